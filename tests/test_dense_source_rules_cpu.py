"""Rules on the dense kernels' sources that no run can show broken."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "litetopk_b200" / "csrc"


def _code(name):
    return re.sub(r"//[^\n]*", "", (CSRC / name).read_text())


def test_a_pair_that_refuses_its_shared_memory_leaves_nothing_unwritten():
    # the merge that follows reads the list of cut sequences; a caller reads results
    code = _code("mla_decode_pair.cuh")
    refusal = code.split("& 1023u) != 0) {")[1].split("return;")[0]
    assert "refuse(p);" in refusal
    body = code.split("void refuse(const Params& p) {")[1].split("\n}")[0]
    assert all(x in body for x in ("p.out)[i] =", "p.lse[i] =", "p.meta[i] = make_int4(-1"))


def test_waits_of_warps_that_read_tensor_memory_end_together():
    # .aligned instructions want the whole warp; a wait that gives up may end for some lanes before others
    for name in ("mla_decode.cu", "mla_decode_pair.cuh"):
        softmax = _code(name).split("if (warp < kSoftmaxWarps) {")[1].split("} else if (warp")[0]
        waits = re.findall(r"(?:mbar_wait|wait_cluster)\([^;]*\);\s*([^;]*);", softmax)
        assert len(waits) >= 3 and all(w.startswith("__syncwarp()") or w.startswith("if (h == 0") for w in waits), (name, waits)
