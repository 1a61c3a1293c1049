"""mla_prefill of more tiles than are cut: those of many keys come first, of all heads; every tile once, whatever the lengths."""
import pytest
import torch

import litetopk_b200 as lt
from test_dense_gpu import DEV, SCALE, _bf16, _cu, _gen, _prefill_compare, _ragged

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,lq,lk", [
    (48, [700, 0, 3, 1500, 257, 256], [700, 9, 2000, 1500, 100, 1200]),       # fewer keys than queries, many keys for few queries
    (300, [512], [512]),
    (40, [1] * 40 + [300], [5] * 39 + [1000, 300]),                           # more sequences than a warp has lanes
])
def test_every_tile_is_done_once(causal, heads, lq, lk):
    g = _gen(heads)
    q, kv, rope, cu_q, starts = _ragged(g, lq, lk, heads)
    kd = kv.to(DEV)
    out = torch.full((cu_q[-1] + 5, heads, 128), 7.0, dtype=torch.bfloat16, device=DEV)
    lse = torch.full((cu_q[-1] + 5, heads), 7.0, device=DEV)
    q_wide = torch.cat((q, _bf16(g, 5, heads, 192)))
    ck = [0]
    for n in lk:
        ck.append(ck[-1] + n)
    lt.mla_prefill(q_wide.to(DEV), kd[..., :128], rope.to(DEV), kd[..., 128:], SCALE, cu_seqlens_q=_cu(cu_q), cu_seqlens_k=_cu(ck), causal=causal, out=out, lse=lse)
    assert bool((out[cu_q[-1]:] == 7).all()) and bool((lse[cu_q[-1]:] == 7).all())
    keep = [0, heads // 2, heads - 1]
    _prefill_compare(q, kv, rope, cu_q, starts, lk, (out[:cu_q[-1]], lse[:cu_q[-1]]), causal, heads=keep, rows={0, 127, 128, 255, 256, 511, 600, 1300})
    # all heads of a head's numbers: every (head, tile) has been written, and alike
    same = kd[:, :1].expand(-1, heads, -1).contiguous()
    a, _ = lt.mla_prefill(q[:, :1].expand(-1, heads, -1).contiguous().to(DEV), same[..., :128], rope.to(DEV), same[..., 128:], SCALE,
                          cu_seqlens_q=_cu(cu_q), cu_seqlens_k=_cu(ck), causal=causal)
    assert torch.equal(a, a[:, :1].expand(-1, heads, -1))


@pytest.mark.parametrize("B", [33, 1000, 1100])
@pytest.mark.parametrize("heads", [1, 3])
def test_batches_of_many_sequences(B, heads):
    g = _gen(B)
    lq = torch.randint(0, 4, (B,), generator=g).tolist()
    lq[B // 2], lq[-1] = 300, 5
    lk = [n + int(torch.randint(0, 3, (1,), generator=g)) for n in lq]
    q, kv, rope, cu_q, starts = _ragged(g, lq, lk, heads)
    ck = starts + [sum(lk)]
    kd = kv.to(DEV)
    out, lse = lt.mla_prefill(q.to(DEV), kd[..., :128], rope.to(DEV), kd[..., 128:], SCALE, cu_seqlens_q=_cu(cu_q), cu_seqlens_k=_cu(ck))
    pick = sorted({0, 1, 31, 32, 33 % B, B // 2, B - 2, B - 1})
    out, lse = out.cpu(), lse.cpu()
    for b in pick:
        _prefill_compare(q[cu_q[b]:cu_q[b + 1]], kv, rope, [0, lq[b]], [starts[b]], [lk[b]], (out[cu_q[b]:cu_q[b + 1]], lse[cu_q[b]:cu_q[b + 1]]))
    # every row has been written: sequences of one key hold its value
    for b in range(B):
        if lk[b] == 1 and lq[b] == 1:
            assert torch.equal(out[cu_q[b]], kv[starts[b], :, 128:])
