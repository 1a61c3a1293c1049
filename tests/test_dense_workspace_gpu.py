"""mla_prefill of calls whose workspace is small: cut into what it holds, and as right as any other."""
import pytest
import torch

import litetopk_b200 as lt
from test_dense_gpu import DEV, SCALE, _cu, _gen, _prefill_compare, _ragged

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lq,lk,heads", [([1], [385], 1), ([1], [513], 3), ([2], [1025], 1), ([1, 0, 1], [400, 5, 700], 2), ([1] * 5, [600] * 5, 1), ([3], [300], 2)])
def test_short_calls(causal, lq, lk, heads):
    g = _gen(sum(lk))
    q, kv, rope, cu_q, starts = _ragged(g, lq, lk, heads)
    kd = kv.to(DEV)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = lt.mla_prefill(q.to(DEV), kd[..., :128], rope.to(DEV), kd[..., 128:], SCALE, cu_seqlens_q=_cu(cu_q), cu_seqlens_k=_cu(starts + [sum(lk)]), causal=causal)
    assert torch.cuda.max_memory_allocated() - before < 16 << 20
    _prefill_compare(q, kv, rope, cu_q, starts, lk, got, causal)
