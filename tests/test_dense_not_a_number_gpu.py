"""mla_decode and mla_prefill of scores that are no number: a row that sees one is NaN, in out and in lse, wherever its sequence is cut; others are as ever."""
import math

import pytest
import torch

import litetopk_b200 as lt
from oracle import dense_oracle as do
from test_dense_gpu import DEV, SCALE, _bf16, _cache, _check, _cu, _gen, _ragged

pytestmark = pytest.mark.gpu


def _none(out, lse):
    assert bool(out.isnan().all()) and bool(lse.isnan().all()), (out.isnan().float().mean(), lse)


def _at(table, block, b, i):
    return int(table[b, i // block]) * block + i % block


def _decode(q, cache, table, lens):
    out, lse = lt.mla_decode(q.to(DEV), cache.to(DEV), table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), SCALE)
    assert lt.mla_decode_status(reset=True)[0] == 0
    return out.cpu(), lse.cpu()


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("heads,q_len,block,lens,place", [
    (16, 1, 64, [3000], 1234),                     # cut into more than eight parts
    (64, 1, 16, [3000], 0),
    (128, 1, 16, [3000], 2999),
    (16, 1, 16, [640] * 40, 333),                  # cut into a few
    (64, 2, 64, [640] * 40, 7),
    (33, 1, 64, [70] * 300, 69),                   # most of them whole
    (66, 2, 32, [70] * 300, 12),
])
def test_decode_of_a_key_that_is_none(packed, heads, q_len, block, lens, place):
    # (among the rope dims: no value is NaN, only the scores)
    g = _gen(heads + len(lens))
    cache, table, rows = _cache(g, lens, block, packed)
    q = _bf16(g, len(lens), q_len, heads, 576)
    b = len(lens) // 2
    row = _at(table, block, b, place)
    rope = cache.view(-1, cache.shape[2])[:, 528:].view(torch.bfloat16) if packed else cache.view(-1, 576)[:, 512:]
    rope[row, 9] = math.nan
    out, lse = _decode(q, cache, table, lens)
    _none(out[b], lse[b])
    keep = sorted({0, heads - 1})
    for x in sorted({0, b - 1, b + 1, len(lens) - 1} - {b}):
        if 0 <= x < len(lens):
            o, s, o_tol, s_tol = do.decode(q[x][:, keep], rows, table[x], lens[x], block, SCALE)
            _check(out[x][:, keep], o, o_tol)
            _check(lse[x][:, keep], s, s_tol)


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("heads,q_len,n", [(4, 3, 130), (40, 3, 65), (128, 1, 2000), (128, 3, 129)])
def test_decode_of_infinite_keys_and_queries_that_are_none(packed, heads, q_len, n):
    # The newest key is infinite in a rope dim: scores +inf, -inf, or unseen.  One head's query is NaN.
    g = _gen(n)
    cache, table, rows = _cache(g, [n], 16, packed)
    q = _bf16(g, 1, q_len, heads, 576)
    q[..., 520] = torch.where(torch.arange(heads) % 2 == 0, 1.0, -1.0).to(torch.bfloat16)
    q[0, :, heads - 2, 3] = math.nan
    rope = cache.view(-1, cache.shape[2])[:, 528:].view(torch.bfloat16) if packed else cache.view(-1, 576)[:, 512:]
    rope[_at(table, 16, 0, n - 1), 8] = math.inf
    out, lse = _decode(q, cache, table, [n])
    _none(out[0, :, heads - 2], lse[0, :, heads - 2])
    _none(out[0, -1, 0:heads - 2:2], lse[0, -1, 0:heads - 2:2])
    for j, h in [(q_len - 1, 1), (q_len - 1, heads - 1)] + ([(0, 0), (q_len - 2, 1)] if q_len > 1 else []):
        see = min(n - q_len + 1 + j, n - 1)            # of the last key the odd heads' weight is nothing
        o, s, o_tol, s_tol = do.decode(q[0, j:j + 1, h:h + 1], rows, table[0], see, 16, SCALE)
        _check(out[0, j:j + 1, h:h + 1], o, o_tol)
        _check(lse[0, j:j + 1, h:h + 1], s, s_tol)


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("heads", [16, 128])
def test_decode_of_values_that_are_none(packed, heads):
    # in the latent: scores and a value at once; and no key at all beside it
    g = _gen(heads)
    cache, table, rows = _cache(g, [200, 0, 90], 16, packed)
    q = _bf16(g, 3, 1, heads, 576)
    if packed:
        cache.view(-1, 656)[_at(table, 16, 0, 100), 300] = 0x7f
    else:
        cache.view(-1, 576)[_at(table, 16, 0, 100), 300] = math.nan
    out, lse = _decode(q, cache, table, [200, 0, 90])
    _none(out[0], lse[0])
    assert bool((out[1] == 0).all()) and bool((lse[1] == math.inf).all())
    o, s, o_tol, s_tol = do.decode(q[2, :, :1], rows, table[2], 90, 16, SCALE)
    _check(out[2, :, :1], o, o_tol)
    _check(lse[2, :, :1], s, s_tol)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("n,m,heads,place", [(300, 300, 2, 130), (77, 77, 3, 0), (6, 4718, 2, 4000), (300, 9001, 2, 100), (200, 60, 2, 30), (1500, 1500, 110, 1400)])
def test_prefill_of_keys_and_queries_that_are_none(causal, n, m, heads, place):
    g = _gen(n + m)
    q, kv, rope, cu_q, starts = _ragged(g, [n], [m], heads)
    kd, qd = kv.to(DEV), q.to(DEV)
    kd[place, 0, 5] = math.nan                         # a key of the first head
    qd[n - 1, heads - 1, 150] = math.nan               # a query of the last
    out, lse = lt.mla_prefill(qd, kd[..., :128], rope.to(DEV), kd[..., 128:], SCALE, causal=causal)
    assert lt.mla_prefill_status(reset=True)[0] == 0
    out, lse = out.cpu(), lse.cpu()
    sees = [max(0, m - n + 1 + i) if causal else m for i in range(n)]
    those = torch.tensor(sees) > place
    _none(out[those, 0], lse[those, 0])
    _none(out[n - 1, heads - 1], lse[n - 1, heads - 1])
    for i in sorted({0, min(127, n - 1), n // 2, n - 1}):
        for h in {0, 1, heads - 1}:
            if (h == 0 and those[i]) or (h == heads - 1 and i == n - 1):
                continue
            o, s, o_tol, s_tol = do.prefill(q[i:i + 1, h:h + 1], kv[:sees[i], h:h + 1, :128], rope[:sees[i]], kv[:sees[i], h:h + 1, 128:], SCALE, causal=False)
            _check(out[i:i + 1, h:h + 1], o, o_tol)
            _check(lse[i:i + 1, h:h + 1], s, s_tol)


@pytest.mark.parametrize("n,m", [(130, 130), (3, 5000)])
def test_prefill_of_infinite_keys(n, m):
    # the last key: +inf for even heads, -inf (no weight) for odd ones
    g = _gen(m)
    heads = 4
    q, kv, rope, cu_q, starts = _ragged(g, [n], [m], heads)
    q[..., 140] = torch.where(torch.arange(heads) % 2 == 0, 1.0, -1.0).to(torch.bfloat16)
    rd, kd = rope.to(DEV), kv.to(DEV)
    rd[m - 1, 12] = math.inf
    out, lse = lt.mla_prefill(q.to(DEV), kd[..., :128], rd, kd[..., 128:], SCALE)
    assert lt.mla_prefill_status(reset=True)[0] == 0
    out, lse = out.cpu(), lse.cpu()
    _none(out[n - 1, ::2], lse[n - 1, ::2])
    for i, h in ((n - 1, 1), (n - 1, 3), (n - 2, 0), (0, 2)):
        see = min(m - n + 1 + i, m - 1)
        o, s, o_tol, s_tol = do.prefill(q[i:i + 1, h:h + 1], kv[:see, h:h + 1, :128], rope[:see], kv[:see, h:h + 1, 128:], SCALE, causal=False)
        _check(out[i:i + 1, h:h + 1], o, o_tol)
        _check(lse[i:i + 1, h:h + 1], s, s_tol)
