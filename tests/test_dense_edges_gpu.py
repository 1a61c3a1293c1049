"""Calls of the dense operators that their documentation allows at its edges: layouts, many tokens, tables without columns, rows far into a cache, several streams."""
import math

import pytest
import torch

import litetopk_b200 as lt
from oracle import dense_oracle as do
from test_dense_gpu import DEV, SCALE, _bf16, _cache, _check, _compare, _gen, _prefill_compare, _ragged

pytestmark = pytest.mark.gpu


def _lens(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("block", [16, 64])
@pytest.mark.parametrize("heads", [16, 64, 128])
def test_a_table_without_columns(packed, block, heads):
    cache = torch.full((4, block, 656 if packed else 576), 255 if packed else math.nan, device=DEV).to(torch.uint8 if packed else torch.bfloat16)
    out, lse = lt.mla_decode(torch.ones((3, heads, 576), dtype=torch.bfloat16, device=DEV), cache, torch.zeros((3, 0), dtype=torch.int32, device=DEV), _lens([5, 0, 9]), SCALE)
    assert lt.mla_decode_status(reset=True)[0] == 0
    assert bool((out == 0).all()) and bool((lse == math.inf).all())


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("heads,q_len", [(12, 1), (12, 3), (40, 2)])
def test_queries_heads_first(packed, heads, q_len):
    g = _gen(heads)
    lens = [70, 0, 200]
    cache, table, rows = _cache(g, lens, 16, packed)
    q = _bf16(g, 3, q_len, heads, 576)
    for order in ((2, 0, 1), (0, 2, 1), (1, 2, 0)):
        back = [order.index(i) for i in range(3)]
        qd = q.to(DEV).permute(*order, 3).contiguous().permute(*back, 3)
        got = lt.mla_decode(qd, cache.to(DEV), table.to(DEV), _lens(lens), SCALE)
        _compare(q, lens, 16, table, rows, got)


@pytest.mark.parametrize("n,m,heads", [(140, 300, 3), (5, 2000, 4)])
def test_prompts_heads_first(n, m, heads):
    g = _gen(n)
    q, kv, rope, cu_q, starts = _ragged(g, [n], [m], heads)
    first = [x.to(DEV).transpose(0, 1).contiguous().transpose(0, 1) for x in (q, kv[..., :128], kv[..., 128:])]
    got = lt.mla_prefill(first[0], first[1], rope.to(DEV), first[2], SCALE)
    _prefill_compare(q, kv, rope, cu_q, starts, [m], got, rows={0, 64, 127, 128})


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("heads,q_len,n", [(128, 60, 130), (1, 700, 800), (20, 300, 250)])
def test_many_tokens_a_sequence(packed, heads, q_len, n):
    g = _gen(q_len)
    lens = [n, 7]
    cache, table, rows = _cache(g, lens, 32, packed)
    q = _bf16(g, 2, q_len, heads, 576)
    out, lse = lt.mla_decode(q.to(DEV), cache.to(DEV), table.to(DEV), _lens(lens), SCALE)
    assert lt.mla_decode_status(reset=True)[0] == 0
    for b, length in enumerate(lens):
        for j in sorted({0, q_len // 2, q_len - 8, q_len - 1}):
            for h in {0, heads - 1}:
                see = max(0, length - q_len + 1 + j)
                o, s, o_tol, s_tol = do.decode(q[b, j:j + 1, h:h + 1], rows, table[b], see, 32, SCALE)
                _check(out[b, j:j + 1, h:h + 1], o, o_tol)
                _check(lse[b, j:j + 1, h:h + 1], s, s_tol)


@pytest.mark.parametrize("packed", [False, True])
def test_rows_behind_the_first_four_gigabytes(packed):
    g = _gen(9)
    pages, T, block = (9_000_000 if packed else 5_000_000) // 64, 300, 64
    cache = torch.zeros((pages, block, 656 if packed else 576), dtype=torch.uint8 if packed else torch.bfloat16, device=DEV)
    own = torch.tensor([pages - 1, pages - 2, 1, pages - 3, 0])
    at = torch.arange(T)
    slots = own[at // block] * block + at % block
    turns = torch.cat((torch.ones((T, 32)), torch.zeros((T, 32))), 1)
    lt.append_kv(_bf16(g, T, 512).to(DEV), _bf16(g, T, 64).to(DEV), at.to(DEV), turns.to(DEV), slots.to(DEV), cache)
    held = cache.view(-1, cache.shape[2])[slots.to(DEV)].cpu()
    rows = torch.stack([do.unpack_row(r) for r in held]) if packed else held
    assert bool((rows.float().abs().sum(1) > 0).all()) and int((cache.view(torch.uint8) != 0).flatten(1).any(1).sum()) == 5
    near = torch.arange(5, dtype=torch.int32)                   # (the rows in a cache of five pages, for the formula)
    rows = torch.cat((rows, torch.zeros((20, 576), dtype=torch.bfloat16)))
    for heads in (16, 128):
        q = _bf16(g, 1, 1, heads, 576)
        out, lse = lt.mla_decode(q.to(DEV), cache, own[None].int().to(DEV), _lens([T]), SCALE)
        keep = [0, heads - 1]
        _compare(q[:, :, keep], [T], block, near[None], rows, (out[:, :, keep].contiguous(), lse[:, :, keep].contiguous()))


def test_calls_on_three_streams_at_once():
    g = torch.Generator(device=DEV).manual_seed(5)

    def randn(*shape):
        return torch.randn(shape, generator=g, device=DEV).bfloat16()
    cache, table = randn(300, 64, 576), torch.randint(0, 300, (40, 30), generator=g, device=DEV).int()
    lens = torch.randint(0, 1920, (40,), generator=g, device=DEV).int()
    q, q2, pq, kv, rope = randn(40, 128, 576), randn(40, 16, 576), randn(1500, 16, 192), randn(1500, 16, 256), randn(1500, 64)
    calls = (lambda: lt.mla_decode(q, cache, table, lens, SCALE), lambda: lt.mla_decode(q2, cache, table, lens, SCALE),
             lambda: lt.mla_prefill(pq, kv[..., :128], rope, kv[..., 128:], SCALE))
    alone = [f() for f in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    for _ in range(30):
        got = []
        for f, s in zip(calls, streams):
            with torch.cuda.stream(s):
                got.append(f())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for x, y in zip(alone, got) for a, b in zip(x, y))
    assert lt.mla_decode_status(reset=True)[0] == lt.mla_prefill_status(reset=True)[0] == 0
