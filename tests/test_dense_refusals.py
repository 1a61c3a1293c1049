"""Calls of the dense operators at the edge of what they take: refused by the C ABI before any CUDA call, or answered."""
import math

import pytest
import torch

import litetopk_b200 as lt
from litetopk_b200 import _lib

P = 0x1000


def test_prefill_refuses_strides_of_nothing(built_lib):
    def call(qt=3200, qh=192, kt=4096, kh=256, kr=64, vt=4096, vh=256, Tq=10, Tk=10, heads=16):
        return built_lib.litedsa_mla_prefill(P, qt, qh, P, kt, kh, P, kr, P, vt, vh, P, P, 2, 0.1, 1, P, P, Tq, Tk, heads, None, 0, None)
    for name in ("qt", "qh", "kt", "kh", "kr", "vt", "vh"):
        assert call(**{name: 0}) == call(**{name: -8}) == _lib.ERR_UNSUPPORTED, name


@pytest.mark.gpu
def test_prefill_names_expanded_operands():
    q = torch.ones((4, 3, 192), dtype=torch.bfloat16, device="cuda:0")
    kv, rope = torch.ones((6, 3, 256), dtype=torch.bfloat16, device="cuda:0"), torch.ones((6, 64), dtype=torch.bfloat16, device="cuda:0")
    shared = kv[:, :1, :128].expand(-1, 3, -1)
    for args, name in (((q, shared, rope, kv[..., 128:]), "k_nope"), ((q, kv[..., :128], rope, shared), "v"), ((q, kv[..., :128], rope[:1].expand(6, -1), kv[..., 128:]), "k_rope"),
                       ((q[:1].expand(4, -1, -1), kv[..., :128], rope, kv[..., 128:]), "q")):
        with pytest.raises(ValueError, match=f"{name} must not be expanded"):
            lt.mla_prefill(*args, 0.1)
        with pytest.raises(ValueError, match=f"{name} must not be expanded"):
            lt.mla_prefill(*args, 0.1, out=torch.empty((4, 3, 128), dtype=torch.bfloat16, device="cuda:0"))
    out, lse = lt.mla_prefill(q, shared.contiguous(), rope, kv[..., 128:], 0.1)
    assert bool((out == 1).all())
    # one key or one head: a stride that is never taken
    one, _ = lt.mla_prefill(q[:, :1], kv[:1, :1, :128].expand(1, 1, -1), rope[:1], kv[:1, :1, 128:], 0.1, causal=False)
    assert bool((one == 1).all())


@pytest.mark.gpu
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("heads", [16, 40, 100])
def test_decode_of_a_cache_without_pages(packed, heads):
    cache = torch.empty((0, 64, 656 if packed else 576), dtype=torch.uint8 if packed else torch.bfloat16, device="cuda:0")
    q = torch.ones((3, heads, 576), dtype=torch.bfloat16, device="cuda:0")
    out, lse = lt.mla_decode(q, cache, torch.zeros((3, 2), dtype=torch.int32, device="cuda:0"), torch.tensor([5, 0, 100], dtype=torch.int32, device="cuda:0"), 0.1)
    assert lt.mla_decode_status(reset=True)[0] == 0
    assert bool((out == 0).all()) and bool((lse == math.inf).all())


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [8, 128])
def test_decode_of_queries_shared_by_sequences(heads):
    # q expanded over the batch, a table with one column, a cache whose blocks are views
    g = torch.Generator().manual_seed(1)
    cache = torch.randn((4, 32, 576), generator=g).bfloat16().cuda()
    q = torch.randn((1, heads, 576), generator=g).bfloat16().cuda()
    table = torch.tensor([[2], [0], [3]], dtype=torch.int32, device="cuda:0")
    lens = torch.tensor([32, 7, 31], dtype=torch.int32, device="cuda:0")
    a = lt.mla_decode(q.expand(3, -1, -1), cache, table, lens, 0.05)
    b = lt.mla_decode(q.repeat(3, 1, 1), cache, table, lens, 0.05)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_decode_refuses_more_keys_than_it_counts(built_lib):
    def call(B, cols, block):
        return built_lib.litedsa_mla_decode(P, 9216, 9216, 576, P, 0, 4, block, block * 1152, P, cols, cols, P, 0.1, P, P, B, 1, 16, None, 0, None)
    assert call(1 << 20, 1 << 20, 256) == call((1 << 31) - 1, 1, 16) == _lib.ERR_UNSUPPORTED
    assert call(1 << 10, 1 << 16, 64) == _lib.ERR_ARG                # no workspace, but no more than that


@pytest.mark.gpu
@pytest.mark.parametrize("heads", [16, 128])
@pytest.mark.parametrize("lens", [[1], [0], [0, 0, 0], [1] * 300, [0] * 149 + [640], [6400, 0, 1, 64, 0, 65], [64 * 148], [64 * 74 + 1, 64]])
def test_decode_deals_out_any_mixture_of_lengths(heads, lens):
    # every key of every sequence once, whoever has it: keys alike, values the key's number's parts
    block, g = 64, torch.Generator().manual_seed(len(lens))
    n = max(lens) // block + 1
    cache = torch.zeros((n, block, 576), dtype=torch.bfloat16)
    at = torch.arange(n * block).view(n, block)
    cache[..., 0], cache[..., 1] = (at % 128).bfloat16(), (at // 128).bfloat16()
    table = torch.arange(n, dtype=torch.int32).repeat(len(lens), 1)
    q = torch.zeros((len(lens), heads, 576), dtype=torch.bfloat16, device="cuda:0")
    out, lse = lt.mla_decode(q, cache.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda:0"), 1.0)
    assert lt.mla_decode_status(reset=True)[0] == 0
    for b in sorted({0, len(lens) // 2, len(lens) - 1, *range(min(len(lens), 6))}):
        keys = torch.arange(lens[b], dtype=torch.float64)
        for d, part in ((0, keys % 128), (1, torch.div(keys, 128, rounding_mode="floor"))):
            want = float(part.mean()) if lens[b] else 0.0
            # equal weights: P = 1, sums of integers below 2^24 in fp32 are exact; the quotient and its rounding to bf16
            assert bool(((out[b, :, d].double().cpu() - want).abs() <= want * (2.0 ** -8 + 2.0 ** -21)).all()), (b, d)
        # log2 of a sum below 2^14 to two units in its last place, 2^-19, times ln 2, and two roundings of a number below 16: 2^-18
        assert bool(((lse[b].double().cpu() - (math.log(lens[b]) if lens[b] else math.inf)).nan_to_num(0.0).abs() <= 2.0 ** -18).all())
