"""mla_decode of more than 64 rows a sequence, which pairs of CTAs share, against the formula in 64 bits (oracle/dense_oracle.py)."""
import pytest
import torch

import litetopk_b200 as lt
from oracle import dense_oracle as do
from test_dense_gpu import DEV, SCALE, _bf16, _cache, _check, _compare, _gen

pytestmark = pytest.mark.gpu


def _lens(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("heads,q_len,block,lens", [
    (65, 1, 16, [0, 1, 15, 16, 17, 31, 32, 33]),     # ends inside, on and behind halves of a CTA's keys
    (66, 2, 32, [47, 48, 49, 63, 64, 65]),           # 132 rows: the second pair has four
    (128, 1, 48, [95, 96, 97, 127, 128, 129, 250]),  # halves on pages that are no power of two
    (127, 3, 128, [1, 2, 3, 200]),                   # tokens that see nothing; pages of two blocks
    (100, 1, 16, [2000, 7, 1]),                      # more blocks than are looked up at a time
    (32, 3, 64, [66, 190]),
])
def test_lengths_pages_and_odd_heads(packed, heads, q_len, block, lens):
    g = _gen(heads + block)
    cache, table, rows = _cache(g, lens, block, packed)
    q = _bf16(g, len(lens), q_len, heads, 576)
    out, lse = lt.mla_decode(q.to(DEV), cache.to(DEV), table.to(DEV), _lens(lens), SCALE)
    keep = sorted({0, 1, heads // 2 - 1, heads // 2, min(63, heads - 1), min(64, heads - 1), heads - 1})
    _compare(q[:, :, keep], lens, block, table, rows, (out[:, :, keep].contiguous(), lse[:, :, keep].contiguous()))


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("block", [16, 64])
@pytest.mark.parametrize("rising", [1.0, -1.0, 0.0])
def test_a_moving_maximum_in_either_cta(packed, block, rising):
    # Scores that climb, fall or lie hundreds apart: by head at another pace, so that the CTAs' rows ask for new maxima at
    # different blocks, or at the same one
    g = _gen(21)
    lens, heads = [1500, 700, 64], 128
    cache, table, values = _cache(g, lens, block, False, poison=False)
    for b, n in enumerate(lens):
        at = torch.arange(n)
        place = table[b].long()[at // block] * block + at % block
        values[place, 512] = (rising * at / 3.0 if rising else torch.where(at % 97 == 3, 300.0, -300.0)).to(torch.bfloat16)
        values[place, 513] = (rising * (n - at) / 3.0 if rising else torch.where(at % 61 == 60, 300.0, -300.0)).to(torch.bfloat16)
    if packed:
        store = torch.empty((values.shape[0], 656), dtype=torch.uint8)
        for i in range(values.shape[0]):
            c, s = do.pack_latent(values[i, :512])
            store[i, :512], store[i, 512:528], store[i, 528:] = c, s.float().view(torch.uint8), values[i, 512:].contiguous().view(torch.uint8)
            values[i] = do.unpack_row(store[i])
        cache = store.view(cache.shape[0], block, 656)
    else:
        cache = values.view(cache.shape)
    q = _bf16(g, 3, 1, heads, 576)
    q[..., 512] = torch.linspace(0, 14, heads).to(torch.bfloat16)
    q[..., 513] = torch.linspace(9, 0, heads).to(torch.bfloat16)
    got = lt.mla_decode(q.to(DEV), cache.to(DEV), table.to(DEV), _lens(lens), SCALE)
    again = lt.mla_decode(q.to(DEV), cache.to(DEV), table.to(DEV), _lens(lens), SCALE)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])
    keep = [0, 1, 30, 62, 63, 64, 65, 90, 127]
    _compare(q[:, :, keep], lens, block, table, values, (got[0][:, :, keep].contiguous(), got[1][:, :, keep].contiguous()))


@pytest.mark.parametrize("packed", [False, True])
def test_pages_that_are_not_there(packed):
    g = _gen(5)
    cache, table, rows = _cache(g, [130, 130], 16, packed)
    q = _bf16(g, 2, 1, 80, 576)
    wrong = table.clone()
    wrong[0, 1], wrong[0, 4], wrong[1, 3], wrong[1, 8] = 1 << 20, -7, cache.shape[0], -(1 << 31)     # zeros
    out, lse = lt.mla_decode(q.to(DEV), cache.to(DEV), wrong.to(DEV), _lens([130, 130]), SCALE)
    blank = torch.cat((rows, torch.zeros((16, 576), dtype=torch.bfloat16)))
    wrong[0, 1] = wrong[0, 4] = wrong[1, 3] = wrong[1, 8] = cache.shape[0]
    keep = [0, 63, 64, 79]
    _compare(q[:, :, keep], [130, 130], 16, wrong, blank, (out[:, :, keep].contiguous(), lse[:, :, keep].contiguous()))


@pytest.mark.parametrize("packed", [False, True])
def test_many_sequences_in_a_replayed_graph(packed):
    # several sequences to a pair, ends and empty ones among them; lengths change between replays
    g = _gen(31)
    B, heads, longest = 400, 72, 200
    cache, table, rows = _cache(g, [longest] * B, 16, packed, poison=False)
    q = _bf16(g, B, 1, heads, 576)
    qd, cd, td, ld = q.to(DEV), cache.to(DEV), table.to(DEV), _lens([longest] * B)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        got = lt.mla_decode(qd, cd, td, ld, SCALE)
    for low, high in ((0, 3), (0, longest + 1)):
        lens = torch.randint(low, high, (B,), generator=g)
        ld.copy_(lens.int())
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.synchronize()
        picks, keep = [0, 1, 2, 133, 134, 250, 398, 399], [0, 63, 64, 71]
        _compare(q[:, :, keep], lens.tolist(), 16, table, rows, (got[0][:, :, keep].contiguous(), got[1][:, :, keep].contiguous()), picks)
        eager = lt.mla_decode(qd, cd, td, ld, SCALE)
        assert torch.equal(eager[0], got[0]) and torch.equal(eager[1], got[1])


def test_queries_with_strides_and_rows_left_alone():
    g = _gen(41)
    lens, heads = [90, 33], 70
    cache, table, rows = _cache(g, lens, 32, False)
    wide = torch.full((2, 2, heads + 3, 600), float("nan"), dtype=torch.bfloat16)
    q = _bf16(g, 2, 2, heads, 576)
    wide[:, :, :heads, :576] = q
    out = torch.full((4, 2, heads, 512), 5.0, dtype=torch.bfloat16, device=DEV)
    lse = torch.full((4, 2, heads), 5.0, device=DEV)
    got = lt.mla_decode(wide.to(DEV)[:, :, :heads, :576], cache.to(DEV), table.to(DEV), _lens(lens), SCALE, out=out[1:3], lse=lse[1:3])
    keep = [0, 63, 64, 69]
    _compare(q[:, :, keep], lens, 32, table, rows, (got[0][:, :, keep].contiguous(), got[1][:, :, keep].contiguous()))
    assert bool((out[::3] == 5).all()) and bool((lse[::3] == 5).all())


def test_many_short_sequences_of_packed_rows():
    # pieces of a block or two: whoever looks ahead reads a length for each, while the others are done with several
    g = _gen(51)
    B, heads, longest = 3000, 128, 129
    cache, table, rows = _cache(g, [longest] * 8, 16, True, poison=False)
    table = table.repeat(B // 8, 1)
    lens = torch.where(torch.arange(B) % 50 == 0, longest, torch.randint(0, 3, (B,), generator=g))
    q = _bf16(g, B, 1, heads, 576)
    for _ in range(3):
        out, lse = lt.mla_decode(q.to(DEV), cache.to(DEV), table.to(DEV), _lens(lens.tolist()), SCALE)
        assert lt.mla_decode_status(reset=True)[0] == 0
    keep, picks = [0, 64, 127], [0, 1, 2, 49, 50, 1500, 2998, 2999]
    _compare(q[:, :, keep], lens.tolist(), 16, table, rows, (out[:, :, keep].contiguous(), lse[:, :, keep].contiguous()), picks)
