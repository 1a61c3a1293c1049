"""append_kv and mla_decode on the GPU against the formulas in 64 bits (oracle/dense_oracle.py, which derives the bounds)."""
import math

import pytest
import torch

import litetopk_b200 as lt
from oracle import dense_oracle as do

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SCALE = 192 ** -0.5


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _bf16(g, *shape, scale=1.0):
    return (torch.randn(shape, generator=g) * scale).to(torch.bfloat16)


def _table(n):
    a = torch.arange(n, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32)
    return torch.cat((a.cos(), a.sin()), 1).float()


def _check(got, ref, bound):
    got = got.cpu().double()
    assert got.shape == ref.shape
    same = (got == ref) | (got.sub(ref).abs() <= bound)
    assert bool(same.all()), (got - ref).abs().sub(bound).max()


# --------------------------------------------------------------------------- append_kv
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,heads,index", [(1, 128, torch.int64), (3, 1, torch.int32), (37, 20, torch.int64), (130, 0, torch.int32)])
def test_append_writes_turned_and_packed_rows(packed, interleaved, T, heads, index):
    g = _gen(T + heads)
    n_pos, blocks, block = 500, 12, 16
    kv = _bf16(g, T, 576)
    kv[0, :128] = 0                                                  # a group of zeros
    if T > 1:
        kv[1, 128:256] *= 1e-30                                      # below what a normal scale brings into range
        kv[2, 200] = 448.0                                           # amax on the border of a scale
        kv[2, 300] = 450.0
    rope, q = _bf16(g, T, 64), _bf16(g, T, max(heads, 1), 192)
    pos = torch.randint(0, n_pos, (T,), generator=g).to(index)
    slots = torch.randperm(blocks * block, generator=g)[:T].to(index)
    table = _table(n_pos)
    width, dt = (656, torch.uint8) if packed else (576, torch.bfloat16)
    store = torch.randint(0, 255, (blocks, block + 1, width), generator=g).to(dt)          # blocks with a gap behind them
    cache = store.to(DEV)
    kd = kv.to(DEV)[:, :512]
    q_abs = _bf16(g, T, max(heads, 1), 576)
    qd, k_out = q_abs.to(DEV), torch.zeros((T, 64), dtype=torch.bfloat16, device=DEV)
    more = dict(q_rope=q.to(DEV)[..., 128:], q_out=qd[..., 512:]) if heads else {}
    lt.append_kv(kd, rope.to(DEV), pos.to(DEV), table.to(DEV), slots.to(DEV), cache[:, :block], interleaved=interleaved, k_out=k_out, **more)
    cos, sin = table[pos.long()].split(32, 1)
    k_ref, k_tol = do.rotate(rope, cos, sin, interleaved), do.rotate_bound(rope, cos, sin, interleaved)
    _check(k_out, k_ref, k_tol + (k_ref.abs() + k_tol) * do.HALF_BF16)
    if heads:
        q_ref, q_tol = do.rotate(q[..., 128:], cos[:, None], sin[:, None], interleaved), do.rotate_bound(q[..., 128:], cos[:, None], sin[:, None], interleaved)
        _check(qd[..., 512:], q_ref, q_tol + (q_ref.abs() + q_tol) * do.HALF_BF16)
    assert torch.equal(qd[..., :512].cpu(), q_abs[..., :512])
    k_bits = k_out.cpu()
    want = store.clone()
    for t in range(T):
        b, i = divmod(int(slots[t]), block)
        if packed:
            codes, scale = do.pack_latent(kv[t, :512])
            want[b, i, :512] = codes
            want[b, i, 512:528] = scale.float().view(torch.uint8)
            want[b, i, 528:] = k_bits[t].view(torch.uint8)
        else:
            want[b, i] = torch.cat((kv[t, :512], k_bits[t]))
    got = cache.cpu()
    if packed:                                                       # -0 and +0 of values that round to nothing are the same value
        a, b = got[..., :512].contiguous().view(torch.float8_e4m3fn).float(), want[..., :512].contiguous().view(torch.float8_e4m3fn).float()
        assert torch.equal(a.nan_to_num(999.0), b.nan_to_num(999.0)) and torch.equal(got[..., 512:], want[..., 512:])
    else:
        assert torch.equal(got.view(torch.int16), want.view(torch.int16))


@pytest.mark.parametrize("packed", [False, True])
def test_append_leaves_out_padding_and_unknown_positions(packed):
    g = _gen(5)
    T, rows, n_pos = 9, 32, 50
    width, dt = (656, torch.uint8) if packed else (576, torch.bfloat16)
    cache = torch.zeros((rows, width), dtype=dt, device=DEV)
    slots = torch.tensor([3, -1, 31, 32, 1 << 40, 7, -(1 << 40), 8, 9], device=DEV)
    pos = torch.tensor([0, 1, 2, 3, 4, 50, 6, -1, 49], device=DEV)
    q = _bf16(g, T, 3, 64).to(DEV)
    before, k_out = q.clone(), torch.full((T, 64), 7.0, dtype=torch.bfloat16, device=DEV)
    lt.append_kv(_bf16(g, T, 512).to(DEV), _bf16(g, T, 64).to(DEV), pos, _table(n_pos).to(DEV), slots, cache, q_rope=q, q_out=q, k_out=k_out)
    written = (cache.view(torch.uint8).view(rows, -1) != 0).any(1).cpu().nonzero()[:, 0].tolist()
    assert written == [3, 9, 31]
    known = torch.tensor([True] * 5 + [False, True, False, True])
    assert torch.equal(q.cpu()[~known], before.cpu()[~known]) and bool((k_out.cpu()[~known] == 7).all())
    assert bool((q.cpu()[1:5] != before.cpu()[1:5]).any(-1).all()) and torch.equal(q.cpu()[0], before.cpu()[0])      # position 0 turns nothing
    assert bool((k_out.cpu()[known] != 7).any(1).all())


def test_append_of_numbers_that_are_none():
    kv = torch.ones((1, 512), dtype=torch.bfloat16)
    kv[0, 5], kv[0, 130], kv[0, 140] = math.nan, math.inf, -math.inf
    cache = torch.zeros((16, 656), dtype=torch.uint8, device=DEV)
    zero = torch.zeros((1,), dtype=torch.int64, device=DEV)
    lt.append_kv(kv.to(DEV), torch.zeros((1, 64), dtype=torch.bfloat16, device=DEV), zero, _table(1).to(DEV), zero, cache)
    row = cache[0].cpu()
    codes, scale = row[:512].view(torch.float8_e4m3fn).float(), row[512:528].clone().view(torch.float32)
    assert math.isnan(codes[5]) and bool(torch.isfinite(scale).all())
    assert codes[130] == 448 and codes[140] == -448
    assert torch.equal(codes[256:] * scale[2], torch.ones(256)) or torch.equal(codes[256:384] * scale[2], torch.ones(128))


# --------------------------------------------------------------------------- mla_decode
def _cache(g, lens, block, packed, pow2=True, extra=2, poison=True, scale=1.0):
    """A paged cache of these lengths, its table and its values; rows that belong to nobody hold NaN and infinities."""
    n = [(x + block - 1) // block for x in lens]
    pages = sum(n) + extra
    order = torch.randperm(pages, generator=g)
    cols = max(max(n), 1)
    table = torch.zeros((len(lens), cols), dtype=torch.int32)
    used = torch.zeros((pages, block), dtype=torch.bool)
    at = 0
    for b, c in enumerate(n):
        table[b, :c] = order[at:at + c]
        for i in range(c):
            used[order[at + i], :min(block, lens[b] - i * block)] = True
        at += c
    rows = _bf16(g, pages * block, 576, scale=scale)
    if packed:
        store = torch.empty((pages * block, 656), dtype=torch.uint8)
        groups = rows[:, :512].float().view(-1, 4, 128)
        s = groups.abs().amax(-1) / 448
        s = torch.exp2(torch.ceil(torch.log2(s))) if pow2 else s
        store[:, :512] = (groups / s[..., None]).view(-1, 512).to(torch.float8_e4m3fn).view(torch.uint8)
        store[:, 512:528] = s.contiguous().view(torch.uint8)
        store[:, 528:] = rows[:, 512:].contiguous().view(torch.uint8)
        codes = store[:, :512].contiguous().view(torch.float8_e4m3fn).float().view(-1, 4, 128)
        rows = torch.cat(((codes * s[..., None]).view(-1, 512).to(torch.bfloat16), rows[:, 512:]), 1)
        if poison:
            store[~used.view(-1)] = 0xff
    else:
        store = rows.clone()
        if poison:
            bad = torch.tensor([math.nan, math.inf, -math.inf])[torch.arange(pages * block * 576) % 3].view(-1, 576).to(torch.bfloat16)
            store[~used.view(-1)] = bad[~used.view(-1)]
    return store.view(pages, block, -1), table, rows


def _compare(q, lens, block, table, rows, got, picks=None, scale=SCALE):
    out, lse = got
    sq = q.shape[1]
    out, lse = out.view(len(lens), sq, q.shape[2], 512), lse.view(len(lens), sq, q.shape[2])
    assert lt.mla_decode_status(reset=True)[0] == 0
    for b in range(len(lens)) if picks is None else picks:
        o, s, o_tol, s_tol = do.decode(q[b], rows, table[b], lens[b], block, scale)
        _check(out[b], o, o_tol)
        _check(lse[b], s, s_tol)


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("heads,q_len,block,lens", [
    (16, 1, 64, [1, 0, 63, 64, 65, 130]),           # ends inside, on and behind a block
    (64, 1, 16, [200, 17, 1000]),                   # four pages to a block
    (1, 1, 32, [5, 700]),
    (128, 1, 64, [129, 1, 64]),                     # two CTAs to a sequence
    (20, 3, 48, [2, 1, 0, 47, 300]),                # tokens that see nothing; pages no power of two
    (8, 2, 128, [500, 2]),                          # 16 rows
    (16, 2, 16, [40, 333]),                         # 32 rows
    (128, 4, 64, [3, 260]),                         # eight CTAs to a sequence
    (33, 1, 64, [65]),
    (16, 9, 64, [12, 150]),                         # three CTAs, the last with 16 rows
])
def test_decode_matches_the_formula(packed, heads, q_len, block, lens):
    g = _gen(heads * q_len + block)
    cache, table, rows = _cache(g, lens, block, packed)
    q = _bf16(g, len(lens), q_len, heads, 576)
    got = lt.mla_decode(q.to(DEV) if q_len > 1 else q[:, 0].to(DEV), cache.to(DEV), table.to(DEV),
                        torch.tensor(lens, dtype=torch.int32, device=DEV), SCALE)
    assert got[0].shape[:-1] == got[1].shape == ((len(lens), q_len, heads) if q_len > 1 else (len(lens), heads))
    _compare(q, lens, block, table, rows, got)


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("heads,B,longest", [(16, 1, 20011), (64, 3, 9000), (16, 400, 300), (128, 90, 400)])
def test_decode_cuts_long_sequences_and_deals_out_many(packed, heads, B, longest):
    g = _gen(B)
    lens = [longest] + torch.randint(0, longest, (B - 1,), generator=g).tolist()
    cache, table, rows = _cache(g, lens, 64, packed)
    q = _bf16(g, B, 1, heads, 576)
    got = lt.mla_decode(q.to(DEV), cache.to(DEV), table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), SCALE)
    # rows are independent: a few sequences, and of those a few heads
    picks = sorted({0, B // 3, B // 2, B - 1})
    keep = sorted({0, 5 % heads, heads - 1})
    out, lse = got
    _compare(q[:, :, keep], lens, 64, table, rows, (out[:, :, keep].contiguous(), lse[:, :, keep].contiguous()), picks)


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("rising", [1.0, -1.0, 0.0])
def test_decode_follows_a_moving_maximum(packed, rising):
    # scores that climb (or fall) by more than the maximum's slack from block to block, or lie hundreds apart
    g = _gen(11)
    n, heads = 1500, 16
    cache, table, rows = _cache(g, [n], 64, False)
    values = rows.clone()
    at = torch.arange(n)
    place = table[0].long()[at // 64] * 64 + at % 64
    ramp = rising * torch.arange(n) / 3.0 if rising else torch.where(torch.arange(n) % 97 == 3, 300.0, -300.0)
    values[place, 512] = ramp.to(torch.bfloat16)
    if packed:
        store = torch.empty((values.shape[0], 656), dtype=torch.uint8)
        for i in range(values.shape[0]):
            c, s = do.pack_latent(values[i, :512])
            store[i, :512], store[i, 512:528], store[i, 528:] = c, s.float().view(torch.uint8), values[i, 512:].contiguous().view(torch.uint8)
            values[i] = do.unpack_row(store[i])
        cache = store.view(cache.shape[0], 64, 656)
    else:
        cache = values.view(cache.shape)
    q = _bf16(g, 1, 1, heads, 576)
    q[..., 512] = torch.linspace(1, 14, heads).to(torch.bfloat16)
    got = lt.mla_decode(q.to(DEV), cache.to(DEV), table.to(DEV), torch.tensor([n], dtype=torch.int32, device=DEV), SCALE)
    _compare(q, [n], 64, table, values, got)


@pytest.mark.parametrize("packed", [False, True])
def test_decode_takes_views_and_given_outputs(packed):
    g = _gen(3)
    lens, heads = [100, 31], 12
    cache, table, rows = _cache(g, lens, 32, packed)
    width = cache.shape[-1]
    wide = torch.full((cache.shape[0], 40, width), 255, dtype=torch.uint8).to(cache.dtype) if packed else torch.full((cache.shape[0], 40, width), math.nan, dtype=cache.dtype)
    wide[:, :32] = cache
    q_wide = torch.full((2, 3, 16, 584), math.nan, dtype=torch.bfloat16)
    q = _bf16(g, 2, 3, heads, 576)
    q_wide[:, :, :heads, :576] = q
    t_wide = torch.full((2, table.shape[1] + 3), 1 << 30, dtype=torch.int32)
    t_wide[:, :table.shape[1]] = table
    out = torch.full((4, 3, heads, 512), 5.0, dtype=torch.bfloat16, device=DEV)
    lse = torch.full((4, 3, heads), 5.0, device=DEV)
    got = lt.mla_decode(q_wide.to(DEV)[:, :, :heads, :576], wide.to(DEV)[:, :32], t_wide.to(DEV)[:, :table.shape[1]],
                        torch.tensor(lens, dtype=torch.int32, device=DEV), SCALE, out=out[1:3], lse=lse[1:3])
    assert got[0].data_ptr() == out[1].data_ptr() and got[1].data_ptr() == lse[1].data_ptr()
    _compare(q, lens, 32, table, rows, got)
    assert bool((out[::3] == 5).all()) and bool((lse[::3] == 5).all())


def test_decode_of_lengths_and_pages_that_are_not_there():
    g = _gen(4)
    cache, table, rows = _cache(g, [64, 64, 64], 16, False)
    q = _bf16(g, 3, 1, 4, 576)
    lens = torch.tensor([-5, 1 << 30, 64], dtype=torch.int32, device=DEV)      # clamped to nothing and to the table's row
    table2 = table.clone()
    table2[2, 1] = 1 << 20                                                     # no such page: zeros
    table2[2, 2] = -7
    got = lt.mla_decode(q.to(DEV), cache.to(DEV), table2.to(DEV), lens, SCALE)
    blank = torch.cat((rows, torch.zeros((16, 576), dtype=torch.bfloat16)))
    table2[2, 1] = table2[2, 2] = blank.shape[0] // 16 - 1
    _compare(q, [0, 64, 64], 16, table2, blank, got)
    pc, pt, prow = _cache(g, [64, 64, 64], 16, True)
    pt2 = pt.clone()
    pt2[2, 1], pt2[2, 2] = 1 << 20, -7
    got = lt.mla_decode(q.to(DEV), pc.to(DEV), pt2.to(DEV), lens, SCALE)
    blank = torch.cat((prow, torch.zeros((16, 576), dtype=torch.bfloat16)))
    pt2[2, 1] = pt2[2, 2] = blank.shape[0] // 16 - 1
    _compare(q, [0, 64, 64], 16, pt2, blank, got)


def test_decode_of_scales_that_are_no_powers_of_two():
    g = _gen(6)
    cache, table, rows = _cache(g, [300], 64, True, pow2=False)
    q = _bf16(g, 1, 1, 64, 576)
    got = lt.mla_decode(q.to(DEV), cache.to(DEV), table.to(DEV), torch.tensor([300], dtype=torch.int32, device=DEV), SCALE)
    _compare(q, [300], 64, table, rows, got)


@pytest.mark.parametrize("packed", [False, True])
def test_decode_is_reproducible_and_follows_new_lengths_in_a_graph(packed):
    g = _gen(8)
    lens = [700, 64, 2000, 1]
    cache, table, rows = _cache(g, [2100] * 4, 64, packed, poison=False)
    q = _bf16(g, 4, 1, 64, 576)
    qd, cd, td = q.to(DEV), cache.to(DEV), table.to(DEV)
    ld = torch.tensor(lens, dtype=torch.int32, device=DEV)
    first = lt.mla_decode(qd, cd, td, ld, SCALE)
    again = lt.mla_decode(qd, cd, td, ld, SCALE)
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    side = torch.cuda.Stream()
    graph, graph2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            got = lt.mla_decode(qd, cd, td, ld, SCALE)
        with torch.cuda.graph(graph2, stream=side):
            got2 = lt.mla_decode(qd, cd, td, ld, SCALE)
    torch.cuda.synchronize()
    for lens in ([700, 64, 2000, 1], [5, 2100, 0, 129]):
        ld.copy_(torch.tensor(lens, dtype=torch.int32))
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):                                # beside the other: each has a workspace of its own
            graph2.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], got2[0]) and torch.equal(got[1], got2[1])
        keep = [0, 40, 63]
        _compare(q[:, :, keep], lens, 64, table, rows, (got[0][:, :, keep].contiguous(), got[1][:, :, keep].contiguous()))


def test_decode_of_no_sequences():
    cache = torch.zeros((2, 16, 576), dtype=torch.bfloat16, device=DEV)
    out, lse = lt.mla_decode(torch.zeros((0, 4, 576), dtype=torch.bfloat16, device=DEV), cache, torch.zeros((0, 1), dtype=torch.int32, device=DEV),
                             torch.zeros((0,), dtype=torch.int32, device=DEV), SCALE)
    assert out.shape == (0, 4, 512) and lse.shape == (0, 4)
    out, lse = lt.mla_decode(torch.ones((1, 4, 576), dtype=torch.bfloat16, device=DEV), cache[:0], torch.zeros((1, 1), dtype=torch.int32, device=DEV),
                             torch.ones((1,), dtype=torch.int32, device=DEV), SCALE)
    assert bool((out == 0).all()) and bool((lse == math.inf).all())  # a cache without blocks holds no key


def test_append_to_nothing():
    z = torch.zeros((1,), dtype=torch.int64, device=DEV)
    kv, kr = torch.ones((1, 512), dtype=torch.bfloat16, device=DEV), torch.ones((1, 64), dtype=torch.bfloat16, device=DEV)
    k_out = torch.zeros_like(kr)
    lt.append_kv(kv, kr, z, _table(1).to(DEV), z, torch.zeros((0, 16, 656), dtype=torch.uint8, device=DEV), k_out=k_out)
    assert torch.equal(k_out, kr)                                     # a cache without rows: the token is padding
    lt.append_kv(kv, kr, z, torch.zeros((0, 64), device=DEV), z, torch.zeros((4, 656), dtype=torch.uint8, device=DEV), k_out=k_out.zero_())
    assert bool((k_out == 0).all())                                   # no positions: it is left out


# --------------------------------------------------------------------------- mla_prefill
def _ragged(g, lq, lk, heads, gap=0, scale=1.0):
    """Operands of sequences of these lengths, ``gap`` rows of NaN and infinities behind each sequence's keys."""
    cu_q = [0]
    for n in lq:
        cu_q.append(cu_q[-1] + n)
    Tk = sum(lk) + gap * len(lk)
    kv = _bf16(g, Tk, heads, 256, scale=scale)
    rope = _bf16(g, Tk, 64)
    q = _bf16(g, cu_q[-1], heads, 192)
    starts, at = [], 0
    for n in lk:
        starts.append(at)
        kv[at + n:at + n + gap] = torch.tensor([math.nan, math.inf, -math.inf])[torch.arange(gap * heads * 256) % 3].view(gap, heads, 256).to(torch.bfloat16)
        rope[at + n:at + n + gap] = math.nan
        at += n + gap
    return q, kv, rope, cu_q, starts


def _prefill_compare(q, kv, rope, cu_q, starts, lk, got, causal=True, heads=None, rows=None, scale=SCALE):
    out, lse = got
    assert lt.mla_prefill_status(reset=True)[0] == 0
    heads = list(range(q.shape[1])) if heads is None else heads
    out, lse = out.cpu()[:, heads], lse.cpu()[:, heads]
    for b in range(len(lk)):
        n, m, k0 = cu_q[b + 1] - cu_q[b], lk[b], starts[b]
        k, v, r = kv[k0:k0 + m][:, heads, :128], kv[k0:k0 + m][:, heads, 128:], rope[k0:k0 + m]
        pick = range(n) if rows is None else sorted({x for x in rows if x < n} | ({n - 1} if n else set()))
        for i in pick:
            see = max(0, m - n + 1 + i) if causal else m
            o, s, o_tol, s_tol = do.prefill(q[cu_q[b] + i:cu_q[b] + i + 1][:, heads], k[:see], r[:see], v[:see], scale, causal=False)
            _check(out[cu_q[b] + i:cu_q[b] + i + 1], o, o_tol)
            _check(lse[cu_q[b] + i:cu_q[b] + i + 1], s, s_tol)


def _cu(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("n,m,heads", [(1, 1, 1), (1, 300, 3), (77, 77, 2), (128, 128, 1), (129, 129, 2), (130, 257, 1), (257, 257, 1), (300, 700, 2),
                                       (5, 3, 2), (200, 60, 1), (3, 0, 2)])
def test_prefill_of_one_sequence(causal, n, m, heads):
    g = _gen(n + m)
    q, kv, rope, cu_q, starts = _ragged(g, [n], [m], heads)
    kd = kv.to(DEV)
    got = lt.mla_prefill(q.to(DEV), kd[..., :128], rope.to(DEV), kd[..., 128:], SCALE, causal=causal)
    _prefill_compare(q, kv, rope, cu_q, starts, [m], got, causal)


@pytest.mark.parametrize("causal", [True, False])
def test_prefill_of_a_ragged_batch_beside_numbers_that_are_none(causal):
    g = _gen(17)
    lq, lk, heads = [3, 0, 130, 1, 260, 40, 7], [3, 5, 130, 400, 300, 11, 0], 3
    q, kv, rope, cu_q, starts = _ragged(g, lq, lk, heads, gap=2)
    kd = kv.to(DEV)
    # a sequence's keys end where the gap begins: its cu_seqlens_k entry and the next one's differ, so the gaps are sequences without queries
    cq, ck = [0], [0]
    for b in range(len(lq)):
        cq += [cu_q[b + 1], cu_q[b + 1]]
        ck += [starts[b] + lk[b], starts[b] + lk[b] + 2]
    got = lt.mla_prefill(q.to(DEV), kd[..., :128], rope.to(DEV), kd[..., 128:], SCALE, cu_seqlens_q=_cu(cq), cu_seqlens_k=_cu(ck), causal=causal)
    _prefill_compare(q, kv, rope, cu_q, starts, lk, got, causal)


@pytest.mark.parametrize("n,m,heads", [(6, 4718, 1), (300, 9001, 2), (1500, 4096, 5)])
def test_prefill_cuts_few_tiles_along_the_keys(n, m, heads):
    g = _gen(n)
    q, kv, rope, cu_q, starts = _ragged(g, [n], [m], heads)
    kd = kv.to(DEV)
    got = lt.mla_prefill(q.to(DEV), kd[..., :128], rope.to(DEV), kd[..., 128:], SCALE)
    _prefill_compare(q, kv, rope, cu_q, starts, [m], got, heads=sorted({0, heads - 1}), rows={0, 127, 128, 255, 256, 700, 1279})


def test_prefill_deals_out_many_tiles():
    g = _gen(23)
    lq = [900, 1, 513] + [17] * 60
    lk = [1000, 130, 513] + [40] * 60
    heads = 40                                                       # 63 sequences: 67 tiles a head
    q, kv, rope, cu_q, starts = _ragged(g, lq, lk, heads)
    kd = kv.to(DEV)
    cu_k = [0]
    for m in lk:
        cu_k.append(cu_k[-1] + m)
    args = (q.to(DEV), kd[..., :128], rope.to(DEV), kd[..., 128:], SCALE)
    got = lt.mla_prefill(*args, cu_seqlens_q=_cu(cu_q), cu_seqlens_k=_cu(cu_k))
    _prefill_compare(q, kv, rope, cu_q, starts, lk, got, heads=[0, 21, 39], rows={0, 130, 256, 600})
    again = lt.mla_prefill(*args, cu_seqlens_q=_cu(cu_q), cu_seqlens_k=_cu(cu_k))
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


@pytest.mark.parametrize("rising", [1.0, -1.0, 0.0])
def test_prefill_follows_a_moving_maximum(rising):
    g = _gen(29)
    n, m, heads = 200, 1300, 2
    q, kv, rope, cu_q, starts = _ragged(g, [n], [m], heads)
    ramp = rising * torch.arange(m) / 3.0 if rising else torch.where(torch.arange(m) % 97 == 3, 300.0, -300.0)
    rope[:, 0] = ramp.to(torch.bfloat16)
    q[:, :, 128] = torch.linspace(-5, 14, n).to(torch.bfloat16)[:, None]
    kd = kv.to(DEV)
    got = lt.mla_prefill(q.to(DEV), kd[..., :128], rope.to(DEV), kd[..., 128:], SCALE)
    _prefill_compare(q, kv, rope, cu_q, starts, [m], got, rows=set(range(0, 200, 9)))
    got = lt.mla_prefill(q.to(DEV), kd[..., :128], rope.to(DEV), kd[..., 128:], 0.0)
    _prefill_compare(q, kv, rope, cu_q, starts, [m], got, rows={0, 150}, scale=0.0)


def test_prefill_takes_views_given_outputs_and_leaves_other_rows():
    g = _gen(31)
    lq, lk, heads = [20, 33], [50, 33], 5
    q, kv, rope, cu_q, starts = _ragged(g, lq, lk, heads)
    Tq, Tk = 53 + 9, 83 + 4
    q_wide = torch.full((Tq, 8, 200), math.nan, dtype=torch.bfloat16)
    q_wide[:53, :heads, :192] = q
    kn = torch.full((Tk, 8, 136), math.nan, dtype=torch.bfloat16)
    vv, rr = kn.clone(), torch.full((Tk, 72), math.nan, dtype=torch.bfloat16)
    kn[:83, :heads, :128], vv[:83, :heads, :128], rr[:83, :64] = kv[..., :128], kv[..., 128:], rope
    out = torch.full((Tq, heads, 128), 5.0, dtype=torch.bfloat16, device=DEV)
    lse = torch.full((Tq, heads), 5.0, device=DEV)
    got = lt.mla_prefill(q_wide.to(DEV)[:, :heads, :192], kn.to(DEV)[:, :heads, :128], rr.to(DEV)[:, :64], vv.to(DEV)[:, :heads, :128], SCALE,
                         cu_seqlens_q=_cu([0, 20, 53]), cu_seqlens_k=_cu([0, 50, 83]), out=out, lse=lse)
    assert got[0].data_ptr() == out.data_ptr()
    _prefill_compare(q, kv, rope, cu_q, starts, lk, (out[:53], lse[:53]))
    assert bool((out[53:] == 5).all()) and bool((lse[53:] == 5).all())


def test_prefill_in_graphs_follows_new_lengths():
    g = _gen(37)
    heads, T = 2, 700
    q, kv, rope, _, _ = _ragged(g, [T], [T], heads)
    qd, kd, rd = q.to(DEV), kv.to(DEV), rope.to(DEV)
    cq, ck = _cu([0, 300, T]), _cu([0, 300, T])
    lt.mla_prefill(qd, kd[..., :128], rd, kd[..., 128:], SCALE, cu_seqlens_q=cq, cu_seqlens_k=ck)
    side, graphs, got = torch.cuda.Stream(), [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    with torch.cuda.stream(side):
        for x in graphs:
            with torch.cuda.graph(x, stream=side):
                got.append(lt.mla_prefill(qd, kd[..., :128], rd, kd[..., 128:], SCALE, cu_seqlens_q=cq, cu_seqlens_k=ck))
    torch.cuda.synchronize()
    for cuts in (([0, 300, 700], [0, 300, 700]), ([0, 0, 513], [0, 100, 700]), ([0, 1, 2], [0, 650, 700])):
        cq.copy_(_cu(cuts[0]))
        ck.copy_(_cu(cuts[1]))
        torch.cuda.synchronize()
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        torch.cuda.synchronize()
        end = cuts[0][-1]
        assert torch.equal(got[0][0][:end], got[1][0][:end]) and torch.equal(got[0][1][:end], got[1][1][:end])
        lk = [cuts[1][1], cuts[1][2] - cuts[1][1]]
        _prefill_compare(q, kv, rope, cuts[0], cuts[1], lk, got[0], rows={0, 129, 255, 256, 299, 400})


def test_prefill_of_nothing():
    e = torch.zeros((0, 2, 192), dtype=torch.bfloat16, device=DEV)
    kv, r = torch.zeros((4, 2, 256), dtype=torch.bfloat16, device=DEV), torch.zeros((4, 64), dtype=torch.bfloat16, device=DEV)
    out, lse = lt.mla_prefill(e, kv[..., :128], r, kv[..., 128:], SCALE)
    assert out.shape == (0, 2, 128) and lse.shape == (0, 2)
    q = torch.ones((3, 2, 192), dtype=torch.bfloat16, device=DEV)
    out = torch.full((3, 2, 128), 5.0, dtype=torch.bfloat16, device=DEV)
    lt.mla_prefill(q, kv[..., :128], r, kv[..., 128:], SCALE, cu_seqlens_q=_cu([0]), cu_seqlens_k=_cu([0]), out=out)
    lt.mla_prefill(q, kv[..., :128], r, kv[..., 128:], SCALE, cu_seqlens_q=_cu([0, 0, 0]), cu_seqlens_k=_cu([0, 2, 4]), out=out)
    assert bool((out == 5).all())
