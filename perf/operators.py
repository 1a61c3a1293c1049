"""The dense side of latent attention as a serving program uses it: writing the paged cache, attending to the whole of it for the
tokens being decoded, and the expanded prefill of prompts.

Operators (``"op"`` of a case):

append      ``append_kv``: the latents of new tokens, with the rotation of their position applied to the 64 rope dims, into rows
            of a paged cache (bf16 rows of 576, or packed rows of 656 bytes: 512 e4m3 codes, 4 fp32 scales, 64 bf16); the
            queries' rope dims are rotated in the same call.
decode      ``mla_decode``: one to a few tokens a sequence against all of its cached rows (absorbed form: keys are the 576 dims
            of a row, values its first 512), with causal masks among the new tokens.
prefill     ``mla_prefill``: the expanded form, 128 + 64 dims of keys and 128 of values a head, over a batch of sequences of their
            own lengths, whose keys may begin before the queries (a cached prefix).

``own`` false: plain torch operations in 32 bits.  Lengths are made from the case alone, values and the order of pages from the seed.
"""
import math

import torch

own = False

DEV = "cuda"
SCALE = 192 ** -0.5                # softmax scale of heads with 128 + 64 dims
MAX_POS = 163840                   # positions of the rotation table


def listed():
    return [
        # one token of one request: nothing but latency
        dict(name="append_1tok", op="append", cache="packed", tokens=1, heads=128, block=64, rows=8192, interleaved=True),
        # a decode step of a batch, a third of it padding, tensor-parallel heads
        dict(name="append_batch", op="append", cache="bf16", tokens=129, heads=16, block=64, rows=65536, interleaved=False),
        # a prefill chunk
        dict(name="append_8k", op="append", cache="packed", tokens=8192, heads=64, block=64, rows=65536, interleaved=True),
        # one request with a short context
        dict(name="decode_1seq_2k", op="decode", cache="bf16", batch=1, q_len=1, heads=64, min_len=2048, max_len=2048, block=64),
        # a batch of odd lengths on packed rows, down to a single token
        dict(name="decode_32seq_packed", op="decode", cache="packed", batch=32, q_len=1, heads=64, min_len=1, max_len=8191, block=64),
        # tensor-parallel heads on long contexts
        dict(name="decode_long_h16", op="decode", cache="bf16", batch=5, q_len=1, heads=16, min_len=65535, max_len=131072, block=64),
        # two tokens a sequence (one of them drafted), all heads on one GPU, small pages
        dict(name="decode_2tok_h128", op="decode", cache="bf16", batch=48, q_len=2, heads=128, min_len=1000, max_len=6001, block=16),
        # a large batch of all heads on packed rows
        dict(name="decode_128seq_packed", op="decode", cache="packed", batch=128, q_len=1, heads=128, min_len=2048, max_len=4096, block=64),
        # a short prompt
        dict(name="prefill_77tok", op="prefill", batch=1, heads=16, min_q=77, max_q=77, min_prefix=0, max_prefix=0),
        # prompts of odd lengths, some behind a cached prefix
        dict(name="prefill_ragged", op="prefill", batch=11, heads=32, min_q=3, max_q=2050, min_prefix=0, max_prefix=1537),
        # a whole prompt, half of a model's heads
        dict(name="prefill_8k", op="prefill", batch=1, heads=64, min_q=8192, max_q=8192, min_prefix=0, max_prefix=0),
        # a chunk at the end of a long prompt
        dict(name="prefill_chunk_32k", op="prefill", batch=1, heads=16, min_q=4096, max_q=4096, min_prefix=28672, max_prefix=28672),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "prefill"])
    if op == "append":
        tokens = _log(rng, 1, 8192)
        return dict(op=op, cache=rng.choice(["bf16", "packed"]), tokens=tokens, heads=rng.choice([8, 16, 24, 32, 64] + [128] * (tokens <= 4096)),
                    block=rng.choice([16, 64, 128]), rows=rng.choice([16384, 65536]), interleaved=rng.choice([True, False]))
    if op == "decode":
        heads, q_len = rng.choice([8, 16, 20, 32, 64, 128]), rng.choice([1, 1, 1, 2, 3, 4])
        longest = _log(rng, q_len, 131072)
        # keys of all sequences, and products of them with the query rows, up to those of the largest listed cases
        most = max(1, min(256, 500000 // longest, 80000000 // (longest * heads * q_len)))
        return dict(op=op, cache=rng.choice(["bf16", "packed"]), batch=_log(rng, 1, most), q_len=q_len, heads=heads,
                    min_len=max(q_len, int(longest * rng.random())), max_len=longest, block=rng.choice([16, 32, 64, 128]))
    heads, longest = rng.choice([1, 8, 16, 20, 32, 64]), _log(rng, 1, 8192)
    prefix = rng.choice([0, 0, _log(rng, 1, 16384)])
    while heads > 1 and heads * longest * (longest / 2 + prefix) > 2.1e9:
        heads //= 2
    most = max(1, min(32, 16384 // longest, int(2.1e9 / (heads * longest * (longest / 2 + prefix)))))
    return dict(op=op, batch=_log(rng, 1, most), heads=heads, min_q=max(1, int(longest * rng.random())), max_q=longest,
                min_prefix=int(prefix * rng.random()), max_prefix=prefix)


# ---------------------------------------------------------------- inputs
def _spread(n, lo, hi, at=0.0):
    """``n`` lengths from ``lo`` to ``hi``, the first of them ``hi``, the second ``lo``, the others spread between."""
    return [hi if i == 0 else lo if i == 1 else lo + int((hi - lo + 1) * ((i * 0.6180339887498949 + at) % 1.0)) for i in range(n)]


def _lengths(case):
    if case["op"] == "decode":
        return _spread(case["batch"], case["min_len"], case["max_len"])
    q = _spread(case["batch"], case["min_q"], case["max_q"])
    return q, [a + b for a, b in zip(q, _spread(case["batch"], case["min_prefix"], case["max_prefix"], 0.37))]


def _padding(case):
    """Tokens at the end of a batch that stand for no request."""
    return case["tokens"] // 3 if case["tokens"] % 2 and case["tokens"] < 1024 else 0


def _table(dtype):
    """[position, cos of 32 angles | sin of 32]; angles of far positions need 64 bits."""
    inv = 10000.0 ** (-torch.arange(32, dtype=torch.float64, device=DEV) / 32)
    a = torch.arange(MAX_POS, dtype=torch.float64, device=DEV)[:, None] * inv
    return torch.cat((a.cos(), a.sin()), 1).to(dtype)


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).to(torch.bfloat16)


def _rows(g, case, rows):
    """A paged cache in use: rows of N(0, 1) latents and rope dims whose dims have scales of their own."""
    kv = _randn(g, rows, 576)
    block = case["block"]
    if case["cache"] == "bf16":
        return kv.view(rows // block, block, 576)
    codes, scale = _quantise(kv[:, :512].float())
    out = torch.empty((rows, 656), dtype=torch.uint8, device=DEV)
    out[:, :512] = codes.view(torch.uint8)
    out[:, 512:528] = scale.view(torch.uint8)
    out[:, 528:] = kv[:, 512:].contiguous().view(torch.uint8)
    return out.view(rows // block, block, 656)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 7919 + 17)
    h = case["heads"]
    s = dict(case=case)
    if case["op"] == "append":
        t = case["tokens"]
        s["cache"] = _rows(g, case, case["rows"])
        s["kv_c"] = _randn(g, t, 576)[:, :512]                     # what the model's down projection leaves: latent | rope
        s["k_rope"] = _randn(g, t, 64)
        s["q"] = _randn(g, t, h, 192)                              # nope | rope dims of every head
        s["q_abs"] = _randn(g, t, h, 576)                          # absorbed queries: the rope dims are to be filled in
        s["k_out"] = torch.empty((t, 64), dtype=torch.bfloat16, device=DEV)
        first = int(torch.randint(0, MAX_POS - t, (1,), generator=g, device=DEV))
        s["positions"] = torch.randint(0, MAX_POS, (t,), generator=g, device=DEV) if t < 1024 else \
            torch.arange(first, first + t, device=DEV)
        slots = torch.randperm(case["rows"], generator=g, device=DEV)[:t]
        if t >= 1024:                                              # a chunk fills page after page
            pages = torch.randperm(case["rows"] // case["block"], generator=g, device=DEV)
            at = torch.arange(t, device=DEV) + 5 % case["block"]
            at = at.clamp(max=case["rows"] - 1)
            slots = pages[at // case["block"]] * case["block"] + at % case["block"]
        if _padding(case):
            slots[-_padding(case):] = -1
        s["slots"] = slots
        s["table"] = _table(torch.float32)
    elif case["op"] == "decode":
        lens, block = _lengths(case), case["block"]
        n = [(x + block - 1) // block for x in lens]
        cols, pages = max(n), sum(n) + 3
        s["cache"] = _rows(g, case, pages * block)
        order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
        table = torch.zeros((case["batch"], cols), dtype=torch.int32, device=DEV)
        at = torch.arange(cols, device=DEV)
        counts = torch.tensor(n, device=DEV)
        starts = counts.cumsum(0) - counts
        inside = at[None, :] < counts[:, None]
        table = torch.where(inside, order[(starts[:, None] + at[None, :]).clamp(max=pages - 1)], table)
        s.update(block_table=table, seq_lens=torch.tensor(lens, dtype=torch.int32, device=DEV), longest=max(lens),
                 q=_randn(g, case["batch"], case["q_len"], h, 576))
    else:
        lq, lk = _lengths(case)
        tq, tk = sum(lq), sum(lk)
        kv = _randn(g, tk, h, 256)                                 # the up projection of the latents: keys | values of every head
        s.update(q=_randn(g, tq, h, 192), k_nope=kv[..., :128], v=kv[..., 128:], k_rope=_randn(g, tk, 64),
                 cu_q=torch.tensor([0] + lq, device=DEV).cumsum(0).to(torch.int32),
                 cu_k=torch.tensor([0] + lk, device=DEV).cumsum(0).to(torch.int32), longest_q=max(lq), longest_k=max(lk))
    return s


# ---------------------------------------------------------------- plain forms
def _quantise(x):
    """e4m3 codes and scales of groups of 128 dims; the scale is the smallest power of two that brings the group into range."""
    x = x.unflatten(-1, (-1, 128))
    m, e = torch.frexp(x.abs().amax(-1))                           # amax = m 2^e, 0.5 <= m < 1; 448 = 0.875 2^9
    e = (e - 9 + (m > 0.875)).clamp(min=-126)
    scale = torch.ldexp(torch.ones_like(m), e)
    return (x / scale[..., None]).flatten(-2).to(torch.float8_e4m3fn), scale


def _rotate(x, cos, sin, interleaved):
    """x [..., 64] with cos and sin [..., 32]"""
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :32], x[..., 32:])
    u, v = a * cos - b * sin, b * cos + a * sin
    return torch.stack((u, v), -1).flatten(-2) if interleaved else torch.cat((u, v), -1)


def _cache_values(cache):
    """What a cache holds, by field."""
    rows = cache.flatten(0, 1)
    if rows.dtype == torch.bfloat16:
        return dict(rows=rows)
    return dict(codes=rows[:, :512].view(torch.float8_e4m3fn), scales=rows[:, 512:528].view(torch.float32), rope=rows[:, 528:].view(torch.bfloat16))


def _append_plain(s):
    inter = s["case"]["interleaved"]
    cs = s["table"][s["positions"]]
    cos, sin = cs[:, :32], cs[:, 32:]
    k = _rotate(s["k_rope"].float(), cos, sin, inter).to(torch.bfloat16)
    q = _rotate(s["q"][..., 128:].float(), cos[:, None], sin[:, None], inter).to(torch.bfloat16)
    s["k_out"].copy_(k)
    s["q_abs"][..., 512:] = q
    rows = s["cache"].view(-1, s["cache"].shape[-1])
    keep = s["slots"] >= 0
    at = s["slots"][keep]
    if rows.dtype == torch.bfloat16:
        rows[at] = torch.cat((s["kv_c"], k), 1)[keep]
    else:
        codes, scale = _quantise(s["kv_c"].float())
        row = torch.cat((codes.view(torch.uint8), scale.view(torch.uint8), k.view(torch.uint8)), 1)
        rows[at] = row[keep]


def _float_rows(rows):
    """Cache rows as 576 values in 32 bits."""
    if rows.dtype == torch.bfloat16:
        return rows.float()
    codes = rows[..., :512].contiguous().view(torch.float8_e4m3fn).float().unflatten(-1, (4, 128))
    scale = rows[..., 512:528].contiguous().view(torch.float32)
    rope = rows[..., 528:].contiguous().view(torch.bfloat16).float()
    return torch.cat(((codes * scale[..., None]).flatten(-2), rope), -1)


def _softmax_rows(s, seen):
    """Softmax of the visible scores and their log-sum-exp; rows that see nothing: 0 and +inf."""
    s = torch.where(seen, s, -math.inf)
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    e = torch.exp(s - m)
    total = e.sum(-1, keepdim=True)
    lse = torch.where(total > 0, m + torch.log(total), math.inf)
    return e / torch.where(total > 0, total, 1.0), lse[..., 0]


def _decode_plain(s):
    case, q = s["case"], s["q"].float()
    b, sq, h, _ = q.shape
    block = case["block"]
    at = torch.arange(s["longest"], device=DEV)
    pages = s["block_table"].long()[:, at // block]                # [b, keys]
    k = _float_rows(s["cache"].flatten(0, 1)[pages * block + at % block])
    lens = s["seq_lens"].long()
    see = lens[:, None] - sq + 1 + torch.arange(sq, device=DEV)    # keys that a token sees
    seen = at < see[:, :, None, None]                              # [b, sq, 1, keys]
    scores = torch.matmul(q.flatten(1, 2), k.transpose(1, 2)).unflatten(1, (sq, h)) * SCALE
    p, lse = _softmax_rows(scores, seen)
    del scores
    out = torch.matmul(p.flatten(1, 2), k[..., :512]).unflatten(1, (sq, h))
    return dict(out=out.to(torch.bfloat16), lse=lse)


def _prefill_plain(s):
    q, cu_q, cu_k = s["q"], s["cu_q"].long(), s["cu_k"].long()
    iq, ik = torch.arange(s["longest_q"], device=DEV), torch.arange(s["longest_k"], device=DEV)
    nq, nk = cu_q.diff(), cu_k.diff()
    rq = (cu_q[:-1, None] + iq).clamp(max=q.shape[0] - 1)          # rows of the padded batch
    rk = (cu_k[:-1, None] + ik).clamp(max=s["k_rope"].shape[0] - 1)
    qp = q[rq].transpose(1, 2).float()                             # [b, h, queries, 192]
    scores = torch.matmul(qp[..., :128], s["k_nope"][rk].permute(0, 2, 3, 1).float())
    scores += torch.matmul(qp[..., 128:], s["k_rope"][rk].transpose(1, 2).float()[:, None])
    scores *= SCALE
    seen = (ik < (nk - nq)[:, None, None] + iq[None, :, None] + 1) & (ik < nk[:, None, None])
    p, lse = _softmax_rows(scores, seen[:, None])
    del scores
    out = torch.matmul(p, s["v"][rk].transpose(1, 2).float()).transpose(1, 2)
    of = torch.repeat_interleave(torch.arange(nq.shape[0], device=DEV), nq, output_size=q.shape[0])
    at = torch.arange(q.shape[0], device=DEV) - cu_q[of]
    return dict(out=out[of, at].to(torch.bfloat16), lse=lse.transpose(1, 2)[of, at])


def run(state):
    op = state["case"]["op"]
    if op == "append":
        if own:
            import litetopk_b200 as lt
            lt.append_kv(state["kv_c"], state["k_rope"], state["positions"], state["table"], state["slots"], state["cache"],
                         interleaved=state["case"]["interleaved"], q_rope=state["q"][..., 128:], q_out=state["q_abs"][..., 512:],
                         k_out=state["k_out"])
        else:
            _append_plain(state)
        return dict(_cache_values(state["cache"]), q=state["q_abs"], k=state["k_out"])
    if op == "decode":
        if own:
            import litetopk_b200 as lt
            out, lse = lt.mla_decode(state["q"], state["cache"], state["block_table"], state["seq_lens"], SCALE)
            return dict(out=out, lse=lse)
        return _decode_plain(state)
    if own:
        import litetopk_b200 as lt
        out, lse = lt.mla_prefill(state["q"], state["k_nope"], state["k_rope"], state["v"], SCALE, cu_seqlens_q=state["cu_q"],
                                  cu_seqlens_k=state["cu_k"], causal=True)
        return dict(out=out, lse=lse)
    return _prefill_plain(state)


# ---------------------------------------------------------------- what a pass cannot do without
def _row_bytes(case):
    return 1152 if case["cache"] == "bf16" else 656


def work(case):
    h = case["heads"]
    if case["op"] == "append":
        t, kept = case["tokens"], case["tokens"] - _padding(case)
        read = kept * 1024 + t * (128 + 16 + 256 + h * 128)
        return dict(bytes=read + kept * _row_bytes(case) + t * (128 + h * 128), flops=t * (h + 1) * 192)
    if case["op"] == "decode":
        lens, sq = _lengths(case), case["q_len"]
        pairs = sum(max(0, n - sq + 1 + j) for n in lens for j in range(sq))
        rows = len(lens) * sq * h
        pages = sum((n + case["block"] - 1) // case["block"] for n in lens)
        return dict(bytes=sum(lens) * _row_bytes(case) + rows * (1152 + 1024 + 4) + 4 * (pages + len(lens)), flops=2 * 1088 * h * pairs)
    lq, lk = _lengths(case)
    pairs = sum(n * (k - n) + n * (n + 1) // 2 for n, k in zip(lq, lk))
    return dict(bytes=sum(lq) * h * (384 + 256 + 4) + sum(lk) * (h * 512 + 128), flops=2 * 320 * h * pairs)


# ---------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    h = case["heads"]
    if case["op"] == "append":
        angles = _table(torch.float64)[s["positions"]]
        rot = torch.complex(angles[:, :32], angles[:, 32:])

        def turned(x, r):                                          # a pair of dims is a complex number, the rotation a product
            x = x.double()
            z = torch.view_as_complex(x.reshape(*x.shape[:-1], 32, 2)) if case["interleaved"] else torch.complex(x[..., :32], x[..., 32:])
            z = z * r
            return torch.view_as_real(z).flatten(-2) if case["interleaved"] else torch.cat((z.real, z.imag), -1)

        k, q = turned(s["k_rope"], rot), turned(s["q"][..., 128:], rot[:, None])
        rows = s["cache"].flatten(0, 1)
        live = torch.nonzero(s["slots"] >= 0)[:, 0]
        at = s["slots"][live]
        res = dict(q=torch.cat((s["q_abs"][..., :512].double(), q), -1), k=k)
        if case["cache"] == "bf16":
            new = rows.double()
            new[at] = torch.cat((s["kv_c"].double(), k), 1)[live]
            return dict(res, rows=new)
        groups = s["kv_c"].double().view(-1, 4, 128)
        scale = 2.0 ** torch.ceil(torch.log2(groups.abs().amax(-1) / 448.0))
        new = {n: v.double() for n, v in _cache_values(s["cache"]).items()}
        new["codes"][at] = (groups / scale[..., None]).flatten(1)[live]
        new["scales"][at] = scale[live]
        new["rope"][at] = k[live]
        return dict(res, **new)
    if case["op"] == "decode":
        sq, block = case["q_len"], case["block"]
        rows = s["cache"].flatten(0, 1)
        out = torch.empty((case["batch"], sq, h, 512), dtype=torch.float64, device=DEV)
        lse = torch.empty((case["batch"], sq, h), dtype=torch.float64, device=DEV)
        for b, n in enumerate(_lengths(case)):
            place = torch.arange(n, device=DEV)
            r = rows[s["block_table"][b, place // block].long() * block + place % block]
            if case["cache"] == "bf16":
                kv = r.double()
            else:
                c = r[:, :512].contiguous().view(torch.float8_e4m3fn).double()
                kv = torch.cat((c * r[:, 512:528].contiguous().view(torch.float32).double().repeat_interleave(128, 1),
                                r[:, 528:].contiguous().view(torch.bfloat16).double()), 1)
            for j in range(sq):
                mine = kv[:max(0, n - sq + 1 + j)]
                x = s["q"][b, j].double() @ mine.T * SCALE
                lse[b, j] = torch.logsumexp(x, -1) if len(mine) else math.inf
                out[b, j] = torch.softmax(x, -1) @ mine[:, :512] if len(mine) else 0.0
        return dict(out=out, lse=lse)
    lq, lk = _lengths(case)
    out = torch.empty((sum(lq), h, 128), dtype=torch.float64, device=DEV)
    lse = torch.empty((sum(lq), h), dtype=torch.float64, device=DEV)
    q0 = k0 = 0
    for n, k in zip(lq, lk):
        hidden = torch.ones((n, k), dtype=torch.bool, device=DEV).triu(k - n + 1)
        for i in range(h):
            keys = torch.cat((s["k_nope"][k0:k0 + k, i], s["k_rope"][k0:k0 + k]), 1).double()
            x = (s["q"][q0:q0 + n, i].double() @ keys.T * SCALE).masked_fill_(hidden, -math.inf)
            lse[q0:q0 + n, i] = torch.logsumexp(x, -1)
            out[q0:q0 + n, i] = torch.softmax(x, -1) @ s["v"][k0:k0 + k, i].double()
        q0, k0 = q0 + n, k0 + k
    return dict(out=out, lse=lse)
