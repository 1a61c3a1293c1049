"""append_kv, mla_prefill and mla_decode together, as a serving program uses them: prompts enter the cache and are attended to, then tokens come one by one.

Heads pick dims of the latent for their keys and values, so that the expanded and the absorbed form hold the same numbers without a rounding between them:
k_nope = latent[key dims of the head], v = latent[value dims of the head], q_absorbed = q_nope at the key dims, and 0.
"""
import pytest
import torch

import litetopk_b200 as lt
from oracle import dense_oracle as do
from test_dense_gpu import DEV, SCALE, _bf16, _check, _gen, _table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("heads,block,prompts", [(4, 16, [70, 1, 133]), (80, 64, [65, 200])])
def test_prompts_then_tokens(packed, interleaved, heads, block, prompts):
    g = _gen(heads + block)
    B, steps = len(prompts), 3
    cols = (max(prompts) + steps + block - 1) // block
    pages = B * cols
    table = torch.randperm(pages, generator=g).view(B, cols).int()
    cache = torch.zeros((pages, block, 656 if packed else 576), dtype=torch.uint8 if packed else torch.bfloat16, device=DEV)
    turns = _table(max(prompts) + steps)
    key_dims = torch.stack([torch.randperm(512, generator=g)[:128] for _ in range(heads)])
    val_dims = torch.stack([torch.randperm(512, generator=g)[:128] for _ in range(heads)])

    def slots_of(b, pos):
        return table[b].long()[pos // block] * block + pos % block

    def append(latent, rope, q, seq, pos):
        """-> what the tokens' queries are after the turn, absorbed [T, heads, 576]; checks the rows written"""
        q_abs = torch.zeros((len(pos), heads, 576), dtype=torch.bfloat16, device=DEV)
        q_abs[..., :512].scatter_(2, key_dims.to(DEV).expand(len(pos), -1, -1), q[..., :128])
        k_out = torch.empty_like(rope)
        slots = torch.tensor([int(slots_of(b, torch.tensor(p))) for b, p in zip(seq, pos)])
        lt.append_kv(latent, rope, torch.tensor(pos, device=DEV), turns.to(DEV), slots.to(DEV), cache, interleaved=interleaved,
                     q_rope=q[..., 128:], q_out=q_abs[..., 512:], k_out=k_out)
        rows = cache.view(-1, cache.shape[2])[slots.to(DEV)]
        assert torch.equal((rows[:, 528:].contiguous().view(torch.bfloat16) if packed else rows[:, 512:]), k_out)
        return q_abs, k_out

    def cached():
        """the cache's rows as attention takes them"""
        flat = cache.view(-1, cache.shape[2])
        return lt.prepare_kv(flat) if packed else flat

    # the prompts, one call for all of them
    seq = [b for b, n in enumerate(prompts) for _ in range(n)]
    pos = [i for n in prompts for i in range(n)]
    T = len(pos)
    latent, rope, q = _bf16(g, T, 512).to(DEV), _bf16(g, T, 64).to(DEV), _bf16(g, T, heads, 192).to(DEV)
    q_abs, _ = append(latent, rope, q, seq, pos)
    cu = torch.tensor([0] + torch.tensor(prompts).cumsum(0).tolist(), dtype=torch.int32, device=DEV)
    q_turned = torch.cat((q[..., :128], q_abs[..., 512:]), 2)

    def expanded(rows):
        return (rows[:, :512][:, key_dims.to(DEV)].contiguous(), rows[:, 512:].contiguous(), rows[:, :512][:, val_dims.to(DEV)].contiguous())

    held = torch.cat([slots_of(b, torch.arange(n)) for b, n in enumerate(prompts)]).to(DEV)
    k_nope, k_rope, v = expanded(cached()[held])
    out, lse = lt.mla_prefill(q_turned, k_nope, k_rope, v, SCALE, cu_seqlens_q=cu, cu_seqlens_k=cu)
    assert lt.mla_prefill_status(reset=True)[0] == 0
    keep = sorted({0, heads // 2, heads - 1})
    for b, n in enumerate(prompts):
        k0, i = int(cu[b]), n - 1
        o, s, o_tol, s_tol = do.prefill(q_turned[k0 + i:k0 + n, keep].cpu(), k_nope[k0:k0 + n, keep].cpu(), k_rope[k0:k0 + n].cpu(), v[k0:k0 + n, keep].cpu(), SCALE)
        _check(out[k0 + i:k0 + n, keep], o, o_tol)
        _check(lse[k0 + i:k0 + n, keep], s, s_tol)

    # the last prompt token again, then tokens one by one: absorbed over the cache, expanded over the same rows, and in 64 bits
    for step in range(steps + 1):
        lens = [n + step for n in prompts]
        if step == 0:
            last = (cu[1:] - 1).long()
            q1, q1_abs = q_turned[last], q_abs[last]
        else:
            latent, rope, q = _bf16(g, B, 512).to(DEV), _bf16(g, B, 64).to(DEV), _bf16(g, B, heads, 192).to(DEV)
            q1_abs, _ = append(latent, rope, q, range(B), [n - 1 for n in lens])
            q1 = torch.cat((q[..., :128], q1_abs[..., 512:]), 2)
        wide, lse1 = lt.mla_decode(q1_abs, cache, table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), SCALE)
        assert lt.mla_decode_status(reset=True)[0] == 0
        held = torch.cat([slots_of(b, torch.arange(n)) for b, n in enumerate(lens)]).to(DEV)
        k_nope, k_rope, v = expanded(cached()[held])
        ck = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device=DEV)
        cq = torch.arange(B + 1, dtype=torch.int32, device=DEV)
        out2, lse2 = lt.mla_prefill(q1, k_nope, k_rope, v, SCALE, cu_seqlens_q=cq, cu_seqlens_k=ck)
        rows = cached().cpu()
        for b in range(B):
            o, s, o_tol, s_tol = do.decode(q1_abs[b:b + 1, keep].cpu(), rows, table[b], lens[b], block, SCALE)
            _check(wide[b:b + 1, keep], o, o_tol)
            _check(lse1[b:b + 1, keep], s, s_tol)
            at = val_dims[keep][None]
            _check(out2[b:b + 1, keep], o.gather(2, at), o_tol.gather(2, at))
            _check(lse2[b:b + 1, keep], s, s_tol)
