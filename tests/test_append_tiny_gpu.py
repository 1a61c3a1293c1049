"""append_kv of numbers below 2^-126, which fp32 holds without a leading one: they are turned and packed like any others."""
import pytest
import torch

import litetopk_b200 as lt
from oracle import dense_oracle as do
from test_dense_gpu import DEV, _check, _gen, _table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("interleaved", [False, True])
def test_tiny_latents_and_rope_dims(interleaved):
    g = _gen(1)
    T, n_pos = 6, 40
    # multiples of 2^-133, the smallest bf16; groups of nothing else, and beside larger numbers
    kv = (torch.randint(-127, 128, (T, 512), generator=g).double() * 2.0 ** -133).to(torch.bfloat16)
    kv[1, :128:3] = 2.0 ** -120
    kv[2, 130] = 1.0
    rope = (torch.randint(-127, 128, (T, 64), generator=g).double() * 2.0 ** -133).to(torch.bfloat16)
    q = (torch.randint(-127, 128, (T, 5, 64), generator=g).double() * 2.0 ** -133).to(torch.bfloat16)
    pos, table, slots = torch.tensor([0, 3, 0, 39, 7, 20]), _table(n_pos), torch.arange(T)
    cache = torch.zeros((16, 656), dtype=torch.uint8, device=DEV)
    qd, k_out = q.to(DEV), torch.zeros((T, 64), dtype=torch.bfloat16, device=DEV)
    lt.append_kv(kv.to(DEV), rope.to(DEV), pos.to(DEV), table.to(DEV), slots.to(DEV), cache, interleaved=interleaved, q_rope=qd, q_out=qd, k_out=k_out)
    rows = cache.cpu()[:T]
    for t in range(T):
        codes, scale = do.pack_latent(kv[t])
        got = rows[t, :512].view(torch.float8_e4m3fn).float()
        assert torch.equal(got, codes.view(torch.float8_e4m3fn).float()), t
        assert torch.equal(rows[t, 512:528].clone().view(torch.float32).double(), scale)
    assert bool((rows[0, :512] & 0x7f).any())
    # position 0 turns nothing
    assert torch.equal(k_out[0].cpu(), rope[0]) and torch.equal(k_out[2].cpu(), rope[2]) and torch.equal(qd[0].cpu(), q[0])
    # products and sums of fp32 are rounded to 2^-149 at best, three of them, the result to half of 2^-133
    cos, sin = table[pos].split(32, 1)
    _check(k_out, do.rotate(rope, cos, sin, interleaved), torch.full((T, 64), 3 * 2.0 ** -149 + 2.0 ** -134, dtype=torch.float64))
    _check(qd, do.rotate(q, cos[:, None], sin[:, None], interleaved), torch.full((T, 5, 64), 3 * 2.0 ** -149 + 2.0 ** -134, dtype=torch.float64))
