"""The sequence of calls that the integration guide shows for the dense operators, run as it stands there."""
import re
from pathlib import Path

import pytest
import torch

from oracle import dense_oracle as do
from test_dense_gpu import DEV, SCALE, _bf16, _check, _gen, _table

pytestmark = pytest.mark.gpu
GUIDE = Path(__file__).resolve().parents[1] / "INTEGRATION.md"


def _turned(x, table, positions):
    cos, sin = table[positions].split(32, 1)
    if x.dim() == 3:
        cos, sin = cos[:, None], sin[:, None]
    ref, tol = do.rotate(x, cos, sin, True), do.rotate_bound(x, cos, sin, True)
    return ref, tol + (ref.abs() + tol) * do.HALF_BF16


@pytest.mark.parametrize("heads,prompts", [(3, [1, 3, 0, 0]), (20, [70, 1, 133])])
def test_the_guides_calls(heads, prompts):
    section = GUIDE.read_text().split("## 5. Dense prefill and decode")[1].split("\n## ")[0]
    code = re.search(r"```python\n(.*?)```", section, re.S).group(1)
    g = _gen(heads)
    B, T, block = len(prompts), sum(prompts), 16
    cols = max(prompts) // block + 1
    table = torch.randperm(B * cols, generator=g).view(B, cols).int()
    seq = [b for b, n in enumerate(prompts) for _ in range(n)]
    pos = [i for n in prompts for i in range(n)]
    slot = [int(table[b, p // block]) * block + p % block for b, p in zip(seq, pos)]
    step_slot = [int(table[b, n // block]) * block + n % block for b, n in enumerate(prompts)]
    turns = _table(max(prompts) + 1)
    cu = torch.tensor([0] + torch.tensor(prompts).cumsum(0).tolist(), dtype=torch.int32, device=DEV)
    host = dict(kv_c=_bf16(g, T, 512), k_rope=_bf16(g, T, 64), q=_bf16(g, T, heads, 192), k_nope=_bf16(g, T, heads, 128), v=_bf16(g, T, heads, 128),
                step_kv_c=_bf16(g, B, 512), step_k_rope=_bf16(g, B, 64), step_q=_bf16(g, B, heads, 192), q_abs=_bf16(g, B, heads, 576))
    names = {n: t.to(DEV) for n, t in host.items()}
    names.update(cos_sin=turns.to(DEV), positions=torch.tensor(pos, device=DEV), slots=torch.tensor(slot, device=DEV), sm_scale=SCALE,
                 k_rope_turned=torch.zeros((T, 64), dtype=torch.bfloat16, device=DEV), cache=torch.zeros((B * cols, block, 656), dtype=torch.uint8, device=DEV),
                 cu_q=cu, cu_k=cu, block_table=table.to(DEV), seq_lens=torch.tensor([n + 1 for n in prompts], dtype=torch.int32, device=DEV),
                 step_positions=torch.tensor(prompts, device=DEV), step_slots=torch.tensor(step_slot, device=DEV))
    exec(compile(code, str(GUIDE), "exec"), names)

    # the prompts: queries and keys turned by their positions, everything attended to
    q, k_rope = names["q"].cpu(), names["k_rope_turned"].cpu()
    assert torch.equal(q[..., :128], host["q"][..., :128])
    _check(q[..., 128:], *_turned(host["q"][..., 128:], turns, torch.tensor(pos)))
    _check(k_rope, *_turned(host["k_rope"], turns, torch.tensor(pos)))
    for b, n in enumerate(prompts):
        if n:
            k0, i = int(cu[b]), max(0, n - 3)
            o, s, o_tol, s_tol = do.prefill(q[k0 + i:k0 + n], host["k_nope"][k0:k0 + n], k_rope[k0:k0 + n], host["v"][k0:k0 + n], SCALE)
            _check(names["out"][k0 + i:k0 + n], o, o_tol)
            _check(names["lse"][k0 + i:k0 + n], s, s_tol)
    # the step
    q_abs = names["q_abs"].cpu()
    assert torch.equal(q_abs[..., :512], host["q_abs"][..., :512])
    _check(q_abs[..., 512:], *_turned(host["step_q"][..., 128:], turns, torch.tensor(prompts)))
    rows = torch.stack([do.unpack_row(r) for r in names["cache"].cpu().view(-1, 656)])
    for b, n in enumerate(prompts):
        o, s, o_tol, s_tol = do.decode(q_abs[b:b + 1], rows, table[b], n + 1, block, SCALE)
        _check(names["step_out"][b:b + 1], o, o_tol)
        _check(names["step_lse"][b:b + 1], s, s_tol)
    # the rows that the sparse operators take
    assert torch.equal(names["kv"].cpu().view(torch.int16), rows.view(torch.int16))
