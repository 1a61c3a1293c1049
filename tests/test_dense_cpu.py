"""Refusals of the dense operators (checked before any CUDA call), and their oracle against plain torch."""
import math

import pytest
import torch

from litetopk_b200 import _lib
from oracle import dense_oracle as do

P = 0x1000


def test_append_refuses_wrong_arguments(built_lib):
    def call(kv_c=P, kr=P, pos=P, cs=P, slots=P, cache=P, packed=1, blocks=4, block=64, pitch=64 * 656, q=P, qo=P, heads=4, T=3, ks=512, css=64,
             qts=256, ko=None):
        return built_lib.litedsa_append_kv(kv_c, ks, kr, 64, pos, 1, cs, 10, css, slots, 1, cache, packed, blocks, block, pitch, 1, q, qts, 64, qo,
                                           256, 64, heads, ko, 64, T, None)
    for name in ("kv_c", "kr", "pos", "cs", "slots", "cache", "q", "qo"):
        assert call(**{name: None}) == _lib.ERR_ARG, name
    assert call(T=-1) == call(block=0) == call(heads=0) == call(pitch=64 * 656 - 16) == call(blocks=-1) == _lib.ERR_SHAPE
    for name in ("kv_c", "kr", "cs", "cache", "q", "qo", "ko"):
        assert call(**{name: P + 8}) == _lib.ERR_UNSUPPORTED, name
    assert call(ks=516) == call(css=66) == call(qts=260) == call(pitch=64 * 656 + 8) == _lib.ERR_UNSUPPORTED
    assert call(T=0) == _lib.OK


def test_decode_refuses_wrong_arguments(built_lib):
    def call(q=P, cache=P, packed=0, blocks=4, block=64, pitch=64 * 1152, table=P, cols=2, lens=P, out=P, lse=P, B=2, q_len=1, heads=16, ws=P,
             size=1 << 40, qb=9216):
        return built_lib.litedsa_mla_decode(q, qb, 9216, 576, cache, packed, blocks, block, pitch, table, cols, cols, lens, 0.1, out, lse, B, q_len,
                                            heads, ws, size, None)
    for name in ("q", "cache", "table", "lens", "out", "lse", "ws"):
        assert call(**{name: None}) == _lib.ERR_ARG, name
    for bad in (dict(B=-1), dict(q_len=0), dict(heads=0), dict(heads=129), dict(cols=-1), dict(block=0), dict(pitch=64 * 1152 - 16), dict(size=64)):
        assert call(**bad) == _lib.ERR_SHAPE, bad
    for bad in (dict(block=8, pitch=8 * 1152), dict(block=40), dict(q=P + 8), dict(cache=P + 2), dict(out=P + 8), dict(qb=9220), dict(pitch=64 * 1152 + 8),
                dict(lse=P + 2), dict(ws=P + 8), dict(cols=1 << 25, block=64)):
        assert call(**bad) == _lib.ERR_UNSUPPORTED, bad
    assert call(B=0) == _lib.OK
    assert built_lib.litedsa_mla_decode_workspace(0, 16) == built_lib.litedsa_mla_decode_workspace(1, 129) == 0


def test_prefill_refuses_wrong_arguments(built_lib):
    def call(q=P, kn=P, kr=P, v=P, cq=P, ck=P, B=2, scale=0.1, out=P, lse=P, Tq=1 << 20, Tk=100, heads=16, ws=None, size=0, qs=3200):
        return built_lib.litedsa_mla_prefill(q, qs, 192, kn, 4096, 256, kr, 64, v, 4096, 256, cq, ck, B, scale, 1, out, lse, Tq, Tk, heads, ws, size, None)
    for name in ("q", "kn", "kr", "v", "cq", "ck", "out", "lse"):
        assert call(**{name: None}) == _lib.ERR_ARG, name
    for bad in (dict(B=-1), dict(cq=None, ck=None), dict(Tq=-1), dict(Tk=-1), dict(heads=0)):
        assert call(**bad) == _lib.ERR_SHAPE, bad
    for bad in (dict(scale=-0.1), dict(scale=math.nan), dict(q=P + 8), dict(kn=P + 8), dict(kr=P + 8), dict(v=P + 8), dict(out=P + 8), dict(lse=P + 2),
                dict(qs=3204), dict(Tq=(1 << 31) - 1, heads=1 << 10)):
        assert call(**bad) == _lib.ERR_UNSUPPORTED, bad
    assert call(Tq=0) == call(Tq=0, q=None, out=None, lse=None) == _lib.OK
    need = built_lib.litedsa_mla_prefill_workspace(64, 4096, 2)
    assert need > 0 and built_lib.litedsa_mla_prefill_workspace(8192, 8192, 64) == built_lib.litedsa_mla_prefill_workspace(64, 64, 2) == 0
    assert call(Tq=64, Tk=4096, heads=2) == _lib.ERR_ARG and call(Tq=64, Tk=4096, heads=2, ws=P, size=need - 1) == _lib.ERR_SHAPE


def test_python_layer_names_what_is_wrong():
    import litetopk_b200 as lt
    cpu = torch.zeros((2, 512), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="kv_c must be a CUDA tensor"):
        lt.append_kv(cpu, cpu[:, :64], torch.zeros(2, dtype=torch.int64), torch.zeros((4, 64)), torch.zeros(2, dtype=torch.int64), torch.zeros((4, 576)))
    with pytest.raises(TypeError, match="kv_c must have dtype"):
        lt.append_kv(cpu.float(), cpu[:, :64], torch.zeros(2, dtype=torch.int64), torch.zeros((4, 64)), torch.zeros(2, dtype=torch.int64), torch.zeros((4, 576)))
    with pytest.raises(TypeError, match="q must have dtype"):
        lt.mla_decode(torch.zeros((1, 4, 576)), None, None, None, 1.0)
    with pytest.raises(ValueError, match="no CPU path"):
        lt.mla_decode(torch.zeros((1, 4, 576), dtype=torch.bfloat16), None, None, None, 1.0)


def test_oracle_agrees_with_plain_torch():
    g = torch.Generator().manual_seed(0)
    q, k = torch.randn((2, 3, 576), generator=g).to(torch.bfloat16), torch.randn((40, 576), generator=g).to(torch.bfloat16)
    o, s, o_tol, s_tol = do.decode(q, k, torch.tensor([1, 0]), 30, 20, 0.1)
    rows = torch.cat((k[20:], k[:20]))[:30].double()
    for j in range(2):
        x = q[j].double() @ rows[:29 + j].T * 0.1
        assert torch.allclose(o[j], torch.softmax(x, -1) @ rows[:29 + j, :512], atol=1e-12) and torch.allclose(s[j], torch.logsumexp(x, -1))
    assert bool((o_tol > 0).all()) and float(o_tol.max()) < 0.05 and float(s_tol.max()) < 2e-3
    o, s, _, _ = do.decode(q, k, torch.tensor([1, 0]), 1, 20, 0.1)
    assert bool((o[0] == 0).all()) and bool((s[0] == math.inf).all()) and torch.equal(o[1], k[20, :512].double().expand(3, 512))
    # the rotation is a product of complex numbers
    x, a = torch.randn((5, 64), generator=g), torch.randn((5, 32), generator=g).double()
    z = torch.view_as_complex(x.double().view(5, 32, 2)) * torch.polar(torch.ones_like(a), a)
    assert torch.allclose(do.rotate(x, a.cos(), a.sin(), True), torch.view_as_real(z).flatten(1))
    codes, scale = do.pack_latent(k[0, :512])
    back = codes.view(torch.float8_e4m3fn).double().view(4, 128) * scale[:, None]
    assert float((back - k[0, :512].double().view(4, 128)).abs().div(k[0, :512].double().abs().view(4, 128) + scale[:, None] * 2.0 ** -6).max()) <= 2.0 ** -4
