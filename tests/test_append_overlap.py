"""append_kv refuses outputs that overlap themselves, which several threads would write."""
import pytest
import torch

import litetopk_b200 as lt
from litetopk_b200 import _lib

P = 0x1000


def test_the_c_call(built_lib):
    def call(token=256, head=64, heads=4, T=3, k=64):
        # (refused before any CUDA call)
        return built_lib.litedsa_append_kv(P, 512, P, 64, P, 1, P, 10, 64, P, 1, P, 1, 4, 64, 64 * 656, 1, P, 256, 64, P, token, head, heads, P, k, T, None)
    for bad in (dict(token=0), dict(head=0), dict(token=192), dict(head=56), dict(token=64, head=128), dict(token=64, head=64), dict(k=0), dict(k=56), dict(T=1, head=0),
                dict(heads=1, token=0), dict(token=-256)):
        assert call(**bad) == _lib.ERR_UNSUPPORTED, bad


@pytest.mark.gpu
def test_what_is_refused_by_name_and_what_is_not():
    dev = "cuda:0"
    T, heads = 3, 4
    args = dict(kv_c=torch.ones((T, 512), dtype=torch.bfloat16, device=dev), k_rope=torch.ones((T, 64), dtype=torch.bfloat16, device=dev),
                positions=torch.zeros(T, dtype=torch.int64, device=dev), cos_sin=torch.cat((torch.ones((1, 32)), torch.zeros((1, 32))), 1).to(dev),
                slots=torch.arange(T, device=dev), kv_cache=torch.zeros((16, 576), dtype=torch.bfloat16, device=dev))
    paged = dict(args, kv_cache=torch.zeros((1, 16, 576), dtype=torch.bfloat16, device=dev))
    q = torch.randn((T, heads, 64), device=dev).bfloat16()
    base = torch.zeros((T * heads * 64,), dtype=torch.bfloat16, device=dev)
    for a in (args, paged):                                # (the general way in, and the short one)
        for out in (base[:64].expand(T, heads, 64), base[:T * 64].view(T, 1, 64).expand(T, heads, 64), base.as_strided((T, heads, 64), (192, 64, 1)),
                    base.as_strided((T, heads, 64), (32, 128, 1))):
            with pytest.raises(ValueError, match="q_out must not overlap itself"):
                lt.append_kv(**a, q_rope=q, q_out=out)
        with pytest.raises(ValueError, match="k_out must not overlap itself"):
            lt.append_kv(**a, k_out=base[:64].expand(T, 64))
        # heads first, a head or a token alone, queries that are one vector
        out = torch.zeros((heads, T, 64), dtype=torch.bfloat16, device=dev).transpose(0, 1)
        lt.append_kv(**a, q_rope=q, q_out=out)
        assert torch.equal(out, q)
        one = torch.zeros((T, 64), dtype=torch.bfloat16, device=dev)
        lt.append_kv(**a, q_rope=q[:, :1], q_out=one[:, None], k_out=torch.zeros((T, 72), dtype=torch.bfloat16, device=dev)[:, 8:])
        assert torch.equal(one, q[:, 0])
        lt.append_kv(**a, q_rope=q[:1, :1].expand(T, heads, 64), q_out=out)
        assert torch.equal(out, q[:1, :1].expand(T, heads, 64))
    first = {n: t[:1] if n not in ("cos_sin", "kv_cache") else t for n, t in paged.items()}
    out = torch.zeros((1, heads, 64), dtype=torch.bfloat16, device=dev)
    lt.append_kv(**first, q_rope=q[:1], q_out=out.as_strided((1, heads, 64), (8, 64, 1)))
    assert torch.equal(out, q[:1])
