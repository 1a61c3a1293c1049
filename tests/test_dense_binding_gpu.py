"""The short way into the dense operators (host_binding.cpp) against the general one (ctypes): the same results bit for bit, and what is
not plain goes the general way, with its results and errors."""
import math

import pytest
import torch

import litetopk_b200 as lt
from litetopk_b200 import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture
def both(monkeypatch):
    """f -> (result of f by the short way, by the general one), and whether the short way took it."""
    host = _lib.host()
    assert host is not None, "the module of host_binding.cpp is missing"

    def run(f):
        took = []

        class Spy:
            def __getattr__(self, name):
                def call(*args):
                    took.append(getattr(host, name)(*args))
                    return took[-1]
                return call
        monkeypatch.setattr(_lib, "_host", Spy())
        short = f()
        monkeypatch.setattr(_lib, "_host", None)
        general = f()
        torch.cuda.synchronize()
        return short, general, [r is not None for r in took]
    return run


def _same(a, b):
    assert len(a) == len(b)
    for x, y in zip(a, b):
        assert x.shape == y.shape and x.dtype == y.dtype and x.stride() == y.stride()
        assert torch.equal(x.view(torch.uint8) if x.dtype == torch.uint8 else x.nan_to_num(7.0), y.view(torch.uint8) if y.dtype == torch.uint8 else y.nan_to_num(7.0))


def _bf16(*shape):
    g = torch.Generator(device=DEV).manual_seed(sum(shape))
    return torch.randn(shape, generator=g, device=DEV).to(torch.bfloat16)


def _append(packed=True, heads=5, index=torch.int64, **kw):
    T = 7
    cache = torch.zeros((4, 16, 656), dtype=torch.uint8, device=DEV) if packed else torch.zeros((4, 16, 576), dtype=torch.bfloat16, device=DEV)
    q_out, k_out = (torch.zeros((T, max(heads, 1), 576), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    args = dict(kv_c=_bf16(T, 576)[:, :512], k_rope=_bf16(T, 64), positions=torch.arange(T, device=DEV).to(index),
                cos_sin=torch.rand((20, 64), generator=torch.Generator(device=DEV).manual_seed(1), device=DEV),
                slots=torch.arange(T, device=DEV).to(index) * 3, kv_cache=cache)
    if heads:
        args.update(q_rope=_bf16(T, heads, 192)[..., 128:], q_out=q_out[..., 512:], k_out=k_out[:, 0, :64])
    lt.append_kv(**{**args, **kw})
    return cache, q_out, k_out


@pytest.mark.parametrize("kw", [{}, dict(packed=False), dict(heads=0), dict(index=torch.int32), dict(interleaved=False)])
def test_append(both, kw):
    short, general, took = both(lambda: _append(**kw))
    assert took == [True]
    _same(short, general)


def _decode(packed=False, q_len=1, block=64, **kw):
    pages = 12
    cache = _bf16(pages, block, 576)
    if packed:
        cache = torch.zeros((pages, block, 656), dtype=torch.uint8, device=DEV)
        rows = pages * block
        table = torch.rand((rows, 64), device=DEV, generator=torch.Generator(device=DEV).manual_seed(2))
        lt.append_kv(_bf16(rows, 512), _bf16(rows, 64), torch.arange(rows, device=DEV), table, torch.arange(rows, device=DEV), cache)
    q = _bf16(3, q_len, 20, 576) if q_len > 1 else _bf16(3, 20, 576)
    args = dict(q=q, kv_cache=cache, block_table=torch.arange(12, dtype=torch.int32, device=DEV).view(3, 4), seq_lens=torch.tensor([1, 4 * block, 70], dtype=torch.int32, device=DEV),
                sm_scale=0.1)
    return lt.mla_decode(**{**args, **kw})


@pytest.mark.parametrize("kw", [{}, dict(packed=True), dict(q_len=3), dict(block=32)])
def test_decode(both, kw):
    short, general, took = both(lambda: _decode(**kw))
    assert took == [True] * (2 if kw.get("packed") else 1)                   # (packed rows are written by append_kv)
    _same(short, general)


def _prefill(T=40, **kw):
    kv = _bf16(T + 9, 3, 256)
    args = dict(q=_bf16(T, 3, 192), k_nope=kv[..., :128], k_rope=_bf16(T + 9, 64), v=kv[..., 128:], sm_scale=0.1)
    return lt.mla_prefill(**{**args, **kw})


def test_prefill(both):
    cu = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)      # noqa: E731
    for kw in ({}, dict(causal=False), dict(cu_seqlens_q=cu(0, 11, 40), cu_seqlens_k=cu(0, 15, 49)), dict(T=900)):
        short, general, took = both(lambda: _prefill(**kw))
        assert took == [True]
        _same(short, general)


def test_what_is_not_plain_goes_the_general_way(both):
    for f in (lambda: _prefill(sm_scale=torch.tensor(0.1)), lambda: _prefill(out=torch.empty((40, 3, 128), dtype=torch.bfloat16, device=DEV)),
              lambda: _prefill(causal=1), lambda: _decode(sm_scale=torch.tensor(0.1)), lambda: _decode(lse=torch.empty((3, 20), device=DEV)),
              lambda: _decode(seq_lens=torch.tensor([1, 9, 256, 9, 70], dtype=torch.int32, device=DEV)[::2].contiguous()[:3], block_table=torch.zeros((3, 0), dtype=torch.int32, device=DEV)),
              lambda: _append(interleaved=1), lambda: _append(kv_cache=torch.zeros((64, 656), dtype=torch.uint8, device=DEV))):
        short, general, took = both(f)
        assert not any(took)
        _same(short, general)


@pytest.mark.parametrize("way", ["short", "general"])
def test_errors_are_the_same_either_way(monkeypatch, way):
    if way == "general":
        monkeypatch.setattr(_lib, "_host", None)
    for call, error in ((lambda: _append(kv_c=_bf16(7, 576)), ValueError), (lambda: _append(k_rope=_bf16(6, 64)), ValueError),
                        (lambda: _append(slots=torch.zeros(7, device=DEV)), TypeError), (lambda: _append(q_out=None), ValueError),
                        (lambda: _append(cos_sin=torch.zeros((20, 64), dtype=torch.float64, device=DEV)), TypeError),
                        (lambda: _append(kv_cache=torch.zeros((4, 16, 576), device=DEV)), TypeError),
                        (lambda: _append(kv_cache=torch.zeros((4, 16, 640), dtype=torch.uint8, device=DEV)), ValueError),
                        (lambda: _append(positions=torch.zeros(7, dtype=torch.int64)), ValueError),
                        (lambda: _decode(block=8), ValueError), (lambda: _decode(q=_bf16(3, 129, 576)), ValueError), (lambda: _decode(q=_bf16(3, 20, 512)), ValueError),
                        (lambda: _decode(q=_bf16(3, 20, 576).float()), TypeError), (lambda: _decode(seq_lens=torch.zeros(3, dtype=torch.int64, device=DEV)), TypeError),
                        (lambda: _decode(block_table=torch.zeros((2, 4), dtype=torch.int32, device=DEV)), ValueError),
                        (lambda: _decode(kv_cache=_bf16(64, 576)), ValueError), (lambda: _decode(seq_lens=torch.zeros(3, dtype=torch.int32)), ValueError),
                        (lambda: _decode(out=torch.empty((3, 20, 576), dtype=torch.bfloat16, device=DEV)), ValueError),
                        (lambda: _prefill(sm_scale=-1.0), ValueError), (lambda: _prefill(sm_scale=math.nan), ValueError), (lambda: _prefill(q=_bf16(40, 3, 128)), ValueError),
                        (lambda: _prefill(k_rope=_bf16(48, 64)), ValueError), (lambda: _prefill(cu_seqlens_q=torch.zeros(2, dtype=torch.int32, device=DEV)), ValueError),
                        (lambda: _prefill(v=_bf16(49, 3, 128).cpu()), ValueError), (lambda: _prefill(q=_bf16(40, 3, 192).half()), TypeError)):
        with pytest.raises(error):
            call()
    wide = _bf16(3, 20, 580)[..., 4:]                                        # rows that do not start on 16 bytes: refused by the library
    for call in (lambda: _decode(q=wide), lambda: _append(k_rope=_bf16(7, 68)[:, 4:]), lambda: _prefill(k_rope=_bf16(49, 68)[:, :64])):
        with pytest.raises(_lib.LiteDSAError) as e:
            call()
        assert e.value.code == _lib.ERR_UNSUPPORTED
