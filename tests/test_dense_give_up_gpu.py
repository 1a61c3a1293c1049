"""Waits that run out in the dense attention kernels: a call returns and says so in its status, and the next call is as right as any.

With the shortest limit a wait gives up that takes longer than some milliseconds.  Some legitimately do where a sequence is long enough:
whoever brings the next piece's queries waits for as long as the present piece takes.  Its keys are a few pages, over and over.
"""
import pytest
import torch

import litetopk_b200 as lt
from litetopk_b200 import api
from test_dense_gpu import DEV, SCALE

pytestmark = pytest.mark.gpu


@pytest.fixture
def limit():
    yield api.set_wait_limit_ns
    api.set_wait_limit_ns(0)


def _gives_up_and_recovers(limit, call, status, sites):
    right = call()
    assert status(reset=True)[0] == 0
    limit(1)
    call()
    assert status(reset=True)[0] in sites
    limit(0)
    again = call()
    assert status(reset=True)[0] == 0
    assert all(torch.equal(a, b) for a, b in zip(right, again))


def _decode(heads, block, packed, sequences, blocks, rising=False):
    g = torch.Generator(device=DEV).manual_seed(heads)
    pages, cols = 2048 // block, 64 * blocks // block
    if packed:
        cache = torch.randint(0, 126, (pages, block, 656), generator=g, device=DEV).to(torch.uint8)
        cache[..., 512:528] = torch.ones(4, device=DEV).view(torch.uint8)
        cache[..., 528:] = torch.randn((pages, block, 64), generator=g, device=DEV).bfloat16().view(torch.uint8)
    else:
        cache = torch.randn((pages, block, 576), generator=g, device=DEV).bfloat16()
    table = torch.randint(0, pages, (sequences, cols), generator=g, device=DEV).int()
    lens = torch.full((sequences,), 64 * blocks, dtype=torch.int32, device=DEV)
    q = torch.randn((sequences, heads, 576), generator=g, device=DEV).bfloat16()
    if rising:                                         # page after page, each with scores far above the one before: maxima move all the time
        table = (torch.arange(cols, device=DEV) * pages // cols).int().repeat(sequences, 1)
        ramp = (torch.arange(pages, device=DEV) * (60 * block / 64)).bfloat16()[:, None]
        if packed:
            cache[..., 528:530] = ramp.view(torch.uint8).view(pages, 1, 2)
        else:
            cache[..., 512] = ramp
        q[..., 512] = 8
    return lambda: lt.mla_decode(q, cache, table, lens, SCALE)


@pytest.mark.parametrize("rising", [False, True])
@pytest.mark.parametrize("packed,block", [(False, 64), (False, 16), (True, 64)])
def test_decode_of_many_rows(limit, packed, block, rising):
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    _gives_up_and_recovers(limit, _decode(128, block, packed, sms, 6000, rising), lt.mla_decode_status, range(1, 10))


@pytest.mark.parametrize("rising", [False, True])
@pytest.mark.parametrize("heads", [16, 64])
@pytest.mark.parametrize("packed,block", [(False, 64), (False, 16), (True, 64)])
def test_decode_of_few_rows(limit, packed, block, heads, rising):
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    _gives_up_and_recovers(limit, _decode(heads, block, packed, 2 * sms, 8000, rising), lt.mla_decode_status, range(1, 10))


def test_decode_with_a_cut_sequence(limit):
    # parts of a launch that gave up are merged like any others; nothing of them is left afterwards
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    _gives_up_and_recovers(limit, _decode(32, 64, False, 2 * sms + 5, 8000), lt.mla_decode_status, range(1, 10))


def _prefill(heads, Tk):
    # (a key's heads begin a row apart in one and the same memory)
    g = torch.Generator(device=DEV).manual_seed(heads)
    rows = [torch.randn((Tk + heads, 128), generator=g, device=DEV, dtype=torch.bfloat16) for _ in range(2)]
    k, v = (x.as_strided((Tk, heads, 128), (128, 128, 1)) for x in rows)
    q = torch.randn((1, heads, 192), generator=g, device=DEV).bfloat16()
    rope = torch.randn((Tk, 64), generator=g, device=DEV, dtype=torch.bfloat16)
    return lambda: lt.mla_prefill(q, k, rope, v, SCALE)


def test_prefill(limit):
    # as many tiles as multiprocessors: whole.  The second tile has no query, so its warps wait for the next work as long as this one takes
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    _gives_up_and_recovers(limit, _prefill(sms, 128 * 6000), lt.mla_prefill_status, range(1, 11))


def test_prefill_of_tiles_that_are_cut(limit):
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    _gives_up_and_recovers(limit, _prefill(sms * 2 // 3, 128 * 24000), lt.mla_prefill_status, range(1, 11))
