"""Calls at the edges of what the 8-bit cache's attention takes."""
import numpy as np
import pytest
import torch

from plain_cache8 import CODES, PlainCache, attention
from test_cache8_gpu import DEV, TYPES, _check_attention, _device_cache, _filled, _i32, _tables, _tolerance, _values

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tc", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_portions_past_the_last_position(tc, dtype):
    """A portion whose positions pass 2^31 - 1 is reported and its rows are left as they were; another beside it is served."""
    from sandyrt_b200.csrc import ops
    from sandyrt_b200.errors import KernelError

    if tc and dtype == torch.float32:
        pytest.skip("the tcgen05 kernel takes bfloat16")
    plain, lists, table = _filled(np.random.default_rng(3), "e4m3", 2, 64, 16, [64, 64])
    dev = _device_cache(plain)
    q = torch.randn(8, 4 * 64, device=DEV).to(dtype)
    want = torch.empty_like(q)
    call = lambda before, out: ops.prefill_attention_8bit(q, dev, table, _i32([0, 4, 8]), _i32(before), out, n_heads=4, max_q_len=4, scale=0.1, tc=tc)
    call([60, 60], want)
    ops.check_kernel_status(DEV)
    for before in (2 ** 31 - 1, 2 ** 31 - 3):
        got = torch.full_like(q, 3.0)
        call([before, 60], got)
        with pytest.raises(KernelError, match="status 16"):
            ops.check_kernel_status(DEV)
        assert bool((got[:4] == 3).all()) and torch.equal(got[4:], want[4:])


@pytest.mark.parametrize("softcap", [0.5, 50.0, 3e3, 1e5, 1e7, 1e30])
@pytest.mark.parametrize("path", ["decode", "mma", "chosen"])
def test_caps_of_every_size(softcap, path):
    """A cap far above the scores changes nothing; its own size does not make their error larger.  Scores of some 30 beside each other."""
    seqs = [(0, 1), (70, 1), (200, 1)] if path == "decode" else [(0, 60), (150, 40)]
    _check_attention("int8", "bf16", 4, 2, 64, 16, seqs, path == "decode", q_scale=8.0, softcap=softcap, tc=False if path == "mma" else None)
    if path != "chosen":
        _check_attention("e4m3", "f32", 4, 2, 64, 16, seqs, path == "decode", softcap=softcap)


def test_caps_that_the_tcgen05_kernel_takes():
    from sandyrt_b200.errors import UnsupportedShape

    _check_attention("int8", "bf16", 4, 2, 64, 16, [(0, 60), (150, 40)], False, q_scale=8.0, softcap=512.0, tc=True)
    with pytest.raises(UnsupportedShape):
        _check_attention("int8", "bf16", 4, 2, 64, 16, [(0, 60)], False, softcap=513.0, tc=True)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("code", list(CODES))
@pytest.mark.parametrize("low", [torch.finfo(torch.float32).min, -1e30, 1e30, float("-inf")])
@pytest.mark.parametrize("decode", [True, False])
def test_biases_as_masks(code, dtype, low, decode):
    """A bias of the type's lowest number, or of -1e30, on every distance: a row is the mean of its values, whose blocks differ in size.  On some
    distances: the others are all that counts (with 1e30 the other way round).  Minus infinity on all: zeros."""
    from sandyrt_b200.csrc import ops

    rng = np.random.default_rng(31)
    hkv, d, ps, H, n = 1, 64, 16, 2, 100
    lists, table, pages = _tables(rng, [-(-n // ps)])
    plain = PlainCache(pages, hkv, ps, d, CODES[code])
    k, v = (_values(rng, n, hkv, d, torch.float64) for _ in range(2))
    v *= torch.exp2(torch.arange(n) // ps % 3 * 3.0)[:, None, None]
    plain.append(k, v, lists, [0, n], [0])
    dev = _device_cache(plain)
    kk, vv = (plain.values(w, lists[0], n) for w in range(2))
    pos = list(range(n - 12, n))
    q = torch.from_numpy(rng.standard_normal((len(pos), H * d))).to(TYPES[dtype])
    every = torch.full((H, 110), low)
    some = torch.zeros(H, 110)
    some[:, 3:40], some[1, 60:] = low, low
    for bias in (every, some):
        out = torch.empty(len(pos), H * d, dtype=TYPES[dtype], device=DEV)
        if decode:
            ops.decode_attention_8bit(q.to(DEV), dev, table, _i32([0] * len(pos)), _i32(pos), out, n_heads=H, scale=0.125, dist_bias=bias.to(DEV))
        else:
            ops.prefill_attention_8bit(q.to(DEV), dev, table, _i32([0, len(pos)]), _i32([pos[0]]), out, n_heads=H, max_q_len=len(pos), scale=0.125, dist_bias=bias.to(DEV))
        ops.check_kernel_status(DEV)
        if bias is every and low == float("-inf"):
            want = torch.zeros(len(pos), H * d, dtype=torch.float64)
        else:
            want = attention(q.double().reshape(len(pos), H, d), kk, vv, pos, scale=0.125, dist_bias=bias.double()).reshape(len(pos), -1)
        assert bool(((out.cpu().double() - want).abs() <= _tolerance(TYPES[dtype], want, vv)).all())
