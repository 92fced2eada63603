"""Attention over the 8-bit cache where one key's weight is far above very many others', which together still count."""
import numpy as np
import pytest
import torch

from plain_cache8 import CODES, PlainCache
from test_cache8_gpu import DEV, TYPES, _device_cache, _i32, _tables, _tolerance

pytestmark = pytest.mark.gpu

BEFORE, D, SCALE = 100_000, 64, 0.125
_made = {}


def _one_key_above(code, first_value, ps):
    """A request of BEFORE + 40 keys whose first has a score 18 nats above the others' (which spread by half a nat around 0) and values
    of `first_value`; the others' values have a mean of 1.  (plain cache, page list, block table, keys, values); queries whose
    first element is 8 see it so."""
    key = (code, first_value, ps)
    if key not in _made:
        rng = np.random.default_rng(21)
        n = BEFORE + 40
        k = torch.from_numpy(rng.standard_normal((n, 1, D)) * 0.5)
        k[:, :, 0] = 0.0
        k[0] = 0.0
        k[0, 0, 0] = 18.0                                       # 8 * 18 / 8
        v = torch.from_numpy(1.0 + 0.3 * rng.standard_normal((n, 1, D)))
        v[0] = first_value
        lists, table, pages = _tables(rng, [-(-n // ps)])
        plain = PlainCache(pages, 1, ps, D, CODES[code])
        # the first key alone in its page, so that the others' codes are not made small beside it
        plain.append(k[:1], v[:1], lists, [0, 1], [0])
        plain.append(k[1:], v[1:], lists, [0, n - 1], [1])
        _made.clear()                                             # one at a time: some 200 MB on the host
        _made[key] = plain, table, plain.values(0, lists[0], n)[:, 0], plain.values(1, lists[0], n)[:, 0]
    return _made[key]


def _check(code, dtype, first_value, path, n, H, splits, ps, tolerance, above=True):
    from sandyrt_b200.csrc import ops

    plain, table, k, v = _one_key_above(code, first_value, ps)
    dev = _device_cache(plain)
    rng = np.random.default_rng(22)
    q = torch.from_numpy(rng.standard_normal((n, H, D))).to(TYPES[dtype])
    q[:, :, 0] = 8.0 if above else 0.0
    out = torch.empty(n, H * D, dtype=TYPES[dtype], device=DEV)
    pos = list(range(BEFORE, BEFORE + n))
    if path == "decode":
        ops.decode_attention_8bit(q.reshape(n, -1).to(DEV), dev, table, _i32([0] * n), _i32(pos), out, n_heads=H, scale=SCALE, num_splits=splits)
    else:
        ops.prefill_attention_8bit(q.reshape(n, -1).to(DEV), dev, table, _i32([0, n]), _i32([BEFORE]), out, n_heads=H, max_q_len=n, scale=SCALE,
                                   num_splits=splits, tc=path == "tcgen05")
    ops.check_kernel_status(DEV)
    s = (q.double().reshape(n * H, D) @ k.T * SCALE).reshape(n, H, -1)
    s = s.masked_fill(torch.arange(s.shape[2])[None, None] > torch.tensor(pos)[:, None, None], float("-inf"))
    want = (torch.softmax(s, dim=2) @ v).reshape(n, -1)
    off = (out.cpu().double() - want).abs()
    assert bool((off <= tolerance(want, v)).all()), (float(off.max()), float(want.abs().max()))


@pytest.mark.parametrize("code", list(CODES))
@pytest.mark.parametrize("first_value", [1.0, 0.0])
@pytest.mark.parametrize("path,n,H,splits", [("decode", 1, 1, 0), ("decode", 3, 4, 0), ("decode", 1, 8, 40), ("prompt", 5, 2, 0), ("prompt", 40, 1, 0)])
def test_small_weights_together_in_float32(code, first_value, path, n, H, splits):
    """100,000 weights of e^-18 = 2^-26 beside one of 1: together 1.5e-3 of the result.  The bound is the calls' own, and where they are all
    there is (the first value 0) 1e-4 of the result besides: scores of up to 26 in units of log 2, whose sums of 64 products
    and rounding are off by some ten times 2^-24 * 26, 1.6e-5 of a weight, and the weights' 22 bits."""
    def tolerance(want, v):
        bound = _tolerance(torch.float32, want, v)
        return bound if first_value else torch.minimum(bound, 1e-4 * want.abs())

    _check(code, "f32", first_value, path, n, H, splits, 64, tolerance)


def test_float32_values_of_many_small_weights_at_heads_of_every_kernel():
    """The same through the kernels of odd pages (rows looked up one by one)."""
    _check("int8", "f32", 0.0, "decode", 2, 3, 0, 37, lambda want, v: 1e-4 * want.abs())
    _check("int8", "f32", 0.0, "prompt", 9, 2, 2, 37, lambda want, v: 1e-4 * want.abs())


@pytest.mark.parametrize("code", list(CODES))
@pytest.mark.parametrize("above", [True, False])
@pytest.mark.parametrize("path,n,H", [("decode", 3, 4), ("decode", 2, 1), ("prompt", 40, 1)])
def test_sums_over_many_keys_in_float32(code, path, n, H, above):
    """100,000 keys walked by one block, so that a warp sums 25,000: small weights are not lost beside what the sums already hold."""
    _check(code, "f32", 1.0, path, n, H, 1, 64, lambda want, v: _tolerance(torch.float32, want, v), above)


def _half_tolerance(want, v):
    """The result's rounding (2^-8 of it) and its two columns' worth of sums (2^-9), and half a step of half precision's smallest numbers,
    2^-25 beside a reference of 2^-7 of the largest weight: 2^-32 of the largest value a key."""
    return want.abs() * (2.0 ** -8 + 2.0 ** -9) + BEFORE * 2.0 ** -32 * float(v.abs().max())


@pytest.mark.parametrize("code", list(CODES))
@pytest.mark.parametrize("first_value", [1.0, 0.0])
@pytest.mark.parametrize("path,n,H,splits", [("decode", 1, 1, 0), ("decode", 3, 4, 1), ("decode", 2, 8, 40), ("prompt", 5, 2, 0), ("prompt", 40, 1, 1), ("tcgen05", 40, 1, 0),
                                             ("tcgen05", 33, 4, 1), ("tcgen05", 40, 2, 8)])
def test_small_weights_together_in_bfloat16(code, first_value, path, n, H, splits):
    """The same as in float32: where the first key's value is 0, as that of a token that takes what attention is left over, the others'
    1.5e-3 are all there is."""
    _check(code, "bf16", first_value, path, n, H, splits, 64, _half_tolerance)


def test_small_weights_together_beside_scales_that_are_no_powers_of_two():
    """The largest weights there are, 2^14 and what a scale is beside its power of two, do not pass half precision's range: scores that
    rise by a little less than what moves the reference, in every tile."""
    from sandyrt_b200.csrc import ops

    n, hkv = 400, 1
    rng = np.random.default_rng(5)
    k = torch.zeros(n, hkv, D, dtype=torch.float64)
    k[:, 0, 0] = torch.arange(n) // 16 % 2 * 9.0                 # with q's first element 8 and scale 1/8: 9 nats, 13 in units of log 2
    v = torch.from_numpy(1.0 + 0.3 * rng.standard_normal((n, hkv, D)))
    lists, table, pages = _tables(rng, [-(-n // 16)])
    plain = PlainCache(pages, hkv, 16, D, torch.int8)
    plain.append(k, v, lists, [0, n], [0])
    plain.scales[1] = (plain.scales[1] * 1.99).float().double()
    dev = _device_cache(plain)
    q = torch.zeros(40, D)
    q[:, 0] = 8.0
    q = q.to(torch.bfloat16)
    kk, vv = (plain.values(w, lists[0], n)[:, 0] for w in range(2))
    for path in ("decode", "prompt", "tcgen05"):
        out = torch.empty(40, D, dtype=torch.bfloat16, device=DEV)
        pos = list(range(n - 40, n))
        if path == "decode":
            ops.decode_attention_8bit(q.to(DEV), dev, table, _i32([0] * 40), _i32(pos), out, n_heads=1, scale=SCALE, num_splits=1)
        else:
            ops.prefill_attention_8bit(q.to(DEV), dev, table, _i32([0, 40]), _i32([n - 40]), out, n_heads=1, max_q_len=40, scale=SCALE, num_splits=1, tc=path == "tcgen05")
        ops.check_kernel_status(DEV)
        want = torch.stack([torch.softmax(kk[:p + 1] @ q[0].double() * SCALE, 0) @ vv[:p + 1] for p in pos])
        # the weights' rounding, and what a scale is beside its power of two times a code: 2^-11 of each term twice
        assert bool(((out.cpu().double() - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -9)).all()), path
