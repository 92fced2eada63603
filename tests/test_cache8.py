"""The 8-bit cache's Python face without a device: what it refuses, and that its plain implementation is what it says."""
import math

import pytest
import torch

from plain_cache8 import CODES, LARGEST, PlainCache, nearest, scale_for
from sandyrt_b200.csrc import ops
from sandyrt_b200.errors import KernelError, UnsupportedShape


def _cache(pages=4, hkv=2, ps=16, d=64, dtype=torch.int8):
    return ops.Cache8.empty(pages, hkv, ps, d, dtype=dtype, device="cpu")


def _i32(*v):
    return torch.tensor(v, dtype=torch.int32)


def _append(cache=None, k=None, v=None, table=None, q_start=None, before=None, max_q_len=3):
    cache = cache or _cache()
    k = torch.zeros(3, 128) if k is None else k
    ops.kv_append_8bit(k, torch.zeros_like(k) if v is None else v, cache, _i32(0, 1).reshape(1, 2) if table is None else table,
                       _i32(0, 3) if q_start is None else q_start, _i32(5) if before is None else before, max_q_len=max_q_len)


def _decode(q=None, cache=None, out=None, table=None, seq=None, pos=None, n_heads=4, **rules):
    q = torch.zeros(2, 256) if q is None else q
    ops.decode_attention_8bit(q, cache or _cache(), _i32(0, 1, 2, 3).reshape(2, 2) if table is None else table, _i32(0, 1) if seq is None else seq,
                              _i32(3, 4) if pos is None else pos, torch.zeros_like(q) if out is None else out, n_heads=n_heads, scale=0.1, **rules)


def _with(cache, **parts):
    for name, t in parts.items():
        setattr(cache, name, t)
    return cache


@pytest.mark.parametrize("call,error,words", [
    (lambda: _append(), KernelError, "CUDA tensors"),
    (lambda: _append(cache=_cache(dtype=torch.uint8)), UnsupportedShape, "float8_e4m3fn or int8"),
    (lambda: _append(cache=_with(_cache(), v=torch.zeros(4, 2, 16, 64, dtype=torch.float8_e4m3fn))), UnsupportedShape, "float8_e4m3fn or int8"),
    (lambda: _append(cache=_cache(d=40), k=torch.zeros(3, 80)), UnsupportedShape, "head sizes"),
    (lambda: _append(cache=_cache(d=272), k=torch.zeros(3, 544)), UnsupportedShape, "head sizes"),
    (lambda: _append(cache=_with(_cache(), k=torch.zeros(4, 2, 16, 64, dtype=torch.int8).transpose(1, 2).contiguous().transpose(1, 2))), KernelError, "dense"),
    (lambda: _append(cache=_with(_cache(), v=torch.zeros(5, 2, 16, 64, dtype=torch.int8))), KernelError, "alike"),
    (lambda: _append(cache=_with(_cache(), k_scale=torch.zeros(4, 3))), KernelError, "scales"),
    (lambda: _append(cache=_with(_cache(), v_scale=torch.zeros(4, 2, dtype=torch.float64))), KernelError, "scales"),
    (lambda: _append(cache=_with(_cache(), k=torch.zeros(1, 2, 16, 64, dtype=torch.int8).expand(4, -1, -1, -1),
                                 v=torch.zeros(1, 2, 16, 64, dtype=torch.int8).expand(4, -1, -1, -1))), KernelError, "overlap"),
    (lambda: _append(k=torch.zeros(3, 120)), KernelError, "rows must be"),
    (lambda: _append(v=torch.zeros(2, 128)), KernelError, "rows must be"),
    (lambda: _append(v=torch.zeros(3, 128, dtype=torch.bfloat16)), KernelError, "rows must be"),
    (lambda: _append(k=torch.zeros(128, 3).t()), KernelError, "rows must be"),
    (lambda: _append(k=torch.zeros(3, 128, dtype=torch.float16)), UnsupportedShape, "float32 or bfloat16"),
    (lambda: _append(q_start=_i32(0, 1, 3)), KernelError, "disagree"),
    (lambda: _append(before=_i32(5, 6)), KernelError, "disagree"),
    (lambda: _append(before=torch.tensor([5])), KernelError, "int32"),
    (lambda: _append(table=_i32(0, 1)), KernelError, "disagree"),
    (lambda: _append(max_q_len=-1), KernelError, "negative"),
    (lambda: _decode(), KernelError, "CUDA tensors"),
    (lambda: _decode(n_heads=3), UnsupportedShape, "do not divide"),
    (lambda: _decode(q=torch.zeros(2, 200)), KernelError, "q and out"),
    (lambda: _decode(out=torch.zeros(2, 256, dtype=torch.bfloat16)), KernelError, "q and out"),
    (lambda: _decode(seq=_i32(0)), KernelError, "disagree"),
    (lambda: _decode(pos=_i32(0, 1, 2)), KernelError, "disagree"),
    (lambda: _decode(window=-1), UnsupportedShape, "negative"),
    (lambda: _decode(softcap=float("nan")), UnsupportedShape, "negative"),
    (lambda: _decode(keep_first=1, chunk=4), UnsupportedShape, "not together"),
    (lambda: _decode(sink=torch.zeros(3)), KernelError, "sink"),
    (lambda: _decode(out_gate=torch.zeros(2, 3)), KernelError, "gate by head"),
    (lambda: _decode(dist_bias=torch.zeros(4, 0)), KernelError, "bias by distance"),
    (lambda: _decode(elem_gate=torch.zeros(2, 5)), KernelError, "gate by element"),
    (lambda: _decode(elem_gate=torch.zeros(2, 8, dtype=torch.bfloat16)), KernelError, "gate by element"),
    (lambda: _decode(num_splits=-1), KernelError, "num_splits"),
    (lambda: _decode(windows=3), TypeError, "windows"),
])
def test_refusals_of_the_cache_kernels(call, error, words):
    with pytest.raises(error, match=words):
        call()


@pytest.mark.parametrize("more,error,words", [
    (dict(), KernelError, "CUDA tensors"),
    (dict(logits=torch.zeros(5, 2).t()), KernelError, "innermost"),
    (dict(logits=torch.zeros(2, 5, dtype=torch.float64)), UnsupportedShape, "float32 or bfloat16"),
    (dict(ids=torch.zeros(2, dtype=torch.int64)), KernelError, "ids"),
    (dict(ids=None), KernelError, "go with"),
    (dict(logprob=torch.zeros(3)), KernelError, "logprob"),
    (dict(entropy=torch.zeros(2, dtype=torch.float64)), KernelError, "entropy"),
    (dict(top_ids=torch.zeros(2, 3, dtype=torch.int32)), KernelError, "go with"),
    (dict(top_ids=torch.zeros(2, 3, dtype=torch.int32), top_logprobs=torch.zeros(2, 2)), KernelError, "top_logprobs"),
    (dict(top_ids=torch.zeros(2, 6, dtype=torch.int32), top_logprobs=torch.zeros(2, 6)), UnsupportedShape, "likeliest"),
    (dict(logits=torch.zeros(2, 50), top_ids=torch.zeros(2, 33, dtype=torch.int32), top_logprobs=torch.zeros(2, 33)), UnsupportedShape, "likeliest"),
    (dict(status=torch.zeros(1)), KernelError, "status"),
])
def test_refusals_of_token_logprobs(more, error, words):
    args = dict(logits=torch.zeros(2, 5), ids=torch.zeros(2, dtype=torch.int32), logprob=torch.zeros(2))
    args.update(more)
    with pytest.raises(error, match=words):
        ops.token_logprobs(args.pop("logits"), args.pop("ids"), args.pop("logprob"), **args)


@pytest.mark.parametrize("code", list(CODES))
def test_a_scale_is_the_smallest_power_of_two(code):
    code = CODES[code]
    for amax in (1e-3, 0.7, 1.0, LARGEST[code], LARGEST[code] * 1.001, 3.3e4, LARGEST[code] * 2.0 ** -20, 1e30):
        s = scale_for(amax, code)
        assert math.log2(s) == int(math.log2(s)) and amax <= LARGEST[code] * s and amax > LARGEST[code] * s / 2
    assert scale_for(0.0, code) == 2.0 ** -100 == scale_for(1e-38, code)


def test_the_plain_rounding_is_the_type_s():
    """Against torch's conversion, at every code, between codes and at ties."""
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    codes = codes[torch.isfinite(codes)].sort().values
    y = torch.cat([codes, (codes[1:] + codes[:-1]) / 2, codes[1:] * 0.3 + codes[:-1] * 0.7])
    assert torch.equal(nearest(y, torch.float8_e4m3fn), y.float().to(torch.float8_e4m3fn).double())


def test_growing_blocks_in_int8_stay_within_one_step():
    """Rounding old codes again at every doubling of the scale costs no more than one step of the last scale together."""
    g = torch.Generator().manual_seed(3)
    cache = PlainCache(1, 1, 16, 16, torch.int8)
    x = torch.randn(16, 1, 16, generator=g, dtype=torch.float64) * torch.exp2(torch.arange(16.0))[:, None, None]
    for t in range(16):
        cache.append(x[t:t + 1], x[t:t + 1], [[0]], [0, 1], [t])
    got = cache.values(0, [0], 16)
    step = float(cache.scales[0][0, 0])
    assert step == scale_for(float(x.abs().max()), torch.int8)
    assert float((got - x).abs().max()) <= step
