"""Numbers that the 8-bit attention's calls cannot hand on are refused by the library's own errors; no device is needed."""
import pytest
import torch

from sandyrt_b200.csrc import ops
from sandyrt_b200.errors import KernelError, UnsupportedShape
from test_cache8 import _cache, _i32


def _decode(scale=0.1, **rules):
    q = torch.zeros(2, 256)
    ops.decode_attention_8bit(q, _cache(), _i32(0, 1, 2, 3).reshape(2, 2), _i32(0, 1), _i32(3, 4), torch.zeros_like(q), n_heads=4, scale=scale, **rules)


def _prompt(scale=0.1, **rules):
    q = torch.zeros(2, 256)
    ops.prefill_attention_8bit(q, _cache(), _i32(0, 1).reshape(1, 2), _i32(0, 2), _i32(3), torch.zeros_like(q), n_heads=4, max_q_len=2, scale=scale, **rules)


@pytest.mark.parametrize("call", [_decode, _prompt])
@pytest.mark.parametrize("rules,error,words", [
    (dict(window=1 << 31), UnsupportedShape, "32-bit"),
    (dict(keep_first=1 << 31, window=5), UnsupportedShape, "32-bit"),
    (dict(chunk=1 << 40), UnsupportedShape, "32-bit"),
    (dict(softcap=float("inf")), UnsupportedShape, "cap at most"),
    (dict(softcap=1e31), UnsupportedShape, "cap at most"),
    (dict(softcap=1e300), UnsupportedShape, "cap at most"),
    (dict(scale=float("nan")), KernelError, "finite"),
    (dict(scale=float("inf")), KernelError, "finite"),
    (dict(scale=-1e300), KernelError, "finite"),
    # the largest there are go on to the next check, which finds no device
    (dict(window=(1 << 31) - 1, keep_first=(1 << 31) - 1), KernelError, "CUDA tensors"),
    (dict(softcap=1e30), KernelError, "CUDA tensors"),
])
def test_numbers_that_do_not_fit(call, rules, error, words):
    with pytest.raises(error, match=words):
        call(**rules)
