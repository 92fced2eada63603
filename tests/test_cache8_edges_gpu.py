"""Calls at the edges of what the 8-bit cache's attention takes."""
import numpy as np
import pytest
import torch

from test_cache8_gpu import DEV, _check_attention, _device_cache, _filled, _i32

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
