"""Calls at the edges of what the 8-bit cache's attention takes."""
import numpy as np
import pytest
import torch

from plain_cache8 import CODES, PlainCache, attention
from test_cache8_gpu import DEV, TYPES, _check_attention, _device_cache, _filled, _i32, _tables, _tolerance, _values

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tc,dtype", [(True, torch.bfloat16), (False, torch.bfloat16), (False, torch.float32)])
def test_portions_past_the_last_position(tc, dtype):
    """A portion whose positions pass 2^31 - 1 is reported and its rows are left as they were; another beside it is served."""
    from sandyrt_b200.csrc import ops
    from sandyrt_b200.errors import KernelError

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


@pytest.mark.parametrize("tc,dtype", [(True, "bf16"), (False, "bf16"), (False, "f32")])
@pytest.mark.parametrize("rules", [{}, dict(window=9, keep_first=2), dict(chunk=8)], ids=lambda r: "-".join(r) or "plain")
def test_portions_padded_in_front(tc, dtype, rules):
    """A portion whose first rows stand at negative positions: zeros there, and the others as without them; a portion of such rows alone."""
    from sandyrt_b200.csrc import ops

    H, d = 4, 64
    plain, lists, table = _filled(np.random.default_rng(6), "int8", 2, d, 16, [50, 20])
    dev = _device_cache(plain)
    q = torch.randn(50 + 7 + 5, H * d, device=DEV).to(TYPES[dtype])
    got, want = torch.full_like(q, float("nan")), torch.empty_like(q)
    call = lambda q, starts, before, out: ops.prefill_attention_8bit(q, dev, table, _i32(starts), _i32(before), out, n_heads=H, max_q_len=60, scale=0.125, tc=tc, **rules)
    call(q, [0, 57, 62], [-7, -5], got)
    call(q[7:57], [0, 50, 50], [0, 0], want[7:57])
    ops.check_kernel_status(DEV)
    assert bool((got[:7] == 0).all()) and bool((got[57:] == 0).all())
    host = [plain.values(w, lists[0], 50) for w in range(2)]
    exact = attention(q[7:57].double().cpu().reshape(50, H, d), *host, list(range(50)), scale=0.125, **rules).reshape(50, -1)
    for out in (got, want):
        assert bool(((out[7:57].cpu().double() - exact).abs() <= _tolerance(TYPES[dtype], exact, host[1])).all())


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("offset", [1, 2, 3])
@pytest.mark.parametrize("decode", [True, False])
def test_rows_off_their_alignment(dtype, offset, decode):
    """Queries and results at any element, row pitches of any size; what is beside them is left as it was."""
    from sandyrt_b200.csrc import ops

    H, d, n = 4, 48, 40
    plain, lists, table = _filled(np.random.default_rng(7), "e4m3", 2, d, 16, [90])
    dev = _device_cache(plain)
    wide = torch.randn(n, H * d + 7, device=DEV).to(TYPES[dtype])
    out = torch.full_like(wide, 5.0)
    q, o = wide[:, offset:offset + H * d], out[:, offset:offset + H * d]
    pos = list(range(50, 90))
    if decode:
        ops.decode_attention_8bit(q, dev, table, _i32([0] * n), _i32(pos), o, n_heads=H, scale=0.14)
    else:
        ops.prefill_attention_8bit(q, dev, table, _i32([0, n]), _i32([50]), o, n_heads=H, max_q_len=n, scale=0.14)
    ops.check_kernel_status(DEV)
    host = [plain.values(w, lists[0], 90) for w in range(2)]
    want = attention(q.double().cpu().reshape(n, H, d), *host, pos, scale=0.14).reshape(n, -1)
    assert bool(((o.cpu().double() - want).abs() <= _tolerance(TYPES[dtype], want, host[1])).all())
    assert bool((out[:, :offset] == 5).all()) and bool((out[:, offset + H * d:] == 5).all())


@pytest.mark.parametrize("dtype", list(TYPES))
def test_hundreds_of_heads_that_share_one(dtype):
    _check_attention("int8", dtype, 300, 1, 16, 16, [(0, 1), (70, 1)], True)
    _check_attention("int8", dtype, 300, 1, 16, 16, [(0, 1), (70, 3)], False)
    _check_attention("e4m3", dtype, 50, 2, 32, 5, [(0, 1), (300, 1)], True, splits=3)          # odd pages, splits joined by a kernel
    _check_attention("e4m3", dtype, 50, 2, 32, 5, [(0, 1), (300, 1)], True, splits=12)
    if dtype == "bf16":
        _check_attention("int8", dtype, 300, 1, 16, 16, [(0, 1), (70, 3)], False, tc=True)


def test_appending_and_reading_in_turn_without_waiting():
    """A token's keys are written, read by single tokens and by a portion of one, and the result goes into the next call, all queued at
    once, on two streams side by side, and as recorded graphs: the same to the bit as with a wait behind every call."""
    from sandyrt_b200.csrc import ops

    S, H, hkv, d, ps, steps, first = 12, 8, 4, 64, 16, 60, 37
    blocks = -(-(first + steps) // ps)

    def made(seed):
        g = torch.Generator(device=DEV).manual_seed(seed)
        r = lambda *shape: torch.randn(*shape, generator=g, device=DEV).to(torch.bfloat16)
        i32 = lambda t: t.to(device=DEV, dtype=torch.int32)
        cache = ops.Cache8.empty(S * blocks, hkv, ps, d, device=DEV)
        for t in (cache.k, cache.v, cache.k_scale, cache.v_scale):
            t.view(torch.uint8).zero_()
        return dict(cache=cache, table=i32(torch.randperm(S * blocks, generator=g, device=DEV)).reshape(S, blocks), first=[r(S * first, hkv * d) for _ in range(2)],
                    new=[r(steps, S, hkv * d) for _ in range(2)], q=r(steps, S, H * d), out=torch.zeros(2, steps, S, H * d, dtype=torch.bfloat16, device=DEV),
                    starts=i32(torch.arange(S + 1) * first), zero=i32(torch.zeros(S)), one=i32(torch.arange(S + 1)), seq=i32(torch.arange(S)),
                    pos=[i32(torch.full((S,), first + i)) for i in range(steps)])

    def run(m, wait=lambda: None):
        ops.kv_append_8bit(*m["first"], m["cache"], m["table"], m["starts"], m["zero"], max_q_len=first)
        wait()
        for i in range(steps):
            ops.kv_append_8bit(m["new"][0][i], m["new"][1][i], m["cache"], m["table"], m["one"], m["pos"][i], max_q_len=1)
            wait()
            ops.decode_attention_8bit(m["q"][i], m["cache"], m["table"], m["seq"], m["pos"][i], m["out"][0, i], n_heads=H, scale=0.125, num_splits=(0, 1, 9)[i % 3])
            wait()
            ops.prefill_attention_8bit(m["out"][0, i], m["cache"], m["table"], m["one"], m["pos"][i], m["out"][1, i], n_heads=H, max_q_len=1, scale=0.125, tc=i % 2 == 0)
            wait()
        return m

    want = [run(made(s), lambda: torch.cuda.synchronize(DEV)) for s in (1, 2)]
    same = lambda m, w: torch.equal(m["out"], w["out"]) and all(torch.equal(getattr(m["cache"], n).view(torch.uint8), getattr(w["cache"], n).view(torch.uint8))
                                                                  for n in ("k", "v", "k_scale", "v_scale"))
    assert bool(torch.isfinite(want[0]["out"]).all()) and not torch.equal(want[0]["out"], want[1]["out"])
    assert same(run(made(1)), want[0])
    streams = [torch.cuda.Stream() for _ in range(2)]
    ms = [made(1), made(2)]
    torch.cuda.synchronize(DEV)
    for m, st in zip(ms, streams):
        with torch.cuda.stream(st):
            run(m)
    torch.cuda.synchronize(DEV)
    assert all(same(m, w) for m, w in zip(ms, want))
    graphs, ms = [], [made(1), made(2)]
    for m in ms:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            run(m)
    for _ in range(3):
        for m in ms:
            m["out"].zero_()
        torch.cuda.synchronize(DEV)
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize(DEV)
        assert all(torch.equal(m["out"], w["out"]) for m, w in zip(ms, want))
    ops.check_kernel_status(DEV)
