"""The 8-bit cache's kernels and the log-probabilities of tokens against their formulas in 64 bits (plain_cache8.py)."""
import math

import numpy as np
import pytest
import torch

from plain_cache8 import CODES, PlainCache, attention, logprobs

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _starts(lens, at=0):
    return [int(v) for v in at + np.concatenate([[0], np.cumsum(lens)])]


def _tables(rng, needs, spare=2):
    """Page lists of requests that need so many pages, in no order, as (lists, table with -1 behind them, pages there are)."""
    total = sum(needs) + spare
    order = rng.permutation(total).tolist()
    lists, at = [], 0
    for n in needs:
        lists.append(order[at:at + n])
        at += n
    width = max(max(needs), 1)
    return lists, _i32([p + [-1] * (width - len(p)) for p in lists]), total


def _device_cache(plain):
    """A device cache with the plain one's codes; where nobody has written, codes and scales that would show."""
    from sandyrt_b200.csrc import ops

    c = ops.Cache8.empty(*plain.codes[0].shape, dtype=plain.code, device=DEV)
    for which, (codes, scales) in enumerate((("k", "k_scale"), ("v", "v_scale"))):
        x = plain.codes[which].float()
        if plain.code == torch.int8:
            getattr(c, codes).copy_(torch.where(torch.isnan(x), torch.tensor(113.0), x).to(torch.int8))
        else:
            getattr(c, codes).copy_(x.to(plain.code))
        getattr(c, scales).copy_(plain.scales[which].float())
    return c


def _same(dev, plain):
    """Whether the device cache holds the plain one's codes and scales; codes nobody wrote are not looked at."""
    for which, (codes, scales) in enumerate((("k", "k_scale"), ("v", "v_scale"))):
        want = plain.codes[which]
        got = getattr(dev, codes).cpu().to(torch.float32).double()
        written = ~torch.isnan(want)
        assert torch.equal(got[written], want[written])
        s_got, s_want = getattr(dev, scales).cpu().double(), plain.scales[which]
        assert torch.equal(torch.isnan(s_got), torch.isnan(s_want)) and torch.equal(s_got[~torch.isnan(s_got)], s_want[~torch.isnan(s_want)])


def _bits(cache):
    return [cache.k.view(torch.uint8).clone(), cache.v.view(torch.uint8).clone(), cache.k_scale.view(torch.int32).clone(), cache.v_scale.view(torch.int32).clone()]


def _values(rng, n, hkv, d, dtype, grow=1.0):
    x = torch.from_numpy(rng.standard_normal((n, hkv, d)) * np.exp(0.7 * rng.standard_normal((n, hkv, 1))) * grow)
    return x.to(dtype)


APPENDS = [  # hkv, d, page size, steps of (tokens each request brings)
    (2, 64, 16, [[5, 17, 0], [1, 1, 1], [1, 1, 40], [30, 1, 1], [1, 1, 1]]),
    (3, 16, 8, [[1], [7], [1], [9], [1]]),
    (1, 256, 64, [[70, 3], [1, 1], [1, 64]]),
    (5, 80, 5, [[4, 1, 11], [2, 2, 2], [1, 0, 1]]),
    (25, 64, 32, [[33], [1], [1]]),
    (2, 112, 1, [[3, 1], [1, 2]]),
]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("code", list(CODES))
@pytest.mark.parametrize("hkv,d,ps,steps", APPENDS)
def test_append_over_several_steps(code, dtype, hkv, d, ps, steps):
    """Codes and scales are those of the formula to the bit, blocks that grow among them; rows of no request are not read; the
    sources are columns of a wider matrix."""
    from sandyrt_b200.csrc import ops

    rng = np.random.default_rng(hkv * 100 + d + ps)
    S = len(steps[0])
    needs = [-(-sum(st[s] for st in steps) // ps) for s in range(S)]
    lists, table, pages = _tables(rng, needs)
    plain = PlainCache(pages, hkv, ps, d, CODES[code])
    dev = _device_cache(plain)
    have = [0] * S
    for i, lens in enumerate(steps):
        first = i % 3                                             # rows in front of the first request and behind the last
        starts = _starts(lens, first)
        n = starts[-1] + 2
        wide = torch.full((n, 3 * hkv * d + 8), float("nan"), dtype=TYPES[dtype], device=DEV)
        k, v = (_values(rng, n, hkv, d, TYPES[dtype], grow=1.7 ** i) for _ in range(2))
        rows = slice(first, starts[-1])
        wide[rows, hkv * d:2 * hkv * d] = k.reshape(n, -1)[rows].to(DEV)
        wide[rows, 2 * hkv * d:3 * hkv * d] = v.reshape(n, -1)[rows].to(DEV)
        ops.kv_append_8bit(wide[:, hkv * d:2 * hkv * d], wide[:, 2 * hkv * d:3 * hkv * d], dev, table, _i32(starts), _i32(have), max_q_len=max(lens))
        ops.check_kernel_status(DEV)
        plain.append(k.double(), v.double(), lists, starts, have)
        have = [h + x for h, x in zip(have, lens)]
        _same(dev, plain)


@pytest.mark.parametrize("offset", [1, 2, 3])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_append_and_read_of_rows_off_their_alignment(dtype, offset):
    from sandyrt_b200.csrc import ops

    rng = np.random.default_rng(offset)
    hkv, d, ps, n = 2, 48, 16, 37
    lists, table, pages = _tables(rng, [3])
    plain = PlainCache(pages, hkv, ps, d, torch.int8)
    dev = _device_cache(plain)
    k, v = (_values(rng, n, hkv, d, TYPES[dtype]) for _ in range(2))
    wide = torch.zeros(2, n, hkv * d + 5, dtype=TYPES[dtype], device=DEV)
    wide[0, :, offset:offset + hkv * d], wide[1, :, offset:offset + hkv * d] = k.reshape(n, -1).to(DEV), v.reshape(n, -1).to(DEV)
    ops.kv_append_8bit(wide[0, :, offset:offset + hkv * d], wide[1, :, offset:offset + hkv * d], dev, table, _i32([0, n]), _i32([0]), max_q_len=n)
    plain.append(k.double(), v.double(), lists, [0, n], [0])
    _same(dev, plain)
    out = torch.full((2, n, hkv * d + 5), 7.0, dtype=TYPES[dtype], device=DEV)
    ops.kv_read_8bit(dev, table, _i32([0]), _i32([0, n]), out[0, :, offset:offset + hkv * d], out[1, :, offset:offset + hkv * d], max_len=n)
    ops.check_kernel_status(DEV)
    for w in range(2):
        assert torch.equal(out[w, :, offset:offset + hkv * d].cpu().double().reshape(n, hkv, d), plain.values(w, lists[0], n))
        assert bool((out[w, :, :offset] == 7).all()) and bool((out[w, :, offset + hkv * d:] == 7).all())


@pytest.mark.parametrize("code", list(CODES))
def test_append_of_zeros_extremes_and_what_is_not_finite(code):
    """Zeros; the smallest and the largest finite numbers; an infinity or a NaN takes its block (one head, keys or values), for
    good until the page starts anew, and no other."""
    from sandyrt_b200.csrc import ops

    big = torch.finfo(torch.float32).max
    hkv, d, ps = 4, 16, 16
    x = torch.ones(18, hkv, d)
    x[:, 0] = 0.0
    x[:, 1] = 1e-42
    x[3, 1] = 2.0 ** -100
    x[:, 2, ::2] = big
    x[5, 3, 7] = float("inf")
    y = torch.ones(18, hkv, d)
    y[2, 0, 0] = float("nan")
    plain = PlainCache(3, hkv, ps, d, CODES[code])
    dev = _device_cache(plain)
    table = _i32([[2, 0]])

    def step(lo, hi):
        ops.kv_append_8bit(x[lo:hi].reshape(hi - lo, -1).to(DEV), y[lo:hi].reshape(hi - lo, -1).to(DEV), dev, table, _i32([0, hi - lo]), _i32([lo]), max_q_len=hi - lo)

    for lo, hi in ((0, 4), (4, 5), (5, 17), (17, 18)):
        step(lo, hi)
        plain.append(x[lo:hi].double().clamp(-1.875 * 2.0 ** 127, 1.875 * 2.0 ** 127).where(torch.isfinite(x[lo:hi]).double() > 0, x[lo:hi].double()),
                     y[lo:hi].double(), [[2, 0]], [0, hi - lo], [lo])
        _same(dev, plain)
    k, v = torch.zeros(18, hkv * d, device=DEV), torch.zeros(18, hkv * d, device=DEV)
    ops.kv_read_8bit(dev, table, _i32([0]), _i32([0, 18]), k, v, max_len=18)
    k, v = k.cpu().reshape(18, hkv, d), v.cpu().reshape(18, hkv, d)
    assert bool((k[:, 0] == 0).all()) and bool((k[3, 1] == 2.0 ** -100).all()) and bool((k[0, 1] == 0).all())
    assert bool(torch.isfinite(k[:, 2]).all()) and bool((k[:, 2, ::2] >= 0.9 * big).all())
    assert bool(torch.isnan(k[:16, 3]).all()) and bool((k[16:, 3] == 1).all())            # the block, and not the next page
    assert bool(torch.isnan(v[:16, 0]).all()) and bool((v[:, 1:] == 1).all())
    # the page is given to another request: whatever it held is forgotten
    ops.kv_append_8bit(torch.ones(1, hkv * d, device=DEV), torch.ones(1, hkv * d, device=DEV), dev, _i32([[2]]), _i32([0, 1]), _i32([0]), max_q_len=1)
    ops.kv_read_8bit(dev, _i32([[2]]), _i32([0]), _i32([0, 1]), k0 := torch.zeros(1, hkv * d, device=DEV), v0 := torch.zeros(1, hkv * d, device=DEV), max_len=1)
    assert bool((k0 == 1).all()) and bool((v0 == 1).all())
    ops.check_kernel_status(DEV)


def test_pages_that_are_not_there():
    """Positions without a page (none in the table, numbers outside the pool, a table too short, negative positions) and rows outside the
    sources are reported and leave everything as it was; what has a page beside them is served."""
    from sandyrt_b200.csrc import ops
    from sandyrt_b200.errors import KernelError

    rng = np.random.default_rng(5)
    hkv, d, ps = 2, 64, 16
    plain = PlainCache(6, hkv, ps, d, torch.int8)
    k, v = (_values(rng, 80, hkv, d, torch.float32) for _ in range(2))
    kd, vd = k.reshape(80, -1).to(DEV), v.reshape(80, -1).to(DEV)
    dev = _device_cache(plain)
    for table, starts, before in (([[3, -1]], [0, 20], [0]), ([[3, 6]], [0, 20], [0]), ([[3]], [0, 20], [0]), ([[3, 99999]], [0, 20], [0])):
        ops.kv_append_8bit(kd, vd, dev, _i32(table), _i32(starts), _i32(before), max_q_len=20)
        with pytest.raises(KernelError, match="status 8"):
            ops.check_kernel_status(DEV)
        plain.append(k[:16].double(), v[:16].double(), [[3]], [0, 16], [0])
        _same(dev, plain)
    was = _bits(dev)
    for table, starts, before in (([[3, 4]], [70, 90], [0]), ([[3, 4]], [-5, 10], [0]), ([[3, 4]], [0, 3], [-9])):
        ops.kv_append_8bit(kd, vd, dev, _i32(table), _i32(starts), _i32(before), max_q_len=20)
        with pytest.raises(KernelError, match="status 8"):
            ops.check_kernel_status(DEV)
        assert all(torch.equal(a, b) for a, b in zip(was, _bits(dev)))
    out = [torch.full((40, hkv * d), 3.0, device=DEV) for _ in range(2)]
    for table, first, starts, good in (([[3, -1]], [0], [2, 22], slice(2, 18)), ([[-1, 3]], [8], [0, 12], slice(8, 8)), ([[3]], [-4], [0, 8], slice(4, 8)),
                                       ([[3]], [0], [30, 44], slice(0, 0))):
        for o in out:
            o.fill_(3.0)
        ops.kv_read_8bit(dev, _i32(table), _i32(first), _i32(starts), out[0], out[1], max_len=20)
        with pytest.raises(KernelError, match="status 16"):
            ops.check_kernel_status(DEV)
        for w, o in enumerate(out):
            rest = torch.ones(40, dtype=torch.bool)
            rest[good] = False
            if table == [[-1, 3]]:
                rest[8:12] = False
            assert bool((o.cpu()[rest] == 3).all())
            if good.stop > good.start:
                lo = 0
                assert torch.equal(o.cpu()[good].double().reshape(-1, hkv, d), plain.values(w, [3], 16)[lo:good.stop - good.start])
    # attention: a visible key without a page is left out
    q = torch.randn(1, 4 * d, device=DEV)
    got, want = torch.empty_like(q), torch.empty_like(q)
    ops.decode_attention_8bit(q, dev, _i32([[3, -1]]), _i32([0]), _i32([19]), got, n_heads=4, scale=0.1)
    with pytest.raises(KernelError, match="status 16"):
        ops.check_kernel_status(DEV)
    ops.decode_attention_8bit(q, dev, _i32([[3, -1]]), _i32([0]), _i32([15]), want, n_heads=4, scale=0.1)
    ops.check_kernel_status(DEV)
    assert torch.equal(got, want)
    for seq in (1, -1, 1 << 30):                                  # a token of no request: zeros
        ops.decode_attention_8bit(q, dev, _i32([[3, -1]]), _i32([seq]), _i32([3]), got, n_heads=4, scale=0.1)
        with pytest.raises(KernelError, match="status 16"):
            ops.check_kernel_status(DEV)
        assert bool((got == 0).all())


# ---- attention --------------------------------------------------------------------------------------------------
def _tolerance(dtype, want, v):
    """bfloat16: the result's rounding (2^-8 of it), P's to half precision (2^-11 of the largest value); float32: q and P in two
    half-precision pieces, sums of up to 256 products and of scores up to some 16, the exponential: below 2e-5 of the largest
    value.  1e-4 of it covers what the two share in bfloat16."""
    top = float(v.abs().max())
    return want.abs() * 2.0 ** -8 + top * (2.0 ** -11 + 1e-4) if dtype == torch.bfloat16 else torch.full_like(want, top * 2e-5)


def _filled(rng, code, hkv, d, ps, totals):
    """A plain cache with so many positions of each request written, and the requests' page lists and table."""
    lists, table, pages = _tables(rng, [max(1, -(-n // ps)) for n in totals])
    plain = PlainCache(pages, hkv, ps, d, CODES[code])
    n = sum(totals)
    k, v = (_values(rng, n, hkv, d, torch.float64) * torch.from_numpy(np.exp(0.8 * rng.standard_normal((1, hkv, d)))) for _ in range(2))
    plain.append(k, v, lists, _starts(totals), [0] * len(totals))
    return plain, lists, table


def _rules_on_host(rules):
    return {k: v.double().cpu() if isinstance(v, torch.Tensor) else v for k, v in rules.items()}


def _check_attention(code, dtype, H, hkv, d, ps, seqs, decode, seed=0, splits=0, q_scale=1.0, more=0.0, tc=None, **rules):
    """seqs: (positions in the cache before, new tokens) of each request; single tokens go to requests in another order."""
    from sandyrt_b200.csrc import ops

    rng = np.random.default_rng(seed * 1000 + H * 7 + d + ps)
    dtype = TYPES[dtype]
    plain, lists, table = _filled(rng, code, hkv, d, ps, [b + n for b, n in seqs])
    dev = _device_cache(plain)
    lens = [n for _, n in seqs]
    starts = _starts(lens, 0 if decode else 1)
    n = starts[-1] + (0 if decode else 2)
    q = torch.from_numpy(rng.standard_normal((n, H * d + 24)) * q_scale).to(dtype).to(DEV)[:, 8:8 + H * d]
    if "elem_gate" in rules:
        rules["elem_gate"] = torch.from_numpy(rng.standard_normal((n, H * rules["elem_gate"] + 3))).to(dtype).to(DEV)[:, :H * rules["elem_gate"]]
    for name, shape in (("sink", (H,)), ("out_gate", (n, H)), ("dist_bias", (H, 29))):
        if name in rules:
            rules[name] = torch.from_numpy(rng.standard_normal(shape)).float().to(DEV)
    out = torch.full((n, H * d + 8), 5.0, dtype=dtype, device=DEV)
    scale = 1.0 / math.sqrt(d)
    if decode:
        order = rng.permutation(len(seqs)).tolist()
        ops.decode_attention_8bit(q, dev, table, _i32(order), _i32([seqs[s][0] for s in order]), out[:, :H * d], n_heads=H, scale=scale,
                                  num_splits=splits, **rules)
        rows = [(s, [t], [seqs[s][0]]) for t, s in enumerate(order)]
    else:
        ops.prefill_attention_8bit(q, dev, table, _i32(starts), _i32([b for b, _ in seqs]), out[:, :H * d], n_heads=H, max_q_len=max(lens),
                                   scale=scale, num_splits=splits, tc=tc, **rules)
        rows = [(s, list(range(starts[s], starts[s + 1])), list(range(b, b + m))) for s, (b, m) in enumerate(seqs)]
    ops.check_kernel_status(DEV)
    got = out.cpu().double()
    assert bool((got[:, H * d:] == 5).all())
    if not decode:
        assert bool((got[0] == 5).all()) and bool((got[-2:] == 5).all())          # rows of no request
    host = _rules_on_host(rules)
    for s, at, pos in rows:
        if not at:
            continue
        total = seqs[s][0] + seqs[s][1]
        k, v = (plain.values(w, lists[s], total) for w in range(2))
        per_row = {n: host[n][at] for n in ("out_gate", "elem_gate") if n in host}
        want = attention(q[at].double().cpu().reshape(len(at), H, d), k, v, pos, scale=scale, **{**host, **per_row}).reshape(len(at), -1)
        assert bool(((got[at, :H * d] - want).abs() <= _tolerance(dtype, want, v) + more * float(v.abs().max())).all()), float((got[at, :H * d] - want).abs().max())


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("code", list(CODES))
@pytest.mark.parametrize("H,hkv,d,ps", [(4, 4, 64, 16), (12, 2, 64, 8), (2, 1, 16, 16), (8, 1, 128, 16), (3, 3, 48, 5), (16, 1, 96, 32), (10, 2, 256, 16),
                                        (6, 2, 80, 64), (25, 1, 32, 16)])
def test_single_tokens(code, dtype, H, hkv, d, ps):
    _check_attention(code, dtype, H, hkv, d, ps, [(0, 1), (1, 1), (15, 1), (16, 1), (63, 1), (130, 1), (257, 1), (700, 1)], True)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("code", list(CODES))
@pytest.mark.parametrize("hkv,group,rules", [(25, 1, {}), (25, 4, dict(window=20, keep_first=3, sink=True))])
def test_single_tokens_of_very_many_requests(code, dtype, hkv, group, rules):
    """Thousands of (token, key/value head) pairs: blocks of two warps."""
    _check_attention(code, dtype, hkv * group, hkv, 64, 16, [((7 * i) % 90 if i % 9 else 0, 1) for i in range(100)], True, **rules)


@pytest.mark.parametrize("splits", [1, 2, 3, 7, 16, 40])
def test_single_tokens_in_so_many_splits(splits):
    _check_attention("e4m3", "bf16", 6, 2, 64, 16, [(0, 1), (300, 1), (511, 1), (640, 1)], True, splits=splits)
    _check_attention("int8", "f32", 4, 4, 128, 8, [(0, 1), (333, 1)], True, splits=splits, window=100, keep_first=9, sink=True)


RULES = [dict(window=1), dict(window=20), dict(window=33, keep_first=5), dict(window=40, keep_first=50, sink=True), dict(softcap=2.0), dict(chunk=24), dict(sink=True),
         dict(out_gate=True, elem_gate=11), dict(dist_bias=True), dict(window=50, softcap=3.0, dist_bias=True, sink=True, out_gate=True, elem_gate=16)]


@pytest.mark.parametrize("rules", RULES, ids=lambda r: "-".join(r))
@pytest.mark.parametrize("decode", [True, False])
@pytest.mark.parametrize("code,dtype,H,hkv,d,ps", [("e4m3", "bf16", 4, 2, 64, 16), ("int8", "f32", 6, 2, 48, 8)])
def test_rules(code, dtype, H, hkv, d, ps, decode, rules):
    seqs = [(0, 1), (70, 1), (200, 1), (47, 1)] if decode else [(0, 40), (90, 1), (0, 0), (33, 70)]
    _check_attention(code, dtype, H, hkv, d, ps, seqs, decode, **dict(rules))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("code", list(CODES))
@pytest.mark.parametrize("H,hkv,d,ps", [(3, 3, 64, 16), (4, 1, 64, 8), (4, 2, 128, 16), (2, 2, 16, 16), (6, 3, 96, 32), (2, 1, 256, 16), (5, 1, 80, 5), (2, 2, 128, 256)])
def test_prompt_portions(code, dtype, H, hkv, d, ps):
    _check_attention(code, dtype, H, hkv, d, ps, [(0, 1), (0, 130), (100, 33), (3, 0), (127, 2), (250, 17)], False)
    _check_attention(code, dtype, H, hkv, d, ps, [(300, 140)], False, seed=1)


@pytest.mark.parametrize("code", list(CODES))
@pytest.mark.parametrize("H,hkv,d,ps", [(2, 2, 64, 16), (2, 2, 128, 32), (12, 3, 64, 48), (8, 1, 128, 16), (3, 1, 64, 256)])
@pytest.mark.parametrize("seqs", [[(0, 1)], [(0, 128)], [(0, 129), (5, 0), (511, 2)], [(0, 300), (130, 40)], [(400, 257)], [(1000, 8), (0, 8)]])
def test_prompt_portions_on_tcgen05(code, H, hkv, d, ps, seqs):
    _check_attention(code, "bf16", H, hkv, d, ps, seqs, False, tc=True)


@pytest.mark.parametrize("code", list(CODES))
@pytest.mark.parametrize("splits", [1, 2, 4, 8])
@pytest.mark.parametrize("H,hkv,d,ps", [(2, 2, 64, 16), (8, 2, 128, 32)])
@pytest.mark.parametrize("seqs,rules", [([(0, 1), (0, 128), (0, 3)], {}), ([(0, 300), (700, 140), (3, 0), (1500, 1)], {}), ([(0, 1000)], {}),
                                        ([(900, 200), (5, 60)], dict(window=200, keep_first=3, sink=True)), ([(400, 260)], dict(chunk=96, out_gate=True, elem_gate=8))])
def test_prompt_portions_on_tcgen05_in_so_many_splits(code, splits, H, hkv, d, ps, seqs, rules):
    _check_attention(code, "bf16", H, hkv, d, ps, seqs, False, splits=splits, tc=True, **rules)


@pytest.mark.parametrize("code", list(CODES))
@pytest.mark.parametrize("splits", [0, 1, 4, 8])
@pytest.mark.parametrize("H,hkv,d,ps", [(3, 3, 16, 16), (6, 2, 32, 16), (8, 2, 48, 32), (4, 4, 80, 16), (5, 1, 96, 16), (2, 2, 112, 48)])
def test_prompt_portions_on_tcgen05_of_other_head_sizes(code, splits, H, hkv, d, ps):
    """The last page of the cache is used, whose rows' ends are the memory's."""
    _check_attention(code, "bf16", H, hkv, d, ps, [(0, 300), (130, 40), (0, 1)], False, splits=splits, tc=True)
    _check_attention(code, "bf16", H, hkv, d, ps, [(700, 90)], False, splits=splits, tc=True, window=100, keep_first=5, sink=True, elem_gate=11)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rules", [r for r in RULES if "dist_bias" not in r], ids=lambda r: "-".join(r))
def test_rules_on_tcgen05(d, rules):
    _check_attention("e4m3", "bf16", 4, 2, d, 16, [(0, 150), (290, 1), (0, 0), (333, 170)], False, tc=True, **dict(rules))


def test_calls_the_tcgen05_kernel_does_not_take():
    from sandyrt_b200.errors import UnsupportedShape

    for H, hkv, d, ps, dtype, rules in ((2, 2, 64, 8, "bf16", {}), (2, 2, 256, 16, "bf16", {}), (2, 2, 64, 16, "bf16", dict(dist_bias=True))):
        with pytest.raises(UnsupportedShape):
            _check_attention("int8", dtype, H, hkv, d, ps, [(0, 70)], False, tc=True, **rules)
    with pytest.raises(UnsupportedShape):
        _check_attention("int8", "f32", 2, 2, 64, 16, [(0, 70)], False, tc=True)


@pytest.mark.parametrize("splits", [1, 2, 5])
def test_prompt_portions_in_so_many_splits(splits):
    _check_attention("int8", "bf16", 4, 2, 64, 16, [(0, 20), (301, 40)], False, splits=splits)
    _check_attention("e4m3", "f32", 2, 1, 128, 16, [(260, 19)], False, splits=splits)


@pytest.mark.parametrize("code", list(CODES))
@pytest.mark.parametrize("decode", [True, False])
@pytest.mark.parametrize("dtype,q_scale", [("bf16", 60.0), ("f32", 60.0), ("bf16", 1e-20), ("f32", 1e-20), ("bf16", 0.0)])
def test_large_and_small_queries(code, dtype, decode, q_scale):
    """Scores of some hundreds: a softmax of one key.  float32's tolerance grows with the scores (their rounding): q_scale 60 gives
    scores of up to some 2,000, 2^-24 * 2000 = 1.2e-4 each, several times."""
    _check_attention(code, dtype, 4, 2, 64, 16, [(0, 1), (100, 1), (400, 1)] if decode else [(0, 50), (100, 33)], decode, q_scale=q_scale,
                     more=2e-3 if q_scale == 60.0 else 0.0)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("decode", [True, False])
def test_values_of_blocks_far_apart_in_size(dtype, decode):
    """Blocks whose values differ by 2^40, the large ones under scores that all but hide them, and the other way round."""
    from sandyrt_b200.csrc import ops

    hkv, d, ps, n = 1, 64, 16, 64
    rng = np.random.default_rng(2)
    plain = PlainCache(4, hkv, ps, d, torch.int8)
    k, v = _values(rng, n, hkv, d, torch.float64), _values(rng, n, hkv, d, torch.float64)
    v[16:32] *= 2.0 ** 40
    v[48:] *= 2.0 ** -30
    k[16:32] = 0.0
    k[16:32, :, 0] = -60.0                                       # with q's first element 8 and scale 1/8: 60 below the others
    plain.append(k, v, [[0, 1, 2, 3]], [0, n], [0])
    dev = _device_cache(plain)
    q = torch.from_numpy(rng.standard_normal((2, d))).to(TYPES[dtype])
    q[:, 0] = 8.0
    out = torch.empty(2, d, dtype=TYPES[dtype], device=DEV)
    table, pos = _i32([[0, 1, 2, 3]]), [47, 63]
    if decode:
        ops.decode_attention_8bit(q.to(DEV), dev, table, _i32([0, 0]), _i32(pos), out, n_heads=1, scale=0.125)
    else:
        for i, p in enumerate(pos):
            ops.prefill_attention_8bit(q[i:i + 1].to(DEV), dev, table, _i32([0, 1]), _i32([p]), out[i:i + 1], n_heads=1, max_q_len=1, scale=0.125)
    ops.check_kernel_status(DEV)
    kk, vv = (plain.values(w, [0, 1, 2, 3], n) for w in range(2))
    for i, p in enumerate(pos):
        s = kk[:p + 1, 0] @ q[i].double() * 0.125
        w = torch.softmax(s, 0)
        want = w @ vv[:p + 1, 0]
        # as a weighted sum: every term off by 2^-11 of itself (bfloat16) or a few 2^-22 and the scores' rounding (float32)
        far = (w[:, None] * vv[:p + 1, 0].abs()).sum(0)
        tol = want.abs() * 2.0 ** -8 + far * (2.0 ** -10) if dtype == "bf16" else far * 3e-5
        # P is a half-precision number beside its largest term: what is 2^-25 below that is gone
        tol = tol + (w[:, None] * vv[:p + 1, 0].abs().amax(1, keepdim=True)).max() * 2.0 ** -18
        assert bool(((out[i].cpu().double() - want).abs() <= tol).all())


@pytest.mark.parametrize("path", ["decode", "prompt", "tcgen05"])
@pytest.mark.parametrize("code", list(CODES))
@pytest.mark.parametrize("kind", ["any numbers", "zeros", "zeros beside large ones"])
def test_scales_that_are_no_power_of_two(code, path, kind):
    """Scales as another program might have them: any numbers, zero for a block of zeros.  And blocks of zeros (2^-100 by appending) beside
    values of 2^50, whose weights must not be missing in the denominator."""
    from sandyrt_b200.csrc import ops

    rng = np.random.default_rng(17)
    hkv, d, ps, H, n = 2, 64, 16, 4, 150
    lists, table, pages = _tables(rng, [-(-n // ps)])
    plain = PlainCache(pages, hkv, ps, d, CODES[code])
    k, v = (_values(rng, n, hkv, d, torch.float64) for _ in range(2))
    if kind != "any numbers":
        k[32:48], v[64:80], v[96:112] = 0.0, 0.0, 0.0
    if kind == "zeros beside large ones":
        v[16:32] *= 2.0 ** 50
        k[16:32] = 0.0
        k[16:32, :, 0] = -20.0                                   # 20 below the others: a weight of e^-20 on values of 2^50
    plain.append(k, v, lists, [0, n], [0])
    if kind != "zeros beside large ones":
        for w in range(2):
            plain.scales[w] = (plain.scales[w] * torch.from_numpy(rng.uniform(0.6, 1.7, plain.scales[w].shape))).float().double()
            plain.scales[w] = torch.where(plain.scales[w] < 2.0 ** -90, torch.zeros(()).double(), plain.scales[w])
    dev = _device_cache(plain)
    q = torch.from_numpy(rng.standard_normal((n, H, d)))
    q[:, :, 0] = 8.0
    q = q.to(torch.bfloat16).reshape(n, -1)
    out = torch.empty(n, H * d, dtype=torch.bfloat16, device=DEV)
    if path == "decode":
        ops.decode_attention_8bit(q.to(DEV), dev, table, _i32([0] * n), _i32(list(range(n))), out, n_heads=H, scale=0.125)
    else:
        ops.prefill_attention_8bit(q.to(DEV), dev, table, _i32([0, n]), _i32([0]), out, n_heads=H, max_q_len=n, scale=0.125, tc=path == "tcgen05")
    ops.check_kernel_status(DEV)
    kk, vv = (plain.values(w, lists[0], n) for w in range(2))
    qq = q.double().reshape(n, H, d)
    want = attention(qq, kk, vv, list(range(n)), scale=0.125)
    # a sum of terms, each off by 2^-11 twice (the weight, and a value times what its scale is beside a power of two); weights below 2^-25
    # of the largest term are gone
    far = attention(qq, kk, vv.abs(), list(range(n)), scale=0.125)
    tol = want.abs() * 2.0 ** -8 + far * 2.0 ** -9 + far.amax(dim=2, keepdim=True) * 2.0 ** -16
    assert bool(((out.cpu().double().reshape(n, H, d) - want).abs() <= tol).all())


def test_positions_behind_the_block_table():
    """Far behind: reported, and nothing is walked for them.  A longest portion that was said too short is reported too."""
    from sandyrt_b200.csrc import ops
    from sandyrt_b200.errors import KernelError

    rng = np.random.default_rng(3)
    hkv, d, ps, H = 2, 64, 16, 4
    plain, lists, table = _filled(rng, "e4m3", hkv, d, ps, [64])
    dev = _device_cache(plain)
    q = torch.randn(4, H * d, device=DEV)
    want, got = torch.empty_like(q), torch.empty_like(q)
    ops.decode_attention_8bit(q, dev, table, _i32([0] * 4), _i32([63] * 4), want, n_heads=H, scale=0.1)
    ops.check_kernel_status(DEV)
    ops.decode_attention_8bit(q, dev, table, _i32([0] * 4), _i32([64, 1000, 2 ** 31 - 17, 2 ** 30]), got, n_heads=H, scale=0.1)
    with pytest.raises(KernelError, match="status 16"):
        ops.check_kernel_status(DEV)
    assert torch.equal(got, want)
    for rules in (dict(window=30), dict(window=30, keep_first=2 ** 30), dict(window=30, keep_first=40)):
        ops.decode_attention_8bit(q, dev, table, _i32([0] * 4), _i32([2 ** 31 - 17] * 4), got, n_heads=H, scale=0.1, **rules)
        with pytest.raises(KernelError, match="status 16"):
            ops.check_kernel_status(DEV)
        assert bool((got == 0).all()) if "keep_first" not in rules else bool(torch.isfinite(got).all())
    b = q.to(torch.bfloat16)
    for tc in (True, False):
        outs = []
        for before in (60, 2 ** 31 - 40):                        # rows at 60..63, and far behind
            o = torch.full_like(b, 3.0)
            ops.prefill_attention_8bit(b, dev, table, _i32([0, 4]), _i32([before]), o, n_heads=H, max_q_len=4, scale=0.1, tc=tc)
            if before > 60:
                with pytest.raises(KernelError, match="status 16"):
                    ops.check_kernel_status(DEV)
            ops.check_kernel_status(DEV)
            outs.append(o)
        assert bool(torch.isfinite(outs[0]).all()) and bool(torch.isfinite(outs[1]).all())
        o = torch.full_like(b, 3.0)
        ops.prefill_attention_8bit(b, dev, table, _i32([0, 4]), _i32([60]), o, n_heads=H, max_q_len=3, scale=0.1, tc=tc)
        with pytest.raises(KernelError, match="status 16"):
            ops.check_kernel_status(DEV)
        assert bool((o == 3).all())
    was = _bits(dev)
    rows = torch.randn(4, hkv * d, device=DEV)
    ops.kv_append_8bit(rows, rows, dev, table, _i32([0, 4]), _i32([0]), max_q_len=3)
    with pytest.raises(KernelError, match="status 8"):
        ops.check_kernel_status(DEV)
    assert all(torch.equal(a, c) for a, c in zip(was, _bits(dev)))
    k, v = torch.full_like(rows, 3.0), torch.full_like(rows, 3.0)
    ops.kv_read_8bit(dev, table, _i32([0]), _i32([0, 4]), k, v, max_len=3)
    with pytest.raises(KernelError, match="status 16"):
        ops.check_kernel_status(DEV)
    assert bool((k == 3).all()) and bool((v == 3).all())


def test_appending_at_the_last_positions_there_are():
    """Positions up to and past 2^31: no page, reported, nothing written."""
    from sandyrt_b200.csrc import ops
    from sandyrt_b200.errors import KernelError

    for ps in (16, 5):
        plain, lists, table = _filled(np.random.default_rng(4), "int8", 2, 64, ps, [20])
        dev = _device_cache(plain)
        was, rows = _bits(dev), torch.randn(4, 128, device=DEV)
        for before in (2 ** 31 - 1, 2 ** 31 - 3, 2 ** 31 - 20, 2 ** 31 - 200, -1, -2 ** 31):
            ops.kv_append_8bit(rows, rows, dev, table, _i32([0, 4]), _i32([before]), max_q_len=4)
            with pytest.raises(KernelError, match="status 8"):
                ops.check_kernel_status(DEV)
            if before != -1:                                         # its second row would be position 0
                out = torch.full_like(rows, 3.0)
                ops.kv_read_8bit(dev, table, _i32([before]), _i32([0, 2]), out, out.clone(), max_len=2)
                with pytest.raises(KernelError, match="status 16"):
                    ops.check_kernel_status(DEV)
                assert bool((out == 3).all())
        with pytest.raises(KernelError, match="32-bit"):
            ops.kv_append_8bit(rows, rows, dev, table, _i32([0, 4]), _i32([0]), max_q_len=2 ** 31)
        ops.check_kernel_status(DEV)
        assert all(torch.equal(x, y) for x, y in zip(was, _bits(dev)))


@pytest.mark.parametrize("code", list(CODES))
@pytest.mark.parametrize("decode", [True, False])
def test_blocks_that_are_not_finite(code, decode):
    """A block with a scale of NaN gives NaN to the rows that see it, and to no other."""
    from sandyrt_b200.csrc import ops

    rng = np.random.default_rng(9)
    hkv, d, ps, H = 2, 64, 16, 4
    plain, lists, table = _filled(rng, code, hkv, d, ps, [90])
    plain.scales[0][lists[0][2], 0] = float("nan")               # keys 32..47 of head 0
    plain.scales[1][lists[0][4], 1] = float("nan")               # values 64..79 of head 1
    dev = _device_cache(plain)
    pos = list(range(20, 90))
    q = torch.from_numpy(rng.standard_normal((len(pos), H * d))).to(torch.bfloat16).to(DEV)
    out = torch.empty_like(q)
    if decode:
        ops.decode_attention_8bit(q, dev, table, _i32([0] * len(pos)), _i32(pos), out, n_heads=H, scale=0.1, window=30)
    else:
        ops.prefill_attention_8bit(q, dev, table, _i32([0, len(pos)]), _i32([20]), out, n_heads=H, max_q_len=len(pos), scale=0.1, window=30)
    ops.check_kernel_status(DEV)
    bad = torch.isnan(out.cpu().reshape(len(pos), H, d))
    for i, p in enumerate(pos):
        sees = [32 <= p and p - 29 <= 47, 64 <= p and p - 29 <= 79]
        for h in range(H):
            assert bool(bad[i, h].all()) == sees[h // 2] and bool(bad[i, h].any()) == sees[h // 2], (p, h)


def test_padded_tokens_and_empty_calls():
    from sandyrt_b200.csrc import ops

    rng = np.random.default_rng(4)
    plain, lists, table = _filled(rng, "e4m3", 2, 64, 16, [40])
    dev = _device_cache(plain)
    q = torch.randn(3, 256, device=DEV)
    out = torch.full_like(q, float("nan"))
    ops.decode_attention_8bit(q, dev, table, _i32([0, 0, 0]), _i32([-1, 39, -7]), out, n_heads=4, scale=0.1, sink=torch.zeros(4, device=DEV))
    ops.check_kernel_status(DEV)
    assert bool((out[[0, 2]] == 0).all()) and bool(torch.isfinite(out[1]).all())
    none = torch.empty(0, 256, device=DEV)
    ops.decode_attention_8bit(none, dev, table, _i32([]), _i32([]), none.clone(), n_heads=4, scale=0.1)
    ops.prefill_attention_8bit(q, dev, table, _i32([0, 0]), _i32([0]), out, n_heads=4, max_q_len=0, scale=0.1)
    ops.prefill_attention_8bit(q, dev, table, _i32([1, 1]), _i32([0]), was := out.clone(), n_heads=4, max_q_len=5, scale=0.1)
    assert torch.equal(was, out)
    ops.kv_append_8bit(none[:, :128], none[:, :128], dev, table, _i32([0, 0]), _i32([0]), max_q_len=0)
    ops.check_kernel_status(DEV)


def test_heads_of_a_page_past_32_bits():
    """Codes that lie more than 2^32 bytes behind the cache's start."""
    from sandyrt_b200.csrc import ops

    hkv, d, ps = 8, 128, 16
    page = hkv * d * ps
    pages = (1 << 32) // page + 10
    codes = [torch.empty(pages, hkv, ps, d, dtype=torch.int8, device=DEV) for _ in range(2)]
    scales = [torch.empty(pages, hkv, device=DEV) for _ in range(2)]
    dev = ops.Cache8(*codes, *scales)
    rng = np.random.default_rng(6)
    lists = [[pages - 1, 3, pages - 4]]
    small = PlainCache(3, hkv, ps, d, torch.int8)
    k, v = (_values(rng, 40, hkv, d, torch.bfloat16) for _ in range(2))
    ops.kv_append_8bit(k.reshape(40, -1).to(DEV), v.reshape(40, -1).to(DEV), dev, _i32(lists), _i32([0, 40]), _i32([0]), max_q_len=40)
    small.append(k.double(), v.double(), [[0, 1, 2]], [0, 40], [0])
    out = [torch.empty(40, hkv * d, device=DEV) for _ in range(2)]
    ops.kv_read_8bit(dev, _i32(lists), _i32([0]), _i32([0, 40]), *out, max_len=40)
    for w in range(2):
        assert torch.equal(out[w].cpu().double().reshape(40, hkv, d), small.values(w, [0, 1, 2], 40))
    q = torch.from_numpy(rng.standard_normal((40, 8 * d))).to(torch.bfloat16)
    got = torch.empty(40, 8 * d, dtype=torch.bfloat16, device=DEV)
    want = attention(q.double().reshape(40, 8, d), small.values(0, [0, 1, 2], 40), small.values(1, [0, 1, 2], 40), list(range(40)), scale=0.09).reshape(40, -1)
    ops.prefill_attention_8bit(q.to(DEV), dev, _i32(lists), _i32([0, 40]), _i32([0]), got, n_heads=8, max_q_len=40, scale=0.09)
    assert bool(((got.cpu().double() - want).abs() <= _tolerance(torch.bfloat16, want, small.values(1, [0, 1, 2], 40))).all())
    ops.decode_attention_8bit(q[39:].to(DEV), dev, _i32(lists), _i32([0]), _i32([39]), got[39:], n_heads=8, scale=0.09)
    assert bool(((got[39:].cpu().double() - want[39:]).abs() <= _tolerance(torch.bfloat16, want, small.values(1, [0, 1, 2], 40))[39:]).all())
    ops.check_kernel_status(DEV)


def test_pages_of_keys_and_values_in_one_arena():
    """Keys and values of a page side by side, as the engine's arenas have them: a page pitch of its own."""
    from sandyrt_b200.csrc import ops

    rng = np.random.default_rng(8)
    hkv, d, ps = 2, 64, 16
    lists, table, pages = _tables(rng, [4])
    arena = torch.zeros(pages, 2, hkv, ps, d, dtype=torch.int8, device=DEV)
    scales = torch.zeros(pages, 2, hkv, device=DEV)
    dev = ops.Cache8(arena[:, 0], arena[:, 1], scales[:, 0], scales[:, 1])
    plain = PlainCache(pages, hkv, ps, d, torch.int8)
    k, v = (_values(rng, 60, hkv, d, torch.bfloat16) for _ in range(2))
    ops.kv_append_8bit(k.reshape(60, -1).to(DEV), v.reshape(60, -1).to(DEV), dev, table, _i32([0, 60]), _i32([0]), max_q_len=60)
    plain.append(k.double(), v.double(), lists, [0, 60], [0])
    plain.scales = [torch.where(torch.isnan(s), torch.zeros(()).double(), s) for s in plain.scales]
    _same(dev, plain)
    q = torch.from_numpy(rng.standard_normal((60, 4 * d))).to(torch.bfloat16)
    out = torch.empty(60, 4 * d, dtype=torch.bfloat16, device=DEV)
    ops.prefill_attention_8bit(q.to(DEV), dev, table, _i32([0, 60]), _i32([0]), out, n_heads=4, max_q_len=60, scale=0.12)
    ops.check_kernel_status(DEV)
    want = attention(q.double().reshape(60, 4, d), plain.values(0, lists[0], 60), plain.values(1, lists[0], 60), list(range(60)), scale=0.12).reshape(60, -1)
    assert bool(((out.cpu().double() - want).abs() <= _tolerance(torch.bfloat16, want, plain.values(1, lists[0], 60))).all())


# ---- together -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("code", list(CODES))
def test_a_prompt_and_its_tokens_in_a_recorded_step(code):
    """Two prompts, then decode steps as a recorded graph on a stream of its own: append, attention, log-probabilities of a step, with
    positions moved on between replays; blocks grow on the way.  Each step is held against the formula on what the cache holds
    by the formula."""
    from sandyrt_b200.csrc import ops

    rng = np.random.default_rng(12)
    H, hkv, d, ps, vocab, top, steps = 4, 2, 64, 16, 777, 5, 20
    lens = [37, 15]
    lists, table, pages = _tables(rng, [-(-(n + steps) // ps) for n in lens])
    plain = PlainCache(pages, hkv, ps, d, CODES[code])
    dev = _device_cache(plain)
    draw = lambda n, grow=1.0: [_values(rng, n, hkv, d, torch.bfloat16, grow) for _ in range(2)]
    k, v = draw(sum(lens))
    ops.kv_append_8bit(k.reshape(-1, hkv * d).to(DEV), v.reshape(-1, hkv * d).to(DEV), dev, table, _i32(_starts(lens)), _i32([0, 0]), max_q_len=max(lens))
    plain.append(k.double(), v.double(), lists, _starts(lens), [0, 0])
    out = torch.empty(sum(lens), H * d, dtype=torch.bfloat16, device=DEV)
    q = torch.from_numpy(rng.standard_normal((sum(lens), H * d))).to(torch.bfloat16)
    ops.prefill_attention_8bit(q.to(DEV), dev, table, _i32(_starts(lens)), _i32([0, 0]), out, n_heads=H, max_q_len=max(lens), scale=0.125)
    at = 0
    for s, n in enumerate(lens):
        kk, vv = (plain.values(w, lists[s], n) for w in range(2))
        want = attention(q[at:at + n].double().reshape(n, H, d), kk, vv, list(range(n)), scale=0.125).reshape(n, -1)
        assert bool(((out[at:at + n].cpu().double() - want).abs() <= _tolerance(torch.bfloat16, want, vv)).all())
        at += n
    # the step's buffers
    kd, vd = (torch.zeros(2, hkv * d, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    qd, od = (torch.zeros(2, H * d, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    head = torch.from_numpy(rng.standard_normal((H * d, vocab)) * 0.2).float().to(DEV)
    logits, ids = torch.zeros(2, vocab, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV)
    lp, ent = torch.zeros(2, device=DEV), torch.zeros(2, device=DEV)
    ti, tl = torch.zeros(2, top, dtype=torch.int32, device=DEV), torch.zeros(2, top, device=DEV)
    pos, starts, seq = _i32(lens), _i32([0, 1, 2]), _i32([0, 1])

    def step():
        ops.kv_append_8bit(kd, vd, dev, table, starts, pos, max_q_len=1)
        ops.decode_attention_8bit(qd, dev, table, seq, pos, od, n_heads=H, scale=0.125, num_splits=2)
        torch.mm(od.float(), head, out=logits)
        ops.token_logprobs(logits, ids, lp, entropy=ent, top_ids=ti, top_logprobs=tl)
        pos.add_(1)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    held = _bits(dev)
    with torch.cuda.stream(stream):
        torch.mm(od.float(), head, out=logits)                    # the library's workspace before the recording
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
    assert all(torch.equal(a, b) for a, b in zip(held, _bits(dev)))          # recording runs nothing
    have = list(lens)
    for i in range(steps):
        k, v = draw(2, 1.3 ** i)
        q = torch.from_numpy(rng.standard_normal((2, H * d))).to(torch.bfloat16)
        with torch.cuda.stream(stream):
            kd.copy_(k.reshape(2, -1)); vd.copy_(v.reshape(2, -1)); qd.copy_(q)
            ids.copy_(torch.tensor([i, vocab - 1 - i], dtype=torch.int32))
            graph.replay()
        stream.synchronize()
        plain.append(k.double(), v.double(), lists, [0, 1, 2], have)
        for s in range(2):
            kk, vv = (plain.values(w, lists[s], have[s] + 1) for w in range(2))
            want = attention(q[s:s + 1].double().reshape(1, H, d), kk, vv, [have[s]], scale=0.125).reshape(-1)
            assert bool(((od[s].cpu().double() - want).abs() <= _tolerance(torch.bfloat16, want, vv)).all())
        _check_logprobs(logits, ids.tolist(), top, lp, ent, ti, tl)
        have = [h + 1 for h in have]
    _same(dev, plain)
    ops.check_kernel_status(DEV)


# ---- log-probabilities ----------------------------------------------------------------------------------------------
def _check_logprobs(x, ids, top, lp, ent, ti, tl):
    """Sums of `vocab` positive terms by threads' 16s and a tree (below 64 additions in a row: 2^-18 of the sum, 4e-6), exponentials
    off by 2^-22 and by their argument's rounding (2^-24 of up to 50), differences and logarithms rounded at values up to some
    50: 1e-5 and 1e-6 of the value."""
    x = x.double().cpu()
    want, want_ent, order, want_top = logprobs(x, ids, top)
    tol = lambda w: 1e-5 + 1e-6 * np.abs(np.where(np.isfinite(w), w, 0.0))
    for got, w in ((lp, want), (ent, want_ent), (tl, want_top)):
        got = got.double().cpu().numpy()
        fine = np.isfinite(w)
        assert np.array_equal(fine, np.isfinite(got)) and np.array_equal(got[~fine], w[~fine])
        off = np.abs(got[fine] - w[fine])
        assert (off <= tol(w)[fine]).all(), float(off.max())
    assert np.array_equal(ti.cpu().numpy(), order)


def _run_logprobs(x, ids, top):
    from sandyrt_b200.csrc import ops

    n = x.shape[0]
    nan = lambda *shape: torch.full(shape, float("nan"), device=DEV)
    lp, ent, tl = nan(n), nan(n), nan(n, top)
    ti = torch.full((n, top), -9, dtype=torch.int32, device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.token_logprobs(x, _i32(ids), lp, entropy=ent, top_ids=ti, top_logprobs=tl, status=status)
    return lp, ent, ti, tl, int(status.item())


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n,vocab,top", [(1, 1, 1), (2, 2, 2), (3, 5, 4), (7, 33, 32), (4, 777, 20), (700, 512, 5), (3, 4097, 32), (1, 8192, 8), (8, 50257, 5), (40, 50257, 32),
                                         (600, 9001, 20), (2, 128256, 1)])
def test_logprobs(dtype, n, vocab, top):
    """Rows at every alignment (a pitch of odd numbers), bfloat16 with its many ties."""
    g = torch.Generator().manual_seed(n + vocab)
    x = (torch.randn(n, vocab + 3, generator=g) * torch.rand(n, 1, generator=g) * 5 - 20).to(TYPES[dtype]).to(DEV)[:, 1:1 + vocab]
    ids = torch.randint(0, vocab, (n,), generator=g).tolist()
    ids[n // 2] = -1
    lp, ent, ti, tl, status = _run_logprobs(x, ids, top)
    assert status == 0
    _check_logprobs(x, ids, top, lp, ent, ti, tl)


@pytest.mark.parametrize("n", [1, 300])
@pytest.mark.parametrize("vocab", [40, 5000, 50257])
def test_logprobs_of_rows_in_an_order(vocab, n):
    """Logits that rise (every one a candidate for the top), that fall, that are all the same, two values in turn, the type's lowest value
    as a mask, minus infinities on all but few."""
    rise = torch.arange(vocab, dtype=torch.float32) / vocab * 3
    few = torch.full((vocab,), float("-inf"))
    few[[0, vocab // 2, vocab - 1]] = torch.tensor([1.0, 2.0, 1.0])
    lowest = torch.full((vocab,), torch.finfo(torch.float32).min)
    lowest[vocab // 3] = 4.0
    kinds = torch.stack([rise, rise.flip(0), torch.zeros(vocab), (torch.arange(vocab) % 2).float(), lowest, few, rise * 1e-30, torch.zeros(vocab) - rise % 0.1])
    x = kinds.repeat(n, 1).to(DEV)
    ids = [(7 * i) % vocab for i in range(x.shape[0])]
    lp, ent, ti, tl, status = _run_logprobs(x, ids, 20)
    assert status == 0
    _check_logprobs(x, ids, 20, lp, ent, ti, tl)


@pytest.mark.parametrize("vocab", [10, 50257])
def test_logprobs_of_rows_without_a_distribution(vocab):
    x = torch.zeros(6, vocab)
    x[0] = float("-inf")
    x[1, 3] = float("inf")
    x[2, vocab - 1] = float("nan")
    x[3, 0] = -float("nan")
    ids = [1, 3, 0, 0, vocab, -2]
    lp, ent, ti, tl, status = _run_logprobs(x.to(DEV), ids, 3)
    assert status == 1
    assert bool(torch.isnan(lp).all())
    assert torch.isnan(ent).cpu().tolist() == [True] * 4 + [False] * 2
    assert bool(torch.isnan(tl[:4]).all()) and bool(torch.isfinite(tl[4:]).all())
    assert ti.cpu().tolist() == [[0, 1, 2], [3, 0, 1], [-1] * 3, [-1] * 3, [0, 1, 2], [0, 1, 2]]
    for bad in (0, 1, 4, 5):                                      # an id outside, and no other fault
        one = torch.zeros(1, dtype=torch.int32, device=DEV)
        from sandyrt_b200.csrc import ops

        ops.token_logprobs(x[bad:bad + 1].to(DEV), _i32([ids[bad]]), torch.zeros(1, device=DEV), status=one)
        assert int(one.item()) == (1 if bad >= 4 else 0)


def test_logprobs_of_parts_alone():
    """Each output without the others, the same to the bit; twice, the same to the bit."""
    from sandyrt_b200.csrc import ops

    x = torch.randn(5, 50257, generator=torch.Generator().manual_seed(1)).to(DEV) * 3
    ids = [4, 9, 50256, 0, 77]
    lp, ent, ti, tl, _ = _run_logprobs(x, ids, 7)
    again = _run_logprobs(x, ids, 7)
    assert all(torch.equal(a, b) for a, b in zip((lp, ent, ti, tl), again[:4]))
    lp2, ent2, ti2, tl2 = torch.zeros_like(lp), torch.zeros_like(ent), torch.zeros_like(ti), torch.zeros_like(tl)
    ops.token_logprobs(x, _i32(ids), lp2)
    ops.token_logprobs(x, None, None, entropy=ent2)
    ops.token_logprobs(x, None, None, top_ids=ti2, top_logprobs=tl2)
    assert torch.equal(lp, lp2) and torch.equal(ent, ent2) and torch.equal(ti, ti2) and torch.equal(tl, tl2)
    ops.token_logprobs(x[:0], _i32([]), lp2[:0])


def test_tensors_on_two_devices_are_refused():
    from sandyrt_b200.csrc import ops
    from sandyrt_b200.errors import KernelError

    with pytest.raises(KernelError, match="tensors on"):
        ops.token_logprobs(torch.zeros(2, 5, device=DEV), torch.zeros(2, dtype=torch.int32), torch.zeros(2, device=DEV))
