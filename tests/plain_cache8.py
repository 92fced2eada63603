"""The 8-bit cache, the attention over it and the log-probabilities of tokens, written out in 64 bits on the host."""
import math

import numpy as np
import torch

CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
LARGEST = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def scale_for(amax, code):
    """The smallest power of two s >= 2^-100 with amax <= largest * s (amax a Python float)."""
    s = 2.0 ** -100
    if amax > LARGEST[code] * s:
        s = 2.0 ** math.ceil(math.log2(amax / LARGEST[code]))
        if s * LARGEST[code] < amax:
            s *= 2
        elif s / 2 * LARGEST[code] >= amax:
            s /= 2
    return s


def nearest(y, code):
    """The code's value nearest to y (float64 tensor), ties to the even one."""
    if code == torch.int8:
        return torch.round(y)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step


class PlainCache:
    """codes (float64 values of the codes) and scales of keys and values; NaN where nobody has written."""

    def __init__(self, pages, hkv, ps, d, code):
        self.code, self.ps = code, ps
        self.codes = [torch.full((pages, hkv, ps, d), float("nan"), dtype=torch.float64) for _ in range(2)]
        self.scales = [torch.full((pages, hkv), float("nan"), dtype=torch.float64) for _ in range(2)]

    def append(self, k, v, table, q_start, before):
        """k, v: [T, hkv, d] float64."""
        for which, x in enumerate((k, v)):
            codes, scales = self.codes[which], self.scales[which]
            for s in range(len(before)):
                t, n, b = q_start[s], q_start[s + 1] - q_start[s], before[s]
                for block in range(b // self.ps, (b + n - 1) // self.ps + 1 if n else 0):
                    lo, hi = max(b, block * self.ps), min(b + n, (block + 1) * self.ps)
                    page, at = table[s][block], lo - block * self.ps
                    for h in range(x.shape[1]):
                        rows = x[t + lo - b:t + hi - b, h]
                        if not bool(torch.isfinite(rows).all()):
                            scales[page, h] = float("nan")
                        else:
                            need = scale_for(float(rows.abs().max()), self.code)
                            if at:
                                old = float(scales[page, h])
                                need = need if need > old else old             # an old NaN stays
                                if need == need and need > old:
                                    codes[page, h, :at] = nearest(codes[page, h, :at] * (old / need), self.code)
                            scales[page, h] = need
                        s_now = float(scales[page, h])
                        codes[page, h, at:at + hi - lo] = nearest(rows / s_now, self.code) if s_now == s_now else 0.0

    def values(self, which, table_row, n):
        """[n, hkv, d]: the first n cached positions of a request."""
        pages = list(table_row[:-(-n // self.ps)])
        x = self.codes[which][pages] * self.scales[which][pages][..., None, None]
        return x.transpose(1, 2).reshape(-1, x.shape[1], x.shape[3])[:n]


def attention(q, k, v, positions, *, scale, window=0, keep_first=0, softcap=0.0, chunk=0, sink=None, out_gate=None, dist_bias=None,
              elem_gate=None):
    """q: [n, H, d] at `positions`; k, v: [L, hkv, d] (float64).  Rows without a visible key are zeros."""
    n, H, d = q.shape
    out = torch.zeros(n, H, d, dtype=torch.float64)
    for i in range(n):
        pos = int(positions[i])
        lo = max(0, pos + 1 - window) if window else 0
        if chunk and pos >= 0:
            lo = max(lo, pos - pos % chunk)
        keys = [j for j in range(pos + 1) if j >= lo or j < keep_first]
        if not keys:
            continue
        kk, vv = k[keys], v[keys]
        for h in range(H):
            g = h * k.shape[1] // H
            s = kk[:, g] @ q[i, h] * scale
            if softcap:
                s = softcap * torch.tanh(s / softcap)
            if dist_bias is not None:
                far = torch.tensor([min(pos - j, dist_bias.shape[1] - 1) for j in keys])
                s = s + dist_bias[h][far]
            m = s.max()
            p = torch.exp(s - m)
            total = p.sum() + (torch.exp(sink[h] - m) if sink is not None else 0.0)
            y = (p / total) @ vv[:, g]
            if out_gate is not None:
                y = y * out_gate[i, h]
            if elem_gate is not None:
                dim = elem_gate.shape[1] // H
                y[:dim] = y[:dim] * torch.sigmoid(elem_gate[i, h * dim:(h + 1) * dim])
            out[i, h] = y
    return out


def logprobs(x, ids, top):
    """x: [n, vocab] float64, finite or minus infinity.  (logprob, entropy, top ids, top logprobs) as float64 / int64 arrays."""
    x = x.numpy()
    m = x.max(axis=1, keepdims=True)
    lz = m + np.log(np.exp(x - m).sum(axis=1, keepdims=True))
    lp = x - lz
    p = np.exp(lp)
    entropy = -np.where(p > 0, p * np.where(p > 0, lp, 0.0), 0.0).sum(axis=1)
    order = np.argsort(-x, axis=1, kind="stable")[:, :top]
    given = np.array([lp[r, i] if i >= 0 else 0.0 for r, i in enumerate(ids)])
    return given, entropy, order, np.take_along_axis(lp, order, axis=1)
