"""Plain 64-bit forms of the decoder operators, on the CPU, and how far float32 kernels may be
from them (first-order bounds, counted roundings)."""
import numpy as np
import torch

U32 = 2.0 ** -24  # half a step of float32, relative
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133}


def f64(t):
    return t.detach().double().cpu().numpy()


def quantize_tokens(x):
    x = f64(x)
    top = np.abs(x).max(-1).astype(np.float32)
    s = np.maximum(top / np.float32(127.0), np.float32(2.0 ** -126))
    good = np.isfinite(top)
    s = np.where(good, s, np.float32(np.nan))
    with np.errstate(invalid="ignore"):
        q = np.where(good[..., None], np.rint(x / s.astype(np.float64)[..., None]), 0.0)
    return q.astype(np.int8), s


def token_qlinear(q, s, w, ws, bias):
    """(y, |sum s ws|), both in 64 bits."""
    p = (q.astype(np.int64) @ w.astype(np.int64)).astype(np.float64) * s.astype(np.float64)[:, None] * ws.astype(np.float64)
    return (p if bias is None else p + bias.astype(np.float64)), np.abs(p)


def token_qlinear_bound(y, p, dtype):
    """The sum to float32, the scales' product, the product and the bias: a rounding each; then dtype's own."""
    return 4 * U32 * (p + np.abs(y)) + HALF[dtype] * np.abs(y) + TINY[dtype]


GRID = {4: np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6]),
        8: np.array([(m / 8.0) * 2.0 ** -6 if e == 0 else (1 + m / 8.0) * 2.0 ** (e - 7) for e in range(16) for m in range(8)][:127])}


def cached(x, bits):
    """What the cache holds for x [..., D]: blocks of 32, a power-of-two scale each."""
    x = f64(x)
    b = x.reshape(-1, 32)
    grid, lo, hi = GRID[bits], *((-125, 125) if bits == 4 else (-117, 119))
    out = np.empty_like(b)
    for i, r in enumerate(b):
        top = np.abs(r).max()
        if not np.isfinite(top):
            out[i] = np.nan
            continue
        e = lo
        while e < hi and (top / 2.0 ** e >= 7.0 if bits == 4 else top / 2.0 ** e > 464.0):
            e += 1
        a = np.abs(r) / 2.0 ** e
        k = np.clip(np.searchsorted(grid, a), 1, len(grid) - 1)
        down, up = a - grid[k - 1], grid[k] - a
        k = np.where((down < up) | ((down == up) & (k % 2 == 1)), k - 1, k)
        out[i] = np.sign(r) * grid[k] * 2.0 ** e
    return out.reshape(x.shape)


def attention(q, k, v, lengths, starts, scale, softcap=0.0, window=0, slopes=None, causal=True, terms=3, dtype=torch.float32,
              absent=None):
    """(out, bound) [rows, heads, D] for k, v: lists of [tokens, kv_heads, D] in 64 bits, one of each sequence.
    absent: for each sequence, which of its tokens lie in no page of the cache."""
    q = f64(q)
    rows, H, D = q.shape
    out, bound = np.full(q.shape, np.nan), np.zeros(q.shape)
    weight = {1: 2.0 ** -8, 2: 2.0 ** -16, 3: 2.0 ** -24}[terms]
    for b, n in enumerate(lengths):
        r0, r1 = starts[b], starts[b + 1]
        for r in range(r0, r1):
            p = n - (r1 - r0) + r - r0
            j = np.arange(n)
            seen = np.ones(n, bool)
            if causal:
                seen &= j <= p
            if window:
                seen &= j > p - window
            if absent is not None:
                seen &= ~absent[b]
            for h in range(H):
                g = h // (H // k[b].shape[1])
                if not seen.any():
                    out[r, h] = 0.0
                    continue
                kk, vv, jj = k[b][seen, g], v[b][seen, g], j[seen]
                a = np.abs(kk) @ np.abs(q[r, h]) * abs(scale)
                s = kk @ q[r, h] * scale
                d = (terms * D + 8) * a + 4 * np.abs(s)
                if softcap:
                    # (in float32 the roundings are a score's own: 6 of its series, or 8 of the cap where that
                    # is no more than four times the score)
                    d = d + 8 * (softcap if terms < 3 else np.minimum(softcap, 4 * np.abs(s)))
                    s = softcap * np.tanh(s / softcap)
                if slopes is not None:
                    t = slopes[h] * (jj - p)
                    s = s + t
                    d = d + 4 * np.abs(t)
                m = s.max()
                e = np.exp(s - m)
                # scores as powers of two (a rounding each of the product, of the difference from the
                # maximum and of the exponential), and the sums over the tokens
                d = U32 * (d + 4 * np.abs(s) + 8 * np.abs(s - m) + 8 + len(jj) + 16)
                w = e / e.sum()
                out[r, h] = w @ vv
                mag = np.abs(vv)
                bound[r, h] = (w * (d + weight)) @ mag + (w @ d) * (w @ mag)
    return out, bound + HALF[dtype] * np.abs(out) + TINY[dtype] + 2.0 ** -60
