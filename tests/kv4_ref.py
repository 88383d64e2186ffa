"""The 4-bit paged KV cache's operators in numpy, in 64 bits (no GPU): the
reference that tests/test_gpu_kv4.py holds the kernels to.

A batch is described by host arrays: tok_start, kv_len, pages; a cache by its
bytes, [n_pages][nkv][page_rows rows of codes, page_rows rows of f16 scales].
"""
import numpy as np

F16_MAX = 65504.0


def page_bytes(rows, nkv, hd):
    return rows * nkv * (hd // 2 + hd // 16)


def quantise(x):
    """x f32 [..., hd] -> (codes uint8 [..., hd / 32, 32], scales f16 [..., hd / 32]):
    the header's steps, every fp32 product and sum rounded."""
    with np.errstate(all="ignore"):
        b = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32).astype(np.float32)
        nan = np.isnan(b).any(-1)
        b = np.clip(np.nan_to_num(b, nan=0.0, posinf=F16_MAX, neginf=-F16_MAX), -F16_MAX, F16_MAX).astype(np.float32)
        m = np.take_along_axis(b, np.abs(b).argmax(-1)[..., None], -1)[..., 0]
        d = m / np.float32(-8.0)
        d16 = d.astype(np.float16)
        inv = np.where(d16 == 0, np.float32(0), np.float32(1) / d).astype(np.float32)
        q = (b * inv[..., None]).astype(np.float32) + np.float32(8.5)
        code = np.minimum(np.trunc(q), 15).astype(np.uint8)
    code[nan] = 8
    d16 = np.where(d16 == 0, np.float16(0), d16)
    d16[nan] = np.float16(np.nan)
    return code, d16


def values(code, d16):
    v = (code.astype(np.float64) - 8.0) * d16.astype(np.float64)[..., None]
    return v.reshape(*v.shape[:-2], -1)


def head_view(cache, page, g, rows, nkv, hd):
    """(codes [rows, hd / 2], scales f16 [rows, hd / 32]) of one head of one page: views."""
    per = rows * (hd // 2 + hd // 16)
    at = (page * nkv + g) * per
    codes = cache[at:at + rows * hd // 2].reshape(rows, hd // 2)
    return codes, cache[at + rows * hd // 2:at + per].view(np.float16).reshape(rows, hd // 32)


def put(cache, page, row, g, rows, nkv, hd, code, d16):
    codes, scales = head_view(cache, page, g, rows, nkv, hd)
    codes[row] = (code[:, :16] | (code[:, 16:] << 4)).reshape(-1)
    scales[row] = d16


def get(cache, page, row, g, rows, nkv, hd):
    codes, scales = head_view(cache, page, g, rows, nkv, hd)
    b = codes[row].reshape(-1, 16)
    return values(np.concatenate([b & 15, b >> 4], -1), scales[row])


def positions(tok_start, kv_len, n_tok):
    """(sequence, position) of each token row; sequence -1: nobody's."""
    out = [(-1, -1)] * n_tok
    for s in range(len(kv_len)):
        n = tok_start[s + 1] - tok_start[s]
        for i in range(n):
            out[tok_start[s] + i] = (s, kv_len[s] - n + i)
    return out


def prep(x, w, pos, eps, rope_dims, base):
    """x [heads, hd] at one position; returns the value and the magnitude its rounding errors scale with."""
    x = x.astype(np.float64)
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    if w is not None:
        y = y * w.astype(np.float64)
    mag, half = np.abs(y), rope_dims // 2
    if half:
        ang = pos * float(base) ** (-np.arange(half) / half)
        c, s = np.cos(ang), np.sin(ang)
        a, b = y[:, :half].copy(), y[:, half:2 * half].copy()
        y[:, :half], y[:, half:2 * half] = a * c - b * s, a * s + b * c
        mag[:, :half] = mag[:, half:2 * half] = np.abs(a) + np.abs(b)
    return y, mag


def attention(q, k, v, scale):
    """One row: q [hd], k and v [rows, hd], all seen.  Returns the output, sum w |v| per
    element, and the largest sum |q k| * scale."""
    if len(k) == 0:
        return np.zeros(len(q)), np.zeros(len(q)), 0.0
    s = (k @ q) * scale
    w = np.exp(s - s.max())
    w /= w.sum()
    return w @ v, w @ np.abs(v), float((np.abs(k) @ np.abs(q)).max() * scale)
