"""64-bit restatements (numpy) of rotary rows, the KV cache and attention for drafted tokens, for the tests."""
import numpy as np

F32, Q80, Q40 = 0, 1, 2


def half_up(x):
    """Nonnegative fp32 values on fp16's grid, halves up (the quantizer's rounding), as float32."""
    x = np.asarray(x, np.float32).astype(np.float64)
    e = np.floor(np.log2(np.maximum(x, 2.0 ** -14)))
    step = 2.0 ** (e - 10)
    y = np.floor(x / step + 0.5) * step
    return np.where(y > 65504.0, np.inf, y).astype(np.float32)


def held(x, qtype):
    """What a cache of this type holds for x [..., head_dim] (fp32 in, fp32 out), in the quantizer's fp32 steps."""
    x = np.asarray(x, np.float32)
    if qtype == F32:
        return x.copy()
    hd = x.shape[-1]
    pad = -hd % 32
    b = np.pad(x, [(0, 0)] * (x.ndim - 1) + [(0, pad)]).reshape(*x.shape[:-1], -1, 32)
    inv_top = np.float32(1) / np.float32(127 if qtype == Q80 else 7)
    d = half_up(np.abs(b).max(-1, keepdims=True) * inv_top)
    with np.errstate(divide="ignore"):
        inv = np.where(d > 0, np.float32(1) / d, np.float32(0)).astype(np.float32)
    y = (b * inv).astype(np.float32)
    if qtype == Q40:
        y = (y + np.float32(8)).astype(np.float32)
    n = np.trunc(y)
    n = n + np.sign(y) * (np.abs(y - n) >= 0.5)
    n = np.clip(n, -127, 127) if qtype == Q80 else np.clip(n, 0, 15) - 8
    n = np.where(np.abs(b).max(-1, keepdims=True) > 0, n, -8 if qtype == Q40 else 0)  # a block of zeros: nibbles 0
    return (n.astype(np.int32).astype(np.float32) * d).reshape(*x.shape[:-1], -1)[..., :hd]


def rotate(x, cos, sin, rot, neox):
    """x [rows, heads, hd] with cos, sin [rows, rot / 2], in the dtype of x."""
    c, s = cos[:, None, :], sin[:, None, :]
    a = np.arange(rot // 2) if neox else 2 * np.arange(rot // 2)
    b = a + rot // 2 if neox else a + 1
    y = x.copy()
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., a] * s + x[..., b] * c
    return y


def sees(mask, t, tokens, n, slots):
    """Bool [slots]: what token t sees of n committed slots and the drafted ones after them."""
    s = np.zeros(slots, bool)
    s[:min(n, slots)] = True
    for j in range(tokens):
        if n + j < slots:
            s[n + j] = (int(mask[t, j // 64]) >> (j % 64)) & 1 if mask is not None else j <= t
    return s


def attention(q, k, v, lens, seqs, mask, scale, max_seq):
    """q [batch, tokens, heads, hd]; k, v [n_seqs, max_seq, kv, hd].  Returns (out, slack): the exact result and, per
    element, what one unit of relative error of the weights moves it by, with the largest sum |q k| scale of the row."""
    b, t, heads, hd = q.shape
    kv = k.shape[2]
    out = np.zeros(q.shape)
    weight = np.zeros(q.shape)
    terms = np.zeros(q.shape)
    for i in range(b):
        n = lens[i]
        if n < 0 or not 0 <= seqs[i] < k.shape[0]:
            continue
        for r in range(t):
            m = sees(None if mask is None else mask[i], r, t, n, max_seq)
            if not m.any():
                continue
            for h in range(heads):
                kk = k[seqs[i], m, h * kv // heads].astype(np.float64)
                vv = v[seqs[i], m, h * kv // heads].astype(np.float64)
                x = kk @ q[i, r, h].astype(np.float64) * scale
                w = np.exp(x - x.max())
                w /= w.sum()
                out[i, r, h] = w @ vv
                weight[i, r, h] = w @ np.abs(vv)
                terms[i, r, h] = (np.abs(kk) @ np.abs(q[i, r, h].astype(np.float64))).max() * scale
    return out, weight, terms
