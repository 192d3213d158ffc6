"""GPU tests of rotary rows (mlb_rope_*), the caller-owned KV cache (mlb_kv_cache_*) and attention for drafted
tokens (mlb_attention_tree) against 64-bit restatements.

Tolerances, fixed by derivation:
  - rotation, quantized writes and reads: bit for bit (every step is an explicitly rounded fp32 operation in the
    order of mlb_rope and mlb_quantize, the cache's scale a product with fl(1/127) or fl(1/7); the table is the host's)
  - attention, per output: out = sum_s w_s V_s with w = softmax(x).  q and the weights carry at least 22 bits
    (2^-22 relative) and every sum is in fp32: a score is off by at most g X, X = scale sum_i |q_i k_i| and
    g = 2^-20 (2^-22 of the split plus fp32 rounding of sums of up to 256 products), and a weight by that twice
    (itself and the normaliser) plus 2^-19 for the exponential, the normaliser's sum and the weighted sum.  So
    |out - exact| <= (2^-19 X_max + 2^-19) sum_s w_s |V_s|, X_max the largest X of the row.
"""
import ctypes

import numpy as np
import pytest

import cached_decoding_ref as ref
from mini_llama_b200 import capi
from mini_llama_b200.device import DeviceArray, KvCache, RopeTable

pytestmark = pytest.mark.gpu

F32, Q80, Q40 = capi.F32, capi.Q8_0, capi.Q4_0
NAME = {F32: "f32", Q80: "q8_0", Q40: "q4_0"}


class Cache:
    """Cache planes on the device with their descriptor."""

    def __init__(self, lib, dev, qtype, n_seqs, n_layers, max_seq, kv, hd, fill=0):
        self.lib, self.dev = lib, dev
        self.desc = capi.KvCache(type=qtype, n_seqs=n_seqs, n_layers=n_layers, max_seq_len=max_seq, n_kv_heads=kv,
                                 head_dim=hd)
        plane, scale = ctypes.c_size_t(), ctypes.c_size_t()
        lib.call("mlb_kv_cache_bytes", ctypes.byref(self.desc), ctypes.byref(plane), ctypes.byref(scale))
        self.plane_bytes, self.scale_bytes = plane.value, scale.value
        self.bufs = [DeviceArray(lib, dev, (n,), np.uint8) for n in (plane.value,) * 2 + (scale.value,) * 2]
        for b in self.bufs:
            lib.call("mlb_memset", dev, b.ptr, fill, b.nbytes)
        self.desc.k, self.desc.v = self.bufs[0].ptr, self.bufs[1].ptr
        if qtype != F32:
            self.desc.k_scale, self.desc.v_scale = self.bufs[2].ptr, self.bufs[3].ptr

    @property
    def ref(self):
        return ctypes.byref(self.desc)

    def write(self, layer, seqs, slots, k, v):
        rows = len(slots)
        kd, vd = (DeviceArray.from_host(self.lib, self.dev, np.asarray(x, np.float32)) for x in (k, v))
        sd = DeviceArray.from_host(self.lib, self.dev, np.asarray(slots, np.int32))
        qd = DeviceArray.from_host(self.lib, self.dev, np.asarray(seqs, np.int32)) if seqs is not None else None
        n = self.desc.n_kv_heads * self.desc.head_dim
        self.lib.call("mlb_kv_cache_write", self.dev, self.ref, layer, rows, qd.ptr if qd else None, sd.ptr, kd.ptr, n,
                      vd.ptr, n)

    def read(self, layer, seqs, slots):
        rows = len(slots)
        shape = (rows, self.desc.n_kv_heads, self.desc.head_dim)
        if layer == capi.ALL_LAYERS:
            shape = (self.desc.n_layers,) + shape
        kd, vd = DeviceArray(self.lib, self.dev, shape), DeviceArray(self.lib, self.dev, shape)
        sd = DeviceArray.from_host(self.lib, self.dev, np.asarray(slots, np.int32))
        qd = DeviceArray.from_host(self.lib, self.dev, np.asarray(seqs, np.int32)) if seqs is not None else None
        n = self.desc.n_kv_heads * self.desc.head_dim
        self.lib.call("mlb_kv_cache_read", self.dev, self.ref, layer, rows, qd.ptr if qd else None, sd.ptr, kd.ptr, n,
                      vd.ptr, n)
        return kd.download(), vd.download()

    def planes(self):
        return [b.download() for b in self.bufs]


def same_bits(a, b):
    return np.array_equal(np.asarray(a, np.float32).view(np.uint32), np.asarray(b, np.float32).view(np.uint32))


# ------------------------------------------------------------------------------------------------ rotary rows
def make_table(lib, dev, n_positions, hd, rot, neox, theta=1e4, scale=None):
    buf = DeviceArray(lib, dev, (n_positions, rot // 2, 2))
    t = capi.RopeTable(n_positions=n_positions, head_dim=hd, rot_dim=rot,
                       rope_type=capi.ROPE_NEOX if neox else capi.ROPE_NORMAL, cos_sin=buf.ptr)
    lib.call("mlb_rope_table_fill", dev, ctypes.byref(t), theta, ctypes.byref(scale) if scale else None)
    return t, buf


@pytest.mark.parametrize("neox", [False, True])
@pytest.mark.parametrize("hd,rot", [(64, 64), (128, 128), (16, 16), (128, 32), (80, 40), (10, 6), (64, 2), (36, 12)])
@pytest.mark.parametrize("rows,in_place", [(1, False), (7, True), (33, False)])
def test_rope_rows(mlb, gpu, neox, hd, rot, rows, in_place):
    heads, kv = 6, 2
    rng = np.random.default_rng(hd * 1000 + rot + rows)
    table, buf = make_table(mlb, gpu, 600, hd, rot, neox)
    cs = buf.download()
    wide = (heads + 2 * kv) * hd + 4  # rows of a fused projection, with a gap
    x = rng.standard_normal((rows, wide)).astype(np.float32)
    pos = rng.integers(0, 600, rows).astype(np.int32)
    xd, pd = DeviceArray.from_host(mlb, gpu, x), DeviceArray.from_host(mlb, gpu, pos)
    q = x[:, :heads * hd].reshape(rows, heads, hd)
    k = x[:, heads * hd:(heads + kv) * hd].reshape(rows, kv, hd)
    c, s = cs[pos, :, 0], cs[pos, :, 1]
    if in_place:
        out = (xd.ptr, wide, xd.ptr + 4 * heads * hd, wide)
    else:
        qo, ko = DeviceArray(mlb, gpu, (rows, heads, hd)), DeviceArray(mlb, gpu, (rows, kv, hd))
        out = (qo.ptr, heads * hd, ko.ptr, kv * hd)
    mlb.call("mlb_rope_rows", gpu, ctypes.byref(table), rows, pd.ptr, xd.ptr, wide, out[0], out[1], heads,
             xd.ptr + 4 * heads * hd, wide, out[2], out[3], kv)
    if in_place:
        y = xd.download()
        assert same_bits(y[:, (heads + kv) * hd:], x[:, (heads + kv) * hd:])
        yq, yk = y[:, :heads * hd].reshape(q.shape), y[:, heads * hd:(heads + kv) * hd].reshape(k.shape)
    else:
        yq, yk = qo.download(), ko.download()
    assert same_bits(yq, ref.rotate(q, c, s, rot, neox))
    assert same_bits(yk, ref.rotate(k, c, s, rot, neox))


@pytest.mark.parametrize("rope_type", [capi.ROPE_NORMAL, capi.ROPE_NEOX])
def test_rope_rows_equals_mlb_rope(mlb, gpu, rope_type):
    """Unscaled whole heads: the bits of the one-row call, at far positions too."""
    heads, kv, hd, theta = 14, 2, 64, 1e6
    rng = np.random.default_rng(3)
    table, _ = make_table(mlb, gpu, 32768, hd, hd, rope_type == capi.ROPE_NEOX, theta)
    pos = np.array([0, 1, 77, 4097, 32767], np.int32)
    q = rng.standard_normal((len(pos), heads, hd)).astype(np.float32)
    k = rng.standard_normal((len(pos), kv, hd)).astype(np.float32)
    qd, kd, pd = (DeviceArray.from_host(mlb, gpu, a) for a in (q, k, pos))
    mlb.call("mlb_rope_rows", gpu, ctypes.byref(table), len(pos), pd.ptr, qd.ptr, heads * hd, qd.ptr, heads * hd, heads,
             kd.ptr, kv * hd, kd.ptr, kv * hd, kv)
    got_q, got_k = qd.download(), kd.download()
    for i, p in enumerate(pos):
        q1, k1 = DeviceArray.from_host(mlb, gpu, q[i]), DeviceArray.from_host(mlb, gpu, k[i])
        mlb.call("mlb_rope", gpu, q1.ptr, k1.ptr, heads, kv, hd, int(p), theta, rope_type)
        assert same_bits(got_q[i], q1.download()) and same_bits(got_k[i], k1.download())


def test_rope_rows_outside_table_and_absent_parts(mlb, gpu):
    """Rows outside the table become NaN (whole heads), others do not change; q or k alone works."""
    hd, rot, heads = 32, 16, 3
    table, buf = make_table(mlb, gpu, 10, hd, rot, True)
    cs = buf.download()
    x = np.random.default_rng(1).standard_normal((4, heads, hd)).astype(np.float32)
    pos = np.array([-1, 9, 10, 0], np.int32)
    xd, pd = DeviceArray.from_host(mlb, gpu, x), DeviceArray.from_host(mlb, gpu, pos)
    n = heads * hd
    mlb.call("mlb_rope_rows", gpu, ctypes.byref(table), 4, pd.ptr, None, 0, None, 0, 0, xd.ptr, n, xd.ptr, n, heads)
    y = xd.download()
    assert np.isnan(y[[0, 2]]).all()
    at = pos[[1, 3]]
    assert same_bits(y[[1, 3]], ref.rotate(x[[1, 3]], cs[at, :, 0], cs[at, :, 1], rot, True))


def test_rope_table_scalings(mlb, gpu):
    """The scaled tables against their formulas in 64 bits: a frequency is fp32 (2^-23 relative of a power and a
    division, 4 ulp), so an angle of position p is off by at most 2^-21 p freq, plus 2^-24 for cos and sin."""
    n, rot, theta, factor, orig = 300, 64, 1e4, 8.0, 64
    i = np.arange(rot // 2)
    f = theta ** (-2.0 * i / rot)
    turns = orig * f / (2 * np.pi)
    d = lambda r: rot * np.log(orig / (r * 2 * np.pi)) / (2 * np.log(theta))  # noqa: E731
    low, high = max(0.0, np.floor(d(32))), min(rot - 1.0, np.ceil(d(1)))
    ramp = np.clip((i - low) / (high - low), 0, 1)
    smooth = np.clip((turns - 1) / (4 - 1), 0, 1)
    want = {capi.ROPE_SCALE_NONE: (f, 1.0), capi.ROPE_SCALE_LINEAR: (f / factor, 1.0),
            capi.ROPE_SCALE_NTK: ((theta * factor ** (rot / (rot - 2))) ** (-2.0 * i / rot), 1.0),
            capi.ROPE_SCALE_YARN: (f / factor * ramp + f * (1 - ramp), 0.1 * np.log(factor) + 1),
            capi.ROPE_SCALE_WAVELENGTH: (f / factor * (1 - smooth) + f * smooth, 1.0)}
    for kind, (freq, mag) in want.items():
        scale = capi.RopeScale(scaling=kind, factor=factor, original_positions=orig)
        _, buf = make_table(mlb, gpu, n, rot, rot, False, theta, scale)
        got = buf.download()
        angle = np.arange(n)[:, None] * freq
        tol = mag * (2.0 ** -21 * angle + 2.0 ** -22)
        assert (np.abs(got[..., 0] - mag * np.cos(angle)) <= tol).all(), kind
        assert (np.abs(got[..., 1] - mag * np.sin(angle)) <= tol).all(), kind


# ------------------------------------------------------------------------------------------------ cache
@pytest.mark.parametrize("qtype", [F32, Q80, Q40], ids=NAME.get)
@pytest.mark.parametrize("kv,hd", [(2, 64), (8, 128), (2, 16), (3, 80), (1, 33), (2, 7), (1, 256)])
@pytest.mark.parametrize("rows", [1, 5, 67])
def test_cache_write_and_read_back(mlb, gpu, qtype, kv, hd, rows):
    n_seqs, layers, max_seq = 3, 2, 45
    rng = np.random.default_rng(rows * 1000 + hd)
    c = Cache(mlb, gpu, qtype, n_seqs, layers, max_seq, kv, hd, fill=0x5A)
    before = c.planes()
    at = rng.permutation(n_seqs * max_seq)[:rows]
    seqs, slots = (at // max_seq).astype(np.int32), (at % max_seq).astype(np.int32)
    k = (rng.standard_normal((rows, kv, hd)) * rng.choice([1e-6, 1e-3, 1.0, 300.0], (rows, kv, 1))).astype(np.float32)
    v = rng.standard_normal((rows, kv, hd)).astype(np.float32)
    k[0, 0] = 0.0
    if rows > 4:  # padding and rows outside are skipped
        slots[1], seqs[2], slots[3], seqs[4] = -1, n_seqs, max_seq, -1
    c.write(1, seqs, slots, k, v)
    got_k, got_v = c.read(1, seqs, slots)
    kept = (slots >= 0) & (slots < max_seq) & (seqs >= 0) & (seqs < n_seqs)
    assert same_bits(got_k[kept], ref.held(k, qtype)[kept]) and same_bits(got_v[kept], ref.held(v, qtype)[kept])
    assert (got_k[~kept] == 0).all() and (got_v[~kept] == 0).all()
    # nothing else changed: as many bytes differ at most as the rows hold
    per_row = kv * (hd * 4 if qtype == F32 else (hd + 31) // 32 * (32 if qtype == Q80 else 16))
    for b, a in zip(before, c.planes()):
        assert (a != b).sum() <= per_row * kept.sum()
    layer0, _ = c.read(0, seqs[kept], slots[kept])
    fresh = Cache(mlb, gpu, qtype, n_seqs, layers, max_seq, kv, hd, fill=0x5A)
    assert same_bits(layer0, fresh.read(0, seqs[kept], slots[kept])[0])


@pytest.mark.parametrize("qtype", [Q80, Q40], ids=NAME.get)
def test_cache_layout_is_the_quantizers(mlb, gpu, qtype):
    """The planes hold the blocks of mlb_quantize (whose scales these inputs share): scales and quants as the header
    lays them out."""
    n_seqs, layers, max_seq, kv, hd = 2, 2, 9, 2, 96
    stored, blocks, qb = 16, 3, 32 if qtype == Q80 else 16
    rng = np.random.default_rng(5)
    x = rng.standard_normal((1, kv, hd)).astype(np.float32)
    c = Cache(mlb, gpu, qtype, n_seqs, layers, max_seq, kv, hd)
    c.write(1, [1], [8], x, -x)
    xd = DeviceArray.from_host(mlb, gpu, x[0])
    out = DeviceArray(mlb, gpu, (kv, blocks, qb + 2), np.uint8)
    mlb.call("mlb_quantize", gpu, qtype, xd.ptr, kv, hd, out.ptr)
    want = out.download()
    planes = c.planes()
    q = planes[0].reshape(n_seqs, layers, kv, stored, blocks, qb)
    d = planes[2].reshape(n_seqs, layers, kv, stored, blocks, 2)
    assert np.array_equal(q[1, 1, :, 8], want[..., 2:]) and np.array_equal(d[1, 1, :, 8], want[..., :2])
    q[1, 1, :, 8], d[1, 1, :, 8] = 0, 0
    assert not q.any() and not d.any()


@pytest.mark.parametrize("qtype", [F32, Q80, Q40], ids=NAME.get)
def test_cache_all_layers_and_default_sequence(mlb, gpu, qtype):
    """One call for every layer equals a call for each; seqs NULL is sequence 0."""
    layers, kv, hd, rows = 3, 2, 64, 4
    rng = np.random.default_rng(8)
    k, v = (rng.standard_normal((layers, rows, kv, hd)).astype(np.float32) for _ in range(2))
    slots = [3, 0, -1, 7]
    a, b = (Cache(mlb, gpu, qtype, 2, layers, 8, kv, hd) for _ in range(2))
    n = kv * hd
    kd, vd = DeviceArray.from_host(mlb, gpu, k), DeviceArray.from_host(mlb, gpu, v)
    sd = DeviceArray.from_host(mlb, gpu, np.array(slots, np.int32))
    mlb.call("mlb_kv_cache_write", gpu, a.ref, capi.ALL_LAYERS, rows, None, sd.ptr, kd.ptr, n, vd.ptr, n)
    for l in range(layers):
        b.write(l, [0] * rows, slots, k[l], v[l])
    for x, y in zip(a.planes(), b.planes()):
        assert np.array_equal(x, y)
    all_k, all_v = a.read(capi.ALL_LAYERS, None, slots)
    for l in range(layers):
        one_k, one_v = b.read(l, None, slots)
        assert same_bits(all_k[l], one_k) and same_bits(all_v[l], one_v)


@pytest.mark.parametrize("qtype", [F32, Q80, Q40], ids=NAME.get)
@pytest.mark.parametrize("neox", [False, True])
@pytest.mark.parametrize("hd,rot", [(64, 64), (128, 64), (80, 80), (36, 20), (16, 16)])
def test_cache_write_rope_equals_the_two_calls(mlb, gpu, qtype, neox, hd, rot):
    heads, kv, rows, max_seq = 6, 2, 9, 30
    rng = np.random.default_rng(hd + rot)
    table, _ = make_table(mlb, gpu, 40, hd, rot, neox)
    q, k, v = (rng.standard_normal((rows, h, hd)).astype(np.float32) for h in (heads, kv, kv))
    slots = rng.permutation(max_seq)[:rows].astype(np.int32)
    pos = rng.integers(0, 40, rows).astype(np.int32)
    pos[2], slots[4] = 40, -1  # a position outside the table, a padding row
    qd, kd, vd, sd, pd = (DeviceArray.from_host(mlb, gpu, a) for a in (q, k, v, slots, pos))
    a, b = (Cache(mlb, gpu, qtype, 1, 1, max_seq, kv, hd) for _ in range(2))
    q1, q2, k2 = (DeviceArray(mlb, gpu, x.shape) for x in (q, q, k))
    n, m = heads * hd, kv * hd
    mlb.call("mlb_kv_cache_write_rope", gpu, a.ref, 0, rows, None, sd.ptr, ctypes.byref(table), pd.ptr, qd.ptr, n, q1.ptr,
             n, heads, kd.ptr, m, vd.ptr, m)
    mlb.call("mlb_rope_rows", gpu, ctypes.byref(table), rows, pd.ptr, qd.ptr, n, q2.ptr, n, heads, kd.ptr, m, k2.ptr, m, kv)
    skip = slots.copy()
    skip[2] = -1
    skipd = DeviceArray.from_host(mlb, gpu, skip)
    mlb.call("mlb_kv_cache_write", gpu, b.ref, 0, rows, None, skipd.ptr, k2.ptr, m, vd.ptr, m)
    got = q1.download()
    assert np.isnan(got[2]).all()
    good = [r for r in range(rows) if r != 2]
    assert same_bits(got[good], q2.download()[good])
    for x, y in zip(a.planes(), b.planes()):
        assert np.array_equal(x, y)


def test_cache_unaligned_rows(mlb, gpu):
    """Rows at odd addresses and strides take the element-wise form, with the same bits."""
    kv, hd, rows = 2, 64, 6
    x = np.random.default_rng(2).standard_normal((rows, kv * hd + 3)).astype(np.float32)
    xd = DeviceArray.from_host(mlb, gpu, x)
    sd = DeviceArray.from_host(mlb, gpu, np.arange(rows, dtype=np.int32))
    back = DeviceArray(mlb, gpu, (rows, kv * hd + 5))
    for qtype in (F32, Q80, Q40):
        c = Cache(mlb, gpu, qtype, 1, 1, 8, kv, hd)
        mlb.call("mlb_kv_cache_write", gpu, c.ref, 0, rows, None, sd.ptr, xd.ptr + 4, kv * hd + 3, xd.ptr + 8, kv * hd + 3)
        k, v = c.read(0, None, list(range(rows)))
        flat = x.reshape(-1)
        rows_at = lambda off: np.stack([flat[off + r * (kv * hd + 3):][:kv * hd] for r in range(rows)])  # noqa: E731
        want_k = ref.held(rows_at(1)[:, :].reshape(rows, kv, hd), qtype)
        assert same_bits(k, want_k)
        mlb.call("mlb_kv_cache_read", gpu, c.ref, 0, rows, None, sd.ptr, back.ptr + 4, kv * hd + 5, None, 0)
        got = back.download().reshape(-1)
        got = np.stack([got[1 + r * (kv * hd + 5):][:kv * hd] for r in range(rows)])
        assert same_bits(got.reshape(rows, kv, hd), want_k)


# ------------------------------------------------------------------------------------------------ attention
def random_tree(rng, tokens):
    words = (tokens + 63) // 64
    seen = np.zeros((tokens, words * 64), np.uint8)
    for i in range(tokens):
        p = int(rng.integers(max(-1, i - 5), i)) if i else -1
        if p >= 0:
            seen[i] = seen[p]
        seen[i, i] = 1
    return np.packbits(seen, axis=-1, bitorder="little").view(np.uint64)


def run_attention(lib, dev, c, layer, q, seqs, lens, max_len, mask, scale=0.0, pad=0):
    b, t, heads, hd = q.shape
    n = heads * hd
    rows = np.full((b * t, n + pad), np.nan, np.float32)
    rows[:, :n] = q.reshape(b * t, n)
    qd = DeviceArray.from_host(lib, dev, rows)
    od = DeviceArray.from_host(lib, dev, np.full((b * t, n + pad), 7.0, np.float32))
    ld = DeviceArray.from_host(lib, dev, np.asarray(lens, np.int32))
    sd = DeviceArray.from_host(lib, dev, np.asarray(seqs, np.int32)) if seqs is not None else None
    md = DeviceArray.from_host(lib, dev, mask) if mask is not None else None
    lib.call("mlb_attention_tree", dev, c.ref, layer, b, t, sd.ptr if sd else None, ld.ptr, max_len,
             md.ptr if md else None, qd.ptr, n + pad, heads, scale, od.ptr, n + pad)
    out = od.download()
    assert (out[:, n:] == 7.0).all(), "the gap between output rows was written"
    return out[:, :n].reshape(b, t, heads, hd)


def assert_attention(got, want, weight, terms, what=""):
    tol = (2.0 ** -19 * terms + 2.0 ** -19) * weight
    err = np.abs(got.astype(np.float64) - want)
    assert np.isfinite(got).all(), what
    assert (err <= tol).all(), f"{what}: {int((err > tol).sum())} of {err.size} outside, worst {float((err / np.maximum(tol, 1e-300)).max()):.2f} times the bound"


def filled(lib, dev, rng, qtype, n_seqs, max_seq, kv, hd, layers=1, layer=0, k_scale=1.0):
    c = Cache(lib, dev, qtype, n_seqs, layers, max_seq, kv, hd, fill=0)
    seqs, slots = np.repeat(np.arange(n_seqs), max_seq), np.tile(np.arange(max_seq), n_seqs)
    k = (k_scale * rng.standard_normal((n_seqs * max_seq, kv, hd))).astype(np.float32)
    v = rng.standard_normal((n_seqs * max_seq, kv, hd)).astype(np.float32)
    c.write(layer, seqs, slots, k, v)
    kk, vv = (ref.held(x, qtype).reshape(n_seqs, max_seq, kv, hd) for x in (k, v))
    return c, kk, vv


SHAPES = [(4, 2, 16), (14, 2, 64), (6, 6, 64), (10, 2, 80), (12, 4, 96), (32, 8, 128), (3, 1, 40), (8, 1, 160), (2, 2, 256),
          (24, 1, 128), (5, 5, 224)]


@pytest.mark.parametrize("qtype", [F32, Q80, Q40], ids=NAME.get)
@pytest.mark.parametrize("heads,kv,hd", SHAPES)
@pytest.mark.parametrize("tokens", [1, 3, 17, 70])
def test_tree_attention(mlb, gpu, qtype, heads, kv, hd, tokens):
    rng = np.random.default_rng(heads * 100 + hd + tokens)
    lens = [0, 1, 37, 64, 130, 300]
    n_seqs, max_seq = len(lens), 300 + tokens + 3
    c, k, v = filled(mlb, gpu, rng, qtype, n_seqs, max_seq, kv, hd, layers=2, layer=1)
    q = rng.standard_normal((n_seqs, tokens, heads, hd)).astype(np.float32)
    seqs = rng.permutation(n_seqs)
    mask = np.stack([random_tree(rng, tokens) for _ in range(n_seqs)]) if tokens > 1 else None
    got = run_attention(mlb, gpu, c, 1, q, seqs, lens, 300, mask, pad=4)
    want = ref.attention(q, k, v, lens, seqs, mask, hd ** -0.5, max_seq)
    assert_attention(got, *want, f"{NAME[qtype]} {heads}/{kv}x{hd} tokens {tokens}")


@pytest.mark.parametrize("qtype", [F32, Q80, Q40], ids=NAME.get)
@pytest.mark.parametrize("heads,kv,hd", [(14, 2, 64), (32, 8, 128), (6, 2, 7), (4, 1, 129)])
def test_chain_without_mask(mlb, gpu, qtype, heads, kv, hd):
    """No mask: a causal piece of a prompt; batch entries in order, odd head sizes and query addresses too."""
    rng = np.random.default_rng(hd)
    tokens, lens = 45, [0, 200]
    c, k, v = filled(mlb, gpu, rng, qtype, 2, 256, kv, hd)
    q = rng.standard_normal((2, tokens, heads, hd)).astype(np.float32)
    got = run_attention(mlb, gpu, c, 0, q, None, lens, 211, None, pad=1)
    assert_attention(got, *ref.attention(q, k, v, lens, [0, 1], None, hd ** -0.5, 256))


@pytest.mark.parametrize("qtype", [F32, Q80, Q40], ids=NAME.get)
@pytest.mark.parametrize("length,tokens", [(5000, 1), (4999, 9), (2047, 64)])
def test_long_and_split(mlb, gpu, qtype, length, tokens):
    """Contexts long enough to be split over CTAs and joined, peaked scores, an explicit scale."""
    rng = np.random.default_rng(length)
    heads, kv, hd, max_seq = 8, 2, 64, length + tokens
    c, k, v = filled(mlb, gpu, rng, qtype, 2, max_seq, kv, hd, k_scale=3.0)
    q = rng.standard_normal((2, tokens, heads, hd)).astype(np.float32)
    mask = np.stack([random_tree(rng, tokens) for _ in range(2)])
    lens = [length, length // 3]
    got = run_attention(mlb, gpu, c, 0, q, None, lens, length, mask, scale=0.2)
    assert_attention(got, *ref.attention(q, k, v, lens, [0, 1], mask, np.float64(np.float32(0.2)), max_seq))


@pytest.mark.parametrize("qtype", [F32, Q80, Q40], ids=NAME.get)
@pytest.mark.parametrize("hd", [64, 128, 160])
def test_rows_that_see_nothing_and_inactive_entries(mlb, gpu, qtype, hd):
    rng = np.random.default_rng(4)
    tokens, heads, kv = 4, 4, 2
    c, k, v = filled(mlb, gpu, rng, qtype, 4, 40, kv, hd)
    q = rng.standard_normal((5, tokens, heads, hd)).astype(np.float32)
    mask = np.stack([random_tree(rng, tokens) for _ in range(5)])
    mask[0, 1] = 0  # an empty row where nothing is committed
    mask[1, 2] = 0  # an empty mask over committed slots: those alone
    mask[2, 3] |= np.uint64(0xFFFFFFFFFFFFFF00)  # bits past the tokens mean nothing
    lens, seqs = [0, 9, 20, -1, 11], [0, 1, 2, 3, 9]
    got = run_attention(mlb, gpu, c, 0, q, seqs, lens, 30, mask)
    assert (got[0, 1] == 0).all() and (got[3] == 0).all() and (got[4] == 0).all()
    assert_attention(got, *ref.attention(q, k, v, lens, seqs, mask, hd ** -0.5, 40))


@pytest.mark.parametrize("qtype", [F32, Q80, Q40], ids=NAME.get)
@pytest.mark.parametrize("hd", [64, 128, 160])
@pytest.mark.parametrize("byte", [0xFF, 0x7C])
def test_unseen_slots_hold_anything(mlb, gpu, qtype, hd, byte):
    """Slots past the tokens, and drafted slots that some rows see and others do not, hold NaN, infinities or huge
    values: rows that do not see them are unchanged."""
    rng = np.random.default_rng(6)
    tokens, heads, kv, n = 6, 8, 2, 50
    c = Cache(mlb, gpu, qtype, 1, 1, 64, kv, hd, fill=byte)
    k, v = (rng.standard_normal((n + tokens, kv, hd)).astype(np.float32) for _ in range(2))
    keep = [s for s in range(n + tokens) if s != n + 2]  # drafted token 2 stays as the fill left it
    c.write(0, None, keep, k[keep], v[keep])
    mask = np.zeros((1, tokens, 1), np.uint64)
    for t in range(tokens):
        mask[0, t, 0] = sum(1 << j for j in range(t + 1) if j != 2)
    mask[0, 2, 0] |= np.uint64(4)
    q = rng.standard_normal((1, tokens, heads, hd)).astype(np.float32)
    got = run_attention(mlb, gpu, c, 0, q, None, [n], 60, mask)
    kk, vv = (np.zeros((1, 64, kv, hd), np.float32) for _ in range(2))
    kk[0, keep], vv[0, keep] = ref.held(k[keep], qtype), ref.held(v[keep], qtype)
    others = [t for t in range(tokens) if t != 2]
    want = [x[:, others] for x in ref.attention(q, kk, vv, [n], [0], mask, hd ** -0.5, 64)]
    assert_attention(got[:, others], *want)


@pytest.mark.parametrize("qtype", [F32, Q80, Q40], ids=NAME.get)
def test_lengths_past_the_bounds(mlb, gpu, qtype):
    """lens above max_len count as max_len; drafted slots past the cache do not exist."""
    rng = np.random.default_rng(7)
    c, k, v = filled(mlb, gpu, rng, qtype, 2, 100, 2, 64)
    q = rng.standard_normal((2, 5, 4, 64)).astype(np.float32)
    got = run_attention(mlb, gpu, c, 0, q, None, [70, 98], 60, None)
    assert_attention(got, *ref.attention(q, k, v, [60, 60], [0, 1], None, 0.125, 100))
    got = run_attention(mlb, gpu, c, 0, q, None, [98, 100], 1 << 30, None)
    assert_attention(got, *ref.attention(q, k, v, [98, 100], [0, 1], None, 0.125, 100))


@pytest.mark.parametrize("qtype", [F32, Q80, Q40], ids=NAME.get)
@pytest.mark.parametrize("k_mag,v_mag,q_mag", [(1e-4, 1e-4, 1e4), (30.0, 2e4, 0.05), (1.0, 1e-3, 1.0)])
def test_magnitudes(mlb, gpu, qtype, k_mag, v_mag, q_mag):
    """Small and large keys, values and queries keep the same relative accuracy."""
    rng = np.random.default_rng(9)
    tokens, heads, kv, hd, n = 5, 8, 2, 128, 200
    c = Cache(mlb, gpu, qtype, 1, 1, 256, kv, hd)
    k = (k_mag * rng.standard_normal((n + tokens, kv, hd))).astype(np.float32)
    v = (v_mag * rng.standard_normal((n + tokens, kv, hd)) * rng.choice([1.0, 1e-3], (n + tokens, 1, 1))).astype(np.float32)
    c.write(0, None, list(range(n + tokens)), k, v)
    q = (q_mag * rng.standard_normal((1, tokens, heads, hd))).astype(np.float32)
    kk, vv = (np.zeros((1, 256, kv, hd), np.float32) for _ in range(2))
    kk[0, :n + tokens], vv[0, :n + tokens] = ref.held(k, qtype), ref.held(v, qtype)
    got = run_attention(mlb, gpu, c, 0, q, None, [n], n, None)
    assert_attention(got, *ref.attention(q, kk, vv, [n], [0], None, hd ** -0.5, 256))


@pytest.mark.parametrize("qtype", [F32, Q80, Q40], ids=NAME.get)
def test_a_dominant_key_with_tiny_values(mlb, gpu, qtype):
    """One slot takes nearly all the weight and holds almost nothing: what the others add still counts."""
    rng = np.random.default_rng(10)
    heads, kv, hd, n = 4, 1, 64, 700
    k, v = (rng.standard_normal((n, kv, hd)).astype(np.float32) for _ in range(2))
    q = np.abs(rng.standard_normal((1, 1, heads, hd))).astype(np.float32)
    k[0], v[0] = 1.5, 1e-5
    c = Cache(mlb, gpu, qtype, 1, 1, 1024, kv, hd)
    c.write(0, None, list(range(n)), k, v)
    kk, vv = (np.zeros((1, 1024, kv, hd), np.float32) for _ in range(2))
    kk[0, :n], vv[0, :n] = ref.held(k, qtype), ref.held(v, qtype)
    got = run_attention(mlb, gpu, c, 0, q, None, [n - 1], n, None)
    assert_attention(got, *ref.attention(q, kk, vv, [n - 1], [0], None, hd ** -0.5, 1024))


def test_fp32_cache_is_the_batched_decode_layout(mlb, gpu):
    """tokens = 1 over an fp32 cache equals mlb_attention_decode_batched (1e-4 mixed, its tolerance)."""
    rng = np.random.default_rng(11)
    batch, heads, kv, hd, max_seq = 3, 14, 2, 64, 200
    c, k, v = filled(mlb, gpu, rng, F32, batch, max_seq, kv, hd, layers=2, layer=1)
    q = rng.standard_normal((batch, 1, heads, hd)).astype(np.float32)
    lens = [5, 150, 77]
    got = run_attention(mlb, gpu, c, 1, q, None, lens, 160, None)
    qd, od = DeviceArray.from_host(mlb, gpu, q), DeviceArray(mlb, gpu, q.shape)
    pd = DeviceArray.from_host(mlb, gpu, np.array(lens, np.int32))
    mlb.call("mlb_attention_decode_batched", gpu, batch, qd.ptr, c.desc.k, c.desc.v, 2, max_seq, 1, pd.ptr, 150, heads, kv,
             hd, od.ptr)
    other = od.download()
    assert (np.abs(got - other) <= 1e-4 * np.maximum(1, np.abs(other))).all()


@pytest.mark.parametrize("qtype", [F32, Q80], ids=NAME.get)
def test_offsets_past_32_bits(mlb, gpu, qtype):
    """The last sequence of a cache whose planes pass 2^32 bytes (and 2^31 elements for fp32)."""
    rng = np.random.default_rng(12)
    kv, hd, max_seq, n_seqs = 8, 128, 1 << 19, 9 if qtype == Q80 else 5
    c = Cache(mlb, gpu, qtype, n_seqs, 1, max_seq, kv, hd)
    assert c.plane_bytes > 1 << 32
    n, tokens = 500, 3
    k, v = (rng.standard_normal((n + tokens, kv, hd)).astype(np.float32) for _ in range(2))
    slots = list(range(n + tokens))
    c.write(0, [n_seqs - 1] * len(slots), slots, k, v)
    got_k, _ = c.read(0, [n_seqs - 1] * len(slots), slots)
    assert same_bits(got_k, ref.held(k, qtype))
    c.write(0, [n_seqs - 1], [max_seq - 1], k[:1], v[:1])
    assert same_bits(c.read(0, [n_seqs - 1], [max_seq - 1])[1], ref.held(v[:1], qtype))
    q = rng.standard_normal((1, tokens, 16, hd)).astype(np.float32)
    got = run_attention(mlb, gpu, c, 0, q, [n_seqs - 1], [n], n, None)
    kk, vv = (ref.held(x, qtype)[None] for x in (k, v))
    assert_attention(got, *ref.attention(q, kk, vv, [n], [0], None, hd ** -0.5, n + tokens))


def test_repeated_calls_and_changing_shapes(mlb, gpu):
    """Calls of different shapes in a row, then the first again: the same bits (workspaces hold nothing over)."""
    first = None
    for heads, kv, hd, n, tokens in [(32, 8, 128, 900, 5), (14, 2, 64, 40, 1), (16, 1, 128, 2500, 20), (32, 8, 128, 900, 5)]:
        g = np.random.default_rng(n + tokens)
        c, k, v = filled(mlb, gpu, g, Q80, 2, n + tokens, kv, hd)
        q = g.standard_normal((2, tokens, heads, hd)).astype(np.float32)
        runs = [run_attention(mlb, gpu, c, 0, q, None, [n, n // 2], n, None) for _ in range(3)]
        assert same_bits(runs[0], runs[1]) and same_bits(runs[0], runs[2])
        if first is None:
            first = runs[0]
    assert same_bits(first, runs[0])


@pytest.mark.parametrize("qtype", [Q80, Q40], ids=NAME.get)
@pytest.mark.parametrize("heads,kv,hd,tokens,length,n_seqs", [(16, 4, 32, 12, 700, 48), (64, 8, 64, 20, 400, 24),
                                                              (33, 1, 128, 1, 1500, 2)])
def test_many_items_to_a_cta(mlb, gpu, qtype, heads, kv, hd, tokens, length, n_seqs):
    """More row groups than SMs, several tiles each: the tensor-memory kernel's roles walk from item to item.  Every
    wait there is bounded; one that expired shows at the synchronisation."""
    rng = np.random.default_rng(length)
    max_seq = length + tokens
    c, k, v = filled(mlb, gpu, rng, qtype, n_seqs, max_seq, kv, hd)
    q = rng.standard_normal((n_seqs, tokens, heads, hd)).astype(np.float32)
    mask = np.stack([random_tree(rng, tokens) for _ in range(n_seqs)])
    lens = [length - 13 * i for i in range(n_seqs)]
    got = run_attention(mlb, gpu, c, 0, q, None, lens, length, mask)
    for _ in range(3):
        assert same_bits(got, run_attention(mlb, gpu, c, 0, q, None, lens, length, mask))
    mlb.sync(gpu)
    some = [0, n_seqs // 2, n_seqs - 1]
    want = ref.attention(q[some], k[some], v[some], [lens[i] for i in some], range(len(some)), mask[some], hd ** -0.5, max_seq)
    assert_attention(got[some], *want)


@pytest.mark.parametrize("qtype", [F32, Q80, Q40], ids=NAME.get)
@pytest.mark.parametrize("max_seq", [1, 5, 16, 31, 100, 129])
@pytest.mark.parametrize("heads,kv,tokens", [(2, 2, 1), (4, 1, 5), (24, 2, 7)])
def test_short_caches(mlb, gpu, qtype, max_seq, heads, kv, tokens):
    """Planes shorter than a unit or a tile of the matrix kernels, filled to their end; few rows and many."""
    rng = np.random.default_rng(max_seq)
    c, k, v = filled(mlb, gpu, rng, qtype, 3, max_seq, kv, 64)
    q = rng.standard_normal((3, tokens, heads, 64)).astype(np.float32)
    mask = np.stack([random_tree(rng, tokens) for _ in range(3)])
    lens = [max(0, max_seq - tokens), max_seq, 0]
    got = run_attention(mlb, gpu, c, 0, q, None, lens, max_seq, mask)
    assert_attention(got, *ref.attention(q, k, v, lens, range(3), mask, 0.125, max_seq))


@pytest.mark.parametrize("qtype", [F32, Q80, Q40], ids=NAME.get)
@pytest.mark.parametrize("hd", [32, 96, 128])
@pytest.mark.parametrize("byte", [0xFF, 0x7C, 0x77])  # fp16 scales: NaN, NaN, 30576
def test_many_rows_past_unseen_slots(mlb, gpu, qtype, hd, byte):
    """More than 32 rows per KV head: a drafted slot that only its own token sees holds NaN or huge values; a row that
    sees nothing, an empty entry and an inactive one are zero, the others unchanged."""
    rng = np.random.default_rng(hd + byte)
    tokens, heads, kv, n, max_seq = 9, 10, 2, 150, 192
    c = Cache(mlb, gpu, qtype, 4, 1, max_seq, kv, hd, fill=byte)
    k, v = (rng.standard_normal((2, n + tokens, kv, hd)).astype(np.float32) for _ in range(2))
    odd = n + 3
    for s in range(2):
        keep = [i for i in range(n + tokens) if s == 1 or i != odd]
        c.write(0, [s] * len(keep), keep, k[s, keep], v[s, keep])
    mask = np.zeros((4, tokens, 1), np.uint64)
    for t in range(tokens):
        mask[:, t, 0] = sum(1 << j for j in range(t + 1) if j != 3 or t == 3)
    mask[1, 6] = 0  # sees what is committed: nothing
    lens, seqs = [n, 0, 50, -1], [0, 1, 7, 0]
    q = rng.standard_normal((4, tokens, heads, hd)).astype(np.float32)
    got = run_attention(mlb, gpu, c, 0, q, seqs, lens, n, mask)
    assert (got[1, 6] == 0).all() and (got[2] == 0).all() and (got[3] == 0).all()
    kk, vv = (np.zeros((2, max_seq, kv, hd), np.float32) for _ in range(2))
    kk[:, :n + tokens], vv[:, :n + tokens] = ref.held(k, qtype), ref.held(v, qtype)
    kk[0, odd] = vv[0, odd] = 0
    want = ref.attention(q[:2], kk, vv, lens[:2], seqs[:2], mask[:2], hd ** -0.5, max_seq)
    others = [t for t in range(tokens) if t != 3]
    assert_attention(got[:1, others], *[x[:1, others] for x in want])
    assert_attention(got[1:2], *[x[1:2] for x in want])


@pytest.mark.parametrize("qtype", [F32, Q80, Q40], ids=NAME.get)
@pytest.mark.parametrize("k_mag,v_mag,q_mag", [(1e-4, 1e-4, 1e4), (30.0, 2e4, 0.05), (5e4, 1.0, 1e-5), (1.0, 1e-3, 1.0)])
def test_magnitudes_of_many_rows(mlb, gpu, qtype, k_mag, v_mag, q_mag):
    """As test_magnitudes, more than 32 rows per KV head; some tiles of 128 slots hold large scales, some do not."""
    rng = np.random.default_rng(13)
    tokens, heads, kv, hd, n = 7, 12, 2, 128, 700
    c = Cache(mlb, gpu, qtype, 1, 1, 768, kv, hd)
    size = np.where(np.arange(n + tokens) // 200 % 2, 1.0, 1e-3)[:, None, None]
    k = (k_mag * size * rng.standard_normal((n + tokens, kv, hd))).astype(np.float32)
    v = (v_mag * size * rng.standard_normal((n + tokens, kv, hd))).astype(np.float32)
    c.write(0, None, list(range(n + tokens)), k, v)
    q = (q_mag * rng.standard_normal((1, tokens, heads, hd))).astype(np.float32)
    kk, vv = (np.zeros((1, 768, kv, hd), np.float32) for _ in range(2))
    kk[0, :n + tokens], vv[0, :n + tokens] = ref.held(k, qtype), ref.held(v, qtype)
    got = run_attention(mlb, gpu, c, 0, q, None, [n], n, None)
    assert_attention(got, *ref.attention(q, kk, vv, [n], [0], None, hd ** -0.5, 768))


def test_empty_calls(mlb, gpu):
    c = Cache(mlb, gpu, Q80, 1, 1, 8, 1, 32)
    mlb.call("mlb_kv_cache_write", gpu, c.ref, 0, 0, None, None, None, 32, None, 32)
    mlb.call("mlb_kv_cache_read", gpu, c.ref, 0, 0, None, None, None, 32, None, 32)
    mlb.call("mlb_attention_tree", gpu, c.ref, 0, 0, 1, None, None, 0, None, None, 32, 1, 0.0, None, 32)
    mlb.call("mlb_attention_tree", gpu, c.ref, 0, 1, 0, None, None, 0, None, None, 32, 1, 0.0, None, 32)
    mlb.sync(gpu)


@pytest.mark.parametrize("qtype", [F32, Q80, Q40], ids=NAME.get)
@pytest.mark.parametrize("heads,kv", [(32, 8), (16, 16)])
@pytest.mark.parametrize("tokens,length", [(12, 20), (12, 100), (24, 90), (16, 1000)])
def test_a_linear_right_behind_attention(mlb, gpu, qtype, heads, kv, tokens, length):
    """The output projection queued right behind an attention call, both behind a longer kernel so that they run back
    to back: the bits of the same calls one by one.  The linear's first kernel is a programmatic dependent of the
    attention's last one; contexts of one unit (nothing to join) and longer ones, results alternating."""
    rng = np.random.default_rng(tokens + length)
    hd, dim = 64, 1024
    n = heads * hd
    c, _, _ = filled(mlb, gpu, rng, qtype, 1, length + tokens, kv, hd)
    up = lambda a: DeviceArray.from_host(mlb, gpu, a)  # noqa: E731
    qs = [up(rng.standard_normal((1, tokens, heads, hd)).astype(np.float32)) for _ in range(2)]
    weights, blocks = up(rng.standard_normal((dim, n)).astype(np.float32)), DeviceArray(mlb, gpu, (dim * n // 32 * 34,), np.uint8)
    mlb.call("mlb_quantize", gpu, Q80, weights.ptr, dim, n, blocks.ptr)
    lens, mask = up(np.array([length], np.int32)), up(random_tree(rng, tokens)[None])
    att, out = DeviceArray(mlb, gpu, (tokens, n)), [DeviceArray(mlb, gpu, (tokens, dim)) for _ in range(6)]
    big = DeviceArray(mlb, gpu, (1 << 31,), np.uint8)

    def attend(i):
        mlb.call("mlb_attention_tree", gpu, c.ref, 0, 1, tokens, None, lens.ptr, length, mask.ptr, qs[i % 2].ptr, n, heads, 0.0,
                 att.ptr, n)

    def project(i):
        mlb.call("mlb_quant_linear", gpu, Q80, att.ptr, blocks.ptr, dim * n // 32, tokens, n, dim, None, out[i].ptr)

    want = []
    for i in range(2):
        attend(i)
        mlb.sync(gpu)
        project(i)
        mlb.sync(gpu)
        want.append(out[i].download())
    assert np.isfinite(want[0]).all() and not same_bits(want[0], want[1])
    for _ in range(5):
        mlb.call("mlb_memset", gpu, att.ptr, 0xFF, att.nbytes)
        mlb.call("mlb_memset", gpu, big.ptr, 0, big.nbytes)
        for i in range(len(out)):
            attend(i)
            project(i)
        mlb.sync(gpu)
        for i, o in enumerate(out):
            assert same_bits(o.download(), want[i % 2]), i


@pytest.mark.parametrize("qtype", [F32, Q80, Q40], ids=NAME.get)
@pytest.mark.parametrize("heads,tokens", [(4, 2), (8, 4), (8, 9)])
@pytest.mark.parametrize("hd", [64, 128, 160])
@pytest.mark.parametrize("n", [40, 300])
@pytest.mark.parametrize("common,outlier", [(0.05, 1e4), (0.05, 1e5), (1.0, 1e5)])
@pytest.mark.parametrize("where", ["early", "block", "middle", "drafted"])
def test_a_large_value_costs_the_others_no_precision(mlb, gpu, qtype, heads, tokens, hd, n, common, outlier, where):
    """One slot (or one block of it) holds large values with next to no weight, or is a drafted one that a single token
    sees: the rest is as exact as without it.  The slot's weight is e^-24 or less, so that the 2^-38 that a weight is off
    by at most adds 2^-38 2e6 / 1 < 2^-17 of what the row sums, within (2^-19 24 + 2^-19) of it."""
    rng = np.random.default_rng(n + hd)
    c = Cache(mlb, gpu, qtype, 1, 1, n + tokens, 1, hd)
    k = (0.3 * rng.standard_normal((n + tokens, 1, hd))).astype(np.float32)
    v = (common * rng.standard_normal((n + tokens, 1, hd))).astype(np.float32)
    q = np.abs(rng.standard_normal((1, tokens, heads, hd))).astype(np.float32)
    at = {"early": 3, "block": 3, "middle": n // 2, "drafted": n + 1}[where]
    part = slice(32, 64) if where == "block" else slice(None)
    v[at, 0, part] = outlier * rng.standard_normal(v[at, 0, part].shape)
    k[at] = -24.0 / (q[0].sum(-1).min() * hd ** -0.5)
    mask = np.zeros((1, tokens, 1), np.uint64)
    for t in range(tokens):
        mask[0, t, 0] = 1 << t
    c.write(0, None, list(range(n + tokens)), k, v)
    kk, vv = ref.held(k, qtype)[None], ref.held(v, qtype)[None]
    got = run_attention(mlb, gpu, c, 0, q, None, [n], n, mask)
    assert_attention(got, *ref.attention(q, kk, vv, [n], [0], mask, hd ** -0.5, n + tokens))


@pytest.mark.parametrize("qtype", [Q80, Q40], ids=NAME.get)
@pytest.mark.parametrize("share", [0.004, 0.5])
def test_tiles_with_large_values_among_many_items(mlb, gpu, qtype, share):
    """Row groups that follow one another in a CTA, some tiles with large V scales and some without: a tile that is
    multiplied twice leaves the waits of the next ones in order (one that expired shows at the synchronisation)."""
    rng = np.random.default_rng(17)
    heads, kv, hd, tokens, length, n_seqs = 64, 8, 64, 20, 400, 24
    c = Cache(mlb, gpu, qtype, n_seqs, 1, length + tokens, kv, hd)
    k, v = (rng.standard_normal((n_seqs, length + tokens, kv, hd)).astype(np.float32) for _ in range(2))
    v *= np.where(rng.random(v.shape[:3]) < share, 4e4, 1.0)[..., None].astype(np.float32)
    for s in range(n_seqs):
        c.write(0, [s] * (length + tokens), list(range(length + tokens)), k[s], v[s])
    q = rng.standard_normal((n_seqs, tokens, heads, hd)).astype(np.float32)
    mask = np.stack([random_tree(rng, tokens) for _ in range(n_seqs)])
    lens = [length - 13 * i for i in range(n_seqs)]
    got = run_attention(mlb, gpu, c, 0, q, None, lens, length, mask)
    assert same_bits(got, run_attention(mlb, gpu, c, 0, q, None, lens, length, mask))
    mlb.sync(gpu)
    some = [0, n_seqs // 2, n_seqs - 1]
    want = ref.attention(q[some], ref.held(k[some], qtype), ref.held(v[some], qtype), [lens[i] for i in some],
                         range(len(some)), mask[some], hd ** -0.5, length + tokens)
    assert_attention(got[some], *want)


@pytest.mark.parametrize("heads,kv,hd,tokens", [(4, 2, 64, 1), (12, 2, 64, 3), (8, 1, 64, 6), (8, 2, 128, 4), (2, 1, 160, 3),
                                                (3, 1, 7, 2)])
def test_fp32_values_up_to_the_largest(mlb, gpu, heads, kv, hd, tokens):
    """Keys and values up to the largest that count as finite, the number below 2^128 (1 - 2^-12).  Each row sees one
    slot, so that no weighted sum of its own passes fp32."""
    rng = np.random.default_rng(hd)
    top = np.array([0x7F7FEFFF], np.uint32).view(np.float32)[0]
    c = Cache(mlb, gpu, F32, 1, 1, 40, kv, hd)
    shape = (tokens, kv, hd)
    k, v = ((top * rng.choice([1.0, -1.0, 0.51, 1 - 2.0 ** -12], shape)).astype(np.float32) for _ in range(2))
    c.write(0, None, list(range(tokens)), k, v)
    q = (1e-30 * rng.standard_normal((1, tokens, heads, hd))).astype(np.float32)
    scale = np.float32(1e-10)
    mask = np.array([[[1 << t] for t in range(tokens)]], np.uint64)
    got = run_attention(mlb, gpu, c, 0, q, None, [0], 0, mask, scale=float(scale))
    assert_attention(got, *ref.attention(q, k[None], v[None], [0], [0], mask, np.float64(scale), tokens))


@pytest.mark.parametrize("qtype", [F32, Q80, Q40], ids=NAME.get)
@pytest.mark.parametrize("heads,kv,hd,tokens", [(8, 2, 64, 1), (16, 2, 64, 3), (24, 2, 128, 5), (8, 2, 160, 3), (6, 2, 7, 2)])
@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("where", ["k", "v", "query"])
def test_committed_values_that_are_not_finite_stay_with_their_rows(mlb, gpu, qtype, heads, kv, hd, tokens, value, where):
    """A committed slot of one KV head of one sequence, or one head of one query token, holds an infinity or NaN: all
    other rows, of the same tile too, are as exact as ever, and calls after it as well."""
    rng = np.random.default_rng(hd + tokens)
    n, max_seq = 70, 96
    c = Cache(mlb, gpu, qtype, 2, 1, max_seq, kv, hd)
    k, v = (rng.standard_normal((2, n + tokens, kv, hd)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((2, tokens, heads, hd)).astype(np.float32)
    x = {"k": k, "v": v}
    if where != "query":
        x[where][0, 33, 1, 2] = value
    for s in range(2):
        c.write(0, [s] * (n + tokens), list(range(n + tokens)), k[s], v[s])
    if qtype != F32 and where != "query":  # the quantizer keeps infinities as a scale, NaN not at all: put the scale in
        at = ((0 * kv + 1) * max_seq + 33) * ((hd + 31) // 32) * 2
        bits = np.array([value], np.float16)
        mlb.call("mlb_memcpy_h2d", gpu, c.bufs[2 if where == "k" else 3].ptr + at, bits.ctypes.data, 2)
        mlb.sync(gpu)
    if where == "query":
        q[0, tokens - 1, heads // 2 + 1, 3] = value
    if where != "query":
        x[where][0, 33, 1, 2] = 0
    kk, vv = ref.held(k, qtype), ref.held(v, qtype)
    safe = np.where(np.isfinite(q), q, 0)
    want = ref.attention(safe, kk, vv, [n, n], [0, 1], None, hd ** -0.5, n + tokens)
    touched = np.zeros((2, tokens, heads), bool)
    if where == "query":
        touched[0, tokens - 1, heads // 2 + 1] = True
    else:
        touched[0, :, heads // 2:] = True
    got = run_attention(mlb, gpu, c, 0, q, None, [n, n], n, None)
    mlb.sync(gpu)
    assert_attention(got[~touched], *[w[~touched] for w in want])
    if where != "k" and not np.isneginf(value):  # an element of V or a whole query: nothing hides it
        assert not np.isfinite(got[touched]).all()


@pytest.mark.parametrize("qtype", [F32, Q80, Q40], ids=NAME.get)
@pytest.mark.parametrize("heads,tokens", [(4, 1), (8, 4), (12, 6)])
@pytest.mark.parametrize("k_mag,q_mag,scale", [(1e-4, 1e36, 1e-33), (3e4, 1e-36, 3e30), (3e4, 1e32, 1e-38)])
def test_queries_and_scales_of_any_size(mlb, gpu, qtype, heads, tokens, k_mag, q_mag, scale):
    """Queries near the ends of fp32's range, with scales that bring the scores back to the order of one."""
    rng = np.random.default_rng(heads)
    hd, n = 128, 150
    c = Cache(mlb, gpu, qtype, 1, 1, n + tokens, 1, hd)
    k = (k_mag * rng.standard_normal((n + tokens, 1, hd))).astype(np.float32)
    v = rng.standard_normal((n + tokens, 1, hd)).astype(np.float32)
    q = (q_mag * rng.standard_normal((1, tokens, heads, hd))).astype(np.float32)
    c.write(0, None, list(range(n + tokens)), k, v)
    kk, vv = ref.held(k, qtype)[None], ref.held(v, qtype)[None]
    factor = float(np.float32(scale))
    got = run_attention(mlb, gpu, c, 0, q, None, [n], n, None, scale=factor)
    assert_attention(got, *ref.attention(q, kk, vv, [n], [0], None, factor, n + tokens))


@pytest.mark.parametrize("qtype", [F32, Q80, Q40], ids=NAME.get)
@pytest.mark.parametrize("heads,tokens", [(4, 1), (8, 4), (12, 6)])
def test_a_single_slot_with_a_score_near_the_lowest(mlb, gpu, qtype, heads, tokens):
    """One visible slot has all the weight, whatever its score: -64 q k down to -2.2e38 (-3.2e38 in powers of two)."""
    rng = np.random.default_rng(tokens)
    hd = 64
    c = Cache(mlb, gpu, qtype, 1, 1, 40, 1, hd)
    k = np.full((tokens, 1, hd), -1e5, np.float32)
    v = rng.standard_normal((tokens, 1, hd)).astype(np.float32)
    q = np.full((1, tokens, heads, hd), 2.2e38 / 64 / 1e5, np.float32)
    q[0, :, ::2] *= 0.6
    c.write(0, None, list(range(tokens)), k, v)
    mask = np.array([[[1 << t] for t in range(tokens)]], np.uint64)
    got = run_attention(mlb, gpu, c, 0, q, None, [0], 0, mask, scale=1.0)
    want = np.broadcast_to(ref.held(v, qtype)[:, 0][None, :, None], got.shape)
    assert (np.abs(got - want) <= 2.0 ** -19 * np.abs(want)).all()


# ------------------------------------------------------------------------------------------------ rows, further
def rows_of_planes(c):
    """The cache's planes as [n_seqs, n_layers, kv, slot, bytes] views of fresh downloads."""
    d, out = c.desc, []
    blocks, stored = (d.head_dim + 31) // 32, (d.max_seq_len + 7) // 8 * 8
    for i, p in enumerate(c.planes()):
        if d.type == F32:
            if i < 2:
                out.append(p.reshape(d.n_seqs, d.n_layers, d.max_seq_len, d.n_kv_heads, d.head_dim * 4).swapaxes(2, 3))
        else:
            width = blocks * (2 if i > 1 else 32 if d.type == Q80 else 16)
            out.append(p.reshape(d.n_seqs, d.n_layers, d.n_kv_heads, stored, width))
    return out


@pytest.mark.parametrize("qtype", [F32, Q80, Q40], ids=NAME.get)
@pytest.mark.parametrize("kv,hd", [(2, 64), (3, 80), (1, 33)])
def test_a_write_touches_its_rows_alone(mlb, gpu, qtype, kv, hd):
    """Every byte of the planes outside the named slots of the named layer stays as it was."""
    rng = np.random.default_rng(hd)
    n_seqs, layers, max_seq, rows = 3, 2, 45, 67
    c = Cache(mlb, gpu, qtype, n_seqs, layers, max_seq, kv, hd, fill=0x5A)
    at = rng.permutation(n_seqs * max_seq)[:rows]
    seqs, slots = (at // max_seq).astype(np.int32), (at % max_seq).astype(np.int32)
    slots[[1, 5]], seqs[[2, 9]], slots[3], seqs[4] = -1, n_seqs, max_seq, -1
    k, v = (rng.standard_normal((rows, kv, hd)).astype(np.float32) for _ in range(2))
    c.write(1, seqs, slots, k, v)
    kept = (slots >= 0) & (slots < max_seq) & (seqs >= 0) & (seqs < n_seqs)
    for p in rows_of_planes(c):
        named = np.zeros(p.shape[:4], bool)
        named[seqs[kept], 1, :, slots[kept]] = True
        assert (p[~named] == 0x5A).all()
        assert (p[named] != 0x5A).any(axis=-1).all()
    got_k, got_v = c.read(1, seqs, slots)
    assert same_bits(got_k[kept], ref.held(k, qtype)[kept]) and same_bits(got_v[kept], ref.held(v, qtype)[kept])


@pytest.mark.parametrize("qtype", [F32, Q80, Q40], ids=NAME.get)
@pytest.mark.parametrize("layers,rows", [(1, 2401), (3, 803)])
def test_large_calls_of_rows(mlb, gpu, qtype, layers, rows):
    """More than 75776 blocks (two to a group of lanes), a remainder, skipped rows: write, rotate and write, read."""
    rng = np.random.default_rng(rows)
    kv, hd, heads, max_seq = 8, 128, 4, rows + 60
    assert layers * rows * kv * hd // 32 > 75776 and rows % 2
    slots = rng.permutation(max_seq)[:rows].astype(np.int32)
    skip = rng.random(rows) < 0.02
    slots[skip] = -1
    slots[-1] = max_seq
    kept = (slots >= 0) & (slots < max_seq)
    k, v = (rng.standard_normal((layers, rows, kv, hd)).astype(np.float32) for _ in range(2))
    up = lambda a: DeviceArray.from_host(mlb, gpu, a)  # noqa: E731
    kd, vd, sd, n = up(k), up(v), up(slots), kv * hd
    layer = capi.ALL_LAYERS if layers > 1 else 0
    c = Cache(mlb, gpu, qtype, 1, layers, max_seq, kv, hd, fill=0x33)
    mlb.call("mlb_kv_cache_write", gpu, c.ref, layer, rows, None, sd.ptr, kd.ptr, n, vd.ptr, n)
    for p in rows_of_planes(c):
        named = np.zeros(p.shape[:4], bool)
        named[:, :, :, slots[kept]] = True
        assert (p[~named] == 0x33).all()
    kr, vr = (DeviceArray.from_host(mlb, gpu, np.full(k.shape, 7, np.float32)) for _ in range(2))
    mlb.call("mlb_kv_cache_read", gpu, c.ref, layer, rows, None, sd.ptr, kr.ptr, n, vr.ptr, n)
    for got, x in ((kr.download(), k), (vr.download(), v)):
        assert same_bits(got[:, kept], ref.held(x, qtype)[:, kept]) and (got[:, ~kept] == 0).all()
    if layers > 1:
        return
    table, buf = make_table(mlb, gpu, max_seq, hd, 64, True)
    cs, pos = buf.download(), rng.integers(0, max_seq, rows).astype(np.int32)
    q = rng.standard_normal((rows, heads, hd)).astype(np.float32)
    qd, qo, pd = up(q), DeviceArray(mlb, gpu, q.shape), up(pos)
    mlb.call("mlb_kv_cache_write_rope", gpu, c.ref, 0, rows, None, sd.ptr, ctypes.byref(table), pd.ptr, qd.ptr, heads * hd,
             qo.ptr, heads * hd, heads, kd.ptr, n, vd.ptr, n)
    mlb.call("mlb_kv_cache_read", gpu, c.ref, 0, rows, None, sd.ptr, kr.ptr, n, vr.ptr, n)
    turn = lambda x: ref.rotate(x, cs[pos, :, 0], cs[pos, :, 1], 64, True)  # noqa: E731
    assert same_bits(qo.download(), turn(q))
    assert same_bits(kr.download()[0, kept], ref.held(turn(k[0]), qtype)[kept])
    assert same_bits(vr.download()[0, kept], ref.held(v[0], qtype)[kept])


@pytest.mark.parametrize("qtype", [F32, Q80, Q40], ids=NAME.get)
def test_unaligned_values(mlb, gpu, qtype):
    """V at odd addresses and strides, written and read."""
    kv, hd, rows, gap = 2, 64, 6, 3
    n = kv * hd
    x = np.random.default_rng(3).standard_normal((rows, n + gap)).astype(np.float32)
    xd = DeviceArray.from_host(mlb, gpu, x)
    sd = DeviceArray.from_host(mlb, gpu, np.arange(rows, dtype=np.int32))
    back = DeviceArray.from_host(mlb, gpu, np.full((rows, n + 5), 7, np.float32))
    c = Cache(mlb, gpu, qtype, 1, 1, 8, kv, hd)
    mlb.call("mlb_kv_cache_write", gpu, c.ref, 0, rows, None, sd.ptr, xd.ptr + 4, n + gap, xd.ptr + 8, n + gap)
    flat = x.reshape(-1)
    want = ref.held(np.stack([flat[2 + r * (n + gap):][:n] for r in range(rows)]).reshape(rows, kv, hd), qtype)
    assert same_bits(c.read(0, None, list(range(rows)))[1], want)
    mlb.call("mlb_kv_cache_read", gpu, c.ref, 0, rows, None, sd.ptr, None, 0, back.ptr + 4, n + 5)
    got = back.download().reshape(-1)
    assert same_bits(np.stack([got[1 + r * (n + 5):][:n] for r in range(rows)]).reshape(rows, kv, hd), want)
    for r in range(rows - 1):
        assert (got[1 + r * (n + 5) + n:1 + (r + 1) * (n + 5)] == 7).all()


def test_python_wrappers(mlb, gpu):
    """RopeTable and KvCache: rotate in place, write, read and attend give what the calls give."""
    rng = np.random.default_rng(21)
    heads, kv, hd, rows = 4, 2, 64, 5
    q, k, v = (rng.standard_normal((rows, h, hd)).astype(np.float32) for h in (heads, kv, kv))
    pos, slots = np.array([4, 0, 9, 2, 7], np.int32), np.arange(rows, dtype=np.int32)
    qd, kd, vd, pd, sd = (DeviceArray.from_host(mlb, gpu, a) for a in (q, k, v, pos, slots))
    table = RopeTable(mlb, gpu, 10, hd, 1e4, capi.ROPE_NEOX)
    cs = table.angles.download()
    table.rotate(rows, pd.ptr, qd.ptr, heads, kd.ptr, kv)
    turned = [ref.rotate(x, cs[pos, :, 0], cs[pos, :, 1], hd, True) for x in (q, k)]
    assert same_bits(qd.download(), turned[0]) and same_bits(kd.download(), turned[1])
    for qtype in (F32, Q80, Q40):
        c = KvCache(mlb, gpu, qtype, 1, 2, 24, kv, hd)
        c.write(1, rows, sd.ptr, kd.ptr, vd.ptr)
        kr, vr = DeviceArray(mlb, gpu, k.shape), DeviceArray(mlb, gpu, v.shape)
        c.read(1, rows, sd.ptr, kr.ptr, vr.ptr)
        kk, vv = ref.held(turned[1], qtype), ref.held(v, qtype)
        assert same_bits(kr.download(), kk) and same_bits(vr.download(), vv)
        lens, out = DeviceArray.from_host(mlb, gpu, np.zeros(1, np.int32)), DeviceArray(mlb, gpu, q.shape)
        c.attend(1, 1, rows, lens.ptr, 0, qd.ptr, heads, out.ptr)
        assert_attention(out.download()[None], *ref.attention(turned[0][None], kk[None], vv[None], [0], [0], None, hd ** -0.5, rows))


@pytest.mark.parametrize("qtype", [F32, Q80, Q40], ids=NAME.get)
@pytest.mark.parametrize("heads,tokens", [(4, 1), (8, 5)])
def test_a_long_context(mlb, gpu, qtype, heads, tokens):
    """40000 slots of one KV head, cut over every CTA."""
    rng = np.random.default_rng(heads)
    hd, n = 64, 40000
    c, k, v = filled(mlb, gpu, rng, qtype, 1, n + tokens, 1, hd, k_scale=2.0)
    q = rng.standard_normal((1, tokens, heads, hd)).astype(np.float32)
    got = run_attention(mlb, gpu, c, 0, q, None, [n], n, None)
    assert_attention(got, *ref.attention(q, k, v, [n], [0], None, hd ** -0.5, n + tokens))


def test_calls_in_a_row_share_the_workspace(mlb, gpu):
    """Attention calls of different shapes queued behind a longer kernel, no download between: the bits of each alone."""
    rng = np.random.default_rng(31)
    shapes = [(Q80, 32, 8, 128, 900, 5), (F32, 14, 2, 64, 3000, 3), (Q40, 16, 1, 128, 2500, 20), (Q80, 4, 1, 64, 5000, 1)]
    up = lambda a: DeviceArray.from_host(mlb, gpu, a)  # noqa: E731
    calls = []
    for qtype, heads, kv, hd, n, tokens in shapes:
        c, _, _ = filled(mlb, gpu, rng, qtype, 1, n + tokens, kv, hd)
        q = up(rng.standard_normal((tokens, heads * hd)).astype(np.float32))
        outs = [DeviceArray(mlb, gpu, (tokens, heads * hd)) for _ in range(3)]
        calls.append((c, tokens, up(np.array([n], np.int32)), n, q, heads, heads * hd, outs))

    def attend(call, out):
        c, tokens, lens, n, q, heads, width, _ = call
        mlb.call("mlb_attention_tree", gpu, c.ref, 0, 1, tokens, None, lens.ptr, n, None, q.ptr, width, heads, 0.0, out.ptr, width)

    want = []
    for call in calls:
        attend(call, call[-1][0])
        want.append(call[-1][0].download())
    big = DeviceArray(mlb, gpu, (1 << 31,), np.uint8)
    mlb.call("mlb_memset", gpu, big.ptr, 0, big.nbytes)
    for i in (1, 2):
        for call in calls:
            attend(call, call[-1][i])
    for call, w in zip(calls, want):
        assert same_bits(call[-1][1].download(), w) and same_bits(call[-1][2].download(), w)
