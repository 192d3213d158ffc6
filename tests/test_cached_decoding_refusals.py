"""Argument checks of mlb_rope_*, mlb_kv_cache_* and mlb_attention_tree: they come before any device work, so a
refused call needs no GPU.  The addresses are never read."""
import ctypes

import pytest

from mini_llama_b200 import capi

P = 1 << 20  # a 16-byte aligned address that nothing reads
BAD, RANGE, UNSUP = capi.MLB_ERR_INVALID_ARGUMENT, capi.MLB_ERR_OUT_OF_RANGE, capi.MLB_ERR_UNSUPPORTED


@pytest.fixture(scope="module")
def lib():
    from mini_llama_b200 import build
    return capi.load(build.build())


def cache(**kw):
    c = dict(type=capi.Q8_0, n_seqs=2, n_layers=2, max_seq_len=64, n_kv_heads=2, head_dim=64, k=P, v=P, k_scale=P, v_scale=P)
    c.update(kw)
    return capi.KvCache(**c)


def table(**kw):
    t = dict(n_positions=16, head_dim=64, rot_dim=64, rope_type=capi.ROPE_NEOX, cos_sin=P)
    t.update(kw)
    return capi.RopeTable(**t)


def ref(x):
    return ctypes.byref(x) if x is not None else None


def refused(lib, want, text, name, *args):
    assert lib.raw(name, *args) == want, lib.last_error()
    assert name in lib.last_error() and text in lib.last_error()


@pytest.mark.parametrize("change,want,text", [
    (dict(type=capi.Q4_1), UNSUP, "F32, Q8_0 or Q4_0"), (dict(type=9), UNSUP, "F32, Q8_0 or Q4_0"),
    (dict(n_seqs=0), BAD, "positive"), (dict(max_seq_len=-1), BAD, "positive"), (dict(n_kv_heads=0), BAD, "positive"),
    (dict(head_dim=0), BAD, "positive"), (dict(n_layers=0), BAD, "positive"), (dict(k=None), BAD, "empty"),
    (dict(v_scale=None), BAD, "scales are null"), (dict(v=P + 8), BAD, "16-byte"), (dict(k_scale=P + 2), BAD, "16-byte"),
    (dict(type=capi.F32, k=P + 2), BAD, "4-byte"), (dict(head_dim=5000), UNSUP, "too large")])
def test_cache_descriptor(lib, change, want, text):
    c = cache(**change)
    refused(lib, want, text, "mlb_kv_cache_write", 0, ref(c), 0, 1, P, P, P, 9999, P, 9999)
    refused(lib, want, text, "mlb_kv_cache_read", 0, ref(c), 0, 1, P, P, P, 9999, P, 9999)
    refused(lib, want, text, "mlb_attention_tree", 0, ref(c), 0, 1, 1, P, P, 8, None, P, 9999, 2, 0.0, P, 9999)


@pytest.mark.parametrize("kw,want,text", [
    (dict(cache=None), BAD, "cache is null"), (dict(layer=2), RANGE, "layer out of range"),
    (dict(layer=-2), RANGE, "layer out of range"), (dict(rows=-1), BAD, "row count"), (dict(slots=None), BAD, "slots is null"),
    (dict(k=None), BAD, "k or v is null"), (dict(v=None), BAD, "k or v is null"), (dict(ks=127), BAD, "stride"),
    (dict(vs=0), BAD, "stride")])
def test_write(lib, kw, want, text):
    a = dict(cache=cache(), layer=0, rows=1, slots=P, k=P, ks=128, v=P, vs=128)
    a.update(kw)
    refused(lib, want, text, "mlb_kv_cache_write", 0, ref(a["cache"]), a["layer"], a["rows"], None, a["slots"], a["k"], a["ks"],
            a["v"], a["vs"])


def test_read(lib):
    c = cache()
    refused(lib, BAD, "k and v are null", "mlb_kv_cache_read", 0, ref(c), 0, 1, None, P, None, 0, None, 0)
    refused(lib, BAD, "stride", "mlb_kv_cache_read", 0, ref(c), 0, 1, None, P, P, 64, None, 0)
    refused(lib, RANGE, "layer", "mlb_kv_cache_read", 0, ref(c), 5, 1, None, P, P, 128, None, 0)


@pytest.mark.parametrize("kw,want,text", [
    (dict(rot_dim=3), BAD, "rot_dim"), (dict(rot_dim=0), BAD, "rot_dim"), (dict(rot_dim=66), BAD, "rot_dim"),
    (dict(n_positions=0), BAD, "positive"), (dict(rope_type=2), BAD, "rope type"), (dict(cos_sin=None), BAD, "empty"),
    (dict(cos_sin=P + 8), BAD, "16-byte")])
def test_rope_table(lib, kw, want, text):
    t = table(**kw)
    refused(lib, want, text, "mlb_rope_rows", 0, ref(t), 1, P, P, 256, P, 256, 4, P, 128, P, 128, 2)
    refused(lib, want, text, "mlb_rope_table_fill", 0, ref(t), 1e4, None)
    refused(lib, want, text, "mlb_kv_cache_write_rope", 0, ref(cache()), 0, 1, P, P, ref(t), P, P, 256, P, 256, 4, P, 128, P, 128)


@pytest.mark.parametrize("kw,text", [
    (dict(scaling=7), "scaling"), (dict(factor=0.5), "factor"), (dict(factor=float("nan")), "factor"),
    (dict(scaling=capi.ROPE_SCALE_YARN, original_positions=0), "original_positions"),
    (dict(scaling=capi.ROPE_SCALE_WAVELENGTH, fast=1.0, slow=4.0), "slow < fast"),
    (dict(scaling=capi.ROPE_SCALE_YARN, attention_factor=-1.0), "attention factor")])
def test_rope_scale(lib, kw, text):
    s = dict(scaling=capi.ROPE_SCALE_LINEAR, factor=2.0, original_positions=64)
    s.update(kw)
    refused(lib, BAD, text, "mlb_rope_table_fill", 0, ref(table()), 1e4, ref(capi.RopeScale(**s)))


def test_rope_rows(lib):
    t = table()
    name = "mlb_rope_rows"
    refused(lib, BAD, "rope table is null", name, 0, None, 1, P, P, 256, P, 256, 4, P, 128, P, 128, 2)
    refused(lib, BAD, "row count", name, 0, ref(t), -1, P, P, 256, P, 256, 4, P, 128, P, 128, 2)
    refused(lib, BAD, "positions", name, 0, ref(t), 1, None, P, 256, P, 256, 4, P, 128, P, 128, 2)
    refused(lib, BAD, "q is null", name, 0, ref(t), 1, P, None, 256, P, 256, 4, P, 128, P, 128, 2)
    refused(lib, BAD, "k stride", name, 0, ref(t), 1, P, P, 256, P, 256, 4, P, 100, P, 128, 2)
    refused(lib, BAD, "equal strides", name, 0, ref(t), 1, P, P, 256, P, 512, 4, P, 128, P, 128, 2)
    refused(lib, BAD, "head count", name, 0, ref(t), 1, P, P, 256, P, 256, -4, P, 128, P, 128, 2)
    refused(lib, BAD, "theta", "mlb_rope_table_fill", 0, ref(t), -1.0, None)


def test_write_rope(lib):
    name = "mlb_kv_cache_write_rope"
    refused(lib, BAD, "different head_dim", name, 0, ref(cache()), 0, 1, P, P, ref(table(head_dim=128)), P, P, 512, P, 512, 4,
            P, 128, P, 128)
    refused(lib, RANGE, "layer", name, 0, ref(cache()), capi.ALL_LAYERS, 1, P, P, ref(table()), P, P, 256, P, 256, 4, P, 128,
            P, 128)
    refused(lib, BAD, "positions", name, 0, ref(cache()), 0, 1, P, P, ref(table()), None, P, 256, P, 256, 4, P, 128, P, 128)


@pytest.mark.parametrize("kw,want,text", [
    (dict(cache=None), BAD, "cache is null"), (dict(layer=2), RANGE, "layer"), (dict(layer=-1), RANGE, "layer"),
    (dict(batch=-1), BAD, "negative"), (dict(tokens=-1), BAD, "negative"), (dict(max_len=-1), BAD, "max_len"),
    (dict(heads=3), BAD, "multiple"), (dict(heads=0), BAD, "multiple"), (dict(lens=None), BAD, "null"),
    (dict(q=None), BAD, "null"), (dict(out=None), BAD, "null"), (dict(qs=255), BAD, "stride"), (dict(os=255), BAD, "stride"),
    (dict(scale=-1.0), BAD, "scale"), (dict(scale=float("inf")), BAD, "scale"), (dict(seqs=None, batch=3), BAD, "sequences"),
    (dict(cache=cache(head_dim=257), qs=9999, os=9999), UNSUP, "256"), (dict(batch=1 << 20, tokens=1 << 12), UNSUP, "too many")])
def test_attention(lib, kw, want, text):
    a = dict(cache=cache(), layer=0, batch=1, tokens=1, seqs=P, lens=P, max_len=8, mask=None, q=P, qs=256, heads=4, scale=0.0,
             out=P, os=256)
    a.update(kw)
    refused(lib, want, text, "mlb_attention_tree", 0, ref(a["cache"]), a["layer"], a["batch"], a["tokens"], a["seqs"], a["lens"],
            a["max_len"], a["mask"], a["q"], a["qs"], a["heads"], a["scale"], a["out"], a["os"])


@pytest.mark.parametrize("qtype,hd,plane,scale", [(capi.F32, 80, 80 * 4 * 13, 0), (capi.Q8_0, 80, 96 * 16, 3 * 2 * 16),
                                                  (capi.Q4_0, 64, 32 * 16, 2 * 2 * 16)])
def test_bytes(lib, qtype, hd, plane, scale):
    """max_seq_len 13 is stored as 16 slots in a quantized cache."""
    c = cache(type=qtype, head_dim=hd, max_seq_len=13, k=None)
    p, s = ctypes.c_size_t(), ctypes.c_size_t()
    lib.call("mlb_kv_cache_bytes", ref(c), ctypes.byref(p), ctypes.byref(s))
    assert (p.value, s.value) == (plane * 2 * 2 * 2, scale * 2 * 2 * 2)


@pytest.mark.parametrize("which,text", [("seqs", "seqs is not 4-byte"), ("slots", "slots is not 4-byte"), ("k", "k is not 4-byte"),
                                        ("v", "v is not 4-byte")])
def test_rows_off_their_boundary(lib, which, text):
    """Pointers that are not on their elements' boundary are refused, not sent to the device."""
    a = dict(seqs=P, slots=P, k=P, v=P)
    a[which] += 2
    for name in ("mlb_kv_cache_write", "mlb_kv_cache_read"):
        refused(lib, BAD, text, name, 0, ref(cache()), 0, 1, a["seqs"], a["slots"], a["k"], 128, a["v"], 128)
    refused(lib, BAD, text, "mlb_kv_cache_write_rope", 0, ref(cache()), 0, 1, a["seqs"], a["slots"], ref(table()), P, P, 256, P,
            256, 4, a["k"], 128, a["v"], 128)


@pytest.mark.parametrize("which,text", [("positions", "positions"), ("q", "q is not"), ("q_out", "q output"), ("k", "k is not"),
                                        ("k_out", "k output")])
def test_rotated_rows_off_their_boundary(lib, which, text):
    a = dict(positions=P, q=P, q_out=4 * P, k=P, k_out=4 * P)
    a[which] += 1
    refused(lib, BAD, text, "mlb_rope_rows", 0, ref(table()), 1, a["positions"], a["q"], 256, a["q_out"], 256, 4, a["k"], 128,
            a["k_out"], 128, 2)
    refused(lib, BAD, "positions", "mlb_kv_cache_write_rope", 0, ref(cache()), 0, 1, P, P, ref(table()), P + 2, P, 256, P, 256, 4,
            P, 128, P, 128)


@pytest.mark.parametrize("which,step,text", [("seqs", 2, "seqs is not 4-byte"), ("lens", 1, "lens is not 4-byte"),
                                             ("mask", 4, "mask is not 8-byte"), ("q", 2, "q is not 4-byte"),
                                             ("out", 2, "out is not 4-byte")])
def test_attention_off_its_boundary(lib, which, step, text):
    a = dict(seqs=P, lens=P, mask=P, q=P, out=P)
    a[which] += step
    refused(lib, BAD, text, "mlb_attention_tree", 0, ref(cache()), 0, 1, 2, a["seqs"], a["lens"], 8, a["mask"], a["q"], 256, 4, 0.0,
            a["out"], 256)
