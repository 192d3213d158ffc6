"""Workloads of the cached-decoding operators: rotary positions for rows, the quantised KV cache (write, read
back) and attention for drafted tokens over it, with their plain forms.

A case is a dict of sizes.  prepare() makes its inputs, run() is one call as a decoding program makes it (with
`own` the library's kernels, else elementary torch operations in fp32), exact() the definition in 64 bits, work()
what the call cannot do without.  Sequences of a batch hold different numbers of tokens, from `min_len` to `len`
in even steps, in an order drawn from the seed.
"""
import ctypes

import numpy as np
import torch

own = False

DEV = "cuda"
F32, Q8, Q4 = "f32", "q8_0", "q4_0"
BITS = {F32: 32, Q8: 8, Q4: 4}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one token of each of 32 sequences, Llama-style heads, positions up to 32 K
        {"name": "rope_step", "op": "rope", "rows": 32, "heads": 32, "kv_heads": 8, "head_dim": 128, "rot_dim": 128,
         "neox": True, "positions": 32768},
        # a long prompt, half of each head rotated, q and k still inside the fused projection's rows
        {"name": "rope_prompt_partial", "op": "rope", "rows": 4096, "heads": 32, "kv_heads": 32, "head_dim": 128,
         "rot_dim": 64, "neox": False, "positions": 8192},
        # one token of each of 64 sequences into an 8-bit cache, and those rows read back
        {"name": "cache_step_q8", "op": "cache", "type": Q8, "batch": 64, "tokens": 1, "kv_heads": 32, "head_dim": 128,
         "capacity": 1024},
        # the drafted tokens of 8 sequences: q and k rotated, k and v written in one call
        {"name": "cache_rope_tree_q8", "op": "cache_rope", "type": Q8, "batch": 8, "tokens": 24, "heads": 14,
         "kv_heads": 2, "head_dim": 64, "rot_dim": 64, "neox": True, "capacity": 4096},
        # a 4 K prompt into a 4-bit cache, and read back
        {"name": "cache_prompt_q4", "op": "cache", "type": Q4, "batch": 1, "tokens": 4096, "kv_heads": 8,
         "head_dim": 128, "capacity": 8192},
        # a stored prefix of 32 K tokens read back (to be moved or inspected)
        {"name": "cache_read_q8", "op": "read", "type": Q8, "batch": 1, "tokens": 32768, "kv_heads": 8, "head_dim": 128,
         "capacity": 32768},
        # the smallest decode call: one sequence, one token, a short context
        {"name": "attn_short_q8", "op": "attention", "type": Q8, "batch": 1, "tokens": 1, "tree": False, "heads": 14,
         "kv_heads": 2, "head_dim": 64, "len": 131, "min_len": 131, "capacity": 256},
        # a batch of ordinary decode steps, sequences of very different lengths
        {"name": "attn_batch_q8", "op": "attention", "type": Q8, "batch": 32, "tokens": 1, "tree": False, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "len": 8192, "min_len": 500, "capacity": 8448},
        # a long context in 4 bits, one token
        {"name": "attn_long_q4", "op": "attention", "type": Q4, "batch": 4, "tokens": 1, "tree": False, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "len": 32768, "min_len": 32768, "capacity": 33024},
        # one sequence's tree of 16 drafted tokens, checked in one call
        {"name": "attn_tree_q8", "op": "attention", "type": Q8, "batch": 1, "tokens": 16, "tree": True, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "len": 8191, "min_len": 8191, "capacity": 8448},
        # large trees for a batch: the case bound by arithmetic
        {"name": "attn_tree_batch_q4", "op": "attention", "type": Q4, "batch": 16, "tokens": 61, "tree": True,
         "heads": 32, "kv_heads": 8, "head_dim": 128, "len": 4096, "min_len": 1024, "capacity": 4352},
        # drafted tokens over the cache as the decode session holds it, 32-bit values
        {"name": "attn_tree_f32", "op": "attention", "type": F32, "batch": 8, "tokens": 7, "tree": True, "heads": 14,
         "kv_heads": 2, "head_dim": 64, "len": 16384, "min_len": 2000, "capacity": 16640},
    ]


HEADS = [(4, 2, 16), (14, 2, 64), (12, 12, 64), (20, 4, 80), (32, 8, 128), (32, 32, 128), (16, 1, 128)]


def _spread(rng, low, high):
    """A whole number of low..high, even over its logarithm."""
    return max(low, min(high, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    heads, kv, hd = rng.choice(HEADS)
    op = rng.choice(["rope", "cache", "cache_rope", "read", "attention", "attention", "attention", "attention"])
    c = {"op": op, "kv_heads": kv, "head_dim": hd}
    if op == "rope":
        c |= {"rows": _spread(rng, 1, 4096), "heads": heads, "rot_dim": rng.choice([hd, hd // 2]),
              "neox": rng.random() < 0.5, "positions": _spread(rng, 64, 32768)}
    elif op in ("cache", "cache_rope", "read"):
        batch = _spread(rng, 1, 64)
        tokens = _spread(rng, 1, 4096 // batch)
        c |= {"type": rng.choice([Q8, Q4]), "batch": batch, "tokens": tokens, "capacity": tokens + _spread(rng, 8, 1024)}
        if op == "cache_rope":
            c |= {"heads": heads, "rot_dim": rng.choice([hd, hd // 2]), "neox": rng.random() < 0.5}
    else:
        batch = _spread(rng, 1, 32)
        tree = rng.random() < 0.6
        tokens = _spread(rng, 2, 80) if tree else rng.choice([1, 1, 1, _spread(rng, 2, 80)])
        kind = rng.choice([Q8, Q8, Q4, F32])
        most = min(32768, (1 << 30) // (BITS[kind] * batch * kv * hd), (1 << 26) // (batch * heads * tokens))
        length = _spread(rng, 1, max(2, most))
        c |= {"type": kind, "batch": batch, "tokens": tokens, "tree": tree, "heads": heads,
              "len": length, "min_len": rng.randint(0, length), "capacity": length + tokens + rng.randint(0, 64)}
    return c


# ------------------------------------------------------------------------------------------------ inputs
def _lens(case):
    b, lo, hi = case["batch"], case["min_len"], case["len"]
    return [hi - (i * (hi - lo)) // max(1, b - 1) for i in range(b)]


def _padded(head_dim):
    return (head_dim + 31) // 32 * 32


def _stored(case):
    """Slots that a quantised cache holds for each sequence: the capacity, rounded up to 8."""
    return (case["capacity"] + 7) // 8 * 8


def _rope_table(positions, rot_dim, theta=10000.0):
    """(cos, sin) pairs [positions][rot_dim / 2][2]."""
    i = torch.arange(rot_dim // 2, device=DEV, dtype=torch.float64)
    angle = torch.arange(positions, device=DEV, dtype=torch.float64)[:, None] * theta ** (-2.0 * i / rot_dim)
    return torch.stack((angle.cos(), angle.sin()), -1).float().contiguous()


def _empty_cache(case):
    """K and V planes of a cache (and their scales), zero."""
    b, kv, hd, kind = case["batch"], case["kv_heads"], case["head_dim"], case["type"]
    if kind == F32:  # [sequence][layer][slot][KV head][head_dim]
        return [torch.zeros(b, 1, case["capacity"], kv, hd, device=DEV) for _ in "kv"], [None, None]
    hp = _padded(hd)  # [sequence][layer][KV head][slot][quants of the padded head]
    planes = [torch.zeros(b, 1, kv, _stored(case), hp * BITS[kind] // 8, dtype=torch.int8 if kind == Q8 else torch.uint8,
                          device=DEV) for _ in "kv"]
    return planes, [torch.zeros(b, 1, kv, _stored(case), hp // 32, dtype=torch.float16, device=DEV) for _ in "kv"]


def _filled_cache(case, g):
    """A cache with N(0, 1) keys and values in every slot."""
    b, kv, hd, kind = case["batch"], case["kv_heads"], case["head_dim"], case["type"]
    planes, scales = _empty_cache(case)
    for which in range(2):
        for s in range(b):
            n = case["capacity"]
            x = torch.randn(n, kv, hd, device=DEV, generator=g)
            if kind == F32:
                planes[which][s, 0] = x
            else:
                q, d = _quantise(x, kind)
                planes[which][s, 0, :, :n] = q.transpose(0, 1)
                scales[which][s, 0, :, :n] = d.transpose(0, 1)
    return planes, scales


def _tree_masks(case, rng):
    """Bit j of row t: drafted token t sees drafted token j (its ancestors and itself), [batch][tokens][words] int64."""
    b, t = case["batch"], case["tokens"]
    seen = np.zeros((b, t, (t + 63) // 64 * 64), dtype=np.uint8)
    for s in range(b):
        for i in range(t):
            parent = rng.integers(max(-1, i - 8), i) if i else -1
            if parent >= 0:
                seen[s, i] = seen[s, parent]
            seen[s, i, i] = 1
    words = np.packbits(seen, axis=-1, bitorder="little").view(np.int64)
    return torch.from_numpy(words.copy()).to(DEV)


def _device_state(s, case):
    """What the library's calls take besides the tensors: the descriptors."""
    from mini_llama_b200 import capi
    s["lib"] = lib = capi.load()
    lib.call("mlb_set_device", 0)
    if "table" in s:
        s["rope"] = capi.RopeTable(n_positions=s["table"].shape[0], head_dim=case["head_dim"], rot_dim=case["rot_dim"],
                                   rope_type=capi.ROPE_NEOX if case["neox"] else capi.ROPE_NORMAL,
                                   cos_sin=s["table"].data_ptr())
    if "planes" in s:
        kind = {F32: capi.F32, Q8: capi.Q8_0, Q4: capi.Q4_0}[case["type"]]
        at = [p.data_ptr() if p is not None else None for p in s["planes"] + s["scales"]]
        s["cache"] = capi.KvCache(type=kind, n_seqs=case["batch"], n_layers=1, max_seq_len=case["capacity"],
                                  n_kv_heads=case["kv_heads"], head_dim=case["head_dim"], k=at[0], v=at[1],
                                  k_scale=at[2], v_scale=at[3])


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    rng = np.random.default_rng(seed)
    kv, hd, op = case["kv_heads"], case["head_dim"], case["op"]
    s = {"case": case}
    if op == "rope":
        rows, heads = case["rows"], case["heads"]
        s["table"] = _rope_table(case["positions"], case["rot_dim"])
        s["positions"] = torch.randint(0, case["positions"], (rows,), device=DEV, generator=g, dtype=torch.int32)
        s["qkv"] = torch.randn(rows, heads + 2 * kv, hd, device=DEV, generator=g)  # a fused projection's rows
        s["q"], s["k"] = s["qkv"][:, :heads], s["qkv"][:, heads:heads + kv]
        s["q_out"] = torch.empty(rows, heads, hd, device=DEV)
        s["k_out"] = torch.empty(rows, kv, hd, device=DEV)
    elif op in ("cache", "cache_rope", "read"):
        b, t = case["batch"], case["tokens"]
        rows = b * t
        s["planes"], s["scales"] = _filled_cache(case, g) if op == "read" else _empty_cache(case)
        first = torch.randint(0, case["capacity"] - t + 1, (b, 1), device=DEV, generator=g, dtype=torch.int32)
        s["slots"] = (first + torch.arange(t, device=DEV, dtype=torch.int32)).reshape(-1).contiguous()
        s["seqs"] = torch.arange(b, device=DEV, dtype=torch.int32).repeat_interleave(t)
        s["k_read"] = torch.empty(rows, kv, hd, device=DEV)
        s["v_read"] = torch.empty(rows, kv, hd, device=DEV)
        if op != "read":
            s["k"] = torch.randn(rows, kv, hd, device=DEV, generator=g)
            s["v"] = torch.randn(rows, kv, hd, device=DEV, generator=g)
        if op == "cache_rope":
            s["table"] = _rope_table(case["capacity"], case["rot_dim"])
            s["positions"] = s["slots"]
            s["q"] = torch.randn(rows, case["heads"], hd, device=DEV, generator=g)
            s["q_out"] = torch.empty_like(s["q"])
    else:
        b, t = case["batch"], case["tokens"]
        s["planes"], s["scales"] = _filled_cache(case, g)
        s["lens"] = torch.tensor([_lens(case)[i] for i in rng.permutation(b)], dtype=torch.int32, device=DEV)
        s["seqs"] = torch.from_numpy(rng.permutation(b).astype(np.int32)).to(DEV)
        s["mask"] = _tree_masks(case, rng) if case["tree"] else None
        s["q"] = torch.randn(b, t, case["heads"], hd, device=DEV, generator=g)
        s["out"] = torch.empty_like(s["q"])
    if own:
        _device_state(s, case)
    torch.cuda.synchronize()
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _half_up(x):
    """x >= 0 rounded to fp16's grid, halves up (the rounding of the framework's quantiser), as fp32."""
    normal = ((x.view(torch.int32) + 0x1000) & ~0x1FFF).view(torch.float32)
    return torch.where(x < 2.0 ** -14, torch.floor(x * 2.0 ** 24 + 0.5) * 2.0 ** -24, normal)


def _round_away(y):
    """y rounded to whole numbers, halves away from zero."""
    whole = torch.trunc(y)
    return whole + torch.sign(y) * ((y - whole).abs() >= 0.5)


def _quantise(x, kind):
    """x [..., head_dim] in blocks of 32: (quants as stored, fp16 scales)."""
    x = torch.nn.functional.pad(x, (0, _padded(x.shape[-1]) - x.shape[-1]))
    x = x.reshape(*x.shape[:-1], -1, 32)
    top = 127.0 if kind == Q8 else 7.0
    d = _half_up(x.abs().amax(-1, keepdim=True) / top)
    inv = torch.where(d > 0, 1.0 / d, torch.zeros_like(d))
    if kind == Q8:
        q = _round_away(x * inv).clamp(-127, 127).to(torch.int8).flatten(-2)
    else:
        n = _round_away(x * inv + 8.0).clamp(0, 15).to(torch.uint8)
        q = (n[..., :16] | (n[..., 16:] << 4)).flatten(-2)
    return q, d.squeeze(-1).half()


def _dequantise(q, d, kind, head_dim):
    """Stored quants [..., bytes] and scales [..., blocks] as fp32 [..., head_dim]."""
    q = q.unflatten(-1, (d.shape[-1], -1))
    n = q.float() if kind == Q8 else torch.cat((q & 15, q >> 4), -1).float() - 8.0
    return (n * d.float()[..., None]).flatten(-2)[..., :head_dim]


def _rotate(x, cos_sin, rot_dim, neox):
    """x [rows, heads, head_dim] rotated by cos_sin [rows, rot_dim / 2, 2]."""
    c, s = cos_sin[:, None, :, 0], cos_sin[:, None, :, 1]
    r = x[..., :rot_dim]
    a, b = (r[..., :rot_dim // 2], r[..., rot_dim // 2:]) if neox else (r[..., 0::2], r[..., 1::2])
    ya, yb = a * c - b * s, a * s + b * c
    y = torch.cat((ya, yb), -1) if neox else torch.stack((ya, yb), -1).flatten(-2)
    return torch.cat((y, x[..., rot_dim:]), -1)


def _plain_write(s, which, x, kind):
    seqs, slots = s["seqs"].long(), s["slots"].long()
    q, d = _quantise(x, kind)
    s["planes"][which][seqs, 0, :, slots] = q
    s["scales"][which][seqs, 0, :, slots] = d


def _plain_read(s, which, case):
    seqs, slots = s["seqs"].long(), s["slots"].long()
    return _dequantise(s["planes"][which][seqs, 0, :, slots], s["scales"][which][seqs, 0, :, slots], case["type"],
                       case["head_dim"])


def _cache_values(s, which, case):
    """The sequences' cached values [batch, kv_heads, capacity, head_dim] in fp32."""
    p = s["planes"][which][s["seqs"].long(), 0]
    if case["type"] == F32:
        return p.transpose(1, 2)
    return _dequantise(p, s["scales"][which][s["seqs"].long(), 0], case["type"], case["head_dim"])


def _visible(s, case, slots):
    """[batch, tokens, slots]: what each drafted token sees."""
    t = case["tokens"]
    lens = s["lens"].long()[:, None, None]
    at = torch.arange(slots, device=DEV)[None, None, :]
    j = at - lens  # the drafted token that the slot holds
    if s["mask"] is None:
        drafted = j <= torch.arange(t, device=DEV)[None, :, None]
    else:
        bits = (s["mask"][..., None] >> torch.arange(64, device=DEV)) & 1
        inside = j.clamp(0, t - 1).expand(case["batch"], t, slots)
        drafted = torch.gather(bits.flatten(-2).bool(), 2, inside)
    return (j < 0) | (drafted & (j < t))


def _plain_attention(s, case):
    b, t, kv, hd = case["batch"], case["tokens"], case["kv_heads"], case["head_dim"]
    n = case["len"] + t
    group = case["heads"] // kv
    k, v = (_cache_values(s, w, case)[:, :, :n] for w in range(2))
    q = s["q"].view(b, t, kv, group, hd).permute(0, 2, 1, 3, 4).reshape(b, kv, t * group, hd)
    x = torch.matmul(q, k.transpose(-1, -2)) * hd ** -0.5
    see = _visible(s, case, n)[:, None, :, None, :].expand(b, 1, t, group, n).reshape(b, 1, t * group, n)
    x = x.masked_fill(~see, float("-inf"))
    p = torch.exp(x - x.amax(-1, keepdim=True))
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    return o.view(b, kv, t, group, hd).permute(0, 2, 1, 3, 4).reshape(b, t, case["heads"], hd)


def _run_plain(s):
    case = s["case"]
    op = case["op"]
    if op == "attention":
        return _plain_attention(s, case)
    if op in ("rope", "cache_rope"):
        at = s["table"][s["positions"].long()]
        q = _rotate(s["q"], at, case["rot_dim"], case["neox"])
        k = _rotate(s["k"], at, case["rot_dim"], case["neox"])
        if op == "rope":
            return [q, k]
    if op != "read":
        _plain_write(s, 0, k if op == "cache_rope" else s["k"], case["type"])
        _plain_write(s, 1, s["v"], case["type"])
    got = [_plain_read(s, 0, case), _plain_read(s, 1, case)]
    return [q] + got if op == "cache_rope" else got


# ------------------------------------------------------------------------------------------------ the library's calls
def _run_own(s):
    case, lib = s["case"], s["lib"]
    op, heads, kv, hd = case["op"], case.get("heads", 0), case["kv_heads"], case["head_dim"]
    if op == "attention":
        b, t = case["batch"], case["tokens"]
        mask = s["mask"].data_ptr() if s["mask"] is not None else None
        lib.call("mlb_attention_tree", 0, ctypes.byref(s["cache"]), 0, b, t, s["seqs"].data_ptr(), s["lens"].data_ptr(),
                 case["len"], mask, s["q"].data_ptr(), heads * hd, heads, 0.0, s["out"].data_ptr(), heads * hd)
        return s["out"]
    if op == "rope":
        wide = (heads + 2 * kv) * hd
        lib.call("mlb_rope_rows", 0, ctypes.byref(s["rope"]), case["rows"], s["positions"].data_ptr(),
                 s["q"].data_ptr(), wide, s["q_out"].data_ptr(), heads * hd, heads,
                 s["k"].data_ptr(), wide, s["k_out"].data_ptr(), kv * hd, kv)
        return [s["q_out"], s["k_out"]]
    rows, seqs, slots = case["batch"] * case["tokens"], s["seqs"].data_ptr(), s["slots"].data_ptr()
    if op == "cache":
        lib.call("mlb_kv_cache_write", 0, ctypes.byref(s["cache"]), 0, rows, seqs, slots, s["k"].data_ptr(), kv * hd,
                 s["v"].data_ptr(), kv * hd)
    elif op == "cache_rope":
        lib.call("mlb_kv_cache_write_rope", 0, ctypes.byref(s["cache"]), 0, rows, seqs, slots, ctypes.byref(s["rope"]),
                 s["positions"].data_ptr(), s["q"].data_ptr(), heads * hd, s["q_out"].data_ptr(), heads * hd, heads,
                 s["k"].data_ptr(), kv * hd, s["v"].data_ptr(), kv * hd)
    lib.call("mlb_kv_cache_read", 0, ctypes.byref(s["cache"]), 0, rows, seqs, slots, s["k_read"].data_ptr(), kv * hd,
             s["v_read"].data_ptr(), kv * hd)
    got = [s["k_read"], s["v_read"]]
    return [s["q_out"]] + got if op == "cache_rope" else got


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------------------------ work
def work(case):
    op, kv, hd = case["op"], case["kv_heads"], case["head_dim"]
    heads = case.get("heads", 0)
    if op == "rope":
        n = case["rows"] * (heads + kv) * hd
        return {"bytes": 8 * n + case["rows"] * (4 + 4 * case["rot_dim"]), "flops": 3 * n}
    if op == "attention":
        t, n = case["tokens"], sum(_lens(case)) + case["batch"] * case["tokens"]
        entry = 4 * hd if case["type"] == F32 else _padded(hd) // 32 * (4 * BITS[case["type"]] + 2)
        return {"bytes": 2 * n * kv * entry + 8 * case["batch"] * t * heads * hd, "flops": 4 * n * t * heads * hd}
    rows = case["batch"] * case["tokens"]
    values = 2 * rows * kv * hd
    held = 2 * rows * kv * _padded(hd) // 32 * (4 * BITS[case["type"]] + 2)
    moved = {"read": held + 4 * values, "cache": 8 * values + 2 * held, "cache_rope": 8 * values + 2 * held}[op]
    if op == "cache_rope":
        moved += 8 * rows * heads * hd + 4 * rows * case["rot_dim"]
    return {"bytes": moved + 8 * rows, "flops": 4 * values}


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_rotated(s, case, x):
    rot, half = case["rot_dim"], case["rot_dim"] // 2
    y = x.double().clone()
    ang = s["table"].double()[s["positions"].long()][:, None]
    for i in range(half):
        a, b = (i, i + half) if case["neox"] else (2 * i, 2 * i + 1)
        c, sn = ang[..., i, 0], ang[..., i, 1]
        y[..., a] = x[..., a].double() * c - x[..., b].double() * sn
        y[..., b] = x[..., a].double() * sn + x[..., b].double() * c
    return y


def _exact_held(x, kind):
    """The values that a cache of this type holds for x (64 bits; the scale is an fp16 number)."""
    hd = x.shape[-1]
    y = torch.zeros_like(x)
    for lo in range(0, hd, 32):
        part = x[..., lo:lo + 32]
        d = part.abs().amax(-1, keepdim=True) / (127 if kind == Q8 else 7)
        step = torch.exp2(torch.floor(torch.log2(d.clamp_min(2.0 ** -14))) - 10)
        d = torch.floor(d / step + 0.5) * step
        n = torch.where(d > 0, part / d, torch.zeros_like(part))
        n = torch.copysign(torch.floor(n.abs() + 0.5), n) if kind == Q8 else torch.floor(n + 8 + 0.5) - 8
        y[..., lo:lo + 32] = d * n.clamp(-127 if kind == Q8 else -8, 127 if kind == Q8 else 7)
    return y


def _exact_stored(s, which, seq, case):
    """One sequence's cache in 64 bits [kv_heads, capacity, head_dim]."""
    p = s["planes"][which][seq, 0]
    if case["type"] == F32:
        return p.double().permute(1, 0, 2)
    d = s["scales"][which][seq, 0].double().repeat_interleave(32, -1)
    if case["type"] == Q8:
        n = p.double()
    else:
        blocks = p.view(*p.shape[:-1], -1, 16).long()
        n = torch.stack((blocks % 16, blocks // 16), -2).flatten(-3).double() - 8
    return (n * d)[..., :case["head_dim"]]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "rope":
        return [_exact_rotated(s, case, s["q"]), _exact_rotated(s, case, s["k"])]
    if op in ("cache", "cache_rope"):
        k = _exact_rotated(s, case, s["k"]) if op == "cache_rope" else s["k"].double()
        held = [_exact_held(k, case["type"]), _exact_held(s["v"].double(), case["type"])]
        return [_exact_rotated(s, case, s["q"])] + held if op == "cache_rope" else held
    if op == "read":
        b, t = case["batch"], case["tokens"]
        at = s["slots"].view(b, t).long()
        return [torch.cat([_exact_stored(s, w, i, case)[:, at[i]].transpose(0, 1) for i in range(b)]) for w in range(2)]
    b, t, heads, kv, hd = (case[x] for x in ("batch", "tokens", "heads", "kv_heads", "head_dim"))
    out = torch.zeros(b, t, heads, hd, dtype=torch.float64, device=DEV)
    for i in range(b):
        n, seq = int(s["lens"][i]), int(s["seqs"][i])
        k, v = (_exact_stored(s, w, seq, case)[:, :n + t] for w in range(2))
        see = torch.ones(t, n + t, dtype=torch.bool, device=DEV)
        if case["tree"]:
            bits = s["mask"][i].cpu().numpy().view(np.uint8)
            see[:, n:] = torch.from_numpy(np.unpackbits(bits, axis=-1, bitorder="little")[:, :t].astype(bool)).to(DEV)
        else:
            see[:, n:] = torch.ones(t, t, device=DEV).tril().bool()
        for h in range(heads):
            x = (s["q"][i, :, h].double() @ k[h * kv // heads].T) / hd ** 0.5
            out[i, :, h] = torch.softmax(x.masked_fill(~see, float("-inf")), -1) @ v[h * kv // heads]
    return out
