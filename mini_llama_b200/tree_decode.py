"""Greedy decoding with drafted tokens over a quantized KV cache, from the op-level calls.

    python -m mini_llama_b200.tree_decode [--model qwen2] [--cache q8_0] [--tokens 128] [--draft 12]

Every step feeds the last token and a tree of guesses about what follows it through the model in one pass:
tree rows go through the linears together, mlb_kv_cache_write_rope rotates q and k and stores K and V (8 or 4
bits, or fp32), mlb_attention_tree attends with all rows at once, each seeing its ancestors.  The guesses come
from the text so far (what followed earlier occurrences of the last tokens), so no second model is needed; the
longest path that the model itself would have chosen is kept, which leaves the greedy text unchanged.  Prints one
JSON line.  It shows the calls in use and is not the fast way to decode: a pass is hundreds of small launches from
Python (630 tokens/s with drafts on the Qwen2-0.5B shape, where the decode session makes 2411).
"""
from __future__ import annotations

import argparse
import json
import time

import numpy as np

from . import capi, synth
from .device import DeviceArray, KvCache, Model, RopeTable

CACHE_TYPES = {"f32": capi.F32, "q8_0": capi.Q8_0, "q4_0": capi.Q4_0}

SPECS = {
    "tiny": dict(vocab_size=256, dim=64, hidden_dim=176, n_layers=2, n_heads=4, n_kv_heads=2, head_dim=16,
                 max_seq_len=512, rope_theta=1e4, rms_norm_eps=1e-5, rope_neox=0, qkv_bias=0, qtype=capi.Q8_0),
    "qwen2": dict(vocab_size=151936, dim=896, hidden_dim=4864, n_layers=24, n_heads=14, n_kv_heads=2, head_dim=64,
                  max_seq_len=1024, rope_theta=1e6, rms_norm_eps=1e-6, rope_neox=1, qkv_bias=1, qtype=capi.Q8_0),
}


def draft_tree(history, size: int, branches: int = 3):
    """Guesses about what follows `history`: (tokens, parents) of at most `size` nodes.  Node 0 is the last token
    (parent -1).  Each branch is what followed an earlier occurrence of the last two tokens (else of the last
    one); common beginnings are shared, and the branches share the nodes evenly."""
    tokens, parents = [history[-1]], [-1]
    found = []
    for n in (2, 1):
        tail = history[-n:]
        for i in range(len(history) - n - 1, -1, -1):
            if len(found) < branches and history[i:i + n] == tail and i + n not in found:
                found.append(i + n)
    ends = [0] * len(found)  # where each branch has come to; they grow by one token in turn
    for step in range(size):
        for j, start in enumerate(found):
            if start + step >= len(history):
                continue
            t = history[start + step]
            child = next((i for i in range(1, len(tokens)) if parents[i] == ends[j] and tokens[i] == t), None)
            if child is None:
                if len(tokens) == size:
                    return tokens, parents
                tokens.append(t)
                parents.append(ends[j])
                child = len(tokens) - 1
            ends[j] = child
    return tokens, parents


def tree_mask(parents) -> np.ndarray:
    """[nodes][words] of 64 bits: each node's ancestors and itself."""
    n = len(parents)
    seen = np.zeros((n, (n + 63) // 64 * 64), np.uint8)
    for i, p in enumerate(parents):
        if p >= 0:
            seen[i] = seen[p]
        seen[i, i] = 1
    return np.packbits(seen, axis=-1, bitorder="little").view(np.uint64)


def accepted_path(tokens, parents, choice):
    """Nodes that the model agrees with, from node 0 down, and the token that follows the last of them."""
    path = [0]
    while True:
        want = choice[path[-1]]
        child = next((i for i in range(1, len(tokens)) if parents[i] == path[-1] and tokens[i] == want), None)
        if child is None:
            return path, want
        path.append(child)


class TreeDecoder:
    """One sequence decoded with drafted tokens; weights are those of a device Model."""

    def __init__(self, model: Model, cache_type: int, max_rows: int = 64):
        self.lib, self.dev, self.model, s = model.lib, model.device, model, model.spec
        self.max_rows, self.len = max_rows, 0
        self.qd, self.kd = s["n_heads"] * s["head_dim"], s["n_kv_heads"] * s["head_dim"]
        new = lambda *shape, dtype=np.float32: DeviceArray(self.lib, self.dev, shape, dtype)  # noqa: E731
        r, d, f = max_rows, s["dim"], s["hidden_dim"]
        self.x, self.normed, self.sum = new(r, d), new(r, d), new(r, d)
        self.q, self.att = new(r, self.qd), new(r, self.qd)
        self.k, self.v = new(s["n_layers"], r, self.kd), new(s["n_layers"], r, self.kd)  # of the last pass
        self.gate, self.up, self.act = new(r, f), new(r, f), new(r, f)
        self.logits, self.choice = new(r, s["vocab_size"]), new(r, dtype=np.int32)
        self.slots, self.positions = new(r, dtype=np.int32), new(r, dtype=np.int32)
        self.lens, self.mask = new(1, dtype=np.int32), new(r, (r + 63) // 64, dtype=np.uint64)
        self.table = RopeTable(self.lib, self.dev, s["max_seq_len"], s["head_dim"], s["rope_theta"],
                               capi.ROPE_NEOX if s["rope_neox"] else capi.ROPE_NORMAL)
        self.cache = KvCache(self.lib, self.dev, cache_type, 1, s["n_layers"], s["max_seq_len"], s["n_kv_heads"],
                             s["head_dim"])

    def _put(self, array: DeviceArray, values):
        a = np.ascontiguousarray(values, dtype=array.dtype)
        self.lib.call("mlb_memcpy_h2d", self.dev, array.ptr, a.ctypes.data, a.nbytes)

    def _linear(self, layer, kind, bias, x, rows, n_in, n_out, y):
        w, _ = self.model.weight(layer, kind)
        b = self.model.weight(layer, bias)[0] if bias is not None and self.model.spec["qkv_bias"] else None
        self.lib.call("mlb_quant_linear", self.dev, self.model.spec["qtype"], x, w, n_out * ((n_in + 31) // 32), rows, n_in,
                      n_out, b, y)

    def _norm(self, layer, kind, rows):
        w, _ = self.model.weight(layer, kind)
        d = self.model.spec["dim"]
        for r in range(rows):
            self.lib.call("mlb_rmsnorm", self.dev, self.x.ptr + 4 * d * r, w, d, self.model.spec["rms_norm_eps"],
                          self.normed.ptr + 4 * d * r)

    def forward(self, tokens, parents) -> list[int]:
        """One pass over tree nodes whose root sits at position self.len; the model's choice after each node."""
        s, n, call = self.model.spec, len(tokens), self.lib.call
        if not 1 <= n <= self.max_rows or len(parents) != n:
            raise ValueError(f"a pass takes 1 to {self.max_rows} nodes with a parent each, not {n} and {len(parents)}")
        if self.len + n > s["max_seq_len"]:
            raise ValueError(f"{n} nodes after {self.len} tokens pass the cache's {s['max_seq_len']} slots")
        d, f, V = s["dim"], s["hidden_dim"], s["vocab_size"]
        depth = []
        for p in parents:
            depth.append(0 if p < 0 else depth[p] + 1)
        self._put(self.slots, [self.len + i for i in range(n)])
        self._put(self.positions, [self.len + i for i in depth])
        self._put(self.lens, [self.len])
        self._put(self.mask, tree_mask(parents))
        emb, _ = self.model.weight(-1, capi.W_EMBEDDING)
        for i, t in enumerate(tokens):
            call("mlb_embedding", self.dev, emb, V, d, int(t), self.x.ptr + 4 * d * i)
        x, normed, total = self.x.ptr, self.normed.ptr, self.sum.ptr
        for l in range(s["n_layers"]):
            k, v = (a.ptr + 4 * l * self.max_rows * self.kd for a in (self.k, self.v))
            self._norm(l, capi.W_ATTN_NORM, n)
            self._linear(l, capi.W_WQ, capi.W_BQ, normed, n, d, self.qd, self.q.ptr)
            self._linear(l, capi.W_WK, capi.W_BK, normed, n, d, self.kd, k)
            self._linear(l, capi.W_WV, capi.W_BV, normed, n, d, self.kd, v)
            self.cache.write_rope(l, n, self.slots.ptr, self.table, self.positions.ptr, self.q.ptr, s["n_heads"], k, v)
            self.cache.attend(l, 1, n, self.lens.ptr, self.len, self.q.ptr, s["n_heads"], self.att.ptr, self.mask.ptr)
            self._linear(l, capi.W_WO, None, self.att.ptr, n, self.qd, d, total)
            call("mlb_add", self.dev, x, total, n * d, x)
            self._norm(l, capi.W_FFN_NORM, n)
            self._linear(l, capi.W_GATE, None, normed, n, d, f, self.gate.ptr)
            self._linear(l, capi.W_UP, None, normed, n, d, f, self.up.ptr)
            call("mlb_silu", self.dev, self.gate.ptr, n * f, self.act.ptr)
            call("mlb_mul", self.dev, self.act.ptr, self.up.ptr, n * f, self.act.ptr)
            self._linear(l, capi.W_DOWN, None, self.act.ptr, n, f, d, total)
            call("mlb_add", self.dev, x, total, n * d, x)
        self._norm(-1, capi.W_FINAL_NORM, n)
        self._linear(-1, capi.W_LM_HEAD, None, normed, n, d, V, self.logits.ptr)
        for i in range(n):
            call("mlb_argmax", self.dev, self.logits.ptr + 4 * V * i, V, self.choice.ptr + 4 * i)
        return [int(c) for c in self.choice.download()[:n]]

    def keep(self, path):
        """Commits the nodes of `path`: their K and V move up to the slots after self.len.  They are written
        again from the pass's rows, the others skipped (slot -1); nothing to do where they are in place."""
        if path != list(range(len(path))):
            slots, positions = np.full(self.max_rows, -1, np.int32), np.zeros(self.max_rows, np.int32)
            for i, node in enumerate(path):
                slots[node] = positions[node] = self.len + i
            self._put(self.slots, slots)
            self._put(self.positions, positions)
            for l in range(self.model.spec["n_layers"]):
                k, v = (a.ptr + 4 * l * self.max_rows * self.kd for a in (self.k, self.v))
                self.cache.write_rope(l, max(path) + 1, self.slots.ptr, self.table, self.positions.ptr, None, 0, k, v)
        self.len += len(path)

    def generate(self, prompt, n_new: int, draft: int):
        """Greedy tokens after `prompt`, at most `draft` tree nodes to a pass: (tokens, passes).  The cache then holds
        the prompt and all of them but the last, which a further call's prompt begins with."""
        history, out, passes = [int(t) for t in prompt], [], 0
        room = self.model.spec["max_seq_len"]
        if not history:
            raise ValueError("the prompt is empty")
        if draft > self.max_rows:
            raise ValueError(f"{draft} nodes to a pass, but the decoder was made for {self.max_rows}")
        if self.len + len(history) + n_new + draft > room:
            raise ValueError(f"the cache's {room} slots are too few for {self.len} + {len(history)} tokens, {n_new} new ones "
                             f"and {draft} drafted")
        for i in range(0, len(history) - 1, self.max_rows):  # the prompt but its last token, as chains
            part = history[i:min(i + self.max_rows, len(history) - 1)]
            self.forward(part, list(range(-1, len(part) - 1)))
            self.len += len(part)
        while len(out) < n_new:
            tokens, parents = draft_tree(history, max(1, draft))
            choice = self.forward(tokens, parents)
            path, follow = accepted_path(tokens, parents, choice)
            if len(path) > n_new - len(out):  # the cache keeps what is returned and no more
                path = path[:n_new - len(out)]
                follow = choice[path[-1]]
            self.keep(path)
            fresh = [tokens[i] for i in path[1:]] + [follow]
            history += fresh
            out += fresh
            passes += 1
        return out, passes


def main(argv=None) -> int:
    ap = argparse.ArgumentParser()
    ap.add_argument("--model", choices=sorted(SPECS), default="qwen2")
    ap.add_argument("--cache", choices=sorted(CACHE_TYPES), default="q8_0")
    ap.add_argument("--prompt", type=int, default=64)
    ap.add_argument("--tokens", type=int, default=128)
    ap.add_argument("--draft", type=int, default=12)
    ap.add_argument("--device", type=int, default=0)
    args = ap.parse_args(argv)
    lib, spec = capi.load(), SPECS[args.model]
    model = Model(lib, args.device, spec)
    model.synthesize(seed=3, tied=True)
    prompt = synth.tokens(args.prompt, 3, spec["vocab_size"])
    line = {"model": args.model, "cache": args.cache, "weights": "synthetic"}
    texts = []
    for name, draft in (("plain", 1), ("drafted", args.draft)):
        decoder = TreeDecoder(model, CACHE_TYPES[args.cache], max(args.draft, 16))
        t0 = time.perf_counter()
        text, passes = decoder.generate(prompt, args.tokens, draft)
        texts.append(text)
        line[name] = {"tokens_s": round(args.tokens / (time.perf_counter() - t0), 1), "passes": passes}
        line["cache_bytes"] = decoder.cache.nbytes()
    line["same_text"] = texts[0] == texts[1]
    print(json.dumps(line), flush=True)
    model.close()
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
