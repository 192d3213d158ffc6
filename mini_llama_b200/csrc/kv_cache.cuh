// The caller-owned KV cache (mlb_kv_cache) as kernels see it, and the checks of
// its descriptor that every entry point makes.
#pragma once

#include "common.cuh"

namespace mlb {

// Strides are in rows of one head (a position's B blocks, or head_dim floats):
// quantized caches keep a head's positions contiguous, fp32 ones a position's
// heads.
struct KvView {
    int type, n_seqs, n_layers, max_seq, n_kv, hd, blocks;
    long long seq_rows, layer_rows;  // row strides of a sequence and of a layer
    int head_rows, slot_rows;        // row strides of a head and of a slot
    int head_slots;                  // slots that a head's plane holds
    void *k, *v;
    __half *ks, *vs;

    __host__ __device__ __forceinline__ long long Row(int seq, int layer, int head, int slot) const {
        return seq * seq_rows + layer * layer_rows + 1LL * head * head_rows + 1LL * slot * slot_rows;
    }
};

// Checks the descriptor's shape, and with `pointers` its planes too.
KvView CheckedKvView(const char* caller, const mlb_kv_cache* cache, bool pointers);
// A pointer that is not on its elements' boundary (null is) would fault on the device.  The text is put together
// only for a refusal: small calls take no longer than their host side.
inline void RequireAligned(const char* caller, const char* name, const void* p, unsigned bytes, const char* part = "") {
    if (reinterpret_cast<uintptr_t>(p) % bytes != 0)
        Require(false, caller, std::string(name) + part + " is not " + std::to_string(bytes) + "-byte aligned");
}
// Checks a layer index (all_ok: MLB_ALL_LAYERS is allowed).
void CheckKvLayer(const char* caller, const KvView& c, int layer, bool all_ok);

}  // namespace mlb
