// What the kernels of mlb_attention_tree share.
#pragma once

#include "kv_cache.cuh"

namespace mlb {

constexpr int kMaxBlocks = 8;  // head_dim up to 256

struct TreeArgs {
    KvView c;
    int layer, batch, tokens, words, max_len;
    const int* seqs;
    const int* lens;
    const uint64_t* mask;
    const float* q;
    size_t q_stride;
    int n_heads, group;
    float scale;
    float* out;
    size_t out_stride;
    int q_vec, out_vec, cache_vec;  // rows (and fp32 cache rows) allow 16-byte accesses
};

// A batch entry's cache sequence and length; sequence -1: inactive.
struct Entry {
    int seq, len, slots;  // slots: what can be seen at all, drafted tokens included
};

__device__ __forceinline__ Entry FindEntry(const TreeArgs& a, int b) {
    Entry e;
    e.seq = a.seqs ? __ldg(a.seqs + b) : b;
    e.len = __ldg(a.lens + b);
    if (e.len < 0 || e.seq < 0 || e.seq >= a.c.n_seqs) {
        e.seq = -1;
        e.len = e.slots = 0;
        return e;
    }
    e.len = min(min(e.len, a.max_len), a.c.max_seq);
    e.slots = static_cast<int>(min(static_cast<long long>(e.len) + a.tokens, static_cast<long long>(a.c.max_seq)));
    return e;
}

// Whether drafted token t (mask row `bits`, null: chain) sees drafted token j.
__device__ __forceinline__ bool SeesDraft(const uint64_t* bits, int t, int j) {
    return bits ? (__ldg(bits + (j >> 6)) >> (j & 63)) & 1 : j <= t;
}


// The matrix-instruction kernels (tree_mma.cuh); false: the shape is not one of
// theirs.
bool LaunchTreeF32(DeviceContext& ctx, const TreeArgs& a);
bool LaunchTreeQ80(DeviceContext& ctx, const TreeArgs& a);
bool LaunchTreeQ40(DeviceContext& ctx, const TreeArgs& a);
// The tensor-memory kernel (tree_tc.cu) for many rows over quantized caches.
bool LaunchTreeTc(DeviceContext& ctx, const TreeArgs& a);

}  // namespace mlb
