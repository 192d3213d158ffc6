// Attention of drafted tokens over the KV cache (mlb_attention_tree): `tokens`
// queries of each sequence against its cached slots, the drafted slots by a bit
// mask, over fp32, Q8_0 and Q4_0 caches.
#include <cmath>

#include "tree_attention.cuh"

namespace mlb {

namespace {

constexpr int kRowWarps = 8;

// Element `e` of a cached head row.
template <int TYPE>
__device__ __forceinline__ float CachedElement(const void* plane, const __half* scales, long long row, int blocks, int hd,
                                               int e) {
    if (TYPE == MLB_F32) return e < hd ? __ldg(static_cast<const float*>(plane) + row * hd + e) : 0.0f;
    const long long at = row * blocks + (e >> 5);
    const float d = __half2float(__ldg(scales + at));
    if (TYPE == MLB_Q8_0) return d * static_cast<float>(__ldg(static_cast<const signed char*>(plane) + at * 32 + (e & 31)));
    const int n = __ldg(static_cast<const unsigned char*>(plane) + at * 16 + (e & 15));
    return d * static_cast<float>((((e & 16) ? n >> 4 : n & 15)) - 8);
}

// Any head size, alignment and length; for what the matrix kernels do not take (fp32
// rows without 16-byte alignment, planes of fewer slots than their unit).  One CTA per
// query row (sequence, token, head): warp w takes every eighth slot from w, lane i
// the elements i, i + 32, .., with a running maximum and sum; the warps' results
// are joined at the end.  Bound: a dot product's latency (shuffles) per slot and warp,
// and each row reads the cache again: 32 heads over 4000 slots of 8 x 256 in Q8_0
// 912 us, the matrix kernel 19.
template <int TYPE>
__global__ void __launch_bounds__(kRowWarps * 32) TreeRowKernel(TreeArgs a) {
    __shared__ float so[kRowWarps][kMaxBlocks * 32];
    __shared__ float sm[kRowWarps], sl[kRowWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int h = blockIdx.x % a.n_heads;
    const long long row = blockIdx.x / a.n_heads;
    const int b = static_cast<int>(row / a.tokens), t = static_cast<int>(row % a.tokens);
    const Entry e = FindEntry(a, b);
    const KvView& c = a.c;
    const float* q = a.q + row * a.q_stride + size_t(h) * c.hd;
    float* out = a.out + row * a.out_stride + size_t(h) * c.hd;
    const uint64_t* bits = a.mask ? a.mask + row * a.words : nullptr;
    float qr[kMaxBlocks], o[kMaxBlocks];
#pragma unroll
    for (int i = 0; i < kMaxBlocks; ++i) {
        qr[i] = i * 32 + lane < c.hd ? __ldg(q + i * 32 + lane) : 0.0f;
        o[i] = 0.0f;
    }
    float m = -INFINITY, l = 0.0f;
    for (int s = warp; s < e.slots; s += kRowWarps) {
        if (s >= e.len && !SeesDraft(bits, t, s - e.len)) continue;
        const long long at = c.Row(e.seq, a.layer, h / a.group, s);
        float x = 0.0f;
#pragma unroll
        for (int i = 0; i < kMaxBlocks; ++i)
            if (i < c.blocks) x = fmaf(qr[i], CachedElement<TYPE>(c.k, c.ks, at, c.blocks, c.hd, i * 32 + lane), x);
        x = WarpSum(x) * a.scale;
        const float top = fmaxf(m, x);
        // a score of -inf (an infinite key or query) weighs nothing
        const float keep = m == -INFINITY ? 0.0f : expf(m - top), w = x == -INFINITY ? 0.0f : expf(x - top);
        m = top;
        l = l * keep + w;
#pragma unroll
        for (int i = 0; i < kMaxBlocks; ++i)
            if (i < c.blocks)
                o[i] = fmaf(w, CachedElement<TYPE>(c.v, c.vs, at, c.blocks, c.hd, i * 32 + lane), o[i] * keep);
    }
    if (lane == 0) {
        sm[warp] = m;
        sl[warp] = l;
    }
#pragma unroll
    for (int i = 0; i < kMaxBlocks; ++i) so[warp][i * 32 + lane] = o[i];
    __syncthreads();
    float top = -INFINITY, sum = 0.0f;
    for (int w = 0; w < kRowWarps; ++w) top = fmaxf(top, sm[w]);
    for (int w = 0; w < kRowWarps; ++w) sum += sl[w] == 0.0f ? 0.0f : sl[w] * expf(sm[w] - top);
    for (int i = threadIdx.x; i < c.hd; i += blockDim.x) {
        float v = 0.0f;
        for (int w = 0; w < kRowWarps; ++w)
            if (sl[w] != 0.0f) v += so[w][i] * expf(sm[w] - top);
        out[i] = sum == 0.0f ? 0.0f : v / sum;
    }
}

// fp32 caches whose rows allow 16-byte copies, and planes of a unit or more.  Above
// 32 rows per KV head the tensor-memory kernel.  At 32, 40 and 64 rows it takes 67.7, 68.8
// and 70.3 us for 8 sequences of 4000 slots, 8 x 128 in Q8_0, the warp-level kernel 61.5,
// 84.0 and 107.3 (Q4_0: 65.0, 65.5, 67.6 against 57.3, 77.8, 99.3); for one of 2000 slots
// 18.4, 18.4, 20.1 against 18.4, 20.5, 22.5.  For one of 8000 it gains later: 32.8, 32.8,
// 34.8 against 28.0, 32.8, 36.9 in Q8_0 and 31.4, 32.8, 34.8 against 26.7, 30.7, 36.5 in
// Q4_0, where the rule by rows alone costs 7 % at 40.
bool LaunchTreeMma(DeviceContext& ctx, const TreeArgs& a) {
    if (a.c.type == MLB_F32) return a.cache_vec && LaunchTreeF32(ctx, a);
    if (1LL * a.tokens * a.group > 32 && LaunchTreeTc(ctx, a)) return true;
    return a.c.type == MLB_Q8_0 ? LaunchTreeQ80(ctx, a) : LaunchTreeQ40(ctx, a);
}

}  // namespace

}  // namespace mlb

using namespace mlb;

extern "C" {

int mlb_attention_tree(int device, const mlb_kv_cache* cache, int layer, int batch, int tokens, const int* seqs,
                       const int* lens, int max_len, const uint64_t* mask, const float* q, size_t q_stride, int n_heads,
                       float scale, float* out, size_t out_stride) {
    return Guard([&] {
        const char* c = "mlb_attention_tree";
        TreeArgs a{};
        a.c = CheckedKvView(c, cache, true);
        CheckKvLayer(c, a.c, layer, false);
        Require(a.c.hd <= kMaxBlocks * 32, c, "head_dim above 256 is not supported", MLB_ERR_UNSUPPORTED);
        Require(batch >= 0 && tokens >= 0, c, "batch or token count is negative");
        Require(max_len >= 0, c, "max_len is negative");
        Require(n_heads > 0 && n_heads % a.c.n_kv == 0, c, "n_heads must be a multiple of n_kv_heads");
        Require(std::isfinite(scale) && scale >= 0.0f, c, "scale must be finite and not negative");
        if (batch == 0 || tokens == 0) return;
        Require(lens && q && out, c, "lens, q or out is null");
        const size_t n = size_t(n_heads) * a.c.hd;
        Require(q_stride >= n && out_stride >= n, c, "row stride is shorter than a row");
        RequireAligned(c, "lens", lens, 4);
        RequireAligned(c, "seqs", seqs, 4);
        RequireAligned(c, "mask", mask, 8);
        RequireAligned(c, "q", q, 4);
        RequireAligned(c, "out", out, 4);
        Require(seqs || batch <= a.c.n_seqs, c, "batch is larger than the cache's sequences");
        Require(1.0 * batch * tokens * n_heads < 2147483648.0, c, "too many query rows", MLB_ERR_UNSUPPORTED);
        a.layer = layer;
        a.batch = batch;
        a.tokens = tokens;
        a.words = (tokens + 63) / 64;
        a.max_len = max_len;
        a.seqs = seqs;
        a.lens = lens;
        a.mask = mask;
        a.q = q;
        a.q_stride = q_stride;
        a.n_heads = n_heads;
        a.group = n_heads / a.c.n_kv;
        a.scale = scale > 0.0f ? scale : 1.0f / std::sqrt(static_cast<float>(a.c.hd));
        a.out = out;
        a.out_stride = out_stride;
        auto vec = [](const void* p, size_t stride) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride % 4 == 0; };
        a.q_vec = a.c.hd % 4 == 0 && vec(q, q_stride);
        a.out_vec = a.c.hd % 4 == 0 && vec(out, out_stride);
        a.cache_vec = a.c.hd % 4 == 0 && vec(a.c.k, 0) && vec(a.c.v, 0);
        DeviceContext& ctx = Ctx(device);
        if (LaunchTreeMma(ctx, a)) return;
        const unsigned grid = static_cast<unsigned>(batch) * tokens * n_heads;
        if (a.c.type == MLB_F32)
            TreeRowKernel<MLB_F32><<<grid, kRowWarps * 32, 0, ctx.stream>>>(a);
        else if (a.c.type == MLB_Q8_0)
            TreeRowKernel<MLB_Q8_0><<<grid, kRowWarps * 32, 0, ctx.stream>>>(a);
        else
            TreeRowKernel<MLB_Q4_0><<<grid, kRowWarps * 32, 0, ctx.stream>>>(a);
        CheckCuda(cudaGetLastError(), "TreeRowKernel");
    });
}

}  // extern "C"
