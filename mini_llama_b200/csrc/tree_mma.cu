// Attention of drafted tokens on the warp-level matrix instructions, for the
// decode regime: few query rows per KV head, the cache read once.
//
// The R = tokens x (query heads per KV head) rows that share a KV head are cut
// into tiles of eight: the N side of mma.m16n8k16.  A warp takes 16 slots of
// the cache at a time (the M side, S^T = K Q^T) for one tile of rows:
//   K      the 16 x head_dim quants, straight from memory into A fragments (the
//          order of the elements within a block is free, as Q is loaded in the
//          same one), as fp16 whole numbers: exact.  Q is scaled per row by a
//          power of two and split into fp16 hi + lo (22 bits), so a block's
//          products are exact up to the fp32 sum; the slot's scale of the block
//          multiplies that sum.
//   softmax  running maximum and sum per row, the maximum moved only when a
//          score passes it by 2^2 (a vote): weights are 2^(x - m + 12) <= 2^14,
//          split into fp16 hi + lo and turned into B fragments by movmatrix.
//   V      O^T = V^T P^T: quants as exact fp16 A fragments again (byte
//          transposition in registers); the slot's scale of a block goes into
//          the weights, P' = hi + lo of p d by one product and two FMAs on half
//          pairs, relative to a power of two per row that covers the largest d
//          seen.  Two MMAs per fragment.
// fp32 caches take the same path with mma.m16n8k8 on tf32 hi + lo pairs (three
// products; no ranges to mind).  A unit's weighted values are summed in fresh
// accumulators and added to the running ones in fp32 with rounding to nearest:
// the matrix unit's own additions truncate, which over a long context would
// cost several times the fp32 rounding.
//
// The units of 16 slots of all (sequence, KV head, row group) items are one
// list, cut evenly over the CTAs (the lengths are on the device, so every CTA
// works the cut out from them): sequences of any lengths balance.  A CTA's warps
// share a stretch of the list, join their results in shared memory, and items
// that are cut between CTAs are joined by the CTA that finishes last (partials
// in the workspace, one counter per item, added in a fixed order).
#include <algorithm>
#include <cmath>

#include "tree_attention.cuh"

namespace mlb {

namespace {

constexpr int kUnit = 16;          // slots of a matrix step
constexpr int kRows = 8;           // query rows of a tile
constexpr float kStart = -1.7e38f; // running maximum before the first score (finite: no inf - inf)
constexpr float kLag = 2.0f;       // how far scores may pass the running maximum, in powers of two
constexpr float kOffset = 12.0f;   // weights are relative to 2^12: at most 2^14, and the fp16 pairs resolve
                                   // 2^-37 of the largest, for slots that weigh little where the heavy ones hold zeros
constexpr int kAhead = 3;          // rounds that the L2 prefetch runs ahead
constexpr float kLog2e = 1.4426950408889634f;

struct TreeSplit {
    int wq;        // row tiles of an item: warps that share its slots
    int groups;    // items of a (sequence, KV head): ceil(R / (8 wq))
    int rows;      // R
    float* parts;  // two partial results per CTA
    int* counters; // per item
    uint32_t magic;
};

__device__ __forceinline__ void Mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void MmaTf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The same with a zero accumulator.
__device__ __forceinline__ void MmaFirst(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}

__device__ __forceinline__ void MmaTf32First(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}

__device__ __forceinline__ void AddTo(float (&o)[4], const float (&d)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] += d[i];
}

__device__ __forceinline__ uint32_t Transpose8x8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

__device__ __forceinline__ float Exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t H2(__half2 v) { return *reinterpret_cast<uint32_t*>(&v); }
__device__ __forceinline__ __half2 AsHalf2(uint32_t v) { return *reinterpret_cast<__half2*>(&v); }

// (x, y) rounded to halves, and what the rounding left, rounded too.
__device__ __forceinline__ void SplitHalf(float x, float y, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    hi = H2(h);
    lo = H2(__floats2half2_rn(x - f.x, y - f.y));
}

// x as tf32 (rounded to nearest, halves up) and the rest, whose low 13 bits the
// matrix unit does not read: together 2^-21 relative at worst.
__device__ __forceinline__ void SplitTf32(float x, uint32_t& hi, uint32_t& lo) {
    hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
    lo = __float_as_uint(x - __uint_as_float(hi));
}

// int8 in bytes 0 and 2 of w as a half pair: byte ^ 0x80 is q + 128, and the half
// 0x6400 + u is 1024 + u.  `magic` (kMagic8, kMagic4) comes from the kernel's
// parameters: as a literal it would not fit the one logic instruction beside the
// mask.
constexpr uint32_t kMagic8 = 0x64806480u, kMagic4 = 0x64006400u;
__device__ __forceinline__ uint32_t EvenBytes(uint32_t w, uint32_t magic) {
    return H2(__hsub2(AsHalf2((w & 0x00ff00ffu) ^ magic), AsHalf2(kMagic8)));  // - (1024 + 128)
}

// The nibbles of bytes 0 and 2: low ones n - 8, high ones n - 8.
__device__ __forceinline__ uint32_t LowNibbles(uint32_t w, uint32_t magic) {
    return H2(__hsub2(AsHalf2((w & 0x000F000Fu) | magic), AsHalf2(0x64086408u)));  // 1024 + n - 1032
}
__device__ __forceinline__ uint32_t HighNibbles(uint32_t w, uint32_t magic) {
    // (1024 + 16 n) / 16 - 72
    return H2(__hfma2(AsHalf2((w & 0x00F000F0u) | magic), AsHalf2(0x2C002C00u), AsHalf2(0xD480D480u)));
}

// The fp16 scales of one slot's blocks, two to a word.
template <int NB>
__device__ __forceinline__ void LoadScales(const __half* p, uint32_t (&d)[(NB + 1) / 2]) {
    if constexpr (NB % 4 == 0) {
#pragma unroll
        for (int i = 0; i < NB / 4; ++i) {
            const uint2 w = __ldg(reinterpret_cast<const uint2*>(p) + i);
            d[2 * i] = w.x;
            d[2 * i + 1] = w.y;
        }
    } else if constexpr (NB % 2 == 0) {
#pragma unroll
        for (int i = 0; i < NB / 2; ++i) d[i] = __ldg(reinterpret_cast<const uint32_t*>(p) + i);
    } else {
        const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
        for (int i = 0; i < NB / 2; ++i) d[i] = __ldg(h + 2 * i) | (uint32_t(__ldg(h + 2 * i + 1)) << 16);
        d[NB / 2] = __ldg(h + NB - 1);
    }
}

template <int N>
__device__ __forceinline__ float ScaleOf(const uint32_t (&d)[N], int b) {
    return b & 1 ? __high2float(AsHalf2(d[b >> 1])) : __low2float(AsHalf2(d[b >> 1]));
}

// The rows, lengths and mask that a warp's step needs, common to both forms.
struct Step {
    int lane, g, c;  // lane = 4 g + c
    int slots, len, tokens, words;
    const uint64_t* mask;  // the batch entry's
    int t0, t1;            // drafted tokens of the thread's two score columns
};

__device__ __forceinline__ bool Sees(const Step& s, int t, int slot) {
    if (slot < s.len) return true;
    if (slot >= s.slots || t >= s.tokens) return false;
    return SeesDraft(s.mask ? s.mask + size_t(t) * s.words : nullptr, t, slot - s.len);
}

// Scores S (C fragment: rows slot g, g + 8; columns query 2c, 2c + 1) to weights
// 2^(x - m + offset), slots from `low` on, with the running maxima m and sums l of the two columns;
// `rescale` gets the factors of a moved maximum.
template <typename Rescale>
__device__ __forceinline__ void Weights(const Step& s, int p0, int low, float (&x)[4], float cs0, float cs1, float offset,
                                        float (&m)[2], float (&l)[2], Rescale&& rescale) {
    if (low + kUnit > s.len) {  // drafted slots, or the end
        const int a = p0 + s.g, b = a + 8;
        if (a < low || !Sees(s, s.t0, a)) x[0] = -INFINITY;
        if (a < low || !Sees(s, s.t1, a)) x[1] = -INFINITY;
        if (b < low || !Sees(s, s.t0, b)) x[2] = -INFINITY;
        if (b < low || !Sees(s, s.t1, b)) x[3] = -INFINITY;
    }
    float top0 = fmaxf(x[0], x[2]) * cs0, top1 = fmaxf(x[1], x[3]) * cs1;
    if (__any_sync(0xffffffffu, top0 > m[0] + kLag || top1 > m[1] + kLag)) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
            top0 = fmaxf(top0, __shfl_xor_sync(0xffffffffu, top0, o));
            top1 = fmaxf(top1, __shfl_xor_sync(0xffffffffu, top1, o));
        }
        const float n0 = fmaxf(m[0], top0), n1 = fmaxf(m[1], top1);
        const float r0 = Exp2(m[0] - n0), r1 = Exp2(m[1] - n1);
        m[0] = n0;
        m[1] = n1;
        l[0] *= r0;
        l[1] *= r1;
        rescale(r0, r1);
    }
    const float o0 = offset - m[0], o1 = offset - m[1];
    x[0] = Exp2(fmaf(x[0], cs0, o0));
    x[1] = Exp2(fmaf(x[1], cs1, o1));
    x[2] = Exp2(fmaf(x[2], cs0, o0));
    x[3] = Exp2(fmaf(x[3], cs1, o1));
    l[0] += x[0] + x[2];
    l[1] += x[1] + x[3];
}

// ---------------------------------------------------------------- quantized caches
// A warp's running result for one tile of rows over Q8_0 / Q4_0 slots.
template <int TYPE, int NB>
struct QuantWarp {
    static constexpr int kQuantBytes = TYPE == MLB_Q8_0 ? 32 : 16;
    static constexpr int kKWords = TYPE == MLB_Q8_0 ? 2 : 1;

    float o[NB][2][4];
    float m[2], l[2], cs[2];
    int e;         // of row g: P' is relative to 2^e
    float bound;   // 2^e
    __half2 down;  // 2^-e
    uint32_t kw[2][NB][kKWords];
    uint32_t kd[2][(NB + 1) / 2];
    const uint8_t *k, *v;
    const __half *ks, *vs;
    int stored;
    uint32_t magic;
    const uint4* qs;  // Q fragments of the tile: [block][half][lane] (hi, hi, lo, lo)

    // First of the four output elements of row tile j (0, 1) of a block that
    // the thread holds in o[.][j][0..1] (its row g) and o[.][j][2..3] (g + 8).
    __device__ __forceinline__ static int Dim(int g, int j, int half) {
        return TYPE == MLB_Q8_0 ? 4 * g + 2 * j + half : 16 * j + 2 * g + half;
    }

    __device__ __forceinline__ static void LayOut(const TreeArgs& a, const Step& s, const float* q, uint4* frags,
                                                  float* undos) {
        // the thread's elements of its row g, in the order of the K fragments
        float x[NB][8], top = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int d0 = b * 32 + (TYPE == MLB_Q8_0 ? 8 * s.c : 4 * s.c);
            const int d1 = TYPE == MLB_Q8_0 ? d0 + 4 : d0 + 16;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int d = half ? d1 : d0;
                if (a.q_vec) {
                    const float4 w = q && d < a.c.hd ? __ldg(reinterpret_cast<const float4*>(q + d))
                                                     : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    x[b][4 * half] = w.x;
                    x[b][4 * half + 1] = w.y;
                    x[b][4 * half + 2] = w.z;
                    x[b][4 * half + 3] = w.w;
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[b][4 * half + i] = q && d + i < a.c.hd ? __ldg(q + d + i) : 0.0f;
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[b][i]));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int up = ScaleExp(top);  // largest |q| into [2^14, 2^15)
        const float sc = Pow2(up), undo = fmaxf(Pow2(-up) * a.scale * kLog2e, 1e-37f);
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float* y = &x[b][4 * i];
                // bytes 0 and 2, then 1 and 3 of a word
                uint4 f;
                SplitHalf(y[0] * sc, y[2] * sc, f.x, f.z);
                SplitHalf(y[1] * sc, y[3] * sc, f.y, f.w);
                frags[(2 * b + i) * 32 + s.lane] = f;
            }
        if (s.c == 0) undos[s.g] = undo;
    }

    // `write`: the warp that lays out the tile's Q fragments.
    __device__ __forceinline__ void Begin(const TreeArgs& a, const TreeSplit& sp, const Step& s, int seq, int head,
                                          const float* q, uint4* frags, float* undos, bool write) {
        qs = frags + s.lane;
        magic = sp.magic;
        const long long row = a.c.Row(seq, a.layer, head, 0);
        k = static_cast<const uint8_t*>(a.c.k) + row * NB * kQuantBytes;
        v = static_cast<const uint8_t*>(a.c.v) + row * NB * kQuantBytes;
        ks = a.c.ks + row * NB;
        vs = a.c.vs + row * NB;
        stored = a.c.head_rows;
        if (write) LayOut(a, s, q, frags, undos);
        m[0] = m[1] = kStart;
        l[0] = l[1] = 0.0f;
        SetPower(-15);
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int i = 0; i < 8; ++i) o[b][i >> 2][i & 3] = 0.0f;
    }

    __device__ __forceinline__ void SetPower(int to) {
        e = to;
        bound = Pow2(to);
        down = __float2half2_rn(Pow2(-to));
    }

    // Slots p0 .. p1 - 1 (p0 a multiple of 16) into the L2.
    __device__ __forceinline__ void Prefetch(const Step& s, int p0, int p1) const {
        if (s.lane != 0) return;
        const uint32_t n = min((p1 + 7) & ~7, stored) - p0;
        BulkPrefetchL2(k + size_t(p0) * NB * kQuantBytes, n * NB * kQuantBytes);
        BulkPrefetchL2(v + size_t(p0) * NB * kQuantBytes, n * NB * kQuantBytes);
        BulkPrefetchL2(ks + size_t(p0) * NB, n * NB * 2);
        BulkPrefetchL2(vs + size_t(p0) * NB, n * NB * 2);
    }

    __device__ __forceinline__ void LoadK(const Step& s, int p0) {
        const uint8_t* row = k + size_t(p0 + s.g) * (NB * kQuantBytes) + 4 * kKWords * s.c;
        const __half* sc = ks + size_t(p0 + s.g) * NB;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const uint8_t* at = row + 8 * r * (NB * kQuantBytes) + b * kQuantBytes;
                if constexpr (TYPE == MLB_Q8_0) {
                    const uint2 w = __ldg(reinterpret_cast<const uint2*>(at));
                    kw[r][b][0] = w.x;
                    kw[r][b][1] = w.y;
                } else {
                    kw[r][b][0] = __ldg(reinterpret_cast<const uint32_t*>(at));
                }
            }
            LoadScales<NB>(sc + 8 * r * NB, kd[r]);
        }
    }

    __device__ __forceinline__ void Scores(float (&x)[4]) const {
        x[0] = x[1] = x[2] = x[3] = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            uint32_t f[2][4];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                if constexpr (TYPE == MLB_Q8_0) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        f[i][r] = EvenBytes(kw[r][b][i], magic);
                        f[i][2 + r] = EvenBytes(kw[r][b][i] >> 8, magic);
                    }
                } else {
                    const uint32_t w = kw[r][b][0], u = w >> 8;
                    f[0][r] = LowNibbles(w, magic);
                    f[0][2 + r] = LowNibbles(u, magic);
                    f[1][r] = HighNibbles(w, magic);
                    f[1][2 + r] = HighNibbles(u, magic);
                }
            }
            float d[4];
            const uint4 q0 = qs[(2 * b) * 32], q1 = qs[(2 * b + 1) * 32];
            MmaFirst(d, f[0], q0.z, q0.w);
            Mma(d, f[1], q1.z, q1.w);
            Mma(d, f[0], q0.x, q0.y);
            Mma(d, f[1], q1.x, q1.y);
            const float d0 = ScaleOf(kd[0], b), d1 = ScaleOf(kd[1], b);
            x[0] = fmaf(d0, d[0], x[0]);
            x[1] = fmaf(d0, d[1], x[1]);
            x[2] = fmaf(d1, d[2], x[2]);
            x[3] = fmaf(d1, d[3], x[3]);
        }
    }

    __device__ __forceinline__ void ScaleColumns(float r0, float r1) {
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                o[b][j][0] *= r0;
                o[b][j][1] *= r1;
                o[b][j][2] *= r0;
                o[b][j][3] *= r1;
            }
    }

    // After the barrier that follows Begin.
    __device__ __forceinline__ void Ready(const Step& s, const float* undos) {
        cs[0] = undos[2 * s.c];
        cs[1] = undos[2 * s.c + 1];
    }

    // One unit of slots from p0, those below `low` another's; its K is loaded,
    // `next` is the K to load.
    __device__ __forceinline__ void Unit(const Step& s, int p0, int low, int next) {
        // slots 2c, 2c + 1, 2c + 8, 2c + 9
        uint32_t vw[NB][TYPE == MLB_Q8_0 ? 4 : 2];
        uint32_t vd[4][(NB + 1) / 2];
        {
            const int p = p0 + 2 * s.c;
            const uint8_t* row = v + size_t(p) * (NB * kQuantBytes) + (kQuantBytes / 8) * s.g;
            const __half* sc = vs + size_t(p) * NB;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int more = (i & 1) + (i >> 1) * 8;
                LoadScales<NB>(sc + more * NB, vd[i]);
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const uint8_t* at = row + more * (NB * kQuantBytes) + b * kQuantBytes;
                    if constexpr (TYPE == MLB_Q8_0) {
                        vw[b][i] = __ldg(reinterpret_cast<const uint32_t*>(at));
                    } else {
                        const uint32_t w = __ldg(reinterpret_cast<const unsigned short*>(at));
                        vw[b][i >> 1] = i & 1 ? vw[b][i >> 1] | (w << 16) : w;
                    }
                }
            }
        }
        float x[4];
        Scores(x);
        if (next >= 0) LoadK(s, next);
        Weights(s, p0, low, x, cs[0], cs[1], kOffset, m, l, [&](float r0, float r1) { ScaleColumns(r0, r1); });
        // weights as B fragments: row (query) g, slots 2c, 2c + 1 (+ 8)
        uint32_t ph0, pl0, ph1, pl1;
        SplitHalf(x[0], x[1], ph0, pl0);
        SplitHalf(x[2], x[3], ph1, pl1);
        ph0 = Transpose8x8(ph0);
        ph1 = Transpose8x8(ph1);
        pl0 = Transpose8x8(pl0);
        pl1 = Transpose8x8(pl1);
        uint32_t d0[NB], d1[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int pick = b & 1 ? 0x7632 : 0x5410;  // block b of two slots
            d0[b] = __byte_perm(vd[0][b >> 1], vd[1][b >> 1], pick);
            d1[b] = __byte_perm(vd[2][b >> 1], vd[3][b >> 1], pick);
        }
        if (low + kUnit > s.len) {  // a slot that is not seen may hold any scale, NaN too
            const uint32_t see0 = __hne2_mask(AsHalf2(ph0), AsHalf2(0u)), see1 = __hne2_mask(AsHalf2(ph1), AsHalf2(0u));
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                d0[b] &= see0;
                d1[b] &= see1;
            }
        }
        __half2 big = __hmax2(AsHalf2(d0[0]), AsHalf2(d1[0]));
#pragma unroll
        for (int b = 1; b < NB; ++b) big = __hmax2(big, __hmax2(AsHalf2(d0[b]), AsHalf2(d1[b])));
        const float top = fmaxf(__low2float(big), __high2float(big));
        if (__any_sync(0xffffffffu, top > bound)) {
            float t = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 2));
            // 2^ne > t, ne within the powers that a half can scale by
            const int ne = max(e, min(15, max(-15, static_cast<int>(__float_as_uint(t) >> 23) - 126)));
            const float f = Pow2(e - ne);
            SetPower(ne);
            ScaleColumns(__shfl_sync(0xffffffffu, f, 8 * s.c), __shfl_sync(0xffffffffu, f, 8 * s.c + 4));
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const __half2 s0 = __hmul2(AsHalf2(d0[b]), down), s1 = __hmul2(AsHalf2(d1[b]), down);
            const __half2 h0 = __hmul2(AsHalf2(ph0), s0), h1 = __hmul2(AsHalf2(ph1), s1);
            const uint32_t l0 = H2(__hfma2(AsHalf2(pl0), s0, __hfma2(AsHalf2(ph0), s0, __hneg2(h0))));
            const uint32_t l1 = H2(__hfma2(AsHalf2(pl1), s1, __hfma2(AsHalf2(ph1), s1, __hneg2(h1))));
            uint32_t f[2][4];
            if constexpr (TYPE == MLB_Q8_0) {
#pragma unroll
                for (int r = 0; r < 2; ++r) {  // slots 2c, 2c + 1, then + 8: bytes of the two side by side
                    const uint32_t low = __byte_perm(vw[b][2 * r], vw[b][2 * r + 1], 0x5410);
                    const uint32_t high = __byte_perm(vw[b][2 * r], vw[b][2 * r + 1], 0x7632);
                    f[0][2 * r] = EvenBytes(low, magic);
                    f[0][2 * r + 1] = EvenBytes(low >> 8, magic);
                    f[1][2 * r] = EvenBytes(high, magic);
                    f[1][2 * r + 1] = EvenBytes(high >> 8, magic);
                }
            } else {
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const uint32_t w = vw[b][r], u = w >> 8;
                    f[0][2 * r] = LowNibbles(w, magic);
                    f[0][2 * r + 1] = LowNibbles(u, magic);
                    f[1][2 * r] = HighNibbles(w, magic);
                    f[1][2 * r + 1] = HighNibbles(u, magic);
                }
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float d[4];
                MmaFirst(d, f[j], l0, l1);
                Mma(d, f[j], H2(h0), H2(h1));
                AddTo(o[b][j], d);
            }
        }
    }

    __device__ __forceinline__ void End(const Step& s) {
        const float f = Pow2(e);
        ScaleColumns(__shfl_sync(0xffffffffu, f, 8 * s.c), __shfl_sync(0xffffffffu, f, 8 * s.c + 4));
    }
};

// ---------------------------------------------------------------- fp32 caches
template <int NB>
struct F32Warp {
    float q[NB][8];
    float o[NB][2][4];
    float m[2], l[2], cs[2];
    const float *k, *v;
    size_t pitch;  // floats between slots
    int hd;

    __device__ __forceinline__ static int Dim(int g, int j, int half) { return 4 * g + 2 * j + half; }

    __device__ __forceinline__ void Begin(const TreeArgs& a, const TreeSplit&, const Step& s, int seq, int head,
                                          const float* qr, uint4*, float*, bool) {
        const long long row = a.c.Row(seq, a.layer, head, 0);
        k = static_cast<const float*>(a.c.k) + row * a.c.hd;
        v = static_cast<const float*>(a.c.v) + row * a.c.hd;
        pitch = size_t(a.c.n_kv) * a.c.hd;
        hd = a.c.hd;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int d = b * 32 + 8 * s.c + i;
                q[b][i] = qr && d < hd ? __ldg(qr + d) : 0.0f;
                o[b][i >> 2][i & 3] = 0.0f;
            }
        cs[0] = cs[1] = fmaxf(a.scale * kLog2e, 1e-37f);
        m[0] = m[1] = kStart;
        l[0] = l[1] = 0.0f;
    }

    __device__ __forceinline__ void Prefetch(const Step& s, int p0, int p1) const {
        // a lane per 128-byte line of the slots' rows
        const int lines = (hd * 4 + 127) / 128;
        for (int i = s.lane; i < (p1 - p0) * lines; i += 32) {
            const int p = p0 + i / lines;
            const size_t at = size_t(p) * pitch + (i % lines) * 32;
            asm volatile("prefetch.global.L2 [%0];" ::"l"(k + at));
            asm volatile("prefetch.global.L2 [%0];" ::"l"(v + at));
        }
    }

    __device__ __forceinline__ void Ready(const Step&, const float*) {}
    __device__ __forceinline__ void LoadK(const Step&, int) {}

    __device__ __forceinline__ void ScaleColumns(float r0, float r1) {
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                o[b][j][0] *= r0;
                o[b][j][1] *= r1;
                o[b][j][2] *= r0;
                o[b][j][3] *= r1;
            }
    }

    __device__ __forceinline__ float4 Load(const float* p, int d) const {
        return d < hd ? __ldg(reinterpret_cast<const float4*>(p + d)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }

    __device__ __forceinline__ void Unit(const Step& s, int p0, int low, int) {
        float x[4] = {0.0f, 0.0f, 0.0f, 0.0f}, rest[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        float4 kr[2][NB][2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const float* row = k + size_t(p0 + s.g + 8 * r) * pitch;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                kr[r][b][0] = Load(row, b * 32 + 8 * s.c);
                kr[r][b][1] = Load(row, b * 32 + 8 * s.c + 4);
            }
        }
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) {  // elements 2i, 2i + 1 of the thread's eight: k = c, c + 4
                const float4 ra = kr[0][b][i >> 1], rb = kr[1][b][i >> 1];
                uint32_t h[4], w[4], qh[2], qw[2];
                SplitTf32(i & 1 ? ra.z : ra.x, h[0], w[0]);
                SplitTf32(i & 1 ? rb.z : rb.x, h[1], w[1]);
                SplitTf32(i & 1 ? ra.w : ra.y, h[2], w[2]);
                SplitTf32(i & 1 ? rb.w : rb.y, h[3], w[3]);
                SplitTf32(q[b][2 * i], qh[0], qw[0]);
                SplitTf32(q[b][2 * i + 1], qh[1], qw[1]);
                MmaTf32(rest, w, qh[0], qh[1]);
                MmaTf32(rest, h, qw[0], qw[1]);
                MmaTf32(x, h, qh[0], qh[1]);
            }
        AddTo(x, rest);
        float4 vr[4][NB];  // slots c, c + 4, c + 8, c + 12
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float* row = v + size_t(p0 + s.c + 4 * i) * pitch;
#pragma unroll
            for (int b = 0; b < NB; ++b) vr[i][b] = Load(row, b * 32 + 4 * s.g);
        }
        Weights(s, p0, low, x, cs[0], cs[1], 0.0f, m, l, [&](float r0, float r1) { ScaleColumns(r0, r1); });
        if (low + kUnit > s.len) {
            bool odd = false;  // a slot that some rows do not see may hold NaN or infinities
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int b = 0; b < NB; ++b)
                    odd = odd || !(fabsf(vr[i][b].x) <= 3.4e38f && fabsf(vr[i][b].y) <= 3.4e38f &&
                                   fabsf(vr[i][b].z) <= 3.4e38f && fabsf(vr[i][b].w) <= 3.4e38f);
            if (__any_sync(0xffffffffu, odd)) {
                Plainly(s, p0, x);
                return;
            }
        }
        // weights as B fragments: query g, slots c and c + 4 (+ 8)
        float pw[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int src = 4 * (s.c + 4 * (i & 1)) + (s.g >> 1);
            const float even = __shfl_sync(0xffffffffu, x[i & 2], src), odd = __shfl_sync(0xffffffffu, x[(i & 2) + 1], src);
            pw[i] = s.g & 1 ? odd : even;
        }
        uint32_t ph[4], pl[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) SplitTf32(pw[i], ph[i], pl[i]);
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float d[4];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float4 va = vr[2 * i][b], vb = vr[2 * i + 1][b];
                    uint32_t h[4], w[4];
                    SplitTf32(j ? va.z : va.x, h[0], w[0]);
                    SplitTf32(j ? va.w : va.y, h[1], w[1]);
                    SplitTf32(j ? vb.z : vb.x, h[2], w[2]);
                    SplitTf32(j ? vb.w : vb.y, h[3], w[3]);
                    i == 0 ? MmaTf32First(d, w, ph[0], ph[1]) : MmaTf32(d, w, ph[2], ph[3]);
                    MmaTf32(d, h, pl[2 * i], pl[2 * i + 1]);
                    MmaTf32(d, h, ph[2 * i], ph[2 * i + 1]);
                }
                AddTo(o[b][j], d);
            }
    }

    // The weighted values of one unit slot by slot, those of weight 0 left out.
    __device__ __forceinline__ void Plainly(const Step& s, int p0, const float (&x)[4]) {
        for (int i = 0; i < kUnit && p0 + i < s.slots; ++i) {  // weights of slots below `low` are 0
            const int src = 4 * (i & 7) + s.c;
            const float w0 = __shfl_sync(0xffffffffu, i < 8 ? x[0] : x[2], src);
            const float w1 = __shfl_sync(0xffffffffu, i < 8 ? x[1] : x[3], src);
            const float* row = v + size_t(p0 + i) * pitch;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const float4 y = Load(row, b * 32 + 4 * s.g);
                const float e[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    float* to = &o[b][d >> 1][(d & 1) * 2];
                    if (w0 != 0.0f) to[0] = fmaf(w0, e[d], to[0]);
                    if (w1 != 0.0f) to[1] = fmaf(w1, e[d], to[1]);
                }
            }
        }
    }

    __device__ __forceinline__ void End(const Step&) {}
};

template <int TYPE, int NB>
struct WarpOf {
    using T = QuantWarp<TYPE, NB>;
};
template <int NB>
struct WarpOf<MLB_F32, NB> {
    using T = F32Warp<NB>;
};

__device__ __forceinline__ long long WarpSum64(long long v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

__device__ __forceinline__ long long EntryUnits(const TreeArgs& a, int b, int items) {
    return 1LL * ((FindEntry(a, b).slots + kUnit - 1) / kUnit) * items;
}

// Four consecutive elements of an output row.
__device__ __forceinline__ void StoreOut(const TreeArgs& a, float* row, int d, const float4& v) {
    if (a.out_vec) {
        if (d < a.c.hd) *reinterpret_cast<float4*>(row + d) = v;
        return;
    }
    const float e[4] = {v.x, v.y, v.z, v.w};
    for (int i = 0; i < 4; ++i)
        if (d + i < a.c.hd) row[d + i] = e[i];
}

__device__ __forceinline__ float* OutRow(const TreeArgs& a, int b, int head, int r) {
    return a.out + (size_t(b) * a.tokens + r / a.group) * a.out_stride + size_t(head * a.group + r % a.group) * a.c.hd;
}

// Sum of partial results: o 2^(m - M) over parts, M their largest maximum.
struct Joined {
    float m = kStart, l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);

    __device__ __forceinline__ void Add(float pm, float pl, const float4& po) {
        const float n = fmaxf(m, pm), a = Exp2(m - n), b = Exp2(pm - n);
        m = n;
        l = l * a + pl * b;
        o.x = o.x * a + po.x * b;
        o.y = o.y * a + po.y * b;
        o.z = o.z * a + po.z * b;
        o.w = o.w * a + po.w * b;
    }
    __device__ __forceinline__ float4 Result() const {
        const float r = l == 0.0f ? 0.0f : 1.0f / l;
        return make_float4(o.x * r, o.y * r, o.z * r, o.w * r);
    }
};

template <int NB>
constexpr int JoinPitch() {
    return NB * 32 + 4;
}

template <int TYPE, int NB, int NW>
__global__ void __launch_bounds__(NW * 32, 1) TreeMmaKernel(TreeArgs a, TreeSplit sp) {
    constexpr int kPitch = JoinPitch<NB>(), kFours = NB * 8;
    extern __shared__ float4 smem4[];
    float* so = reinterpret_cast<float*>(smem4);  // [NW][kRows][kPitch]
    float* sm = so + NW * kRows * kPitch;         // [NW][kRows]
    float* sl = sm + NW * kRows;
    float* su = sl + NW * kRows;                            // [4][kRows]
    uint4* sq = reinterpret_cast<uint4*>(su + 4 * kRows);   // [wq][2 NB][32], quantized caches
    __shared__ int s_last;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int nt = warp % sp.wq, wp = warp / sp.wq, wps = NW / sp.wq;
    const int items = a.c.n_kv * sp.groups, item_rows = kRows * sp.wq;

    // entries with nothing to see
    for (int b = blockIdx.x; b < a.batch; b += gridDim.x) {
        if (FindEntry(a, b).slots != 0) continue;
        for (int t = warp; t < a.tokens; t += NW)
            for (int i = lane; i < a.n_heads * a.c.hd; i += 32)
                a.out[(size_t(b) * a.tokens + t) * a.out_stride + i] = 0.0f;
    }

    // the cut: all units in a row, an even stretch for each CTA
    long long total = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 32)
        total += WarpSum64(b0 + lane < a.batch ? EntryUnits(a, b0 + lane, items) : 0);
    if (total == 0) return;
    const long long want = (total + wps - 1) / wps;  // a unit for each warp at least
    const long long ctas = want < gridDim.x ? want : gridDim.x;
    if (blockIdx.x >= ctas) return;
    long long cur = total * blockIdx.x / ctas;
    const long long end = total * (blockIdx.x + 1) / ctas;
    // the entry of the first unit
    int b = 0;
    long long first = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 32) {
        const long long n = b0 + lane < a.batch ? EntryUnits(a, b0 + lane, items) : 0;
        const long long chunk = WarpSum64(n);
        if (cur >= first + chunk) {
            first += chunk;
            continue;
        }
        long long incl = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long t = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += t;
        }
        const int at = __ffs(__ballot_sync(0xffffffffu, first + incl > cur)) - 1;
        first += __shfl_sync(0xffffffffu, incl - n, at);
        b = b0 + at;
        break;
    }

    Step s;
    s.lane = lane;
    s.g = lane >> 2;
    s.c = lane & 3;
    s.tokens = a.tokens;
    s.words = a.words;
    typename WarpOf<TYPE, NB>::T w;
    while (cur < end) {
        const Entry e = FindEntry(a, b);
        const int units = (e.slots + kUnit - 1) / kUnit;
        if (cur - first >= 1LL * units * items) {  // the next entry
            first += 1LL * units * items;
            ++b;
            continue;
        }
        const int item = static_cast<int>((cur - first) / units);
        const int u0 = static_cast<int>((cur - first) - 1LL * item * units);
        const int u1 = static_cast<int>(end - cur < units - u0 ? u0 + (end - cur) : units);
        const int head = item / sp.groups, row0 = (item - head * sp.groups) * item_rows;

        // ---- this warp's units of the item
        const int tile = row0 + nt * kRows;
        s.slots = e.slots;
        s.len = e.len;
        s.mask = a.mask ? a.mask + size_t(b) * a.tokens * a.words : nullptr;
        s.t0 = (tile + 2 * s.c) / a.group;
        s.t1 = (tile + 2 * s.c + 1) / a.group;
        float* to = so + (warp * kRows + 2 * s.c) * kPitch;
        const bool live = tile < sp.rows;
        if (live) {
            const int r = tile + s.g;
            const float* q = r < sp.rows ? a.q + (size_t(b) * a.tokens + r / a.group) * a.q_stride +
                                               size_t(head * a.group + r % a.group) * a.c.hd
                                         : nullptr;
            w.Begin(a, sp, s, e.seq, head, q, sq + nt * 2 * NB * 32, su + nt * kRows, wp == 0);
            // the last unit of the plane may hold 8 slots only: it starts earlier and leaves out the others
            const int top = a.c.head_slots - kUnit;
            // a round is a unit of every warp; the warps take turns to prefetch one
            const int span = wps * kUnit;
            if (nt == 0 && wp < kAhead && u0 * kUnit + (wp + 1) * span < e.slots && (wp + 1) * wps < u1 - u0)
                w.Prefetch(s, u0 * kUnit + (wp + 1) * span, min(min(u0 * kUnit + (wp + 2) * span, u1 * kUnit), e.slots));
            if (u0 + wp < u1) w.LoadK(s, min((u0 + wp) * kUnit, top));
        }
        if (TYPE != MLB_F32) __syncthreads();
        if (live) {
            w.Ready(s, su + nt * kRows);
            const int top = a.c.head_slots - kUnit, span = wps * kUnit;
            int u = u0 + wp;
            for (int round = 0; u < u1; u += wps, ++round) {
                const int ahead = (u0 + (round + kAhead + 1) * wps) * kUnit;
                if (nt == 0 && round % wps == wp && ahead < min(u1 * kUnit, e.slots))
                    w.Prefetch(s, ahead, min(min(ahead + span, u1 * kUnit), e.slots));
                w.Unit(s, min(u * kUnit, top), u * kUnit, u + wps < u1 ? min((u + wps) * kUnit, top) : -1);
            }
            w.End(s);
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) {
                w.l[0] += __shfl_xor_sync(0xffffffffu, w.l[0], o);
                w.l[1] += __shfl_xor_sync(0xffffffffu, w.l[1], o);
            }
#pragma unroll
            for (int k = 0; k < NB; ++k)
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int d = k * 32 + w.Dim(s.g, j, h);
                        to[d] = w.o[k][j][2 * h];
                        to[kPitch + d] = w.o[k][j][2 * h + 1];
                    }
            if (s.g == 0) {
                sm[warp * kRows + 2 * s.c] = w.m[0];
                sm[warp * kRows + 2 * s.c + 1] = w.m[1];
                sl[warp * kRows + 2 * s.c] = w.l[0];
                sl[warp * kRows + 2 * s.c + 1] = w.l[1];
            }
        }
        __syncthreads();

        // ---- join the warps
        const bool whole = u0 == 0 && u1 == units;
        const size_t part_floats = size_t(item_rows) * (NB * 32 + 2);
        float* part = sp.parts + (2 * size_t(blockIdx.x) + (u0 == 0 ? 1 : 0)) * part_floats;
        const int live_rows = min(item_rows, sp.rows - row0);
        for (int i = threadIdx.x; i < live_rows * kFours; i += NW * 32) {
            const int r = i / kFours, d = (i - r * kFours) * 4;
            Joined x;
            for (int k = 0; k < wps; ++k) {
                const int at = (k * sp.wq + r / kRows) * kRows + r % kRows;
                x.Add(sm[at], sl[at], *reinterpret_cast<const float4*>(so + at * kPitch + d));
            }
            if (whole) {
                StoreOut(a, OutRow(a, b, head, row0 + r), d, x.Result());
            } else {
                __stcg(reinterpret_cast<float4*>(part + r * NB * 32 + d), x.o);
                if (d == 0) {
                    __stcg(part + item_rows * NB * 32 + r, x.m);
                    __stcg(part + item_rows * (NB * 32 + 1) + r, x.l);
                }
            }
        }

        // ---- join the CTAs that share the item: the last to arrive adds them up
        if (!whole) {
            const long long i0 = cur - u0, i1 = i0 + units - 1;  // the item's first and last unit
            const int c0 = static_cast<int>(((i0 + 1) * ctas - 1) / total), c1 = static_cast<int>(((i1 + 1) * ctas - 1) / total);
            __threadfence();
            __syncthreads();
            if (threadIdx.x == 0) {
                int* counter = sp.counters + size_t(b) * items + item;
                s_last = atomicAdd(counter, 1) == c1 - c0;
                if (s_last) *counter = 0;  // every contributor has arrived
            }
            __syncthreads();
            if (s_last) {
                __threadfence();
                // parts: the first CTA's begins at the item's start where it holds its first unit
                for (int i = threadIdx.x; i < live_rows * kFours; i += NW * 32) {
                    const int r = i / kFours, d = (i - r * kFours) * 4;
                    Joined x;
                    for (int k = c0; k <= c1; k += 4) {
                        float pm[4], pl[4];
                        float4 po[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            if (k + j > c1) break;
                            const float* p = sp.parts + (2 * size_t(k + j) + (k + j == c0 ? 1 : 0)) * part_floats;
                            pm[j] = __ldcg(p + item_rows * NB * 32 + r);
                            pl[j] = __ldcg(p + item_rows * (NB * 32 + 1) + r);
                            po[j] = __ldcg(reinterpret_cast<const float4*>(p + r * NB * 32 + d));
                        }
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if (k + j <= c1) x.Add(pm[j], pl[j], po[j]);
                    }
                    StoreOut(a, OutRow(a, b, head, row0 + r), d, x.Result());
                }
            }
        }
        __syncthreads();
        cur += u1 - u0;
    }
}

int* Counters(DeviceContext& ctx, size_t n) {
    if (n <= ctx.tree_counter_count) return ctx.tree_counters;
    if (ctx.tree_counters) CheckCuda(cudaFreeAsync(ctx.tree_counters, ctx.stream), "cudaFreeAsync");
    ctx.tree_counters = nullptr;
    ctx.tree_counter_count = 0;
    const size_t want = std::max<size_t>(n, 4096);
    void* p = nullptr;
    CheckCuda(cudaMallocFromPoolAsync(&p, want * sizeof(int), ctx.pool, ctx.stream), "cudaMallocFromPoolAsync(counters)");
    CheckCuda(cudaMemsetAsync(p, 0, want * sizeof(int), ctx.stream), "cudaMemsetAsync(counters)");
    ctx.tree_counters = static_cast<int*>(p);
    ctx.tree_counter_count = want;
    return ctx.tree_counters;
}

template <int TYPE, int NB>
void Launch(DeviceContext& ctx, const TreeArgs& a) {
    // registers per thread bound the warps: fp32 units hold twice the values
    #ifndef TREE_NW
#define TREE_NW 12
#endif
    constexpr int NW = TYPE == MLB_F32 && NB > 2 ? 8 : TREE_NW;
    TreeSplit sp{};
    sp.rows = a.tokens * a.group;
    sp.wq = sp.rows <= kRows ? 1 : (sp.rows <= 2 * kRows ? 2 : 4);
    sp.groups = static_cast<int>(CeilDiv(sp.rows, kRows * sp.wq));
    const size_t items = size_t(a.c.n_kv) * sp.groups;
    // an upper bound of the units, from the caller's bound of the lengths
    const long long slots = std::min<long long>(1LL * std::min(a.max_len, a.c.max_seq) + a.tokens, a.c.max_seq);
    const long long units = 1LL * a.batch * items * CeilDiv(slots, kUnit), per_cta = NW / sp.wq;
    const int grid = static_cast<int>(std::max(1LL, std::min<long long>(ctx.sm_count, (units + per_cta - 1) / per_cta)));
    const size_t part = size_t(kRows) * sp.wq * (NB * 32 + 2) * sizeof(float);
    sp.parts = static_cast<float*>(Workspace(ctx, 2 * size_t(grid) * part));
    sp.magic = TYPE == MLB_Q8_0 ? kMagic8 : kMagic4;
    sp.counters = Counters(ctx, size_t(a.batch) * items);
    constexpr size_t smem = (size_t(NW) * kRows * (JoinPitch<NB>() + 2) + 4 * kRows) * sizeof(float) +
                            (TYPE == MLB_F32 ? 0 : 4 * 2 * NB * 32 * sizeof(uint4));
    auto* kernel = TreeMmaKernel<TYPE, NB, NW>;
    if (smem > 48 * 1024)
        CheckCuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem),
                  "cudaFuncSetAttribute(TreeMmaKernel)");
    kernel<<<grid, NW * 32, smem, ctx.stream>>>(a, sp);
    CheckCuda(cudaGetLastError(), "TreeMmaKernel");
}

template <int TYPE>
bool LaunchBlocks(DeviceContext& ctx, const TreeArgs& a) {
    switch (a.c.blocks) {
        case 1: Launch<TYPE, 1>(ctx, a); return true;
        case 2: Launch<TYPE, 2>(ctx, a); return true;
        case 3: Launch<TYPE, 3>(ctx, a); return true;
        case 4: Launch<TYPE, 4>(ctx, a); return true;
        default: return false;
    }
}

}  // namespace

bool LaunchTreeMma(DeviceContext& ctx, const TreeArgs& a) {
    if (a.c.head_slots < kUnit) return false;  // a unit is 16 slots
    if (a.c.type == MLB_F32) return a.cache_vec && LaunchBlocks<MLB_F32>(ctx, a);
    return a.c.type == MLB_Q8_0 ? LaunchBlocks<MLB_Q8_0>(ctx, a) : LaunchBlocks<MLB_Q4_0>(ctx, a);
}

}  // namespace mlb
