// Attention of drafted tokens on the warp-level matrix instructions: few query
// rows per KV head, the cache read once.
//
// The R = tokens x (query heads per KV head) rows that share a KV head are cut
// into tiles of eight: the N side of mma.m16n8k16.  A warp takes 16 slots of
// the cache at a time (the M side, S^T = K Q^T) for a tile of rows (fp32: NT = 1 or 2):
//   K      the 16 x head_dim quants as A fragments (the order of the elements
//          within a block is free, as Q is laid out in the same one), fp16 whole
//          numbers: exact.  Q is scaled per row by a power of two and split into
//          fp16 hi + lo (22 bits), so a block's products are exact up to the
//          fp32 sum; the slot's scale of the block multiplies that sum.
//   softmax  running maximum and sum per row, the maximum moved only when a
//          score passes it by 2^2 (a vote): weights are 2^(x - m + 12) <= 2^14,
//          split into fp16 hi + lo and turned into B fragments by movmatrix.
//   V      O^T = V^T P^T: quants as exact fp16 A fragments again (byte
//          transposition in registers); the slot's scale of a block goes into
//          the weights, P' = hi + lo of p d by one product and two FMAs on half
//          pairs, relative to a power of two that all scales of the unit lie close
//          below, so that d 2^-e is a normal half, exact.  Where they spread wider
//          (one slot with large values among others) the unit is summed in fp32, slot
//          by slot.  Two MMAs per fragment.
// fp32 caches take the same path with mma.m16n8k8 on tf32 hi + lo pairs (three
// products; no ranges to mind).  A unit's weighted values are summed in fresh
// accumulators and added to the running ones in fp32 with rounding to nearest:
// the matrix unit's own additions truncate, which over a long context would
// cost several times the fp32 rounding.
//
// Bound: a decode step over long sequences (4 rows, 32 sequences, 304 MB in Q8_0)
// runs at 4.1 TB/s, 62 % of the copy rate; the instructions of a unit (conversion,
// fragments, softmax) take about as long as its bytes, and overlap them in part.
// In 4 bits (151 MB, 32 K slots) it is the instructions: 2.5 TB/s.  Neither the issue
// slots (58 and 55 %) nor a pipe is full: with three warps to a scheduler the
// dependences within a unit show.  From 16 rows on it is instructions and matrix products,
// for fp32 the tf32 products (three for one: 49 % of the tensor pipe's cycles).
//
// The units (32 slots, fp32 16) of all (sequence, KV head, row group) items are one
// list, cut evenly over the CTAs (the lengths are on the device, so every CTA
// works the cut out from them): sequences of any lengths balance.  A CTA's
// stretch is dealt out to groups of WQ warps, a tile (fp32: or two) of the item's rows
// each; a group brings its units into a ring of S stages in shared memory
// (cp.async, S - 1 units ahead; rows an odd number of 16-byte chunks apart, so
// every fragment load is free of bank conflicts) and meets at a named barrier
// once per unit.  The groups join their results in shared memory, and a second
// kernel joins the items that are cut between CTAs (partials in the workspace,
// added in a fixed order).
#pragma once

#include <algorithm>
#include <cmath>

#include "tree_attention.cuh"

namespace mlb {

namespace {

constexpr int kSlots = 16;          // slots of a matrix step
constexpr int kRows = 8;            // query rows of a tile
constexpr float kStart = -3.4028235e38f;  // running maximum before the first score (the lowest finite: no inf - inf)
constexpr float kLag = 2.0f;        // how far scores may pass the running maximum, in powers of two
constexpr float kOffset = 12.0f;    // weights are relative to 2^12: at most 2^14, and the fp16 pairs resolve
                                    // 2^-37 of the largest, for slots that weigh little where the heavy ones hold zeros
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLeast = 1e-45f;  // a score factor is not 0: no inf * 0

constexpr int kSmShared = 226 * 1024;  // shared memory of an SM for its CTAs
constexpr int kMaxStages = 4;

struct TreeSplit {
    int groups;    // items of a (sequence, KV head): ceil(R / (8 NT WQ))
    int rows;      // R
    float* parts;  // two partial results per CTA
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

// Exponent s with (top * 2^s) in [2^14, 2^15), for queries of any size: ScaleExp of the linears stops at 2^100 either
// way.  Below 2^-112 the result stays smaller, with bits to spare, so that 2^-s is a normal number.
__device__ __forceinline__ int QueryExp(float top) {
    if (!(top > 0.0f) || !isfinite(top)) return 0;
    return min(126, 14 - (static_cast<int>(__float_as_uint(top) >> 23) - 127));
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
// matrix unit does not read: together 2^-21 relative at worst.  From 2^128 (1 - 2^-12)
// on the rounding carries to infinity; a form without that (keeping the largest, or
// cutting instead of rounding) cost 4 to 13 %, so the header states the limit.
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

// The fp16 scales of one slot's blocks in shared memory, two to a word.
template <int NB>
__device__ __forceinline__ void LoadScales(const __half* p, uint32_t (&d)[(NB + 1) / 2]) {
    if constexpr (NB % 4 == 0) {
#pragma unroll
        for (int i = 0; i < NB / 4; ++i) {
            const uint2 w = reinterpret_cast<const uint2*>(p)[i];
            d[2 * i] = w.x;
            d[2 * i + 1] = w.y;
        }
    } else if constexpr (NB % 2 == 0) {
#pragma unroll
        for (int i = 0; i < NB / 2; ++i) d[i] = reinterpret_cast<const uint32_t*>(p)[i];
    } else {
        const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
        for (int i = 0; i < NB / 2; ++i) d[i] = h[2 * i] | (uint32_t(h[2 * i + 1]) << 16);
        d[NB / 2] = h[NB - 1];
    }
}

template <int N>
__device__ __forceinline__ float ScaleOf(const uint32_t (&d)[N], int b) {
    return b & 1 ? __high2float(AsHalf2(d[b >> 1])) : __low2float(AsHalf2(d[b >> 1]));
}

// The rows, lengths and mask that a warp's step needs, common to all forms.
struct Step {
    int lane, g, c;  // lane = 4 g + c
    int slots, len, tokens, words;
    const uint64_t* mask;  // the batch entry's
};

// Without branches, so that the mask words of several slots load together.
__device__ __forceinline__ bool Sees(const Step& s, int t, int slot) {
    const int j = min(max(slot - s.len, 0), s.tokens - 1), row = min(t, s.tokens - 1);
    const bool draft = s.mask ? (__ldg(s.mask + size_t(row) * s.words + (j >> 6)) >> (j & 63)) & 1 : j <= row;
    return slot < s.len || (draft && slot < s.slots);
}

// Whether a largest score `top` moves the running maximum m (both before their factor cs).
__device__ __forceinline__ bool Passes(float top, float m, float cs) {
    return (top - m) * cs > kLag;
}
// A part's maximum with its factor, in powers of two; l: the sum of its weights (0: nothing seen).
__device__ __forceinline__ float Scaled(float m, float cs, float l) { return l > 0.0f ? fmaxf(m * cs, kStart) : kStart; }

// One tile of rows: drafted tokens, running maxima and sums of the thread's two
// score columns (queries 2c, 2c + 1).  The maxima are scores before their factor: only
// differences are multiplied by it, so that scores of any size weigh 2^0 at their maximum.
struct Columns {
    int t0, t1;
    float m[2], l[2], cs[2];

    __device__ __forceinline__ void Begin(int t_a, int t_b) {
        t0 = t_a;
        t1 = t_b;
        m[0] = m[1] = kStart;
        l[0] = l[1] = 0.0f;
    }

    // Scores (C fragments: rows slot g, g + 8; columns query 2c, 2c + 1) of the H
    // steps of a unit at p0, slots from `low` on, to weights 2^(x - m + offset);
    // `edge`: not every row sees all of it.  `rescale` gets the factors of a
    // moved maximum.
    template <int H, typename Rescale>
    __device__ __forceinline__ void Weights(const Step& s, int p0, int low, bool edge, float (&x)[H][4], float offset,
                                            Rescale&& rescale) {
        if (edge) {  // drafted slots, or the end
            bool see[H][4];
#pragma unroll
            for (int h = 0; h < H; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int slot = p0 + h * kSlots + s.g + (i >> 1) * 8;
                    see[h][i] = slot >= low && Sees(s, i & 1 ? t1 : t0, slot);
                }
#pragma unroll
            for (int h = 0; h < H; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (!see[h][i]) x[h][i] = -INFINITY;
        }
        float top0 = fmaxf(x[0][0], x[0][2]), top1 = fmaxf(x[0][1], x[0][3]);
#pragma unroll
        for (int h = 1; h < H; ++h) {
            top0 = fmaxf(top0, fmaxf(x[h][0], x[h][2]));
            top1 = fmaxf(top1, fmaxf(x[h][1], x[h][3]));
        }
        if (__any_sync(0xffffffffu, Passes(top0, m[0], cs[0]) || Passes(top1, m[1], cs[1]))) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) {
                top0 = fmaxf(top0, __shfl_xor_sync(0xffffffffu, top0, o));
                top1 = fmaxf(top1, __shfl_xor_sync(0xffffffffu, top1, o));
            }
            const float n0 = fmaxf(m[0], top0), n1 = fmaxf(m[1], top1);
            const float r0 = Exp2((m[0] - n0) * cs[0]), r1 = Exp2((m[1] - n1) * cs[1]);
            m[0] = n0;
            m[1] = n1;
            l[0] *= r0;
            l[1] *= r1;
            rescale(r0, r1);
        }
#pragma unroll
        for (int h = 0; h < H; ++h) {
            x[h][0] = Exp2(fmaf(x[h][0] - m[0], cs[0], offset));
            x[h][1] = Exp2(fmaf(x[h][1] - m[1], cs[1], offset));
            x[h][2] = Exp2(fmaf(x[h][2] - m[0], cs[0], offset));
            x[h][3] = Exp2(fmaf(x[h][3] - m[1], cs[1], offset));
            l[0] += x[h][0] + x[h][2];
            l[1] += x[h][1] + x[h][3];
        }
    }
};

// O^T fragments of one tile: [block][row tile][C fragment].
template <int NB>
struct Values {
    float o[NB][2][4];

    __device__ __forceinline__ void Clear() {
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int i = 0; i < 8; ++i) o[b][i >> 2][i & 3] = 0.0f;
    }
    __device__ __forceinline__ void Scale(float r0, float r1) {
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
};

// 16 bytes to shared memory, `bytes` (16 or 0) of them read and the rest zeros.
__device__ __forceinline__ void CopyChunk(uint32_t to, const void* from, int bytes = 16) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}

// Shared-memory loads by 32-bit address; volatile: they stay behind the waits.
__device__ __forceinline__ uint32_t LoadWord(uint32_t at, int more) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at + more));
    return v;
}
__device__ __forceinline__ uint32_t LoadHalf(uint32_t at, int more) {
    uint16_t v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(at + more));
    return v;
}

// ---------------------------------------------------------------- quantized caches
// A warp's running result for a tile of rows over Q8_0 / Q4_0 slots, two steps of
// 16 slots to a unit: half the sums of the fresh accumulators and half the loads
// of Q of one step.
template <int TYPE, int NB>
struct QuantWarp {
    static constexpr int H = 2;
    static constexpr int kUnit = kSlots * H;
    static constexpr int kQuantBytes = TYPE == MLB_Q8_0 ? 32 : 16;
    static constexpr int kChunks = NB * kQuantBytes / 16;  // of a row
    // Rows of eight chunks are stored with chunk j at j ^ (row % 8), others an odd number of chunks apart: either
    // way the rows that a fragment load touches lie in different banks.
    static constexpr bool kXor = TYPE == MLB_Q8_0 && kChunks == 8;
    static constexpr int kPitch = kXor ? 128 : (kChunks | 1) * 16;
    static constexpr int kPlane = kUnit * kPitch, kScales = kUnit * NB * 2;
    static constexpr int kStageBytes = kPlane + kScales;   // of K, and of V
    static_assert(!kXor || kStageBytes % 128 == 0, "the chunk bits of a stage's address are free");
    static constexpr int kFrags = 2 * NB;                  // uint4 per lane and tile: (hi, hi, lo, lo)

    Values<NB> v[1];
    Columns col[1];
    // P' is relative to 2^e, and takes scales above 2^(e - kSpan): with fewer binades than the 14 of the normal halves
    // the products with small weights keep the rest.  (Every nonzero scale for the lowest e.)
    static constexpr int kSpan = 10, kLowest = -15, kHighest = 15;  // powers that a half can scale by
    __half2 bound, least;  // 2^e, 2^(e - kSpan)
    __half2 down;          // 2^-e
    // weights of the unit as B fragments: row (query) g, slots 2c, 2c + 1 (+ 8), hi and lo
    uint32_t ph[H][2], pl[H][2];
    bool edge;         // not every row sees all of the unit
    uint32_t magic;
    const uint8_t *kp, *vp;  // the head's planes
    const __half *ksp, *vsp;

    // Output element of a block in o[.][j][0..1] (half 0: row g of the fragment)
    // or o[.][j][2..3] (half 1: row g + 8).
    __device__ __forceinline__ static int Dim(int g, int j, int half) {
        return TYPE == MLB_Q8_0 ? 4 * g + 2 * j + half : 16 * j + 2 * g + half;
    }

    // Q fragments of one tile (rows q of row g; null: none) and its score factors.
    __device__ __forceinline__ static void LayOut(const TreeArgs& a, const Step& s, const float* q, uint4* frags,
                                                  float* undos) {
        // the thread's elements of its row g in the order of the K fragments: 4c .. 4c + 3 and 16 further
        float x[NB][8], top = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int d = b * 32 + 16 * half + 4 * s.c;
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
        const int up = QueryExp(top);  // largest |q| into [2^14, 2^15)
        const float sc = Pow2(up), undo = fmaxf(Pow2(-up) * a.scale * kLog2e, kLeast);
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

    __device__ __forceinline__ void SetPower(int to) {
        bound = __float2half2_rn(Pow2(to));
        least = __float2half2_rn(to > kLowest ? Pow2(to - kSpan) : 0.0f);
        down = __float2half2_rn(Pow2(-to));
    }

    __device__ __forceinline__ void Begin(const TreeArgs& a, const TreeSplit& sp, int seq, int head) {
        magic = sp.magic;
        const long long row = a.c.Row(seq, a.layer, head, 0);
        kp = static_cast<const uint8_t*>(a.c.k) + row * NB * kQuantBytes;
        vp = static_cast<const uint8_t*>(a.c.v) + row * NB * kQuantBytes;
        ksp = a.c.ks + row * NB;
        vsp = a.c.vs + row * NB;
        v[0].Clear();
        SetPower(kLowest);
    }

    // K (or V) of the unit at p0 into a ring stage, by the COUNT threads of a group.
    template <int COUNT>
    __device__ __forceinline__ static void Copy(const uint8_t* plane, const __half* scales, uint32_t stage, int p0, int id) {
        const uint8_t* from = plane + size_t(p0) * (NB * kQuantBytes);
        constexpr int kAll = kUnit * kChunks;
#pragma unroll
        for (int j = 0; j < (kAll + COUNT - 1) / COUNT; ++j) {
            const int i = id + j * COUNT;
            if (kAll % COUNT != 0 && i >= kAll) break;
            const int row = i / kChunks, chunk = i % kChunks;
            CopyChunk(stage + row * kPitch + (kXor ? chunk ^ (row & 7) : chunk) * 16, from + i * 16);
        }
        constexpr int kSc = kScales / 16;
        static_assert(kSc <= COUNT, "a piece of scales to a thread");
        if (id < kSc) CopyChunk(stage + kPlane + id * 16, scales + size_t(p0) * NB + id * 8);
    }
    template <int COUNT>
    __device__ __forceinline__ void CopyK(uint32_t stage, int p0, int id) const {
        Copy<COUNT>(kp, ksp, stage, p0, id);
    }
    template <int COUNT>
    __device__ __forceinline__ void CopyV(uint32_t stage, int p0, int id) const {
        Copy<COUNT>(vp, vsp, stage, p0, id);
    }

    // Scores and weights of the unit at p0, its K staged; slots below `low` are
    // another unit's.
    __device__ __forceinline__ void Keys(const Step& s, const uint8_t* stage, const uint4* frags, int p0, int low) {
        edge = low + kUnit > s.len;
        float x[H][4];
#pragma unroll
        for (int h = 0; h < H; ++h) x[h][0] = x[h][1] = x[h][2] = x[h][3] = 0.0f;
        {
            const __half* sc = reinterpret_cast<const __half*>(stage + kPlane) + s.g * NB;
            uint32_t kd[2 * H][(NB + 1) / 2];
#pragma unroll
            for (int r = 0; r < 2 * H; ++r) LoadScales<NB>(sc + 8 * r * NB, kd[r]);
            // (with kXor the address bits of the chunk hold g, and chunk j is one exclusive or away)
            const uint32_t row = SmemAddr(stage) + s.g * kPitch + 4 * s.c + (kXor ? s.g * 16 : 0);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const uint4 q0 = frags[2 * b * 32];
                const uint4 q1 = frags[(2 * b + 1) * 32];
#pragma unroll
                for (int h = 0; h < H; ++h) {
                    uint32_t f[2][4];
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const int step = (8 * r + h * kSlots) * kPitch;
                        if constexpr (TYPE == MLB_Q8_0) {
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                const int chunk = (2 * b + i) * 16;
                                const uint32_t w = kXor ? LoadWord(row ^ chunk, step) : LoadWord(row, step + chunk);
                                f[i][r] = EvenBytes(w, magic);
                                f[i][2 + r] = EvenBytes(w >> 8, magic);
                            }
                        } else {
                            const uint32_t w = LoadWord(row, step + b * 16), u = w >> 8;
                            f[0][r] = LowNibbles(w, magic);
                            f[0][2 + r] = LowNibbles(u, magic);
                            f[1][r] = HighNibbles(w, magic);
                            f[1][2 + r] = HighNibbles(u, magic);
                        }
                    }
                    const float d0 = ScaleOf(kd[2 * h], b), d1 = ScaleOf(kd[2 * h + 1], b);
                    float d[4];
                    MmaFirst(d, f[0], q0.z, q0.w);
                    Mma(d, f[1], q1.z, q1.w);
                    Mma(d, f[0], q0.x, q0.y);
                    Mma(d, f[1], q1.x, q1.y);
                    float(&to)[4] = x[h];
                    to[0] = fmaf(d0, d[0], to[0]);
                    to[1] = fmaf(d0, d[1], to[1]);
                    to[2] = fmaf(d1, d[2], to[2]);
                    to[3] = fmaf(d1, d[3], to[3]);
                }
            }
        }
        col[0].Weights(s, p0, low, edge, x, kOffset, [&](float r0, float r1) { v[0].Scale(r0, r1); });
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                SplitHalf(x[h][2 * i], x[h][2 * i + 1], ph[h][i], pl[h][i]);
                ph[h][i] = Transpose8x8(ph[h][i]);
                pl[h][i] = Transpose8x8(pl[h][i]);
            }
    }

    // The power for the unit's scales; false: they spread too wide for one.  They lie side by side, a word or a few to a
    // lane; zeros do not matter, and what slots that are not seen hold may at worst choose the plain form.
    __device__ __forceinline__ bool Choose(const Step& s, const uint8_t* stage) {
        const uint32_t* sc = reinterpret_cast<const uint32_t*>(stage + kPlane) + s.lane;
        __half2 big = AsHalf2(0u), small = AsHalf2(0x7C007C00u);
#pragma unroll
        for (int i = 0; i < kScales / 4; i += 32) {
            const uint32_t d = kScales / 4 % 32 == 0 || i + s.lane < kScales / 4 ? sc[i] & 0x7fff7fffu : 0u;
            big = __hmax2(big, AsHalf2(d));
            small = __hmin2(small, AsHalf2(d | (__heq2_mask(AsHalf2(d), AsHalf2(0u)) & 0x7C007C00u)));
        }
        if (!__any_sync(0xffffffffu, !(__hble2(big, bound) && __hbgt2(small, least)))) return true;
        const uint32_t most = __reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(__low2float(big), __high2float(big))));
        SetPower(min(kHighest, max(kLowest, static_cast<int>(most >> 23) - 126)));  // 2^e > the largest
        return __all_sync(0xffffffffu, __hbgt2(small, least));
    }

    // The weighted values of the unit, its V staged.
    __device__ __forceinline__ void Sum(const Step& s, const uint8_t* stage) {
        if (!Choose(s, stage)) {
            Plainly(s, stage);
            return;
        }
        uint32_t d[H][2][NB];  // the scales of slots 2c, 2c + 1 (+ 8) as half pairs
        {
            const __half* sc = reinterpret_cast<const __half*>(stage + kPlane) + 2 * s.c * NB;
#pragma unroll
            for (int h = 0; h < H; ++h)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    uint32_t va[(NB + 1) / 2], vb[(NB + 1) / 2];
                    LoadScales<NB>(sc + (i * 8 + h * kSlots) * NB, va);
                    LoadScales<NB>(sc + (i * 8 + h * kSlots + 1) * NB, vb);
#pragma unroll
                    for (int b = 0; b < NB; ++b)
                        d[h][i][b] = __byte_perm(va[b >> 1], vb[b >> 1], b & 1 ? 0x7632 : 0x5410);
                }
        }
        const float up = __low2float(bound);
        const uint32_t row = SmemAddr(stage) + 2 * s.c * kPitch +
                             (kXor ? ((s.g >> 2) ^ (2 * s.c)) * 16 + 4 * (s.g & 3) : (kQuantBytes / 8) * s.g);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            float t[2][4];
#pragma unroll
            for (int h = 0; h < H; ++h) {
                uint32_t f[2][4];
#pragma unroll
                for (int r = 0; r < 2; ++r) {  // slots 2c, 2c + 1, then + 8
                    const int step = (8 * r + h * kSlots) * kPitch, chunk = b * kQuantBytes;
                    if constexpr (TYPE == MLB_Q8_0) {
                        const uint32_t w0 = kXor ? LoadWord(row ^ chunk, step) : LoadWord(row, step + chunk);
                        const uint32_t w1 = kXor ? LoadWord(row ^ (chunk + 16), step + kPitch)
                                                 : LoadWord(row, step + chunk + kPitch);
                        // bytes of the two slots side by side
                        const uint32_t low2 = __byte_perm(w0, w1, 0x5410), high2 = __byte_perm(w0, w1, 0x7632);
                        f[0][2 * r] = EvenBytes(low2, magic);
                        f[0][2 * r + 1] = EvenBytes(low2 >> 8, magic);
                        f[1][2 * r] = EvenBytes(high2, magic);
                        f[1][2 * r + 1] = EvenBytes(high2 >> 8, magic);
                    } else {
                        const uint32_t w = LoadHalf(row, step + chunk) | (LoadHalf(row, step + chunk + kPitch) << 16);
                        const uint32_t u = w >> 8;
                        f[0][2 * r] = LowNibbles(w, magic);
                        f[0][2 * r + 1] = LowNibbles(u, magic);
                        f[1][2 * r] = HighNibbles(w, magic);
                        f[1][2 * r + 1] = HighNibbles(u, magic);
                    }
                }
                uint32_t hi[2], lo[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    uint32_t di = d[h][i][b];
                    if (edge) di &= __hne2_mask(AsHalf2(ph[h][i]), AsHalf2(0u));  // a slot not seen may hold NaN
                    const __half2 sc = __hmul2(AsHalf2(di), down);
                    const __half2 p = AsHalf2(ph[h][i]), y = __hmul2(p, sc);
                    hi[i] = H2(y);
                    lo[i] = H2(__hfma2(AsHalf2(pl[h][i]), sc, __hfma2(p, sc, __hneg2(y))));
                }
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    h == 0 ? MmaFirst(t[j], f[j], lo[0], lo[1]) : Mma(t[j], f[j], lo[0], lo[1]);
                    Mma(t[j], f[j], hi[0], hi[1]);
                }
            }
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) v[0].o[b][j][i] = fmaf(t[j][i], up, v[0].o[b][j][i]);
        }
    }

    // The same in fp32 slot by slot, those of weight 0 left out: exact for scales of any spread.  Some five times a
    // unit's usual time (32 sequences of 500 to 8192 slots, Q8_0: 72 us, with one slot in 500 two thousand times the
    // others 90, with every unit of this kind 217).
    __device__ __forceinline__ void Plainly(const Step& s, const uint8_t* stage) {
#pragma unroll 2
        for (int r = 0; r < kUnit; ++r) {
            const int i = (r >> 3) & 1;
            const uint32_t hi = r < kSlots ? (i ? ph[0][1] : ph[0][0]) : (i ? ph[1][1] : ph[1][0]);
            const uint32_t lo = r < kSlots ? (i ? pl[0][1] : pl[0][0]) : (i ? pl[1][1] : pl[1][0]);
            const float2 h = __half22float2(AsHalf2(hi)), l = __half22float2(AsHalf2(lo));
            const float w = r & 1 ? h.y + l.y : h.x + l.x;  // of query g
            const int src = 8 * s.c + ((r & 7) >> 1);
            const float w0 = __shfl_sync(0xffffffffu, w, src), w1 = __shfl_sync(0xffffffffu, w, src + 4);
            const uint8_t* row = stage + r * kPitch;
            const __half* scales = reinterpret_cast<const __half*>(stage + kPlane) + r * NB;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                float x[2][2];  // as Dim
                if constexpr (TYPE == MLB_Q8_0) {
                    const int chunk = 2 * b + (s.g >> 2);
                    const uint32_t q = *reinterpret_cast<const uint32_t*>(row + (kXor ? chunk ^ (r & 7) : chunk) * 16 + 4 * (s.g & 3));
#pragma unroll
                    for (int k = 0; k < 4; ++k) x[k >> 1][k & 1] = static_cast<float>(static_cast<int8_t>(q >> (8 * k)));
                } else {
                    const uint32_t q = *reinterpret_cast<const uint16_t*>(row + b * 16 + 2 * s.g);
#pragma unroll
                    for (int k = 0; k < 4; ++k) x[k >> 1][k & 1] = static_cast<float>(static_cast<int>((q >> (8 * (k & 1) + 4 * (k >> 1))) & 15) - 8);
                }
                const float d = __half2float(scales[b]);
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        if (w0 != 0.0f) v[0].o[b][j][2 * k] = fmaf(w0, d * x[j][k], v[0].o[b][j][2 * k]);
                        if (w1 != 0.0f) v[0].o[b][j][2 * k + 1] = fmaf(w1, d * x[j][k], v[0].o[b][j][2 * k + 1]);
                    }
            }
        }
    }
};

// ---------------------------------------------------------------- fp32 caches
template <int NB, int NT>
struct F32Warp {
    static constexpr int kUnit = kSlots;
    static constexpr int kChunks = NB * 8;
    static constexpr int kPitch = (kChunks | 1) * 16;
    static constexpr int kStageBytes = kUnit * kPitch;  // of K, and of V
    static constexpr int kFrags = 4 * NB;

    Values<NB> v[NT];
    Columns col[NT];
    float p[NT][4];  // weights of the unit, as the scores' C fragments
    bool edge;       // not every row sees all of the unit
    const float *kp, *vp;
    int pitch;  // floats between slots
    int hd;

    __device__ __forceinline__ static int Dim(int g, int j, int half) { return 4 * g + 2 * j + half; }

    __device__ __forceinline__ static void LayOut(const TreeArgs& a, const Step& s, const float* q, uint4* frags,
                                                  float* undos) {
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i) {  // elements 2i, 2i + 1 of the thread's eight: k = c, c + 4
                const int d = b * 32 + 8 * s.c + 2 * i;
                uint4 f;
                SplitTf32(q && d < a.c.hd ? __ldg(q + d) : 0.0f, f.x, f.z);
                SplitTf32(q && d + 1 < a.c.hd ? __ldg(q + d + 1) : 0.0f, f.y, f.w);
                frags[(4 * b + i) * 32 + s.lane] = f;
            }
        if (s.c == 0) undos[s.g] = fmaxf(a.scale * kLog2e, kLeast);
    }

    __device__ __forceinline__ void Begin(const TreeArgs& a, const TreeSplit&, int seq, int head) {
        const long long row = a.c.Row(seq, a.layer, head, 0);
        hd = a.c.hd;
        kp = static_cast<const float*>(a.c.k) + row * hd;
        vp = static_cast<const float*>(a.c.v) + row * hd;
        pitch = a.c.n_kv * hd;
#pragma unroll
        for (int n = 0; n < NT; ++n) v[n].Clear();
    }

    template <int COUNT>
    __device__ __forceinline__ void Copy(const float* plane, uint32_t stage, int p0, int id) const {
        constexpr int kAll = kUnit * kChunks;
#pragma unroll 4
        for (int j = 0; j < (kAll + COUNT - 1) / COUNT; ++j) {
            const int i = id + j * COUNT;
            if (kAll % COUNT != 0 && i >= kAll) break;
            const int r = i / kChunks, d = i % kChunks * 4, bytes = d < hd ? 16 : 0;
            CopyChunk(stage + r * kPitch + d * 4, plane + size_t(p0 + r) * pitch + (d < hd ? d : 0), bytes);
        }
    }
    template <int COUNT>
    __device__ __forceinline__ void CopyK(uint32_t stage, int p0, int id) const {
        Copy<COUNT>(kp, stage, p0, id);
    }
    template <int COUNT>
    __device__ __forceinline__ void CopyV(uint32_t stage, int p0, int id) const {
        Copy<COUNT>(vp, stage, p0, id);
    }

    __device__ __forceinline__ void Keys(const Step& s, const uint8_t* stage, const uint4* frags, int p0, int low) {
        edge = low + kUnit > s.len;
        float x[NT][1][4], rest[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) x[n][0][i] = rest[n][i] = 0.0f;
        const float* row = reinterpret_cast<const float*>(stage + s.g * kPitch) + 8 * s.c;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float4 ra = *reinterpret_cast<const float4*>(row + b * 32 + 4 * h);
                const float4 rb = *reinterpret_cast<const float4*>(row + 8 * (kPitch / 4) + b * 32 + 4 * h);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    uint32_t hi[4], lo[4];
                    SplitTf32(i ? ra.z : ra.x, hi[0], lo[0]);
                    SplitTf32(i ? rb.z : rb.x, hi[1], lo[1]);
                    SplitTf32(i ? ra.w : ra.y, hi[2], lo[2]);
                    SplitTf32(i ? rb.w : rb.y, hi[3], lo[3]);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const uint4 q = frags[(n * kFrags + 4 * b + 2 * h + i) * 32];
                        MmaTf32(rest[n], lo, q.x, q.y);
                        MmaTf32(rest[n], hi, q.z, q.w);
                        MmaTf32(x[n][0], hi, q.x, q.y);
                    }
                }
            }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            AddTo(x[n][0], rest[n]);
            col[n].Weights(s, p0, low, edge, x[n], 0.0f, [&](float r0, float r1) { v[n].Scale(r0, r1); });
#pragma unroll
            for (int i = 0; i < 4; ++i) p[n][i] = x[n][0][i];
        }
    }

    __device__ __forceinline__ void Sum(const Step& s, const uint8_t* stage) {
        const float* vrow = reinterpret_cast<const float*>(stage + 2 * s.c * kPitch) + 4 * s.g;
        if (edge) {  // a slot that some rows do not see may hold NaN or infinities
            bool odd = false;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const float4 y = *reinterpret_cast<const float4*>(vrow + ((i & 1) + (i >> 1) * 8) * (kPitch / 4) + b * 32);
                    odd = odd || !(fabsf(y.x) <= 3.4e38f && fabsf(y.y) <= 3.4e38f && fabsf(y.z) <= 3.4e38f &&
                                   fabsf(y.w) <= 3.4e38f);
                }
            if (__any_sync(0xffffffffu, odd)) {
#pragma unroll
                for (int n = 0; n < NT; ++n) Plainly(s, stage, n);
                return;
            }
        }
        // weights as B fragments: query g, slots 2c and 2c + 1 (+ 8)
        uint32_t ph[NT][4], pl[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int src = 4 * (2 * s.c + (i & 1)) + (s.g >> 1);
                const float even = __shfl_sync(0xffffffffu, p[n][i & 2], src);
                const float other = __shfl_sync(0xffffffffu, p[n][(i & 2) + 1], src);
                SplitTf32(s.g & 1 ? other : even, ph[n][i], pl[n][i]);
            }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            float4 y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                y[i] = *reinterpret_cast<const float4*>(vrow + ((i & 1) + (i >> 1) * 8) * (kPitch / 4) + b * 32);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float t[NT][4];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float4 va = y[2 * i], vb = y[2 * i + 1];
                    uint32_t hi[4], lo[4];
                    SplitTf32(j ? va.z : va.x, hi[0], lo[0]);
                    SplitTf32(j ? va.w : va.y, hi[1], lo[1]);
                    SplitTf32(j ? vb.z : vb.x, hi[2], lo[2]);
                    SplitTf32(j ? vb.w : vb.y, hi[3], lo[3]);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        i == 0 ? MmaTf32First(t[n], lo, ph[n][0], ph[n][1]) : MmaTf32(t[n], lo, ph[n][2], ph[n][3]);
                        MmaTf32(t[n], hi, pl[n][2 * i], pl[n][2 * i + 1]);
                        MmaTf32(t[n], hi, ph[n][2 * i], ph[n][2 * i + 1]);
                    }
                }
#pragma unroll
                for (int n = 0; n < NT; ++n) AddTo(v[n].o[b][j], t[n]);
            }
        }
    }

    // The weighted values of one unit slot by slot, those of weight 0 left out.
    __device__ __forceinline__ void Plainly(const Step& s, const uint8_t* stage, int n) {
        const float(&x)[4] = p[n];
        const float* row = reinterpret_cast<const float*>(stage) + 4 * s.g;
        for (int i = 0; i < kUnit; ++i) {
            const int src = 4 * (i & 7) + s.c;
            const float w0 = __shfl_sync(0xffffffffu, i < 8 ? x[0] : x[2], src);
            const float w1 = __shfl_sync(0xffffffffu, i < 8 ? x[1] : x[3], src);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const float4 y = *reinterpret_cast<const float4*>(row + i * (kPitch / 4) + b * 32);
                const float e[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    float* to = &v[n].o[b][d >> 1][(d & 1) * 2];
                    if (w0 != 0.0f) to[0] = fmaf(w0, e[d], to[0]);
                    if (w1 != 0.0f) to[1] = fmaf(w1, e[d], to[1]);
                }
            }
        }
    }
};

template <int TYPE, int NB, int NT>
struct WarpOf {
    static_assert(NT == 1, "quantized caches: a tile per warp");
    using T = QuantWarp<TYPE, NB>;
};
template <int NB, int NT>
struct WarpOf<MLB_F32, NB, NT> {
    using T = F32Warp<NB, NT>;
};

// Units of a batch entry: `unit` slots each, for all its items.
__device__ __forceinline__ unsigned EntryUnits(const TreeArgs& a, int b, unsigned unit, unsigned items) {
    return (unsigned(FindEntry(a, b).slots) + unit - 1) / unit * items;
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

// The list of all units, cut evenly over the CTAs: the first `extra` take one
// more.  A warp works it out together.
struct Cut {
    unsigned total, ctas, each, extra;

    // `groups`: units that a CTA works on at a time; `small`: an item that a CTA keeps to itself, as joining its parts
    // would take longer (131 slots of 2 x 64 in Q8_0: 7.8 us whole, 10.2 cut).
    __device__ __forceinline__ Cut(const TreeArgs& a, unsigned unit, unsigned items, unsigned groups, unsigned small,
                                   unsigned grid) {
        const int lane = threadIdx.x & 31;
        unsigned live = 0;
        total = 0;
        for (int b0 = 0; b0 < a.batch; b0 += 32) {
            const unsigned n = b0 + lane < a.batch ? EntryUnits(a, b0 + lane, unit, items) : 0;
            total += __reduce_add_sync(0xffffffffu, n);
            live += __popc(__ballot_sync(0xffffffffu, n != 0));
        }
        // a unit for each group, or an item for each CTA, at least
        const unsigned whole = min(live * items, total);
        ctas = max(1u, min(total <= small * whole ? whole : max((total + groups - 1) / groups, whole), grid));
        each = total / ctas;
        extra = total - each * ctas;
    }
    __device__ __forceinline__ unsigned Start(unsigned cta) const { return cta * each + min(cta, extra); }
    __device__ __forceinline__ unsigned Owner(unsigned at) const {
        const unsigned high = extra * (each + 1);
        return at < high ? at / (each + 1) : extra + (at - high) / each;
    }
    // The batch entry of unit `at`, and that entry's first unit.
    __device__ __forceinline__ int Find(const TreeArgs& a, unsigned unit, unsigned items, unsigned at, unsigned& first) const {
        const int lane = threadIdx.x & 31;
        first = 0;
        for (int b0 = 0; b0 < a.batch; b0 += 32) {
            const unsigned n = b0 + lane < a.batch ? EntryUnits(a, b0 + lane, unit, items) : 0;
            unsigned incl = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned t = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += t;
            }
            const unsigned past = __ballot_sync(0xffffffffu, first + incl > at);
            if (past) {
                const int to = __ffs(past) - 1;
                first += __shfl_sync(0xffffffffu, incl - n, to);
                return b0 + to;
            }
            first += __shfl_sync(0xffffffffu, incl, 31);
        }
        return a.batch;
    }
};

// Shared memory: the ring of every group (S stages of K, then S of V), which the
// joining of the groups reuses, the Q fragments and the score factors.  PER_SM
// CTAs share an SM, so that one joins or starts while another computes.
template <int TYPE, int NB, int NT, int WQ, int NW, int PER_SM>
struct TreeShape {
    using Warp = typename WarpOf<TYPE, NB, NT>::T;
    static constexpr int kGroups = NW / WQ;
    static constexpr int kRowsOf = kRows * NT;        // of a warp
    static constexpr int kItemRows = kRowsOf * WQ;
    static constexpr int kPitch = NB * 32 + 4;        // of a row in the join
    static constexpr int kFragBytes = WQ * NT * Warp::kFrags * 32 * 16;
    static constexpr int kJoinBytes = NW * kRowsOf * (kPitch + 2) * 4;
    static constexpr int kUndoBytes = WQ * kRowsOf * 4;
    static constexpr int kMaxShared = kSmShared / PER_SM - 1024;
    static constexpr int kFit = (kMaxShared - kFragBytes - kUndoBytes) / (kGroups * 2 * Warp::kStageBytes);
    static constexpr int kStages = kFit < kMaxStages ? kFit : kMaxStages;
    static constexpr int kRingBytes = kStages * 2 * Warp::kStageBytes;  // of a group
    static constexpr int kTop = (kGroups * kRingBytes > kJoinBytes ? kGroups * kRingBytes : kJoinBytes);
    static constexpr int kBytes = (kTop + 15) / 16 * 16 + kFragBytes + kUndoBytes;
    static_assert(kStages >= 2, "a ring has two stages at least");
    static_assert(kBytes <= kMaxShared, "shared memory");
    static_assert(kGroups <= 15, "a named barrier per group");
};

template <int TYPE, int NB, int NT, int WQ, int NW, int PER_SM>
__global__ void __launch_bounds__(NW * 32, PER_SM) TreeMmaKernel(TreeArgs a, TreeSplit sp) {
    using Shape = TreeShape<TYPE, NB, NT, WQ, NW, PER_SM>;
    using Warp = typename Shape::Warp;
    constexpr int kPitch = Shape::kPitch, kFours = NB * 8, kItemRows = Shape::kItemRows, kStages = Shape::kStages;
    constexpr int kUnit = Warp::kUnit, kStageBytes = Warp::kStageBytes;
    constexpr unsigned kGroups = Shape::kGroups;
    extern __shared__ __align__(128) uint4 smem4[];
    uint8_t* ring = reinterpret_cast<uint8_t*>(smem4);
    float* so = reinterpret_cast<float*>(smem4);                 // join: [NW][8 NT][kPitch]
    float* sm = so + NW * Shape::kRowsOf * kPitch;               // [NW][8 NT]
    float* sl = sm + NW * Shape::kRowsOf;
    uint4* sq = reinterpret_cast<uint4*>(ring + (Shape::kTop + 15) / 16 * 16);  // [WQ NT][kFrags][32]
    float* su = reinterpret_cast<float*>(sq + Shape::kFragBytes / 16);          // [WQ NT][8]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int wq = warp % WQ, group = warp / WQ;
    const unsigned items = a.c.n_kv * sp.groups;

    // entries with nothing to see
    for (int b = blockIdx.x; b < a.batch; b += gridDim.x) {
        if (FindEntry(a, b).slots != 0) continue;
        for (int t = warp; t < a.tokens; t += NW)
            for (int i = lane; i < a.n_heads * a.c.hd; i += 32)
                a.out[(size_t(b) * a.tokens + t) * a.out_stride + i] = 0.0f;
    }

    GridDepLaunch();  // the joining kernel may come up as CTAs leave
    const Cut cut(a, kUnit, items, kGroups, 2 * kGroups, gridDim.x);
    if (cut.total == 0 || blockIdx.x >= cut.ctas) return;
    unsigned cur = cut.Start(blockIdx.x);
    const unsigned end = cut.Start(blockIdx.x + 1);
    unsigned first;
    int b = cut.Find(a, kUnit, items, cur, first);

    Step s;
    s.lane = lane;
    s.g = lane >> 2;
    s.c = lane & 3;
    s.tokens = a.tokens;
    s.words = a.words;
    const int last_unit = a.c.head_slots - kUnit;
    constexpr int kRing = kStages * kStageBytes;  // of K, then of V
    const uint8_t* ring_ptr = ring + group * Shape::kRingBytes;
    const uint32_t ring_at = SmemAddr(ring_ptr);
    Warp w;
    while (cur < end) {
        const Entry e = FindEntry(a, b);
        const unsigned units = (e.slots + kUnit - 1) / kUnit;
        if (cur - first >= units * items) {  // the next entry
            first += units * items;
            ++b;
            continue;
        }
        const unsigned item = (cur - first) / units;
        const int u0 = cur - first - item * units;
        const int u1 = min(u0 + (end - cur), units);
        const int head = item / sp.groups, row0 = (item - head * sp.groups) * kItemRows;
        const int tile = row0 + wq * Shape::kRowsOf;  // the warp's first row
        s.slots = e.slots;
        s.len = e.len;
        s.mask = a.mask ? a.mask + size_t(b) * a.tokens * a.words : nullptr;

        // ---- the ring's first units, then the Q fragments
        w.Begin(a, sp, e.seq, head);
        // K runs half a unit ahead of V: its stage is free again once the scores are done
        int k_from = u0 + group, v_from = k_from;  // the units to copy next
        int k_into = 0, v_into = 0;                // their stages
        const int id = wq * 32 + lane;
        // the last unit of a plane may hold fewer slots: it starts earlier and leaves the others out
        auto copy_k = [&] {
            if (k_from < u1) w.template CopyK<WQ * 32>(ring_at + k_into, min(k_from * kUnit, last_unit), id);
            asm volatile("cp.async.commit_group;" ::: "memory");
            k_from += kGroups;
            k_into = k_into + kStageBytes == kRing ? 0 : k_into + kStageBytes;
        };
        auto copy_v = [&] {
            if (v_from < u1) w.template CopyV<WQ * 32>(ring_at + kRing + v_into, min(v_from * kUnit, last_unit), id);
            asm volatile("cp.async.commit_group;" ::: "memory");
            v_from += kGroups;
            v_into = v_into + kStageBytes == kRing ? 0 : v_into + kStageBytes;
        };
#pragma unroll
        for (int k = 0; k < kStages - 1; ++k) {
            copy_k();
            copy_v();
        }
        copy_k();
        for (int n = warp; n < WQ * NT; n += NW) {
            const int r = row0 + n * kRows + s.g;
            const float* q = r < sp.rows ? a.q + (size_t(b) * a.tokens + r / a.group) * a.q_stride +
                                               size_t(head * a.group + r % a.group) * a.c.hd
                                         : nullptr;
            Warp::LayOut(a, s, q, sq + n * Warp::kFrags * 32, su + n * kRows);
        }
        __syncthreads();
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int r = tile + n * kRows + 2 * s.c;
            const float* undo = su + (wq * NT + n) * kRows + 2 * s.c;
            w.col[n].Begin(r / a.group, (r + 1) / a.group);
            w.col[n].cs[0] = undo[0];
            w.col[n].cs[1] = undo[1];
        }

        // ---- the group's units
        const uint4* frags = sq + wq * NT * Warp::kFrags * 32 + lane;
        // all copies but the 2 (S - 1) latest have landed, and every warp of the group is here
        auto meet = [&] {
            asm volatile("cp.async.wait_group %0;" ::"n"(2 * (kStages - 1)) : "memory");
            if (WQ == 1)
                __syncwarp();
            else
                asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(WQ * 32) : "memory");
        };
        int stage = 0;
        for (int u = u0 + group; u < u1; u += kGroups) {
            meet();  // this unit's K is there, the last unit's V has been read
            copy_v();
            if (tile < sp.rows) w.Keys(s, ring_ptr + stage, frags, min(u * kUnit, last_unit), u * kUnit);
            meet();  // its V is there, its K has been read
            copy_k();
            if (tile < sp.rows) w.Sum(s, ring_ptr + kRing + stage);
            stage = stage + kStageBytes == kRing ? 0 : stage + kStageBytes;
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();  // the ring is free for the join
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            Columns& col = w.col[n];
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) {
                col.l[0] += __shfl_xor_sync(0xffffffffu, col.l[0], o);
                col.l[1] += __shfl_xor_sync(0xffffffffu, col.l[1], o);
            }
            const int at = warp * Shape::kRowsOf + n * kRows + 2 * s.c;
            float* to = so + at * kPitch;
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int d = i * 32 + w.Dim(s.g, j, h);
                        to[d] = w.v[n].o[i][j][2 * h];
                        to[kPitch + d] = w.v[n].o[i][j][2 * h + 1];
                    }
            if (s.g == 0) {
                sm[at] = Scaled(col.m[0], col.cs[0], col.l[0]);
                sm[at + 1] = Scaled(col.m[1], col.cs[1], col.l[1]);
                sl[at] = col.l[0];
                sl[at + 1] = col.l[1];
            }
        }
        __syncthreads();

        // ---- join the groups
        const bool whole = u0 == 0 && u1 == int(units);
        constexpr size_t kPart = size_t(kItemRows) * (NB * 32 + 2);
        float* part = sp.parts + (2 * size_t(blockIdx.x) + (u0 == 0 ? 1 : 0)) * kPart;
        const int live_rows = min(kItemRows, sp.rows - row0);
        for (int i = threadIdx.x; i < live_rows * kFours; i += NW * 32) {
            const int r = i / kFours, d = (i - r * kFours) * 4;
            Joined x;
#pragma unroll 4
            for (unsigned j = 0; j < kGroups; ++j) {
                const int at = j * kItemRows + r;  // warp j WQ + its wq
                x.Add(sm[at], sl[at], *reinterpret_cast<const float4*>(so + at * kPitch + d));
            }
            if (whole) {
                StoreOut(a, OutRow(a, b, head, row0 + r), d, x.Result());
            } else {
                __stcg(reinterpret_cast<float4*>(part + r * NB * 32 + d), x.o);
                if (d == 0) {
                    __stcg(part + kItemRows * NB * 32 + r, x.m);
                    __stcg(part + kItemRows * (NB * 32 + 1) + r, x.l);
                }
            }
        }

        __syncthreads();
        cur += u1 - u0;
    }
}

// Items that are cut between CTAs: `share` warps to a row add up its parts, in
// the order of the CTAs, and one of them joins their sums.  blockIdx.x: item,
// blockIdx.y: rows, kJoinWarps / share of them at a time.
constexpr int kJoinWarps = 8;
constexpr int kJoinBatch = 4;  // parts in flight

template <int NB, bool SHARED>
__global__ void __launch_bounds__(kJoinWarps * 32) TreeJoinKernel(TreeArgs a, TreeSplit sp, int unit, int groups, int small,
                                                                  int item_rows, int grid, int shared) {
    const int share = SHARED ? shared : 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned items = a.c.n_kv * sp.groups;
    const int b = blockIdx.x / items;
    const unsigned item = blockIdx.x - b * items;
    const Cut cut(a, unit, items, groups, small, grid);
    const unsigned units = EntryUnits(a, b, unit, 1);
    unsigned first = 0;  // of the entry
    for (int b0 = 0; b0 < b; b0 += 32)
        first += __reduce_add_sync(0xffffffffu, b0 + lane < b ? EntryUnits(a, b0 + lane, unit, items) : 0);
    // CTAs with nothing to join wait too: the next kernel may be a dependent of this one, whose wait covers the main
    // kernel only if this one has not ended before it.
    GridDepWait();
    if (units == 0) return;
    const unsigned u0 = first + item * units;
    const unsigned c0 = cut.Owner(u0), c1 = cut.Owner(u0 + units - 1);
    if (c0 == c1) return;
    const int head = item / sp.groups, row0 = (item - head * sp.groups) * item_rows;
    const int rows = min(item_rows, sp.rows - row0), at_once = kJoinWarps / share;
    const size_t part = size_t(item_rows) * (NB * 32 + 2);
    const unsigned each = (c1 - c0 + share) / share;  // parts of a warp
    const unsigned begin = c0 + warp % share * each, end = min(begin + each, c1 + 1);
    constexpr int kFours = NB * 8;
    for (int base = blockIdx.y * at_once; base < rows; base += gridDim.y * at_once) {
#pragma unroll
        for (int d0 = 0; d0 < kFours; d0 += 32) {
            const int r = base + warp / share, d = min(d0 + lane, kFours - 1) * 4;
            Joined x;
            if (r < rows)
                for (unsigned k = begin; k < end; k += kJoinBatch) {
                    float pm[kJoinBatch], pl[kJoinBatch];
                    float4 po[kJoinBatch];
#pragma unroll
                    for (int j = 0; j < kJoinBatch; ++j) {
                        // a CTA has two parts: of the item that it goes on with, and of one that it begins
                        const unsigned cta = min(k + j, end - 1);
                        const float* p = sp.parts + (2 * size_t(cta) + (cut.Start(cta) <= u0 ? 1 : 0)) * part;
                        pm[j] = __ldcg(p + item_rows * NB * 32 + r);
                        pl[j] = __ldcg(p + item_rows * (NB * 32 + 1) + r);
                        po[j] = __ldcg(reinterpret_cast<const float4*>(p + r * NB * 32 + d));
                    }
#pragma unroll
                    for (int j = 0; j < kJoinBatch; ++j)
                        if (k + j < end) x.Add(pm[j], pl[j], po[j]);
                }
            if constexpr (SHARED) {
                __shared__ float sm[kJoinWarps], sl[kJoinWarps];
                __shared__ float4 so[kJoinWarps][32];
                if (lane == 0) {
                    sm[warp] = x.m;
                    sl[warp] = x.l;
                }
                so[warp][lane] = x.o;
                __syncthreads();
                if (warp % share == 0)
                    for (int j = 1; j < share; ++j) x.Add(sm[warp + j], sl[warp + j], so[warp + j][lane]);
                __syncthreads();
            }
            if (r < rows && warp % share == 0 && d0 + lane < kFours) StoreOut(a, OutRow(a, b, head, row0 + r), d, x.Result());
        }
    }
}

// Comes up while the main kernel's last CTAs run.  Warps share a row where an item
// is cut into more parts than one has in flight.
template <int NB>
void LaunchJoin(DeviceContext& ctx, const TreeArgs& a, const TreeSplit& sp, int unit, int groups, int small, int item_rows,
                int grid) {
    const int all = a.batch * a.c.n_kv * sp.groups;
    int share = 1;
    while (share < kJoinWarps && 1LL * share * kJoinBatch * all < grid) share *= 2;
    // as many rows at once as do not make many more CTAs than the device holds
    const int rows = std::min(item_rows, sp.rows);
    const int per_item = std::max(1, std::min<int>(CeilDiv(rows * share, kJoinWarps), 16 * ctx.sm_count / all));
    Launch("TreeJoinKernel", share > 1 ? TreeJoinKernel<NB, true> : TreeJoinKernel<NB, false>, dim3(all, per_item),
           dim3(kJoinWarps * 32), 0, ctx.stream, true, a, sp, unit, groups, small, item_rows, grid, share);
}

template <int TYPE, int NB, int NT, int WQ, int NW, int PER_SM>
bool LaunchShape(DeviceContext& ctx, const TreeArgs& a) {
    using Shape = TreeShape<TYPE, NB, NT, WQ, NW, PER_SM>;
    TreeSplit sp{};
    sp.rows = a.tokens * a.group;
    sp.groups = static_cast<int>(CeilDiv(sp.rows, Shape::kItemRows));
    const unsigned long long items = 1ull * a.c.n_kv * sp.groups;
    // an upper bound of the units, from the caller's bound of the lengths
    const long long slots = std::min<long long>(1LL * std::min(a.max_len, a.c.max_seq) + a.tokens, a.c.max_seq);
    const double units = double(a.batch) * double(items) * double(CeilDiv(slots, Shape::Warp::kUnit));
    if (units >= 2147483648.0 || a.c.head_slots < Shape::Warp::kUnit) return false;
    const int grid = static_cast<int>(std::min<double>(
        PER_SM * ctx.sm_count, std::max(std::ceil(units / Shape::kGroups), double(a.batch) * double(items))));
    sp.parts = static_cast<float*>(
        Workspace(ctx, 2 * size_t(grid) * Shape::kItemRows * (NB * 32 + 2) * sizeof(float)));
    sp.magic = TYPE == MLB_Q8_0 ? kMagic8 : kMagic4;
    auto* kernel = TreeMmaKernel<TYPE, NB, NT, WQ, NW, PER_SM>;
    static int configured[64] = {};
    if (ctx.device >= 64 || !configured[ctx.device]) {
        CheckCuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::kBytes),
                  "cudaFuncSetAttribute(TreeMmaKernel)");
        if (ctx.device < 64) configured[ctx.device] = 1;
    }
    kernel<<<grid, NW * 32, Shape::kBytes, ctx.stream>>>(a, sp);
    CheckCuda(cudaGetLastError(), "TreeMmaKernel");
    if (grid == 1) return true;  // nothing is cut
    LaunchJoin<NB>(ctx, a, sp, Shape::Warp::kUnit, Shape::kGroups, 2 * Shape::kGroups, Shape::kItemRows, grid);
    return true;
}

// Rows per KV head choose the tiles.  Up to 8: a tile, every warp its own slots;
// more: two warps share slots, a tile each, a group of 16 rows after the other (the
// second reads the cache from L2).  8 sequences of 4000 slots, 8 x 128 in Q8_0: 16
// rows 36.9 us (groups of 8: 39.2), 32 rows 61.3 (63.0); in Q4_0 34.8 (36.9), 57.3 (59.4).
// Three CTAs of four warps begin and end their items independently: 32 sequences
// of 500 to 8192 slots, four rows, took 73 us, with two CTAs of six warps 84.
// fp32 caches are bound by the tf32 products: above 32 rows two tiles to a warp
// halve the splits of K and V (49 rows, 2 x 64, 8 sequences of 2000 to 16384 slots:
// 65 us, one tile 77; 32 rows of 8000 slots: 24.4 against 20.6).  Heads of more
// than 64 elements leave no room for that: four warps a group above 16 rows (32 rows,
// 8 x 4000 slots of 8 x 128: 117 us, two warps 133), two above 8 (16 rows: 76 us, one 103).
// Heads of more than 128: one CTA per SM, as many groups as shared memory holds
// (4 rows, 4000 slots of 8 x 256: Q8_0 19.5 us, Q4_0 18.4, fp32 36.9).
template <int TYPE, int NB>
bool LaunchRows(DeviceContext& ctx, const TreeArgs& a) {
    const long long rows = 1LL * a.tokens * a.group;
    if constexpr (NB > 4) {
        constexpr int NW = TYPE == MLB_F32 ? 3 : 6;
        if (rows <= kRows) return LaunchShape<TYPE, NB, 1, 1, NW, 1>(ctx, a);
        return LaunchShape<TYPE, NB, 1, 2, TYPE == MLB_F32 ? 4 : 8, 1>(ctx, a);
    } else if constexpr (TYPE == MLB_F32 && NB > 2) {
        if (rows <= kRows) return LaunchShape<TYPE, NB, 1, 1, 3, 2>(ctx, a);
        if (rows <= 2 * kRows) return LaunchShape<TYPE, NB, 1, 2, 4, 2>(ctx, a);
        return LaunchShape<TYPE, NB, 1, 4, 4, 2>(ctx, a);
    } else {
        if (rows <= kRows) return LaunchShape<TYPE, NB, 1, 1, 4, 3>(ctx, a);
        if constexpr (TYPE == MLB_F32)
            if (rows > 4 * kRows) return LaunchShape<TYPE, NB, 2, 2, 4, 3>(ctx, a);
        return LaunchShape<TYPE, NB, 1, 2, 4, 3>(ctx, a);
    }
}

template <int TYPE>
bool LaunchBlocks(DeviceContext& ctx, const TreeArgs& a) {
    switch (a.c.blocks) {
        case 1: return LaunchRows<TYPE, 1>(ctx, a);
        case 2: return LaunchRows<TYPE, 2>(ctx, a);
        case 3: return LaunchRows<TYPE, 3>(ctx, a);
        case 4: return LaunchRows<TYPE, 4>(ctx, a);
        case 5: return LaunchRows<TYPE, 5>(ctx, a);
        case 6: return LaunchRows<TYPE, 6>(ctx, a);
        case 7: return LaunchRows<TYPE, 7>(ctx, a);
        case 8: return LaunchRows<TYPE, 8>(ctx, a);
        default: return false;
    }
}

}  // namespace
}  // namespace mlb
