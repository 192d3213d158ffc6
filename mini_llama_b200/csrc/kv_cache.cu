// Rotary positions of rows and the caller-owned KV cache: table fill, row
// rotation, quantizing writes (with the rotation fused where asked for) and
// reads.  C-ABI: mlb_rope_table_fill, mlb_rope_rows, mlb_kv_cache_*.
//
// Everything here is bound by memory: a call reads its rows once and writes
// them once.  A rotation unit is four pairs (two 16-byte loads, two of the
// table, two stores); a cache unit is four elements of a 32-element block, so
// the eight lanes of a block share its maximum by shuffles and store its quants
// as 32 contiguous bytes (Q4_0: 16).  Measured, each call by itself: 4096 rows of 64 x 128
// rotated 47 us (5.7 TB/s); 4096 rows of K and V of 8 x 128 written to Q4_0 / Q8_0 / fp32
// 16.4 / 15.0 / 14.4 us (2.3 / 2.8 / 4.7 TB/s) and read 12.3 / 12.3 / 14.3 (3.1 / 3.5 / 4.7),
// with 32 query heads rotated and written 43 / 43 / 39 (4.1 / 4.2 / 5.2); 32768 rows
// written 96 / 94 / 83 (3.2 / 3.6 / 6.4) and read 68 / 68 / 84 (4.5 / 5.0 / 6.4); decode
// steps of a few rows 4.5 to 6.5 us, a launch.  So fp32 rows run at the copy rate,
// and the quantizing write at half of it.  Each kernel has a form for shapes,
// strides or addresses that do not allow 16-byte accesses.  All arithmetic uses
// explicitly rounded operations: rotations equal mlb_rope's and blocks mlb_quantize's
// bit for bit, except that a scale is amax times fl(1/127) or fl(1/7) where
// mlb_quantize divides, which differs in the last bit of about one Q4_0 scale in 40 000.
#include <algorithm>
#include <cmath>
#include <type_traits>
#include <vector>

#include "kv_cache.cuh"

namespace mlb {

namespace {

constexpr int kThreads = 256;
constexpr int kBlockLanes = 8;  // lanes per 32-element block, four elements each
constexpr int kGroups = kThreads / kBlockLanes;
// Blocks per group of lanes: one while that fills the device with fewer than
// kManyCtas CTAs (latency), else kUnits with their loads in flight together (a read
// of 32768 rows of 8 x 128 in Q8_0: 90 us with one, 68 with two, 74 with four).
constexpr int kUnits = 2;
constexpr unsigned kManyCtas = 148 * 8 * kUnits;

struct RopeView {
    const float2* cs;
    int n_positions, rot, neox;
};

// Rows of q or k to rotate.
struct RotRows {
    const float* in;
    float* out;
    size_t in_stride, out_stride;
    int heads;
    int copy;  // the part past rot_dim has to be copied
};

__device__ __forceinline__ float2 Rotate(float a, float b, float2 cs) {
    return make_float2(__fsub_rn(__fmul_rn(a, cs.x), __fmul_rn(b, cs.y)),
                       __fadd_rn(__fmul_rn(a, cs.y), __fmul_rn(b, cs.x)));
}

__host__ __device__ __forceinline__ int RotUnits(int hd, int rot, bool vec) {
    return vec ? hd / 8 : rot / 2 + (hd - rot);
}

// Unit u of one head: four pairs (VEC) or one, or as many elements past the
// rotated part.  `cs` is the position's table row, null for a position outside.
template <bool VEC>
__device__ __forceinline__ void RotateUnit(const RotRows& t, const RopeView& r, int hd, size_t row, int head, int u,
                                           const float2* cs) {
    const float* in = t.in + row * t.in_stride + size_t(head) * hd;
    float* out = t.out + row * t.out_stride + size_t(head) * hd;
    const int half = r.rot / 2;
    if (VEC) {
        const bool turn = u < r.rot / 8;
        if (!turn && !t.copy && cs) return;
        const int a = turn ? (r.neox ? 4 * u : 8 * u) : 8 * u;
        const int b = turn && r.neox ? a + half : a + 4;
        float4 x = *reinterpret_cast<const float4*>(in + a);
        float4 y = *reinterpret_cast<const float4*>(in + b);
        if (!cs) {
            x = y = make_float4(NAN, NAN, NAN, NAN);
        } else if (turn) {
            const float4 c0 = __ldg(reinterpret_cast<const float4*>(cs + 4 * u));
            const float4 c1 = __ldg(reinterpret_cast<const float4*>(cs + 4 * u + 2));
            const float2 p0 = make_float2(c0.x, c0.y), p1 = make_float2(c0.z, c0.w);
            const float2 p2 = make_float2(c1.x, c1.y), p3 = make_float2(c1.z, c1.w);
            if (r.neox) {
                const float2 r0 = Rotate(x.x, y.x, p0), r1 = Rotate(x.y, y.y, p1);
                const float2 r2 = Rotate(x.z, y.z, p2), r3 = Rotate(x.w, y.w, p3);
                x = make_float4(r0.x, r1.x, r2.x, r3.x);
                y = make_float4(r0.y, r1.y, r2.y, r3.y);
            } else {
                const float2 r0 = Rotate(x.x, x.y, p0), r1 = Rotate(x.z, x.w, p1);
                const float2 r2 = Rotate(y.x, y.y, p2), r3 = Rotate(y.z, y.w, p3);
                x = make_float4(r0.x, r0.y, r1.x, r1.y);
                y = make_float4(r2.x, r2.y, r3.x, r3.y);
            }
        }
        *reinterpret_cast<float4*>(out + a) = x;
        *reinterpret_cast<float4*>(out + b) = y;
    } else if (u < half) {
        const int a = r.neox ? u : 2 * u, b = r.neox ? u + half : 2 * u + 1;
        const float2 y = cs ? Rotate(in[a], in[b], __ldg(cs + u)) : make_float2(NAN, NAN);
        out[a] = y.x;
        out[b] = y.y;
    } else {
        const int e = r.rot + (u - half);
        if (t.copy || !cs) out[e] = cs ? in[e] : NAN;
    }
}

__device__ __forceinline__ const float2* TableRow(const RopeView& r, int pos) {
    return pos >= 0 && pos < r.n_positions ? r.cs + size_t(pos) * (r.rot / 2) : nullptr;
}

// Unit i of rows x (q heads, then k heads) x units.
template <bool VEC>
__device__ __forceinline__ void RotateIndex(unsigned i, unsigned total, const RotRows& q, const RotRows& k,
                                            const RopeView& r, int hd, const int* positions) {
    if (i >= total) return;
    const unsigned units = RotUnits(hd, r.rot, VEC), per_row = (q.heads + k.heads) * units;
    const unsigned row = i / per_row, in_row = i - row * per_row;
    const int head = in_row / units, u = in_row - head * units;
    const float2* cs = TableRow(r, __ldg(positions + row));
    if (head < q.heads)
        RotateUnit<VEC>(q, r, hd, row, head, u, cs);
    else
        RotateUnit<VEC>(k, r, hd, row, head - q.heads, u, cs);
}

template <bool VEC>
__global__ void __launch_bounds__(kThreads) RopeRowsKernel(RotRows q, RotRows k, RopeView r, int hd, unsigned total,
                                                           const int* positions) {
    RotateIndex<VEC>(blockIdx.x * kThreads + threadIdx.x, total, q, k, r, hd, positions);
}

// ---------------------------------------------------------------- cache rows
// Elements e0 .. e0 + 3 of a head (zeros past head_dim), rotated when cs is set.
template <bool VEC, bool ROPE>
__device__ __forceinline__ void LoadFour(const float* in, int e0, int hd, const RopeView& r, const float2* cs,
                                         float (&x)[4]) {
    if (VEC) {
        const float4 a = e0 < hd ? __ldg(reinterpret_cast<const float4*>(in + e0)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = e0 + j < hd ? __ldg(in + e0 + j) : 0.0f;
    }
    if (!ROPE || !cs) return;
    const int half = r.rot / 2;
    if (VEC && e0 < r.rot) {
        if (r.neox) {
            const bool second = e0 >= half;
            const int i = second ? e0 - half : e0;
            const float4 o = __ldg(reinterpret_cast<const float4*>(in + (second ? i : e0 + half)));
            const float4 c0 = __ldg(reinterpret_cast<const float4*>(cs + i));
            const float4 c1 = __ldg(reinterpret_cast<const float4*>(cs + i + 2));
            const float other[4] = {o.x, o.y, o.z, o.w};
            const float2 p[4] = {make_float2(c0.x, c0.y), make_float2(c0.z, c0.w), make_float2(c1.x, c1.y),
                                 make_float2(c1.z, c1.w)};
#pragma unroll
            for (int j = 0; j < 4; ++j)
                x[j] = second ? Rotate(other[j], x[j], p[j]).y : Rotate(x[j], other[j], p[j]).x;
        } else {
            const float4 c = __ldg(reinterpret_cast<const float4*>(cs + e0 / 2));
            const float2 r0 = Rotate(x[0], x[1], make_float2(c.x, c.y));
            const float2 r1 = Rotate(x[2], x[3], make_float2(c.z, c.w));
            x[0] = r0.x; x[1] = r0.y; x[2] = r1.x; x[3] = r1.y;
        }
    } else if (!VEC) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int e = e0 + j;
            if (e >= r.rot) continue;
            const bool second = r.neox ? e >= half : (e & 1);
            const int i = r.neox ? (second ? e - half : e) : e / 2;
            const int p = r.neox ? (second ? i : e + half) : e ^ 1;
            const float o = __ldg(in + p);
            const float2 c = __ldg(cs + i);
            x[j] = second ? Rotate(o, x[j], c).y : Rotate(x[j], o, c).x;
        }
    }
}

__device__ __forceinline__ int Clamp(int v, int lo, int hi) { return v < lo ? lo : (v > hi ? hi : v); }

// Stores four elements of block `blk` of one cache row, lane l of the block's
// eight; `live` lanes only store, every lane of the warp takes part.
template <int TYPE>
__device__ __forceinline__ void StoreFour(void* plane, __half* scales, long long row, int blocks, int blk, int l, int hd,
                                          bool live, bool vec, const float (&x)[4]) {
    if (TYPE == MLB_F32) {
        if (!live) return;
        float* o = static_cast<float*>(plane) + row * hd + blk * 32 + 4 * l;
        const int left = hd - (blk * 32 + 4 * l);
        if (vec && left >= 4) {
            *reinterpret_cast<float4*>(o) = make_float4(x[0], x[1], x[2], x[3]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j < left) o[j] = x[j];
        }
        return;
    }
    float mx = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
#pragma unroll
    for (int o = 1; o < kBlockLanes; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    const uint16_t d = mx > 0.0f ? F32ToF16Ref(__fmul_rn(mx, TYPE == MLB_Q8_0 ? 1.0f / 127.0f : 1.0f / 7.0f)) : 0;
    const float stored = HalfBits(d);
    const float inv = stored == 0.0f ? 0.0f : __fdiv_rn(1.0f, stored);
    uint32_t word = 0;
    if (TYPE == MLB_Q8_0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int n = Clamp(static_cast<int>(roundf(__fmul_rn(x[j], inv))), -127, 127);
            word |= static_cast<uint32_t>(n & 0xff) << (8 * j);
        }
        if (live) static_cast<uint32_t*>(plane)[(row * blocks + blk) * 8 + l] = word;
    } else {
        // the quantizer's all-zero block: scale 0 and nibbles 0
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int n = Clamp(static_cast<int>(roundf(__fadd_rn(__fmul_rn(x[j], inv), 8.0f))), 0, 15);
            word |= static_cast<uint32_t>(mx > 0.0f ? n : 0) << (8 * j);
        }
        const uint32_t high = __shfl_down_sync(0xffffffffu, word, 4);  // elements 16 .. 31
        if (live && l < 4) static_cast<uint32_t*>(plane)[(row * blocks + blk) * 4 + l] = word | (high << 4);
    }
    if (live && l == 0) scales[row * blocks + blk] = __ushort_as_half(d);
}

struct CacheRows {
    const int* seqs;
    const int* slots;
    int rows;
    size_t k_stride, v_stride;
};

// The block that a group of eight lanes works on.
struct BlockAt {
    unsigned row;
    int head, blk;
    long long at;  // cache row; -1: outside
};

__device__ __forceinline__ BlockAt FindBlock(const KvView& c, const CacheRows& w, unsigned g, int layer) {
    BlockAt b{0, 0, 0, -1};
    const unsigned per_row = c.n_kv * c.blocks;
    b.row = g / per_row;
    const unsigned rest = g - b.row * per_row;
    b.head = rest / c.blocks;
    b.blk = rest - b.head * c.blocks;
    const int seq = w.seqs ? __ldg(w.seqs + b.row) : 0, slot = __ldg(w.slots + b.row);
    if (seq >= 0 && seq < c.n_seqs && slot >= 0 && slot < c.max_seq) b.at = c.Row(seq, layer, b.head, slot);
    return b;
}

// Blocks of 32 elements of K and V: CTA (x, layer), UNITS of them for each group
// of eight lanes, their loads together; with ROPE the CTAs past kv_ctas rotate q.
template <int TYPE, bool VEC, bool ROPE, int UNITS>
__global__ void __launch_bounds__(kThreads) KvWriteRowsKernel(KvView c, CacheRows w, int layer0, const float* k,
                                                              const float* v, unsigned total, unsigned kv_ctas, RopeView r,
                                                              const int* positions, RotRows q, unsigned q_total) {
    if (ROPE && blockIdx.x >= kv_ctas) {
        const RotRows none{};
        RotateIndex<VEC>((blockIdx.x - kv_ctas) * kThreads + threadIdx.x, q_total, q, none, r, c.hd, positions);
        return;
    }
    const int l = threadIdx.x % kBlockLanes, layer = layer0 + blockIdx.y;
    // Every step for all units before the next, without branches, so that their
    // loads are in flight together; a unit past the end repeats the last block.
    BlockAt b[UNITS];
    bool live[UNITS];
    float xk[UNITS][4], xv[UNITS][4];
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
        const unsigned g = (blockIdx.x * UNITS + u) * kGroups + threadIdx.x / kBlockLanes;
        b[u] = FindBlock(c, w, min(g, total - 1), layer);
        live[u] = g < total && b[u].at >= 0;
    }
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
        const float2* cs = nullptr;
        if (ROPE) {
            const int pos = __ldg(positions + b[u].row);
            live[u] = live[u] && TableRow(r, pos);
            cs = r.cs + size_t(Clamp(pos, 0, r.n_positions - 1)) * (r.rot / 2);
        }
        const size_t src = size_t(blockIdx.y) * w.rows + b[u].row, head = size_t(b[u].head) * c.hd;
        LoadFour<VEC, ROPE>(k + src * w.k_stride + head, b[u].blk * 32 + 4 * l, c.hd, r, cs, xk[u]);
        LoadFour<VEC, false>(v + src * w.v_stride + head, b[u].blk * 32 + 4 * l, c.hd, r, nullptr, xv[u]);
    }
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
        StoreFour<TYPE>(c.k, c.ks, b[u].at, c.blocks, b[u].blk, l, c.hd, live[u], VEC, xk[u]);
        StoreFour<TYPE>(c.v, c.vs, b[u].at, c.blocks, b[u].blk, l, c.hd, live[u], VEC, xv[u]);
    }
}

template <int TYPE>
__device__ __forceinline__ void LoadCached(const void* plane, const __half* scales, long long at, int blocks, int blk, int l,
                                           int hd, bool vec, float (&x)[4]) {
    if (TYPE == MLB_F32) {
        const float* in = static_cast<const float*>(plane) + at * hd;
        const int e0 = blk * 32 + 4 * l;
        if (vec) {
            if (e0 < hd) {
                const float4 a = *reinterpret_cast<const float4*>(in + e0);
                x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (e0 + j < hd) x[j] = in[e0 + j];
        }
        return;
    }
    const float d = __half2float(scales[at * blocks + blk]);
    if (TYPE == MLB_Q8_0) {
        const uint32_t w = static_cast<const uint32_t*>(plane)[(at * blocks + blk) * 8 + l];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = __fmul_rn(d, static_cast<float>(static_cast<int8_t>(w >> (8 * j))));
    } else {
        const uint32_t w = static_cast<const uint32_t*>(plane)[(at * blocks + blk) * 4 + (l & 3)] >> (l & 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = __fmul_rn(d, static_cast<float>(static_cast<int>((w >> (8 * j)) & 15) - 8));
    }
}

template <bool VEC>
__device__ __forceinline__ void StoreRow(float* out, int e0, int hd, const float (&x)[4]) {
    if (VEC) {
        if (e0 < hd) *reinterpret_cast<float4*>(out + e0) = make_float4(x[0], x[1], x[2], x[3]);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (e0 + j < hd) out[e0 + j] = x[j];
    }
}

template <int TYPE, bool VEC, int UNITS>
__global__ void __launch_bounds__(kThreads) KvReadRowsKernel(KvView c, CacheRows w, int layer0, float* k, float* v,
                                                             unsigned total) {
    const int l = threadIdx.x % kBlockLanes;
    BlockAt b[UNITS];
    float xk[UNITS][4], xv[UNITS][4];
#pragma unroll
    for (int u = 0; u < UNITS; ++u)
        b[u] = FindBlock(c, w, min((blockIdx.x * UNITS + u) * kGroups + threadIdx.x / kBlockLanes, total - 1),
                         layer0 + blockIdx.y);
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
        const long long at = b[u].at >= 0 ? b[u].at : 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) xk[u][j] = xv[u][j] = 0.0f;
        if (k) LoadCached<TYPE>(c.k, c.ks, at, c.blocks, b[u].blk, l, c.hd, VEC, xk[u]);
        if (v) LoadCached<TYPE>(c.v, c.vs, at, c.blocks, b[u].blk, l, c.hd, VEC, xv[u]);
    }
#pragma unroll
    for (int u = 0; u < UNITS; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            xk[u][j] = b[u].at >= 0 ? xk[u][j] : 0.0f;
            xv[u][j] = b[u].at >= 0 ? xv[u][j] : 0.0f;
        }
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
        if ((blockIdx.x * UNITS + u) * kGroups + threadIdx.x / kBlockLanes >= total) break;
        const size_t dst = size_t(blockIdx.y) * w.rows + b[u].row, head = size_t(b[u].head) * c.hd;
        if (k) StoreRow<VEC>(k + dst * w.k_stride + head, b[u].blk * 32 + 4 * l, c.hd, xk[u]);
        if (v) StoreRow<VEC>(v + dst * w.v_stride + head, b[u].blk * 32 + 4 * l, c.hd, xv[u]);
    }
}

// ---------------------------------------------------------------- host checks
bool Aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

RopeView CheckedRope(const char* c, const mlb_rope_table* t) {
    Require(t != nullptr, c, "rope table is null");
    Require(t->n_positions > 0 && t->head_dim > 0, c, "rope table shape must be positive");
    Require(t->rot_dim >= 2 && t->rot_dim % 2 == 0 && t->rot_dim <= t->head_dim, c,
            "rot_dim must be even and within head_dim");
    Require(t->rope_type == MLB_ROPE_NORMAL || t->rope_type == MLB_ROPE_NEOX, c, "unknown rope type");
    Require(t->cos_sin != nullptr, c, "rope table is empty");
    Require(Aligned16(t->cos_sin), c, "rope table is not 16-byte aligned");
    return {reinterpret_cast<const float2*>(t->cos_sin), t->n_positions, t->rot_dim, t->rope_type == MLB_ROPE_NEOX};
}

// Whether pairs of four fit the table rows and the head.
bool RopeVec(const RopeView& r, int hd) { return r.rot % 8 == 0 && hd % 8 == 0; }

bool RowsVec(const void* p, size_t stride) { return Aligned16(p) && stride % 4 == 0; }

unsigned Checked32(const char* c, unsigned long long n) {
    Require(n < (1ull << 31), c, "too many elements for one call", MLB_ERR_UNSUPPORTED);
    return static_cast<unsigned>(n);
}

// Rows to rotate (heads 0: absent).
RotRows CheckedRot(const char* c, const char* name, const float* in, size_t in_stride, float* out, size_t out_stride,
                   int heads, int hd, int rot) {
    if (heads == 0) return {};
    Require(in && out, c, std::string(name) + " is null");
    const size_t n = size_t(heads) * hd;
    Require(in_stride >= n && out_stride >= n, c, std::string(name) + " stride is shorter than a row");
    Require(in != out || in_stride == out_stride, c, std::string(name) + " in place needs equal strides");
    RequireAligned(c, name, in, 4);
    RequireAligned(c, name, out, 4, " output");
    return {in, out, in_stride, out_stride, heads, in != out && rot < hd};
}

bool RotVec(const RotRows& t) { return t.heads == 0 || (RowsVec(t.in, t.in_stride) && RowsVec(t.out, t.out_stride)); }

// f(std::integral_constant<int, type>) for the cache's type.
template <typename F>
void ByType(int type, F&& f) {
    if (type == MLB_F32)
        f(std::integral_constant<int, MLB_F32>{});
    else if (type == MLB_Q8_0)
        f(std::integral_constant<int, MLB_Q8_0>{});
    else
        f(std::integral_constant<int, MLB_Q4_0>{});
}

template <bool ROPE>
void LaunchKvWrite(const char* caller, DeviceContext& ctx, const KvView& c, const CacheRows& w, int layer0, int layers,
                   const float* k, const float* v, const RopeView& r, const int* positions, const RotRows& q) {
    bool vec = c.hd % 4 == 0 && RowsVec(k, w.k_stride) && RowsVec(v, w.v_stride) && Aligned16(c.k) && Aligned16(c.v);
    if (ROPE) vec = vec && RopeVec(r, c.hd) && RotVec(q);
    const unsigned total = Checked32(caller, 1ull * w.rows * c.n_kv * c.blocks);
    const unsigned q_total = Checked32(caller, 1ull * w.rows * q.heads * RotUnits(c.hd, ROPE ? r.rot : 0, vec));
    const bool many = vec && CeilDiv(total, kGroups) * layers >= kManyCtas;
    const unsigned kv_ctas = CeilDiv(total, kGroups * (many ? kUnits : 1));
    const dim3 grid(kv_ctas + CeilDiv(q_total, kThreads), layers);
    auto go = [&](auto kernel) {
        kernel<<<grid, kThreads, 0, ctx.stream>>>(c, w, layer0, k, v, total, kv_ctas, r, positions, q, q_total);
        CheckCuda(cudaGetLastError(), "KvWriteRowsKernel");
    };
    auto type = [&](auto t) {
        constexpr int T = decltype(t)::value;
        if (many)
            go(KvWriteRowsKernel<T, true, ROPE, kUnits>);
        else
            vec ? go(KvWriteRowsKernel<T, true, ROPE, 1>) : go(KvWriteRowsKernel<T, false, ROPE, 1>);
    };
    ByType(c.type, type);
}

void CheckKvRows(const char* c, const KvView& v, int rows, const int* seqs, const int* slots, const void* k, size_t k_stride,
                 const void* vv, size_t v_stride) {
    Require(rows >= 0, c, "row count is negative");
    if (rows == 0) return;
    Require(slots != nullptr, c, "slots is null");
    const size_t n = size_t(v.n_kv) * v.hd;
    Require((!k || k_stride >= n) && (!vv || v_stride >= n), c, "row stride is shorter than a row");
    RequireAligned(c, "seqs", seqs, 4);
    RequireAligned(c, "slots", slots, 4);
    RequireAligned(c, "k", k, 4);
    RequireAligned(c, "v", vv, 4);
}

// The pair frequencies of a table, scaled, in fp32.
std::vector<float> Frequencies(const char* c, int rot, float theta, const mlb_rope_scale* s, float* magnitude) {
    *magnitude = 1.0f;
    const int kind = s ? s->scaling : MLB_ROPE_SCALE_NONE;
    Require(kind >= MLB_ROPE_SCALE_NONE && kind <= MLB_ROPE_SCALE_WAVELENGTH, c, "unknown rope scaling");
    const double factor = kind == MLB_ROPE_SCALE_NONE ? 1.0 : s->factor;
    Require(std::isfinite(factor) && factor >= 1.0, c, "scaling factor must be at least 1");
    const bool by_turns = kind == MLB_ROPE_SCALE_YARN || kind == MLB_ROPE_SCALE_WAVELENGTH;
    double fast = 0.0, slow = 0.0;
    if (by_turns) {
        Require(s->original_positions > 0, c, "original_positions must be positive");
        const bool preset = s->fast == 0.0f && s->slow == 0.0f;
        fast = preset ? (kind == MLB_ROPE_SCALE_YARN ? 32.0 : 4.0) : s->fast;
        slow = preset ? 1.0 : s->slow;
        Require(std::isfinite(fast) && slow > 0.0 && fast > slow, c, "turn counts must satisfy 0 < slow < fast");
    }
    if (kind == MLB_ROPE_SCALE_NTK && rot > 2)
        theta = static_cast<float>(theta * std::pow(factor, double(rot) / (rot - 2)));
    const int half = rot / 2;
    std::vector<float> f(half);
    for (int i = 0; i < half; ++i)
        f[i] = 1.0f / std::pow(theta, static_cast<float>(2 * i) / static_cast<float>(rot));
    constexpr double kTurn = 6.283185307179586476925;
    double low = 0.0, high = 0.0;
    if (kind == MLB_ROPE_SCALE_YARN) {
        Require(theta > 1.0f, c, "YaRN needs theta above 1");
        // pair index at which a frequency turns n times within the original positions
        auto index = [&](double n) {
            return rot * std::log(s->original_positions / (n * kTurn)) / (2.0 * std::log(double(theta)));
        };
        low = std::max(0.0, std::floor(index(fast)));
        high = std::min(rot - 1.0, std::ceil(index(slow)));
        if (high <= low) high = low + 0.001;
        Require(s->attention_factor >= 0.0f && std::isfinite(s->attention_factor), c, "attention factor must be >= 0");
        *magnitude = s->attention_factor > 0.0f ? s->attention_factor : static_cast<float>(0.1 * std::log(factor) + 1.0);
    }
    for (int i = 0; i < half; ++i) {
        const double g = f[i];
        double kept = 1.0;  // share of the unscaled frequency
        if (kind == MLB_ROPE_SCALE_LINEAR) kept = 0.0;
        if (kind == MLB_ROPE_SCALE_YARN) kept = 1.0 - std::min(1.0, std::max(0.0, (i - low) / (high - low)));
        if (kind == MLB_ROPE_SCALE_WAVELENGTH) {
            const double turns = s->original_positions * g / kTurn;
            kept = std::min(1.0, std::max(0.0, (turns - slow) / (fast - slow)));
        }
        if (kept < 1.0) f[i] = static_cast<float>(g * kept + g / factor * (1.0 - kept));
    }
    return f;
}

}  // namespace

KvView CheckedKvView(const char* c, const mlb_kv_cache* cache, bool pointers) {
    Require(cache != nullptr, c, "cache is null");
    Require(cache->type == MLB_F32 || cache->type == MLB_Q8_0 || cache->type == MLB_Q4_0, c,
            "cache type must be F32, Q8_0 or Q4_0", MLB_ERR_UNSUPPORTED);
    Require(cache->n_seqs > 0 && cache->n_layers > 0 && cache->max_seq_len > 0 && cache->n_kv_heads > 0 &&
                cache->head_dim > 0,
            c, "cache shape must be positive");
    Require(cache->head_dim <= 4096 && cache->n_kv_heads <= 4096 && cache->max_seq_len <= (1 << 28), c,
            "cache shape is too large", MLB_ERR_UNSUPPORTED);
    KvView v{};
    v.type = cache->type;
    v.n_seqs = cache->n_seqs;
    v.n_layers = cache->n_layers;
    v.max_seq = cache->max_seq_len;
    v.n_kv = cache->n_kv_heads;
    v.hd = cache->head_dim;
    v.blocks = (v.hd + 31) / 32;
    const bool f32 = v.type == MLB_F32;
    const int slots = f32 ? v.max_seq : (v.max_seq + 7) / 8 * 8;
    v.head_rows = f32 ? 1 : slots;
    v.head_slots = slots;
    v.slot_rows = f32 ? v.n_kv : 1;
    v.layer_rows = 1LL * v.n_kv * slots;
    v.seq_rows = v.layer_rows * v.n_layers;
    Require(1.0 * v.seq_rows * v.n_seqs * v.blocks * 128.0 < 9.0e18, c, "cache shape is too large", MLB_ERR_UNSUPPORTED);
    if (!pointers) return v;
    Require(cache->k && cache->v, c, "cache is empty");
    if (!f32) {
        Require(cache->k_scale && cache->v_scale, c, "cache scales are null");
        Require(Aligned16(cache->k) && Aligned16(cache->v) && Aligned16(cache->k_scale) && Aligned16(cache->v_scale), c,
                "cache planes are not 16-byte aligned");
    } else {
        Require(((reinterpret_cast<uintptr_t>(cache->k) | reinterpret_cast<uintptr_t>(cache->v)) & 3) == 0, c,
                "cache planes are not 4-byte aligned");
    }
    v.k = cache->k;
    v.v = cache->v;
    v.ks = static_cast<__half*>(cache->k_scale);
    v.vs = static_cast<__half*>(cache->v_scale);
    return v;
}

void CheckKvLayer(const char* c, const KvView& v, int layer, bool all_ok) {
    if (all_ok && layer == MLB_ALL_LAYERS) {
        Require(v.n_layers <= 65535, c, "too many layers for one call", MLB_ERR_UNSUPPORTED);
        return;
    }
    Require(layer >= 0 && layer < v.n_layers, c, "layer out of range", MLB_ERR_OUT_OF_RANGE);
}

}  // namespace mlb

using namespace mlb;

extern "C" {

int mlb_rope_table_fill(int device, const mlb_rope_table* table, float theta, const mlb_rope_scale* scale) {
    return Guard([&] {
        const char* c = "mlb_rope_table_fill";
        CheckedRope(c, table);
        Require(std::isfinite(theta) && theta > 0.0f, c, "theta must be positive");
        float magnitude = 1.0f;
        const std::vector<float> f = Frequencies(c, table->rot_dim, theta, scale, &magnitude);
        const int half = table->rot_dim / 2;
        std::vector<float> cs(size_t(table->n_positions) * half * 2);
        for (int p = 0; p < table->n_positions; ++p) {
            float* row = cs.data() + size_t(p) * half * 2;
            for (int i = 0; i < half; ++i) {
                const float angle = static_cast<float>(p) * f[i];
                row[2 * i] = std::cos(angle) * magnitude;
                row[2 * i + 1] = std::sin(angle) * magnitude;
            }
        }
        DeviceContext& ctx = Ctx(device);
        CheckCuda(cudaMemcpyAsync(table->cos_sin, cs.data(), cs.size() * sizeof(float), cudaMemcpyHostToDevice, ctx.stream),
                  "cudaMemcpyAsync(rope table)");
        CheckCuda(cudaStreamSynchronize(ctx.stream), "cudaStreamSynchronize(rope table)");
    });
}

int mlb_rope_rows(int device, const mlb_rope_table* table, int rows, const int* positions, const float* q, size_t q_stride,
                  float* q_out, size_t q_out_stride, int n_heads, const float* k, size_t k_stride, float* k_out,
                  size_t k_out_stride, int n_kv_heads) {
    return Guard([&] {
        const char* c = "mlb_rope_rows";
        const RopeView r = CheckedRope(c, table);
        const int hd = table->head_dim;
        Require(rows >= 0, c, "row count is negative");
        Require(n_heads >= 0 && n_kv_heads >= 0, c, "head count is negative");
        if (rows == 0 || (n_heads == 0 && n_kv_heads == 0)) return;
        Require(positions != nullptr, c, "positions is null");
        RequireAligned(c, "positions", positions, 4);
        const RotRows tq = CheckedRot(c, "q", q, q_stride, q_out, q_out_stride, n_heads, hd, r.rot);
        const RotRows tk = CheckedRot(c, "k", k, k_stride, k_out, k_out_stride, n_kv_heads, hd, r.rot);
        const bool vec = RopeVec(r, hd) && RotVec(tq) && RotVec(tk);
        const unsigned total =
            Checked32(c, 1ull * rows * (1ull * n_heads + n_kv_heads) * RotUnits(hd, r.rot, vec));
        DeviceContext& ctx = Ctx(device);
        const unsigned grid = CeilDiv(total, kThreads);
        if (vec)
            RopeRowsKernel<true><<<grid, kThreads, 0, ctx.stream>>>(tq, tk, r, hd, total, positions);
        else
            RopeRowsKernel<false><<<grid, kThreads, 0, ctx.stream>>>(tq, tk, r, hd, total, positions);
        CheckCuda(cudaGetLastError(), "RopeRowsKernel");
    });
}

int mlb_kv_cache_bytes(const mlb_kv_cache* cache, size_t* plane_bytes, size_t* scale_bytes) {
    return Guard([&] {
        const char* c = "mlb_kv_cache_bytes";
        const KvView v = CheckedKvView(c, cache, false);
        const size_t rows = size_t(v.seq_rows) * v.n_seqs;
        if (plane_bytes)
            *plane_bytes = v.type == MLB_F32 ? rows * v.hd * 4 : rows * v.blocks * (v.type == MLB_Q8_0 ? 32 : 16);
        if (scale_bytes) *scale_bytes = v.type == MLB_F32 ? 0 : rows * v.blocks * 2;
    });
}

int mlb_kv_cache_write(int device, const mlb_kv_cache* cache, int layer, int rows, const int* seqs, const int* slots,
                       const float* k, size_t k_stride, const float* v, size_t v_stride) {
    return Guard([&] {
        const char* c = "mlb_kv_cache_write";
        const KvView view = CheckedKvView(c, cache, true);
        CheckKvLayer(c, view, layer, true);
        CheckKvRows(c, view, rows, seqs, slots, k, k_stride, v, v_stride);
        if (rows == 0) return;
        Require(k && v, c, "k or v is null");
        const bool all = layer == MLB_ALL_LAYERS;
        LaunchKvWrite<false>(c, Ctx(device), view, {seqs, slots, rows, k_stride, v_stride}, all ? 0 : layer,
                             all ? view.n_layers : 1, k, v, {}, nullptr, {});
    });
}

int mlb_kv_cache_write_rope(int device, const mlb_kv_cache* cache, int layer, int rows, const int* seqs, const int* slots,
                            const mlb_rope_table* table, const int* positions, const float* q, size_t q_stride,
                            float* q_out, size_t q_out_stride, int n_heads, const float* k, size_t k_stride,
                            const float* v, size_t v_stride) {
    return Guard([&] {
        const char* c = "mlb_kv_cache_write_rope";
        const KvView view = CheckedKvView(c, cache, true);
        CheckKvLayer(c, view, layer, false);
        const RopeView r = CheckedRope(c, table);
        Require(table->head_dim == view.hd, c, "rope table and cache have different head_dim");
        CheckKvRows(c, view, rows, seqs, slots, k, k_stride, v, v_stride);
        Require(n_heads >= 0, c, "head count is negative");
        if (rows == 0) return;
        Require(k && v, c, "k or v is null");
        Require(positions != nullptr, c, "positions is null");
        RequireAligned(c, "positions", positions, 4);
        const RotRows tq = CheckedRot(c, "q", q, q_stride, q_out, q_out_stride, n_heads, view.hd, r.rot);
        LaunchKvWrite<true>(c, Ctx(device), view, {seqs, slots, rows, k_stride, v_stride}, layer, 1, k, v, r, positions,
                            tq);
    });
}

int mlb_kv_cache_read(int device, const mlb_kv_cache* cache, int layer, int rows, const int* seqs, const int* slots,
                      float* k, size_t k_stride, float* v, size_t v_stride) {
    return Guard([&] {
        const char* c = "mlb_kv_cache_read";
        const KvView view = CheckedKvView(c, cache, true);
        CheckKvLayer(c, view, layer, true);
        CheckKvRows(c, view, rows, seqs, slots, k, k_stride, v, v_stride);
        if (rows == 0) return;
        Require(k || v, c, "k and v are null");
        const bool all = layer == MLB_ALL_LAYERS;
        const bool vec = view.hd % 4 == 0 && (!k || RowsVec(k, k_stride)) && (!v || RowsVec(v, v_stride)) &&
                         Aligned16(view.k) && Aligned16(view.v);
        const unsigned total = Checked32(c, 1ull * rows * view.n_kv * view.blocks);
        const unsigned layers = all ? view.n_layers : 1;
        const bool many = vec && CeilDiv(total, kGroups) * layers >= kManyCtas;
        const dim3 grid(CeilDiv(total, kGroups * (many ? kUnits : 1)), layers);
        DeviceContext& ctx = Ctx(device);
        const CacheRows w{seqs, slots, rows, k_stride, v_stride};
        auto go = [&](auto kernel) {
            kernel<<<grid, kThreads, 0, ctx.stream>>>(view, w, all ? 0 : layer, k, v, total);
            CheckCuda(cudaGetLastError(), "KvReadRowsKernel");
        };
        ByType(view.type, [&](auto t) {
            constexpr int T = decltype(t)::value;
            if (many)
                go(KvReadRowsKernel<T, true, kUnits>);
            else
                vec ? go(KvReadRowsKernel<T, true, 1>) : go(KvReadRowsKernel<T, false, 1>);
        });
    });
}

}  // extern "C"
