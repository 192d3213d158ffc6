// Attention of many drafted rows over a quantized cache on the 5th-generation
// tensor cores (tcgen05): more than 32 rows per KV head, where the matrix work
// of the warp-level kernel (tree_mma.cuh) outgrows the cache's bytes.
//
// An item is 128 query rows (tokens x query heads of one KV head, zeros past
// their end) against a stretch of the cache, 128 slots to a tile:
//   S = Q K^T     128 x 128, three MMA products: K = d q is exact as fp16 hi + lo
//                 (19 bits: hi = rn(d q), lo = fma(d, q, -hi); fp16(d) is a
//                 multiple of 2^-24, so subnormal scales too), Q is scaled per row
//                 by a power of two and split into hi + lo (22 bits), the lo lo
//                 product is dropped (2^-22)
//   softmax       a row's running maximum m, moved when a score passes it by 2^2;
//                 weights 2^(x - m + 12) <= 2^14 as fp16 hi + lo, written over the
//                 scores: 16 columns become 8 of hi and 8 of lo
//   O = P V       128 x head_dim, A from tensor memory, V = hi + lo as K, stored as it
//                 lies in the cache (the N side contiguous); a fresh accumulator per
//                 tile, added to the running rows in registers in fp32 (the matrix
//                 unit's own sums truncate)
// Where |d q| could pass fp16's range (a scale of 2^8 or more) quants are taken times
// 2^-9, undone in fp32: a K slot by itself (its other blocks then resolve to 2^-16);
// a V tile with such scales is multiplied twice, first its other blocks as they are,
// then these.  So no slot's values depend on another's.  Slots that only some rows see
// may hold any bytes: K touches its own column only; a V scale that is not finite in a
// drafted slot becomes 0 and the rows that see it NaN in that block.
//
// Measured: 61-token trees of 16 sequences of 1024 to 4096 slots, 32 / 8 x 128 in Q4_0
// 187 us, 673 TFLOP/s of fp16 products (41 % of the measured matrix rate); where one
// slot in 500 has a large V scale 208.  A tile takes some 7950 cycles, the softmax warps' time: 2460 of them the weights, 1700 the
// maximum and the scores' wait, 1150 the item's start and end; the MMAs alone 3100.
//
// Bound: the MMAs, 6 x 128 x 128 x head_dim multiply-adds a tile (64 cycles for
// 128 x 128 x 16), and the shared memory that they, the images' stores and the
// other loads share.  One CTA per SM, roles by warp:
//   0-7    softmax and accumulation: row = lane of tensor memory, two threads to a
//          row (64 slots, half of head_dim each); scores are read twice, for the
//          maximum and for the weights, so that a thread holds 16 at a time.  Q goes
//          into tensor memory once per item: as an A operand there it leaves half of
//          shared memory's bandwidth to the producers
//   8-15   producers: quants in registers an image ahead,
//          converted into the operand images (no swizzle: 16-byte chunks of eight
//          elements, chunk c of row r at 2064 c + 16 r)
//   16     tensor memory (17-19 idle); issues all MMAs: QK(i + 1) before PV(i), so that
//          the tensor pipe works while the weights of tile i + 1 and the images of
//          the next tiles are made
// Tensor memory: two buffers of scores and weights, Q, one O.  Shared memory: two
// images of K, one of V.  The cut of the items over the CTAs and the joining of cut
// items are those of tree_mma.cuh.  Every wait is bounded; an expired one sets the
// device status word, every role leaves, and issued MMAs are waited for before
// tensor memory is freed.
#include "tree_mma.cuh"

namespace mlb {

namespace {

constexpr int kTile = 128;       // slots of a tile and rows of an item
constexpr int kSoftWarps = 8;    // softmax warps
constexpr int kProdWarps = 8;    // producer warps
constexpr int kMmaWarp = kSoftWarps + kProdWarps;
constexpr int kTcWarps = kMmaWarp + 4;  // a whole warpgroup, for the register split
// Registers of a softmax, a producer and an MMA thread: five warpgroups launched
// with 96 each, 2 x 136 + 2 x 80 + 48 of their 5 x 96.  (A launch with fewer would leave
// setmaxnreg waiting for good: the launcher checks the compiled number.)
constexpr int kSoftRegs = 136, kProdRegs = 80, kMmaRegs = 48, kLaunchRegs = 96;
static_assert(2 * kSoftRegs + 2 * kProdRegs + kMmaRegs <= 5 * kLaunchRegs, "setmaxnreg draws on the launch's registers");
constexpr int kProducers = kProdWarps * 32;
constexpr int kQCol = 2 * kTile, kOCol = 3 * kTile;  // tensor-memory columns of Q and of O
constexpr int kChunkPitch = 16 * kTile + 16;  // bytes between the chunks of eight elements in an image
constexpr uint64_t kTcWait = 2000000000ull;
constexpr int kInfoBufs = 4;     // images of K, and of V, whose flags are kept

struct TcTreeShared {
    uint64_t q_full, v_full, v_empty, o_full, o_empty, drain;
    uint64_t soft, prod;  // meetings of the softmax and of the producer threads
    uint64_t s_full[2], p_full[2], k_full[2], k_empty[2];
    uint32_t tmem;
    int abort;
    float top[2][2][kTile];  // [parity][half][row]: the largest scores of a tile
    float sum[2][kTile];     // the largest |q|
    float last[2][kTile];    // sums of the weights
    uint32_t flag[2][kProdWarps];
    int k_big[kInfoBufs], v_info[kInfoBufs];  // kOdd, kMore
    uint32_t k_bits[kInfoBufs][kTile / 32];      // slots of K taken times 2^-9, where k_big
    uint32_t v_bad[kInfoBufs][4][kTile / 32];  // [image][block][slots]: scales that are not finite, drafted slots
};
// Of an image of V: v_bad holds something; a second one of the same tile follows, of its large scales times 2^-9.
constexpr int kOdd = 1, kMore = 2;
constexpr int kTcHeaderBytes = 7168;
static_assert(sizeof(TcTreeShared) <= kTcHeaderBytes, "header");

__device__ __forceinline__ void Fail(TcTreeShared& sh, int* status) {
    atomicCAS(status, 0, MLB_ERR_DEVICE_TIMEOUT);
    *reinterpret_cast<volatile int*>(&sh.abort) = 1;
}

// Waits for a phase; false (status set, abort raised) when it gave up.  One
// thread's wait, and a whole warp's, which gives all its lanes the same answer.
__device__ __forceinline__ bool WaitOne(TcTreeShared& sh, uint64_t* bar, uint32_t parity, int* status) {
    const volatile int* abort = &sh.abort;
    if (MbarWaitFor(bar, parity, kTcWait, abort)) return true;
    if (!*abort) Fail(sh, status);
    return false;
}
__device__ __forceinline__ bool Wait(TcTreeShared& sh, uint64_t* bar, uint32_t parity, int* status) {
    return __all_sync(0xffffffffu, WaitOne(sh, bar, parity, status));
}

__device__ __forceinline__ void Arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(SmemAddr(bar)) : "memory");
}
__device__ __forceinline__ void Commit(uint32_t one, uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %1, 0;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(SmemAddr(bar)),
        "r"(one)
        : "memory");
}
__device__ __forceinline__ void FenceBefore() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void FenceAfter() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void FenceAsync() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// A meeting of a role's warps: bounded, as every wait, so that nobody is left
// behind when one of them gives up.
__device__ __forceinline__ bool Meet(TcTreeShared& sh, uint64_t* bar, uint32_t& phase, int* status) {
    Arrive(bar);
    return Wait(sh, bar, phase++ & 1, status);
}

// Shared-memory descriptor, no swizzle: lead = bytes between the two 8-element
// chunks of K (K-major) or between groups of 8 K (MN-major), stride = bytes
// between groups of 8 rows (K-major) or of 8 N (MN-major).
__device__ __forceinline__ uint64_t Descriptor(uint32_t addr, uint32_t lead, uint32_t stride) {
    return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | (static_cast<uint64_t>((lead >> 4) & 0x3FFFu) << 16) |
           (static_cast<uint64_t>((stride >> 4) & 0x3FFFu) << 32) | (1ull << 46);
}
// kind::f16, fp16 operands, fp32 accumulators, M = 128; bit 16: B is MN-major.
__device__ __forceinline__ uint32_t Instruction(int n, bool b_mn) {
    return (1u << 4) | (b_mn ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) | (8u << 24);
}

// One lane of the (converged) warp.
__device__ __forceinline__ uint32_t ElectOne() {
    uint32_t e;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(e));
    return e;
}
// A from tensor memory, B from shared memory; the whole warp comes here with the
// same operands, so that they stay in uniform registers, and `one` lane issues.
template <bool ACCUMULATE>
__device__ __forceinline__ void MmaTensor(uint32_t one, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 e, %0, 0;\n\tsetp.ne.b32 p, %5, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%1], [%2], %3, %4, {%6, %6, %6, %6}, p;\n\t}\n" ::"r"(one),
        "r"(d), "r"(a), "l"(b), "r"(idesc), "n"(ACCUMULATE ? 1 : 0), "r"(0));
}

// 16 columns of the warp's 32 lanes.
__device__ __forceinline__ void Load16(uint32_t at, float* v) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
        "[%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(at));
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void Load8(uint32_t at, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(at));
}
__device__ __forceinline__ void Store8(uint32_t at, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(at), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]));
}
__device__ __forceinline__ void WaitLoad() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void WaitStore() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Exponents of the weights of a pair of scores, (x - m) cs + offset: two adds and two FMAs as one of each.
__device__ __forceinline__ void Exponents(float& x, float& y, uint64_t minus_m, uint64_t cs, uint64_t offset) {
    asm("{\n\t.reg .b64 t;\n\tmov.b64 t, {%0, %1};\n\tadd.rn.f32x2 t, t, %2;\n\tfma.rn.f32x2 t, t, %3, %4;\n\t"
        "mov.b64 {%0, %1}, t;\n\t}\n"
        : "+f"(x), "+f"(y)
        : "l"(minus_m), "l"(cs), "l"(offset));
}
__device__ __forceinline__ uint64_t Pair(float x, float y) {
    return static_cast<uint64_t>(__float_as_uint(x)) | (static_cast<uint64_t>(__float_as_uint(y)) << 32);
}

// The items of a CTA, one after the other; every role walks them alike.
struct Walk {
    unsigned cur, end, first;
    int b;
    // of the current item
    Entry e;
    unsigned units;
    int u0, u1, head, row0;

    __device__ __forceinline__ bool Next(const TreeArgs& a, const TreeSplit& sp, unsigned items) {
        while (cur < end) {
            e = FindEntry(a, b);
            units = (e.slots + kTile - 1) / kTile;
            if (cur - first >= units * items) {
                first += units * items;
                ++b;
                continue;
            }
            const unsigned item = (cur - first) / units;
            u0 = cur - first - item * units;
            u1 = min(u0 + (end - cur), units);
            head = item / sp.groups;
            row0 = (item - head * sp.groups) * kTile;
            cur += u1 - u0;
            return true;
        }
        return false;
    }
};

// Which of the 32 slots from s0 row t sees, of `slots` slots, `len` of them committed.
__device__ __forceinline__ uint32_t SeenBits(const uint64_t* mask, int words, int tokens, int t, int s0, int len, int slots) {
    const int n = min(max(len - s0, 0), 32);           // committed ones
    uint32_t seen = n == 32 ? 0xffffffffu : (1u << n) - 1;
    const int live = min(max(slots - s0, 0), 32);      // drafted or committed
    if (n < live && t < tokens) {
        const int j0 = s0 + n - len;  // the first drafted token here
        uint64_t bits;
        if (mask) {
            const uint64_t* row = mask + size_t(t) * words + (j0 >> 6);
            bits = __ldg(row) >> (j0 & 63);
            if ((j0 & 63) != 0 && (j0 >> 6) + 1 < words) bits |= __ldg(row + 1) << (64 - (j0 & 63));
        } else {
            bits = t >= j0 ? (t - j0 >= 63 ? ~0ull : (2ull << (t - j0)) - 1) : 0;
        }
        const uint32_t in = live == 32 ? 0xffffffffu : (1u << live) - 1;
        seen |= (static_cast<uint32_t>(bits) << n) & in;
    }
    return seen;
}

// hi and lo of d times a half pair, into two words.
__device__ __forceinline__ void Product(uint32_t pair, __half2 d, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __hmul2(AsHalf2(pair), d);
    hi = H2(h);
    lo = H2(__hfma2(AsHalf2(pair), d, __hneg2(h)));
}

// A producer's share of a tile of K or V: 16-byte pieces of quants.  Eight
// neighbouring threads take kSide pieces of 8 / kSide rows, so that loads are
// whole sectors and the images' stores hit eight different groups of banks.
template <int TYPE, int NB>
struct Share {
    static constexpr int kPieces = NB * (TYPE == MLB_Q8_0 ? 2 : 1);  // of a row
    static constexpr int kMost = TYPE == MLB_Q8_0 ? 4 : 2;
    static constexpr int kSide = kPieces % kMost == 0 ? kMost : (kPieces % 2 == 0 ? 2 : 1);
    static constexpr int kTasks = (kPieces * kTile + kProducers - 1) / kProducers;
    uint4 q[kTasks];
    unsigned short d[kTasks];

    __device__ __forceinline__ static int Row(int j, int id) { return (j * kProducers + id) / kSide % kTile; }
    __device__ __forceinline__ static int Piece(int j, int id) {
        return (j * kProducers + id) / (kSide * kTile) * kSide + id % kSide;
    }
    __device__ __forceinline__ static bool Has(int j, int id) {
        return kPieces * kTile % kProducers == 0 || j * kProducers + id < kPieces * kTile;
    }
    __device__ __forceinline__ static int Block(int piece) { return TYPE == MLB_Q8_0 ? piece >> 1 : piece; }

    // Rows of the tile at p0; those from `slots` on count as zeros.
    __device__ __forceinline__ void Load(const uint8_t* plane, const __half* scales, int p0, int slots, int last, int id) {
#pragma unroll
        for (int j = 0; j < kTasks; ++j) {
            d[j] = 0;
            if (!Has(j, id)) continue;
            const int at = p0 + Row(j, id), row = min(at, last), piece = Piece(j, id);
            q[j] = __ldg(reinterpret_cast<const uint4*>(plane + size_t(row) * (kPieces * 16)) + piece);
            d[j] = __ldg(reinterpret_cast<const unsigned short*>(scales + size_t(row) * NB + Block(piece)));
            if (at >= slots) d[j] = 0;
        }
    }
    __device__ __forceinline__ static bool IsLarge(unsigned short d) { return (d & 0x7fffu) >= 0x5C00u; }  // 2^8, infinity, NaN
    __device__ __forceinline__ bool Big() const {
        bool big = false;
#pragma unroll
        for (int j = 0; j < kTasks; ++j) big = big || IsLarge(d[j]);
        return big;
    }
    // Takes out the scales that are not finite of rows from `from` on; whether there was one.
    __device__ __forceinline__ bool TakeOdd(int from, int id) {
        bool odd = false;
#pragma unroll
        for (int j = 0; j < kTasks; ++j)
            if ((d[j] & 0x7C00u) == 0x7C00u && Row(j, id) >= from) {
                odd = true;
                d[j] = 0;
            }
        return odd;
    }
    // Piece q with the scale d into an image, within each group of four elements in the order 0, 2, 1, 3.
    // BIG: the quants times `factor` (the scale itself could lose bits).
    template <bool BIG>
    __device__ __forceinline__ static void Convert(uint8_t* image, int row, int piece, const uint4& q, unsigned short d,
                                                   uint32_t magic, uint32_t factor) {
        constexpr int kLo = NB * 4 * kChunkPitch;  // of the lo image
        const __half2 s = __half2half2(__ushort_as_half(d));
        uint8_t* to = image + piece * ((TYPE == MLB_Q8_0 ? 2 : 4) * kChunkPitch) + row * 16;
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int c = 0; c < (TYPE == MLB_Q8_0 ? 2 : 4); ++c) {  // eight elements each
            const uint32_t w0 = w[2 * (c & 1)], w1 = w[2 * (c & 1) + 1];
            uint32_t p[4];
            if constexpr (TYPE == MLB_Q8_0) {
                p[0] = EvenBytes(w0, magic);
                p[1] = EvenBytes(w0 >> 8, magic);
                p[2] = EvenBytes(w1, magic);
                p[3] = EvenBytes(w1 >> 8, magic);
            } else {
                p[0] = c < 2 ? LowNibbles(w0, magic) : HighNibbles(w0, magic);
                p[1] = c < 2 ? LowNibbles(w0 >> 8, magic) : HighNibbles(w0 >> 8, magic);
                p[2] = c < 2 ? LowNibbles(w1, magic) : HighNibbles(w1, magic);
                p[3] = c < 2 ? LowNibbles(w1 >> 8, magic) : HighNibbles(w1 >> 8, magic);
            }
            if constexpr (BIG)
#pragma unroll
                for (int i = 0; i < 4; ++i) p[i] = H2(__hmul2(AsHalf2(p[i]), AsHalf2(factor)));
            uint4 hi, lo;
            Product(p[0], s, hi.x, lo.x);
            Product(p[1], s, hi.y, lo.y);
            Product(p[2], s, hi.z, lo.z);
            Product(p[3], s, hi.w, lo.w);
            *reinterpret_cast<uint4*>(to + c * kChunkPitch) = hi;
            *reinterpret_cast<uint4*>(to + c * kChunkPitch + kLo) = lo;
            asm volatile("" ::: "memory");  // one chunk's registers at a time
        }
    }
    __device__ __forceinline__ void Convert(uint8_t* image, int id, uint32_t magic) const {
#pragma unroll
        for (int j = 0; j < kTasks; ++j)
            if (Has(j, id)) Convert<false>(image, Row(j, id), Piece(j, id), q[j], d[j], magic, 0);
    }
    // A tile with large scales, read again (rare, and so without registers of its own): quants times `large` in the rows
    // whose bit is set in `down` (null: in the blocks with a large scale), times `other` in the rest.  Scales that are
    // not finite count as 0 from row `odd_from` on.
    __device__ __forceinline__ static void ConvertLarge(uint8_t* image, const uint8_t* plane, const __half* scales, int p0,
                                                        int slots, int last, int odd_from, int id, uint32_t magic,
                                                        const uint32_t* down, uint32_t large, uint32_t other) {
#pragma unroll 1
        for (int j = 0; j < kTasks; ++j) {
            if (!Has(j, id)) break;
            const int at = Row(j, id), row = min(p0 + at, last), piece = Piece(j, id);
            const uint4 x = __ldg(reinterpret_cast<const uint4*>(plane + size_t(row) * (kPieces * 16)) + piece);
            unsigned short y = __ldg(reinterpret_cast<const unsigned short*>(scales + size_t(row) * NB + Block(piece)));
            if (p0 + at >= slots || ((y & 0x7C00u) == 0x7C00u && at >= odd_from)) y = 0;
            const bool take = down ? (down[at >> 5] >> (at & 31)) & 1 : IsLarge(y);
            Convert<true>(image, at, piece, x, y, magic, take ? large : other);
        }
    }
};

template <int TYPE, int NB>
__global__ void __launch_bounds__(kTcWarps * 32, 1) TreeTcKernel(TreeArgs a, TreeSplit sp, int* status) {
    constexpr int HD = NB * 32, kImage = NB * 4 * kChunkPitch;  // one fp16 image
    constexpr int kHalf = HD / 2;                         // head_dim of a softmax thread
    extern __shared__ __align__(1024) uint8_t tc_smem[];
    TcTreeShared& sh = *reinterpret_cast<TcTreeShared*>(tc_smem);
    uint8_t* ki = tc_smem + kTcHeaderBytes;  // two buffers of hi, lo
    uint8_t* vi = ki + 4 * kImage;           // hi, lo
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned items = a.c.n_kv * sp.groups;

    // entries with nothing to see
    for (int b = blockIdx.x; b < a.batch; b += gridDim.x) {
        if (FindEntry(a, b).slots != 0) continue;
        for (int t = warp; t < a.tokens; t += kTcWarps)
            for (int i = lane; i < a.n_heads * a.c.hd; i += 32)
                a.out[(size_t(b) * a.tokens + t) * a.out_stride + i] = 0.0f;
    }
    GridDepLaunch();  // the joining kernel may come up as CTAs leave
    const Cut cut(a, kTile, items, 1, 1, gridDim.x);
    if (cut.total == 0 || blockIdx.x >= cut.ctas) return;
    Walk walk;
    walk.cur = cut.Start(blockIdx.x);
    walk.end = cut.Start(blockIdx.x + 1);
    walk.b = cut.Find(a, kTile, items, walk.cur, walk.first);

    if (threadIdx.x == 0) {
        MbarInit(&sh.q_full, kSoftWarps * 32);
        MbarInit(&sh.v_full, kProdWarps * 32);
        MbarInit(&sh.v_empty, 1);
        MbarInit(&sh.o_full, 1);
        MbarInit(&sh.o_empty, kSoftWarps * 32);
        MbarInit(&sh.drain, 1);
        MbarInit(&sh.soft, kSoftWarps * 32);
        MbarInit(&sh.prod, kProdWarps * 32);
        for (int i = 0; i < 2; ++i) {
            MbarInit(&sh.p_full[i], kSoftWarps * 32);
            MbarInit(&sh.s_full[i], 1);
            MbarInit(&sh.k_full[i], kProdWarps * 32);
            MbarInit(&sh.k_empty[i], 1);
        }
        FenceMbarInit();
        sh.abort = 0;
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(SmemAddr(&sh.tmem)));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
    }
    FenceBefore();
    __syncthreads();
    FenceAfter();
    const uint32_t tmem = sh.tmem;

    if (warp < kSoftWarps) {
        // ------------------------------------------------ softmax and accumulation
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftRegs));
        const int half = warp >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t lanes = tmem + ((static_cast<uint32_t>(warp & 3) * 32) << 16);
        int it = 0, pv = 0;  // tiles, and images of V, so far
        uint32_t met = 0;
        bool ok = true;
        while (ok && walk.Next(a, sp, items)) {
            const int r = walk.row0 + row;
            const bool live = r < sp.rows;
            const int t = r / a.group;
            float cs;
            {  // this thread's half of the row of Q
                const float* q = live ? a.q + (size_t(walk.b) * a.tokens + t) * a.q_stride +
                                            size_t(walk.head * a.group + r % a.group) * a.c.hd
                                      : nullptr;
                float x[kHalf], top = 0.0f;
#pragma unroll
                for (int i = 0; i < kHalf; i += 4) {
                    const int d = half * kHalf + i;
                    if (a.q_vec) {
                        const float4 w = q && d < a.c.hd ? __ldg(reinterpret_cast<const float4*>(q + d))
                                                         : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        x[i] = w.x;
                        x[i + 1] = w.y;
                        x[i + 2] = w.z;
                        x[i + 3] = w.w;
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; ++j) x[i + j] = q && d + j < a.c.hd ? __ldg(q + d + j) : 0.0f;
                    }
                }
#pragma unroll
                for (int i = 0; i < kHalf; ++i) top = fmaxf(top, fabsf(x[i]));
                // (its own words: the tiles' maxima of the last item may still be read)
                sh.sum[half][row] = top;
                if (!(ok = Meet(sh, &sh.soft, met, status))) break;
                top = fmaxf(sh.sum[0][row], sh.sum[1][row]);
                const int up = QueryExp(top);
                const float sc = Pow2(up);
                cs = fmaxf(Pow2(-up) * a.scale * kLog2e, kLeast);
#pragma unroll
                for (int i = 0; i < kHalf; i += 16) {  // a k step: 8 columns of hi, 8 of lo
                    uint32_t hi[8], lo[8];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {  // the images' order 0, 2, 1, 3
                        const float* y = x + i + 4 * j;
                        SplitHalf(y[0] * sc, y[2] * sc, hi[2 * j], lo[2 * j]);
                        SplitHalf(y[1] * sc, y[3] * sc, hi[2 * j + 1], lo[2 * j + 1]);
                    }
                    Store8(lanes + kQCol + half * kHalf + i, hi);
                    Store8(lanes + kQCol + half * kHalf + i + 8, lo);
                }
                WaitStore();
                FenceBefore();
                Arrive(&sh.q_full);
            }
            float o[kHalf], m = kStart, l0 = 0.0f, l1 = 0.0f, m_of_o = kStart, m_last = kStart;
            uint32_t poison = 0;
#pragma unroll
            for (int i = 0; i < kHalf; ++i) o[i] = 0.0f;
            const uint64_t* mask = a.mask ? a.mask + size_t(walk.b) * a.tokens * a.words : nullptr;

            // Tile u's weights, then O of tile u - 1 (whose PV has had the time of a QK to finish).  The code of the
            // roles together has to stay in the instruction cache: loops are unrolled only where registers ask for it.
            for (int u = walk.u0; u <= walk.u1; ++u) {
                if (u < walk.u1) {
                    const uint32_t scores = lanes + (it & 1) * kTile + half * 64;
                    if (!(ok = Wait(sh, &sh.s_full[it & 1], (it >> 1) & 1, status))) break;
                    FenceAfter();
                    const bool edge = (u + 1) * kTile > walk.e.len;
                    if (sh.k_big[it % kInfoBufs]) {
#pragma unroll 1
                        for (int i = 0; i < 64; i += 8) {
                            const uint32_t down = sh.k_bits[it % kInfoBufs][(half * 64 + i) >> 5] >> (i & 31);
                            uint32_t x[8];
                            Load8(scores + i, x);
                            WaitLoad();
#pragma unroll
                            for (int j = 0; j < 8; ++j)
                                if ((down >> j) & 1) x[j] = __float_as_uint(__uint_as_float(x[j]) * 512.0f);
                            Store8(scores + i, x);
                        }
                        WaitStore();
                    }
                    // 16 scores, those that the row does not see taken out
                    auto get = [&](float (&x)[16], int i) {
                        Load16(scores + i, x);
                        uint32_t seen = 0xffffu;
                        if (edge)
                            seen = SeenBits(mask, a.words, a.tokens, t, u * kTile + half * 64 + i, walk.e.len, walk.e.slots);
                        WaitLoad();
                        if (edge)
#pragma unroll
                            for (int j = 0; j < 16; ++j)
                                if (!((seen >> j) & 1)) x[j] = -INFINITY;
                    };
                    float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
                    for (int i = 0; i < 64; i += 16) {
                        float x[16];
                        get(x, i);
#pragma unroll
                        for (int j = 0; j < 16; ++j) tops[j & 3] = fmaxf(tops[j & 3], x[j]);
                    }
                    float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
                    sh.top[it & 1][half][row] = top;
                    if (!(ok = Meet(sh, &sh.soft, met, status))) break;
                    top = fmaxf(top, sh.top[it & 1][half ^ 1][row]);
                    m_last = m;
                    if (Passes(top, m, cs)) {
                        const float f = Exp2((m - top) * cs);
                        l0 *= f;
                        l1 *= f;
                        m = top;
                    }
#pragma unroll 1
                    for (int i = 0; i < 64; i += 16) {
                        float x[16];
                        get(x, i);
                        uint32_t hi[8], lo[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            Exponents(x[2 * j], x[2 * j + 1], Pair(-m, -m), Pair(cs, cs), Pair(kOffset, kOffset));
                            const float p0 = Exp2(x[2 * j]), p1 = Exp2(x[2 * j + 1]);
                            l0 += p0;
                            l1 += p1;
                            SplitHalf(p0, p1, hi[j], lo[j]);
                        }
                        Store8(scores + i, hi);
                        Store8(scores + i + 8, lo);
                    }
                    WaitStore();
                    FenceBefore();
                    Arrive(&sh.p_full[it & 1]);
                } else {
                    m_last = m;
                }
                if (u > walk.u0) {
                    if (!(ok = Wait(sh, &sh.o_full, pv & 1, status))) break;
                    FenceAfter();
                    const float keep = Exp2((m_of_o - m_last) * cs);
                    m_of_o = m_last;
#pragma unroll
                    for (int i = 0; i < kHalf; i += 16) {
                        float d[16];
                        Load16(lanes + kOCol + half * kHalf + i, d);
                        WaitLoad();
#pragma unroll
                        for (int j = 0; j < 16; ++j) o[i + j] = fmaf(o[i + j], keep, d[j]);
                    }
                    const int info = sh.v_info[pv % kInfoBufs];
                    if (info & kOdd)
#pragma unroll 1
                        for (int k = 0; k < kTile / 32; ++k) {
                            const uint32_t seen =
                                SeenBits(mask, a.words, a.tokens, t, (u - 1) * kTile + 32 * k, walk.e.len, walk.e.slots);
                            for (int b = 0; b < NB; ++b)
                                if (seen & sh.v_bad[pv % kInfoBufs][b][k]) poison |= 1u << b;
                        }
                    FenceBefore();
                    Arrive(&sh.o_empty);
                    ++pv;
                    if (info & kMore) {  // the tile's large scales
                        if (!(ok = Wait(sh, &sh.o_full, pv & 1, status))) break;
                        FenceAfter();
#pragma unroll
                        for (int i = 0; i < kHalf; i += 8) {
                            uint32_t d[8];
                            Load8(lanes + kOCol + half * kHalf + i, d);
                            WaitLoad();
#pragma unroll
                            for (int j = 0; j < 8; ++j) o[i + j] = fmaf(__uint_as_float(d[j]), 512.0f, o[i + j]);
                        }
                        FenceBefore();
                        Arrive(&sh.o_empty);
                        ++pv;
                    }
                }
                if (u < walk.u1) ++it;
            }
            if (!ok) break;
            // ---- the row's result, or its part of it
            sh.last[half][row] = l0 + l1;
            if (!(ok = Meet(sh, &sh.soft, met, status))) break;
            const float l = sh.last[0][row] + sh.last[1][row];
            if (live) {
#pragma unroll
                for (int i = 0; i < kHalf; ++i)
                    if ((poison >> ((half * kHalf + i) / 32)) & 1) o[i] = NAN;
                if (walk.u0 == 0 && walk.u1 == int(walk.units)) {
                    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                    float* out = OutRow(a, walk.b, walk.head, r);
#pragma unroll
                    for (int i = 0; i < kHalf; i += 4)  // back from the order 0, 2, 1, 3
                        StoreOut(a, out, half * kHalf + i, make_float4(o[i] * inv, o[i + 2] * inv, o[i + 1] * inv, o[i + 3] * inv));
                } else {
                    float* part = sp.parts + (2 * size_t(blockIdx.x) + (walk.u0 == 0 ? 1 : 0)) * (size_t(kTile) * (HD + 2));
#pragma unroll
                    for (int i = 0; i < kHalf; i += 4)
                        __stcg(reinterpret_cast<float4*>(part + row * HD + half * kHalf + i),
                               make_float4(o[i], o[i + 2], o[i + 1], o[i + 3]));
                    if (half == 0) {
                        __stcg(part + kTile * HD + row, Scaled(m, cs, l));
                        __stcg(part + kTile * (HD + 1) + row, l);
                    }
                }
            }
            __syncwarp();
        }
    } else if (warp < kSoftWarps + kProdWarps) {
        // ------------------------------------------------ producers
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kProdRegs));
        const int id = threadIdx.x - kSoftWarps * 32;
        int kt = 0, vt = 0;  // images of K and V so far
        uint32_t met = 0;
        bool ok = true;
        // what the producers' `bits` hold together
        auto together = [&](uint32_t bits) {
            bits = __reduce_or_sync(0xffffffffu, bits);
            const uint32_t side = met & 1;
            if (lane == 0) sh.flag[side][id / 32] = bits;
            ok = Meet(sh, &sh.prod, met, status);
            bits = 0;
#pragma unroll
            for (int i = 0; i < kProdWarps; ++i) bits |= sh.flag[side][i];
            return bits;
        };
        while (ok && walk.Next(a, sp, items)) {
            const long long base = a.c.Row(walk.e.seq, a.layer, walk.head, 0);
            constexpr int kRowBytes = Share<TYPE, NB>::kPieces * 16;
            const uint8_t* kp = static_cast<const uint8_t*>(a.c.k) + base * kRowBytes;
            const uint8_t* vp = static_cast<const uint8_t*>(a.c.v) + base * kRowBytes;
            const __half *ks = a.c.ks + base * NB, *vs = a.c.vs + base * NB;
            // The images in the order of their use: K(0), K(1), V(0), K(2), V(1), ..; the quants of the next one are
            // under way while this one waits for its place.
            const int tiles = walk.u1 - walk.u0, all = 2 * tiles;
            auto is_v = [&](int i) { return (i >= 2 && !(i & 1)) || i == all - 1; };
            auto tile = [&](int i) { return walk.u0 + (is_v(i) ? (i == all - 1 ? tiles - 1 : i / 2 - 1) : (i + 1) / 2); };
            Share<TYPE, NB> r;
            r.Load(kp, ks, walk.u0 * kTile, walk.e.slots, a.c.head_slots - 1, id);
#pragma unroll 1
            for (int i = 0; i < all; ++i) {
                const bool v = is_v(i);
                const int u = tile(i);
                // a drafted slot's V scale that is not finite is taken out and noted
                const bool odd = v && r.TakeOdd(walk.e.len - u * kTile, id);
                const uint32_t flags = together((r.Big() ? 1u : 0u) | (odd ? 2u : 0u));
                if (!ok) break;
                const bool big = flags & 1, any = flags & 2;
                const int n = v ? vt++ : kt++;
                if (v) {
                    if (n > 0 && !(ok = Wait(sh, &sh.v_empty, (n - 1) & 1, status))) break;
                } else {
                    if (n > 1 && !(ok = Wait(sh, &sh.k_empty[n & 1], ((n >> 1) - 1) & 1, status))) break;
                }
                if (any && id < kTile) {  // a row for each of four warps' threads
                    const int at = u * kTile + id;
                    for (int b = 0; b < NB; ++b) {
                        const unsigned short d =
                            __ldg(reinterpret_cast<const unsigned short*>(vs + size_t(min(at, a.c.head_slots - 1)) * NB + b));
                        const bool bad = (d & 0x7C00u) == 0x7C00u && at >= walk.e.len && at < walk.e.slots;
                        const uint32_t bits = __ballot_sync(0xffffffffu, bad);
                        if (lane == 0) sh.v_bad[n % kInfoBufs][b][id / 32] = bits;
                    }
                }
                const bool twice = v && big;  // a tile of V with large scales goes out as two images
                if (id == 0) (v ? sh.v_info : sh.k_big)[n % kInfoBufs] = v ? (any ? kOdd : 0) | (twice ? kMore : 0) : int(big);
                uint8_t* image = v ? vi : ki + (n & 1) * 2 * kImage;
                if (!big) {
                    r.Convert(image, id, sp.magic);
                } else {
                    uint32_t* down = sh.k_bits[n % kInfoBufs];
                    if (!v) {  // the slots that need it
                        if (id < kTile) {
                            const size_t at = min(u * kTile + id, a.c.head_slots - 1);
                            bool large = false;
                            for (int b = 0; b < NB; ++b)
                                large = large || r.IsLarge(__ldg(reinterpret_cast<const unsigned short*>(ks + at * NB + b)));
                            const uint32_t bits = __ballot_sync(0xffffffffu, large);
                            if (lane == 0) down[id / 32] = bits;
                        }
                        if (!(ok = Meet(sh, &sh.prod, met, status))) break;
                    }
                    constexpr uint32_t kOne = 0x3C003C00u, kDown = 0x18001800u;  // 1, 2^-9
                    r.ConvertLarge(image, v ? vp : kp, v ? vs : ks, u * kTile, walk.e.slots, a.c.head_slots - 1,
                                   v ? walk.e.len - u * kTile : kTile, id, sp.magic, v ? nullptr : down, v ? 0 : kDown, kOne);
                    if (twice) {
                        FenceAsync();
                        Arrive(&sh.v_full);
                        if (!(ok = Wait(sh, &sh.v_empty, n & 1, status))) break;
                        ++vt;
                        if (id == 0) sh.v_info[(n + 1) % kInfoBufs] = 0;
                        r.ConvertLarge(image, vp, vs, u * kTile, walk.e.slots, a.c.head_slots - 1, walk.e.len - u * kTile, id,
                                       sp.magic, nullptr, kDown, 0);
                    }
                }
                FenceAsync();
                Arrive(v ? &sh.v_full : &sh.k_full[n & 1]);
                if (i + 1 < all) {
                    const bool w = is_v(i + 1);
                    r.Load(w ? vp : kp, w ? vs : ks, tile(i + 1) * kTile, walk.e.slots, a.c.head_slots - 1, id);
                }
            }
        }
    } else if (warp >= kMmaWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kMmaRegs));
    }
    if (warp == kMmaWarp) {
        // ------------------------------------------------ MMA issue
        const uint32_t qk = Instruction(kTile, false), pv_op = Instruction(HD, true);
        // K-major images: chunks of K kChunkPitch bytes apart, groups of 8 rows 128
        const uint64_t kd = Descriptor(SmemAddr(ki), kChunkPitch, 128);
        // V: groups of 8 slots 128 bytes apart, groups of 8 of head_dim kChunkPitch
        const uint64_t vd = Descriptor(SmemAddr(vi), 128, kChunkPitch);
        constexpr uint64_t kLoStep = kImage >> 4, kKStep = (2 * kChunkPitch) >> 4, kVStep = 256 >> 4;
        const uint32_t one = ElectOne(), base = __shfl_sync(0xffffffffu, tmem, 0);
        int it = 0, pv = 0, item = 0;  // tiles, images of V, items
        bool ok = true;
        while (ok && walk.Next(a, sp, items)) {
            if (!(ok = Wait(sh, &sh.q_full, item & 1, status))) break;
            ++item;
            for (int u = walk.u0; u <= walk.u1; ++u) {
                if (u < walk.u1) {  // QK of tile `it`
                    if (!(ok = Wait(sh, &sh.k_full[it & 1], (it >> 1) & 1, status))) break;
                    // The weights that lay in this buffer, of tile it - 2, have been multiplied: its PV is the one issued
                    // last, but at the start of an item, where PV(it - 1) has been issued after O(it - 2) was read.
                    if (pv > 0 && u > walk.u0 && !(ok = Wait(sh, &sh.o_full, (pv - 1) & 1, status))) break;
                    FenceAfter();
                    const uint32_t d = base + (it & 1) * kTile, q = base + kQCol;
                    const uint64_t k = kd + (it & 1) * 2 * kLoStep;
                    MmaTensor<false>(one, d, q + 8, k, qk);
#pragma unroll
                    for (int s = 1; s < HD / 16; ++s) MmaTensor<true>(one, d, q + 16 * s + 8, k + s * kKStep, qk);
#pragma unroll
                    for (int s = 0; s < HD / 16; ++s) MmaTensor<true>(one, d, q + 16 * s, k + kLoStep + s * kKStep, qk);
#pragma unroll
                    for (int s = 0; s < HD / 16; ++s) MmaTensor<true>(one, d, q + 16 * s, k + s * kKStep, qk);
                    Commit(one, &sh.k_empty[it & 1]);
                    Commit(one, &sh.s_full[it & 1]);
                }
                const int n = it - 1;  // PV of the tile before
                if (u > walk.u0 && !(ok = Wait(sh, &sh.p_full[n & 1], (n >> 1) & 1, status))) break;
#pragma unroll 1
                for (bool more = u > walk.u0; more; ++pv) {
                    if (!(ok = Wait(sh, &sh.v_full, pv & 1, status))) break;
                    if (pv > 0 && !(ok = Wait(sh, &sh.o_empty, (pv - 1) & 1, status))) break;  // the last O has been read
                    FenceAfter();
                    const uint32_t p = base + (n & 1) * kTile;
                    MmaTensor<false>(one, base + kOCol, p + 8, vd, pv_op);
#pragma unroll
                    for (int s = 1; s < kTile / 16; ++s)
                        MmaTensor<true>(one, base + kOCol, p + 16 * s + 8, vd + s * kVStep, pv_op);
#pragma unroll
                    for (int s = 0; s < kTile / 16; ++s)
                        MmaTensor<true>(one, base + kOCol, p + 16 * s, vd + kLoStep + s * kVStep, pv_op);
#pragma unroll
                    for (int s = 0; s < kTile / 16; ++s) MmaTensor<true>(one, base + kOCol, p + 16 * s, vd + s * kVStep, pv_op);
                    Commit(one, &sh.v_empty);
                    Commit(one, &sh.o_full);
                    more = sh.v_info[pv % kInfoBufs] & kMore;
                }
                if (!ok) break;
                if (u < walk.u1) ++it;
            }
        }
        // every MMA issued has finished before tensor memory is freed
        Commit(one, &sh.drain);
        if (!MbarWaitFor(&sh.drain, 0, kTcWait, nullptr)) Fail(sh, status);
    }
    FenceBefore();
    __syncthreads();
    if (warp == kMmaWarp) {
        FenceAfter();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    }
}

template <int TYPE, int NB>
bool LaunchTc(DeviceContext& ctx, const TreeArgs& a) {
    TreeSplit sp{};
    sp.rows = a.tokens * a.group;
    sp.groups = static_cast<int>(CeilDiv(sp.rows, kTile));
    const unsigned long long items = 1ull * a.c.n_kv * sp.groups;
    const long long slots = std::min<long long>(1LL * std::min(a.max_len, a.c.max_seq) + a.tokens, a.c.max_seq);
    const double units = double(a.batch) * double(items) * double(CeilDiv(slots, kTile));
    if (units >= 2147483648.0) return false;
    const int grid = static_cast<int>(std::min<double>(ctx.sm_count, units));
    sp.parts = static_cast<float*>(Workspace(ctx, 2 * size_t(grid) * kTile * (NB * 32 + 2) * sizeof(float)));
    sp.magic = TYPE == MLB_Q8_0 ? kMagic8 : kMagic4;
    constexpr int kBytes = kTcHeaderBytes + 6 * NB * 4 * kChunkPitch;
    auto* kernel = TreeTcKernel<TYPE, NB>;
    static int configured[64] = {};
    if (ctx.device >= 64 || !configured[ctx.device]) {
        CheckCuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes),
                  "cudaFuncSetAttribute(TreeTcKernel)");
        cudaFuncAttributes attr;
        CheckCuda(cudaFuncGetAttributes(&attr, kernel), "cudaFuncGetAttributes(TreeTcKernel)");
        Require(attr.numRegs >= kLaunchRegs, "mlb_attention_tree", "compiled with too few registers", MLB_ERR_UNSUPPORTED);
        if (ctx.device < 64) configured[ctx.device] = 1;
    }
    kernel<<<grid, kTcWarps * 32, kBytes, ctx.stream>>>(a, sp, ctx.status);
    CheckCuda(cudaGetLastError(), "TreeTcKernel");
    if (grid == 1) return true;  // nothing is cut
    LaunchJoin<NB>(ctx, a, sp, kTile, 1, 1, kTile, grid);
    return true;
}

template <int TYPE>
bool LaunchTcBlocks(DeviceContext& ctx, const TreeArgs& a) {
    switch (a.c.blocks) {
        case 1: return LaunchTc<TYPE, 1>(ctx, a);
        case 2: return LaunchTc<TYPE, 2>(ctx, a);
        case 3: return LaunchTc<TYPE, 3>(ctx, a);
        case 4: return LaunchTc<TYPE, 4>(ctx, a);
        default: return false;
    }
}

}  // namespace

bool LaunchTreeTc(DeviceContext& ctx, const TreeArgs& a) {
    if (a.c.type == MLB_F32) return false;
    return a.c.type == MLB_Q8_0 ? LaunchTcBlocks<MLB_Q8_0>(ctx, a) : LaunchTcBlocks<MLB_Q4_0>(ctx, a);
}

}  // namespace mlb
