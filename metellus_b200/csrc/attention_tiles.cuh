// Paged attention of one token per sequence in tiles of 16 or 32 tokens a warp.
//
// For each sequence and key-value head: S^T = K Q^T (16 tokens x 8 query heads a product),
// the softmax over the tokens in one pass (running maximum m, l = sum exp2(s - m), O = sum
// exp2(s - m) v, rescaled when m grows), and O^T += V^T P^T. What bounds it is HBM: K and V
// are read once and used by one token's query heads only (2 flops a query head for each
// element), so everything here serves the loads:
//
// * The tokens are the rows (M) of the matrix instructions and the query heads their 8
//   columns: a group of 4 or 8 query heads wastes little of them, and 16 columns (NT = 2)
//   serve larger groups. K's fragments come by ldmatrix, V's by its transposing form; S^T's
//   accumulators become P^T's operands by transposing 8 x 8 blocks in registers.
// * Every warp works alone, without barriers: it streams tiles through its own ring of S
//   stages in shared memory (16-byte asynchronous copies, page by page), and while one
//   waits where a head ends, the others of its SM go on.
// * The tiles of all sequences lie on one line that is cut into equal ranges: a ragged batch
//   or one long sequence keeps every SM at work. Neighbouring warps take the heads of one range,
//   whose rows are neighbours in memory. A sequence that a cut crosses leaves parts (m, l, O) of
//   its heads in the workspace, and a second kernel joins them; it is launched early and
//   waits for the first on the device.
//
// Measured (bf16, 32 query heads on 8 of 128, pages of 16 in random order; replayed from graphs, as all
// times here): 64 sequences of 4096 to 8192 tokens 246 us = 6.6 TB/s, the copy rate; 16 of 37 to 4001 28 us =
// 4.4 TB/s; 1 of 120001 82 us = 6.0 TB/s; 1 of 100 7.6 us. The matrix pipe is busy 14 % of the time and a third of the issue slots are
// used, so its 16-row form loses nothing here, and the 128-row form of tcgen05 would cut a line of
// tiles eight times as coarsely and tie the warps of a block to one another's loads. What is left at
// short lines are the ends: lengths, then page numbers, then rows have to arrive before the first
// product (4 us), SMs finish up to 3 us apart, and the join takes 2 to 3 us.
//
// 8-bit codes become fp16 in registers, exactly; K's scales multiply the scores, V's the
// probabilities. 32-bit queries (and 32-bit caches) are split into pieces whose products
// together keep at least 22 bits.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <atomic>
#include <type_traits>

#include "mt_paged_attention.h"

namespace mt {
namespace tiles {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct TileArgs {
    AttentionArgs a;
    int items;       // of a sequence: kv_heads * row blocks; warp w works on item w % items of range w / items
    int row_chunks;  // 16-byte pieces of a cache row
    int q_chunks;    // 16-byte pieces of a query row, 0 where it cannot be copied in pieces
    int out_quads;   // output rows can be written four elements at a time
    int whole;       // a range a sequence: nothing is cut
    FastDiv ranges, per_range, row_blocks;  // divisors: ranges, items, blocks of NT * 8 query heads in a group
    // workspace: two parts a warp, (m, l) and O of NT * 8 rows each. Part 2 w belongs to a
    // sequence that began before warp w's range, part 2 w + 1 to one that ends behind it.
    float2* part_ml;
    float* part_o;
};

// ---- instructions ------------------------------------------------------------------------

__device__ inline uint32_t smem_address(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// kBeyond: a row of 8-bit codes is 128 bytes or less, and the next one is another warp's of the
// same block: L2 fetches 256 bytes (e4m3, 32 sequences of 8192, 64 query heads on 8 of 128: 99.0 us, with 128 bytes 99.8).
template <bool kBeyond> __device__ inline void copy16(uint32_t dst, const void* src, bool really) {
    if constexpr (kBeyond)
        asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(really ? 16 : 0));
    else
        asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(really ? 16 : 0));
}
__device__ inline void copy4(uint32_t dst, const void* src, bool really) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(really ? 4 : 0));
}
__device__ inline void copies_commit() { asm volatile("cp.async.commit_group;"); }
__device__ inline void copies_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
template <int N> __device__ inline void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ inline void load_matrices(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ inline void load_transposed(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ inline uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ inline float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <int CT>
__device__ inline void product(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (CT == MT_F32)
        asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else if constexpr (CT == MT_BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// ---- operands ------------------------------------------------------------------------------

template <class T> __device__ inline T rounded(float x);
template <> __device__ inline float rounded<float>(float x) { return x; }
template <> __device__ inline __half rounded<__half>(float x) { return __float2half_rn(x); }
template <> __device__ inline __nv_bfloat16 rounded<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

__device__ inline void store4(float* to, float4 y) { *(float4*)to = y; }
__device__ inline void store4(__half* to, float4 y) {
    *(__half2*)to = __floats2half2_rn(y.x, y.y);
    *(__half2*)(to + 2) = __floats2half2_rn(y.z, y.w);
}
__device__ inline void store4(__nv_bfloat16* to, float4 y) {
    *(__nv_bfloat162*)to = __floats2bfloat162_rn(y.x, y.y);
    *(__nv_bfloat162*)(to + 2) = __floats2bfloat162_rn(y.z, y.w);
}

// Two floats as one register of 16-bit operands (bf16 for a bf16 cache, else fp16).
template <bool kBf16> __device__ inline uint32_t pack(float lo, float hi) {
    if constexpr (kBf16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return reinterpret_cast<const uint32_t&>(v);
    } else {
        const __half2 v = __floats2half2_rn(lo, hi);
        return reinterpret_cast<const uint32_t&>(v);
    }
}
template <bool kBf16> __device__ inline float2 unpack(uint32_t x) {
    if constexpr (kBf16) return __bfloat1622float2(reinterpret_cast<const __nv_bfloat162&>(x));
    else return __half22float2(reinterpret_cast<const __half2&>(x));
}

// The upper 11 significant bits of a float, to nearest: what a tf32 operand keeps.
__device__ inline uint32_t upper(float x) { return (__float_as_uint(x) + 0x1000u) & 0xffffe000u; }

// Four codes as fp16, exactly: bytes 0, 1 and 2, 3 of x (kPairs), or 0, 2 and 1, 3.
template <int CT, bool kPairs> __device__ inline void decode(uint32_t x, uint32_t& lo, uint32_t& hi) {
    if constexpr (CT == MT_I8) {
        // 0x6400 | u is 1024 + u; with u = code + 128, 1152 more than the code
        x ^= 0x80808080u;
        const __half2 off = __half2half2(__ushort_as_half(0x6480));
        const uint32_t a = __byte_perm(x, 0x64646464u, kPairs ? 0x4140 : 0x4240);
        const uint32_t b = __byte_perm(x, 0x64646464u, kPairs ? 0x4342 : 0x4341);
        const __half2 u = __hsub2(reinterpret_cast<const __half2&>(a), off), v = __hsub2(reinterpret_cast<const __half2&>(b), off);
        lo = reinterpret_cast<const uint32_t&>(u);
        hi = reinterpret_cast<const uint32_t&>(v);
    } else {
        if constexpr (!kPairs) x = __byte_perm(x, 0, 0x3120);
        asm("{ .reg .b16 l, h; mov.b32 {l, h}, %2; cvt.rn.f16x2.e4m3x2 %0, l; cvt.rn.f16x2.e4m3x2 %1, h; }"
            : "=r"(lo), "=r"(hi) : "r"(x));
    }
}

// ---- shapes --------------------------------------------------------------------------------

template <int CT, class Q, int DP, int NT> struct Shape {
    static constexpr bool kQ32 = sizeof(Q) == 4;
    static constexpr int EB = CT == MT_F32 ? 4 : CT == MT_F16 || CT == MT_BF16 ? 2 : 1;
    static constexpr bool kScaled = EB == 1, kBf16 = CT == MT_BF16;
    // The matrix pipe truncates what it adds to an accumulator, so a long chain of products
    // drifts. For 32-bit outputs chains are short (4 steps of a score, one tile of O) and
    // are added up in fp32, rounded to nearest; smaller pieces have a chain of their own. fp32, heads of
    // 128, 18 sequences up to 2280: off by 3.9e-7 (in fp32 throughout 7.6e-7; in one chain 1.7e-6).
    static constexpr bool kExact = kQ32;
    // For 16-bit outputs O's chains are kChain tiles long, and added up in the workspace. 1770 tiles of values
    // around 1 come out 1.5e-5 too small (7e-6 with 64), in one chain 2.4e-4, fp16's
    // half step. 64 sequences of 4096 to 8192 tokens, bf16: 246.4 us, in one chain 243.7, 64 tiles 248; a sum
    // a tile, in registers, would cost up to 14 % (16-bit) and 31 % (8-bit, 16 heads a warp).
    static constexpr int kChain = 128;
    static constexpr int ROW = DP * EB;               // bytes of a (padded) cache row
    static constexpr int CPR = ROW / 16;              // its 16-byte pieces
    // tokens a tile: 8-bit rows are short, and a tile's chain of instructions takes as long
    static constexpr int TW = kScaled && DP <= 128 ? 32 : 16, TB = TW / 16;
    static constexpr int STAGE = 2 * TW * ROW + (kScaled ? 256 : 0);  // rows of K, of V, scales of 32 tokens each
    // Whether step c of a row's pairs of pieces may be behind its end: rows are longer than half of
    // DP, but for DP = 32
    __host__ __device__ static constexpr bool may_end(int c) { return DP == 32 ? c >= 1 : 4 * c >= CPR; }
    static constexpr int KS = CT == MT_F32 ? DP / 8 : DP / 16;    // steps of K Q^T
    // pieces of a query: fp16 11 bits, bf16 8 bits, tf32 11 bits each
    static constexpr int QP = CT == MT_F32 ? 2 : !kQ32 ? 1 : kBf16 ? 3 : 2;
    // pieces of a probability: enough that the output's own rounding is what shows (with one of fp16, off by
    // up to 2^-12, 5 % of the bf16 outputs over 2 to 8 tokens were rounded the wrong way; at no cost in time)
    static constexpr int PP = CT == MT_F32 ? 2 : kQ32 ? QP : 2;
    // queries that fp16 may not hold are divided by a power of two per row
    static constexpr bool kNormed = CT != MT_F32 && !kBf16 && (kQ32 || kScaled);
    // A 16-bit cache's next rows are asked for in two bursts a tile, K's before the scores and V's behind
    // them (64 sequences of 6144, bf16: 248 us, in one burst 253). 8-bit and 32-bit tiles, whose products take
    // longer, lose by it (e4m3 99 -> 101, fp32 108 -> 110).
    static constexpr bool kTwoBursts = EB == 2;
    // The exponents' base m is raised only when a score passes it by more than kSlack (a factor of
    // 2^4), which after a head's first tiles is rare. fp16 probabilities are held times
    // 2^11, so that they stay below 2^15; the smallest, 2^-24, is 2^-35 of 1. Those of an 8-bit cache are
    // multiplied by V's scales before they are fp16, and held in units of 2^-11 of the largest scale, or, where
    // that is kSpread times a head's largest product or more, of 2^-5 of the product. (In units of the scale
    // alone a token that has no weight cost the others their bits: float32 queries, one token's scale 10^8
    // times the others': off by 5.5e-4, now 2.3e-7.)
    static constexpr float kSlack = 4.0f, kOffset = CT == MT_F16 ? 11.0f : 0.0f;
    static constexpr float kLeastUnit = 1.17549435e-38f, kSpread = 64.0f;  // 2^-126, 2^6
    // A part's queries come into shared memory as they are, while the part before is worked
    // on; then they stay in registers as operands, or, where O leaves too few, in shared memory.
    // Those that are operands as they are (one piece) need no second place, and come late.
    static constexpr bool kQReg = KS * 2 * NT * QP + DP / 4 * NT <= (EB == 4 ? 192 : 168), kQRaw = !kQReg && QP == 1 && !kNormed;
    static constexpr int ROWS = NT * 8;
    static constexpr int QROW = DP * (kQ32 ? 4 : 2), QPIECES = QROW / 16, QSPREAD = QPIECES < 8 ? QPIECES - 1 : 7;
    static constexpr int Q_BYTES = ROWS * QROW + (kQReg || kQRaw ? 0 : KS * NT * QP * 256);
    static constexpr int warp_bytes(int stages) { return stages * STAGE + Q_BYTES + 128; }
    // stages and resident blocks: 3 blocks an SM (12 warps, 168 registers, enough for O of 64 each;
    // 4 for heads of 32) with 3 stages at least, else 2 blocks, else one. With one warp a scheduler instead of two, bf16
    // under float32 queries took 79 us for 41 us of bytes (now 49).
    static constexpr int kMost = 227 * 1024;          // of shared memory a block
    static constexpr bool fits(int warps, int stages, int blocks) {
        return warps * warp_bytes(stages) <= kMost && blocks * (warps * warp_bytes(stages) + 1024) <= 228 * 1024;
    }
    // warps a block: 4, or where two blocks of them do not fit, 6 of 32-bit rows with 2 stages (their
    // products take long: 8 heads of 128, 16 sequences of 4096 tokens 107 us, 120 with 4 warps), else
    // as many as fit
    static constexpr int NW = !fits(4, 2, 2) && fits(6, 2, 1) ? 6 : fits(4, 2, 1) ? 4 : fits(3, 2, 1) ? 3 : 2;
    static constexpr int kMany = fits(NW, 3, 4) && DP * NT <= 32 ? 4 : fits(NW, 3, 3) && DP * NT <= 128 ? 3 : fits(NW, 2, 2) ? 2 : 1;
    static constexpr int S = fits(NW, 4, kMany) ? 4 : fits(NW, 3, kMany) ? 3 : 2;
    static constexpr int WARP = warp_bytes(S), SMEM = NW * WARP;
    static constexpr int BLOCKS = kMany;
    static_assert(SMEM <= kMost, "a block's shared memory");
};

// Where 16-byte piece c of row r lies, so that 8 rows' pieces of one column fall in
// different banks.
template <int CPR> __device__ inline int swizzled(int r, int c) {
    if constexpr (CPR >= 8) return r * CPR + (c ^ (r & 7));
    else return r * CPR + (c ^ (r / (8 / CPR) & (CPR - 1)));
}

// Where a warp is on the line of tiles.
struct Cursor {
    int b, begin, end, tiles, tile;
    int next, next_length;  // the next sequence with tokens
};

// The tokens [begin, end) that a sequence of `length` shows, and its tiles.
template <int TW> __device__ inline void enter_sequence(Cursor& c, const TileArgs& t, int length) {
    c.end = min(max(length, 0), t.a.max_tokens);
    c.begin = c.end > t.a.window ? c.end - t.a.window : 0;
    c.tiles = (c.end - c.begin + TW - 1) / TW;
}
__device__ inline int length_of(const TileArgs& t, int b) { return t.a.lengths[(int64_t)b * t.a.length_seq]; }

// The cuts of the line of all sequences' tiles: every range gets tiles / ranges, the first ones
// one more. Every warp works them out for itself, without barriers: each lane sums a run of
// sequences, and a scan over the lanes finds the one that a range begins in.
template <int TW> struct Cuts {
    const TileArgs& t;
    int b0, b1, mine;  // this lane's sequences and their tiles
    uint32_t base, more;

    __device__ int tiles_of(int b, Cursor& c) const {
        enter_sequence<TW>(c, t, length_of(t, b));
        return c.tiles;
    }
    __device__ explicit Cuts(const TileArgs& args) : t(args), mine(0) {
        const int per = (t.a.batch + 31) / 32, lane = threadIdx.x & 31;
        b0 = min(lane * per, t.a.batch);
        b1 = min(b0 + per, t.a.batch);
        Cursor c;
        for (int b = b0; b < b1; ++b) mine += tiles_of(b, c);
        base = t.ranges.div((uint32_t)__reduce_add_sync(0xffffffffu, mine), &more);
    }
    __device__ int first(uint32_t range) const { return (int)(range * base + min(range, more)); }
    __device__ int owner(uint32_t tile) const {
        const uint32_t big = more * (base + 1);
        return (int)(tile < big ? tile / (base + 1) : more + (tile - big) / base);  // base is not 0 in the second
    }
    // The tiles of the sequences before b (all lanes of a warp call it).
    __device__ int before(int b) const {
        Cursor c;
        int n = 0;
        for (int i = b0; i < min(b1, b); ++i) n += tiles_of(i, c);
        return __reduce_add_sync(0xffffffffu, n);
    }
    // The cursor at a range's first tile; returns how many tiles the range has.
    __device__ int locate(int range, Cursor& c) const {
        const int lane = threadIdx.x & 31, target = first(range), count = first(range + 1) - target;
        int upto = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, upto, d);
            if (lane >= d) upto += o;
        }
        const uint32_t who = __ballot_sync(0xffffffffu, target < upto);
        if (!who || count == 0) return 0;  // behind the end
        const int src = __ffs(who) - 1;
        int b = b0, p = upto - mine, length = 0;
        if (lane == src)
            for (; b < b1; ++b) {
                length = length_of(t, b);
                enter_sequence<TW>(c, t, length);
                if (target < p + c.tiles) break;
                p += c.tiles;
            }
        c.b = __shfl_sync(0xffffffffu, b, src);
        p = __shfl_sync(0xffffffffu, p, src);
        enter_sequence<TW>(c, t, __shfl_sync(0xffffffffu, length, src));
        c.tile = target - p;
        return count;
    }
};

// kPadded: rows are shorter than DP. Only that form looks for their end: with the tests in it, the
// other would be 5 to 30 % slower (bf16, 16 sequences of 4096 tokens, 8 heads of 256: 91 us, 115);
// it takes 44 us at 80 dims, 97 of fp32, where products of whole DPs took 47, 157.
template <int CT, class Q, int DP, int NT, bool kPadded>
__global__ void __launch_bounds__(Shape<CT, Q, DP, NT>::NW * 32, Shape<CT, Q, DP, NT>::BLOCKS)
attention_tiles(const __grid_constant__ TileArgs t) {
    using Z = Shape<CT, Q, DP, NT>;
    constexpr int TW = Z::TW, TB = Z::TB, S = Z::S, CPR = Z::CPR, ROWS = Z::ROWS, QP = Z::QP, PP = Z::PP, KS = Z::KS;
    constexpr bool kScaled = Z::kScaled, kBf16 = Z::kBf16;
    extern __shared__ __align__(128) unsigned char smem[];
    const AttentionArgs& a = t.a;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, quad = lane & 3, oct = lane >> 2;
    unsigned char* const ring = smem + warp * Z::WARP;
    unsigned char* const sm_raw = ring + S * Z::STAGE;                    // queries as they are
    uint2* const sm_q = (uint2*)(sm_raw + ROWS * Z::QROW);                // and as operands, where not in registers
    int4* const sm_meta = (int4*)(ring + Z::WARP - 128);

    const int me = blockIdx.x * (blockDim.x >> 5) + warp;
    uint32_t item;
    const int range = (int)t.per_range.div((uint32_t)me, &item);
    uint32_t row_block;
    const int kv_head = (int)t.row_blocks.div(item, &row_block);
    const int head0 = kv_head * a.group + (int)row_block * ROWS, rows = min(ROWS, a.group - (int)row_block * ROWS);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    Cursor in{};
    int tiles;
    if (t.whole) {
        if (range >= a.batch) return;
        in.b = range;
        in.tile = 0;
        enter_sequence<TW>(in, t, length_of(t, in.b));
        tiles = in.tiles;
    } else {
        if (range >= (int)t.ranges.d) return;
        tiles = Cuts<TW>(t).locate(range, in);
    }
    auto find_next = [&]() {
        do ++in.next;
        while (in.next < a.batch && (in.next_length = length_of(t, in.next)) <= 0);
    };
    in.next = in.b;
    if (tiles > in.tiles - in.tile) find_next();

    // -- a tile to fetch: lane l looks after token l's rows of K and V
    struct Step {
        int b, next, page, flags;  // page: -1 for no token
        uint32_t at;         // the token's place in it
    };
    constexpr int kFirst = 1, kLast = 2, kFromStart = 4, kEnds = 8, kMore = 16;  // of a part; its sequence's ends; parts follow
    int left = tiles;
    bool from_start = in.tile == 0, fresh = true;
    auto look_up = [&]() {
        Step s;
        s.b = in.b;
        s.next = in.next;
        const int token = in.begin + in.tile * TW + (lane & (TW - 1));
        const uint32_t j = a.page.div((uint32_t)token, &s.at);
        s.page = token < in.end ? a.tables[(int64_t)in.b * a.table_seq + j] : -1;
        const bool ends = in.tile + 1 == in.tiles;
        s.flags = (fresh ? kFirst : 0) | (left > in.tiles - in.tile ? kMore : 0) | (ends || left == 1 ? kLast : 0) | (from_start ? kFromStart : 0) | (ends ? kEnds : 0);
        --left;
        fresh = false;
        if (++in.tile == in.tiles) {
            in.tile = 0;
            fresh = from_start = true;
            in.b = in.next;
            enter_sequence<TW>(in, t, in.next_length);
            if (left > in.tiles) find_next();
        }
        return s;
    };
    // of 16 tokens, lanes 16 .. 31 look after V
    const bool is_v = TW == 16 && lane >= 16;
    const uint32_t row_page = is_v ? a.v_rows.page : a.k_rows.page, row_token = is_v ? a.v_rows.token : a.k_rows.token;
    const int64_t head_bytes = (int64_t)kv_head * Z::EB;
    // the piece of a row that this lane copies, where a row has no more than 32
    const int row_chunks = kPadded ? t.row_chunks : CPR;
    const unsigned char* const k_base = (const unsigned char*)a.cache.k.ptr + head_bytes * a.cache.k.head + (CPR <= 32 ? lane % CPR * 16 : 0);
    const unsigned char* const v_base = (const unsigned char*)a.cache.v.ptr + head_bytes * a.cache.v.head + (CPR <= 32 ? lane % CPR * 16 : 0);
    const unsigned char* const k_scales = (const unsigned char*)a.cache.k_scale.ptr + (int64_t)kv_head * a.cache.k_scale.head * 4;
    const unsigned char* const v_scales = (const unsigned char*)a.cache.v_scale.ptr + (int64_t)kv_head * a.cache.v_scale.head * 4;
    // where the rows of the tile being asked for are, and which of them there are
    uint32_t k_row = 0, v_row = 0, there_mask = 0;
    constexpr uint32_t kAll = TW == 32 ? 0xffffffffu : 0xffffu;
    auto find_rows = [&](const Step& s, int slot) {
        const bool valid = s.page >= 0 && s.page < a.cache.pages;
        there_mask = __ballot_sync(0xffffffffu, valid) & kAll;
        const uint32_t page = valid ? (uint32_t)s.page : 0u, at = valid ? s.at : 0u;
        k_row = page * row_page + at * row_token;
        v_row = TW == 32 ? page * a.v_rows.page + at * a.v_rows.token : k_row;
        if (lane == 0) sm_meta[slot] = make_int4(s.b, s.flags, (int)there_mask, s.next);
        if constexpr (kScaled) {
            const uint32_t to = smem_address(ring + slot * Z::STAGE) + 2 * TW * Z::ROW;
            const uint32_t zk = page * a.k_scale_rows.page + at * a.k_scale_rows.token;
            const uint32_t zv = page * a.v_scale_rows.page + at * a.v_scale_rows.token;
            copy4(to + lane * 4, k_scales + (uint64_t)zk * a.k_scale_rows.unit, valid);
            copy4(to + (32 + lane) * 4, v_scales + (uint64_t)zv * a.v_scale_rows.unit, valid);
        }
    };
    auto copy_rows = [&](int slot, auto of_v, auto whole_tile) {
        constexpr bool kV = decltype(of_v)::value, kWhole = decltype(whole_tile)::value;
        constexpr int kCopies = TW * CPR / 32, kUnroll = kWhole || kCopies < 4 ? kCopies : 4;  // the rarer case's code stays small
        const uint32_t to = smem_address(ring + slot * Z::STAGE) + (kV ? TW * Z::ROW : 0);
#pragma unroll kUnroll
        for (int i = 0; i < TW * CPR / 32; ++i) {
            const int r = (i * 32 + lane) / CPR, piece = (i * 32 + lane) % CPR;
            const uint32_t number = __shfl_sync(0xffffffffu, kV ? v_row : k_row, r + (kV && TW == 16 ? 16 : 0));
            const unsigned char* const from = (kV ? v_base : k_base) + (uint64_t)number * (kV ? a.v_rows.unit : a.k_rows.unit) +
                                              (CPR <= 32 ? 0 : piece * 16);
            const uint32_t dst = to + swizzled<CPR>(r, piece) * 16;
            if constexpr (kWhole) {
                if (piece < row_chunks) copy16<kScaled>(dst, from, true);
            } else {
                // absent tokens: V must be zeros (their probability is 0, and 0 * NaN is not); K's
                // scores are replaced
                const bool there = there_mask >> r & 1;
                if (piece < row_chunks && (kV || there)) copy16<kScaled>(dst, from, there);
            }
        }
    };
    auto fetch = [&](int slot, auto of_v) {
        if (there_mask == kAll) copy_rows(slot, of_v, std::true_type{});
        else if (there_mask) copy_rows(slot, of_v, std::false_type{});
    };
    // Behind a row's last piece K is zeros, as the queries are there; V's columns are not used. Copies
    // leave it alone, a part's end (which uses a stage otherwise) puts it back.
    auto clear_padding = [&](int slot) {
        for (int i = lane; i < TW * (CPR - row_chunks); i += 32) {
            const int r = i % TW, piece = row_chunks + i / TW;
            *(uint4*)(ring + slot * Z::STAGE + swizzled<CPR>(r, piece) * 16) = make_uint4(0, 0, 0, 0);
        }
    };
    constexpr std::false_type kKeys{};
    constexpr std::true_type kValues{};

    // -- a part's queries: asked for early, taken when it begins. Their rows' 16-byte pieces are
    // exchanged as the cache's are.
    auto q_place = [](int r, int d) {
        const int byte = d * (int)sizeof(Q);
        return r * Z::QROW + ((byte >> 4 ^ (r & Z::QSPREAD)) << 4 | (byte & 15));
    };
    auto ask_queries = [&](int b) {
        const Q* const q = (const Q*)a.q + (int64_t)b * a.q_seq + (int64_t)head0 * a.q_head;
        const uint32_t to = smem_address(sm_raw);
        if (t.q_chunks)
            for (int i = lane; i < rows * t.q_chunks; i += 32) {
                const int r = i / t.q_chunks, piece = i - r * t.q_chunks;
                copy16<false>(to + r * Z::QROW + (piece ^ (r & Z::QSPREAD)) * 16, (const unsigned char*)(q + (int64_t)r * a.q_head) + piece * 16, true);
            }
        else
            for (int i = lane; i < rows * a.cache.head_dim; i += 32) {
                const int r = i / a.cache.head_dim, d = i - r * a.cache.head_dim;
                *(Q*)(sm_raw + q_place(r, d)) = q[(int64_t)r * a.q_head + d];
            }
    };
    // in the order that the products take them: four lanes a row
    uint2 qf[Z::kQReg ? KS : 1][NT][QP];
    float qscale[NT][2];
    auto lay_out = [&](int n, int dim) {
        const int r = n * 8 + oct;
        if constexpr (QP == 1 && !Z::kNormed) {
            // operands as they are
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                const int d = k * 16 + quad * 2;
                qf[k][n][0] = make_uint2(d < dim ? *(const uint32_t*)(sm_raw + q_place(r, d)) : 0u,
                                         d + 8 < dim ? *(const uint32_t*)(sm_raw + q_place(r, d + 8)) : 0u);
            }
            qscale[n][0] = qscale[n][1] = a.scale * kLog2e;
            return;
        }
        constexpr int XS = CT == MT_F32 ? 2 : 4;
        float x[KS][XS];
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int i = 0; i < XS; i += XS / 2) {
                const int d = CT == MT_F32 ? k * 8 + quad + i * 4
                              : kScaled ? k * 16 + quad * 4 + i : k * 16 + quad * 2 + i * 4;
                if constexpr (CT == MT_F32) {
                    x[k][i] = d < dim ? (float)*(const Q*)(sm_raw + q_place(r, d)) : 0.0f;
                } else {  // head_dim is even here
                    float2 v = make_float2(0.0f, 0.0f);
                    if (d < dim) {
                        const unsigned char* const at = sm_raw + q_place(r, d);
                        if constexpr (sizeof(Q) == 4) v = *(const float2*)at;
                        else v = unpack<std::is_same<Q, __nv_bfloat16>::value>(*(const uint32_t*)at);
                    }
                    x[k][i] = v.x;
                    x[k][i + 1] = v.y;
                }
            }
        float factor = a.scale * kLog2e;
        if constexpr (Z::kNormed) {
            float top = 0.0f;
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int i = 0; i < XS; ++i) top = fmaxf(top, fabsf(x[k][i]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // 2^-e with 2^e <= top: exponents of both within fp32's normal range
            const uint32_t e = min(max(__float_as_uint(top) >> 23, 1u), 252u);
            const float down = __uint_as_float((254u - e) << 23);
            factor *= __uint_as_float(e << 23);
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int i = 0; i < XS; ++i) x[k][i] *= down;
        }
        // row oct's factor, to the lanes that hold column oct of a product
#pragma unroll
        for (int i = 0; i < 2; ++i) qscale[n][i] = __shfl_sync(0xffffffffu, factor, (quad * 2 + i) * 4);
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int p = 0; p < QP; ++p) {
                uint2 y;
                if constexpr (CT == MT_F32) {
                    if (p == 0) {
                        y = make_uint2(upper(x[k][0]), upper(x[k][1]));
                        x[k][0] -= __uint_as_float(y.x);
                        x[k][1] -= __uint_as_float(y.y);
                    } else {
                        y = make_uint2(__float_as_uint(x[k][0]), __float_as_uint(x[k][1]));
                    }
                } else {
                    y = make_uint2(pack<kBf16>(x[k][0], x[k][1]), pack<kBf16>(x[k][2], x[k][3]));
                    if (p + 1 < QP) {
                        const float2 g0 = unpack<kBf16>(y.x), g1 = unpack<kBf16>(y.y);
                        x[k][0] -= g0.x;
                        x[k][1] -= g0.y;
                        x[k][2] -= g1.x;
                        x[k][3] -= g1.y;
                    }
                }
                if constexpr (Z::kQReg) qf[k][n][p] = y;
                else sm_q[((k * NT + n) * QP + p) * 32 + lane] = y;  // read back by this lane alone
            }
    };
    auto take_queries = [&]() {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int dim = n * 8 + oct < rows ? a.cache.head_dim : 0;  // behind it: zeros
            if constexpr (Z::kQRaw) {
                // products read the rows themselves: zeros where nothing was copied
                for (int d = dim + quad; d < DP; d += 4) *(Q*)(sm_raw + q_place(n * 8 + oct, d)) = Q(0.0f);
                qscale[n][0] = qscale[n][1] = a.scale * kLog2e;
            } else {
                lay_out(n, dim);
            }
        }
    };
    auto query = [&](int k, int n, int p) {
        if constexpr (Z::kQReg) {
            return qf[k][n][p];
        } else if constexpr (Z::kQRaw) {
            // dims 16 k + quad * 2 and 8 more: pieces 2 k and 2 k + 1
            const unsigned char* const row = sm_raw + (n * 8 + oct) * Z::QROW + quad * 4;
            return make_uint2(*(const uint32_t*)(row + ((2 * k ^ oct) << 4)), *(const uint32_t*)(row + (((2 * k + 1) ^ oct) << 4)));
        } else {
            return sm_q[((k * NT + n) * QP + p) * 32 + lane];
        }
    };

    if (tiles > 0) ask_queries(in.b);
    copies_commit();
    if constexpr (kPadded)
        for (int s = 0; s < S; ++s) clear_padding(s);
    // the first tiles' pages are looked up together
    Step ahead[S];
#pragma unroll
    for (int s = 0; s < S; ++s)
        if (s < tiles) ahead[s] = look_up();
#pragma unroll
    for (int s = 0; s < S - 1; ++s) {
        if (s < tiles) {
            find_rows(ahead[s], s);
            fetch(s, kKeys);
            fetch(s, kValues);
        }
        copies_commit();
    }
    Step next = ahead[S - 1];

    // Sequences without tokens have no tiles: every range looks after some of them. Batches are padded
    // with many in a row; as a tile each they all came to one warp, 124 us in place of 86 for fp16, 146
    // sequences of 133 to 639 tokens and 36 without any, 16 heads of 128.
    for (int64_t b = range; b < a.batch; b += t.ranges.d)
        if (min(length_of(t, (int)b), a.max_tokens) <= 0) {
            for (int i = lane; i < rows * a.cache.head_dim; i += 32) {
                const int r = i / a.cache.head_dim, d = i - r * a.cache.head_dim;
                ((Q*)a.out)[b * a.out_seq + (int64_t)(head0 + r) * a.out_head + d] = Q(0.0f);
            }
            if (a.lse && lane < rows) a.lse[b * a.lse_seq + (int64_t)(head0 + lane) * a.lse_head] = -INFINITY;
        }

    // per query head: the largest score when the base was set, the base of the exponents (less the
    // offset), and the score above which it is set again
    float o[DP / 16][NT][4], m[NT][2], base[NT][2], limit[NT][2], l[NT][2];
    auto inverse = [](float power) { return __uint_as_float((254u << 23) - __float_as_uint(power)); };  // of a power of two
    // 8-bit caches: O, and the products of probabilities and scales, are in units of this power of two; scales
    // up to `roof` cannot take a product out of fp16's range
    float unit[NT][2], roof = 0.0f;
    int slot = 0, in_part = S;  // tiles of this part so far
    // O of a part's earlier tiles lies where the part's own is left at its end, each lane's accumulators, and
    // what they are relative to beside it. (Sequences taken whole, without a workspace, are shorter than kChain.)
    auto place_of = [&](int flags) { return (int64_t)me * 2 + (flags & kFromStart ? 1 : 0); };
    auto add_earlier = [&](int flags) {
        const float* const from = t.part_o + place_of(flags) * (ROWS * DP) + lane;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float2 then = t.part_ml[place_of(flags) * ROWS + n * 8 + quad * 2 + i];
                float by = exp2_fast(then.x - base[n][i]);
                if constexpr (kScaled) by *= then.y / unit[n][i];
#pragma unroll
                for (int d = 0; d < DP / 16; ++d)
#pragma unroll
                    for (int j = i; j < 4; j += 2) o[d][n][j] += from[((d * NT + n) * 4 + j) * 32] * by;
            }
    };
    auto leave = [&](int flags) {
        if (in_part > Z::kChain) add_earlier(flags);
        __syncwarp();
        float* const to = t.part_o + place_of(flags) * (ROWS * DP) + lane;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (oct == 0) t.part_ml[place_of(flags) * ROWS + n * 8 + quad * 2 + i] = make_float2(m[n][i] == -INFINITY ? -INFINITY : base[n][i], unit[n][i]);
#pragma unroll
                for (int d = 0; d < DP / 16; ++d)
#pragma unroll
                    for (int j = i; j < 4; j += 2) {
                        to[((d * NT + n) * 4 + j) * 32] = o[d][n][j];
                        o[d][n][j] = 0.0f;
                    }
            }
        __syncwarp();
    };
    for (int tile = 0; tile < tiles; ++tile) {
        __syncwarp();
        // the tile S - 1 ahead goes into the last one's stage
        const bool ask = tile + S - 1 < tiles;
        const int ask_slot = slot == 0 ? S - 1 : slot - 1;
        if (ask) {
            find_rows(next, ask_slot);
            fetch(ask_slot, kKeys);
            if constexpr (!Z::kTwoBursts) fetch(ask_slot, kValues);
            if (left > 0) next = look_up();
        } else {
            asm volatile("griddepcontrol.launch_dependents;");
        }
        const int4 meta = sm_meta[slot];
        ++in_part;
        if (meta.y & kFirst) {
            // the part's queries, while its tiles are on their way: the first part's are the oldest copy;
            // another's were asked for when the last part began, and have been waited for if that is
            // S tiles ago
            if (Z::kQRaw && tile > 0) ask_queries(meta.x);
            if (tile == 0) copies_wait<S - 1>();
            else if (Z::kQRaw || in_part <= S) copies_wait_all();
            __syncwarp();
            take_queries();
            __syncwarp();
            if (!Z::kQRaw && (meta.y & kMore)) ask_queries(meta.w);
            in_part = 1;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    m[n][i] = limit[n][i] = -INFINITY;
                    base[n][i] = -Z::kOffset;
                    l[n][i] = 0.0f;
                    unit[n][i] = Z::kLeastUnit;
                }
            roof = 0.0f;
#pragma unroll
            for (int d = 0; d < DP / 16; ++d)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[d][n][i] = 0.0f;
        }
        copies_wait<S - 2>();  // this turn's are not committed yet
        __syncwarp();
        const uint32_t mask = (uint32_t)meta.z;
        unsigned char* const stage = ring + slot * Z::STAGE;
        const uint32_t k_at = smem_address(stage), v_at = k_at + TW * Z::ROW;
        if (Z::kTwoBursts && ask && !mask) fetch(ask_slot, kValues);
        if (mask) {
            // S^T: s[.][.][0], [1] are token oct, heads quad * 2 + 0, 1; [2], [3] token oct + 8. The
            // largest pieces' products go into `part` first where they are kept apart, and those of smaller
            // ones into `small`: added to s each, they would be truncated to its steps.
            float s[TB][NT][4];
#pragma unroll
            for (int b = 0; b < TB; ++b) {
                // where they are not, `part` takes every second step: two short chains of products
                float part[NT][4], small[NT][4];
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[b][n][i] = part[n][i] = small[n][i] = 0.0f;
                auto times_queries = [&](int k, const uint32_t (&x)[4]) {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int p = 0; p < QP; ++p) {
                            const uint2 q = query(k, n, p);
                            product<CT>(Z::kExact ? p == 0 ? part[n] : small[n] : k % 2 == 1 ? part[n] : s[b][n], x, q.x, q.y);
                        }
                    if constexpr (Z::kExact) {
                        if (k % 4 == 3 || (!kPadded && k == KS - 1)) {
#pragma unroll
                            for (int n = 0; n < NT; ++n)
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    s[b][n][i] += part[n][i];
                                    part[n][i] = 0.0f;
                                }
                        }
                    }
                };
#pragma unroll
                for (int c = 0; c < CPR / 2; ++c) {
                    if (kPadded && Z::may_end(c) && 2 * c >= row_chunks) break;
                    uint32_t r[4];
                    load_matrices(r, k_at + swizzled<CPR>(b * 16 + (lane & 15), 2 * c + (lane >> 4)) * 16);
                    if constexpr (CT == MT_F32) {
                        uint32_t hi[4], lo[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            hi[i] = upper(__uint_as_float(r[i]));
                            lo[i] = __float_as_uint(__uint_as_float(r[i]) - __uint_as_float(hi[i]));
                        }
                        times_queries(c, hi);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            const uint2 q = query(c, n, 0);
                            product<CT>(small[n], lo, q.x, q.y);
                        }
                    } else if constexpr (kScaled) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            uint32_t x[4];
                            decode<CT, true>(r[2 * h], x[0], x[2]);
                            decode<CT, true>(r[2 * h + 1], x[1], x[3]);
                            times_queries(2 * c + h, x);
                        }
                    } else {
                        times_queries(c, r);
                    }
                }
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if constexpr (!Z::kExact || kPadded) s[b][n][i] += part[n][i];
                        // of an infinite key the largest pieces alone make the score: what is left of an infinity is NaN
                        if constexpr (Z::kExact && (QP > 1 || CT == MT_F32))
                            if (fabsf(s[b][n][i]) != INFINITY) s[b][n][i] += small[n][i];
                    }
            }
            if constexpr (kScaled) {
                const float* z = (const float*)(stage + 2 * TW * Z::ROW);
#pragma unroll
                for (int b = 0; b < TB; ++b)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float ks = z[b * 16 + h * 8 + oct];
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            s[b][n][2 * h] *= ks;
                            s[b][n][2 * h + 1] *= ks;
                        }
                    }
            }
            if (mask != kAll) {
#pragma unroll
                for (int b = 0; b < TB; ++b)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (!(mask >> (b * 16 + (i >> 1) * 8 + oct) & 1)) s[b][n][i] = -INFINITY;
            }
            float vs[TB][2], keep[NT][2], most_v = 0.0f;
            bool grown = false;
            if constexpr (kScaled) {
                const float* z = (const float*)(stage + 2 * TW * Z::ROW) + 32;
#pragma unroll
                for (int b = 0; b < TB; ++b)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        vs[b][h] = z[b * 16 + h * 8 + oct];
                        most_v = fmaxf(most_v, fabsf(vs[b][h]));
                    }
                grown = most_v > roof;
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float top = -INFINITY;
#pragma unroll
                    for (int b = 0; b < TB; ++b) top = fmaxf(top, fmaxf(s[b][n][i], s[b][n][2 + i]));
                    grown |= top > limit[n][i];
                    keep[n][i] = 1.0f;
                }
            // scores are compared and kept as the products give them; qscale turns them into exponents
            const bool rescale = __any_sync(0xffffffffu, grown);
            if (rescale) {
                if constexpr (kScaled)
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) most_v = fmaxf(most_v, __shfl_xor_sync(0xffffffffu, most_v, d));
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float top = m[n][i];
#pragma unroll
                        for (int b = 0; b < TB; ++b) top = fmaxf(top, fmaxf(s[b][n][i], s[b][n][2 + i]));
#pragma unroll
                        for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                        const float now = top == -INFINITY ? 0.0f : top * qscale[n][i];
                        const float k = m[n][i] == -INFINITY ? 0.0f : exp2_fast((base[n][i] + Z::kOffset) - now);
                        m[n][i] = top;
                        base[n][i] = now - Z::kOffset;
                        // (with the division that rounds to nearest 1 sequence of 100 tokens, int8, takes 9.4 us, so 8.4)
                        limit[n][i] = top == -INFINITY ? top : top + __fdividef(Z::kSlack, qscale[n][i]);
                        l[n][i] *= k;
                        keep[n][i] = k;
                    }
            }
            if (Z::kTwoBursts && ask) fetch(ask_slot, kValues);
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int b = 0; b < TB; ++b)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            float& x = s[b][n][2 * h + i];
                            x = exp2_fast(fmaf(x, qscale[n][i], -base[n][i]));
                            l[n][i] += x;
                        }
            if constexpr (kScaled) {
#pragma unroll
                for (int b = 0; b < TB; ++b)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[b][n][i] *= vs[b][i >> 1];
                if (rescale) {
                    // the next power of two
                    auto above = [](float x) { return __uint_as_float((min(__float_as_uint(x) >> 23, 252u) + 1) << 23); };
                    roof = INFINITY;
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            float most = 0.0f;
#pragma unroll
                            for (int b = 0; b < TB; ++b) most = fmaxf(most, fmaxf(fabsf(s[b][n][i]), fabsf(s[b][n][2 + i])));
#pragma unroll
                            for (int d = 4; d < 32; d <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
                            // (a unit that is much smaller than before could take O out of fp32's range)
                            const float before = __uint_as_float(__float_as_uint(unit[n][i] * keep[n][i]) & 0xff800000u);
                            const float now = fmaxf(fmaxf(above(most), fminf(above(most_v), above(most) * Z::kSpread)) * 0x1p-11f,
                                                    fmaxf(before, Z::kLeastUnit));
                            if (keep[n][i] > 0.0f) keep[n][i] *= unit[n][i] * inverse(now);
                            unit[n][i] = now;
                            roof = fminf(roof, now * 0x1p11f);
                        }
                }
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float per = inverse(unit[n][i & 1]);
#pragma unroll
                        for (int b = 0; b < TB; ++b) s[b][n][i] *= per;
                    }
            }
            if constexpr (!Z::kExact) {
                if (rescale) {
#pragma unroll
                    for (int d = 0; d < DP / 16; ++d)
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int i = 0; i < 4; ++i) o[d][n][i] *= keep[n][i & 1];
                }
            }
            uint32_t pf[TB][NT][2 * PP];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int b = 0; b < TB; ++b) {
                    if constexpr (CT == MT_F32) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const uint32_t x = __float_as_uint(s[b][n][2 * h]), y = __float_as_uint(s[b][n][2 * h + 1]);
                            const uint32_t low = transpose8x8(__byte_perm(x, y, 0x5410)), high = transpose8x8(__byte_perm(x, y, 0x7632));
                            pf[b][n][2 * h] = __byte_perm(low, high, 0x5410);
                            pf[b][n][2 * h + 1] = __byte_perm(low, high, 0x7632);
                        }
                    } else {
#pragma unroll
                        for (int p = 0; p < PP; ++p)
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const uint32_t y = pack<kBf16>(s[b][n][2 * h], s[b][n][2 * h + 1]);
                                pf[b][n][2 * p + h] = transpose8x8(y);
                                if (p + 1 < PP) {
                                    const float2 g = unpack<kBf16>(y);
                                    s[b][n][2 * h] -= g.x;
                                    s[b][n][2 * h + 1] -= g.y;
                                }
                            }
                    }
                }
            }
            // O^T: rows are 16 dims, columns heads as above. Where chains are kept short, a tile's
            // product is added to the rescaled O.
            auto add_up = [&](int d, int n, const float (&x)[4]) {
#pragma unroll
                for (int i = 0; i < 4; ++i) o[d][n][i] = o[d][n][i] * keep[n][i & 1] + x[i];
            };
            if constexpr (CT == MT_F32) {
                const float* v = (const float*)(stage + TW * Z::ROW);
#pragma unroll
                for (int d = 0; d < DP / 16; ++d) {
                    if (kPadded && Z::may_end(2 * d) && 4 * d >= row_chunks) break;
                    float tile_o[NT][4] = {};
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        // operand column j is token 8 h + 2 j, column j + 4 the one after: free of bank
                        // conflicts, and the order in which the probabilities lie
                        uint32_t hi[4], lo[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int token = 8 * h + 2 * quad + (i >> 1), dim = 16 * d + oct + 8 * (i & 1);
                            const float x = v[swizzled<CPR>(token, dim >> 2) * 4 + (dim & 3)];
                            hi[i] = upper(x);
                            lo[i] = __float_as_uint(x - __uint_as_float(hi[i]));
                        }
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            const float p0 = __uint_as_float(pf[0][n][2 * h]), p1 = __uint_as_float(pf[0][n][2 * h + 1]);
                            const uint32_t h0 = upper(p0), h1 = upper(p1);
                            product<CT>(tile_o[n], lo, h0, h1);
                            product<CT>(tile_o[n], hi, __float_as_uint(p0 - __uint_as_float(h0)),
                                        __float_as_uint(p1 - __uint_as_float(h1)));
                            product<CT>(tile_o[n], hi, h0, h1);
                        }
                    }
#pragma unroll
                    for (int n = 0; n < NT; ++n) add_up(d, n, tile_o[n]);
                }
            } else {
                // 16 dims of 16-bit rows are two pieces, of 8-bit ones one
#pragma unroll
                for (int c = 0; c < CPR / 2; ++c) {
                    if (kPadded && Z::may_end(c) && 2 * c >= row_chunks) break;
                    uint32_t r[TB][4];
#pragma unroll
                    for (int b = 0; b < TB; ++b)
                        load_transposed(r[b], kScaled ? v_at + swizzled<CPR>(b * 16 + (lane & 15), 2 * c + (lane >> 4)) * 16
                                                      : v_at + swizzled<CPR>((lane & 7) + (lane >> 4) * 8, 2 * c + (lane >> 3 & 1)) * 16);
#pragma unroll
                    for (int h = 0; h < (kScaled ? 2 : 1); ++h) {
                        const int d = kScaled ? 2 * c + h : c;
                        float tile_o[NT][4] = {};
#pragma unroll
                        for (int b = 0; b < TB; ++b) {
                            // 8 bits: bytes 0, 2 are two tokens' even dim, bytes 1, 3 their odd one
                            uint32_t x[4];
                            if constexpr (kScaled) {
                                decode<CT, false>(r[b][2 * h], x[0], x[1]);
                                decode<CT, false>(r[b][2 * h + 1], x[2], x[3]);
                            } else {
#pragma unroll
                                for (int i = 0; i < 4; ++i) x[i] = r[b][i];
                            }
#pragma unroll
                            for (int n = 0; n < NT; ++n)
#pragma unroll
                                for (int p = PP - 1; p >= 0; --p)
                                    product<CT>(Z::kExact ? tile_o[n] : o[d][n], x, pf[b][n][2 * p], pf[b][n][2 * p + 1]);
                        }
                        if constexpr (Z::kExact)
#pragma unroll
                            for (int n = 0; n < NT; ++n) add_up(d, n, tile_o[n]);
                    }
                }
            }
        }
        copies_commit();
        if (!Z::kExact && in_part % Z::kChain == 0 && !(meta.y & kLast)) leave(meta.y);
        if (meta.y & kLast) {
            if (!Z::kExact && in_part > Z::kChain) add_earlier(meta.y);
            // -- the part ends: from the accumulators' layout to rows by way of this tile's stage, into which
            // nothing will be fetched before the next tile
            __syncwarp();
            const int dim = a.cache.head_dim;
            const bool whole = (meta.y & kFromStart) && (meta.y & kEnds);
            const int64_t part = (int64_t)me * 2 + (meta.y & kFromStart ? 1 : 0);
            Q* const out = (Q*)a.out + (int64_t)meta.x * a.out_seq + (int64_t)head0 * a.out_head;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                if (n * 8 >= rows) break;
                float* const mine = (float*)stage;  // [8][DP]
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float sum = l[n][i];
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
                    const bool none = m[n][i] == -INFINITY && sum == 0.0f;
                    // what sums are relative to, as an exponent
                    const float exponent = m[n][i] == -INFINITY ? -INFINITY : base[n][i];
                    const int r = quad * 2 + i, row = n * 8 + r;
                    float f = !whole ? 1.0f : none ? 0.0f : 1.0f / sum;
                    if constexpr (kScaled) f *= unit[n][i];
#pragma unroll
                    for (int d = 0; d < DP / 16; ++d) {
                        const int d0 = 16 * d + (kScaled ? 2 * oct : oct), d1 = d0 + (kScaled ? 1 : 8);
                        mine[r * DP + (d0 ^ quad * 8)] = o[d][n][i] * f;
                        mine[r * DP + (d1 ^ quad * 8)] = o[d][n][2 + i] * f;
                    }
                    if (oct == 0 && row < rows) {
                        if (!whole)
                            t.part_ml[part * ROWS + row] = make_float2(exponent, sum);
                        else if (a.lse)
                            a.lse[(int64_t)meta.x * a.lse_seq + (int64_t)(head0 + row) * a.lse_head] =
                                (exponent + log2f(sum)) * kLn2;
                    }
                }
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 8 * DP / 128; ++i) {
                    const int r = (i * 32 + lane) / (DP / 4), d = (i * 32 + lane) % (DP / 4) * 4;
                    if (n * 8 + r < rows) {
                        const float4 y = *(const float4*)(mine + r * DP + (d ^ (r >> 1) * 8));
                        if (!whole) {
                            *(float4*)(t.part_o + (part * ROWS + n * 8 + r) * DP + d) = y;
                        } else if (d < dim) {
                            Q* const to = out + (int64_t)(n * 8 + r) * a.out_head + d;
                            if (t.out_quads) {
                                store4(to, y);
                            } else {
                                to[0] = rounded<Q>(y.x);
                                if (d + 1 < dim) to[1] = rounded<Q>(y.y);
                                if (d + 2 < dim) to[2] = rounded<Q>(y.z);
                                if (d + 3 < dim) to[3] = rounded<Q>(y.w);
                            }
                        }
                    }
                }
                __syncwarp();
            }
            if constexpr (kPadded) clear_padding(slot);
        }
        if (++slot == S) slot = 0;
    }
    copies_wait_all();
}

// Joins the parts of sequences that cuts crossed: block (x, y) the rows y * together .. of an
// item whose tiles lie in several ranges. Which ones is known from the lengths, so it is
// found out while attention_tiles still runs. x / items is a sequence, or, where there are
// fewer ranges than sequences, a range: it stands for the sequence that it starts in the
// middle of, if that ends in it. A block is teams of `lanes` threads, 4 dims each: all of DP, or,
// for long chains of few rows, a slice of it (blockIdx.z), which leaves more teams. They take
// `together` rows at a time, and of each row every teams / together-th part (all powers of two).
// 1 sequence of 30000 tokens, 1 head of 256, 888 parts: 17 us, 47 with 8 teams of whole rows.
constexpr int kLeastLanes = 8;

template <class Q, int DP, int ROWS, int TW>
__global__ void __launch_bounds__(DP * 2) join_parts(const __grid_constant__ TileArgs t, int by_sequence, int together, int lanes) {
    constexpr int kThreads = DP * 2;
    __shared__ float4 sm_o[kThreads];
    __shared__ float2 sm_ml[kThreads / kLeastLanes];
    const AttentionArgs& a = t.a;
    asm volatile("griddepcontrol.launch_dependents;");
    uint32_t item, row_block;
    const int x = (int)t.per_range.div(blockIdx.x, &item);
    const int head0 = (int)t.row_blocks.div(item, &row_block) * a.group + (int)row_block * ROWS;
    const int rows = min(ROWS, a.group - (int)row_block * ROWS);
    const int lane = threadIdx.x % lanes, team = threadIdx.x / lanes, teams = kThreads / lanes;
    const int side = team / together, sides = teams / together, r = blockIdx.y * together + team % together;
    const int d0 = (blockIdx.z * lanes + lane) * 4;
    int b, first = 0, count = 0;  // count: parts to join, none or several
    Cursor c;
    const Cuts<TW> cuts(t);
    if (by_sequence) {
        b = x;
        const int begin = cuts.before(b), tiles = cuts.tiles_of(b, c);
        if (tiles > 0) {
            first = cuts.owner(begin);
            count = cuts.owner(begin + tiles - 1) - first + 1;
        }
    } else {
        const int tiles = cuts.locate(x, c);
        b = c.b;
        if (tiles > 0 && c.tile > 0 && c.tiles - c.tile <= tiles) {
            first = cuts.owner(cuts.first(x) - c.tile);
            count = x - first + 1;
        }
    }
    // every block waits, those without work too: what comes after this kernel waits for it alone
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (count <= 1) return;
    // every team takes every sides-th part, four at a time
    float m = -INFINITY, l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    auto take = [&](float2 ml, float4 y) {
        const float top = fmaxf(m, ml.x), base = top == -INFINITY ? 0.0f : top;
        const float keep = exp2_fast(m - base), f = exp2_fast(ml.x - base);
        // NaN scores leave m at -inf and l, o NaN: 0 * NaN passes them on
        m = top;
        l = l * keep + ml.y * f;
        o.x = o.x * keep + y.x * f;
        o.y = o.y * keep + y.y * f;
        o.z = o.z * keep + y.z * f;
        o.w = o.w * keep + y.w * f;
    };
    if (r < rows)
        for (int i = side; i < count; i += 4 * sides) {
            float2 ml[4];
            float4 y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int part = i + j * sides;
                if (part < count) {
                    const int64_t row = (((int64_t)(first + part) * t.items + item) * 2 + (part == 0 ? 1 : 0)) * ROWS + r;
                    ml[j] = t.part_ml[row];
                    y[j] = *(const float4*)(t.part_o + row * DP + d0);
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (i + j * sides < count) take(ml[j], y[j]);
        }
    for (int half = sides / 2; half > 0; half /= 2) {
        // the upper half of a row's teams hands over to the lower one, each in a place of its own, which no
        // later turn writes
        if (side >= half && side < 2 * half) {
            sm_o[threadIdx.x] = o;
            if (lane == 0) sm_ml[team] = make_float2(m, l);
        }
        __syncthreads();
        if (side < half) take(sm_ml[team + half * together], sm_o[threadIdx.x + half * together * lanes]);
    }
    if (side != 0 || r >= rows) return;
    const bool none = m == -INFINITY && l == 0.0f;
    const float per = 1.0f / l;
    const float y[4] = {o.x, o.y, o.z, o.w};
    Q* out = (Q*)a.out + (int64_t)b * a.out_seq + (int64_t)(head0 + r) * a.out_head + d0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (d0 + i < a.cache.head_dim) out[i] = rounded<Q>(none ? 0.0f : y[i] * per);
    if (d0 == 0 && a.lse) a.lse[(int64_t)b * a.lse_seq + (int64_t)(head0 + r) * a.lse_head] = (m + log2f(l)) * kLn2;
}

// ---- launch ------------------------------------------------------------------------------------

constexpr int kMaxDevices = 16;

template <int CT, class Q, int DP, int NT>
int launch(const AttentionArgs& a, bool run, void* workspace, uint64_t* bytes, int dev, cudaStream_t st) {
    using Z = Shape<CT, Q, DP, NT>;
    TileArgs t;
    t.a = a;
    const int row_blocks = (a.group + Z::ROWS - 1) / Z::ROWS;
    t.row_blocks = FastDiv((uint32_t)row_blocks);
    t.items = a.cache.kv_heads * row_blocks;
    t.per_range = FastDiv((uint32_t)t.items);
    t.row_chunks = a.cache.head_dim * Z::EB / 16;
    const int64_t q16 = 16 / (int)sizeof(Q);
    t.q_chunks = a.cache.head_dim % q16 == 0 && (uintptr_t)a.q % 16 == 0 && a.q_seq % q16 == 0 && a.q_head % q16 == 0
                     ? (int)(a.cache.head_dim / q16) : 0;
    t.out_quads = a.cache.head_dim % 4 == 0 && (uintptr_t)a.out % (4 * sizeof(Q)) == 0 && a.out_seq % 4 == 0 && a.out_head % 4 == 0;
    int sms;
    if (int rc = sm_count(dev, &sms)) return rc;
    const int64_t tokens = a.max_tokens < a.window ? a.max_tokens : a.window;
    const int64_t most = tokens > 0 ? (tokens + Z::TW - 1) / Z::TW : 1;
    if (a.batch * most > INT32_MAX || (int64_t)a.batch * t.items > INT32_MAX - 64)
        return bad_argument("paged_attention: the tables' width allows over 2^31 - 1 tiles of %d tokens", Z::TW);
    // A range a sequence where none has more than a few tiles: that costs less than a join. The more
    // so, the more of the warps that fit the GPU at once the sequences occupy: then a join has many
    // parts, and cutting gives each warp less to gain. Long tiles make up for a join sooner. us, whole
    // and cut: bf16, 8 heads of 128, 1 sequence of 4 tiles 8.3, 7.6; 40 sequences (a quarter of the
    // warps) of 6 tiles 10.4, 11.6, of 12 tiles 16.5, 13.1; 110 (three quarters) of 16 tiles 22.9,
    // 29.3 (of 1 to 16 tiles 21.4, 23.8); fp32, 8 heads of 256, 8 sequences of 2 tiles 17.2, 16.0, of 4 tiles 28.1, 15.8.
    // (Tables that are wider than the sequences hide short ones: those are cut.)
    // Otherwise as many ranges as those warps can take the heads of, or fewer where there cannot be as
    // many tiles.
    const int64_t resident = (int64_t)sms * Z::BLOCKS * Z::NW, used = (int64_t)a.batch * t.items;
    constexpr int kTile = Z::TW * DP * (Z::EB == 4 ? 2 : 1), kFew = kTile <= 1024 ? 4 : kTile <= 2048 ? 3 : kTile <= 4096 ? 2 : 1;
    constexpr int kMore = Z::EB == 4 || Z::TW == 32 ? 5 : 15;
    const double share = used <= resident ? (double)used / (double)resident : 0.0;
    t.whole = (double)most <= kFew + kMore * share * (1.0 + share);
    static_assert(kFew + 2 * kMore < Z::kChain, "whole sequences have no workspace");
    int64_t ranges = resident / t.items;
    if (ranges < 1) ranges = 1;
    if (ranges > a.batch * most) ranges = a.batch * most;
    if (t.whole) ranges = a.batch;
    const int64_t warps = ranges * t.items;
    const uint64_t ml_bytes = (uint64_t)warps * 2 * Z::ROWS * 8;
    *bytes = t.whole ? 0 : ml_bytes + (uint64_t)warps * 2 * Z::ROWS * DP * 4;
    if (!run) return 0;
    t.ranges = FastDiv((uint32_t)ranges);
    t.part_ml = (float2*)workspace;
    t.part_o = (float*)((char*)workspace + ml_bytes);
    auto kernel = t.row_chunks < Z::CPR ? attention_tiles<CT, Q, DP, NT, true> : attention_tiles<CT, Q, DP, NT, false>;
    static std::atomic<bool> ready[2][kMaxDevices];  // calls of several threads may come first at once
    std::atomic<bool>& is_ready = ready[t.row_chunks < Z::CPR][dev];
    if (!is_ready) {
        RT_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Z::SMEM));
        is_ready = true;
    }
    // warps of whole sequences are spread over the SMs, where one block fits them at a time
    const int64_t spread = (warps + sms - 1) / sms;
    const int per_block = t.whole && Z::BLOCKS == 1 && spread < Z::NW ? (int)spread : Z::NW;
    RT_CHECK(launch_early(kernel, dim3((unsigned)((warps + per_block - 1) / per_block)), dim3(per_block * 32), per_block * Z::WARP, st, t));
    if (t.whole) return 0;
    const bool by_sequence = a.batch <= ranges;
    // long chains of few items: a block a row; short ones of many: rows together, so that the
    // blocks fit the GPU about once
    const int64_t joined = (by_sequence ? a.batch : ranges) * t.items, rows = a.group < Z::ROWS ? a.group : Z::ROWS;
    int together = 1, lanes = DP / 4;
    while (together < 8 && joined * ((rows + together - 1) / together) > (int64_t)sms * 4) together *= 2;
    // rows in slices while each team has more than one turn of 4 parts (as many as the ranges make on average)
    const int64_t parts = by_sequence ? ranges / a.batch : 2;
    while (together == 1 && lanes > kLeastLanes && parts > DP * 2 / lanes * 4 && joined * rows * (DP / 4 / lanes) < (int64_t)sms * 2) lanes /= 2;
    RT_CHECK(launch_early(join_parts<Q, DP, Z::ROWS, Z::TW>,
                          dim3((unsigned)joined, (unsigned)((rows + together - 1) / together), (unsigned)(DP / 4 / lanes)), dim3(DP * 2), 0, st, t,
                          (int)by_sequence, together, lanes));
    return 0;
}

// Over 8 query heads a key-value head: 16 of them a warp, or 8, so that neighbouring warps read the
// same rows, which one of them finds in L2. 16 halve what the SMs read, and a warp then has fewer
// registers left and twice as much to hand over; they win where a warp has many tiles (as far as
// the tables' width tells). us by sixteens and by eights: bf16, 2 heads of 128, 32 query heads, 16 sequences of
// 2048 tokens (4 tiles a warp) 21.3, 17.2; of 8192 (14) 40.0, 38.5; of 16384 (28) 58.6, 67.1; 64 of
// 32768 (221) 326, 465. fp16, 1 head of 256: 7 of 16384 (12) 50.6, 36.8; 32 of 16384 (55) 120, 122.
// 16 heads of the widest rows leave too few registers where elements are not 16 bits: fp32 over 64 dims 426,
// 392 at 110 tiles a warp; int8 over 128, float32 queries, 32 of 16384 of 256 dims 178, 142, bfloat16 134, 121.
template <int CT, class Q, int DP>
int by_group(const AttentionArgs& a, bool run, void* workspace, uint64_t* bytes, int dev, cudaStream_t st) {
    using Z = Shape<CT, Q, DP, 2>;
    if constexpr (Z::EB == 2 || DP <= (Z::EB == 4 ? 64 : 128)) {
        int sms;
        if (int rc = sm_count(dev, &sms)) return rc;
        const int64_t tiles = (a.max_tokens < a.window ? a.max_tokens : a.window) / Z::TW;
        const int64_t lines = (int64_t)a.cache.kv_heads * ((a.group + Z::ROWS - 1) / Z::ROWS);
        if (a.group > 8 && a.batch * lines * tiles >= 20LL * sms * Z::BLOCKS * Z::NW)
            return launch<CT, Q, DP, 2>(a, run, workspace, bytes, dev, st);
    }
    return launch<CT, Q, DP, 1>(a, run, workspace, bytes, dev, st);
}

template <int CT, class Q> int by_shape(const AttentionArgs& a, bool run, void* workspace, uint64_t* bytes, int dev, cudaStream_t st) {
    const int dim = a.cache.head_dim;
    // (bf16 heads of 32, 8 of them, 16 sequences of 4096 tokens: 20 us, 33 as half of 64)
    if (dim <= 32) return by_group<CT, Q, 32>(a, run, workspace, bytes, dev, st);
    if (dim <= 64) return by_group<CT, Q, 64>(a, run, workspace, bytes, dev, st);
    if (dim <= 128) return by_group<CT, Q, 128>(a, run, workspace, bytes, dev, st);
    return by_group<CT, Q, 256>(a, run, workspace, bytes, dev, st);
}

}  // namespace tiles
}  // namespace mt
