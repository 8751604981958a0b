// Paged attention of one token per sequence in tiles of 16 tokens a warp.
//
// For each sequence and key-value head: S^T = K Q^T (16 tokens x 8 query heads), the
// softmax over the tokens in one pass (running maximum m, l = sum exp2(s - m), O = sum
// exp2(s - m) v, rescaled when m grows), and O^T += V^T P^T. What bounds it is HBM: K and V
// are read once and used by one token's query heads only (2 flops a query head for each
// element), so everything here serves the loads:
//
// * The tokens are the rows (M) of the matrix instructions and the query heads their 8
//   columns: a group of 4 or 8 query heads wastes little of them, and 16 columns (NT = 2)
//   serve larger groups. K's fragments come by ldmatrix, V's by its transposing form; S^T's
//   accumulators become P^T's operands by transposing 8 x 8 blocks in registers.
// * Each warp streams its own 16 of a unit's tokens through a ring of S stages in shared
//   memory (16-byte asynchronous copies, page by page), so no barrier stands between a
//   copy and its use; warps meet only where a head's part ends.
// * Units (64 tokens of one sequence and head) of all sequences lie on one line that is
//   cut into equal ranges, one a block: a ragged batch or one long sequence keeps every SM
//   at work. A head that a cut crosses leaves parts (m, l, O) in the workspace, and a second
//   kernel joins them; it is launched early and waits for the first on the device.
//
// 8-bit codes become fp16 in registers, exactly; K's scales multiply the scores, V's the
// probabilities. 32-bit queries (and 32-bit caches) are split into pieces whose products
// together keep at least 22 bits.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "mt_paged_attention.h"

namespace mt {
namespace tiles {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct TileArgs {
    AttentionArgs a;
    int items;       // per sequence: kv_heads * row blocks
    int row_blocks;  // blocks of NT * 8 query heads in a group
    int row_chunks;  // 16-byte pieces of a cache row
    // workspace: two parts a block, (m, l) and O of NT * 8 rows each, and what they are of
    int4* meta;
    float2* part_ml;
    float* part_o;
};

// What a block's first part is (meta[block].z), for the join.
enum { kNoPart = 0, kMiddle = 1, kEnd = 2, kIdle = 3 };

// ---- instructions ------------------------------------------------------------------------

__device__ inline uint32_t smem_address(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ inline void copy16(uint32_t dst, const void* src, bool really) {
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(really ? 16 : 0));
}
__device__ inline void copy4(uint32_t dst, const void* src, bool really) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(really ? 4 : 0));
}
__device__ inline void copies_commit() { asm volatile("cp.async.commit_group;"); }
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

// Two codes (bytes lo_byte and hi_byte of x) as fp16, exactly.
template <int CT, int kLo, int kHi> __device__ inline uint32_t decode(uint32_t x) {
    if constexpr (CT == MT_I8) {
        // 0x6400 | u is 1024 + u; with u = code + 128, 1152 more than the code
        const uint32_t u = __byte_perm(x ^ 0x80808080u, 0x64646464u, kLo | 0x40 | kHi << 8 | 0x4000);
        const __half2 v = __hsub2(reinterpret_cast<const __half2&>(u), __half2half2(__ushort_as_half(0x6480)));
        return reinterpret_cast<const uint32_t&>(v);
    } else {
        const uint32_t two = __byte_perm(x, 0, kLo | kHi << 4);
        uint32_t v;
        asm("{ .reg .b16 h, l; mov.b32 {l, h}, %1; cvt.rn.f16x2.e4m3x2 %0, l; }" : "=r"(v) : "r"(two));
        return v;
    }
}

// ---- shapes --------------------------------------------------------------------------------

template <int CT, bool kQ32, int DP, int NT> struct Shape {
    static constexpr int EB = CT == MT_F32 ? 4 : CT == MT_F16 || CT == MT_BF16 ? 2 : 1;
    static constexpr bool kScaled = EB == 1, kBf16 = CT == MT_BF16;
    // The matrix pipe truncates what it adds to an accumulator, so a long chain of products
    // drifts. For 32-bit outputs chains are short (4 steps of a score, 16 tokens of O) and
    // are added up in fp32, rounded to nearest.
    static constexpr bool kExact = kQ32;
    static constexpr int ROW = DP * EB;               // bytes of a (padded) cache row
    static constexpr int CPR = ROW / 16;              // its 16-byte pieces
    static constexpr int NW = ROW >= 1024 ? 2 : 4;    // warps a block
    static constexpr int KT = 16 * NW;                // tokens a unit
    static constexpr int STAGE = 32 * ROW + (kScaled ? 128 : 0);  // 16 rows of K, of V, their scales
    static constexpr int S = ROW <= 128 ? 4 : 3;      // stages
    static constexpr int KS = CT == MT_F32 ? DP / 8 : DP / 16;    // steps of K Q^T
    // pieces of a query: fp16 11 bits, bf16 8 bits, tf32 11 bits each
    static constexpr int QP = CT == MT_F32 ? 2 : !kQ32 ? 1 : kBf16 ? 3 : 2;
    // queries that fp16 may not hold are divided by a power of two per row
    static constexpr bool kNormed = CT != MT_F32 && !kBf16 && (kQ32 || kScaled);
    // fp16 probabilities are held times 2^15: the smallest, 2^-24, is 2^-39 of the largest
    static constexpr float kOffset = CT == MT_F16 || kScaled ? 15.0f : 0.0f;
    static constexpr bool kQReg = KS * 2 * NT * QP <= 64;         // queries in registers, else in shared memory
    static constexpr int ROWS = NT * 8;
    static constexpr int Q_BYTES = KS * NT * QP * 256;
    static constexpr int SMALL = NW * S * 16 + NW * ROWS * 8 + ROWS * 4 + 64;
    static constexpr int SMEM = NW * S * STAGE + Q_BYTES + SMALL;
    static constexpr int kFit = 227 * 1024 / (SMEM + 1024);
    static constexpr int BLOCKS = kFit > 4 ? 4 : kFit < 1 ? 1 : kFit;  // resident blocks an SM
};

// Where 16-byte piece c of row r lies, so that 8 rows' pieces of one column fall in
// different banks.
template <int CPR> __device__ inline int swizzled(int r, int c) {
    if constexpr (CPR >= 8) return r * CPR + (c ^ (r & 7));
    else return r * CPR + (c ^ (r / (8 / CPR) & (CPR - 1)));
}

// Where a block is on the line of units.
struct Cursor {
    int b, begin, end, tiles, item, tile, next_length;
};

template <int KT> __device__ inline void enter_sequence(Cursor& c, const TileArgs& t, int length) {
    const int n = min(max(length, 0), t.a.max_tokens);
    c.end = n;
    c.begin = n > t.a.window ? n - t.a.window : 0;
    c.tiles = max(1, (n - c.begin + KT - 1) / KT);  // a sequence without tokens has one empty unit
    c.next_length = c.b + 1 < t.a.batch ? t.a.lengths[(int64_t)(c.b + 1) * t.a.length_seq] : 0;
}

template <int CT, class Q, int DP, int NT>
__global__ void __launch_bounds__(Shape<CT, sizeof(Q) == 4, DP, NT>::NW * 32, Shape<CT, sizeof(Q) == 4, DP, NT>::BLOCKS)
attention_tiles(const __grid_constant__ TileArgs t) {
    using Z = Shape<CT, sizeof(Q) == 4, DP, NT>;
    constexpr int NW = Z::NW, KT = Z::KT, S = Z::S, CPR = Z::CPR, ROWS = Z::ROWS, QP = Z::QP, KS = Z::KS;
    constexpr bool kScaled = Z::kScaled, kBf16 = Z::kBf16;
    extern __shared__ __align__(128) unsigned char smem[];
    const AttentionArgs& a = t.a;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, quad = lane & 3, oct = lane >> 2;

    unsigned char* const ring = smem + warp * (S * Z::STAGE);
    uint2* const sm_q = (uint2*)(smem + NW * S * Z::STAGE);
    int4* const sm_meta = (int4*)((unsigned char*)sm_q + Z::Q_BYTES) + warp * S;
    float2* const sm_ml = (float2*)((unsigned char*)sm_q + Z::Q_BYTES + NW * S * 16);  // [NW][ROWS]
    float* const sm_qscale = (float*)(sm_ml + NW * ROWS);
    int64_t* const sm_start = (int64_t*)(sm_qscale + ROWS);  // total, prefix, sequence

    asm volatile("griddepcontrol.launch_dependents;");

    // -- this block's range of units: every thread sums some sequences' tiles, a scan finds
    // the sequence that the range starts in
    int64_t left;
    Cursor in;
    {
        const int per = (a.batch + NW * 32 - 1) / (NW * 32);
        const int b0 = threadIdx.x * per, b1 = min(b0 + per, a.batch);
        int64_t mine = 0;
        for (int b = b0; b < b1; ++b) {
            const int n = min(max(a.lengths[(int64_t)b * a.length_seq], 0), a.max_tokens);
            mine += max(1, (min(n, a.window) + KT - 1) / KT);
        }
        int64_t upto = mine;
        for (int d = 1; d < 32; d <<= 1) {
            const int64_t o = __shfl_up_sync(0xffffffffu, upto, d);
            if (lane >= d) upto += o;
        }
        int64_t* const sums = (int64_t*)smem;  // per warp; the ring is not in use yet
        if (lane == 31) sums[warp] = upto;
        __syncthreads();
        int64_t total = 0, before = 0;
        for (int w = 0; w < NW; ++w) {
            if (w < warp) before += sums[w];
            total += sums[w];
        }
        const int64_t units = total * t.items;
        const int64_t u0 = units * blockIdx.x / gridDim.x, u1 = units * (blockIdx.x + 1) / gridDim.x;
        left = u1 - u0;
        int64_t p = before + upto - mine;
        const int64_t target = u0 / t.items;
        if (left > 0 && p <= target && target < p + mine) {
            for (int b = b0; b < b1; ++b) {
                const int n = min(max(a.lengths[(int64_t)b * a.length_seq], 0), a.max_tokens);
                const int64_t tiles = max(1, (min(n, a.window) + KT - 1) / KT);
                if (target < p + tiles) {
                    sm_start[0] = p;
                    sm_start[1] = b;
                    break;
                }
                p += tiles;
            }
        }
        __syncthreads();
        if (left == 0) {
            if (threadIdx.x == 0) t.meta[blockIdx.x] = make_int4(0, 0, kIdle, 0);
            return;
        }
        in.b = (int)sm_start[1];
        enter_sequence<KT>(in, t, a.lengths[(int64_t)in.b * a.length_seq]);
        const int64_t within = u0 - sm_start[0] * t.items;
        in.item = (int)(within / in.tiles);
        in.tile = (int)(within % in.tiles);
    }
    const int units = (int)left;

    // -- fetching: lane l < 16 finds token l's row of K, lane l + 16 its row of V
    bool from_start = in.tile == 0, fresh = true;
    int page_id = -1;
    auto look_up = [&]() {
        const int token = in.begin + in.tile * KT + warp * 16 + (lane & 15);
        page_id = token < in.end ? a.tables[(int64_t)in.b * a.table_seq + a.page.div((uint32_t)token)] : -1;
    };
    look_up();
    auto fetch = [&](int slot) {
        unsigned char* const stage = ring + slot * Z::STAGE;
        const uint32_t to = smem_address(stage);
        const int token = in.begin + in.tile * KT + warp * 16 + (lane & 15);
        const bool valid = token < in.end && page_id >= 0 && page_id < a.cache.pages;
        const uint32_t mask = __ballot_sync(0xffffffffu, valid) & 0xffffu;
        const int head = in.item / t.row_blocks;
        uint32_t at = 0;
        if (valid) a.page.div((uint32_t)token, &at);
        const CacheView& c = lane < 16 ? a.cache.k : a.cache.v;
        const unsigned char* row = (const unsigned char*)c.ptr;
        if (valid) row += ((int64_t)page_id * c.page + (int64_t)at * c.token + (int64_t)head * c.head) * Z::EB;
        if (lane == 0) {
            const bool ends = in.tile + 1 == in.tiles, last = ends || left == 1;
            sm_meta[slot] = make_int4(in.b, in.item, (int)mask, (fresh ? 1 : 0) | (last ? 2 : 0) | (from_start ? 4 : 0) | (ends ? 8 : 0));
        }
        if constexpr (kScaled) {
            const CacheView& z = lane < 16 ? a.cache.k_scale : a.cache.v_scale;
            const float* s = (const float*)z.ptr;
            if (valid) s += (int64_t)page_id * z.page + (int64_t)at * z.token + (int64_t)head * z.head;
            copy4(to + 32 * Z::ROW + lane * 4, s, valid);
        }
        if (mask) {
#pragma unroll
            for (int which = 0; which < 2; ++which)
#pragma unroll
                for (int i = 0; i < 16 * CPR / 32; ++i) {
                    const int r = (i * 32 + lane) / CPR, piece = (i * 32 + lane) % CPR;
                    const unsigned char* from =
                        (const unsigned char*)__shfl_sync(0xffffffffu, (unsigned long long)row, r + 16 * which);
                    const bool real = piece < t.row_chunks, there = mask >> r & 1;
                    const uint32_t dst = to + which * 16 * Z::ROW + swizzled<CPR>(r, piece) * 16;
                    // absent tokens: V must be zeros (their probability is 0, and 0 * NaN is not);
                    // K's scores are replaced. Padding: K must be zeros, V's columns are not used.
                    if (which == 0 ? (there || !real) : real) copy16(dst, from + (real ? piece * 16 : 0), real && there);
                }
        }
        // on to the next unit
        --left;
        fresh = false;
        if (left > 0) {
            if (++in.tile == in.tiles) {
                in.tile = 0;
                fresh = from_start = true;
                if (++in.item == t.items) {
                    in.item = 0;
                    ++in.b;
                    enter_sequence<KT>(in, t, in.next_length);
                }
            }
            look_up();
        }
    };

    // -- queries of a part as operands, in the order that the products take them: warp nt
    // holds rows nt * 8 .. + 7, four lanes a row
    auto stage_queries = [&](int b, int item) {
        if (warp >= NT) return;
        const int r = warp * 8 + oct, in_group = (item % t.row_blocks) * ROWS + r, dim = a.cache.head_dim;
        const bool there = in_group < a.group;
        const Q* q = (const Q*)a.q + (int64_t)b * a.q_seq + (int64_t)(item / t.row_blocks * a.group + (there ? in_group : 0)) * a.q_head;
        float x[KS][CT == MT_F32 ? 2 : 4], top = 0.0f;
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int i = 0; i < (CT == MT_F32 ? 2 : 4); ++i) {
                const int d = CT == MT_F32 ? k * 8 + quad + i * 4
                              : kScaled ? k * 16 + quad * 4 + i : k * 16 + quad * 2 + (i & 1) + (i >> 1) * 8;
                x[k][i] = there && d < dim ? (float)q[d] : 0.0f;
                top = fmaxf(top, fabsf(x[k][i]));
            }
        float factor = a.scale * kLog2e;
        if constexpr (Z::kNormed) {
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // 2^-e with 2^e <= top: exponents of both within fp32's normal range
            const uint32_t e = min(max(__float_as_uint(top) >> 23, 1u), 252u);
            const float down = __uint_as_float((254u - e) << 23);
            factor *= __uint_as_float(e << 23);
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) x[k][i] *= down;
        }
        if (quad == 0) sm_qscale[r] = factor;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            if constexpr (CT == MT_F32) {
                const uint32_t h0 = upper(x[k][0]), h1 = upper(x[k][1]);
                sm_q[((k * NT + warp) * QP + 0) * 32 + lane] = make_uint2(h0, h1);
                sm_q[((k * NT + warp) * QP + 1) * 32 + lane] =
                    make_uint2(__float_as_uint(x[k][0] - __uint_as_float(h0)), __float_as_uint(x[k][1] - __uint_as_float(h1)));
            } else {
#pragma unroll
                for (int p = 0; p < QP; ++p) {
                    const uint32_t y0 = pack<kBf16>(x[k][0], x[k][1]), y1 = pack<kBf16>(x[k][2], x[k][3]);
                    sm_q[((k * NT + warp) * QP + p) * 32 + lane] = make_uint2(y0, y1);
                    if (p + 1 < QP) {
                        const float2 g0 = unpack<kBf16>(y0), g1 = unpack<kBf16>(y1);
                        x[k][0] -= g0.x;
                        x[k][1] -= g0.y;
                        x[k][2] -= g1.x;
                        x[k][3] -= g1.y;
                    }
                }
            }
        }
    };
    stage_queries(in.b, in.item);
    const int first_item = in.item, first_b = in.b;
    int first_kind = kNoPart;

#pragma unroll
    for (int s = 0; s < S - 1; ++s) {
        if (left > 0) fetch(s);
        copies_commit();
    }
    __syncthreads();  // queries

    uint2 qf[Z::kQReg ? KS : 1][NT][QP];
    float o[DP / 16][NT][4], m[NT][2], l[NT][2], qscale[NT][2];
    float v_unit = 0.0f;  // O is in units of this power of two (8-bit caches)

    int slot = 0;
    for (int unit = 0; unit < units; ++unit) {
        __syncwarp();
        if (left > 0) fetch(slot == 0 ? S - 1 : slot - 1);
        copies_commit();
        copies_wait<S - 1>();
        __syncwarp();
        const int4 meta = sm_meta[slot];
        const uint32_t mask = (uint32_t)meta.z;
        unsigned char* const stage = ring + slot * Z::STAGE;
        const uint32_t k_at = smem_address(stage), v_at = k_at + 16 * Z::ROW;
        if (meta.w & 1) {
            if constexpr (Z::kQReg)
#pragma unroll
                for (int k = 0; k < KS; ++k)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int p = 0; p < QP; ++p) qf[k][n][p] = sm_q[((k * NT + n) * QP + p) * 32 + lane];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    m[n][i] = -INFINITY;
                    l[n][i] = 0.0f;
                    qscale[n][i] = sm_qscale[n * 8 + quad * 2 + i];
                }
#pragma unroll
            for (int d = 0; d < DP / 16; ++d)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[d][n][i] = 0.0f;
            v_unit = 1.17549435e-38f;  // 2^-126
        }
        if (mask) {
            // S^T: c[0], c[1] are token oct, heads quad * 2 + 0, 1; c[2], c[3] token oct + 8
            float s[NT][4], part[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[n][i] = part[n][i] = 0.0f;
            auto query = [&](int k, int n, int p) {
                return Z::kQReg ? qf[Z::kQReg ? k : 0][n][p] : sm_q[((k * NT + n) * QP + p) * 32 + lane];
            };
            // the largest pieces' products go into `part`, the others into s
            auto times_queries = [&](int k, const uint32_t (&x)[4]) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int p = 0; p < QP; ++p) {
                        const uint2 q = query(k, n, p);
                        product<CT>(p == 0 && Z::kExact ? part[n] : s[n], x, q.x, q.y);
                    }
                if constexpr (Z::kExact) {
                    if (k % 4 == 3 || k == KS - 1) {
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                s[n][i] += part[n][i];
                                part[n][i] = 0.0f;
                            }
                    }
                }
            };
#pragma unroll
            for (int c = 0; c < CPR / 2; ++c) {
                uint32_t r[4];
                load_matrices(r, k_at + swizzled<CPR>(lane & 15, 2 * c + (lane >> 4)) * 16);
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
                        product<CT>(s[n], lo, q.x, q.y);
                    }
                } else if constexpr (kScaled) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t x[4] = {decode<CT, 0, 1>(r[2 * h]), decode<CT, 0, 1>(r[2 * h + 1]),
                                               decode<CT, 2, 3>(r[2 * h]), decode<CT, 2, 3>(r[2 * h + 1])};
                        times_queries(2 * c + h, x);
                    }
                } else {
                    times_queries(c, r);
                }
            }
            float ks[2] = {1.0f, 1.0f}, vs[2] = {1.0f, 1.0f}, shrink = 1.0f;
            if constexpr (kScaled) {
                const float* z = (const float*)(stage + 32 * Z::ROW);
                ks[0] = z[oct];
                ks[1] = z[oct + 8];
                vs[0] = z[16 + oct];
                vs[1] = z[16 + oct + 8];
                float top = fmaxf(fabsf(vs[0]), fabsf(vs[1]));
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                // the power of two above the largest scale so far
                const float unit = __uint_as_float((min(__float_as_uint(top) >> 23, 252u) + 1) << 23);
                if (unit > v_unit) {
                    shrink = v_unit / unit;
                    v_unit = unit;
                }
                const float per = 1.0f / v_unit;
                vs[0] *= per;
                vs[1] *= per;
            }
            const bool seen[2] = {(mask >> oct & 1) != 0, (mask >> (oct + 8) & 1) != 0};
            uint32_t pf[NT][CT == MT_F32 ? 4 : 2 * QP];
            bool grown = shrink != 1.0f;
            float keep[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float s0 = seen[0] ? s[n][i] * (qscale[n][i] * ks[0]) : -INFINITY;
                    const float s1 = seen[1] ? s[n][2 + i] * (qscale[n][i] * ks[1]) : -INFINITY;
                    float top = fmaxf(s0, s1);
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                    top = fmaxf(top, m[n][i]);
                    const float base = top == -INFINITY ? 0.0f : top;
                    keep[n][i] = exp2_fast(m[n][i] - base);
                    grown |= top > m[n][i];
                    m[n][i] = top;
                    const float p0 = exp2_fast(s0 - base + Z::kOffset), p1 = exp2_fast(s1 - base + Z::kOffset);
                    l[n][i] = l[n][i] * keep[n][i] + (p0 + p1);
                    s[n][i] = kScaled ? p0 * vs[0] : p0;
                    s[n][2 + i] = kScaled ? p1 * vs[1] : p1;
                }
                if constexpr (CT == MT_F32) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t x = __float_as_uint(s[n][2 * h]), y = __float_as_uint(s[n][2 * h + 1]);
                        const uint32_t low = transpose8x8(__byte_perm(x, y, 0x5410)), high = transpose8x8(__byte_perm(x, y, 0x7632));
                        pf[n][2 * h] = __byte_perm(low, high, 0x5410);
                        pf[n][2 * h + 1] = __byte_perm(low, high, 0x7632);
                    }
                } else {
#pragma unroll
                    for (int p = 0; p < QP; ++p)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const uint32_t y = pack<kBf16>(s[n][2 * h], s[n][2 * h + 1]);
                            pf[n][2 * p + h] = transpose8x8(y);
                            if (p + 1 < QP) {
                                const float2 g = unpack<kBf16>(y);
                                s[n][2 * h] -= g.x;
                                s[n][2 * h + 1] -= g.y;
                            }
                        }
                }
            }
            if (!Z::kExact && __any_sync(0xffffffffu, grown)) {
#pragma unroll
                for (int d = 0; d < DP / 16; ++d)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[d][n][i] *= kScaled ? keep[n][i & 1] * shrink : keep[n][i & 1];
            }
            // O^T: rows are 16 dims, columns heads as above
            auto add_up = [&](int d, int n, const float (&x)[4]) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    o[d][n][i] = o[d][n][i] * (kScaled ? keep[n][i & 1] * shrink : keep[n][i & 1]) + x[i];
            };
            if constexpr (CT == MT_F32) {
                const float* v = (const float*)(stage + 16 * Z::ROW);
#pragma unroll
                for (int d = 0; d < DP / 16; ++d) {
                    float x16[NT][4] = {};
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
                            const float p0 = __uint_as_float(pf[n][2 * h]), p1 = __uint_as_float(pf[n][2 * h + 1]);
                            const uint32_t h0 = upper(p0), h1 = upper(p1);
                            product<CT>(x16[n], lo, h0, h1);
                            product<CT>(x16[n], hi, __float_as_uint(p0 - __uint_as_float(h0)),
                                        __float_as_uint(p1 - __uint_as_float(h1)));
                            product<CT>(x16[n], hi, h0, h1);
                        }
                    }
#pragma unroll
                    for (int n = 0; n < NT; ++n) add_up(d, n, x16[n]);
                }
            } else if constexpr (kScaled) {
#pragma unroll
                for (int c = 0; c < CPR / 2; ++c) {
                    uint32_t r[4];
                    load_transposed(r, v_at + swizzled<CPR>(lane & 15, 2 * c + (lane >> 4)) * 16);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        // bytes 0, 2 are two tokens' even dim, bytes 1, 3 their odd one
                        const uint32_t x[4] = {decode<CT, 0, 2>(r[2 * h]), decode<CT, 1, 3>(r[2 * h]),
                                               decode<CT, 0, 2>(r[2 * h + 1]), decode<CT, 1, 3>(r[2 * h + 1])};
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            float x16[4] = {};
#pragma unroll
                            for (int p = QP - 1; p >= 0; --p)
                                product<CT>(Z::kExact ? x16 : o[2 * c + h][n], x, pf[n][2 * p], pf[n][2 * p + 1]);
                            if constexpr (Z::kExact) add_up(2 * c + h, n, x16);
                        }
                    }
                }
            } else {
#pragma unroll
                for (int d = 0; d < DP / 16; ++d) {
                    uint32_t r[4];
                    load_transposed(r, v_at + swizzled<CPR>((lane & 7) + (lane >> 4) * 8, 2 * d + (lane >> 3 & 1)) * 16);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        float x16[4] = {};
#pragma unroll
                        for (int p = QP - 1; p >= 0; --p)
                            product<CT>(Z::kExact ? x16 : o[d][n], r, pf[n][2 * p], pf[n][2 * p + 1]);
                        if constexpr (Z::kExact) add_up(d, n, x16);
                    }
                }
            }
        }
        if (meta.w & 2) {
            // -- the part ends: join the warps' (m, l, O). Each warp's O goes to its own stage of this
            // unit, which nothing will be fetched into before the last barrier below.
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float sum = l[n][i];
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
                    if (oct == 0) sm_ml[warp * ROWS + n * 8 + quad * 2 + i] = make_float2(m[n][i], sum);
                }
            __syncthreads();
            const int item = meta.y, head0 = item / t.row_blocks * a.group + item % t.row_blocks * ROWS;
            const int rows = min(ROWS, a.group - item % t.row_blocks * ROWS), dim = a.cache.head_dim;
            const bool whole = (meta.w & 12) == 12;
            const int part = blockIdx.x * 2 + (meta.w & 4 ? 1 : 0);
            if (!(meta.w & 4)) first_kind = meta.w & 8 ? kEnd : kMiddle;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                if (n * 8 >= rows) break;
                float* const mine = (float*)stage;  // [8][DP]
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int r = quad * 2 + i;
                    float top = -INFINITY;
#pragma unroll
                    for (int w = 0; w < NW; ++w) top = fmaxf(top, sm_ml[w * ROWS + n * 8 + r].x);
                    float f = m[n][i] == -INFINITY ? 0.0f : exp2_fast(m[n][i] - top);
                    if constexpr (kScaled) f *= v_unit;
#pragma unroll
                    for (int d = 0; d < DP / 16; ++d) {
                        const int d0 = 16 * d + (kScaled ? 2 * oct : oct), d1 = d0 + (kScaled ? 1 : 8);
                        mine[r * DP + (d0 ^ quad * 8)] = o[d][n][i] * f;
                        mine[r * DP + (d1 ^ quad * 8)] = o[d][n][2 + i] * f;
                    }
                }
                __syncthreads();
                for (int r = warp; r < 8 && n * 8 + r < rows; r += NW) {
                    float top = -INFINITY, sum = 0.0f;
#pragma unroll
                    for (int w = 0; w < NW; ++w) top = fmaxf(top, sm_ml[w * ROWS + n * 8 + r].x);
#pragma unroll
                    for (int w = 0; w < NW; ++w) {
                        const float2 ml = sm_ml[w * ROWS + n * 8 + r];
                        sum += ml.x == -INFINITY ? ml.y : ml.y * exp2_fast(ml.x - top);
                    }
                    const bool none = top == -INFINITY && sum == 0.0f;
                    const float per = none ? 0.0f : 1.0f / sum;
                    for (int d = lane; d < dim; d += 32) {
                        float x = 0.0f;
#pragma unroll
                        for (int w = 0; w < NW; ++w)
                            x += ((const float*)(smem + w * (S * Z::STAGE) + slot * Z::STAGE))[r * DP + (d ^ (r >> 1) * 8)];
                        if (whole)
                            ((Q*)a.out)[(int64_t)meta.x * a.out_seq + (int64_t)(head0 + n * 8 + r) * a.out_head + d] =
                                rounded<Q>(none ? 0.0f : x * per);
                        else
                            t.part_o[((int64_t)part * ROWS + n * 8 + r) * DP + d] = x;
                    }
                    if (lane == 0) {
                        if (!whole)
                            t.part_ml[(int64_t)part * ROWS + n * 8 + r] = make_float2(top, sum);
                        else if (a.lse)
                            a.lse[(int64_t)meta.x * a.lse_seq + (int64_t)(head0 + n * 8 + r) * a.lse_head] =
                                (top + log2f(sum) - Z::kOffset) * kLn2;
                    }
                }
                if (n == NT - 1 || (n + 1) * 8 >= rows) {
                    if (unit + 1 < units) {
                        const int4 next = sm_meta[slot + 1 == S ? 0 : slot + 1];
                        stage_queries(next.x, next.y);
                    }
                }
                __syncthreads();
            }
        }
        if (++slot == S) slot = 0;
    }
    copies_wait<0>();
    if (threadIdx.x == 0) t.meta[blockIdx.x] = make_int4(first_b, first_item, first_kind, 0);
}

// Joins the parts of heads that cuts crossed. Block (c, r): if the part that block c of
// attention_tiles started in ended there, it is the last of a chain that goes back to the
// block where that head began; row r of the chain's (m, l, O) becomes the output.
constexpr int kJoinThreads = 128;

template <class Q, int DP, int ROWS>
__global__ void __launch_bounds__(kJoinThreads) join_parts(const __grid_constant__ TileArgs t, float offset) {
    extern __shared__ float weight[];  // of each part of the chain, then the first one's place
    __shared__ float red[2][kJoinThreads / 32];
    __shared__ int sm_first;
    const AttentionArgs& a = t.a;
    const int c = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int4 end = t.meta[c];
    const int r = blockIdx.y, row_block = end.y % t.row_blocks;
    if (end.z != kEnd || row_block * ROWS + r >= a.group) return;
    // back to the block whose last part began the head
    int first = -1;
    for (int hi = c - 1; first < 0 && hi >= 0; hi -= kJoinThreads) {
        const int p = hi - (int)threadIdx.x;
        const int kind = p >= 0 ? t.meta[p].z : kMiddle;
        if (threadIdx.x == 0) sm_first = -1;
        __syncthreads();
        if (kind == kNoPart || kind == kEnd) atomicMax(&sm_first, p);
        __syncthreads();
        first = sm_first;
        __syncthreads();
    }
    if (first < 0) return;  // not reached: the first block's first part begins a head
    const int count = c - first + 1;
    auto place = [&](int i) { return (int64_t)((first + i) * 2 + (i == 0 ? 1 : 0)) * ROWS + r; };
    float top = -INFINITY;
    for (int i = threadIdx.x; i < count; i += kJoinThreads)
        if (i == 0 || t.meta[first + i].z != kIdle) top = fmaxf(top, t.part_ml[place(i)].x);
    for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    if (lane == 0) red[0][warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kJoinThreads / 32; ++w) top = fmaxf(top, red[0][w]);
    float sum = 0.0f;
    for (int i = threadIdx.x; i < count; i += kJoinThreads) {
        float f = 0.0f;
        if (i == 0 || t.meta[first + i].z != kIdle) {
            const float2 ml = t.part_ml[place(i)];
            f = ml.x == -INFINITY ? (ml.y == 0.0f ? 0.0f : 1.0f) : exp2_fast(ml.x - top);
            sum += ml.y * f;
        } else {
            f = -1.0f;  // an idle block: its memory holds nothing
        }
        weight[i] = f;
    }
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (lane == 0) red[1][warp] = sum;
    __syncthreads();
    sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kJoinThreads / 32; ++w) sum += red[1][w];
    const int head = end.y / t.row_blocks * a.group + row_block * ROWS + r;
    const bool none = top == -INFINITY && sum == 0.0f;
    const float per = none ? 0.0f : 1.0f / sum;
    for (int d = threadIdx.x; d < a.cache.head_dim; d += kJoinThreads) {
        float x = 0.0f;
#pragma unroll 4
        for (int i = 0; i < count; ++i) {
            const float f = weight[i];
            if (f >= 0.0f || f != f) x += f * t.part_o[place(i) * DP + d];
        }
        ((Q*)a.out)[(int64_t)end.x * a.out_seq + (int64_t)head * a.out_head + d] = rounded<Q>(none ? 0.0f : x * per);
    }
    if (threadIdx.x == 0 && a.lse)
        a.lse[(int64_t)end.x * a.lse_seq + (int64_t)head * a.lse_head] = (top + log2f(sum) - offset) * kLn2;
}

// ---- launch ------------------------------------------------------------------------------------

constexpr int kMaxDevices = 16;

template <int CT, class Q, int DP, int NT>
int launch(const AttentionArgs& a, void* workspace, uint64_t* bytes, int dev, cudaStream_t st) {
    using Z = Shape<CT, sizeof(Q) == 4, DP, NT>;
    TileArgs t;
    t.a = a;
    t.row_blocks = (a.group + Z::ROWS - 1) / Z::ROWS;
    t.items = a.cache.kv_heads * t.row_blocks;
    t.row_chunks = a.cache.head_dim * Z::EB / 16;
    int sms;
    if (int rc = sm_count(dev, &sms)) return rc;
    // as many blocks as fit the GPU at once, or fewer where there cannot be as many units
    const int64_t tokens = a.max_tokens < a.window ? a.max_tokens : a.window;
    const int64_t most = (tokens + Z::KT - 1) / Z::KT, resident = (int64_t)sms * Z::BLOCKS;
    int64_t blocks = (int64_t)a.batch * t.items * (most > 0 ? most : 1);
    if (blocks > resident) blocks = resident;
    const uint64_t meta_bytes = (uint64_t)blocks * 16, ml_bytes = (uint64_t)blocks * 2 * Z::ROWS * 8;
    *bytes = meta_bytes + ml_bytes + (uint64_t)blocks * 2 * Z::ROWS * DP * 4;
    if (!workspace) return 0;
    t.meta = (int4*)workspace;
    t.part_ml = (float2*)((char*)workspace + meta_bytes);
    t.part_o = (float*)((char*)workspace + meta_bytes + ml_bytes);
    auto kernel = attention_tiles<CT, Q, DP, NT>;
    static bool ready[kMaxDevices] = {};
    if (!ready[dev]) {
        RT_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Z::SMEM));
        ready[dev] = true;
    }
    kernel<<<(unsigned)blocks, Z::NW * 32, Z::SMEM, st>>>(t);
    RT_CHECK(cudaGetLastError());
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks, a.group < Z::ROWS ? a.group : Z::ROWS);
    cfg.blockDim = dim3(kJoinThreads);
    cfg.dynamicSmemBytes = (size_t)blocks * 4;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    RT_CHECK(cudaLaunchKernelEx(&cfg, join_parts<Q, DP, Z::ROWS>, (const TileArgs)t, Z::kOffset));
    return 0;
}

template <int CT, class Q> int by_shape(const AttentionArgs& a, void* workspace, uint64_t* bytes, int dev, cudaStream_t st) {
    const int dim = a.cache.head_dim;
    const bool wide = a.group > 8;
    if (dim <= 64) return wide ? launch<CT, Q, 64, 2>(a, workspace, bytes, dev, st) : launch<CT, Q, 64, 1>(a, workspace, bytes, dev, st);
    if (dim <= 128) return wide ? launch<CT, Q, 128, 2>(a, workspace, bytes, dev, st) : launch<CT, Q, 128, 1>(a, workspace, bytes, dev, st);
    return wide ? launch<CT, Q, 256, 2>(a, workspace, bytes, dev, st) : launch<CT, Q, 256, 1>(a, workspace, bytes, dev, st);
}

}  // namespace tiles
}  // namespace mt
