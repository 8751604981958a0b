// Paged attention for any head_dim and alignment: one warp reads one key row at a time.
//
// Softmax in one pass: with the running maximum m of the scores, l = sum exp(s - m) and
// o = sum exp(s - m) v; a new maximum m' scales l and o by exp(m - m'). Every warp of a sequence's
// blocks keeps its own (m, l, o) over runs of 4 tokens; they are joined at the end.
//
// It serves what tiles cannot: rows that are not whole 16-byte pieces, caches whose rows have no 32-bit
// numbers, scales that are not positive. Instructions bound it (a dot product's 5 exchanges for each
// query head and token): bf16, 32 query heads on 8 of 100, 64 sequences of 1024 tokens 518 us (32 at the
// copy rate; heads of 104, in tiles, 50). Few sequences are split over clusters of up to 8 blocks:
// 1 of 16384 tokens 258 us, 2.6 ms in one block each, a token at a time.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cooperative_groups.h>

#include "mt_paged_attention.h"

namespace mt {

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kRows = 8;                       // query heads of one key-value head a block holds
constexpr int kPerLane = kMaxHeadDim / 32;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

template <class T> __device__ inline T rounded(float x);
template <> __device__ inline float rounded<float>(float x) { return x; }
template <> __device__ inline __half rounded<__half>(float x) { return __float2half_rn(x); }
template <> __device__ inline __nv_bfloat16 rounded<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// exp2(m_old - m_new), 0 where there was nothing before (m_new may be -inf then too)
__device__ inline float rescale(float m_old, float m_new) {
    return m_old == -INFINITY ? 0.0f : exp2f(m_old - m_new);
}

// Blocks blockIdx.x % splits of a cluster share a sequence's tokens: kChunk at a time a warp, whose rows
// are asked for together.
constexpr int kChunk = 4;

template <class Q, class C>
__global__ void __launch_bounds__(kThreads) attention_rows(const AttentionArgs a, int splits) {
    constexpr bool kScaled = sizeof(C) == 1;
    __shared__ float sm_m[kWarps][kRows], sm_l[kWarps][kRows], sm_o[kWarps][kMaxHeadDim];
    __shared__ float block_m[kRows], block_l[kRows], block_o[kRows][kMaxHeadDim];
    asm volatile("griddepcontrol.launch_dependents;\n\tgriddepcontrol.wait;" ::: "memory");
    const cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, split = (int)(blockIdx.x % splits);
    const int64_t b = blockIdx.x / splits;
    const int g = blockIdx.y, r0 = blockIdx.z * kRows;
    const int rows = min(kRows, a.group - r0), dim = a.cache.head_dim;
    const int n = min(max(a.lengths[b * a.length_seq], 0), a.max_tokens);
    const int first = n > a.window ? n - a.window : 0;
    float q[kRows][kPerLane], o[kRows][kPerLane], m[kRows], l[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        m[r] = -INFINITY;
        l[r] = 0.0f;
        const Q* row = (const Q*)a.q + b * a.q_seq + (int64_t)(g * a.group + r0 + r) * a.q_head;
#pragma unroll
        for (int i = 0; i < kPerLane; ++i) {
            const int d = lane + 32 * i;
            q[r][i] = r < rows && d < dim ? (float)row[d] : 0.0f;
            o[r][i] = 0.0f;
        }
    }
    // n and a chunk's end are below 2^31 - 1024
    for (int64_t t0 = first + (int64_t)(split * kWarps + warp) * kChunk; t0 < n; t0 += (int64_t)splits * kWarps * kChunk) {
        // lanes 0 .. kChunk - 1 look up a token's place each
        uint32_t at = 0;
        int page = -1;
        if (lane < kChunk && t0 + lane < n) {
            const uint32_t j = a.page.div((uint32_t)(t0 + lane), &at);
            page = a.tables[b * a.table_seq + j];
            if (page >= a.cache.pages) page = -1;
        }
        C k[kChunk][kPerLane], v[kChunk][kPerLane];
        float ks[kChunk], vs[kChunk];
        bool there[kChunk];
#pragma unroll
        for (int c = 0; c < kChunk; ++c) {
            const int64_t p = __shfl_sync(0xffffffffu, page, c), u = __shfl_sync(0xffffffffu, at, c);
            there[c] = p >= 0;
            ks[c] = vs[c] = 1.0f;
            if (!there[c]) continue;
            const C* krow = (const C*)a.cache.k.ptr + p * a.cache.k.page + u * a.cache.k.token + g * a.cache.k.head;
            const C* vrow = (const C*)a.cache.v.ptr + p * a.cache.v.page + u * a.cache.v.token + g * a.cache.v.head;
#pragma unroll
            for (int i = 0; i < kPerLane; ++i) {
                const int d = lane + 32 * i;
                k[c][i] = d < dim ? krow[d] : C(0.0f);
                v[c][i] = d < dim ? vrow[d] : C(0.0f);
            }
            if constexpr (kScaled) {
                const CacheView &zk = a.cache.k_scale, &zv = a.cache.v_scale;
                ks[c] = ((const float*)zk.ptr)[p * zk.page + u * zk.token + g * zk.head];
                vs[c] = ((const float*)zv.ptr)[p * zv.page + u * zv.token + g * zv.head];
            }
        }
#pragma unroll
        for (int c = 0; c < kChunk; ++c) {
            if (!there[c]) continue;
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                if (r >= rows) break;
                float s = 0.0f;
#pragma unroll
                for (int i = 0; i < kPerLane; ++i) s = fmaf(q[r][i], (float)k[c][i], s);
#pragma unroll
                for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
                s *= ks[c] * a.scale * kLog2e;
                const float top = fmaxf(m[r], s);
                const float keep = rescale(m[r], top), p = s == -INFINITY ? 0.0f : exp2f(s - top);
                m[r] = top;
                l[r] = l[r] * keep + p;
#pragma unroll
                for (int i = 0; i < kPerLane; ++i) o[r][i] = o[r][i] * keep + p * ((float)v[c][i] * vs[c]);
            }
        }
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r)
        if (lane == 0) {
            sm_m[warp][r] = m[r];
            sm_l[warp][r] = l[r];
        }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        if (r >= rows) break;
        float top = -INFINITY, sum = 0.0f;
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm_m[w][r]);
        for (int w = 0; w < kWarps; ++w) sum += sm_l[w][r] * rescale(sm_m[w][r], top);
        const float keep = rescale(m[r], top);
#pragma unroll
        for (int i = 0; i < kPerLane; ++i) sm_o[warp][lane + 32 * i] = o[r][i] * keep;
        __syncthreads();
        for (int d = threadIdx.x; d < dim; d += kThreads) {
            float x = 0.0f;
            for (int w = 0; w < kWarps; ++w) x += sm_o[w][d];
            block_o[r][d] = x;
        }
        if (threadIdx.x == 0) {
            block_m[r] = top;
            block_l[r] = sum;
        }
        __syncthreads();
    }
    // the cluster's blocks join theirs, some rows each
    cluster.sync();
    for (int r = split; r < rows; r += splits) {
        float top = -INFINITY, sum = 0.0f, x[kMaxHeadDim / kThreads] = {};
        for (int s = 0; s < splits; ++s) top = fmaxf(top, *cluster.map_shared_rank(&block_m[r], s));
        for (int s = 0; s < splits; ++s) {
            const float keep = rescale(*cluster.map_shared_rank(&block_m[r], s), top);
            sum += *cluster.map_shared_rank(&block_l[r], s) * keep;
            for (int d = threadIdx.x, i = 0; d < dim; d += kThreads, ++i) x[i] += *cluster.map_shared_rank(&block_o[r][d], s) * keep;
        }
        const int64_t head = g * a.group + r0 + r;
        for (int d = threadIdx.x, i = 0; d < dim; d += kThreads, ++i)
            ((Q*)a.out)[b * a.out_seq + head * a.out_head + d] = rounded<Q>(sum == 0.0f && top == -INFINITY ? 0.0f : x[i] / sum);
        if (a.lse && threadIdx.x == 0) a.lse[b * a.lse_seq + head * a.lse_head] = (top + log2f(sum)) * kLn2;
    }
    cluster.sync();  // until all have read
}

template <class Q, class C> int launch(const AttentionArgs& a, int sms, cudaStream_t st) {
    const int row_blocks = (a.group + kRows - 1) / kRows;
    // a sequence's tokens in up to 8 blocks, as long as there are SMs for them and chunks for their warps
    const int64_t tokens = a.max_tokens < a.window ? a.max_tokens : a.window;
    unsigned splits = 1;
    while (splits < 8 && (int64_t)a.batch * a.cache.kv_heads * row_blocks * splits < sms && tokens > (int64_t)splits * kWarps * kChunk)
        splits *= 2;
    const dim3 grid((unsigned)a.batch * splits, a.cache.kv_heads, row_blocks);
    RT_CHECK(launch_clusters(splits, attention_rows<Q, C>, grid, kThreads, 0, st, a, (int)splits));
    return 0;
}

template <class Q> int launch8(const AttentionArgs& a, int sms, cudaStream_t st) {
    return a.cache.dtype == MT_I8 ? launch<Q, int8_t>(a, sms, st) : launch<Q, __nv_fp8_e4m3>(a, sms, st);
}

}  // namespace

int attend_by_rows(const AttentionArgs& a, int dev, cudaStream_t st) {
    int sms;
    if (int rc = sm_count(dev, &sms)) return rc;
    const int q = a.q_type, c = a.cache.dtype;
    if (a.cache.scaled()) {
        if (q == MT_F32) return launch8<float>(a, sms, st);
        if (q == MT_F16) return launch8<__half>(a, sms, st);
        return launch8<__nv_bfloat16>(a, sms, st);
    }
    if (c == MT_F32) return launch<float, float>(a, sms, st);
    if (c == MT_F16) return q == MT_F32 ? launch<float, __half>(a, sms, st) : launch<__half, __half>(a, sms, st);
    return q == MT_F32 ? launch<float, __nv_bfloat16>(a, sms, st) : launch<__nv_bfloat16, __nv_bfloat16>(a, sms, st);
}

}  // namespace mt
