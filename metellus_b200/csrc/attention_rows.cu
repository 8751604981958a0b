// Paged attention for any head_dim and alignment: one warp reads one key row at a time.
//
// Softmax in one pass: with the running maximum m of the scores, l = sum exp(s - m) and
// o = sum exp(s - m) v; a new maximum m' scales l and o by exp(m - m'). Every warp of a
// block keeps its own (m, l, o) over every eighth token; they are joined at the end.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

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

template <class Q, class C>
__global__ void __launch_bounds__(kThreads) attention_rows(const AttentionArgs a) {
    constexpr bool kScaled = sizeof(C) == 1;
    __shared__ float sm_m[kWarps][kRows], sm_l[kWarps][kRows], sm_o[kWarps][kMaxHeadDim];
    asm volatile("griddepcontrol.launch_dependents;\n\tgriddepcontrol.wait;" ::: "memory");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int b = blockIdx.x, g = blockIdx.y, r0 = blockIdx.z * kRows;
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
    for (int t = first + warp; t < n; t += kWarps) {
        uint32_t at;
        const uint32_t j = a.page.div((uint32_t)t, &at);
        const int page = a.tables[b * a.table_seq + j];
        if (page < 0 || page >= a.cache.pages) continue;
        const C* krow = (const C*)a.cache.k.ptr + page * a.cache.k.page + at * a.cache.k.token + g * a.cache.k.head;
        const C* vrow = (const C*)a.cache.v.ptr + page * a.cache.v.page + at * a.cache.v.token + g * a.cache.v.head;
        float ks = 1.0f, vs = 1.0f;
        if constexpr (kScaled) {
            const CacheView &zk = a.cache.k_scale, &zv = a.cache.v_scale;
            ks = ((const float*)zk.ptr)[page * zk.page + at * zk.token + g * zk.head];
            vs = ((const float*)zv.ptr)[page * zv.page + at * zv.token + g * zv.head];
        }
        float k[kPerLane], v[kPerLane];
#pragma unroll
        for (int i = 0; i < kPerLane; ++i) {
            const int d = lane + 32 * i;
            k[i] = d < dim ? (float)krow[d] : 0.0f;
            v[i] = d < dim ? (float)vrow[d] * vs : 0.0f;
        }
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            if (r >= rows) break;
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < kPerLane; ++i) s = fmaf(q[r][i], k[i], s);
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
            s *= ks * a.scale * kLog2e;
            const float top = fmaxf(m[r], s);
            const float keep = rescale(m[r], top), p = s == -INFINITY ? 0.0f : exp2f(s - top);
            m[r] = top;
            l[r] = l[r] * keep + p;
#pragma unroll
            for (int i = 0; i < kPerLane; ++i) o[r][i] = o[r][i] * keep + p * v[i];
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
        const int head = g * a.group + r0 + r;
        for (int d = threadIdx.x; d < dim; d += kThreads) {
            float x = 0.0f;
            for (int w = 0; w < kWarps; ++w) x += sm_o[w][d];
            ((Q*)a.out)[b * a.out_seq + head * a.out_head + d] = rounded<Q>(sum == 0.0f && top == -INFINITY ? 0.0f : x / sum);
        }
        if (a.lse && threadIdx.x == 0)
            a.lse[b * a.lse_seq + head * a.lse_head] = (top + log2f(sum)) * kLn2;
        __syncthreads();
    }
}

template <class Q, class C> int launch(const AttentionArgs& a, cudaStream_t st) {
    const dim3 grid(a.batch, a.cache.kv_heads, (a.group + kRows - 1) / kRows);
    RT_CHECK(launch_early(attention_rows<Q, C>, grid, kThreads, 0, st, a));
    return 0;
}

template <class Q> int launch8(const AttentionArgs& a, cudaStream_t st) {
    return a.cache.dtype == MT_I8 ? launch<Q, int8_t>(a, st) : launch<Q, __nv_fp8_e4m3>(a, st);
}

}  // namespace

int attend_by_rows(const AttentionArgs& a, cudaStream_t st) {
    const int q = a.q_type, c = a.cache.dtype;
    if (a.cache.scaled()) {
        if (q == MT_F32) return launch8<float>(a, st);
        if (q == MT_F16) return launch8<__half>(a, st);
        return launch8<__nv_bfloat16>(a, st);
    }
    if (c == MT_F32) return launch<float, float>(a, st);
    if (c == MT_F16) return q == MT_F32 ? launch<float, __half>(a, st) : launch<__half, __half>(a, st);
    return q == MT_F32 ? launch<float, __nv_bfloat16>(a, st) : launch<__nv_bfloat16, __nv_bfloat16>(a, st);
}

}  // namespace mt
