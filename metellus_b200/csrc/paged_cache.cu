// Writing a paged key-value cache and reading it back (mt_cache_write, mt_cache_read).
//
// HBM alone bounds both: each element is read once and written once, and between the two a
// token's head stays in registers, its rows of K and of V together: 16 elements a thread,
// head_dim / 16 threads a row, so that a row's addresses cost little beside its elements. Rows that
// cannot be moved 8 elements at a time take a warp each, element by element.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <type_traits>

#include "mt_paged.h"

namespace mt {

const char* dtype_name(int dtype) {
    static const char* const names[] = {"float32", "float16", "bfloat16", "int8", "float8_e4m3", "int32", "int64"};
    return dtype >= 0 && dtype <= MT_I64 ? names[dtype] : "unknown";
}

int64_t elements(const mt_array& a) {
    int64_t n = 1;
    for (int i = 0; i < a.ndim; ++i) n *= a.shape[i];
    return n;
}

int check_array(const char* who, const char* name, const mt_array* a, int ndim, uint32_t dtypes, bool last1) {
    if (!a) return bad_argument("%s: %s is missing", who, name);
    if (a->ndim != ndim) return bad_argument("%s: %s must have %d dimensions, not %d", who, name, ndim, a->ndim);
    if (a->dtype < 0 || a->dtype > MT_I64 || !(dtypes >> a->dtype & 1))
        return bad_argument("%s: %s cannot be %s", who, name, dtype_name(a->dtype));
    double bytes = bytes_of(a->dtype);
    for (int i = 0; i < ndim; ++i) {
        if (a->shape[i] < 0) return bad_argument("%s: %s has a negative extent", who, name);
        if (a->shape[i] > 1 && a->strides[i] < 0) return bad_argument("%s: %s has a negative stride", who, name);
        bytes *= (double)a->shape[i];
    }
    if (bytes > 4e18) return bad_argument("%s: %s is too large", who, name);
    if (last1 && a->shape[ndim - 1] > 1 && a->strides[ndim - 1] != 1)
        return bad_argument("%s: the last dimension of %s must be contiguous", who, name);
    if (elements(*a) > 0) {
        if (!a->ptr) return bad_argument("%s: %s has no memory", who, name);
        if ((uintptr_t)a->ptr % bytes_of(a->dtype))
            return bad_argument("%s: %s is not aligned to its elements", who, name);
    }
    return 0;
}

int check_written(const char* who, const char* name, const mt_array& a) {
    if (elements(a) == 0) return 0;
    for (int i = 0; i < a.ndim; ++i)
        if (a.shape[i] > 1 && a.strides[i] == 0)
            return bad_argument("%s: %s is written and must not be a broadcast (stride 0)", who, name);
    return 0;
}

static bool same_shape(const mt_array& a, const mt_array& b, int n) {
    for (int i = 0; i < n; ++i)
        if (a.shape[i] != b.shape[i]) return false;
    return true;
}

static CacheView view_of(const mt_array& a) {
    CacheView v;
    if (a.ndim < 3) return v;
    v.ptr = a.ptr;
    v.page = a.strides[0];
    v.token = a.strides[1];
    v.head = a.strides[2];
    return v;
}

int check_cache(const char* who, const mt_paged_cache* c, bool written, CacheShape* out) {
    if (!c) return bad_argument("%s: the cache is missing", who);
    const uint32_t types = 1u << MT_F32 | 1u << MT_F16 | 1u << MT_BF16 | 1u << MT_I8 | 1u << MT_E4M3;
    if (int rc = check_array(who, "k_cache", &c->k, 4, types, true)) return rc;
    if (int rc = check_array(who, "v_cache", &c->v, 4, types, true)) return rc;
    if (c->k.dtype != c->v.dtype) return bad_argument("%s: k_cache and v_cache must have one type", who);
    if (!same_shape(c->k, c->v, 4)) return bad_argument("%s: k_cache and v_cache must have one shape", who);
    const int64_t* s = c->k.shape;
    if (s[1] < 1 || s[2] < 1 || s[3] < 1)
        return bad_argument("%s: page_size, kv_heads and head_dim of the cache must be positive", who);
    if (s[3] > kMaxHeadDim) return bad_argument("%s: head_dim %lld is over %d", who, (long long)s[3], kMaxHeadDim);
    if (s[0] > INT32_MAX || s[1] > INT32_MAX || s[2] > 65535 || s[0] * s[1] > INT32_MAX)
        return bad_argument("%s: a cache holds at most 2^31 - 1 tokens of 65535 heads", who);
    const bool scaled = c->k.dtype == MT_I8 || c->k.dtype == MT_E4M3;
    for (int i = 0; i < 2; ++i) {
        const mt_array& z = i ? c->v_scale : c->k_scale;
        const char* name = i ? "v_scale" : "k_scale";
        if (!scaled) {
            if (z.ndim) return bad_argument("%s: a cache of %s has no %s", who, dtype_name(c->k.dtype), name);
            continue;
        }
        if (!z.ndim) return bad_argument("%s: a cache of %s needs %s", who, dtype_name(c->k.dtype), name);
        if (int rc = check_array(who, name, &z, 3, 1u << MT_F32, false)) return rc;
        if (!same_shape(z, c->k, 3))
            return bad_argument("%s: %s must be [pages, page_size, kv_heads] of the cache", who, name);
        if (written)
            if (int rc = check_written(who, name, z)) return rc;
    }
    if (written) {
        if (int rc = check_written(who, "k_cache", c->k)) return rc;
        if (int rc = check_written(who, "v_cache", c->v)) return rc;
    }
    out->dtype = c->k.dtype;
    out->pages = (int)s[0];
    out->page_size = (int)s[1];
    out->kv_heads = (int)s[2];
    out->head_dim = (int)s[3];
    out->k = view_of(c->k);
    out->v = view_of(c->v);
    if (scaled) {
        out->k_scale = view_of(c->k_scale);
        out->v_scale = view_of(c->v_scale);
    }
    return 0;
}

bool rows_aligned(const mt_array& a, int align) {
    if ((uintptr_t)a.ptr % align) return false;
    for (int i = 0; i + 1 < a.ndim; ++i)
        if (a.shape[i] > 1 && a.strides[i] * bytes_of(a.dtype) % align) return false;
    return true;
}

}  // namespace mt

namespace {

using namespace mt;

// Rows outside the cache: [tokens, heads, head_dim], last stride 1.
struct RowsView {
    void* ptr;
    int64_t token, head;
};

struct RowArgs {
    RowsView rows[2];      // k, v
    CacheView cache[2];
    CacheView scale[2];
    const void* slots;
    int64_t slot_stride;
    int slots64;
    int total_slots, head_dim, first, count;  // which of k, v: first .. first + count - 1
    int pieces;                               // rows can be moved 8 elements at a time (cache_*_pieces)
    int64_t row_count;                         // tokens * heads
    FastDiv heads, page;
};

template <class T> __device__ inline float to_float(T x) { return (float)x; }
template <> __device__ inline float to_float(__nv_fp8_e4m3 x) { return (float)x; }
template <> __device__ inline float to_float(int8_t x) { return (float)x; }

template <class T> __device__ inline T from_float(float x);
template <> __device__ inline float from_float<float>(float x) { return x; }
template <> __device__ inline __half from_float<__half>(float x) { return __float2half_rn(x); }
template <> __device__ inline __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// What a row is divided by: its scale s, as pairs of numbers for the instructions that take two
// elements. Rows of scales up to 1e-30 are raised by 2^96 first, both exactly, for 1 / s to be a
// number, and cut to `top`, the largest code: scales of a few of fp32's smallest steps are rounded
// so far that quotients would pass it.
struct Divisor {
    uint64_t minus_s, per, quarter;
    template <int N> __device__ Divisor(float s, float (&x)[N], float top) {
        if (s <= 1e-30f) {
            s *= 0x1p96f;
#pragma unroll
            for (int i = 0; i < N; ++i) x[i] = fminf(fmaxf(x[i] * 0x1p96f, -top * s), top * s);
        }
        const float y = 1.0f / s;
        minus_s = both(-s, -s), per = both(y, y), quarter = both(0.25f * y, 0.25f * y);
    }
    static __device__ uint64_t both(float a, float b) {
        uint64_t y;
        asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(a), "f"(b));
        return y;
    }

    // x / s, rounded so that it rounds to the code that x / s itself is nearest to (of two as near the
    // even one). x / s in fp32 can be rounded onto, or over, the border between two codes. t = x / s up
    // to 2 ulps; g = 9 t - (9 t - t), Veltkamp's way to drop t's last bits, is the multiple of 8 ulps
    // next to it, so x / s is within 6 ulps of g. Borders have 8 leading bits at most: none but g itself
    // is as near to x / s, and all that counts is on which side of g it lies: the sign of r = x - g s, which one fma gives exactly (where g is a border, s > 1e-30 keeps
    // it from underflow). g + r / 4s, rounded up, and down, and both moves added: g where r is 0, else a
    // number between g and x / s, or the next to g on that side. The last sum rounds down so that
    // -0 stays what it is.
    // 9 instructions for two elements and no branch. 2^25 elements fp16 -> e4m3, whose quotients often
    // are borders: 26 us (15.6 at the copy rate); 57 with a check that sent rows next to a border a slower
    // way, 28 with the sign of r taken in integers.
    __device__ float2 quotients(float x0, float x1) const {
        constexpr uint64_t kNine = 0x4110000041100000ull, kMinus1 = 0xBF800000BF800000ull;
        const uint64_t x = both(x0, x1);
        float2 y;
        asm("{.reg .b64 t, c, g, r, u, d, e, q;\n\t"
            "mul.rn.f32x2 t, %2, %3;\n\t"
            "mul.rn.f32x2 c, t, %6;\n\t"
            "fma.rn.f32x2 e, t, %7, c;\n\t"
            "fma.rn.f32x2 g, e, %7, c;\n\t"
            "fma.rn.f32x2 r, g, %4, %2;\n\t"
            "fma.rp.f32x2 u, r, %5, g;\n\t"
            "fma.rm.f32x2 d, r, %5, g;\n\t"
            "fma.rn.f32x2 e, g, %7, u;\n\t"
            "add.rm.f32x2 q, d, e;\n\t"
            "mov.b64 {%0, %1}, q;}"
            : "=f"(y.x), "=f"(y.y) : "l"(x), "l"(per), "l"(minus_s), "l"(quarter), "l"(kNine), "l"(kMinus1));
        return y;
    }
};

constexpr float kBig = 12582912.0f;  // 1.5 * 2^23: its ulp is 1, so adding it rounds to whole numbers

template <class C> struct Code;
template <> struct Code<int8_t> {
    static constexpr float kLargest = 127.0f;
    static __device__ int8_t of(float x, const Divisor& by) { return (int8_t)__float_as_uint(by.quotients(x, x).x + kBig); }
    static __device__ uint32_t bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
        return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
    }
    static __device__ uint32_t pack4(const float* x, const Divisor& by) {
        const float2 a = by.quotients(x[0], x[1]), b = by.quotients(x[2], x[3]);  // their low bytes, with kBig added
        return bytes(__float_as_uint(a.x + kBig), __float_as_uint(a.y + kBig), __float_as_uint(b.x + kBig), __float_as_uint(b.y + kBig));
    }
    static __device__ void unpack4(uint32_t y, float* x) {
#pragma unroll
        for (int i = 0; i < 4; ++i)  // 2^23 + (code + 128), less 2^23 + 128
            x[i] = __uint_as_float(__byte_perm(y ^ 0x80808080u, 0x4B000000u, 0x7540 | i)) - 8388736.0f;
    }
};
template <> struct Code<__nv_fp8_e4m3> {
    static constexpr float kLargest = 448.0f;
    static __device__ __nv_fp8_e4m3 of(float x, const Divisor& by) { return __nv_fp8_e4m3(by.quotients(x, x).x); }
    static __device__ uint32_t pack4(const float* x, const Divisor& by) {
        return __nv_cvt_float2_to_fp8x2(by.quotients(x[0], x[1]), __NV_SATFINITE, __NV_E4M3) |
               (uint32_t)__nv_cvt_float2_to_fp8x2(by.quotients(x[2], x[3]), __NV_SATFINITE, __NV_E4M3) << 16;
    }
    static __device__ void unpack4(uint32_t y, float* x) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(y >> (i * 16)), __NV_E4M3);
            const float2 f = __half22float2(*(const __half2*)&h);
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    }
};

// A row's largest magnitude; NaN if it has one. Then its scale, NaN too if that is not finite.
__device__ inline float largest(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
template <class C> __device__ inline float scale_of(float top) {
    return top < INFINITY ? top / Code<C>::kLargest : __uint_as_float(0x7fc00000u);
}

// Two 16-bit elements as a word.
template <class T> __device__ inline uint32_t word(float lo, float hi) {
    if constexpr (std::is_same<T, __half>::value) {
        const __half2 v = __floats2half2_rn(lo, hi);
        return reinterpret_cast<const uint32_t&>(v);
    } else {
        const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return reinterpret_cast<const uint32_t&>(v);
    }
}
template <class T> __device__ inline float2 floats(uint32_t w) {
    if constexpr (std::is_same<T, __half>::value) return __half22float2(reinterpret_cast<const __half2&>(w));
    else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// A thread's elements of a row, from and to memory, in runs whose neighbours belong to the
// next thread, so that a warp's accesses are of whole lines: runs of 4 where that fills 16
// bytes on one side, else of 8.
template <int kElements, int kThreads, int kRun> struct Piece {
    static constexpr int kRuns = kElements / kRun;
    int lane;
    __device__ int at(int run) const { return (run * kThreads + lane) * kRun; }

    __device__ void load(const float* p, int dim, float* x) const {
#pragma unroll
        for (int i = 0; i < kRuns; ++i)
            if (at(i) < dim) {
                const float4 a = *(const float4*)(p + at(i));
                x[4 * i] = a.x, x[4 * i + 1] = a.y, x[4 * i + 2] = a.z, x[4 * i + 3] = a.w;
            }
    }
    __device__ void store(float* p, int dim, const float* x) const {
#pragma unroll
        for (int i = 0; i < kRuns; ++i)
            if (at(i) < dim) *(float4*)(p + at(i)) = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
    }
    // 16-bit elements: two to a word
    template <class T> __device__ void load(const T* p, int dim, float* x) const {
#pragma unroll
        for (int i = 0; i < kRuns; ++i)
            if (at(i) < dim) {
                uint32_t w[kRun / 2];
                if constexpr (kRun == 4) {
                    const uint2 a = *(const uint2*)(p + at(i));
                    w[0] = a.x, w[1] = a.y;
                } else {
                    const uint4 a = *(const uint4*)(p + at(i));
                    w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
                }
#pragma unroll
                for (int k = 0; k < kRun / 2; ++k) {
                    const float2 f = floats<T>(w[k]);
                    x[kRun * i + 2 * k] = f.x, x[kRun * i + 2 * k + 1] = f.y;
                }
            }
    }
    template <class T> __device__ void store(T* p, int dim, const float* x) const {
#pragma unroll
        for (int i = 0; i < kRuns; ++i)
            if (at(i) < dim) {
                uint32_t w[kRun / 2];
#pragma unroll
                for (int k = 0; k < kRun / 2; ++k) w[k] = word<T>(x[kRun * i + 2 * k], x[kRun * i + 2 * k + 1]);
                if constexpr (kRun == 4) *(uint2*)(p + at(i)) = make_uint2(w[0], w[1]);
                else *(uint4*)(p + at(i)) = make_uint4(w[0], w[1], w[2], w[3]);
            }
    }
    template <class C> __device__ void store_codes(C* p, int dim, float (&x)[kElements], float s) const {
        uint32_t w[kElements / 4] = {};
        if (s > 0.0f) {
            const Divisor by(s, x, Code<C>::kLargest);
#pragma unroll
            for (int k = 0; k < kElements / 4; ++k) w[k] = Code<C>::pack4(x + 4 * k, by);
        }
#pragma unroll
        for (int i = 0; i < kRuns; ++i)
            if (at(i) < dim) {
                if constexpr (kRun == 4) *(uint32_t*)(p + at(i)) = w[i];
                else *(uint2*)(p + at(i)) = make_uint2(w[2 * i], w[2 * i + 1]);
            }
    }
    template <class C> __device__ void load_codes(const C* p, int dim, float* x) const {
#pragma unroll
        for (int i = 0; i < kRuns; ++i)
            if (at(i) < dim) {
                uint32_t w[kRun / 4];
                if constexpr (kRun == 4) {
                    w[0] = *(const uint32_t*)(p + at(i));
                } else {
                    const uint2 a = *(const uint2*)(p + at(i));
                    w[0] = a.x, w[1] = a.y;
                }
#pragma unroll
                for (int k = 0; k < kRun / 4; ++k) Code<C>::unpack4(w[k], x + kRun * i + 4 * k);
            }
    }
};
template <class X, class C, int kElements, int kThreads>
using PieceOf = Piece<kElements, kThreads, sizeof(X) == 4 || sizeof(C) == 4 || kElements == 4 ? 4 : 8>;

__device__ inline int64_t slot_of(const RowArgs& a, int64_t token) {
    return a.slots64 ? ((const int64_t*)a.slots)[token * a.slot_stride]
                     : (int64_t)((const int32_t*)a.slots)[token * a.slot_stride];
}

__device__ inline int64_t cache_offset(const CacheView& c, uint32_t page, uint32_t token, uint32_t head) {
    return (int64_t)page * c.page + (int64_t)token * c.token + (int64_t)head * c.head;
}

constexpr int kRowThreads = 256;
constexpr int kPerLane = kMaxHeadDim / 32;

template <class X, class C>
__global__ void __launch_bounds__(kRowThreads) cache_write_rows(const RowArgs a) {
    asm volatile("griddepcontrol.launch_dependents;\n\tgriddepcontrol.wait;" ::: "memory");
    constexpr bool kScaled = sizeof(C) == 1;
    const int lane = threadIdx.x & 31, which = a.first + blockIdx.y;
    const int64_t stride = (int64_t)gridDim.x * (kRowThreads / 32);
    for (int64_t row = (int64_t)blockIdx.x * (kRowThreads / 32) + (threadIdx.x >> 5); row < a.row_count; row += stride) {
        uint32_t head;
        const uint32_t token = a.heads.div((uint32_t)row, &head);
        const int64_t slot = slot_of(a, token);
        if (slot < 0 || slot >= a.total_slots) continue;
        uint32_t at;
        const uint32_t page = a.page.div((uint32_t)slot, &at);
        const X* x = (const X*)a.rows[which].ptr + (int64_t)token * a.rows[which].token + (int64_t)head * a.rows[which].head;
        C* c = (C*)a.cache[which].ptr + cache_offset(a.cache[which], page, at, head);
        float v[kPerLane];
#pragma unroll
        for (int i = 0; i < kPerLane; ++i) v[i] = lane + 32 * i < a.head_dim ? to_float(x[lane + 32 * i]) : 0.0f;
        if constexpr (kScaled) {
            float top = 0.0f;
#pragma unroll
            for (int i = 0; i < kPerLane; ++i) top = largest(top, fabsf(v[i]));
#pragma unroll
            for (int i = 1; i < 32; i <<= 1) top = largest(top, __shfl_xor_sync(0xffffffffu, top, i));
            const float s = scale_of<C>(top);
            if (lane == 0)
                ((float*)a.scale[which].ptr)[cache_offset(a.scale[which], page, at, head)] = s;
            const bool none = !(s > 0.0f);
            const Divisor by(s, v, Code<C>::kLargest);
#pragma unroll
            for (int i = 0; i < kPerLane; ++i)
                if (lane + 32 * i < a.head_dim) c[lane + 32 * i] = none ? C(0.0f) : Code<C>::of(v[i], by);
        } else {
#pragma unroll
            for (int i = 0; i < kPerLane; ++i)
                if (lane + 32 * i < a.head_dim) c[lane + 32 * i] = from_float<C>(v[i]);
        }
    }
}

template <class X, class C>
__global__ void __launch_bounds__(kRowThreads) cache_read_rows(const RowArgs a) {
    asm volatile("griddepcontrol.launch_dependents;\n\tgriddepcontrol.wait;" ::: "memory");
    constexpr bool kScaled = sizeof(C) == 1;
    const int lane = threadIdx.x & 31, which = a.first + blockIdx.y;
    const int64_t stride = (int64_t)gridDim.x * (kRowThreads / 32);
    for (int64_t row = (int64_t)blockIdx.x * (kRowThreads / 32) + (threadIdx.x >> 5); row < a.row_count; row += stride) {
        uint32_t head;
        const uint32_t token = a.heads.div((uint32_t)row, &head);
        const int64_t slot = slot_of(a, token);
        const bool there = slot >= 0 && slot < a.total_slots;
        uint32_t at;
        const uint32_t page = a.page.div(there ? (uint32_t)slot : 0u, &at);
        X* x = (X*)a.rows[which].ptr + (int64_t)token * a.rows[which].token + (int64_t)head * a.rows[which].head;
        const C* c = (const C*)a.cache[which].ptr + cache_offset(a.cache[which], page, at, head);
        float s = 1.0f;
        if constexpr (kScaled)
            if (there) s = ((const float*)a.scale[which].ptr)[cache_offset(a.scale[which], page, at, head)];
#pragma unroll
        for (int i = 0; i < kPerLane; ++i) {
            const int d = lane + 32 * i;
            if (d < a.head_dim) x[d] = from_float<X>(there ? (kScaled ? to_float(c[d]) * s : to_float(c[d])) : 0.0f);
        }
    }
}

// The same in pieces: kThreads threads (a power of two) a row, kElements of it a thread. With
// many rows 16 or 24 elements, and the rows of K and of V together; with few, where a call takes as
// long as one thread's work does, 4 or 8, and K and V in different blocks (gridDim.y = 2).
template <class X, class C, int kElements, int kThreads>
__global__ void __launch_bounds__(kRowThreads) cache_write_pieces(const RowArgs a) {
    asm volatile("griddepcontrol.launch_dependents;\n\tgriddepcontrol.wait;" ::: "memory");
    constexpr bool kScaled = sizeof(C) == 1;
    constexpr int kGroups = kRowThreads / kThreads;
    constexpr bool kBoth = kElements >= 16;
    const PieceOf<X, C, kElements, kThreads> piece{(int)(threadIdx.x % kThreads)};
    const int from = kBoth ? 0 : blockIdx.y, to = kBoth ? 2 : from + 1;
    const uint32_t count = (uint32_t)a.row_count;
    // every thread of a warp takes every turn: a row's threads exchange their largest elements
    for (uint32_t base = blockIdx.x * kGroups; base < count; base += gridDim.x * kGroups) {
        const uint32_t row = base + threadIdx.x / kThreads;
        uint32_t head, at;
        const uint32_t token = a.heads.div(row < count ? row : 0, &head);
        const int64_t slot = row < count ? slot_of(a, token) : -1;
        float x[kBoth ? 2 : 1][kElements] = {};
        if (row < count)
#pragma unroll
            for (int i = from; i < to; ++i)
                piece.load((const X*)a.rows[i].ptr + (int64_t)token * a.rows[i].token + (int64_t)head * a.rows[i].head, a.head_dim,
                           x[kBoth ? i : 0]);
        const bool there = slot >= 0 && slot < a.total_slots;
        const uint32_t page = a.page.div(there ? (uint32_t)slot : 0, &at);
#pragma unroll
        for (int i = from; i < to; ++i) {
            auto& xi = x[kBoth ? i : 0];
            C* const c = (C*)a.cache[i].ptr + cache_offset(a.cache[i], page, at, head);
            if constexpr (kScaled) {
                float top = 0.0f;
#pragma unroll
                for (int k = 0; k < kElements; ++k) top = largest(top, fabsf(xi[k]));
#pragma unroll
                for (int k = 1; k < kThreads; k <<= 1) top = largest(top, __shfl_xor_sync(0xffffffffu, top, k));
                if (!there) continue;
                const float s = scale_of<C>(top);
                if (piece.lane == 0) ((float*)a.scale[i].ptr)[cache_offset(a.scale[i], page, at, head)] = s;
                piece.store_codes(c, a.head_dim, xi, s);
            } else {
                if (there) piece.store(c, a.head_dim, xi);
            }
        }
    }
}

template <class X, class C, int kElements, int kThreads>
__global__ void __launch_bounds__(kRowThreads) cache_read_pieces(const RowArgs a) {
    asm volatile("griddepcontrol.launch_dependents;\n\tgriddepcontrol.wait;" ::: "memory");
    constexpr bool kScaled = sizeof(C) == 1;
    constexpr int kGroups = kRowThreads / kThreads;
    constexpr bool kBoth = kElements >= 16;
    const PieceOf<X, C, kElements, kThreads> piece{(int)(threadIdx.x % kThreads)};
    const int from = kBoth ? 0 : blockIdx.y, to = kBoth ? 2 : from + 1;
    const uint32_t count = (uint32_t)a.row_count;
    for (uint32_t row = blockIdx.x * kGroups + threadIdx.x / kThreads; row < count; row += gridDim.x * kGroups) {
        uint32_t head, at;
        const uint32_t token = a.heads.div(row, &head);
        const int64_t slot = slot_of(a, token);
        const bool there = slot >= 0 && slot < a.total_slots;
        const uint32_t page = a.page.div(there ? (uint32_t)slot : 0, &at);
        float x[kBoth ? 2 : 1][kElements] = {}, s[2] = {1.0f, 1.0f};
        if (there)
#pragma unroll
            for (int i = from; i < to; ++i) {
                if (!a.rows[i].ptr) continue;
                float* const xi = x[kBoth ? i : 0];
                const C* const c = (const C*)a.cache[i].ptr + cache_offset(a.cache[i], page, at, head);
                if constexpr (kScaled) {
                    s[i] = ((const float*)a.scale[i].ptr)[cache_offset(a.scale[i], page, at, head)];
                    piece.load_codes(c, a.head_dim, xi);
                } else {
                    piece.load(c, a.head_dim, xi);
                }
            }
#pragma unroll
        for (int i = from; i < to; ++i) {
            if (!a.rows[i].ptr) continue;
            float* const xi = x[kBoth ? i : 0];
            if constexpr (kScaled)
#pragma unroll
                for (int k = 0; k < kElements; ++k) xi[k] *= s[i];
            piece.store((X*)a.rows[i].ptr + (int64_t)token * a.rows[i].token + (int64_t)head * a.rows[i].head, a.head_dim, xi);
        }
    }
}

template <class X, class C, int kElements, int kThreads>
int launch_pieces(bool write, const RowArgs& a, int sms, cudaStream_t st) {
    const int64_t groups = kRowThreads / kThreads, want = (a.row_count + groups - 1) / groups;
    const int64_t resident = (int64_t)sms * 4;  // 64 registers a thread
    const dim3 grid((unsigned)(want < resident ? want : resident), kElements >= 16 ? 1 : 2);
    if (write)
        RT_CHECK(launch_early(cache_write_pieces<X, C, kElements, kThreads>, grid, kRowThreads, 0, st, a));
    else
        RT_CHECK(launch_early(cache_read_pieces<X, C, kElements, kThreads>, grid, kRowThreads, 0, st, a));
    return 0;
}

template <class X, class C>
int launch_rows(bool write, const RowArgs& a, int sms, cudaStream_t st) {
    if (a.pieces) {
        // few: not even one block an SM at 16 elements a thread. One token of 16 sequences, 8 heads of
        // 128, bf16 to e4m3: 2.5 us with 4 elements a thread, 5.5 with 16.
        const bool few = a.row_count * ((a.head_dim + 15) / 16) < (int64_t)sms * kRowThreads;
        // Many: 16 elements, or 24 where 5 or 6 threads would not be a power of two. 2^25 elements fp16 ->
        // e4m3 in rows of 32: 26 us, 53 with 4 threads a row; of 80: 34 us, 44 with 8 threads of 16.
        if (a.head_dim <= 32 && !few) return launch_pieces<X, C, 16, 2>(write, a, sms, st);
        if (a.head_dim <= 64) return few ? launch_pieces<X, C, 4, 16>(write, a, sms, st) : launch_pieces<X, C, 16, 4>(write, a, sms, st);
        if (a.head_dim > 64 && a.head_dim <= 96 && !few) return launch_pieces<X, C, 24, 4>(write, a, sms, st);
        if (a.head_dim <= 128) return few ? launch_pieces<X, C, 4, 32>(write, a, sms, st) : launch_pieces<X, C, 16, 8>(write, a, sms, st);
        return few ? launch_pieces<X, C, 8, 32>(write, a, sms, st) : launch_pieces<X, C, 16, 16>(write, a, sms, st);
    }
    const int64_t want = (a.row_count + kRowThreads / 32 - 1) / (kRowThreads / 32);
    const dim3 grid((unsigned)(want < (int64_t)sms * 8 ? want : (int64_t)sms * 8), a.count);
    if (write)
        RT_CHECK(launch_early(cache_write_rows<X, C>, grid, kRowThreads, 0, st, a));
    else
        RT_CHECK(launch_early(cache_read_rows<X, C>, grid, kRowThreads, 0, st, a));
    return 0;
}

template <class X>
int launch_cache_type(int dtype, bool write, const RowArgs& a, int sms, cudaStream_t st) {
    switch (dtype) {
        case MT_F32: return launch_rows<X, float>(write, a, sms, st);
        case MT_F16: return launch_rows<X, __half>(write, a, sms, st);
        case MT_BF16: return launch_rows<X, __nv_bfloat16>(write, a, sms, st);
        case MT_I8: return launch_rows<X, int8_t>(write, a, sms, st);
        default: return launch_rows<X, __nv_fp8_e4m3>(write, a, sms, st);
    }
}

int move_rows(const char* who, bool write, int dev, const mt_array* k, const mt_array* v, const mt_paged_cache* cache,
              const mt_array* slots, void* stream) {
    CacheShape c;
    if (int rc = check_cache(who, cache, write, &c)) return rc;
    if (!k && !v) return bad_argument("%s: k and v are missing", who);
    const uint32_t types = 1u << MT_F32 | 1u << MT_F16 | 1u << MT_BF16;
    if (int rc = check_array(who, "slots", slots, 1, 1u << MT_I32 | 1u << MT_I64, false)) return rc;
    RowArgs a{};
    int dtype = -1;
    bool pieces = c.head_dim % 8 == 0;
    for (int i = 0; i < 2; ++i) {
        const mt_array* x = i ? v : k;
        const char* name = i ? "v" : "k";
        if (!x) continue;
        if (int rc = check_array(who, name, x, 3, types, true)) return rc;
        if (x->shape[1] != c.kv_heads || x->shape[2] != c.head_dim)
            return bad_argument("%s: %s must be [tokens, %d, %d] as the cache's heads are", who, name, c.kv_heads, c.head_dim);
        if (x->shape[0] != slots->shape[0])
            return bad_argument("%s: %s has %lld tokens, slots %lld", who, name, (long long)x->shape[0],
                                (long long)slots->shape[0]);
        if (dtype >= 0 && dtype != x->dtype) return bad_argument("%s: k and v must have one type", who);
        dtype = x->dtype;
        if (!write)
            if (int rc = check_written(who, name, *x)) return rc;
        a.rows[i] = {x->ptr, x->strides[0], x->strides[1]};
        const int align = 8 * bytes_of(c.dtype) < 16 ? 8 : 16;
        pieces = pieces && rows_aligned(*x, 16) && rows_aligned(i ? cache->v : cache->k, align);
    }
    a.pieces = pieces;
    a.first = k ? 0 : 1;
    a.count = (k ? 1 : 0) + (v ? 1 : 0);
    const int64_t tokens = slots->shape[0];
    if (tokens > INT32_MAX / c.kv_heads) return bad_argument("%s: over 2^31 - 1 rows in one call", who);
    if (tokens == 0) return 0;
    if (c.pages == 0 && write) return 0;  // every slot is outside the cache
    a.cache[0] = c.k;
    a.cache[1] = c.v;
    a.scale[0] = c.k_scale;
    a.scale[1] = c.v_scale;
    a.slots = slots->ptr;
    a.slot_stride = slots->strides[0];
    a.slots64 = slots->dtype == MT_I64;
    a.total_slots = c.pages * c.page_size;
    a.head_dim = c.head_dim;
    a.row_count = tokens * c.kv_heads;
    a.heads = FastDiv((uint32_t)c.kv_heads);
    a.page = FastDiv((uint32_t)c.page_size);
    cudaStream_t st;
    OnDevice on;
    RT_CHECK(on.enter(dev));
    if (int rc = call_stream(dev, stream, &st)) return rc;
    int sms;
    if (int rc = sm_count(dev, &sms)) return rc;
    switch (dtype) {
        case MT_F32: return launch_cache_type<float>(c.dtype, write, a, sms, st);
        case MT_F16: return launch_cache_type<__half>(c.dtype, write, a, sms, st);
        default: return launch_cache_type<__nv_bfloat16>(c.dtype, write, a, sms, st);
    }
}

}  // namespace

extern "C" {

int mt_cache_write(int dev, const mt_array* k, const mt_array* v, const mt_paged_cache* cache, const mt_array* slots,
                   void* stream) {
    if (!k || !v) return bad_argument("cache_write: k and v are both needed");
    return move_rows("cache_write", true, dev, k, v, cache, slots, stream);
}

int mt_cache_read(int dev, const mt_paged_cache* cache, const mt_array* slots, const mt_array* k, const mt_array* v,
                  void* stream) {
    return move_rows("cache_read", false, dev, k, v, cache, slots, stream);
}

}  // extern "C"
