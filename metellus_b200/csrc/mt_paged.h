// Paged key-value cache: what the host checks and the kernels share.
#ifndef METELLUS_MT_PAGED_H
#define METELLUS_MT_PAGED_H

#include <cstdint>

#include "mt_host.h"

namespace mt {

constexpr int kMaxHeadDim = 256;

// Quotient and remainder by a divisor that is known on the host: for n < 2^31,
// n / d = (umulhi(n, magic) + n) >> shift with shift = ceil(log2 d).
struct FastDiv {
    uint32_t d = 1, magic = 0, shift = 0;
    FastDiv() = default;
    explicit FastDiv(uint32_t divisor) : d(divisor) {
        while ((1ull << shift) < d) ++shift;
        magic = (uint32_t)(((1ull << 32) * ((1ull << shift) - d)) / d + 1);
    }
    __host__ __device__ uint32_t div(uint32_t n) const {
#ifdef __CUDA_ARCH__
        return (__umulhi(n, magic) + n) >> shift;
#else
        return (uint32_t)((((uint64_t)n * magic >> 32) + n) >> shift);
#endif
    }
    __host__ __device__ uint32_t div(uint32_t n, uint32_t* rem) const {
        const uint32_t q = div(n);
        *rem = n - q * d;
        return q;
    }
};

// One of a cache's arrays: element (page, token, head[, dim]).
struct CacheView {
    void* ptr = nullptr;
    int64_t page = 0, token = 0, head = 0;  // strides in elements
};

// Cache geometry after the checks.
struct CacheShape {
    int dtype = 0, pages = 0, page_size = 1, kv_heads = 1, head_dim = 1;
    CacheView k, v, k_scale, v_scale;
    bool scaled() const { return dtype == MT_I8 || dtype == MT_E4M3; }
};

inline int bytes_of(int dtype) {
    switch (dtype) {
        case MT_F32: case MT_I32: return 4;
        case MT_F16: case MT_BF16: return 2;
        case MT_I8: case MT_E4M3: return 1;
        case MT_I64: return 8;
        default: return 0;
    }
}

const char* dtype_name(int dtype);
// Number of elements (0 for an empty array).
int64_t elements(const mt_array& a);
// An array of `ndim` dimensions of one of the types in `dtypes` (a bit set), with a pointer (unless empty) aligned to its
// element, positive extents in range and, where `last1`, the last stride 1 (any where that extent is 1).
int check_array(const char* who, const char* name, const mt_array* a, int ndim, uint32_t dtypes, bool last1);
// No two elements of an array that is written may share an address: rejects zero strides.
int check_written(const char* who, const char* name, const mt_array& a);
int check_cache(const char* who, const mt_paged_cache* cache, bool written, CacheShape* out);
// Whether rows of `row_bytes` bytes at this array's addresses start on `align` bytes (all strides but the last).
bool rows_aligned(const mt_array& a, int align);

}  // namespace mt

#endif
