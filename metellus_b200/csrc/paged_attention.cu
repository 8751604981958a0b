// Attention of one new token per sequence over a paged key-value cache
// (mt_paged_attention): argument checks and the choice of the kernel.
#include <cmath>

#include "mt_paged_attention.h"

namespace mt {

namespace {

// Whether an array's rows, whose strides are multiples of `least` bytes, can be numbered in 32 bits.
bool number_rows(const CacheView& view, const CacheShape& c, int bytes, uint32_t least, RowNumbers* out) {
    const int64_t page = view.page * bytes, token = view.token * bytes;
    uint32_t unit = least;
    while (unit < (1u << 20) && page % (2 * unit) == 0 && token % (2 * unit) == 0) unit *= 2;
    *out = {(uint32_t)(page / unit), (uint32_t)(token / unit), unit};
    const double last = (double)(c.pages - 1) * (double)(page / unit) + (double)(c.page_size - 1) * (double)(token / unit);
    return last < 4294967296.0;
}

int check_attention(const char* who, const mt_array* q, const mt_paged_cache* cache, const mt_array* tables,
                    int64_t window, AttentionArgs* a, int* batch, int* heads, bool* tiled) {
    CacheShape c;
    if (int rc = check_cache(who, cache, false, &c)) return rc;
    if (int rc = check_array(who, "q", q, 3, 1u << MT_F32 | 1u << MT_F16 | 1u << MT_BF16, true)) return rc;
    if (q->shape[2] != c.head_dim)
        return bad_argument("%s: q has head_dim %lld, the cache %d", who, (long long)q->shape[2], c.head_dim);
    if (q->shape[1] < 1 || q->shape[1] % c.kv_heads)
        return bad_argument("%s: %lld query heads are not a multiple of %d key-value heads", who,
                            (long long)q->shape[1], c.kv_heads);
    if (q->shape[1] > 65535 || q->shape[0] > 65535 * 32)
        return bad_argument("%s: at most %d sequences of 65535 heads", who, 65535 * 32);
    if (q->dtype != MT_F32 && !c.scaled() && q->dtype != c.dtype)
        return bad_argument("%s: q of %s does not go with a cache of %s", who, dtype_name(q->dtype),
                            dtype_name(c.dtype));
    if (window < 0) return bad_argument("%s: window must not be negative", who);
    if (int rc = check_array(who, "tables", tables, 2, 1u << MT_I32, true)) return rc;
    if (tables->shape[0] != q->shape[0])
        return bad_argument("%s: tables has %lld rows, q %lld", who, (long long)tables->shape[0], (long long)q->shape[0]);
    // the kernels count tokens in int, up to a few hundred past the end
    if (tables->shape[1] > (INT32_MAX - 1024) / c.page_size)
        return bad_argument("%s: the tables' width allows over 2^31 - 1025 tokens", who);
    a->q = q->ptr;
    a->q_seq = q->strides[0];
    a->q_head = q->strides[1];
    a->cache = c;
    a->tables = (const int32_t*)tables->ptr;
    a->table_seq = tables->strides[0];
    a->max_tokens = (int)tables->shape[1] * c.page_size;
    a->page = FastDiv((uint32_t)c.page_size);
    a->group = (int)(q->shape[1] / c.kv_heads);
    a->q_type = q->dtype;
    *batch = a->batch = (int)q->shape[0];
    *heads = (int)q->shape[1];
    a->window = window == 0 || window > INT32_MAX ? INT32_MAX : (int)window;
    const int bytes = bytes_of(c.dtype);
    *tiled = c.head_dim * bytes % 16 == 0 && rows_aligned(cache->k, 16) && rows_aligned(cache->v, 16) &&
             number_rows(c.k, c, bytes, 16, &a->k_rows) && number_rows(c.v, c, bytes, 16, &a->v_rows);
    if (*tiled && c.scaled())
        *tiled = number_rows(c.k_scale, c, 4, 4, &a->k_scale_rows) && number_rows(c.v_scale, c, 4, 4, &a->v_scale_rows);
    return 0;
}

int attend_tiles(const AttentionArgs& a, bool run, void* workspace, uint64_t* bytes, int dev, cudaStream_t st) {
    switch (a.cache.dtype) {
        case MT_F32: return attend_tiles_f32(a, run, workspace, bytes, dev, st);
        case MT_F16: return attend_tiles_f16(a, run, workspace, bytes, dev, st);
        case MT_BF16: return attend_tiles_bf16(a, run, workspace, bytes, dev, st);
        case MT_I8: return attend_tiles_i8(a, run, workspace, bytes, dev, st);
        default: return attend_tiles_e4m3(a, run, workspace, bytes, dev, st);
    }
}

}  // namespace

}  // namespace mt

using namespace mt;

extern "C" {

int mt_paged_attention_workspace(int dev, const mt_array* q, const mt_paged_cache* cache, const mt_array* tables,
                                 int64_t window, uint64_t* bytes) {
    const char* who = "paged_attention_workspace";
    AttentionArgs a{};
    int batch, heads;
    bool tiled;
    if (!bytes) return bad_argument("%s: bytes is missing", who);
    if (int rc = check_attention(who, q, cache, tables, window, &a, &batch, &heads, &tiled)) return rc;
    *bytes = 0;
    return batch == 0 || !tiled ? 0 : attend_tiles(a, false, nullptr, bytes, dev, nullptr);
}

int mt_paged_attention(int dev, const mt_array* q, const mt_paged_cache* cache, const mt_array* tables,
                       const mt_array* lengths, const mt_array* out, const mt_array* lse, double scale,
                       int64_t window, void* workspace, uint64_t workspace_bytes, void* stream) {
    const char* who = "paged_attention";
    AttentionArgs a{};
    int batch, heads;
    bool tiled;
    if (int rc = check_attention(who, q, cache, tables, window, &a, &batch, &heads, &tiled)) return rc;
    if (int rc = check_array(who, "lengths", lengths, 1, 1u << MT_I32, false)) return rc;
    if (lengths->shape[0] != batch)
        return bad_argument("%s: lengths has %lld entries, q %d sequences", who, (long long)lengths->shape[0], batch);
    if (int rc = check_array(who, "out", out, 3, 1u << q->dtype, true)) return rc;
    for (int i = 0; i < 3; ++i)
        if (out->shape[i] != q->shape[i]) return bad_argument("%s: out must have q's shape", who);
    if (int rc = check_written(who, "out", *out)) return rc;
    if (lse) {
        if (int rc = check_array(who, "lse", lse, 2, 1u << MT_F32, false)) return rc;
        if (lse->shape[0] != batch || lse->shape[1] != heads)
            return bad_argument("%s: lse must be [batch, heads]", who);
        if (int rc = check_written(who, "lse", *lse)) return rc;
        a.lse = (float*)lse->ptr;
        a.lse_seq = lse->strides[0];
        a.lse_head = lse->strides[1];
    }
    if (!std::isfinite((float)scale)) return bad_argument("%s: scale must be finite", who);
    if (batch == 0) return 0;
    a.lengths = (const int32_t*)lengths->ptr;
    a.length_seq = lengths->strides[0];
    a.out = out->ptr;
    a.out_seq = out->strides[0];
    a.out_head = out->strides[1];
    a.scale = (float)scale;
    cudaStream_t st;
    OnDevice on;
    RT_CHECK(on.enter(dev));
    if (int rc = call_stream(dev, stream, &st)) return rc;
    if (!tiled || !(a.scale > 0.0f)) return attend_by_rows(a, dev, st);  // tiles mask and compare scores before they are scaled
    uint64_t need = 0;
    if (int rc = attend_tiles(a, false, nullptr, &need, dev, st)) return rc;
    if (need && !workspace && !stream) {
        // this library's stream: workspace from its pool, given back in the stream's order
        RT_CHECK(cudaMallocAsync(&workspace, need, st));
        const int rc = attend_tiles(a, true, workspace, &need, dev, st);
        RT_CHECK(cudaFreeAsync(workspace, st));
        return rc;
    }
    if (need && (!workspace || workspace_bytes < need))
        return bad_argument("%s: the workspace has %llu bytes, %llu are needed", who,
                            (unsigned long long)(workspace ? workspace_bytes : 0), (unsigned long long)need);
    if ((uintptr_t)workspace % 16) return bad_argument("%s: the workspace is not 16-byte aligned", who);
    return attend_tiles(a, true, workspace, &need, dev, st);
}

}  // extern "C"
