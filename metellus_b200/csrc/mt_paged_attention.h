// Paged attention: arguments after the checks, and the kernels' entry points.
#ifndef METELLUS_MT_PAGED_ATTENTION_H
#define METELLUS_MT_PAGED_ATTENTION_H

#include "mt_paged.h"

namespace mt {

// Rows of a cache array by 32-bit numbers: row (p, t) of a head is (p * page + t * token) * unit bytes
// behind the head's first. unit: the largest power of two that divides the strides.
struct RowNumbers {
    uint32_t page = 0, token = 0, unit = 0;
};

struct AttentionArgs {
    const void* q;
    int64_t q_seq, q_head;  // strides in elements
    void* out;
    int64_t out_seq, out_head;
    float* lse;  // may be null
    int64_t lse_seq, lse_head;
    const int32_t* tables;
    int64_t table_seq;
    const int32_t* lengths;
    int64_t length_seq;
    CacheShape cache;
    RowNumbers k_rows, v_rows, k_scale_rows, v_scale_rows;  // for the tiles
    FastDiv page;
    int q_type, batch, group, max_tokens, window;
    float scale;
};

// Any head_dim and alignment: one warp a key row (attention_rows.cu).
int attend_by_rows(const AttentionArgs& a, int dev, cudaStream_t st);

// Rows of the cache that 16-byte copies can fetch: tiles on the matrix pipe
// (attention_tiles.cuh), split over the sequences' lengths. `bytes`: the workspace needed,
// which is all that is found out unless `run`.
int attend_tiles_f32(const AttentionArgs& a, bool run, void* workspace, uint64_t* bytes, int dev, cudaStream_t st);
int attend_tiles_f16(const AttentionArgs& a, bool run, void* workspace, uint64_t* bytes, int dev, cudaStream_t st);
int attend_tiles_bf16(const AttentionArgs& a, bool run, void* workspace, uint64_t* bytes, int dev, cudaStream_t st);
int attend_tiles_i8(const AttentionArgs& a, bool run, void* workspace, uint64_t* bytes, int dev, cudaStream_t st);
int attend_tiles_e4m3(const AttentionArgs& a, bool run, void* workspace, uint64_t* bytes, int dev, cudaStream_t st);

}  // namespace mt

#endif
