// Paged attention in tiles over a cache of bf16 (a file of its own: they compile in parallel).
#include "attention_tiles.cuh"

namespace mt {

int attend_tiles_bf16(const AttentionArgs& a, bool run, void* workspace, uint64_t* bytes, int dev, cudaStream_t st) {
    if (a.q_type == MT_BF16) return tiles::by_shape<MT_BF16, __nv_bfloat16>(a, run, workspace, bytes, dev, st);
    return tiles::by_shape<MT_BF16, float>(a, run, workspace, bytes, dev, st);
}

}  // namespace mt
