// Paged attention in tiles over a cache of int8 (a file of its own: they compile in parallel).
#include "attention_tiles.cuh"

namespace mt {

int attend_tiles_i8(const AttentionArgs& a, bool run, void* workspace, uint64_t* bytes, int dev, cudaStream_t st) {
    if (a.q_type == MT_F16) return tiles::by_shape<MT_I8, __half>(a, run, workspace, bytes, dev, st);
    if (a.q_type == MT_BF16) return tiles::by_shape<MT_I8, __nv_bfloat16>(a, run, workspace, bytes, dev, st);
    return tiles::by_shape<MT_I8, float>(a, run, workspace, bytes, dev, st);
}

}  // namespace mt
