// Paged attention in tiles over a cache of f16 (a file of its own: they compile in parallel).
#include "attention_tiles.cuh"

namespace mt {

int attend_tiles_f16(const AttentionArgs& a, bool run, void* workspace, uint64_t* bytes, int dev, cudaStream_t st) {
    if (a.q_type == MT_F16) return tiles::by_shape<MT_F16, __half>(a, run, workspace, bytes, dev, st);
    return tiles::by_shape<MT_F16, float>(a, run, workspace, bytes, dev, st);
}

}  // namespace mt
