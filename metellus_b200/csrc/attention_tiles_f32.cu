// Paged attention in tiles over a cache of f32 (a file of its own: they compile in parallel).
#include "attention_tiles.cuh"

namespace mt {

int attend_tiles_f32(const AttentionArgs& a, bool run, void* workspace, uint64_t* bytes, int dev, cudaStream_t st) {
    return tiles::by_shape<MT_F32, float>(a, run, workspace, bytes, dev, st);
}

}  // namespace mt
