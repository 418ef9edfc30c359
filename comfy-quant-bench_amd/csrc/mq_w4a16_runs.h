// The order in which a wave of the w4a16 kernel takes its steps, apart from what a step does. Plain integers: the
// host checks it for every cut of the work.
#pragma once

#include <cstdint>

namespace mq {

// A wave takes `share` consecutive steps of every chunk of x (the workgroup's waves together `chunk_steps`) through a ring
// of KB places. Every chunk of every tile begins at place 0, so a run is counted in whole rounds of the ring: the places
// behind the share stay empty.
template <int W>
__host__ __device__ __forceinline__ int w4_share(int chunk_steps) {
    return (chunk_steps + W - 1) / W;
}
template <int KB>
__host__ __device__ __forceinline__ int w4_run(int share) {
    return (share + KB - 1) / KB * KB;
}

// The steps that are fetched into the places one after the other: step `blk` of tile `tile`, if any() says so.
template <bool THROUGH>
struct W4Fetch {
    int tile, blk;      // of the next place
    int at;             // of the run
    __host__ __device__ __forceinline__ W4Fetch(int first_tile, int wave, int share) : tile(first_tile), blk(wave * share), at(0) {}
    __host__ __device__ __forceinline__ bool any(int share, int steps, int tiles) const {
        return at < share && blk < steps && (!THROUGH || tile < tiles);
    }
    // on to the next place: of this run, of the wave's run of the next chunk, or (THROUGH) of the next tile
    __host__ __device__ __forceinline__ void next(int wave, int share, int run, int chunk_steps, int steps, int tile_step) {
        ++blk;
        if (++at < run) return;
        at = 0;
        blk += chunk_steps - run;
        if (THROUGH && blk - wave * share >= steps) {   // the runs of the last chunk are done
            blk = wave * share;
            tile += tile_step;
        }
    }
};

}  // namespace mq
