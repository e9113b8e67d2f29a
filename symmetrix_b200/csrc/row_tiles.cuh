// Tiles of rows that never mix groups: what a CTA of the linears with adapters finds its work with. (Linears of routed rows walk degrees and blocks of
// columns as well, in an order of their own: csrc/grouped_f32.cuh, csrc/grouped_f64.cuh.)
#pragma once

namespace smx {
namespace {

// Rows of a tile: pairs [pair0, pair0 + ...) of one group, rows counted in components from row0 of the group.
struct TileRows { int group; long long first_pair, row0, rows; };

// The tile-th tile of `size` rows, groups one after the other (group `groups`: the pairs behind the last group, if `tail`); false, and the number
// of tiles, if there is none. Called by one warp.
__device__ __forceinline__ bool find_tile(const int* __restrict__ offsets, int groups, bool tail, long long pairs, int comps, int size, long long tile,
                                          TileRows& out, long long& tiles_in_all) {
    const int lane = threadIdx.x & 31;
    long long run = 0;
    for (int g0 = 0; g0 <= groups; g0 += 32) {
        const int g = g0 + lane;
        long long first = 0, rows = 0;
        if (g < groups || (g == groups && tail)) {
            first = offsets[g];
            rows = ((g < groups ? offsets[g + 1] : pairs) - first) * comps;
        }
        const long long tiles = (rows + size - 1) / size;
        long long incl = tiles;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const long long up = __shfl_up_sync(0xffffffffu, incl, d);
            if (lane >= d) incl += up;
        }
        const long long begin = run + incl - tiles;
        const unsigned hit = __ballot_sync(0xffffffffu, tile >= begin && tile < begin + tiles);
        if (hit) {
            const int src = __ffs(hit) - 1;
            out.group = __shfl_sync(0xffffffffu, g, src);
            out.first_pair = __shfl_sync(0xffffffffu, first, src);
            const long long b = __shfl_sync(0xffffffffu, begin, src), r = __shfl_sync(0xffffffffu, rows, src);
            out.row0 = (tile - b) * size;
            out.rows = min(static_cast<long long>(size), r - out.row0);
            return true;
        }
        run += __shfl_sync(0xffffffffu, incl, 31);
    }
    tiles_in_all = run;
    return false;
}

}  // namespace
}  // namespace smx
