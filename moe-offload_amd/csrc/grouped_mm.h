// What the grouped products of unquantised experts share: the operands' description, the check of a
// call's arguments, and the search for a block's tile.
#pragma once
#include "moe_common.h"

namespace gmm {

constexpr int kMaxSeg = 1024;

// Rows r of segment s: seg_start[s] .. seg_start[s + 1] - 1, weights of slot seg_slot[s] (s where null).
struct Segs {
    const int32_t* start;
    const int32_t* slot;
    int n_seg, n_rows, n_slots, fill;
};

// Block index -> work item, keeping consecutive items on one XCD (blocks are dealt to the 8 XCDs round
// robin), so that the blocks of one row tile find its rows in that XCD's L2.
__device__ __forceinline__ uint32_t xcd_order(uint32_t b, uint32_t nb) {
    const uint32_t per = nb / 8, rem = nb % 8, x = b % 8, i = b / 8;
    return x < rem ? x * (per + 1) + i : rem * (per + 1) + (x - rem) * per + i;
}

// Rows and slot of virtual segment v: 0 the rows before the first segment, 1 .. n_seg the segments, and
// n_seg + 1 the rows behind the last.  slot < 0: rows that no weights apply to; they have no tiles
// unless they are to be filled with zeros.
__device__ __forceinline__ void seg_rows(const Segs& S, int v, int& r0, int& r1, int& slot) {
    auto at = [&](int i) {
        const int r = S.start[i];
        return r < 0 ? 0 : r > S.n_rows ? S.n_rows : r;
    };
    slot = -1;
    if (v == 0) {
        r0 = 0;
        r1 = at(0);
    } else if (v <= S.n_seg) {
        r0 = at(v - 1);
        r1 = at(v);
        slot = S.slot ? S.slot[v - 1] : v - 1;
        if (slot >= S.n_slots) slot = -1;
    } else {
        r0 = at(S.n_seg);
        r1 = S.n_rows;
    }
    if (r1 < r0) r1 = r0;
    if (slot < 0 && !S.fill) r1 = r0;
}

__device__ __forceinline__ uint32_t tiles_of(int rows, int bm) { return ((uint32_t)rows + bm - 1) / (uint32_t)bm; }

struct Tile {
    int r0, r1, slot, col;            // rows of the tile, weights' slot (-1: none), column tile
};

// The row tile (bm rows of one segment at most) and column tile of this block; false: none is left for it.
// Every thread sums the tiles of its own few segments, a scan over the block turns the sums into first
// tiles, and the thread whose segments hold the block's item publishes it.
template <int THREADS>
__device__ __forceinline__ bool find_tile(const Segs& S, int bm, int n_col, Tile& out) {
    __shared__ uint32_t wave_sum[THREADS / 64];
    __shared__ int found[3];
    const int t = threadIdx.x, lane = t & 63, wv = t >> 6;
    const int n_virtual = S.n_seg + 2, per = (n_virtual + THREADS - 1) / THREADS;
    const int v0 = t * per, v1 = v0 + per < n_virtual ? v0 + per : n_virtual;
    int r0 = 0, r1 = 0, slot = -1;
    uint32_t sum = 0;
    for (int v = v0; v < v1; ++v) {
        seg_rows(S, v, r0, r1, slot);
        sum += tiles_of(r1 - r0, bm);
    }
    uint32_t inc = sum;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t o = __shfl_up(inc, d, 64);
        if (lane >= d) inc += o;
    }
    if (lane == 63) wave_sum[wv] = inc;
    __syncthreads();
    uint32_t first = inc - sum, total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
        if (w < wv) first += wave_sum[w];
        total += wave_sum[w];
    }
    if (blockIdx.x >= (uint64_t)total * n_col) return false;
    const uint32_t item = xcd_order(blockIdx.x, total * (uint32_t)n_col), row_tile = item / (uint32_t)n_col;
    if (row_tile >= first && row_tile < first + sum) {
        uint32_t p = first;
        for (int v = v0; v < v1; ++v) {
            seg_rows(S, v, r0, r1, slot);
            const uint32_t c = tiles_of(r1 - r0, bm);
            if (row_tile < p + c) {
                const int a = r0 + (int)(row_tile - p) * bm;
                found[0] = a;
                found[1] = a + bm < r1 ? a + bm : r1;
                found[2] = slot;
                break;
            }
            p += c;
        }
    }
    __syncthreads();
    out.r0 = __builtin_amdgcn_readfirstlane(found[0]);
    out.r1 = __builtin_amdgcn_readfirstlane(found[1]);
    out.slot = __builtin_amdgcn_readfirstlane(found[2]);
    out.col = (int)(item % (uint32_t)n_col);
    return true;
}

}  // namespace gmm
