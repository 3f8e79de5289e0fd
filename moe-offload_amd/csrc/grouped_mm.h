// What the grouped products of unquantised experts and the adapters share: the search for a block's rows, loads
// from global memory straight into LDS, and the matrix unit's operands read from there.
#pragma once
#include "moe_common.h"

namespace gmm {

constexpr int kMaxSeg = 1024;
constexpr int kMaxSide = 1 << 30;     // rows, columns and contractions: sums of two of them and a tile stay below 2^31
constexpr int64_t kMaxThreads = 0xFFFFFFFF;                   // of a launch, in a dimension

// Rows r of segment s: seg_start[s] .. seg_start[s + 1] - 1, weights of slot seg_slot[s] (s where null).
struct Segs {
    const int32_t* start;
    const int32_t* slot;
    int n_seg, n_rows, n_slots, fill;
};

// dx[rows[r]] = W_u^T (dv[3 rows[r]] + dv[3 rows[r] + 1] + dv[3 rows[r] + 2]), W_u [n][k] of dtype, dv three bf16 parts
// of a value each (bf16_parts); zeros for rows of no segment.  dry: launches nothing, -1 if one launch does not take it.
int dx_of_parts(const void* dv, const int32_t* rows, int n_rows, const int32_t* seg_start, int n_seg, const void* w,
                int64_t w_stride, int n, int k, void* dx, int64_t lddx, int dtype, bool dry, hipStream_t s);

// Block index -> work item, keeping consecutive items on one XCD (blocks are dealt to the 8 XCDs round
// robin), so that the blocks of one row tile find its rows in that XCD's L2.
__device__ __forceinline__ uint32_t xcd_order(uint32_t b, uint32_t nb) {
    const uint32_t per = nb / 8, rem = nb % 8, x = b % 8, i = b / 8;
    return x < rem ? x * (per + 1) + i : rem * (per + 1) + (x - rem) * per + i;
}

// Weights' gradients: blocks of one segment are as long as it is.  Up to kManySegs segments each is dealt to all 8 XCDs in
// runs of `run` items; more of them even out over whole shares of one XCD each, which read a row once.  us of gradients,
// dealt and in whole shares: 16 experts of 4096 x 1024, 1024 rows on average, with mm_dx 396 and 437 (of 1024 rows each, dw
// alone, 145 both ways), 8 adapters of 4096 tokens, all of lora_grad, 62.5 and 76.1; 512 experts of 1024 x 2048, 40 rows, 999 and 914.
constexpr int kManySegs = 128;

__device__ __forceinline__ uint32_t dealt(uint32_t b, uint32_t nb, uint32_t run) {
    const uint32_t i = b / 8;
    return b < nb / (8 * run) * (8 * run) ? (i / run * 8 + b % 8) * run + i % run : b;
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
// scratch: THREADS / 64 + 3 words of LDS, free again once every thread is back.
// Every thread sums the tiles of its own few segments, a scan over the block turns the sums into first
// tiles, and the thread whose segments hold the block's item publishes it.  (No thread does where seg_start is not in
// order and the sums wrap: the block then has no rows.)
template <int THREADS>
__device__ __forceinline__ bool find_tile(const Segs& S, int bm, int n_col, uint32_t* scratch, Tile& out) {
    uint32_t* wave_sum = scratch;
    int* found = (int*)(scratch + THREADS / 64);
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
    if (t == 0) found[0] = found[1] = 0;
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
    return out.r0 < out.r1;
}

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

template <typename T>
__device__ __forceinline__ f32x4 mfma(uint4 a, uint4 b, f32x4 c) {
    if constexpr (__is_same(T, _Float16))
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// An fp32 value as the sum of three bf16 values, each the upper half of what the ones before it leave: all of its 24 bits,
// over fp32's range (rounded parts would overflow near the largest values).  An infinity or NaN stays in the first part.
__device__ __forceinline__ void bf16_parts(float v, __bf16 (&p)[3]) {
    const bool fine = __builtin_fabsf(v) < __builtin_inff();
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        p[k] = fine ? __builtin_bit_cast(__bf16, (uint16_t)(__builtin_bit_cast(uint32_t, v) >> 16)) : (__bf16)v;
        v = fine ? v - (float)p[k] : 0.f;
    }
}

// c + a b, or (FIRST false) c + b a, where b is a part of such a value.  bf16: as it is.  fp16: a's 11 bits are two bf16
// values, the upper 8 and the other 3, so no value needs a scale.  (The fp32 matrix unit takes 16 times as long as one
// 16-bit product, two parts times three 6 times.)
template <typename T, bool FIRST = true>
__device__ __forceinline__ f32x4 mfma_parts(uint4 a, uint4 b, f32x4 c) {
    auto add = [&](uint4 part) { c = FIRST ? mfma<__bf16>(part, b, c) : mfma<__bf16>(b, part, c); };
    if constexpr (__is_same(T, _Float16)) {
        typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
        const f16x8 w = __builtin_bit_cast(f16x8, a);
        u16x8 hi, lo;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float f = (float)w[e];
            const uint32_t top = __builtin_bit_cast(uint32_t, f) & 0xFFFF0000u;
            const float rest = f - __builtin_bit_cast(float, top);
            hi[e] = (uint16_t)(top >> 16);                                     // (a NaN's quiet bit is among them)
            lo[e] = (uint16_t)(__builtin_bit_cast(uint32_t, __builtin_fmaxf(rest, -256.f)) >> 16);
        }
        add(__builtin_bit_cast(uint4, hi));
        add(__builtin_bit_cast(uint4, lo));
    } else {
        add(a);
    }
    return c;
}

template <typename T>
__device__ __forceinline__ uint2 round4(f32x4 v) {
    typedef T t4 __attribute__((ext_vector_type(4)));
    const t4 r = {(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
    return __builtin_bit_cast(uint2, r);
}

template <typename T>
__device__ __forceinline__ f32x4 widen4(uint2 w) {
    typedef T t4 __attribute__((ext_vector_type(4)));
    const t4 r = __builtin_bit_cast(t4, w);
    return (f32x4){(float)r[0], (float)r[1], (float)r[2], (float)r[3]};
}

// Two subtiles' 4 adjacent 16-bit results per lane -> 8 adjacent: lanes 16-31 and 48-63 take the second
// subtile.  Returns the 16 bytes and which subtile (0, 1) and half (0, 1) of its 16 columns they are.
__device__ __forceinline__ uint4 pair8(uint2 a, uint2 b) {
    const auto x = __builtin_amdgcn_permlane16_swap(a.x, b.x, false, false);
    const auto y = __builtin_amdgcn_permlane16_swap(a.y, b.y, false, false);
    return make_uint4(x[0], y[0], x[1], y[1]);
}

// 16 bytes out, past the caches.  Results are read again by the next launch at the earliest, and their lines
// wait in L2 for a write that then meets the next tile's loads: us with and without, weights' gradient 1024 x 2048 of 512 x
// 40 rows 377 and 607, 4096 x 1024 of 16 x 256 rows 63 and 74, mm 4096 x 1024 of 16 x 2048 rows 258 and 276, mm_dx 1024 x
// 2048 of 512 x 40 rows 431 and 441, gate_up 1024 x 4096 of 16 x 2048 rows 478 and 485.
__device__ __forceinline__ void store16(void* to, uint4 v) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    __builtin_nontemporal_store(__builtin_bit_cast(u32x4, v), (u32x4*)to);
}

// What an operand's lanes read where it has nothing: contraction indexes past the end.
static __device__ uint4 g_zero16;

// 16 bytes per lane from global memory straight into LDS: lane l's land at lds + 16 l (lds wave-uniform).
// The issuing code waits for them itself (vmcnt), and no register receives data.  m0, where the instruction finds the LDS
// address, is an operand, so that the compiler knows what it holds.
__device__ __forceinline__ void load_to_lds(const void* g, uint32_t lds) {
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"{m0}"(lds), "v"(g) : "memory");
}

constexpr int kBC = 64;                                       // contraction indexes per step
typedef __attribute__((address_space(3))) uint8_t lds_u8;

// Row of a step's image, along which the other index runs -> which 32-byte block trades places with block 0:
// the rows that one transposing read touches (4 of each of two or four lane groups) get eight different ones, or
// as many as a row of W values has.
template <int W>
__device__ __forceinline__ int turn(int row) {
    if constexpr (W >= 128) return (row & 3) | ((row >> 3) & 1) << 2;
    else if constexpr (W == 64) return row & 3;
    else return W == 32 ? row >> 3 & 1 : 0;              // rows of 64 bytes: 4 rows are 4 places already
}

// One operand's fragments for v_mfma_f32_16x16x32: lane (n, kq) holds c = 32 ks + 8 kq .. + 7 of row / column n.
// ALONG false: the image has a row per tile row, 64 values (128 bytes) each, 16-byte unit u of row r at u ^ (r & 7).
// ALONG true: a row per c, W values each, read transposed by ds_read_b64_tr_b16 (lane i of 16 gives the address of
// 4 columns of row i / 4 and receives column i of 4 rows).
template <bool ALONG, int W, int SUBS>
struct Frags {
    uint32_t at[ALONG ? SUBS : 2];

    __device__ __forceinline__ void init(uint32_t base, int first, int lane) {
        const int n = lane & 15, kq = lane >> 4;
        if constexpr (ALONG) {
            const int row = kq * 8 + (n >> 2);
#pragma unroll
            for (int s = 0; s < SUBS; ++s)
                at[s] = base + row * (W * 2) + (((first >> 4) + s) ^ turn<W>(row)) * 32 + (n & 3) * 8;
        } else {
            at[0] = base + (first + n) * 128 + (kq ^ (n & 7)) * 16;
            at[1] = base + (first + n) * 128 + ((kq + 4) ^ (n & 7)) * 16;
        }
    }

    __device__ __forceinline__ uint4 read(uint32_t stage, int s, int ks) const {
        if constexpr (ALONG) {
            typedef short s16x4 __attribute__((ext_vector_type(4)));
            typedef __attribute__((address_space(3))) s16x4* ptr;
            const uint32_t p = at[s] + stage + ks * 32 * (W * 2);
            const uint2 lo = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(uintptr_t)p));
            const uint2 hi = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(uintptr_t)(p + 4 * (W * 2))));
            return make_uint4(lo.x, lo.y, hi.x, hi.y);
        } else {
            typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
            typedef __attribute__((address_space(3))) const u32x4* ptr;
            const u32x4 v = *(ptr)(uintptr_t)(at[ks] + stage + s * 2048);
            return make_uint4(v[0], v[1], v[2], v[3]);
        }
    }
};

}  // namespace gmm
