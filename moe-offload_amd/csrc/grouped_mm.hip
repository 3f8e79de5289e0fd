// Matrix products of sorted rows by their experts' unquantised weights (fp16 or bf16), with gradients.
//
// Segment u covers the sorted rows r in [seg_start[u], seg_start[u + 1]) and uses W_u = w[seg_slot[u]]
// ([n][k]; slot u where seg_slot is null):
//     mm       y[row_out[r]]  = s_u  W_u   x[row_in[r]]
//     gate_up  h[r]           = silu(g) * u,  (g, u) = W_u x[row_in[r]]   (W_u: inter gate rows, inter up rows)
//     mm_dx    dx[row_out[r]] = s_u  W_u^T dy[row_in[r]]
//       with gu, the (g, u) of a gate_up whose h the product W_u took:  the gradient of (g, u) instead,
//       dg = dh u sig(g) (1 + g (1 - sig(g))),  du = dh g sig(g),  dh = s_u W_u^T dy[row_in[r]]
//     mm_dw    dW_u           = s_u  sum over r of u of  dy[row_dy[r]] x[row_x[r]]^T      (no rows: zeros)
// Sums in fp32 (MFMA), one rounding to the output's type at the end.  The reference multiplies its sorted
// rows by 2-bit experts only (mlx-qwen38/prefill_qproj.py:18-40); these are the same products for the
// weights before quantisation.
//
// All four are one tile product  out[p][q] = sum over c of P[p][c] Q[q][c]  with q the direction in which
// the output is contiguous; an operand is either contiguous in c (x, dy; W for mm) or has its c along the
// rows of memory (W for mm_dx, both operands for mm_dw).  The matrix unit takes Q as its first operand,
// so a lane of the result holds four adjacent q of one p.
#include <hip/hip_bf16.h>

#include <algorithm>
#include <type_traits>

#include "grouped_mm.h"

namespace {

using namespace gmm;

enum { kMM = 0, kGateUp = 1, kDx = 2, kDxGlu = 3, kDw = 4, kDxParts = 5 };

struct Args {
    Segs S;
    const void* p;               // rows (x, or dy)
    const void* q;               // weights, or x for the weights' gradient
    void* out;
    const int32_t* row_p;
    const int32_t* row_q;
    const int32_t* row_out;
    const float* scale;
    const void* gu;              // mm_dx: the pre-activations
    void* gu_out;                // gate_up: where they go (may be null)
    int64_t ldp, ldq, ldo, ldgu; // elements from row to row; ldq from slot to slot where q is weights; ldo of mm_dw likewise
    int n_p, n_q, n_out;         // rows of p, q and out that exist
    int np, nq, nc;              // extents: output columns in p (mm_dw) and q, and the contraction
    int out_f32;
    int span;                    // column tiles per block
    int fold;                    // kDxParts: the weights' rows, which the contraction goes through three times
    int dry;                     // only whether one launch takes the call
};

// A block of WP x WQ waves computes `span` tiles of BP x BQ results side by side in q.  A step of 64 contraction
// indexes goes from global memory to LDS without passing registers while the step before it is multiplied, the
// next tile's first step during the last of this one: two images, one barrier per step.
// Few rows per segment: memory bounds it (gate_up of 512 x 10 rows, 1280 x 2560, 570 us, 5.9 TB/s, matrix unit 17% busy;
// weights' gradient over 512 x 40 rows, 1024 x 2048, 457 us, 4.6 TB/s written).  Many: the matrix unit and, with short
// contractions, a tile's results (8192 x 8192 x 8192 795 us, 1385 TFLOP/s; 16 x 2048 rows, 4096 x 1024, 289 us, 950).
template <typename T, int OP, int BP, int BQ, int WP, int WQ, int BLOCKS>
__global__ __launch_bounds__(64 * WP * WQ, BLOCKS) void k_grouped(Args a) {
    constexpr int kWaves = WP * WQ, SP = BP / WP / 16, SQ = BQ / WQ / 16;
    constexpr bool kAlongP = OP == kDw, kAlongQ = OP >= kDx;
    constexpr int kLoadsP = BP / 8 / kWaves, kLoadsQ = BQ / 8 / kWaves;        // 1 KiB each
    constexpr uint32_t kStageP = BP * 128, kStage = (BP + BQ) * 128;
    constexpr int kQStep = OP == kGateUp ? BQ / 2 : BQ;                        // output columns of a tile
    static_assert(SQ % 2 == 0 && kLoadsP >= 1 && kLoadsQ >= 1, "");
    constexpr bool kThroughLds = OP == kDxGlu || (OP != kGateUp && BP >= 128);
    static_assert(!kThroughLds || (SQ == 4 && kStage / kWaves >= 4096), "");
    constexpr int kIdx = 1024;                                                 // mm_dw: rows whose numbers are held
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * kStage];
    __shared__ int2 idx[OP == kDw ? kIdx : 1];
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_u8*)lds;
    const int t = threadIdx.x, lane = t & 63, wv = __builtin_amdgcn_readfirstlane(t >> 6);
    const int inter = a.nq;                                                    // gate_up, and mm_dx with gu
    const int tiles = (a.nq + kQStep - 1) / kQStep, groups = (tiles + a.span - 1) / a.span;
    int r0, r1, slot, tile, p0 = 0, nc = a.nc, seg = 0;
    if constexpr (OP == kDw) {
        const int tp = (a.np + BP - 1) / BP;
        const uint32_t run = ((uint32_t)groups * tp + 7) / 8;
        const uint32_t item = a.S.n_seg < kManySegs ? dealt(blockIdx.x, gridDim.x, run) : xcd_order(blockIdx.x, gridDim.x);
        seg = item / (groups * tp);
        p0 = (int)(item / groups % tp) * BP;
        tile = (int)(item % groups) * a.span;
        seg_rows(a.S, seg + 1, r0, r1, slot);
        nc = r1 - r0;
    } else {
        Tile at;
        __shared__ uint32_t scratch[kWaves + 3];
        if (!find_tile<64 * kWaves>(a.S, BP, groups, scratch, at)) return;
        r0 = at.r0;
        r1 = at.r1;
        slot = at.slot;
        tile = at.col * a.span;
        if (slot < 0 || a.n_p == 0) nc = 0;
    }
    const int end = tile + a.span < tiles ? tile + a.span : tiles;
    const T* P = (const T*)a.p;
    const T* Q = (const T*)a.q;
    if constexpr (OP != kDw) Q += (int64_t)(slot < 0 ? 0 : slot) * a.ldq;

    // Where this lane's 16 bytes of each of its wave's next loads are.  Rows past the tile, and rows that do not
    // exist, read some row that does: their results are not stored, or replaced by zeros.  Contraction indexes past
    // the end read zeros.
    const T* zero = (const T*)&g_zero16;
    asm("" : "+s"(zero));                                                      // kept in registers
    const T* pp[kLoadsP];
    const T* qp[kLoadsQ];
    constexpr int kUnitsP = BP / 8, kUnitsQ = BQ / 8;                          // ALONG: 16-byte units per row of the image
    const int cu = ((lane & 7) ^ (lane >> 3)) * 8;                             // not ALONG: first c of the 16 bytes
    auto along_row = [&](int j, int loads, int units) { return (wv * loads + j) * (64 / units) + lane / units; };
    // The rows of x or dy, the same in every step.  mm_dw: numbers of the rows [c0, c1) of dy and x, -1 for one that is
    // missing on either side: zeros on the one would still meet an infinity on the other.
    int rp[kLoadsP];
    auto hold_rows = [&](int c0, int c1) {
        static_assert(OP != kDw || BP == BQ, "both operands' loads of a step have the same rows");
        for (int c = c0 + t; c < c1; c += 64 * kWaves) {
            const int v = a.row_p ? a.row_p[r0 + c] : r0 + c, x = a.row_q ? a.row_q[r0 + c] : r0 + c;
            const bool both = v >= 0 && v < a.n_p && x >= 0 && x < a.n_q;
            idx[c - c0] = make_int2(both ? v : -1, both ? x : -1);
        }
    };
    if constexpr (OP != kDw) {
#pragma unroll
        for (int j = 0; j < kLoadsP; ++j) {
            int r = r0 + (wv * kLoadsP + j) * 8 + (lane >> 3);
            r = r < r1 ? r : r1 - 1;
            const int v = a.row_p ? a.row_p[r] : r;
            rp[j] = v >= 0 && v < a.n_p ? v : 0;
        }
    }
    // mm_dw of more rows than are held: tile by tile, kIdx of them [part0, part1) at a time
    const bool parts = OP == kDw && nc > kIdx;
    int part0 = 0, part1 = nc;
    int load_tile = tile, load_c = 0;                                          // the step that is loaded next
    auto place = [&]() {
        const bool any = load_tile < end;
        const int q0 = load_tile * kQStep;
        if constexpr (OP == kDw) {
#pragma unroll
            for (int j = 0; j < kLoadsP; ++j) {
                const int row = along_row(j, kLoadsP, kUnitsP), col = (lane % kUnitsP ^ 2 * turn<BP>(row)) * 8;
                const int c = load_c + row;
                const int2 v = idx[any && c < part1 ? c - part0 : 0];
                const bool ok = any && c < part1 && v.x >= 0;
                pp[j] = ok ? P + v.x * a.ldp + (p0 + col < a.np ? p0 + col : 0) : zero;
                qp[j] = ok ? Q + v.y * a.ldq + (q0 + col < a.nq ? q0 + col : 0) : zero;
            }
        } else {
            const bool ok = any && load_c + cu < nc;
#pragma unroll
            for (int j = 0; j < kLoadsP; ++j) pp[j] = ok ? P + rp[j] * a.ldp + load_c + cu : zero;
#pragma unroll
            for (int j = 0; j < kLoadsQ; ++j) {
                if constexpr (kAlongQ) {
                    const int row = along_row(j, kLoadsQ, kUnitsQ), q = q0 + (lane % kUnitsQ ^ 2 * turn<BQ>(row)) * 8;
                    const int c = load_c + row, w = OP != kDxParts || c < a.fold ? c : c < 2 * a.fold ? c - a.fold : c - 2 * a.fold;
                    qp[j] = any && c < nc ? Q + (int64_t)w * a.nq + (q < a.nq ? q : 0) : zero;
                } else {
                    const int row = (wv * kLoadsQ + j) * 8 + (lane >> 3);
                    int64_t q;
                    if constexpr (OP == kGateUp) {
                        // a wave's first SQ / 2 subtiles are gate rows, the others the up rows of the same outputs
                        const int sub = row / 16 % SQ;
                        int c = q0 + row / (SQ * 16) * (SQ * 8) + sub % (SQ / 2) * 16 + row % 16;
                        c = c < inter ? c : inter - 1;
                        q = c + (sub < SQ / 2 ? 0 : inter);
                    } else {
                        q = q0 + row < a.nq ? q0 + row : a.nq - 1;
                    }
                    qp[j] = ok ? Q + q * a.nc + load_c + cu : zero;
                }
            }
        }
    };
    auto advance = [&]() {
        load_c += kBC;
        if (OP != kDw && OP != kDxParts && load_tile < end && load_c + kBC <= nc) {    // wave-uniform; past the end all stay at zero
#pragma unroll
            for (int j = 0; j < kLoadsP; ++j) pp[j] += kBC;
#pragma unroll
            for (int j = 0; j < kLoadsQ; ++j) qp[j] += kAlongQ ? (int64_t)kBC * a.nq : kBC;
            return;
        }
        if (load_c >= part1) {
            load_c = 0;
            load_tile = parts ? end : load_tile + 1;
            if (OP == kDw && BP == 128 && nc <= kBC && load_tile < end && (load_tile + 1) * BQ <= a.nq) {
                // the same rows again, further right: no row numbers, no multiplications (lanes without a row stay at zero)
#pragma unroll
                for (int j = 0; j < kLoadsQ; ++j) qp[j] += qp[j] == zero ? 0 : BQ;
                return;
            }
        }
        place();
    };
    auto load = [&](int d, uint32_t stage) {
        if (d < kLoadsP) load_to_lds(pp[d], lds0 + stage + (wv * kLoadsP + d) * 1024);
        else load_to_lds(qp[d - kLoadsP], lds0 + stage + kStageP + (wv * kLoadsQ + d - kLoadsP) * 1024);
    };
    constexpr int kLoads = kLoadsP + kLoadsQ;

    const int wp = wv / WQ, wq = wv % WQ, n = lane & 15, kq = lane >> 4;
    Frags<kAlongP, BP, SP> fp;
    Frags<kAlongQ, BQ, SQ> fq;
    fp.init(lds0, wp * SP * 16, lane);
    fq.init(lds0 + kStageP, wq * SQ * 16, lane);
    const float s = a.scale && slot >= 0 && (OP != kDw || nc > 0) ? a.scale[slot] : 1.0f;   // (dw of no rows: zeros, whatever the scale)
    // 16-byte stores: lane (n, kq) of a pair of subtiles holds columns 8 (kq / 2) .. + 7 of subtile kq % 2
    const int pair_col = (kq & 1) * 16 + (kq >> 1) * 8;
    // the output row of this lane's row in each subtile (-1: none); bit i of dead: its results are zeros
    int orow[SP];
    uint32_t dead_rows = 0;
    if constexpr (OP != kDw) {
#pragma unroll
        for (int i = 0; i < SP; ++i) {
            const int r = r0 + wp * SP * 16 + i * 16 + n;
            orow[i] = -1;
            if (r < r1) {
                const int v = a.row_p ? a.row_p[r] : 0, o = a.row_out ? a.row_out[r] : r;
                if (slot < 0 || (a.row_p && (v < 0 || v >= a.n_p))) dead_rows |= 1u << i;
                orow[i] = o < a.n_out ? o : -1;
            }
        }
    }
    auto multiply = [](uint4 q, uint4 p, f32x4 c) {
        if constexpr (OP == kDxParts) return mfma_parts<T>(q, p, c);
        else return mfma<T>(q, p, c);
    };
    uint32_t stage = 0;
    bool landed = false;                                                       // the next step's loads have been waited for
    auto start = [&](int c0) {
        load_tile = tile;
        load_c = c0;
        place();
#pragma unroll
        for (int d = 0; d < kLoads; ++d) load(d, stage);
        advance();
    };
    if (nc > 0 && !parts) {
        if constexpr (OP == kDw) {
            hold_rows(0, nc);
            __syncthreads();
        }
        start(0);
    }
#pragma unroll 1
    for (; tile < end; ++tile) {
        const int q0 = tile * kQStep;
        f32x4 acc[SP][SQ] = {};
#pragma unroll 1
        for (int c0 = 0; c0 < nc; c0 += kBC) {
            if (OP == kDw && parts && c0 % kIdx == 0) {
                part0 = c0;
                part1 = c0 + kIdx < nc ? c0 + kIdx : nc;
                __syncthreads();                                               // the rows held so far are all placed
                hold_rows(part0, part1);
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");               // the part before's loads past its end
                __syncthreads();
                start(part0);
            }
            // this wave's loads of the step have landed and its reads of the step before are done; past the barrier, so are
            // everyone's
            if (landed) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            landed = false;
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            const uint32_t fill = kStage - stage;
            // The step's second half is read from LDS, and the next step's loads are issued, between the first half's
            // products, row by row (past the last step they fetch zeros that nobody reads)
            uint4 vp[2][SP], vq[2][SQ];
#pragma unroll
            for (int j = 0; j < SQ; ++j) vq[0][j] = fq.read(stage, j, 0);
#pragma unroll
            for (int i = 0; i < SP; ++i) vp[0][i] = fp.read(stage, i, 0);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < SP; ++i) {
                // (of eight rows from the middle on: by then half of the first half's registers are free)
                constexpr int kFrom = SP > 4 ? SP / 2 : 0, kEach = SP > 4 ? 2 : 1;
                if (i == kFrom) {
#pragma unroll
                    for (int j = 0; j < SQ; ++j) vq[1][j] = fq.read(stage, j, 1);
                }
                if (i >= kFrom) {
#pragma unroll
                    for (int e = (i - kFrom) * kEach; e < (i - kFrom + 1) * kEach; ++e) vp[1][e] = fp.read(stage, e, 1);
                }
#pragma unroll
                for (int j = 0; j < SQ; ++j) acc[i][j] = multiply(vq[0][j], vp[0][i], acc[i][j]);
#pragma unroll
                for (int d = i * kLoads / SP; d < (i + 1) * kLoads / SP; ++d) load(d, fill);
                __builtin_amdgcn_sched_barrier(0);
            }
            advance();
#pragma unroll
            for (int i = 0; i < SP; ++i)
#pragma unroll
                for (int j = 0; j < SQ; ++j) acc[i][j] = multiply(vq[1][j], vp[1][i], acc[i][j]);
            stage = fill;
        }
        // The next tile's first step is waited for before the stores: in the loop the wait would take them in.
        if (BP < 256 && nc > 0 && tile + 1 < end) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            landed = !parts;
        }
        if constexpr (kThroughLds) {
            // The results go through the image just multiplied, a part of it for each wave, and out in whole lines: a lane
            // of the matrix unit's result has 8 or 16 bytes of a row and its neighbour another row's, each a cache access
            // of its own, and a store past the caches wants whole lines (mm 4096 x 1024, 16 x 2048 rows to places in no
            // order: 258 us, and 276 straight from the registers; weights' gradient over 512 x 40 rows, 1024 x 2048, 377 and
            // 687).  Tiles of 64 rows have too few steps to pay for the barrier (mm of 100 x 47 rows, 1152 x 320: 20.3 us, and
            // 19.5 without), but silu's gradient reads (g, u) in whole lines too this way.
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();                                      // everyone has read the image
            asm volatile("" ::: "memory");
            int l = lane;
            asm volatile("" : "+v"(l));                                        // no addresses are kept over the products
            const int n = l & 15, kq = l >> 4;
            const uint32_t area = lds0 + (kStage - stage) + wv * (kStage / kWaves);
            typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
            typedef __attribute__((address_space(3))) u32x4* lds16;
            const int col = q0 + wq * SQ * 16;
            // row m % 16 of the wave's subtile row i: where its results go in out's elements, -1 if nowhere
            auto row_at = [&](int i, int m) -> int64_t {
                if constexpr (OP == kDw) {
                    const int o = p0 + wp * SP * 16 + i * 16 + m;
                    return o < a.np ? (int64_t)seg * a.ldo + (int64_t)o * a.nq : -1;
                } else {
                    const int o = __shfl(orow[i], m, 64);
                    return o < 0 ? -1 : (int64_t)o * a.ldo;
                }
            };
            // kPass subtile rows at a time, rows of UNITS 16-byte units; unit u of row r is at u ^ (r & 7) in its low bits
            auto result = [&](int i, int j) { return (dead_rows >> i & 1) ? f32x4{} : acc[i][j] * s; };
            auto pass = [&](auto bytes_c, auto* dst) {
                constexpr int kBytes = decltype(bytes_c)::value, UNITS = SQ * kBytes, kRowsPer = 64 / UNITS;
                constexpr int kFit = kStage / kWaves / (UNITS * 256), kPass = kFit < SP ? kFit : SP;
                static_assert(SP % kPass == 0, "");
                auto at = [&](int row, int u) { return area + (uint32_t)(row * UNITS + (u ^ (row & 7))) * 16; };
#pragma unroll
                for (int i0 = 0; i0 < SP; i0 += kPass) {
#pragma unroll
                    for (int i = 0; i < kPass; ++i)
                        if constexpr (kBytes == 4) {
#pragma unroll
                            for (int j = 0; j < SQ; ++j)
                                *(lds16)(uintptr_t)at(i * 16 + n, 4 * j + kq) = __builtin_bit_cast(u32x4, result(i0 + i, j));
                        } else {
#pragma unroll
                            for (int j = 0; j < SQ; j += 2)
                                *(lds16)(uintptr_t)at(i * 16 + n, 2 * j + (kq & 1) * 2 + (kq >> 1)) = __builtin_bit_cast(
                                    u32x4, pair8(round4<T>(result(i0 + i, j)), round4<T>(result(i0 + i, j + 1))));
                        }
#pragma unroll
                    for (int it = 0; it < kPass * 16 / kRowsPer; ++it) {
                        const int row = it * kRowsPer + l / UNITS, u = l % UNITS, c = col + u * (16 / kBytes);
                        const u32x4 v = *(lds16)(uintptr_t)at(row, u);
                        const int64_t o = row_at(i0 + it * kRowsPer / 16, row & 15);
                        if (o >= 0 && c < a.nq) store16(dst + o + c, __builtin_bit_cast(uint4, v));
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            };
            if constexpr (OP == kDxGlu) {
                // dh in fp32, one subtile row at a time; a lane then has 8 adjacent columns of a row, of dh and of (g, u)
                auto at = [&](int row, int u) { return area + (uint32_t)(row * 16 + (u ^ (row & 7))) * 16; };
                const int u8 = l & 7, c = col + u8 * 8;
#pragma unroll
                for (int i = 0; i < SP; ++i) {
                    uint4 gv[2], uv[2];
                    int64_t o[2];
#pragma unroll
                    for (int it = 0; it < 2; ++it) {
                        const int m = it * 8 + (l >> 3), r = r0 + wp * SP * 16 + i * 16 + m;
                        o[it] = row_at(i, m);
                        const uint32_t dead = __shfl(dead_rows, m, 64);                 // (by every lane, before any condition)
                        const bool ok = o[it] >= 0 && c < inter && !(dead >> i & 1);
                        const T* gr = ok ? (const T*)a.gu + (int64_t)r * a.ldgu + c : zero;
                        gv[it] = *(const uint4*)gr;
                        uv[it] = *(const uint4*)(ok ? gr + inter : zero);
                    }
#pragma unroll
                    for (int j = 0; j < SQ; ++j) *(lds16)(uintptr_t)at(n, 4 * j + kq) = __builtin_bit_cast(u32x4, result(i, j));
#pragma unroll
                    for (int it = 0; it < 2; ++it) {
                        const int m = it * 8 + (l >> 3);
                        uint2 dg[2], du[2];
#pragma unroll
                        for (int b = 0; b < 2; ++b) {
                            const f32x4 dh = __builtin_bit_cast(f32x4, *(lds16)(uintptr_t)at(m, 2 * u8 + b));
                            const f32x4 g = widen4<T>(b ? make_uint2(gv[it].z, gv[it].w) : make_uint2(gv[it].x, gv[it].y));
                            const f32x4 u = widen4<T>(b ? make_uint2(uv[it].z, uv[it].w) : make_uint2(uv[it].x, uv[it].y));
                            f32x4 vg, vu;
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                // sig is 0 or 1 from -200 and 200 on; an infinity (g past fp16's range) would meet a zero
                                const float low = g[e] < -200.f ? -200.f : g[e], both = low > 200.f ? 200.f : low;
                                const float sg = 1.0f / (1.0f + __expf(-low));
                                vg[e] = dh[e] * u[e] * sg * (1.0f + both * (1.0f - sg));
                                vu[e] = dh[e] * low * sg;
                            }
                            dg[b] = round4<T>(vg);
                            du[b] = round4<T>(vu);
                        }
                        if (o[it] >= 0 && c < inter) {
                            T* d = (T*)a.out + o[it] + c;
                            store16(d, make_uint4(dg[0].x, dg[0].y, dg[1].x, dg[1].y));
                            store16(d + inter, make_uint4(du[0].x, du[0].y, du[1].x, du[1].y));
                        }
                    }
                }
            } else if (OP == kDw && a.out_f32) {
                pass(std::integral_constant<int, 4>(), (float*)a.out);
            } else {
                pass(std::integral_constant<int, 2>(), (T*)a.out);
            }
            continue;
        }
#pragma unroll
        for (int i = 0; i < SP; ++i) {
            const int m = wp * SP * 16 + i * 16 + n;
            if constexpr (OP == kDw) {
                const int64_t row = (int64_t)seg * a.ldo + (int64_t)(p0 + m) * a.nq;
                const bool live = p0 + m < a.np;
                if (a.out_f32) {
#pragma unroll
                    for (int j = 0; j < SQ; ++j) {
                        const int q = q0 + wq * SQ * 16 + j * 16 + kq * 4;
                        if (live && q < a.nq)
                            store16((float*)a.out + row + q, __builtin_bit_cast(uint4, acc[i][j] * s));
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < SQ; j += 2) {
                        const uint4 v = pair8(round4<T>(acc[i][j] * s), round4<T>(acc[i][j + 1] * s));
                        const int q = q0 + wq * SQ * 16 + j * 16 + pair_col;
                        if (live && q < a.nq) store16((T*)a.out + row + q, v);
                    }
                }
                continue;
            }
            const int r = r0 + m, o = orow[i];
            const bool live = o >= 0, dead = dead_rows >> i & 1;
            if constexpr (OP == kGateUp) {
                uint2 h[SQ / 2], g2[SQ / 2], u2[SQ / 2];
#pragma unroll
                for (int j = 0; j < SQ / 2; ++j) {
                    f32x4 g = acc[i][j], u = acc[i][j + SQ / 2], hv;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        g[e] = dead ? 0.f : g[e];
                        u[e] = dead ? 0.f : u[e];
                        hv[e] = g[e] / (1.0f + __expf(-g[e])) * u[e];
                    }
                    h[j] = round4<T>(hv);
                    g2[j] = round4<T>(g);
                    u2[j] = round4<T>(u);
                }
                if constexpr (SQ / 2 == 1) {
                    const int c = q0 + wq * 16 + kq * 4;
                    if (live && c < inter) {
                        *(uint2*)((T*)a.out + (int64_t)r * a.ldo + c) = h[0];
                        if (a.gu_out) {
                            *(uint2*)((T*)a.gu_out + (int64_t)r * a.ldgu + c) = g2[0];
                            *(uint2*)((T*)a.gu_out + (int64_t)r * a.ldgu + inter + c) = u2[0];
                        }
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < SQ / 2; j += 2) {
                        const int c = q0 + wq * SQ * 8 + j * 16 + pair_col;
                        const uint4 vh = pair8(h[j], h[j + 1]);
                        if (live && c < inter) store16((T*)a.out + (int64_t)r * a.ldo + c, vh);
                        if (a.gu_out) {
                            const uint4 vg = pair8(g2[j], g2[j + 1]), vu = pair8(u2[j], u2[j + 1]);
                            if (live && c < inter) {
                                store16((T*)a.gu_out + (int64_t)r * a.ldgu + c, vg);
                                store16((T*)a.gu_out + (int64_t)r * a.ldgu + inter + c, vu);
                            }
                        }
                    }
                }
            } else {
#pragma unroll
                for (int j = 0; j < SQ; j += 2) {
                    const f32x4 zero = {};
                    const uint4 v = pair8(round4<T>(dead ? zero : acc[i][j] * s), round4<T>(dead ? zero : acc[i][j + 1] * s));
                    const int q = q0 + wq * SQ * 16 + j * 16 + pair_col;
                    if (live && q < a.nq) store16((T*)a.out + (int64_t)o * a.ldo + q, v);
                }
            }
        }
    }
    // the last step's loads write LDS that is another block's once this one has ended
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// A few rows per segment (decoding): one wave per 16 rows of a segment and 16 weight rows (mm: 16 columns; gate_up: 8
// gate rows and the 8 up rows of the same outputs), which it streams through an LDS ring of its own, kFewRing steps of
// 64 ahead, without a barrier.  Loads that put the weights straight into the matrix unit's layout would take 16 bytes
// per lane from 16 rows at a time, four times the cache accesses.  The steps are k_grouped's, in its order, so a row's
// result has the same bits whichever of the two a call's size selects.  gate_up of 1024 x 2048 for one token's 10 experts:
// 14 us, 42 MB at 3 TB/s; what bounds it is one wave's way through its 32 steps.
constexpr int kFewRing = 8;
constexpr int few_step(int op) { return op == kGateUp ? 8 : 16; }             // output columns of a wave of k_grouped_few

template <typename T, int OP>
__global__ __launch_bounds__(64) void k_grouped_few(Args a) {
    constexpr int kQStep = few_step(OP);
    constexpr uint32_t kStage = 4096;                                          // 16 weight rows, 16 rows of x
    __shared__ __attribute__((aligned(1024))) uint8_t lds[kFewRing * kStage];
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_u8*)lds;
    const int lane = threadIdx.x, n = lane & 15, kq = lane >> 4;
    Tile at;
    if (!find_tile<64>(a.S, 16, (a.nq + kQStep - 1) / kQStep, (uint32_t*)lds, at)) return;
    const int slot = at.slot, q0 = at.col * kQStep, nc = slot < 0 || a.n_p == 0 ? 0 : a.nc, steps = (nc + kBC - 1) / kBC;
    const T* zero = (const T*)&g_zero16;
    const T* Q = (const T*)a.q + (int64_t)(slot < 0 ? 0 : slot) * a.ldq;
    // this lane's 16 bytes of each load: row lane / 8 of its 8 rows
    const int cu = ((lane & 7) ^ (lane >> 3)) * 8;
    const T* pp[2];
    const T* qp[2];
    uint32_t live_p = 0;                                                       // rows of x that do not exist read zeros
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int r = at.r0 + j * 8 + (lane >> 3);
        int v = -1;
        if (r < at.r1) v = a.row_p ? a.row_p[r] : r;
        if (v >= 0 && v < a.n_p) live_p |= 1u << j;
        pp[j] = (const T*)a.p + (int64_t)(live_p >> j & 1 ? v : 0) * a.ldp + cu;
        int64_t c = q0 + (OP == kGateUp ? 0 : j * 8) + (lane >> 3);
        c = c < a.nq ? c : a.nq - 1;
        qp[j] = Q + (OP == kGateUp ? c + (int64_t)j * a.nq : c) * nc + cu;
    }
    auto issue = [&](int s) {
        const uint32_t to = lds0 + (uint32_t)(s % kFewRing) * kStage;
        const bool in = s * kBC + cu < nc;                                     // (also past the last step)
#pragma unroll
        for (int j = 0; j < 2; ++j) load_to_lds(in ? qp[j] + s * kBC : zero, to + j * 1024);
#pragma unroll
        for (int j = 0; j < 2; ++j) load_to_lds(in && live_p >> j & 1 ? pp[j] + s * kBC : zero, to + 2048 + j * 1024);
    };
    Frags<false, 16, 1> fp, fq;
    fq.init(lds0, 0, lane);
    fp.init(lds0 + 2048, 0, lane);
    f32x4 acc = {};
    if (steps > 0) {
#pragma unroll
        for (int s = 0; s < kFewRing; ++s) issue(s);
    }
#pragma unroll 1
    for (int s = 0; s < steps; ++s) {
        const uint32_t stage = (uint32_t)(s % kFewRing) * kStage;
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"((kFewRing - 1) * 4) : "memory");     // loads return in order
        const uint4 q0v = fq.read(stage, 0, 0), p0v = fp.read(stage, 0, 0), q1v = fq.read(stage, 0, 1), p1v = fp.read(stage, 0, 1);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                            // read before the next load overwrites it
        issue(s + kFewRing);
        acc = mfma<T>(q0v, p0v, acc);
        acc = mfma<T>(q1v, p1v, acc);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                                  // LDS is another block's after this one
    // lane (n, kq): row n, columns 4 kq .. + 3
    const int r = at.r0 + n;
    bool live = r < at.r1, dead = slot < 0;
    int o = r;
    if (live) {
        if (a.row_p) {
            const int v = a.row_p[r];
            dead |= v < 0 || v >= a.n_p;
        }
        if (OP == kMM && a.row_out) o = a.row_out[r];
        live = o >= 0 && o < a.n_out;
    }
    if (dead) acc = (f32x4){0.f, 0.f, 0.f, 0.f};
    if constexpr (OP == kGateUp) {
        // gate columns 4 kq .. + 3 in the lower two lane groups, the same outputs' up values 32 lanes further
        f32x4 up, h;
#pragma unroll
        for (int e = 0; e < 4; ++e) up[e] = __shfl_xor(acc[e], 32, 64);
#pragma unroll
        for (int e = 0; e < 4; ++e) h[e] = acc[e] / (1.0f + __expf(-acc[e])) * up[e];
        const int c = q0 + (kq & 1) * 4;
        if (!live || c >= a.nq) return;
        if (kq < 2) *(uint2*)((T*)a.out + (int64_t)r * a.ldo + c) = round4<T>(h);
        if (a.gu_out) *(uint2*)((T*)a.gu_out + (int64_t)r * a.ldgu + (kq < 2 ? 0 : a.nq) + c) = round4<T>(acc);
    } else {
        const int c = q0 + kq * 4;
        const float s = a.scale && slot >= 0 ? a.scale[slot] : 1.0f;
        if (live && c < a.nq) *(uint2*)((T*)a.out + (int64_t)o * a.ldo + c) = round4<T>(acc * s);
    }
}

// Row tiles of a call as far as the host knows it: as many segments as can have rows have a tile, and but for one of them
// a last tile that is half full.
int64_t row_tiles(const Args& a, int bp) {
    const int64_t segs = std::min(a.S.n_seg, a.S.n_rows);
    return std::max((a.S.n_rows + (segs - 1) * (bp / 2) + bp - 1) / bp, segs);
}

// Sets the column tiles per block and returns the blocks, or -1.
template <int OP, int BP, int BQ, int THREADS>
int64_t blocks_of(Args& a) {
    const int qstep = OP == kGateUp ? BQ / 2 : BQ, tiles = (a.nq + qstep - 1) / qstep;
    int64_t rows, most, steps;                                // row tiles expected and at most, steps per tile
    if constexpr (OP == kDw) {
        rows = most = (int64_t)a.S.n_seg * ((a.np + BP - 1) / BP);
        steps = (int64_t)a.S.n_rows / a.S.n_seg / kBC + 1;
    } else {
        rows = row_tiles(a, BP);
        most = (int64_t)a.S.n_rows / BP + (a.S.n_seg + 2 < a.S.n_rows ? a.S.n_seg + 2 : a.S.n_rows);
        steps = (a.nc + kBC - 1) / kBC;
    }
    // Column tiles per block: short tiles share one block's start (the search for its rows, the first load's way) while
    // that leaves 1024 blocks.  us per launch at 1, 2, 4 and 16 tiles: weights' gradient 4096 x 1024 of 16 x 256 rows (4
    // steps) 68, 61, 57, 77, 1024 x 2048 of 512 x 40 rows (1 step) 594, 449, 402, 381; mm 4096 x 1024 of 16 x 512 rows (16
    // steps) 77, 69, 122, 422.  Tiles of 64 rows wait for memory and have three blocks per CU to do so: mm_dx 1024 x 2048 of
    // 512 x 40 rows (16 steps) 431, 436, 456, 469.
    const int64_t target = OP == kDw ? 16 : BP == 64 ? 8 : 32;
    const int64_t span = std::min(target / steps, rows * tiles / 1024);
    a.span = (int)std::max<int64_t>(1, std::min<int64_t>(span, tiles));
    const int64_t groups = (tiles + a.span - 1) / a.span;
    if (most > kMaxThreads / THREADS / groups) {
        moe_set_error("grouped product: %lld x %lld tiles are more than one launch takes", (long long)most, (long long)groups);
        return -1;
    }
    return most * groups;
}

template <typename T, int OP, int BP, int BQ, int WP, int WQ, int BLOCKS>
int launch_tiles(Args a, hipStream_t s) {
    const int64_t blocks = blocks_of<OP, BP, BQ, 64 * WP * WQ>(a);
    if (blocks < 0) return -1;
    if (a.dry) return 0;
    hipLaunchKernelGGL((k_grouped<T, OP, BP, BQ, WP, WQ, BLOCKS>), dim3((uint32_t)blocks), dim3(64 * WP * WQ), 0, s, a);
    HIP_TRY(hipGetLastError());
    return 0;
}

// Tiles of 256 x 256 (one block per CU) multiply 1.3 times as fast as tiles of 128 x 128 (two per CU) once every CU has
// one, but there are a quarter of them: TFLOP/s of 128 and 256, bf16, 16 segments: mm 4096 x 1024 of 2048 rows each 778
// and 955, of 1024 rows 893 and 1020; 1024 x 4096 of 2048 rows 912 and 1158; weights' gradient 4096 x 1024 of 1024 rows
// 648 and 926; one segment, 8192 x 8192 x 8192, 952 and 1385 (the library's product: 1370); 2048 rows of 4096 x 2048
// (512 and 128 tiles) 920 and 655.  Rows per tile are what the host can expect of ragged segments.
bool big_tiles(int64_t tiles128, int64_t tiles256) {
    return (tiles256 + 255) / 256 * 256 * 4 * 10 < (tiles128 + 511) / 512 * 512 * 13;
}

// Tiles of 64 x 64 (1024 blocks at a time, half the work each) or 64 x 128 (768): both wait for memory, so the rounds of
// blocks count.  us of mm with 64 x 64 and 64 x 128: 100 x 10 rows, 1152 x 1024, (900 tiles of 128) 38 and 42; 64 x 1 rows,
// 2048 x 2048, (1024) 125 and 133; 500 rows, 2048 x 4096, (128) 37 and 42; 40 x 12 rows, 2048 x 1024, (640) 32 and 28; 100
// x 1 rows, 2048 x 512, (1600) 42 and 39; mm_dx of 512 x 40 rows, 1024 x 2048, (8192) 485 and 442.
bool narrow_tiles(int64_t tiles) { return (2 * tiles + 1023) / 1024 * 512 * 115 < (tiles + 767) / 768 * 768 * 100; }

template <typename T, int OP>
int launch_few(const Args& a, hipStream_t s) {
    const int qstep = few_step(OP);
    const int64_t rows = (int64_t)a.S.n_rows / 16 + std::min(a.S.n_seg + 2, a.S.n_rows), tiles = (a.nq + qstep - 1) / qstep;
    hipLaunchKernelGGL((k_grouped_few<T, OP>), dim3((uint32_t)(rows * tiles)), dim3(64), 0, s, a);
    HIP_TRY(hipGetLastError());
    return 0;
}

// The tiles of a weights' gradient.
enum { kDw256, kDw128, kDw64 };

int dw_tiles(const Args& a) {
    const int64_t per_seg = a.S.n_rows / std::max(a.S.n_seg, 1);
    auto tiles = [&](int b) { return (int64_t)a.S.n_seg * ((a.np + b - 1) / b) * ((a.nq + b - 1) / b); };
    // with few rows the output's bytes bound it, and either size wins somewhere: us with tiles of 128 and of 256, 512 x 80
    // rows, 1280 x 2560, 1101 and 1177, 128 x 64 rows, 4096 x 1024, 204 and 210, 64 x 100 rows, 2048 x 1024, 76 and 78, 512 x
    // 40 rows, 1024 x 2048, 377 and 380 (ragged, with mm_dx, 914 and 851); from 512 rows on the rounds of blocks decide
    if (per_seg >= 512 && big_tiles(tiles(128), tiles(256))) return kDw256;
    // narrow ones: tiles of 128 would be half empty, and few (8 x 512 rows, 64 x 2048: 13.9 us with them, 9.4 with 64's).
    // Where not every CU gets one of 128, more and shorter steps of 64 are done sooner too: 2 x 4000 rows, 512 x 1024, 66 and
    // 41 us, 1113 rows, 2272 x 96, 22.7 and 12.9, 8 x 300 rows, 1024 x 512, 11.4 and 10.7
    if (a.np <= 64 || a.nq <= 64 || tiles(128) <= 256) return kDw64;
    return kDw128;
}

template <typename T, int OP>
int launch(const Args& a, hipStream_t s) {
    if constexpr (OP == kDw) {
        switch (dw_tiles(a)) {
            case kDw256: return launch_tiles<T, OP, 256, 256, 2, 4, 2>(a, s);
            case kDw128: return launch_tiles<T, OP, 128, 128, 2, 2, 2>(a, s);
            default: return launch_tiles<T, OP, 64, 64, 2, 2, 4>(a, s);
        }
    } else {
        const int64_t per_seg = a.S.n_rows / std::max(a.S.n_seg, 1);
        auto cols = [&](int bq) { return (a.nq + (OP == kGateUp ? bq / 2 : bq) - 1) / (OP == kGateUp ? bq / 2 : bq); };
        // A wave per 16 rows and 16 columns where that leaves no SIMD with more than one: us, and with tiles, gate_up of 512 x
        // 2048 for 10 rows of 10 segments 14 and 26, mm of 100 rows, 2048 x 4096, (896 waves) 24 and 35, 1000 rows, 256 x
        // 4096, (1008) 15.5 and 21.5; 100 rows, 4096 x 1024, (1792) 16.5 and 10.9, 100 x 6 rows, 1152 x 320, (7200) 35 and 18
        if constexpr (OP == kMM || OP == kGateUp) {
            if (row_tiles(a, 16) * ((a.nq + few_step(OP) - 1) / few_step(OP)) <= 1024) return launch_few<T, OP>(a, s);
        }
        // Tiles of 64 rows waste less of short segments, tiles of 128 read the weights half as often: us of either, mm of
        // 512 segments, 1024 x 2048, 48 rows each 406 and 411, 64 rows 425 and 427, 80 rows 515 and 438; 64 segments, 2048 x
        // 1024, 64 rows 54 and 51, 96 rows 74 and 58; 512 segments of 1 to 80 rows, mm_dx 521 and 534; and where not every
        // CU gets one of 128, mm of 4 x 300 rows, 1024 x 2048, 23 and 27
        if (per_seg <= 48 || row_tiles(a, 128) * cols(128) <= 256) {
            if constexpr (OP != kDxGlu) {
                if (narrow_tiles(row_tiles(a, 64) * cols(128))) return launch_tiles<T, OP, 64, 64, 2, 2, 4>(a, s);
            }
            return launch_tiles<T, OP, 64, 128, 2, 2, 3>(a, s);
        }
        if (big_tiles(row_tiles(a, 128) * cols(128), row_tiles(a, 256) * cols(256)))
            return launch_tiles<T, OP, 256, 256, 2, 4, 2>(a, s);
        return launch_tiles<T, OP, 128, 128, 2, 2, 2>(a, s);
    }
}

template <int OP>
int launch_typed(const Args& a, int dtype, hipStream_t s) {
    return dtype ? launch<__bf16, OP>(a, s) : launch<_Float16, OP>(a, s);
}

bool bad(const char* who, const char* what) {
    moe_set_error("%s: %s", who, what);
    return true;
}

// Whether a matrix of `rows` rows may be read or written in 16-byte pieces of `width` elements.
bool bad_matrix(const char* who, const char* name, const void* p, int64_t ld, int64_t width, int64_t rows) {
    if (rows < 0 || width <= 0 || width % 8 || ld % 8 || (rows > 1 && ld < width) || ld < 0) {
        moe_set_error("%s: %s: %lld rows of %lld elements at a step of %lld (multiples of 8 wanted)", who, name,
                      (long long)rows, (long long)width, (long long)ld);
        return true;
    }
    if (rows > 0 && (!p || (uintptr_t)p % 16)) {
        moe_set_error("%s: %s: null or not 16-byte aligned", who, name);
        return true;
    }
    return false;
}

bool bad_segs(const char* who, const Segs& S, int n, int k, int dtype, const void* w) {
    if (dtype != 0 && dtype != 1) return bad(who, "dtype is 0 (fp16) or 1 (bf16)");
    if (S.n_seg < 0 || S.n_seg > kMaxSeg || S.n_rows < 0 || S.n_rows > kMaxSide || S.n_slots < 0 || n < 0 || n > kMaxSide ||
        k < 0 || k > kMaxSide) {
        moe_set_error("%s: n_seg=%d (0..%d) n_rows=%d n_slots=%d matrices of %d x %d (up to %d)", who, S.n_seg, kMaxSeg, S.n_rows,
                      S.n_slots, n, k, kMaxSide);
        return true;
    }
    if (!S.start) return bad(who, "seg_start is null");
    if (S.n_slots > 0 && !w) return bad(who, "no weights");
    return false;
}

}  // namespace

int gmm::dx_of_parts(const void* dv, const int32_t* rows, int n_rows, const int32_t* seg_start, int n_seg, const void* w,
                     int64_t w_stride, int n, int k, void* dx, int64_t lddx, int dtype, bool dry, hipStream_t s) {
    Args a = {};
    a.dry = dry;
    a.S = Segs{seg_start, nullptr, n_seg, n_rows, n_seg, 1};
    a.p = dv, a.q = w, a.out = dx, a.row_p = a.row_out = rows;
    a.ldp = 3 * (int64_t)n, a.ldq = w_stride, a.ldo = lddx, a.n_p = a.n_out = n_rows, a.nq = k, a.nc = 3 * n, a.fold = n;
    return launch_typed<kDxParts>(a, dtype, s);
}

extern "C" {

int moe_grouped_mm(const void* x, int64_t ldx, int n_x, const int32_t* row_in, const int32_t* seg_start,
                   const int32_t* seg_slot, int n_seg, int n_rows, const void* w, int64_t w_stride, int n_slots, int n,
                   int k, const float* scale, void* y, int64_t ldy, int n_y, const int32_t* row_out, int dtype, int fill,
                   void* stream) {
    const char* who = "grouped_mm";
    Args a = {};
    a.S = Segs{seg_start, seg_slot, n_seg, n_rows, n_slots, fill};
    if (bad_segs(who, a.S, n, k, dtype, w) || bad_matrix(who, "x", x, ldx, k, n_x) ||
        bad_matrix(who, "w", w, w_stride, k, n_slots) || bad_matrix(who, "y", y, ldy, n, n_y))
        return -1;
    if (n_slots > 1 && w_stride < (int64_t)n * k) return bad(who, "w_stride is less than a matrix"), -1;
    if ((!row_in && n_rows > n_x) || (!row_out && n_rows > n_y)) return bad(who, "more rows than x or y has"), -1;
    if (n_rows == 0 || n_y == 0) return 0;
    a.p = x, a.q = w, a.out = y, a.row_p = row_in, a.row_out = row_out, a.scale = scale;
    a.ldp = ldx, a.ldq = w_stride, a.ldo = ldy, a.n_p = n_x, a.n_out = n_y, a.nq = n, a.nc = k;
    return launch_typed<kMM>(a, dtype, (hipStream_t)stream);
}

int moe_grouped_gate_up(const void* x, int64_t ldx, int n_x, const int32_t* row_in, const int32_t* seg_start,
                        const int32_t* seg_slot, int n_seg, int n_rows, const void* w, int64_t w_stride, int n_slots,
                        int inter, int hidden, void* h, int64_t ldh, void* gu, int64_t ldgu, int dtype, int fill,
                        void* stream) {
    const char* who = "grouped_gate_up";
    Args a = {};
    a.S = Segs{seg_start, seg_slot, n_seg, n_rows, n_slots, fill};
    if (bad_segs(who, a.S, inter, hidden, dtype, w) || bad_matrix(who, "x", x, ldx, hidden, n_x) ||
        bad_matrix(who, "w", w, w_stride, hidden, n_slots) || bad_matrix(who, "h", h, ldh, inter, n_rows) ||
        (gu && bad_matrix(who, "gu", gu, ldgu, 2 * (int64_t)inter, n_rows)))
        return -1;
    if (n_slots > 1 && w_stride < 2 * (int64_t)inter * hidden) return bad(who, "w_stride is less than a matrix"), -1;
    if (!row_in && n_rows > n_x) return bad(who, "more rows than x has"), -1;
    if (n_rows == 0) return 0;
    a.p = x, a.q = w, a.out = h, a.row_p = row_in, a.gu_out = gu;
    a.ldp = ldx, a.ldq = w_stride, a.ldo = ldh, a.ldgu = ldgu, a.n_p = n_x, a.n_out = n_rows, a.nq = inter, a.nc = hidden;
    return launch_typed<kGateUp>(a, dtype, (hipStream_t)stream);
}

int moe_grouped_mm_dx(const void* dy, int64_t lddy, int n_dy, const int32_t* row_in, const int32_t* seg_start,
                      const int32_t* seg_slot, int n_seg, int n_rows, const void* w, int64_t w_stride, int n_slots, int n,
                      int k, const float* scale, const void* gu, int64_t ldgu, void* dx, int64_t lddx, int n_dx,
                      const int32_t* row_out, int dtype, int fill, void* stream) {
    const char* who = "grouped_mm_dx";
    Args a = {};
    a.S = Segs{seg_start, seg_slot, n_seg, n_rows, n_slots, fill};
    if (bad_segs(who, a.S, n, k, dtype, w) || bad_matrix(who, "dy", dy, lddy, n, n_dy) ||
        bad_matrix(who, "w", w, w_stride, k, n_slots) ||
        bad_matrix(who, "dx", dx, lddx, (gu ? 2 : 1) * (int64_t)k, n_dx) ||
        (gu && bad_matrix(who, "gu", gu, ldgu, 2 * (int64_t)k, n_rows)))
        return -1;
    if (n_slots > 1 && w_stride < (int64_t)n * k) return bad(who, "w_stride is less than a matrix"), -1;
    if ((!row_in && n_rows > n_dy) || (!row_out && n_rows > n_dx)) return bad(who, "more rows than dy or dx has"), -1;
    if (n_rows == 0 || n_dx == 0) return 0;
    a.p = dy, a.q = w, a.out = dx, a.row_p = row_in, a.row_out = row_out, a.scale = scale, a.gu = gu;
    a.ldp = lddy, a.ldq = w_stride, a.ldo = lddx, a.ldgu = ldgu, a.n_p = n_dy, a.n_out = n_dx, a.nq = k, a.nc = n;
    return gu ? launch_typed<kDxGlu>(a, dtype, (hipStream_t)stream) : launch_typed<kDx>(a, dtype, (hipStream_t)stream);
}

int moe_grouped_mm_dw(const void* dy, int64_t lddy, int n_dy, const int32_t* row_dy, const void* x, int64_t ldx, int n_x,
                      const int32_t* row_x, const int32_t* seg_start, int n_seg, int n_rows, int n, int k,
                      const float* scale, void* dw, int64_t dw_stride, int out_f32, int dtype, void* stream) {
    const char* who = "grouped_mm_dw";
    Args a = {};
    a.S = Segs{seg_start, nullptr, n_seg, n_rows, n_seg, 0};
    if (bad_segs(who, a.S, n, k, dtype, dw) || bad_matrix(who, "dy", dy, lddy, n, n_dy) ||
        bad_matrix(who, "x", x, ldx, k, n_x) || bad_matrix(who, "dw", dw, dw_stride, k, n_seg))
        return -1;
    if (n_seg > 1 && dw_stride < (int64_t)n * k) return bad(who, "dw_stride is less than a matrix"), -1;
    if ((!row_dy && n_rows > n_dy) || (!row_x && n_rows > n_x)) return bad(who, "more rows than dy or x has"), -1;
    if (n_seg == 0) return 0;
    a.p = dy, a.q = x, a.out = dw, a.row_p = row_dy, a.row_q = row_x, a.scale = scale;
    a.ldp = lddy, a.ldq = ldx, a.ldo = dw_stride, a.n_p = n_dy, a.n_q = n_x, a.np = n, a.nq = k, a.out_f32 = out_f32;
    return launch_typed<kDw>(a, dtype, (hipStream_t)stream);
}

}  // extern "C"
