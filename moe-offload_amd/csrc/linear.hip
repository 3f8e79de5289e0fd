// A projection that all tokens share (the router, a shared expert), with what surrounds it in the same launch, and its
// gradients:
//     z = x W^T + bias,   y = act(z) + residual        (bias and residual may be absent; z is kept where it is asked for)
//     dz = dy act'(z),    dx = dz W,   dW = dz^T x,   dbias = the sum of dz over the tokens
// act: none, silu, gelu (z times the normal distribution's integral) or the squared relu.  x, W, bias, residual and z are
// fp16 or bf16, y too or fp32, sums and everything between a load and a store fp32.
//
// All three products are one tile product  out[p][q] = sum over c of P[p][c] Q[q][c]  as the grouped products' are
// (grouped_mm.h: loads straight into LDS, operands along or across a row of memory), without rows to look up: x and W have c
// along a row, W for dx has it along the column, dz and x for dW both.
//
// dz goes to the matrix unit as it came where it is dy itself, in the inputs' type.  Where it is computed, or dy is fp32, one value of
// 16 bits would add an error as large as the results' own rounding (fp16, 1999 x 2560 x 640 through silu: 2.9e-4 of the norm
// for 2.1e-4), and fp16 has no place for all that dy may hold.  So it goes in parts, images one after another in the contraction:
//   kParts   bf16 values, each with the next 8 of its bits, over fp32's range: two for results of 16 bits (2^-15 of a value is lost at
//            most), three for fp32 ones (nothing is).  fp16's x and W, two bf16 values each, take every product twice.
//   kHalves  for fp16 dy through slopes that are never above 1.13, and results of 16 bits: dz / 2 as two fp16 values, the
//            second times 2^10 (2^-21 of a value is lost, or 2^-33), half the products of kParts.
// us of both gradients through silu, fp16, as one value, in kHalves and in kParts: 1999 x 2560 x 640 28 43 80, 8192 x 4096 x 4096 440 841
// 1554; bf16, as one value and in kParts: 28 45, 430 801.
#include <algorithm>
#include <type_traits>

#include "grouped_mm.h"
#include "lane_reduce.h"

namespace {

using namespace gmm;

enum { kActNone = 0, kActSilu = 1, kActGelu = 2, kActRelu2 = 3 };

// The normal distribution's integral up to -m, m >= 0, times exp(m^2 / 2), as a polynomial in t = 1 / (1 + 0.27 m): fitted to its relative
// error for m up to 20 (least squares over 4000 Chebyshev points, weighted anew until the largest was least), 2.4e-8 of the value;
// in fp32, with the exponential, (m^2 / 2 + 4) steps of 2^-23 of it.
__device__ __forceinline__ float normal_tail(float m) {
    const float t = __builtin_amdgcn_rcpf(1.f + 0.27f * m);
    constexpr float c[] = {0.10772167f, 0.107526444f, 0.10192253f, 0.071631186f, 0.10876759f, -0.070522137f, 0.17089182f, -0.12700342f,
                           0.029064333f};
    float poly = c[8];
#pragma unroll
    for (int i = 7; i >= 0; --i) poly = c[i] + t * poly;
    return t * poly * __builtin_amdgcn_exp2f(m * m * -0.72134752f);
}

// The activations, and their slopes.  Where exponentials have left fp32's range both are at their limits, taken from arguments
// that are not infinite: an infinity would meet a zero.  A NaN stays one.
template <int ACT>
__device__ __forceinline__ float activation(float z) {
    if constexpr (ACT == kActRelu2) return z < 0.f ? 0.f : z * z;
    if constexpr (ACT == kActSilu) {
        const float low = z < -200.f ? -200.f : z;
        return low / (1.0f + __expf(-low));
    }
    if constexpr (ACT == kActGelu) {
        const float m = fminf(fabsf(z), 200.f);                                // z N(z) = max(z, 0) - |z| N(-|z|)
        return (z < 0.f ? 0.f : z) - m * normal_tail(m);
    }
    return z;
}

template <int ACT>
__device__ __forceinline__ float slope(float z) {
    if constexpr (ACT == kActRelu2) return z < 0.f ? 0.f : 2.f * z;
    const float low = z < -200.f ? -200.f : z, both = low > 200.f ? 200.f : low;
    if constexpr (ACT == kActSilu) {
        const float sg = 1.0f / (1.0f + __expf(-low));
        return sg * (1.0f + both * (1.0f - sg));
    }
    if constexpr (ACT == kActGelu) {
        const float tail = normal_tail(fabsf(both));
        return (both < 0.f ? tail : 1.f - tail) + both * 0.39894228f * __expf(-0.5f * both * both);
    }
    return 1.f;
}

// Calls f with the activation as a type: one branch for many values.
template <typename F>
__device__ __forceinline__ void by_act(int act, const F& f) {
    if (act == kActNone) f(std::integral_constant<int, kActNone>());
    else if (act == kActSilu) f(std::integral_constant<int, kActSilu>());
    else if (act == kActGelu) f(std::integral_constant<int, kActGelu>());
    else f(std::integral_constant<int, kActRelu2>());
}

// What a product does with its results: z = sum + bias, out = act(z) + res.
struct Epilogue {
    const void* bias;
    const void* res;
    void* z;
    int64_t ldr, ldz;
    int act, out_f32;
};

struct Product {
    const void* p;
    const void* q;
    void* out;
    int64_t ldp, ldq, ldo;       // elements from row to row of memory
    int np, nq, nc;              // extents: rows and columns of out, and the contraction
    int parts, part_c;           // the contraction in parts of part_c, each with sums of its own (fp32, [parts][np][nq]; not dx)
    int terms;                   // kParts, kHalves: P is the sum of so many images, one after another from p on,
    int64_t term_p;              // so many elements apart; the contraction goes over all of them
};

enum { kForward = 0, kDx = 1, kDw = 2 };
enum { kWhole = 0, kParts = 1, kHalves = 2 };                                  // how P comes

constexpr float kSecondHalf = 0x1p-10f;                                        // of kHalves, the first image

template <typename T>
__device__ __forceinline__ uint4 round8(const f32x4 (&v)[2]) {
    const uint2 lo = round4<T>(v[0]), hi = round4<T>(v[1]);
    return make_uint4(lo.x, lo.y, hi.x, hi.y);
}

template <typename T>
__device__ __forceinline__ void widen8(uint4 v, f32x4 (&f)[2]) {
    f[0] = widen4<T>(make_uint2(v.x, v.y));
    f[1] = widen4<T>(make_uint2(v.z, v.w));
}

// 8 adjacent columns of a row out: act(sum + bias) + res, and z.
template <typename T>
__device__ __forceinline__ void finish8(const Product& a, const Epilogue& e, int64_t r, int c, const f32x4 (&sum)[2],
                                        const f32x4 (&bias)[2], uint4 res) {
    f32x4 z[2], y[2], rs[2];
    widen8<T>(res, rs);
    by_act(e.act, [&](auto act) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            z[h] = sum[h] + bias[h];
#pragma unroll
            for (int i = 0; i < 4; ++i) y[h][i] = activation<decltype(act)::value>(z[h][i]) + rs[h][i];
        }
    });
    if (e.z) store16((T*)e.z + r * e.ldz + c, round8<T>(z));
    if (e.out_f32) {
        float* d = (float*)a.out + r * a.ldo + c;
        store16(d, __builtin_bit_cast(uint4, y[0]));
        store16(d + 4, __builtin_bit_cast(uint4, y[1]));
    } else {
        store16((T*)a.out + r * a.ldo + c, round8<T>(y));
    }
}

// c + q p, and in kParts p, a bf16 part of a value, goes with q of T: fp16's 11 bits are two bf16 values, the upper 8 and
// the other 3.  An infinite q is infinite in both, and of one that the first holds whole the second is as good as nothing, but not
// zero: so the sum is infinite where q p is, and a NaN only where that is one.
template <typename T, int MODE>
__device__ __forceinline__ f32x4 multiply(uint4 q, uint4 p, f32x4 c) {
    if constexpr (MODE == kParts && __is_same(T, _Float16)) {
        typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
        const uint32_t v[4] = {q.x, q.y, q.z, q.w};
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const f16x2 both = __builtin_bit_cast(f16x2, v[e]), top = __builtin_bit_cast(f16x2, v[e] & 0xFFF8FFF8u);
            // up to 7 of the value's last steps, 32 at most; of an infinity -256, which the infinity below outweighs
            const f16x2 rest = __builtin_elementwise_max(both - top, (f16x2)(-256.f));
            uint32_t t[2], r[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                t[k] = __builtin_bit_cast(uint32_t, (float)top[k]);
                r[k] = __builtin_bit_cast(uint32_t, __builtin_fmaf((float)both[k], 0x1p-40f, (float)rest[k]));
            }
            hi[e] = __builtin_amdgcn_perm(t[1], t[0], 0x07060302);             // upper halves (a NaN's quiet bit is among them)
            lo[e] = __builtin_amdgcn_perm(r[1], r[0], 0x07060302);
        }
        c = mfma<__bf16>(make_uint4(hi[0], hi[1], hi[2], hi[3]), p, c);
        return mfma<__bf16>(make_uint4(lo[0], lo[1], lo[2], lo[3]), p, c);
    } else {
        return mfma<T>(q, p, c);
    }
}

template <int BP, int BQ>
__host__ __device__ inline int64_t tiles_in(const Product& a) {
    return ((int64_t)a.np + BP - 1) / BP * (((int64_t)a.nq + BQ - 1) / BQ);
}

// Item -> tile: panels of PANEL columns of tiles, row by row in each, so that the tiles that an XCD works on at a time (its items
// follow each other) are a square rather than a line, and share their rows of both operands in its L2.
template <int BP, int BQ, int PANEL>
__device__ __forceinline__ void tile_at(const Product& a, uint32_t item, int& p0, int& q0) {
    const uint32_t tp = (a.np + BP - 1) / BP, tq = (a.nq + BQ - 1) / BQ, full = tp * PANEL;
    const uint32_t panel = item / full, left = tq - panel * PANEL, width = left < PANEL ? left : PANEL, i = item - panel * full;
    p0 = (int)(i / width) * BP;
    q0 = (int)(panel * PANEL + i % width) * BQ;
}

// What bounds it: full grids of large tiles the matrix unit and what feeds it (8192 x 4096 x 4096 bf16 in 256 x 256: 190-205 us, 1340-1450
// TFLOP/s, 1.4 us a step and 8 at a tile's ends; the library's product 177-185), grids of one tile per CU the steps' latencies (4096 x 2048 x
// 512 in 128 x 64: 12.5-14.3 us on one box and another, 0.3 us a step, the waves waiting for 48% of it, the matrix unit busy for 28%, LDS for
// 30%; the library's 15).  In panels: 4096 x 4096 x 4096 in tiles of 64 205 us, 294 in lines, of 256 105 and 113.  Tiles of 256 x 256 by
// four waves of 128 x 128, which read LDS less, took 106-121 for it: a wave alone on its SIMD waits for every load that it issues.
//
// One tile of BP x BQ results by WP x WQ waves, or SPLIT = 2 times as many that take turns at the steps.  A step of 64 contraction
// indexes goes from global memory to LDS without passing registers, RING - 1 steps ahead of the one that is multiplied: with one
// tile per block nothing else hides the way through memory.  One barrier per step (and two steps, of SPLIT = 2), at its start or,
// in large tiles, in its middle, where half of the next step's operands are read from LDS behind this one's products.
template <typename T, int KIND, typename C, int MODE = kWhole>
__device__ __forceinline__ void tile_product(const Product& a, const Epilogue& e, uint32_t item, uint8_t* lds) {
    constexpr int BP = C::BP, BQ = C::BQ, WP = C::WP, WQ = C::WQ, RING = C::RING, SPLIT = C::SPLIT;
    constexpr int kWaves = WP * WQ, SP = BP / WP / 16, SQ = BQ / WQ / 16;
    constexpr bool kAlongP = KIND == kDw, kAlongQ = KIND != kForward;
    constexpr int kLoadsP = BP / 8 / kWaves, kLoadsQ = BQ / 8 / kWaves, kLoads = kLoadsP + kLoadsQ;   // 1 KiB each
    constexpr uint32_t kStageP = BP * 128, kStage = (BP + BQ) * 128;
    static_assert((SQ == 2 || SQ == 4) && BP % (8 * kWaves) == 0 && BQ % (8 * kWaves) == 0 && RING * kStage / kWaves >= SQ * 1024, "");
    const int t = threadIdx.x, lane = t & 63, all = __builtin_amdgcn_readfirstlane(t >> 6), turn_of = all / kWaves, wv = all % kWaves;
    const uint32_t lds_all = (uint32_t)(uintptr_t)(lds_u8*)lds, lds0 = lds_all + turn_of * RING * kStage;
    const T* P = (const T*)a.p;
    const T* Q = (const T*)a.q;
    int nc = a.nc;
    int64_t part = 0;
    if (KIND != kDx && a.parts > 1) {
        const uint32_t tiles = (uint32_t)tiles_in<BP, BQ>(a);
        part = item / tiles;
        item -= (uint32_t)part * tiles;
        P += part * a.part_c * (kAlongP ? a.ldp : 1);
        Q += part * a.part_c * (kAlongQ ? a.ldq : 1);
        nc = (int)std::min<int64_t>(nc - part * a.part_c, a.part_c);
    }
    // P's images follow each other in the contraction, each as whole steps
    int term = 0;
    const int whole = (nc + kBC - 1) / kBC * kBC;
    const uint32_t all_c = MODE == kWhole ? nc : (uint32_t)a.terms * whole;
    int p0, q0;
    tile_at<BP, BQ, C::PANEL>(a, item, p0, q0);
    const T* zero = (const T*)&g_zero16;
    asm("" : "+s"(zero));                                                      // kept in registers
    // Where this lane's 16 bytes of each of its wave's next loads are.  Rows and columns past the end read some that exist:
    // their results are not stored.  Contraction indexes past the end read zeros.
    const T* pp[kLoadsP];
    const T* qp[kLoadsQ];
    const int cu = ((lane & 7) ^ (lane >> 3)) * 8;                             // not ALONG: first c of the 16 bytes
    int load_c = turn_of * kBC;
    auto place_one = [&](auto along, auto width, const T* base, int64_t ld, int first, int n, int wave_loads, int j) -> const T* {
        constexpr int W = decltype(width)::value, kUnits = W / 8;
        if constexpr (decltype(along)::value) {
            const int row = (wv * wave_loads + j) * (64 / kUnits) + lane / kUnits, col = first + (lane % kUnits ^ 2 * turn<W>(row)) * 8;
            const int c = load_c + row;
            return c < nc ? base + c * ld + (col < n ? col : 0) : zero;
        } else {
            const int r = first + (wv * wave_loads + j) * 8 + (lane >> 3);
            return load_c + cu < nc ? base + (r < n ? r : n - 1) * ld + load_c + cu : zero;
        }
    };
    auto place = [&]() {
        if constexpr (MODE != kWhole) {
            for (; load_c >= whole && term < a.terms; ++term) {
                load_c -= whole;
                P += a.term_p;
            }
            if (term == a.terms) nc = 0;
        }
#pragma unroll
        for (int j = 0; j < kLoadsP; ++j)
            pp[j] = place_one(std::integral_constant<bool, kAlongP>(), std::integral_constant<int, BP>(), P, a.ldp, p0, a.np, kLoadsP, j);
#pragma unroll
        for (int j = 0; j < kLoadsQ; ++j)
            qp[j] = place_one(std::integral_constant<bool, kAlongQ>(), std::integral_constant<int, BQ>(), Q, a.ldq, q0, a.nq, kLoadsQ, j);
    };
    auto advance = [&]() {
        load_c += SPLIT * kBC;
        if (load_c + kBC <= nc) {
#pragma unroll
            for (int j = 0; j < kLoadsP; ++j) pp[j] += kAlongP ? SPLIT * kBC * a.ldp : SPLIT * kBC;
#pragma unroll
            for (int j = 0; j < kLoadsQ; ++j) qp[j] += kAlongQ ? SPLIT * kBC * a.ldq : SPLIT * kBC;
        } else {
            place();
        }
    };
    auto load = [&](int d, uint32_t stage) {
        if (d < kLoadsP) load_to_lds(pp[d], lds0 + stage + (wv * kLoadsP + d) * 1024);
        else load_to_lds(qp[d - kLoadsP], lds0 + stage + kStageP + (wv * kLoadsQ + d - kLoadsP) * 1024);
    };
    const int wp = wv / WQ, wq = wv % WQ;
    Frags<kAlongP, BP, SP> fp;
    Frags<kAlongQ, BQ, SQ> fq;
    fp.init(lds0, wp * SP * 16, lane);
    fq.init(lds0 + kStageP, wq * SQ * 16, lane);
    f32x4 acc[SP][SQ] = {};
    place();
    auto wait = [&](auto outstanding) {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(decltype(outstanding)::value * kLoads) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    auto after = [](uint32_t stage) { return stage + kStage == RING * kStage ? 0 : stage + kStage; };
    // Both loops: us of forward products of 4096 x 4096 x 4096 in 256 x 256 100 and 104, 2048 x 2048 x 2048 in 128 x 128 20.8 and
    // 21.7, 4096 x 2048 x 512 in 128 x 64 13.3 and 13.0, 1024 x 1024 x 1024 in 64 x 64 7.2 and 6.6; of both gradients, which read LDS
    // with twice as many instructions, 8192 x 2048 x 2048 in 256 x 128 117 and 120, 2048 x 2048 x 1024 in 128 x 128, four steps in the
    // ring, 23.6 and 21.2.
    constexpr bool kHalfAhead = BP * BQ >= 128 * 128 && (KIND == kForward || RING < 4);
    static_assert(!kHalfAhead || SPLIT == 1, "");
    constexpr int kAhead = kHalfAhead ? RING : RING - 1;                       // steps that are loaded before the first product
    uint4 vp[2][SP], vq[2][SQ];
    uint32_t stage = 0;
    bool second = MODE == kHalves;                                             // the sums are those of the second halves
    auto scale_sums = [&](float by) {
#pragma unroll
        for (int i = 0; i < SP; ++i)
#pragma unroll
            for (int j = 0; j < SQ; ++j) acc[i][j] *= by;
    };
    auto first_halves_from = [&](uint32_t c) {
        if (MODE == kHalves && second && c >= (uint32_t)whole) {
            scale_sums(kSecondHalf);
            second = false;
        }
    };
#pragma unroll
    for (int s = 0; s < kAhead; ++s) {
#pragma unroll
        for (int d = 0; d < kLoads; ++d) load(d, s * kStage);
        advance();
    }
    if constexpr (kHalfAhead) {
        // One barrier, in the middle of a step: past it everyone's loads of the next step have landed, and everyone's reads of this
        // one are done, so that the loads of the step RING on go where it was.  The reads and loads come one by one between the
        // products: a wave that issues many together waits for the unit that takes them, and its products with it.
        auto read_some = [&](auto half, uint32_t from, int i) {
            constexpr int H = decltype(half)::value, kReads = SP + SQ;
#pragma unroll
            for (int x = 0; x < kReads; ++x) {
                if (x < i * kReads / (SP - 1) || x >= (i + 1) * kReads / (SP - 1)) continue;
                if (x > 0 && x <= SQ) vq[H][x - 1] = fq.read(from, x - 1, H);
                else vp[H][x == 0 ? 0 : x - SQ] = fp.read(from, x == 0 ? 0 : x - SQ, H);
            }
        };
        const std::integral_constant<int, 0> first;
        const std::integral_constant<int, 1> second;
        wait(std::integral_constant<int, RING - 1>());
#pragma unroll
        for (int i = 0; i < SP - 1; ++i) read_some(first, stage, i);
#pragma unroll 1
        for (uint32_t c0 = 0; c0 < all_c; c0 += kBC) {
            const uint32_t next = after(stage);
            first_halves_from(c0);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < SP; ++i) {
                if (i < SP - 1) read_some(second, stage, i);
#pragma unroll
                for (int j = 0; j < SQ; ++j) acc[i][j] = multiply<T, MODE>(vq[0][j], vp[0][i], acc[i][j]);
                __builtin_amdgcn_sched_barrier(0);
            }
            wait(std::integral_constant<int, RING - 2>());
#pragma unroll
            for (int i = 0; i < SP; ++i) {
                if (i < SP - 1) read_some(first, next, i);
#pragma unroll
                for (int d = i * kLoads / SP; d < (i + 1) * kLoads / SP; ++d) load(d, stage);
#pragma unroll
                for (int j = 0; j < SQ; ++j) acc[i][j] = multiply<T, MODE>(vq[1][j], vp[1][i], acc[i][j]);
                __builtin_amdgcn_sched_barrier(0);
            }
            advance();
            stage = next;
        }
    } else {
        uint32_t fill = (RING - 1) * kStage;
#pragma unroll 1
        for (uint32_t c0 = 0; c0 < all_c; c0 += SPLIT * kBC) {
            // this wave's loads of the step have landed and its reads of the step before are done; past the barrier, so are
            // everyone's
            wait(std::integral_constant<int, RING - 2>());
            first_halves_from(c0 + turn_of * kBC);
#pragma unroll
            for (int j = 0; j < SQ; ++j) vq[0][j] = fq.read(stage, j, 0);
#pragma unroll
            for (int i = 0; i < SP; ++i) vp[0][i] = fp.read(stage, i, 0);
            __builtin_amdgcn_sched_barrier(0);
            // the step's second half is read from LDS, and the loads ahead are issued, between the first half's products
#pragma unroll
            for (int i = 0; i < SP; ++i) {
                if (i == 0) {
#pragma unroll
                    for (int j = 0; j < SQ; ++j) vq[1][j] = fq.read(stage, j, 1);
                }
                vp[1][i] = fp.read(stage, i, 1);
#pragma unroll
                for (int j = 0; j < SQ; ++j) acc[i][j] = multiply<T, MODE>(vq[0][j], vp[0][i], acc[i][j]);
#pragma unroll
                for (int d = i * kLoads / SP; d < (i + 1) * kLoads / SP; ++d) load(d, fill);
                __builtin_amdgcn_sched_barrier(0);
            }
            advance();
#pragma unroll
            for (int i = 0; i < SP; ++i)
#pragma unroll
                for (int j = 0; j < SQ; ++j) acc[i][j] = multiply<T, MODE>(vq[1][j], vp[1][i], acc[i][j]);
            stage = after(stage);
            fill = after(fill);
        }
    }
    if constexpr (MODE == kHalves) scale_sums(second ? 2.f * kSecondHalf : 2.f);
    // The results go through LDS, one of a wave's subtile rows at a time: a lane of the matrix unit's result has 4 columns of
    // a row and its neighbour another row's; out of LDS 8 columns, and whole lines side by side.  (The loads past the last
    // step write there too, so they are waited for.)
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) u32x4* lds16;
    constexpr int kUnits = SQ * 2, kRowsPer = 64 / kUnits, kIts = 16 / kRowsPer;
    constexpr int kOwn = SP / SPLIT;                                           // subtile rows that a wave finishes
    if constexpr (SPLIT == 2) {
        // the waves of a turn hand the other's half of the rows over and add what they get
        static_assert(2 * kWaves * kOwn * SQ * 1024 <= SPLIT * RING * kStage, "");
        auto box = [&](int turn, int i, int j) {
            return lds_all + (uint32_t)((((turn * kWaves + wv) * kOwn + i) * SQ + j) * 1024 + lane * 16);
        };
#pragma unroll
        for (int i = 0; i < kOwn; ++i)
#pragma unroll
            for (int j = 0; j < SQ; ++j)
                *(lds16)(uintptr_t)box(turn_of, i, j) = __builtin_bit_cast(u32x4, turn_of ? acc[i][j] : acc[kOwn + i][j]);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kOwn; ++i)
#pragma unroll
            for (int j = 0; j < SQ; ++j)
                acc[i][j] = (turn_of ? acc[kOwn + i][j] : acc[i][j]) + __builtin_bit_cast(f32x4, *(lds16)(uintptr_t)box(1 - turn_of, i, j));
        __syncthreads();
    }
    int l = lane;
    asm volatile("" : "+v"(l));                                                // no addresses are kept over the products
    const int l16 = l & 15, lq = l >> 4, u8 = l % kUnits, c = q0 + wq * SQ * 16 + u8 * 8;
    const uint32_t area = lds_all + all * (SQ * 1024);
    auto at = [&](int row, int u) { return area + (uint32_t)(row * SQ * 4 + (u ^ (row & 7))) * 16; };
    const bool in = c < a.nq;
    f32x4 bias[2] = {};
    if (KIND == kForward && e.bias && in) widen8<T>(*(const uint4*)((const T*)e.bias + c), bias);
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
        uint4 rv[kIts];
        int row[kIts];
#pragma unroll
        for (int it = 0; it < kIts; ++it) {
            const int r = p0 + wp * SP * 16 + (turn_of * kOwn + i) * 16 + it * kRowsPer + l / kUnits;
            row[it] = r < a.np && in ? r : -1;
            rv[it] = make_uint4(0, 0, 0, 0);
            if (KIND == kForward && e.res && row[it] >= 0) rv[it] = *(const uint4*)((const T*)e.res + row[it] * e.ldr + c);
        }
#pragma unroll
        for (int j = 0; j < SQ; ++j) *(lds16)(uintptr_t)at(l16, 4 * j + lq) = __builtin_bit_cast(u32x4, acc[i][j]);
#pragma unroll
        for (int it = 0; it < kIts; ++it) {
            const int m = it * kRowsPer + l / kUnits;
            const f32x4 sum[2] = {__builtin_bit_cast(f32x4, *(lds16)(uintptr_t)at(m, 2 * u8)),
                                  __builtin_bit_cast(f32x4, *(lds16)(uintptr_t)at(m, 2 * u8 + 1))};
            if (row[it] < 0) continue;
            if ((KIND == kDw && e.out_f32) || (KIND == kForward && a.parts > 1)) {
                float* d = (float*)a.out + (part * a.np + row[it]) * a.ldo + c;
                store16(d, __builtin_bit_cast(uint4, sum[0]));
                store16(d + 4, __builtin_bit_cast(uint4, sum[1]));
            } else if constexpr (KIND == kForward) {
                finish8<T>(a, e, row[it], c, sum, bias, rv[it]);
            } else {
                store16((T*)a.out + row[it] * a.ldo + c, round8<T>(sum));
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    }
}

// A tile's sides, its waves, how many share the steps, its ring, the waves per SIMD that registers are kept for (of one block of eight
// waves, as LDS holds no second, or of two blocks of four), the panel.
template <int BP_, int BQ_, int WP_, int WQ_, int SPLIT_, int RING_, int PER_SIMD_, int PANEL_>
struct Tiles {
    static constexpr int BP = BP_, BQ = BQ_, WP = WP_, WQ = WQ_, SPLIT = SPLIT_, RING = RING_, PER_SIMD = PER_SIMD_, PANEL = PANEL_;
    static constexpr int kThreads = 64 * WP * WQ * SPLIT, kLds = SPLIT * RING * (BP + BQ) * 128;
};

template <typename T, typename C>
__global__ __launch_bounds__(C::kThreads, C::PER_SIMD) void k_linear(Product a, Epilogue e) {
    __shared__ __attribute__((aligned(1024))) uint8_t lds[C::kLds];
    tile_product<T, kForward, C>(a, e, xcd_order(blockIdx.x, gridDim.x), lds);
}

// y from the parts of its contraction, in their order: a thread has 8 columns of a row.
template <typename T>
__global__ __launch_bounds__(256) void k_linear_join(const float* __restrict__ sums, int parts, Product a, Epilogue e) {
    const uint32_t units = a.nq / 8;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, r = i / units;
    const int c = (int)(i - r * units) * 8;
    if (r >= a.np) return;
    f32x4 s[2] = {}, bias[2] = {};
    const float* from = sums + r * a.nq + c;
    const int64_t step = (int64_t)a.np * a.nq;
    uint4 res = make_uint4(0, 0, 0, 0);
    if (e.res) res = *(const uint4*)((const T*)e.res + r * e.ldr + c);
    if (e.bias) widen8<T>(*(const uint4*)((const T*)e.bias + c), bias);
#pragma unroll 4
    for (int k = 0; k < parts; ++k) {
        s[0] += *(const f32x4*)(from + k * step);
        s[1] += *(const f32x4*)(from + k * step + 4);
    }
    finish8<T>(a, e, r, c, s, bias, res);
}

// What k_linear_dz left of the bias's gradient: [blocks][n], summed in order by a block of 64 columns and 4 parts of the rows.
struct BiasSums {
    const float* sums;
    void* db;
    int blocks, n;
};

template <typename T, int THREADS>
__device__ __forceinline__ void sum_bias(const BiasSums& b, uint32_t item, float* lds) {
    constexpr int kParts = THREADS / 64;
    const int c = (int)item * 64 + (threadIdx.x & 63), part = threadIdx.x >> 6;
    float s = 0.f;
    if (c < b.n) {
        const int from = (int)((int64_t)b.blocks * part / kParts), to = (int)((int64_t)b.blocks * (part + 1) / kParts);
#pragma unroll 8
        for (int i = from; i < to; ++i) s += b.sums[(int64_t)i * b.n + c];
    }
    lds[threadIdx.x] = s;
    __syncthreads();
    if (part == 0 && c < b.n) {
        for (int i = 1; i < kParts; ++i) s += lds[i * 64 + threadIdx.x];
        ((T*)b.db)[c] = (T)s;
    }
}

// All gradients behind dz in one launch: the tiles of dW (longer, as a rule) before those of dx, then the bias's.  A product of no
// rows is not there.
template <typename T, typename C, int MODE>
__global__ __launch_bounds__(C::kThreads, C::PER_SIMD) void k_linear_grads(Product dw, Product dx, BiasSums b, int dw_f32) {
    __shared__ __attribute__((aligned(1024))) uint8_t lds[C::kLds];
    const uint32_t n_dw = (uint32_t)tiles_in<C::BP, C::BQ>(dw) * dw.parts, n_dx = (uint32_t)tiles_in<C::BP, C::BQ>(dx);
    const uint32_t i = blockIdx.x;
    Epilogue e = {};
    e.out_f32 = dw_f32;
    if (i < n_dw) tile_product<T, kDw, C, MODE>(dw, e, xcd_order(i, n_dw), lds);
    else if (i < n_dw + n_dx) tile_product<T, kDx, C, MODE>(dx, e, xcd_order(i - n_dw, n_dx), lds);
    else sum_bias<T, C::kThreads>(b, i - n_dw - n_dx, (float*)lds);
}

// dW from its parts, in their order, and behind those blocks the bias's gradient.
struct Parts {
    const float* sums;
    void* dw;
    int64_t n;                   // elements of dW, a multiple of 8
    int parts, f32;
};

template <typename T>
__global__ __launch_bounds__(256) void k_linear_parts(Parts p, uint32_t blocks, BiasSums b) {
    __shared__ float lds[256];
    if (blockIdx.x >= blocks) {
        sum_bias<T, 256>(b, blockIdx.x - blocks, lds);
        return;
    }
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
    if (i >= p.n) return;
    f32x4 s[2] = {};
#pragma unroll 4
    for (int k = 0; k < p.parts; ++k) {
        s[0] += *(const f32x4*)(p.sums + k * p.n + i);
        s[1] += *(const f32x4*)(p.sums + k * p.n + i + 4);
    }
    if (p.f32) {
        *(f32x4*)((float*)p.dw + i) = s[0];
        *(f32x4*)((float*)p.dw + i + 4) = s[1];
    } else {
        *(uint4*)((T*)p.dw + i) = round8<T>(s);
    }
}

// Up to 256 tiles of 16 x 16, and up to 16 tokens, where a tile of 64 rows would be mostly empty.  us of these and of the tiles above:
// 8 x 2048 x 2048 5.7 and 8.3, 24 x 2048 x 2048 (256 of them) 6.4 and 8.4, 64 x 2048 x 512 (128) 6.5 and 8.3; 48 x 2048 x 2048 (384)
// 9.9 and 8.4, 512 x 2048 x 512 (1024) 17.8 and 8.6.  8 x 2048 x 2048: 8.5 MB at 1.5 TB/s, one run through memory and back.
//
// Few results: a block has 16 x 16 of them, its waves take turns at the steps, and their sums meet in LDS.  Rows of both
// operands come straight into the matrix unit's layout, four of a wave's steps under way at once, and no wave waits for another
// before the end.
constexpr int kFewWaves = 8;

template <typename T>
__global__ __launch_bounds__(64 * kFewWaves) void k_linear_few(Product a, Epilogue e) {
    constexpr int kAhead = 4;
    __shared__ f32x4 part[kFewWaves][64];
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, kq = lane >> 4;
    const uint32_t item = xcd_order(blockIdx.x, gridDim.x), tp = (a.np + 15) / 16;
    const int p0 = (int)(item % tp) * 16, q0 = (int)(item / tp) * 16, steps = (a.nc + kBC - 1) / kBC;
    const T* W = (const T*)a.q + (int64_t)(q0 + n < a.nq ? q0 + n : a.nq - 1) * a.ldq + kq * 8;
    const T* X = (const T*)a.p + (int64_t)(p0 + n < a.np ? p0 + n : a.np - 1) * a.ldp + kq * 8;
    f32x4 acc = {};
    const T* zero = (const T*)&g_zero16;
    for (int s = wv; s < steps; s += kFewWaves * kAhead) {
        uint4 w[kAhead][2], x[kAhead][2];
        auto read = [&](auto inside) {
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
#pragma unroll
                for (int ks = 0; ks < 2; ++ks) {
                    const int c = (s + u * kFewWaves) * kBC + ks * 32;
                    const bool in = decltype(inside)::value || c + kq * 8 < a.nc;
                    w[u][ks] = *(const uint4*)(in ? W + c : zero);
                    x[u][ks] = *(const uint4*)(in ? X + c : zero);
                }
        };
        if ((s + (kAhead - 1) * kFewWaves + 1) * kBC <= a.nc) read(std::true_type());
        else read(std::false_type());
        __builtin_amdgcn_sched_barrier(0);                                     // all loads before the first wait
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) acc = mfma<T>(w[u][ks], x[u][ks], acc);
    }
    part[wv][lane] = acc;
    __syncthreads();
    // a thread has 8 columns of a row: lane (n, kq) of a result has columns 4 kq .. + 3 of row n
    const int half = threadIdx.x & 1, row = threadIdx.x >> 1, c = q0 + half * 8;
    if (row >= 16 || p0 + row >= a.np || c >= a.nq) return;
    f32x4 sum[2] = {}, bias[2] = {};
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int w = 0; w < kFewWaves; ++w) sum[h] += part[w][(half * 2 + h) * 16 + row];
    if (e.bias) widen8<T>(*(const uint4*)((const T*)e.bias + c), bias);
    finish8<T>(a, e, p0 + row, c, sum, bias, e.res ? *(const uint4*)((const T*)e.res + (p0 + row) * e.ldr + c) : make_uint4(0, 0, 0, 0));
}

constexpr int kDzThreads = 256;

struct DzArgs {
    const void* dy;
    const void* z;               // null: dz = dy
    void* dz;                    // null: only the sums
    int parts, halves;           // images of dz, 2 or 3, one after another; those of kHalves
    float* sums;                 // [row blocks][n], null: none wanted
    int64_t lddy, ldz;
    int n_rows, n, act;
    int rows;                    // of a block
};

// A thread has 8 columns of every eighth row of its block; the rows' sums meet in LDS.  1999 x 640 fp16 through silu 6.4-7.0 us
// (4.2-6.6 with one image): 10.2 MB, a load, an exponential and stores after one another.
//
// The images of kParts: a value's upper 16 bits, then those of what is left, the last one rounded; of kHalves: the rest of the rounding
// below, then that.  All have the value's sign, and none is zero (the smallest there is stands for nothing) unless the value is,
// or is below the type's range, 2^-23 of kHalves: an infinity that they meet in a product stays one.
__device__ __forceinline__ void dz_parts(float v, int parts, __bf16 (&p)[3]) {
    const bool fine = fabsf(v) < __builtin_inff();
    const uint32_t sign = __float_as_uint(v) & 1u << 31;
    const bool any = v != 0.f;
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        p[k] = fine && k + 1 < parts ? __builtin_bit_cast(__bf16, (uint16_t)(__float_as_uint(v) >> 16)) : (__bf16)v;
        if (fine) v -= (float)p[k];
        if (any && fabsf(v) < 0x1p-126f) v = __uint_as_float(sign | 1u << 23);
    }
}

__device__ __forceinline__ void dz_halves(float v, _Float16 (&p)[3]) {
    const float u = 0.5f * v;
    p[1] = (_Float16)__builtin_amdgcn_cvt_pkrtz(u, 0.f)[0];
    p[0] = fabsf(u) < __builtin_inff() ? (_Float16)((u - (float)p[1]) * (1.f / kSecondHalf)) : p[1];
    const uint16_t tiny = (uint16_t)((__float_as_uint(v) >> 16 & 0x8000u) | 1u);
    if (v != 0.f && p[0] == (_Float16)0.f) p[0] = __builtin_bit_cast(_Float16, tiny);
}

template <typename T, bool F32>
__global__ __launch_bounds__(kDzThreads) void k_linear_dz(DzArgs a) {
    __shared__ f32x4 part[8][32][2];
    const int t = threadIdx.x, u = t & 31, sub = t >> 5, c = (blockIdx.x * 32 + u) * 8;
    const int64_t r0 = (int64_t)blockIdx.y * a.rows, r1 = r0 + a.rows < a.n_rows ? r0 + a.rows : a.n_rows;
    f32x4 sum[2] = {};
    if (c < a.n) {
#pragma unroll 2
        for (int64_t r = r0 + sub; r < r1; r += 8) {
            f32x4 d[2];
            if constexpr (F32) {
                d[0] = *(const f32x4*)((const float*)a.dy + r * a.lddy + c);
                d[1] = *(const f32x4*)((const float*)a.dy + r * a.lddy + c + 4);
            } else {
                widen8<T>(*(const uint4*)((const T*)a.dy + r * a.lddy + c), d);
            }
            if (a.z) {
                f32x4 z[2];
                widen8<T>(*(const uint4*)((const T*)a.z + r * a.ldz + c), z);
                by_act(a.act, [&](auto act) {
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int e = 0; e < 4; ++e) d[h][e] *= slope<decltype(act)::value>(z[h][e]);
                });
            }
            if (a.dz) {
                auto images = [&](auto type, auto&& split) {
                    using I = decltype(type);
                    typedef I i8 __attribute__((ext_vector_type(8)));
                    i8 image[3];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        I p[3];
                        split(d[e / 4][e % 4], p);
#pragma unroll
                        for (int k = 0; k < 3; ++k) image[k][e] = p[k];
                    }
#pragma unroll
                    for (int k = 0; k < 3; ++k)
                        if (k < a.parts) *(i8*)((I*)a.dz + ((int64_t)k * a.n_rows + r) * a.n + c) = image[k];
                };
                if (__is_same(T, _Float16) && a.halves) images(_Float16(), [](float v, _Float16 (&p)[3]) { dz_halves(v, p); p[2] = p[0]; });
                else images(__bf16(), [&](float v, __bf16 (&p)[3]) { dz_parts(v, a.parts, p); });
            }
            sum[0] += d[0];
            sum[1] += d[1];
        }
    }
    if (!a.sums) return;
    part[sub][u][0] = sum[0];
    part[sub][u][1] = sum[1];
    __syncthreads();
    if (sub == 0 && c < a.n) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            f32x4 s = part[0][u][h];
            for (int i = 1; i < 8; ++i) s += part[i][u][h];
            *(f32x4*)(a.sums + (int64_t)blockIdx.y * a.n + c + h * 4) = s;
        }
    }
}

// The rows of a block of k_linear_dz: about 1024 blocks, at most 256 of them below each other (what the bias's sums wait for).
int dz_rows(int n_tok, int n) {
    const int64_t cols = ((int64_t)n + 255) / 256, down = std::max<int64_t>(1, std::min<int64_t>(256, 1024 / cols));
    return (int)std::max<int64_t>(8, (n_tok + down * 8 - 1) / (down * 8) * 8);
}
int dz_blocks(int n_tok, int n) { return (int)(((int64_t)n_tok + dz_rows(n_tok, n) - 1) / dz_rows(n_tok, n)); }

bool bad_matrix(const char* who, const char* name, const void* p, int64_t ld, int64_t width, int64_t rows) {
    if (ld % 8 || (rows > 1 && ld < width) || ld < 0) {
        moe_set_error("%s: %s: rows of %lld elements at a step of %lld (a multiple of 8 wanted)", who, name, (long long)width,
                      (long long)ld);
        return true;
    }
    if (rows > 0 && (!p || (uintptr_t)p % 16)) {
        moe_set_error("%s: %s: null or not 16-byte aligned", who, name);
        return true;
    }
    return false;
}

bool bad_sizes(const char* who, int n_tok, int n_in, int n_out, int act, int dtype) {
    if (n_tok < 0 || n_tok > kMaxSide || n_in < 8 || n_in % 8 || n_in > kMaxSide || n_out < 8 || n_out % 8 || n_out > kMaxSide ||
        act < kActNone || act > kActRelu2 || (dtype != 0 && dtype != 1)) {
        moe_set_error("%s: n_tok=%d n_in=%d n_out=%d (multiples of 8, up to 2^30) act=%d (0 none, 1 silu, 2 gelu, 3 squared relu) "
                      "dtype=%d (0 fp16, 1 bf16)", who, n_tok, n_in, n_out, act, dtype);
        return true;
    }
    return false;
}

bool too_many(const char* who, int64_t blocks, int threads) {
    if (blocks <= kMaxThreads / threads) return false;
    moe_set_error("%s: %lld tiles are more than one launch takes", who, (long long)blocks);
    return true;
}

uint64_t round_up(uint64_t v) { return (v + 255) / 256 * 256; }

// The tiles there are, with 0.01 us of a step where a CU has one of their blocks, and two (side by side those of four waves, one after the
// other those of eight), as measured, of dz as it came.  us per forward product in
// their order, chosen *: 1024 x 1024 x 1024 6.8* 7.0 8.4 9.2 10.5 12.3 15.4 20 26; 1030 x 72 x 1856 6.9 5.1* 7.5 6.1 6.2 8.1 8.5 10.5
// 13; 4096 x 2048 x 512 17.6 15.1 14.0* 15.1 16.9 20 25 35 42; 2048 x 2048 x 2048 35 29 26.7 23.8 20.5* 26.5 27.5 36 42; 3000 x 2048 x 2048
// 47 39 36 34 37 29 28.4* 36 42; 5000 x 4096 x 2056 158 131 131 110 95 101 101 75.6* 86; 4096 x 4096 x 4096 228 190 178 148 131 118 113 135
// 99.7*.  Both gradients, without 192 x 256: 333 x 640 x 2560 13.6* 12.7 15 15 19 24 28 47; 1999 x 2560 x 640 37 28 29 25 22.9* 26 28 42;
// 2048 x 2048 x 2048 65 53 53 44 40 34 33.2* 46; 4096 x 2048 x 512 44 33 33 30* 34 46 47 76; 8192 x 4096 x 4096 882 1050 734 716 563 480 455
// 393*.
template <bool FORWARD, typename F>
int each_tiles(const F& f) {
    f(Tiles<64, 64, 2, 2, 2, 3, 2, 8>(), 21, 40);
    f(Tiles<64, 64, 2, 2, 1, 4, 2, 8>(), 22, 37);
    f(Tiles<128, 64, 4, 2, 1, 4, 2, 8>(), 32, 63);
    f(Tiles<128, 64, 2, 2, 1, 3, 2, 8>(), 32, 54);
    f(Tiles<128, 128, 2, 4, 1, 4, 2, 6>(), 44, 89);
    f(Tiles<128, 128, 2, 2, 1, 2, 2, 8>(), 60, 85);
    f(Tiles<256, 128, 4, 2, 1, 3, 2, 6>(), 80, 163);
    if constexpr (FORWARD) f(Tiles<192, 256, 2, 4, 1, 2, 2, 4>(), 107, 213);   // (an image along the other index has a power of two)
    f(Tiles<256, 256, 2, 4, 1, 2, 2, 4>(), 138, 273);
    return 0;
}

// Calls run(tiles) with those that are done first: with one product, as many steps as a CU's blocks have; with two, whose blocks follow
// each other as CUs get free, the sum of all steps over the CUs, but at least those of the longest tile.
// split: fp16's values are taken apart on the way to the matrix unit, by every wave for its own columns: a step has WP BQ / 8 subtiles of
// them for a CU's four vector units, of 36 operations each.
template <bool FORWARD, typename R>
int best_tiles(const Product& a, const Product& b, bool split, const R& run) {
    int64_t best = INT64_MAX;
    int pick = 0, i = 0;
    auto steps = [](const Product& p) { return ((int64_t)(p.parts > 1 ? p.part_c : p.nc) / kBC + 1) * p.terms; };
    each_tiles<FORWARD>([&](auto tiles, int one, int two) {
        using C = decltype(tiles);
        if (split) one += C::WP * C::BQ / 5, two += C::WP * C::BQ / 5 * 2;
        const int64_t ta = tiles_in<C::BP, C::BQ>(a) * a.parts, tb = tiles_in<C::BP, C::BQ>(b) * b.parts;
        int64_t cost;
        if (ta == 0 || tb == 0) {
            const int64_t n = (ta + tb + 255) / 256;
            cost = (ta ? steps(a) : steps(b)) * (n / 2 * two + n % 2 * one);
        } else {
            cost = std::max((ta * steps(a) + tb * steps(b)) * two / 512, std::max(steps(a), steps(b)) * one);
        }
        if (cost < best) best = cost, pick = i;
        ++i;
    });
    int rc = -1;
    i = 0;
    each_tiles<FORWARD>([&](auto tiles, int, int) {
        if (i++ == pick) rc = run(tiles);
    });
    return rc;
}

// The length of a part, whole steps, and the parts of up to so many that have something then.
int part_of(int64_t nc, int64_t parts) { return (int)((nc + parts * kBC - 1) / (parts * kBC) * kBC); }
int parts_of(int64_t nc, int64_t parts) { return parts < 2 || nc < 1 ? 1 : (int)((nc - 1) / part_of(nc, parts) + 1); }

// Results few enough for k_linear_few.
bool few_results(int n_tok, int n_out) { return n_tok <= 16 || ((int64_t)n_tok + 15) / 16 * (((int64_t)n_out + 15) / 16) <= 256; }

// The parts of a forward product's contraction: as many as give every CU a tile of 64 x 64, of 8 steps or more, if a tile is rid of
// 30 steps that way, which pays for the second launch.  us with 1, 2, 4, 8 parts: 32 x 4096 x 4096 (64 steps) 14.2 12.7 10.5* 11.8, 256 x
// 4096 x 1024 15.1 12.8 10.8* 12.9, 128 x 4096 x 1024 13.4 12.0 10.1 10.1*, 100 x 2560 x 640 (40) 9.5 9.8 8.4 8.9 (5: 8.6*), 128 x 2048
// x 2048 (32) 8.6* 10.2 9.4 11.6.
int forward_parts(int n_tok, int n_in, int n_out) {
    if (n_tok < 1 || few_results(n_tok, n_out)) return 1;
    const int64_t tiles = ((int64_t)n_tok + 63) / 64 * (((int64_t)n_out + 63) / 64), steps = (int64_t)n_in / kBC;
    const int64_t parts = std::min(256 / tiles, steps / 8);
    return parts < 2 || steps * (parts - 1) < 30 * parts ? 1 : parts_of(n_in, parts);
}

template <typename T>
int forward(const Product& a, const Epilogue& e, void* workspace, hipStream_t s) {
    const int64_t tiles16 = tiles_in<16, 16>(a);
    if (few_results(a.np, a.nq)) {
        if (too_many("linear", tiles16, 64 * kFewWaves)) return -1;
        hipLaunchKernelGGL((k_linear_few<T>), dim3((uint32_t)tiles16), dim3(64 * kFewWaves), 0, s, a, e);
        HIP_TRY(hipGetLastError());
        return 0;
    }
    Product sums = a;
    if (a.parts > 1) sums.out = workspace, sums.ldo = a.nq;
    return best_tiles<true>(sums, Product{}, false, [&](auto tiles) {
        using C = decltype(tiles);
        const int64_t blocks = tiles_in<C::BP, C::BQ>(a) * a.parts, joins = ((int64_t)a.np * (a.nq / 8) + 255) / 256;
        if (too_many("linear", blocks, C::kThreads) || (a.parts > 1 && too_many("linear", joins, 256))) return -1;
        hipLaunchKernelGGL((k_linear<T, C>), dim3((uint32_t)blocks), dim3(C::kThreads), 0, s, sums, e);
        HIP_TRY(hipGetLastError());
        if (a.parts > 1) {
            hipLaunchKernelGGL((k_linear_join<T>), dim3((uint32_t)joins), dim3(256), 0, s, (const float*)workspace, a.parts, a, e);
            HIP_TRY(hipGetLastError());
        }
        return 0;
    });
}

// The parts of dW's contraction, the tokens: as many as give every CU a tile of 64 x 64, of 16 steps or more.  us of both gradients
// with 1, 2, 4, 8, 16 parts: 8192 x 512 x 256 28.9 21.5 15.4 14.4* 15.7, 8192 x 2048 x 64 45 48 28 25* 22, 4096 x 2048 x 128 26.6 19.4
// 16.0* 18 22, 4096 x 2048 x 512 32.2* 33.1 30.3 35 59.
int dw_parts(int n_tok, int n_out, int n_in) {
    const int64_t tiles = ((int64_t)n_out + 63) / 64 * (((int64_t)n_in + 63) / 64), steps = (int64_t)n_tok / kBC;
    return parts_of(n_tok, std::min(256 / tiles, steps / 16));
}

template <typename T, int MODE>
int gradients(const DzArgs* dz, int dy_f32, const Product& dw, int dw_f32, const Product& dx, const BiasSums& b, const Parts& p,
              hipStream_t s) {
    return best_tiles<false>(dw, dx, __is_same(T, _Float16) && MODE == kParts, [&](auto tiles) {
        using C = decltype(tiles);
        const bool parts = dw.parts > 1 && dw.np > 0;
        // what one launch does not take is refused before anything is queued
        const int64_t sums = b.db ? ((int64_t)b.n + 63) / 64 : 0, adds = parts ? (p.n / 8 + 255) / 256 : 0;
        const int64_t blocks = tiles_in<C::BP, C::BQ>(dw) * dw.parts + tiles_in<C::BP, C::BQ>(dx) + (parts ? 0 : sums);
        if (too_many("linear_grad", blocks, C::kThreads) || too_many("linear_grad", adds + sums, 256)) return -1;
        if (dz && dz->n_rows > 0) {
            const dim3 grid((dz->n + 255) / 256, dz_blocks(dz->n_rows, dz->n));
            if (dy_f32) hipLaunchKernelGGL((k_linear_dz<T, true>), grid, dim3(kDzThreads), 0, s, *dz);
            else hipLaunchKernelGGL((k_linear_dz<T, false>), grid, dim3(kDzThreads), 0, s, *dz);
            HIP_TRY(hipGetLastError());
        }
        if (blocks > 0) {
            hipLaunchKernelGGL((k_linear_grads<T, C, MODE>), dim3((uint32_t)blocks), dim3(C::kThreads), 0, s, dw, dx, b, parts || dw_f32);
            HIP_TRY(hipGetLastError());
        }
        if (parts) {
            hipLaunchKernelGGL((k_linear_parts<T>), dim3((uint32_t)(adds + sums)), dim3(256), 0, s, p, (uint32_t)adds, b);
            HIP_TRY(hipGetLastError());
        }
        return 0;
    });
}

// Images of dz for a dW of 16 bits or of fp32; dx, always of 16 bits, takes the first two.
constexpr int kDzParts = 2, kDzPartsF32 = 3;

// The workspace: dz (as a dW of fp32 takes it), the sums that the bias's gradient is made of, dW's parts.
struct Layout {
    uint64_t sums, parts, bytes;
};

Layout layout(int n_tok, int n_in, int n_out, bool own_dz, bool want_dw, bool want_db) {
    Layout l;
    l.sums = own_dz ? round_up(2 * (uint64_t)(want_dw ? kDzPartsF32 : kDzParts) * n_tok * n_out) : 0;
    l.parts = l.sums + (want_db ? round_up(4 * (uint64_t)dz_blocks(n_tok, n_out) * n_out) : 0);
    const int parts = want_dw ? dw_parts(n_tok, n_out, n_in) : 1;
    l.bytes = l.parts + (parts > 1 ? 4 * (uint64_t)parts * n_out * n_in : 0);
    return l;
}

}  // namespace

extern "C" uint64_t moe_linear_workspace_bytes(int n_tok, int n_in, int n_out) {
    if (n_tok < 1 || n_in < 1 || n_out < 1) return 0;
    const int parts = forward_parts(n_tok, n_in, n_out);
    return parts > 1 ? 4 * (uint64_t)parts * n_tok * n_out : 0;
}

extern "C" int moe_linear(const void* x, int64_t ldx, const void* w, const void* bias, const void* residual, int64_t ldr, int n_tok,
                          int n_in, int n_out, int act, int dtype, int out_f32, void* workspace, void* z, int64_t ldz, void* y,
                          int64_t ldy, void* stream) {
    const char* who = "linear";
    if (bad_sizes(who, n_tok, n_in, n_out, act, dtype) || bad_matrix(who, "x", x, ldx, n_in, n_tok) ||
        bad_matrix(who, "w", w, n_in, n_in, n_out) || (bias && bad_matrix(who, "bias", bias, n_out, n_out, 1)) ||
        (residual && bad_matrix(who, "residual", residual, ldr, n_out, n_tok)) ||
        (z && bad_matrix(who, "z", z, ldz, n_out, n_tok)) || bad_matrix(who, "y", y, ldy, n_out, n_tok))
        return -1;
    if (n_tok == 0) return 0;
    const int parts = forward_parts(n_tok, n_in, n_out);
    if (parts > 1 && (!workspace || (uintptr_t)workspace % 16)) {
        moe_set_error("linear: the workspace is null or not 16-byte aligned");
        return -1;
    }
    const Product a = {x, w, y, ldx, n_in, ldy, n_tok, n_out, n_in, parts, part_of(n_in, parts), 1, 0};
    const Epilogue e = {bias, residual, z, ldr, ldz, act, out_f32};
    const hipStream_t s = (hipStream_t)stream;
    return dtype ? forward<__bf16>(a, e, workspace, s) : forward<_Float16>(a, e, workspace, s);
}

extern "C" uint64_t moe_linear_grad_workspace_bytes(int n_tok, int n_in, int n_out, int act, int dy_f32, int want_dw, int want_db) {
    if (n_tok < 0 || n_in < 1 || n_out < 1) return 0;
    return layout(n_tok, n_in, n_out, act != kActNone || dy_f32, want_dw, want_db).bytes;
}

extern "C" int moe_linear_grad(const void* dy, int64_t lddy, int dy_f32, const void* x, int64_t ldx, const void* w, const void* z,
                               int64_t ldz, int n_tok, int n_in, int n_out, int act, int dtype, void* workspace, void* dx, void* dw,
                               int dw_f32, void* db, void* stream) {
    const char* who = "linear_grad";
    const hipStream_t s = (hipStream_t)stream;
    const bool own_dz = act != kActNone || dy_f32;
    if (bad_sizes(who, n_tok, n_in, n_out, act, dtype) || bad_matrix(who, "dy", dy, lddy, n_out, n_tok) ||
        (act != kActNone && bad_matrix(who, "z", z, ldz, n_out, n_tok)) || (dw && bad_matrix(who, "x", x, ldx, n_in, n_tok)) ||
        (dx && (bad_matrix(who, "w", w, n_in, n_in, n_out) || bad_matrix(who, "dx", dx, n_in, n_in, n_tok))) ||
        (dw && bad_matrix(who, "dw", dw, n_in, n_in, n_out)))
        return -1;
    const Layout at = layout(n_tok, n_in, n_out, own_dz, dw != nullptr, db != nullptr);
    if (at.bytes > 0 && (!workspace || (uintptr_t)workspace % 16)) {
        moe_set_error("linear_grad: the workspace is null or not 16-byte aligned");
        return -1;
    }
    void* dz = own_dz && (dx || dw) ? workspace : nullptr;
    const void* rows = own_dz ? dz : dy;
    const int64_t ld = own_dz ? n_out : lddy;
    float* sums = db ? (float*)((char*)workspace + at.sums) : nullptr;
    const int images = dw && dw_f32 ? kDzPartsF32 : kDzParts;
    const bool halves = dtype == 0 && !dy_f32 && (act == kActSilu || act == kActGelu) && images == kDzParts;
    const DzArgs d = {dy, act != kActNone ? z : nullptr, dz, images, halves, sums, lddy, ldz, n_tok, n_out, act, dz_rows(n_tok, n_out)};
    const int parts = dw ? dw_parts(n_tok, n_out, n_in) : 1;
    void* into = parts > 1 ? (char*)workspace + at.parts : dw;
    const Product gw = {rows, x, into, ld, ldx, n_in, dw ? n_out : 0, n_in, n_tok, parts, part_of(n_tok, parts),
                        own_dz ? images : 1, (int64_t)n_tok * n_out};
    const Product gx = {rows, w, dx, ld, n_in, n_in, dx ? n_tok : 0, n_in, n_out, 1, 0, own_dz ? kDzParts : 1,
                        (int64_t)n_tok * n_out};
    const BiasSums b = {sums, db, dz_blocks(n_tok, n_out), n_out};
    const Parts p = {(const float*)into, dw, (int64_t)n_out * n_in, parts, dw_f32};
    const DzArgs* need = dz || db ? &d : nullptr;
    if (dtype) return own_dz ? gradients<__bf16, kParts>(need, dy_f32, gw, dw_f32, gx, b, p, s)
                             : gradients<__bf16, kWhole>(need, dy_f32, gw, dw_f32, gx, b, p, s);
    if (!own_dz) return gradients<_Float16, kWhole>(need, dy_f32, gw, dw_f32, gx, b, p, s);
    return halves ? gradients<_Float16, kHalves>(need, dy_f32, gw, dw_f32, gx, b, p, s)
                  : gradients<_Float16, kParts>(need, dy_f32, gw, dw_f32, gx, b, p, s);
}
