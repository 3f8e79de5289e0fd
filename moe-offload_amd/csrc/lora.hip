// Low-rank adapters of many requests at once beside a shared projection.
//
// Token t belongs to a request with adapter i = ids[t]:   out[t] = base[t] + s_i B_i (A_i x[t]),
// A_i [rank][n_in], B_i [n_out][rank]; an id outside the adapters leaves out[t] = base[t].  base is the
// shared projection's output (a grouped product, the 2-bit experts' rows, a router's logits) and may be
// out itself.  v = A_i x is written and read in fp32 between the two products, and out is rounded once.
//
// Two launches.  k_lora_v multiplies 16 or 32 tokens by up to 32 ranks per block, the contraction dealt to its waves.
// k_lora_out multiplies v by B's rows and adds base; on the 16-bit matrix unit v is a sum of 16-bit parts: all of its bits
// for bf16, 22 of them for fp16 (split8).  Both take their operands through LDS in loads of whole lines.  The tokens of a
// tile may have different adapters: the tile is multiplied by each adapter that occurs in it and every token keeps its own
// adapter's result.  In a batch of prompts that is one adapter nearly always; for few tokens the adapters of a tile go to
// blocks of their own.
//
// The gradients: dv[t] = s_i B_i^T dy[t] beside v in one launch, then over the tokens sorted by adapter dx = A_i^T dv (a
// grouped product), and dA_i = sum dv x^T, dB_i = s_i sum dy v^T in one launch.  v and dv are three bf16 parts each there,
// which are all of their fp32 bits whatever their magnitude: two rounded parts would lose bits, and two fp16 parts also the
// values past 65504 and, step by step, those below 2^-14, where a gradient's are.
#include <hip/hip_bf16.h>

#include <algorithm>
#include <initializer_list>

#include "../../include/moe_offload.h"
#include "grouped_mm.h"

namespace {

using namespace gmm;

template <typename T>
__device__ __forceinline__ void widen8(uint4 w, float* v) {
    typedef T t8 __attribute__((ext_vector_type(8)));
    const t8 r = __builtin_bit_cast(t8, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)r[i];
}

// The adapters of a tile of 16 ST tokens, each once in the order of their first tokens: calls f(adapter, which of this
// lane's tokens have it) for the ones numbered first, first + step, ...  Wave-uniform.
template <int ST, typename F>
__device__ __forceinline__ void each_adapter(const int (&id)[ST], const bool (&has)[ST], int first, int step, F f) {
    uint32_t todo[ST];
    for (int m = 0; m < ST; ++m) todo[m] = (uint32_t)__ballot(has[m]) & 0xFFFFu;
    for (int j = 0;; ++j) {
        int i = -1;
#pragma unroll
        for (int m = ST - 1; m >= 0; --m)
            if (todo[m]) i = __builtin_amdgcn_readlane(id[m], __builtin_ctz(todo[m]));
        if (i < 0) return;
        bool mine[ST];
#pragma unroll
        for (int m = 0; m < ST; ++m) {
            mine[m] = has[m] && id[m] == i;
            todo[m] &= ~(uint32_t)__ballot(mine[m]);
        }
        if (j >= first && (j - first) % step == 0) f(i, mine);
    }
}

constexpr int kVWaves = 4;      // (8, one block per CU: lora_add of 64 tokens 8.9 us, with 4 8.7; lora_grad of 4096 64.7 and 62.5)
constexpr int kVRing = 2;

// v[t][j] = s_i W_i[j] x[t] for 16 ST tokens (blockIdx.x) and 16 SR ranks (blockIdx.y), where W_i[j] is row j of A_i, or
// (ALONG) column j of B_i [nc][rank].  Each wave multiplies every fourth step of 64 along the contraction, through an LDS
// ring of its own (two steps of the tokens' and the ranks' operands); the waves' sums are added in their order.  O: fp32, or
// bf16 where v is an operand of a product next: rows 3 t .. 3 t + 2 are the parts of v[t].  4096 tokens, rank 64, 2560: 13 us for
// 24 MB, a block per 32 tokens and 32 ranks, whose waves' few steps (10) are mostly the loads' way; v and dv for the
// gradients, 2560 and 2048, 20 us for 40 MB.
template <typename T, int SR, int ST, bool ALONG, typename O>
__device__ __forceinline__ void ranks_of(uint8_t* lds, int z, int n_z, const T* __restrict__ x, int64_t ldx,
                                         const T* __restrict__ W, int64_t w_stride, const int32_t* __restrict__ ids,
                                         const float* __restrict__ scale, int n_tok, int n_ad, int nc, int rank,
                                         O* __restrict__ v) {
    constexpr int kLoads = 2 * (ST + SR);
    constexpr uint32_t kStage = kLoads * 1024;
    static_assert(SR * ST <= kVWaves, "a wave per subtile of the sums");
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, kq = lane >> 4;
    const uint32_t ring = (uint32_t)(uintptr_t)(lds_u8*)lds + wv * kVRing * kStage;
    const int j0 = blockIdx.y * (16 * SR), cu = ((lane & 7) ^ (lane >> 3)) * 8;
    const T* zero = (const T*)&g_zero16;
    asm("" : "+s"(zero));
    int64_t t[ST];
    const T* xp[2 * ST];
    int id[ST];
    bool has[ST];
#pragma unroll
    for (int m = 0; m < ST; ++m) {
        t[m] = ((int64_t)blockIdx.x * ST + m) * 16 + n;
        id[m] = t[m] < n_tok ? ids[t[m]] : -1;
        has[m] = id[m] >= 0 && id[m] < n_ad;
    }
#pragma unroll
    for (int j = 0; j < 2 * ST; ++j) {
        const int64_t r = (int64_t)blockIdx.x * 16 * ST + j * 8 + (lane >> 3);
        xp[j] = x + (r < n_tok ? r : n_tok - 1) * ldx + cu;
    }
    Frags<false, 16, ST> fx;
    Frags<ALONG, 16 * SR, SR> fw;
    fx.init(ring, 0, lane);
    fw.init(ring + ST * 2048, 0, lane);
    const int steps = ((nc + 63) / 64 - wv + kVWaves - 1) / kVWaves;           // wv, wv + 4, ...
    each_adapter<ST>(id, has, z, n_z, [&](int i, const bool (&mine)[ST]) {
        const float si = scale ? scale[i] : 1.0f;
        const T* wp[2 * SR];
        int first_c[2 * SR];                                                   // of the lane's 16 bytes, in a step
#pragma unroll
        for (int j = 0; j < 2 * SR; ++j) {
            if constexpr (ALONG) {
                const int row = j * (32 / SR) + lane / (2 * SR), q = j0 + (lane % (2 * SR) ^ 2 * turn<16 * SR>(row)) * 8;
                first_c[j] = q < rank ? row : nc;                              // (ranks past the end: zeros)
                wp[j] = W + (int64_t)i * w_stride + (int64_t)row * rank + q;
            } else {
                const int r = j0 + j * 8 + (lane >> 3);
                first_c[j] = cu;
                wp[j] = W + (int64_t)i * w_stride + (int64_t)(r < rank ? r : rank - 1) * nc + cu;
            }
        }
        auto issue = [&](int s) {
            const int c = (s * kVWaves + wv) * 64;                             // (also past the last step)
            const uint32_t to = ring + (uint32_t)(s % kVRing) * kStage;
#pragma unroll
            for (int j = 0; j < 2 * ST; ++j) load_to_lds(c + cu < nc ? xp[j] + c : zero, to + j * 1024);
#pragma unroll
            for (int j = 0; j < 2 * SR; ++j)
                load_to_lds(c + first_c[j] < nc ? wp[j] + (ALONG ? (int64_t)c * rank : c) : zero, to + (2 * ST + j) * 1024);
        };
        f32x4 acc[SR][ST] = {};
#pragma unroll
        for (int s = 0; s < kVRing; ++s) issue(s);
#pragma unroll 1
        for (int s = 0; s < steps; ++s) {
            const uint32_t stage = (uint32_t)(s % kVRing) * kStage;
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"((kVRing - 1) * kLoads) : "memory");   // loads return in order
            uint4 xv[2][ST], wr[2][SR];
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
                for (int m = 0; m < ST; ++m) xv[ks][m] = fx.read(stage, m, ks);
#pragma unroll
                for (int r = 0; r < SR; ++r) wr[ks][r] = fw.read(stage, r, ks);
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                        // read before the next load overwrites it
            issue(s + kVRing);
#pragma unroll
            for (int ks = 0; ks < 2; ++ks)
#pragma unroll
                for (int r = 0; r < SR; ++r)
#pragma unroll
                    for (int m = 0; m < ST; ++m) acc[r][m] = mfma<T>(wr[ks][r], xv[ks][m], acc[r][m]);
        }
        // the sums trade places through the rings, which are idle once every wave's loads have landed
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        f32x4(*part)[SR * ST][64] = (f32x4(*)[SR * ST][64])lds;
#pragma unroll
        for (int r = 0; r < SR; ++r)
#pragma unroll
            for (int m = 0; m < ST; ++m) part[wv][r * ST + m][lane] = acc[r][m];
        __syncthreads();
        if (wv < SR * ST) {
            const int r = wv / ST, j = j0 + r * 16 + kq * 4;
            f32x4 sum = part[0][wv][lane];
#pragma unroll
            for (int w = 1; w < kVWaves; ++w) sum += part[w][wv][lane];
            sum *= si;
#pragma unroll
            for (int m = 0; m < ST; ++m)
                if (wv % ST == m && mine[m] && j < rank) {
                    if constexpr (sizeof(O) == 4) *(f32x4*)(v + t[m] * rank + j) = sum;
                    else {
                        typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
                        bf16x4 part[3];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            __bf16 p[3];
                            bf16_parts(sum[e], p);
#pragma unroll
                            for (int k = 0; k < 3; ++k) part[k][e] = p[k];
                        }
#pragma unroll
                        for (int k = 0; k < 3; ++k) *(bf16x4*)(v + (3 * t[m] + k) * rank + j) = part[k];
                    }
                }
        }
        __syncthreads();
    });
}

template <int SR, int ST>
constexpr uint32_t kRings = kVWaves * kVRing * 2 * (ST + SR) * 1024;

template <typename T, int SR, int ST>
__global__ __launch_bounds__(64 * kVWaves) void k_lora_v(const T* x, int64_t ldx, const T* A, int64_t a_stride, const int32_t* ids,
                                                         const float* scale, int n_tok, int n_ad, int n_in, int rank, float* v) {
    __shared__ __attribute__((aligned(1024))) uint8_t lds[kRings<SR, ST>];
    ranks_of<T, SR, ST, false, float>(lds, blockIdx.z, gridDim.z, x, ldx, A, a_stride, ids, scale, n_tok, n_ad, n_in, rank, v);
}

// The gradients' v = A_i x[t] and dv = s_i B_i^T dy[t], one in the even blocks of the third dimension, one in the odd.
template <typename T, int SR, int ST>
__global__ __launch_bounds__(64 * kVWaves) void k_lora_v_dv(const T* x, int64_t ldx, const T* A, int64_t a_stride, const T* dy,
                                                            int64_t lddy, const T* B, int64_t b_stride, const int32_t* ids,
                                                            const float* scale, int n_tok, int n_ad, int n_in, int n_out, int rank,
                                                            __bf16* v, __bf16* dv) {
    __shared__ __attribute__((aligned(1024))) uint8_t lds[kRings<SR, ST>];
    const int z = blockIdx.z >> 1, n_z = gridDim.z >> 1;
    if (blockIdx.z & 1)
        ranks_of<T, SR, ST, true, __bf16>(lds, z, n_z, dy, lddy, B, b_stride, ids, scale, n_tok, n_ad, n_out, rank, dv);
    else
        ranks_of<T, SR, ST, false, __bf16>(lds, z, n_z, x, ldx, A, a_stride, ids, nullptr, n_tok, n_ad, n_in, rank, v);
}

// Blocks of a tile's adapters: up to 256 tokens each gets its own (16 tokens have 16 at most).  One after another and side
// by side, us of lora_add, 2048 x 2048: 8 tokens of 8 adapters, rank 16, 34 and 9.6, 200 tokens, 4 to an adapter, 22 and
// 10.6; but 1000 tokens, 100 to an adapter, 2560 x 2560, rank 64, 20.8 and 32.9: most of the blocks find none left.
template <int ST>
uint32_t split_of(int n_tok) {
    return ST == 1 && n_tok <= 256 ? (uint32_t)(n_tok < 16 ? n_tok : 16) : 1;
}

template <typename T, int ST>
int lora_v_dv(const T* x, int64_t ldx, const T* A, int64_t a_stride, const T* dy, int64_t lddy, const T* B, int64_t b_stride,
              const int32_t* ids, const float* scale, int n_tok, int n_ad, int n_in, int n_out, int rank, __bf16* v,
              __bf16* dv, hipStream_t s) {
    const uint32_t tiles = (uint32_t)(((int64_t)n_tok + 16 * ST - 1) / (16 * ST)), split = 2 * split_of<ST>(n_tok);
    // (a tile of 32 ranks for 16: lora_add of 4096 tokens, rank 16, 28.1 us, and 26.8 with a tile of 16)
    if (rank <= 16)
        hipLaunchKernelGGL((k_lora_v_dv<T, 1, ST>), dim3(tiles, 1, split), dim3(64 * kVWaves), 0, s, x, ldx, A,
                           a_stride, dy, lddy, B, b_stride, ids, scale, n_tok, n_ad, n_in, n_out, rank, v, dv);
    else
        hipLaunchKernelGGL((k_lora_v_dv<T, 2, ST>), dim3(tiles, (rank + 31) / 32, split), dim3(64 * kVWaves), 0, s, x, ldx, A,
                           a_stride, dy, lddy, B, b_stride, ids, scale, n_tok, n_ad, n_in, n_out, rank, v, dv);
    HIP_TRY(hipGetLastError());
    return 0;
}

// Tokens of a tile: 32 use each load of an adapter twice, 16 are more blocks.  us of lora_add with 32 and 16, rank 64, 2560 x
// 2560: 4096 tokens 33 and 36 with inputs from memory, 34 and 29 with all in cache; 1000 tokens 24 and 21; lora_grad of
// 4096 tokens, 2560 x 2048, 62.5 and 64.1.
constexpr int kFewTokens = 1024;

template <typename T>
int lora_v_dv_typed(const void* x, int64_t ldx, const void* A, int64_t a_stride, const void* dy, int64_t lddy, const void* B,
                    int64_t b_stride, const int32_t* ids, const float* scale, int n_tok, int n_ad, int n_in, int n_out, int rank,
                    __bf16* v, __bf16* dv, hipStream_t s) {
    auto f = n_tok <= kFewTokens ? lora_v_dv<T, 1> : lora_v_dv<T, 2>;
    return f((const T*)x, ldx, (const T*)A, a_stride, (const T*)dy, lddy, (const T*)B, b_stride, ids, scale, n_tok, n_ad, n_in, n_out,
             rank, v, dv, s);
}

// fp32 values as sums of values of T.  bf16: three parts, which are the value itself.  fp16 values are first scaled by a
// power of two per token, so that the largest is just below 2^15, and two parts of 11 bits each are 22 bits, or 2^-40 of the
// token's largest value: what is lost is a tenth of a percent of half a step of out's type.  An infinity or NaN stays in the
// first part.
template <typename T>
constexpr int kParts = __is_same(T, _Float16) ? 2 : 3;

template <typename T>
__device__ __forceinline__ void split8(const float* v, uint4 (&part)[kParts<T>]) {
    typedef T t8 __attribute__((ext_vector_type(8)));
    t8 p[kParts<T>];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        if constexpr (kParts<T> == 3) {
            __bf16 q[3];
            bf16_parts(v[e], q);
#pragma unroll
            for (int k = 0; k < 3; ++k) p[k][e] = q[k];
        } else {
            p[0][e] = (T)v[e];
            p[1][e] = (T)(__builtin_fabsf(v[e]) < __builtin_inff() ? v[e] - (float)p[0][e] : 0.f);
        }
    }
#pragma unroll
    for (int k = 0; k < kParts<T>; ++k) part[k] = __builtin_bit_cast(uint4, p[k]);
}

// out = base + B_i v for 16 ST tokens (blockIdx.x) and 128 columns per wave.  The wave's eight subtiles of 16
// columns are dealt out so that lane n has the columns 8 n .. 8 n + 7, one of each: 16 bytes per token, and 16 lanes' are
// one row's 256.  B's rows and v go through LDS, 64 ranks at a time, in loads of whole lines: loaded straight into the
// matrix unit's layout every lane's 16 bytes are a cache access of their own, and those set the pace (4096 tokens, rank 64,
// 2560 columns: 42 us that way, 20 this way, 2.2 TB/s of base and out; waits 47% of the time).
template <typename T, int ST>
__global__ __launch_bounds__(256, 2) void k_lora_out(const T* base, int64_t ldb, const float* __restrict__ v,
                                                        const T* __restrict__ B, int64_t b_stride, const int32_t* __restrict__ ids,
                                                        int n_tok, int n_ad, int n_out, int rank, T* out, int64_t ldo) {
    constexpr int W = 4, SC = 8, kVLoads = ST;
    constexpr uint32_t kB = 128 * 128;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[W * kB + 4 * ST * 1024];
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, kq = lane >> 4;
    const uint32_t lds_b = (uint32_t)(uintptr_t)(lds_u8*)lds + wv * kB, lds_v = (uint32_t)(uintptr_t)(lds_u8*)lds + W * kB;
    const int first = ((int)blockIdx.y * W + wv) * 128, q = first + n * 8;
    const bool in_q = q < n_out;
    const T* zero = (const T*)&g_zero16;
    asm("" : "+s"(zero));
    const int64_t t0 = (int64_t)blockIdx.x * 16 * ST;
    int id[ST];
    bool has[ST];
#pragma unroll
    for (int m = 0; m < ST; ++m) {
        const int64_t t = t0 + m * 16 + n;
        id[m] = t < n_tok ? ids[t] : -1;
        has[m] = id[m] >= 0 && id[m] < n_ad;
    }
    // result lane (n, kq): columns q .. q + 7 of tokens 4 kq .. + 3
    uint4 bs[ST][4];
#pragma unroll
    for (int m = 0; m < ST; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t r = t0 + m * 16 + kq * 4 + i;
            bs[m][i] = *(const uint4*)(r < n_tok && in_q ? base + r * ldb + q : zero);
        }
    auto put = [&](uint32_t tokens, int m, int i, uint4 r) {
        if (tokens >> (kq * 4 + i) & 1 && in_q) *(uint4*)(out + (t0 + m * 16 + kq * 4 + i) * ldo + q) = r;
    };
    // tokens without an adapter are copied by the first of a tile's blocks
    if (base != out && blockIdx.z == 0)
#pragma unroll
        for (int m = 0; m < ST; ++m) {
            const uint32_t none = (uint32_t)__ballot(t0 + m * 16 + n < n_tok && !has[m]) & 0xFFFFu;
            if (none)
#pragma unroll
                for (int i = 0; i < 4; ++i) put(none, m, i, bs[m][i]);
        }
    each_adapter<ST>(id, has, blockIdx.z, gridDim.z, [&](int i, const bool (&mine)[ST]) {
        const T* Bi = B + (int64_t)i * b_stride;
        // columns past the end read the last ones', whose results are not stored (both ends are multiples of 8)
        auto load_chunk = [&](int k0) {
            int l = lane;
            asm volatile("" : "+v"(l));                                        // no addresses are kept over the products
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const int top = first + j * 8 < n_out ? first + j * 8 : n_out - 8, u = ((l & 7) ^ (j & 7)) * 8;
                const T* p = Bi + (int64_t)top * rank + k0 + ((l >> 3) * rank + u);
                load_to_lds(k0 + u < rank ? p : zero, lds_b + j * 1024);
            }
#pragma unroll
            for (int j = 0; j < kVLoads; ++j) {
                const int row = (wv * kVLoads + j) * 4 + (l >> 4), k = k0 + ((l & 15) ^ (row & 15)) * 4;
                const float* p = v + t0 * rank + (row * rank + k);
                load_to_lds(k < rank && row < 16 * ST && t0 + row < n_tok ? (const void*)p : zero, lds_v + (wv * kVLoads + j) * 1024);
            }
        };
        auto read_v = [&](int m, int ks, float* w) {
            typedef __attribute__((address_space(3))) const f32x4* ptr;
            const uint32_t at = lds_v + (m * 16 + n) * 256;
            const f32x4 lo = *(ptr)(uintptr_t)(at + ((8 * ks + 2 * kq) ^ n) * 16), hi = *(ptr)(uintptr_t)(at + ((8 * ks + 2 * kq + 1) ^ n) * 16);
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = lo[e], w[4 + e] = hi[e];
        };
        auto landed = [&]() {
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
        };
        load_chunk(0);
        // fp16: the power of two of this lane's token in each tile, from its largest |v|
        float up[ST], down[ST];
#pragma unroll
        for (int m = 0; m < ST; ++m) up[m] = down[m] = 1.f;
        if constexpr (kParts<T> == 2) {
            float most[ST] = {};
            for (int k0 = 64; k0 < rank; k0 += 64)                             // what the first 64 ranks leave
                for (int m = 0; m < ST; ++m)
                    for (int k = k0 + kq * 8; k < k0 + 64 && k < rank; k += 32)
                        for (int e = 0; e < 8; ++e)
                            most[m] = fmaxf(most[m], mine[m] ? __builtin_fabsf(v[(t0 + m * 16 + n) * rank + k + e]) : 0.f);
            landed();
#pragma unroll
            for (int m = 0; m < ST; ++m) {
#pragma unroll
                for (int ks = 0; ks < 2; ++ks) {
                    float w[8];
                    read_v(m, ks, w);
#pragma unroll
                    for (int e = 0; e < 8; ++e) most[m] = fmaxf(most[m], __builtin_fabsf(w[e]));
                }
                most[m] = fmaxf(most[m], __shfl_xor(most[m], 16, 64));
                most[m] = fmaxf(most[m], __shfl_xor(most[m], 32, 64));
                if (most[m] > 0.f && most[m] < __builtin_inff()) {
                    // 2^100 or 2^-113 at most: what is smaller yet than 2^-85 is 0 in the result's type
                    int e = 15 - __builtin_amdgcn_frexp_expf(most[m]);
                    e = e > 100 ? 100 : e < -113 ? -113 : e;
                    up[m] = ldexpf(1.f, e);
                    down[m] = ldexpf(1.f, -e);
                }
            }
        } else {
            landed();
        }
        f32x4 acc[ST][SC] = {};
#pragma unroll 1
        for (int k0 = 0;; k0 += 64) {
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                if (k0 + ks * 32 >= rank) break;
                uint4 part[ST][kParts<T>];
#pragma unroll
                for (int m = 0; m < ST; ++m) {
                    float w[8];
                    read_v(m, ks, w);
#pragma unroll
                    for (int e = 0; e < 8; ++e) w[e] *= up[m];
                    split8<T>(w, part[m]);
                }
#pragma unroll
                for (int s = 0; s < SC; ++s) {
                    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
                    typedef __attribute__((address_space(3))) const u32x4* ptr;
                    const u32x4 r = *(ptr)(uintptr_t)(lds_b + (8 * n + s) * 128 + ((4 * ks + kq) ^ (n & 7)) * 16);
                    const uint4 b = make_uint4(r[0], r[1], r[2], r[3]);
#pragma unroll
                    for (int m = 0; m < ST; ++m)
#pragma unroll
                        for (int k = 0; k < kParts<T>; ++k) acc[m][s] = mfma<T>(part[m][k], b, acc[m][s]);
                }
            }
            // everyone has read this chunk (and, after the last, the next adapter's may overwrite it)
            landed();
            if (k0 + 64 >= rank) break;
            load_chunk(k0 + 64);
            landed();
        }
#pragma unroll
        for (int m = 0; m < ST; ++m) {
            const uint32_t tokens = (uint32_t)__ballot(mine[m]) & 0xFFFFu;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                typedef T t8 __attribute__((ext_vector_type(8)));
                float w[8];
                t8 r;
                widen8<T>(bs[m][e], w);
                const float back = __shfl(down[m], kq * 4 + e, 64);
#pragma unroll
                for (int s = 0; s < SC; ++s) r[s] = (T)fmaf(acc[m][s][e], back, w[s]);
                put(tokens, m, e, __builtin_bit_cast(uint4, r));
            }
        }
    });
}

// da_i = sum over adapter i's tokens of dv x^T, or (DA false) db_i = s_i sum of dy v^T; order[r] is the r-th token in the
// order of the adapters, `parts` holds dv or v.
struct DwArgs {
    const void* wide;                 // x or dy
    int64_t ld;
    const __bf16* parts;
    int n_wide;
    int span;                         // tiles per block, side by side along the wide operand
    const float* scale;
    void* out;
};

// A block computes `span` tiles of 64 x 64 results of one adapter.  A step of 64 tokens is one image of the wide operand and
// one of each part, straight from memory to LDS while the step before it is multiplied (the next tile's first during the
// last of this one): a wide row is loaded once and multiplied by all three parts.  Four waves, 32 x 32 results each, multiply
// the step's first 32 tokens and four its others, and their sums are added at the end: the longest segment's steps one after
// another are what bounds it (4096 tokens of 8 adapters, rank 64, 2560 and 2048 wide: 21 us in bf16, 32 in fp16, whose two
// parts are made in registers; four waves and steps of 32 tokens 25 and 38; without the loads or without the products hardly
// less).
constexpr int kDwTile = 64, kDwWaves = 8, kDwStep = 8 * kDwWaves, kDwHeld = 1024;     // kDwHeld: tokens whose numbers are in LDS
constexpr uint32_t kDwImage = kDwStep * kDwTile * 2, kDwStage = 4 * kDwImage;

template <typename T, bool DA>
__device__ __forceinline__ void dw_tiles(uint8_t* lds, const DwArgs& a, const int32_t* __restrict__ order,
                                         const int32_t* __restrict__ seg_start, int n_tok, int n_ad, int rank, uint32_t block,
                                         uint32_t blocks) {
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, kq = lane >> 4;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_u8*)lds;
    const int tiles = (a.n_wide + kDwTile - 1) / kDwTile, groups = (tiles + a.span - 1) / a.span, rt = (rank + kDwTile - 1) / kDwTile;
    const uint32_t run = ((uint32_t)groups * rt + 7) / 8;
    const uint32_t item = n_ad < kManySegs ? dealt(block, blocks, run) : xcd_order(block, blocks);
    const int seg = item / (groups * rt), j0 = (int)(item / groups % rt) * kDwTile, tile0 = (int)(item % groups) * a.span;
    const int end = tile0 + a.span < tiles ? tile0 + a.span : tiles;
    const Segs S{seg_start, nullptr, n_ad, n_tok, n_ad, 0};
    int r0, r1, slot;
    seg_rows(S, seg + 1, r0, r1, slot);
    const int steps = (r1 - r0 + kDwStep - 1) / kDwStep;

    // A wave loads 8 tokens of each image, a lane 16 bytes of its token's row; tokens past the end read zeros.
    const int row = wv * 8 + (lane >> 3), col = ((lane & 7) ^ 2 * turn<kDwTile>(row)) * 8;
    const T* zero = (const T*)&g_zero16;
    asm("" : "+s"(zero));
    const int64_t part_col = j0 + col < rank ? j0 + col : 0;                   // (columns past the end are not stored)
    int* held = (int*)(lds + 2 * kDwStage);
    auto load = [&](int t, int tile, uint32_t stage) {
        const int c = tile * kDwTile + col;
        const uint32_t to = lds0 + stage + wv * 1024;
        load_to_lds(t >= 0 ? (const T*)a.wide + t * a.ld + (c < a.n_wide ? c : 0) : zero, to);
        const __bf16* p = a.parts + (int64_t)t * 3 * rank + part_col;
#pragma unroll
        for (int k = 0; k < 3; ++k) load_to_lds(t >= 0 ? (const void*)(p + k * rank) : zero, to + (k + 1) * kDwImage);
    };
    const int w0 = (wv & 1) * 32, p0 = (wv >> 1 & 1) * 32, half = wv >> 2;     // this wave's results in the tile, and tokens
    Frags<true, kDwTile, 2> fw, fp;
    fw.init(lds0, w0, lane);
    fp.init(lds0 + kDwImage, p0, lane);
    const float s = a.scale && steps > 0 ? a.scale[seg] : 1.0f;               // (no tokens: zeros, whatever the scale)
    const int np = DA ? rank : a.n_wide, nq = DA ? a.n_wide : rank;
    int next = 0, next_tile = tile0, chunk = -1;                               // the step that is loaded next; tokens held
    uint32_t stage = 0;
    auto advance = [&]() {
        const int c = next * kDwStep;
        if (c / kDwHeld != chunk) {
            chunk = c / kDwHeld;
            __syncthreads();                                                   // everyone has read the numbers held so far
            for (int i = threadIdx.x; i < kDwHeld; i += 64 * kDwWaves) held[i] = r0 + c + i < r1 ? order[r0 + c + i] : -1;
            __syncthreads();
        }
        load(held[c % kDwHeld + row], next_tile, stage);
        if (++next == steps) next = 0, ++next_tile;
    };
    if (steps > 0) advance();
#pragma unroll 1
    for (int tile = tile0; tile < end; ++tile) {
        f32x4 acc[2][2] = {};                                                  // [rows of out][along them]
#pragma unroll 1
        for (int step = 0; step < steps; ++step) {
            // this wave's loads of the step have landed and its reads of the step before are done; past the barrier, so are
            // everyone's
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            const uint32_t at = stage;
            stage = kDwStage - stage;
            if (next_tile < end) advance();
            uint4 w[2], p[3][2];
#pragma unroll
            for (int i = 0; i < 2; ++i) w[i] = fw.read(at, i, half);
#pragma unroll
            for (int k = 0; k < 3; ++k)
#pragma unroll
                for (int i = 0; i < 2; ++i) p[k][i] = fp.read(at + k * kDwImage, i, half);
#pragma unroll
            for (int k = 0; k < 3; ++k)
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        if constexpr (DA) acc[i][j] = mfma_parts<T>(w[j], p[k][i], acc[i][j]);
                        else acc[i][j] = mfma_parts<T, false>(w[i], p[k][j], acc[i][j]);
                    }
        }
        if (r1 - r0 > kDwStep / 2) {
            // through the image just multiplied
            typedef __attribute__((address_space(3))) f32x4* ptr;
            const uint32_t mine = lds0 + (kDwStage - stage) + ((wv & 3) * 256 + lane) * 16;
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();                                      // everyone has read it
            asm volatile("" ::: "memory");
            if (half) {
#pragma unroll
                for (int i = 0; i < 4; ++i) *(ptr)(uintptr_t)(mine + i * 1024) = acc[i >> 1][i & 1];
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            if (!half) {
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[i >> 1][i & 1] += *(ptr)(uintptr_t)(mine + i * 1024);
            }
        }
        if (half) continue;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = (DA ? j0 + p0 : tile * kDwTile + w0) + i * 16 + n;
            const int c = (DA ? tile * kDwTile + w0 : j0 + p0) + (kq & 1) * 16 + (kq >> 1) * 8;
            const uint4 v = pair8(round4<T>(acc[i][0] * s), round4<T>(acc[i][1] * s));
            if (r < np && c < nq) store16((T*)a.out + ((int64_t)seg * np + r) * nq + c, v);
        }
    }
}

// Both in one launch, the first n_a blocks da's.
template <typename T>
__global__ __launch_bounds__(64 * kDwWaves, 4) void k_lora_dw(DwArgs a, DwArgs b, const int32_t* order, const int32_t* seg_start, int n_tok,
                                                    int n_ad, int rank, uint32_t n_a) {
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * kDwStage + kDwHeld * 4];
    if (blockIdx.x < n_a) dw_tiles<T, true>(lds, a, order, seg_start, n_tok, n_ad, rank, blockIdx.x, n_a);
    else dw_tiles<T, false>(lds, b, order, seg_start, n_tok, n_ad, rank, blockIdx.x - n_a, gridDim.x - n_a);
}

// Sets the tiles per block and returns the blocks.  Tiles of short segments share a block's start while that leaves 1024
// blocks.  us of the gradients of 4096 tokens at 1, 2, 4, 8 and 16 tiles: 512 adapters, rank 16, 2048 x 2048 (one step) 413,
// -, 344, 332, 325; 64 adapters, rank 128, 2560 x 2560 (two steps expected) 143, 137, 147, 153, -.
int64_t dw_blocks(DwArgs& a, int n_tok, int n_ad, int rank) {
    const int64_t tiles = (a.n_wide + kDwTile - 1) / kDwTile, rows = (int64_t)n_ad * ((rank + kDwTile - 1) / kDwTile);
    const int64_t steps = (int64_t)n_tok / n_ad / kDwStep + 1;
    a.span = (int)std::max<int64_t>(1, std::min<int64_t>({steps == 1 ? 16 : 4 / steps, rows * tiles / 1024, tiles}));
    return rows * ((tiles + a.span - 1) / a.span);
}

template <typename T>
int lora_dw(DwArgs a, DwArgs b, const int32_t* order, const int32_t* seg_start, int n_tok, int n_ad, int rank, bool dry, hipStream_t s) {
    const int64_t n_a = dw_blocks(a, n_tok, n_ad, rank), n_b = dw_blocks(b, n_tok, n_ad, rank);
    if (n_a + n_b > kMaxThreads / (64 * kDwWaves)) {
        moe_set_error("lora_grad: %lld tiles are more than one launch takes", (long long)(n_a + n_b));
        return -1;
    }
    if (dry) return 0;
    hipLaunchKernelGGL((k_lora_dw<T>), dim3((uint32_t)(n_a + n_b)), dim3(64 * kDwWaves), 0, s, a, b, order, seg_start, n_tok, n_ad, rank,
                       (uint32_t)n_a);
    HIP_TRY(hipGetLastError());
    return 0;
}

template <typename T, int ST>
int lora_add(const T* base, int64_t ldb, const T* x, int64_t ldx, const T* A, int64_t a_stride, const T* B, int64_t b_stride,
             const int32_t* ids, const float* scale, int n_tok, int n_ad, int n_in, int n_out, int rank, float* v, T* out,
             int64_t ldo, hipStream_t s) {
    const uint32_t tiles = (uint32_t)(((int64_t)n_tok + 16 * ST - 1) / (16 * ST));
    const uint32_t split = split_of<ST>(n_tok);
    if (n_ad > 0) {
        if (rank <= 16)
            hipLaunchKernelGGL((k_lora_v<T, 1, ST>), dim3(tiles, 1, split), dim3(64 * kVWaves), 0, s, x, ldx, A,
                               a_stride, ids, scale, n_tok, n_ad, n_in, rank, v);
        else
            hipLaunchKernelGGL((k_lora_v<T, 2, ST>), dim3(tiles, (rank + 31) / 32, split), dim3(64 * kVWaves), 0, s, x, ldx, A,
                               a_stride, ids, scale, n_tok, n_ad, n_in, rank, v);
        HIP_TRY(hipGetLastError());
    }
    hipLaunchKernelGGL((k_lora_out<T, ST>), dim3(tiles, (n_out + 511) / 512, split), dim3(256), 0, s, base, ldb, v, B, b_stride, ids,
                       n_tok, n_ad, n_out, rank, out, ldo);
    HIP_TRY(hipGetLastError());
    return 0;
}

template <typename T>
int lora_add_typed(const void* base, int64_t ldb, const void* x, int64_t ldx, const void* A, int64_t a_stride, const void* B,
                   int64_t b_stride, const int32_t* ids, const float* scale, int n_tok, int n_ad, int n_in, int n_out, int rank,
                   float* v, void* out, int64_t ldo, hipStream_t s) {
    auto f = n_tok <= kFewTokens ? lora_add<T, 1> : lora_add<T, 2>;
    return f((const T*)base, ldb, (const T*)x, ldx, (const T*)A, a_stride, (const T*)B, b_stride, ids, scale, n_tok, n_ad, n_in,
             n_out, rank, v, (T*)out, ldo, s);
}

constexpr int kMaxOut = (1 << 23) - 8;                        // the second grid dimension, 512 columns each, and its loads
constexpr int kMaxTok = (int)(kMaxThreads / 256) * 32;        // blocks of 256 threads for 32 tokens each

// The shapes and strides that both entry points take; base or dy is [n_tok][n_out].
bool bad_shapes(const char* who, int dtype, int n_tok, int n_ad, int n_in, int n_out, int rank, int64_t ldx, int64_t ldy,
                int64_t a_stride, int64_t b_stride) {
    if ((dtype != 0 && dtype != 1) || n_tok < 0 || n_ad < 0 || n_in <= 0 || n_out <= 0 || rank <= 0 || n_in % 8 ||
        n_out % 8 || rank % 8 || rank > 256 || n_out > kMaxOut || n_in > kMaxSide || n_tok > kMaxTok) {
        moe_set_error("%s: dtype=%d n_tok=%d n_ad=%d n_in=%d n_out=%d rank=%d (multiples of 8, rank <= 256, n_out < 2^23, n_in <= "
                      "2^30, n_tok <= %d)",
                      who, dtype, n_tok, n_ad, n_in, n_out, rank, kMaxTok);
        return true;
    }
    if (ldx % 8 || ldy % 8 || a_stride % 8 || b_stride % 8 || (n_tok > 1 && (ldx < n_in || ldy < n_out)) ||
        (n_ad > 1 && (a_stride < (int64_t)rank * n_in || b_stride < (int64_t)rank * n_out))) {
        moe_set_error("%s: strides must be multiples of 8 and not less than a row or matrix", who);
        return true;
    }
    return false;
}

bool bad_pointers(const char* who, std::initializer_list<const void*> ps) {
    for (const void* p : ps)
        if (!p || (uintptr_t)p % 16) {
            moe_set_error("%s: a pointer is null or not 16-byte aligned", who);
            return true;
        }
    return false;
}

uint64_t up16(uint64_t v) { return (v + 15) / 16 * 16; }

}  // namespace

extern "C" uint64_t moe_lora_workspace_bytes(int n_tok, int rank) {
    return n_tok > 0 && rank > 0 ? (uint64_t)n_tok * rank * 4 : 0;
}

extern "C" int moe_lora_add(const void* base, int64_t ld_base, const void* x, int64_t ldx, const void* a, int64_t a_stride,
                            const void* b, int64_t b_stride, const int32_t* ids, const float* scale, int n_tok, int n_ad,
                            int n_in, int n_out, int rank, int dtype, void* workspace, void* out, int64_t ld_out,
                            void* stream) {
    const char* who = "lora_add";
    if (bad_shapes(who, dtype, n_tok, n_ad, n_in, n_out, rank, ldx, ld_base, a_stride, b_stride)) return -1;
    if (ld_out % 8 || (n_tok > 1 && (ld_out < n_out || (out == base && ld_out != ld_base)))) {
        moe_set_error("%s: ld_out=%lld (ld_base=%lld)", who, (long long)ld_out, (long long)ld_base);
        return -1;
    }
    if (n_tok == 0) return 0;
    if (!ids) {
        moe_set_error("%s: ids is null", who);
        return -1;
    }
    if (bad_pointers(who, {base, x, out, workspace}) || (n_ad > 0 && bad_pointers(who, {a, b}))) return -1;
    auto f = dtype ? lora_add_typed<__bf16> : lora_add_typed<_Float16>;
    return f(base, ld_base, x, ldx, a, a_stride, b, b_stride, ids, scale, n_tok, n_ad, n_in, n_out, rank, (float*)workspace,
             out, ld_out, (hipStream_t)stream);
}

extern "C" uint64_t moe_lora_grad_workspace_bytes(int n_tok, int n_ad, int rank) {
    if (n_tok < 0 || n_ad < 1 || rank <= 0) return 0;
    return 2 * up16((uint64_t)n_tok * rank * 6) + 2 * up16((uint64_t)n_tok * 4) + up16((uint64_t)(n_ad + 1) * 4) +
           moe_expert_plan_workspace_bytes(n_tok, n_ad);
}

extern "C" int moe_lora_grad(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* a, int64_t a_stride,
                             const void* b, int64_t b_stride, const int32_t* ids, const float* scale, int n_tok, int n_ad,
                             int n_in, int n_out, int rank, int dtype, void* workspace, void* dx, int64_t lddx, void* da,
                             void* db, void* stream) {
    const char* who = "lora_grad";
    if (bad_shapes(who, dtype, n_tok, n_ad, n_in, n_out, rank, ldx, lddy, a_stride, b_stride)) return -1;
    if (n_ad < 1 || n_ad > gmm::kMaxSeg || lddx % 8 || (n_tok > 1 && lddx < n_in)) {
        moe_set_error("%s: n_ad=%d (1..%d) lddx=%lld", who, n_ad, gmm::kMaxSeg, (long long)lddx);
        return -1;
    }
    if (n_tok > 0 && !ids) {
        moe_set_error("%s: ids is null", who);
        return -1;
    }
    if (bad_pointers(who, {a, b, da, db, workspace}) || (n_tok > 0 && bad_pointers(who, {dy, x, dx}))) return -1;
    uint8_t* p = (uint8_t*)workspace;
    auto take = [&](uint64_t bytes) {
        uint8_t* q = p;
        p += up16(bytes);
        return q;
    };
    __bf16* v = (__bf16*)take((uint64_t)n_tok * rank * 6);
    __bf16* dv = (__bf16*)take((uint64_t)n_tok * rank * 6);
    int32_t* order = (int32_t*)take((uint64_t)n_tok * 4);
    int32_t* same = (int32_t*)take((uint64_t)n_tok * 4);
    int32_t* seg = (int32_t*)take((uint64_t)(n_ad + 1) * 4);
    auto v_dv = dtype ? lora_v_dv_typed<__bf16> : lora_v_dv_typed<_Float16>;
    auto dw = dtype ? lora_dw<__bf16> : lora_dw<_Float16>;
    const auto dx_dw = [&](bool dry) {
        return (n_tok > 0 && gmm::dx_of_parts(dv, order, n_tok, seg, n_ad, a, a_stride, rank, n_in, dx, lddx, dtype, dry,
                                              (hipStream_t)stream)) ||
               dw(DwArgs{x, ldx, dv, n_in, 1, nullptr, da}, DwArgs{dy, lddy, v, n_out, 1, scale, db}, order, seg, n_tok, n_ad, rank,
                  dry, (hipStream_t)stream);
    };
    // the tokens sorted by adapter: a token's row number everywhere but in seg is its own.  Without tokens da and db are the
    // products over empty segments.
    if (dx_dw(true) || moe_expert_plan(ids, n_tok, 1, n_ad, p, same, order, seg, stream) ||
        (n_tok > 0 && v_dv(x, ldx, a, a_stride, dy, lddy, b, b_stride, ids, scale, n_tok, n_ad, n_in, n_out, rank, v, dv,
                           (hipStream_t)stream)) ||
        dx_dw(false))
        return -1;
    return 0;
}
