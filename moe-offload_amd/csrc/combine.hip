// The weighted sum of each token's per-expert rows, and its gradients:
//     out[t] = residual[t] + sum over j of w[t][j] y[t k + j]         (the residual may be absent)
//     dy[t k + j] = w[t][j] dout[t],     dw[t][j] = <dout[t], y[t k + j]>
// y, residual, dout and dy fp16 or bf16, out too or fp32, w and dw fp32; sums in fp32, in the order of j, one rounding at
// the end.  A place of weight 0 adds nothing whatever its row holds, and so do its gradients: dy is 0, and dw, which a
// weight that happens to be 0 has too, is 0 where it would not be finite.  moe_pair_combine (mlx-qwen38/loader.py:964-965) is
// the sum of fp16 rows by fp16 scores, of inference.
#include <hip/hip_fp16.h>

#include "lane_reduce.h"
#include "moe_common.h"

namespace {

constexpr int kCombineThreads = 256;
constexpr int64_t kCombineBlocks = 1 << 22;    // more work than they hold: a block takes several items

typedef float f32x8 __attribute__((ext_vector_type(8)));

template <typename T>
__device__ __forceinline__ f32x8 widen8(uint4 v) {
    typedef T t8 __attribute__((ext_vector_type(8)));
    return __builtin_convertvector(__builtin_bit_cast(t8, v), f32x8);
}

template <typename T>
__device__ __forceinline__ uint4 round8(f32x8 v) {
    typedef T t8 __attribute__((ext_vector_type(8)));
    return __builtin_bit_cast(uint4, __builtin_convertvector(v, t8));
}

struct CombineArgs {
    const void* y;
    const float* weights;
    const void* residual;
    void* out;
    int64_t ldy, ldr, ldo;
    int n_tok, k, hidden;
};

// A thread has 8 columns of a token, and kAtOnce of its rows under way at once: memory bounds it, 4096 tokens of 10 x 2560 fp16 38
// us (6.6 TB/s), 512 tokens 4.3 (7.3, out of the last-level cache; 7.8 with one row at a time).
template <typename T, bool F32>
__global__ __launch_bounds__(kCombineThreads) void k_combine(CombineArgs a) {
    constexpr int kAtOnce = 5;
    const uint32_t units = a.hidden / 8;
    const int64_t items = (int64_t)a.n_tok * units;
    for (int64_t i = (int64_t)blockIdx.x * kCombineThreads + threadIdx.x; i < items; i += (int64_t)gridDim.x * kCombineThreads) {
        // (a division of 64 bits is a loop of its own)
        const int64_t t = items <= 0xFFFFFFFF ? (uint32_t)i / units : i / units;
        const int c = (int)(i - t * units) * 8;
        const T* y = (const T*)a.y + t * a.k * a.ldy + c;
        const float* w = a.weights + t * a.k;
        uint4 res = make_uint4(0, 0, 0, 0);
        if (a.residual) res = *(const uint4*)((const T*)a.residual + t * a.ldr + c);
        f32x8 sum = {};
        for (int j0 = 0; j0 < a.k; j0 += kAtOnce) {
            uint4 v[kAtOnce];
            float wj[kAtOnce];
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j) {
                const bool in = j0 + j < a.k;
                v[j] = *(const uint4*)(y + (in ? j0 + j : 0) * a.ldy);
                wj[j] = in ? w[j0 + j] : 0.f;
            }
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j)
                if (wj[j] != 0.f) sum += wj[j] * widen8<T>(v[j]);
        }
        sum += widen8<T>(res);
        if constexpr (F32) *(f32x8*)((float*)a.out + t * a.ldo + c) = sum;
        else *(uint4*)((T*)a.out + t * a.ldo + c) = round8<T>(sum);
    }
}

struct CombineGradArgs {
    const void* dout;
    const void* y;
    const float* weights;
    void* dy;
    float* dweights;
    int64_t ldd, ldy, lddy;
    int n_tok, k, hidden;
};

// A wave has a (token, place), and finds dout again in L2 for the token's other places.  dy goes past the caches: 8192 tokens of
// 4 x 4096 bf16 104 us (5.8 TB/s), 110 through them; 4096 of 10 x 2560 72 and 83.
template <typename T>
__global__ __launch_bounds__(kCombineThreads) void k_combine_grad(CombineGradArgs a) {
    const int lane = threadIdx.x & 63, units = a.hidden / 8;
    const int64_t pairs = (int64_t)a.n_tok * a.k, step = (int64_t)gridDim.x * (kCombineThreads / 64);
    for (int64_t p = (int64_t)blockIdx.x * (kCombineThreads / 64) + (threadIdx.x >> 6); p < pairs; p += step) {
        const T* d = (const T*)a.dout + p / a.k * a.ldd;
        const float w = a.weights[p];
        const bool none = w == 0.f;
        float dot = 0.f;
#pragma unroll 2
        for (int u = lane; u < units; u += 64) {
            const f32x8 dv = widen8<T>(*(const uint4*)(d + u * 8));
            const f32x8 v = widen8<T>(*(const uint4*)((const T*)a.y + p * a.ldy + u * 8));
            typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
            __builtin_nontemporal_store(__builtin_bit_cast(u32x4, round8<T>(none ? (f32x8)(0.f) : w * dv)), (u32x4*)((T*)a.dy + p * a.lddy + u * 8));
#pragma unroll
            for (int e = 0; e < 8; ++e) dot += dv[e] * v[e];
        }
        dot = lanes::group_sum<64>(dot);
        if (none && !(fabsf(dot) < __builtin_inff())) dot = 0.f;
        if (lane == 0) a.dweights[p] = dot;
    }
}

bool bad_rows(const char* who, const char* name, const void* p, int64_t ld, int hidden, int64_t rows) {
    if (ld % 8 || (rows > 1 && ld < hidden) || ld < 0) {
        moe_set_error("%s: %s: rows of %d elements at a step of %lld (a multiple of 8 wanted)", who, name, hidden, (long long)ld);
        return true;
    }
    if (rows > 0 && (!p || (uintptr_t)p % 16)) {
        moe_set_error("%s: %s: null or not 16-byte aligned", who, name);
        return true;
    }
    return false;
}

bool bad_sizes(const char* who, int n_tok, int k, int hidden, int dtype) {
    if (n_tok < 0 || k < 1 || (int64_t)n_tok * k > (1 << 30) || hidden < 8 || hidden % 8 || hidden > (1 << 30) ||
        (dtype != 0 && dtype != 1)) {
        moe_set_error("%s: n_tok=%d k=%d (up to 2^30 rows) hidden=%d (a multiple of 8) dtype=%d (0 fp16, 1 bf16)", who, n_tok, k,
                      hidden, dtype);
        return true;
    }
    return false;
}

dim3 combine_grid(int64_t items, int per) {
    const int64_t blocks = (items + per - 1) / per;
    return dim3((uint32_t)(blocks < kCombineBlocks ? blocks : kCombineBlocks));
}

template <typename T>
int launch_combine(const CombineArgs& a, int out_f32, hipStream_t s) {
    const dim3 grid = combine_grid((int64_t)a.n_tok * (a.hidden / 8), kCombineThreads);
    if (out_f32) hipLaunchKernelGGL((k_combine<T, true>), grid, dim3(kCombineThreads), 0, s, a);
    else hipLaunchKernelGGL((k_combine<T, false>), grid, dim3(kCombineThreads), 0, s, a);
    HIP_TRY(hipGetLastError());
    return 0;
}

template <typename T>
int launch_combine_grad(const CombineGradArgs& a, hipStream_t s) {
    hipLaunchKernelGGL((k_combine_grad<T>), combine_grid((int64_t)a.n_tok * a.k, kCombineThreads / 64), dim3(kCombineThreads), 0, s, a);
    HIP_TRY(hipGetLastError());
    return 0;
}

}  // namespace

extern "C" int moe_combine(const void* y, int64_t ldy, const float* weights, const void* residual, int64_t ldr, int n_tok, int k,
                           int hidden, int dtype, int out_f32, void* out, int64_t ldo, void* stream) {
    const char* who = "combine";
    if (bad_sizes(who, n_tok, k, hidden, dtype) || bad_rows(who, "y", y, ldy, hidden, (int64_t)n_tok * k) ||
        (residual && bad_rows(who, "residual", residual, ldr, hidden, n_tok)) || bad_rows(who, "out", out, ldo, hidden, n_tok))
        return -1;
    if (n_tok == 0) return 0;
    if (!weights) {
        moe_set_error("combine: null pointer");
        return -1;
    }
    const CombineArgs a = {y, weights, residual, out, ldy, ldr, ldo, n_tok, k, hidden};
    return dtype ? launch_combine<__bf16>(a, out_f32, (hipStream_t)stream) : launch_combine<_Float16>(a, out_f32, (hipStream_t)stream);
}

extern "C" int moe_combine_grad(const void* dout, int64_t ldd, const void* y, int64_t ldy, const float* weights, int n_tok, int k,
                                int hidden, int dtype, void* dy, int64_t lddy, float* dweights, void* stream) {
    const char* who = "combine_grad";
    const int64_t rows = (int64_t)n_tok * k;
    if (bad_sizes(who, n_tok, k, hidden, dtype) || bad_rows(who, "dout", dout, ldd, hidden, n_tok) ||
        bad_rows(who, "y", y, ldy, hidden, rows) || bad_rows(who, "dy", dy, lddy, hidden, rows))
        return -1;
    if (n_tok == 0) return 0;
    if (!weights || !dweights) {
        moe_set_error("combine_grad: null pointer");
        return -1;
    }
    const CombineGradArgs a = {dout, y, weights, dy, dweights, ldd, ldy, lddy, n_tok, k, hidden};
    return dtype ? launch_combine_grad<__bf16>(a, (hipStream_t)stream) : launch_combine_grad<_Float16>(a, (hipStream_t)stream);
}
