// Low-rank adapters of many requests at once beside a shared projection.
//
// Token t belongs to a request with adapter i = ids[t]:   out[t] = base[t] + s_i B_i (A_i x[t]),
// A_i [rank][n_in], B_i [n_out][rank]; an id outside the adapters leaves out[t] = base[t].  base is the
// shared projection's output (a grouped product, the 2-bit experts' rows, a router's logits) and may be
// out itself.  v = A_i x stays in fp32 between the two products, and out is rounded once.
#include <hip/hip_bf16.h>

#include "moe_common.h"

namespace {

template <typename T>
__device__ __forceinline__ void widen8(uint4 w, float* v) {
    typedef T t8 __attribute__((ext_vector_type(8)));
    const t8 r = __builtin_bit_cast(t8, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)r[i];
}

// v[t][j] = s_i A_i[j] x[t]: one wave per (t, j).
template <typename T>
__global__ __launch_bounds__(256) void k_lora_v(const T* __restrict__ x, int64_t ldx, const T* __restrict__ A, int64_t a_stride,
                                                const int32_t* __restrict__ ids, const float* __restrict__ scale, int n_tok,
                                                int n_ad, int n_in, int rank, float* __restrict__ v) {
    const int lane = threadIdx.x & 63;
    const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int t = (int)(w / rank), j = (int)(w % rank);
    if (t >= n_tok) return;
    const int i = ids[t];
    if (i < 0 || i >= n_ad) return;
    const T* a = A + (int64_t)i * a_stride + (int64_t)j * n_in;
    const T* xr = x + (int64_t)t * ldx;
    float sum = 0.f;
    for (int c = lane * 8; c < n_in; c += 512) {
        float av[8], xv[8];
        widen8<T>(*(const uint4*)(a + c), av);
        widen8<T>(*(const uint4*)(xr + c), xv);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = fmaf(av[e], xv[e], sum);
    }
    for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d, 64);
    if (lane == 0) v[(int64_t)t * rank + j] = (scale ? scale[i] : 1.0f) * sum;
}

template <typename T>
__global__ __launch_bounds__(256) void k_lora_out(const T* base, int64_t ldb, const float* __restrict__ v,
                                                  const T* __restrict__ B, int64_t b_stride, const int32_t* __restrict__ ids,
                                                  int n_ad, int n_out, int rank, T* out, int64_t ldo) {
    const int64_t t = blockIdx.x;
    const int n = blockIdx.y * 256 + threadIdx.x;
    if (n >= n_out) return;
    const int i = ids[t];
    float sum = 0.f;
    if (i >= 0 && i < n_ad) {
        const T* b = B + (int64_t)i * b_stride + (int64_t)n * rank;
        for (int j = 0; j < rank; j += 8) {
            float bv[8];
            widen8<T>(*(const uint4*)(b + j), bv);
#pragma unroll
            for (int e = 0; e < 8; ++e) sum = fmaf(bv[e], v[t * rank + j + e], sum);
        }
    } else if (base == out) {
        return;
    }
    out[t * ldo + n] = (T)((float)base[t * ldb + n] + sum);
}

template <typename T>
int lora_add(const void* base, int64_t ldb, const void* x, int64_t ldx, const void* A, int64_t a_stride, const void* B,
             int64_t b_stride, const int32_t* ids, const float* scale, int n_tok, int n_ad, int n_in, int n_out, int rank,
             float* v, void* out, int64_t ldo, hipStream_t s) {
    const int64_t waves = (int64_t)n_tok * rank;
    hipLaunchKernelGGL((k_lora_v<T>), dim3((uint32_t)((waves + 3) / 4)), dim3(256), 0, s, (const T*)x, ldx, (const T*)A,
                       a_stride, ids, scale, n_tok, n_ad, n_in, rank, v);
    HIP_TRY(hipGetLastError());
    hipLaunchKernelGGL((k_lora_out<T>), dim3(n_tok, (n_out + 255) / 256), dim3(256), 0, s, (const T*)base, ldb, v,
                       (const T*)B, b_stride, ids, n_ad, n_out, rank, (T*)out, ldo);
    HIP_TRY(hipGetLastError());
    return 0;
}

}  // namespace

extern "C" uint64_t moe_lora_workspace_bytes(int n_tok, int rank) {
    return n_tok > 0 && rank > 0 ? (uint64_t)n_tok * rank * 4 : 0;
}

extern "C" int moe_lora_add(const void* base, int64_t ld_base, const void* x, int64_t ldx, const void* a, int64_t a_stride,
                            const void* b, int64_t b_stride, const int32_t* ids, const float* scale, int n_tok, int n_ad,
                            int n_in, int n_out, int rank, int dtype, void* workspace, void* out, int64_t ld_out,
                            void* stream) {
    if ((dtype != 0 && dtype != 1) || n_tok < 0 || n_ad < 0 || n_in <= 0 || n_out <= 0 || rank <= 0 || n_in % 8 ||
        n_out % 8 || rank % 8 || rank > 256) {
        moe_set_error("lora_add: dtype=%d n_tok=%d n_ad=%d n_in=%d n_out=%d rank=%d (multiples of 8, rank <= 256)", dtype,
                      n_tok, n_ad, n_in, n_out, rank);
        return -1;
    }
    if (ldx % 8 || ld_base % 8 || ld_out % 8 || a_stride % 8 || b_stride % 8 ||
        (n_tok > 1 && (ldx < n_in || ld_base < n_out || ld_out < n_out)) ||
        (n_ad > 1 && (a_stride < (int64_t)rank * n_in || b_stride < (int64_t)rank * n_out))) {
        moe_set_error("lora_add: strides must be multiples of 8 and not less than a row or matrix");
        return -1;
    }
    if (n_tok == 0) return 0;
    if (!base || !x || !ids || !out || !workspace || (n_ad > 0 && (!a || !b))) {
        moe_set_error("lora_add: null pointer");
        return -1;
    }
    if (((uintptr_t)base | (uintptr_t)x | (uintptr_t)a | (uintptr_t)b | (uintptr_t)out | (uintptr_t)workspace) % 16) {
        moe_set_error("lora_add: pointers must be 16-byte aligned");
        return -1;
    }
    if (((int64_t)n_tok * rank + 3) / 4 > 0x7FFFFFFF || (n_out + 255) / 256 > 65535) {
        moe_set_error("lora_add: n_tok=%d x rank=%d or n_out=%d is more than one launch takes", n_tok, rank, n_out);
        return -1;
    }
    auto f = dtype ? lora_add<__bf16> : lora_add<_Float16>;
    return f(base, ld_base, x, ldx, a, a_stride, b, b_stride, ids, scale, n_tok, n_ad, n_in, n_out, rank, (float*)workspace,
             out, ld_out, (hipStream_t)stream);
}
