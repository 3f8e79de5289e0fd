// Low-rank adapters of many requests at once beside a shared projection.
//
// Token t belongs to a request with adapter i = ids[t]:   out[t] = base[t] + s_i B_i (A_i x[t]),
// A_i [rank][n_in], B_i [n_out][rank]; an id outside the adapters leaves out[t] = base[t].  base is the
// shared projection's output (a grouped product, the 2-bit experts' rows, a router's logits) and may be
// out itself.  v = A_i x stays in fp32 between the two products, and out is rounded once.
//
// Two launches.  k_lora_v: 16 tokens and up to 32 ranks per block, the contraction split over its waves, both
// operands from global memory straight in the matrix unit's layout (each byte of x is used for 16 ranks at a
// time, so staging would gain nothing).  k_lora_out: 16 tokens and 64 output columns per block, v and B in the
// fp32 matrix unit, so v keeps its bits and its range.  The tokens of a tile may have different adapters: the
// tile is multiplied by each adapter that occurs in it and every token keeps its own adapter's result.  In a
// batch of prompts that is one adapter nearly always; for few tokens the adapters of a tile go to blocks of
// their own.
#include <hip/hip_bf16.h>

#include <initializer_list>

#include "../../include/moe_offload.h"
#include "grouped_mm.h"

namespace {

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

// What lanes past the end of a row read.
__device__ uint4 g_zero16;

constexpr int kVWaves = 8;

// v[t][j] = s_i A_i[j] x[t] for 16 ST tokens (blockIdx.x) and 16 SR ranks (blockIdx.y), an eighth of the row per wave.
template <typename T, int SR, int ST>
__global__ __launch_bounds__(64 * kVWaves, 4) void k_lora_v(const T* __restrict__ x, int64_t ldx, const T* __restrict__ A,
                                                            int64_t a_stride, const int32_t* __restrict__ ids,
                                                            const float* __restrict__ scale, int n_tok, int n_ad, int n_in,
                                                            int rank, float* __restrict__ v) {
    constexpr int U = 8 / (SR * ST) < 4 ? 4 : 8 / (SR * ST);                   // steps of 32 whose loads are under way at once
    __shared__ f32x4 part[kVWaves][SR * ST][64];
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, kq = lane >> 4;
    const int j0 = blockIdx.y * (16 * SR);
    const T* zero = (const T*)&g_zero16;
    int64_t t[ST];
    const T* xr[ST];
    int id[ST];
    bool has[ST];
#pragma unroll
    for (int m = 0; m < ST; ++m) {
        t[m] = ((int64_t)blockIdx.x * ST + m) * 16 + n;
        xr[m] = x + (t[m] < n_tok ? t[m] : (int64_t)n_tok - 1) * ldx + kq * 8;
        id[m] = t[m] < n_tok ? ids[t[m]] : -1;
        has[m] = id[m] >= 0 && id[m] < n_ad;
    }
    const int steps = (n_in + 31) / 32, per = (steps + kVWaves - 1) / kVWaves;
    const int s0 = wv * per, s1 = s0 + per < steps ? s0 + per : steps;
    each_adapter<ST>(id, has, blockIdx.z, gridDim.z, [&](int i, const bool (&mine)[ST]) {
        const T* ar[SR];
#pragma unroll
        for (int s = 0; s < SR; ++s) {
            const int j = j0 + s * 16 + n;
            ar[s] = A + (int64_t)i * a_stride + (int64_t)(j < rank ? j : rank - 1) * n_in + kq * 8;
        }
        f32x4 acc[SR][ST] = {};
#pragma unroll 1
        for (int s = s0; s < s1; s += U) {
            uint4 xv[ST][U], av[SR][U];
            const bool whole = s + U <= s1 && (s + U) * 32 <= n_in;            // wave-uniform
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int c = (s + u) * 32;
                const bool in = whole || (s + u < s1 && c + kq * 8 < n_in);
#pragma unroll
                for (int m = 0; m < ST; ++m) xv[m][u] = *(const uint4*)(in ? xr[m] + c : zero);
#pragma unroll
                for (int r = 0; r < SR; ++r) av[r][u] = *(const uint4*)(in ? ar[r] + c : zero);
            }
            __builtin_amdgcn_sched_barrier(0);                                 // all of them before the first product
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int r = 0; r < SR; ++r)
#pragma unroll
                    for (int m = 0; m < ST; ++m) acc[r][m] = mfma<T>(av[r][u], xv[m][u], acc[r][m]);
        }
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
            const float si = scale ? scale[i] : 1.0f;
#pragma unroll
            for (int m = 0; m < ST; ++m)
                if (wv % ST == m && mine[m] && j < rank) *(f32x4*)(v + t[m] * rank + j) = sum * si;
        }
        __syncthreads();
    });
}

// out = base + B_i v for 16 ST tokens (blockIdx.x) and 64 SC columns (blockIdx.y), 16 SC to a wave.
template <typename T, int SC, int ST>
__global__ __launch_bounds__(256) void k_lora_out(const T* base, int64_t ldb, const float* __restrict__ v,
                                                  const T* __restrict__ B, int64_t b_stride, const int32_t* __restrict__ ids,
                                                  int n_tok, int n_ad, int n_out, int rank, T* out, int64_t ldo) {
    typedef T t4 __attribute__((ext_vector_type(4)));
    const int lane = threadIdx.x & 63, n = lane & 15, kq = lane >> 4;
    const int q0 = (blockIdx.y * 4 + (threadIdx.x >> 6)) * (16 * SC);
    if (q0 >= n_out) return;
    const T* zero = (const T*)&g_zero16;
    int64_t t[ST];
    int id[ST];
    bool has[ST], got[ST];
    t4 bs[ST][SC];                             // lane (n, kq): columns 4 kq .. + 3 of token n
    f32x4 acc[ST][SC];
#pragma unroll
    for (int m = 0; m < ST; ++m) {
        t[m] = ((int64_t)blockIdx.x * ST + m) * 16 + n;
        id[m] = t[m] < n_tok ? ids[t[m]] : -1;
        has[m] = id[m] >= 0 && id[m] < n_ad;
        got[m] = false;
#pragma unroll
        for (int s = 0; s < SC; ++s) {
            const int q = q0 + s * 16 + kq * 4;
            bs[m][s] = *(const t4*)(base + (t[m] < n_tok ? t[m] : 0) * ldb + (q < n_out ? q : 0));
        }
    }
    each_adapter<ST>(id, has, blockIdx.z, gridDim.z, [&](int i, const bool (&mine)[ST]) {
        const T* br[SC];
#pragma unroll
        for (int s = 0; s < SC; ++s) {
            const int q = q0 + s * 16 + n;
            br[s] = B + (int64_t)i * b_stride + (int64_t)(q < n_out ? q : n_out - 1) * rank + kq * 8;
        }
        f32x4 one[ST][SC] = {};
        uint4 bv[SC];
        f32x4 lo[ST], hi[ST];
        auto fetch = [&](int k0) {
            const bool in = k0 + kq * 8 < rank;
#pragma unroll
            for (int s = 0; s < SC; ++s) bv[s] = *(const uint4*)(in ? br[s] + k0 : zero);
#pragma unroll
            for (int m = 0; m < ST; ++m) {
                const float* p = v + t[m] * rank + k0 + kq * 8;
                lo[m] = *(const f32x4*)(in && mine[m] ? p : (const float*)zero);
                hi[m] = *(const f32x4*)(in && mine[m] ? p + 4 : (const float*)zero);
            }
        };
        fetch(0);
#pragma unroll 1
        for (int k0 = 0; k0 < rank; k0 += 32) {
            float bw[SC][8];
            f32x4 l[ST], h[ST];
#pragma unroll
            for (int s = 0; s < SC; ++s) widen8<T>(bv[s], bw[s]);
#pragma unroll
            for (int m = 0; m < ST; ++m) l[m] = lo[m], h[m] = hi[m];
            if (k0 + 32 < rank) fetch(k0 + 32);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int e = 0; e < 8; ++e)
#pragma unroll
                for (int m = 0; m < ST; ++m)
#pragma unroll
                    for (int s = 0; s < SC; ++s)
                        one[m][s] = __builtin_amdgcn_mfma_f32_16x16x4f32(bw[s][e], e < 4 ? l[m][e] : h[m][e - 4], one[m][s], 0, 0, 0);
        }
#pragma unroll
        for (int m = 0; m < ST; ++m)
            if (mine[m]) {
                got[m] = true;
#pragma unroll
                for (int s = 0; s < SC; ++s) acc[m][s] = one[m][s];
            }
    });
    // a token without an adapter is written by the first block of its tile
#pragma unroll
    for (int m = 0; m < ST; ++m) {
        if (t[m] >= n_tok || !(got[m] || (!has[m] && blockIdx.z == 0 && base != out))) continue;
#pragma unroll
        for (int s = 0; s < SC; ++s) {
            const int q = q0 + s * 16 + kq * 4;
            t4 r = bs[m][s];
            if (got[m])
#pragma unroll
                for (int e = 0; e < 4; ++e) r[e] = (T)((float)r[e] + acc[m][s][e]);
            if (q < n_out) *(t4*)(out + t[m] * ldo + q) = r;
        }
    }
}

template <typename T, int ST>
int lora_add(const T* base, int64_t ldb, const T* x, int64_t ldx, const T* A, int64_t a_stride, const T* B, int64_t b_stride,
             const int32_t* ids, const float* scale, int n_tok, int n_ad, int n_in, int n_out, int rank, float* v, T* out,
             int64_t ldo, hipStream_t s) {
    const uint32_t tiles = (uint32_t)(((int64_t)n_tok + 16 * ST - 1) / (16 * ST));
    // up to 256 tokens a tile's adapters get blocks of their own (16 tokens have 16 at most)
    const uint32_t split = ST == 1 && n_tok <= 256 ? (uint32_t)(n_tok < 16 ? n_tok : 16) : 1;
    if (n_ad > 0) {
        if (rank <= 16)
            hipLaunchKernelGGL((k_lora_v<T, 1, ST>), dim3(tiles, 1, split), dim3(64 * kVWaves), 0, s, x, ldx, A, a_stride, ids,
                               scale, n_tok, n_ad, n_in, rank, v);
        else
            hipLaunchKernelGGL((k_lora_v<T, 2, ST>), dim3(tiles, (rank + 31) / 32, split), dim3(64 * kVWaves), 0, s, x, ldx, A,
                               a_stride, ids, scale, n_tok, n_ad, n_in, rank, v);
        HIP_TRY(hipGetLastError());
    }
    if ((int64_t)tiles * n_out < 512 * 256)
        hipLaunchKernelGGL((k_lora_out<T, 1, ST>), dim3(tiles, (n_out + 63) / 64, split), dim3(256), 0, s, base, ldb, v, B,
                           b_stride, ids, n_tok, n_ad, n_out, rank, out, ldo);
    else
        hipLaunchKernelGGL((k_lora_out<T, 4, ST>), dim3(tiles, (n_out + 255) / 256, split), dim3(256), 0, s, base, ldb, v, B,
                           b_stride, ids, n_tok, n_ad, n_out, rank, out, ldo);
    HIP_TRY(hipGetLastError());
    return 0;
}

template <typename T>
int lora_add_typed(const void* base, int64_t ldb, const void* x, int64_t ldx, const void* A, int64_t a_stride, const void* B,
                   int64_t b_stride, const int32_t* ids, const float* scale, int n_tok, int n_ad, int n_in, int n_out, int rank,
                   float* v, void* out, int64_t ldo, hipStream_t s) {
    auto f = n_tok <= 1024 ? lora_add<T, 1> : lora_add<T, 2>;
    return f((const T*)base, ldb, (const T*)x, ldx, (const T*)A, a_stride, (const T*)B, b_stride, ids, scale, n_tok, n_ad, n_in,
             n_out, rank, v, (T*)out, ldo, s);
}

// The shapes and strides that both entry points take; base or dy is [n_tok][n_out].
bool bad_shapes(const char* who, int dtype, int n_tok, int n_ad, int n_in, int n_out, int rank, int64_t ldx, int64_t ldy,
                int64_t a_stride, int64_t b_stride) {
    if ((dtype != 0 && dtype != 1) || n_tok < 0 || n_ad < 0 || n_in <= 0 || n_out <= 0 || rank <= 0 || n_in % 8 ||
        n_out % 8 || rank % 8 || rank > 256 || (n_out + 63) / 64 > 65535) {
        moe_set_error("%s: dtype=%d n_tok=%d n_ad=%d n_in=%d n_out=%d rank=%d (multiples of 8, rank <= 256, n_out < 2^22)",
                      who, dtype, n_tok, n_ad, n_in, n_out, rank);
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
    return 2 * up16((uint64_t)n_tok * rank * 2) + 2 * up16((uint64_t)n_tok * 4) + up16((uint64_t)(n_ad + 1) * 4) +
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
    const int64_t mat = (int64_t)rank * n_in;
    void* v = take((uint64_t)n_tok * rank * 2);
    void* dv = take((uint64_t)n_tok * rank * 2);
    int32_t* order = (int32_t*)take((uint64_t)n_tok * 4);
    int32_t* same = (int32_t*)take((uint64_t)n_tok * 4);
    int32_t* seg = (int32_t*)take((uint64_t)(n_ad + 1) * 4);
    // rows sorted by adapter; v and dv are in that order.  Without tokens da and db are the products over empty segments
    if (moe_expert_plan(ids, n_tok, 1, n_ad, p, same, order, seg, stream) ||
        moe_grouped_mm(x, ldx, n_tok, order, seg, nullptr, n_ad, n_tok, a, a_stride, n_ad, rank, n_in, nullptr, v, rank, n_tok,
                       nullptr, dtype, 1, stream) ||
        moe_grouped_mm_dx(dy, lddy, n_tok, order, seg, nullptr, n_ad, n_tok, b, b_stride, n_ad, n_out, rank, scale, nullptr, 0,
                          dv, rank, n_tok, nullptr, dtype, 1, stream) ||
        moe_grouped_mm_dx(dv, rank, n_tok, nullptr, seg, nullptr, n_ad, n_tok, a, a_stride, n_ad, rank, n_in, nullptr, nullptr,
                          0, dx, lddx, n_tok, order, dtype, 1, stream) ||
        moe_grouped_mm_dw(dv, rank, n_tok, nullptr, x, ldx, n_tok, order, seg, n_ad, n_tok, rank, n_in, nullptr, da, mat, 0,
                          dtype, stream) ||
        moe_grouped_mm_dw(dy, lddy, n_tok, order, v, rank, n_tok, nullptr, seg, n_ad, n_tok, n_out, rank, scale, db,
                          (int64_t)rank * n_out, 0, dtype, stream))
        return -1;
    return 0;
}
