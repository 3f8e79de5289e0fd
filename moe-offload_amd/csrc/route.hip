// Routing of a batch: each token's experts and their weights from the router's logits l, and the weights' gradient.
//
//     s = softmax(l) or sigmoid(l);    c = s + bias, or l itself where there is no bias (its order is the scores' own)
//     groups of n_exp / n_group adjacent experts: a group's value is the sum of its group_best largest c (of s, where
//     there is no bias and group_best > 1); the topk_group groups of the largest values are kept
//     ids = the k largest c of the experts kept, in descending order;   w_j = scale s[id_j] (/ the sum of all k)
// Equals go to the lowest index.  An expert whose logit or bias is -inf or NaN is never chosen; places that remain
// have id -1 and weight 0.  A NaN among a row's logits makes its weights NaN.  Infinite logits have the weights'
// limits: several +inf share a softmax evenly.
//
// With g = scale dw over the places with an id, p the weights before the scale, u = l[id], the gradient in the logits is
//     softmax, renormalised   dl[id_j] += p_j (g_j - sum p g)
//     softmax                 dl[e] = s_e (sum of g_j with id_j = e, - sum p g)      for every expert
//     sigmoid, renormalised   dl[id_j] += p_j sig(-u_j) (g_j - sum p g)
//     sigmoid                 dl[id_j] += s_j sig(-u_j) g_j
// and the bias has none.  The reference routes one token (mlx-qwen38/loader.py:903-908), by softmax alone.
//
// A wave takes a token.  Comparisons are exact: logits as they come, and sums of a score and a bias in 64 bits, where
// 32 would let experts trade places whose values differ by less than their rounding.
#include <hip/hip_fp16.h>

#include "lane_reduce.h"
#include "moe_common.h"

namespace {

constexpr int kRouteMaxExp = 1024;
constexpr int kRouteMaxK = 32;
constexpr int kRouteMaxGroups = 64;
constexpr int kRouteThreads = 256, kRouteWaves = kRouteThreads / 64;
constexpr int kRouteBlocks = 1 << 20;       // more tokens than they hold: a block takes several

struct RouteArgs {
    const void* logits;
    const float* bias;
    int32_t* ids;
    float* weights;
    int64_t ld;
    int n_tok, n_exp, k, n_group, topk_group, group_best;
    float scale;
};

struct RouteGradArgs {
    const void* logits;
    const int32_t* ids;
    const float* dweights;
    void* dlogits;
    int64_t ld, ldd;
    int n_tok, n_exp, k;
    float scale;
};

template <typename T>
__device__ __forceinline__ float widen(T v) { return (float)v; }

// exp(l - m) for l <= m: 1 where they are equal (infinite or not), 0 for -inf.
__device__ __forceinline__ float exp_below(float l, float m) {
    return l == -__builtin_inff() ? 0.f : l == m ? 1.f : expf(l - m);
}
__device__ __forceinline__ double exp_below(double l, double m) {
    return l == -__builtin_inf() ? 0.0 : l == m ? 1.0 : exp(l - m);
}

__device__ __forceinline__ float sigmoid(float l) { return 1.f / (1.f + expf(-l)); }
__device__ __forceinline__ double sigmoid(double l) { return 1.0 / (1.0 + exp(-l)); }

// Order of doubles as unsigned integers; -0 is 0.  Never 0, which stands for "not to be chosen".
__device__ __forceinline__ uint64_t order_key(double c) {
    const uint64_t b = (uint64_t)__double_as_longlong(c + 0.0);
    return b >> 63 ? ~b : b | 1ull << 63;
}

__device__ __forceinline__ uint64_t wave_max_u64(uint64_t v) {
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t o = __shfl_xor(v, d, 64);
        v = o > v ? o : v;
    }
    return v;
}

__device__ __forceinline__ float wave_max_f32(float v) {
    for (int d = 1; d < 64; d <<= 1) v = fmaxf(v, __shfl_xor(v, d, 64));
    return v;
}

// The k weights' parts before the scale, a place per lane (id < 0: none): softmax or sigmoid over the chosen ones.
// Scores of any magnitude keep their bits: both are taken relative to the largest.
template <bool SIGMOID>
__device__ __forceinline__ float renormalised(float l, bool has) {
    float top = wave_max_f32(has ? l : -__builtin_inff());
    float v;
    if constexpr (SIGMOID) {
        top = fminf(top, 0.f);
        v = has ? exp_below(fminf(l, 0.f), top) / (1.f + expf(-fabsf(l))) : 0.f;
    } else {
        v = has ? exp_below(l, top) : 0.f;
    }
    const float sum = lanes::group_sum<64>(v);
    return sum > 0.f ? v / sum : v;
}

template <typename T, bool SIGMOID, bool RENORM>
__global__ __launch_bounds__(kRouteThreads) void k_route(RouteArgs a) {
    constexpr int P = kRouteMaxExp / 64;
    __shared__ double group_in[kRouteWaves][kRouteMaxExp];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const int per = a.n_exp / a.n_group;
    for (int64_t t = (int64_t)blockIdx.x * kRouteWaves + wv; t < a.n_tok; t += (int64_t)gridDim.x * kRouteWaves) {
        const T* row = (const T*)a.logits + t * a.ld;
        float l[P];
        bool nan = false;
        float top = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int e = lane + 64 * i;
            l[i] = e < a.n_exp ? widen(row[e]) : -__builtin_inff();
            nan |= l[i] != l[i];
            top = fmaxf(top, l[i]);
        }
        nan = __any(nan);
        top = wave_max_f32(top);
        double sum = 0;
        if constexpr (!SIGMOID) {
#pragma unroll
            for (int i = 0; i < P; ++i) sum += l[i] == l[i] ? exp_below((double)l[i], (double)top) : 0.0;
            sum = lanes::wave_sum_f64(sum);
        }
        uint64_t key[P];
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int e = lane + 64 * i;
            key[i] = 0;
            if (e >= a.n_exp) continue;
            bool ok = l[i] > -__builtin_inff();
            double c = l[i];
            const double s = SIGMOID ? sigmoid((double)l[i]) : exp_below((double)l[i], (double)top) / sum;
            if (a.bias) {
                c = s + (double)a.bias[e];
                ok &= c > -__builtin_inf();
            }
            if (ok) key[i] = order_key(c);
            if (a.n_group > 1) group_in[wv][e] = !ok ? -__builtin_inf() : a.bias || a.group_best == 1 ? c : s;
        }
        if (a.n_group > 1) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_wave_barrier();
            double first = -__builtin_inf(), second = first;
            if (lane < a.n_group)
                for (int i = 0; i < per; ++i) {
                    const double v = group_in[wv][lane * per + i];
                    if (v > first) second = first, first = v;
                    else if (v > second) second = v;
                }
            if (a.group_best > 1 && second > -__builtin_inf()) first += second;
            // lanes whose group comes before this one's
            int before = 0;
            for (int g = 0; g < a.n_group; ++g) {
                const double v = __shfl(first, g, 64);
                before += v > first || (v == first && g < lane);
            }
            const uint64_t kept = __ballot(lane < a.n_group && before < a.topk_group);
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const int e = lane + 64 * i;
                if (e < a.n_exp && !(kept >> (e / per) & 1)) key[i] = 0;
            }
            __builtin_amdgcn_wave_barrier();
        }
        int id = -1;
        float mine = -__builtin_inff();
        for (int j = 0; j < a.k; ++j) {
            uint64_t best = 0;
#pragma unroll
            for (int i = 0; i < P; ++i) best = key[i] > best ? key[i] : best;
            best = wave_max_u64(best);
            if (best == 0) break;
            uint32_t at = ~0u;
#pragma unroll
            for (int i = P - 1; i >= 0; --i) at = key[i] == best ? (uint32_t)(lane + 64 * i) : at;
            for (int d = 1; d < 64; d <<= 1) at = min(at, __shfl_xor(at, d, 64));
            float v = 0.f;
#pragma unroll
            for (int i = 0; i < P; ++i)
                if (at == (uint32_t)(lane + 64 * i)) {
                    v = l[i];
                    key[i] = 0;
                }
            v = __shfl(v, at & 63, 64);
            if (lane == j) id = (int)at, mine = v;
        }
        float w;
        if constexpr (RENORM) w = renormalised<SIGMOID>(mine, id >= 0);
        else if constexpr (SIGMOID) w = sigmoid(mine);
        else w = id >= 0 ? exp_below(mine, top) / (float)sum : 0.f;
        w = nan ? __builtin_nanf("") : id < 0 ? 0.f : w * a.scale;
        if (lane < a.k) {
            a.ids[t * a.k + lane] = id;
            a.weights[t * a.k + lane] = w;
        }
    }
}

template <typename T, bool SIGMOID, bool RENORM>
__global__ __launch_bounds__(kRouteThreads) void k_route_grad(RouteGradArgs a) {
    constexpr int P = kRouteMaxExp / 64;
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    for (int64_t t = (int64_t)blockIdx.x * kRouteWaves + wv; t < a.n_tok; t += (int64_t)gridDim.x * kRouteWaves) {
        const T* row = (const T*)a.logits + t * a.ld;
        T* out = (T*)a.dlogits + t * a.ldd;
        int id = -1;
        float l = -__builtin_inff(), g = 0.f;
        if (lane < a.k) {
            id = a.ids[t * a.k + lane];
            if (id < 0 || id >= a.n_exp) id = -1;
            if (id >= 0) {
                l = widen(row[id]);
                g = a.scale * a.dweights[t * a.k + lane];
            }
        }
        float s[P], v;
        if constexpr (!SIGMOID && !RENORM) {
            float x[P], top = -__builtin_inff();
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const int e = lane + 64 * i;
                x[i] = e < a.n_exp ? widen(row[e]) : -__builtin_inff();
                top = fmaxf(top, x[i]);
            }
            top = wave_max_f32(top);
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < P; ++i) sum += s[i] = exp_below(x[i], top);
            sum = lanes::group_sum<64>(sum);
            const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
#pragma unroll
            for (int i = 0; i < P; ++i) s[i] *= inv;
            v = g;
            const float dot = lanes::group_sum<64>(id >= 0 ? exp_below(l, top) * inv * g : 0.f);
            float d[P];
#pragma unroll
            for (int i = 0; i < P; ++i) d[i] = -dot;
            for (int j = 0; j < a.k; ++j) {
                const int at = __shfl(id, j, 64);
                const float add = __shfl(v, j, 64);
#pragma unroll
                for (int i = 0; i < P; ++i)
                    if (at == lane + 64 * i) d[i] += add;
            }
#pragma unroll
            for (int i = 0; i < P; ++i)
                if (lane + 64 * i < a.n_exp) out[lane + 64 * i] = (T)(s[i] * d[i]);
        } else {
            if constexpr (RENORM) {
                const float p = renormalised<SIGMOID>(l, id >= 0);
                const float dot = lanes::group_sum<64>(id >= 0 ? p * g : 0.f);
                v = p * (g - dot);
                if constexpr (SIGMOID) v *= sigmoid(-l);
            } else {
                v = sigmoid(l) * sigmoid(-l) * g;
            }
#pragma unroll
            for (int i = 0; i < P; ++i) s[i] = 0.f;
            for (int j = 0; j < a.k; ++j) {
                const int at = __shfl(id, j, 64);
                const float add = __shfl(v, j, 64);
#pragma unroll
                for (int i = 0; i < P; ++i)
                    if (at == lane + 64 * i) s[i] += add;
            }
#pragma unroll
            for (int i = 0; i < P; ++i)
                if (lane + 64 * i < a.n_exp) out[lane + 64 * i] = (T)s[i];
        }
    }
}

bool bad_route(const char* who, const void* logits, int64_t ld, int n_tok, int n_exp, int k, int score, int renorm, int dtype) {
    if (n_tok < 0 || n_exp < 1 || n_exp > kRouteMaxExp || k < 1 || k > kRouteMaxK || k > n_exp || ld < n_exp) {
        moe_set_error("%s: n_tok=%d n_exp=%d (1..%d) k=%d (1..%d, at most n_exp) at a step of %lld", who, n_tok, n_exp, kRouteMaxExp,
                      k, kRouteMaxK, (long long)ld);
        return true;
    }
    if ((score != 0 && score != 1) || (renorm != 0 && renorm != 1) || dtype < 0 || dtype > 2) {
        moe_set_error("%s: score=%d renorm=%d (0, 1) dtype=%d (0 fp16, 1 bf16, 2 fp32)", who, score, renorm, dtype);
        return true;
    }
    if (n_tok > 0 && !logits) {
        moe_set_error("%s: null pointer", who);
        return true;
    }
    return false;
}

template <typename T, typename A, typename L>
int by_rule(int score, int renorm, const A& a, const L& launch) {
    if (score) return renorm ? launch(T(), std::true_type(), std::true_type()) : launch(T(), std::true_type(), std::false_type());
    return renorm ? launch(T(), std::false_type(), std::true_type()) : launch(T(), std::false_type(), std::false_type());
}

template <typename A, typename L>
int by_type(int dtype, int score, int renorm, const A& a, const L& launch) {
    if (dtype == 0) return by_rule<_Float16>(score, renorm, a, launch);
    if (dtype == 1) return by_rule<__bf16>(score, renorm, a, launch);
    return by_rule<float>(score, renorm, a, launch);
}

dim3 route_grid(int n_tok) {
    const int64_t blocks = ((int64_t)n_tok + kRouteWaves - 1) / kRouteWaves;
    return dim3((uint32_t)(blocks < kRouteBlocks ? blocks : kRouteBlocks));
}

}  // namespace

extern "C" int moe_route(const void* logits, int64_t ld, int n_tok, int n_exp, int k, int score, int renorm, const float* bias,
                         int n_group, int topk_group, int group_best, float scale, int dtype, int32_t* ids, float* weights,
                         void* stream) {
    const char* who = "route";
    if (bad_route(who, logits, ld, n_tok, n_exp, k, score, renorm, dtype)) return -1;
    if (n_group < 1 || n_group > kRouteMaxGroups || n_exp % n_group || topk_group < 1 || topk_group > n_group ||
        (group_best != 1 && group_best != 2)) {
        moe_set_error("route: n_group=%d (1..%d, a divisor of n_exp=%d) topk_group=%d (1..n_group) group_best=%d (1, 2)", n_group,
                      kRouteMaxGroups, n_exp, topk_group, group_best);
        return -1;
    }
    if (n_tok == 0) return 0;
    if (!ids || !weights) {
        moe_set_error("route: null pointer");
        return -1;
    }
    const RouteArgs a = {logits, bias, ids, weights, ld, n_tok, n_exp, k, n_group, topk_group, group_best, scale};
    const hipStream_t s = (hipStream_t)stream;
    return by_type(dtype, score, renorm, a, [&](auto type, auto sigmoid, auto renorm_) {
        using T = decltype(type);
        hipLaunchKernelGGL((k_route<T, decltype(sigmoid)::value, decltype(renorm_)::value>), route_grid(n_tok), dim3(kRouteThreads),
                           0, s, a);
        HIP_TRY(hipGetLastError());
        return 0;
    });
}

extern "C" int moe_route_grad(const float* dweights, const void* logits, int64_t ld, const int32_t* ids, int n_tok, int n_exp, int k,
                              int score, int renorm, float scale, int dtype, void* dlogits, int64_t ldd, void* stream) {
    const char* who = "route_grad";
    if (bad_route(who, logits, ld, n_tok, n_exp, k, score, renorm, dtype)) return -1;
    if (ldd < n_exp) {
        moe_set_error("route_grad: gradients at a step of %lld", (long long)ldd);
        return -1;
    }
    if (n_tok == 0) return 0;
    if (!ids || !dweights || !dlogits) {
        moe_set_error("route_grad: null pointer");
        return -1;
    }
    const RouteGradArgs a = {logits, ids, dweights, dlogits, ld, ldd, n_tok, n_exp, k, scale};
    const hipStream_t s = (hipStream_t)stream;
    return by_type(dtype, score, renorm, a, [&](auto type, auto sigmoid, auto renorm_) {
        using T = decltype(type);
        hipLaunchKernelGGL((k_route_grad<T, decltype(sigmoid)::value, decltype(renorm_)::value>), route_grid(n_tok),
                           dim3(kRouteThreads), 0, s, a);
        HIP_TRY(hipGetLastError());
        return 0;
    });
}
