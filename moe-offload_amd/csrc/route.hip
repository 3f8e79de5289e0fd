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
// 32 would let experts trade places whose values differ by less than their rounding.  What the 64 bits cost is spent on few
// tokens only: values in 32 bits, with a bound of their error, decide unless two of them are closer than twice that; then
// those that are in question are computed in 64 bits.
//
// The k largest: the k-th largest of the 64 lanes' own maxima, rounded down to 16 bits by a search from bit 31 on (a
// ballot each), is below the k-th largest of all, and few more than k values are above it.  These come one to a lane
// through LDS, and each counts the others above it, which is its place.  Where more than 64 are above (equal logits), k
// rounds of a maximum over the wave find them (k rounds for all: 108 us for 16384 tokens of 512, 12 this way).
//
// The vector unit bounds it: 16384 tokens of 512 fp32 logits, top-10, 11.8 us (79% busy, some 310 operations per token; 35 MB at
// 3 TB/s), of 1024 17.5, of 64 7.0, which is what so many waves take to come and go; top-32 of 512 18; of 512 with a bias 20 (sigmoid) and
// 24 (softmax), whatever its size. 5001 tokens of 240 with a bias and groups 10.5 (74% busy).
// Several tokens per wave, the next one's row read ahead, took 13.5 for the first: more registers, no fewer operations.
#include <hip/hip_fp16.h>

#include "lane_reduce.h"
#include "moe_common.h"

namespace {

constexpr int kRouteMaxExp = 1024;
constexpr int kRouteMaxK = 32;
constexpr int kRouteMaxGroups = 64;
constexpr int kRouteThreads = 256, kRouteWaves = kRouteThreads / 64;
constexpr int kRouteMost = 1 << 24;         // tokens of a launch

constexpr float kInf = __builtin_inff();

struct RouteArgs {
    const void* logits;
    const float* bias;
    int32_t* ids;
    float* weights;
    int64_t ld;
    int n_tok, n_exp, k, n_group, topk_group, group_best;
    int dtype, sigmoid, renorm;
    int wide;                    // rows may be read in pieces of a lane's adjacent values
    int group_size, group_shift; // experts of a group, lanes that look through it: 2^group_shift
    uint32_t group_div;          // e / (n_exp / n_group) = e * group_div >> 20
    float scale;
};

struct RouteGradArgs {
    const void* logits;
    const int32_t* ids;
    const float* dweights;
    void* dlogits;
    int64_t ld, ldd;
    int n_tok, n_exp, k;
    int dtype, sigmoid, renorm, wide, wide_out;
    float scale;
};

// exp(l - m) for l <= m: 1 where they are equal (infinite or not), 0 for -inf.
__device__ __forceinline__ float exp_below(float l, float m) { return l == -kInf ? 0.f : l == m ? 1.f : expf(l - m); }
__device__ __forceinline__ double exp_below(double l, double m) { return l == -__builtin_inf() ? 0.0 : l == m ? 1.0 : exp(l - m); }

__device__ __forceinline__ float sigmoid(float l) { return 1.f / (1.f + expf(-l)); }
__device__ __forceinline__ double sigmoid(double l) { return 1.0 / (1.0 + exp(-l)); }

// Order of floats as unsigned integers; -0 is 0.  0 stands for "not to be chosen": -inf and NaN.
__device__ __forceinline__ uint32_t order_key(float c) {
    const uint32_t b = __float_as_uint(c + 0.f);
    return c > -kInf ? b >> 31 ? ~b : b | 1u << 31 : 0u;
}
__device__ __forceinline__ float order_value(uint32_t k) { return __uint_as_float(k >> 31 ? k & ~(1u << 31) : ~k); }
__device__ __forceinline__ uint64_t order_key(double c) {
    const uint64_t b = (uint64_t)__double_as_longlong(c + 0.0);
    return c > -__builtin_inf() ? b >> 63 ? ~b : b | 1ull << 63 : 0ull;
}
__device__ __forceinline__ double order_value(uint64_t k) { return __longlong_as_double((long long)(k >> 63 ? k & ~(1ull << 63) : ~k)); }

template <typename F>
__device__ __forceinline__ uint32_t wave_reduce_u32(uint32_t v, const F& f) {
    v = f(v, lanes::partner<1>(v));
    v = f(v, lanes::partner<2>(v));
    v = f(v, lanes::partner<4>(v));
    v = f(v, lanes::partner<8>(v));
    auto p = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = f((uint32_t)p[0], (uint32_t)p[1]);
    p = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return f((uint32_t)p[0], (uint32_t)p[1]);
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    return wave_reduce_u32(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}
__device__ __forceinline__ uint32_t wave_min(uint32_t v) {
    return wave_reduce_u32(v, [](uint32_t a, uint32_t b) { return a < b ? a : b; });
}
__device__ __forceinline__ float wave_max(float v) {
    return __uint_as_float(wave_reduce_u32(__float_as_uint(v), [](uint32_t a, uint32_t b) {
        return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    }));
}
__device__ __forceinline__ uint64_t wave_max(uint64_t v) {
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t o = __shfl_xor(v, d, 64);
        v = o > v ? o : v;
    }
    return v;
}

__device__ __forceinline__ uint32_t lane_value(uint32_t v, int lane) { return (uint32_t)__builtin_amdgcn_readlane((int)v, lane); }
__device__ __forceinline__ float lane_value(float v, int lane) { return __uint_as_float(lane_value(__float_as_uint(v), lane)); }

// Lane's value i of P is expert (i / V) 64 V + lane V + i % V: V adjacent ones are one load.
template <int P>
struct Row {
    static constexpr int V = P < 4 ? P : 4;
    static __device__ __forceinline__ int at(int lane, int i) { return i / V * 64 * V + lane * V + i % V; }

    template <typename T>
    static __device__ __forceinline__ void read(const T* row, int n, bool wide, int lane, float (&l)[P]) {
        typedef T tv __attribute__((ext_vector_type(V)));
#pragma unroll
        for (int c = 0; c < P / V; ++c) {
            const int e = at(lane, c * V);
            if (wide && e + V <= n) {
                if constexpr (V == 1) {
                    l[c] = (float)row[e];
                } else {
                    const tv v = *(const tv*)(row + e);
#pragma unroll
                    for (int i = 0; i < V; ++i) l[c * V + i] = (float)v[i];
                }
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) l[c * V + i] = e + i < n ? (float)row[e + i] : -kInf;
            }
        }
    }

    // Infinity below stands for the values past the row's end.
    static __device__ __forceinline__ void read(const void* p, int64_t at, int dtype, int n, bool wide, int lane, float (&l)[P]) {
        if (dtype == 2) read((const float*)p + at, n, wide, lane, l);
        else if (dtype == 1) read((const __bf16*)p + at, n, wide, lane, l);
        else read((const _Float16*)p + at, n, wide, lane, l);
    }

    template <typename T>
    static __device__ __forceinline__ void write(T* row, int n, bool wide, int lane, const float (&l)[P]) {
        typedef T tv __attribute__((ext_vector_type(V)));
#pragma unroll
        for (int c = 0; c < P / V; ++c) {
            const int e = at(lane, c * V);
            if (wide && e + V <= n) {
                if constexpr (V == 1) {
                    row[e] = (T)l[c];
                } else {
                    tv v;
#pragma unroll
                    for (int i = 0; i < V; ++i) v[i] = (T)l[c * V + i];
                    *(tv*)(row + e) = v;
                }
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (e + i < n) row[e + i] = (T)l[c * V + i];
            }
        }
    }

    static __device__ __forceinline__ void write(void* p, int64_t at, int dtype, int n, bool wide, int lane, const float (&l)[P]) {
        if (dtype == 2) write((float*)p + at, n, wide, lane, l);
        else if (dtype == 1) write((__bf16*)p + at, n, wide, lane, l);
        else write((_Float16*)p + at, n, wide, lane, l);
    }
};

__device__ __forceinline__ float read_one(const void* p, int64_t at, int dtype) {
    return dtype == 2 ? ((const float*)p)[at] : dtype == 1 ? (float)((const __bf16*)p)[at] : (float)((const _Float16*)p)[at];
}

// What LDS holds goes from lanes to other lanes of the same wave only.
__device__ __forceinline__ void wave_lds_fence() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_wave_barrier();
}

// A lane's part of the k weights before the scale, softmax or sigmoid over the chosen ones: scores of any magnitude keep
// their bits, both are taken relative to the largest.
__device__ __forceinline__ float renormalised(bool sig, float l, bool has) {
    float top = wave_max(has ? l : -kInf), v = 0.f;
    if (sig) {
        top = fminf(top, 0.f);
        if (has) v = exp_below(fminf(l, 0.f), top) / (1.f + expf(-fabsf(l)));
    } else if (has) {
        v = exp_below(l, top);
    }
    const float sum = lanes::group_sum<64>(v);
    return sum > 0.f ? v / sum : v;
}

// The chosen ones as they end up: a lane's expert and logit, its place among the k, whether it has one.  Lanes n .. k - 1
// stand for the places that nobody has.
struct Chosen {
    int id, place, n;
    float l;
    bool has;
};

// The k largest in k rounds, equals from the lowest index on: key[i] of lane's value i, 0 for none.
template <int P, typename K>
__device__ __forceinline__ Chosen in_rounds(K (&key)[P], const float (&l)[P], int k, int lane) {
    Chosen c = {-1, lane, 0, 0.f, false};
    for (int j = 0; j < k; ++j) {
        K best = 0;
#pragma unroll
        for (int i = 0; i < P; ++i) best = key[i] > best ? key[i] : best;
        best = wave_max(best);
        if (best == 0) break;
        uint32_t at = ~0u;
#pragma unroll
        for (int i = P - 1; i >= 0; --i) at = key[i] == best ? (uint32_t)Row<P>::at(lane, i) : at;
        at = wave_min(at);
        uint32_t v = 0;
#pragma unroll
        for (int i = 0; i < P; ++i)
            if (at == (uint32_t)Row<P>::at(lane, i)) {
                v = __float_as_uint(l[i]);
                key[i] = 0;
            }
        v = __shfl(v, (int)at / Row<P>::V % 64, 64);
        if (lane == j) c.id = (int)at, c.l = __uint_as_float(v), c.has = true;
        ++c.n;
    }
    return c;
}

// Values above `from` (a key, at least 1), one to a lane: their keys and experts.  How many there are; more than 64: none is
// moved.
template <int P>
__device__ __forceinline__ int gather_above(const uint32_t (&key)[P], uint32_t from, uint64_t* lds, int lane, uint32_t& mine, int& id) {
    uint64_t who[P];
    int n = 0;
#pragma unroll
    for (int i = 0; i < P; ++i) {
        who[i] = __ballot(key[i] >= from);
        n += __popcll(who[i]);
    }
    if (n > 64) return n;
    int base = 0;
#pragma unroll
    for (int i = 0; i < P; ++i) {
        if (who[i] == 0) continue;
        const int to = base + __builtin_amdgcn_mbcnt_hi((uint32_t)(who[i] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who[i], 0));
        if (key[i] >= from) lds[to] = (uint64_t)key[i] << 32 | (uint32_t)Row<P>::at(lane, i);
        base += __popcll(who[i]);
    }
    wave_lds_fence();
    const uint64_t v = lane < n ? lds[lane] : 0;
    wave_lds_fence();
    mine = (uint32_t)(v >> 32);
    id = (int)(uint32_t)v;
    return n;
}

// A key not above the k-th largest of the lanes' keys, and so not above the k-th largest of all; at least 1.
__device__ __forceinline__ uint32_t not_above_kth(uint32_t lane_max, int k) {
    uint32_t from = 0;
#pragma unroll
    for (int bit = 31; bit >= 16; --bit) {
        const uint32_t c = from | 1u << bit;
        if (__popcll(__ballot(lane_max >= c)) >= k) from = c;
    }
    return from ? from : 1u;
}

// The softmax's sum in 64 bits.
template <int P>
__device__ __forceinline__ double exact_sum(const float (&l)[P], float top) {
    double sum = 0;
#pragma unroll
    for (int i = 0; i < P; ++i) {
        sum += l[i] == l[i] ? exp_below((double)l[i], (double)top) : 0.0;
        __builtin_amdgcn_sched_barrier(0);                                     // one at a time: registers before speed, here
    }
    return lanes::wave_sum_f64(sum);
}

__device__ __forceinline__ double exact_score(const RouteArgs& a, double l, float top, double sum) {
    return a.sigmoid ? sigmoid(l) : exp_below(l, (double)top) / sum;
}

// The values of a lane that W lanes, or a mirror of the W next, are between: fit for sums and maxima over 16 lanes.
template <int W>
__device__ __forceinline__ float partner(float v) { return __uint_as_float(lanes::partner<W>(__float_as_uint(v))); }
template <int W>
__device__ __forceinline__ double partner(double v) { return lanes::partner_f64<W>(v); }

// With L = 2^group_shift, the values of group g are lanes g L .. g L + L - 1's to look through.  first: the largest of those in LDS,
// and for group_best = 2 the second largest added, in all of its lanes.  size: the magnitudes of those that are finite.
template <typename F>
__device__ __forceinline__ F best_of_group(const RouteArgs& a, const F* lds, int lane, F& size) {
    const int per = a.group_size, L = 1 << a.group_shift, g = lane >> a.group_shift;
    F first = -(F)kInf, second = first;
    auto least = [](F x, F y) { return x < y ? x : y; };
    auto most = [](F x, F y) { return x > y ? x : y; };
    if (g < a.n_group)
        for (int i = lane & (L - 1); i < per; i += L) {
            const F v = lds[g * per + i];
            second = most(second, least(v, first));
            first = most(first, v);
        }
    auto merge = [&](F f, F s) {
        second = most(most(second, s), least(first, f));
        first = most(first, f);
    };
    if (L > 1) merge(partner<1>(first), partner<1>(second));
    if (L > 2) merge(partner<2>(first), partner<2>(second));
    if (L > 4) merge(partner<4>(first), partner<4>(second));
    if (L > 8) merge(partner<8>(first), partner<8>(second));
    for (int d = 16; d < L; d <<= 1) merge(__shfl_xor(first, d, 64), __shfl_xor(second, d, 64));
    const bool both = a.group_best > 1 && second > -(F)kInf;
    const F f = first < 0 ? -first : first, s = second < 0 ? -second : second;
    size = f < (F)kInf ? f : 0;
    if (!both) return first;
    if (!(f < (F)kInf && s < (F)kInf)) return first + second;
    // the sum of two finite values is more than no value, and less than an infinite one, also where 32 bits do not hold it
    const F limit = sizeof(F) == 4 ? (F)0x1.fffffep127f : (F)kInf;
    size = least(f + s, limit);
    return least(most(first + second, -limit), limit);
}

// Experts of the groups that stay keep their keys.  value[i]: what the groups are compared by, -inf for experts that are never
// chosen; err: a bound of its score's error.  The group's own magnitudes bound the rounding of its sums: an expert that a bias of
// -1e9 keeps out leaves the others' bounds alone.  Where that does not decide, the values in 64 bits do.
template <int P>
__device__ __forceinline__ void keep_groups(const RouteArgs& a, const float (&l)[P], float top, const float (&value)[P], float err,
                                            bool exact, double* lds, int lane, uint32_t (&key)[P]) {
    const int shift = a.group_shift, g = lane >> shift;
    const bool one = g < a.n_group && g << shift == lane;
    float* lds32 = (float*)lds;
#pragma unroll
    for (int i = 0; i < P; ++i) lds32[Row<P>::at(lane, i)] = value[i];
    wave_lds_fence();
    float size;
    const float v = best_of_group(a, (const float*)lds32, lane, size);
    wave_lds_fence();
    int before = 0;
    for (int h = 0; h < a.n_group; ++h) {
        const float o = lane_value(v, h << shift);
        before += o > v || (o == v && h < g);
    }
    bool stays = one && before < a.topk_group;
    if (!exact) {
        const float off = (float)a.group_best * err + size * 0x1p-21f;
        const float least = -wave_max(stays ? off - v : -kInf), most = wave_max(one && !stays ? v + off : -kInf);
        if (most > -kInf && !(least > most)) {
            const double sum = a.sigmoid ? 0.0 : exact_sum<P>(l, top);
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const int e = Row<P>::at(lane, i);
                double c = exact_score(a, (double)l[i], top, sum);
                if (a.bias && e < a.n_exp) c += (double)a.bias[e];
                lds[e] = key[i] == 0 ? -(double)kInf : c;
                __builtin_amdgcn_sched_barrier(0);
            }
            wave_lds_fence();
            double none;
            const double w = best_of_group(a, (const double*)lds, lane, none);
            wave_lds_fence();
            before = 0;
            for (int h = 0; h < a.n_group; ++h) {
                const double o = __shfl(w, h << shift, 64);
                before += o > w || (o == w && h < g);
            }
            stays = one && before < a.topk_group;
        }
    }
    const uint64_t kept = __ballot(stays);
#pragma unroll
    for (int i = 0; i < P; ++i)
        if (!(kept >> ((Row<P>::at(lane, i) * a.group_div >> 20 << shift) & 63) & 1)) key[i] = 0;
}

// The k largest of more than 64 sums of a score and a bias that 32 bits do not tell apart, in 64 bits and k rounds.  key: 0 for
// experts that are out.
template <int P>
__device__ __forceinline__ Chosen exact_rounds(const RouteArgs& a, const float (&l)[P], float top, const uint32_t (&key)[P], int lane) {
    const double sum = a.sigmoid ? 0.0 : exact_sum<P>(l, top);
    uint64_t key64[P];
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const int e = Row<P>::at(lane, i);
        key64[i] = key[i] ? order_key(exact_score(a, (double)l[i], top, sum) + (double)a.bias[e < a.n_exp ? e : 0]) : 0;
        __builtin_amdgcn_sched_barrier(0);
    }
    return in_rounds<P>(key64, l, a.k, lane);
}

// GENERAL: a bias or groups.
template <int P, bool GENERAL>
__global__ __launch_bounds__(kRouteThreads) void k_route(RouteArgs a) {
    __shared__ double lds_all[kRouteWaves][GENERAL && P > 1 ? 64 * P : 64];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    double* lds = lds_all[wv];
    const int64_t t = (int64_t)blockIdx.x * kRouteWaves + wv;
    if (t >= a.n_tok) return;
    float l[P];
    Row<P>::read(a.logits, t * a.ld, a.dtype, a.n_exp, a.wide, lane, l);
    bool nan = false;
    float top = -kInf, sum = 0.f;
#pragma unroll
    for (int i = 0; i < P; ++i) {
        nan |= l[i] != l[i];
    }
    nan = __any(nan);
    if (!a.sigmoid && (!a.renorm || GENERAL)) {
#pragma unroll
        for (int i = 0; i < P; ++i) top = fmaxf(top, l[i]);
        top = wave_max(top);
        // (__expf: 16384 x 512 13.0 us, weights 6.1e-8 of their norm from 64 bits; expf 14.9 and 5.2e-8)
#pragma unroll
        for (int i = 0; i < P; ++i) sum += l[i] == top ? 1.f : l[i] > -kInf ? __expf(l[i] - top) : 0.f;
        sum = lanes::group_sum<64>(sum);
    }
    uint32_t key[P];
    float s_top = 0.f, s_err = 0.f;
    if constexpr (GENERAL) {
        float value[P];
        const float inv = 1.f / sum;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int e = Row<P>::at(lane, i);
            const bool in = l[i] > -kInf;
            float s = 0.f;
            if (a.bias || a.group_best > 1) {
                s = a.sigmoid ? __builtin_amdgcn_rcpf(1.f + __expf(-l[i])) : (l[i] == top ? 1.f : __expf(l[i] - top)) * inv;
                s_top = fmaxf(s_top, in ? s : 0.f);
            }
            float c = l[i];
            if (a.bias) c = in ? s + a.bias[e] : -kInf;
            key[i] = order_key(c);
            value[i] = key[i] == 0 ? -kInf : a.bias || a.group_best == 1 ? c : s;
        }
        s_top = wave_max(s_top);
        // an exponential's argument x is rounded, which its value shows |x| times: at most 0.4 of what x exp(-x) can be (times 1 - s
        // in a sigmoid); the sums and functions around it, of s itself.  The sum with a bias adds half a step of its own.
        s_err = ((a.sigmoid ? 8.f : 24.f) * s_top + 0.4f) * 0x1p-22f;
        if (a.n_group > 1) keep_groups<P>(a, l, top, value, s_err, !a.bias && a.group_best == 1, lds, lane, key);
    } else {
#pragma unroll
        for (int i = 0; i < P; ++i) key[i] = order_key(l[i]);
    }
    Chosen c;
    uint32_t lane_max = key[0];
#pragma unroll
    for (int i = 1; i < P; ++i) lane_max = key[i] > lane_max ? key[i] : lane_max;
    uint32_t from = not_above_kth(lane_max, a.k);
    if (GENERAL && a.bias && from > 1) {
        // what may be above it in truth: a value further below is also larger in magnitude, by no more than it is further, so the
        // threshold's own magnitude bounds both roundings
        const float at = order_value(from);
        const uint32_t lower = fabsf(at) < kInf ? order_key(at - (4 * s_err + fabsf(at) * 0x1p-21f)) : from;
        from = lower ? lower : 1u;
    }
    uint32_t mine;
    c.n = gather_above<P>(key, from, (uint64_t*)lds, lane, mine, c.id);
    c.has = lane < c.n;
    c.place = 0;
    if (c.n > 64) {
        if (GENERAL && a.bias) c = exact_rounds<P>(a, l, top, key, lane);
        else c = in_rounds<P>(key, l, a.k, lane);
    } else if (GENERAL && a.bias) {
        const float v = order_value(mine);
        // (the candidates' magnitudes: the others do not meet here)
        const float off = 2 * (s_err + wave_max(c.has && fabsf(v) < kInf ? fabsf(v) : 0.f) * 0x1p-23f);
        int near = 0;                                                          // within both bounds of this lane's, itself among them
        for (int j = 0; j < c.n; ++j) {
            const float o = lane_value(v, j);
            c.place += o > v;
            near += !(fabsf(o - v) > off);
        }
        float b = 0.f;
        c.l = 0.f;
        if (c.has) {
            c.l = read_one(a.logits, t * a.ld + c.id, a.dtype);
            b = a.bias[c.id];
        }
        const bool close = c.has && near > 1;
        if (__any(close)) {
            const double all = a.sigmoid ? 0.0 : exact_sum<P>(l, top);             // (by every lane, before any condition)
            const uint64_t key64 = c.has ? order_key(exact_score(a, (double)c.l, top, all) + (double)b) : 0;
            c.place = 0;
            for (int j = 0; j < c.n; ++j) {
                const uint64_t o = (uint64_t)lane_value((uint32_t)(key64 >> 32), j) << 32 | lane_value((uint32_t)key64, j);
                c.place += o > key64 || (o == key64 && (int)lane_value((uint32_t)c.id, j) < c.id);
            }
        }
    } else {
        const uint64_t own = (uint64_t)mine << 32 | (uint32_t)~c.id;
        for (int j = 0; j < c.n; ++j) c.place += ((uint64_t)lane_value(mine, j) << 32 | lane_value((uint32_t)~c.id, j)) > own;
        c.l = order_value(mine);
    }
    c.has = c.has && c.place < a.k;
    float w;
    if (a.renorm) w = renormalised(a.sigmoid, c.l, c.has);
    else if (a.sigmoid) w = sigmoid(c.l);
    else w = exp_below(c.l, top) / sum;
    int id = c.id, place = c.place;
    bool write = c.has;
    if (!c.has && lane >= c.n && lane < a.k) {
        write = true;
        id = -1;
        place = lane;
        w = 0.f;
    }
    if (write) {
        a.ids[t * a.k + place] = id;
        a.weights[t * a.k + place] = nan ? __builtin_nanf("") : id < 0 ? 0.f : w * a.scale;
    }
}

// A wave per token; the places' values meet their experts in LDS, and the row leaves in whole pieces: 8192 tokens of 512, plain
// softmax, fp32, 9.6 us (34 MB at 3.5 TB/s, the vector unit 63% busy; every logit's exponential), 15.4 with a comparison of each
// expert with each place instead.
template <int P>
__global__ __launch_bounds__(kRouteThreads) void k_route_grad(RouteGradArgs a) {
    constexpr int V = Row<P>::V;
    __shared__ __attribute__((aligned(16))) float lds_all[kRouteWaves][64 * P];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    float* lds = lds_all[wv];
    typedef float fv __attribute__((ext_vector_type(V)));
    const int64_t t = (int64_t)blockIdx.x * kRouteWaves + wv;
    if (t >= a.n_tok) return;
    const bool all = !a.sigmoid && !a.renorm;
    float x[P];
    if (all) Row<P>::read(a.logits, t * a.ld, a.dtype, a.n_exp, a.wide, lane, x);
    int id = -1;
    float l = -kInf, g = 0.f;
    if (lane < a.k) {
        id = a.ids[t * a.k + lane];
        if ((uint32_t)id >= (uint32_t)a.n_exp) id = -1;
        if (id >= 0) {
            l = read_one(a.logits, t * a.ld + id, a.dtype);
            g = a.scale * a.dweights[t * a.k + lane];
        }
    }
#pragma unroll
    for (int c = 0; c < P / V; ++c) *(fv*)(lds + Row<P>::at(lane, c * V)) = (fv)(0.f);
    float v, dot = 0.f;
    if (all) {
        float top = -kInf, sum = 0.f;
#pragma unroll
        for (int i = 0; i < P; ++i) top = fmaxf(top, x[i]);
        top = wave_max(top);
        // (__expf: 8192 x 512 9.5 us, 7.1e-8 of the norm from 64 bits; expf 10.4 and 6.5e-8)
#pragma unroll
        for (int i = 0; i < P; ++i) sum += x[i] = x[i] == -kInf ? 0.f : x[i] == top ? 1.f : __expf(x[i] - top);
        sum = lanes::group_sum<64>(sum);
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
        for (int i = 0; i < P; ++i) x[i] *= inv;
        v = g;
        dot = lanes::group_sum<64>(id >= 0 ? exp_below(l, top) * inv * g : 0.f);
    } else if (a.renorm) {
        const float p = renormalised(a.sigmoid, l, id >= 0);
        v = p * (g - lanes::group_sum<64>(id >= 0 ? p * g : 0.f));
        if (a.sigmoid) v *= sigmoid(-l);
    } else {
        v = sigmoid(l) * sigmoid(-l) * g;
    }
    // places of one expert add up, in their order, and all write the sum
    float add = 0.f;
    for (int j = 0; j < a.k; ++j) {
        const int oid = (int)lane_value((uint32_t)id, j);
        const float o = lane_value(v, j);
        add += oid == id ? o : 0.f;
    }
    wave_lds_fence();
    if (id >= 0) lds[id] = add;
    wave_lds_fence();
#pragma unroll
    for (int c = 0; c < P / V; ++c) {
        const fv d = *(const fv*)(lds + Row<P>::at(lane, c * V));
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float& o = x[c * V + i];
            if (all) o *= d[i] - dot;
            else o = d[i];
        }
    }
    Row<P>::write(a.dlogits, t * a.ldd, a.dtype, a.n_exp, a.wide_out, lane, x);
}

// Whether rows at a step of ld elements of the type may be read a lane's adjacent values at a time.
bool wide_rows(const void* p, int64_t ld, int dtype, int v) {
    const int size = dtype == 2 ? 4 : 2;
    return (uintptr_t)p % (v * size) == 0 && ld % v == 0;
}

// The values per lane: 1, 2, 4, 8 or 16.
template <typename L>
int by_width(int n_exp, const L& launch) {
    if (n_exp <= 64) return launch(std::integral_constant<int, 1>());
    if (n_exp <= 128) return launch(std::integral_constant<int, 2>());
    if (n_exp <= 256) return launch(std::integral_constant<int, 4>());
    if (n_exp <= 512) return launch(std::integral_constant<int, 8>());
    return launch(std::integral_constant<int, 16>());
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

// Launches as many times as the tokens need, each with its own rows.
template <typename A, typename L>
int launch_tokens(A a, int64_t logit_bytes, int64_t out_bytes, const L& launch) {
    for (int64_t left = a.n_tok; left > 0; left -= kRouteMost) {
        a.n_tok = (int)(left < kRouteMost ? left : kRouteMost);
        launch(a, dim3((uint32_t)((a.n_tok + kRouteWaves - 1) / kRouteWaves)));
        HIP_TRY(hipGetLastError());
        a.logits = (const char*)a.logits + kRouteMost * logit_bytes;
        a.ids += (int64_t)kRouteMost * a.k;
        if constexpr (std::is_same<A, RouteArgs>::value) {
            a.weights += (int64_t)kRouteMost * a.k;
        } else {
            a.dweights += (int64_t)kRouteMost * a.k;
            a.dlogits = (char*)a.dlogits + kRouteMost * out_bytes;
        }
    }
    return 0;
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
    const hipStream_t s = (hipStream_t)stream;
    return by_width(n_exp, [&](auto width) {
        constexpr int P = decltype(width)::value;
        RouteArgs a = {logits, bias, ids, weights, ld, n_tok, n_exp, k, n_group, topk_group, group_best, dtype, score, renorm};
        a.wide = wide_rows(logits, ld, dtype, Row<P>::V);
        a.group_size = n_exp / n_group;
        while (n_group << (a.group_shift + 1) <= 64) ++a.group_shift;
        a.group_div = (1u << 20) / (uint32_t)(n_exp / n_group) + 1;
        a.scale = scale;
        return launch_tokens(a, ld * (dtype == 2 ? 4 : 2), 0, [&](const RouteArgs& part, dim3 grid) {
            if (bias || n_group > 1) hipLaunchKernelGGL((k_route<P, true>), grid, dim3(kRouteThreads), 0, s, part);
            else hipLaunchKernelGGL((k_route<P, false>), grid, dim3(kRouteThreads), 0, s, part);
        });
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
    const hipStream_t s = (hipStream_t)stream;
    return by_width(n_exp, [&](auto width) {
        constexpr int P = decltype(width)::value;
        RouteGradArgs a = {logits, ids, dweights, dlogits, ld, ldd, n_tok, n_exp, k, dtype, score, renorm};
        a.wide = wide_rows(logits, ld, dtype, Row<P>::V);
        a.wide_out = wide_rows(dlogits, ldd, dtype, Row<P>::V);
        a.scale = scale;
        const int size = dtype == 2 ? 4 : 2;
        return launch_tokens(a, ld * size, ldd * size, [&](const RouteGradArgs& part, dim3 grid) {
            hipLaunchKernelGGL((k_route_grad<P>), grid, dim3(kRouteThreads), 0, s, part);
        });
    });
}
