// Row plan of a batch on the GPU: the (token, k) expert ids, flattened, in a stable order by expert.
//
// With ids e_p of the pairs p = token * k + j, row r of the plan is the pair order[r], where order sorts
// the pairs by (e_p, p); row_out[r] = order[r], row_token[r] = order[r] / k, and segment e is rows
// seg_start[e] .. seg_start[e + 1] - 1.  Ids outside 0 .. n_exp - 1 (a padded token, a dropped pair) are
// one class of their own behind the last segment.  The host does the same in prefill.resident_plan
// (mlx-qwen38/loader.py:583-591), after a copy of the ids to the host.
//
// A counting sort: each wave counts the ids of its own contiguous part of the pairs in a table of its
// own, one pass over the tables turns the counts into first rows, and the waves go through their parts
// again, 64 pairs at a time in order.  A pair's row is its class's running row of this wave plus the
// number of equal ids in lower lanes, from one ballot per bit of the id.  No atomic's order shows: the
// counting atomics add to integers of which only the sums are read.
#include "moe_common.h"

namespace {

constexpr int kPlanWaves = 16;
constexpr int kPlanThreads = 64 * kPlanWaves;
constexpr int kPlanMaxExp = 1024;

__device__ __forceinline__ int id_class(int id, int n_exp) { return (unsigned)id < (unsigned)n_exp ? id : n_exp; }

__global__ __launch_bounds__(kPlanThreads) void k_expert_plan(const int32_t* __restrict__ ids, int n_ids, int k, int n_exp,
                                                              int bits, int32_t* __restrict__ row_token,
                                                              int32_t* __restrict__ row_out,
                                                              int32_t* __restrict__ seg_start) {
    __shared__ int hist[kPlanWaves * (kPlanMaxExp + 1)];
    __shared__ int wave_total[kPlanWaves];
    const int t = threadIdx.x, lane = t & 63, wv = __builtin_amdgcn_readfirstlane(t >> 6);
    const int classes = n_exp + 1;
    for (int i = t; i < kPlanWaves * classes; i += kPlanThreads) hist[i] = 0;
    __syncthreads();
    const int batches = (n_ids - 1) / 64 + 1, per = (batches + kPlanWaves - 1) / kPlanWaves;
    const int b0 = wv * per, b1 = b0 + per < batches ? b0 + per : batches;
    int* mine = hist + wv * classes;
    for (int b = b0; b < b1; ++b) {
        const int p = b * 64 + lane;
        if (p < n_ids) atomicAdd(&mine[id_class(ids[p], n_exp)], 1);
    }
    __syncthreads();
    // counts -> first rows: thread c takes classes c and c + 1024
    int sum = 0;
    if (t < classes)
        for (int w = 0; w < kPlanWaves; ++w) sum += hist[w * classes + t];
    int inc = sum;
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(inc, d, 64);
        if (lane >= d) inc += o;
    }
    if (lane == 63) wave_total[wv] = inc;
    __syncthreads();
    int first = inc - sum;
    for (int w = 0; w < wv; ++w) first += wave_total[w];
    if (t < classes) {
        seg_start[t] = first;
        int run = first;
        for (int w = 0; w < kPlanWaves; ++w) {
            const int c = hist[w * classes + t];
            hist[w * classes + t] = run;
            run += c;
        }
    }
    if (t == kPlanThreads - 1 && classes > kPlanThreads) {
        // 1024 experts: the class of the ids outside them is one more than there are threads
        int run = first + sum;
        seg_start[n_exp] = run;
        for (int w = 0; w < kPlanWaves; ++w) {
            const int c = hist[w * classes + n_exp];
            hist[w * classes + n_exp] = run;
            run += c;
        }
    }
    __syncthreads();
    for (int b = b0; b < b1; ++b) {
        const int p = b * 64 + lane;
        const bool in = p < n_ids;
        const int c = in ? id_class(ids[p], n_exp) : 0;
        uint64_t same = __ballot(in);
        for (int i = 0; i < bits; ++i) {
            const uint64_t v = __ballot((c >> i) & 1);
            same &= ((c >> i) & 1) ? v : ~v;
        }
        const int below = __popcll(same & ((1ull << lane) - 1ull));
        const int row = in ? mine[c] + below : 0;
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (in && below == 0) mine[c] = row + __popcll(same);
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (in) {
            row_out[row] = p;
            row_token[row] = p / k;
        }
    }
}

}  // namespace

extern "C" int moe_expert_plan(const int32_t* ids, int n_ids, int k, int n_exp, int32_t* row_token, int32_t* row_out,
                               int32_t* seg_start, void* stream) {
    if (n_ids < 0 || k <= 0 || n_ids % k || n_exp < 1 || n_exp > kPlanMaxExp) {
        moe_set_error("expert_plan: n_ids=%d must be a multiple of k=%d, n_exp=%d in 1..%d", n_ids, k, n_exp, kPlanMaxExp);
        return -1;
    }
    if (!seg_start || (n_ids > 0 && (!ids || !row_token || !row_out))) {
        moe_set_error("expert_plan: null pointer");
        return -1;
    }
    int bits = 0;
    while ((n_exp >> bits) != 0) ++bits;
    hipLaunchKernelGGL(k_expert_plan, dim3(1), dim3(kPlanThreads), 0, (hipStream_t)stream, ids, n_ids, k, n_exp, bits,
                       row_token, row_out, seg_start);
    HIP_TRY(hipGetLastError());
    return 0;
}
