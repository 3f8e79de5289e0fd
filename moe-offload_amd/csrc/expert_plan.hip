// Row plan of a batch on the GPU: the (token, k) expert ids, flattened, in a stable order by expert.
//
// With ids e_p of the pairs p = token * k + j, row r of the plan is the pair order[r], where order sorts
// the pairs by (e_p, p); row_out[r] = order[r], row_token[r] = order[r] / k, and segment e is rows
// seg_start[e] .. seg_start[e + 1] - 1.  Ids outside 0 .. n_exp - 1 (a padded token, a dropped pair) are
// one class of their own behind the last segment.  The host does the same in prefill.resident_plan
// (mlx-qwen38/loader.py:583-591), after a copy of the ids to the host.
//
// A counting sort.  Each wave counts the ids of its own contiguous part of the pairs in a table of its own;
// the counts of all waves before it, of its class, and of all lower classes give its first row; then it
// goes through its part again, 64 pairs at a time in order, and a pair's row is its class's running row of
// this wave plus the number of equal ids in lower lanes, from one ballot per bit of the id.  Its counts
// come from the same ballots, kept in registers for the first 256 pairs: an atomic per pair serialises
// where few experts, or adapters, take most of them (4096 pairs of 8 classes: 14.4 us that way, 6.5 this
// way).  No atomic's order shows: those of k_plan_count add to integers of which only the sums are read.
//
// Up to kPlanOne pairs take one block and one launch (4096 pairs: 6.5 us; as two launches of two blocks 4.0
// and 4.4).  More are dealt to up to kPlanBlocks blocks: a first launch writes each block's counts to the
// workspace, in the second every block adds up the others' itself (a column per thread, so that no third
// launch has to scan them).  The steps' latencies bound it, not its bytes: 640 pairs of 512 experts 4.2 us,
// 163840 pairs 3.1 and 10.5 us (2 MB; with 1024 pairs per block instead of 2048 2.9 and 12.1, with 4096
// 3.3 and 12.5).
#include "moe_common.h"

namespace {

constexpr int kPlanWaves = 16;
constexpr int kPlanThreads = 64 * kPlanWaves;
constexpr int kPlanMaxExp = 1024;
constexpr int kPlanOne = 4096;        // pairs that one block takes alone
constexpr int kPlanBlocks = 256;
constexpr int kPlanHeld = 4;          // batches of a wave whose ids stay in registers between its two passes
constexpr int kPlanPairs = 2048;      // pairs per block, at least, where there are several

__host__ __device__ inline int plan_blocks(int n_ids) {
    if (n_ids <= kPlanOne) return 1;
    const int n = (n_ids - 1) / kPlanPairs + 1;
    return n < kPlanBlocks ? n : kPlanBlocks;
}

__device__ __forceinline__ int id_class(int id, int n_exp) { return (unsigned)id < (unsigned)n_exp ? id : n_exp; }

// The batches of 64 pairs [b0, b1) of one of the grid's waves, numbered in pair order.
__device__ __forceinline__ void wave_part(int n_ids, int wave, int waves, int& b0, int& b1) {
    const int batches = (n_ids - 1) / 64 + 1, per = batches / waves, rest = batches % waves;
    b0 = wave * per + (wave < rest ? wave : rest);
    b1 = b0 + per + (wave < rest ? 1 : 0);
    if (n_ids == 0) b1 = b0;
}

// The lanes with this lane's class: how many of them are lower, and how many there are.
__device__ __forceinline__ void equal_lanes(int c, bool in, int bits, int lane, int& below, int& count) {
    uint64_t same = __ballot(in);
    for (int i = 0; i < bits; ++i) {
        const uint64_t v = __ballot((c >> i) & 1);
        same &= ((c >> i) & 1) ? v : ~v;
    }
    below = __popcll(same & ((1ull << lane) - 1ull));
    count = __popcll(same);
}

__global__ __launch_bounds__(kPlanThreads) void k_plan_count(const int32_t* __restrict__ ids, int n_ids, int n_exp,
                                                             int32_t* __restrict__ counts) {
    __shared__ int hist[kPlanMaxExp + 1];
    const int t = threadIdx.x, lane = t & 63, classes = n_exp + 1;
    for (int i = t; i < classes; i += kPlanThreads) hist[i] = 0;
    __syncthreads();
    int b0, b1;
    wave_part(n_ids, blockIdx.x * kPlanWaves + (t >> 6), gridDim.x * kPlanWaves, b0, b1);
    for (int b = b0; b < b1; ++b) {
        const int64_t p = (int64_t)b * 64 + lane;
        if (p < n_ids) atomicAdd(&hist[id_class(ids[p], n_exp)], 1);
    }
    __syncthreads();
    for (int i = t; i < classes; i += kPlanThreads) counts[(size_t)blockIdx.x * classes + i] = hist[i];
}

__global__ __launch_bounds__(kPlanThreads) void k_plan_place(const int32_t* __restrict__ ids, int n_ids, int k, int n_exp,
                                                             int bits, const int32_t* __restrict__ counts,
                                                             int32_t* __restrict__ row_token, int32_t* __restrict__ row_out,
                                                             int32_t* __restrict__ seg_start) {
    __shared__ int hist[kPlanWaves * (kPlanMaxExp + 1)];
    __shared__ int wave_total[kPlanWaves];
    const int t = threadIdx.x, lane = t & 63, wv = __builtin_amdgcn_readfirstlane(t >> 6);
    const int classes = n_exp + 1;
    for (int i = t; i < kPlanWaves * classes; i += kPlanThreads) hist[i] = 0;
    __syncthreads();
    int b0, b1;
    wave_part(n_ids, blockIdx.x * kPlanWaves + wv, gridDim.x * kPlanWaves, b0, b1);
    int* mine = hist + wv * classes;
    // batch b of this wave: its ids' classes (-1: no pair), and each lane's place among the equal ones
    struct Batch { int c, below, count; };
    auto read = [&](int b) {
        const int64_t p = (int64_t)b * 64 + lane;
        return b < b1 && p < n_ids ? id_class(ids[p], n_exp) : -1;
    };
    auto rank = [&](int id) {
        Batch v;
        v.c = id;
        equal_lanes(id < 0 ? 0 : id, id >= 0, bits, lane, v.below, v.count);
        return v;
    };
    // mine[c] += count by the lowest of the equal lanes; returns what it was
    auto add = [&](const Batch& v) {
        const int was = v.c >= 0 ? mine[v.c] : 0;
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (v.c >= 0 && v.below == 0) mine[v.c] = was + v.count;
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        return was;
    };
    Batch held[kPlanHeld];
#pragma unroll
    for (int i = 0; i < kPlanHeld; ++i) held[i].c = read(b0 + i);
#pragma unroll
    for (int i = 0; i < kPlanHeld; ++i)
        if (b0 + i < b1) {
            held[i] = rank(held[i].c);
            add(held[i]);
        }
    for (int b = b0 + kPlanHeld; b < b1; ++b) add(rank(read(b)));
    // thread c: the pairs of class c in all blocks, and in the blocks before this one
    int all = 0, before = 0;
    if (gridDim.x > 1 && t < classes) {
#pragma unroll 16
        for (int b = 0; b < (int)gridDim.x; ++b) {
            const int c = counts[(size_t)b * classes + t];
            all += c;
            before += b < (int)blockIdx.x ? c : 0;
        }
    }
    __syncthreads();
    if (gridDim.x == 1 && t < classes)
        for (int w = 0; w < kPlanWaves; ++w) all += hist[w * classes + t];
    int inc = all;
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(inc, d, 64);
        if (lane >= d) inc += o;
    }
    if (lane == 63) wave_total[wv] = inc;
    __syncthreads();
    int first = inc - all;
    for (int w = 0; w < wv; ++w) first += wave_total[w];
    auto place = [&](int c, int from, int skip) {
        if (blockIdx.x == 0) seg_start[c] = from;
        int run = from + skip;
        for (int w = 0; w < kPlanWaves; ++w) {
            const int n = hist[w * classes + c];
            hist[w * classes + c] = run;
            run += n;
        }
    };
    if (t < classes) place(t, first, before);
    if (t == kPlanThreads - 1 && classes > kPlanThreads) {
        // 1024 experts: the class of the ids outside them is one more than there are threads
        int skip = 0;
        for (int b = 0; b < (int)blockIdx.x; ++b) skip += counts[(size_t)b * classes + n_exp];
        place(n_exp, first + all, skip);
    }
    __syncthreads();
    auto place_batch = [&](int b, const Batch& v) {
        const int row = add(v) + v.below;
        if (v.c >= 0) {
            const int p = (int)((int64_t)b * 64 + lane);
            row_out[row] = p;
            row_token[row] = p / k;
        }
    };
#pragma unroll
    for (int i = 0; i < kPlanHeld; ++i)
        if (b0 + i < b1) place_batch(b0 + i, held[i]);
    for (int b = b0 + kPlanHeld; b < b1; ++b) place_batch(b, rank(read(b)));
}

}  // namespace

extern "C" uint64_t moe_expert_plan_workspace_bytes(int n_ids, int n_exp) {
    if (n_ids <= 0 || n_exp < 1 || n_exp > kPlanMaxExp || plan_blocks(n_ids) == 1) return 0;
    return (uint64_t)plan_blocks(n_ids) * (n_exp + 1) * 4;
}

extern "C" int moe_expert_plan(const int32_t* ids, int n_ids, int k, int n_exp, void* workspace, int32_t* row_token,
                               int32_t* row_out, int32_t* seg_start, void* stream) {
    if (n_ids < 0 || k <= 0 || n_ids % k || n_exp < 1 || n_exp > kPlanMaxExp) {
        moe_set_error("expert_plan: n_ids=%d must be a multiple of k=%d, n_exp=%d in 1..%d", n_ids, k, n_exp, kPlanMaxExp);
        return -1;
    }
    if (!seg_start || (n_ids > 0 && (!ids || !row_token || !row_out)) ||
        (!workspace && moe_expert_plan_workspace_bytes(n_ids, n_exp) > 0)) {
        moe_set_error("expert_plan: null pointer");
        return -1;
    }
    const hipStream_t s = (hipStream_t)stream;
    const int blocks = plan_blocks(n_ids);
    int bits = 0;
    while ((n_exp >> bits) != 0) ++bits;
    if (blocks > 1) {
        hipLaunchKernelGGL(k_plan_count, dim3(blocks), dim3(kPlanThreads), 0, s, ids, n_ids, n_exp, (int32_t*)workspace);
        HIP_TRY(hipGetLastError());
    }
    hipLaunchKernelGGL(k_plan_place, dim3(blocks), dim3(kPlanThreads), 0, s, ids, n_ids, k, n_exp, bits,
                       (const int32_t*)workspace, row_token, row_out, seg_start);
    HIP_TRY(hipGetLastError());
    return 0;
}
