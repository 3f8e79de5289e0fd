// The norm of a step's gradients, and the gradients scaled to at most a given norm:
//     norm = sqrt(sum of g^2 over all tensors),    out = g min(1, max_norm / (norm + 1e-6))
// Tensors are fp16, bf16 or fp32 in any mixture, of any length, starting anywhere.  Squares are summed in 64 bits (one of
// 1e20 has no square in 32), each block's part kept apart and the parts added in their order, so a call's result has
// the same bits every time.
//
// Memory bounds it: 806 MB of bf16 129 us for the squares (6.2 TB/s), 270 for the scaling into other buffers (6.0 TB/s both ways).
// The gradients are read twice, as the factor is known only once all of them have been.
//
// Three launches: the blocks' sums of squares, their sum with the factor, the scaling.  What the kernels know of the tensors
// comes with the launch itself (a table of up to kTable ranges; a longer list takes several launches), so that nothing on
// the host has to outlive the call and a captured graph holds it all.
#include <algorithm>
#include <new>
#include <vector>

#include "lane_reduce.h"
#include "moe_common.h"

namespace {

constexpr int kTable = 96;                 // ranges of a launch: the table stays below the 4 KiB that a launch's arguments have
constexpr int kClipThreads = 256;
constexpr int kChunk = 16384;              // elements of a block
constexpr uint32_t kMostChunks = 1u << 23; // of a launch (2^31 threads)
// Blocks of a launch of the squares, eight per CU, each with a sum: one block adds 24,600 sums in 10 us, these in 4.7.
constexpr uint32_t kSquareBlocks = 2048;
constexpr int kHead = 16;                  // bytes of the workspace before the blocks' sums: the factor

struct Range {
    const void* p;
    void* out;
    int64_t n;                             // elements
};

// Range r has the launch's chunks first[r] .. first[r + 1] - 1.  Its chunks start at the 16-byte line that its first element
// lies in.
struct Table {
    Range range[kTable];
    uint32_t first[kTable + 1];
    uint8_t type[kTable];
    int n;
};

__device__ __forceinline__ int range_of(const Table& t, uint32_t chunk) {
    int lo = 0, hi = t.n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (t.first[mid] <= chunk) lo = mid;
        else hi = mid;
    }
    return lo;
}

template <typename T>
constexpr int kPer = 16 / (int)sizeof(T);

// Calls f(values, i, from, to) for this thread's groups of kPer elements i .. i + kPer - 1 of a chunk, of which from .. to - 1
// (counted from i) are the range's.  A chunk that is the range's as a whole is loaded at once.
template <typename T, typename F>
__device__ __forceinline__ void for_chunk(const Range& r, uint32_t chunk, const F& f) {
    typedef T tv __attribute__((ext_vector_type(kPer<T>)));
    constexpr int kGroups = kChunk / (kPer<T> * kClipThreads), kAtOnce = 8;
    const int64_t skew = ((uintptr_t)r.p % 16) / sizeof(T), first = (int64_t)chunk * kChunk - skew;
    const int64_t i0 = first + (int64_t)threadIdx.x * kPer<T>;
    if (first >= 0 && first + kChunk <= r.n) {
        const tv* p = (const tv*)((const T*)r.p + i0);
#pragma unroll
        for (int j0 = 0; j0 < kGroups; j0 += kAtOnce) {
            tv v[kAtOnce];
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j) v[j] = p[(j0 + j) * kClipThreads];
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j) f(v[j], i0 + (int64_t)(j0 + j) * kClipThreads * kPer<T>, 0, kPer<T>);
        }
        return;
    }
    for (int j = 0; j < kGroups; ++j) {
        const int64_t i = i0 + (int64_t)j * kClipThreads * kPer<T>;
        const int from = i < 0 ? (int)(i > -kPer<T> ? -i : kPer<T>) : 0, to = i + kPer<T> <= r.n ? kPer<T> : i < r.n ? (int)(r.n - i) : 0;
        if (from >= to) continue;
        tv v = {};
        if (from == 0 && to == kPer<T>) {
            v = *(const tv*)((const T*)r.p + i);
        } else {
#pragma unroll
            for (int e = 0; e < kPer<T>; ++e)
                if (e >= from && e < to) v[e] = ((const T*)r.p)[i + e];
        }
        f(v, i, from, to);
    }
}

template <typename T>
__device__ __forceinline__ double squares(const Range& r, uint32_t chunk) {
    double sum = 0;
    for_chunk<T>(r, chunk, [&](auto v, int64_t, int, int) {                    // (zeros where the range has none)
#pragma unroll
        for (int e = 0; e < kPer<T>; ++e) sum += (double)(float)v[e] * (double)(float)v[e];
    });
    return sum;
}

__device__ __forceinline__ double block_sum(double v, double* scratch) {
    v = lanes::wave_sum_f64(v);
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
    for (int w = 0; w < (int)blockDim.x / 64; ++w) v += scratch[w];
    return v;
}

__global__ __launch_bounds__(kClipThreads) void k_clip_squares(Table t, uint32_t chunks, double* __restrict__ sums) {
    __shared__ double scratch[kClipThreads / 64];
    double v = 0;
    for (uint32_t c = blockIdx.x; c < chunks; c += gridDim.x) {
        const int i = range_of(t, c);
        const uint32_t chunk = c - t.first[i];
        const int type = t.type[i];
        v += type == 0 ? squares<_Float16>(t.range[i], chunk)
             : type == 1 ? squares<__bf16>(t.range[i], chunk) : squares<float>(t.range[i], chunk);
    }
    const double sum = block_sum(v, scratch);
    if (threadIdx.x == 0) sums[blockIdx.x] = sum;
}

__global__ __launch_bounds__(1024) void k_clip_norm(const double* __restrict__ sums, int64_t n, double max_norm, float* __restrict__ factor,
                                                    float* __restrict__ norm) {
    __shared__ double scratch[16];
    double v = 0;
    for (int64_t i = threadIdx.x; i < n; i += 1024) v += sums[i];
    v = block_sum(v, scratch);
    if (threadIdx.x == 0) {
        const double root = sqrt(v), f = max_norm / (root + 1e-6);
        *norm = (float)root;
        *factor = f >= 1.0 ? 1.f : (float)f;                                   // (a NaN stays one)
    }
}

template <typename T>
__device__ __forceinline__ void scale(const Range& r, uint32_t chunk, float f) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    const bool aligned = ((uintptr_t)r.p - (uintptr_t)r.out) % 16 == 0;
    for_chunk<T>(r, chunk, [&](auto v, int64_t i, int from, int to) {
        T* o = (T*)r.out + i;
#pragma unroll
        for (int e = 0; e < kPer<T>; ++e) v[e] = (T)((float)v[e] * f);
        if (aligned && from == 0 && to == kPer<T>) {
            __builtin_nontemporal_store(__builtin_bit_cast(u32x4, v), (u32x4*)o);
        } else {
#pragma unroll
            for (int e = 0; e < kPer<T>; ++e)
                if (e >= from && e < to) o[e] = v[e];
        }
    });
}

// Chunks from the last to the first: some of what the squares' pass read last is still in the caches (all of a call on 806 MB
// 417 us, and 425 from the first on).
__global__ __launch_bounds__(kClipThreads) void k_clip_scale(Table t, uint32_t chunks, const float* __restrict__ factor) {
    const float f = *factor;
    const uint32_t c = chunks - 1 - blockIdx.x;
    const int i = range_of(t, c);
    const Range r = t.range[i];
    if (f == 1.f && r.p == r.out) return;
    const uint32_t chunk = c - t.first[i];
    const int type = t.type[i];
    if (type == 0) scale<_Float16>(r, chunk, f);
    else if (type == 1) scale<__bf16>(r, chunk, f);
    else scale<float>(r, chunk, f);
}

int size_of(int type) { return type == 2 ? 4 : 2; }

uint64_t chunks_of(const void* p, int64_t n, int type) {
    const uint64_t skew = ((uintptr_t)p % 16) / size_of(type);
    return n > 0 ? (skew + (uint64_t)n + kChunk - 1) / kChunk : 0;
}

struct Item {
    Range r;
    int type;
};

// Whether something is written where something else is read or written.
bool overlap(const std::vector<Item>& items) {
    struct Span { uintptr_t a, b; bool out; };
    std::vector<Span> spans;
    spans.reserve(2 * items.size());
    for (const Item& it : items) {
        const uintptr_t bytes = (uintptr_t)it.r.n * size_of(it.type), g = (uintptr_t)it.r.p, o = (uintptr_t)it.r.out;
        if (g != o) spans.push_back({g, g + bytes, false});
        spans.push_back({o, o + bytes, true});
    }
    std::sort(spans.begin(), spans.end(), [](const Span& x, const Span& y) { return x.a < y.a; });
    uintptr_t all = 0, out = 0;
    for (const Span& s : spans) {
        if (s.a < (s.out ? all : out)) return true;
        all = std::max(all, s.b);
        if (s.out) out = std::max(out, s.b);
    }
    return false;
}

int clip(int n, const void* const* grads, void* const* outs, const int64_t* sizes, const int32_t* types, double max_norm,
         void* workspace, float* norm, hipStream_t s) {
    // Ranges of neighbours in memory are one: gradients that are views of a flat buffer, in its order, need one launch
    // however many they are (384 of them 0.13 ms on the host as ranges of their own, 0.01 as one).
    std::vector<Item> items;
    for (int i = 0; i < n; ++i) {
        if (sizes[i] == 0) continue;
        void* out = outs ? outs[i] : nullptr;
        if (!items.empty()) {
            Item& l = items.back();
            const int64_t bytes = l.r.n * size_of(l.type);
            if (l.type == types[i] && (const char*)l.r.p + bytes == grads[i] && (!outs || (char*)l.r.out + bytes == out)) {
                l.r.n += sizes[i];
                continue;
            }
        }
        items.push_back({{grads[i], out, sizes[i]}, types[i]});
    }
    if (outs && overlap(items)) {
        moe_set_error("clip_grads: what is written overlaps another tensor");
        return -1;
    }
    double* sums = (double*)((char*)workspace + kHead);
    float* factor = (float*)workspace;
    // Calls launch(table, chunks) for as many ranges as one takes at a time.
    auto launches = [&](auto&& launch) {
        Table t;
        t.n = 0;
        t.first[0] = 0;
        auto flush = [&]() {
            if (t.n == 0) return hipSuccess;
            launch(t, t.first[t.n]);
            t.n = 0;
            return hipGetLastError();
        };
        for (const Item& it : items) {
            // a range of more chunks than a launch takes is cut at a chunk's end, where its address is aligned
            Range r = it.r;
            while (r.n > 0) {
                const int64_t skew = ((uintptr_t)r.p % 16) / size_of(it.type);
                const uint64_t room = kMostChunks - t.first[t.n], want = chunks_of(r.p, r.n, it.type), have = std::min(room, want);
                const int64_t take = have == want ? r.n : (int64_t)have * kChunk - skew;
                t.range[t.n] = {r.p, r.out, take};
                t.type[t.n] = (uint8_t)it.type;
                t.first[t.n + 1] = t.first[t.n] + (uint32_t)have;
                ++t.n;
                r.p = (const char*)r.p + take * size_of(it.type);
                if (r.out) r.out = (char*)r.out + take * size_of(it.type);
                r.n -= take;
                if (t.n == kTable || t.first[t.n] == kMostChunks)
                    if (const hipError_t e = flush()) return e;
            }
        }
        return flush();
    };
    int64_t blocks = 0;
    HIP_TRY(launches([&](const Table& t, uint32_t chunks) {
        const uint32_t grid = chunks < kSquareBlocks ? chunks : kSquareBlocks;
        hipLaunchKernelGGL(k_clip_squares, dim3(grid), dim3(kClipThreads), 0, s, t, chunks, sums + blocks);
        blocks += grid;
    }));
    hipLaunchKernelGGL(k_clip_norm, dim3(1), dim3(1024), 0, s, sums, blocks, max_norm, factor, norm);
    HIP_TRY(hipGetLastError());
    if (!outs) return 0;
    HIP_TRY(launches([&](const Table& t, uint32_t chunks) {
        hipLaunchKernelGGL(k_clip_scale, dim3(chunks), dim3(kClipThreads), 0, s, t, chunks, factor);
    }));
    return 0;
}

}  // namespace

extern "C" uint64_t moe_clip_workspace_bytes(int n, int64_t n_elements) {
    // every tensor may end in a chunk of its own, and start in the middle of a 16-byte line
    if (n < 0 || n_elements < 0) return 0;
    return kHead + 8 * ((uint64_t)n_elements / kChunk + 2 * (uint64_t)n + 1);
}

extern "C" int moe_clip_grads(int n, const void* const* grads, void* const* outs, const int64_t* sizes, const int32_t* types,
                              double max_norm, void* workspace, float* norm, void* stream) {
    if (n < 0 || !workspace || (uintptr_t)workspace % 16 || !norm || (n > 0 && (!grads || !sizes || !types))) {
        moe_set_error("clip_grads: n=%d, or a null pointer, or a workspace that is not 16-byte aligned", n);
        return -1;
    }
    if (!(max_norm >= 0)) {
        moe_set_error("clip_grads: max_norm=%g", max_norm);
        return -1;
    }
    for (int i = 0; i < n; ++i) {
        if (types[i] < 0 || types[i] > 2 || sizes[i] < 0 || sizes[i] > ((int64_t)1 << 40)) {
            moe_set_error("clip_grads: tensor %d: type %d (0 fp16, 1 bf16, 2 fp32), %lld elements (up to 2^40)", i, types[i],
                          (long long)sizes[i]);
            return -1;
        }
        const uintptr_t a = (uintptr_t)grads[i], b = outs ? (uintptr_t)outs[i] : a;
        if (sizes[i] > 0 && (!a || !b || (a | b) % size_of(types[i]))) {
            moe_set_error("clip_grads: tensor %d: null or not aligned to its elements", i);
            return -1;
        }
    }
    try {
        return clip(n, grads, outs, sizes, types, max_norm, workspace, norm, (hipStream_t)stream);
    } catch (const std::exception& e) {
        moe_set_error("clip_grads: %s", e.what());
        return -1;
    }
}
