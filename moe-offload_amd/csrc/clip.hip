// The norm of a step's gradients, and the gradients scaled to at most a given norm:
//     norm = sqrt(sum of g^2 over all tensors),    out = g min(1, max_norm / (norm + 1e-6))
// Tensors are fp16, bf16 or fp32 in any mixture, of any length, starting anywhere.  Squares are summed in 64 bits (one of
// 1e20 has no square in 32), each block's part kept apart and the parts added in their order, so a call's result has
// the same bits every time.
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

// Calls f(i, whole) for this thread's groups of kPer elements of a chunk: elements i .. i + kPer - 1 of the range, of which
// some lie outside 0 .. n - 1 where whole is false.
template <typename T, typename F>
__device__ __forceinline__ void for_chunk(const Range& r, uint32_t chunk, const F& f) {
    const int64_t skew = ((uintptr_t)r.p % 16) / sizeof(T);
    const int64_t from = (int64_t)chunk * kChunk - skew;
#pragma unroll 4
    for (int j = 0; j < kChunk / (kPer<T> * kClipThreads); ++j) {
        const int64_t i = from + (int64_t)(j * kClipThreads + threadIdx.x) * kPer<T>;
        if (i >= r.n || i <= -kPer<T>) continue;
        f(i, i >= 0 && i + kPer<T> <= r.n);
    }
}

template <typename T>
__device__ __forceinline__ double squares(const Range& r, uint32_t chunk) {
    typedef T tv __attribute__((ext_vector_type(kPer<T>)));
    double sum = 0;
    for_chunk<T>(r, chunk, [&](int64_t i, bool whole) {
        const T* p = (const T*)r.p + i;
        if (whole) {
            const tv v = *(const tv*)p;
#pragma unroll
            for (int e = 0; e < kPer<T>; ++e) sum += (double)(float)v[e] * (double)(float)v[e];
        } else {
            for (int e = 0; e < kPer<T>; ++e)
                if (i + e >= 0 && i + e < r.n) sum += (double)(float)p[e] * (double)(float)p[e];
        }
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

__global__ __launch_bounds__(kClipThreads) void k_clip_squares(Table t, double* __restrict__ sums) {
    __shared__ double scratch[kClipThreads / 64];
    const int i = range_of(t, blockIdx.x);
    const uint32_t chunk = blockIdx.x - t.first[i];
    const int type = t.type[i];
    const double v = type == 0 ? squares<_Float16>(t.range[i], chunk)
                     : type == 1 ? squares<__bf16>(t.range[i], chunk) : squares<float>(t.range[i], chunk);
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
    typedef T tv __attribute__((ext_vector_type(kPer<T>)));
    const bool aligned = ((uintptr_t)r.p - (uintptr_t)r.out) % 16 == 0;
    for_chunk<T>(r, chunk, [&](int64_t i, bool whole) {
        const T* p = (const T*)r.p + i;
        T* o = (T*)r.out + i;
        if (whole && aligned) {
            tv v = *(const tv*)p;
#pragma unroll
            for (int e = 0; e < kPer<T>; ++e) v[e] = (T)((float)v[e] * f);
            *(tv*)o = v;
        } else {
            for (int e = 0; e < kPer<T>; ++e)
                if (i + e >= 0 && i + e < r.n) o[e] = (T)((float)p[e] * f);
        }
    });
}

__global__ __launch_bounds__(kClipThreads) void k_clip_scale(Table t, const float* __restrict__ factor) {
    const float f = *factor;
    const int i = range_of(t, blockIdx.x);
    const Range r = t.range[i];
    if (f == 1.f && r.p == r.out) return;
    const uint32_t chunk = blockIdx.x - t.first[i];
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

// Whether something is written where something else is read or written.
bool overlap(int n, const void* const* grads, void* const* outs, const int64_t* sizes, const int32_t* types) {
    struct Span { uintptr_t a, b; bool out; };
    std::vector<Span> spans;
    spans.reserve(2 * (size_t)n);
    for (int i = 0; i < n; ++i) {
        if (sizes[i] == 0) continue;
        const uintptr_t bytes = (uintptr_t)sizes[i] * size_of(types[i]), g = (uintptr_t)grads[i], o = (uintptr_t)outs[i];
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
    // ranges of neighbours in memory are one
    struct Item { Range r; int type; };
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
    double* sums = (double*)((char*)workspace + kHead);
    float* factor = (float*)workspace;
    auto launches = [&](auto&& launch) {
        Table t;
        t.n = 0;
        t.first[0] = 0;
        uint64_t before = 0;
        auto flush = [&]() {
            if (t.n == 0) return hipSuccess;
            launch(t, before);
            before += t.first[t.n];
            t.n = 0;
            return hipGetLastError();
        };
        constexpr uint64_t kMost = 1u << 23;                                   // blocks of a launch (2^31 threads)
        for (const Item& it : items) {
            // a range of more chunks than a launch takes is cut at a chunk's end, where its address is aligned
            Range r = it.r;
            while (r.n > 0) {
                const int64_t skew = ((uintptr_t)r.p % 16) / size_of(it.type);
                const uint64_t room = kMost - t.first[t.n], want = chunks_of(r.p, r.n, it.type), have = std::min(room, want);
                const int64_t take = have == want ? r.n : (int64_t)have * kChunk - skew;
                t.range[t.n] = {r.p, r.out, take};
                t.type[t.n] = (uint8_t)it.type;
                t.first[t.n + 1] = t.first[t.n] + (uint32_t)have;
                ++t.n;
                r.p = (const char*)r.p + take * size_of(it.type);
                if (r.out) r.out = (char*)r.out + take * size_of(it.type);
                r.n -= take;
                if (t.n == kTable || t.first[t.n] == kMost)
                    if (const hipError_t e = flush()) return e;
            }
        }
        return flush();
    };
    uint64_t chunks = 0;
    HIP_TRY(launches([&](const Table& t, uint64_t before) {
        hipLaunchKernelGGL(k_clip_squares, dim3(t.first[t.n]), dim3(kClipThreads), 0, s, t, sums + before);
        chunks = before + t.first[t.n];
    }));
    hipLaunchKernelGGL(k_clip_norm, dim3(1), dim3(1024), 0, s, sums, (int64_t)chunks, max_norm, factor, norm);
    HIP_TRY(hipGetLastError());
    if (!outs) return 0;
    HIP_TRY(launches([&](const Table& t, uint64_t) {
        hipLaunchKernelGGL(k_clip_scale, dim3(t.first[t.n]), dim3(kClipThreads), 0, s, t, factor);
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
        if (outs && overlap(n, grads, outs, sizes, types)) {
            moe_set_error("clip_grads: what is written overlaps another tensor");
            return -1;
        }
        return clip(n, grads, outs, sizes, types, max_norm, workspace, norm, (hipStream_t)stream);
    } catch (const std::exception& e) {
        moe_set_error("clip_grads: %s", e.what());
        return -1;
    }
}
