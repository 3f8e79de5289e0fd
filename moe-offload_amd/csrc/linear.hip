// A projection that all tokens share (the router, a shared expert), with what surrounds it in the same launch, and its
// gradients:
//     z = x W^T + bias,   y = act(z) + residual        (bias and residual may be absent; z is kept where it is asked for)
//     dz = dy act'(z),    dx = dz W,   dW = dz^T x,   dbias = the sum of dz over the tokens
// act: none, silu, gelu (z times the normal distribution's integral) or the squared relu.  x, W, bias, residual and z are
// fp16 or bf16, y too or fp32, sums and everything between a load and a store fp32.  The products are the grouped
// products' kernels (grouped_mm.hip) over one segment of all tokens; this file has the entry points and dz.
//
// dz is rounded to the inputs' type before the matrix unit takes it, unless it is dy as it came: half a step of each
// value, the same as that of the products' own results, and independent from value to value.
#include "grouped_mm.h"
#include "lane_reduce.h"

namespace {

using namespace gmm;

constexpr int kDzThreads = 256;
constexpr int kDzRows = 64;                // tokens of a block, of 256 columns

struct DzArgs {
    const void* dy;
    const void* z;               // null: dz = dy
    void* dz;                    // null: only the sums
    float* sums;                 // [row blocks][n], null: none wanted
    int64_t lddy, ldz;
    int n_rows, n, act;
};

// A thread has 8 columns of every eighth row of its block; the rows' sums meet in LDS.
template <typename T, bool F32>
__global__ __launch_bounds__(kDzThreads) void k_linear_dz(DzArgs a) {
    __shared__ f32x4 part[8][32][2];
    const int t = threadIdx.x, u = t & 31, sub = t >> 5, c = (blockIdx.x * 32 + u) * 8;
    const int r0 = (int)blockIdx.y * kDzRows;
    f32x4 sum[2] = {};
    if (c < a.n) {
        for (int i = sub; i < kDzRows && r0 + i < a.n_rows; i += 8) {
            const int64_t r = r0 + i;
            f32x4 d[2];
            if constexpr (F32) {
                d[0] = *(const f32x4*)((const float*)a.dy + r * a.lddy + c);
                d[1] = *(const f32x4*)((const float*)a.dy + r * a.lddy + c + 4);
            } else {
                const uint4 v = *(const uint4*)((const T*)a.dy + r * a.lddy + c);
                d[0] = widen4<T>(make_uint2(v.x, v.y));
                d[1] = widen4<T>(make_uint2(v.z, v.w));
            }
            if (a.z) {
                const uint4 v = *(const uint4*)((const T*)a.z + r * a.ldz + c);
                const f32x4 z0 = widen4<T>(make_uint2(v.x, v.y)), z1 = widen4<T>(make_uint2(v.z, v.w));
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    d[0][e] *= slope(a.act, z0[e]);
                    d[1][e] *= slope(a.act, z1[e]);
                }
            }
            if (a.dz) {
                const uint2 lo = round4<T>(d[0]), hi = round4<T>(d[1]);
                *(uint4*)((T*)a.dz + r * a.n + c) = make_uint4(lo.x, lo.y, hi.x, hi.y);
            }
            sum[0] += d[0];
            sum[1] += d[1];
        }
    }
    if (!a.sums) return;
    part[sub][u][0] = sum[0];
    part[sub][u][1] = sum[1];
    __syncthreads();
    if (sub == 0 && c < a.n) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            f32x4 s = part[0][u][h];
            for (int i = 1; i < 8; ++i) s += part[i][u][h];
            *(f32x4*)(a.sums + (int64_t)blockIdx.y * a.n + c + h * 4) = s;
        }
    }
}

template <typename T>
__global__ __launch_bounds__(64) void k_linear_db(const float* __restrict__ sums, int blocks, int n, T* __restrict__ db) {
    const int c = blockIdx.x * 64 + threadIdx.x;
    if (c >= n) return;
    float s = 0.f;
    for (int b = 0; b < blocks; ++b) s += sums[(int64_t)b * n + c];
    db[c] = (T)s;
}

bool bad_matrix(const char* who, const char* name, const void* p, int64_t ld, int64_t width, int64_t rows) {
    if (ld % 8 || (rows > 1 && ld < width) || ld < 0) {
        moe_set_error("%s: %s: rows of %lld elements at a step of %lld (a multiple of 8 wanted)", who, name, (long long)width, (long long)ld);
        return true;
    }
    if (rows > 0 && (!p || (uintptr_t)p % 16)) {
        moe_set_error("%s: %s: null or not 16-byte aligned", who, name);
        return true;
    }
    return false;
}

bool bad_sizes(const char* who, int n_tok, int n_in, int n_out, int act, int dtype) {
    if (n_tok < 0 || n_tok > kMaxSide || n_in < 8 || n_in % 8 || n_in > kMaxSide || n_out < 8 || n_out % 8 || n_out > kMaxSide ||
        act < kActNone || act > kActRelu2 || (dtype != 0 && dtype != 1)) {
        moe_set_error("%s: n_tok=%d n_in=%d n_out=%d (multiples of 8, up to 2^30) act=%d (0 none, 1 silu, 2 gelu, 3 squared relu) "
                      "dtype=%d (0 fp16, 1 bf16)", who, n_tok, n_in, n_out, act, dtype);
        return true;
    }
    return false;
}

uint64_t round_up(uint64_t v) { return (v + 255) / 256 * 256; }

int row_blocks(int n_tok) { return (int)(((int64_t)n_tok + kDzRows - 1) / kDzRows); }

template <typename T>
int launch_dz(const DzArgs& a, int dy_f32, void* db, hipStream_t s) {
    const int blocks = row_blocks(a.n_rows), cols = (a.n + 255) / 256;
    if (blocks > 0) {
        const dim3 grid(cols, blocks);
        if (dy_f32) hipLaunchKernelGGL((k_linear_dz<T, true>), grid, dim3(kDzThreads), 0, s, a);
        else hipLaunchKernelGGL((k_linear_dz<T, false>), grid, dim3(kDzThreads), 0, s, a);
        HIP_TRY(hipGetLastError());
    }
    if (db) {
        hipLaunchKernelGGL((k_linear_db<T>), dim3((a.n + 63) / 64), dim3(64), 0, s, a.sums, blocks, a.n, (T*)db);
        HIP_TRY(hipGetLastError());
    }
    return 0;
}

}  // namespace

extern "C" int moe_linear(const void* x, int64_t ldx, const void* w, const void* bias, const void* residual, int64_t ldr, int n_tok,
                          int n_in, int n_out, int act, int dtype, int out_f32, void* z, int64_t ldz, void* y, int64_t ldy,
                          void* stream) {
    const char* who = "linear";
    if (bad_sizes(who, n_tok, n_in, n_out, act, dtype) || bad_matrix(who, "x", x, ldx, n_in, n_tok) ||
        bad_matrix(who, "w", w, n_in, n_in, n_out) || (bias && bad_matrix(who, "bias", bias, n_out, n_out, 1)) ||
        (residual && bad_matrix(who, "residual", residual, ldr, n_out, n_tok)) ||
        (z && bad_matrix(who, "z", z, ldz, n_out, n_tok)) || bad_matrix(who, "y", y, ldy, n_out, n_tok))
        return -1;
    if (n_tok == 0) return 0;
    const Linear l = {x, w, bias, residual, y, z, ldx, ldr, ldy, ldz, n_tok, n_out, n_in, act, out_f32};
    return gmm::linear(l, dtype, (hipStream_t)stream);
}

extern "C" uint64_t moe_linear_grad_workspace_bytes(int n_tok, int n_out, int act, int dy_f32, int want_db) {
    if (n_tok < 0 || n_out < 0) return 0;
    const uint64_t dz = act != kActNone || dy_f32 ? round_up(2 * (uint64_t)n_tok * n_out) : 0;
    return dz + (want_db ? 4 * (uint64_t)row_blocks(n_tok) * n_out : 0);
}

extern "C" int moe_linear_grad(const void* dy, int64_t lddy, int dy_f32, const void* x, int64_t ldx, const void* w, const void* z,
                               int64_t ldz, int n_tok, int n_in, int n_out, int act, int dtype, void* workspace, void* dx, void* dw,
                               int dw_f32, void* db, void* stream) {
    const char* who = "linear_grad";
    const hipStream_t s = (hipStream_t)stream;
    const bool own_dz = act != kActNone || dy_f32;
    if (bad_sizes(who, n_tok, n_in, n_out, act, dtype) || bad_matrix(who, "dy", dy, lddy, n_out, n_tok) ||
        (act != kActNone && bad_matrix(who, "z", z, ldz, n_out, n_tok)) || (dw && bad_matrix(who, "x", x, ldx, n_in, n_tok)) ||
        (dx && (bad_matrix(who, "w", w, n_in, n_in, n_out) || bad_matrix(who, "dx", dx, n_in, n_in, n_tok))) ||
        (dw && bad_matrix(who, "dw", dw, n_in, n_in, n_out)))
        return -1;
    if (moe_linear_grad_workspace_bytes(n_tok, n_out, act, dy_f32, db != nullptr) > 0 && (!workspace || (uintptr_t)workspace % 16)) {
        moe_set_error("linear_grad: the workspace is null or not 16-byte aligned");
        return -1;
    }
    if (row_blocks(n_tok) > 65535) {
        moe_set_error("linear_grad: n_tok=%d (up to %d)", n_tok, 65535 * kDzRows);
        return -1;
    }
    void* dz = own_dz && (dx || dw) ? workspace : nullptr;
    const void* rows = own_dz ? dz : dy;
    const int64_t ld = own_dz ? n_out : lddy;
    // what one launch does not take is refused before anything is queued
    auto dx_of = [&](bool dry) { return !dx || n_tok == 0 ? 0 : linear_dx(rows, ld, w, dx, n_tok, n_out, n_in, dtype, dry, s); };
    auto dw_of = [&](bool dry) { return !dw ? 0 : linear_dw(rows, ld, x, ldx, dw, n_tok, n_out, n_in, dw_f32, dtype, dry, s); };
    if (dx_of(true) || dw_of(true)) return -1;
    if (dz || db) {
        const uint64_t skip = own_dz ? round_up(2 * (uint64_t)n_tok * n_out) : 0;
        const DzArgs a = {dy, act != kActNone ? z : nullptr, dz, db ? (float*)((char*)workspace + skip) : nullptr, lddy, ldz, n_tok, n_out, act};
        if (dtype ? launch_dz<__bf16>(a, dy_f32, db, s) : launch_dz<_Float16>(a, dy_f32, db, s)) return -1;
    }
    return dx_of(false) || dw_of(false) ? -1 : 0;
}
