// Matrix products of sorted rows by their experts' unquantised weights (fp16 or bf16), with gradients.
//
// Segment u covers the sorted rows r in [seg_start[u], seg_start[u + 1]) and uses W_u = w[seg_slot[u]]
// ([n][k]; slot u where seg_slot is null):
//     mm       y[row_out[r]]  = s_u  W_u   x[row_in[r]]
//     gate_up  h[r]           = silu(g) * u,  (g, u) = W_u x[row_in[r]]   (W_u: inter gate rows, inter up rows)
//     mm_dx    dx[row_out[r]] = s_u  W_u^T dy[row_in[r]]
//       with gu, the (g, u) of a gate_up whose h the product W_u took:  the gradient of (g, u) instead,
//       dg = dh u sig(g) (1 + g (1 - sig(g))),  du = dh g sig(g),  dh = s_u W_u^T dy[row_in[r]]
//     mm_dw    dW_u           = s_u  sum over r of u of  dy[row_dy[r]] x[row_x[r]]^T      (no rows: zeros)
// Sums in fp32 (MFMA), one rounding to the output's type at the end.  The reference multiplies its sorted
// rows by 2-bit experts only (mlx-qwen38/prefill_qproj.py:18-40); these are the same products for the
// weights before quantisation.
//
// All four are one tile product  out[p][q] = sum over c of P[p][c] Q[q][c]  with q the direction in which
// the output is contiguous; an operand is either contiguous in c (x, dy; W for mm) or has its c along the
// rows of memory (W for mm_dx, both operands for mm_dw).  The matrix unit takes Q as its first operand,
// so a lane of the result holds four adjacent q of one p.
#include <hip/hip_bf16.h>

#include "grouped_mm.h"

namespace {

using gmm::Segs;
using gmm::Tile;

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

enum { kMM = 0, kGateUp = 1, kDx = 2, kDxGlu = 3, kDw = 4 };

struct Args {
    Segs S;
    const void* p;               // rows (x, or dy)
    const void* q;               // weights, or x for the weights' gradient
    void* out;
    const int32_t* row_p;
    const int32_t* row_q;
    const int32_t* row_out;
    const float* scale;
    const void* gu;              // mm_dx: the pre-activations
    void* gu_out;                // gate_up: where they go (may be null)
    int64_t ldp, ldq, ldo, ldgu; // elements from row to row; ldq from slot to slot where q is weights; ldo of mm_dw likewise
    int n_p, n_q, n_out;         // rows of p, q and out that exist
    int np, nq, nc;              // extents: output columns in p (mm_dw) and q, and the contraction
    int out_f32;
};

template <typename T>
__device__ __forceinline__ f32x4 mfma(uint4 a, uint4 b, f32x4 c) {
    if constexpr (__is_same(T, _Float16))
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

template <typename T>
__device__ __forceinline__ uint2 round4(const float* v) {
    typedef T t4 __attribute__((ext_vector_type(4)));
    const t4 r = {(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
    return __builtin_bit_cast(uint2, r);
}

template <typename T>
__device__ __forceinline__ void widen4(uint2 w, float* v) {
    typedef T t4 __attribute__((ext_vector_type(4)));
    const t4 r = __builtin_bit_cast(t4, w);
    for (int i = 0; i < 4; ++i) v[i] = (float)r[i];
}

constexpr int kBP = 64, kBQ = 64, kBC = 32, kLd = kBC + 8;

template <typename T, int OP>
__global__ __launch_bounds__(256) void k_grouped(Args a) {
    __shared__ __attribute__((aligned(16))) uint16_t lp[kBP * kLd];
    __shared__ __attribute__((aligned(16))) uint16_t lq[kBQ * kLd];
    const int t = threadIdx.x, lane = t & 63, wv = t >> 6;
    const int qstep = OP == kGateUp ? kBQ / 2 : kBQ;          // output columns of a tile
    const int inter = a.nq;                                    // gate_up, and mm_dx with gu
    int r0, r1, slot, q0, p0 = 0, nc = a.nc, seg = 0;
    if constexpr (OP == kDw) {
        const int tq = (a.nq + kBQ - 1) / kBQ, tp = (a.np + kBP - 1) / kBP;
        const uint32_t item = gmm::xcd_order(blockIdx.x, gridDim.x);
        seg = item / (tq * tp);
        p0 = (int)(item / tq % tp) * kBP;
        q0 = (int)(item % tq) * kBQ;
        Segs S = a.S;
        gmm::seg_rows(S, seg + 1, r0, r1, slot);
        nc = r1 - r0;
    } else {
        Tile tile;
        if (!gmm::find_tile<256>(a.S, kBP, (a.nq + qstep - 1) / qstep, tile)) return;
        r0 = tile.r0;
        r1 = tile.r1;
        slot = tile.slot;
        q0 = tile.col * qstep;
        if (slot < 0) nc = 0;
    }
    const T* P = (const T*)a.p;
    const T* Q = (const T*)a.q;
    if constexpr (OP != kDw) Q += (int64_t)(slot < 0 ? 0 : slot) * a.ldq;

    // this thread's 16 bytes of each operand per step
    const int crow = t >> 2, cch = (t & 3) * 8;                // contiguous in c: row, first c
    const int trow = t >> 3, tch = (t & 7) * 8;                // c along the rows: c, first column
    const T* prow = nullptr;
    const T* qrow = nullptr;
    if constexpr (OP != kDw) {
        const int r = r0 + crow;
        if (r < r1) {
            const int v = a.row_p ? a.row_p[r] : r;
            if (v >= 0 && v < a.n_p) prow = P + (int64_t)v * a.ldp;
        }
    }
    if constexpr (OP == kMM) {
        if (q0 + crow < a.nq) qrow = Q + (int64_t)(q0 + crow) * a.nc;
    }
    if constexpr (OP == kGateUp) {
        // the tile's 64 weight rows: per wave column 16 gate rows, then the 16 up rows of the same outputs
        const int c = q0 + (crow >> 5) * 16 + (crow & 15);
        if (c < inter) qrow = Q + (int64_t)(c + ((crow >> 4) & 1) * inter) * a.nc;
    }
    const uint4 zero = make_uint4(0, 0, 0, 0);
    f32x4 acc[2][2] = {};
    const int wp = (wv >> 1) * 32, wq = (wv & 1) * 32, n = lane & 15, kq = lane >> 4;
    for (int c0 = 0; c0 < nc; c0 += kBC) {
        uint4 vp = zero, vq = zero;
        if constexpr (OP == kDw) {
            const int r = r0 + c0 + trow;
            if (r < r1) {
                const int v = a.row_p ? a.row_p[r] : r, x = a.row_q ? a.row_q[r] : r;
                if (v >= 0 && v < a.n_p && x >= 0 && x < a.n_q) {
                    if (p0 + tch < a.np) vp = *(const uint4*)(P + (int64_t)v * a.ldp + p0 + tch);
                    if (q0 + tch < a.nq) vq = *(const uint4*)(Q + (int64_t)x * a.ldq + q0 + tch);
                }
            }
        } else {
            if (prow && c0 + cch < nc) vp = *(const uint4*)(prow + c0 + cch);
            if constexpr (OP == kDx || OP == kDxGlu) {
                if (c0 + trow < nc && q0 + tch < a.nq) vq = *(const uint4*)(Q + (int64_t)(c0 + trow) * a.nq + q0 + tch);
            } else {
                if (qrow && c0 + cch < nc) vq = *(const uint4*)(qrow + c0 + cch);
            }
        }
        __syncthreads();
        auto put = [&](uint16_t* l, uint4 v, bool along) {
            if (along) {
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int i = 0; i < 8; ++i) l[(tch + i) * kLd + trow] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
            } else {
                *(uint4*)(l + crow * kLd + cch) = v;
            }
        };
        put(lp, vp, OP == kDw);
        put(lq, vq, OP >= kDx);
        __syncthreads();
        uint4 fp[2], fq[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            fp[i] = *(const uint4*)(lp + (wp + i * 16 + n) * kLd + kq * 8);
            fq[i] = *(const uint4*)(lq + (wq + i * 16 + n) * kLd + kq * 8);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) acc[i][j] = mfma<T>(fq[j], fp[i], acc[i][j]);
    }
    const float s = a.scale && slot >= 0 ? a.scale[slot] : 1.0f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int m = wp + i * 16 + n;
        if constexpr (OP == kDw) {
            if (p0 + m >= a.np) continue;
            for (int j = 0; j < 2; ++j) {
                const int q = q0 + wq + j * 16 + kq * 4;
                if (q >= a.nq) continue;
                float v[4];
                for (int e = 0; e < 4; ++e) v[e] = acc[i][j][e] * s;
                const int64_t at = (int64_t)seg * a.ldo + (int64_t)(p0 + m) * a.nq + q;
                if (a.out_f32) *(float4*)((float*)a.out + at) = make_float4(v[0], v[1], v[2], v[3]);
                else *(uint2*)((T*)a.out + at) = round4<T>(v);
            }
            continue;
        }
        const int r = r0 + m;
        if (r >= r1) continue;
        if constexpr (OP == kGateUp) {
            const int c = q0 + (wv & 1) * 16 + kq * 4;
            if (c >= inter) continue;
            float g[4], u[4], h[4];
            for (int e = 0; e < 4; ++e) {
                g[e] = acc[i][0][e];
                u[e] = acc[i][1][e];
                h[e] = g[e] / (1.0f + __expf(-g[e])) * u[e];
            }
            *(uint2*)((T*)a.out + (int64_t)r * a.ldo + c) = round4<T>(h);
            if (a.gu_out) {
                *(uint2*)((T*)a.gu_out + (int64_t)r * a.ldgu + c) = round4<T>(g);
                *(uint2*)((T*)a.gu_out + (int64_t)r * a.ldgu + inter + c) = round4<T>(u);
            }
        } else {
            const int o = a.row_out ? a.row_out[r] : r;
            if (o < 0 || o >= a.n_out) continue;
            for (int j = 0; j < 2; ++j) {
                const int q = q0 + wq + j * 16 + kq * 4;
                if (q >= a.nq) continue;
                float v[4];
                for (int e = 0; e < 4; ++e) v[e] = acc[i][j][e] * s;
                T* d = (T*)a.out + (int64_t)o * a.ldo + q;
                if constexpr (OP == kDxGlu) {
                    float g[4], u[4], dg[4], du[4];
                    const T* gr = (const T*)a.gu + (int64_t)r * a.ldgu + q;
                    widen4<T>(*(const uint2*)gr, g);
                    widen4<T>(*(const uint2*)(gr + inter), u);
                    for (int e = 0; e < 4; ++e) {
                        const float sg = 1.0f / (1.0f + __expf(-g[e]));
                        dg[e] = slot < 0 ? 0.f : v[e] * u[e] * sg * (1.0f + g[e] * (1.0f - sg));
                        du[e] = slot < 0 ? 0.f : v[e] * g[e] * sg;
                    }
                    *(uint2*)d = round4<T>(dg);
                    *(uint2*)(d + inter) = round4<T>(du);
                } else {
                    *(uint2*)d = round4<T>(v);
                }
            }
        }
    }
}

template <typename T, int OP>
int launch(const Args& a, hipStream_t s) {
    uint64_t blocks;
    if constexpr (OP == kDw) {
        blocks = (uint64_t)a.S.n_seg * ((a.nq + kBQ - 1) / kBQ) * ((a.np + kBP - 1) / kBP);
    } else {
        const int qstep = OP == kGateUp ? kBQ / 2 : kBQ;
        const uint64_t segs = (uint64_t)(a.S.n_seg + 2 < a.S.n_rows ? a.S.n_seg + 2 : a.S.n_rows);
        blocks = ((uint64_t)a.S.n_rows / kBP + segs) * ((a.nq + qstep - 1) / qstep);
    }
    if (blocks > 0x7FFFFFFFu) {
        moe_set_error("grouped product: %llu tiles are more than one launch takes", (unsigned long long)blocks);
        return -1;
    }
    hipLaunchKernelGGL((k_grouped<T, OP>), dim3((uint32_t)blocks), dim3(256), 0, s, a);
    HIP_TRY(hipGetLastError());
    return 0;
}

template <int OP>
int launch_typed(const Args& a, int dtype, hipStream_t s) {
    return dtype ? launch<__bf16, OP>(a, s) : launch<_Float16, OP>(a, s);
}

bool bad(const char* who, const char* what) {
    moe_set_error("%s: %s", who, what);
    return true;
}

// Whether a matrix of `rows` rows may be read or written in 16-byte pieces of `width` elements.
bool bad_matrix(const char* who, const char* name, const void* p, int64_t ld, int64_t width, int64_t rows, int dtype_bytes) {
    if (rows < 0 || width <= 0 || width % 8 || ld % 8 || (rows > 1 && ld < width) || ld < 0) {
        moe_set_error("%s: %s: %lld rows of %lld elements at a step of %lld (multiples of 8 wanted)", who, name,
                      (long long)rows, (long long)width, (long long)ld);
        return true;
    }
    if (rows > 0 && (!p || (uintptr_t)p % 16)) {
        moe_set_error("%s: %s: null or not 16-byte aligned", who, name);
        return true;
    }
    (void)dtype_bytes;
    return false;
}

bool bad_segs(const char* who, const Segs& S, int dtype, const void* w) {
    if (dtype != 0 && dtype != 1) return bad(who, "dtype is 0 (fp16) or 1 (bf16)");
    if (S.n_seg < 0 || S.n_seg > gmm::kMaxSeg || S.n_rows < 0 || S.n_slots < 0) {
        moe_set_error("%s: n_seg=%d (0..%d) n_rows=%d n_slots=%d", who, S.n_seg, gmm::kMaxSeg, S.n_rows, S.n_slots);
        return true;
    }
    if (!S.start) return bad(who, "seg_start is null");
    if (S.n_slots > 0 && !w) return bad(who, "no weights");
    return false;
}

}  // namespace

extern "C" {

int moe_grouped_mm(const void* x, int64_t ldx, int n_x, const int32_t* row_in, const int32_t* seg_start,
                   const int32_t* seg_slot, int n_seg, int n_rows, const void* w, int64_t w_stride, int n_slots, int n,
                   int k, const float* scale, void* y, int64_t ldy, int n_y, const int32_t* row_out, int dtype, int fill,
                   void* stream) {
    const char* who = "grouped_mm";
    Args a = {};
    a.S = Segs{seg_start, seg_slot, n_seg, n_rows, n_slots, fill};
    if (bad_segs(who, a.S, dtype, w) || bad_matrix(who, "x", x, ldx, k, n_x, 2) ||
        bad_matrix(who, "w", w, w_stride, k, n_slots, 2) || bad_matrix(who, "y", y, ldy, n, n_y, 2))
        return -1;
    if (n_slots > 1 && w_stride < (int64_t)n * k) return bad(who, "w_stride is less than a matrix"), -1;
    if ((!row_in && n_rows > n_x) || (!row_out && n_rows > n_y)) return bad(who, "more rows than x or y has"), -1;
    if (n_rows == 0 || n_y == 0) return 0;
    a.p = x, a.q = w, a.out = y, a.row_p = row_in, a.row_out = row_out, a.scale = scale;
    a.ldp = ldx, a.ldq = w_stride, a.ldo = ldy, a.n_p = n_x, a.n_out = n_y, a.nq = n, a.nc = k;
    return launch_typed<kMM>(a, dtype, (hipStream_t)stream);
}

int moe_grouped_gate_up(const void* x, int64_t ldx, int n_x, const int32_t* row_in, const int32_t* seg_start,
                        const int32_t* seg_slot, int n_seg, int n_rows, const void* w, int64_t w_stride, int n_slots,
                        int inter, int hidden, void* h, int64_t ldh, void* gu, int64_t ldgu, int dtype, int fill,
                        void* stream) {
    const char* who = "grouped_gate_up";
    Args a = {};
    a.S = Segs{seg_start, seg_slot, n_seg, n_rows, n_slots, fill};
    if (bad_segs(who, a.S, dtype, w) || bad_matrix(who, "x", x, ldx, hidden, n_x, 2) ||
        bad_matrix(who, "w", w, w_stride, hidden, n_slots, 2) || bad_matrix(who, "h", h, ldh, inter, n_rows, 2) ||
        (gu && bad_matrix(who, "gu", gu, ldgu, 2 * (int64_t)inter, n_rows, 2)))
        return -1;
    if (inter > 0x3FFFFFFF) return bad(who, "inter is too large"), -1;
    if (n_slots > 1 && w_stride < 2 * (int64_t)inter * hidden) return bad(who, "w_stride is less than a matrix"), -1;
    if (!row_in && n_rows > n_x) return bad(who, "more rows than x has"), -1;
    if (n_rows == 0) return 0;
    a.p = x, a.q = w, a.out = h, a.row_p = row_in, a.gu_out = gu;
    a.ldp = ldx, a.ldq = w_stride, a.ldo = ldh, a.ldgu = ldgu, a.n_p = n_x, a.n_out = n_rows, a.nq = inter, a.nc = hidden;
    return launch_typed<kGateUp>(a, dtype, (hipStream_t)stream);
}

int moe_grouped_mm_dx(const void* dy, int64_t lddy, int n_dy, const int32_t* row_in, const int32_t* seg_start,
                      const int32_t* seg_slot, int n_seg, int n_rows, const void* w, int64_t w_stride, int n_slots, int n,
                      int k, const float* scale, const void* gu, int64_t ldgu, void* dx, int64_t lddx, int n_dx,
                      const int32_t* row_out, int dtype, int fill, void* stream) {
    const char* who = "grouped_mm_dx";
    Args a = {};
    a.S = Segs{seg_start, seg_slot, n_seg, n_rows, n_slots, fill};
    if (bad_segs(who, a.S, dtype, w) || bad_matrix(who, "dy", dy, lddy, n, n_dy, 2) ||
        bad_matrix(who, "w", w, w_stride, k, n_slots, 2) ||
        bad_matrix(who, "dx", dx, lddx, (gu ? 2 : 1) * (int64_t)k, n_dx, 2) ||
        (gu && bad_matrix(who, "gu", gu, ldgu, 2 * (int64_t)k, n_rows, 2)))
        return -1;
    if (n_slots > 1 && w_stride < (int64_t)n * k) return bad(who, "w_stride is less than a matrix"), -1;
    if ((!row_in && n_rows > n_dy) || (!row_out && n_rows > n_dx)) return bad(who, "more rows than dy or dx has"), -1;
    if (n_rows == 0 || n_dx == 0) return 0;
    a.p = dy, a.q = w, a.out = dx, a.row_p = row_in, a.row_out = row_out, a.scale = scale, a.gu = gu;
    a.ldp = lddy, a.ldq = w_stride, a.ldo = lddx, a.ldgu = ldgu, a.n_p = n_dy, a.n_out = n_dx, a.nq = k, a.nc = n;
    return gu ? launch_typed<kDxGlu>(a, dtype, (hipStream_t)stream) : launch_typed<kDx>(a, dtype, (hipStream_t)stream);
}

int moe_grouped_mm_dw(const void* dy, int64_t lddy, int n_dy, const int32_t* row_dy, const void* x, int64_t ldx, int n_x,
                      const int32_t* row_x, const int32_t* seg_start, int n_seg, int n_rows, int n, int k,
                      const float* scale, void* dw, int64_t dw_stride, int out_f32, int dtype, void* stream) {
    const char* who = "grouped_mm_dw";
    Args a = {};
    a.S = Segs{seg_start, nullptr, n_seg, n_rows, n_seg, 0};
    if (bad_segs(who, a.S, dtype, dw) || bad_matrix(who, "dy", dy, lddy, n, n_dy, 2) ||
        bad_matrix(who, "x", x, ldx, k, n_x, 2) || bad_matrix(who, "dw", dw, dw_stride, k, n_seg, out_f32 ? 4 : 2))
        return -1;
    if (n_seg > 1 && dw_stride < (int64_t)n * k) return bad(who, "dw_stride is less than a matrix"), -1;
    if ((!row_dy && n_rows > n_dy) || (!row_x && n_rows > n_x)) return bad(who, "more rows than dy or x has"), -1;
    if (n_seg == 0) return 0;
    a.p = dy, a.q = x, a.out = dw, a.row_p = row_dy, a.row_q = row_x, a.scale = scale;
    a.ldp = lddy, a.ldq = ldx, a.ldo = dw_stride, a.n_p = n_dy, a.n_q = n_x, a.np = n, a.nq = k, a.out_f32 = out_f32;
    return launch_typed<kDw>(a, dtype, (hipStream_t)stream);
}

}  // extern "C"
