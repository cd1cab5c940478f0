// Layer norm over the last axis, forward and backward, for fp32 and bf16 rows of up to 32 KB.
//
//   mean = sum_c x / C,  rstd = 1 / sqrt(sum_c (x - mean)^2 / C + eps),  xh = (x - mean) rstd
//   y  = xh w + b
//   g  = dy w
//   dx = rstd (g - sum_c g / C - xh sum_c(g xh) / C),   dw = sum_rows dy xh,   db = sum_rows dy
//
// Replaces the reference's layernorm_forward_kernel (a block per row, tree reduction in shared memory), its
// layernorm_input_grad_kernel and its layernorm_param_grad_kernel, which reads x and dy a second time
// (src/inferno/cuda/cudalayernorm.cu:16-160, 212-400; modules: src/inferno/modules/layernorm.cpp:25-98).
//
// Memory-bound: a row is read once into registers, and everything is computed from there, so the variance is the sum of squared
// differences from the mean and not a difference of two sums.  A row belongs to 32, 128 or 512 threads (LnShape), each of which holds
// up to four 16-byte chunks of it: a row of one warp needs no barrier.  The backward's threads keep their columns from row to row and
// sum dw and db in registers; a block's sums meet in the workspace, which ln_finish_kernel adds up in a fixed order.  All sums are
// fp32; the only rounding to fewer bits is that of the results.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "sm100_ptx.cuh"

namespace ib200 {

struct LnRows {
    const void* x;
    long x_pitch;          // elements from row to row
    const void* dy;        // backward
    long dy_pitch;
    const void* w;         // [C], or null: ones
    const void* b;         // [C], or null: zeros
    int param_bf16;        // type of w and b
    void* out;             // y or dx, dense
    float* mean;           // [M]: written by the forward (or null), read by the backward
    float* rstd;
    float* part;           // backward: dw and db sums of each block, [blocks][2][C], or null
    int M, C;
    float eps;
};

// TPR threads per row, chunks of 16 bytes, NV of them per thread.  ALIGNED: rows begin on 16 bytes and hold whole chunks; a thread's chunk
// is then 16 contiguous bytes.  Otherwise the same columns are dealt out element by element, so that a warp's loads still run together.
template <class T_, int TPR_, int NV_, bool ALIGNED_>
struct LnShape {
    using T = T_;
    static constexpr int TPR = TPR_, NV = NV_, VEC = 16 / sizeof(T_), WARPS = TPR_ / 32;
    static constexpr bool ALIGNED = ALIGNED_;
    static constexpr int THREADS = TPR_ == 32 ? 256 : TPR_, ROWS = THREADS / TPR_;      // per block
    static constexpr int CHUNK_COLS = TPR_ * VEC;                                       // columns of one chunk of all threads
    static constexpr int BWD_BLOCKS = 512 / THREADS;                                    // of the backward, resident per SM
};

__device__ __forceinline__ float ln_to_float(float v) { return v; }
__device__ __forceinline__ float ln_to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void ln_from_float(float v, float& o) { o = v; }
__device__ __forceinline__ void ln_from_float(float v, __nv_bfloat16& o) { o = __float2bfloat16(v); }

// Column of element e of chunk v of thread t; past the row's end: C and more.
template <class S>
__device__ __forceinline__ int ln_col(int v, int e, int t) {
    return S::ALIGNED ? (v * S::TPR + t) * S::VEC + e : v * S::CHUNK_COLS + e * S::TPR + t;
}
__device__ __forceinline__ void ln_unpack(const uint4& u, float (&f)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        f[2 * e] = __uint_as_float(w[e] << 16);
        f[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
    }
}
__device__ __forceinline__ void ln_unpack(const uint4& u, float (&f)[4]) {
    f[0] = __uint_as_float(u.x);
    f[1] = __uint_as_float(u.y);
    f[2] = __uint_as_float(u.z);
    f[3] = __uint_as_float(u.w);
}
// One chunk of a row; zeros past its end.
template <class S>
__device__ __forceinline__ void ln_load(const typename S::T* row, int v, int t, int C, float (&f)[S::VEC]) {
    if constexpr (S::ALIGNED) {
        const int c = ln_col<S>(v, 0, t);
        uint4 u = make_uint4(0, 0, 0, 0);
        if (c < C) u = *reinterpret_cast<const uint4*>(row + c);
        ln_unpack(u, f);
    } else {
#pragma unroll
        for (int e = 0; e < S::VEC; ++e) {
            const int c = ln_col<S>(v, e, t);
            f[e] = c < C ? ln_to_float(row[c]) : 0.f;
        }
    }
}
// The same columns of weight or bias.
template <class S, class P>
__device__ __forceinline__ void ln_load_param_as(const P* p, int v, int t, int C, float (&f)[S::VEC]) {
    if constexpr (S::ALIGNED) {
        const int c = ln_col<S>(v, 0, t);
#pragma unroll
        for (int e = 0; e < S::VEC; ++e) f[e] = 0.f;
        if (c >= C) return;
        if constexpr (sizeof(P) == 4) {
#pragma unroll
            for (int q = 0; q < S::VEC / 4; ++q) {
                const float4 u = *reinterpret_cast<const float4*>(p + c + 4 * q);
                f[4 * q] = u.x; f[4 * q + 1] = u.y; f[4 * q + 2] = u.z; f[4 * q + 3] = u.w;
            }
        } else {
#pragma unroll
            for (int q = 0; q < S::VEC / 4; ++q) {
                const uint2 u = *reinterpret_cast<const uint2*>(p + c + 4 * q);
                f[4 * q] = __uint_as_float(u.x << 16);
                f[4 * q + 1] = __uint_as_float(u.x & 0xffff0000u);
                f[4 * q + 2] = __uint_as_float(u.y << 16);
                f[4 * q + 3] = __uint_as_float(u.y & 0xffff0000u);
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < S::VEC; ++e) {
            const int c = ln_col<S>(v, e, t);
            f[e] = c < C ? ln_to_float(p[c]) : 0.f;
        }
    }
}
template <class S>
__device__ __forceinline__ void ln_load_param(const void* p, int bf16, float none, int v, int t, int C, float (&f)[S::VEC]) {
    if (!p) {
#pragma unroll
        for (int e = 0; e < S::VEC; ++e) f[e] = none;
    } else if (bf16) {
        ln_load_param_as<S>(static_cast<const __nv_bfloat16*>(p), v, t, C, f);
    } else {
        ln_load_param_as<S>(static_cast<const float*>(p), v, t, C, f);
    }
}
template <class S>
__device__ __forceinline__ void ln_store(typename S::T* row, int v, int t, int C, const float (&f)[S::VEC]) {
    if constexpr (S::ALIGNED) {
        const int c = ln_col<S>(v, 0, t);
        if (c >= C) return;
        uint4 u;
        if constexpr (S::VEC == 8) u = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
        else u = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
        *reinterpret_cast<uint4*>(row + c) = u;
    } else {
#pragma unroll
        for (int e = 0; e < S::VEC; ++e) {
            const int c = ln_col<S>(v, e, t);
            if (c < C) ln_from_float(f[e], row[c]);
        }
    }
}

// Sums of a and b over the threads of a row.  `turn` alternates between two sets of slots, so that one barrier per sum is enough: a slot
// is written again only after the next sum's barrier, which every thread reaches after it has read.
template <class S>
__device__ __forceinline__ float2 ln_row_sum(float a, float b, float2 (*slots)[16], int turn) {
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) {
        a += __shfl_xor_sync(0xffffffffu, a, m);
        b += __shfl_xor_sync(0xffffffffu, b, m);
    }
    if constexpr (S::WARPS > 1) {
        float2* s = slots[turn & 1];
        if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = make_float2(a, b);
        __syncthreads();
        a = b = 0.f;
#pragma unroll
        for (int w = 0; w < S::WARPS; ++w) {
            a += s[w].x;
            b += s[w].y;
        }
    }
    return make_float2(a, b);
}

template <class S>
__global__ void __launch_bounds__(S::THREADS) ln_fwd_kernel(const LnRows p) {
    using T = typename S::T;
    __shared__ float2 slots[2][16];
    pdl_wait();
    pdl_trigger();
    const int t = threadIdx.x % S::TPR;
    const int r = blockIdx.x * S::ROWS + threadIdx.x / S::TPR;
    if (r >= p.M) return;                  // a whole row's threads
    const T* row = static_cast<const T*>(p.x) + static_cast<long>(r) * p.x_pitch;
    float x[S::NV][S::VEC];
    float s = 0.f;
#pragma unroll
    for (int v = 0; v < S::NV; ++v) {
        ln_load<S>(row, v, t, p.C, x[v]);
#pragma unroll
        for (int e = 0; e < S::VEC; ++e) s += x[v][e];
    }
    const float inv = 1.f / static_cast<float>(p.C);
    const float mean = ln_row_sum<S>(s, 0.f, slots, 0).x * inv;
    float q = 0.f, left = 0.f;
#pragma unroll
    for (int v = 0; v < S::NV; ++v)
#pragma unroll
        for (int e = 0; e < S::VEC; ++e) {
            x[v][e] -= mean;
            if (ln_col<S>(v, e, t) < p.C) {
                q += x[v][e] * x[v][e];
                left += x[v][e];
            }
        }
    // what rounding has left of the mean: it counts where a row's mean is much larger than its spread
    const float2 s2 = ln_row_sum<S>(q, left, slots, 1);
    const float dm = s2.y * inv;
    const float rstd = rsqrtf(fmaxf(s2.x * inv - dm * dm, 0.f) + p.eps);
    if (t == 0 && p.mean) {
        p.mean[r] = mean + dm;
        p.rstd[r] = rstd;
    }
    const float shift = -dm * rstd;
    T* out = static_cast<T*>(p.out) + static_cast<long>(r) * p.C;
#pragma unroll
    for (int v = 0; v < S::NV; ++v) {
        float w[S::VEC], b[S::VEC];
        ln_load_param<S>(p.w, p.param_bf16, 1.f, v, t, p.C, w);
        ln_load_param<S>(p.b, p.param_bf16, 0.f, v, t, p.C, b);
#pragma unroll
        for (int e = 0; e < S::VEC; ++e) x[v][e] = (x[v][e] * rstd + shift) * w[e] + b[e];
        ln_store<S>(out, v, t, p.C, x[v]);
    }
}

template <class S>
__global__ void __launch_bounds__(S::THREADS, S::BWD_BLOCKS) ln_bwd_kernel(const LnRows p) {
    using T = typename S::T;
    __shared__ float2 slots[2][16];
    pdl_wait();
    pdl_trigger();
    const int t = threadIdx.x % S::TPR;
    const float inv = 1.f / static_cast<float>(p.C);
    float dw[S::NV][S::VEC], db[S::NV][S::VEC];
#pragma unroll
    for (int v = 0; v < S::NV; ++v)
#pragma unroll
        for (int e = 0; e < S::VEC; ++e) dw[v][e] = db[v][e] = 0.f;
    int turn = 0;
    for (long r = static_cast<long>(blockIdx.x) * S::ROWS + threadIdx.x / S::TPR; r < p.M; r += static_cast<long>(gridDim.x) * S::ROWS, ++turn) {
        const T* xr = static_cast<const T*>(p.x) + r * p.x_pitch;
        const T* gr = static_cast<const T*>(p.dy) + r * p.dy_pitch;
        const float mean = p.mean[r], rstd = p.rstd[r];
        float xh[S::NV][S::VEC], g[S::NV][S::VEC];
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int v = 0; v < S::NV; ++v) {
            ln_load<S>(xr, v, t, p.C, xh[v]);
            ln_load<S>(gr, v, t, p.C, g[v]);
        }
#pragma unroll
        for (int v = 0; v < S::NV; ++v) {
            float w[S::VEC];
            ln_load_param<S>(p.w, p.param_bf16, 1.f, v, t, p.C, w);
#pragma unroll
            for (int e = 0; e < S::VEC; ++e) {
                xh[v][e] = (xh[v][e] - mean) * rstd;      // past the row's end: something finite, and g is zero there
                dw[v][e] += g[v][e] * xh[v][e];
                db[v][e] += g[v][e];
                g[v][e] *= w[e];
                s1 += g[v][e];
                s2 += g[v][e] * xh[v][e];
            }
        }
        const float2 s = ln_row_sum<S>(s1, s2, slots, turn);
        const float c1 = s.x * inv, c2 = s.y * inv;
        if (p.out) {
            T* out = static_cast<T*>(p.out) + r * p.C;
#pragma unroll
            for (int v = 0; v < S::NV; ++v) {
#pragma unroll
                for (int e = 0; e < S::VEC; ++e) g[v][e] = rstd * (g[v][e] - c1 - xh[v][e] * c2);
                ln_store<S>(out, v, t, p.C, g[v]);
            }
        }
    }
    if (!p.part) return;
    float* part = p.part + static_cast<long>(blockIdx.x) * 2 * p.C;
    if constexpr (S::ROWS == 1) {
#pragma unroll
        for (int v = 0; v < S::NV; ++v)
#pragma unroll
            for (int e = 0; e < S::VEC; ++e) {
                const int c = ln_col<S>(v, e, t);
                if (c < p.C) {
                    part[c] = dw[v][e];
                    part[p.C + c] = db[v][e];
                }
            }
    } else {
        // the block's warps have the same columns: add them up a chunk at a time
        __shared__ float sums[S::ROWS][S::CHUNK_COLS + 4];
#pragma unroll
        for (int v = 0; v < S::NV; ++v)
#pragma unroll
            for (int which = 0; which < 2; ++which) {
                __syncthreads();
#pragma unroll
                for (int e = 0; e < S::VEC; ++e) sums[threadIdx.x >> 5][ln_col<S>(0, e, t)] = which ? db[v][e] : dw[v][e];
                __syncthreads();
                for (int i = threadIdx.x; i < S::CHUNK_COLS; i += S::THREADS) {
                    const int c = v * S::CHUNK_COLS + i;
                    float a = 0.f;
#pragma unroll
                    for (int w = 0; w < S::ROWS; ++w) a += sums[w][i];
                    if (c < p.C) part[which * p.C + c] = a;
                }
            }
    }
}

// dw and db from the blocks' sums, in the order of the blocks: 32 columns a block, eight threads a column; grid y 0: dw, 1: db.
constexpr int kLnFinishCols = 32;
__global__ void __launch_bounds__(256) ln_finish_kernel(const float* __restrict__ part, int blocks, int C, void* __restrict__ dw, void* __restrict__ db, int bf16) {
    pdl_wait();
    pdl_trigger();
    __shared__ float sums[8][kLnFinishCols];
    void* out = blockIdx.y ? db : dw;
    if (!out) return;
    const int lane = threadIdx.x & 31, grp = threadIdx.x >> 5, c = blockIdx.x * kLnFinishCols + lane;
    float s = 0.f;
    if (c < C)
#pragma unroll 8
        for (int j = grp; j < blocks; j += 8) s += part[(static_cast<long>(j) * 2 + blockIdx.y) * C + c];
    sums[grp][lane] = s;
    __syncthreads();
    if (grp == 0 && c < C) {
#pragma unroll
        for (int g = 1; g < 8; ++g) s += sums[g][lane];
        if (bf16) static_cast<__nv_bfloat16*>(out)[c] = __float2bfloat16(s);
        else static_cast<float*>(out)[c] = s;
    }
}

}  // namespace ib200
