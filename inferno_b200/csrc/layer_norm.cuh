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
// Memory-bound: a row is read from global memory once, into the ring, and everything is computed from there, so the variance is the sum of
// squared differences from the mean and not a difference of two sums.  (bf16 rows that do not begin on 4 bytes, which no asynchronous copy can fetch,
// have no ring: they are read from global memory in each pass, three times forward and twice backward.)  A row belongs to 32, 64, 128, 256 or 512 threads (LnShape), each of
// which has up to four 16-byte chunks of it: a row of one warp needs no barrier.  The backward's threads keep their columns from row to row
// and sum dw and db in registers; a block's sums meet in the workspace, which ln_finish_kernel adds up in a fixed order.  All sums are
// fp32; the only rounding to fewer bits is that of the results.
// Measured (us; floor at the measured copy rate): bf16 16384 x 8192 forward 101 (82), backward 126 (123); 16384 x 4096 55 (41), 68 (61); 16384 x 768 10.8 (7.7),
// 19.8 (11.5); fp32 16384 x 1024 27 (20), 37 (31).  The forward is bound by issue slots (0.75 a cycle), the backward by memory.
// Further off: narrow rows, where lanes of a row's warp have nothing to do (24 of 32 at 64 bf16 columns) and what is done per row counts, bf16 196608 x 64
// 44 (7.7), 56 (11.5), 98304 x 128 23 (7.7), 32 (11.5); rows in pieces of 4 bytes, 32768 x 778 39 (15.6), 51 (23.4) next to 28 and 39 for 776 columns;
// rows of odd bf16 width, 32768 x 777 53 (15.5), 79 (23.3).
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

// TPR threads per row, chunks of 16 bytes, NV of them per thread.  AU: elements per access.  Where rows, weight and bias begin on 16 bytes and hold
// whole chunks it is a chunk (ALIGNED), PT being the type of weight and bias; otherwise 4 bytes or a single bf16, dealt out to the threads in
// turn, so that a warp's accesses still run together, and the type of weight and bias is looked up.
constexpr int kLnBwdThreads = 512;      // a block of the backward, one per SM: as few blocks' sums as there can be
template <class T_, class PT_, int TPR_, int NV_, int AU_>
struct LnShape {
    using T = T_;
    using PT = PT_;
    static constexpr int TPR = TPR_, NV = NV_, VEC = 16 / sizeof(T_), WARPS = TPR_ / 32;
    static constexpr int AU = AU_;
    static constexpr bool ALIGNED = AU_ * sizeof(T_) == 16, RING = AU_ * sizeof(T_) >= 4;      // (asynchronous copies are of 4 bytes at least)
    static constexpr int FWD_THREADS = TPR_ < 256 ? 256 : TPR_, FWD_ROWS = FWD_THREADS / TPR_, FWD_BLOCKS = 1024 / FWD_THREADS;      // blocks resident per SM
    static constexpr int BWD_ROWS = kLnBwdThreads / TPR_;
    static constexpr int CHUNK_COLS = TPR_ * VEC;                                       // columns of one chunk of all threads
    static constexpr int STAGES = 2;                                                    // rows of a thread's ring: this one and the next
    static constexpr int PARAM_UNITS = sizeof(PT_) * VEC / 16 ? sizeof(PT_) * VEC / 16 : 1;      // 16-byte units of a chunk's weights
    static constexpr int FWD_SMEM = RING ? STAGES * NV_ * FWD_THREADS * 16 : 0;
    static constexpr int BWD_RING = RING ? (STAGES * 2 + PARAM_UNITS) * NV_ * kLnBwdThreads * 16 : 0;
    static constexpr int BWD_SUMS = kLnBwdThreads * VEC * 4;                            // one chunk's columns of every row at work, in the ring's place
    static constexpr int BWD_SMEM = BWD_RING > BWD_SUMS ? BWD_RING : BWD_SUMS;
};

__device__ __forceinline__ float ln_to_float(float v) { return v; }
__device__ __forceinline__ float ln_to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void ln_from_float(float v, float& o) { o = v; }
__device__ __forceinline__ void ln_from_float(float v, __nv_bfloat16& o) { o = __float2bfloat16(v); }

// Column of element e of chunk v of thread t; past the row's end: C and more.
template <class S>
__device__ __forceinline__ int ln_col(int v, int e, int t) {
    return v * S::CHUNK_COLS + (e / S::AU * S::TPR + t) * S::AU + e % S::AU;
}
// A chunk in registers: pairs of fp32, for the packed arithmetic (two lanes an instruction: with single ones the issue slots, not the memory, bound
// the forward).
template <class S>
struct LnChunk {
    uint64_t f[S::VEC / 2];
};
__device__ __forceinline__ uint64_t ln_pair_bf16(uint32_t w) { return pack_f32x2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
__device__ __forceinline__ void ln_unpack(const uint4& u, uint64_t (&f)[4]) {
    f[0] = ln_pair_bf16(u.x);
    f[1] = ln_pair_bf16(u.y);
    f[2] = ln_pair_bf16(u.z);
    f[3] = ln_pair_bf16(u.w);
}
__device__ __forceinline__ void ln_unpack(const uint4& u, uint64_t (&f)[2]) {
    f[0] = pack_f32x2(__uint_as_float(u.x), __uint_as_float(u.y));
    f[1] = pack_f32x2(__uint_as_float(u.z), __uint_as_float(u.w));
}
// Elements of p one by one, `none` past the row's end (rows that do not begin on 16 bytes).
template <class S, class P>
__device__ __forceinline__ void ln_gather(const P* p, float none, int v, int t, int C, LnChunk<S>& k) {
#pragma unroll
    for (int e = 0; e < S::VEC; e += 2) {
        const int c0 = ln_col<S>(v, e, t), c1 = ln_col<S>(v, e + 1, t);
        k.f[e / 2] = pack_f32x2(c0 < C ? ln_to_float(p[c0]) : none, c1 < C ? ln_to_float(p[c1]) : none);
    }
}
// The same columns of weight or bias, `none` where there is none.
template <class S>
__device__ __forceinline__ void ln_unpack_param(const uint4 (&u)[S::PARAM_UNITS], LnChunk<S>& k) {
    if constexpr (sizeof(typename S::PT) == 4) {
#pragma unroll
        for (int q = 0; q < S::VEC / 4; ++q) {
            k.f[2 * q] = pack_f32x2(__uint_as_float(u[q].x), __uint_as_float(u[q].y));
            k.f[2 * q + 1] = pack_f32x2(__uint_as_float(u[q].z), __uint_as_float(u[q].w));
        }
    } else {
        const uint32_t w[4] = {u[0].x, u[0].y, u[0].z, u[0].w};
#pragma unroll
        for (int i = 0; i < S::VEC / 2; ++i) k.f[i] = ln_pair_bf16(w[i]);
    }
}
template <class S>
__device__ __forceinline__ void ln_load_param(const void* p, int bf16, float none, int v, int t, int C, LnChunk<S>& k) {
    if constexpr (S::ALIGNED) {
        const int c = ln_col<S>(v, 0, t);
        if (p && c < C) {
            const uint4* src = reinterpret_cast<const uint4*>(static_cast<const typename S::PT*>(p) + c);
            uint4 u[S::PARAM_UNITS];
#pragma unroll
            for (int q = 0; q < S::PARAM_UNITS; ++q) u[q] = src[q];
            ln_unpack_param<S>(u, k);
        } else {
#pragma unroll
            for (int i = 0; i < S::VEC / 2; ++i) k.f[i] = pack_f32x2(none, none);
        }
    } else if (!p) {
#pragma unroll
        for (int i = 0; i < S::VEC / 2; ++i) k.f[i] = pack_f32x2(none, none);
    } else if constexpr (S::AU == 2) {               // pairs, which begin on their own size
#pragma unroll
        for (int i = 0; i < S::VEC / 2; ++i) {
            const int c = ln_col<S>(v, 2 * i, t);
            if (c >= C) k.f[i] = pack_f32x2(none, none);
            else if (bf16) k.f[i] = ln_pair_bf16(*reinterpret_cast<const uint32_t*>(static_cast<const __nv_bfloat16*>(p) + c));
            else k.f[i] = *reinterpret_cast<const uint64_t*>(static_cast<const float*>(p) + c);
        }
    } else if (bf16) {
        ln_gather<S>(static_cast<const __nv_bfloat16*>(p), none, v, t, C, k);
    } else {
        ln_gather<S>(static_cast<const float*>(p), none, v, t, C, k);
    }
}
template <class S>
__device__ __forceinline__ void ln_store(typename S::T* row, int v, int t, int C, const LnChunk<S>& k) {
    float f[S::VEC];
#pragma unroll
    for (int i = 0; i < S::VEC / 2; ++i) unpack_f32x2(k.f[i], f[2 * i], f[2 * i + 1]);
    if constexpr (S::ALIGNED) {
        const int c = ln_col<S>(v, 0, t);
        if (c >= C) return;
        uint4 u;
        if constexpr (S::VEC == 8) u = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
        else u = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
        *reinterpret_cast<uint4*>(row + c) = u;
    } else if constexpr (S::AU == 2) {
#pragma unroll
        for (int e = 0; e < S::VEC; e += 2) {
            const int c = ln_col<S>(v, e, t);
            if (c < C) *reinterpret_cast<uint32_t*>(row + c) = pack_bf16x2(f[e], f[e + 1]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < S::VEC; ++e) {
            const int c = ln_col<S>(v, e, t);
            if (c < C) ln_from_float(f[e], row[c]);
        }
    }
}
__device__ __forceinline__ float ln_pair_sum(uint64_t p) {
    float a, b;
    unpack_f32x2(p, a, b);
    return a + b;
}

// Sums of a (and b) over the threads of a row.  `turn` alternates between two sets of slots, so that one barrier per sum is enough: a slot
// is written again only after the next sum's barrier, which every thread reaches after it has read.  Each row of a block has a barrier of its own.
template <class S, bool BOTH>
__device__ __forceinline__ float2 ln_row_sum(float a, float b, float2 (*slots)[16], int turn) {
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) {
        a += __shfl_xor_sync(0xffffffffu, a, m);
        if (BOTH) b += __shfl_xor_sync(0xffffffffu, b, m);
    }
    if constexpr (S::WARPS > 1) {
        const int warp = threadIdx.x >> 5, first = warp / S::WARPS * S::WARPS;
        float2* s = slots[turn & 1];
        if ((threadIdx.x & 31) == 0) s[warp] = make_float2(a, b);
        asm volatile("bar.sync %0, %1;" ::"r"(1 + warp / S::WARPS), "n"(S::TPR) : "memory");
        a = b = 0.f;
#pragma unroll
        for (int w = 0; w < S::WARPS; ++w) {
            a += s[first + w].x;
            if (BOTH) b += s[first + w].y;
        }
    }
    return make_float2(a, b);
}

// ---- a thread's ring in shared memory: its own chunks of the rows to come ----
// Filled by 16-byte asynchronous copies and read by the thread that asked for them, so that waiting for the thread's own copies is all the
// synchronisation there is.  [stage][chunk][thread]: a warp's accesses run together.
__device__ __forceinline__ void ln_copy_async(uint4* dst, const void* src, bool inside) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(inside ? 16 : 0) : "memory");
}
__device__ __forceinline__ void ln_copy_async4(void* dst, const void* src, bool inside) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(inside ? 4 : 0) : "memory");
}
__device__ __forceinline__ void ln_copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING>
__device__ __forceinline__ void ln_copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory"); }
template <class S, int THREADS>
__device__ __forceinline__ void ln_request(uint4* slots, const typename S::T* row, int t, int C) {
#pragma unroll
    for (int v = 0; v < S::NV; ++v) {
        uint4* slot = slots + v * THREADS + threadIdx.x;
        if constexpr (S::ALIGNED) {
            const int c = ln_col<S>(v, 0, t);
            ln_copy_async(slot, row + (c < C ? c : 0), c < C);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int c = ln_col<S>(v, i * S::AU, t);
                ln_copy_async4(reinterpret_cast<uint32_t*>(slot) + i, row + (c < C ? c : 0), c < C);
            }
        }
    }
}

template <class S>
__global__ void __launch_bounds__(S::FWD_THREADS, S::FWD_BLOCKS) ln_fwd_kernel(const LnRows p) {
    using T = typename S::T;
    extern __shared__ uint4 ring[];
    __shared__ float2 slots[2][16];
    pdl_wait();
    pdl_trigger();
    const int t = threadIdx.x % S::TPR;
    const long first = static_cast<long>(blockIdx.x) * S::FWD_ROWS + threadIdx.x / S::TPR, step = static_cast<long>(gridDim.x) * S::FWD_ROWS;
    const T* x0 = static_cast<const T*>(p.x);
    if constexpr (S::RING) {
        if (first < p.M) ln_request<S, S::FWD_THREADS>(ring, x0 + first * p.x_pitch, t, p.C);
        ln_copy_commit();
    }
    const float inv = 1.f / static_cast<float>(p.C);
    int stage = 0;
    for (long r = first; r < p.M; r += step) {
        if constexpr (S::RING) {
            if (r + step < p.M) ln_request<S, S::FWD_THREADS>(ring + (stage ^ 1) * S::NV * S::FWD_THREADS, x0 + (r + step) * p.x_pitch, t, p.C);
            ln_copy_commit();
            ln_copy_wait<1>();
        }
        // A chunk of the row, less `minus`; zeros past the row's end.  Read again in each of the three passes rather than held in fp32: with 32 registers
        // less there are twice as many rows at work on an SM.
        auto chunk = [&](int v, uint64_t minus, bool centred, LnChunk<S>& x) {
            if constexpr (S::RING) {
                ln_unpack(ring[(stage * S::NV + v) * S::FWD_THREADS + threadIdx.x], x.f);
            } else {
                ln_gather<S>(x0 + r * p.x_pitch, 0.f, v, t, p.C, x);
            }
            if (!centred) return;
#pragma unroll
            for (int i = 0; i < S::VEC / 2; ++i) x.f[i] = fadd2(x.f[i], minus);
        };
        uint64_t s = 0;
#pragma unroll
        for (int v = 0; v < S::NV; ++v) {
            LnChunk<S> x;
            chunk(v, 0, false, x);
#pragma unroll
            for (int i = 0; i < S::VEC / 2; ++i) s = fadd2(s, x.f[i]);
        }
        const float mean = ln_row_sum<S, false>(ln_pair_sum(s), 0.f, slots, 0).x * inv;
        const uint64_t minus = pack_f32x2(-mean, -mean);
        uint64_t q = 0, left = 0;
#pragma unroll
        for (int v = 0; v < S::NV; ++v) {
            LnChunk<S> x;
            chunk(v, minus, true, x);
            if constexpr (S::ALIGNED) {
                if (ln_col<S>(v, 0, t) >= p.C) continue;
            } else {
#pragma unroll
                for (int e = 0; e < S::VEC; e += 2) {
                    float a, b;
                    unpack_f32x2(x.f[e / 2], a, b);
                    x.f[e / 2] = pack_f32x2(ln_col<S>(v, e, t) < p.C ? a : 0.f, ln_col<S>(v, e + 1, t) < p.C ? b : 0.f);
                }
            }
#pragma unroll
            for (int i = 0; i < S::VEC / 2; ++i) {
                q = ffma2(x.f[i], x.f[i], q);
                left = fadd2(left, x.f[i]);
            }
        }
        // what rounding has left of the mean: it counts where a row's mean is much larger than its spread
        const float2 s2 = ln_row_sum<S, true>(ln_pair_sum(q), ln_pair_sum(left), slots, 1);
        const float dm = s2.y * inv;
        const float rstd = rsqrtf(fmaxf(s2.x * inv - dm * dm, 0.f) + p.eps);
        if (t == 0 && p.mean) {
            p.mean[r] = mean + dm;
            p.rstd[r] = rstd;
        }
        const uint64_t scale = pack_f32x2(rstd, rstd), shift = pack_f32x2(-dm * rstd, -dm * rstd);
        T* out = static_cast<T*>(p.out) + r * p.C;
#pragma unroll
        for (int v = 0; v < S::NV; ++v) {
            LnChunk<S> x, w, b;
            ln_load_param<S>(p.w, p.param_bf16, 1.f, v, t, p.C, w);
            ln_load_param<S>(p.b, p.param_bf16, 0.f, v, t, p.C, b);
            chunk(v, minus, true, x);
#pragma unroll
            for (int i = 0; i < S::VEC / 2; ++i) x.f[i] = ffma2(ffma2(x.f[i], scale, shift), w.f[i], b.f[i]);
            ln_store<S>(out, v, t, p.C, x);
        }
        stage ^= 1;
    }
}

template <class S>
__global__ void __launch_bounds__(kLnBwdThreads, 1) ln_bwd_kernel(const LnRows p) {
    using T = typename S::T;
    constexpr int ROW = 2 * S::NV * kLnBwdThreads;
    extern __shared__ uint4 ring[];
    __shared__ float2 slots[2][16];
    pdl_wait();
    pdl_trigger();
    const int t = threadIdx.x % S::TPR;
    const long first = static_cast<long>(blockIdx.x) * S::BWD_ROWS + threadIdx.x / S::TPR, step = static_cast<long>(gridDim.x) * S::BWD_ROWS;
    const T *x0 = static_cast<const T*>(p.x), *g0 = static_cast<const T*>(p.dy);
    auto request = [&](int s, long r) {
        ln_request<S, kLnBwdThreads>(ring + s * ROW, x0 + r * p.x_pitch, t, p.C);
        ln_request<S, kLnBwdThreads>(ring + s * ROW + S::NV * kLnBwdThreads, g0 + r * p.dy_pitch, t, p.C);
    };
    uint4* wsave = ring + S::STAGES * ROW;      // the thread's weights
    float mean = 0.f, rstd = 0.f;
    if (first < p.M) {
        mean = p.mean[first];
        rstd = p.rstd[first];
    }
    if constexpr (S::RING) {
        if (p.w) {
#pragma unroll
            for (int v = 0; v < S::NV; ++v) {
                uint4* save = wsave + v * S::PARAM_UNITS * kLnBwdThreads + threadIdx.x;
                if constexpr (S::ALIGNED) {
                    const int c = ln_col<S>(v, 0, t);
                    const uint4* src = reinterpret_cast<const uint4*>(static_cast<const typename S::PT*>(p.w) + (c < p.C ? c : 0));
#pragma unroll
                    for (int q = 0; q < S::PARAM_UNITS; ++q) ln_copy_async(save + q * kLnBwdThreads, src + q, c < p.C);
                } else {                           // as fp32, whatever they are
                    LnChunk<S> w;
                    ln_load_param<S>(p.w, p.param_bf16, 1.f, v, t, p.C, w);
#pragma unroll
                    for (int q = 0; q < S::PARAM_UNITS; ++q)
                        save[q * kLnBwdThreads] = make_uint4(static_cast<uint32_t>(w.f[2 * q]), static_cast<uint32_t>(w.f[2 * q] >> 32),
                                                             static_cast<uint32_t>(w.f[2 * q + 1]), static_cast<uint32_t>(w.f[2 * q + 1] >> 32));
                }
            }
        }
        if (first < p.M) request(0, first);
        ln_copy_commit();
    }
    const float inv = 1.f / static_cast<float>(p.C);
    LnChunk<S> dw2[S::NV], db2[S::NV];
#pragma unroll
    for (int v = 0; v < S::NV; ++v)
#pragma unroll
        for (int i = 0; i < S::VEC / 2; ++i) dw2[v].f[i] = db2[v].f[i] = 0;
    int turn = 0, stage = 0;
    for (long r = first; r < p.M; r += step, ++turn) {
        float next_mean = 0.f, next_rstd = 0.f;
        if (r + step < p.M) {
            next_mean = p.mean[r + step];
            next_rstd = p.rstd[r + step];
        }
        if constexpr (S::RING) {
            if (r + step < p.M) request(stage ^ 1, r + step);
            ln_copy_commit();
            ln_copy_wait<1>();
        }
        auto weight = [&](int v, LnChunk<S>& w) {
            if constexpr (S::RING) {
                if (p.w) {
                    uint4 u[S::PARAM_UNITS];
#pragma unroll
                    for (int q = 0; q < S::PARAM_UNITS; ++q) u[q] = wsave[(v * S::PARAM_UNITS + q) * kLnBwdThreads + threadIdx.x];
                    ln_unpack_param<S>(u, w);
                } else {
#pragma unroll
                    for (int i = 0; i < S::VEC / 2; ++i) w.f[i] = pack_f32x2(1.f, 1.f);
                }
            } else {
                ln_load_param<S>(p.w, p.param_bf16, 1.f, v, t, p.C, w);
            }
        };
        // One chunk of both rows, xh and g: read again for the second pass rather than held, which would cost the registers that the sums are in.
        const uint64_t scale = pack_f32x2(rstd, rstd), minus = pack_f32x2(-mean, -mean);
        auto chunk = [&](int v, LnChunk<S>& x, LnChunk<S>& g) {
            if constexpr (S::RING) {
                ln_unpack(ring[stage * ROW + v * kLnBwdThreads + threadIdx.x], x.f);
                ln_unpack(ring[stage * ROW + (S::NV + v) * kLnBwdThreads + threadIdx.x], g.f);
            } else {
                ln_gather<S>(x0 + r * p.x_pitch, 0.f, v, t, p.C, x);
                ln_gather<S>(g0 + r * p.dy_pitch, 0.f, v, t, p.C, g);
            }
#pragma unroll
            for (int i = 0; i < S::VEC / 2; ++i) x.f[i] = fmul2(fadd2(x.f[i], minus), scale);      // past the row's end: something finite, and g is zero there
        };
        uint64_t s1 = 0, s2 = 0;
#pragma unroll
        for (int v = 0; v < S::NV; ++v) {
            LnChunk<S> x, g, w;
            chunk(v, x, g);
            weight(v, w);
#pragma unroll
            for (int i = 0; i < S::VEC / 2; ++i) {
                dw2[v].f[i] = ffma2(g.f[i], x.f[i], dw2[v].f[i]);
                db2[v].f[i] = fadd2(db2[v].f[i], g.f[i]);
                const uint64_t gw = fmul2(g.f[i], w.f[i]);
                s1 = fadd2(s1, gw);
                s2 = ffma2(gw, x.f[i], s2);
            }
        }
        const float2 s = ln_row_sum<S, true>(ln_pair_sum(s1), ln_pair_sum(s2), slots, turn);
        if (p.out) {
            // dx = rstd g - rstd c1 - xh rstd c2
            const float c1 = -s.x * inv * rstd, c2 = -s.y * inv * rstd;
            const uint64_t add = pack_f32x2(c1, c1), slope = pack_f32x2(c2, c2);
            T* out = static_cast<T*>(p.out) + r * p.C;
#pragma unroll
            for (int v = 0; v < S::NV; ++v) {
                LnChunk<S> x, g, w;
                chunk(v, x, g);
                weight(v, w);
#pragma unroll
                for (int i = 0; i < S::VEC / 2; ++i) g.f[i] = ffma2(fmul2(g.f[i], w.f[i]), scale, ffma2(x.f[i], slope, add));
                ln_store<S>(out, v, t, p.C, g);
            }
        }
        mean = next_mean;
        rstd = next_rstd;
        stage ^= 1;
    }
    if (!p.part) return;
    // The rows at work have the same columns: a chunk of each is laid out in the ring's place and added up, dw first, then db.
    float* part = p.part + static_cast<long>(blockIdx.x) * 2 * p.C;
    float* sums = reinterpret_cast<float*>(ring) + threadIdx.x / S::TPR * S::CHUNK_COLS;
    ln_copy_wait<0>();
#pragma unroll
    for (int v = 0; v < S::NV; ++v)
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < S::VEC / 2; ++i) {
                float lo, hi;
                unpack_f32x2(which ? db2[v].f[i] : dw2[v].f[i], lo, hi);
                sums[ln_col<S>(0, 2 * i, t)] = lo;
                sums[ln_col<S>(0, 2 * i + 1, t)] = hi;
            }
            __syncthreads();
            for (int i = threadIdx.x; i < S::CHUNK_COLS; i += kLnBwdThreads) {
                const int c = v * S::CHUNK_COLS + i;
                float a = 0.f;
#pragma unroll
                for (int w = 0; w < S::BWD_ROWS; ++w) a += reinterpret_cast<const float*>(ring)[w * S::CHUNK_COLS + i];
                if (c < p.C) part[which * p.C + c] = a;
            }
        }
}

// dw and db from the blocks' sums, in the order of the blocks: 32 columns a block, sixteen threads a column; grid y 0: dw, 1: db.
constexpr int kLnFinishCols = 32;
__global__ void __launch_bounds__(512) ln_finish_kernel(const float* __restrict__ part, int blocks, int C, void* __restrict__ dw, void* __restrict__ db, int bf16) {
    pdl_wait();
    pdl_trigger();
    __shared__ float sums[16][kLnFinishCols];
    void* out = blockIdx.y ? db : dw;
    if (!out) return;
    const int lane = threadIdx.x & 31, grp = threadIdx.x >> 5, c = blockIdx.x * kLnFinishCols + lane;
    float s = 0.f;
    if (c < C)
#pragma unroll 10
        for (int j = grp; j < blocks; j += 16) s += part[(static_cast<long>(j) * 2 + blockIdx.y) * C + c];
    sums[grp][lane] = s;
    __syncthreads();
    if (grp == 0 && c < C) {
#pragma unroll
        for (int g = 1; g < 16; ++g) s += sums[g][lane];
        if (bf16) static_cast<__nv_bfloat16*>(out)[c] = __float2bfloat16(s);
        else static_cast<float*>(out)[c] = s;
    }
}

}  // namespace ib200
