// y = act(x w + bias) + residual for up to 16 rows of x: one token, or a few that are decoded together.
//
// Nothing but the bytes of w counts here (2048 x 8192: 34 MB, 5.1 us at the measured copy rate), so the kernel is built to stream w [K, N] once, in the
// order in which it lies, with many loads on their way, and without shared memory between a load and its product.  A warp takes 16 rows of
// w by 64 columns at a time: lane t loads 16 bytes of rows 2q, 2q + 1, 2q + 8, 2q + 9 (q = t % 4) at columns 8 (t / 4), which are exactly the
// (k, n) that it has to hold for eight m16n8k16 products, if product e is given the columns 8 n + e: the order of the columns among the
// products is free, and two rows are woven into pairs by a byte permutation.  The rows of x, padded to 16, are the other operand; at this
// size the warp-level MMA costs nothing and needs neither descriptors nor tensor memory.
// The eight warps of a block share 64 columns and take the rows of w in turn; blocks of a cluster split the rows further, until the chip is full.
// The sums meet in shared memory, of the cluster's blocks through distributed shared memory, in a fixed order, and whoever adds them up does
// the epilogue.
#pragma once

#include "linear_gemm.cuh"

namespace ib200 {

struct FewRows {
    const __nv_bfloat16* x;        // [M, K], M <= 16
    const __nv_bfloat16* w;        // [K, N]
    const void* bias;              // [N], or null
    int bias_bf16, gelu;
    const __nv_bfloat16* residual; // [M, N], or null
    __half* slope;                 // gelu', or null
    __nv_bfloat16* y;
    int M, N, K;
    int steps;                     // of 16 rows of w, per block
};
constexpr int kFewMaxRows = 16, kFewCols = 64, kFewWarps = 8, kFewBatch = 4;

__device__ __forceinline__ uint4 ld_stream(const void* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ void mma_16x8x16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t cluster_addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(cluster_addr) : "memory");
    return v;
}

// Grid: strips of 64 columns times the cluster's blocks (SPLIT, along K).
template <int SPLIT>
__global__ void __launch_bounds__(kFewWarps * 32, 2) linear_few_kernel(const FewRows p) {
    __shared__ float part[kFewWarps][kFewMaxRows][kFewCols + 4];
    __shared__ float total[kFewMaxRows][kFewCols];
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, q = lane & 3, g = lane >> 2;
    const int strip = blockIdx.x / SPLIT, rank = blockIdx.x % SPLIT;
    const int col = strip * kFewCols + 8 * g;
    const int last = min((p.K + 15) / 16, (rank + 1) * p.steps);
    float acc[8][4];
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[e][i] = 0.f;
    for (int s0 = rank * p.steps + warp; s0 < last; s0 += kFewBatch * kFewWarps) {
        uint4 w[kFewBatch][4];
        uint32_t a[kFewBatch][4];
#pragma unroll
        for (int u = 0; u < kFewBatch; ++u) {
            const int s = s0 + u * kFewWarps;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int k = 16 * s + 2 * q + (i & 1) + 8 * (i >> 1);
                w[u][i] = s < last && k < p.K && col < p.N ? ld_stream(p.w + static_cast<long>(k) * p.N + col) : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int xr = g + 8 * (i & 1), k = 16 * s + 2 * q + 8 * (i >> 1);
                a[u][i] = s < last && k < p.K && xr < p.M ? *reinterpret_cast<const uint32_t*>(p.x + static_cast<long>(xr) * p.K + k) : 0u;
            }
        }
#pragma unroll
        for (int u = 0; u < kFewBatch; ++u) {
            const uint32_t lo[4] = {w[u][0].x, w[u][0].y, w[u][0].z, w[u][0].w}, lo1[4] = {w[u][1].x, w[u][1].y, w[u][1].z, w[u][1].w};
            const uint32_t hi[4] = {w[u][2].x, w[u][2].y, w[u][2].z, w[u][2].w}, hi1[4] = {w[u][3].x, w[u][3].y, w[u][3].z, w[u][3].w};
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t pick = e & 1 ? 0x7632u : 0x5410u;      // the odd or the even column of a pair, of two rows
                mma_16x8x16(acc[e], a[u], __byte_perm(lo[e / 2], lo1[e / 2], pick), __byte_perm(hi[e / 2], hi1[e / 2], pick));
            }
        }
    }
    // what the epilogue will need, asked for ahead of the barriers
    const int row = threadIdx.x / (kFewCols / 4), c4 = threadIdx.x % (kFewCols / 4) * 4, c = strip * kFewCols + c4;
    const bool mine = row < p.M && c < p.N && static_cast<int>(threadIdx.x % SPLIT) == rank;      // the blocks share the adding up
    const long at = static_cast<long>(row) * p.N + c;
    uint4 bias = make_uint4(0, 0, 0, 0);
    uint2 res = make_uint2(0, 0);
    if (mine) {
        if (p.bias && p.bias_bf16) {
            const uint2 b = *reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(p.bias) + c);
            bias.x = b.x;
            bias.y = b.y;
        } else if (p.bias) {
            bias = *reinterpret_cast<const uint4*>(static_cast<const float*>(p.bias) + c);
        }
        if (p.residual) res = *reinterpret_cast<const uint2*>(p.residual + at);
    }
    // product e of column index n is column 8 n + e: a thread has columns 16 q .. 16 q + 15 of rows g and g + 8
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float* dst = &part[warp][g + 8 * (i >> 1)][16 * q + 8 * (i & 1)];
        *reinterpret_cast<float4*>(dst) = make_float4(acc[0][i], acc[1][i], acc[2][i], acc[3][i]);
        *reinterpret_cast<float4*>(dst + 4) = make_float4(acc[4][i], acc[5][i], acc[6][i], acc[7][i]);
    }
    __syncthreads();
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](const float4& v) { sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w; };
    if (row < p.M) {
#pragma unroll
        for (int w = 0; w < kFewWarps; ++w) add(*reinterpret_cast<const float4*>(&part[w][row][c4]));
    }
    if constexpr (SPLIT > 1) {
        *reinterpret_cast<float4*>(&total[row][c4]) = sum;
        cluster_sync_all();
        if (mine) {
            const uint32_t src = smem_u32(&total[row][c4]);
            float4 v[SPLIT];
#pragma unroll
            for (int r = 0; r < SPLIT; ++r) v[r] = ld_cluster_f4(mapa_u32(src, r));
            sum = v[0];
#pragma unroll
            for (int r = 1; r < SPLIT; ++r) add(v[r]);
        }
    }
    if (mine) {
        uint64_t v[2] = {pack_f32x2(sum.x, sum.y), pack_f32x2(sum.z, sum.w)};
        if (p.bias) {
            v[0] = fadd2(v[0], p.bias_bf16 ? unpack_bf16x2(bias.x) : pack_f32x2(__uint_as_float(bias.x), __uint_as_float(bias.y)));
            v[1] = fadd2(v[1], p.bias_bf16 ? unpack_bf16x2(bias.y) : pack_f32x2(__uint_as_float(bias.z), __uint_as_float(bias.w)));
        }
        uint32_t slope[2], out[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            if (p.gelu) v[e] = gelu_with_slope2(v[e], slope[e]);
            if (p.residual) v[e] = fadd2(v[e], unpack_bf16x2(e ? res.y : res.x));
            out[e] = pack_bf16_pair(v[e]);
        }
        *reinterpret_cast<uint2*>(p.y + at) = make_uint2(out[0], out[1]);
        if (p.slope) *reinterpret_cast<uint2*>(p.slope + at) = make_uint2(slope[0], slope[1]);
    }
    if constexpr (SPLIT > 1) cluster_sync_all();                           // no block leaves while another may still read its sums
}

}  // namespace ib200
