// y = act(x w + bias) + residual for up to 32 rows of x: one token, or a few that are decoded together.
//
// Nothing but the bytes of w counts here (2048 x 8192: 34 MB, 5.1 us at the measured copy rate), so the kernel is built to stream w [K, N] once with as
// many bytes on their way as an SM can hold.  (A plain loop of 16-byte loads reads that matrix in 14.4, 10.3 and 8.2 us with 64, 128 and
// 256 KB on their way per SM, whatever the width of a block's strip.)  Each warp has a ring of three boxes of 64 rows by 64 columns, 8 KB each,
// which one of its lanes has the TMA unit fill: 192 KB per SM, and no register, barrier or other thread stands between a box and its use.
// (Sixteen loads a thread in registers, 128 KB per SM: 10.9 us; the same by 16-byte asynchronous copies into slots per thread: 14.)
// A lane (q = t % 4, g = t / 4) reads 16 bytes of rows 2q, 2q + 1, 2q + 8, 2q + 9 at columns 8g, no bank twice, and these are exactly the (k, n) that it
// has to hold for eight m16n8k16 products, if product e is given the columns 8 n + e: the order of the columns among the products is free,
// and two rows are woven into pairs by a byte permutation.  The rows of x, padded to 16 or 32, are the other operand; at this size the
// warp-level MMA costs nothing and needs neither descriptors nor tensor memory.
// The eight warps of a block share 64 columns and take the boxes in turn; blocks of a cluster split the rows further, until every SM has
// a block.  The sums meet in shared memory, of the cluster's blocks through distributed shared memory, in a fixed order, and whoever adds
// them up does the epilogue.
// Measured, us: 1 x 2048 x 8192 9.0 (3.7 TB/s, launch included), 1 x 1024 x 4096 4.2, 32 x 1024 x 4096 7.0; two of them, 4096 -> 16384 -> 4096, 50 (5.4 TB/s).
#pragma once

#include "linear_gemm.cuh"

namespace ib200 {

struct FewRows {
    const __nv_bfloat16* x;        // [M, K], M <= 32
    const void* bias;              // [N], or null
    int bias_bf16, gelu;
    const __nv_bfloat16* residual; // [M, N], or null
    __half* slope;                 // gelu', or null
    __nv_bfloat16* y;
    int M, N, K;
    int steps;                     // of 64 rows of w, per block
    int* status;
};
constexpr int kFewMaxRows = 32, kFewCols = 64, kFewStep = 64, kFewWarps = 8, kFewDepth = 3, kFewBox = kFewStep * kFewCols * 2;
constexpr int kFewSmem = kFewWarps * kFewDepth * kFewBox + 1024;
static_assert(kFewWarps * kFewMaxRows * (kFewCols + 4) * 4 <= kFewWarps * kFewDepth * kFewBox, "the warps' sums take the ring's place");

__device__ __forceinline__ void mma_16x8x16(float (&c)[4], const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t cluster_addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(cluster_addr) : "memory");
    return v;
}

// Grid: strips of 64 columns times the cluster's blocks (SPLIT, along K).  ROWS: 16 or 32.
template <int SPLIT, int ROWS>
__global__ void __launch_bounds__(kFewWarps * 32, 1) linear_few_kernel(const __grid_constant__ CUtensorMap wmap, const FewRows p) {
    extern __shared__ uint8_t few_smem[];
    constexpr int MT = ROWS / 16;
    __shared__ float total[ROWS][kFewCols];
    __shared__ uint64_t bars[kFewWarps][kFewDepth];
    __shared__ int abort_flag;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, q = lane & 3, g = lane >> 2;
    const int strip = blockIdx.x / SPLIT, rank = blockIdx.x % SPLIT;
    const int first = rank * p.steps + warp, last = min((p.K + kFewStep - 1) / kFewStep, (rank + 1) * p.steps);
    uint8_t* boxes = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(few_smem) + 1023) & ~static_cast<uintptr_t>(1023));
    uint8_t* mybox = boxes + warp * kFewDepth * kFewBox;
    const ResidentAbortCtx ab{&abort_flag, p.status};
    if (tid == 0) abort_flag = 0;
    if (lane == 0) {
        for (int u = 0; u < kFewDepth; ++u) mbar_init(&bars[warp][u], 1);
        fence_mbar_init();
        tma_prefetch_desc(&wmap);
    }
    __syncthreads();
    pdl_wait();
    pdl_trigger();

    auto request = [&](int slot, int s) {          // lane 0
        mbar_arrive_expect_tx(&bars[warp][slot], kFewBox);
        tma_load_3d(mybox + slot * kFewBox, &wmap, &bars[warp][slot], strip * kFewCols, s * kFewStep, 0);
    };
    if (lane == 0) {
#pragma unroll
        for (int u = 0; u < kFewDepth; ++u)
            if (first + u * kFewWarps < last) request(u, first + u * kFewWarps);
    }
    // x of a step: of each 16 of its columns, 2q, 2q + 1 and 2q + 8, 2q + 9 of rows g and g + 8 (and 16 more)
    auto load_x = [&](int s, uint32_t (&a)[4][4 * MT]) {
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
#pragma unroll
            for (int i = 0; i < 4 * MT; ++i) {
                const int row = g + 8 * (i & 1) + 16 * (i >> 2), k = kFewStep * s + 16 * kk + 2 * q + 8 * (i >> 1 & 1);
                a[kk][i] = s < last && k < p.K && row < p.M ? *reinterpret_cast<const uint32_t*>(p.x + static_cast<long>(row) * p.K + k) : 0u;
            }
    };
    uint32_t a[4][4 * MT];
    load_x(first, a);
    // what the epilogue will need: the thread adds up four columns of one row in each 16
    const int c4 = tid % (kFewCols / 4) * 4, c = strip * kFewCols + c4;
    const bool my_share = c < p.N && tid % SPLIT == rank;               // the blocks share the adding up
    uint4 bias = make_uint4(0, 0, 0, 0);
    uint2 res[MT];
    if (my_share) {
        if (p.bias && p.bias_bf16) {
            const uint2 b = *reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(p.bias) + c);
            bias.x = b.x;
            bias.y = b.y;
        } else if (p.bias) {
            bias = *reinterpret_cast<const uint4*>(static_cast<const float*>(p.bias) + c);
        }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int row = 16 * m + tid / (kFewCols / 4);
        res[m] = my_share && p.residual && row < p.M ? *reinterpret_cast<const uint2*>(p.residual + static_cast<long>(row) * p.N + c) : make_uint2(0, 0);
    }
    float acc[MT][8][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[m][e][i] = 0.f;
    uint32_t slot = 0, phase = 0;
    for (int s = first; s < last; s += kFewWarps) {
        uint32_t next[4][4 * MT];
        load_x(s + kFewWarps, next);
        mbar_wait(&bars[warp][slot], phase, ab, 40);
        const uint8_t* box = mybox + slot * kFewBox;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
            uint32_t w[4][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint4 v = *reinterpret_cast<const uint4*>(box + sw128_offset(16 * kk + 2 * q + (i & 1) + 8 * (i >> 1), g));
                w[i][0] = v.x; w[i][1] = v.y; w[i][2] = v.z; w[i][3] = v.w;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t pick = e & 1 ? 0x7632u : 0x5410u;      // the odd or the even column of a pair, of two rows
                const uint32_t b0 = __byte_perm(w[0][e / 2], w[1][e / 2], pick), b1 = __byte_perm(w[2][e / 2], w[3][e / 2], pick);
#pragma unroll
                for (int m = 0; m < MT; ++m) mma_16x8x16(acc[m][e], &a[kk][4 * m], b0, b1);
            }
        }
        __syncwarp();                              // every lane has read the box
        if (lane == 0 && s + kFewDepth * kFewWarps < last) request(slot, s + kFewDepth * kFewWarps);
        if (++slot == kFewDepth) { slot = 0; phase ^= 1; }
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
#pragma unroll
            for (int i = 0; i < 4 * MT; ++i) a[kk][i] = next[kk][i];
    }
    __syncthreads();                               // the ring's place is free for the warps' sums
    if (*static_cast<volatile int*>(&abort_flag) != 0) {
        for (int i = 0; i < 64; ++i) __nanosleep(1000);      // copies that are still on their way land before the block's memory is given back
    }
    float(*part)[ROWS][kFewCols + 4] = reinterpret_cast<float(*)[ROWS][kFewCols + 4]>(boxes);
    // product e of column index n is column 8 n + e: a thread has columns 16 q .. 16 q + 15 of rows g and g + 8
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float* dst = &part[warp][16 * m + g + 8 * (i >> 1)][16 * q + 8 * (i & 1)];
            *reinterpret_cast<float4*>(dst) = make_float4(acc[m][0][i], acc[m][1][i], acc[m][2][i], acc[m][3][i]);
            *reinterpret_cast<float4*>(dst + 4) = make_float4(acc[m][4][i], acc[m][5][i], acc[m][6][i], acc[m][7][i]);
        }
    __syncthreads();
    float4 sum[MT];
    auto add = [](float4& s, const float4& v) { s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w; };
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int row = 16 * m + tid / (kFewCols / 4);
        sum[m] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (row < p.M) {
#pragma unroll
            for (int w = 0; w < kFewWarps; ++w) add(sum[m], *reinterpret_cast<const float4*>(&part[w][row][c4]));
        }
        if (SPLIT > 1) *reinterpret_cast<float4*>(&total[row][c4]) = sum[m];
    }
    if constexpr (SPLIT > 1) cluster_sync_all();
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int row = 16 * m + tid / (kFewCols / 4);
        if (!my_share || row >= p.M) continue;
        if constexpr (SPLIT > 1) {
            const uint32_t src = smem_u32(&total[row][c4]);
            float4 v[SPLIT];
#pragma unroll
            for (int r = 0; r < SPLIT; ++r) v[r] = ld_cluster_f4(mapa_u32(src, r));
            sum[m] = v[0];
#pragma unroll
            for (int r = 1; r < SPLIT; ++r) add(sum[m], v[r]);
        }
        uint64_t v[2] = {pack_f32x2(sum[m].x, sum[m].y), pack_f32x2(sum[m].z, sum[m].w)};
        if (p.bias) {
            v[0] = fadd2(v[0], p.bias_bf16 ? unpack_bf16x2(bias.x) : pack_f32x2(__uint_as_float(bias.x), __uint_as_float(bias.y)));
            v[1] = fadd2(v[1], p.bias_bf16 ? unpack_bf16x2(bias.y) : pack_f32x2(__uint_as_float(bias.z), __uint_as_float(bias.w)));
        }
        const long at = static_cast<long>(row) * p.N + c;
        uint32_t slope[2], out[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            if (p.gelu) v[e] = gelu_with_slope2(v[e], slope[e]);
            if (p.residual) v[e] = fadd2(v[e], unpack_bf16x2(e ? res[m].y : res[m].x));
            out[e] = pack_bf16_pair(v[e]);
        }
        *reinterpret_cast<uint2*>(p.y + at) = make_uint2(out[0], out[1]);
        if (p.slope) *reinterpret_cast<uint2*>(p.slope + at) = make_uint2(slope[0], slope[1]);
    }
    if constexpr (SPLIT > 1) cluster_sync_all();                           // no block leaves while another may still read its sums
}

}  // namespace ib200
