// bf16 GEMM with fp32 accumulation and an optional bias epilogue for sm_100a: the projections either side of
// attention (qkv = x Wqkv + b before it, y W_out + b after it), forward and backward.
//
// Replaces, for those two layers, the reference's Linear::forward = matmul(x, W) + b
// (src/inferno/modules/linear.cpp:99-106 -> cublas_mm_row_major, src/inferno/cuda/cudamatmul.cu:1058-1112, plus the
// broadcast add kernel, src/inferno/cuda/cudaadd.cu:20-142) and the two GEMMs of its backward, MMBackward
// (src/inferno/gradfn/mmbackward.cpp:36-98): dX = dY W^T and dW = X^T dY.  The reference materialises every transpose with
// a copy kernel; here a transposed operand is only a different shared-memory descriptor (MN-major instead of K-major).
//
//   C[M, N] = A[M, K] * B[K, N] (+ bias[N])
//   a_mn = 0: A stored [M rows, K contiguous]        a_mn = 1: A stored [K rows, M contiguous]  (A = X^T)
//   b_mn = 1: B stored [K rows, N contiguous]        b_mn = 0: B stored [N rows, K contiguous] (B = W^T)
//
// A pair of CTAs (cta_group::2) owns a 256 x 256 output tile, each CTA 128 of its rows.  Per k-step of 16 a CTA then reads
// 4 KB of A and 4 KB of B (its half of B's rows) for 128 x 256 products: with the copies that fill the ring, 128 bytes per
// clock of shared memory, exactly what the SM can move while the tensor pipe needs 128 clocks.  The one-CTA form of the same
// tile (128 x 256) moves 192 bytes per clock and was bound by it: 16384 x 768 x 2304 in 46.5 us against 36 us at the rate of
// a library GEMM.
//
// One warp of each CTA streams A / B k-slices of 64 through a TMA ring, one lane of the even CTA's MMA warp issues 256x256x16
// MMAs into one of two 256-column TMEM accumulators, and eight warps drain the other accumulator (TMEM -> registers -> +bias ->
// TMA store), so the epilogue of a tile overlaps the main loop of the next.
//
// Measured, us: 8192 x 1024 x 4096 47 (1470 TFLOP/s), with a residual 54, GELU 49, GELU with its slope kept 59; 16384 x 768 x 2304 43, 48, 47, 57.  The operands of a
// pair at the tensor pipe's full rate are 64 bytes per clock and SM, all that an SM takes from L2: what an epilogue reads or writes more is added.
//
// One launch runs up to two products ("tasks"), so that dX and dW of a projection share a grid:
//   task 0 is cut into whole tiles, dealt out round-robin;
//   task 1 is either cut the same way (its tiles follow task 0's), or, when it has too few tiles for the chip and a long K
//   (a weight gradient: K = tokens), into contiguous runs of k-slices, one per CTA pair, sized so that every pair ends up
//   with the same number of k-slices over both tasks.  The partial tiles meet by TMA reduction: in an fp32 workspace, zeroed
//   before and rounded once to bf16 afterwards by linear_finish_kernel, or, for callers without a workspace, in the zeroed
//   bf16 output itself (one rounding per partial, at most eight).  A forward with a fused epilogue,
//   and the dX of a few rows, are cut into equal parts, each with an fp32 matrix of its own, which linear_fused_finish_kernel adds up in
//   order: nothing to zero, and the result repeats.
#pragma once

#include <cuda_fp16.h>

#include <type_traits>

#include "sm100_ptx.cuh"

namespace ib200 {

// What the epilogue of task 0 does.  Each is a kernel of its own: a run-time branch would put every form's registers and code into the others.
enum : int {
    kEpiPlain = 0,         // c = acc; of parts of a tile, added up (with the bias in the first)
    kEpiResidual = 1,      // c = acc + bias + aux
    kEpiGelu = 2,          // z = acc + bias;  c = gelu(z) (+ aux);  gelu'(z) kept as fp16 if it is wanted
    kEpiSlope = 3,         // c = acc aux with aux = gelu'(z), and the column sums of c
    kEpiBias = 4,          // c = acc + bias, of whole tiles
    kEpiSlab = 5,          // c = acc; a part of a tile of task 1 goes to its slab
};
template <int EPI>
constexpr bool kEpiFused = EPI == kEpiResidual || EPI == kEpiGelu || EPI == kEpiSlope;

struct GemmTraits {
    static constexpr int BM = 256, BN = 256, BK = 64;            // tile of a CTA pair
    static constexpr int CM = BM / 2, CN = BN / 2;               // rows of A and of B that one CTA loads
    static constexpr int STAGES = 6;
    static constexpr int A_BYTES = CM * BK * 2;                  // 16 KB
    static constexpr int B_BYTES = CN * BK * 2;                  // 16 KB
    static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
    static constexpr int STAGING_BYTES = 32 * 128;               // epilogue staging of one warp
    static constexpr int EPI_WARPS = 8;                          // two per 32 rows of the tile, each with half of its columns
    static constexpr int THREADS = EPI_WARPS * 32 + 64;          // and the TMA warp and the MMA warp
    static constexpr uint32_t TM_COLS = 512;
};
// Shared memory of a kernel form.  The fused epilogues bring a second 4 KB tile per epilogue warp (what is added or multiplied, or the second
// output), which takes the place of one of the ring's six stages.
template <int EPI>
struct GemmSmem {
    static constexpr int STAGES = kEpiFused<EPI> ? 5 : GemmTraits::STAGES;
    static constexpr int OFF_OUT = STAGES * GemmTraits::STAGE_BYTES;
    static constexpr int OFF_AUX = OFF_OUT + GemmTraits::EPI_WARPS * GemmTraits::STAGING_BYTES;
    static constexpr int OFF_BAR = OFF_AUX + (kEpiFused<EPI> ? GemmTraits::EPI_WARPS * GemmTraits::STAGING_BYTES : 0);
    static constexpr int BYTES = OFF_BAR + 256 + 1024;
    static_assert(BYTES <= 232448, "shared memory budget");
    static_assert((2 * STAGES + 4 + GemmTraits::EPI_WARPS) * 8 + 8 <= 256, "barriers");
};

struct GemmTask {
    int M, N;
    int tiles_m, tiles;    // tiles = 0: no such task
    int k_slices;          // of 64
    int a_mn, b_mn;
    int band_tiles;        // tiles of a band of eight tile rows, and its reciprocal
    float band_inv;
};

enum : int { kPartWhole = 0, kPartReduceBf16 = 1, kPartReduceF32 = 2, kPartSlab = 3 };

struct GemmParams {
    GemmTask t[2];
    int split;             // task 1: kPartWhole, or how partial tiles are added up
    int slabs;             // kPartSlab: parts of a tile
    // split runs: pair c starts at k-slice total1 * (min(c, heavy) * w_heavy + max(0, c - heavy) * w_light) / w_total of task 1
    int heavy;
    long long w_heavy, w_light, w_total;
    const void* bias;      // [N] of task 0 (task 1 when it is the only one), or null
    int bias_bf16;
    int has_aux;           // kEpiGelu: a residual is added
    int keep_slope;        // kEpiGelu: gelu'(z) is kept
    float* colsum;         // kEpiSlope: column sums of each 32 rows, [ceil(M / 32)][N], or null
    int* status;
};

__host__ __device__ __forceinline__ int gemm_split_start(const GemmParams& p, int pair) {
    const long long total = static_cast<long long>(p.t[1].tiles) * p.t[1].k_slices;
    const long long w = (pair < p.heavy ? pair : p.heavy) * p.w_heavy + (pair > p.heavy ? pair - p.heavy : 0) * p.w_light;
    return static_cast<int>(total * w / p.w_total);
}

// The parts of one CTA pair, in order: its run of split task-1 slices first, then its whole tiles.
struct GemmPart {
    int task, m0, n0, ks0, ks1;
    bool partial;          // added to other parts of its tile
};
constexpr int kBandRows = 8;
struct GemmWalk {
    const GemmParams& p;
    int pair, pairs;
    int f, hi;             // split run
    int tile;              // next whole tile
    __device__ __forceinline__ GemmWalk(const GemmParams& prm, int pair_, int pairs_) : p(prm), pair(pair_), pairs(pairs_), f(0), hi(0), tile(pair_) {
        if (p.split != kPartWhole) {
            f = gemm_split_start(p, pair);
            hi = gemm_split_start(p, pair + 1);
        }
    }
    __device__ __forceinline__ bool next(GemmPart& q) {
        int t;
        if (f < hi) {
            const GemmTask& k = p.t[1];
            t = f / k.k_slices;
            q.task = 1;
            q.ks0 = f - t * k.k_slices;
            q.ks1 = min(k.k_slices, q.ks0 + (hi - f));
            q.partial = true;
            f += q.ks1 - q.ks0;
        } else {
            const int whole = p.t[0].tiles + (p.split == kPartWhole ? p.t[1].tiles : 0);
            if (tile >= whole) return false;
            q.task = tile < p.t[0].tiles ? 0 : 1;
            t = q.task ? tile - p.t[0].tiles : tile;
            q.ks0 = 0;
            q.ks1 = p.t[q.task].k_slices;
            q.partial = false;
            tile += pairs;
        }
        // tiles are numbered in bands of eight tile rows, so that the pairs at work share few rows of A and few columns of B in L2
        // (16384 x 768 x 2304 and 8192^3: 3 % and 5 % over one column of tiles after the other)
        // (the quotient by its reciprocal, put right by one where that was off: integer divisions cost an epilogue warp 500 cycles a tile)
        const GemmTask& k = p.t[q.task];
        int band = static_cast<int>(static_cast<float>(t) * k.band_inv), r = t - band * k.band_tiles;
        if (r < 0) { --band; r += k.band_tiles; }
        if (r >= k.band_tiles) { ++band; r -= k.band_tiles; }
        const int rows = min(kBandRows, k.tiles_m - band * kBandRows);
        const int down = rows == kBandRows ? r / kBandRows : r / rows;
        q.m0 = (band * kBandRows + r - down * rows) * GemmTraits::BM;
        q.n0 = down * GemmTraits::BN;
        return true;
    }
};

// The tensor maps of a launch: operands and outputs of the two tasks, and what a split task 1 is added into (its bf16 output,
// the fp32 accumulation workspace) or, slab by slab, stored to.
// aux: what a fused epilogue reads beside its tile; keep: where it leaves gelu'(z).
struct GemmMaps {
    CUtensorMap a[2], b[2], c[2], sum, aux, keep;
};

// Two columns of bias (col is even) as they are stored: converted where they are used, the load waits for nobody.
__device__ __forceinline__ uint2 load_bias2(const GemmParams& p, int col) {
    if (!p.bias_bf16) return *reinterpret_cast<const uint2*>(static_cast<const float*>(p.bias) + col);
    return make_uint2(*reinterpret_cast<const uint32_t*>(static_cast<const __nv_bfloat16*>(p.bias) + col), 0u);
}
__device__ __forceinline__ uint64_t bias_pair(const GemmParams& p, uint2 b) {
    return p.bias_bf16 ? pack_f32x2(__uint_as_float(b.x << 16), __uint_as_float(b.x & 0xffff0000u)) : pack_f32x2(__uint_as_float(b.x), __uint_as_float(b.y));
}

// gelu in its tanh form is z s(2u) with the logistic function s and u = sqrt(2 / pi) (z + 0.044715 z^3): 0.5 (1 + tanh u) = s(2u).  As one exponential
// and one reciprocal it keeps its relative precision where 1 + tanh u cancels, and both ends come out right without a branch (e^-2u is 0 or
// infinite).  Constants: -2 sqrt(2 / pi) log2 e, and that times 0.044715.
constexpr float kGeluExp1 = -2.302208198f, kGeluExp3 = kGeluExp1 * 0.044715f;
constexpr float kGeluDu1 = 1.595769122f, kGeluDu3 = kGeluDu1 * 3.f * 0.044715f;      // d(2u)/dz = kGeluDu1 + kGeluDu3 z^2
// Two at a time: the polynomials in packed fp32, an exponential and a reciprocal each (gelu of 64 elements a thread: about 290 issue slots, 510 one by one).
__device__ __forceinline__ uint64_t splat2(float a) { return pack_f32x2(a, a); }
__device__ __forceinline__ uint64_t gelu_gate2(uint64_t z, uint64_t zz) {            // s(2u)
    float a, b;
    unpack_f32x2(fmul2(z, ffma2(splat2(kGeluExp3), zz, splat2(kGeluExp1))), a, b);
    unpack_f32x2(fadd2(pack_f32x2(fast_exp2(a), fast_exp2(b)), splat2(1.f)), a, b);
    return pack_f32x2(fast_rcp(a), fast_rcp(b));
}
__device__ __forceinline__ uint64_t gelu2(uint64_t z) { return fmul2(z, gelu_gate2(z, fmul2(z, z))); }
// The backward needs gelu'(z) = s + z (2u)' s (1 - s) and nothing else of z, and all of it is at hand here, so the slope is what is kept, as
// fp16: off by 2^-11 of itself, an eighth of what the gradient loses when it is rounded to bf16, or by 2^-25 where it is below 2^-14 in magnitude (z under
// about -4.4: up to 2 % at z = -5, and 0 under about -5.6, where what reaches the gradient is 2^-25 of dy).  (With z kept as bf16 the gradients are half as far off
// again as their rounding leaves them, and with z kept in any type their kernels pay for the exponentials once more: 8192 x 4096, dy -> dz
// 62 us, 127 us for the product that does it in its epilogue.)  Beyond 16 the slope is 0 or 1 to the last bit, so z is limited
// there, where the formula would meet infinity times zero; a NaN is kept by s.
constexpr float kGeluFlat = 16.f;
__device__ __forceinline__ uint64_t gelu_with_slope2(uint64_t z, uint32_t& slope) {
    float a, b;
    unpack_f32x2(z, a, b);
    const uint64_t zc = pack_f32x2(clamp_abs(a, kGeluFlat), clamp_abs(b, kGeluFlat)), zz = fmul2(zc, zc);
    const uint64_t s = gelu_gate2(z, zz);
    unpack_f32x2(ffma2(fmul2(zc, ffma2(splat2(kGeluDu3), zz, splat2(kGeluDu1))), fmul2(s, ffma2(s, splat2(-1.f), splat2(1.f))), s), a, b);
    const __half2 h = __floats2half2_rn(a, b);
    slope = *reinterpret_cast<const uint32_t*>(&h);
    return fmul2(z, s);
}
__device__ __forceinline__ uint64_t unpack_half2(uint32_t w) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    return pack_f32x2(f.x, f.y);
}
__device__ __forceinline__ uint64_t unpack_bf16x2(uint32_t w) { return pack_f32x2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
__device__ __forceinline__ uint32_t pack_bf16_pair(uint64_t p) {
    float a, b;
    unpack_f32x2(p, a, b);
    return pack_bf16x2(a, b);
}

template <int EPI>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(GemmTraits::THREADS, 1)
gemm_bf16_kernel(const __grid_constant__ GemmMaps maps, const __grid_constant__ GemmParams prm) {
    using TR = GemmTraits;
    using SM = GemmSmem<EPI>;
    constexpr int BN = TR::BN, BK = TR::BK, NS = SM::STAGES, kTmaWarp = TR::EPI_WARPS, kMmaWarp = TR::EPI_WARPS + 1;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint8_t* sOut = smem + SM::OFF_OUT;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + SM::OFF_BAR);
    uint64_t* full = bars;                  // [NS]  TMA of both CTAs -> MMA (used in the even CTA)
    uint64_t* empty = full + NS;            // [NS]  MMA -> TMA (in both)
    uint64_t* acc_full = empty + NS;        // [2]   MMA -> epilogue (in both)
    uint64_t* acc_empty = acc_full + 2;     // [2]   the epilogues of both CTAs -> MMA (used in the even CTA)
    uint64_t* aux_full = acc_empty + 2;     // [EPI_WARPS]  TMA -> that warp (fused epilogues)
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(aux_full + TR::EPI_WARPS);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = cluster_ctarank();
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    ResidentAbortCtx ab{abort_flag, prm.status};

    if (tid == 0) {
        *abort_flag = 0;
        for (int s = 0; s < NS; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        for (int b = 0; b < 2; ++b) { mbar_init(&acc_full[b], 1); mbar_init(&acc_empty[b], 2 * TR::EPI_WARPS); }
        if (kEpiFused<EPI>)
            for (int w = 0; w < TR::EPI_WARPS; ++w) mbar_init(&aux_full[w], 1);
        fence_mbar_init();
    }
    if (warp == kMmaWarp) { tmem_alloc_pair(tmem_slot, TR::TM_COLS); tmem_relinquish_pair(); }
    if (warp == kTmaWarp && lane == 0) {
        for (int t = 0; t < 2; ++t)
            if (prm.t[t].tiles) { tma_prefetch_desc(&maps.a[t]); tma_prefetch_desc(&maps.b[t]); tma_prefetch_desc(&maps.c[t]); }
    }
    tc_fence_before_sync();
    cluster_sync_all();                     // the other CTA's barriers exist before anything signals them
    tc_fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    pdl_wait();

    GemmWalk walk(prm, pair, pairs);
    GemmPart q;
    if (warp == kTmaWarp) {
        // ------------------------------ TMA producer (each CTA loads its halves) ------------------------------
        // Like the MMA warp, this one stays converged and predicates the copies on an elected lane: a lone lane in a divergent
        // branch took 714 cycles to issue a k-slice, longer than the 512 the tensor pipe needs for it.
        const bool leader = elect_one_lane();
        uint32_t s = 0, phase = 0, used = 0;     // ring position
        const uint32_t full0 = mapa_u32(smem_u32(full), 0);
        while (walk.next(q)) {
            const GemmTask& k = prm.t[q.task];
            const CUtensorMap *ma = &maps.a[q.task], *mb = &maps.b[q.task];
            const int m0 = q.m0 + static_cast<int>(rank) * TR::CM, n0 = q.n0 + static_cast<int>(rank) * TR::CN;
            const bool a_mn = k.a_mn, b_mn = k.b_mn;
            for (int ks = q.ks0; ks < q.ks1; ++ks) {
                mbar_wait(&empty[s], phase ^ 1, ab, 10);
                const uint32_t bar = full0 + s * 8;
                uint8_t* sa = smem + s * TR::STAGE_BYTES;
                uint8_t* sb = sa + TR::A_BYTES;
                const int k0 = ks * BK;
                if (leader) {
                    if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * TR::STAGE_BYTES);
                    if (!a_mn) {
                        tma_load_3d_pair(sa, ma, bar, k0, m0, 0);                          // [128 m-rows x 64 k]
                    } else {
                        tma_load_3d_pair(sa, ma, bar, m0, k0, 0);                          // two panels [64 k-rows x 64 m]
                        tma_load_3d_pair(sa + BK * 128, ma, bar, m0 + 64, k0, 0);
                    }
                    if (!b_mn) {
                        tma_load_3d_pair(sb, mb, bar, k0, n0, 0);                          // [128 n-rows x 64 k]
                    } else {
                        tma_load_3d_pair(sb, mb, bar, n0, k0, 0);                          // two panels [64 k-rows x 64 n]
                        tma_load_3d_pair(sb + BK * 128, mb, bar, n0 + 64, k0, 0);
                    }
                }
                if (++s == NS) { s = 0; phase ^= 1; }
                if (used < NS) ++used;
            }
        }
        if (leader) pdl_trigger();
        // the last MMAs' arrivals on this CTA's empty barriers must have landed before the CTA leaves
        for (; used > 0; --used) {
            mbar_wait(&empty[s], phase ^ 1, ab, 11);
            if (++s == NS) { s = 0; phase ^= 1; }
        }
    } else if (warp == kMmaWarp) {
        // ------------------------------ MMA issuer (even CTA) ------------------------------
        // The warp stays converged; only the MMA / commit instructions are predicated on one elected lane (commits are
        // then free, where a lone lane in a divergent branch pays ~44 cycles of tensor-pipe time for each).
        if (rank == 0) {
            const bool leader = elect_one_lane();
            uint32_t s = 0, phase = 0, n = 0;
            for (; walk.next(q); ++n) {
                const GemmTask& k = prm.t[q.task];
                const uint32_t idesc = make_idesc(kFmtBF16, TR::BM, TR::BN, k.a_mn ? kMajorMN : kMajorK, k.b_mn ? kMajorMN : kMajorK);
                const uint32_t a_step = k.a_mn ? 2048u >> 4 : 32u >> 4, b_step = k.b_mn ? 2048u >> 4 : 32u >> 4;
                const uint32_t a_lo0 = sdesc_lo(smem_u32(smem), k.a_mn ? BK * 128 : 16), b_lo0 = sdesc_lo(smem_u32(smem + TR::A_BYTES), k.b_mn ? BK * 128 : 16);
                const uint32_t buf = n & 1, acc = tmem + buf * BN;
                mbar_wait_cluster(&acc_empty[buf], ((n >> 1) & 1) ^ 1, ab, 20);            // both epilogues have drained this accumulator
                tc_fence_after_sync();
                for (int ks = q.ks0; ks < q.ks1; ++ks) {
                    mbar_wait(&full[s], phase, ab, 21);
                    tc_fence_after_sync();
                    const uint32_t a_lo = a_lo0 + s * (TR::STAGE_BYTES >> 4), b_lo = b_lo0 + s * (TR::STAGE_BYTES >> 4);
#pragma unroll
                    for (int j = 0; j < BK / 16; ++j)
                        if (leader) umma_ss_f16_pair(acc, sdesc_join(a_lo + j * a_step), sdesc_join(b_lo + j * b_step), idesc, (ks != q.ks0) || j != 0);
                    if (leader) umma_commit_pair(&empty[s]);
                    if (++s == NS) { s = 0; phase ^= 1; }
                }
                if (leader) umma_commit_pair(&acc_full[buf]);
            }
        }
    } else {
        // ------------------------------ epilogue (32 rows a warp, half of the tile's columns) ------------------------------
        // Every warp works for itself: it stages 32 rows x 64 columns in its own 4 KB and has the TMA unit store them (or add them to the other parts
        // of the tile), so no barrier ties the warps together.  Registers straight to global memory (a 32-byte sector per thread) took 6200
        // cycles a tile, at three cycles per sector, and 2800 more in the release of the accumulator, which had to wait for the stores; four
        // warps that shared staging panels under named barriers took 7300.
        // The accumulator comes in one of two layouts:
        // - a row per lane (tmem_ld_x32) where nothing is done with it, and for the parts of a product that is cut, whose fp32 goes out 16 bytes a lane
        //   (backward of 1000 x 768 x 768, us: 15.0; pairs, stored 8 bytes at a time, 15.5; added in memory straight from the registers 16.1);
        // - pairs of columns of four rows (tmem_ld_16x256b_x8), the same columns in each, where there is an epilogue: a step's bias is eight shuffles, and
        //   the arithmetic is packed.  With a row per lane each element's bias came by a shuffle, and two warps a scheduler could not hide it all:
        //   15000 cycles a 256 x 256 tile with GELU and z, 10800 with a residual (8192 x 1024 x 4096: 69.7 and 56.8 us).
        // A kernel has one of them, but for kEpiSlope, which shares its launch with a weight gradient.  Code that a launch does not run slows down the
        // code that it does: backward of 2048 x 512 x 512, 1000 x 768 x 768 and 2048 x 768 x 256, whose dW is cut, us: 14.0, 15.1 and 13.8 with both layouts
        // in one kernel, 14.1, 15.0 and 13.6 with parts that are added up and slabs in one, 13.7, 14.7 and 12.9 apart.  Forward of
        // 2048 x 512 x 512 and 16384 x 768 x 768, whole tiles with a bias: 7.7 and 18.0 in one kernel, 7.4 and 17.8 apart.
        const int h = warp >> 2, row0 = (warp & 3) * 32;
        const uint32_t lane_base = static_cast<uint32_t>(row0) << 16;
        uint8_t* stage = sOut + warp * TR::STAGING_BYTES;
        uint8_t* second = smem + SM::OFF_AUX + warp * TR::STAGING_BYTES;      // fused forms: what is read beside the accumulator, or a second output
        const uint32_t free_bar[2] = {mapa_u32(smem_u32(&acc_empty[0]), 0), mapa_u32(smem_u32(&acc_empty[1]), 0)};
        const int colf = h * (BN / 2);
        auto tile_free = [&] {                                   // the last copies have read the staging tiles
            if (lane == 0) tma_store_wait_read_all();
            __syncwarp();
        };
        auto release = [&](uint32_t buf) {                       // every column of the accumulator is in registers: hand it back to the MMA warp
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster_relaxed(free_bar[buf]);
        };
        // 32 rows x 128 bytes, a row per lane: to their place, or added to what is there (rows and columns past M and N are clipped by the copy)
        auto stage_out = [&](const CUtensorMap* m, bool add, int col, int row, int z, const uint4 (&w)[8]) {
            tile_free();
#pragma unroll
            for (int c = 0; c < 8; ++c) st_shared_sw128(stage, lane, c, w[c]);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                if (add) tma_reduce_add_3d(m, stage, col, row, z);
                else tma_store_3d(m, stage, col, row, z);
                tma_store_commit();
            }
        };
        auto stage_out_f32 = [&](const uint32_t (&r)[2][32], int col, int row, int slab, int N) {
            uint4 w[8];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
#pragma unroll
                for (int c = 0; c < 8; ++c) w[c] = make_uint4(r[half][4 * c], r[half][4 * c + 1], r[half][4 * c + 2], r[half][4 * c + 3]);
                if (col + 32 * half < N) stage_out(&maps.sum, EPI != kEpiSlab, col + 32 * half, row, slab, w);
            }
        };
        uint32_t n = 0;
        if constexpr (EPI == kEpiPlain || EPI == kEpiSlab) {
            const int slab = EPI == kEpiSlab ? pair % prm.slabs : 0;
            for (; walk.next(q); ++n) {
                const GemmTask& k = prm.t[q.task];
                const uint32_t buf = n & 1;
                const int row = q.m0 + static_cast<int>(rank) * TR::CM + row0;
                const bool with_bias = EPI == kEpiPlain && prm.bias && q.ks0 == 0;       // the part that starts the tile's K range brings the bias in
                const bool f32_part = q.partial && (EPI == kEpiSlab || prm.split == kPartReduceF32);
                const CUtensorMap* mc = q.partial ? &maps.sum : &maps.c[q.task];
                // two columns of bias per lane and 64-column step, fetched under the wait and handed round by shuffles (broadcast loads in
                // the element loop queued behind the MMAs' operand reads for 2000 cycles and more)
                float2 bias0 = make_float2(0.f, 0.f), bias1 = bias0;
                if (with_bias) {
                    const int col = q.n0 + colf + 2 * lane;
                    if (col < k.N) unpack_f32x2(bias_pair(prm, load_bias2(prm, col)), bias0.x, bias0.y);
                    if (col + 64 < k.N) unpack_f32x2(bias_pair(prm, load_bias2(prm, col + 64)), bias1.x, bias1.y);
                }
                mbar_wait(&acc_full[buf], (n >> 1) & 1, ab, 30);
                tc_fence_after_sync();
#pragma unroll 1
                for (int c0 = colf; c0 < colf + BN / 2; c0 += 64) {
                    const int col = q.n0 + c0;
                    uint32_t v[2][32];
                    tmem_ld_x32(tmem + buf * BN + c0 + lane_base, v[0]);
                    tmem_ld_x32(tmem + buf * BN + c0 + 32 + lane_base, v[1]);
                    tmem_wait_ld();
                    if (c0 != colf) release(buf);
                    if (row >= k.M || col >= k.N) continue;
                    if (with_bias) {
                        const float2 bc = c0 != colf ? bias1 : bias0;
#pragma unroll
                        for (int e = 0; e < 64; ++e) v[e / 32][e % 32] = __float_as_uint(__uint_as_float(v[e / 32][e % 32]) + __shfl_sync(0xffffffffu, e & 1 ? bc.y : bc.x, e / 2));
                    }
                    if (f32_part) {
                        stage_out_f32(v, col, row, slab, k.N);
                        continue;
                    }
                    uint4 w[8];
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        const uint32_t* x = &v[c / 4][c % 4 * 8];
                        auto two = [&](int e) { return pack_bf16x2(__uint_as_float(x[e]), __uint_as_float(x[e + 1])); };
                        w[c] = make_uint4(two(0), two(2), two(4), two(6));
                    }
                    stage_out(mc, EPI == kEpiPlain && q.partial, col, row, 0, w);
                }
            }
        } else {
            const bool has_aux = EPI == kEpiResidual || EPI == kEpiSlope || (EPI == kEpiGelu && prm.has_aux);
            const int pair_col = 2 * (lane & 3);
            uint32_t aux_n = 0;
            auto request_aux = [&](const GemmPart& p, int c0) {      // the step's 32 x 64 tile; one at a time is on its way or being read
                const int row = p.m0 + static_cast<int>(rank) * TR::CM + row0, col = p.n0 + c0;
                if (has_aux && p.task == 0 && row < prm.t[0].M && col < prm.t[0].N && lane == 0) {
                    mbar_arrive_expect_tx(&aux_full[warp], TR::STAGING_BYTES);
                    tma_load_3d(second, &maps.aux, &aux_full[warp], col, row, 0);
                }
            };
            uint2 bias = make_uint2(0u, 0u);                         // of columns 2 lane, 2 lane + 1 of a step, handed round by shuffles
            auto request_bias = [&](const GemmPart& p, int c0) {
                const int col = p.n0 + c0 + 2 * lane;
                if (EPI != kEpiSlope && prm.bias && col < prm.t[p.task].N) bias = load_bias2(prm, col);
            };
            bool more = walk.next(q);
            if (more) {
                request_aux(q, colf);
                request_bias(q, colf);
            }
            for (; more; ++n) {
                const GemmTask& k = prm.t[q.task];
                const bool fused = kEpiFused<EPI> && q.task == 0;
                const uint32_t buf = n & 1;
                const int row = q.m0 + static_cast<int>(rank) * TR::CM + row0;
                const bool with_bias = EPI != kEpiSlope && prm.bias;
                const bool f32_part = EPI == kEpiSlope && q.partial;      // (dW beside it, in fp32; the other forms run whole tiles)
                mbar_wait(&acc_full[buf], (n >> 1) & 1, ab, 30);
                tc_fence_after_sync();
                GemmPart ahead;
                bool more_ahead = false;
#pragma unroll 1
                for (int c0 = colf; c0 < colf + BN / 2; c0 += 64) {
                    const int col = q.n0 + c0;
                    const bool inside = row < k.M && col < k.N, last = c0 != colf;
                    uint32_t r[2][32];
                    if (f32_part) {
                        tmem_ld_x32(tmem + buf * BN + c0 + lane_base, r[0]);
                        tmem_ld_x32(tmem + buf * BN + c0 + 32 + lane_base, r[1]);
                    } else {
                        tmem_ld_16x256b_x8(tmem + buf * BN + c0 + lane_base, r[0]);
                        tmem_ld_16x256b_x8(tmem + buf * BN + c0 + lane_base + (16u << 16), r[1]);
                    }
                    tmem_wait_ld();
                    if (last) release(buf);
                    if (f32_part && inside) stage_out_f32(r, col, row, 0, k.N);
                    // rows 8i + lane / 4, columns 8j + pair_col
                    uint64_t v[4][8];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const uint32_t* x = &r[i >> 1][4 * j + 2 * (i & 1)];
                            v[i][j] = pack_f32x2(__uint_as_float(x[0]), __uint_as_float(x[1]));
                        }
                    if (with_bias) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const uint32_t lo = __shfl_sync(0xffffffffu, bias.x, 4 * j + (lane & 3));
                            const uint64_t b = bias_pair(prm, make_uint2(lo, prm.bias_bf16 ? 0u : __shfl_sync(0xffffffffu, bias.y, 4 * j + (lane & 3))));
#pragma unroll
                            for (int i = 0; i < 4; ++i) v[i][j] = fadd2(v[i][j], b);
                        }
                    }
                    if (last) {
                        more_ahead = walk.next(ahead);
                        if (more_ahead) request_bias(ahead, colf);
                    } else {
                        request_bias(q, c0 + 64);
                    }
                    auto request_next_aux = [&] {                    // once every lane has read the tile that is there
                        if (!last) request_aux(q, c0 + 64);
                        else if (more_ahead) request_aux(ahead, colf);
                    };
                    if (!inside || !fused) request_next_aux();
                    if (!inside || f32_part) continue;
                    tile_free();
                    if (!fused) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const uint32_t w[4] = {pack_bf16_pair(v[0][j]), pack_bf16_pair(v[1][j]), pack_bf16_pair(v[2][j]), pack_bf16_pair(v[3][j])};
                            st_matrix_sw128(stage, lane, j, w);
                        }
                        fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) {
                            tma_store_3d(&maps.c[q.task], stage, col, row, 0);
                            tma_store_commit();
                        }
                        continue;
                    }
                    if constexpr (kEpiFused<EPI>) {
                        uint64_t sum[8];
                        // One body for each combination: with the choice made element by element no two exponentials overlap (8192 x 1024 x 4096 with GELU
                        // 53.7 -> 56.2 us, 16384 x 768 x 2304 54 -> 60).
                        auto form = [&](auto keep_, auto aux_) {
                            constexpr bool KEEP = decltype(keep_)::value, AUX = decltype(aux_)::value;
                            uint32_t w[8][4];
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                uint32_t slope[4], a[4];
                                if (AUX) ld_matrix_sw128(second, lane, j, a);
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    if (EPI == kEpiGelu) v[i][j] = KEEP ? gelu_with_slope2(v[i][j], slope[i]) : gelu2(v[i][j]);
                                    if (EPI == kEpiSlope) v[i][j] = fmul2(v[i][j], unpack_half2(a[i]));
                                    else if (AUX) v[i][j] = fadd2(v[i][j], unpack_bf16x2(a[i]));
                                    w[j][i] = pack_bf16_pair(v[i][j]);
                                }
                                if (EPI == kEpiSlope) sum[j] = fadd2(fadd2(v[0][j], v[1][j]), fadd2(v[2][j], v[3][j]));
                                if (KEEP) st_matrix_sw128(stage, lane, j, slope);
                                if (!KEEP || !AUX) st_matrix_sw128(KEEP ? second : stage, lane, j, w[j]);
                            }
                            fence_proxy_async_smem();
                            __syncwarp();
                            if (lane == 0) {
                                if (KEEP) tma_store_3d(&maps.keep, stage, col, row, 0);
                                if (!KEEP || !AUX) tma_store_3d(&maps.c[0], KEEP ? second : stage, col, row, 0);
                                tma_store_commit();
                            }
                            if (AUX) request_next_aux();
                            if (KEEP && AUX) {               // the second tile is the residual's: c goes out of the first one, behind the slope
                                tile_free();
#pragma unroll
                                for (int j = 0; j < 8; ++j) st_matrix_sw128(stage, lane, j, w[j]);
                                fence_proxy_async_smem();
                                __syncwarp();
                                if (lane == 0) {
                                    tma_store_3d(&maps.c[0], stage, col, row, 0);
                                    tma_store_commit();
                                }
                            }
                        };
                        if (has_aux) {
                            mbar_wait(&aux_full[warp], aux_n & 1, ab, 31);
                            ++aux_n;
                        }
                        constexpr std::true_type yes{};
                        constexpr std::false_type no{};
                        if constexpr (EPI != kEpiGelu) form(no, yes);
                        else if (prm.keep_slope) has_aux ? form(yes, yes) : form(yes, no);
                        else has_aux ? form(no, yes) : form(no, no);
                        if (EPI == kEpiSlope && prm.colsum) {
                            // the eight lanes that share columns add up their rows' sums, each ending with one of the eight pairs (rows past M are zeros)
#pragma unroll
                            for (int half = 4; half > 0; half >>= 1) {
                                const bool upper = lane & (4 * half);
#pragma unroll
                                for (int j = 0; j < half; ++j) {
                                    const uint64_t send = upper ? sum[j] : sum[j + half], keep = upper ? sum[j + half] : sum[j];
                                    sum[j] = fadd2(keep, __shfl_xor_sync(0xffffffffu, static_cast<unsigned long long>(send), 4 * half));
                                }
                            }
                            const int at = col + 8 * (lane >> 2) + pair_col;
                            if (at < k.N) *reinterpret_cast<uint64_t*>(prm.colsum + static_cast<long>(row >> 5) * k.N + at) = sum[0];
                        }
                    }
                }
                more = more_ahead;
                q = ahead;
            }
        }
        if (lane == 0) tma_store_wait_read_all();    // the CTA may leave once its shared memory has been read; the writes complete on their own
    }

    tc_fence_before_sync();
    __syncthreads();
    if (*abort_flag != 0) {
        for (int i = 0; i < 64; ++i) __nanosleep(1000);
    }
    cluster_sync_all();                     // neither CTA leaves while the other may still signal it or use its half of an MMA
    if (warp == kMmaWarp) tmem_dealloc_pair(tmem, TR::TM_COLS);
}

// The backward's helper ahead of the GEMMs: column sums of dY [M, N] (the bias gradient: the reference's sum_to_shape after
// the broadcast add, src/inferno/core/broadcastops.cpp) as one row of partial sums per row slab, and the zeroing of the
// fp32 accumulation workspace.  Block (x, y): 256 columns, rows y * rows_per_block ...; a warp reads 512 contiguous bytes
// of a row (16 bytes a lane) and keeps four rows in flight.  HBM-bound: one read of dY.
// SLOPE: x is dy, `slope` the kept gelu'(z); dz = dy slope is written for the two products that follow, and its columns, not dy's, are summed
// (before they are rounded): two reads and a write.
constexpr int kColsumCols = 256, kMaxColsumSlabs = 128;
template <bool SLOPE>
__global__ void __launch_bounds__(256) linear_prep_kernel(const __nv_bfloat16* __restrict__ x, const __half* __restrict__ slope, __nv_bfloat16* __restrict__ dz,
                                                          float* __restrict__ part, int M, int N, int rows_per_block, int atomic, float4* __restrict__ zero,
                                                          long zero4) {
    pdl_wait();
    pdl_trigger();
    // The accumulators are zeroed behind the reads where there are only reads, and ahead of them where dz is written as well: backward of
    // 8192 x 1024 x 4096 117.4 us (ahead: 120.2), with GELU 138.7 (behind: 141.2); 16384 x 768 x 768 with GELU 51.9 (54.1).
    auto clear = [&] {
        const long step = static_cast<long>(gridDim.x) * gridDim.y * blockDim.x;
        for (long i = (static_cast<long>(blockIdx.y) * gridDim.x + blockIdx.x) * blockDim.x + threadIdx.x; i < zero4; i += step) zero[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    };
    if (SLOPE || !part) clear();
    if (!SLOPE && !part) return;
    __shared__ float sums[8][kColsumCols + 4];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int col = blockIdx.x * kColsumCols + lane * 8;
    const int row1 = min(M, static_cast<int>(blockIdx.y + 1) * rows_per_block);
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    auto add = [&](const uint4& v) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            acc[2 * e] += __uint_as_float(w[e] << 16);
            acc[2 * e + 1] += __uint_as_float(w[e] & 0xffff0000u);
        }
    };
    if (SLOPE && col < N) {
        const uint4* src = reinterpret_cast<const uint4*>(x + col);
        const uint4* ssrc = reinterpret_cast<const uint4*>(slope + col);
        uint4* dst = reinterpret_cast<uint4*>(dz + col);
        const long pitch = N / 8;
        auto product = [&](long at, const uint4& g4, const uint4& s4) {
            const uint32_t g[4] = {g4.x, g4.y, g4.z, g4.w}, f[4] = {s4.x, s4.y, s4.z, s4.w};
            uint32_t o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float a, b;
                unpack_f32x2(fmul2(unpack_bf16x2(g[e]), unpack_half2(f[e])), a, b);
                acc[2 * e] += a;
                acc[2 * e + 1] += b;
                o[e] = pack_bf16x2(a, b);
            }
            dst[at] = make_uint4(o[0], o[1], o[2], o[3]);
        };
        int row = blockIdx.y * rows_per_block + warp;
        for (; row + 24 < row1; row += 32) {
            uint4 g[4], f[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                g[u] = src[(row + 8 * u) * pitch];
                f[u] = ssrc[(row + 8 * u) * pitch];
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) product((row + 8 * u) * pitch, g[u], f[u]);
        }
        for (; row < row1; row += 8) product(row * pitch, src[row * pitch], ssrc[row * pitch]);
    }
    if (!SLOPE && col < N) {
        const uint4* src = reinterpret_cast<const uint4*>(x + col);
        const long pitch = N / 8;
        int row = blockIdx.y * rows_per_block + warp;
        for (; row + 24 < row1; row += 32) {
            uint4 v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) v[u] = src[(row + 8 * u) * pitch];
#pragma unroll
            for (int u = 0; u < 4; ++u) add(v[u]);
        }
        for (; row < row1; row += 8) add(src[row * pitch]);
    }
    if (!part) return;
    if (!SLOPE) clear();
#pragma unroll
    for (int e = 0; e < 8; ++e) sums[warp][lane * 8 + e] = acc[e];
    __syncthreads();
    const int c = blockIdx.x * kColsumCols + threadIdx.x;
    if (c < N) {
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) s += sums[w][threadIdx.x];
        if (atomic) atomicAdd(part + c, s);                              // no workspace: the slabs meet in the zeroed output
        else part[static_cast<long>(blockIdx.y) * N + c] = s;
    }
}

// The backward's helper behind the GEMMs, for up to two projections: dW = bf16(fp32 accumulator), 8 elements per thread, and db = the sum
// of the row slabs' partial sums, in a fixed order.  The first `db_blocks` blocks of a job do its db, 32 columns each (eight threads a column).
constexpr int kFinishCols = 32;
struct FinishJob {
    const float4* acc;     // or null
    uint4* out;
    long n8;
    const float* part;     // [slabs][N]
    int slabs, N;
    void* db;              // or null
    int db_bf16, db_blocks;
};
struct FinishJobs {
    FinishJob j[2];
};
__global__ void __launch_bounds__(256) linear_finish_kernel(const __grid_constant__ FinishJobs jobs) {
    pdl_wait();
    pdl_trigger();
    const int all_db = jobs.j[0].db_blocks + jobs.j[1].db_blocks;
    if (static_cast<int>(blockIdx.x) < all_db) {
        const bool second = static_cast<int>(blockIdx.x) >= jobs.j[0].db_blocks;
        const FinishJob& k = jobs.j[second];
        __shared__ float sums[8][kFinishCols];
        const int lane = threadIdx.x & 31, grp = threadIdx.x >> 5, c = (blockIdx.x - (second ? jobs.j[0].db_blocks : 0)) * kFinishCols + lane;
        float s = 0.f;
        if (c < k.N)
#pragma unroll 4
            for (int j = grp; j < k.slabs; j += 8) s += k.part[static_cast<long>(j) * k.N + c];
        sums[grp][lane] = s;
        __syncthreads();
        if (grp == 0 && c < k.N) {
#pragma unroll
            for (int g = 1; g < 8; ++g) s += sums[g][lane];
            if (k.db_bf16) static_cast<__nv_bfloat16*>(k.db)[c] = __float2bfloat16(s);
            else static_cast<float*>(k.db)[c] = s;
        }
        return;
    }
    const long step = static_cast<long>(gridDim.x - all_db) * blockDim.x;
    const long first = (static_cast<long>(blockIdx.x) - all_db) * blockDim.x + threadIdx.x;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const FinishJob& k = jobs.j[q];
        if (!k.acc) continue;
        for (long i = first; i < k.n8; i += step) {
            const float4 a = k.acc[2 * i], b = k.acc[2 * i + 1];
            k.out[i] = make_uint4(pack_bf16x2(a.x, a.y), pack_bf16x2(a.z, a.w), pack_bf16x2(b.x, b.y), pack_bf16x2(b.z, b.w));
        }
    }
}

// Behind a product that was cut along K into slabs: their sum, and the epilogue on it, 8 elements per thread.
struct FusedFinish {
    const float4* acc;          // [slabs][M][N]
    int slabs;
    const void* bias;
    int bias_bf16, gelu;
    const uint4* residual;      // or null
    uint4* slope;               // gelu'(z), fp16, or null
    uint4* y;
    long n8;
    int N;
};
__global__ void __launch_bounds__(256) linear_fused_finish_kernel(const FusedFinish p) {
    pdl_wait();
    pdl_trigger();
    const long step = static_cast<long>(gridDim.x) * blockDim.x;
    for (long i = static_cast<long>(blockIdx.x) * blockDim.x + threadIdx.x; i < p.n8; i += step) {
        uint64_t v[4] = {0, 0, 0, 0};
#pragma unroll 4
        for (int j = 0; j < p.slabs; ++j) {
            const float4 a = p.acc[2 * (i + j * p.n8)], b = p.acc[2 * (i + j * p.n8) + 1];
            v[0] = fadd2(v[0], pack_f32x2(a.x, a.y));
            v[1] = fadd2(v[1], pack_f32x2(a.z, a.w));
            v[2] = fadd2(v[2], pack_f32x2(b.x, b.y));
            v[3] = fadd2(v[3], pack_f32x2(b.z, b.w));
        }
        const int col = static_cast<int>(i * 8 % p.N);
        uint32_t o[4];
        const uint4 r4 = p.residual ? p.residual[i] : make_uint4(0, 0, 0, 0);
        const uint32_t r[4] = {r4.x, r4.y, r4.z, r4.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (p.bias)
                v[e] = fadd2(v[e], p.bias_bf16 ? unpack_bf16x2(reinterpret_cast<const uint32_t*>(static_cast<const __nv_bfloat16*>(p.bias) + col)[e])
                                               : reinterpret_cast<const uint64_t*>(static_cast<const float*>(p.bias) + col)[e]);
            if (p.gelu) v[e] = gelu_with_slope2(v[e], o[e]);
        }
        if (p.slope) p.slope[i] = make_uint4(o[0], o[1], o[2], o[3]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (p.residual) v[e] = fadd2(v[e], unpack_bf16x2(r[e]));
            o[e] = pack_bf16_pair(v[e]);
        }
        p.y[i] = make_uint4(o[0], o[1], o[2], o[3]);
    }
}

}  // namespace ib200
