// Losses at the vocabulary projection (sm_100a): cross entropy and top-k
// distillation over logits z = H * W^T that are never kept, with the gradients
// of H and W.
//
// Mathematics. Row t of H (T x D) has the logits z_v = h_t . w_v. With
// p = softmax(z / tau) over the vocabulary and a sparse target distribution q
// (one token for the cross entropy, the softmax of a teacher's kept logits for
// the distillation; entries of one index add up)
//   loss_t = tau^2 * sum_k q_k (log q_k + lse_t - z_{i_k} / tau),
//   lse_t  = log sum_v exp(z_v / tau),
//   dloss_t / dz_v = tau * (p_v - q_v).
//
// Forward: one pass over W. A persistent tcgen05 GEMM computes 256-column
// tiles of z in TMEM; its epilogue keeps, for every row and tile, the running
// maximum m and s = sum exp((z - m) / tau) and copies out the logits at the
// row's targets. 8 bytes per (row, tile) leave the SM instead of 1024. A small
// kernel, in a small call the last block of the product, merges the tiles in order
// and forms the loss.
//
// Backward: the vocabulary is walked in pieces. For each piece, the logits are
// recomputed and turned into G = g_t (p - q) in 16 bits (T x piece), then
//   dH += G W_piece     (fp32, added piece after piece in stream order)
//   dW_piece = G^T H    (rounded once)
// G is the operand both products read, so it stays the operands' type: its
// rounding is half a step of the type for each term, which most of what a gradient is
// off by comes from (bf16: 1.9e-3 to 2.5e-3 of its norm, 1.7e-3 from rounding the
// result alone; fp16: 2.5e-4 to 3.0e-4 and 2.1e-4). In 32 bits, or as two numbers, it
// would double both products. The factor common to all rows
// is applied after the products, in 32 bits, so that |G| <= 1; half precision holds
// G times 2^14 (kHalfScale), since its steps below 2^-14 are 2^-24 wide whatever the
// value and most probabilities over a large vocabulary are there. Weights of the rows
// (a gradient for each row's loss) leave G as powers of two: bf16 has the exponents to
// hold them all the same; half precision does not, so there a row's power of two goes
// to its row of dH in 32 bits, and to dW on a copy of H (weigh_kernel).
//
// Rows without a target are gathered out first: they cost nothing, and what
// they hold (padding, infinities, NaN) meets no other row. W and H keep their
// row-major layout in all three products; where the contraction runs down the
// rows, the operand tile goes to the tensor cores in its MN-major form.
#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdlib>
#include <cstring>
#include <mutex>

#include <cuda_fp16.h>

#include "internal.h"
#include "ptx.cuh"

namespace b200 {
namespace vl {

constexpr int kBK = 64;
constexpr int kBN = 256;          // columns of a tile; 128 where wider ones leave SMs idle
constexpr int kRowsPerCta = 128;
// Eight epilogue warps, two for each TMEM quadrant (32 rows), each with half of
// the tile's columns. Four warps left the exponentials and the staging of a tile
// exposed up to D = 1024 (768 x 32000 x 64: 28 us for the statistics, 36 us for
// G).
constexpr int kEpiWarps = 8;
constexpr int kThreads = 64 + 32 * kEpiWarps;
constexpr int kEpiBufBytes = 32 * 128;
// k-slices between two drains of the statistics' accumulators. The tensor cores
// add to a 32-bit accumulator without rounding to nearest: over D = 4096 the lost
// bits add up to 5e-6 of a logit. Sums of 512 products (256 in single CTAs, whose
// calls wait for the weight anyway) are added up in registers instead, rounded to
// nearest. Sums of 1024 would be 1 % faster and as far off as a plain sum in 32 bits.
constexpr int kDrainMost = 8;
template <int kCtaGroup>
constexpr int kDrain = kCtaGroup == 1 ? 4 : kDrainMost;
constexpr int kQueue = 4;
constexpr int kNoCol = INT_MAX;
constexpr int kMaxTop = 256;      // teacher logits per row
constexpr int kMaxSplits = 16;    // runs of the contraction of dH or dW
constexpr float kLog2e = 1.4426950408889634f;
// G in half precision: 2^14 of its 65504 for 1, so full precision from 2^-28 on. 128256
// flat logits without it: dW of tokens that are no target off by a relative 2.1e-3
// instead of 2.2e-4.
constexpr float kHalfScale = 16384.0f;
// Limits of what a CTA waits for before it leaves: loads and products that it has
// started end within microseconds.
constexpr unsigned long long kLeaveNs = 10000000, kSettleNs = 50000;

// The products. Operands: Stats, Grad: A = H, B = W (both K-major); Dh: A = G
// (K-major), B = W (MN-major); Dw: A = G, B = H (both MN-major). StatsShort is
// Stats over at most kDrainMost k-slices, DwParts leaves runs of Dw's contraction
// as partial sums.
enum Op { kStats = 0, kStatsShort = 1, kGrad = 2, kDh = 3, kDw = 4, kDwParts = 5 };
__host__ __device__ constexpr bool is_stats(int op) { return op == kStats || op == kStatsShort; }
__host__ __device__ constexpr bool is_dw(int op) { return op == kDw || op == kDwParts; }

// What the first kernels of a call leave in the workspace for the others.
struct Head {
    int status;       // device status word
    int counter[4];   // tile scheduler: next tile, finished clusters; dW's own pair
    int g_piece;      // the last piece whose G is known to be complete, from 1
    int ticket;       // finished blocks of the merge kernel
    int n_rows;       // rows that the products run over
    int n_valid;      // rows with a loss, if the rows' kernel ran
    int compact;      // 1: the rows are those of the gathered copy of H
    float alpha;      // factor common to all rows of G, applied after the products
    int g_exponent;   // weights of rows: the exponent of the largest finite one
    unsigned h_most;  // and of the largest finite |h| 2^(row's exponent - g_exponent), its bits
};

// kSubM = 2 (Dw in pairs): a tile is two blocks of 256 rows that share their B
// operand, one in each accumulator: 48 KiB of operands for 2 x 4.2 MFLOP of a CTA
// instead of 32 KiB for 4.2. The start of a tile then waits for the last one's rows
// to be read out of TMEM, which dW's short epilogue allows (8192 rows x 32000 x 4096:
// 1312 against 1411 us) and G's exponentials do not (2000 x 50001 x 1024: 146 against
// 134 us).
template <int kCtaGroup, int kTileN, int kSubM = 1>
struct Cfg {
    static_assert(kTileN == kBN || (kTileN == 128 && kCtaGroup == 1), "unsupported tile width");
    static_assert(kSubM == 1 || (kSubM == 2 && kCtaGroup == 2), "unsupported tile height");
    static constexpr int kStages = kSubM == 2 || (kCtaGroup == 1 && kTileN == kBN) ? 4 : 6;
    static constexpr int kASubBytes = kRowsPerCta * kBK * 2;
    static constexpr int kABytes = kASubBytes * kSubM;
    static constexpr int kBRows = kTileN / kCtaGroup;
    static constexpr int kBBytes = kBRows * kBK * 2;
    static constexpr int kStageBytes = kABytes + kBBytes;
    static constexpr int kSubRows = kRowsPerCta * kCtaGroup;
    static constexpr int kTileM = kSubRows * kSubM;
    static constexpr int kEpiOffset = kStages * kStageBytes;
    static constexpr int kEpiBytes = kEpiWarps * kEpiBufBytes;
    static constexpr int kBarOffset = kEpiOffset + kEpiBytes;
    static constexpr int kBarCount = 2 * kStages + 5 + 2 * kQueue;
    static constexpr int kBarBytes = kBarCount * 8 + 16 + 4 * kQueue;
    static constexpr int kSmemBytes = kBarOffset + kBarBytes + 1024;
    static_assert(kStageBytes % 1024 == 0, "ring slots must keep 1024-byte alignment");
    static_assert(kSmemBytes <= 232448, "exceeds the 227 KB opt-in shared memory");
};

// Runs of a contraction over `slices` k-slices whose product has `tiles` tiles
// for `slots` clusters: the fewest k-slices on the longest cluster, with what a
// further run's sums cost to write and read again (in k-slices, 1 / 16ths).
__host__ __device__ inline unsigned runs_cost(unsigned s, unsigned tiles, unsigned slots, unsigned slices, unsigned run_cost16) {
    const unsigned rounds = (tiles * s + slots - 1) / slots;
    const unsigned long long cost =
        16ull * rounds * ((slices + s - 1) / s) + static_cast<unsigned long long>(run_cost16) * (s - 1);
    return cost < 0xfffffffeull ? static_cast<unsigned>(cost) : 0xfffffffeu;
}

// The rows that carry a loss are known on the device alone, so the kernels choose,
// all of them the same: a warp tries a number of runs per lane.
__device__ __forceinline__ int runs_for_warp(int tiles, int slots, int slices, int most, int run_cost16) {
    static_assert(kMaxSplits <= 32, "a lane for each number of runs");
    if (most == 1) return 1;
    const int s = static_cast<int>(threadIdx.x & 31) + 1;
    const unsigned cost = s <= min(most, slices) ? runs_cost(s, tiles, slots, slices, run_cost16) : 0xffffffffu;
    const unsigned least = __reduce_min_sync(0xffffffffu, cost);
    return __ffs(__ballot_sync(0xffffffffu, cost == least));
}

enum RowFlag { kNoLoss = 0, kLoss = 1, kBad = 2 };  // kBad: a target outside the vocabulary

constexpr int kMergeWarps = 8;

struct MergeParams {
    Head* head;
    const float2* part;
    long long part_ld;
    int tiles;            // half tiles
    int warps_per_row;    // merge_kernel: 1 or kMergeWarps
    int lanes;            // 0: merge_kernel follows; otherwise the product's last block merges, so many lanes a row
    int rows, top, reduction;
    int count;            // 1: nobody has counted the rows with a loss
    const int* inv;
    const int* flag;
    const float* eq;
    const float* zsel;
    float c2, inv_tau, tau2;
    float* lse;
    float* target_logp;    // [rows][top]
    float* row_loss;   // reduction none: the result
    float* loss;
};

struct Params {
    Head* head;
    unsigned long long timeout_ns;
    int fp16;             // operand type: 1 fp16, 0 bf16 (kHalf where it is packed)
    int rows;             // rows of the call
    int m;                // Dw: rows of the piece; otherwise from the head
    int n;                // columns of the product: piece (Stats, Grad) or D
    int k;                // contraction: D (Stats, Grad) or piece (Dh); Dw: from the head
    int v0;               // first vocabulary row of the piece
    int group_m;          // m-blocks per raster group
    int a_bytes;          // bytes of a block of A: rows beyond the call's are not loaded
    int early;            // Stats: the operands are the call's own, all rows in their order
    int splits;           // Dh, DwParts: runs of the contraction at most
    int run_slots;        // clusters that they are chosen for
    int run_slices;       // Dh: k-slices of the first piece (all pieces are cut alike)
    int run_cost16;
    int rows_pad;         // Dh, DwParts: rows between two splits' partial sums
    int accumulate;       // Dh: 1 add to the partial sums, 0 write them
    int piece_no;         // Dh, Dw, DwParts: the piece, from 1
    // Stats, Grad. One target per row (cross entropy): ecol and zsel (Stats) go by
    // the gathered row, rowmap and eq are null. A teacher's: by the row of the call.
    const int* rowmap;    // gathered row -> row
    const unsigned short* epos;  // [rows][epos_ld]: first entry at or behind each half tile
    long long epos_ld;
    const int* ecol;      // [rows][top] ascending target columns, kNoCol behind the last
    const float* eq;      // [rows][top] their probabilities
    float* zsel;          // Stats: [rows][top] logits at the targets; Grad: their log-probabilities
    float2* part;         // Stats: [gathered row][part_ld half tiles] (maximum, sum of exponentials)
    long long part_ld;
    const float4* rgrad;  // Grad: [gathered row] (g_t, -lse_t log2(e), g_t (p - 1) at the one target, its exponent), g_t in G's scale
    int top;
    float c2;             // log2(e) / tau
    MergeParams merge;    // Stats
};

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
}

// Shared-memory descriptor of an MN-major operand tile written by TMA in
// 64-column x 64-row boxes with 128-byte swizzle: atoms of 64 columns x 8 rows
// (1024 bytes) follow each other down the contraction (stride-dimension
// offset 1024), the next 64 columns start one box later (leading-dimension
// offset 8192).
__device__ __forceinline__ uint64_t smem_desc_mn_sw128(uint32_t smem_addr) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((smem_addr >> 4) & 0x3FFFu);
    d |= static_cast<uint64_t>(8192u >> 4) << 16;
    d |= static_cast<uint64_t>(1024u >> 4) << 32;
    d |= static_cast<uint64_t>(1u) << 46;
    d |= static_cast<uint64_t>(2u) << 61;
    return d;
}

// Arrival on a barrier of either CTA of the pair, ordered within the own CTA
// only: it hands back something that was read (a tile id, an accumulator), no
// written data. The cluster-scope release waits for every earlier store to
// global memory, about 1400 cycles per tile and warp.
__device__ __forceinline__ void mbar_arrive_pair(uint32_t cluster_bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}

// Four bytes into the peer's shared memory; they and the count on the peer's
// barrier arrive together, so the peer waits as for a TMA load.
__device__ __forceinline__ void st_async_u32(uint32_t cluster_addr, uint32_t v, uint32_t cluster_bar) {
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];"
                 ::"r"(cluster_addr), "r"(v), "r"(cluster_bar) : "memory");
}

// Two TMEM columns of the warp's 32 lanes.
__device__ __forceinline__ void tmem_ld_cols(uint32_t taddr0, uint32_t taddr1, float& z0, float& z1) {
    uint32_t r0, r1;
    __syncwarp();
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r0) : "r"(taddr0));
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r1) : "r"(taddr1));
    asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(r0), "+r"(r1)::"memory");
    z0 = __uint_as_float(r0);
    z1 = __uint_as_float(r1);
}

// Adds a staged fp32 box to global memory (each element once per launch, so
// the order of additions is the order of the launches).
__device__ __forceinline__ void tma_reduce_add_2d(const void* tmap, uint32_t src, int32_t x, int32_t y) {
    asm volatile(
        "cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3}], [%1];"
        ::"l"(reinterpret_cast<uint64_t>(tmap)), "r"(src), "r"(x), "r"(y)
        : "memory");
}

__device__ __forceinline__ void st_release_gpu(int* addr, int v) {
    asm volatile("st.release.gpu.global.b32 [%0], %1;" ::"l"(addr), "r"(v) : "memory");
}

// Global memory seen by ordinary loads so far is seen by TMA loads from here on.
__device__ __forceinline__ void fence_proxy_async() { asm volatile("fence.proxy.async.global;" ::: "memory"); }

// Time for what went to the other CTA of the pair, or is counted there, to land.
__device__ __forceinline__ void settle() {
    const uint64_t t0 = globaltimer_ns();
    for (int i = 0; i < 100000 && globaltimer_ns() - t0 < kSettleNs; ++i) __nanosleep(1000);
}

// 2^x by the hardware's approximation (off by about 2^-22 of the result, results
// below 2^-126 are zeros): every use is a term of a sum of exponentials or a
// probability.
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The smaller one; NaN where either is.
__device__ __forceinline__ float min_nan(float a, float b) {
    float y;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

// The reference point of a sum of exponentials: the maximum, or 0 where it is
// infinite (all terms are then 0, or one is infinite, without a NaN from
// inf - inf).
__device__ __forceinline__ float finite_or_zero(float m) { return fabsf(m) == INFINITY ? 0.0f : m; }

// What a sum of exponentials against `from` is multiplied by to stand against `to`.
// A sum against -inf is empty: nothing, not 0 times the overflow of exp(0 - to).
__device__ __forceinline__ float rescale(float from, float to, float c2) {
    return from == -INFINITY ? 0.0f : exp2_approx((finite_or_zero(from) - finite_or_zero(to)) * c2);
}

// Half tiles j0, j0 + step, ... of a row: the maximum first, then the sums against
// it, eight at a time. What other blocks wrote is read from L2.
__device__ __forceinline__ void merge_parts(const MergeParams& p, int i, int j0, int step, float& m, float& s) {
    const float2* part = p.part + i * p.part_ld;
    for (; j0 < p.tiles; j0 += 8 * step) {
        float2 v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
            v[j] = j0 + j * step < p.tiles ? __ldcg(part + j0 + j * step) : make_float2(-INFINITY, 0.0f);
        float mx = m;
#pragma unroll
        for (int j = 0; j < 8; ++j) mx = fmaxf(mx, v[j].x);
        s *= rescale(m, mx, p.c2);
#pragma unroll
        for (int j = 0; j < 8; ++j) s += v[j].y * rescale(v[j].x, mx, p.c2);
        m = mx;
    }
}

// The same over groups of `lanes` lanes.
__device__ __forceinline__ void merge_lanes(const MergeParams& p, int lanes, float& m, float& s) {
    float mx = m;
    for (int o = lanes / 2; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    s *= rescale(m, mx, p.c2);
    for (int o = lanes / 2; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    m = mx;
}

// A row's results by a group of lanes from its flag, its gathered number and the
// logit at its one target; `row` beyond the last: nothing to write.
__device__ __forceinline__ void merge_row(const MergeParams& p, int row, int f, float z_one, int i, bool failed, float m,
                                          float s, int lane, int lanes) {
    // Log-probabilities at the targets as differences from the maximum: next to lse,
    // which is rounded to its own size, those near 0 would be lost.
    const float ref = finite_or_zero(m), logs = logf(s);
    const bool there = row < p.rows;
    // A launch that was given up leaves no number that a backward pass could go on from.
    if (there && lane == 0) p.lse[row] = failed ? NAN : (i >= 0 ? logs + ref * p.inv_tau : 0.0f);
    float v = 0.0f;
    if (f == kLoss && p.eq == nullptr) {
        v = logs - (z_one - ref);
        if (lane == 0) p.target_logp[row] = -v;
    } else if (f != kLoss) {
        // Nothing reads these, but no output keeps what was in its memory.
        if (there)
            for (int k = lane; k < p.top; k += lanes) p.target_logp[static_cast<long long>(row) * p.top + k] = 0.0f;
    } else {
        const long long e = static_cast<long long>(row) * p.top;
        for (int k = lane; k < p.top; k += lanes) {
            const float qv = p.eq[e + k];
            const float logp = (__ldcg(p.zsel + e + k) - ref) * p.inv_tau - logs;
            p.target_logp[e + k] = logp;
            if (qv != 0.0f) v += qv * (logf(qv) - logp);
        }
    }
    if (p.eq != nullptr) {
        for (int o = lanes / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        v *= p.tau2;
    }
    // A target outside the vocabulary, or a launch that was given up, is no number.
    if (f == kBad || failed) v = NAN;
    if (there && lane == 0) p.row_loss[row] = v;
}

// The rows' sum, and their mean over those with a loss, by one block; in 64 bits,
// which over many rows keeps the rows' own precision.
template <int kBlock>
__device__ __forceinline__ void merge_sum(const MergeParams& p, double (&sums)[kBlock / 32], int (&counts)[kBlock / 32]) {
    double sum = 0.0;
    for (int r = threadIdx.x; r < p.rows; r += kBlock) sum += static_cast<double>(__ldcg(p.row_loss + r));
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    int n = 0;
    if (p.count) {
        for (int r = threadIdx.x; r < p.rows; r += kBlock) n += p.flag[r] != kNoLoss;
        n = __reduce_add_sync(0xffffffffu, n);
    }
    if (threadIdx.x % 32 == 0) {
        sums[threadIdx.x / 32] = sum;
        counts[threadIdx.x / 32] = n;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kBlock / 32; ++w) {
            sum += sums[w];
            n += counts[w];
        }
        if (p.reduction == B200_VL_MEAN) sum /= max(p.count ? n : p.head->n_valid, 1);
        *p.loss = static_cast<float>(sum);
    }
}

template <int kCtaGroup, int kTileN, int kOp, bool kHalf, int kSubM>
__global__ void __launch_bounds__(kThreads, 1)
vocab_gemm_kernel(const __grid_constant__ CUtensorMap tmA0, const __grid_constant__ CUtensorMap tmA1,
                  const __grid_constant__ CUtensorMap tmB0, const __grid_constant__ CUtensorMap tmB1,
                  const __grid_constant__ CUtensorMap tmD, const Params p) {
    using C = Cfg<kCtaGroup, kTileN, kSubM>;
    static_assert(kSubM == 1 || kOp == kDw, "one accumulator is read while the other is filled");
    constexpr int kStages = C::kStages;
    constexpr int kHalfN = kTileN / 2;
    constexpr int kTmemCols = 2 * kTileN;  // two accumulators
    constexpr bool kPair = kCtaGroup == 2;
    constexpr int kDrain = vl::kDrain<kCtaGroup>;
    constexpr bool kAMn = is_dw(kOp);
    constexpr bool kBMn = kOp == kDh || is_dw(kOp);
    constexpr int kBoxBytes = 64 * kBK * 2;  // an MN-major box

    int* const status_word = &p.head->status;
    // Launch contract: uniform across the grid, checked before any barrier.
    if (blockDim.x != kThreads || blockDim.y != 1 || blockDim.z != 1 ||
        (kPair && cluster_nctarank() != 2) || (gridDim.x % kCtaGroup) != 0) {
        if (threadIdx.x == 0) report_status(status_word, B200_DEV_BAD_LAUNCH);
        return;
    }

    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                               ~static_cast<uintptr_t>(1023));
    const uint32_t sbase = smem_u32(smem);
    const uint32_t full0 = sbase + C::kBarOffset;
    const uint32_t empty0 = full0 + 8 * kStages;
    const uint32_t tfull0 = empty0 + 8 * kStages;
    const uint32_t tempty0 = tfull0 + 16;
    const uint32_t qfull0 = tempty0 + 16;
    const uint32_t qempty0 = qfull0 + 8 * kQueue;
    const uint32_t done0 = qempty0 + 8 * kQueue;  // the products' end, for their issuer alone
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::kBarOffset + C::kBarCount * 8);
    volatile int* ring = reinterpret_cast<volatile int*>(smem + C::kBarOffset + C::kBarCount * 8 + 16);
    const uint32_t ring_addr = smem_u32(const_cast<int*>(ring));

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t rank = kPair ? cluster_ctarank() : 0;
    const int num_clusters = gridDim.x / kCtaGroup;
    const int cluster = blockIdx.x / kCtaGroup;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(full0 + 8 * s, 1);
            mbar_init(empty0 + 8 * s, 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(tfull0 + 8 * a, 1);
            mbar_init(tempty0 + 8 * a, kEpiWarps * kCtaGroup);
        }
        // A queued tile id is read by the MMA issuer and the epilogue warps of the
        // leader, and in pair mode also by the peer's producer and epilogue warps.
        for (int q = 0; q < kQueue; ++q) {
            mbar_init(qfull0 + 8 * q, 1);
            mbar_init(qempty0 + 8 * q, (kEpiWarps + 1) * kCtaGroup);
        }
        mbar_init(done0, 1);
        fence_barrier_init();
        // The peer's slots are filled by asynchronous stores, each armed before the
        // leader may write it.
        if (rank == 1)
            for (int q = 0; q < kQueue; ++q) mbar_arrive_expect_tx(qfull0 + 8 * q, 4);
    }
    if (warp == 0 && lane == 0) {
        tma_prefetch_desc(&tmA0);
        tma_prefetch_desc(&tmB0);
        if (!is_stats(kOp)) tma_prefetch_desc(&tmD);
    }
    if (warp == 1) {
        tmem_alloc<kCtaGroup>(smem_u32(tmem_slot), kTmemCols);
        tmem_relinquish<kCtaGroup>();
    }
    tc_fence_before();
    if constexpr (kPair) cluster_sync(); else __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
    // Nothing in global memory is touched before the previous kernel is done, with
    // one exception: where the operands are the call's own and no row is left out
    // (early), the first tile is loaded and multiplied meanwhile. The kernels before
    // this one in the call write neither, and the first of them began when everything
    // before the call was done. Each role then waits before it touches the workspace, the
    // status word included (a 512^3 forward pass as a graph: 16.5 -> 14.5 us).
    const bool early = is_stats(kOp) && p.early;
    int* status = early ? nullptr : status_word;
    if constexpr (is_dw(kOp)) {
        // dW needs G and not the product before it, which is dH: it fills the SMs that
        // dH leaves, and waits for dH's end at its own (512^3 step as a graph: 43.1 ->
        // 39.0 us; 8192 x 128256 x 4096: 25.15-25.33 -> 24.99 ms). dH is launched
        // first, waits for G and says so; without its word, dW waits for all that came
        // before.
        if (ld_acquire_gpu(&p.head->g_piece) != p.piece_no) griddep_wait();
        fence_proxy_async();
    } else if (!early) {
        griddep_wait();
    }
    if constexpr (kOp == kDh) {
        if (threadIdx.x == 0) {
            if (blockIdx.x == 0) st_release_gpu(&p.head->g_piece, p.piece_no);
            griddep_launch_dependents();
        }
    }
    int* const counter = p.head->counter + (is_dw(kOp) ? 2 : 0);

    const int n_rows = early ? p.rows : p.head->n_rows;
    const bool compact = !early && p.head->compact != 0;
    // Of H, the gathered copy where rows were left out. Without a single row the
    // products still run over one block of zero rows: dW is then written as zeros.
    const CUtensorMap* tmA = ((is_stats(kOp) || kOp == kGrad) && compact) ? &tmA1 : &tmA0;
    const CUtensorMap* tmB = (is_dw(kOp) && compact) ? &tmB1 : &tmB0;
    const int m_ext = is_dw(kOp) ? p.m : (is_stats(kOp) ? n_rows : max(n_rows, 1));
    const int k_ext = is_dw(kOp) ? max(n_rows, 1) : p.k;
    const int num_m = (m_ext + C::kTileM - 1) / C::kTileM;
    const int num_n = (p.n + kTileN - 1) / kTileN;
    const int num_k = (k_ext + kBK - 1) / kBK;
    const int tiles_mn = num_m * num_n;
    constexpr bool kSplit = kOp == kDh || kOp == kDwParts;
    const int splits =
        kSplit ? runs_for_warp(tiles_mn, p.run_slots, kOp == kDh ? p.run_slices : num_k, p.splits, p.run_cost16) : 1;
    const int num_tiles = tiles_mn * splits;

    // Tile id -> blocks and k-slices. Groups of m-blocks walk all n-blocks, so
    // the tiles in flight share rows of both operands in L2.
    struct Tile {
        int mb, nb, kb0, kb1, split;
        int subs;  // blocks of rows that the tile has
    };
    auto tile_of = [&](int t) {
        Tile w;
        w.split = 0;
        w.kb0 = 0;
        w.kb1 = num_k;
        if constexpr (kSplit) {
            w.split = t / tiles_mn;
            t -= w.split * tiles_mn;
            w.kb0 = static_cast<int>(static_cast<long long>(num_k) * w.split / splits);
            w.kb1 = static_cast<int>(static_cast<long long>(num_k) * (w.split + 1) / splits);
        }
        const int per_group = p.group_m * num_n;
        const int g = t / per_group;
        const int first = g * p.group_m;
        const int gsize = min(p.group_m, num_m - first);
        const int r = t - g * per_group;
        w.mb = first + r % gsize;
        w.nb = r / gsize;
        w.subs = kSubM == 1 || m_ext - w.mb * C::kTileM <= C::kSubRows ? 1 : 2;
        return w;
    };
    auto queue_wait = [&](uint32_t qs, uint32_t qph, int code) -> bool {
        return mbar_wait(qfull0 + 8 * qs, qph, status, p.timeout_ns, code);
    };
    auto queue_release = [&](uint32_t qs) {
        if constexpr (kPair) mbar_arrive_pair(mapa_shared(qempty0 + 8 * qs, 0));
        else mbar_arrive(qempty0 + 8 * qs);
    };

    if (warp == 0) {
        // ------------------------------------------------------------ producer
        if (elect_one()) {
            uint32_t stage = 0, phase = 0, qs = 0, qph = 0;
            long long issued = 0;
            bool ok = true;
            // The first tile is the cluster's own number, later ones come from the
            // launch-wide counter.
            int next = cluster;
            bool waited = !early;
            bool ended = false;  // every tile has been loaded
            while (ok) {
                int t;
                if (rank == 0) {
                    if (!mbar_wait(qempty0 + 8 * qs, qph ^ 1, status, p.timeout_ns,
                                   B200_DEV_TIMEOUT_PRODUCER)) {
                        break;
                    }
                    t = next;
                    if (t >= num_tiles) {
                        t = -1;
                        if (!waited) griddep_wait();
                        __threadfence();
                        if (atomicAdd(&counter[1], 1) == num_clusters - 1) {
                            // Every cluster has made its last fetch: ready for the next launch.
                            atomicExch(&counter[0], 0);
                            atomicExch(&counter[1], 0);
                        }
                    }
                    ring[qs] = t;
                    if constexpr (kPair)
                        st_async_u32(mapa_shared(ring_addr + 4 * qs, 1), static_cast<uint32_t>(t),
                                     mapa_shared(qfull0 + 8 * qs, 1));
                    mbar_arrive(qfull0 + 8 * qs);
                } else {
                    if (!queue_wait(qs, qph, B200_DEV_TIMEOUT_PRODUCER)) break;
                    t = ring[qs];
                    // Armed for the slot's next turn before the slot is handed back.
                    if (t >= 0) mbar_arrive_expect_tx(qfull0 + 8 * qs, 4);
                    queue_release(qs);
                }
                if (++qs == kQueue) { qs = 0; qph ^= 1; }
                if (t < 0) {
                    ended = true;
                    griddep_launch_dependents();
                    break;
                }
                const Tile w = tile_of(t);
                const int a_m = w.mb * C::kTileM + static_cast<int>(rank) * kRowsPerCta;
                const int b_n = w.nb * kTileN + static_cast<int>(rank) * C::kBRows;
                // The next tile id is fetched two ring depths before the last k-slice:
                // early enough to hide the round trip, late enough that a fast cluster
                // does not take two tiles while a slow one has none.
                const int fetch_kb = max(w.kb0, w.kb1 - 2 * kStages);
                // Single CTAs, which a small number of rows takes, stream W from HBM: each
                // tile starts at another column, so that those in flight do not all read
                // the same 128 bytes of rows a power of two apart (one token over 128256 x
                // 4096: 185.3 against 195.6 us, 64 tokens 193.5 and 197.6; other widths
                // alike).
                int turn = 0;
                if constexpr (!kPair && !kBMn) turn = static_cast<int>(13u * w.nb % static_cast<unsigned>(num_k));
                if (rank == 0 && w.kb0 == w.kb1) next = atomicAdd(&counter[0], 1) + num_clusters;
                for (int kb = w.kb0; kb < w.kb1; ++kb) {
                    if (rank == 0 && kb == fetch_kb && waited) next = atomicAdd(&counter[0], 1) + num_clusters;
                    if (!mbar_wait(empty0 + 8 * stage, phase ^ 1, status, p.timeout_ns,
                                   B200_DEV_TIMEOUT_PRODUCER)) {
                        ok = false;
                        break;
                    }
                    const uint32_t sa = sbase + stage * C::kStageBytes;
                    const uint32_t sb = sa + C::kABytes;
                    const uint32_t fb = full0 + 8 * stage;
                    const uint32_t bar = kPair ? mapa_shared(fb, 0) : fb;
                    if (rank == 0) mbar_arrive_expect_tx(fb, kCtaGroup * (p.a_bytes * w.subs + C::kBBytes));
                    auto load = [&](uint32_t dst, const CUtensorMap* map, int x, int y) {
                        if constexpr (kPair) tma_load_2d_pair(dst, map, bar, x, y);
                        else tma_load_2d(dst, map, bar, x, y);
                    };
                    const int kc = (kb + turn < w.kb1 ? kb + turn : kb + turn - num_k) * kBK;
#pragma unroll
                    for (int sm = 0; sm < kSubM; ++sm) {
                        if (sm >= w.subs) break;
                        const uint32_t dst = sa + sm * C::kASubBytes;
                        const int row = a_m + sm * C::kSubRows;
                        if constexpr (kAMn) {
#pragma unroll
                            for (int i = 0; i < kRowsPerCta / 64; ++i)
                                load(dst + i * kBoxBytes, tmA, row + 64 * i, kc);
                        } else {
                            load(dst, tmA, kc, row);
                        }
                    }
                    if constexpr (kBMn) {
                        const int y = kOp == kDh ? p.v0 + kc : kc;
#pragma unroll
                        for (int i = 0; i < C::kBRows / 64; ++i)
                            load(sb + i * kBoxBytes, tmB, b_n + 64 * i, y);
                    } else {
                        load(sb, tmB, kc, p.v0 + b_n);
                    }
                    ++issued;
                    if (++stage == kStages) { stage = 0; phase ^= 1; }
                }
                if (!waited) {
                    griddep_wait();
                    status = status_word;
                    waited = true;
                    if (rank == 0) next = atomicAdd(&counter[0], 1) + num_clusters;
                }
            }
            if (!waited) griddep_wait();
            // This CTA (pair) leaves only when the loads into its ring have landed. At a
            // normal end the other roles wait longer than that anyway; where one of them
            // has given up, perhaps without a status word to say so, this is the only wait.
            if (rank == 0) {
                for (int s = 0; s < kStages; ++s) {
                    if (issued <= s) continue;
                    const long long last = ((issued - 1 - s) / kStages) * kStages + s;
                    mbar_wait(full0 + 8 * s, static_cast<uint32_t>((last / kStages) & 1), nullptr, kLeaveNs, 0);
                }
            }
            // A peer that has run ahead of a leader that gave up has loads that no barrier
            // counts, and a leader may have sent it a tile id just now.
            if (kPair && (!ended || status_failed(status_word))) settle();
        }
        __syncwarp();
    } else if (warp == 1) {
        // --------------------------------------------------------- MMA issuer
        if (rank == 0 && elect_one()) {
            const uint32_t fmt = p.fp16 ? 0u : 1u;
            const uint32_t idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | ((kAMn ? 1u : 0u) << 15) |
                                   ((kBMn ? 1u : 0u) << 16) | ((kTileN >> 3) << 17) |
                                   (((kRowsPerCta * kCtaGroup) >> 4) << 24);
            uint32_t stage = 0, phase = 0, unit = 0, qs = 0, qph = 0;
            bool ok = true;
            while (ok) {
                if (!queue_wait(qs, qph, B200_DEV_TIMEOUT_MMA_FULL)) break;
                const int t = ring[qs];
                queue_release(qs);
                if (++qs == kQueue) { qs = 0; qph ^= 1; }
                if (t < 0) break;
                const Tile w = tile_of(t);
                if (w.kb0 == w.kb1) continue;
                // The products of a block of rows with the k-slice in ring slot `st`.
                auto multiply = [&](uint32_t slot, int sm, uint32_t st, bool first) {
                    const uint32_t sa = sbase + st * C::kStageBytes + sm * C::kASubBytes;
                    const uint32_t sb = sbase + st * C::kStageBytes + C::kABytes;
#pragma unroll
                    for (int k = 0; k < kBK / 16; ++k) {
                        // 16 elements down the contraction: 32 bytes inside a K-major row,
                        // 16 rows of 128 bytes in an MN-major box.
                        const uint64_t da = kAMn ? smem_desc_mn_sw128(sa + 2048 * k) : smem_desc_sw128(sa + 32 * k);
                        const uint64_t db = kBMn ? smem_desc_mn_sw128(sb + 2048 * k) : smem_desc_sw128(sb + 32 * k);
                        umma_bf16<kCtaGroup>(tmem_base + slot * kTileN, da, db, idesc, !first || k != 0 ? 1u : 0u);
                    }
                };
                auto commit = [&](uint32_t bar) {
                    if constexpr (!kPair) {
                        umma_commit<1>(bar);
                    } else {
                        umma_commit<2>(mapa_shared(bar, 0));
                        umma_commit<2>(mapa_shared(bar, 1));
                    }
                };
                auto wait_slot = [&](uint32_t u) -> bool {
                    if (!mbar_wait(tempty0 + 8 * (u & 1), ((u >> 1) & 1) ^ 1, status, p.timeout_ns,
                                   B200_DEV_TIMEOUT_MMA_TMEM)) {
                        return false;
                    }
                    tc_fence_after();
                    return true;
                };
                auto wait_full = [&](uint32_t st, uint32_t ph) -> bool {
                    if (!mbar_wait(full0 + 8 * st, ph, status, p.timeout_ns, B200_DEV_TIMEOUT_MMA_FULL)) return false;
                    tc_fence_after();
                    return true;
                };
                auto next_stage = [&](uint32_t& st, uint32_t& ph) {
                    if (++st == kStages) { st = 0; ph ^= 1; }
                };
                if (kSubM == 1 || w.subs == 1) {
                    for (int kb = w.kb0; kb < w.kb1; ++kb) {
                        // A unit is what one accumulator sums up: the whole contraction, or
                        // kDrain k-slices of it for the statistics.
                        const int in_unit = kOp == kStats ? (kb - w.kb0) % kDrain : kb - w.kb0;
                        ok = (in_unit != 0 || wait_slot(unit)) && wait_full(stage, phase);
                        if (!ok) break;
                        multiply(unit & 1, 0, stage, in_unit == 0);
                        commit(empty0 + 8 * stage);
                        next_stage(stage, phase);
                        if (kb + 1 == w.kb1 || (kOp == kStats && in_unit == kDrain - 1)) {
                            commit(tfull0 + 8 * (unit & 1));
                            ++unit;
                        }
                    }
                } else {
                    // Two blocks of rows: the first one runs ahead over the ring while the
                    // second one's accumulator is still being read; those ring slots are
                    // held until the second has used them too.
                    const int slices = w.kb1 - w.kb0, head = min(kStages, slices);
                    const uint32_t slot0 = unit & 1, slot1 = slot0 ^ 1;
                    uint32_t st = stage, ph = phase;
                    ok = wait_slot(unit);
                    for (int i = 0; ok && i < head; ++i) {
                        ok = wait_full(st, ph);
                        if (!ok) break;
                        multiply(slot0, 0, st, i == 0);
                        if (i == slices - 1) commit(tfull0 + 8 * slot0);
                        next_stage(st, ph);
                    }
                    ok = ok && wait_slot(unit + 1);
                    for (int i = 0; ok && i < head; ++i) {
                        multiply(slot1, 1, stage, i == 0);
                        if (i == slices - 1) commit(tfull0 + 8 * slot1);
                        commit(empty0 + 8 * stage);
                        next_stage(stage, phase);
                    }
                    for (int i = head; ok && i < slices; ++i) {
                        ok = wait_full(stage, phase);
                        if (!ok) break;
                        multiply(slot0, 0, stage, false);
                        if (i == slices - 1) commit(tfull0 + 8 * slot0);
                        multiply(slot1, 1, stage, false);
                        if (i == slices - 1) commit(tfull0 + 8 * slot1);
                        commit(empty0 + 8 * stage);
                        next_stage(stage, phase);
                    }
                    unit += 2;
                }
                if (status == nullptr) {
                    griddep_wait();
                    status = status_word;
                }
            }
            // The products read the rings and write the accumulators of the CTA (pair): it
            // leaves when they have ended, although an epilogue that gave up does not wait.
            umma_commit<kCtaGroup>(kPair ? mapa_shared(done0, 0) : done0);
            mbar_wait(done0, 0, nullptr, kLeaveNs, 0);
        }
        __syncwarp();
    } else {
        // ----------------------------------------------------------- epilogue
        if (early) {
            griddep_wait();
            status = status_word;
        }
        const int q = warp & 3;  // TMEM lane quadrant this warp may access
        const int half = (warp - 2) >> 2;
        const uint32_t sbuf = sbase + C::kEpiOffset + (warp - 2) * kEpiBufBytes;
        const uint32_t row_addr = sbuf + lane * 128;
        uint32_t unit = 0, qs = 0, qph = 0;
        const float alpha = kOp == kDw ? p.head->alpha : 1.0f;
        // The warp leaves as a whole: what follows a wait is warp-wide.
        auto wait_unit = [&]() -> bool {
            const bool got = mbar_wait<false, true>(tfull0 + 8 * (unit & 1), (unit >> 1) & 1, status, p.timeout_ns,
                                                    B200_DEV_TIMEOUT_EPILOGUE);
            if (!__all_sync(0xffffffffu, got)) return false;
            tc_fence_after();
            return true;
        };
        // Accumulator fully read: hand it back to the MMA issuer.
        auto release_unit = [&]() {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                const uint32_t bar = tempty0 + 8 * (unit & 1);
                if constexpr (!kPair) mbar_arrive(bar);
                else mbar_arrive_pair(mapa_shared(bar, 0));
            }
            ++unit;
        };
        // One 32-row x 128-byte chunk of the warp into its staging buffer, once the
        // last store has read it; `store` sends it off.
        auto stage_chunk = [&](const uint32_t (&pk)[32]) {
            if (lane == 0) bulk_wait_group_read<0>();
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                st_shared_v4(row_addr + ((j ^ (lane & 7)) << 4), pk[4 * j], pk[4 * j + 1], pk[4 * j + 2],
                             pk[4 * j + 3]);
            }
        };
        auto store_chunk = [&](int x, int y, bool add) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                if (add) tma_reduce_add_2d(&tmD, sbuf, x, y);
                else tma_store_2d(&tmD, sbuf, x, y);
                bulk_commit_group();
            }
        };
        Tile w{};
        int sm = 0;  // block of rows of the tile that comes next
        auto pack = [](float lo, float hi) { return kHalf ? pack_half2(lo, hi) : pack_bf16x2(lo, hi); };

        while (true) {
            if (sm == 0) {
                if (!__all_sync(0xffffffffu, queue_wait(qs, qph, B200_DEV_TIMEOUT_EPILOGUE))) break;
                const int t = ring[qs];
                __syncwarp();
                if (lane == 0) queue_release(qs);
                if (++qs == kQueue) { qs = 0; qph ^= 1; }
                if (t < 0) break;
                w = tile_of(t);
                if (w.kb0 == w.kb1) continue;
            }
            const int row0 = w.mb * C::kTileM + sm * C::kSubRows + static_cast<int>(rank) * kRowsPerCta + q * 32;
            sm = sm + 1 < w.subs ? sm + 1 : 0;
            const int col0 = w.nb * kTileN + half * kHalfN;  // first column of this warp
            const uint32_t t_lane = tmem_base + half * kHalfN + (static_cast<uint32_t>(q * 32) << 16);

            // The row's targets: position of the first one in the warp's columns and
            // behind the last, and up to four columns. A row of a teacher may have
            // several in a tile; a load for each as it is reached would cost the warp its
            // latency every time, a search for the first one two more (together 14 % of
            // the statistics of 4096 rows with 128 logits).
            const int grow = row0 + lane;  // row of the products
            const bool active = grow < n_rows;
            const int first = p.v0 + col0;
            int pos = 0, end = 0, cur = kNoCol, ahead1 = kNoCol, ahead2 = kNoCol, ahead3 = kNoCol, used = 0;
            long long ebase = grow;
            float4 rg = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            auto col_at = [&](int i) { return i < end ? __ldg(p.ecol + ebase + i) : kNoCol; };
            auto load_four = [&]() {
                cur = col_at(pos);
                ahead1 = col_at(pos + 1);
                ahead2 = col_at(pos + 2);
                ahead3 = col_at(pos + 3);
            };
            auto load_targets = [&]() {
                if (!active) return;
                if constexpr (kOp == kGrad) rg = __ldg(p.rgrad + grow);
                if (p.rowmap == nullptr) {
                    cur = __ldg(p.ecol + grow);
                    return;
                }
                const int r = __ldg(p.rowmap + grow);
                const unsigned short* e = p.epos + r * p.epos_ld + first / kHalfN;
                pos = __ldg(e);
                end = __ldg(e + 1);
                ebase = static_cast<long long>(r) * p.top;
                load_four();
            };
            // Statistics over several units: a bit for each column of the warp that is the
            // row's target.
            constexpr int kWords = kHalfN / 32;
            auto find_targets = [&](unsigned (&bits)[kWords]) {
#pragma unroll
                for (int g = 0; g < kWords; ++g) bits[g] = 0;
                auto add = [&](int col) {
                    const unsigned at = static_cast<unsigned>(col - first);
                    if (at >= kHalfN) return;  // kNoCol and other tiles' columns too
#pragma unroll
                    for (int g = 0; g < kWords; ++g)
                        if (at / 32 == g) bits[g] |= 1u << (at % 32);
                };
                if (!active) return;
                if (p.rowmap == nullptr) {
                    add(__ldg(p.ecol + grow));
                    return;
                }
                const int r = __ldg(p.rowmap + grow);
                const unsigned short* e = p.epos + r * p.epos_ld + first / kHalfN;
                pos = __ldg(e);
                end = __ldg(e + 1);
                ebase = static_cast<long long>(r) * p.top;
                for (int i = pos; i < end; i += 4) {
                    int c[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) c[j] = col_at(i + j);
#pragma unroll
                    for (int j = 0; j < 4; ++j) add(c[j]);
                }
                ebase += pos;
            };
            auto advance = [&]() {
                cur = ahead1;
                ahead1 = ahead2;
                ahead2 = ahead3;
                ++pos;
                if (p.rowmap != nullptr && (++used & 3) == 0) load_four();
            };

            // Keeps the logits at the row's targets among the 32 columns of `r` that start
            // at `lo`. A register cannot be picked by a lane's own number: each lane
            // writes its row to the warp's buffer and reads its own columns back, as many
            // steps as the fullest row has (one step per column of the warp: 37 against
            // 29 us for 3537 rows of 115 logits over 807 x 384).
            auto targets_in = [&](int lo) { return cur >= lo && cur < lo + 32; };
            auto keep_targets = [&](const uint32_t (&r)[32], int lo) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    st_shared_v4(row_addr + ((j ^ (lane & 7)) << 4), r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
                while (targets_in(lo)) {
                    const int i = cur - lo;
                    float z;
                    asm volatile("ld.shared.f32 %0, [%1];"
                                 : "=f"(z) : "r"(row_addr + (((i >> 2) ^ (lane & 7)) << 4) + (i & 3) * 4) : "memory");
                    p.zsel[ebase + pos] = z;
                    advance();
                }
                __syncwarp();
            };
            // The statistics over several units look the targets up between two of them:
            // the first accumulator of a tile is not kept waiting.
            if constexpr (kOp == kStatsShort || kOp == kGrad) load_targets();
            if (!wait_unit()) break;
            const uint32_t t_row = t_lane + (unit & 1) * kTileN;
            if constexpr (kOp == kStats) {
                float acc[kHalfN];
#pragma unroll
                for (int g = 0; g < kHalfN / 32; ++g) tmem_ld_32x32b_x32(t_row + 32 * g, reinterpret_cast<uint32_t(&)[32]>(acc[32 * g]));
                tmem_ld_wait();
                release_unit();
                unsigned targets[kWords];
                find_targets(targets);
                bool ok = true;
#pragma unroll 1
                for (int kb = w.kb0 + kDrain; kb < w.kb1; kb += kDrain) {
                    if (kb > w.kb0 + kDrain) release_unit();
                    ok = wait_unit();
                    if (!ok) break;
                    const uint32_t t_next = t_lane + (unit & 1) * kTileN;
#pragma unroll
                    for (int g = 0; g < kHalfN / 32; ++g) {
                        uint32_t r[32];
                        tmem_ld_32x32b_x32(t_next + 32 * g, r);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 32; ++i) acc[32 * g + i] += __uint_as_float(r[i]);
                    }
                }
                if (!ok) break;
                // Logits at the targets: a register cannot be picked by number, a TMEM
                // column can. Where a row has a target here, the sums go back over the last
                // unit's accumulator; all lanes read each target's column, two at a time,
                // those that want it keep it. Marks instead of a list of columns in which
                // the warp looks for the lowest: 421 -> 377 us for 6970 rows of 102 logits
                // over 30798 x 680, 372 -> 361 for 2048 rows of 64 over 32000 x 4096.
                unsigned wanted = 0;
#pragma unroll
                for (int g = 0; g < kWords; ++g) wanted |= targets[g];
                if (__any_sync(0xffffffffu, wanted != 0)) {
                    const uint32_t t_last = t_lane + (unit & 1) * kTileN;
#pragma unroll
                    for (int g = 0; g < kWords; ++g)
                        tmem_st_32x32b_x32(t_last + 32 * g, reinterpret_cast<uint32_t(&)[32]>(acc[32 * g]));
                    tmem_st_wait();
                    float* to = p.zsel + ebase;
#pragma unroll 1
                    for (int g = 0; g < kWords; ++g) {
                        const unsigned mine = targets[0];
#pragma unroll
                        for (int i = 1; i < kWords; ++i) targets[i - 1] = targets[i];
                        unsigned cols = __reduce_or_sync(0xffffffffu, mine);
#pragma unroll 1
                        while (cols != 0) {
                            const unsigned low = cols & (0u - cols), rest = cols ^ low;
                            const unsigned next = rest & (0u - rest);
                            cols = rest ^ next;
                            float z0, z1;
                            tmem_ld_cols(t_last + 32 * g + __ffs(low) - 1, t_last + 32 * g + __ffs(next ? next : low) - 1, z0, z1);
                            if (mine & low) *to++ = z0;
                            if (mine & next) *to++ = z1;
                        }
                    }
                }
                release_unit();
                const int left = p.n - col0;  // columns of the vocabulary in this half
                if (left <= 0) continue;
                if (left < kHalfN) {
#pragma unroll
                    for (int i = 0; i < kHalfN; ++i)
                        if (i >= left) acc[i] = -INFINITY;
                }
                float m4[4] = {acc[0], acc[1], acc[2], acc[3]};
#pragma unroll
                for (int i = 4; i < kHalfN; ++i) m4[i & 3] = fmaxf(m4[i & 3], acc[i]);
                const float m = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
                const float ref = finite_or_zero(m);
                float s4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int i = 0; i < kHalfN; ++i) s4[i & 3] += exp2_approx((acc[i] - ref) * p.c2);
                if (active)
                    p.part[grow * p.part_ld + 2 * w.nb + half] =
                        make_float2(m, (s4[0] + s4[1]) + (s4[2] + s4[3]));
            } else if constexpr (kOp == kStatsShort) {
                // One accumulator holds the whole contraction: 32 columns at a time from
                // TMEM, with a running maximum. A tenth of the code above, which a small
                // call would wait for (5 us of instruction fetches).
                float m = -INFINITY, s = 0.0f;
#pragma unroll 1
                for (int c = 0; c < kHalfN / 32; ++c) {
                    const int left = p.n - (col0 + c * 32);
                    if (left <= 0) break;
                    uint32_t r[32];
                    tmem_ld_32x32b_x32(t_row + c * 32, r);
                    tmem_ld_wait();
                    if (left < 32) {
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (i >= left) r[i] = __float_as_uint(-INFINITY);
                    }
                    float m4[4] = {m, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int i = 0; i < 32; ++i) m4[i & 3] = fmaxf(m4[i & 3], __uint_as_float(r[i]));
                    const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
                    const float ref = finite_or_zero(mx);
                    float s4[4] = {s * rescale(m, mx, p.c2), 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int i = 0; i < 32; ++i) s4[i & 3] += exp2_approx((__uint_as_float(r[i]) - ref) * p.c2);
                    s = (s4[0] + s4[1]) + (s4[2] + s4[3]);
                    m = mx;
                    if (__any_sync(0xffffffffu, targets_in(first + c * 32))) keep_targets(r, first + c * 32);
                }
                release_unit();
                if (active && col0 < p.n)
                    p.part[grow * p.part_ld + 2 * w.nb + half] = make_float2(m, s);
            } else if constexpr (kOp == kGrad) {
#pragma unroll 1
                for (int c = 0; c < kHalfN / 64; ++c) {
                    uint32_t r0[32], r1[32], pk[32];
                    tmem_ld_32x32b_x32(t_row + c * 64, r0);
                    tmem_ld_32x32b_x32(t_row + c * 64 + 32, r1);
                    tmem_ld_wait();
                    const int x = col0 + c * 64;
                    const int left = p.n - x;
                    // At most 1: where z / tau has no digits left behind the point, its
                    // difference from lse may come out above 0. Times a weight below 2, half
                    // precision has room for less than 2 in G's scale. NaN stays NaN.
                    auto grad = [&](uint32_t z) {
                        return rg.x * exp2_approx(min_nan(fmaf(__uint_as_float(z), p.c2, rg.y), 0.0f));
                    };
                    if (left < 64) {
                        // Columns beyond the piece are zeros of the product that contracts
                        // over them, whatever the accumulator holds: logits of -inf.
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            if (i >= left) r0[i] = __float_as_uint(-INFINITY);
                            if (i + 32 >= left) r1[i] = __float_as_uint(-INFINITY);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        pk[i] = pack(grad(r0[2 * i]), grad(r0[2 * i + 1]));
                        pk[16 + i] = pack(grad(r1[2 * i]), grad(r1[2 * i + 1]));
                    }
                    // So are rows without a loss.
#pragma unroll
                    for (int i = 0; i < 32; ++i) pk[i] = active ? pk[i] : 0u;
                    if (row0 >= p.rows) continue;  // nothing of the call in these rows
                    stage_chunk(pk);
                    // The targets' columns again, p - q from the forward pass's
                    // log-probabilities: where p is near q, this product's logits (added
                    // up without rounding to nearest) against a rounded lse are too far off.
                    const int lo = p.v0 + x;
                    while (cur >= lo && cur < lo + 64) {
                        float g = rg.z;
                        if (p.rowmap != nullptr) {
                            const float logp = __ldg(p.zsel + ebase + pos), qv = __ldg(p.eq + ebase + pos);
                            g = rg.x * (exp2_approx(logp * kLog2e) - qv);
                        }
                        const int i = cur - lo;
                        asm volatile("st.shared.u16 [%0], %1;"
                                     ::"r"(row_addr + (((i >> 3) ^ (lane & 7)) << 4) + (i & 7) * 2),
                                     "h"(static_cast<uint16_t>(pack(g, 0.0f) & 0xffffu)) : "memory");
                        advance();
                    }
                    __syncwarp();
                    store_chunk(x, row0, false);
                }
                release_unit();
            } else if constexpr (kSplit) {
#pragma unroll 1
                for (int c = 0; c < kHalfN / 32; ++c) {
                    uint32_t r[32];
                    tmem_ld_32x32b_x32(t_row + c * 32, r);
                    tmem_ld_wait();
                    const int x = col0 + c * 32;
                    if (x >= p.n) break;
                    stage_chunk(r);
                    store_chunk(x, w.split * p.rows_pad + row0, p.accumulate != 0);
                }
                release_unit();
            } else {
                // The whole block rounded into registers before any store: with two blocks
                // per tile no other accumulator is free meanwhile.
                uint32_t pk[kHalfN / 64][32];
#pragma unroll
                for (int c = 0; c < kHalfN / 64; ++c) {
                    uint32_t r0[32], r1[32];
                    tmem_ld_32x32b_x32(t_row + c * 64, r0);
                    tmem_ld_32x32b_x32(t_row + c * 64 + 32, r1);
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        pk[c][i] = pack(alpha * __uint_as_float(r0[2 * i]), alpha * __uint_as_float(r0[2 * i + 1]));
                        pk[c][16 + i] = pack(alpha * __uint_as_float(r1[2 * i]), alpha * __uint_as_float(r1[2 * i + 1]));
                    }
                }
                release_unit();
#pragma unroll
                for (int c = 0; c < kHalfN / 64; ++c) {
                    const int x = col0 + c * 64;
                    if (x >= p.n || row0 >= p.m) break;
                    stage_chunk(pk[c]);
                    store_chunk(x, p.v0 + row0, false);
                }
            }
        }
        if (lane == 0) bulk_wait_group<0>();
        __syncwarp();
    }

    // Whatever follows dW waits for dW alone, and needs dH too.
    if constexpr (is_dw(kOp)) griddep_wait();

    // Teardown: every role is done with TMEM and with the peer's barriers.
    if (is_stats(kOp) && p.merge.lanes != 0) __threadfence();
    tc_fence_before();
    if constexpr (kPair) cluster_sync(); else __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc<kCtaGroup>(tmem_base, kTmemCols);
    }
    if constexpr (is_stats(kOp)) {
        // Little to merge: the block that finishes last does it.
        const MergeParams& mp = p.merge;
        if (mp.lanes == 0) return;
        __shared__ double sums[kThreads / 32];
        __shared__ int counts[kThreads / 32];
        __shared__ int last;
        if (threadIdx.x == 0) last = atomicAdd(&p.head->ticket, 1) == static_cast<int>(gridDim.x) - 1;
        __syncthreads();
        if (!last) return;
        __threadfence();
        const bool failed = __ldcg(&p.head->status) != 0;
        const int sub = threadIdx.x & (mp.lanes - 1);
        for (int r0 = 0; r0 < mp.rows; r0 += kThreads / mp.lanes) {
            const int row = r0 + threadIdx.x / mp.lanes;
            const int i = row < mp.rows ? mp.inv[row] : -1;
            const int f = row < mp.rows ? mp.flag[row] : kNoLoss;
            const float z_one = i >= 0 && mp.eq == nullptr ? __ldcg(mp.zsel + i) : 0.0f;
            float m = -INFINITY, s = 0.0f;
            if (i >= 0) merge_parts(mp, i, sub, mp.lanes, m, s);
            merge_lanes(mp, mp.lanes, m, s);
            merge_row(mp, row, f, z_one, i, failed, m, s, sub, mp.lanes);
        }
        if (mp.reduction == B200_VL_NONE) return;
        __syncthreads();
        merge_sum<kThreads>(mp, sums, counts);
    }
}

// ---------------------------------------------------------------------------
// Rows, targets, teachers
// ---------------------------------------------------------------------------

__device__ __forceinline__ long long index_at(const void* idx, int bytes, long long i) {
    return bytes == 8 ? __ldg(static_cast<const long long*>(idx) + i)
                      : static_cast<long long>(__ldg(static_cast<const int*>(idx) + i));
}

__device__ __forceinline__ float teacher_at(const void* t, int dtype, long long i) {
    if (dtype == B200_VL_F32) return __ldg(static_cast<const float*>(t) + i);
    const unsigned short u = __ldg(static_cast<const unsigned short*>(t) + i);
    if (dtype == B200_VL_BF16) return __uint_as_float(static_cast<uint32_t>(u) << 16);
    return __half2float(__ushort_as_half(u));
}

struct TeacherParams {
    const void* index;
    const void* teacher;
    int index_bytes, teacher_dtype;
    long long ld_index, ld_teacher;
    int rows, vocab, top;
    float inv_tau;
    int half;             // columns of a half tile
    long long epos_ld;
    int* ecol;
    float* eq;
    unsigned short* epos;
    int* flag;
    float* zsel;          // forward: logits at the targets, zeros behind a row's last
    // Where the products run over all rows in their order: nothing is left to number.
    Head* head;           // or null: the rows' kernel follows
    int* rowmap;
    int* inv;
};

// A block turns one row of a teacher's logits into its target distribution:
// softmax over the entries that are there, sorted by column, entries of one
// column added up in the order given. 2 x 8 bytes per entry in, 8 out. It also
// leaves where in the row each half tile of the vocabulary begins. What it takes is
// latency: sorting steps and, for every half tile, a search (two rows of 109 over
// 108645 columns: 20 us with a warp per row, 8 with four). Many rows of few entries
// take a warp each instead (7844 rows of 6: 10 against 16 us).
template <int kTeacherThreads>
__global__ void __launch_bounds__(kTeacherThreads) teacher_kernel(const TeacherParams p, int pad) {
    constexpr int kWarps = kTeacherThreads / 32;
    __shared__ unsigned long long key[kMaxTop];
    __shared__ float prob[kMaxTop];
    __shared__ unsigned cols[kMaxTop];
    __shared__ float red[2][kWarps];
    __shared__ int heads_of[kWarps];
    griddep_launch_dependents();
    const int t = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    float mx = -INFINITY;
    bool any = false, bad = false, nan = false;
    for (int k = tid; k < pad; k += kTeacherThreads) {
        float l = -INFINITY;
        unsigned col = kNoCol;
        if (k < p.top) {
            const long long c = index_at(p.index, p.index_bytes, t * p.ld_index + k);
            if (c >= p.vocab) bad = true;
            else if (c >= 0) {
                l = teacher_at(p.teacher, p.teacher_dtype, t * p.ld_teacher + k);
                if (l != -INFINITY) {
                    col = static_cast<unsigned>(c);
                    any = true;
                    if (!(l < INFINITY)) nan = true;  // NaN or +inf: no distribution
                }
            }
        }
        key[k] = (static_cast<unsigned long long>(col) << 32) | static_cast<unsigned>(k);
        prob[k] = l;
        mx = fmaxf(mx, l);
    }
    for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    if (lane == 0) red[0][warp] = mx;
    any = __syncthreads_or(any);
    bad = __syncthreads_or(bad);
    nan = __syncthreads_or(nan);
    for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, red[0][w]);
    float sum = 0.0f;
    for (int k = tid; k < pad; k += kTeacherThreads) {
        // The difference first: a logit of the type's lowest value is one, whatever tau.
        const float e = prob[k] == -INFINITY ? 0.0f : expf((prob[k] - mx) * p.inv_tau);
        prob[k] = e;
        sum += e;
    }
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) red[1][warp] = sum;
    __syncthreads();
    sum = red[1][0];
    for (int w = 1; w < kWarps; ++w) sum += red[1][w];
    const float inv = nan ? NAN : 1.0f / sum;
    // Bitonic sort of (column, position).
    for (int size = 2; size <= pad; size <<= 1) {
        for (int stride = size >> 1; stride; stride >>= 1) {
            for (int i = tid; i < pad / 2; i += kTeacherThreads) {
                const int lo = 2 * i - (i & (stride - 1));
                const int hi = lo + stride;
                const unsigned long long a = key[lo], b = key[hi];
                if ((a > b) == ((lo & size) == 0)) {
                    key[lo] = b;
                    key[hi] = a;
                }
            }
            __syncthreads();
        }
    }
    int out = 0;
    int* ecol = p.ecol + static_cast<long long>(t) * p.top;
    float* eq = p.eq + static_cast<long long>(t) * p.top;
    for (int base = 0; base < pad; base += kTeacherThreads) {
        const int i = base + tid;
        unsigned col = kNoCol;
        bool first = false;
        if (i < pad) {
            col = static_cast<unsigned>(key[i] >> 32);
            first = col != kNoCol && (i == 0 || static_cast<unsigned>(key[i - 1] >> 32) != col);
        }
        const unsigned heads = __ballot_sync(0xffffffffu, first);
        if (lane == 0) heads_of[warp] = __popc(heads);
        __syncthreads();
        int o = out + __popc(heads & ((1u << lane) - 1));
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) o += heads_of[w];
            out += heads_of[w];
        }
        if (first) {
            float v = 0.0f;
            for (int j = i; j < pad && static_cast<unsigned>(key[j] >> 32) == col; ++j)
                v += prob[static_cast<unsigned>(key[j])];
            ecol[o] = static_cast<int>(col);
            cols[o] = col;
            eq[o] = v * inv;
        }
        __syncthreads();
    }
    for (int i = out + tid; i < p.top; i += kTeacherThreads) {
        ecol[i] = kNoCol;
        eq[i] = 0.0f;
        if (p.zsel != nullptr) p.zsel[static_cast<long long>(t) * p.top + i] = 0.0f;
    }
    if (tid == 0) {
        p.flag[t] = bad ? kBad : (any ? kLoss : kNoLoss);
        if (p.head != nullptr) {
            p.rowmap[t] = t;
            p.inv[t] = bad || any ? t : -1;
            if (t == 0) {
                Head h = {};
                h.n_rows = p.rows;
                h.alpha = 1.0f;
                *p.head = h;
            }
        }
    }
    unsigned short* epos = p.epos + t * p.epos_ld;
    for (long long j = tid; j < p.epos_ld; j += kTeacherThreads) {
        const long long col = j * p.half;
        int lo = 0, hi = out;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (cols[mid] < col) lo = mid + 1;
            else hi = mid;
        }
        epos[j] = static_cast<unsigned short>(lo);
    }
}

struct RowsParams {
    Head* head;
    const void* target;   // cross entropy; null: the flags are the teachers'
    int index_bytes;
    long long ignore;
    int rows, vocab;
    int gather;           // 0: the products run over all rows, in their order
    int copy_all;         // 1: they run over the gathered copy even if no row is left out
    int reduction;
    int* flag;
    int* ecol;            // cross entropy: written here
    int* rowmap;
    int* inv;             // row -> gathered row, -1 without a loss
    const float* grad;    // backward: what comes from above
    const float* lse;
    const float* target_logp;
    float4* rgrad;        // see Params
    float tau;
    float scale;          // of G
    int split;            // weights of rows: 1 leaves their exponents out of G
    const uint4* hidden;  // gather: H, and where its copy goes
    uint4* copy;
    long long ld, ld_copy;
    int vecs;             // 16-byte units of a row
};

// Numbers the rows that have a loss, in order, leaves the factors of the backward
// pass, and copies the rows of H that have a loss (a block of rows of zeros follows
// the last one) unless every row has one and starts on a 128-byte line. Four rows
// per thread and step. Every block counts all rows, so that none waits for another;
// of each group of four rows one block writes what is written, and copies. Latency
// and the copy bound it (2048 of 4096 rows of 8 KiB: 13 us, where a block that numbers
// and a launch that copies took 17 and a launch more).
__global__ void __launch_bounds__(1024) rows_kernel(const RowsParams p) {
    constexpr int kPer = 4, kChunk = 1024 * kPer;
    __shared__ int warp_sum[32];
    __shared__ float warp_max[32];
    __shared__ int base;
    __shared__ int4 numbers[1024];  // inv of a chunk
    // What follows may set itself up, and load what the call was given, from the
    // start; it waits for this kernel's end before it looks at the workspace.
    griddep_launch_dependents();
    griddep_wait();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // Four rows as one access wherever all four are there: one row at a time, 16
    // bytes apart between lanes, took 14 us for 8192 rows.
    auto classify = [&](int t0, int (&f)[kPer], int (&col)[kPer]) {
        const bool four = p.target == nullptr && t0 + kPer <= p.rows;
        if (four) {
            const int4 v = *reinterpret_cast<const int4*>(p.flag + t0);
            f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
        }
        int count = 0;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            col[j] = kNoCol;
            if (!four) f[j] = kNoLoss;
            if (!four && t0 + j < p.rows) {
                if (p.target != nullptr) {
                    const long long c = index_at(p.target, p.index_bytes, t0 + j);
                    f[j] = c == p.ignore ? kNoLoss : (c >= 0 && c < p.vocab ? kLoss : kBad);
                    col[j] = f[j] == kLoss ? static_cast<int>(c) : kNoCol;
                } else {
                    f[j] = p.flag[t0 + j];
                }
            }
            count += f[j] != kNoLoss;
        }
        return count;
    };
    // What must be known of all rows first: whether one is left out, and the largest
    // finite gradient (what is infinite or NaN stays in its own row).
    bool copying = p.gather && p.copy_all;
    const bool per_row = p.rgrad != nullptr && p.reduction == B200_VL_NONE;
    const bool counting = p.gather && !copying && p.rows > kChunk;
    float gmax = 0.0f;
    if (per_row || counting) {
        int left_out = 0;
        for (int t0 = tid * kPer; t0 < p.rows; t0 += kChunk) {
            int f[kPer], col[kPer];
            left_out += classify(t0, f, col) != min(kPer, p.rows - t0);
            if (per_row) {
#pragma unroll
                for (int j = 0; j < kPer; ++j) {
                    const float g = f[j] != kNoLoss ? fabsf(p.grad[t0 + j]) : 0.0f;
                    if (isfinite(g)) gmax = fmaxf(gmax, g);
                }
            }
        }
        for (int o = 16; o; o >>= 1) gmax = fmaxf(gmax, __shfl_xor_sync(0xffffffffu, gmax, o));
        if (lane == 0) warp_max[warp] = gmax;
        left_out = __syncthreads_or(left_out);
        if (counting) copying = left_out != 0;
        for (int i = 0; i < 32; ++i) gmax = fmaxf(gmax, warp_max[i]);
    }
    // G holds the weights over the largest one's power of two, below 2 (times the scale),
    // or each over its own: exact, and no row's gradient depends on another row's weight.
    const int g_exponent = gmax > 0.0f ? ilogbf(gmax) : 0;
    if (tid == 0) base = 0;
    __syncthreads();
    for (int r0 = 0; r0 < p.rows; r0 += kChunk) {
        const int t0 = r0 + tid * kPer;
        const bool four = t0 + kPer <= p.rows;
        const bool mine = t0 < p.rows && (t0 / kPer) % gridDim.x == blockIdx.x;
        int f[kPer], col[kPer];
        const int count = classify(t0, f, col);
        // Rows with a loss before this thread's first one: scan in the warp, then
        // over the warps.
        int upto = count;
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += u;
        }
        if (lane == 31) warp_sum[warp] = upto;
        __syncthreads();
        if (warp == 0) {
            int v = warp_sum[lane];
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, v, o);
                if (lane >= o) v += u;
            }
            warp_sum[lane] = v;
        }
        __syncthreads();
        if (p.gather && !copying && !counting) copying = warp_sum[31] != p.rows;
        int at = base + (warp ? warp_sum[warp - 1] : 0) + upto - count;
        const int at0 = p.gather ? at : t0;
        int inv[kPer];
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const bool in = f[j] != kNoLoss;
            inv[j] = in ? (p.gather ? at : t0 + j) : -1;
            at += in;
        }
        const int4 quad = make_int4(inv[0], inv[1], inv[2], inv[3]);
        if (copying) numbers[tid] = quad;
        if (mine) {
            const bool together = four && (at0 & 3) == 0 && (count == kPer || !p.gather);
            if (four) {
                *reinterpret_cast<int4*>(p.inv + t0) = quad;
                if (p.target != nullptr) *reinterpret_cast<int4*>(p.flag + t0) = make_int4(f[0], f[1], f[2], f[3]);
            }
            if (together) {
                *reinterpret_cast<int4*>(p.rowmap + at0) = make_int4(t0, t0 + 1, t0 + 2, t0 + 3);
                if (p.target != nullptr) *reinterpret_cast<int4*>(p.ecol + at0) = make_int4(col[0], col[1], col[2], col[3]);
            }
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
                const int t = t0 + j;
                if (t >= p.rows) continue;
                if (!four) {
                    p.inv[t] = inv[j];
                    if (p.target != nullptr) p.flag[t] = f[j];
                }
                const int i = p.gather ? inv[j] : t;
                if (i < 0) continue;
                if (!together) {
                    p.rowmap[i] = t;
                    if (p.target != nullptr) p.ecol[i] = col[j];
                }
                if (p.rgrad == nullptr) continue;
                float g = 1.0f;
                int exponent = g_exponent;
                if (per_row) {
                    g = p.grad[t];
                    // A weight of 0 is no reason to scale H by anything.
                    if (p.split && isfinite(g) && f[j] != kBad) exponent = g != 0.0f ? ilogbf(g) : g_exponent - 200;
                    g = scalbnf(g, -exponent);
                }
                g *= p.scale;
                const float own = __int_as_float(exponent);
                // p - 1 at the one target, without the difference of two numbers near 1.
                const float below = p.target != nullptr ? expm1f(p.target_logp[t]) : 0.0f;
                p.rgrad[i] = f[j] == kBad ? make_float4(NAN, NAN, NAN, own)
                                          : make_float4(g, -p.lse[t] * kLog2e, g * below, own);
            }
        }
        __syncthreads();
        if (copying) {
            // A warp per row: of the block's groups of four in this chunk, the e-th row.
            const int first = r0 / kPer;
            const int own = first + (blockIdx.x + gridDim.x - first % gridDim.x) % gridDim.x;
            for (int e = warp;; e += 32) {
                const int quad_no = own + (e >> 2) * static_cast<int>(gridDim.x) - first;
                const int t = r0 + quad_no * kPer + (e & 3);
                if (quad_no >= 1024 || t >= p.rows) break;
                const int i = reinterpret_cast<const int*>(numbers)[quad_no * kPer + (e & 3)];
                if (i < 0) continue;
                const uint4* src = p.hidden + t * p.ld;
                uint4* dst = p.copy + i * p.ld_copy;
                for (int v0 = lane; v0 < p.vecs; v0 += 32 * 8) {
                    uint4 x[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (v0 + 32 * j < p.vecs) x[j] = __ldg(src + v0 + 32 * j);
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (v0 + 32 * j < p.vecs) dst[v0 + 32 * j] = x[j];
                }
            }
        }
        if (tid == 0) base += warp_sum[31];
        __syncthreads();
    }
    const int n_valid = base;
    if (copying) {
        const int end = min(p.rows, (max(n_valid, 1) + 255) / 256 * 256);
        for (int i = n_valid + blockIdx.x * 32 + warp; i < end; i += gridDim.x * 32) {
            uint4* dst = p.copy + i * p.ld_copy;
            for (int v = lane; v < p.vecs; v += 32) dst[v] = make_uint4(0, 0, 0, 0);
        }
    }
    if (blockIdx.x == 0 && tid == 0) {
        Head h;
        h.status = 0;
        for (int i = 0; i < 4; ++i) h.counter[i] = 0;
        h.g_piece = 0;
        h.ticket = 0;
        h.n_valid = n_valid;
        h.n_rows = p.gather ? n_valid : p.rows;
        h.compact = copying;
        h.alpha = 1.0f;
        if (p.rgrad != nullptr) {
            if (per_row) h.alpha = scalbnf(p.tau, g_exponent);
            else h.alpha = p.grad[0] * p.tau / (p.reduction == B200_VL_MEAN ? static_cast<float>(max(n_valid, 1)) : 1.0f);
            h.alpha /= p.scale;
        }
        h.g_exponent = g_exponent;
        h.h_most = 0;
        *p.head = h;
    }
}

// Weights of rows in half precision: dW = sum_t g_t (p - q)_t h_t runs over a copy of H
// that holds each row's power of two, so that G is free of it. The copy is scaled by one
// more power of two for all rows, its largest element then at 2^14 or above: rows of
// 2^-24 of that weight keep what is left of half precision's 40 binades. Exact but for
// elements below 2^-14, which lose less than 2^-39 of the largest. Weights folded
// into G instead cost rows of 1/1000 of the largest weight a third of their dW and 0.4 %
// of their dH at 32064 tokens. The copy takes one more pass over H for its
// largest element; both are bound by reading H.
struct WeighParams {
    Head* head;
    const float4* rgrad;
    const uint4* hidden;  // H, and the gathered copy of it
    const uint4* copy;
    uint4* weighed;
    long long ld, ld_copy;
    int rows, vecs;
    float tau;            // in G's scale
};

constexpr int kWeighWarps = 8;

__device__ __forceinline__ const uint4* weigh_source(const WeighParams& p, int i) {
    return p.head->compact ? p.copy + i * p.ld_copy : p.hidden + i * p.ld;
}

__global__ void __launch_bounds__(32 * kWeighWarps) weigh_most_kernel(const WeighParams p) {
    __shared__ unsigned mosts[kWeighWarps];
    griddep_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n = p.head->n_rows, g_exponent = p.head->g_exponent;
    unsigned most = 0;
    for (int i = blockIdx.x * kWeighWarps + warp; i < n; i += gridDim.x * kWeighWarps) {
        const uint4* src = weigh_source(p, i);
        unsigned m = 0;  // magnitudes order like their bits
        auto finite = [&](unsigned bits) { if (bits < 0x7c00u) m = max(m, bits); };
        for (int v = lane; v < p.vecs; v += 32) {
            const uint4 x = __ldg(src + v);
            for (const unsigned w : {x.x, x.y, x.z, x.w}) {
                finite(w & 0x7fffu);
                finite((w >> 16) & 0x7fffu);
            }
        }
        m = __reduce_max_sync(0xffffffffu, m);
        const float h = __half2float(__ushort_as_half(static_cast<unsigned short>(m)));
        most = max(most, __float_as_uint(scalbnf(h, __float_as_int(p.rgrad[i].w) - g_exponent)));
    }
    if (lane == 0) mosts[warp] = most;
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int w = 0; w < kWeighWarps; ++w) most = max(most, mosts[w]);
    atomicMax(&p.head->h_most, most);  // a maximum: whatever the order
}

__global__ void __launch_bounds__(32 * kWeighWarps) weigh_kernel(const WeighParams p) {
    griddep_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n = p.head->n_rows, g_exponent = p.head->g_exponent;
    const float most = __uint_as_float(p.head->h_most);
    const int up = most > 0.0f ? max(0, min(60, 14 - ilogbf(most))) : 0;
    if (blockIdx.x == 0 && threadIdx.x == 0) p.head->alpha = scalbnf(p.tau, g_exponent - up);
    // Rows of zeros behind the last one: dW's contraction runs over whole k-slices.
    const int end = min(p.rows, (max(n, 1) + 255) / 256 * 256);
    for (int i = blockIdx.x * kWeighWarps + warp; i < end; i += gridDim.x * kWeighWarps) {
        uint4* dst = p.weighed + i * p.ld_copy;
        if (i >= n) {
            for (int v = lane; v < p.vecs; v += 32) dst[v] = make_uint4(0, 0, 0, 0);
            continue;
        }
        const uint4* src = weigh_source(p, i);
        const float factor = scalbnf(1.0f, __float_as_int(p.rgrad[i].w) - g_exponent + up);
        auto times = [&](uint32_t w) {
            const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&w));
            return pack_half2(x.x * factor, x.y * factor);
        };
        for (int v = lane; v < p.vecs; v += 32) {
            const uint4 x = __ldg(src + v);
            dst[v] = make_uint4(times(x.x), times(x.y), times(x.z), times(x.w));
        }
    }
}

// A warp, or all eight of a block where there are few long rows, merges a row's half
// tiles in a fixed order and forms its loss; the last block to finish adds the
// rows in order. Reads 8 bytes per (row, half tile).
__global__ void __launch_bounds__(32 * kMergeWarps) merge_kernel(const MergeParams p) {
    __shared__ float sm[kMergeWarps], ss[kMergeWarps];
    __shared__ double sums[kMergeWarps];
    __shared__ int counts[kMergeWarps];
    __shared__ int last;
    griddep_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int row = blockIdx.x * (kMergeWarps / p.warps_per_row) + warp / p.warps_per_row;
    const int i = row < p.rows ? p.inv[row] : -1;
    const int f = row < p.rows ? p.flag[row] : kNoLoss;
    const bool failed = p.head->status != 0;
    const float z_one = i >= 0 && p.eq == nullptr ? __ldcg(p.zsel + i) : 0.0f;
    float m = -INFINITY, s = 0.0f;
    if (i >= 0) merge_parts(p, i, (warp % p.warps_per_row) * 32 + lane, 32 * p.warps_per_row, m, s);
    merge_lanes(p, 32, m, s);
    if (p.warps_per_row > 1) {
        if (lane == 0) {
            sm[warp] = m;
            ss[warp] = s;
        }
        __syncthreads();
        for (int w = 0; w < kMergeWarps; ++w) m = fmaxf(m, sm[w]);
        s = 0.0f;
        for (int w = 0; w < kMergeWarps; ++w) s += ss[w] * rescale(sm[w], m, p.c2);
    }
    const bool leader = row < p.rows && warp % p.warps_per_row == 0;
    merge_row(p, leader ? row : p.rows, leader ? f : kNoLoss, z_one, i, failed, m, s, lane, 32);
    if (p.reduction == B200_VL_NONE) return;
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) last = atomicAdd(&p.head->ticket, 1) == static_cast<int>(gridDim.x) - 1;
    __syncthreads();
    if (!last) return;
    __threadfence();
    merge_sum<32 * kMergeWarps>(p, sums, counts);
}

struct FinishParams {
    const Head* head;
    const int* inv;
    const float* part_h;  // dH: [splits][rows_pad][ld_part]
    const float* part_w;  // dW: the same over the vocabulary, or null: written by the product
    long long ld_part, stride_h, stride_w;
    int splits_h, splits_w, rows, hidden, vocab, fp16;
    int width;            // threads of a row: 32 to 256
    int tile_m_h, slots_h, slots_w, slices_h, cost16_h, cost16_w;  // of runs_for, as in the products
    const float4* rgrad;  // weights of rows: their exponents, where G is free of them
    float tau;            // in G's scale
    void* d_hidden;
    void* d_weight;
};

// Adds the splits of dH (and of dW) in order, applies the common (or the row's) factor, rounds,
// and puts the rows of dH back in their places; rows without a loss get zeros.
// 4 bytes read per split and 2 written for each element. Short rows share a block
// (step of 4000 x 8000 x 256 as a graph: 111 us, 123 with a block for each row).
__global__ void __launch_bounds__(256) finish_kernel(const FinishParams p) {
    griddep_wait();
    const bool failed = p.head->status != 0;
    const float alpha = p.head->alpha;
    const int vecs = p.hidden / 8;
    const int n_rows = max(p.head->n_rows, 1);
    const int num_n = (p.hidden + kBN - 1) / kBN;
    const int splits_h = runs_for_warp((n_rows + p.tile_m_h - 1) / p.tile_m_h * num_n, p.slots_h, p.slices_h, p.splits_h, p.cost16_h);
    const int splits_w = p.part_w == nullptr ? 1
                                             : runs_for_warp((p.vocab + kBN - 1) / kBN * num_n, p.slots_w, (n_rows + kBK - 1) / kBK,
                                                        p.splits_w, p.cost16_w);
    const int rows_h = p.d_hidden != nullptr ? p.rows : 0;
    const int rows_w = p.d_weight != nullptr && (failed || p.part_w != nullptr) ? p.vocab : 0;
    const int groups = 256 / p.width, at = threadIdx.x & (p.width - 1);
    const long long all = static_cast<long long>(rows_h) + rows_w;
    for (long long r = static_cast<long long>(blockIdx.x) * groups + threadIdx.x / p.width; r < all;
         r += static_cast<long long>(gridDim.x) * groups) {
        const bool is_h = r < rows_h;
        const int t = static_cast<int>(is_h ? r : r - rows_h);
        const int i = is_h ? p.inv[t] : t;
        const int splits = is_h ? splits_h : splits_w;
        const long long stride = is_h ? p.stride_h : p.stride_w;
        const float* part = (is_h ? p.part_h : p.part_w) + max(i, 0) * p.ld_part;
        const float factor = is_h && p.rgrad != nullptr ? scalbnf(p.tau, __float_as_int(p.rgrad[max(i, 0)].w)) : alpha;
        uint4* out = static_cast<uint4*>(is_h ? p.d_hidden : p.d_weight) + static_cast<long long>(t) * vecs;
        for (int v = at; v < vecs; v += p.width) {
            float x[8] = {};
            if (i >= 0 && !failed) {
                for (int s = 0; s < splits; ++s) {
                    const float4* src = reinterpret_cast<const float4*>(part + s * stride) + 2 * v;
                    const float4 a = __ldcs(src), b = __ldcs(src + 1);
                    x[0] += a.x; x[1] += a.y; x[2] += a.z; x[3] += a.w;
                    x[4] += b.x; x[5] += b.y; x[6] += b.z; x[7] += b.w;
                }
            }
            uint32_t o[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                // Never a silent half of a gradient: a launch that was given up leaves NaN.
                const float lo = failed ? NAN : (i >= 0 ? factor * x[2 * j] : 0.0f);
                const float hi = failed ? NAN : (i >= 0 ? factor * x[2 * j + 1] : 0.0f);
                o[j] = p.fp16 ? pack_half2(lo, hi) : pack_bf16x2(lo, hi);
            }
            out[v] = make_uint4(o[0], o[1], o[2], o[3]);
        }
    }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
static int runs_for(int tiles, int slots, int slices, int most, int run_cost16) {
    int best = 1;
    for (int s = 2; s <= most && s <= slices; ++s)
        if (runs_cost(s, tiles, slots, slices, run_cost16) < runs_cost(best, tiles, slots, slices, run_cost16)) best = s;
    return best;
}

static int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
static int64_t align_up(int64_t a, int64_t b) { return ceil_div(a, b) * b; }

// Room for G: this, or as much as H itself takes (one 256-column block at least).
constexpr int64_t kPieceBytes = int64_t(256) << 20;
constexpr int64_t kPartialBytes = int64_t(256) << 20;
// What the last block of the product merges in the time of a launch: rows x (half
// tiles or targets), and those of one row. (26 rows over 718 columns 15.7 -> 13.0 us,
// 8 over 32000 17.2 -> 16.0, 512 over 512 16.5 -> 15.9; beyond: 64 over 32000 16.4 ->
// 22.4, one over 128256 181 -> 184.)
constexpr int64_t kMergeHere = 4096, kMergeRowHere = 512;
// A piece of G that is still in L2 (126 MB) when the second product reads it.
constexpr int64_t kL2Piece = int64_t(48) << 20;

struct Layout {
    int cta_group, tile_n;          // tiles of the logits (Stats, Grad)
    int cta_group_h;                // tiles of dH, 256 wide
    int64_t tile_m, tile_m_h, piece, pieces, rows_pad;
    int64_t splits_h, splits_w, slices_h;  // runs of dH's and dW's contractions at most
    int cost16_h, cost16_w;
    int sub_w;                             // blocks of 256 rows per tile of dW
    // Offsets in the workspace.
    int64_t flag, rowmap, inv, ecol, eq, epos;           // both directions
    int64_t zsel, part, row_loss, gathered_forward;
    int64_t rgrad, gathered_backward, weighed, g, part_h, part_w;
    int64_t epos_ld;
    int64_t ld_gathered, ld_part;                        // row pitches on 128-byte lines
    int64_t bytes_forward, bytes_backward;
    bool gather_forward;
    bool split;           // weights of rows leave G (RowsParams)
    int merge_lanes;      // of MergeParams
};

static int check_desc(const B200VocabLossDesc* d) {
    if (d == nullptr) {
        set_error("desc must not be NULL");
        return B200_ERR_INVALID_ARGUMENT;
    }
    const int64_t kMax = (int64_t(1) << 31) - 1;
    if (d->rows < 0 || d->vocab < 1 || d->hidden < 1) {
        set_error("(rows,vocab,hidden)=(%lld,%lld,%lld): rows must be >= 0, vocab and hidden >= 1",
                  (long long)d->rows, (long long)d->vocab, (long long)d->hidden);
        return B200_ERR_INVALID_ARGUMENT;
    }
    // Tile arithmetic is in 32 bits: leave room for a block behind the end.
    if (d->rows > kMax - 8192 || d->vocab > kMax - 8192 || d->hidden > kMax - 8192) {
        set_error("(rows,vocab,hidden)=(%lld,%lld,%lld): every extent must be below 2^31 - 8192",
                  (long long)d->rows, (long long)d->vocab, (long long)d->hidden);
        return B200_ERR_UNSUPPORTED;
    }
    // Byte counts are in 64 bits, with room for what is kept of each.
    if (d->rows > (int64_t(1) << 46) / d->hidden || d->vocab > (int64_t(1) << 46) / d->hidden ||
        d->rows > (int64_t(1) << 50) / d->vocab) {
        set_error("(rows,vocab,hidden)=(%lld,%lld,%lld): operands must be below 2^46 elements, logits below 2^50",
                  (long long)d->rows, (long long)d->vocab, (long long)d->hidden);
        return B200_ERR_UNSUPPORTED;
    }
    if (d->hidden % 8 != 0) {
        set_error("hidden=%lld: rows must be whole 16-byte units for TMA (hidden %% 8 == 0)", (long long)d->hidden);
        return B200_ERR_UNSUPPORTED;
    }
    if (d->dtype != B200_VL_BF16 && d->dtype != B200_VL_F16) {
        set_error("dtype=%lld is neither B200_VL_BF16 nor B200_VL_F16", (long long)d->dtype);
        return B200_ERR_INVALID_ARGUMENT;
    }
    if (d->ld_hidden < d->hidden || d->ld_weight < d->hidden) {
        set_error("row pitches %lld, %lld are smaller than hidden=%lld", (long long)d->ld_hidden,
                  (long long)d->ld_weight, (long long)d->hidden);
        return B200_ERR_INVALID_ARGUMENT;
    }
    if (d->ld_hidden % 8 != 0 || d->ld_weight % 8 != 0) {
        set_error("row pitches %lld, %lld must be multiples of 8 elements (16 bytes)", (long long)d->ld_hidden,
                  (long long)d->ld_weight);
        return B200_ERR_UNSUPPORTED;
    }
    if (d->index_bytes != 4 && d->index_bytes != 8) {
        set_error("index_bytes=%lld is neither 4 nor 8", (long long)d->index_bytes);
        return B200_ERR_INVALID_ARGUMENT;
    }
    if (d->reduction != B200_VL_NONE && d->reduction != B200_VL_MEAN && d->reduction != B200_VL_SUM) {
        set_error("reduction=%lld is not one of NONE(0), MEAN(1), SUM(2)", (long long)d->reduction);
        return B200_ERR_INVALID_ARGUMENT;
    }
    if (d->top < 0 || d->top > kMaxTop) {
        set_error("top=%lld: a teacher's row holds 1 to %d logits (0: cross entropy)", (long long)d->top, kMaxTop);
        return B200_ERR_UNSUPPORTED;
    }
    if (d->top > 0) {
        if (d->teacher_dtype != B200_VL_F32 && d->teacher_dtype != B200_VL_BF16 && d->teacher_dtype != B200_VL_F16) {
            set_error("teacher_dtype=%lld is not one of BF16(0), F16(1), F32(2)", (long long)d->teacher_dtype);
            return B200_ERR_INVALID_ARGUMENT;
        }
        if (d->ld_index < d->top || d->ld_teacher < d->top) {
            set_error("row pitches %lld, %lld of the teacher are smaller than top=%lld", (long long)d->ld_index,
                      (long long)d->ld_teacher, (long long)d->top);
            return B200_ERR_INVALID_ARGUMENT;
        }
        // Its inverse and its square stay far inside 32 bits.
        if (!(d->temperature >= 0x1p-20 && d->temperature <= 0x1p20)) {
            set_error("temperature=%g must be between 2^-20 and 2^20", d->temperature);
            return B200_ERR_INVALID_ARGUMENT;
        }
    } else if (d->temperature != 1.0) {
        set_error("temperature=%g: the cross entropy has temperature 1", d->temperature);
        return B200_ERR_INVALID_ARGUMENT;
    }
    return B200_OK;
}

// The host's choices for a call: a function of the sizes and the SM count alone.
// Costs are in k-slices of a 256 x 256 pair tile (about 0.27 us).
static Layout layout_for(const B200VocabLossDesc& d, int64_t sms) {
    Layout l{};
    const int64_t T = std::max<int64_t>(d.rows, 1), K = std::max<int64_t>(d.top, 1);
    const int64_t V = d.vocab, D = d.hidden;
    const int64_t pairs = std::max<int64_t>(sms / 2, 1);
    const int64_t kd = ceil_div(D, kBK), kt = ceil_div(T, kBK);
    // Tiles of the logits: pairs 256 x 256, or single CTAs 128 x 256 or 128 x 128
    // where those finish in fewer rounds. A k-slice takes the longer of its products
    // (512 cycles for 128 x 256 columns of a CTA) and its operands' way from L2 to the
    // SM (57 bytes per cycle measured with all SMs reading, 32 KiB in 575 cycles; in
    // proportion with fewer), and a tile at least its epilogue.
    struct Shape { int cta_group, tile_n; };
    double best_rounds = 0.0;
    for (const Shape& c : {Shape{2, 256}, Shape{1, 256}, Shape{1, 128}}) {
        if (c.cta_group == 2 && T <= kRowsPerCta) continue;
        const int64_t tiles = ceil_div(T, kRowsPerCta * c.cta_group) * ceil_div(V, c.tile_n);
        const int64_t at_once = std::max<int64_t>(sms / c.cta_group, 1);
        const int64_t rows_a = c.cta_group == 2 ? kRowsPerCta : std::min<int64_t>(kRowsPerCta, align_up(T, 8));
        const double bytes = static_cast<double>(rows_a + c.tile_n / c.cta_group) / 256.0;
        const double slice =
            std::max(c.tile_n / 256.0, bytes * std::min(1.0, static_cast<double>(tiles) / static_cast<double>(at_once)));
        const double rounds = static_cast<double>(ceil_div(tiles, at_once)) *
                              (std::max(slice * static_cast<double>(kd), 8.0 * c.tile_n / 256) + 4.0);
        if (l.cta_group == 0 || rounds < best_rounds) {
            best_rounds = rounds;
            l.cta_group = c.cta_group;
            l.tile_n = c.tile_n;
        }
    }
    l.tile_m = kRowsPerCta * l.cta_group;
    l.cta_group_h = T <= kRowsPerCta ? 1 : 2;
    l.tile_m_h = kRowsPerCta * l.cta_group_h;
    l.rows_pad = align_up(T, l.tile_m_h);
    l.ld_gathered = align_up(D, 64);
    l.ld_part = align_up(D, 32);
    // The forward pass gathers only to save products (its rows do not meet): not
    // where all tiles run at once anyway (2.5 us of a 17 us call).
    const int64_t parts = ceil_div(V, l.tile_n / 2), longest = std::max(parts, d.top);
    l.merge_lanes = 0;
    if (T * longest <= kMergeHere && longest <= kMergeRowHere)
        for (l.merge_lanes = 1; l.merge_lanes < 32 && 8 * l.merge_lanes < longest;) l.merge_lanes *= 2;
    l.gather_forward = ceil_div(T, l.tile_m) * ceil_div(V, l.tile_n) > sms / l.cta_group && T > l.tile_m;
    // Piece of the vocabulary (in blocks of 256) and runs of the contractions of dH
    // and dW: the least k-slices on the longest cluster, over the three products of
    // all pieces, with eight k-slices for each launch's start and end. Widths: all
    // that G has room for, up to 64 between half of that and all of it where that is
    // not the whole vocabulary, and what stays in L2 between the three products, since
    // with a short D the way of G through HBM takes longer than the products. A further
    // run of a contraction writes and reads its sums once more, a further piece reads
    // and writes dH's sums.
    const int64_t blocks_v = ceil_div(V, kBN), nb = ceil_div(D, kBN), mb = l.rows_pad / l.tile_m_h;
    const int64_t slots_h = std::max<int64_t>(sms / l.cta_group_h, 1);
    const int64_t slots = std::max<int64_t>(sms / l.cta_group, 1);
    const int64_t most =
        std::max<int64_t>(1, std::min(blocks_v, std::max(kPieceBytes, 2 * l.rows_pad * D) / (2 * kBN * l.rows_pad)));
    const int64_t least = most == blocks_v ? most : std::max<int64_t>(1, most / 2);
    const int64_t step = std::max<int64_t>(1, (most - least) / 64);
    const int64_t in_l2 = std::max<int64_t>(1, kL2Piece / (2 * kBN * l.rows_pad));
    const int64_t run_bytes = int64_t(1800) << 10;  // bytes in the time of a k-slice
    auto splits_most = [&](int64_t tiles, int64_t slots_, int64_t rows) -> int64_t {
        if (tiles >= 4 * slots_) return 1;
        return std::max<int64_t>(1, std::min<int64_t>(kMaxSplits, kPartialBytes / (4 * rows * l.ld_part)));
    };
    auto rounds_of = [](int64_t tiles, int64_t slots_) { return ceil_div(tiles, slots_); };
    // dW of n blocks of columns in tiles of one or two blocks: with two, a tile's start
    // waits for TMEM (8 k-slices); with one, its operands keep all SMs 8 % below the
    // products' rate over many rounds.
    auto dw_blocks = [&](int64_t n, int64_t sub) {
        const int64_t rounds = rounds_of(ceil_div(n, sub) * nb, pairs);
        if (sub == 2) return rounds * (2 * kt + 8);
        return rounds >= 4 ? rounds * kt * 27 / 25 : rounds * kt;
    };
    auto cost16 = [&](int64_t rows) { return static_cast<int>(std::min<int64_t>(16 * 8 * rows * l.ld_part / run_bytes, 1 << 24)); };
    int64_t best = -1;
    for (int64_t i = in_l2 < least ? -1 : 0; least + i * step <= most; ++i) {
        const int64_t b = i < 0 ? in_l2 : least + i * step;
        const int64_t pieces = ceil_div(blocks_v, b), rest = blocks_v - (pieces - 1) * b;
        auto both = [&](auto cost) { return (pieces - 1) * cost(b) + cost(rest); };
        // What G costs a product that writes or reads it, where it does not stay in L2.
        auto hbm = [&](int64_t n) { return n > in_l2 ? 2 * l.rows_pad * n * kBN / run_bytes : 0; };
        const int64_t grad = both([&](int64_t n) {
            return std::max(rounds_of(ceil_div(T, l.tile_m) * ceil_div(n * kBN, l.tile_n), slots) * std::max<int64_t>(kd, 8), hbm(n)) + 8;
        });
        const int64_t slices_h = std::min(ceil_div(V, kBK), b * (kBN / kBK));
        const int64_t s_h = runs_for(static_cast<int>(mb * nb), static_cast<int>(slots_h), static_cast<int>(slices_h),
                                     static_cast<int>(splits_most(mb * nb, slots_h, l.rows_pad)), cost16(l.rows_pad));
        const int64_t dh = both([&](int64_t n) {
            return std::max(rounds_of(mb * nb * s_h, slots_h) * ceil_div(n * (kBN / kBK), s_h), hbm(n)) + 8;
        }) + 8 * l.rows_pad * l.ld_part * (s_h - 1 + pieces - 1) / run_bytes;
        auto dw_of = [&](int64_t s) {
            auto products = [&](int64_t n) {
                return s > 1 ? rounds_of(n * nb * s, pairs) * ceil_div(kt, s) : std::min(dw_blocks(n, 1), dw_blocks(n, 2));
            };
            return both([&](int64_t n) { return std::max(products(n), hbm(n)) + 8; }) +
                   (s > 1 ? 6 + 8 * b * kBN * l.ld_part * s / run_bytes : 0);
        };
        int64_t s_w = pieces > 1 ? 1
                                 : runs_for(static_cast<int>(b * nb), static_cast<int>(pairs), static_cast<int>(kt),
                                            static_cast<int>(splits_most(b * nb, pairs, b * kBN)), cost16(b * kBN));
        if (dw_of(1) <= dw_of(s_w)) s_w = 1;
        const int64_t dw = dw_of(s_w);
        const int64_t cost = grad + dh + dw;
        if (best < 0 || cost < best) {
            best = cost;
            l.piece = b * kBN;
            l.pieces = pieces;
            l.splits_h = s_h;
            l.splits_w = s_w;
            l.sub_w = s_w == 1 && dw_blocks(b, 2) < dw_blocks(b, 1) ? 2 : 1;
            l.slices_h = slices_h;
        }
    }
    // Room for twice the runs of dH that all rows would take: fewer rows may carry a
    // loss, which leaves clusters for more.
    l.splits_h = std::min({2 * l.splits_h, splits_most(mb * nb, slots_h, l.rows_pad), l.slices_h});
    l.cost16_h = cost16(l.rows_pad);
    l.cost16_w = cost16(l.piece);
    int64_t at = 256;
    auto take = [&](int64_t bytes) {
        const int64_t here = at;
        at = align_up(at + bytes, 256);
        return here;
    };
    l.flag = take(4 * T);
    l.rowmap = take(4 * T);
    l.inv = take(4 * T);
    l.ecol = take(4 * T * K);
    l.eq = take(d.top > 0 ? 4 * T * K : 0);
    // One entry for each half tile of the padded vocabulary and one behind them.
    l.epos_ld = ceil_div(V, kBN) * (2 * kBN / l.tile_n) + 1;
    l.epos = take(d.top > 0 ? 2 * T * l.epos_ld : 0);
    const int64_t common = at;
    l.zsel = take(4 * T * K);
    l.part = take(8 * ceil_div(V, l.tile_n / 2) * T);
    l.row_loss = take(4 * T);
    l.gathered_forward = take(l.gather_forward ? 2 * T * l.ld_gathered : 0);
    l.bytes_forward = at;
    at = common;
    l.rgrad = take(16 * T);
    l.gathered_backward = take(2 * T * l.ld_gathered);
    l.split = d.dtype == B200_VL_F16 && d.reduction == B200_VL_NONE;
    l.weighed = take(l.split ? 2 * T * l.ld_gathered : 0);
    l.g = take(2 * T * l.piece);
    l.part_h = take(4 * l.splits_h * l.rows_pad * l.ld_part);
    l.part_w = take(l.splits_w > 1 ? 4 * l.splits_w * l.piece * l.ld_part : 0);
    l.bytes_backward = at;
    return l;
}

using KernelFn = void (*)(CUtensorMap, CUtensorMap, CUtensorMap, CUtensorMap, CUtensorMap, Params);

struct Variant {
    int cta_group, tile_n, op, sub_m;
    bool fp16;
    KernelFn fn;
    int smem;
};

template <int kCtaGroup, int kTileN, int kOp, bool kHalf = false, int kSubM = 1>
static Variant variant() {
    return {kCtaGroup, kTileN, kOp, kSubM, kHalf, vocab_gemm_kernel<kCtaGroup, kTileN, kOp, kHalf, kSubM>,
            Cfg<kCtaGroup, kTileN, kSubM>::kSmemBytes};
}

// Every product in the shapes that the layout can choose.
static const Variant* variants(int* count) {
    static const Variant all[] = {
        variant<2, 256, kStats>(), variant<1, 256, kStats>(), variant<1, 128, kStats>(),
        variant<2, 256, kStatsShort>(), variant<1, 256, kStatsShort>(), variant<1, 128, kStatsShort>(),
        variant<2, 256, kGrad, false>(), variant<1, 256, kGrad, false>(), variant<1, 128, kGrad, false>(),
        variant<2, 256, kGrad, true>(), variant<1, 256, kGrad, true>(), variant<1, 128, kGrad, true>(),
        variant<2, 256, kDh>(), variant<1, 256, kDh>(),
        variant<2, 256, kDw, false>(), variant<2, 256, kDw, true>(), variant<2, 256, kDwParts>(),
        variant<2, 256, kDw, false, 2>(), variant<2, 256, kDw, true, 2>(),
    };
    *count = static_cast<int>(sizeof(all) / sizeof(all[0]));
    return all;
}

static const Variant* variant_of(int cta_group, int tile_n, int op, bool fp16, int sub_m) {
    int n = 0;
    const Variant* all = variants(&n);
    const bool half = fp16 && (op == kGrad || op == kDw);
    for (int i = 0; i < n; ++i)
        if (all[i].cta_group == cta_group && all[i].tile_n == tile_n && all[i].op == op && all[i].fp16 == half &&
            all[i].sub_m == sub_m)
            return all + i;
    return nullptr;
}

struct DeviceState {
    bool ready = false;
    int sms = 0;
    int pairs = 0;
};

static int device_state(DeviceState* out) {
    constexpr int kMaxDevices = 64;
    static DeviceState cache[kMaxDevices];
    static std::mutex mu;
    int device = 0;
    B200_CUDA_TRY(cudaGetDevice(&device));
    // Binds the device's context to a thread that has not called the runtime yet
    // (autograd's backward threads): the tensor maps are encoded by the driver.
    B200_CUDA_TRY(cudaSetDevice(device));
    DeviceProps props;
    int rc = device_props(device, &props);
    if (rc != B200_OK) return rc;
    if (props.cc_major != 10 || props.cc_minor != 0) {
        set_error("device %d has compute capability %d.%d; this library is built for sm_100a (10.0)", device,
                  props.cc_major, props.cc_minor);
        return B200_ERR_UNSUPPORTED;
    }
    std::lock_guard<std::mutex> lock(mu);
    DeviceState& s = cache[device];
    if (!s.ready) {
        int n = 0;
        const Variant* all = variants(&n);
        for (int i = 0; i < n; ++i)
            B200_CUDA_TRY(cudaFuncSetAttribute(reinterpret_cast<const void*>(all[i].fn),
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, all[i].smem));
        // Loaded now, not at a first launch that a stream capture may hold.
        cudaFuncAttributes loaded;
        for (const void* fn : {reinterpret_cast<const void*>(teacher_kernel<32>), reinterpret_cast<const void*>(teacher_kernel<128>),
                               reinterpret_cast<const void*>(rows_kernel),
                               reinterpret_cast<const void*>(weigh_most_kernel), reinterpret_cast<const void*>(weigh_kernel),
                               reinterpret_cast<const void*>(merge_kernel),
                               reinterpret_cast<const void*>(finish_kernel)})
            B200_CUDA_TRY(cudaFuncGetAttributes(&loaded, fn));
        cudaLaunchConfig_t cfg = {};
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = 2;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.gridDim = dim3(props.sm_count & ~1, 1, 1);
        cfg.blockDim = dim3(kThreads, 1, 1);
        cfg.dynamicSmemBytes = all[0].smem;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        int clusters = 0;
        const cudaError_t err = cudaOccupancyMaxActiveClusters(&clusters, reinterpret_cast<const void*>(all[0].fn), &cfg);
        if (err != cudaSuccess || clusters <= 0) {
            cudaGetLastError();
            clusters = props.sm_count / 2;
        }
        s.sms = props.sm_count;
        s.pairs = std::max(clusters, 1);
        s.ready = true;
    }
    *out = s;
    return B200_OK;
}

// Programmatic dependent launch is on unless B200_PDL=0, as for the GEMM's plans.
static bool pdl_on() {
    const char* e = std::getenv("B200_PDL");
    return e == nullptr || e[0] != '0';
}

// Launches that follow another kernel of the same call start their set-up while
// it ends (programmatic dependent launch); each waits for it before it touches
// global memory.
template <typename... KArgs, typename... Args>
static int launch(void (*fn)(KArgs...), int grid, int block, int smem, int cluster, bool dependent, cudaStream_t stream,
                  Args... args) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (cluster > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = cluster;
        attr[n].val.clusterDim.y = 1;
        attr[n++].val.clusterDim.z = 1;
    }
    if (dependent && pdl_on()) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    cfg.gridDim = dim3(grid, 1, 1);
    cfg.blockDim = dim3(block, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = n;
    B200_CUDA_TRY(cudaLaunchKernelEx(&cfg, fn, static_cast<KArgs>(args)...));
    return B200_OK;
}

struct Call {
    const B200VocabLossDesc* d;
    Layout l;
    DeviceState dev;
    uint8_t* ws;
    cudaStream_t stream;
    CUtensorMapDataType type;
    template <typename T>
    T* at(int64_t offset) const { return reinterpret_cast<T*>(ws + offset); }
    Head* head() const { return reinterpret_cast<Head*>(ws); }
};

static int check_pointers(std::initializer_list<std::pair<const void*, const char*>> ptrs) {
    for (const auto& p : ptrs) {
        if (p.first == nullptr) {
            set_error("%s must be a device pointer", p.second);
            return B200_ERR_INVALID_ARGUMENT;
        }
    }
    return B200_OK;
}

static int check_aligned(std::initializer_list<std::pair<const void*, const char*>> ptrs) {
    for (const auto& p : ptrs) {
        if (reinterpret_cast<uintptr_t>(p.first) % 16 != 0) {
            set_error("%s %p is not 16-byte aligned (TMA requirement)", p.second, p.first);
            return B200_ERR_UNSUPPORTED;
        }
    }
    return B200_OK;
}

static int map_2d(const Call& c, CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int64_t ld,
                  int box_rows, int box_cols) {
    return encode_tmap_2d(map, c.type, 2, base, rows, cols, ld, box_rows, box_cols, CU_TENSOR_MAP_SWIZZLE_128B);
}

static float g_scale(const B200VocabLossDesc& d) { return d.dtype == B200_VL_F16 ? kHalfScale : 1.0f; }

// Targets, row numbers and the gathered copy of H.
static int launch_rows(const Call& c, const void* index, const void* teacher, const void* hidden, bool gather,
                       int64_t gathered, const float* grad, const float* lse,
                       const float* target_logp) {
    const B200VocabLossDesc& d = *c.d;
    const Layout& l = c.l;
    if (d.top > 0) {
        TeacherParams t{};
        t.index = index;
        t.teacher = teacher;
        t.index_bytes = static_cast<int>(d.index_bytes);
        t.teacher_dtype = static_cast<int>(d.teacher_dtype);
        t.ld_index = d.ld_index;
        t.ld_teacher = d.ld_teacher;
        t.rows = static_cast<int>(d.rows);
        t.vocab = static_cast<int>(d.vocab);
        t.top = static_cast<int>(d.top);
        t.inv_tau = static_cast<float>(1.0 / d.temperature);
        t.half = l.tile_n / 2;
        t.epos_ld = l.epos_ld;
        t.epos = c.at<unsigned short>(l.epos);
        t.ecol = c.at<int>(l.ecol);
        t.eq = c.at<float>(l.eq);
        t.flag = c.at<int>(l.flag);
        t.zsel = grad == nullptr ? c.at<float>(l.zsel) : nullptr;
        if (!gather) {
            t.head = c.head();
            t.rowmap = c.at<int>(l.rowmap);
            t.inv = c.at<int>(l.inv);
        }
        int pad = 2;
        while (pad < t.top) pad *= 2;
        const int rc = pad <= 32 && d.rows > 8 * c.dev.sms
                           ? launch(teacher_kernel<32>, static_cast<int>(d.rows), 32, 0, 1, false, c.stream, t, pad)
                           : launch(teacher_kernel<128>, static_cast<int>(d.rows), 128, 0, 1, false, c.stream, t, pad);
        if (rc != B200_OK || !gather) return rc;
    }
    RowsParams r{};
    r.head = c.head();
    r.target = d.top > 0 ? nullptr : index;
    r.index_bytes = static_cast<int>(d.index_bytes);
    r.ignore = d.ignore_index;
    r.rows = static_cast<int>(d.rows);
    r.vocab = static_cast<int>(d.vocab);
    r.gather = gather;
    // Rows that do not start on 128-byte lines cost every tile a fifth more sectors
    // (768 x 50001 x 1016, pitch 1016 against 1024: 72 against 61 us).
    r.copy_all = gather && d.ld_hidden % 64 != 0 && d.rows > 1;
    r.reduction = static_cast<int>(d.reduction);
    r.flag = c.at<int>(l.flag);
    r.ecol = c.at<int>(l.ecol);
    r.rowmap = c.at<int>(l.rowmap);
    r.inv = c.at<int>(l.inv);
    r.grad = grad;
    r.lse = lse;
    r.target_logp = target_logp;
    r.rgrad = grad != nullptr ? c.at<float4>(l.rgrad) : nullptr;
    r.tau = static_cast<float>(d.temperature);
    r.scale = g_scale(d);
    r.split = l.split;
    r.hidden = static_cast<const uint4*>(hidden);
    r.copy = c.at<uint4>(gathered);
    r.ld = d.ld_hidden / 8;
    r.ld_copy = l.ld_gathered / 8;
    r.vecs = static_cast<int>(d.hidden / 8);
    const int64_t blocks = gather ? std::min<int64_t>(ceil_div(d.rows, 8), c.dev.sms) : 1;
    return launch(rows_kernel, static_cast<int>(blocks), 1024, 0, 1, d.top > 0, c.stream, r);
}

// The copy of H with the rows' weights.
static int launch_weigh(const Call& c, const void* hidden) {
    const B200VocabLossDesc& d = *c.d;
    const Layout& l = c.l;
    WeighParams w{};
    w.head = c.head();
    w.rgrad = c.at<float4>(l.rgrad);
    w.hidden = static_cast<const uint4*>(hidden);
    w.copy = c.at<uint4>(l.gathered_backward);
    w.weighed = c.at<uint4>(l.weighed);
    w.ld = d.ld_hidden / 8;
    w.ld_copy = l.ld_gathered / 8;
    w.rows = static_cast<int>(d.rows);
    w.vecs = static_cast<int>(d.hidden / 8);
    w.tau = static_cast<float>(d.temperature) / g_scale(d);
    const int blocks = static_cast<int>(std::min<int64_t>(ceil_div(d.rows, kWeighWarps), 4 * c.dev.sms));
    const int rc = launch(weigh_most_kernel, blocks, 32 * kWeighWarps, 0, 1, true, c.stream, w);
    return rc != B200_OK ? rc : launch(weigh_kernel, blocks, 32 * kWeighWarps, 0, 1, true, c.stream, w);
}

static Params base_params(const Call& c) {
    const B200VocabLossDesc& d = *c.d;
    Params p{};
    p.head = c.head();
    p.timeout_ns = wait_timeout_ns();
    p.fp16 = d.dtype == B200_VL_F16;
    p.rows = static_cast<int>(d.rows);
    p.splits = 1;
    p.rowmap = d.top > 0 ? c.at<int>(c.l.rowmap) : nullptr;
    p.epos = c.at<unsigned short>(c.l.epos);
    p.epos_ld = c.l.epos_ld;
    p.ecol = c.at<int>(c.l.ecol);
    p.eq = d.top > 0 ? c.at<float>(c.l.eq) : nullptr;
    p.top = static_cast<int>(std::max<int64_t>(d.top, 1));
    p.c2 = static_cast<float>(1.4426950408889634 / d.temperature);
    return p;
}

// Raster groups of about 4096 rows of A whose panel stays within 64 MiB.
static int group_for(int64_t tile_m, int64_t k) {
    const double rows = std::min(4096.0, 64.0 * 1024 * 1024 / (2.0 * std::max<int64_t>(k, 64)));
    return std::max(2, std::min(32, static_cast<int>(rows / tile_m + 0.5)));
}

static int64_t slots_of(const Call& c, int cta_group) { return cta_group == 2 ? c.dev.pairs : c.dev.sms; }

static int launch_gemm(const Call& c, int op, int cta_group, int tile_n, int sub_m, int64_t tiles, const CUtensorMap& a0,
                       const CUtensorMap& a1, const CUtensorMap& b0, const CUtensorMap& b1, const CUtensorMap& dmap,
                       const Params& p) {
    const Variant* v = variant_of(cta_group, tile_n, op, p.fp16, sub_m);
    if (v == nullptr) {
        set_error("internal error: no kernel for product %d with %d x %d tiles", op, kRowsPerCta * cta_group * sub_m,
                  tile_n);
        return B200_ERR_INTERNAL;
    }
    const int grid = static_cast<int>(std::max<int64_t>(1, std::min(tiles, slots_of(c, cta_group)))) * cta_group;
    return launch(v->fn, grid, kThreads, v->smem, cta_group, true, c.stream, a0, a1, b0, b1, dmap, p);
}

// Rows of an A tile that are loaded: all 128, or in single-CTA tiles the rows of
// the call. What a tile holds beyond them reaches only rows that nobody reads.
static int a_rows(const B200VocabLossDesc& d, int cta_group) {
    return cta_group == 1 ? static_cast<int>(std::min<int64_t>(kRowsPerCta, align_up(d.rows, 8))) : kRowsPerCta;
}

static int begin(const B200VocabLossDesc* d, void* workspace, int64_t bytes, bool backward, void* stream, Call* c) {
    int rc = device_state(&c->dev);
    if (rc != B200_OK) return rc;
    c->d = d;
    c->l = layout_for(*d, c->dev.sms);
    c->ws = static_cast<uint8_t*>(workspace);
    c->stream = static_cast<cudaStream_t>(stream);
    c->type = d->dtype == B200_VL_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const int64_t need = backward ? c->l.bytes_backward : c->l.bytes_forward;
    if (bytes < need) {
        set_error("workspace of %lld bytes is smaller than the %lld needed", (long long)bytes, (long long)need);
        return B200_ERR_INVALID_ARGUMENT;
    }
    if (reinterpret_cast<uintptr_t>(workspace) % 256 != 0) {
        set_error("workspace %p is not 256-byte aligned", workspace);
        return B200_ERR_INVALID_ARGUMENT;
    }
    return B200_OK;
}

static int forward(const B200VocabLossDesc* d, const void* hidden, const void* weight, const void* index,
                   const void* teacher, float* loss, float* lse, float* target_logp, void* workspace, int64_t bytes,
                   void* stream) {
    int rc = check_desc(d);
    if (rc != B200_OK) return rc;
    if (d->rows == 0) {
        set_error("rows=0: there is nothing to launch");
        return B200_ERR_UNSUPPORTED;
    }
    rc = check_pointers({{hidden, "hidden"}, {weight, "weight"}, {index, "index"}, {loss, "loss"}, {lse, "lse"},
                         {target_logp, "target_logp"}, {workspace, "workspace"}});
    if (rc == B200_OK && d->top > 0) rc = check_pointers({{teacher, "teacher"}});
    if (rc == B200_OK) rc = check_aligned({{hidden, "hidden"}, {weight, "weight"}});
    if (rc != B200_OK) return rc;
    Call c{};
    rc = begin(d, workspace, bytes, false, stream, &c);
    if (rc != B200_OK) return rc;
    const Layout& l = c.l;
    CUtensorMap a0, a1, b;
    const int box_n = l.tile_n / l.cta_group, box_m = a_rows(*d, l.cta_group);
    rc = map_2d(c, &a0, hidden, d->rows, d->hidden, d->ld_hidden, box_m, kBK);
    if (rc == B200_OK)
        rc = l.gather_forward ? map_2d(c, &a1, c.at<void>(l.gathered_forward), d->rows, d->hidden, l.ld_gathered, box_m, kBK)
                              : (a1 = a0, B200_OK);
    if (rc == B200_OK) rc = map_2d(c, &b, weight, d->vocab, d->hidden, d->ld_weight, box_n, kBK);
    if (rc != B200_OK) return rc;
    rc = launch_rows(c, index, teacher, hidden, l.gather_forward, l.gathered_forward, nullptr, nullptr, nullptr);
    if (rc != B200_OK) return rc;
    Params p = base_params(c);
    p.n = static_cast<int>(d->vocab);
    p.k = static_cast<int>(d->hidden);
    p.group_m = group_for(l.tile_m, d->hidden);
    p.zsel = c.at<float>(l.zsel);
    p.part = c.at<float2>(l.part);
    p.early = !l.gather_forward;
    p.part_ld = ceil_div(d->vocab, l.tile_n / 2);
    p.a_bytes = box_m * kBK * 2;
    MergeParams m{};
    m.head = c.head();
    m.part = p.part;
    m.part_ld = p.part_ld;
    m.tiles = static_cast<int>(p.part_ld);
    // A block for each row pays where there are few rows of many half tiles (one row of
    // 2004: 21.0 against 21.9 us; 1000 of 235 33.1 and 37.4, 1021 of 391 41.4 and 45.0).
    m.warps_per_row = d->rows <= c.dev.sms && m.tiles > 512 ? kMergeWarps : 1;
    m.lanes = l.merge_lanes;
    m.rows = static_cast<int>(d->rows);
    m.top = p.top;
    m.reduction = static_cast<int>(d->reduction);
    m.count = d->reduction == B200_VL_MEAN && d->top > 0 && !l.gather_forward;
    m.inv = c.at<int>(l.inv);
    m.flag = c.at<int>(l.flag);
    m.eq = p.eq;
    m.zsel = p.zsel;
    m.c2 = p.c2;
    m.inv_tau = static_cast<float>(1.0 / d->temperature);
    m.tau2 = static_cast<float>(d->temperature * d->temperature);
    m.lse = lse;
    m.target_logp = target_logp;
    m.row_loss = d->reduction == B200_VL_NONE ? loss : c.at<float>(l.row_loss);
    m.loss = loss;
    p.merge = m;
    rc = launch_gemm(c, d->hidden <= kDrainMost * kBK ? kStatsShort : kStats, l.cta_group, l.tile_n, 1,
                     ceil_div(d->rows, l.tile_m) * ceil_div(d->vocab, l.tile_n), a0, a1, b, b, b, p);
    if (rc != B200_OK || m.lanes != 0) return rc;
    return launch(merge_kernel, static_cast<int>(ceil_div(d->rows, kMergeWarps / m.warps_per_row)), 32 * kMergeWarps, 0, 1,
                  true, c.stream, m);
}

static int backward(const B200VocabLossDesc* d, const void* hidden, const void* weight, const void* index,
                    const void* teacher, const float* lse, const float* target_logp, const float* grad_loss,
                    void* d_hidden, void* d_weight, void* workspace, int64_t bytes, void* stream) {
    int rc = check_desc(d);
    if (rc != B200_OK) return rc;
    if (d->rows == 0 || (d_hidden == nullptr && d_weight == nullptr)) {
        set_error("rows=%lld with %s: there is nothing to launch", (long long)d->rows,
                  d_hidden == nullptr && d_weight == nullptr ? "no gradient asked for" : "gradients to write");
        return B200_ERR_UNSUPPORTED;
    }
    rc = check_pointers({{hidden, "hidden"}, {weight, "weight"}, {index, "index"}, {lse, "lse"},
                         {target_logp, "target_logp"}, {grad_loss, "grad_loss"}, {workspace, "workspace"}});
    if (rc == B200_OK && d->top > 0) rc = check_pointers({{teacher, "teacher"}});
    if (rc == B200_OK)
        rc = check_aligned({{hidden, "hidden"}, {weight, "weight"}, {d_hidden, "d_hidden"}, {d_weight, "d_weight"}});
    if (rc != B200_OK) return rc;
    Call c{};
    rc = begin(d, workspace, bytes, true, stream, &c);
    if (rc != B200_OK) return rc;
    const Layout& l = c.l;
    void* hg = c.at<void>(l.gathered_backward);
    void* g = c.at<void>(l.g);
    CUtensorMap h_k, hg_k, h_mn, hg_mn, w_k, w_mn, g_st, g_k, g_mn, dh_st, dw_st;
    const bool weigh = l.split && d_weight != nullptr;
    std::memset(&dw_st, 0, sizeof(dw_st));
    const int64_t T = d->rows, V = d->vocab, D = d->hidden;
    const int box_m = a_rows(*d, l.cta_group), box_m_h = a_rows(*d, l.cta_group_h);
    rc = map_2d(c, &h_k, hidden, T, D, d->ld_hidden, box_m, kBK);
    if (rc == B200_OK) rc = map_2d(c, &hg_k, hg, T, D, l.ld_gathered, box_m, kBK);
    if (rc == B200_OK)
        rc = weigh ? map_2d(c, &h_mn, c.at<void>(l.weighed), T, D, l.ld_gathered, kBK, 64)
                   : map_2d(c, &h_mn, hidden, T, D, d->ld_hidden, kBK, 64);
    if (rc == B200_OK) rc = weigh ? (hg_mn = h_mn, B200_OK) : map_2d(c, &hg_mn, hg, T, D, l.ld_gathered, kBK, 64);
    if (rc == B200_OK) rc = map_2d(c, &w_k, weight, V, D, d->ld_weight, l.tile_n / l.cta_group, kBK);
    if (rc == B200_OK) rc = map_2d(c, &w_mn, weight, V, D, d->ld_weight, kBK, 64);
    if (rc == B200_OK) rc = map_2d(c, &g_st, g, T, l.piece, l.piece, 32, 64);
    if (rc == B200_OK) rc = map_2d(c, &g_k, g, T, l.piece, l.piece, box_m_h, kBK);
    if (rc == B200_OK) rc = map_2d(c, &g_mn, g, T, l.piece, l.piece, kBK, 64);
    auto partial_map = [&](CUtensorMap* map, int64_t offset, int64_t rows) {
        return encode_tmap_2d(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, c.at<void>(offset), rows, D, l.ld_part, 32, 32,
                              CU_TENSOR_MAP_SWIZZLE_128B);
    };
    if (rc == B200_OK) rc = partial_map(&dh_st, l.part_h, l.splits_h * l.rows_pad);
    if (rc == B200_OK && d_weight != nullptr)
        rc = l.splits_w > 1 ? partial_map(&dw_st, l.part_w, l.splits_w * l.piece) : map_2d(c, &dw_st, d_weight, V, D, D, 32, 64);
    if (rc != B200_OK) return rc;
    rc = launch_rows(c, index, teacher, hidden, true, l.gathered_backward, grad_loss, lse, target_logp);
    if (rc == B200_OK && weigh) rc = launch_weigh(c, hidden);
    for (int64_t v0 = 0; rc == B200_OK && v0 < V; v0 += l.piece) {
        const int64_t vp = std::min(l.piece, V - v0);
        Params p = base_params(c);
        p.v0 = static_cast<int>(v0);
        p.rgrad = c.at<float4>(l.rgrad);
        p.zsel = const_cast<float*>(target_logp);
        p.n = static_cast<int>(vp);
        p.k = static_cast<int>(D);
        p.group_m = group_for(l.tile_m, D);
        p.a_bytes = box_m * kBK * 2;
        p.piece_no = static_cast<int>(v0 / l.piece) + 1;
        rc = launch_gemm(c, kGrad, l.cta_group, l.tile_n, 1, ceil_div(T, l.tile_m) * ceil_div(vp, l.tile_n), h_k, hg_k, w_k,
                         w_k, g_st, p);
        if (rc == B200_OK && d_hidden != nullptr) {
            Params q = p;
            q.n = static_cast<int>(D);
            q.k = static_cast<int>(vp);
            q.group_m = group_for(l.tile_m_h, l.piece);
            q.a_bytes = box_m_h * kBK * 2;
            q.splits = static_cast<int>(l.splits_h);
            q.run_slots = static_cast<int>(slots_of(c, l.cta_group_h));
            q.run_slices = static_cast<int>(l.slices_h);
            q.run_cost16 = l.cost16_h;
            q.rows_pad = static_cast<int>(l.rows_pad);
            q.accumulate = v0 > 0;
            rc = launch_gemm(c, kDh, l.cta_group_h, kBN, 1, l.rows_pad / l.tile_m_h * ceil_div(D, kBN) * l.splits_h, g_k, g_k,
                             w_mn, w_mn, dh_st, q);
        }
        if (rc == B200_OK && d_weight != nullptr) {
            Params q = p;
            q.m = static_cast<int>(vp);
            q.n = static_cast<int>(D);
            q.group_m = group_for(2 * kRowsPerCta * l.sub_w, T);
            q.a_bytes = kRowsPerCta * kBK * 2;
            q.splits = static_cast<int>(l.splits_w);
            q.run_slots = static_cast<int>(slots_of(c, 2));
            q.run_cost16 = l.cost16_w;
            q.rows_pad = static_cast<int>(l.piece);
            rc = launch_gemm(c, l.splits_w > 1 ? kDwParts : kDw, 2, kBN, l.sub_w,
                             ceil_div(vp, 2 * kRowsPerCta * l.sub_w) * ceil_div(D, kBN) * l.splits_w, g_mn, g_mn, h_mn, hg_mn, dw_st, q);
        }
    }
    if (rc != B200_OK) return rc;
    FinishParams f{};
    f.head = c.head();
    f.inv = c.at<int>(l.inv);
    f.part_h = c.at<float>(l.part_h);
    f.part_w = d_weight != nullptr && l.splits_w > 1 ? c.at<float>(l.part_w) : nullptr;
    f.ld_part = l.ld_part;
    f.stride_h = l.rows_pad * l.ld_part;
    f.stride_w = l.piece * l.ld_part;
    f.splits_h = static_cast<int>(l.splits_h);
    f.splits_w = static_cast<int>(l.splits_w);
    f.tile_m_h = static_cast<int>(l.tile_m_h);
    f.slots_h = static_cast<int>(slots_of(c, l.cta_group_h));
    f.slots_w = static_cast<int>(slots_of(c, 2));
    f.slices_h = static_cast<int>(l.slices_h);
    f.cost16_h = l.cost16_h;
    f.cost16_w = l.cost16_w;
    f.rows = static_cast<int>(T);
    f.hidden = static_cast<int>(D);
    f.vocab = static_cast<int>(V);
    f.fp16 = d->dtype == B200_VL_F16;
    f.rgrad = l.split ? c.at<float4>(l.rgrad) : nullptr;
    f.tau = static_cast<float>(d->temperature) / g_scale(*d);
    f.d_hidden = d_hidden;
    f.d_weight = d_weight;
    for (f.width = 256; f.width > 32 && f.width / 2 >= D / 8;) f.width /= 2;
    const int64_t rows = (d_hidden != nullptr ? T : 0) + (f.part_w != nullptr ? V : 0);
    const int64_t blocks = std::min<int64_t>(ceil_div(rows, 256 / f.width), 8 * c.dev.sms);
    return launch(finish_kernel, static_cast<int>(std::max<int64_t>(1, blocks)), 256, 0, 1, true, c.stream, f);
}

}  // namespace vl
}  // namespace b200

extern "C" {

size_t b200_vocab_loss_desc_size(void) { return sizeof(B200VocabLossDesc); }
size_t b200_vocab_loss_info_size(void) { return sizeof(B200VocabLossInfo); }

int b200_vocab_loss_info(const B200VocabLossDesc* desc, int sm_count, B200VocabLossInfo* out) {
    B200_ABI_GUARD_BEGIN
    b200::clear_error();
    if (out == nullptr || sm_count < 1) {
        b200::set_error("out must not be NULL and sm_count=%d must be positive", sm_count);
        return B200_ERR_INVALID_ARGUMENT;
    }
    std::memset(out, 0, sizeof(*out));
    const int rc = b200::vl::check_desc(desc);
    if (rc != B200_OK) return rc;
    const b200::vl::Layout l = b200::vl::layout_for(*desc, sm_count);
    out->cta_group = l.cta_group;
    out->tile_m = l.tile_m;
    out->tile_n = l.tile_n;
    out->tile_m_weight = 2 * b200::vl::kRowsPerCta * l.sub_w;
    out->piece = l.piece;
    out->pieces = l.pieces;
    out->splits_hidden = l.splits_h;
    out->splits_weight = l.splits_w;
    out->workspace_forward = l.bytes_forward;
    out->workspace_backward = l.bytes_backward;
    const int64_t teacher = desc->top > 0 ? 1 : 0;
    out->launches_forward = desc->rows == 0 ? 0 : 2 + (l.gather_forward ? teacher : 0) + (l.merge_lanes == 0 ? 1 : 0);
    out->launches_backward = desc->rows == 0 ? 0 : 2 + teacher + (l.split ? 2 : 0) + 3 * l.pieces;
    return B200_OK;
    B200_ABI_GUARD_END
}

int b200_vocab_loss_forward(const B200VocabLossDesc* desc, const void* hidden, const void* weight,
                            const void* index, const void* teacher, float* loss, float* lse,
                            float* target_logp, void* workspace, int64_t workspace_bytes, void* stream) {
    B200_ABI_GUARD_BEGIN
    b200::clear_error();
    return b200::vl::forward(desc, hidden, weight, index, teacher, loss, lse, target_logp, workspace, workspace_bytes, stream);
    B200_ABI_GUARD_END
}

int b200_vocab_loss_backward(const B200VocabLossDesc* desc, const void* hidden, const void* weight,
                             const void* index, const void* teacher, const float* lse,
                             const float* target_logp, const float* grad_loss, void* d_hidden, void* d_weight,
                             void* workspace, int64_t workspace_bytes, void* stream) {
    B200_ABI_GUARD_BEGIN
    b200::clear_error();
    return b200::vl::backward(desc, hidden, weight, index, teacher, lse, target_logp, grad_loss, d_hidden, d_weight,
                              workspace, workspace_bytes, stream);
    B200_ABI_GUARD_END
}

}  // extern "C"
