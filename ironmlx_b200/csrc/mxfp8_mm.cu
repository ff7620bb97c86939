// y = dequantize(x_q) . dequantize(w)^T with both operands in mxfp8 (e4m3 codes, one power of two for 32 values):
//   y[m, n] = bf16( sum over the blocks g of 2^(sx + sw - 254) * sum over k in g of qx * qw )
// That is what tcgen05.mma.kind::mxf8f6f4.block_scale computes, K = 32 a step with one scale a row and step, sums in fp32:
// nothing is dequantized, the codes go from memory to the tensor cores by TMA alone.  (The tensor cores cut an addition off, they
// do not round it: a sum of in / 32 steps loses in 2^-30.5 of it if all its terms have one sign, 2^-18 at 5120, next to 2^-9 of
// the output's rounding.  Tensor memory has no room for more sums at 256 columns.)
//
// Both operands have the same form, so that one kernel serves both orientations: P (128 rows, the lanes of the accumulator) and
// Q (NT rows, its columns), both K-major with 128-byte swizzle, 128 codes a stage.
//   few rows of x   P = weight, Q = the rows (SWAP): the weight's bytes bound it, its tiles are spread over the SMs
//   many rows       P = the rows, Q = weight: the tensor cores bound it.  Tiles of 256 rows by pairs of CTAs
//                   (cta_group::2), each of which brings half of Q.
// Few tiles for the GPU: the K range of a tile is cut over the CTAs of a cluster; each leaves its fp32 sums in shared memory,
// sends every other CTA its columns in one bulk copy (a row, 2048 -> 8192, cut in two: 7.7 us, read by the receiver
// 8.7, sent word by word 9.5, when the rest took 0.7 longer than now) and adds its own over all of them, in rank order.
//
// Scales lie in memory as the format has them, [rows, in / 32] bytes.  The MMA reads them from tensor memory, four K steps in
// a word, row r in lane r mod 32 of column r / 32: four warps fetch them as 16-byte pieces a row (four stages at a time, one
// fetch ahead; as words where rows do not start on 16 bytes), write them into that order beside the stage, and tcgen05.cp takes
// them over, ordered before the MMAs that follow it.  A stage's slot in tensor memory is written again no sooner than its shared
// memory, whose release waits for the MMAs that read both.  Rows and blocks past the end get the scale 1 and, from TMA, codes of
// zero.
//
// Eleven warps: 0..3 epilogue, 4..7 scales, 8 MMA and tensor memory, 9 loads, 10 (of a pair) tells CTA 0, whose warp 8 issues
// the MMAs of both, what has arrived in its own.  Two accumulators alternate, so that the next tile's MMAs run beside the
// epilogue; 2 x 256 columns leave no room for the scales: at NT = 256 the two share 60 columns, which the epilogue takes out
// first.  Every wait is bounded; on expiry what is in flight is waited for, tensor memory is freed, the status word is set and
// the tiles concerned are NaN.
//
// On a B200, the kernel alone: 8192 rows, 2048 -> 8192, 102 us, 2.7 PFLOP/s, 81% of twice cuBLAS' bf16 rate (in a loop of
// seconds the power limit makes it 122 to 125 us); 777 rows, 4096 -> 2048, 12.2 us; 64 rows, 2048 -> 152064, 55 to 59 us, 6.2 to 5.8 TB/s; one row,
// 2048 -> 8192, 7 us, of which 4 are a launch's and the ring's filling.  What a K step of 128 costs beside its MMAs bounds all that
// is not large: 340 cycles for the warp that issues them, before it issued by predicates and looked ahead 600.
#include <atomic>
#include <type_traits>

#include "tcgen05.cuh"
#include "../../include/ironmlx_b200_testing.h"

namespace imx {

namespace {

using namespace tc;

constexpr size_t kStatusBytes = 256;
constexpr int kMxThreads = 352;
constexpr int kMxK = 128;                          // codes of a row in a stage
constexpr int kMxMaxStages = 10;
constexpr int kMxGroups = 2;                       // groups of four K steps whose scales are in shared memory
constexpr int kMxMaxSplits = 8;                    // CTAs of a cluster that cut the K range of a tile
constexpr int kMxMost = 0x7fffff00;                // rows of either operand, and their length: a tile that starts below ends within 31 bits
std::atomic<int> g_mx_give_up{0};                  // see imx_testing_mxfp8_give_up

template <int NT, bool SWAP, bool PAIR>
struct Plan {
    static constexpr int kQParts = NT > 128 ? 2 : 1;                     // 128-row parts of Q's scales
    static constexpr int kQRows = PAIR ? NT / 2 : NT;                    // rows of Q that a CTA brings
    static constexpr int kTile = (128 + kQRows) * kMxK;
    static constexpr int kSf = 512 * (1 + kQParts);                      // scales of a K step
    static constexpr int kGroup = 4 * kSf;                               // ... of the four that a row's 16 bytes hold
    // epilogue: 32 rows x 64 outputs for each of its warps; SWAP: the tile's fp32 sums, a part from each CTA of the cluster
    static constexpr int kOut = SWAP ? 128 * NT * 4 : 4 * 4096;
    static constexpr int kFit = (int)((227 * 1024 - 4096 - kMxGroups * kGroup - kOut) / kTile);
    static constexpr int kMost = NT == 256 ? 5 : kMxMaxStages;           // (so that the accumulators share 64 columns at most)
    static constexpr int kStages = kFit < kMost ? kFit : kMost;
    static constexpr int kSfCols = 4 * (1 + kQParts);
    static constexpr int kSf0 = NT == 256 ? 512 - kStages * kSfCols : 256;   // columns of the scales, a place for every stage, ...
    static constexpr int kAcc1 = NT == 256 ? kSf0 - 256 : NT;            // ... of the second accumulator
    static constexpr int kLag = NT == 256 ? 1 : 2;                       // a tile's MMAs wait for the drain of the kLag-th before
    static constexpr size_t kSmem = (size_t)kStages * kTile + kMxGroups * kGroup + kOut + 2048;
    static_assert(kSmem >= kClusterSmem, "beside another kernel that waits in a cluster");
    static_assert(kSf0 + kStages * kSfCols <= 512 && (NT < 256 || kAcc1 >= 192), "tensor memory");
};

struct MxBars {
    uint64_t full[kMxMaxStages];        // the stage's codes
    uint64_t both[kMxMaxStages];        // pairs, in CTA 0: both CTAs have their codes and scales
    uint64_t empty[kMxMaxStages];
    uint64_t scales[kMxGroups];
    uint64_t used[kMxGroups];           // the MMAs of the group have read its scales
    uint64_t acc_full[2];
    uint64_t drained[2];                // by accumulator, so that no wait can be two phases behind
    uint64_t sums;                      // the parts of this CTA's columns have arrived from the cluster
    uint64_t retired;                   // after an expired wait: the MMAs issued before it
    uint32_t tmem_base;
    int abort;
    int cluster_gave_up;                // K range cut: a CTA of the cluster has (set by that CTA, in all of them)
};

struct MxArgs {
    const uint8_t* ps;
    const uint8_t* qs;
    int p_rows, q_rows, in;
    __nv_bfloat16* y;
    int n_out;
    int tiles, tiles_q;
    int height;                         // rows of P in a tile (SWAP: 128 or fewer)
    int stage_bytes;                    // that the loads of a stage bring
    int y_map;                          // y leaves by TMA (rows that start on 16 bytes)
    int piece_p, piece_q;               // bytes on which the scales' rows start: 16 (and no row ends in a group), 4 or 1
    int spin_limit;
    int give_up;
    int32_t* status;
};
struct MxMaps {
    CUtensorMap p, q, y;
};

// kind::mxf8f6f4, e4m3 x e4m3, ue8m0 scales, M = m, N = n; K step kk of the four that share a word of scales
__device__ __forceinline__ uint32_t mx_idesc(int m, int n, int kk) {
    return (1u << 23) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 7) << 27) | ((uint32_t)kk << 4) | ((uint32_t)kk << 29);
}
template <bool PAIR>
__device__ __forceinline__ void umma_mx(uint32_t me, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb, uint32_t accumulate) {
    if (PAIR)
        asm volatile(
            "{\n\t.reg .pred p, q;\n\t"
            "setp.ne.b32 p, %6, 0;\n\t"
            "setp.ne.b32 q, %7, 0;\n\t"
            "@q tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
            ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate), "r"(me)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p, q;\n\t"
            "setp.ne.b32 p, %6, 0;\n\t"
            "setp.ne.b32 q, %7, 0;\n\t"
            "@q tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
            ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate), "r"(me)
            : "memory");
}
// 32 x 16 bytes of shared memory -> four columns of all four 32-lane parts (of both CTAs of a pair, each from its own)
template <bool PAIR>
__device__ __forceinline__ void tmem_copy_scales(uint32_t me, uint32_t taddr, uint32_t smem) {
    const uint64_t desc = (uint64_t)((smem >> 4) & 0x3fffu) | (8ull << 16) | (8ull << 32) | (1ull << 46);     // no swizzle, 8 rows of 16 bytes together
    if (PAIR)
        asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t@q tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;\n\t}" ::"r"(taddr), "l"(desc), "r"(me) : "memory");
    else
        asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t@q tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;\n\t}" ::"r"(taddr), "l"(desc), "r"(me) : "memory");
}
__device__ __forceinline__ void st_shared(uint32_t addr, uint32_t v) { asm volatile("st.shared.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }
__device__ __forceinline__ void st_shared4(uint32_t addr, uint4 v) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, uint32_t src, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"((uint64_t)map), "r"(src), "r"(x), "r"(y) : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// The stores' source may be written again; ... and they are done.
__device__ __forceinline__ void tma_store_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void tma_store_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
// Shared memory of this CTA into that of CTA `rank` of the cluster, counted there by the barrier at this CTA's offset `bar`.
__device__ __forceinline__ void copy_to_peer(uint32_t dst, uint32_t src, uint32_t bytes, uint32_t bar, uint32_t rank) {
    asm volatile(
        "{\n\t.reg .b32 ra, rb;\n\t"
        "mapa.shared::cluster.u32 ra, %0, %4;\n\t"
        "mapa.shared::cluster.u32 rb, %3, %4;\n\t"
        "cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [ra], [%1], %2, [rb];\n\t}"
        ::"r"(dst), "r"(src), "r"(bytes), "r"(bar), "r"(rank)
        : "memory");
}
// One word of CTA `rank`'s shared memory, at this CTA's offset of it.
__device__ __forceinline__ void st_cluster_int(uint32_t addr, int v, uint32_t rank) {
    asm volatile("{\n\t.reg .b32 ra;\n\tmapa.shared::cluster.u32 ra, %0, %2;\n\tst.shared::cluster.s32 [ra], %1;\n\t}" ::"r"(addr), "r"(v), "r"(rank) : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ int ld_cluster_int(uint32_t addr, uint32_t rank) {
    int v;
    asm volatile("{\n\t.reg .b32 ra;\n\tmapa.shared::cluster.u32 ra, %1, %2;\n\tld.shared::cluster.s32 %0, [ra];\n\t}" : "=r"(v) : "r"(addr), "r"(rank) : "memory");
    return v;
}

// Scales of a row for the four K steps of a group (16 blocks), in the words that they lie in: what is loaded is not touched until
// finish_scales, a group later.  (8192 rows, 2080 -> 8192, whose rows of scales start anywhere: 140 us, byte by byte 252.)
struct RowScales {
    uint32_t w[5];
};
// ALL16: every row's groups are 16-byte pieces (the other ways beside this one cost it 5%).
template <bool ALL16>
__device__ __forceinline__ RowScales load_scales(const uint8_t* row, int group, int blocks, int piece, const uint8_t* first, const uint8_t* last) {
    RowScales s;
    const uint8_t* p = row + group * 16;
    if (ALL16 || piece == 16) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
        s.w[0] = v.x;
        s.w[1] = v.y;
        s.w[2] = v.z;
        s.w[3] = v.w;
        s.w[4] = 0;
        return s;
    }
    if (piece == 4) {                         // (whole words then, up to the end of the row)
#pragma unroll
        for (int i = 0; i < 4; ++i) s.w[i] = group * 16 + 4 * i < blocks ? __ldg(reinterpret_cast<const uint32_t*>(p) + i) : 0x7f7f7f7fu;
        s.w[4] = 0;
        return s;
    }
    const uint8_t* word = reinterpret_cast<const uint8_t*>((uintptr_t)p & ~(uintptr_t)3);
    const uint8_t* end = p + min(16, blocks - group * 16);
#pragma unroll
    for (int i = 0; i < 5; ++i, word += 4) {
        s.w[i] = 0;
        if (word >= end) continue;
        if (word >= first && word + 4 <= last) {
            s.w[i] = __ldg(reinterpret_cast<const uint32_t*>(word));
        } else {                              // the array's first or last word, not all of which is its own
            for (int j = 0; j < 4; ++j)
                if (word + j >= first && word + j < last) s.w[i] |= (uint32_t)__ldg(word + j) << (8 * j);
        }
    }
    return s;
}
// ... 1 (127) past the end of the row.
template <bool ALL16>
__device__ __forceinline__ uint4 finish_scales(const RowScales& s, const uint8_t* row, int group, int blocks, int piece) {
    if (ALL16 || piece != 1) return make_uint4(s.w[0], s.w[1], s.w[2], s.w[3]);
    const int n = blocks - group * 16, shift = (int)((uintptr_t)row & 3) * 8;
    uint32_t v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[i] = __funnelshift_r(s.w[i], s.w[i + 1], shift);
        const int keep = n - 4 * i;
        const uint32_t own = keep >= 4 ? 0xffffffffu : (keep <= 0 ? 0u : (1u << (8 * keep)) - 1u);
        v[i] = (v[i] & own) | (0x7f7f7f7fu & ~own);
    }
    return make_uint4(v[0], v[1], v[2], v[3]);
}

// Four values of an output row, whatever of them lies below n_out.
__device__ __forceinline__ void store4(__nv_bfloat16* y, size_t row, int n, int n_out, float4 v, bool whole) {
    __nv_bfloat16* at = y + row * n_out + n;
    const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
    if (whole && n + 4 <= n_out) {
        uint2 o;
        o.x = *reinterpret_cast<const uint32_t*>(&a);
        o.y = *reinterpret_cast<const uint32_t*>(&b);
        *reinterpret_cast<uint2*>(at) = o;
        return;
    }
    if (n < n_out) at[0] = a.x;
    if (n + 1 < n_out) at[1] = a.y;
    if (n + 2 < n_out) at[2] = b.x;
    if (n + 3 < n_out) at[3] = b.y;
}

template <int NT, bool SWAP, bool PAIR>
__global__ void __launch_bounds__(kMxThreads, 1)
mxfp8_mm_kernel(const MxArgs a, const int lg_splits, const __grid_constant__ MxMaps maps) {
    using P = Plan<NT, SWAP, PAIR>;
    static_assert(!PAIR || !SWAP, "pairs: tiles of many rows");
    extern __shared__ unsigned char smem_raw[];
    __shared__ MxBars bars;
    unsigned char* base = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    // 1024-byte aligned: the stages, then the epilogue's, then the scales
    const uint32_t sbase = smem_u32(base), out_base = sbase + P::kStages * P::kTile, sf_base = out_base + P::kOut;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    volatile int* abort_flag = &bars.abort;

    // Warp 9 prepares the barriers, tells the others so and goes on to the loads, of which a full ring takes microseconds to
    // issue; it needs nothing of what the others prepare.
    if (warp == 9) {
        for (int s = lane; s < P::kStages; s += 32) {
            mbar_init(smem_u32(&bars.full[s]), 1);
            mbar_init(smem_u32(&bars.both[s]), 2);
            mbar_init(smem_u32(&bars.empty[s]), 1);
        }
        if (lane < 2) {
            mbar_init(smem_u32(&bars.scales[lane]), 4);
            mbar_init(smem_u32(&bars.used[lane]), 1);
            mbar_init(smem_u32(&bars.acc_full[lane]), 1);
            mbar_init(smem_u32(&bars.drained[lane]), PAIR ? 8 : 4);
        }
        if (lane == 2) {
            mbar_init(smem_u32(&bars.sums), 1);
            mbar_init(smem_u32(&bars.retired), 1);
            bars.abort = 0;
            bars.cluster_gave_up = 0;
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 8) {
        if (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars.tmem_base)), "r"(512u) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars.tmem_base)), "r"(512u) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    __syncwarp();
    tc_fence_before();
    if (warp == 9) asm volatile("bar.arrive 2, %0;" ::"n"(kMxThreads) : "memory");
    else asm volatile("bar.sync 2, %0;" ::"n"(kMxThreads) : "memory");
    // the peers' barriers are there before anyone arrives on them
    if (PAIR || (SWAP && lg_splits > 0)) cluster_arrive();
    if (PAIR && warp != 9) cluster_wait();
    tc_fence_after();
    const uint32_t tmem = warp == 9 ? 0u : __shfl_sync(0xffffffffu, bars.tmem_base, 0);

    // a cluster a tile when the K range is cut, else every CTA (pair) takes every stride-th tile whole
    const int splits = 1 << lg_splits, rank = PAIR || (SWAP && lg_splits > 0) ? (int)cluster_ctarank() : 0;
    const int spin = SWAP && a.give_up > 1 && a.give_up - 2 != rank ? kSpin : a.spin_limit;
    const int steps = (a.in + kMxK - 1) / kMxK, lg_cluster = PAIR ? 1 : lg_splits;
    const int k0 = PAIR ? 0 : (steps * rank) >> lg_splits, k1 = PAIR ? steps : (steps * (rank + 1)) >> lg_splits;
    const int first = (int)blockIdx.x >> lg_cluster, stride = (int)gridDim.x >> lg_cluster;
    constexpr int kPRows = PAIR ? 256 : 128;                 // rows of P in a tile
    const int p_own = PAIR ? rank * 128 : 0;                 // ... of which this CTA's start here
    auto place = [&](int t, int& p0, int& q0) {              // of a tile (in P, this CTA's half)
        const int p = a.tiles_q == 1 ? t : (int)((unsigned)t / (unsigned)a.tiles_q);
        p0 = p * (SWAP ? a.height : kPRows) + p_own;
        q0 = (t - p * a.tiles_q) * NT;
    };
    // K range cut: columns of the tile that CTA r of the cluster adds (none past the last row of Q)
    const int lg_own = 31 - __clz(NT) - lg_splits;
    int p_first, q_first;
    place(first, p_first, q_first);
    auto sum_cols = [&](int r) { return max(0, min(1 << lg_own, a.q_rows - q_first - (r << lg_own))); };
    bool met = false;                                        // this warp has waited for the cluster's start
    int copied = 0;                                          // stages the loader has started

    if (warp == 9) {
        int s = 0;
        uint32_t ph = 0;
        bool ok = true;
        for (int t = first; t < a.tiles && ok; t += stride) {
            int p0, q0;
            place(t, p0, q0);
            for (int k = k0; k < k1; ++k) {
                if (!mbar_wait(smem_u32(&bars.empty[s]), ph ^ 1u, abort_flag, spin)) {
                    ok = false;
                    break;
                }
                if (lane == 0) {
                    const uint32_t st = sbase + (uint32_t)s * P::kTile, bar = smem_u32(&bars.full[s]);
                    mbar_expect_tx(bar, (uint32_t)a.stage_bytes);
                    tma_load_2d(st, &maps.p, k * kMxK, p0, bar);
                    tma_load_2d(st + 128 * kMxK, &maps.q, k * kMxK, q0 + (PAIR ? rank * P::kQRows : 0), bar);
                }
                __syncwarp();
                ++copied;
                if (++s == P::kStages) {
                    s = 0;
                    ph ^= 1u;
                }
            }
        }
        if (PAIR) cluster_wait();
    } else if (warp == 10) {
        // pairs: tells CTA 0, which issues the MMAs, what has arrived here
        int s = 0, g = 0;
        uint32_t ph = 0, g_ph = 0;
        bool ok = true;
        for (int t = PAIR ? first : a.tiles; t < a.tiles && ok; t += stride)
            for (int k = k0; k < k1; ++k) {
                if (!mbar_wait(smem_u32(&bars.full[s]), ph, abort_flag, spin) ||
                    ((k == k0 || (k & 3) == 0) && !mbar_wait(smem_u32(&bars.scales[g]), g_ph, abort_flag, spin))) {
                    ok = false;
                    break;
                }
                if (lane == 0) mbar_arrive_cta0(smem_u32(&bars.both[s]));
                __syncwarp();
                if ((k & 3) == 3 || k == k1 - 1) {
                    g_ph ^= (uint32_t)(g == kMxGroups - 1);
                    g = g == kMxGroups - 1 ? 0 : g + 1;
                }
                if (++s == P::kStages) {
                    s = 0;
                    ph ^= 1u;
                }
            }
    } else if (warp == 8 && (!PAIR || rank == 0)) {
        const uint32_t flag = smem_u32(&bars.abort);
        int s = 0, g = 0, done = 0;
        uint32_t ph = 0, g_ph = 0;
        const uint32_t me = elect_one() ? 1u : 0u;
        uint32_t ready = 0;
        for (int t = first; t < a.tiles; t += stride, ++done) {
            const int before = done - P::kLag;               // the tile whose drain makes room for this one
            if (before >= 0) mbar_wait_on(smem_u32(&bars.drained[before & 1]), (uint32_t)(before >> 1) & 1u, flag, spin);
            tc_fence_after();
            const uint32_t acc = tmem + ((done & 1) ? (uint32_t)P::kAcc1 : 0u);
            for (int k = k0; k < k1; ++k) {
                const bool last = (k & 3) == 3 || k == k1 - 1;           // of the group
                if (PAIR) {
                    mbar_wait_on(smem_u32(&bars.both[s]), ph, flag, spin, ready);
                } else {
                    mbar_wait_on(smem_u32(&bars.full[s]), ph, flag, spin, ready);
                    if (k == k0 || (k & 3) == 0) mbar_wait_on(smem_u32(&bars.scales[g]), g_ph, flag, spin);
                }
                tc_fence_after();
                // (the next stage, looked at while this one's MMAs are issued: a wait that need not be costs 80 cycles)
                const bool wrap = s + 1 == P::kStages;
                ready = mbar_peek(smem_u32(PAIR ? &bars.both[wrap ? 0 : s + 1] : &bars.full[wrap ? 0 : s + 1]), ph ^ (uint32_t)wrap);
                const uint32_t st = sbase + (uint32_t)s * P::kTile, sf = sf_base + (uint32_t)(g * P::kGroup + (k & 3) * P::kSf);
                const uint32_t sp = tmem + (uint32_t)(P::kSf0 + s * P::kSfCols), sq = sp + 4;
                tmem_copy_scales<PAIR>(me, sp, sf);
#pragma unroll
                for (int h = 0; h < P::kQParts; ++h) tmem_copy_scales<PAIR>(me, sq + 4 * h, sf + 512 * (1 + h));
#pragma unroll
                for (int kk = 0; kk < 4; ++kk)
                    umma_mx<PAIR>(me, acc, smem_desc(st) + 2 * kk, smem_desc(st + 128 * kMxK) + 2 * kk, mx_idesc(kPRows, NT, kk), sp, sq,
                                  (k > k0 || kk > 0) ? 1u : 0u);
                umma_commit_if<PAIR>(me, smem_u32(&bars.empty[s]));
                if (last) umma_commit_if<PAIR>(me, smem_u32(&bars.used[g]));
                if (k == k1 - 1) umma_commit_if<PAIR>(me, smem_u32(&bars.acc_full[done & 1]));
                __syncwarp();
                if (++s == P::kStages) {
                    s = 0;
                    ph ^= 1u;
                }
                if (last) {
                    g_ph ^= (uint32_t)(g == kMxGroups - 1);
                    g = g == kMxGroups - 1 ? 0 : g + 1;
                }
            }
        }
    } else if (warp == 8) {
    } else if (warp >= 4) {
        // Scales: a row of P and one or two of Q per thread (rows to threads so that a warp's 32 words fill 128 bytes of the
        // order above), a group of four K steps at a time, the next one on its way, a tile ahead into L2
        const int sf_row = (lane >> 3) * 32 + (warp & 3) * 8 + (lane & 7), blocks = a.in / 32, g0 = k0 >> 2, groups = ((k1 - 1) >> 2) - g0 + 1;
        const uint32_t at = sf_base + (uint32_t)((sf_row & 31) * 16 + (sf_row >> 5) * 4);
        const uint8_t* row[1 + P::kQParts];
        auto rows_of = [&](int t) {
            int p0, q0;
            place(t, p0, q0);
            row[0] = p0 + sf_row < a.p_rows ? a.ps + (size_t)(p0 + sf_row) * blocks : nullptr;
#pragma unroll
            for (int h = 0; h < P::kQParts; ++h) {
                const int r = h * 128 + sf_row;
                row[1 + h] = r < NT && q0 + r < a.q_rows ? a.qs + (size_t)(q0 + r) * blocks : nullptr;
            }
        };
        auto bring = [&](auto all16) {
            constexpr bool ALL16 = decltype(all16)::value;
            const uint8_t *p_end = a.ps + (size_t)a.p_rows * blocks, *q_end = a.qs + (size_t)a.q_rows * blocks;
            RowScales next[1 + P::kQParts];
            auto fetch = [&](int i) {
#pragma unroll
                for (int j = 0; j < 1 + P::kQParts; ++j)
                    if (row[j] != nullptr) next[j] = load_scales<ALL16>(row[j], g0 + i, blocks, j == 0 ? a.piece_p : a.piece_q, j == 0 ? a.ps : a.qs, j == 0 ? p_end : q_end);
            };
            auto prefetch = [&](int from) {
                for (int b = from; b < min(k1 * 4, blocks); b += 32)
#pragma unroll
                    for (int j = 0; j < 1 + P::kQParts; ++j)
                        if (row[j] != nullptr) asm volatile("prefetch.global.L2 [%0];" ::"l"(row[j] + b));
            };
            uint4 v[1 + P::kQParts];
            rows_of(first);
            fetch(0);
            prefetch(g0 * 16 + 32);
            int g = 0;
            uint32_t g_ph = 0;
            bool ok = true;
            for (int t = first; t < a.tiles && ok; t += stride) {
                for (int i = 0; i < groups; ++i) {
#pragma unroll
                    for (int j = 0; j < 1 + P::kQParts; ++j)
                        v[j] = row[j] != nullptr ? finish_scales<ALL16>(next[j], row[j], g0 + i, blocks, j == 0 ? a.piece_p : a.piece_q) : make_uint4(0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu, 0x7f7f7f7fu);
                    if (i + 1 < groups) {
                        fetch(i + 1);
                    } else if (t + stride < a.tiles) {
                        rows_of(t + stride);
                        fetch(0);
                        prefetch(g0 * 16 + 32);
                    }
                    if (!mbar_wait(smem_u32(&bars.used[g]), g_ph ^ 1u, abort_flag, spin)) {
                        ok = false;
                        break;
                    }
#pragma unroll
                    for (int j = 0; j < 1 + P::kQParts; ++j) {
                        const uint32_t to = at + (uint32_t)(g * P::kGroup + j * 512);
                        st_shared(to, v[j].x);
                        st_shared(to + P::kSf, v[j].y);
                        st_shared(to + 2 * P::kSf, v[j].z);
                        st_shared(to + 3 * P::kSf, v[j].w);
                    }
                    fence_async_proxy();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&bars.scales[g]));
                    if (++g == kMxGroups) {
                        g = 0;
                        g_ph ^= 1u;
                    }
                }
            }
        };
        if (a.piece_p == 16 && a.piece_q == 16) bring(std::true_type{});
        else bring(std::false_type{});
    } else {
        const int l = warp * 32 + lane;                      // lane of the accumulator
        const uint32_t quarter = (uint32_t)(warp * 32) << 16;
        constexpr int kChunks = NT >= 32 ? NT / 32 : 1;
        constexpr int kPairs = (kChunks + 1) / 2;
        const uint32_t out_own = out_base + (uint32_t)(warp * 4096), out_row = out_own + (uint32_t)(lane * 128);
        int done = 0;
        for (int t = first; t < a.tiles; t += stride, ++done) {
            int p0, q0;
            place(t, p0, q0);
            const int buf = done & 1;
            if (!mbar_wait(smem_u32(&bars.acc_full[buf]), (uint32_t)(done >> 1) & 1u, abort_flag, spin)) break;
            tc_fence_after();
            const uint32_t acc = tmem + quarter + (buf ? (uint32_t)P::kAcc1 : 0u);
            for (int pr = 0; pr < kPairs; ++pr) {
                // the columns that the two accumulators share come first
                const int c0 = NT == 256 && buf == 0 ? (2 * pr + 6) & 7 : 2 * pr;
                uint32_t v[2][32];
                tmem_ld32(acc + (uint32_t)(c0 * 32), v[0]);
                if (kChunks > 1) tmem_ld32(acc + (uint32_t)(c0 * 32 + 32), v[1]);
                if (pr == (NT == 256 ? 0 : kPairs - 1)) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        if (PAIR) mbar_arrive_cta0(smem_u32(&bars.drained[buf]));
                        else mbar_arrive(smem_u32(&bars.drained[buf]));
                    }
                }
#pragma unroll
                for (int h = 0; h < (kChunks > 1 ? 2 : 1); ++h) {
                    const int c = (c0 + h) * 32;
                    if (SWAP && lg_splits > 0) {
                        // into the stages' place, [column][lane]
                        float* part = reinterpret_cast<float*>(base) + c * 128 + l;
#pragma unroll
                        for (int i = 0; i < (NT < 32 ? NT : 32); ++i)
                            if (q0 + c + i < a.q_rows) part[i * 128] = __uint_as_float(v[h][i]);
                    } else if (SWAP) {
                        if (p0 + l < a.n_out && l < a.height) {
                            __nv_bfloat16* at = a.y + (size_t)(q0 + c) * a.n_out + p0 + l;
#pragma unroll
                            for (int i = 0; i < (NT < 32 ? NT : 32); ++i)
                                if (q0 + c + i < a.q_rows) at[(size_t)i * a.n_out] = __float2bfloat16_rn(__uint_as_float(v[h][i]));
                        }
                    } else if (a.y_map) {
                        // 32 rows x 64 columns a warp, 128-byte swizzle
                        if (h == 0) {
                            if (lane == 0) tma_store_read();
                            __syncwarp();
                        }
#pragma unroll
                        for (int i = 0; i < 32; i += 8) {
                            uint32_t o[4];
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const __nv_bfloat162 b = __floats2bfloat162_rn(__uint_as_float(v[h][i + 2 * j]), __uint_as_float(v[h][i + 2 * j + 1]));
                                o[j] = *reinterpret_cast<const uint32_t*>(&b);
                            }
                            st_shared4(out_row + (uint32_t)((((h * 4 + i / 8) ^ lane) & 7) * 16), make_uint4(o[0], o[1], o[2], o[3]));
                        }
                        if (h == 1) {
                            fence_async_proxy();
                            __syncwarp();
                            if (lane == 0 && p0 + warp * 32 < a.p_rows && q0 + c0 * 32 < a.n_out) tma_store_2d(&maps.y, out_own, q0 + c0 * 32, p0 + warp * 32);
                        }
                    } else if (p0 + l < a.p_rows) {
                        __nv_bfloat16* at = a.y + (size_t)(p0 + l) * a.n_out;
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (q0 + c + i < a.n_out) at[q0 + c + i] = __float2bfloat16_rn(__uint_as_float(v[h][i]));
                    }
                }
            }
        }
        if (!SWAP && lane == 0) tma_store_done();
        if (SWAP && lg_splits > 0) {
            // each CTA's columns to it, [sender][column][lane]; it adds them.  (All of them send, also a CTA that has given up, so
            // that what a CTA waits for comes.)
            fence_async_proxy();
            asm volatile("bar.sync 1, 128;" ::: "memory");
            cluster_wait();
            met = true;
            if (warp == 0 && elect_one()) {
                mbar_expect_tx(smem_u32(&bars.sums), (uint32_t)((sum_cols(rank) * 512) << lg_splits));
                for (int r = 0; r < splits; ++r)
                    if (sum_cols(r) > 0)
                        copy_to_peer(out_base + (uint32_t)(rank << lg_own) * 512u, sbase + (uint32_t)(r << lg_own) * 512u, (uint32_t)sum_cols(r) * 512u,
                                     smem_u32(&bars.sums), (uint32_t)r);
            }
            __syncwarp();
        }
        if (SWAP && lg_splits > 0 && mbar_wait(smem_u32(&bars.sums), 0u, abort_flag, spin)) {
            const int p0 = p_first, q0 = q_first + (rank << lg_own), cols = sum_cols(rank);
            const float4* parts = reinterpret_cast<const float4*>(base + P::kStages * P::kTile);
            const bool whole = ((uintptr_t)a.y % 8) == 0 && a.n_out % 4 == 0;
            for (int i = tid; i < cols * 32; i += 128) {
                const int col = i >> 5, n = (i & 31) * 4;
                if (p0 + n >= a.n_out) continue;
                float4 sum = parts[col * 32 + (i & 31)];
                for (int c = 1; c < splits; ++c) {
                    const float4 v = parts[((c << lg_own) + col) * 32 + (i & 31)];
                    sum = make_float4(sum.x + v.x, sum.y + v.y, sum.z + v.z, sum.w + v.w);
                }
                store4(a.y, (size_t)(q0 + col), p0 + n, a.n_out, sum, whole);
            }
        }
    }
    __syncthreads();
    const bool gave_up = bars.abort != 0;
    if (gave_up) {
        if (warp == 8 && (!PAIR || rank == 0)) {
            if (elect_one()) {
                if (PAIR) umma_commit_own_pair(smem_u32(&bars.retired));
                else umma_commit(smem_u32(&bars.retired));
            }
            __syncwarp();
            mbar_drain(smem_u32(&bars.retired), 0u);
        } else if (warp == 9) {
            for (int k = max(0, copied - P::kStages); k < copied; ++k)
                mbar_drain(smem_u32(&bars.full[k % P::kStages]), (uint32_t)(k / P::kStages) & 1u);
        }
        __syncthreads();
    }
    if (PAIR) cluster_sync();                                // neither CTA's arrivals and MMAs outlive the other
    if (warp == 8) {
        if (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
    bool bad = gave_up;
    if (PAIR) {
        bad = bad || ld_cluster_int(smem_u32(&bars.abort), (uint32_t)(rank ^ 1)) != 0;
        cluster_sync();
    }
    if (SWAP && lg_splits > 0) {
        if (!met) cluster_wait();
        if (gave_up && tid < splits) st_cluster_int(smem_u32(&bars.cluster_gave_up), 1, (uint32_t)tid);
        // nobody leaves while another CTA may copy into its shared memory or out of it: all copies have been issued here, and a
        // CTA that has waited for its sums has all that come to it
        cluster_arrive();
        cluster_wait();
        if (bars.cluster_gave_up != 0) {                     // (then some may not have waited; the same in all CTAs)
            if (warp == 0) mbar_drain(smem_u32(&bars.sums), 0u);
            cluster_arrive();
            cluster_wait();
            bad = true;
        }
    }
    if (bad) {
        if (tid == 0) atomicExch(a.status, 4);
        for (int t = first; t < a.tiles; t += stride) {
            int p0, q0;
            place(t, p0, q0);
            for (int i = tid; i < 128 * NT; i += kMxThreads) {
                const int p = p0 + i / NT, q = q0 + i % NT;
                if (p < a.p_rows && q < a.q_rows && (!SWAP || i / NT < a.height)) a.y[SWAP ? (size_t)q * a.n_out + p : (size_t)p * a.n_out + q] = __float2bfloat16_rn(__uint_as_float(0x7fc00000u));
            }
        }
    }
}

template <int NT, bool SWAP, bool PAIR = false>
int set_up() {
    IMX_CHECK_CUDA(cudaFuncSetAttribute(mxfp8_mm_kernel<NT, SWAP, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Plan<NT, SWAP, PAIR>::kSmem));
    return IMX_OK;
}

struct Call {
    const uint8_t *x, *xs, *w, *ws;
    int m, n_out, in;
    __nv_bfloat16* y;
    int32_t* status;
    int sms;
    cudaStream_t stream;
};

template <int NT, bool SWAP, bool PAIR = false>
int launch(const Call& c, int lg_splits, int height = PAIR ? 256 : 128) {
    const int splits = 1 << lg_splits;
    MxArgs a = {};
    a.ps = SWAP ? c.ws : c.xs;
    a.qs = SWAP ? c.xs : c.ws;
    a.p_rows = SWAP ? c.n_out : c.m;
    a.q_rows = SWAP ? c.m : c.n_out;
    a.in = c.in;
    a.y = c.y;
    a.n_out = c.n_out;
    a.tiles_q = ceil_div(a.q_rows, NT);
    a.height = height;
    const long tiles = (long)ceil_div(a.p_rows, height) * a.tiles_q;
    IMX_REQUIRE(tiles <= 0x7fffffffL / kMxMaxSplits, "mxfp8_matmul: too many outputs");
    a.tiles = (int)tiles;
    auto piece = [&](const uint8_t* s) { return (uintptr_t)s % 16 == 0 && c.in % 512 == 0 ? 16 : ((uintptr_t)s % 4 == 0 && c.in % 128 == 0 ? 4 : 1); };
    a.piece_p = piece(a.ps);
    a.piece_q = piece(a.qs);
    a.give_up = g_mx_give_up.load();
    a.spin_limit = a.give_up == 0 ? kSpin : 0;
    a.status = c.status;
    // rows of x that do not exist are not brought: what the lanes hold in their place reaches no output
    const int p_box = SWAP ? height : (c.m < 128 ? (c.m + 7) & ~7 : 128);
    a.stage_bytes = (p_box + Plan<NT, SWAP, PAIR>::kQRows) * kMxK;
    MxMaps maps;
    IMX_TRY(encode_tensor_map_2d(SWAP ? c.w : c.x, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, (size_t)a.p_rows, (size_t)c.in, (size_t)c.in, kMxK, p_box, 128, true, &maps.p));
    IMX_TRY(encode_tensor_map_2d(SWAP ? c.x : c.w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, (size_t)a.q_rows, (size_t)c.in, (size_t)c.in, kMxK, Plan<NT, SWAP, PAIR>::kQRows, 128,
                                 true, &maps.q));
    a.y_map = !SWAP && (uintptr_t)c.y % 16 == 0 && c.n_out % 8 == 0;
    if (a.y_map)
        IMX_TRY(encode_tensor_map_2d(c.y, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, (size_t)c.m, (size_t)c.n_out, (size_t)c.n_out * 2, 64, 32, 128, true, &maps.y));
    cudaLaunchConfig_t cfg = {};
    const int cluster = PAIR ? 2 : splits, most = c.sms / 2 * (PAIR ? 1 : 2);
    cfg.gridDim = dim3((unsigned)(lg_splits > 0 ? a.tiles * splits : (a.tiles < most ? a.tiles : most) * cluster));
    cfg.blockDim = dim3(kMxThreads);
    cfg.dynamicSmemBytes = Plan<NT, SWAP, PAIR>::kSmem;
    cfg.stream = c.stream;
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)cluster;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    IMX_CHECK_CUDA(cudaLaunchKernelEx(&cfg, mxfp8_mm_kernel<NT, SWAP, PAIR>, a, lg_splits, maps)); IMX_LAUNCHED();
    return IMX_OK;
}

// Which kernel: the least of a model of their times in us, a part that does not shrink and a time for each K step of each wave
// of tiles, fitted to the kernels alone on a B200 (2048 -> 8192 unless said; measured, in brackets the model):
//   1 row     S16 6.9 (7.0), S16 cut in 2 7.1 (7.5);   2048 -> 512  S16 cut in 1, 2, 4, 8  6.1, 5.6, 5.0, 5.1
//   64 rows   S64 9.5 (9.4), S64 cut in 2 10.2 (9.8), N64 7.7 (7.7);   4096 -> 2048  S64 cut in 4 8.5 (8.8), N64 9.6 (10.6)
//   256 rows  N64 11.1 (10.6), N128 9.1 (9.0), P128 9.7 (9.5), P256 11.9 (12.1)
//   777 rows 4096 -> 2048  N64 16.7 (16.5), N128 12.6 (12.6), P128 12.8 (12.8), P256 17.4 (17.8)
//   1024 rows N128 20.8 (19.8), P128 19.4 (19.5), P256 17.4 (17.8);   8192 rows  N128 130, P128 115, P256 99
//   64 rows 2048 -> 152064  S64 55, N64 63, N128 58, P128 70, P256 68 (memory: 52)
// Clusters of eight that fill the GPU find no place together: 4096 -> 2048, 1 row, cut in 8 (128 CTAs) 11.3, in 4 6.7.
int run(const Call& c) {
    const int steps = ceil_div(c.in, kMxK);
    enum { S16, S32, S64, N64, N128, P128, P256 } best = P256;
    int best_lg = 0;
    float least = 1e30f;
    auto offer = [&](decltype(best) kernel, int lg, float fixed, long tiles, int at_once, float step) {
        const long waves = (tiles + at_once - 1) / at_once;
        const float us = fixed + (float)waves * (float)ceil_div(steps, 1 << lg) * step;
        if (us < least) {
            least = us;
            best = kernel;
            best_lg = lg;
        }
    };
    const int nt = c.m <= 16 ? 16 : (c.m <= 32 ? 32 : 64);
    const long tiles = (long)ceil_div(c.n_out, 128) * ceil_div(c.m, nt);
    for (int lg = 0; lg < 4 && (lg == 0 || (tiles << lg <= (lg == 3 ? 64 : c.sms) && steps >= 2 << lg)); ++lg)
        offer(nt == 16 ? S16 : (nt == 32 ? S32 : S64), lg, 3.4f + 0.044f * nt + (lg > 0 ? 1.f : 0.f) + (lg > 0 && tiles << lg > c.sms / 2 ? 1.f : 0.f), tiles,
              lg > 0 ? (int)tiles : c.sms, nt == 64 ? 0.2f : 0.18f);
    const long rows128 = ceil_div(c.m, 128);
    offer(N64, 0, 4.7f, rows128 * ceil_div(c.n_out, 64), c.sms, 0.185f);
    offer(N128, 0, 5.4f, rows128 * ceil_div(c.n_out, 128), c.sms, 0.225f);
    offer(P128, 0, 6.1f, (long)ceil_div(c.m, 256) * ceil_div(c.n_out, 128), c.sms / 2, 0.21f);
    offer(P256, 0, 6.3f, (long)ceil_div(c.m, 256) * ceil_div(c.n_out, 256), c.sms / 2, 0.36f);
    // More than one wave of weight tiles: all of them as low as the number of waves allows, so that the last is full too.  64
    // rows, 2048 -> 152064 (9 waves for 8.03 of 128 outputs) 55.3 us, with 128 56.7; 8 rows, 2048 -> 40000, 17.8 and 19.9.
    int height = 128;
    if (best <= S64 && best_lg == 0 && tiles > c.sms) {
        const long per_q = (tiles + c.sms - 1) / c.sms * c.sms / ceil_div(c.m, nt);
        height = (int)((c.n_out + per_q - 1) / per_q + 3) & ~3;
    }
    switch (best) {
        case S16: return launch<16, true>(c, best_lg, height);
        case S32: return launch<32, true>(c, best_lg, height);
        case S64: return launch<64, true>(c, best_lg, height);
        case N64: return launch<64, false>(c, 0);
        case N128: return launch<128, false>(c, 0);
        case P128: return launch<128, false, true>(c, 0);
        default: return launch<256, false, true>(c, 0);
    }
}

}  // namespace

// Test hook (include/ironmlx_b200_testing.h).
void testing_mxfp8_give_up(int on) { g_mx_give_up.store(on); }

}  // namespace imx

using namespace imx;

extern "C" {

void imx_testing_mxfp8_give_up(int on) { testing_mxfp8_give_up(on); }

int imx_mxfp8_matmul_scratch_bytes(int m, int n_out, int in, size_t* bytes) {
    IMX_REQUIRE(bytes != nullptr && m >= 0 && n_out > 0 && in > 0 && in % 32 == 0, "mxfp8_matmul_scratch_bytes: bad arguments");
    *bytes = kStatusBytes;
    return IMX_OK;
}

int imx_mxfp8_matmul(const void* x_q, const void* x_scales, int m, const imx_qtensor* w, int n_out, int in, void* y,
                     void* scratch, size_t scratch_bytes, void* stream) {
    IMX_REQUIRE(m >= 0 && n_out > 0 && in > 0 && in % 32 == 0,
                "mxfp8_matmul: sizes (%d rows, %d -> %d) must be positive, the input dimension a multiple of 32", m, in, n_out);
    IMX_REQUIRE(m <= kMxMost && n_out <= kMxMost && in <= kMxMost, "mxfp8_matmul: rows, outputs and inputs of at most %d", kMxMost);
    if (m == 0) return IMX_OK;
    IMX_REQUIRE(x_q && x_scales && w && w->w && w->scales && y, "mxfp8_matmul: rows, weight and their scales, and y are required");
    IMX_REQUIRE(w->biases == nullptr, "mxfp8_matmul: an mxfp8 weight has no biases");
    IMX_REQUIRE((uintptr_t)x_q % 16 == 0 && (uintptr_t)w->w % 16 == 0, "mxfp8_matmul: rows and weight must be 16-byte aligned");
    IMX_REQUIRE((uintptr_t)y % 2 == 0, "mxfp8_matmul: y must be aligned to its bf16 values");
    if (scratch == nullptr || (uintptr_t)scratch % 256 != 0 || scratch_bytes < kStatusBytes) {
        set_error("mxfp8_matmul: 256-byte aligned scratch of %zu bytes needed, %zu given", kStatusBytes, scratch_bytes);
        return IMX_ERR_WORKSPACE;
    }
    const size_t yb = (size_t)m * n_out * 2, xb = (size_t)m * in, wb = (size_t)n_out * in;
    IMX_REQUIRE(!overlap(y, yb, x_q, xb) && !overlap(y, yb, x_scales, xb / 32) && !overlap(y, yb, w->w, wb) &&
                !overlap(y, yb, w->scales, wb / 32) && !overlap(y, yb, scratch, kStatusBytes), "mxfp8_matmul: y overlaps another array");
    DeviceInfo di;
    IMX_TRY(current_device(&di));
    if (device_needs_setup(di.ordinal, kSetupMxfp8)) {       // once per device
        IMX_TRY((set_up<16, true>()));
        IMX_TRY((set_up<32, true>()));
        IMX_TRY((set_up<64, true>()));
        IMX_TRY((set_up<64, false>()));
        IMX_TRY((set_up<128, false>()));
        IMX_TRY((set_up<128, false, true>()));
        IMX_TRY((set_up<256, false, true>()));
        device_mark_setup(di.ordinal, kSetupMxfp8);
    }
    return run(Call{(const uint8_t*)x_q, (const uint8_t*)x_scales, (const uint8_t*)w->w, (const uint8_t*)w->scales, m, n_out, in,
                    (__nv_bfloat16*)y, (int32_t*)scratch, di.sms, (cudaStream_t)stream});
}

}  // extern "C"
