// Low-rank adapters of many requests beside a shared projection: row t with the adapter j = ids[t] gets
//   out[t] = bf16( y[t] + scale[j] * (x[t] . a[j]^T) . b[j]^T ),   a[j]: [rank, in], b[j]: [n_out, rank]
// and a row whose id is outside [0, count) gets out[t] = y[t].
//
// One launch does both products.  A cluster of CTAs takes a unit, up to 16 (64) rows of one adapter: each CTA multiplies its
// part of the input dimension, the cluster adds the parts through its shared memories, in one order, and each CTA multiplies
// its part of the output columns.  Sums are in fp32; for the second product the scaled low-rank row becomes three bf16 numbers
// that add up to it exactly (8 bits each of its 24), three MMAs for one.
// Which rows make up a unit every CTA finds out by itself from the ids: the units of an adapter are its rows in batch order,
// so that the result does not depend on who runs when.  Rows without an adapter are units of their own that are copied.
//
// Two kernels (times on a B200, of the kernels alone):
//   few rows (at most 128): a and b are read once and go straight into the fragments of mma.sync, whose k order is permuted so
//     that a lane's 16 bytes are four k pairs.  Bound by latency, of memory (each lane brings what it alone reads, through a
//     ring of cp.async) and of the cluster's two meetings: one row of rank 16, 2048 -> 8192, takes 5.0 us; 48 rows of 40
//     adapters of rank 32, 4096 -> 2048 (16 MB: 2.5 us at the copy bandwidth), 11.6 us.
//   many rows: tiles of 64 rows by tcgen05.mma, x and y gathered by cp.async, a and b brought by TMA.  8192 rows of rank 64,
//     2048 -> 8192, take 69 us, 318 MB at 4.6 TB/s: y comes and leaves in 37 us (268 MB; a third of the writes is left in L2),
//     but the ids (4.6 us), x . a^T (6.1 us), the cluster's exchange and the low-rank rows' way into tensor memory (5.4 us) come
//     before it, for all CTAs at the same time.  With mma.sync by the warps that copy it was 113 us; rank 128, one CTA an SM,
//     takes 108 us (229).  777 rows of rank 16 take 16 us, each phase a latency or two.
#include <atomic>

#include "tcgen05.cuh"
#include "../../include/ironmlx_b200_testing.h"

namespace imx {

namespace {

constexpr int kMaxRank = 256;
constexpr int kThreads = 256;
constexpr size_t kStatusBytes = 256;
constexpr int kMostColumns = 1 << 30;         // of x and y: columns past the end of a row are counted in 31 bits
std::atomic<int> g_low_rank_give_up{0};       // see imx_testing_low_rank_give_up

struct LowRankArgs {
    const __nv_bfloat16* y;
    const __nv_bfloat16* x;
    const __nv_bfloat16* a;
    const __nv_bfloat16* b;
    const float* scale;
    const int32_t* ids;
    __nv_bfloat16* out;
    int n, in, n_out, count, rank;
    int wide;                 // y and out: rows of whole 16-byte pieces
    int spin_limit, give_up;
    int32_t* status;
};

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ uint32_t peer_addr(uint32_t addr, int rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ float ld_peer(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float4 ld_peer4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void st_peer4(uint32_t addr, uint4 v) {
    asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// v = hi + mid + lo, each the next 8 of its 24 bits: bf16 numbers in the upper halves of 32 bits.  (Cut off, not rounded: hi is
// finite where v is; what is not finite stays in hi.)
__device__ __forceinline__ float upper(float v) { return __uint_as_float(__float_as_uint(v) & 0xffff0000u); }
__device__ __forceinline__ float after_upper(float v) {
    const float left = v - upper(v);
    return left == left ? left : 0.f;
}
__device__ __forceinline__ uint32_t pack2(float a, float b) { return __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632); }       // two upper halves

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {
    const int n = there ? 16 : 0;             // the rest is filled with zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void copy4(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ uint4 ld_shared16(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}

// Four 8 x 8 matrices of 16-bit values; lane l gives the address of row l % 8 of matrix l / 8.
__device__ __forceinline__ void ld_matrices(uint32_t addr, uint32_t (&v)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void st_matrices(uint32_t addr, const uint32_t (&v)[4]) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
}

// ── few rows ────────────────────────────────────────────────────────────────
constexpr int kFewRows = 128;                 // rows of a launch
constexpr int kFewUnit = 16;
// Each lane has a ring of 16-byte pieces in shared memory for what it alone will read, filled by cp.async: in registers there
// is room for two or three pieces on their way (2.6 TB/s).  RB: blocks of 32 values of the rank, 1, 2, 4 or 8.
__host__ __device__ constexpr int ring_pieces(int rb) { return rb == 8 ? 18 : (rb == 4 ? 15 : 12); }
// Dynamic shared memory: the rings, this CTA's sums [row][rank], and in one place the warps' parts of them, [k part][row][rank]
// (8 parts of ranks up to 32, 4 up to 64, 2 up to 128), and afterwards the low-rank rows as hi, mid and lo: [part][row][rb * 32],
// in odd rows the pieces of 64 bytes that make up 128 the other way round, so that lanes that read together are in different
// banks (a padded row would leave no room for two CTAs of a rank of 256).
struct FewPlan {
    int sums_at, part_at, bytes;
    __host__ __device__ FewPlan(int rank, int rb) {
        sums_at = kThreads * ring_pieces(rb) * 16;
        part_at = sums_at + kFewUnit * rank * 4;
        const int parts = 8 / rb, a = parts > 1 ? parts * kFewUnit * rank * 4 : 0, b = 3 * kFewUnit * rb * 32 * 2;
        bytes = part_at + (a > b ? a : b);
    }
};

struct FewShared {
    int32_t ids[kFewRows];
    uint8_t same[kFewRows];                   // rows before with the same id
    uint32_t leads[kFewRows / 32];            // rows that lead a unit, a bit each
    int32_t rows[kFewUnit];
};

// The rows (in s.rows) and the adapter of a unit; returns how many, 0 where there is no such unit.  Row i leads a unit if a
// multiple of 16 rows before it have its id; units are numbered in the order of their leaders.
__device__ __forceinline__ int find_unit(const LowRankArgs& p, FewShared& s, int unit, int& id) {
    const int i = threadIdx.x, lane = i & 31;
    int own = -1;
    if (i < kFewRows) {
        own = i < p.n ? p.ids[i] : -1;
        own = own >= 0 && own < p.count ? own : -1;
        s.ids[i] = own;
    }
    __syncthreads();
    int same = 0;
    if (i < kFewRows) {
        for (int j = 0; j < (i & ~31) && i < p.n; j += 4) {
            const int4 v = *reinterpret_cast<const int4*>(&s.ids[j]);
            same += (v.x == own) + (v.y == own) + (v.z == own) + (v.w == own);
        }
        const unsigned alike = __match_any_sync(0xffffffffu, i < p.n ? own : -2 - lane);
        same += __popc(alike & ((1u << lane) - 1u));
        const unsigned leads = __ballot_sync(0xffffffffu, i < p.n && same % kFewUnit == 0);
        if (lane == 0) s.leads[i >> 5] = leads;
        s.same[i] = (uint8_t)same;
    }
    __syncthreads();
    int leader = -1, here = unit;
#pragma unroll
    for (int b = 0; b < kFewRows / 32; ++b) {
        unsigned m = s.leads[b];
        if (leader < 0 && here < __popc(m)) {
            for (; here > 0; --here) m &= m - 1;
            leader = b * 32 + __ffs(m) - 1;
        }
        here -= __popc(m);
    }
    if (leader < 0) return 0;
    id = s.ids[leader];
    const int at = same - s.same[leader];
    const bool mine = i < p.n && own == id && at >= 0 && at < kFewUnit;
    if (mine) s.rows[at] = i;
    return __syncthreads_count(mine);
}

// `clusters` clusters of `ctas` CTAs a unit: each cluster multiplies x . a^T for itself and takes a part of the columns.
// TP: tiles of eight values of the rank that a warp multiplies (1, 2 or 4; RB > 1: 4).
// Two CTAs an SM above a rank of 32: three would leave 80 registers (rank 64, 128 rows of 16 and 120 adapters 15.4 and 32.9 us,
// with two 13.7 and 27.7; 48 rows of 40 adapters, which fill three, 16.4 and 17.3).
constexpr int few_ctas(int rb) { return rb <= 1 ? 3 : 2; }
template <int RB, int TP>
__global__ void __launch_bounds__(kThreads, few_ctas(RB))
low_rank_few_kernel(const LowRankArgs p, const int ctas, const int clusters) {
    __shared__ __align__(16) FewShared s;
    extern __shared__ __align__(16) unsigned char dyn[];
    constexpr int kPiece = kThreads * 16;     // bytes between a lane's pieces
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
    const int c = (int)blockIdx.x & (ctas - 1);
    int id = -1;
    const int shift = 31 - __clz(ctas), cut = shift + 31 - __clz(clusters);       // (both are powers of two)
    const int m = find_unit(p, s, (int)blockIdx.x >> cut, id);
    if (m == 0) return;                       // fewer units than clusters: the whole cluster leaves
    // output columns of this CTA, in tiles of eight
    const int tiles = (p.n_out + 7) / 8, part_of = (int)blockIdx.x & ((1 << cut) - 1);
    const int t0 = (int)((long)tiles * part_of >> cut), t1 = (int)((long)tiles * (part_of + 1) >> cut);
    if (id < 0) {
        if (p.out != p.y)
            for (int r = 0; r < m; ++r) {
                const size_t at = (size_t)s.rows[r] * p.n_out;
                for (int n = t0 * 8 + tid; n < min(t1 * 8, p.n_out); n += kThreads) p.out[at + n] = p.y[at + n];
            }
        return;
    }
    const float sc = p.scale != nullptr ? p.scale[id] : 1.f;
    // a lane multiplies the rows g and g + 8 of the unit
    const int row0 = s.rows[min(g, m - 1)], row1 = s.rows[min(g + 8, m - 1)];
    const bool has0 = g < m, has1 = g + 8 < m, more = m > 8;
    const int rank = p.rank;
    const FewPlan pl(rank, RB);
    float* sums = reinterpret_cast<float*>(dyn + pl.sums_at);
    float* parts = reinterpret_cast<float*>(dyn + pl.part_at);
    __nv_bfloat16* low_rows = reinterpret_cast<__nv_bfloat16*>(dyn + pl.part_at);
    const uint32_t own = smem_addr(dyn) + (uint32_t)tid * 16u;
    const __nv_bfloat16* a = p.a + (size_t)id * rank * p.in;
    const __nv_bfloat16* b = p.b + (size_t)id * p.n_out * rank;

    // x . a^T: a warp takes TP tiles of the rank, every RB-th, and one of 8 / RB parts of the k blocks of 32
    constexpr int kWk = 8 / RB;
    const int wr = warp & (RB - 1), wk = warp / RB, rt = rank / 8;
    float acc[TP][4] = {};
    {
        constexpr int kPieces = TP + 2, kDepth = ring_pieces(RB) / kPieces;
        const int blocks = (p.in + 31) / 32, b0 = (int)((long)blocks * c >> shift), b1 = (int)((long)blocks * (c + 1) >> shift);
        const int n = (b1 - b0 - wk + kWk - 1) / kWk;                     // blocks of this warp
        int k = (b0 + wk) * 32 + q * 8;                                   // of the next load
        const __nv_bfloat16* x0 = p.x + (size_t)row0 * p.in + k;
        const __nv_bfloat16* x1 = p.x + (size_t)row1 * p.in + k;
        const __nv_bfloat16* aw = a + (size_t)(wr * 8 + g) * p.in + k;
        const size_t tile = (size_t)(8 * RB) * p.in;
        int left = n;
        uint32_t to = own;
        auto load = [&]() {
            if (left > 0) {
                const bool in = k < p.in;
                copy16(to, in && has0 ? x0 : p.x, in && has0);
                if (more) copy16(to + kPiece, in && has1 ? x1 : p.x, in && has1);
#pragma unroll
                for (int i = 0; i < TP; ++i)
                    if (wr + i * RB < rt) copy16(to + (2 + i) * kPiece, in ? aw + i * tile : a, in);
            }
            copies_commit();
            --left;
            k += kWk * 32;
            x0 += kWk * 32;
            x1 += kWk * 32;
            aw += kWk * 32;
            to += kPieces * kPiece;
            if (to == own + kDepth * kPieces * kPiece) to = own;
        };
#pragma unroll
        for (int i = 0; i < kDepth; ++i) load();
        uint32_t from = own;
        for (int i = 0; i < n; ++i) {
            copies_wait<kDepth - 1>();
            const uint4 v0 = ld_shared16(from), v1 = more ? ld_shared16(from + kPiece) : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int t = 0; t < TP; ++t) {
                if (wr + t * RB >= rt) break;
                const uint4 w = ld_shared16(from + (2 + t) * kPiece);
                mma(acc[t], v0.x, v1.x, v0.y, v1.y, w.x, w.y);
                mma(acc[t], v0.z, v1.z, v0.w, v1.w, w.z, w.w);
            }
            load();
            from += kPieces * kPiece;
            if (from == own + kDepth * kPieces * kPiece) from = own;
        }
        copies_wait<0>();
    }
    // The second product's pieces, b and y of a tile of output columns each: the first are on their way while the cluster meets.
    constexpr int kPieces = RB + 1, kDepth = ring_pieces(RB) / kPieces;
    const bool pairs = p.n_out % 2 == 0 && (((uintptr_t)p.y | (uintptr_t)p.out) % 4) == 0;
    const int n = (t1 - t0 - warp + 7) >> 3;                              // tiles of this warp, every eighth
    int left = n, row = (t0 + warp) * 8 + g, col = (t0 + warp) * 8 + 2 * q;    // of the next load: row of b, column of y
    const __nv_bfloat16* bw = b + (size_t)row * rank + q * 8;
    const __nv_bfloat16* y0 = p.y + (size_t)row0 * p.n_out + col;
    const __nv_bfloat16* y1 = p.y + (size_t)row1 * p.n_out + col;
    uint32_t to = own;
    auto load = [&]() {
        if (left > 0) {
#pragma unroll
            for (int kb = 0; kb < RB; ++kb) {
                const bool there = row < p.n_out && kb * 32 + q * 8 < rank;
                copy16(to + (1 + kb) * kPiece, there ? bw + kb * 32 : b, there);
            }
            if (pairs && col < p.n_out) {
                if (has0) copy4(to, y0);
                if (more && has1) copy4(to + 4, y1);
            }
        }
        copies_commit();
        --left;
        row += 64;
        col += 64;
        bw += 64 * rank;
        y0 += 64;
        y1 += 64;
        to += kPieces * kPiece;
        if (to == own + kDepth * kPieces * kPiece) to = own;
    };
#pragma unroll
    for (int i = 0; i < kDepth; ++i) load();
    float* part = kWk > 1 ? parts + wk * kFewUnit * rank : sums;          // (with one part the warps' tiles are the sums)
#pragma unroll
    for (int i = 0; i < TP; ++i) {
        const int t = wr + i * RB;
        if (t >= rt) break;
        float* d = part + t * 8 + 2 * q;
        d[g * rank] = acc[i][0];
        d[g * rank + 1] = acc[i][1];
        d[(g + 8) * rank] = acc[i][2];
        d[(g + 8) * rank + 1] = acc[i][3];
    }
    if (kWk > 1) {
        __syncthreads();
        for (int i = tid; i < m * rank; i += kThreads) {
            float v = 0.f;
#pragma unroll
            for (int k = 0; k < kWk; ++k) v += parts[k * kFewUnit * rank + i];
            sums[i] = v;
        }
    }
    if (ctas > 1) cluster_sync();
    else __syncthreads();
    for (int i = tid; i < kFewUnit * RB * 32; i += kThreads) {
        const int r = i / (RB * 32), k = i % (RB * 32);
        float v = 0.f;
        if (r < m && k < rank) {
            const uint32_t at = smem_addr(&sums[r * rank + k]);
            if (ctas > 1) {
                float u[8];                   // all on their way before the first is added
#pragma unroll
                for (int peer = 0; peer < 8; ++peer) u[peer] = peer < ctas ? ld_peer(peer_addr(at, peer)) : 0.f;
#pragma unroll
                for (int peer = 0; peer < 8; ++peer) v += u[peer];
            } else {
                v = sums[r * rank + k];
            }
            v *= sc;
        }
        const float left = after_upper(v), part[3] = {v, left, left - upper(left)};
#pragma unroll
        for (int h = 0; h < 3; ++h)
            low_rows[(h * kFewUnit + r) * RB * 32 + (RB > 1 ? k ^ ((r & 1) * 32) : k)] = __ushort_as_bfloat16((unsigned short)(__float_as_uint(part[h]) >> 16));
    }
    if (ctas > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");     // this CTA has read the others' sums
    __syncthreads();

    // + t . b^T
    const uint4* low_even = reinterpret_cast<const uint4*>(low_rows) + g * RB * 4 + (RB > 1 ? (g & 1) * 4 : 0) + q;     // of even blocks, odd ones
    const uint4* low_odd = low_even - (g & 1) * 8;
    auto low_at = [&](int kb, int h, int r) { return (kb & 1 ? low_odd : low_even)[(h * kFewUnit + r * 8) * RB * 4 + kb * 4]; };     // hi, mid, lo; rows g and g + 8
    // Up to a rank of 128 the low-rank rows stay in registers (read for every tile they cost a rank of 128 half of its time), of
    // ranks above 64 hi and mid alone (lo from shared memory: 128 rows of 2 adapters 17.3 us, all three, with spills, 18.1).
    constexpr int kKept = RB <= 4 ? RB : 1, kParts = RB == 4 ? 2 : 3;
    uint4 low[kKept][kParts][2];
#pragma unroll
    for (int kb = 0; kb < kKept; ++kb)
#pragma unroll
        for (int h = 0; h < kParts; ++h)
#pragma unroll
            for (int r = 0; r < 2; ++r) low[kb][h][r] = low_at(kb, h, r);
    size_t at0 = (size_t)row0 * p.n_out + (t0 + warp) * 8 + 2 * q, at1 = (size_t)row1 * p.n_out + (t0 + warp) * 8 + 2 * q;
    int out_col = (t0 + warp) * 8 + 2 * q;
    uint32_t from = own;
    auto write = [&](size_t at, uint32_t y, float d0, float d1) {
        if (pairs) {
            const float2 v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&y));
            *reinterpret_cast<__nv_bfloat162*>(p.out + at) = __floats2bfloat162_rn(v.x + d0, v.y + d1);
        } else {
            p.out[at] = __float2bfloat16_rn(__bfloat162float(p.y[at]) + d0);
            if (out_col + 1 < p.n_out) p.out[at + 1] = __float2bfloat16_rn(__bfloat162float(p.y[at + 1]) + d1);
        }
    };
    for (int i = 0; i < n; ++i) {
        copies_wait<kDepth - 1>();
        float d[4] = {0.f, 0.f, 0.f, 0.f}, e[4] = {0.f, 0.f, 0.f, 0.f};
        const uint4 yv = ld_shared16(from);
#pragma unroll
        for (int kb = 0; kb < RB; ++kb) {
            const uint4 w = ld_shared16(from + (1 + kb) * kPiece);
            const int i0 = kKept == RB ? kb : 0;
            if (kKept != RB) {
#pragma unroll
                for (int h = 0; h < kParts; ++h) {
                    low[0][h][0] = low_at(kb, h, 0);
                    if (more) low[0][h][1] = low_at(kb, h, 1);
                }
            }
            // (two sums, lo in both by turns: one for mid and lo would make the chain of MMAs twice as long)
            const uint4 h0 = low[i0][0][0], h1 = low[i0][0][1], m0 = low[i0][1][0], m1 = low[i0][1][1];
            const uint4 l0 = kParts == 3 ? low[i0][kParts - 1][0] : low_at(kb, 2, 0), l1 = kParts == 3 ? low[i0][kParts - 1][1] : low_at(kb, 2, 1);
            mma(e, l0.x, l1.x, l0.y, l1.y, w.x, w.y);
            mma(d, l0.z, l1.z, l0.w, l1.w, w.z, w.w);
            mma(e, m0.x, m1.x, m0.y, m1.y, w.x, w.y);
            mma(d, h0.x, h1.x, h0.y, h1.y, w.x, w.y);
            mma(e, m0.z, m1.z, m0.w, m1.w, w.z, w.w);
            mma(d, h0.z, h1.z, h0.w, h1.w, w.z, w.w);
        }
        if (out_col < p.n_out) {
            if (has0) write(at0, yv.x, d[0] + e[0], d[1] + e[1]);
            if (more && has1) write(at1, yv.y, d[2] + e[2], d[3] + e[3]);
        }
        load();
        at0 += 64;
        at1 += 64;
        out_col += 64;
        from += kPieces * kPiece;
        if (from == own + kDepth * kPieces * kPiece) from = own;
    }
    copies_wait<0>();
    if (ctas > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");       // ... and they this one's
}

struct FewKernel {
    const void* kernel;
    int rb;
};
FewKernel few_kernel(int rank) {
    if (rank <= 8) return {(const void*)low_rank_few_kernel<1, 1>, 1};
    if (rank <= 16) return {(const void*)low_rank_few_kernel<1, 2>, 1};
    if (rank <= 32) return {(const void*)low_rank_few_kernel<1, 4>, 1};
    if (rank <= 64) return {(const void*)low_rank_few_kernel<2, 4>, 2};
    if (rank <= 128) return {(const void*)low_rank_few_kernel<4, 4>, 4};
    return {(const void*)low_rank_few_kernel<8, 4>, 8};
}

// ── many rows ───────────────────────────────────────────────────────────────
constexpr int kTileRows = 64;
constexpr int kCols = 64;                     // columns of a stage, of the input first, then of the output
constexpr int kMaxBins = 2048;                // adapters + 1
constexpr int kBlockRows = 8192;              // rows of a launch: each CTA looks through all their ids
constexpr int kBlock = kTileRows * 128;       // bytes of 64 rows of 64 values in the MMA's K-major layout with 128-byte swizzle

constexpr int kTileThreads = kThreads + 64;    // eight warps that copy and write out, one that issues the MMAs, one that loads a and b
constexpr int kMaxStages = 5;
constexpr size_t kPrefetch = (size_t)64 << 20;     // bytes of x that L2 takes in and keeps until they are read

struct TileShared {
    int32_t rows[kTileRows];
    int32_t warp_count[8];
    int32_t n_rows, id, first;
    uint64_t rows_there[kMaxStages];          // the stage's rows of x (eight warps)
    uint64_t loaded[kMaxStages];              // ... its part of a or b (TMA)
    uint64_t used[kMaxStages];                // its MMAs are done
    uint64_t sums_there[2], sums_free[2];     // second product: a stage's sums, and its place in tensor memory
    uint64_t retired;
    uint32_t tmem_base;
    int abort;
};
struct TileMaps {
    CUtensorMap a, b;
};

// NJ: blocks of 32 values of the rank (1, 2, 4 or 8).  The first product's sums have a place of their own up to a rank of 128
// only: below 65 the stages and the low-rank rows of two CTAs fill an SM, and the sums go where the last stage of the first
// product was; beyond 128 they take the stages' place.
struct TilePlan {
    int r16, blocks;                          // rank rounded up to 16; blocks of 64 of it
    int stages, stage, sums_at, low_at, low_pitch, bytes;  // low_at: the low-rank rows, fp32, low_pitch values apart (no bank twice)
    __host__ __device__ constexpr TilePlan(int rank, int nj) : r16(0), blocks(0), stages(0), stage(0), sums_at(0), low_at(0), low_pitch(0), bytes(0) {
        r16 = (rank + 15) & ~15;
        blocks = (r16 + 63) / 64;
        stages = nj <= 4 ? 5 : 3;
        const int first = kBlock + r16 * 128, second = blocks * kBlock + kTileRows * 128;
        stage = ((first > second ? first : second) + 1023) & ~1023;
        low_at = stages * stage;
        low_pitch = r16 + 4;
        const int end = low_at + kTileRows * low_pitch * 4;
        sums_at = nj == 4 ? end : 0;
        bytes = end + (nj == 4 ? kTileRows * r16 * 4 : 0);
        if (nj > 2 && bytes + 1024 < (int)kClusterSmem) bytes = (int)kClusterSmem - 1024;
    }
    constexpr size_t smem() const { return (size_t)bytes + 1024; }
};
static_assert(TilePlan(8, 1).smem() >= kTileSmem && TilePlan(40, 2).smem() >= kTileSmem, "beside another kernel that waits in a cluster");

// (On their way until tmem_wait.)  16 lanes x 8 columns a count: thread t gets of each block of eight columns lane t / 4, columns 2 (t % 4), +1, and the same of
// lane t / 4 + 8, as an mma.sync leaves its sums.
__device__ __forceinline__ void tmem_ld_16x16(uint32_t taddr, float (&v)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
                 : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait(float (&v)[8]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7])::"memory");
}
__device__ __forceinline__ void tmem_ld_16x32(uint32_t taddr, uint32_t (&u)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]), "=r"(u[9]),
                   "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15])
                 : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait(uint32_t (&u)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(u[0]), "+r"(u[1]), "+r"(u[2]), "+r"(u[3]), "+r"(u[4]), "+r"(u[5]), "+r"(u[6]), "+r"(u[7]), "+r"(u[8]), "+r"(u[9]),
                   "+r"(u[10]), "+r"(u[11]), "+r"(u[12]), "+r"(u[13]), "+r"(u[14]), "+r"(u[15])::"memory");
}

// Eight warps gather x, and y, by cp.async; a ninth issues the MMAs, a tenth brings a and b by TMA.  In the second product a warp
// copies, adds and writes 16 rows x 32 columns that no other warp touches, so that the warps meet nowhere but at the
// accumulators (with a __syncthreads and the MMAs' issue in every stage 8192 tokens of rank 16 took 97 us).
// `clusters` clusters a unit: each multiplies x . a^T for itself and takes a part of the columns.
// WIDE: rows of y and of out are whole 16-byte pieces.
template <int NJ, bool WIDE>
__global__ void __launch_bounds__(kTileThreads, NJ <= 2 ? 2 : 1)
low_rank_tile_kernel(const LowRankArgs p, const int ctas, const int clusters, const __grid_constant__ TileMaps maps) {
    extern __shared__ unsigned char smem_raw[];
    __shared__ TileShared s;
    unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    const TilePlan pl(p.rank, NJ);
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const int shift = 31 - __clz(ctas), cut = shift + 31 - __clz(clusters);       // (both are powers of two)
    const int unit = (int)blockIdx.x >> cut, c = (int)blockIdx.x & (ctas - 1);
    const int spin = p.give_up > 1 && p.give_up - 2 != c ? kSpin : p.spin_limit;
    // First of all the tensor memory: an SM starts its second CTA only when the first has given up the permit to allocate (with
    // the allocation behind the ids half of the CTAs of 8192 rows started 6.7 us late, of 777 rows 3.2).
    // The first product's sums; in their place two stages' of the second, and from column 128 on its A, see below.
    static_assert(NJ > 2 || 2 * (128 + 2 * 16 * NJ) <= 512, "two CTAs an SM");
    // (The tensor cores cut each addition off, not round it: a sum of 172 K steps is off by up to 2^-18, as much as 16 bits of the
    // low-rank row.  So the first product has several sums, a stage each in turn, which are added in the end.)
    constexpr uint32_t kTmem = NJ <= 2 ? 256 : 512, kLowAt = 128, kLowCols = 16 * NJ;
    constexpr int kSums = NJ <= 4 ? 4 : 2;
    static_assert(kSums * NJ * 32 <= (int)kTmem && kLowAt + 2 * kLowCols <= kTmem, "tensor memory");
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_u32(&s.tmem_base)), "r"(kTmem) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // (Which kernels are beside this one on an SM: internal.h.)
    auto give_back = [&]() {
        if (warp == 9) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(s.tmem_base), "r"(kTmem) : "memory");
    };
    // Units of this block of rows: adapter 0's rows in tiles of 64, adapter 1's, ..., at last the rows without one.  A warp
    // has an eighth of the ids, 32 at a time in batch order, all of them in registers: as loads of the loops below, one after
    // the other, they took 22 us.
    int32_t* bins = reinterpret_cast<int32_t*>(smem);
    const int n_bins = p.count + 1;
    constexpr int kIds = kBlockRows / kThreads;
    const int groups = warp < 8 ? (p.n + kThreads - 1) / kThreads : 0, from = warp * groups * 32;
    int bin[kIds];
    // (in lots of eight: what is done for none of the ids of a small batch costs it 2 us)
    auto lots = [&](auto&& each) {
#pragma unroll
        for (int i = 0; i < kIds; ++i) {
            if (i % 8 == 0 && i >= groups) break;
            each(i);
        }
    };
#pragma unroll
    for (int i = 0; i < kIds; ++i) bin[i] = -1;
    lots([&](int i) {
        const int r = from + i * 32 + lane;
        if (i < groups && r < p.n) bin[i] = p.ids[r];
    });
    lots([&](int i) {
        if (i < groups && from + i * 32 + lane < p.n && (bin[i] < 0 || bin[i] >= p.count)) bin[i] = p.count;
    });
    // While the others count, memory would be idle: x on its way into L2, a part of the rows by each CTA.
    if (warp == 9 && (size_t)p.n * p.in * 2 <= kPrefetch)
        for (long r = (long)p.n * blockIdx.x / gridDim.x + lane; r < (long)p.n * (blockIdx.x + 1) / gridDim.x; r += 32) {
            const int j = p.ids[r];
            if (j >= 0 && j < p.count)
                asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p.x + (size_t)r * p.in), "r"(p.in * 2) : "memory");
        }
    __syncwarp();
    for (int i = tid; i < n_bins; i += kTileThreads) bins[i] = 0;
    if (tid == 0) {
        s.n_rows = 0;
        s.abort = 0;
        for (int i = 0; i < kMaxStages; ++i) {
            tc::mbar_init(tc::smem_u32(&s.rows_there[i]), 8);
            tc::mbar_init(tc::smem_u32(&s.loaded[i]), 1);
            tc::mbar_init(tc::smem_u32(&s.used[i]), 1);
        }
        for (int i = 0; i < 2; ++i) {
            tc::mbar_init(tc::smem_u32(&s.sums_there[i]), 1);
            tc::mbar_init(tc::smem_u32(&s.sums_free[i]), 8);
        }
        tc::mbar_init(tc::smem_u32(&s.retired), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    // A group of 32 inside a prompt is one addition, lane i's for group i, all groups of an adapter's one; the ids of the others
    // are added one by one.  (One after the other the groups took 120 cycles each.)
    int all = -1;                             // the adapter of the whole of group `lane`
    lots([&](int i) {
        const int first = __shfl_sync(0xffffffffu, bin[i], 0);
        const bool whole = __all_sync(0xffffffffu, bin[i] == first);
        if (whole && lane == i) all = first;
    });
    const unsigned alike = __match_any_sync(0xffffffffu, all), whole = __ballot_sync(0xffffffffu, all >= 0);
    if (all >= 0 && lane == __ffs(alike) - 1) atomicAdd(&bins[all], 32 * __popc(alike));
    lots([&](int i) {
        if (!(whole >> i & 1u) && bin[i] >= 0) atomicAdd(&bins[bin[i]], 1);
    });
    __syncthreads();
    if (warp == 0) {
        int before = 0;
        for (int base = 0; base < n_bins; base += 32) {
            const int rows = base + lane < n_bins ? bins[base + lane] : 0, units = (rows + kTileRows - 1) / kTileRows;
            int up_to = units;
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const int v = __shfl_up_sync(0xffffffffu, up_to, o);
                if (lane >= o) up_to += v;
            }
            const int mine = unit - before - (up_to - units);
            if (mine >= 0 && mine < units) {
                s.id = base + lane;
                s.first = mine * kTileRows;
                s.n_rows = min(kTileRows, rows - s.first);
            }
            before += __shfl_sync(0xffffffffu, up_to, 31);
        }
    }
    __syncthreads();
    const int m = s.n_rows, id = s.id, skip = s.first;
    if (m == 0) {                             // fewer units than clusters: the whole cluster leaves
        give_back();
        return;
    }
    {
        // the unit's rows: those of the bin from the skip-th on, in batch order; lane i has group i
        unsigned hit = 0;
        lots([&](int i) {
            const unsigned h = __ballot_sync(0xffffffffu, bin[i] == id);
            if (lane == i) hit = h;
        });
        int up_to = __popc(hit);
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const int v = __shfl_up_sync(0xffffffffu, up_to, o);
            if (lane >= o) up_to += v;
        }
        if (lane == 31 && warp < 8) s.warp_count[warp] = up_to;
        __syncthreads();
        int start = up_to - __popc(hit) - skip;
        for (int w = 0; w < min(warp, 8); ++w) start += s.warp_count[w];
        unsigned todo = __ballot_sync(0xffffffffu, hit != 0 && start < m && start + __popc(hit) > 0);
        while (todo != 0) {
            const int i = __ffs(todo) - 1;
            todo &= todo - 1;
            const unsigned h = __shfl_sync(0xffffffffu, hit, i);
            const int at = __shfl_sync(0xffffffffu, start, i) + __popc(h & ((1u << lane) - 1u));
            if ((h >> lane & 1u) && at >= 0 && at < m) s.rows[at] = from + i * 32 + lane;
        }
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, s.tmem_base, 0);
    // chunks of the input and of the output dimension that this CTA takes
    const int ik = (p.in + kCols - 1) / kCols, on = (p.n_out + kCols - 1) / kCols;
    const int part_of = (int)blockIdx.x & ((1 << cut) - 1);
    const int k0 = (int)((long)ik * c >> shift), k1 = (int)((long)ik * (c + 1) >> shift);
    const int n0 = (int)((long)on * part_of >> cut), n1 = (int)((long)on * (part_of + 1) >> cut);
    if (id == p.count) {
        give_back();
        if (p.out != p.y)
            for (int r = warp; r < m; r += kTileThreads / 32) {
                const size_t at = (size_t)s.rows[r] * p.n_out;
                const int end = min(n1 * kCols, p.n_out);
                if (WIDE)
                    for (int n = n0 * kCols + lane * 8; n < end; n += 256) *reinterpret_cast<uint4*>(p.out + at + n) = *reinterpret_cast<const uint4*>(p.y + at + n);
                else
                    for (int n = n0 * kCols + lane; n < end; n += 32) p.out[at + n] = p.y[at + n];
            }
        return;
    }
    const int rank = p.rank, r16 = pl.r16, n_blocks = pl.blocks;
    constexpr int S = NJ <= 4 ? 5 : 3;                     // (TilePlan::stages)
    const uint32_t base = tc::smem_u32(smem);
    // both products' stages in one line, stage i in the place i mod S: x or y, then a or b
    const int n_in = k1 - k0, total = n_in + (n1 - n0);
    const int early = NJ <= 4 ? total : n_in;              // (beyond a rank of 128 the second product's wait for the sums to leave)
    volatile int* abort_flag = &s.abort;
    int issued = 0;                                        // stages whose a or b is on its way

    if (warp == 9) {
        int slot = 0;
        uint32_t ph = 1;                                   // of the MMAs that free the place, the first of which need not be waited for
        bool ok = true;
        auto fill = [&](int upto) {
            for (; issued < upto && ok; ++issued) {
                ok = tc::mbar_wait(tc::smem_u32(&s.used[slot]), ph, abort_flag, spin);
                if (!ok) break;
                if (lane == 0) {
                    const uint32_t to = base + (uint32_t)(slot * pl.stage + kBlock), bar = tc::smem_u32(&s.loaded[slot]);
                    if (issued < n_in) {
                        tc::mbar_expect_tx(bar, (uint32_t)(r16 * 128));
                        tc::tma_load_2d(to, &maps.a, (k0 + issued) * kCols, id * rank, bar);
                    } else {
                        tc::mbar_expect_tx(bar, (uint32_t)(n_blocks * kBlock));
                        for (int kb = 0; kb < n_blocks; ++kb)
                            tc::tma_load_2d(to + kb * kBlock, &maps.b, kb * 64, id * p.n_out + (n0 + issued - n_in) * kCols, bar);
                    }
                }
                __syncwarp();
                if (++slot == S) {
                    slot = 0;
                    ph ^= 1u;
                }
            }
        };
        // (no further than the places that the first product leaves free; the sums take one, or all, until the cluster has met twice)
        fill(min(n_in + S - 1, early));
        if (ctas > 1) cluster_sync();
        else __syncthreads();
        if (ctas > 1) cluster_sync();
        else __syncthreads();
        fill(total);
    } else if (warp == 8) {
        const uint32_t flag = tc::smem_u32(&s.abort), me = tc::elect_one() ? 1u : 0u;
        int slot = 0;
        uint32_t ph = 0;
        auto next_stage = [&]() {
            if (++slot == S) {
                slot = 0;
                ph ^= 1u;
            }
        };
        for (int i = 0; i < n_in; ++i) {
            tc::mbar_wait_on(tc::smem_u32(&s.rows_there[slot]), ph, flag, spin);
            tc::mbar_wait_on(tc::smem_u32(&s.loaded[slot]), ph, flag, spin);
            tc::tc_fence_after();
            const uint32_t st = base + (uint32_t)(slot * pl.stage), idesc = tc::idesc_for(64, r16) | (1u << 7) | (1u << 10);      // bf16
#pragma unroll
            for (int kk = 0; kk < kCols / 16; ++kk)
                tc::umma_ss_if(me, tmem + (uint32_t)((i % kSums) * NJ * 32), tc::smem_desc(st) + 2 * kk, tc::smem_desc(st + kBlock) + 2 * kk, idesc,
                               i >= kSums || kk > 0 ? 1u : 0u);
            tc::umma_commit_if<false>(me, tc::smem_u32(&s.used[slot]));
            __syncwarp();
            next_stage();
        }
        // the low-rank rows are made by the others
        if (ctas > 1) cluster_sync();
        else __syncthreads();
        if (ctas > 1) cluster_sync();
        else __syncthreads();
        asm volatile("bar.sync 1, %0;" ::"n"(kThreads + 32) : "memory");   // ... and in tensor memory
        tc::tc_fence_after();
        const uint32_t idesc = tc::idesc_for(128, kCols) | (1u << 7) | (1u << 10);
        const int kks = r16 / 16;
        for (int e = 0; e < total - n_in; ++e) {
            tc::mbar_wait_on(tc::smem_u32(&s.loaded[slot]), ph, flag, spin);
            if (e >= 2) tc::mbar_wait_on(tc::smem_u32(&s.sums_free[e & 1]), (uint32_t)((e - 2) >> 1) & 1u, flag, spin);
            tc::tc_fence_after();
            const uint32_t d = tmem + (uint32_t)((e & 1) * 64);
            const uint64_t b_desc = tc::smem_desc(base + (uint32_t)(slot * pl.stage + kBlock));
#pragma unroll
            for (int part = 1; part >= 0; --part)          // (the small ones first)
#pragma unroll
                for (int kk = 0; kk < 2 * NJ; ++kk)
                    if (kk < kks)
                        tc::umma_ts_if(me, d, tmem + kLowAt + (uint32_t)(part * kLowCols + kk * 8),
                                       b_desc + (uint64_t)((kk >> 2) * (kBlock >> 4) + 2 * (kk & 3)), idesc, part == 0 || kk > 0 ? 1u : 0u);
            tc::umma_commit_if<false>(me, tc::smem_u32(&s.used[slot]));
            tc::umma_commit_if<false>(me, tc::smem_u32(&s.sums_there[e & 1]));
            __syncwarp();
            next_stage();
        }
    } else {
        const int rt = warp & 3, half = warp >> 2, g = lane >> 2, q = lane & 3;    // the warp's 16 rows, and its half of the columns
        auto wait = [&](uint64_t& bar, int phase) { tc::mbar_wait(tc::smem_u32(&bar), (uint32_t)phase & 1u, abort_flag, spin); };
        const float sc = p.scale != nullptr ? p.scale[id] : 1.f;
        // What a thread copies is the same in every stage but for the columns: a piece of two rows of x, or of y.
        const int cr = tid >> 3, cc = (tid & 7) * 8;
        const __nv_bfloat16* xr[2];
        const __nv_bfloat16* yr[2];
        __nv_bfloat16* to_own[2];
        uint32_t y_at[2];                     // of the piece in the stage
        bool has[2], has_own[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            has[i] = cr + 32 * i < m;
            xr[i] = p.x + (size_t)s.rows[has[i] ? cr + 32 * i : 0] * p.in + k0 * kCols + cc;
            const int r = rt * 16 + g + 8 * i;
            has_own[i] = r < m;
            const size_t at = (size_t)s.rows[has_own[i] ? r : 0] * p.n_out + n0 * kCols + half * 32 + q * 8;
            yr[i] = p.y + at;
            to_own[i] = p.out + at;
            y_at[i] = (uint32_t)(r * 128 + (((half * 4 + q) ^ (r & 7)) * 16));
        }
        const uint32_t x_at = (uint32_t)(cr * 128 + (((tid & 7) ^ (cr & 7)) * 16));
        int in_left = p.in - k0 * kCols - cc, y_left = p.n_out - n0 * kCols - half * 32 - q * 8;      // columns of x and of y up to the end
        int next = 0;                         // stage to copy next
        uint32_t to = base;                   // its place
        auto copy = [&](int upto) {
            if (next < upto) {
                if (next < n_in) {
                    const bool in = in_left > 0;
#pragma unroll
                    for (int i = 0; i < 2; ++i) copy16(to + x_at + i * 32 * 128, in && has[i] ? xr[i] : p.x, in && has[i]);
                    in_left -= kCols;
                    xr[0] += kCols;
                    xr[1] += kCols;
                } else {
                    if (WIDE) {
#pragma unroll
                        for (int i = 0; i < 2; ++i)
                            if (y_left > 0 && has_own[i]) copy16(to + y_at[i], yr[i], true);
                    }
                    y_left -= kCols;
                    yr[0] += kCols;
                    yr[1] += kCols;
                }
                ++next;
                to += pl.stage;
                if (to == base + (uint32_t)(S * pl.stage)) to = base;
            }
            copies_commit();
        };
        auto arrived = [&]() {                // the oldest of S - 1 copies
            if (NJ <= 4) copies_wait<3>();
            else copies_wait<1>();
        };
        for (int i = 0; i < S - 1; ++i) copy(early);
        for (int i = 0; i < n_in; ++i) {
            arrived();
            tc::fence_async_proxy();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(tc::smem_u32(&s.rows_there[i % S]));
            if (i > 0) wait(s.used[(i - 1) % S], (i - 1) / S);             // the place of the next copy is free
            copy(early);
        }
        // the low-rank rows: this CTA's part of the sums, then all of them in every CTA
        auto sums_of = [&](int cta) {         // their place in a CTA
            return NJ <= 2 ? (((int)((long)ik * (cta + 1) >> shift) - (int)((long)ik * cta >> shift) + S - 1) % S) * pl.stage : pl.sums_at;
        };
        float* sums = reinterpret_cast<float*>(smem + sums_of(c));
        if (n_in > 0) wait(s.used[(n_in - 1) % S], (n_in - 1) / S);
        tc::tc_fence_after();
        const bool gave_up = *abort_flag != 0;             // a CTA that has makes the low-rank rows NaN, and so all outputs of the cluster
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const int t = half + 2 * j;
            if (t * 16 >= r16) break;
            float v[8] = {}, u[kSums][8];
#pragma unroll
            for (int k = 0; k < kSums; ++k)
                if (k < n_in) tmem_ld_16x16(tmem + ((uint32_t)(rt * 32) << 16) + (uint32_t)(k * NJ * 32 + t * 16), u[k]);
#pragma unroll
            for (int k = 0; k < kSums; ++k) {
                if (k >= n_in) break;
                tmem_wait(u[k]);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] += u[k][i];
            }
            if (gave_up)
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(0x7fc00000u);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float* d = sums + (rt * 16 + g) * r16 + t * 16 + h * 8 + 2 * q;
                *reinterpret_cast<float2*>(d) = make_float2(v[4 * h], v[4 * h + 1]);
                *reinterpret_cast<float2*>(d + 8 * r16) = make_float2(v[4 * h + 2], v[4 * h + 3]);
            }
        }
        tc::tc_fence_before();
        if (ctas > 1) cluster_sync();
        else __syncthreads();
        const int pieces = r16 / 8;
        // A CTA makes every ctas-th piece of eight values, ctas lanes one: each brings a CTA's part, they add them by a tree (the
        // order is the same for all), and each writes the piece into one CTA.  By one lane it took 2.3 us, twice as long.
        const int peer = lane & (ctas - 1), parts_at = sums_of(peer);
        for (int li = tid >> shift; (li - (lane >> shift)) * ctas + c < m * pieces; li += kThreads >> shift) {       // (what is in the other rows reaches no output)
            const int i = li * ctas + c, r = i / pieces, j = i - r * pieces;
            const bool mine = i < m * pieces;
            float v[8] = {};
            if (mine) {
                const uint32_t at = base + (uint32_t)(parts_at + (r * r16 + j * 8) * 4), src = ctas > 1 ? peer_addr(at, peer) : at;
                const float4 u = ld_peer4(src), w = ld_peer4(src + 16);
                v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
                v[4] = w.x; v[5] = w.y; v[6] = w.z; v[7] = w.w;
            }
            for (int d = 1; d < ctas; d *= 2)
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] += __shfl_xor_sync(0xffffffffu, v[e], d);
            if (!mine) continue;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = j * 8 < rank ? v[e] * sc : 0.f;                     // (past the rank: another adapter's)
            const uint32_t at = base + (uint32_t)(pl.low_at + (r * pl.low_pitch + j * 8) * 4), dst = ctas > 1 ? peer_addr(at, peer) : at;
            st_peer4(dst, make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])));
            st_peer4(dst + 16, make_uint4(__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7])));
        }
        asm volatile("fence.proxy.async.shared::cluster;" ::: "memory");   // (TMA writes where the sums were)
        if (ctas > 1) cluster_sync();
        else __syncthreads();
        // The second product's A is the same in every stage and lies in tensor memory, so that its MMAs read b alone from shared
        // memory, whose bandwidth the copies of y need (a call on 8192 rows of rank 64: 78.4 us, with A there, too, 86 to 91): hi
        // and mid of a warp's 16 rows in its 32 lanes, and in columns behind them lo and zeros.
        {
            const float* row = reinterpret_cast<const float*>(smem + pl.low_at) + (rt * 16 + (lane & 15)) * pl.low_pitch;
            const uint32_t keep = lane < 16 ? 0xffffffffu : 0u;
#pragma unroll 1
            for (int jb = 0; jb < NJ; ++jb) {
                uint32_t cols[16] = {};
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int k = jb * 32 + i * 4;
                    if (k >= r16) break;
                    const float4 f = *reinterpret_cast<const float4*>(row + k);
                    const float l0 = after_upper(f.x), l1 = after_upper(f.y), l2 = after_upper(f.z), l3 = after_upper(f.w);
                    if (half == 0) {
                        cols[2 * i] = pack2(lane < 16 ? f.x : l0, lane < 16 ? f.y : l1);
                        cols[2 * i + 1] = pack2(lane < 16 ? f.z : l2, lane < 16 ? f.w : l3);
                    } else {
                        cols[2 * i] = pack2(l0 - upper(l0), l1 - upper(l1)) & keep;
                        cols[2 * i + 1] = pack2(l2 - upper(l2), l3 - upper(l3)) & keep;
                    }
                }
                tc::tmem_st16(tmem + ((uint32_t)(rt * 32) << 16) + kLowAt + (uint32_t)(half * (int)kLowCols + jb * 16), cols);
            }
            tc::tmem_st_wait();
            tc::tc_fence_before();
            asm volatile("bar.arrive 1, %0;" ::"n"(kThreads + 32) : "memory");
        }
        if (NJ > 4)
            for (int i = 0; i < S - 1; ++i) copy(total);
        int n = n0 * kCols;                                // first column of the stage
        uint32_t y = base + (uint32_t)((n_in % S) * pl.stage);                   // ... and its place
        const uint32_t frag_at = (uint32_t)((rt * 16 + (lane & 7)) * 128 + (((half * 4 + (lane >> 3)) ^ (lane & 7)) * 16));
        // Rows that start on 4 bytes, not on 16: a lane's own values two at a time, a stage ahead (5034 outputs, 2579 rows of rank
        // 128: 74 us; 5033 outputs, one by one when they are needed, 186).  Rows of an odd number are left at that.
        const bool pairs = !WIDE && p.n_out % 2 == 0 && (((uintptr_t)p.y | (uintptr_t)p.out) % 4) == 0;
        const size_t row_at[2] = {(size_t)s.rows[has_own[0] ? rt * 16 + g : 0] * p.n_out, (size_t)s.rows[has_own[1] ? rt * 16 + g + 8 : 0] * p.n_out};
        uint32_t ahead[2][4];
        auto fetch = [&](int from) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int col = from + half * 32 + j * 8 + 2 * q;
                    ahead[h][j] = has_own[h] && col < p.n_out ? *reinterpret_cast<const uint32_t*>(p.y + row_at[h] + col) : 0u;
                }
        };
        if (pairs && total > n_in) fetch(n);
        for (int e = 0; e < total - n_in; ++e) {
            wait(s.sums_there[e & 1], e >> 1);
            tc::tc_fence_after();
            uint32_t u[16], u_mid[16], v[2][4];
            const uint32_t sums_at = tmem + ((uint32_t)(rt * 32) << 16) + (uint32_t)((e & 1) * 64 + half * 32);
            tmem_ld_16x32(sums_at, u);
            tmem_ld_16x32(sums_at + (16u << 16), u_mid);
            arrived();
            __syncwarp();
            if (WIDE) {
#pragma unroll
                for (int h = 0; h < 2; ++h) ld_matrices(y + frag_at + h * 1024, v[h]);
            }
            tmem_wait(u);
            tmem_wait(u_mid);
            tc::tc_fence_before();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(tc::smem_u32(&s.sums_free[e & 1]));
            float d[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) d[i] = __uint_as_float(u[i]) + __uint_as_float(u_mid[i]);
            if (WIDE) {
                // added in y's place, which is read and written as 8 x 8 matrices (the sums' layout), out in 16-byte pieces
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v[h][j]));
                        const __nv_bfloat162 o = __floats2bfloat162_rn(f.x + d[4 * j + 2 * h], f.y + d[4 * j + 2 * h + 1]);
                        v[h][j] = *reinterpret_cast<const uint32_t*>(&o);
                    }
                    st_matrices(y + frag_at + h * 1024, v[h]);
                }
                __syncwarp();
                const bool in = n + half * 32 + q * 8 < p.n_out;
                const uint4 o0 = ld_shared16(y + y_at[0]), o1 = ld_shared16(y + y_at[1]);
                if (has_own[0] && in) *reinterpret_cast<uint4*>(to_own[0]) = o0;
                if (has_own[1] && in) *reinterpret_cast<uint4*>(to_own[1]) = o1;
            } else if (pairs) {
                uint32_t now[2][4];
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int j = 0; j < 4; ++j) now[h][j] = ahead[h][j];
                if (e + 1 < total - n_in) fetch(n + kCols);
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int col = n + half * 32 + j * 8 + 2 * q;
                        if (!has_own[h] || col >= p.n_out) continue;
                        const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&now[h][j]));
                        const __nv_bfloat162 o = __floats2bfloat162_rn(f.x + d[4 * j + 2 * h], f.y + d[4 * j + 2 * h + 1]);
                        *reinterpret_cast<__nv_bfloat162*>(p.out + row_at[h] + col) = o;
                    }
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int h = 0; h < 4; ++h) {
                        const int col = n + half * 32 + j * 8 + 2 * q + (h & 1);
                        if (has_own[h >> 1] && col < p.n_out) {
                            const size_t at = row_at[h >> 1] + col;
                            p.out[at] = __float2bfloat16_rn(__bfloat162float(p.y[at]) + d[4 * j + h]);
                        }
                    }
            }
            n += kCols;
            to_own[0] += kCols;
            to_own[1] += kCols;
            y += pl.stage;
            if (y == base + (uint32_t)(S * pl.stage)) y = base;
            copy(total);                                   // into the place of the stage before this one, of y if not of x: see above
        }
        copies_wait<0>();
    }
    __syncthreads();
    if (s.abort != 0) {                                    // a wait ran out: NaN in this CTA's columns (after the exchange in these alone)
        if (warp == 8) {
            if (tc::elect_one()) tc::umma_commit(tc::smem_u32(&s.retired));
            __syncwarp();
            tc::mbar_drain(tc::smem_u32(&s.retired), 0u);
        } else if (warp == 9) {
            for (int i = max(0, issued - S); i < issued; ++i) tc::mbar_drain(tc::smem_u32(&s.loaded[i % S]), (uint32_t)(i / S) & 1u);
        }
        if (tid == 0) atomicExch(p.status, 5);
        for (int r = warp; r < m; r += kTileThreads / 32)
            for (int col = n0 * kCols + lane; col < min(n1 * kCols, p.n_out); col += 32)
                p.out[(size_t)s.rows[r] * p.n_out + col] = __float2bfloat16_rn(__uint_as_float(0x7fc00000u));
        __syncthreads();
    }
    give_back();
}

struct TileKernel {
    const void* kernel;
    int nj;
};
template <bool WIDE>
TileKernel tile_kernel_of(int rank) {
    if (rank <= 32) return {(const void*)low_rank_tile_kernel<1, WIDE>, 1};
    if (rank <= 64) return {(const void*)low_rank_tile_kernel<2, WIDE>, 2};
    if (rank <= 128) return {(const void*)low_rank_tile_kernel<4, WIDE>, 4};
    return {(const void*)low_rank_tile_kernel<8, WIDE>, 8};
}
TileKernel tile_kernel(int rank, bool wide) { return wide ? tile_kernel_of<true>(rank) : tile_kernel_of<false>(rank); }

int launch_clusters(const void* kernel, unsigned grid, int threads, int ctas, size_t smem, cudaStream_t stream, void** args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)ctas;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    IMX_CHECK_CUDA(cudaLaunchKernelExC(&cfg, kernel, args)); IMX_LAUNCHED();
    return IMX_OK;
}

// 128 rows, 2048 -> 4096, by the two kernels, in us: 16 adapters of rank 16, 64, 128  9.5, 13.9, 21.4 and (tiles) 12.9, 15.8, 29.5;
// 120 adapters  17.6, 28.5, 53.2 and 29.5, 35.8, 65.4; 2 adapters  8.8, 12.1, 17.5 and 9.2, 12.0, 16.1.  So up to 128 rows are
// few; so are, 128 at a time, more of them where the tile kernel cannot count the adapters or name b's rows in 31 bits.
int launch_low_rank(LowRankArgs p, int sms, cudaStream_t stream) {
    const int rows = p.n, step = rows <= kFewRows || p.count >= kMaxBins || (long)p.count * p.n_out > 0x7fffffffL ? kFewRows : kBlockRows;
    const LowRankArgs whole = p;
    TileMaps maps;
    if (step != kFewRows) {
        const int r16 = (p.rank + 15) & ~15;
        IMX_TRY(encode_tensor_map_2d(p.a, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, (size_t)p.count * p.rank, (size_t)p.in, (size_t)p.in * 2, kCols, r16, 128,
                                     true, &maps.a));
        IMX_TRY(encode_tensor_map_2d(p.b, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, (size_t)p.count * p.n_out, (size_t)p.rank, (size_t)p.rank * 2, 64, kCols, 128,
                                     true, &maps.b));
    }
    for (size_t r0 = 0; r0 < (size_t)rows; r0 += step) {     // (31 bits do not count the end of the last block of 2^31 - 1 rows)
        p.n = rows - (int)r0 < step ? rows - (int)r0 : step;
        p.x = whole.x + r0 * p.in;
        p.y = whole.y + r0 * p.n_out;
        p.out = whole.out + r0 * p.n_out;
        p.ids = whole.ids + r0;
        int ctas = 1;
        void* args[] = {&p, &ctas, nullptr, nullptr};
        if (step == kFewRows) {
            // Units: no more than every 16th row leads because 16 have gone before, and one of every id.  A cluster up to
            // CTAs for three on every SM (two, where registers or rings leave room for no more): 48 rows of 40 adapters with two 12.4
            // us, with one 14.0, with three 11.7.  More clusters of a unit repeat x . a^T and pay while SMs are idle: one row,
            // 2048 -> 8192, 5.5 us, in one cluster 8.1.
            const FewKernel few = few_kernel(p.rank);
            const int ids = p.count < p.n ? p.count + 1 : p.n, bound = p.n / kFewUnit + ids, units = bound < p.n ? bound : p.n;
            while (ctas < 8 && units * ctas * 2 <= few_ctas(few.rb) * sms) ctas *= 2;
            int clusters = 1;
            while (clusters < 16 && units * ctas * clusters * 2 <= sms && p.n_out >= 128 * ctas * clusters) clusters *= 2;
            args[2] = &clusters;
            IMX_TRY(launch_clusters(few.kernel, (unsigned)(units * ctas * clusters), kThreads, ctas, (size_t)FewPlan(p.rank, few.rb).bytes, stream, args));
            continue;
        }
        // No more units than these; CTAs for two on every SM (for one 8192 rows of rank 64 take 103 us, for four 98, not 82):
        // clusters of up to eight for a unit (777 rows of rank 16: clusters of 8, 4, 2, 1 take 20.4, 21.2, 23.8, 24.4 us),
        // then several of them (200 rows, 2048 -> 8192, with one 18.4 us, with more 16.2).
        const int units = p.n / kTileRows + (p.count + 1 < p.n ? p.count + 1 : p.n);
        while (ctas < 8 && units * ctas * 2 <= 2 * sms) ctas *= 2;
        int clusters = 1;
        while (clusters < 8 && units * ctas * clusters * 2 <= 2 * sms && p.n_out >= 2 * kCols * ctas * clusters) clusters *= 2;
        const TileKernel tile = tile_kernel(p.rank, p.wide != 0);
        args[2] = &clusters;
        args[3] = &maps;
        IMX_TRY(launch_clusters(tile.kernel, (unsigned)(units * ctas * clusters), kTileThreads, ctas, TilePlan(p.rank, tile.nj).smem(), stream, args));
    }
    return IMX_OK;
}

}  // namespace

// Test hook (include/ironmlx_b200_testing.h).
void testing_low_rank_give_up(int on) { g_low_rank_give_up.store(on); }

}  // namespace imx

using namespace imx;

extern "C" void imx_testing_low_rank_give_up(int on) { testing_low_rank_give_up(on); }

extern "C" int imx_low_rank_scratch_bytes(int n_rows, int in, int n_out, int count, int rank, size_t* bytes) {
    IMX_REQUIRE(bytes != nullptr && n_rows >= 0 && in > 0 && n_out > 0 && count > 0 && rank > 0 && rank <= kMaxRank,
                "low_rank_scratch_bytes: bad arguments");
    *bytes = kStatusBytes;
    return IMX_OK;
}

extern "C" int imx_low_rank_add(const void* y, const void* x, int n_rows, int in, const imx_adapters* ad, const int32_t* ids, int n_out,
                                void* out, void* scratch, size_t scratch_bytes, void* stream) {
    IMX_REQUIRE(n_rows >= 0 && n_out > 0 && in > 0 && in % 8 == 0,
                "low_rank_add: sizes (%d rows, %d -> %d) must be positive, the input dimension a multiple of 8", n_rows, in, n_out);
    IMX_REQUIRE(in <= kMostColumns && n_out <= kMostColumns, "low_rank_add: dimensions of at most %d", kMostColumns);
    if (n_rows == 0) return IMX_OK;
    IMX_REQUIRE(y && x && ad && ids && out, "low_rank_add: y, x, adapters, ids and out are required");
    IMX_REQUIRE(ad->a && ad->b && ad->count > 0, "low_rank_add: at least one adapter is required");
    IMX_REQUIRE(ad->rank > 0 && ad->rank % 8 == 0 && ad->rank <= kMaxRank,
                "low_rank_add: the rank (%d) must be a multiple of 8, at most %d", ad->rank, kMaxRank);
    IMX_REQUIRE((((uintptr_t)x | (uintptr_t)ad->a | (uintptr_t)ad->b) % 16) == 0, "low_rank_add: x, a and b must be 16-byte aligned");
    IMX_REQUIRE((((uintptr_t)ids | (uintptr_t)ad->scale) % 4) == 0, "low_rank_add: ids and scale must be aligned to their values");
    IMX_REQUIRE((((uintptr_t)y | (uintptr_t)out) % 2) == 0, "low_rank_add: y and out must be aligned to their bf16 values");
    if (scratch == nullptr || (uintptr_t)scratch % 256 != 0 || scratch_bytes < kStatusBytes) {
        set_error("low_rank_add: 256-byte aligned scratch of %zu bytes needed, %zu given", kStatusBytes, scratch_bytes);
        return IMX_ERR_WORKSPACE;
    }
    const size_t ob = (size_t)n_rows * n_out * 2;
    IMX_REQUIRE(out == y || !overlap(out, ob, y, ob), "low_rank_add: out overlaps y without being it");
    IMX_REQUIRE(!overlap(out, ob, x, (size_t)n_rows * in * 2) && !overlap(out, ob, ids, (size_t)n_rows * 4) &&
                !overlap(out, ob, ad->a, (size_t)ad->count * ad->rank * in * 2) &&
                !overlap(out, ob, ad->b, (size_t)ad->count * ad->rank * n_out * 2) &&
                !overlap(out, ob, ad->scale, (size_t)ad->count * 4) && !overlap(out, ob, scratch, kStatusBytes), "low_rank_add: out overlaps another array");
    DeviceInfo di;
    IMX_TRY(current_device(&di));
    if (device_needs_setup(di.ordinal, kSetupLowRank)) {     // once per device
        for (int rank : {8, 16, 32, 64, 128, 256}) {
            const FewKernel few = few_kernel(rank);
            IMX_CHECK_CUDA(cudaFuncSetAttribute(few.kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, FewPlan(rank, few.rb).bytes));
            for (bool wide : {false, true}) {
                const TileKernel tile = tile_kernel(rank, wide);
                IMX_CHECK_CUDA(cudaFuncSetAttribute(tile.kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)TilePlan(rank, tile.nj).smem()));
            }
        }
        device_mark_setup(di.ordinal, kSetupLowRank);
    }
    const int give_up = g_low_rank_give_up.load();
    const int wide = n_out % 8 == 0 && (((uintptr_t)y | (uintptr_t)out) % 16) == 0;
    return launch_low_rank(LowRankArgs{(const __nv_bfloat16*)y, (const __nv_bfloat16*)x, (const __nv_bfloat16*)ad->a, (const __nv_bfloat16*)ad->b,
                                       ad->scale, ids, (__nv_bfloat16*)out, n_rows, in, n_out, ad->count, ad->rank, wide,
                                       give_up == 0 ? kSpin : 0, give_up, (int32_t*)scratch},
                           di.sms, (cudaStream_t)stream);
}
