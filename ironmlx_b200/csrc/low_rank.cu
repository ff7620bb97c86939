// Low-rank adapters of many requests beside a shared projection: row t with the adapter j = ids[t] gets
//   out[t] = bf16( y[t] + scale[j] * (x[t] . a[j]^T) . b[j]^T ),   a[j]: [rank, in], b[j]: [n_out, rank]
// and a row whose id is outside [0, count) gets out[t] = y[t].
//
// One launch does both products.  A cluster of CTAs takes a unit, up to 16 (64) rows of one adapter: each CTA multiplies its
// part of the input dimension, the cluster adds the parts through its shared memories, in rank order, and each CTA multiplies
// its part of the output columns.  Sums are in fp32; for the second product the scaled low-rank row becomes two bf16 numbers,
// hi + lo (16 bits: with one, its rounding would weigh as much as the output's), two MMAs for one.
// Which rows make up a unit every CTA finds out by itself from the ids: the units of an adapter are its rows in batch order,
// so that the result does not depend on who runs when.  Rows without an adapter are units of their own that are copied.
//
// Two kernels, both bound by memory:
//   few rows (at most 128 a launch): a and b are read once and go straight into the fragments of mma.sync, whose k order is
//     permuted so that a lane's 16 bytes are four k pairs; latency counts, a cluster of eight spreads a unit's adapter.
//   many rows: tiles of 64 rows; x with a, then y with b, come in stages of 64 columns by cp.async, four in flight; out
//     leaves through y's place in shared memory in 16-byte pieces.
#include "internal.h"

namespace imx {

namespace {

constexpr int kMaxRank = 256;
constexpr int kThreads = 256;

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
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
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
__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&v)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(addr) : "memory");
}
// v = hi + lo to 16 bits (what is not finite stays in hi)
__device__ __forceinline__ void split2(float v, __nv_bfloat16& hi, __nv_bfloat16& lo) {
    hi = __float2bfloat16_rn(v);
    const float h = __bfloat162float(hi);
    lo = __float2bfloat16_rn(isfinite(h) ? v - h : 0.f);
}
__device__ __forceinline__ uint32_t pack2(__nv_bfloat16 a, __nv_bfloat16 b) { return (uint32_t)__bfloat16_as_ushort(a) | (uint32_t)__bfloat16_as_ushort(b) << 16; }

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

// ── few rows ────────────────────────────────────────────────────────────────
constexpr int kFewRows = 128;                 // rows of a launch
constexpr int kFewUnit = 16;
// Each lane has a ring of 16-byte pieces in shared memory for what it alone will read, filled by cp.async: in registers there
// is room for two or three pieces on their way (2.6 TB/s).  RB: blocks of 32 values of the rank, 1, 2, 4 or 8.
__host__ __device__ constexpr int ring_pieces(int rb) { return rb == 8 ? 18 : (rb == 4 ? 15 : 12); }
// Dynamic shared memory: the rings, this CTA's sums [row][rank], and in one place the warps' parts of them, [k part][row][rank]
// (8 parts of ranks up to 32, 4 up to 64, 2 up to 128), and afterwards the low-rank rows as hi and lo.
struct FewPlan {
    int pitch, sums_at, part_at, lo_at, bytes;       // pitch: values of a row of hi or lo
    __host__ __device__ FewPlan(int rank, int rb) {
        pitch = rb * 32 + 8;
        sums_at = kThreads * ring_pieces(rb) * 16;
        part_at = sums_at + kFewUnit * rank * 4;
        lo_at = part_at + kFewUnit * pitch * 2;
        const int parts = 8 / rb, a = parts > 1 ? parts * kFewUnit * rank * 4 : 0, b = 2 * kFewUnit * pitch * 2;
        bytes = part_at + (a > b ? a : b);
    }
};

struct FewShared {
    int32_t ids[kFewRows];
    int32_t same[kFewRows];                   // rows before with the same id
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
        s.same[i] = same;
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
template <int RB, int TP>
__global__ void __launch_bounds__(kThreads, RB <= 2 ? 3 : 2)
low_rank_few_kernel(const LowRankArgs p, const int ctas, const int clusters) {
    __shared__ __align__(16) FewShared s;
    extern __shared__ __align__(16) unsigned char dyn[];
    constexpr int kPiece = kThreads * 16;     // bytes between a lane's pieces
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
    const int c = ctas > 1 ? (int)cluster_rank() : 0;
    int id = -1;
    const int cluster = blockIdx.x / ctas, unit = cluster / clusters;
    const int m = find_unit(p, s, unit, id);
    if (m == 0) return;                       // fewer units than clusters: the whole cluster leaves
    // output columns of this CTA, in tiles of eight
    const int tiles = (p.n_out + 7) / 8, part_of = (cluster - unit * clusters) * ctas + c;
    const int t0 = (int)((long)tiles * part_of / (ctas * clusters)), t1 = (int)((long)tiles * (part_of + 1) / (ctas * clusters));
    if (id < 0) {
        if (p.out != p.y)
            for (int r = 0; r < m; ++r) {
                const size_t at = (size_t)s.rows[r] * p.n_out;
                for (int n = t0 * 8 + tid; n < min(t1 * 8, p.n_out); n += kThreads) p.out[at + n] = p.y[at + n];
            }
        return;
    }
    // a lane multiplies the rows g and g + 8 of the unit
    const int row0 = s.rows[min(g, m - 1)], row1 = s.rows[min(g + 8, m - 1)];
    const bool has0 = g < m, has1 = g + 8 < m, more = m > 8;
    const int rank = p.rank;
    const FewPlan pl(rank, RB);
    float* sums = reinterpret_cast<float*>(dyn + pl.sums_at);
    float* parts = reinterpret_cast<float*>(dyn + pl.part_at);
    __nv_bfloat16* hi = reinterpret_cast<__nv_bfloat16*>(dyn + pl.part_at);
    __nv_bfloat16* lo = reinterpret_cast<__nv_bfloat16*>(dyn + pl.lo_at);
    const uint32_t own = smem_addr(dyn) + (uint32_t)tid * 16u;
    const __nv_bfloat16* a = p.a + (size_t)id * rank * p.in;
    const __nv_bfloat16* b = p.b + (size_t)id * p.n_out * rank;

    // x . a^T: a warp takes TP tiles of the rank, every RB-th, and one of 8 / RB parts of the k blocks of 32
    constexpr int kWk = 8 / RB;
    const int wr = warp & (RB - 1), wk = warp / RB, rt = rank / 8;
    float acc[TP][4] = {};
    {
        constexpr int kPieces = TP + 2, kDepth = ring_pieces(RB) / kPieces;
        const int blocks = (p.in + 31) / 32, b0 = blocks * c / ctas, b1 = blocks * (c + 1) / ctas;
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
    const float sc = p.scale != nullptr ? p.scale[id] : 1.f;
    for (int i = tid; i < kFewUnit * RB * 32; i += kThreads) {
        const int r = i / (RB * 32), k = i % (RB * 32);
        float v = 0.f;
        if (r < m && k < rank) {
            const uint32_t at = smem_addr(&sums[r * rank + k]);
            for (int peer = 0; peer < ctas; ++peer) v += ctas > 1 ? ld_peer(peer_addr(at, peer)) : sums[r * rank + k];
            v *= sc;
        }
        split2(v, hi[r * pl.pitch + k], lo[r * pl.pitch + k]);
    }
    if (ctas > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");     // this CTA has read the others' sums
    __syncthreads();

    // + t . b^T
    const uint4* h0 = reinterpret_cast<const uint4*>(hi + g * pl.pitch + q * 8);
    const uint4* h1 = reinterpret_cast<const uint4*>(hi + (g + 8) * pl.pitch + q * 8);
    const uint4* l0 = reinterpret_cast<const uint4*>(lo + g * pl.pitch + q * 8);
    const uint4* l1 = reinterpret_cast<const uint4*>(lo + (g + 8) * pl.pitch + q * 8);
    constexpr int kKept = RB <= 2 ? RB : 1;   // up to a rank of 64 the low-rank rows stay in registers
    uint4 vh0[kKept], vh1[kKept], vl0[kKept], vl1[kKept];
#pragma unroll
    for (int kb = 0; kb < kKept; ++kb) {
        vh0[kb] = h0[kb * 4];
        vh1[kb] = h1[kb * 4];
        vl0[kb] = l0[kb * 4];
        vl1[kb] = l1[kb * 4];
    }
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
            const int i0 = RB <= 2 ? kb : 0;
            if (RB > 2) {
                vh0[0] = h0[kb * 4];
                vh1[0] = h1[kb * 4];
                vl0[0] = l0[kb * 4];
                vl1[0] = l1[kb * 4];
            }
            mma(d, vh0[i0].x, vh1[i0].x, vh0[i0].y, vh1[i0].y, w.x, w.y);
            mma(e, vl0[i0].x, vl1[i0].x, vl0[i0].y, vl1[i0].y, w.x, w.y);
            mma(d, vh0[i0].z, vh1[i0].z, vh0[i0].w, vh1[i0].w, w.z, w.w);
            mma(e, vl0[i0].z, vl1[i0].z, vl0[i0].w, vl1[i0].w, w.z, w.w);
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
// Stages of columns in shared memory: what fits with two CTAs on an SM (one from a rank of 65 on).
__host__ __device__ constexpr int tile_stages(int rank) { return rank > 128 ? 2 : (rank > 32 ? 4 : 6); }
constexpr int kMaxBins = 2048;                // adapters + 1
constexpr int kBlockRows = 8192;              // rows of a launch: each CTA looks through all their ids
constexpr int kColPitch = (kCols / 8 + 1) * 16;   // bytes; an odd number of 16-byte pieces: eight rows meet no bank twice

struct TileShared {
    int32_t rows[kTileRows];
    int32_t warp_count[8];
    int32_t n_rows, id, first;
};

// Offsets in the dynamic shared memory.
struct TilePlan {
    int r16, pitch;                           // rank rounded up to 16; bytes of a row of it
    int stage, sums_at, hi_at, lo_at, bytes;
    __host__ __device__ explicit TilePlan(int rank) {
        r16 = (rank + 15) & ~15;
        pitch = ((r16 / 8) | 1) * 16;
        const int first = (kTileRows + r16) * kColPitch, second = kTileRows * kColPitch + kCols * pitch;
        stage = first > second ? first : second;
        sums_at = tile_stages(rank) * stage;
        hi_at = sums_at + kTileRows * r16 * 4;
        lo_at = hi_at + kTileRows * pitch;
        bytes = lo_at + kTileRows * pitch;
    }
};

// NJ: tiles of 16 values of the rank that a warp multiplies (rank up to 32 NJ).
template <int NJ>
__global__ void __launch_bounds__(kThreads, NJ <= 2 ? 2 : 1)
low_rank_tile_kernel(const LowRankArgs p, const int ctas) {
    constexpr int kTileStages = tile_stages(32 * NJ);
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ TileShared s;
    const TilePlan pl(p.rank);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int unit = blockIdx.x / ctas, c = ctas > 1 ? (int)cluster_rank() : 0;
    // Units of this block of rows: adapter 0's rows in tiles of 64, adapter 1's, ..., at last the rows without one.  A warp
    // has an eighth of the ids, 32 at a time in batch order, all of them in registers: as loads of the loops below, one after
    // the other, they took 22 us.
    int32_t* bins = reinterpret_cast<int32_t*>(smem);
    const int n_bins = p.count + 1;
    constexpr int kIds = kBlockRows / kThreads;
    const int groups = (p.n + kThreads - 1) / kThreads, from = warp * groups * 32;
    int bin[kIds];
#pragma unroll
    for (int i = 0; i < kIds; ++i) {
        const int r = from + i * 32 + lane;
        bin[i] = i < groups && r < p.n ? p.ids[r] : -1;
        if (i < groups && r < p.n && (bin[i] < 0 || bin[i] >= p.count)) bin[i] = p.count;
    }
    for (int i = tid; i < n_bins; i += kThreads) bins[i] = 0;
    if (tid == 0) s.n_rows = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kIds; ++i) {
        if (i >= groups) break;
        const unsigned alike = __match_any_sync(0xffffffffu, bin[i]);
        if (bin[i] >= 0 && lane == __ffs(alike) - 1) atomicAdd(&bins[bin[i]], __popc(alike));
    }
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
    if (m == 0) return;
    {
        // the unit's rows: those of the bin from the skip-th on, in batch order
        int n = 0;
#pragma unroll
        for (int i = 0; i < kIds; ++i) n += __popc(__ballot_sync(0xffffffffu, bin[i] == id));
        if (lane == 0) s.warp_count[warp] = n;
        __syncthreads();
        n = -skip;
        for (int w = 0; w < warp; ++w) n += s.warp_count[w];
#pragma unroll
        for (int i = 0; i < kIds; ++i) {
            const unsigned hit = __ballot_sync(0xffffffffu, bin[i] == id);
            const int at = n + __popc(hit & ((1u << lane) - 1u));
            if ((hit >> lane & 1u) && at >= 0 && at < m) s.rows[at] = from + i * 32 + lane;
            n += __popc(hit);
        }
    }
    __syncthreads();
    // chunks of the input and of the output dimension that this CTA takes
    const int ik = (p.in + kCols - 1) / kCols, on = (p.n_out + kCols - 1) / kCols;
    const int k0 = ik * c / ctas, k1 = ik * (c + 1) / ctas, n0 = on * c / ctas, n1 = on * (c + 1) / ctas;
    if (id == p.count) {
        if (p.out != p.y)
            for (int r = warp; r < m; r += 8) {
                const size_t at = (size_t)s.rows[r] * p.n_out;
                const int end = min(n1 * kCols, p.n_out);
                if (p.wide)
                    for (int n = n0 * kCols + lane * 8; n < end; n += 256) *reinterpret_cast<uint4*>(p.out + at + n) = *reinterpret_cast<const uint4*>(p.y + at + n);
                else
                    for (int n = n0 * kCols + lane; n < end; n += 32) p.out[at + n] = p.y[at + n];
            }
        return;
    }
    const int rank = p.rank, r16 = pl.r16;
    const __nv_bfloat16* a = p.a + (size_t)id * rank * p.in;
    const __nv_bfloat16* b = p.b + (size_t)id * p.n_out * rank;
    const uint32_t base = smem_addr(smem);
    // What a thread copies is the same in every stage but for the columns: of x and y a piece of two rows, of a and b NJ pieces.
    const int cr = tid >> 3, cc = (tid & 7) * 8;
    const __nv_bfloat16* xr[2];
    const __nv_bfloat16* yr[2];
    bool has[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        has[i] = cr + 32 * i < m;
        const size_t row = s.rows[has[i] ? cr + 32 * i : 0];
        xr[i] = p.x + row * p.in + cc;
        yr[i] = p.y + row * p.n_out + cc;
    }
    const int pieces = r16 / 8;
    int b_left[NJ], b_to[NJ];                 // rows of b up to the end (0: zeros, below: nothing), and where the piece goes
    const __nv_bfloat16* b_from[NJ];
#pragma unroll
    for (int i = 0; i < NJ; ++i) {
        const int e = tid + i * kThreads, r = e / pieces, j = e - r * pieces;
        b_left[i] = r < kCols ? (j * 8 < rank ? p.n_out - n0 * kCols - r : 0) : -(1 << 30);
        b_from[i] = b + (size_t)(n0 * kCols + r) * rank + j * 8;
        b_to[i] = kTileRows * kColPitch + r * pl.pitch + j * 16;
    }
    const uint32_t own = base + cr * kColPitch + cc * 2;
    int in_left = p.in - k0 * kCols - cc, out_left = p.n_out - n0 * kCols - cc;      // columns of x and of y up to the end
    const __nv_bfloat16* a_from = a + (size_t)cr * p.in + k0 * kCols + cc;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        xr[i] += k0 * kCols;
        yr[i] += n0 * kCols;
    }
    // the next stage of the first product: 64 rows of x and the rank's rows of a, 64 columns each
    auto load_in = [&](uint32_t st) {
        const bool in = in_left > 0;
#pragma unroll
        for (int i = 0; i < 2; ++i) copy16(own + st + i * 32 * kColPitch, in && has[i] ? xr[i] : p.x, in && has[i]);
#pragma unroll
        for (int i = 0; i < NJ; ++i)
            if (cr + 32 * i < r16) {
                const bool there = in && cr + 32 * i < rank;
                copy16(own + st + (kTileRows + 32 * i) * kColPitch, there ? a_from + (size_t)(32 * i) * p.in : a, there);
            }
        in_left -= kCols;
        a_from += kCols;
        xr[0] += kCols;
        xr[1] += kCols;
    };
    // ... of the second: 64 rows of y (where they are whole pieces) and 64 of b
    auto load_out = [&](uint32_t st) {
        if (p.wide) {
            const bool in = out_left > 0;
#pragma unroll
            for (int i = 0; i < 2; ++i) copy16(own + st + i * 32 * kColPitch, in && has[i] ? yr[i] : p.y, in && has[i]);
        }
#pragma unroll
        for (int i = 0; i < NJ; ++i) {
            if (b_left[i] > -(1 << 29)) copy16(base + st + b_to[i], b_left[i] > 0 ? b_from[i] : b, b_left[i] > 0);
            b_left[i] -= kCols;
            b_from[i] += kCols * rank;
        }
        out_left -= kCols;
        yr[0] += kCols;
        yr[1] += kCols;
    };
    const int rt = warp & 3, half = warp >> 2;     // the warp's 16 rows, and its half of the rank's or the columns' tiles
    // (ldmatrix: lanes 0..15 give the rows of the first eight columns, 16..31 those of the next)
    const int lr = lane & 15, lc = (lane >> 4) * 16;
    const int total = (k1 - k0) + (n1 - n0);       // both products' stages in one line
    const uint32_t ring = (uint32_t)(kTileStages * pl.stage);
    int loaded = 0;
    uint32_t to_stage = 0, at_stage = 0;           // offsets of the stage to fill next and of the one to use next
    auto load = [&]() {
        if (loaded < k1 - k0) load_in(to_stage);
        else if (loaded < total) load_out(to_stage);
        copies_commit();
        ++loaded;
        to_stage += pl.stage;
        if (to_stage == ring) to_stage = 0;
    };
    auto next_stage = [&]() {
        at_stage += pl.stage;
        if (at_stage == ring) at_stage = 0;
    };
    for (int i = 0; i < kTileStages - 1; ++i) load();
    float acc[NJ][8] = {};
    int it = 0;
    for (; it < k1 - k0; ++it) {
        copies_wait<kTileStages - 2>();
        __syncthreads();
        load();
        const uint32_t xs = base + at_stage, as = xs + kTileRows * kColPitch;
        next_stage();
#pragma unroll
        for (int kk = 0; kk < kCols / 16; ++kk) {
            uint32_t va[4];
            ldmatrix4(xs + (rt * 16 + lr) * kColPitch + kk * 32 + lc, va);
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const int t = half + 2 * j;
                if (t * 16 >= r16) break;
                uint32_t vb[4];
                ldmatrix4(as + (t * 16 + lr) * kColPitch + kk * 32 + lc, vb);
                float(&d0)[4] = *reinterpret_cast<float(*)[4]>(&acc[j][0]);
                float(&d1)[4] = *reinterpret_cast<float(*)[4]>(&acc[j][4]);
                mma(d0, va[0], va[1], va[2], va[3], vb[0], vb[2]);
                mma(d1, va[0], va[1], va[2], va[3], vb[1], vb[3]);
            }
        }
    }
    // the low-rank rows: this CTA's part of the sums, then all of them as hi + lo in every CTA
    const int g = lane >> 2, q = lane & 3;
    float* sums = reinterpret_cast<float*>(smem + pl.sums_at);
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
        const int t = half + 2 * j;
        if (t * 16 >= r16) break;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float* d = sums + (rt * 16 + g) * r16 + t * 16 + h * 8 + 2 * q;
            *reinterpret_cast<float2*>(d) = make_float2(acc[j][4 * h], acc[j][4 * h + 1]);
            *reinterpret_cast<float2*>(d + 8 * r16) = make_float2(acc[j][4 * h + 2], acc[j][4 * h + 3]);
        }
    }
    if (ctas > 1) cluster_sync();
    else __syncthreads();
    const float sc = p.scale != nullptr ? p.scale[id] : 1.f;
    for (int i = tid * ctas + c; i < kTileRows * pieces; i += kThreads * ctas) {
        const int r = i / pieces, j = i - r * pieces;
        float v[8] = {};
        const uint32_t at = base + pl.sums_at + (uint32_t)(r * r16 + j * 8) * 4u;
        for (int peer = 0; peer < ctas; ++peer) {
            const uint32_t from = ctas > 1 ? peer_addr(at, peer) : at;
            const float4 u = ld_peer4(from), w = ld_peer4(from + 16);
            v[0] += u.x; v[1] += u.y; v[2] += u.z; v[3] += u.w;
            v[4] += w.x; v[5] += w.y; v[6] += w.z; v[7] += w.w;
        }
        __nv_bfloat16 hi[8], lo[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) split2(v[e] * sc, hi[e], lo[e]);
        const uint4 vh = make_uint4(pack2(hi[0], hi[1]), pack2(hi[2], hi[3]), pack2(hi[4], hi[5]), pack2(hi[6], hi[7]));
        const uint4 vl = make_uint4(pack2(lo[0], lo[1]), pack2(lo[2], lo[3]), pack2(lo[4], lo[5]), pack2(lo[6], lo[7]));
        const uint32_t to = base + (uint32_t)(r * pl.pitch + j * 16);
        for (int peer = 0; peer < ctas; ++peer) {
            const uint32_t dst = ctas > 1 ? peer_addr(to, peer) : to;
            st_peer4(dst + pl.hi_at, vh);
            st_peer4(dst + pl.lo_at, vl);
        }
    }
    if (ctas > 1) cluster_sync();
    else __syncthreads();
    // up to a rank of 64 the low-rank rows stay in registers
    constexpr int kKept = NJ <= 2 ? 2 * NJ : 0;
    uint32_t kh[kKept > 0 ? kKept : 1][4], kl[kKept > 0 ? kKept : 1][4];
    const uint32_t hi_own = base + pl.hi_at + (rt * 16 + lr) * pl.pitch + lc, lo_own = hi_own + pl.lo_at - pl.hi_at;
#pragma unroll
    for (int kk = 0; kk < kKept; ++kk)
        if (kk * 16 < r16) {
            ldmatrix4(hi_own + kk * 32, kh[kk]);
            ldmatrix4(lo_own + kk * 32, kl[kk]);
        }
    __nv_bfloat16* to_own[2];
    bool has_own[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = rt * 16 + (lane >> 2) + 8 * i;
        has_own[i] = r < m;
        to_own[i] = p.out + (size_t)s.rows[has_own[i] ? r : 0] * p.n_out + n0 * kCols + half * 32 + (lane & 3) * 8;
    }
    int n = n0 * kCols;                            // first column of the stage
    for (; it < total; ++it) {
        copies_wait<kTileStages - 2>();
        __syncthreads();
        load();
        unsigned char* ys_p = smem + at_stage;
        next_stage();
        const uint32_t bs = smem_addr(ys_p) + kTileRows * kColPitch + (half * 32 + lr) * pl.pitch + lc;
        float d[4][4] = {};                   // four tiles of eight columns of the warp's 32
        auto step = [&](const uint32_t (&vh)[4], const uint32_t (&vl)[4], int kk) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                uint32_t vb[4];
                ldmatrix4(bs + j * 16 * pl.pitch + kk * 32, vb);
                mma(d[2 * j], vh[0], vh[1], vh[2], vh[3], vb[0], vb[2]);
                mma(d[2 * j + 1], vh[0], vh[1], vh[2], vh[3], vb[1], vb[3]);
                mma(d[2 * j], vl[0], vl[1], vl[2], vl[3], vb[0], vb[2]);
                mma(d[2 * j + 1], vl[0], vl[1], vl[2], vl[3], vb[1], vb[3]);
            }
        };
        if (kKept > 0) {
#pragma unroll
            for (int kk = 0; kk < kKept; ++kk)
                if (kk * 16 < r16) step(kh[kk], kl[kk], kk);
        } else {
#pragma unroll 2
            for (int kk = 0; kk < r16 / 16; ++kk) {
                uint32_t vh[4], vl[4];
                ldmatrix4(hi_own + kk * 32, vh);
                ldmatrix4(lo_own + kk * 32, vl);
                step(vh, vl, kk);
            }
        }
        if (p.wide) {
            // added in y's place, out in 16-byte pieces: 16 rows x 32 columns that no other warp touches
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    __nv_bfloat162* at = reinterpret_cast<__nv_bfloat162*>(ys_p + (rt * 16 + g + 8 * h) * kColPitch + (half * 32 + j * 8 + 2 * q) * 2);
                    const float2 v = __bfloat1622float2(*at);
                    *at = __floats2bfloat162_rn(v.x + d[j][2 * h], v.y + d[j][2 * h + 1]);
                }
            __syncwarp();
            const int r0 = rt * 16 + (lane >> 2), col = half * 32 + (lane & 3) * 8;
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (has_own[i] && n + col < p.n_out)
                    *reinterpret_cast<uint4*>(to_own[i]) = *reinterpret_cast<const uint4*>(ys_p + (r0 + 8 * i) * kColPitch + col * 2);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = rt * 16 + g + 8 * (e >> 1), col = n + half * 32 + j * 8 + 2 * q + (e & 1);
                    if (r < m && col < p.n_out) {
                        const size_t at = (size_t)s.rows[r] * p.n_out + col;
                        p.out[at] = __float2bfloat16_rn(__bfloat162float(p.y[at]) + d[j][e]);
                    }
                }
        }
        n += kCols;
        to_own[0] += kCols;
        to_own[1] += kCols;
    }
    copies_wait<0>();
}

int launch_clusters(const void* kernel, unsigned grid, int ctas, size_t smem, cudaStream_t stream, void** args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(kThreads);
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

int launch_low_rank(LowRankArgs p, int sms, cudaStream_t stream) {
    const int rows = p.n, step = rows <= kFewRows || p.count >= kMaxBins ? kFewRows : kBlockRows;
    const LowRankArgs whole = p;
    for (int r0 = 0; r0 < rows; r0 += step) {
        p.n = rows - r0 < step ? rows - r0 : step;
        p.x = whole.x + (size_t)r0 * p.in;
        p.y = whole.y + (size_t)r0 * p.n_out;
        p.out = whole.out + (size_t)r0 * p.n_out;
        p.ids = whole.ids + r0;
        int ctas = 1;
        void* args[] = {&p, &ctas, nullptr};
        if (step == kFewRows) {
            const FewKernel few = few_kernel(p.rank);
            while (ctas < 8 && p.n * ctas * 2 <= (few.rb <= 2 ? 3 : 2) * sms) ctas *= 2;
            int clusters = 1;
            while (clusters < 16 && p.n * ctas * clusters * 2 <= sms && p.n_out >= 128 * ctas * clusters) clusters *= 2;
            args[2] = &clusters;
            IMX_TRY(launch_clusters(few.kernel, (unsigned)(p.n * ctas * clusters), ctas, (size_t)FewPlan(p.rank, few.rb).bytes, stream, args));
            continue;
        }
        // no more units than these; CTAs for two on every SM
        const int units = p.n / kTileRows + (p.count + 1 < p.n ? p.count + 1 : p.n);
        while (ctas < 8 && units * ctas * 2 <= 2 * sms) ctas *= 2;
        const void* kernel = p.rank <= 32 ? (const void*)low_rank_tile_kernel<1> : (p.rank <= 64 ? (const void*)low_rank_tile_kernel<2>
                                          : (p.rank <= 128 ? (const void*)low_rank_tile_kernel<4> : (const void*)low_rank_tile_kernel<8>));
        IMX_TRY(launch_clusters(kernel, (unsigned)(units * ctas), ctas, (size_t)TilePlan(p.rank).bytes, stream, args));
    }
    return IMX_OK;
}

}  // namespace

}  // namespace imx

using namespace imx;

extern "C" int imx_low_rank_add(const void* y, const void* x, int n_rows, int in, const imx_adapters* ad, const int32_t* ids, int n_out,
                                void* out, void* stream) {
    IMX_REQUIRE(n_rows >= 0 && n_out > 0 && in > 0 && in % 8 == 0,
                "low_rank_add: sizes (%d rows, %d -> %d) must be positive, the input dimension a multiple of 8", n_rows, in, n_out);
    if (n_rows == 0) return IMX_OK;
    IMX_REQUIRE(y && x && ad && ids && out, "low_rank_add: y, x, adapters, ids and out are required");
    IMX_REQUIRE(ad->a && ad->b && ad->count > 0, "low_rank_add: at least one adapter is required");
    IMX_REQUIRE(ad->rank > 0 && ad->rank % 8 == 0 && ad->rank <= kMaxRank,
                "low_rank_add: the rank (%d) must be a multiple of 8, at most %d", ad->rank, kMaxRank);
    IMX_REQUIRE((((uintptr_t)x | (uintptr_t)ad->a | (uintptr_t)ad->b) % 16) == 0, "low_rank_add: x, a and b must be 16-byte aligned");
    IMX_REQUIRE((((uintptr_t)ids | (uintptr_t)ad->scale) % 4) == 0, "low_rank_add: ids and scale must be aligned to their values");
    IMX_REQUIRE((((uintptr_t)y | (uintptr_t)out) % 2) == 0, "low_rank_add: y and out must be aligned to their bf16 values");
    const size_t ob = (size_t)n_rows * n_out * 2;
    IMX_REQUIRE(out == y || !overlap(out, ob, y, ob), "low_rank_add: out overlaps y without being it");
    IMX_REQUIRE(!overlap(out, ob, x, (size_t)n_rows * in * 2) && !overlap(out, ob, ids, (size_t)n_rows * 4) &&
                !overlap(out, ob, ad->a, (size_t)ad->count * ad->rank * in * 2) &&
                !overlap(out, ob, ad->b, (size_t)ad->count * ad->rank * n_out * 2) &&
                !overlap(out, ob, ad->scale, (size_t)ad->count * 4), "low_rank_add: out overlaps another array");
    DeviceInfo di;
    IMX_TRY(current_device(&di));
    if (device_needs_setup(di.ordinal, kSetupLowRank)) {     // once per device
        const void* kernels[4] = {(const void*)low_rank_tile_kernel<1>, (const void*)low_rank_tile_kernel<2>, (const void*)low_rank_tile_kernel<4>,
                                  (const void*)low_rank_tile_kernel<8>};
        for (int i = 0; i < 4; ++i) IMX_CHECK_CUDA(cudaFuncSetAttribute(kernels[i], cudaFuncAttributeMaxDynamicSharedMemorySize, TilePlan(32 << i).bytes));
        for (int rank : {8, 16, 32, 64, 128, 256}) {
            const FewKernel few = few_kernel(rank);
            IMX_CHECK_CUDA(cudaFuncSetAttribute(few.kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, FewPlan(rank, few.rb).bytes));
        }
        device_mark_setup(di.ordinal, kSetupLowRank);
    }
    const int wide = n_out % 8 == 0 && (((uintptr_t)y | (uintptr_t)out) % 16) == 0;
    return launch_low_rank(LowRankArgs{(const __nv_bfloat16*)y, (const __nv_bfloat16*)x, (const __nv_bfloat16*)ad->a, (const __nv_bfloat16*)ad->b,
                                       ad->scale, ids, (__nv_bfloat16*)out, n_rows, in, n_out, ad->count, ad->rank, wide},
                           di.sms, (cudaStream_t)stream);
}
