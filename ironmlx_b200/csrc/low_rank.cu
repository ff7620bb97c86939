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
__device__ __forceinline__ uint4 ldg16(const __nv_bfloat16* p) { return __ldg(reinterpret_cast<const uint4*>(p)); }
// v = hi + lo to 16 bits (what is not finite stays in hi)
__device__ __forceinline__ void split2(float v, __nv_bfloat16& hi, __nv_bfloat16& lo) {
    hi = __float2bfloat16_rn(v);
    const float h = __bfloat162float(hi);
    lo = __float2bfloat16_rn(isfinite(h) ? v - h : 0.f);
}
__device__ __forceinline__ uint32_t pack2(__nv_bfloat16 a, __nv_bfloat16 b) { return (uint32_t)__bfloat16_as_ushort(a) | (uint32_t)__bfloat16_as_ushort(b) << 16; }

// ── few rows ────────────────────────────────────────────────────────────────
constexpr int kFewRows = 128;                 // rows of a launch
constexpr int kFewUnit = 16;
constexpr int kFewCtas = 8;                   // CTAs of a cluster

struct FewShared {
    int32_t ids[kFewRows];
    int32_t rows[kFewUnit];
    int32_t n_rows, id;
    float part[2048];                         // [k part][row][rank] of the warps: 8 parts of up to 8, 4 of 24, 2 of 56
    float sum[kFewUnit * kMaxRank];           // [row][rank] of this CTA's part of the input dimension
    __align__(16) __nv_bfloat16 hi[kFewUnit][kMaxRank + 8], lo[kFewUnit][kMaxRank + 8];
};

__global__ void __launch_bounds__(kThreads)
low_rank_few_kernel(const LowRankArgs p) {
    __shared__ FewShared s;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q = lane & 3;
    const int unit = blockIdx.x / kFewCtas, c = (int)cluster_rank();
    // Row i leads a unit if a multiple of 16 rows before it have its id; units are numbered in the order of their leaders.
    if (tid < kFewRows) {
        const int id = tid < p.n ? p.ids[tid] : -1;
        s.ids[tid] = id >= 0 && id < p.count ? id : -1;
    }
    if (tid == 0) s.n_rows = 0;
    __syncthreads();
    if (warp == 0) {
        int before = 0;
        bool found = false;
        for (int base = 0; base < p.n && !found; base += 32) {
            const int i = base + lane, id = s.ids[i];
            int same = 0;
            for (int j = 0; j < base; j += 4) {
                const int4 v = *reinterpret_cast<const int4*>(&s.ids[j]);
                same += (v.x == id) + (v.y == id) + (v.z == id) + (v.w == id);
            }
            const unsigned alike = __match_any_sync(0xffffffffu, i < p.n ? id : -2 - lane);
            same += __popc(alike & ((1u << lane) - 1u));
            const unsigned leads = __ballot_sync(0xffffffffu, i < p.n && same % kFewUnit == 0);
            const int here = unit - before;
            if (here < __popc(leads)) {
                // the unit's leader is the here-th set bit; its rows are it and the next 15 with its id
                unsigned m = leads;
                for (int k = 0; k < here; ++k) m &= m - 1;
                const int src = __ffs(m) - 1, leader = base + src, lead_id = __shfl_sync(0xffffffffu, id, src);
                int n = 0;
                for (int b2 = leader & ~31; b2 < p.n && n < kFewUnit; b2 += 32) {
                    const int r = b2 + lane;
                    const unsigned hit = __ballot_sync(0xffffffffu, r >= leader && r < p.n && s.ids[r] == lead_id);
                    const int at = n + __popc(hit & ((1u << lane) - 1u));
                    if ((hit >> lane & 1u) && at < kFewUnit) s.rows[at] = r;
                    n += __popc(hit);
                }
                if (lane == 0) {
                    s.n_rows = min(n, kFewUnit);
                    s.id = lead_id;
                }
                found = true;
            }
            before += __popc(leads);
        }
    }
    __syncthreads();
    const int m = s.n_rows, id = s.id;
    if (m == 0) return;                       // fewer units than clusters: the whole cluster leaves
    // output columns of this CTA, in tiles of eight
    const int tiles = (p.n_out + 7) / 8, t0 = tiles * c / kFewCtas, t1 = tiles * (c + 1) / kFewCtas;
    if (id < 0) {
        if (p.out != p.y)
            for (int r = 0; r < m; ++r) {
                const size_t at = (size_t)s.rows[r] * p.n_out;
                for (int n = t0 * 8 + tid; n < min(t1 * 8, p.n_out); n += kThreads) p.out[at + n] = p.y[at + n];
            }
        return;
    }
    const int rank = p.rank, rt = rank / 8;   // rank in tiles of eight
    const __nv_bfloat16* a = p.a + (size_t)id * rank * p.in;
    const __nv_bfloat16* b = p.b + (size_t)id * p.n_out * rank;
    const uint4 zero = make_uint4(0, 0, 0, 0);

    // x . a^T: warps over tiles of the rank (up to four each) and over k
    const int lg_wr = rt >= 8 ? 3 : (rt >= 4 ? 2 : (rt >= 2 ? 1 : 0)), wr = warp & ((1 << lg_wr) - 1), wk = warp >> lg_wr, n_wk = 8 >> lg_wr;
    const int blocks = (p.in + 31) / 32, b0 = blocks * c / kFewCtas, b1 = blocks * (c + 1) / kFewCtas;
    float acc[4][4] = {};
    {
        const __nv_bfloat16* x0 = p.x + (size_t)s.rows[min(g, m - 1)] * p.in;
        const __nv_bfloat16* x1 = p.x + (size_t)s.rows[min(g + 8, m - 1)] * p.in;
#pragma unroll 2
        for (int kb = b0 + wk; kb < b1; kb += n_wk) {
            const int k = kb * 32 + q * 8;
            const bool in = k < p.in;
            const uint4 v0 = in && g < m ? ldg16(x0 + k) : zero, v1 = in && g + 8 < m ? ldg16(x1 + k) : zero;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int t = wr + (i << lg_wr);
                if (t >= rt) break;
                const uint4 w = in ? ldg16(a + (size_t)(t * 8 + g) * p.in + k) : zero;
                mma(acc[i], v0.x, v1.x, v0.y, v1.y, w.x, w.y);
                mma(acc[i], v0.z, v1.z, v0.w, v1.w, w.z, w.w);
            }
        }
    }
    const int pitch = n_wk > 1 ? rt * 8 : 0;  // (with one part the warps' tiles are the sums)
    float* part = n_wk > 1 ? s.part + wk * kFewUnit * pitch : s.sum;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int t = wr + (i << lg_wr);
        if (t >= rt) break;
        float* d = part + t * 8 + 2 * q;
        d[g * rank] = acc[i][0];
        d[g * rank + 1] = acc[i][1];
        d[(g + 8) * rank] = acc[i][2];
        d[(g + 8) * rank + 1] = acc[i][3];
    }
    __syncthreads();
    if (n_wk > 1) {
        for (int i = tid; i < m * rank; i += kThreads) {
            float v = 0.f;
            for (int k = 0; k < n_wk; ++k) v += s.part[k * kFewUnit * pitch + i];
            s.sum[i] = v;
        }
    }
    cluster_sync();
    const float sc = p.scale != nullptr ? p.scale[id] : 1.f;
    const int blocks_r = (rank + 31) / 32;
    for (int i = tid; i < kFewUnit * blocks_r * 32; i += kThreads) {
        const int r = i / (blocks_r * 32), k = i - r * blocks_r * 32;
        float v = 0.f;
        if (r < m && k < rank) {
            const uint32_t at = smem_addr(&s.sum[r * rank + k]);
#pragma unroll
            for (int peer = 0; peer < kFewCtas; ++peer) v += ld_peer(peer_addr(at, peer));
            v *= sc;
        }
        split2(v, s.hi[r][k], s.lo[r][k]);
    }
    __syncthreads();

    // + t . b^T
    const bool pairs = p.n_out % 2 == 0 && (((uintptr_t)p.y | (uintptr_t)p.out) % 4) == 0;
    const size_t at0 = (size_t)s.rows[min(g, m - 1)] * p.n_out, at1 = (size_t)s.rows[min(g + 8, m - 1)] * p.n_out;
    const uint4* h0 = reinterpret_cast<const uint4*>(&s.hi[g][q * 8]);
    const uint4* h1 = reinterpret_cast<const uint4*>(&s.hi[g + 8][q * 8]);
    const uint4* l0 = reinterpret_cast<const uint4*>(&s.lo[g][q * 8]);
    const uint4* l1 = reinterpret_cast<const uint4*>(&s.lo[g + 8][q * 8]);
#pragma unroll 4
    for (int t = t0 + warp; t < t1; t += 8) {
        float d[4] = {0.f, 0.f, 0.f, 0.f};
        const __nv_bfloat16* br = b + (size_t)(t * 8 + g) * rank + q * 8;
        for (int kb = 0; kb < blocks_r; ++kb) {
            const uint4 w = t * 8 + g < p.n_out && kb * 32 + q * 8 < rank ? ldg16(br + kb * 32) : zero;
            const uint4 vh0 = h0[kb * 4], vh1 = h1[kb * 4], vl0 = l0[kb * 4], vl1 = l1[kb * 4];
            mma(d, vh0.x, vh1.x, vh0.y, vh1.y, w.x, w.y);
            mma(d, vh0.z, vh1.z, vh0.w, vh1.w, w.z, w.w);
            mma(d, vl0.x, vl1.x, vl0.y, vl1.y, w.x, w.y);
            mma(d, vl0.z, vl1.z, vl0.w, vl1.w, w.z, w.w);
        }
        const int n = t * 8 + 2 * q;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (g + 8 * h >= m || n >= p.n_out) continue;
            const size_t at = (h ? at1 : at0) + n;
            if (pairs) {
                const float2 v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(p.y + at));
                *reinterpret_cast<__nv_bfloat162*>(p.out + at) = __floats2bfloat162_rn(v.x + d[2 * h], v.y + d[2 * h + 1]);
            } else {
                p.out[at] = __float2bfloat16_rn(__bfloat162float(p.y[at]) + d[2 * h]);
                if (n + 1 < p.n_out) p.out[at + 1] = __float2bfloat16_rn(__bfloat162float(p.y[at + 1]) + d[2 * h + 1]);
            }
        }
    }
    cluster_sync();                           // the others have read this CTA's sums
}

// ── many rows ───────────────────────────────────────────────────────────────
constexpr int kTileRows = 64;
constexpr int kCols = 64;                     // columns of a stage, of the input first, then of the output
__host__ __device__ constexpr int tile_stages(int rank) { return rank > 128 ? 2 : 4; }
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
    int stage, stages_at, sums_at, hi_at, lo_at, bytes;
    __host__ __device__ explicit TilePlan(int rank) {
        r16 = (rank + 15) & ~15;
        pitch = ((r16 / 8) | 1) * 16;
        const int first = (kTileRows + r16) * kColPitch, second = kTileRows * kColPitch + kCols * pitch;
        stage = first > second ? first : second;
        stages_at = 0;
        sums_at = tile_stages(rank) * stage;
        hi_at = sums_at + kTileRows * r16 * 4;
        lo_at = hi_at + kTileRows * pitch;
        bytes = lo_at + kTileRows * pitch;
    }
};

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {
    const int n = there ? 16 : 0;             // the rest is filled with zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

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
    // Units of this block of rows: adapter 0's rows in tiles of 64, adapter 1's, ..., at last the rows without one.
    int32_t* bins = reinterpret_cast<int32_t*>(smem);
    const int n_bins = p.count + 1;
    for (int i = tid; i < n_bins; i += kThreads) bins[i] = 0;
    if (tid == 0) s.n_rows = 0;
    __syncthreads();
    auto bin_of = [&](int i) {
        const int id = p.ids[i];
        return id >= 0 && id < p.count ? id : p.count;
    };
    for (int i = tid; i < ((p.n + 31) & ~31); i += kThreads) {
        const int bin = i < p.n ? bin_of(i) : -1;
        const unsigned alike = __match_any_sync(0xffffffffu, bin);
        if (bin >= 0 && lane == __ffs(alike) - 1) atomicAdd(&bins[bin], __popc(alike));
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
        // the unit's rows: those of the bin from the skip-th on, in batch order; a warp looks through an eighth
        const int per = ((p.n + 255) / 256) * 32, from = warp * per, to = min(from + per, p.n);
        int n = 0;
        for (int base = from; base < to; base += 32) n += __popc(__ballot_sync(0xffffffffu, base + lane < to && bin_of(base + lane) == id));
        if (lane == 0) s.warp_count[warp] = n;
        __syncthreads();
        n = -skip;
        for (int w = 0; w < warp; ++w) n += s.warp_count[w];
        for (int base = from; base < to && n < m; base += 32) {
            const unsigned hit = __ballot_sync(0xffffffffu, base + lane < to && bin_of(base + lane) == id);
            const int at = n + __popc(hit & ((1u << lane) - 1u));
            if ((hit >> lane & 1u) && at >= 0 && at < m) s.rows[at] = base + lane;
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
    // a stage of the first product: 64 rows of x and the rank's rows of a, 64 columns each
    auto load_in = [&](int k, int st) {
        const uint32_t xs = base + pl.stages_at + st * pl.stage, as = xs + kTileRows * kColPitch;
        for (int i = tid; i < kTileRows * 8; i += kThreads) {
            const int r = i >> 3, col = k * kCols + (i & 7) * 8;
            const bool there = r < m && col < p.in;
            copy16(xs + r * kColPitch + (i & 7) * 16, there ? p.x + (size_t)s.rows[r] * p.in + col : p.x, there);
        }
        for (int i = tid; i < r16 * 8; i += kThreads) {
            const int r = i >> 3, col = k * kCols + (i & 7) * 8;
            const bool there = r < rank && col < p.in;
            copy16(as + r * kColPitch + (i & 7) * 16, there ? a + (size_t)r * p.in + col : a, there);
        }
    };
    // ... of the second: 64 rows of y (where they are whole pieces) and 64 of b
    const int pieces = r16 / 8;
    auto load_out = [&](int n, int st) {
        const uint32_t ys = base + pl.stages_at + st * pl.stage, bs = ys + kTileRows * kColPitch;
        if (p.wide)
            for (int i = tid; i < kTileRows * 8; i += kThreads) {
                const int r = i >> 3, col = n * kCols + (i & 7) * 8;
                const bool there = r < m && col < p.n_out;
                copy16(ys + r * kColPitch + (i & 7) * 16, there ? p.y + (size_t)s.rows[r] * p.n_out + col : p.y, there);
            }
        for (int i = tid; i < kCols * pieces; i += kThreads) {
            const int r = i / pieces, j = i - r * pieces, row = n * kCols + r;
            const bool there = row < p.n_out && j * 8 < rank;
            copy16(bs + r * pl.pitch + j * 16, there ? b + (size_t)row * rank + j * 8 : b, there);
        }
    };
    const int rt = warp & 3, half = warp >> 2;     // the warp's 16 rows, and its half of the rank's or the columns' tiles
    // (ldmatrix: lanes 0..15 give the rows of the first eight columns, 16..31 those of the next)
    const int lr = lane & 15, lc = (lane >> 4) * 16;
    const int total = (k1 - k0) + (n1 - n0);       // both products' stages in one line
    auto load = [&](int i) {
        if (i < k1 - k0) load_in(k0 + i, i % kTileStages);
        else if (i < total) load_out(n0 + i - (k1 - k0), i % kTileStages);
        copies_commit();
    };
    for (int i = 0; i < kTileStages - 1; ++i) load(i);
    float acc[NJ][8] = {};
    int it = 0;
    for (; it < k1 - k0; ++it) {
        copies_wait<kTileStages - 2>();
        __syncthreads();
        load(it + kTileStages - 1);
        const uint32_t xs = base + pl.stages_at + (it % kTileStages) * pl.stage, as = xs + kTileRows * kColPitch;
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
    for (; it < total; ++it) {
        copies_wait<kTileStages - 2>();
        __syncthreads();
        load(it + kTileStages - 1);
        const int n = n0 + it - (k1 - k0);
        unsigned char* ys_p = smem + pl.stages_at + (it % kTileStages) * pl.stage;
        const uint32_t ys = smem_addr(ys_p), bs = ys + kTileRows * kColPitch;
        float d[4][4] = {};                   // four tiles of eight columns of the warp's 32
#pragma unroll 2
        for (int kk = 0; kk < r16 / 16; ++kk) {
            uint32_t vh[4], vl[4];
            ldmatrix4(base + pl.hi_at + (rt * 16 + lr) * pl.pitch + kk * 32 + lc, vh);
            ldmatrix4(base + pl.lo_at + (rt * 16 + lr) * pl.pitch + kk * 32 + lc, vl);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                uint32_t vb[4];
                ldmatrix4(bs + (half * 32 + j * 16 + lr) * pl.pitch + kk * 32 + lc, vb);
                mma(d[2 * j], vh[0], vh[1], vh[2], vh[3], vb[0], vb[2]);
                mma(d[2 * j + 1], vh[0], vh[1], vh[2], vh[3], vb[1], vb[3]);
                mma(d[2 * j], vl[0], vl[1], vl[2], vl[3], vb[0], vb[2]);
                mma(d[2 * j + 1], vl[0], vl[1], vl[2], vl[3], vb[1], vb[3]);
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
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = rt * 16 + (lane >> 2) + 8 * i, col = half * 32 + (lane & 3) * 8;
                if (r < m && n * kCols + col < p.n_out)
                    *reinterpret_cast<uint4*>(p.out + (size_t)s.rows[r] * p.n_out + n * kCols + col) = *reinterpret_cast<const uint4*>(ys_p + r * kColPitch + col * 2);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = rt * 16 + g + 8 * (e >> 1), col = n * kCols + half * 32 + j * 8 + 2 * q + (e & 1);
                    if (r < m && col < p.n_out) {
                        const size_t at = (size_t)s.rows[r] * p.n_out + col;
                        p.out[at] = __float2bfloat16_rn(__bfloat162float(p.y[at]) + d[j][e]);
                    }
                }
        }
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
        void* args[] = {&p, nullptr};
        if (step == kFewRows) {
            IMX_TRY(launch_clusters((const void*)low_rank_few_kernel, (unsigned)(p.n * kFewCtas), kFewCtas, 0, stream, args));
            continue;
        }
        // no more units than these; CTAs for two on every SM
        const int units = p.n / kTileRows + (p.count + 1 < p.n ? p.count + 1 : p.n);
        int ctas = 1;
        while (ctas < 8 && units * ctas * 2 <= 2 * sms) ctas *= 2;
        args[1] = &ctas;
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
        device_mark_setup(di.ordinal, kSetupLowRank);
    }
    const int wide = n_out % 8 == 0 && (((uintptr_t)y | (uintptr_t)out) % 16) == 0;
    return launch_low_rank(LowRankArgs{(const __nv_bfloat16*)y, (const __nv_bfloat16*)x, (const __nv_bfloat16*)ad->a, (const __nv_bfloat16*)ad->b,
                                       ad->scale, ids, (__nv_bfloat16*)out, n_rows, in, n_out, ad->count, ad->rank, wide},
                           di.sms, (cudaStream_t)stream);
}
