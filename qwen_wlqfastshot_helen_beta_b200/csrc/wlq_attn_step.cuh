// Attention of few query rows (a decoding step: the new tokens of a sequence
// times the query heads of a kv head are at most 16) over the paged cache.
//
// HBM-bound: the cache is read once.  The key tiles of all sequences and kv
// heads, 64 keys each, form one list that is shared out evenly over the CTAs
// whatever the sequences' lengths are; a CTA walks its share, one segment per
// (sequence, kv head) it touches.  Few tiles are shared out by equal parts of
// each sequence instead, one per CTA.  Where a segment is only a part, its
// unnormalised output and statistics go to the workspace, and the CTA that
// delivers a (sequence, kv head)'s last part adds the parts up in the order
// of the keys: one launch, and results that do not depend on timing.
//
// A CTA is one TMA producer warp, which keeps the ring of tiles full across
// segments, and four consumer warps with 16 keys of each tile.  Scores are
// computed transposed, S^T = K Q^T: the 16 keys are the MMA's rows and the
// query rows its 8 columns, so 7 query heads of a group waste one column of
// eight instead of nine rows of sixteen.  The probabilities change layout in
// registers (movmatrix) and O^T += V^T P^T follows.
//
// 8-bit caches: the tensor cores take the e4m3 codes as fp16 (exact), the
// scales are applied to the scores and folded into the probabilities.  The
// queries become fp16 with a power of two per row (exact but for values
// 2^-29 of the row's largest).  A probability p times its value's scale 2^e
// is kept relative to the largest such product of the row (m1), the sum of
// the p relative to the largest score (m0), so neither the scales' spread
// nor rows of zeros cost any precision.
// What bounds it: long caches the memory (32 sequences of 16384 tokens, 28
// heads over 4, D 128: 16-bit 180 us, 6.0 TB/s, 91 % of the measured copy rate;
// 8-bit 104 us, 5.2 TB/s: a page of one head is then 2 KB at a random place).
// Short ones a chain of round trips: finding the share 1.6 us, first tile 1.5,
// a tile 0.4 to 0.75, the warps' merge and the output 1.2, joining parts 2 to 3
// (one sequence of 64 tokens 8 us, of 1501 12 us).  Scores transposed, one
// 16-key MMA per warp and tile: with two groups of 16 keys per warp the time
// per key stayed the same.
#pragma once

#include "wlq_attn_row.cuh"
#include "wlq_internal.h"

namespace wlq {

namespace {

constexpr int kStepKeys = 64;      // keys of a tile, 16 per consumer warp
constexpr int kStepThreads = 160;  // 4 consumer warps, 1 producer warp

struct StepParams {
    CUtensorMap tm_k, tm_v;
    AttnParams a;
    float* part;        // [2 * CTAs][8 NT][D] parts' outputs, two slots per CTA
    float* stat;        // [2 * CTAs][8 NT][4] their m1, m0, sum
    uint32_t* arrived;  // [B * Hkv] parts delivered; zero between calls
};

template <int D, bool Q8, int NT>
struct StepPlan {
    static constexpr int kRowsMax = 8 * NT;
    static constexpr int kSide = kStepKeys * D * (Q8 ? 1 : 2);  // k or v of a tile
    static constexpr int kStage = 2 * kSide + (Q8 ? 1024 : 0);  // 8-bit: the rows' scales behind them
    static constexpr int kMerge = 2 * kRowsMax * D * 4;         // two warps' outputs
    static constexpr int kStat = 5 * kRowsMax * 4 * 4;           // the warps' statistics, then the segment's
    static constexpr int kCtas = NT == 1 ? 3 : 2;               // per SM
    static constexpr int kFit = ((kCtas == 3 ? 74 : 112) * 1024 - 1024 - 256 - kMerge - kStat) / kStage;
    static constexpr int kStages = kFit > 8 ? 8 : kFit;
    static constexpr int kMergeOff = kStages * kStage;
    static constexpr int kStatOff = kMergeOff + kMerge;
    static constexpr int kBarOff = kStatOff + kStat;
    static constexpr int kAlloc = kBarOff + 256 + 1024;
    static_assert(kStages >= 2, "tiles in flight");
};

struct StepSeq {
    int rows, tiles, len, n, first;
};

__device__ __forceinline__ StepSeq step_seq(const AttnParams& p, int b, int rows_max) {
    StepSeq s;
    s.first = b;
    s.n = 1;
    if (p.cu) {
        s.first = p.cu[b];
        s.n = p.cu[b + 1] - s.first;
    }
    if (s.first < 0 || s.n < 0 || (int64_t)s.first + s.n > p.T) s.n = 0;  // rows outside q are nobody's
    s.len = (int)max((int64_t)0, min((int64_t)p.kv_lens[b], p.table_cols << p.log2_page));
    s.rows = min(s.n * p.G, rows_max);
    // an empty sequence's rows (zeros) still have to be written: one tile without keys
    s.tiles = s.n ? max(1, (s.len + kStepKeys - 1) / kStepKeys) : 0;
    return s;
}

// a * b / c (rounded up by `up`), in 32 bits where the product fits: a 64-bit
// division takes several times as long, and a cut needs a handful.
__device__ __forceinline__ int mul_div(uint32_t a, uint32_t b, uint32_t c, bool up) {
    const uint64_t x = (uint64_t)a * b + (up ? c - 1 : 0u);
    return (x >> 32) == 0 ? (int)((uint32_t)x / c) : (int)(x / c);
}

// The list's G - 1 cuts, at even distances; a cut within `slack` tiles of a
// sequence's (and kv head's) end moves there, so that a part is worth the
// joining it costs.
struct StepCuts {
    int total, G, slack;
    __device__ __forceinline__ int raw(int c) const { return mul_div(c, total, G, false); }
    // the cuts inside tiles [base, base + n): c in [lo, hi]
    __device__ __forceinline__ void inside(int base, int n, int& lo, int& hi) const {
        lo = mul_div(base + slack + 1, G, total, true);
        hi = n > slack ? mul_div(base + n - slack, G, total, true) - 1 : lo - 1;
    }
    __device__ __forceinline__ int moved(int at, int base, int n) const {
        return at - base <= slack ? base : (base + n - at <= slack ? base + n : at);
    }
};

// The tiles of one CTA, segment by segment.
struct StepWalk {
    int it, it1;      // this CTA's tiles of the list
    int b, cum;       // current sequence, tiles of the list before it
    StepSeq s;
    // the segment: kv head, tiles [t0, t1) of the sequence, list index of tile 0
    int hk, t0, t1, base;
    int parts, part;  // parts > 0: the segment is all there is, part number `part` of its sequence and kv head

    __device__ __forceinline__ bool next(const AttnParams& p, int rows_max) {
        if (parts) {
            const bool first = it == 0;
            it = 1;
            return first;
        }
        if (it >= it1) return false;
        while (it >= cum + s.tiles * p.Hkv) {
            cum += s.tiles * p.Hkv;
            s = step_seq(p, ++b, rows_max);
        }
        hk = (it - cum) / s.tiles;
        base = cum + hk * s.tiles;
        t0 = it - base;
        t1 = min(s.tiles, t0 + (it1 - it));
        it += t1 - t0;
        return true;
    }
};

// Parts of about T tiles.
__device__ __forceinline__ int parts_of(int tiles, int T) { return tiles ? max(1, (tiles + (T >> 1)) / T) : 0; }

__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t v) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
    return d;
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t addr, uint32_t (&a)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t (&a)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint2 lds64u(uint32_t a) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void bar_sync_step() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
__device__ __forceinline__ float4 ldcg4(const float* a) {
    float4 v;
    asm volatile("ld.global.cg.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(a)
                 : "memory");
    return v;
}
__device__ __forceinline__ float2 ldcg2(const float* a) {
    float2 v;
    asm volatile("ld.global.cg.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "l"(a) : "memory");
    return v;
}
// n += v; what this warp wrote before is visible to whoever adds after it, and the other way round.
__device__ __forceinline__ uint32_t add_acq_rel(uint32_t* n, uint32_t v) {
    uint32_t old;
    asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], %2;" : "=r"(old) : "l"(n), "r"(v) : "memory");
    return old;
}
// Barrier of the four consumer warps; whether `v` holds for all of them.
__device__ __forceinline__ bool bar_and_step(bool v) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "bar.red.and.pred q, 1, 128, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r)
        : "r"((uint32_t)v)
        : "memory");
    return r != 0;
}
// 2^(a - b) where b may be -inf (nothing seen yet)
__device__ __forceinline__ float rescale(float a, float b) { return a == b ? 1.f : ex2(a - (b == -INFINITY ? 0.f : b)); }

// One finished row: x = (m1, m0, sum, -), a this lane's E values relative to 2^m1.
template <typename T, int E>
__device__ __forceinline__ void store_row(const AttnParams& p, int hk, int first, int r, int lane, const float (&a)[E],
                                          const float4 x) {
    const float f = x.z > 0.f ? rescale(x.x, x.y) / x.z : (x.z == x.z ? 0.f : x.z);
    const int tk = r / p.G;
    uint16_t* d = p.out + (int64_t)(first + tk) * p.o_tok + (hk * p.G + r - tk * p.G) * p.o_head + lane * E;
#pragma unroll
    for (int j = 0; j < E; j += 2) *reinterpret_cast<uint32_t*>(d + j) = pack2<T>(a[j] * f, a[j + 1] * f);
}

// Adds up the parts of one (sequence, kv head), by the four consumer warps, a
// row per warp and round: the parts' statistics in a lane each, the outputs of
// eight parts in flight together.  The sums have a fixed order.  Part 0 is CTA
// c0's last, part i > 0 the first of CTA c0 + i.
template <typename T, int D, int NT>
__device__ __forceinline__ void join_parts(const StepParams& sp, int rows, int hk, int first, int c0, int parts, int warp,
                                           int lane) {
    constexpr int RM = 8 * NT, E = D / 32, U = 8;
    for (int rb = warp; rb < rows; rb += 8) {  // rows rb, rb + 4
        float a[2][E], a1[2], a0[2], sum[2];
#pragma unroll
        for (int z = 0; z < 2; ++z) {
            a1[z] = a0[z] = -INFINITY;
            sum[z] = 0.f;
#pragma unroll
            for (int j = 0; j < E; ++j) a[z][j] = 0.f;
        }
        for (int p0 = 0; p0 < parts; p0 += 32) {
            const int n = min(32, parts - p0), mine = p0 + min(lane, n - 1);
            float4 x[2];
            float f[2];
#pragma unroll
            for (int z = 0; z < 2; ++z)
                x[z] = ldcg4(sp.stat + ((int64_t)(2 * (c0 + mine) + (mine == 0)) * RM + min(rb + 4 * z, RM - 1)) * 4);
            for (int i0 = 0; i0 < n; i0 += U) {
                float4 v[2][U];
#pragma unroll
                for (int z = 0; z < 2; ++z)
#pragma unroll
                    for (int y = 0; y < U; ++y) {
                        const int i = p0 + min(i0 + y, n - 1);
                        const float* src =
                            sp.part + ((int64_t)(2 * (c0 + i) + (i == 0)) * RM + min(rb + 4 * z, RM - 1)) * D + lane * E;
                        if constexpr (E == 4) {
                            v[z][y] = ldcg4(src);
                        } else {
                            const float2 t = ldcg2(src);
                            v[z][y] = make_float4(t.x, t.y, 0.f, 0.f);
                        }
                    }
                if (i0 == 0) {  // (with the outputs on their way)
#pragma unroll
                    for (int z = 0; z < 2; ++z) {
                        if (lane >= n) x[z] = make_float4(-INFINITY, -INFINITY, 0.f, 0.f);
                        float b1 = fmaxf(a1[z], x[z].x), b0 = fmaxf(a0[z], x[z].y);
#pragma unroll
                        for (int d = 16; d; d >>= 1) {
                            b1 = fmaxf(b1, __shfl_xor_sync(0xffffffffu, b1, d));
                            b0 = fmaxf(b0, __shfl_xor_sync(0xffffffffu, b0, d));
                        }
                        const float keep = rescale(a1[z], b1);
                        f[z] = rescale(x[z].x, b1);
                        sum[z] = sum[z] * rescale(a0[z], b0) + x[z].z * rescale(x[z].y, b0);  // per lane, added up at the end
                        a1[z] = b1, a0[z] = b0;
#pragma unroll
                        for (int j = 0; j < E; ++j) a[z][j] *= keep;
                    }
                }
#pragma unroll
                for (int z = 0; z < 2; ++z)
#pragma unroll
                    for (int y = 0; y < U; ++y) {
                        const float g = __shfl_sync(0xffffffffu, f[z], min(i0 + y, 31));
                        if (i0 + y < n) {
                            a[z][0] += v[z][y].x * g;
                            a[z][1] += v[z][y].y * g;
                            if constexpr (E == 4) {
                                a[z][2] += v[z][y].z * g;
                                a[z][3] += v[z][y].w * g;
                            }
                        }
                    }
            }
        }
#pragma unroll
        for (int z = 0; z < 2; ++z) {
            const int r = rb + 4 * z;
#pragma unroll
            for (int d = 16; d; d >>= 1) sum[z] += __shfl_xor_sync(0xffffffffu, sum[z], d);
            if (r < rows) store_row<T, E>(sp.a, hk, first, r, lane, a[z], make_float4(a1[z], a0[z], sum[z], 0.f));
        }
    }
}

template <typename T, int D, bool Q8, int NT>
__global__ void __launch_bounds__(kStepThreads, StepPlan<D, Q8, NT>::kCtas) attn_step_kernel(const __grid_constant__ StepParams sp) {
    using P = StepPlan<D, Q8, NT>;
    using MT = typename std::conditional<Q8, __half, T>::type;  // the MMAs' operand type
    constexpr int NS = P::kStages, KK = D / 16, RM = P::kRowsMax;
    const AttnParams& p = sp.a;
    extern __shared__ uint8_t smem_raw[];
    __shared__ int plan[10];
    __shared__ uint32_t last_part;
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t sb = (raw + 1023u) & ~1023u;
    uint8_t* sgen = smem_raw + (sb - raw);
    const uint32_t bars = sb + P::kBarOff;
    auto full = [&](int s) { return bars + 8u * s; };
    auto empty = [&](int s) { return bars + 8u * (NS + s); };
    float* merge = reinterpret_cast<float*>(sgen + P::kMergeOff);
    float* wstat = reinterpret_cast<float*>(sgen + P::kStatOff);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 128) {
        for (int s = 0; s < NS; ++s) {
            mbar_init(full(s), Q8 ? 33 : 1);  // the producer's bytes; its lanes' copies of the scales
            mbar_init(empty(s), 4);
        }
        mbar_fence_init();
        tma_prefetch_desc(&sp.tm_k);
        tma_prefetch_desc(&sp.tm_v);
    }
    if (warp == 0) {
        int total = 0, units = 0, tiles0 = 0;  // tiles0: of this lane's sequence among the first 32
        for (int b0 = 0; b0 < p.B; b0 += 32) {
            const int tiles = b0 + lane < p.B ? step_seq(p, b0 + lane, RM).tiles : 0;
            if (b0 == 0) tiles0 = tiles;
            total += tiles;
            units += tiles > 0;
        }
        total = __reduce_add_sync(0xffffffffu, total) * p.Hkv;
        units = __reduce_add_sync(0xffffffffu, units) * p.Hkv;
        // n tiles of a (sequence, kv head) in P parts take n / P * 0.75 us and, for P > 1, 3 us + P * 0.05 us to be
        // joined: least at P = sqrt(15 n), and worth it from 6 tiles on.  Where such parts, `size` tiles each, are no more
        // than the CTAs, every CTA has one: a sequence's parts are alike, whatever the other sequences' lengths are.
        // Equal parts (even cuts), us, 8-bit: 1 x 1501 11.6 (13.4), 1 x 16384 20 (25), 32 x 1280 18.2 (21.0), 32 x 3000 29 (33), 100
        // x 500 18.7 (17.7); beyond 16 tiles a CTA they are alike (64 x 2048 45.8 (42.6), 32 x 8192 59.8 (60.8)).
        const int grid = (int)gridDim.x;
        int size = 0, parts = 0, part = 0, hk = 0;
        if (total / grid < 16 && units <= grid) {
            const float n = (float)total / (float)max(units, 1);
            size = n < 6.f ? 6 : max(1, (int)(n / fminf(n, sqrtf(15.f * n)) + 0.5f));
            for (int tries = 0; tries < 6; ++tries) {
                int sum = parts_of(tiles0, size);
                for (int b0 = 32; b0 < p.B; b0 += 32)
                    sum += b0 + lane < p.B ? parts_of(step_seq(p, b0 + lane, RM).tiles, size) : 0;
                sum = __reduce_add_sync(0xffffffffu, sum) * p.Hkv;
                if (sum <= grid) break;
                size = tries == 5 ? 0 : mul_div(size, sum, grid, false) + 1;  // 0: shared out evenly after all
            }
        }
        // Otherwise the list of tiles is cut evenly; a part is worth 4 tiles or more.
        StepCuts cuts;
        cuts.total = total;
        cuts.G = max(1, min(total, grid));
        cuts.slack = min(max(total / cuts.G / 2, 4), 8);
        // this CTA's first tile and the next one's, each with the sequence it lies in
        int first = 0, cum0 = 0, at = total, end = total;
        if (size) {
            at = end = 0;
            int before = 0;
            for (int b0 = 0; b0 < p.B; b0 += 32) {
                const int tiles = b0 == 0 ? tiles0 : b0 + lane < p.B ? step_seq(p, b0 + lane, RM).tiles : 0;
                const int ps = parts_of(tiles, size), cum = before + warp_scan(ps * p.Hkv, lane);
                const unsigned hit = __ballot_sync(0xffffffffu, (int)blockIdx.x < cum);
                if (hit) {
                    const int l = __ffs(hit) - 1;
                    first = b0 + l;
                    parts = __shfl_sync(0xffffffffu, ps, l);
                    const int n = __shfl_sync(0xffffffffu, tiles, l);
                    const int x = (int)blockIdx.x - __shfl_sync(0xffffffffu, cum - ps * p.Hkv, l);
                    hk = x / parts;
                    part = x - hk * parts;
                    at = part * n / parts;
                    end = (part + 1) * n / parts;
                    break;
                }
                before = __shfl_sync(0xffffffffu, cum, 31);
            }
        } else if ((int)blockIdx.x < cuts.G) {
            const int r0 = cuts.raw(blockIdx.x), r1 = cuts.raw(blockIdx.x + 1);
            int before = 0;
            for (int b0 = 0; b0 < p.B && before <= r1; b0 += 32) {
                const int tiles = b0 == 0 ? tiles0 : b0 + lane < p.B ? step_seq(p, b0 + lane, RM).tiles : 0;
                const int mine = tiles * p.Hkv, cum = before + warp_scan(mine, lane) - mine;
                // (sequences' tiles are disjoint: one lane of one round at most has either)
                const bool h0 = r0 >= cum && r0 < cum + mine, h1 = r1 >= cum && r1 < cum + mine;
                int m0 = 0, m1 = 0;
                if (h0) {
                    const int base = cum + (r0 - cum) / tiles * tiles;
                    m0 = cuts.moved(r0, base, tiles);
                }
                if (h1) {
                    const int base = cum + (r1 - cum) / tiles * tiles;
                    m1 = cuts.moved(r1, base, tiles);
                }
                const unsigned a0 = __ballot_sync(0xffffffffu, h0), a1 = __ballot_sync(0xffffffffu, h1);
                if (a0) {
                    const int l = __ffs(a0) - 1;
                    first = b0 + l;
                    cum0 = __shfl_sync(0xffffffffu, cum, l);
                    at = __shfl_sync(0xffffffffu, m0, l);
                }
                if (a1) end = __shfl_sync(0xffffffffu, m1, __ffs(a1) - 1);
                before = __shfl_sync(0xffffffffu, cum + mine, 31);
            }
        }
        if (lane == 0) {
            plan[0] = total;
            plan[1] = first;
            plan[2] = cum0;
            plan[3] = cuts.G;
            plan[4] = cuts.slack;
            plan[5] = at;
            plan[6] = end;
            plan[7] = parts;
            plan[8] = part;
            plan[9] = hk;
        }
    }
    __syncthreads();
    StepWalk w;
    w.it = plan[5];
    w.it1 = plan[6];
    if (w.it >= w.it1) return;
    w.parts = plan[7];
    w.part = plan[8];
    StepCuts cuts;
    cuts.total = plan[0];
    cuts.G = plan[3];
    cuts.slack = plan[4];
    w.b = plan[1];
    w.cum = plan[2];
    w.s = step_seq(p, w.b, RM);
    if (w.parts) {
        w.t0 = w.it;
        w.t1 = w.it1;
        w.hk = plan[9];
        w.it = 0;
    }

    if (warp == 4) {
        // ------------------------------------------------------ producer
        const int box = min(p.page_size, kStepKeys);  // keys of one copy
        int g = 0;
        bool ok = true;
        while (ok && w.next(p, RM)) {
            int ids = 0;  // page of this lane's 16 keys of a window of 8 tiles; one outside the pool reads as zeros
            for (int t = w.t0; t < w.t1; ++t, ++g) {
                const int x = (t - w.t0) & 7;
                if (x == 0) {
                    const int key = t * kStepKeys + lane * 16;
                    ids = key < w.s.len ? p.table[(int64_t)w.b * p.table_cols + (key >> p.log2_page)] : -1;
                    if (ids < 0 || ids >= p.num_pages) ids = (int)p.num_pages;
                }
                const int kb = t * kStepKeys;
                const int pieces = (max(0, min(kStepKeys, w.s.len - kb)) + box - 1) / box;
                const int s = g % NS, use = g / NS;
                const int key = kb + (lane & 3) * 16;  // 16 keys per lane, twice
                const int id = __shfl_sync(0xffffffffu, ids, 4 * x + (lane & 3));
                const int y = key & (p.page_size - 1);
                if (use > 0 && !(ok = warp_wait(empty(s), (use - 1) & 1))) break;
                if (lane == 0) mbar_arrive_expect_tx(full(s), pieces * box * 2 * D * (Q8 ? 1 : 2));
                __syncwarp();
                const uint32_t dst = sb + s * P::kStage;
                if constexpr (Q8) {
                    // the rows' scales, 16 bytes a lane: a copy of its own for them would cost the TMA unit as much as
                    // the codes' (3.7 TB/s of cache with it, 16 sequences of 16384 tokens)
                    if (lane < 8) {
                        const int64_t row = ((int64_t)id * p.Hkv + w.hk) * p.page_size + y;
                        cp_async16(dst + 2 * P::kSide + lane * 16, (lane < 4 ? p.k_exp : p.v_exp) + (id < p.num_pages ? row : 0),
                                   id < p.num_pages);
                    }
                    cp_async_arrive(full(s));
                }
                if (lane < 4 && (lane * 16) % box == 0 && lane * 16 < pieces * box) {
                    const int z = id * p.Hkv + w.hk;
                    if constexpr (Q8) {
                        tma_load_3d(dst + lane * 16 * D, &sp.tm_k, full(s), 0, y, z);
                        tma_load_3d(dst + P::kSide + lane * 16 * D, &sp.tm_v, full(s), 0, y, z);
                    } else {
#pragma unroll
                        for (int h = 0; h < D / 64; ++h) {
                            const uint32_t d = dst + h * kStepKeys * 128 + lane * 16 * 128;
                            tma_load_3d(d, &sp.tm_k, full(s), h * 64, y, z);
                            tma_load_3d(d + P::kSide, &sp.tm_v, full(s), h * 64, y, z);
                        }
                    }
                }
            }
        }
        // no copy may still be landing when the CTA exits
        for (int j = g > NS ? g - NS : 0; j < g; ++j) mbar_wait(full(j % NS), (j / NS) & 1);
        return;
    }

    // --------------------------------------------------------- consumers
    const int gq = lane >> 2, tq = lane & 3;
    int g = 0;
    bool ok = true;
    // the parts of the segment's (sequence, kv head), the first of them CTA c0's
    auto parts_around = [&](int& c0) {
        c0 = (int)blockIdx.x - w.part;
        if (w.parts) return w.parts;
        int hi;
        cuts.inside(w.base, w.s.tiles, c0, hi);
        --c0;
        return hi - c0 + 1;
    };
    // counts this CTA's part as delivered (one thread); whether it is the last
    auto deliver = [&](int parts) {
        uint32_t* n = sp.arrived + w.b * p.Hkv + w.hk;
        const bool last = add_acq_rel(n, 1u) == (uint32_t)(parts - 1);
        if (last) *n = 0u;  // every part is here: nobody else looks at it in this call
        return last;
    };
    while (ok && w.next(p, RM)) {
        const StepSeq s = w.s;
        const int past = s.len - s.n;
        // q as the MMAs' B operand: row 8 nt + gq, the head values this lane's k indexes stand for
        uint32_t qf[NT][KK][2];
        float fac[NT][2];  // scale of the scores of rows 8 nt + 2 tq, + 1
        int lim[NT][2];    // their last visible key
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int r = 8 * nt + gq;
            const bool in = r < s.rows;
            const int tk = in ? r / p.G : 0;
            const uint16_t* src = p.q + (int64_t)(s.first + tk) * p.q_tok + (w.hk * p.G + (in ? r - tk * p.G : 0)) * p.q_head;
            if constexpr (Q8) {
                constexpr int C = D / 32;  // 8-value chunks of this lane: its 16-code chunks of a key
                uint4 v[C];
                float f[C][8], top = 0.f;
#pragma unroll
                for (int x = 0; x < C; ++x) v[x] = keep_if(in, ldg16(src + tq * (D / 4) + 8 * x));
#pragma unroll
                for (int x = 0; x < C; ++x) {
                    const uint32_t u[4] = {v[x].x, v[x].y, v[x].z, v[x].w};
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        f[x][i] = ActTraits<T>::bits_to_f32((uint16_t)(u[i >> 1] >> (16 * (i & 1))));
                        top = fmaxf(top, fabsf(f[x][i]));
                    }
                }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                // 2^14 <= largest * 2^-e < 2^15 (a row of zeros, or of subnormals, as it is)
                const int eb = min(254, max(15, (int)(__float_as_uint(top) >> 23)));  // e = eb - 127 - 14
                const float down = __uint_as_float((uint32_t)(127 + 141 - eb) << 23);
                const float up = __uint_as_float((uint32_t)(eb - 14) << 23) * p.scale_log2;
                fac[nt][0] = __shfl_sync(0xffffffffu, up, 8 * tq);
                fac[nt][1] = __shfl_sync(0xffffffffu, up, 8 * tq + 4);
#pragma unroll
                for (int x = 0; x < C; ++x)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const __half2 h = __floats2half2_rn(f[x][2 * i] * down, f[x][2 * i + 1] * down);
                        qf[nt][2 * x + (i >> 1)][i & 1] = *reinterpret_cast<const uint32_t*>(&h);
                    }
            } else {
#pragma unroll
                for (int k = 0; k < KK; ++k)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint32_t v = *reinterpret_cast<const uint32_t*>(src + 16 * k + 2 * tq + 8 * i);
                        qf[nt][k][i] = in ? v : 0u;
                    }
                fac[nt][0] = fac[nt][1] = p.scale_log2;
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) lim[nt][i] = min(s.len - 1, past + (8 * nt + 2 * tq + i) / p.G);
        }
        float o[KK][NT][4];
        float m1[NT][2], m0[NT][2], l[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int i = 0; i < 2; ++i) m1[nt][i] = m0[nt][i] = -INFINITY, l[nt][i] = 0.f;
#pragma unroll
            for (int k = 0; k < KK; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[k][nt][i] = 0.f;
        }

        for (int t = w.t0; t < w.t1; ++t, ++g) {
            const int st = g % NS;
            if (!(ok = warp_wait(full(st), (g / NS) & 1))) break;
            const int kb = t * kStepKeys + warp * 16;
            if (kb < s.len) {
                const uint32_t ks = sb + st * P::kStage, vs = ks + P::kSide;
                const int k0 = warp * 16;
                float c[2][NT][4];
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) c[h][nt][i] = 0.f;
                if constexpr (Q8) {
                    uint4 a[D / 64], b[D / 64];
#pragma unroll
                    for (int x = 0; x < D / 64; ++x) {
                        const int r0 = k0 + gq, r1 = r0 + 8, ch = (D / 64) * tq + x;
                        if constexpr (D == 128) {
                            a[x] = lds128(ks + r0 * 128 + (((ch ^ r0) & 7) << 4));
                            b[x] = lds128(ks + r1 * 128 + (((ch ^ r1) & 7) << 4));
                        } else {
                            a[x] = lds128(ks + r0 * 64 + (((ch ^ (r0 >> 1)) & 3) << 4));
                            b[x] = lds128(ks + r1 * 64 + (((ch ^ (r1 >> 1)) & 3) << 4));
                        }
                    }
#pragma unroll
                    for (int x = 0; x < D / 64; ++x) {
                        const uint32_t wa[4] = {a[x].x, a[x].y, a[x].z, a[x].w}, wb[4] = {b[x].x, b[x].y, b[x].z, b[x].w};
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint32_t f[4] = {e4m3x2_to_f16x2(wa[i]), e4m3x2_to_f16x2(wb[i]),
                                                   e4m3x2_to_f16x2(wa[i] >> 16), e4m3x2_to_f16x2(wb[i] >> 16)};
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
                                Mma16816<MT>::run(c[i & 1][nt], f, qf[nt][4 * x + i][0], qf[nt][4 * x + i][1]);
                        }
                    }
                } else {
                    const int r = k0 + (lane & 15);
#pragma unroll
                    for (int k = 0; k < KK; ++k) {
                        uint32_t f[4];
                        const int ch = 2 * (k & 3) + (lane >> 4);
                        ldmatrix_x4(ks + (k >> 2) * kStepKeys * 128 + r * 128 + (((ch ^ r) & 7) << 4), f);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) Mma16816<MT>::run(c[k & 1][nt], f, qf[nt][k][0], qf[nt][k][1]);
                    }
                }
                // scores in powers of two; x0 of a key's value scale 2^ve
                float ke[2] = {1.f, 1.f}, ve[2] = {0.f, 0.f};
                if constexpr (Q8) {
                    const uint32_t es = ks + 2 * P::kSide + k0 + gq;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        ke[h] = exp2_biased(lds8(es + 8 * h));
                        ve[h] = (float)((int)lds8(es + kStepKeys + 8 * h) - 127);
                    }
                }
                float sc[NT][4];
                bool grow = false;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int key = kb + gq + 8 * (i >> 1);
                        float x = (c[0][nt][i] + c[1][nt][i]) * fac[nt][i & 1];
                        if constexpr (Q8) x *= ke[i >> 1];
                        x = key <= lim[nt][i & 1] ? x : -INFINITY;
                        sc[nt][i] = x;
                        grow |= x - m0[nt][i & 1] > 8.f;
                        if constexpr (Q8) grow |= x + ve[i >> 1] - m1[nt][i & 1] > 8.f;
                    }
                if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float f1[2];
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            float a = fmaxf(m0[nt][i], fmaxf(sc[nt][i], sc[nt][i + 2]));
                            float b = fmaxf(m1[nt][i], fmaxf(sc[nt][i] + ve[0], sc[nt][i + 2] + ve[1]));
#pragma unroll
                            for (int d = 4; d < 32; d <<= 1) {
                                a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, d));
                                if constexpr (Q8) b = fmaxf(b, __shfl_xor_sync(0xffffffffu, b, d));
                            }
                            if constexpr (!Q8) b = a;
                            l[nt][i] *= rescale(m0[nt][i], a);
                            f1[i] = rescale(m1[nt][i], b);
                            m0[nt][i] = a;
                            m1[nt][i] = b;
                        }
#pragma unroll
                        for (int k = 0; k < KK; ++k)
#pragma unroll
                            for (int i = 0; i < 4; ++i) o[k][nt][i] *= f1[i & 1];
                    }
                }
                // probabilities: this lane's keys gq, gq + 8 -> B fragments with keys 2 tq ..
                uint32_t pf[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float x[2];
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const float r0 = m0[nt][i] == -INFINITY ? 0.f : m0[nt][i];
                            const float e = ex2(sc[nt][2 * h + i] - r0);
                            l[nt][i] += e;
                            x[i] = e;
                            if constexpr (Q8) {
                                const float r1 = m1[nt][i] == -INFINITY ? 0.f : m1[nt][i];
                                x[i] = ex2(sc[nt][2 * h + i] + ve[h] - r1);
                            }
                        }
                        pf[nt][h] = movmatrix_trans(pack2<MT>(x[0], x[1]));
                    }
                const int behind = s.len - kb;  // keys of the 16 that exist
                if constexpr (Q8) {
                    constexpr int W = D / 32;  // words of 4 codes of a lane: its chunk of each of 4 keys
                    uint32_t v[4][W];
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const int kx = 2 * tq + (x & 1) + 8 * (x >> 1), r = k0 + kx;
                        if constexpr (D == 128) {
                            const uint4 q = lds128(vs + r * 128 + (((gq ^ r) & 7) << 4));
                            v[x][0] = q.x, v[x][1] = q.y, v[x][2] = q.z, v[x][3] = q.w;
                        } else {
                            const uint2 q = lds64u(vs + r * 64 + ((((gq >> 1) ^ (r >> 1)) & 3) << 4) + (gq & 1) * 8);
                            v[x][0] = q.x, v[x][1] = q.y;
                        }
                        if (behind < 16 && kx >= behind) {
#pragma unroll
                            for (int y = 0; y < W; ++y) v[x][y] = 0u;
                        }
                    }
#pragma unroll
                    for (int y = 0; y < W; ++y)
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const uint32_t sel = j ? 0x7362u : 0x5140u;
                            const uint32_t a = prmt(v[0][y], v[1][y], sel), b = prmt(v[2][y], v[3][y], sel);
                            const uint32_t f[4] = {e4m3x2_to_f16x2(a), e4m3x2_to_f16x2(a >> 16), e4m3x2_to_f16x2(b),
                                                   e4m3x2_to_f16x2(b >> 16)};
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) Mma16816<MT>::run(o[2 * y + j][nt], f, pf[nt][0], pf[nt][1]);
                        }
                } else {
                    const int r = k0 + (lane & 7) + 8 * (lane >> 4);
                    uint32_t keep[2] = {0xffffffffu, 0xffffffffu};
                    if (behind < 16) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int kx = 2 * tq + 8 * h;
                            keep[h] = (kx < behind ? 0xffffu : 0u) | (kx + 1 < behind ? 0xffff0000u : 0u);
                        }
                    }
#pragma unroll
                    for (int k = 0; k < KK; ++k) {
                        uint32_t f[4];
                        const int ch = 2 * (k & 3) + ((lane >> 3) & 1);
                        ldmatrix_x4_trans(vs + (k >> 2) * kStepKeys * 128 + r * 128 + (((ch ^ r) & 7) << 4), f);
                        if (behind < 16) {
                            f[0] &= keep[0], f[1] &= keep[0];
                            f[2] &= keep[1], f[3] &= keep[1];
                        }
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) Mma16816<MT>::run(o[k][nt], f, pf[nt][0], pf[nt][1]);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(empty(st));
        }
        // ------------------------------- the segment's result, in warp 0
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) l[nt][i] += __shfl_xor_sync(0xffffffffu, l[nt][i], d);
                if (gq == 0)
                    *reinterpret_cast<float4*>(wstat + (warp * RM + 8 * nt + 2 * tq + i) * 4) =
                        make_float4(m1[nt][i], m0[nt][i], l[nt][i], 0.f);
            }
        if (!(ok = bar_and_step(ok))) break;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float f[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float4 x[4];
#pragma unroll
                for (int y = 0; y < 4; ++y)
                    x[y] = *reinterpret_cast<const float4*>(wstat + (y * RM + 8 * nt + 2 * tq + i) * 4);
                const float a = fmaxf(fmaxf(x[0].x, x[1].x), fmaxf(x[2].x, x[3].x));
                const float b = fmaxf(fmaxf(x[0].y, x[1].y), fmaxf(x[2].y, x[3].y));
                f[i] = rescale(m1[nt][i], a);
                float sum = 0.f;
#pragma unroll
                for (int y = 0; y < 4; ++y) sum += x[y].z * rescale(x[y].y, b);
                m1[nt][i] = a;
                m0[nt][i] = b;
                l[nt][i] = sum;
            }
#pragma unroll
            for (int k = 0; k < KK; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[k][nt][i] *= f[i & 1];
        }
        auto out_to = [&](int y) {
#pragma unroll
            for (int k = 0; k < KK; ++k)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    *reinterpret_cast<float4*>(merge + (((y * KK + k) * NT + nt) * 32 + lane) * 4) =
                        make_float4(o[k][nt][0], o[k][nt][1], o[k][nt][2], o[k][nt][3]);
        };
        auto add_from = [&](int y) {
#pragma unroll
            for (int k = 0; k < KK; ++k)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const float4 x = *reinterpret_cast<const float4*>(merge + (((y * KK + k) * NT + nt) * 32 + lane) * 4);
                    o[k][nt][0] += x.x, o[k][nt][1] += x.y, o[k][nt][2] += x.z, o[k][nt][3] += x.w;
                }
        };
        if (warp >= 2) out_to(warp - 2);
        bar_sync_step();
        if (warp < 2) add_from(warp);
        if (warp == 1) out_to(1);
        bar_sync_step();
        if (warp == 0) {
            add_from(1);
            unsigned bad = 0;  // rows with a value that is not finite
            if (s.n > 1) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float x = 0.f;
#pragma unroll
                        for (int k = 0; k < KK; ++k) x = fmaf(o[k][nt][i], 0.f, fmaf(o[k][nt][2 + i], 0.f, x));
                        if (x != x) bad |= 1u << (8 * nt + 2 * tq + i);
                    }
                bad = __reduce_or_sync(0xffffffffu, bad);
            }
            out_to(0);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    if (gq == 0)
                        *reinterpret_cast<float4*>(wstat + (4 * RM + 8 * nt + 2 * tq + i) * 4) =
                            make_float4(m1[nt][i], m0[nt][i], l[nt][i], __uint_as_float(bad));
        }
        bar_sync_step();
        // a row per warp and round, E values of it per lane
        const bool whole = w.t0 == 0 && w.t1 == s.tiles;
        constexpr int E = D / 32;
        const int slot = 2 * (int)blockIdx.x + (w.t0 == 0);
        for (int rb = warp; rb < s.rows; rb += 8) {  // rows rb, rb + 4
            float4 x[2];
            float a[2][E];
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                const int r = min(rb + 4 * y, RM - 1);
                x[y] = *reinterpret_cast<const float4*>(wstat + (4 * RM + r) * 4);
#pragma unroll
                for (int j = 0; j < E; ++j) {
                    // where warp 0's lane and register of (row r, value d) went
                    const int d = lane * E + j;
                    const int k = Q8 ? (d % (D / 8)) >> 1 : d >> 4, gl = Q8 ? d / (D / 8) : d & 7, h = Q8 ? d & 1 : (d >> 3) & 1;
                    a[y][j] = merge[((k * NT + (r >> 3)) * 32 + gl * 4 + ((r & 7) >> 1)) * 4 + 2 * h + (r & 1)];
                }
            }
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                const int r = rb + 4 * y;
                if (r >= s.rows) break;
                // with several new tokens, keys a row does not see may have spoilt it (a sum that is NaN is so by what it sees)
                if (s.n > 1 && ((__float_as_uint(x[y].w) >> r) & 1) && x[y].z == x[y].z) {
                    constexpr int kSource = Q8 ? kPaged8 : kPaged;
                    const int seen = max(0, min(s.len, past + r / p.G + 1)), j0 = w.t0 * kStepKeys;
                    const RowOf u{w.b, w.hk, s.first};
                    if (last_not_finite<T, D, kSource>(p, u, max(seen, j0), min(s.len, w.t1 * kStepKeys), lane) >= 0) {
                        row_alone<T, D, kSource>(p, u, r, j0, seen, lane, a[y], x[y].x, x[y].z);
                        x[y].y = x[y].x;
                    }
                }
                if (whole) {
                    store_row<T, E>(p, w.hk, s.first, r, lane, a[y], x[y]);
                } else {
                    float* d = sp.part + ((int64_t)slot * RM + r) * D + lane * E;
#pragma unroll
                    for (int j = 0; j < E; j += 2) *reinterpret_cast<float2*>(d + j) = make_float2(a[y][j], a[y][j + 1]);
                    if (lane == 0) *reinterpret_cast<float4*>(sp.stat + ((int64_t)slot * RM + r) * 4) = x[y];
                }
            }
        }
        // its parts: the one a CTA ends its share with (slot 1), then those that begin with a cut (slot 0)
        if (!whole) {
            int c0;
            const int parts = parts_around(c0);
            bar_sync_step();
            if (threadIdx.x == 0) last_part = deliver(parts);
            bar_sync_step();
            if (last_part) join_parts<T, D, NT>(sp, s.rows, w.hk, s.first, c0, parts, warp, lane);
        }
    }
    // A CTA that gave up still counts its parts: the counters are zero again after the call, whose output is undefined
    // (the device error word says so), and the next call finds them as it must.
    if (!ok && threadIdx.x == 0) {
        do {
            int c0;
            if (w.t0 != 0 || w.t1 != w.s.tiles) deliver(parts_around(c0));
        } while (w.next(p, RM));
    }
}

// Counters of the (sequence, kv head) pairs ahead of the parts; their place
// does not depend on the call, so that what one call leaves zero the next
// one finds zero.
constexpr size_t kStepCounters = WLQ_ATTENTION_ZERO_BYTES / 4;


template <typename T, int D, bool Q8, int NT>
int launch_step(const AttnParams& a, cudaStream_t stream) {
    using P = StepPlan<D, Q8, NT>;
    StepParams sp;
    sp.a = a;
    int rc;
    const CUtensorMapDataType dt = Q8                            ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                   : (ActTraits<T>::kIsF16) ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    constexpr int es = Q8 ? 1 : 2;
    const uint64_t pg = (uint64_t)a.num_pages * a.Hkv, ps = a.page_size;
    const CUtensorMapSwizzle sw = Q8 && D == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B;
    const uint32_t box = Q8 ? D : 64, keys = a.page_size < kStepKeys ? a.page_size : kStepKeys;
    if ((rc = encode_3d(&sp.tm_k, dt, a.k_cache, D, ps, pg, D * es, ps * D * es, box, keys, 1, sw, "k_cache")) ||
        (rc = encode_3d(&sp.tm_v, dt, a.v_cache, D, ps, pg, D * es, ps * D * es, box, keys, 1, sw, "v_cache")))
        return rc;
    // no more CTAs than the table has tiles for
    const int64_t tiles = (int64_t)a.B * a.Hkv * std::max<int64_t>(1, ((a.table_cols << a.log2_page) + kStepKeys - 1) / kStepKeys);
    const int grid = (int)std::min<int64_t>(P::kCtas * device_sm_count(), tiles);
    sp.arrived = static_cast<uint32_t*>(a.ws);
    sp.stat = reinterpret_cast<float*>(sp.arrived + kStepCounters);
    sp.part = sp.stat + (size_t)2 * grid * P::kRowsMax * 4;
    auto kernel = attn_step_kernel<T, D, Q8, NT>;
    static OncePerDevice limit;
    if ((rc = allow_shared_memory(limit, kernel, P::kAlloc, "attn_step_kernel shared memory"))) return rc;
    kernel<<<grid, kStepThreads, P::kAlloc, stream>>>(sp);
    return check_cuda(cudaGetLastError(), "attn_step_kernel");
}

template <typename T>
int launch_step_any(const AttnParams& a, cudaStream_t stream) {
    const bool one = a.max_q * a.G <= 8;
    if (a.k_exp) {
        if (a.D == 64) return one ? launch_step<T, 64, true, 1>(a, stream) : launch_step<T, 64, true, 2>(a, stream);
        return one ? launch_step<T, 128, true, 1>(a, stream) : launch_step<T, 128, true, 2>(a, stream);
    }
    if (a.D == 64) return one ? launch_step<T, 64, false, 1>(a, stream) : launch_step<T, 64, false, 2>(a, stream);
    return one ? launch_step<T, 128, false, 1>(a, stream) : launch_step<T, 128, false, 2>(a, stream);
}

}  // namespace

}  // namespace wlq
