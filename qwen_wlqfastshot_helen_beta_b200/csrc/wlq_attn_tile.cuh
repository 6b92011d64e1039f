// Attention of many query rows: 256 rows of one kv head against tiles of 128
// keys on the tensor cores (tcgen05, scores and outputs in TMEM).
//
// With s_ij = q_i . k_j, o_i = sum_j 2^(c s_ij - M_i) v_j / sum_j 2^(c s_ij -
// M_i), c = scale log2(e), the sums taken tile by tile with a running
// reference M_i; both sums carry the same factor, so M_i only has to keep the
// exponentials in range.  It is raised, and the output accumulator rescaled,
// only when a probability would pass 2^14 (fp16 ends at 2^16): no precision is
// lost, they are floating-point numbers and the sum is fp32, and after the
// first tiles the accumulator is hardly ever touched.
//
// A tile's 128 rows are whole tokens of one sequence times the G query heads
// of one kv head, token-major (128 / G tokens, rounded down), so that a short
// prompt or a chunk of few tokens fills its tiles whatever G is, every row of
// a tile needs about the same keys, and q comes and the output goes as one
// TMA box of tokens x heads.
//
// Roles (one CTA per SM):
//   warps 0..3, 4..7  softmax of rows 0..127 and 128..255, a thread per row:
//                     scores TMEM -> registers, maximum, exponentials, the
//                     16-bit probabilities back into TMEM over the scores;
//                     the output through the q tile's shared memory
//   warp 8            issues the MMAs: S = Q K^T (both from shared memory),
//                     O += P V (P from TMEM).  The order P0 V, S0, P1 V, S1
//                     lets the tensor cores work on one half's tiles while
//                     the other half's softmax runs; with a warp for each half
//                     both halves fell into step, softmax beside softmax (514
//                     us for a prompt of 8192 tokens and 28 heads, 439 so)
//   warp 9            TMA producer of q and of the k and v tiles: packed rows,
//                     or one copy per page
//   warps 12..19      8-bit caches: the pages' codes land in a staging ring
//                     and are written as the 16-bit tiles the MMAs read,
//                     code * 2^e, which is exact
//
// What bounds it: the chain of one half, softmax (2000 cycles: scores read 200,
// maximum 450, 128 exponentials a thread 1350) then P V and the next S (1024),
// against 2048 cycles of MMAs for a pair of tiles; a pair takes 3300 (61 % of
// the tensor pipe's cycles).  One prompt of 8192 tokens, 28 heads over 4, D 128,
// bf16, values spread as activations are, call after call under the power cap:
// 454 us, 1.06 PFLOP/s of the causal products, 64 % of the measured cuBLAS
// burst rate; normal values, a call at a time: 382 us, 1.26 PFLOP/s.  The latter
// way 4 x 512 new tokens over 16384 cached ones take 458 us from 16-bit pages of 16
// tokens, 441 from pages of 64, and 580 us from 8-bit ones, where writing and
// reading the 16-bit tiles beside the MMAs' operands takes the shared memory's
// rate (and 96 registers a thread spill 64 to 76 bytes in the softmax groups).
// Tried: a polynomial for a part of the exponentials (1.5 % faster for
// prompts, 4 to 15 % slower over pages); exponentials before the maximum (10 %
// slower); references that rise by 2^8 (4 % slower than by 2^14); prompts' row
// tiles by length over all sequences (0 to 3 % slower than sequence by sequence).
//
// Every mbarrier wait is bounded; a wait that runs out sets the device error
// word and the CTA winds down, releasing its TMEM.
#pragma once

#include <algorithm>

#include "wlq_attn_row.cuh"
#include "wlq_internal.h"

namespace wlq {

namespace {

constexpr int kRowsT = 128;   // query rows of one tile (MMA M)
constexpr int kRows = 256;    // query rows of one CTA
constexpr int kKeys = 128;    // keys of one tile
constexpr float kGrow = 14.f; // powers of two a row's maximum may pass its reference by
constexpr int kConvWarps = 8; // warps that turn codes into 16-bit tiles

struct TileParams {
    CUtensorMap tm_q, tm_o, tm_k, tm_v;
    AttnParams a;
    int* joins;   // numbers of row tiles that several CTAs share (few parts, many), then a Join for each
    float* part;  // [split CTAs][D / 4][kRows][4] unnormalised outputs of a part of the keys
    float* stat;  // [split CTAs][kRows][2] their row maxima (times c) and sums
    int sms;
    int nt;       // tokens of a tile: 128 / G
};

template <int D, int SRC>
struct TilePlan {
    static constexpr int kHalves = D / 64;           // 128-byte-wide column blocks of a tile
    static constexpr int kBlock = kKeys * 128;       // bytes of one block
    static constexpr int kTileBytes = kBlock * kHalves;
    static constexpr int kQBytes = 2 * kTileBytes;
    static constexpr int kStageBytes = kKeys * D + kKeys;  // 8-bit codes of one tile and their rows' scales
    static constexpr int kStages = SRC == kPaged8 ? 2 : 0;
    static constexpr int kBudget = 227 * 1024 - 2048 - kQBytes - kStages * kStageBytes;
    static constexpr int kFit = kBudget / kTileBytes;
    static constexpr int kSlots = kFit > 8 ? 8 : kFit;
    static constexpr int kKvOff = kQBytes;
    static constexpr int kStageOff = kKvOff + kSlots * kTileBytes;
    static constexpr int kBarOff = kStageOff + kStages * kStageBytes;
    static constexpr int kAlloc = kBarOff + 512 + 1024;  // barriers, alignment slack
    // registers a thread: the softmax groups hold a row's 128 scores; the
    // groups' shares add up to what the block is launched with (168 x 3, 96 x 5)
    static constexpr int kThreads = SRC == kPaged8 ? 640 : 384;
    static constexpr int kRegsSoftmax = SRC == kPaged8 ? 168 : 208, kRegsOther = SRC == kPaged8 ? 48 : 88;
    static_assert(2 * kRegsSoftmax + (kThreads / 128 - 2) * kRegsOther == 65536 / kThreads / 8 * 8 * (kThreads / 128),
                  "register shares");
    // the next k and v tiles are waited for while this one's still hold theirs
    static_assert(kSlots >= 4, "k and v tiles in flight");
};

// A row tile whose keys several CTAs share: the first part's slot (the next
// ones follow Hkv apart), the parts, and the rows.
struct alignas(8) Join {
    int slot, parts, tok0, n, first, hk;
};

// What one CTA works on.
struct Unit {
    int b, hk;        // sequence, kv head
    int tok0, n;      // its first token in the sequence, tokens of the sequence
    int first;        // first query token of the sequence in q
    int past;         // token t sees keys <= past + t
    int len;          // keys of the sequence
    int tile0, tiles; // key tiles [tile0, tile0 + tiles)
    int slot;         // partial result slot, or -1: the whole row is here
};

struct Seq {
    int tiles, rtiles, len, n, first;
};

template <bool PAGED>
__device__ __forceinline__ Seq seq_of(const AttnParams& p, int nt, int b) {
    Seq s;
    if (p.cu) {
        s.first = p.cu[b];
        s.n = p.cu[b + 1] - s.first;
    } else {
        s.first = b;
        s.n = 1;
    }
    // rows outside q are nobody's
    if (s.first < 0 || s.n < 0 || (int64_t)s.first + s.n > p.T) s.n = 0;
    s.len = s.n;
    if (PAGED) s.len = (int)max((int64_t)0, min((int64_t)p.kv_lens[b], p.table_cols << p.log2_page));
    s.rtiles = (s.n + 2 * nt - 1) / (2 * nt);
    s.tiles = (s.len + kKeys - 1) / kKeys;
    return s;
}

constexpr int kJoinListBytes = 64 * 1024;  // (at least two parts each: at most 4 * 148 / 2 entries)
constexpr int kFewTiles = 4;    // key tiles of a part, at least
// CTAs an SM where rows are shared, at most (4 x 512 tokens over 1501 .. 16384
// 8-bit ones: 213 us, 224 with three)
constexpr int kPartsPerSm = 4;
constexpr int kLanesSeqs = 32;  // sequences whose split is searched for

// Key tiles of one part (paged form), found by one warp: a sequence with more
// tiles is shared by several CTAs.  Up to 32 sequences: of 16 sizes the one
// with the least waves of CTAs times a part's duration (its tiles, about 3
// more for starting and ending, and once 6 for joining the parts).  More
// sequences: an even share of all tiles.  The search's time, the even share's in
// brackets (us, 28 heads over 4, D 128, 16-bit): 8 x 40 tokens over 16384 124 (143),
// 1 x 512 over 16384 133 (146), 4 x 64 over 8192 57 (60), 4 x 128 over 4096 51 (52); but
// where one wave of CTAs does all, 1 x 64 over 16384 36 (28), 1 x 64 over 65536 87 (65), 3
// x 196 over 3071 43 (36): the host launches up to four CTAs an SM for the search, and
// those without work wait for an SM until the others end.
__device__ __forceinline__ int tiles_per_part(const AttnParams& p, int nt, int sms, int lane) {
    if (p.B > kLanesSeqs) {
        int64_t w = 0;
        for (int b = lane; b < p.B; b += 32) {
            const Seq s = seq_of<true>(p, nt, b);
            w += (int64_t)s.rtiles * s.tiles;
        }
        return (int)max((int64_t)kFewTiles, (warp_sum(w) * p.Hkv + sms - 1) / sms);
    }
    Seq s{};
    if (lane < p.B) s = seq_of<true>(p, nt, lane);
    const int most = __reduce_max_sync(0xffffffffu, s.rtiles ? s.tiles : 0);
    const int units = s.rtiles * p.Hkv;
    int best = most, cost = 0x7fffffff;
    for (int parts = 1; parts <= 64; parts += parts < 8 ? 1 : parts / 4) {
        const int per = (most + parts - 1) / parts;
        if (parts > 1 && per < kFewTiles) break;
        const int sp = (s.tiles + per - 1) / max(per, 1);
        const int ctas = __reduce_add_sync(0xffffffffu, units * max(sp, 1));
        const int shared = __reduce_add_sync(0xffffffffu, sp > 1 ? units * sp : 0);
        if (shared && ctas > kPartsPerSm * sms) break;
        const int c = (ctas + sms - 1) / sms * (per + 3) + (shared ? 6 : 0);
        if (c < cost) {
            cost = c;
            best = per;
        }
    }
    return max(best, 1);
}
__device__ __forceinline__ int parts_of(const Seq& s, int per) { return s.rtiles ? max(1, (s.tiles + per - 1) / per) : 0; }

// The work of CTA c, found by one warp: sequences in order, row tiles from
// the last (the longest, where the mask is causal) to the first, then parts
// of the keys, then heads.  False if there is none.
template <bool PAGED>
__device__ __forceinline__ bool find_unit(const AttnParams& p, int nt, int sms, int c, int lane, Unit& u) {
    const int per = PAGED ? tiles_per_part(p, nt, sms, lane) : 0;
    int before = 0, slots = 0;  // CTAs of earlier sequences, those of them that hold parts
    for (int b0 = 0; b0 < p.B; b0 += 32) {
        const int b = b0 + lane;
        Seq s{};
        int sp = 0;
        if (b < p.B) {
            s = seq_of<PAGED>(p, nt, b);
            sp = PAGED ? parts_of(s, per) : (s.rtiles ? 1 : 0);
        }
        const int mine = s.rtiles * sp * p.Hkv, part = sp > 1 ? mine : 0;
        const int cum = warp_scan(mine, lane), pcum = warp_scan(part, lane);
        const unsigned hit = __ballot_sync(0xffffffffu, c < before + cum);
        if (hit) {
            const int l = __ffs(hit) - 1;
            const int x = c - before - __shfl_sync(0xffffffffu, cum - mine, l);  // CTA within the sequence
            const int slot0 = slots + __shfl_sync(0xffffffffu, pcum - part, l);
            sp = __shfl_sync(0xffffffffu, sp, l);
            s.rtiles = __shfl_sync(0xffffffffu, s.rtiles, l);
            s.tiles = __shfl_sync(0xffffffffu, s.tiles, l);
            s.len = __shfl_sync(0xffffffffu, s.len, l);
            s.n = __shfl_sync(0xffffffffu, s.n, l);
            s.first = __shfl_sync(0xffffffffu, s.first, l);
            u.b = b0 + l;
            u.hk = x % p.Hkv;
            const int y = x / p.Hkv;
            const int part_no = y % sp;
            u.tok0 = (s.rtiles - 1 - y / sp) * 2 * nt;
            u.n = s.n;
            u.first = s.first;
            u.len = s.len;
            u.past = s.len - s.n;
            // keys the last token sees
            const int seen = p.causal ? max(0, min(s.len, u.past + min(u.tok0 + 2 * nt, s.n))) : s.len;
            const int need = (seen + kKeys - 1) / kKeys;
            u.tile0 = sp > 1 ? min(need, part_no * per) : 0;
            u.tiles = (sp > 1 ? min(need, u.tile0 + per) : need) - u.tile0;
            u.slot = sp > 1 ? slot0 + x : -1;
            return true;
        }
        before += __shfl_sync(0xffffffffu, cum, 31);
        slots += __shfl_sync(0xffffffffu, pcum, 31);
    }
    return false;
}

// The lists of joins, written by one warp of CTA 0: those of up to
// kJoinWarps parts, which take a warp a piece, from the front, the others, which
// take a block a piece, from the back.  Chunk and join (us, all joins by blocks
// in brackets): 4 x 128 over 4096 51 (64), 3 x 196 over 3071 43 (58), 8 x 40 over 16384 125
// (134), 1 x 64 over 4096, 8 parts, 23.5 (21.8); with all by warps 1 x 64 over 16384 41
// instead of 36, over 65536 96 instead of 87.
constexpr int kJoinWarps = 8;
constexpr int kMaxJoins = (kJoinListBytes - 8) / (int)sizeof(Join);

__device__ __forceinline__ void list_joins(const AttnParams& p, int nt, int sms, int lane, int* out) {
    const int per = tiles_per_part(p, nt, sms, lane);
    Join* list = reinterpret_cast<Join*>(out + 2);
    int few = 0, many = 0, slots = 0;
    for (int b0 = 0; b0 < p.B; b0 += 32) {
        const int b = b0 + lane;
        Seq s{};
        int sp = 0;
        if (b < p.B) {
            s = seq_of<true>(p, nt, b);
            sp = parts_of(s, per);
        }
        const int mine = sp > 1 ? s.rtiles * p.Hkv : 0;
        const int nf = sp <= kJoinWarps ? mine : 0, nm = mine - nf;
        const int at_f = few + warp_scan(nf, lane) - nf, at_m = many + warp_scan(nm, lane) - nm;
        const int slot = slots + warp_scan(mine * sp, lane) - mine * sp;
        for (int x = 0; x < mine; ++x) {
            const int rt = x / p.Hkv, hk = x - rt * p.Hkv;
            list[nf ? at_f + x : kMaxJoins - 1 - (at_m + x)] =
                Join{slot + rt * sp * p.Hkv + hk, sp, (s.rtiles - 1 - rt) * 2 * nt, s.n, s.first, hk};
        }
        few = __shfl_sync(0xffffffffu, at_f + nf, 31);
        many = __shfl_sync(0xffffffffu, at_m + nm, 31);
        slots = __shfl_sync(0xffffffffu, slot + mine * sp, 31);
    }
    if (lane == 0) {
        out[0] = few;
        out[1] = many;
    }
}

// ------------------------------------------------------------ tcgen05 extras

// Descriptor of a tile stored as its transpose (the MMA's N contiguous): 128
// key rows of 64 values in the 128-byte swizzle, 8-row atoms of 1024 bytes
// along K, the next 64 columns of N one block further.
__device__ __forceinline__ uint64_t umma_desc_mn_sw128(uint32_t saddr, uint32_t block) {
    uint64_t d = 0;
    d |= (uint64_t)((saddr >> 4) & 0x3FFFu);
    d |= (uint64_t)(block >> 4) << 16;
    d |= (uint64_t)(1024u >> 4) << 32;
    d |= (uint64_t)1u << 46;
    d |= (uint64_t)2u << 61;
    return d;
}

// One lane of a converged warp: 1 there, 0 in the others.
__device__ __forceinline__ uint32_t elect_one() {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(r));
    return r;
}
// The MMAs and the commit of wlq_sm100.cuh, issued where `me` is set.
__device__ __forceinline__ void umma_f16_if(uint32_t me, uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                            uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(me)
        : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem]: A is M x 16 16-bit values, two per column
__device__ __forceinline__ void umma_f16_ts_if(uint32_t me, uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc,
                                               uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(tmem_d), "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(me)
        : "memory");
}
__device__ __forceinline__ void umma_commit_if(uint32_t me, uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
        ::"r"(bar), "r"(me)
        : "memory");
}

__device__ __forceinline__ void tmem_st_32x32b_x32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};"
        ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
          "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
          "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]),
          "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, uint32_t src, int x, int y, int z) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];"
                 ::"l"(reinterpret_cast<uint64_t>(map)), "r"(src), "r"(x), "r"(y), "r"(z)
                 : "memory");
}
__device__ __forceinline__ void tma_store_wait() {  // until this thread's stores have read their source
    asm volatile("cp.async.bulk.commit_group;\n\tcp.async.bulk.wait_group.read 0;" ::: "memory");
}
// Barrier of one half's 128 softmax threads; whether `v` holds for any.
__device__ __forceinline__ bool bar_or_half(int t, bool v) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "bar.red.or.pred q, %2, 128, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r)
        : "r"((uint32_t)v), "r"(1 + t)
        : "memory");
    return r != 0;
}

// Two fp32 operations in one instruction.
__device__ __forceinline__ uint64_t f2_pack(float a, float b) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ void f2_unpack(uint64_t v, float& a, float& b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

__device__ __forceinline__ uint64_t f2_mul(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// 16 e4m3 codes times 2^(e - 127) as 16-bit values, exact where the type has
// them: in fp16 by one packed product after the conversion (scales outside
// fp16's normal range and everything in bf16 through fp32).
template <typename T>
__device__ __forceinline__ void codes_to_16(uint4 q, uint32_t e, uint32_t (&o)[8]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
    if (ActTraits<T>::kIsF16 && e >= 113 && e <= 142) {
        const uint32_t s16 = (e - 112) << 10;  // 2^(e - 127)
        const uint32_t s2 = s16 | (s16 << 16);
#pragma unroll
        for (int y = 0; y < 8; ++y) {
            const uint32_t h = e4m3x2_to_f16x2(y & 1 ? w[y >> 1] >> 16 : w[y >> 1]);
            const __half2 v = __hmul2(*reinterpret_cast<const __half2*>(&h), *reinterpret_cast<const __half2*>(&s2));
            o[y] = *reinterpret_cast<const uint32_t*>(&v);
        }
        return;
    }
    const float sc = exp2_biased(e);
    const uint64_t sc2 = f2_pack(sc, sc);
#pragma unroll
    for (int y = 0; y < 8; ++y) {
        const uint32_t h = e4m3x2_to_f16x2(y & 1 ? w[y >> 1] >> 16 : w[y >> 1]);
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
        float a, b;
        f2_unpack(f2_mul(f2_pack(f.x, f.y), sc2), a, b);
        o[y] = pack2<T>(a, b);
    }
}

// Byte offset of 16-byte chunk c (of 8 values) of row r in a tile: blocks of
// 64 columns, the chunk index XORed with row % 8 inside a 128-byte row (the
// layout TMA writes and tcgen05 reads).
__device__ __forceinline__ uint32_t tile_chunk(int r, int c) {
    return (uint32_t)((c >> 3) * (kKeys * 128) + r * 128 + (((c ^ r) & 7) << 4));
}

template <typename T, int D, int SRC>
__global__ void __launch_bounds__(TilePlan<D, SRC>::kThreads, 1) attn_tile_kernel(const __grid_constant__ TileParams tp) {
    using P = TilePlan<D, SRC>;
    constexpr int NS = P::kSlots, NST = P::kStages;
    constexpr bool kPagedSrc = SRC != kPacked;
    const AttnParams& p = tp.a;
    extern __shared__ uint8_t smem_raw[];
    __shared__ Unit su;
    __shared__ int work_here;
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t sb = (raw + 1023u) & ~1023u;
    uint8_t* sgen = smem_raw + (sb - raw);
    const uint32_t bars = sb + P::kBarOff;
    const uint32_t q_full = bars, v_fixed = bars + 8u;
    auto s_full = [&](int t) { return bars + 8u * (2 + t); };    // scores of half t are in TMEM
    auto p_full = [&](int t, int h) { return bars + 8u * (4 + 2 * t + h); };  // probabilities of its keys 64 h .. are
    auto pv_done = [&](int t) { return bars + 8u * (8 + t); };   // its output is complete
    auto full = [&](int s) { return bars + 8u * (10 + s); };
    auto empty = [&](int s) { return bars + 8u * (10 + NS + s); };
    auto st_full = [&](int s) { return bars + 8u * (10 + 2 * NS + s); };
    auto st_empty = [&](int s) { return bars + 8u * (10 + 2 * NS + NST + s); };
    const uint32_t tmem_slot = bars + 8u * (10 + 2 * NS + 2 * NST);
    auto slot = [&](int s) { return sb + P::kKvOff + s * P::kTileBytes; };
    auto stage = [&](int s) { return sb + P::kStageOff + s * P::kStageBytes; };

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (warp == 0) {
        Unit u;
        const bool any = find_unit<kPagedSrc>(p, tp.nt, tp.sms, (int)blockIdx.x, lane, u);
        if (lane == 0) {
            su = u;
            work_here = any;
        }
    }
    if (threadIdx.x == 32) {
        mbar_init(q_full, 1);
        mbar_init(v_fixed, 1);
        for (int t = 0; t < 2; ++t) {
            mbar_init(s_full(t), 1);
            mbar_init(p_full(t, 0), 4);
            mbar_init(p_full(t, 1), 4);
            mbar_init(pv_done(t), 1);
        }
        for (int s = 0; s < NS; ++s) {
            mbar_init(full(s), SRC == kPaged8 ? kConvWarps : 1);
            mbar_init(empty(s), 1);
        }
        for (int s = 0; s < NST; ++s) {
            mbar_init(st_full(s), 33);  // the producer's bytes; its lanes' copies of the scales
            mbar_init(st_empty(s), kConvWarps);
        }
        mbar_fence_init();
        tma_prefetch_desc(&tp.tm_q);
        tma_prefetch_desc(&tp.tm_k);
        tma_prefetch_desc(&tp.tm_v);
        tma_prefetch_desc(&tp.tm_o);
    }
    if (warp == 8) {  // beside the search
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(sgen + P::kBarOff + (tmem_slot - bars));
    if (!work_here) {
        if (kPagedSrc && blockIdx.x == 0 && threadIdx.x < 2) tp.joins[threadIdx.x] = 0;
        if (warp == 8) tmem_dealloc(tmem, 512);
        return;
    }
    const Unit& u = su;  // read where it is used: its fields would take the softmax threads' registers
    const int n = u.tiles;
    const int halves = u.tok0 + tp.nt < u.n ? 2 : 1;
    const int key0 = u.tile0 * kKeys;
    // keys past the sequence's end in the last tile here
    const int last_keys = min(kKeys, u.len - (key0 + (n - 1) * kKeys));

    if (warp < 8) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(P::kRegsSoftmax));
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(P::kRegsOther));

    if (warp < 8) {
        // ------------------------------------------------------- softmax
        const int t = warp >> 2;
        const int r = threadIdx.x & 127;  // row of the tile
        const int tok = u.tok0 + t * tp.nt + r / p.G;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + t * 128 + lanes, to = tmem + 256 + t * D + lanes;
        const float c = p.scale_log2;
        // the row's last visible key, and the first one any row of the half cannot see
        const int lim = p.causal ? min(u.len - 1, u.past + tok) : u.len - 1;
        const int lim0 = p.causal ? min(u.len - 1, u.past + u.tok0 + t * tp.nt) : u.len - 1;
        // rows past the tile's tokens or the sequence compute whatever is there, and have no say in the others'
        const bool mine = r < tp.nt * p.G && tok < u.n;
        float m = -INFINITY;
        uint64_t l2 = f2_pack(0.f, 0.f);
        bool ok = true;
        if (t < halves) {
            const bool frees = r == 0 && t == halves - 1;  // hands the k and v slots back
            int sv = NS - 1, sk = 0;                       // slots of V_i-1 and K_i
            for (int i = 0; i < n; ++i) {
                if (!(ok = warp_wait(s_full(t), i & 1))) break;
                tc_fence_after_sync();
                // the scores of both halves are there, so nothing reads this tile's k any more, nor the last one's v
                if (frees) {
                    mbar_arrive(empty(sk));
                    if (i > 0) mbar_arrive(empty(sv));
                }
                sv = sv + 2 >= NS ? sv + 2 - NS : sv + 2;
                sk = sk + 2 >= NS ? sk + 2 - NS : sk + 2;
                uint32_t s[4][32];
#pragma unroll
                for (int k = 0; k < 4; ++k) tmem_ld_32x32b_x32(ts + 32 * k, s[k]);
                tmem_ld_wait();
                const int kb = key0 + i * kKeys;
                if (kb + kKeys - 1 > lim0) {
                    const int see = lim - kb;
#pragma unroll
                    for (int k = 0; k < 128; ++k)
                        if (k > see) s[k >> 5][k & 31] = 0xff800000u;
                }
                float mx[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    mx[k] = __uint_as_float(s[k][0]);
#pragma unroll
                    for (int j = 1; j < 31; j += 2)
                        mx[k] = max3(mx[k], __uint_as_float(s[k][j]), __uint_as_float(s[k][j + 1]));
                    mx[k] = fmaxf(mx[k], __uint_as_float(s[k][31]));
                }
                const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                if (__any_sync(0xffffffffu, mine && (top - m) * c > kGrow)) {
                    const float mn = fmaxf(m, top);
                    const float f = mn == m ? 1.f : ex2((m - mn) * c);
                    m = mn;
                    float la, lb;
                    f2_unpack(l2, la, lb);
                    l2 = f2_pack(la * f, lb * f);
                    if (i > 0) {
                        // (this tile's scores were computed after the last one's products)
#pragma unroll 1
                        for (int k = 0; k < D / 32; ++k) {
                            uint32_t o[32];
                            tmem_ld_32x32b_x32(to + 32 * k, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
                            tmem_st_32x32b_x32(to + 32 * k, o);
                        }
                    }
                }
                const float neg = m == -INFINITY ? 0.f : -m * c;
                const uint64_t c2 = f2_pack(c, c), n2 = f2_pack(neg, neg);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    uint32_t w[32];
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        const uint32_t* x = &s[2 * k + (j >> 4)][(2 * j) & 31];
                        float a, b;
                        f2_unpack(f2_fma(f2_pack(__uint_as_float(x[0]), __uint_as_float(x[1])), c2, n2), a, b);
                        a = ex2(a);
                        b = ex2(b);
                        l2 = f2_add(l2, f2_pack(a, b));
                        w[j] = pack2<T>(a, b);
                    }
                    tmem_st_32x32b_x32(ts + 32 * k, w);
                    tmem_st_wait();
                    tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(p_full(t, k));
                }
            }
            // ------------------------------------------------------ output
            float la, lb;
            f2_unpack(l2, la, lb);
            float l = la + lb;
            if (n > 0 && ok) ok = warp_wait(pv_done(t), 0);
            tc_fence_after_sync();
            const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
            float4* pdst = u.slot < 0 ? nullptr
                                      : reinterpret_cast<float4*>(tp.part) + (int64_t)u.slot * (D / 4) * kRows + t * kRowsT + r;
            const uint32_t tile = sb + t * P::kTileBytes;  // this half's q, which no MMA reads any more
            float bad = 0.f;
#pragma unroll 1
            for (int k = 0; k < D / 64; ++k) {
                uint32_t o[2][32];
                if (n > 0) {
                    tmem_ld_32x32b_x32(to + 64 * k, o[0]);
                    tmem_ld_32x32b_x32(to + 64 * k + 32, o[1]);
                    tmem_ld_wait();
                } else {
#pragma unroll
                    for (int j = 0; j < 32; ++j) o[0][j] = o[1][j] = 0u;
                }
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    float f[32];
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        f[j] = __uint_as_float(o[y][j]);
                        bad = fmaf(f[j], 0.f, bad);  // NaN where a value is not finite
                    }
                    if (pdst) {
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            if (mine) pdst[(16 * k + 8 * y + j) * kRows] = make_float4(f[4 * j], f[4 * j + 1], f[4 * j + 2], f[4 * j + 3]);
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            sts128(tile + tile_chunk(r, 8 * k + 4 * y + j),
                                   make_uint4(pack2<T>(f[8 * j] * inv, f[8 * j + 1] * inv),
                                              pack2<T>(f[8 * j + 2] * inv, f[8 * j + 3] * inv),
                                              pack2<T>(f[8 * j + 4] * inv, f[8 * j + 5] * inv),
                                              pack2<T>(f[8 * j + 6] * inv, f[8 * j + 7] * inv)));
                    }
                }
            }
            if (pdst)
                *reinterpret_cast<float2*>(tp.stat + ((int64_t)u.slot * kRows + t * kRowsT + r) * 2) = make_float2(m * c, l);
            // rows that values behind the mask have spoilt (a sum that is NaN is so by what the row sees)
            const int end = key0 + n * kKeys;
            unsigned again = __ballot_sync(0xffffffffu, ok && mine && end - 1 > lim && bad != bad && l == l);
            if (again) {
                const int j0 = __reduce_min_sync(0xffffffffu, (again >> lane) & 1 ? lim + 1 : end);
                const int last = last_not_finite<T, D, SRC>(p, RowOf{u.b, u.hk, u.first}, max(j0, key0), min(u.len, end), lane);
                again &= __ballot_sync(0xffffffffu, lim < last);
            }
            if (!pdst) {
                fence_proxy_async_smem();
                const bool plain = bar_or_half(t, again != 0 || !ok) || u.tok0 + (t + 1) * tp.nt > u.n;
                if (!plain) {
                    if (r == 0) {
#pragma unroll
                        for (int h = 0; h < P::kHalves; ++h)
                            tma_store_3d(&tp.tm_o, tile + h * P::kBlock, h * 64, u.hk * p.G, u.first + u.tok0 + t * tp.nt);
                        tma_store_wait();
                    }
                } else {
                    // the sequence ends inside the tile (or rows follow): a warp's 32 rows, chunk by chunk
                    constexpr int C = D / 8, S = 32 / C;
                    const int ch = lane % C, rw = (r & ~31) + lane / C;
                    int tw = rw / p.G, hw = rw - tw * p.G;
                    const int qs = S / p.G, rs = S - qs * p.G;
#pragma unroll
                    for (int i = 0; i < C; ++i) {
                        const uint4 x = lds128(tile + tile_chunk(rw + i * S, ch));
                        if (tw < tp.nt && u.tok0 + t * tp.nt + tw < u.n)
                            *reinterpret_cast<uint4*>(p.out + (int64_t)(u.first + u.tok0 + t * tp.nt + tw) * p.o_tok +
                                                      (u.hk * p.G + hw) * p.o_head + ch * 8) = x;
                        tw += qs;
                        hw += rs;
                        if (hw >= p.G) {
                            hw -= p.G;
                            ++tw;
                        }
                    }
                }
            }
            __syncwarp();
            while (again) {
                const int x = __ffs(again) - 1;
                again &= again - 1;
                const int rx = (r & ~31) + x, tx = __shfl_sync(0xffffffffu, tok, x), hx = rx % p.G;
                const int j1 = __shfl_sync(0xffffffffu, lim, x) + 1;
                float o[D / 32], mx, lx;
                row_alone<T, D, SRC>(p, RowOf{u.b, u.hk, u.first}, tx * p.G + hx, key0, min(j1, end), lane, o, mx, lx);
                if (u.slot < 0) {
                    const float ix = lx > 0.f ? 1.f / lx : (lx == lx ? 0.f : lx);
                    uint16_t* d = p.out + (int64_t)(u.first + tx) * p.o_tok + (u.hk * p.G + hx) * p.o_head + lane * (D / 32);
#pragma unroll
                    for (int j = 0; j < D / 32; j += 2)
                        *reinterpret_cast<uint32_t*>(d + j) = pack2<T>(o[j] * ix, o[j + 1] * ix);
                } else {
                    const int64_t at = (int64_t)u.slot * kRows + t * kRowsT + rx;
#pragma unroll
                    for (int j = 0; j < D / 32; ++j) {
                        const int d = lane * (D / 32) + j;
                        tp.part[(((int64_t)u.slot * (D / 4) + (d >> 2)) * kRows + t * kRowsT + rx) * 4 + (d & 3)] = o[j];
                    }
                    if (lane == 0) {
                        tp.stat[at * 2] = mx;
                        tp.stat[at * 2 + 1] = lx;
                    }
                }
            }
        }
    } else if (warp == 8) {
        // ------------------------------------------------------ MMA issue
        // The whole warp runs the loop and one lane of it issues: addresses and descriptors are then the same in all
        // lanes by construction, and stay in uniform registers, where the MMAs want them.
        if (n > 0) {
            constexpr uint32_t fmt = ActTraits<T>::kIsF16 ? 0u : 1u;
            constexpr uint32_t id_s = umma_idesc_f16(fmt, kRowsT, kKeys);
            constexpr uint32_t id_o = umma_idesc_f16(fmt, kRowsT, D) | (1u << 16);  // V is stored with N contiguous
            constexpr uint32_t kTile16 = P::kTileBytes >> 4, kBlock16 = P::kBlock >> 4;
            // descriptors hold addresses in units of 16 bytes: a tile's or block's offset is added to them as it is
            const uint64_t dq = umma_desc_sw128(sb), dk = umma_desc_sw128(slot(0)), dv = umma_desc_mn_sw128(slot(0), P::kBlock);
            const uint32_t me = elect_one();
            const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
            auto issue_s = [&](int t, int sl) {
                const uint64_t q0 = dq + (uint32_t)t * kTile16, k0 = dk + (uint32_t)sl * kTile16;
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    const uint32_t off = (k >> 2) * kBlock16 + (k & 3) * 2;
                    umma_f16_if(me, tm + t * 128, q0 + off, k0 + off, id_s, k > 0);
                }
            };
            const int nh = __shfl_sync(0xffffffffu, halves, 0), nn = __shfl_sync(0xffffffffu, n, 0);
            const bool fix = SRC != kPaged8 && last_keys < kKeys;
            bool ok = warp_wait(q_full, 0) && warp_wait(full(0), 0);
            tc_fence_after_sync();
            for (int t = 0; ok && t < nh; ++t) {
                issue_s(t, 0);
                umma_commit_if(me, s_full(t));
            }
            // tiles arrive as K0 V0 K1 V1 ...
            int sv = 1 % NS, sk = 2 % NS, pv = 0, pk = 2 / NS & 1;  // slots of V_i and K_i+1, their phases
            auto arrived = [&](int i) {
                return warp_wait(full(sv), pv) && (i + 1 < nn ? warp_wait(full(sk), pk) : !fix || warp_wait(v_fixed, 0));
            };
            ok = ok && arrived(0);
            for (int i = 0; ok && i < nn; ++i) {
                const bool more = i + 1 < nn;
                const uint64_t v0 = dv + (uint32_t)sv * kTile16;
                const int slot_k = sk;
                for (int t = 0; t < nh; ++t) {
                    const uint32_t ts = tm + t * 128, to = tm + 256 + t * D;
                    // the first 64 keys' products run while the other probabilities are computed
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (!(ok = warp_wait(p_full(t, h), i & 1))) break;
                        tc_fence_after_sync();
#pragma unroll
                        for (int k = 4 * h; k < 4 * h + 4; ++k)
                            umma_f16_ts_if(me, to, ts + 8 * k, v0 + k * 128, id_o, i > 0 || k > 0);
                    }
                    if (!ok) break;
                    // one commit a tile (the next scores, over P in TMEM: the MMAs of a thread run in order); the
                    // slots are handed back by the softmax that sees it: a commit holds the issuing thread up until
                    // the MMAs before it are nearly done, so the next tiles' arrival is looked at before it
                    if (more) issue_s(t, slot_k);
                    if (t + 1 == nh) {
                        sv += 2, sk += 2;
                        if (sv >= NS) sv -= NS, pv ^= 1;
                        if (sk >= NS) sk -= NS, pk ^= 1;
                        if (more) ok = arrived(i + 1);
                    }
                    umma_commit_if(me, more ? s_full(t) : pv_done(t));
                }
            }
        }
        __syncwarp();
    } else if (warp == 9) {
        // -------------------------------------------------- TMA producer
        bool ok = true;
        int g = 0;
        constexpr int NR = SRC == kPaged8 ? NST : NS;
        auto rfull = [&](int s) { return SRC == kPaged8 ? st_full(s) : full(s); };
        auto rempty = [&](int s) { return SRC == kPaged8 ? st_empty(s) : empty(s); };
        if (lane == 0 && n > 0) {
            mbar_arrive_expect_tx(q_full, halves * P::kHalves * tp.nt * p.G * 128);
            for (int t = 0; t < halves; ++t)
#pragma unroll
                for (int h = 0; h < P::kHalves; ++h)
                    tma_load_3d(sb + t * P::kTileBytes + h * P::kBlock, &tp.tm_q, q_full, h * 64, u.hk * p.G,
                                u.first + u.tok0 + t * tp.nt);
        }
        int ids = 0;  // paged: the page of this lane's 16 keys of a window of 4 tiles; one outside the pool reads as zeros
        for (int i = 0; i < n && ok; ++i) {
            const int kb = key0 + i * kKeys;
            int id = 0, y = 0, keys = kKeys;
            if constexpr (kPagedSrc) {
                if ((i & 3) == 0) {
                    const int key = min(kb + lane * 16, u.len - 1);
                    ids = p.table[(int64_t)u.b * p.table_cols + (key >> p.log2_page)];
                    if (ids < 0 || ids >= p.num_pages) ids = (int)p.num_pages;
                }
                id = __shfl_sync(0xffffffffu, ids, 8 * (i & 3) + (lane & 7));
                y = (kb + (lane & 7) * 16) & (p.page_size - 1);
                keys = (min(kKeys, u.len - kb) + p.page_size - 1) & -p.page_size;  // whole pages
            }
            for (int kv = 0; kv < 2 && ok; ++kv, ++g) {
                const int s = g % NR, use = g / NR;
                if (use > 0 && !(ok = warp_wait(rempty(s), (use - 1) & 1))) break;
                const CUtensorMap* map = kv ? &tp.tm_v : &tp.tm_k;
                if constexpr (SRC == kPacked) {
                    if (lane == 0) {
                        mbar_arrive_expect_tx(rfull(s), P::kTileBytes);
#pragma unroll
                        for (int h = 0; h < P::kHalves; ++h)
                            tma_load_3d(slot(s) + h * P::kBlock, map, rfull(s), h * 64, u.hk, u.first + kb);
                    }
                } else {
                    if (lane == 0) mbar_arrive_expect_tx(rfull(s), keys * (SRC == kPaged8 ? D : 2 * D));
                    __syncwarp();
                    if constexpr (SRC == kPaged8) {
                        const bool in = id < p.num_pages;
                        const int64_t row = ((int64_t)(in ? id : 0) * p.Hkv + u.hk) * p.page_size + y;
                        if (lane < 8) cp_async16(stage(s) + kKeys * D + lane * 16, (kv ? p.v_exp : p.k_exp) + row, in);
                        cp_async_arrive(rfull(s));
                    }
                    if (lane * 16 < keys && y == 0) {  // a page begins here (tiles begin with a page)
                        const int z = id * p.Hkv + u.hk;
                        if constexpr (SRC == kPaged8) {
                            tma_load_3d(stage(s) + lane * 16 * D, map, rfull(s), 0, 0, z);
                        } else {
#pragma unroll
                            for (int h = 0; h < P::kHalves; ++h)
                                tma_load_3d(slot(s) + h * P::kBlock + lane * 16 * 128, map, rfull(s), h * 64, 0, z);
                        }
                    }
                }
            }
        }
        if (SRC != kPaged8 && ok && n > 0 && last_keys < kKeys) {
            // v rows behind the sequence's end: zeros, as their probabilities are
            const int gl = 2 * n - 1, s = gl % NS;
            if ((ok = warp_wait(full(s), (gl / NS) & 1))) {
                for (int x = last_keys * (D / 8) + lane; x < kKeys * (D / 8); x += 32)
                    sts128(slot(s) + tile_chunk(x / (D / 8), x % (D / 8)), make_uint4(0u, 0u, 0u, 0u));
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(v_fixed);
            }
        }
        // no copy may still be landing when the CTA exits
        if (n > 0) warp_wait(q_full, 0);
        for (int j = g > NR ? g - NR : 0; j < g; ++j) mbar_wait(rfull(j % NR), (j / NR) & 1);
    } else if (warp == 10) {
        if constexpr (kPagedSrc) {
            if (blockIdx.x == 0) list_joins(p, tp.nt, tp.sms, lane, tp.joins);
        }
    } else if constexpr (SRC == kPaged8) {
        if (warp >= 12) {
            // ------------------------------------------- codes -> 16-bit tiles
            constexpr int C = D / 16;             // 16-code chunks of a row
            constexpr int R = 32 * kConvWarps / C;  // rows of one round
            const int tid = threadIdx.x - 384;
            const int ch = tid % C, r0 = tid / C;
            bool ok = true;
            for (int i = 0; i < n && ok; ++i) {
                const int kb = key0 + i * kKeys;
                const int keys = min(kKeys, u.len - kb);
                for (int kv = 0; kv < 2 && ok; ++kv) {
                    const int g = 2 * i + kv, st = g % NST, s = g % NS;
                    if (!(ok = warp_wait(st_full(st), (g / NST) & 1))) break;
                    if (g >= NS && !(ok = warp_wait(empty(s), (g / NS - 1) & 1))) break;
#pragma unroll
                    for (int x = 0; x < kKeys / R; ++x) {
                        const int r = r0 + x * R;
                        uint4 lo = make_uint4(0u, 0u, 0u, 0u), hi = lo;
                        if (r < keys) {
                            const uint4 q = lds128(stage(st) + r * D + ch * 16);
                            uint32_t o[8];
                            codes_to_16<T>(q, lds8(stage(st) + kKeys * D + r), o);
                            lo = make_uint4(o[0], o[1], o[2], o[3]);
                            hi = make_uint4(o[4], o[5], o[6], o[7]);
                        }
                        // (the two column blocks' lanes write their chunks in opposite order: no bank twice)
                        const int odd = (ch >> 2) & 1;
                        sts128(slot(s) + tile_chunk(r, 2 * ch + odd), odd ? hi : lo);
                        sts128(slot(s) + tile_chunk(r, 2 * ch + 1 - odd), odd ? lo : hi);
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(full(s));
                        mbar_arrive(st_empty(st));
                    }
                }
            }
        }
    }
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 8) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, 512);
    }
}

// Joins the parts of the row tiles whose keys several CTAs shared.  A piece of
// work is 32 rows (a lane each) of 16 columns.  Up to eight parts: a piece per
// warp.  More: a piece per block, its parts go to the eight warps in turn, and
// the warps' sums are added in their order.  Either way the order of the sums does
// not depend on timing.
template <typename T, int D>
__global__ void __launch_bounds__(32 * kJoinWarps) attn_tile_join_kernel(const __grid_constant__ TileParams tp) {
    const AttnParams& p = tp.a;
    __shared__ float sh[kJoinWarps][18][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int kPieces = (kRows / 32) * (D / 16), kGroups = kPieces / kJoinWarps;
    const int groups = tp.joins[0] * kGroups, items = groups + tp.joins[1] * kPieces;
    const Join* list = reinterpret_cast<const Join*>(tp.joins + 2);
    for (int i = blockIdx.x; i < items; i += gridDim.x) {
        const bool many = i >= groups;
        const Join j = list[many ? kMaxJoins - 1 - (i - groups) / kPieces : i / kGroups];
        // the 16 columns vary fastest: a group of 8 pieces shares its rows' statistics
        const int piece = many ? (i - groups) % kPieces : (i % kGroups) * kJoinWarps + warp;
        const int rg = piece / (D / 16), col = piece % (D / 16);
        const int r = rg * 32 + lane, rt = r & (kRowsT - 1), tk = j.tok0 + (r >> 7) * tp.nt + rt / p.G;
        const bool mine = rt < tp.nt * p.G && tk < j.n;
        if (!__any_sync(0xffffffffu, mine)) continue;  // many: the same for all warps
        float m = -INFINITY, l = 0.f, o[16];
#pragma unroll
        for (int x = 0; x < 16; ++x) o[x] = 0.f;
#pragma unroll 2
        for (int s = many ? warp : 0; s < j.parts; s += many ? kJoinWarps : 1) {
            const int64_t at = j.slot + s * p.Hkv;
            const float2 st = *reinterpret_cast<const float2*>(tp.stat + (at * kRows + r) * 2);
            float4 v[4];
#pragma unroll
            for (int x = 0; x < 4; ++x)
                v[x] = reinterpret_cast<const float4*>(tp.part)[(at * (D / 4) + col * 4 + x) * kRows + r];
            const float mn = fmaxf(m, st.x), ref = mn == -INFINITY ? 0.f : mn;
            const float keep = exp2f(m - ref), f = exp2f(st.x - ref);
            m = mn;
            l = l * keep + st.y * f;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                o[4 * x] = o[4 * x] * keep + v[x].x * f;
                o[4 * x + 1] = o[4 * x + 1] * keep + v[x].y * f;
                o[4 * x + 2] = o[4 * x + 2] * keep + v[x].z * f;
                o[4 * x + 3] = o[4 * x + 3] * keep + v[x].w * f;
            }
        }
        uint16_t* out = p.out + (int64_t)(j.first + tk) * p.o_tok + (j.hk * p.G + rt % p.G) * p.o_head + col * 16;
        if (!many) {
            const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
            if (mine)
#pragma unroll
                for (int x = 0; x < 2; ++x)
                    reinterpret_cast<uint4*>(out)[x] =
                        make_uint4(pack2<T>(o[8 * x] * inv, o[8 * x + 1] * inv), pack2<T>(o[8 * x + 2] * inv, o[8 * x + 3] * inv),
                                   pack2<T>(o[8 * x + 4] * inv, o[8 * x + 5] * inv),
                                   pack2<T>(o[8 * x + 6] * inv, o[8 * x + 7] * inv));
            continue;
        }
        sh[warp][16][lane] = m;
        sh[warp][17][lane] = l;
#pragma unroll
        for (int x = 0; x < 16; ++x) sh[warp][x][lane] = o[x];
        __syncthreads();
        float all = -INFINITY, sum = 0.f;
#pragma unroll
        for (int y = 0; y < kJoinWarps; ++y) all = fmaxf(all, sh[y][16][lane]);
        const float ref = all == -INFINITY ? 0.f : all;
        float a[2] = {0.f, 0.f};  // this warp's two of the 16 columns
#pragma unroll
        for (int y = 0; y < kJoinWarps; ++y) {
            const float f = exp2f(sh[y][16][lane] - ref);
            sum += sh[y][17][lane] * f;
            a[0] += sh[y][2 * warp][lane] * f;
            a[1] += sh[y][2 * warp + 1][lane] * f;
        }
        const float inv = sum > 0.f ? 1.f / sum : (sum == sum ? 0.f : sum);
        if (mine) *reinterpret_cast<uint32_t*>(out + 2 * warp) = pack2<T>(a[0] * inv, a[1] * inv);
        __syncthreads();
    }
}

template <typename T, int D, int SRC>
int launch_tile(const AttnParams& a, cudaStream_t stream) {
    using P = TilePlan<D, SRC>;
    TileParams tp;
    tp.a = a;
    tp.sms = device_sm_count();
    tp.nt = kRowsT / a.G;
    int rc;
    const CUtensorMapDataType act = ActTraits<T>::kIsF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    // the strides of a single head or token are never used
    const uint64_t qt = a.T == 1 ? D * 2 : a.q_tok * 2, qh = a.Hq == 1 ? D * 2 : a.q_head * 2;
    const uint64_t ot = a.T == 1 ? D * 2 : a.o_tok * 2, oh = a.Hq == 1 ? D * 2 : a.o_head * 2;
    if ((rc = encode_3d(&tp.tm_q, act, a.q, D, a.Hq, a.T, qh, qt, 64, a.G, tp.nt, CU_TENSOR_MAP_SWIZZLE_128B, "q")) ||
        (rc = encode_3d(&tp.tm_o, act, a.out, D, a.Hq, a.T, oh, ot, 64, a.G, tp.nt, CU_TENSOR_MAP_SWIZZLE_128B, "out")))
        return rc;
    const CUtensorMapDataType dt = SRC == kPaged8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : act;
    if constexpr (SRC == kPacked) {
        const uint64_t kh = a.Hkv == 1 ? D * 2 : a.k_head * 2, vh = a.Hkv == 1 ? D * 2 : a.v_head * 2;
        const uint64_t kt = a.T == 1 ? D * 2 : a.k_tok * 2, vt = a.T == 1 ? D * 2 : a.v_tok * 2;
        if ((rc = encode_3d(&tp.tm_k, dt, a.k, D, a.Hkv, a.T, kh, kt, 64, 1, kKeys, CU_TENSOR_MAP_SWIZZLE_128B, "k")) ||
            (rc = encode_3d(&tp.tm_v, dt, a.v, D, a.Hkv, a.T, vh, vt, 64, 1, kKeys, CU_TENSOR_MAP_SWIZZLE_128B, "v")))
            return rc;
    } else {
        constexpr int es = SRC == kPaged8 ? 1 : 2;
        const uint64_t pg = (uint64_t)a.num_pages * a.Hkv, ps = a.page_size;
        const CUtensorMapSwizzle sw = SRC == kPaged8 ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B;
        const uint32_t box = SRC == kPaged8 ? D : 64;
        if ((rc = encode_3d(&tp.tm_k, dt, a.k_cache, D, ps, pg, D * es, ps * D * es, box, ps, 1, sw, "k_cache")) ||
            (rc = encode_3d(&tp.tm_v, dt, a.v_cache, D, ps, pg, D * es, ps * D * es, box, ps, 1, sw, "v_cache")))
            return rc;
    }
    tp.joins = reinterpret_cast<int*>(static_cast<uint8_t*>(a.ws) + WLQ_ATTENTION_ZERO_BYTES);
    static_assert(sizeof(Join) == 24, "the list's entries");
    tp.part = reinterpret_cast<float*>(tp.joins) + kJoinListBytes / 4;
    tp.stat = tp.part + (size_t)kPartsPerSm * tp.sms * kRows * D;
    // the most CTAs there can be work for: those beyond what there is start, search and end, 1.7 us per 148 of them
    // (3 x 196 tokens over 3071, 10 heads over 5, D 64: 23.3 us, 28.8 with 3 x 148 CTAs more than row tiles)
    int64_t grid = (a.T / (2 * tp.nt) + a.B) * a.Hkv;
    const int64_t tiles = SRC == kPacked ? 0 : ((a.table_cols << a.log2_page) + kKeys - 1) / kKeys;
    const bool shares = tiles > kFewTiles;
    if (shares) {
        // an even share: a row tile that is split has more than an SM's share, and so adds at most that many parts
        const int64_t most = a.B > kLanesSeqs ? grid + tp.sms : std::max(grid, (int64_t)kPartsPerSm * tp.sms);
        grid = std::min(grid * ((tiles + kFewTiles - 1) / kFewTiles), most);
    }
    if (grid > 0x7fffffff) return fail(WLQ_ERR_UNSUPPORTED, "attention: %lld row tiles in one call", (long long)grid);
    auto kernel = attn_tile_kernel<T, D, SRC>;
    static OncePerDevice limit;
    if ((rc = allow_shared_memory(limit, kernel, P::kAlloc, "attn_tile_kernel shared memory"))) return rc;
    kernel<<<(unsigned)grid, P::kThreads, P::kAlloc, stream>>>(tp);
    if ((rc = check_cuda(cudaGetLastError(), "attn_tile_kernel"))) return rc;
    if (shares) {
        attn_tile_join_kernel<T, D><<<4 * tp.sms, 32 * kJoinWarps, 0, stream>>>(tp);
        rc = check_cuda(cudaGetLastError(), "attn_tile_join_kernel");
    }
    return rc;
}

template <typename T>
int launch_tile_any(const AttnParams& a, cudaStream_t stream) {
    if (!a.k_cache) return a.D == 64 ? launch_tile<T, 64, kPacked>(a, stream) : launch_tile<T, 128, kPacked>(a, stream);
    if (a.k_exp) return a.D == 64 ? launch_tile<T, 64, kPaged8>(a, stream) : launch_tile<T, 128, kPaged8>(a, stream);
    return a.D == 64 ? launch_tile<T, 64, kPaged>(a, stream) : launch_tile<T, 128, kPaged>(a, stream);
}

}  // namespace

}  // namespace wlq
