// paged_attn.cuh — attention over the paged 8-bit cache (kv_cache.cuh): what the
// kernels share, and the kernel for few query rows (decode).
//
// Row (token i, head hq) of a sequence with q_len new tokens and kv_len cached
// ones (the new ones included) sees the keys j < limit, limit = kv_len - q_len
// + i + 1 (causal) or kv_len:
//   z_j = scale * k_scale[page(j)] * <q, kc_j>,  out = sum_j softmax(z)_j v_scale[page(j)] vc_j
// and lse = log sum_j exp(z_j). A row that sees nothing gives 0 and -inf.
//
// Numbers. An int8 or e4m3 code is exact in fp16, so the products run on fp16
// tensor cores with the page scales applied in fp32 around them. q is brought
// to fp16 by a power of two per row: one term holds an fp16 or bf16 value
// exactly; an fp32 value takes two (22 bits, the second the rounding error of
// the first). What enters the second product is a key's contribution P_j =
// 2^(z_j - ref) * v_scale[page(j)] / unit, the same way: one fp16 term for 16-bit
// outputs, two for fp32. The unit is a power of two near the first pages' scales,
// ref a whole number per row that follows the row's largest contribution, not its
// largest score: set so that this one lies in [2^5, 2^6), and moved when one would
// pass 2^15. So a row keeps 2^-30 of its largest contribution (half a step of
// fp16's smallest numbers) however far the scales of pages lie apart that it
// does not see or gives no weight. (With a unit that followed the largest scale
// of the tile, one page of 10^6 times the other scales left the others five
// bits.) ref moves once or twice in a row's life; set only 3 (in log2) under its
// limit, some row of a warp moved it in every second or third tile, and each
// time O is rescaled. The row sums of 2^(z_j - ref) are fp32, which has room for
// scales 2^60 to either side of the first pages'. Sums are fp32.
// The tensor cores cut a sum's bits below fp32 off instead of rounding them, so
// every accumulation step loses a little on the same side (fp32 q, a row over
// 9000 keys, 1130 steps: 1.6e-5 off in the 2-norm; 272 steps: 3.5e-6). After
// some 100 steps the accumulators are therefore added into the workspace,
// rounded to nearest (attn_flush4), and begin at 0 again, and second terms of q
// and P are added before first ones, into small sums: 2.6e-6 and 1.9e-6 where
// fp32 products and a fp32 softmax are 2.2e-6 off. The flushes cost 2 % of a decode
// step over 100k keys, 7 % of a fp32 chunk (every 8 tiles instead of 6: 3 % less, 3.0e-6).
//
// Work. The query rows of one kv head and sequence, (token, head of the group)
// in that order, form row tiles of kRows rows; a unit is (sequence, row tile,
// kv head) with its visible keys in tiles. All units in a row, each as long as
// its tiles plus what beginning it costs in tiles (START), form one range that is
// cut into equal shares, one per CTA: ragged batches, causal triangles and one
// long sequence balance alike (without START a CTA could draw a dozen units of
// one tile: 32 ragged requests took 231 us, equal ones 127). A unit that is cut leaves
// partial sums, softmax reference and row sums in the workspace, which
// attn_combine_kernel joins in key order (same split, same result).
#pragma once

#include <cuda.h>

#include "common.cuh"
#include "gemm_tc.cuh"   // TMA and mbarrier helpers
#include "kv_cache.cuh"

namespace cpq {

constexpr int kAttnMaxSeqs = 1024;

struct alignas(64) AttnArgs {
    CUtensorMap tmap_k, tmap_v;  // codes as [D / 128][n_pages * n_head_kv * block][128] bytes, box 128 x min(block, 32) x D / 128
    const uint8_t *k, *v;
    const float *k_scale, *v_scale;
    int64_t n_pages;
    int block, hkv;
    const void *q;
    int64_t qs_tok, qs_head;     // elements
    void *out;
    int64_t os_tok, os_head;
    float *lse;                  // [t][hkv * group], or null
    int type;                    // of q and out
    int wide;                    // q and out: 16-byte aligned rows
    int t, group, n_seqs;
    const int32_t *seq_start, *kv_len, *table;
    int64_t table_stride;
    int max_blocks, causal;
    float scale_log2;            // softmax scale * log2(e)
    int min_share;               // a CTA's share is at least this many places
    // workspace: two slots per CTA (the unit that ends in it, the unit that begins in it)
    float *part_o;               // [slot][kRows][D]
    float2 *part_ml;             // [slot][kRows]: softmax reference, row sum
    int4 *part_hdr;              // [slot]: sequence, row tile, kv head, 0 unused | 1 goes on | 2 the unit's end
    float4 *acc;                 // [CTA][kAttnAcc / 16 * D]: what accumulators held before; each element is one thread's
};
constexpr int kAttnAcc = 512;    // bytes of acc per CTA and dim (128 rows, or 8 warps of 16 accumulator rows)

// ---- the split ------------------------------------------------------------------

struct AttnSeq {
    int row0, q, kv, seen;  // first token, tokens, keys, keys the table has blocks for
};

__device__ __forceinline__ AttnSeq attn_seq(const AttnArgs &a, int s) {
    AttnSeq r;
    r.row0 = min(max(a.seq_start[s], 0), a.t);
    r.q = min(max(a.seq_start[s + 1], r.row0), a.t) - r.row0;
    r.kv = max(a.kv_len[s], 0);
    r.seen = min(r.kv, a.max_blocks * a.block);
    return r;
}

// Keys that the rows [r * rows, (r + 1) * rows) see together.
__device__ __forceinline__ int attn_kv_end(const AttnSeq &s, int r, int rows, int group, int causal) {
    if (!causal) return s.seen;
    const int last = (min(s.q * group, (r + 1) * rows) - 1) / group;
    return min(max(s.kv - s.q + last + 1, 0), s.seen);
}

__device__ __forceinline__ int attn_row_tiles(const AttnSeq &s, int rows, int group) { return (s.q * group + rows - 1) / rows; }

// Where a CTA's share begins.
struct AttnPlan {
    int s, r, h, at, left;  // unit, place in it (START places, then its tiles), and the share's places
};

// Fills the plan (all threads of the CTA; barriers inside). through: scratch of
// kAttnMaxSeqs + 1 ints, free again afterwards. A unit with no visible key
// counts one tile, so that some CTA writes its rows. Also marks the CTA's
// workspace slots unused, before any is written.
template <int ROWS, int TILE, int START>
__device__ __forceinline__ void attn_make_plan(const AttnArgs &a, AttnPlan &p, int *through) {
    if (threadIdx.x < 2) a.part_hdr[2 * blockIdx.x + threadIdx.x] = make_int4(0, 0, 0, 0);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, n_warps = blockDim.x >> 5;
    auto places = [&](const AttnSeq &s, int r) {
        return START + max(1, (attn_kv_end(s, r, ROWS, a.group, a.causal) + TILE - 1) / TILE);
    };
    for (int s = tid; s < a.n_seqs; s += blockDim.x) {
        const AttnSeq q = attn_seq(a, s);
        const int n = attn_row_tiles(q, ROWS, a.group);
        int w = -1;  // many row tiles: counted by a warp below
        if (n <= 4) {
            w = 0;
            for (int r = 0; r < n; r++) w += places(q, r);
        }
        through[s + 1] = w < 0 ? -1 : w * a.hkv;
    }
    __syncthreads();
    for (int s = warp; s < a.n_seqs; s += n_warps) {
        if (through[s + 1] >= 0) continue;
        const AttnSeq q = attn_seq(a, s);
        const int n = attn_row_tiles(q, ROWS, a.group);
        int w = 0;
        for (int r = lane; r < n; r += 32) w += places(q, r);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
        __syncwarp();
        if (lane == 0) through[s + 1] = w * a.hkv;
    }
    __syncthreads();
    if (warp == 0) {
        int sum = 0;
        for (int s0 = 0; s0 < a.n_seqs; s0 += 32) {
            int w = s0 + lane < a.n_seqs ? through[s0 + lane + 1] : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, w, o);
                if (lane >= o) w += u;
            }
            if (s0 + lane < a.n_seqs) through[s0 + lane + 1] = sum + w;
            sum += __shfl_sync(0xffffffffu, w, 31);
        }
        if (lane == 0) through[0] = 0;
        __syncwarp();
        const int n_cta = max(1, min(int(gridDim.x), sum / a.min_share));
        const int c = blockIdx.x;
        const int x0 = c < n_cta ? int(int64_t(sum) * c / n_cta) : sum;
        const int x1 = c < n_cta ? int(int64_t(sum) * (c + 1) / n_cta) : sum;
        int s = 0, r = 0, h = 0, at = 0;
        if (x1 > x0) {
            int lo = 0, hi = a.n_seqs;  // the last sequence that begins at or before x0 (and so has places there)
            while (hi - lo > 1) {
                const int mid = (lo + hi) / 2;
                if (through[mid] <= x0) lo = mid;
                else hi = mid;
            }
            s = lo;
            int rem = x0 - through[s];
            const AttnSeq q = attn_seq(a, s);
            const int n = attn_row_tiles(q, ROWS, a.group);
            for (int r0 = 0; r0 < n; r0 += 32) {  // row tiles in order, each with its hkv units
                const int mine = r0 + lane < n ? places(q, r0 + lane) * a.hkv : 0;
                int w = mine;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int u = __shfl_up_sync(0xffffffffu, w, o);
                    if (lane >= o) w += u;
                }
                const unsigned after = __ballot_sync(0xffffffffu, w > rem);
                if (after) {
                    const int i = __ffs(int(after)) - 1;
                    const int before = __shfl_sync(0xffffffffu, w - mine, i);
                    const int per = __shfl_sync(0xffffffffu, mine, i) / a.hkv;
                    r = r0 + i;
                    h = min(max((rem - before) / per, 0), a.hkv - 1);  // (within bounds whatever seq_start holds)
                    at = min(max((rem - before) - h * per, 0), per - 1);
                    break;
                }
                rem -= __shfl_sync(0xffffffffu, w, 31);
            }
        }
        if (lane == 0) p.s = s, p.r = r, p.h = h, p.at = at, p.left = x1 - x0;
    }
    __syncthreads();
}

// One unit's part in this CTA.
struct AttnUnit {
    int s, r, h;
    AttnSeq seq;
    int kv_end, t0, t1, n;  // keys seen, tiles [t0, t1) of n here
};

// Walks the CTA's units; every role of the CTA does so by itself.
template <int ROWS, int TILE, int START>
struct AttnWalk {
    const AttnArgs &a;
    int s, r, h, at, left;
    AttnSeq seq;
    __device__ AttnWalk(const AttnArgs &a_, const AttnPlan &p) : a(a_), s(p.s), r(p.r), h(p.h), at(p.at), left(p.left) {
        if (left > 0) seq = attn_seq(a, s);
    }
    __device__ bool next(AttnUnit &u) {
        if (left <= 0) return false;
        u.s = s, u.r = r, u.h = h;
        u.seq = seq;
        u.kv_end = attn_kv_end(seq, r, ROWS, a.group, a.causal);
        u.n = max(1, (u.kv_end + TILE - 1) / TILE);
        const int to = min(START + u.n, at + left);
        u.t0 = max(0, at - START);
        u.t1 = max(0, to - START);
        left -= to - at;
        at = 0;
        if (u.t1 == u.t0) return false;  // the share ends before the unit's first tile
        if (++h == a.hkv) {
            h = 0;
            if (++r == attn_row_tiles(seq, ROWS, a.group)) {
                r = 0;
                while (left > 0 && ++s < a.n_seqs) {
                    seq = attn_seq(a, s);
                    if (seq.q > 0) break;
                }
            }
        }
        return true;
    }
};

// The workspace slot of a cut unit: 0 when it began in an earlier CTA, 1 when it begins here.
__device__ __forceinline__ int attn_slot(const AttnUnit &u) { return 2 * int(blockIdx.x) + (u.t0 == 0 ? 1 : 0); }

// The page of a sequence's block b, or -1 when it is no page of the pool (its
// keys then count as absent).
__device__ __forceinline__ int attn_page(const AttnArgs &a, int s, int b) {
    if (b >= a.max_blocks) return -1;
    const int page = a.table[int64_t(s) * a.table_stride + b];
    return page >= 0 && int64_t(page) < a.n_pages ? page : -1;
}

__device__ __forceinline__ float attn_q_at(const AttnArgs &a, int64_t i) {
    if (a.type == CPQ_TYPE_F32) return static_cast<const float *>(a.q)[i];
    if (a.type == CPQ_TYPE_F16) return __half2float(static_cast<const __half *>(a.q)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16 *>(a.q)[i]);
}

__device__ __forceinline__ void attn_out_at(const AttnArgs &a, int64_t i, float v) {
    if (a.type == CPQ_TYPE_F32) static_cast<float *>(a.out)[i] = v;
    else if (a.type == CPQ_TYPE_F16) static_cast<__half *>(a.out)[i] = __float2half_rn(v);
    else static_cast<__nv_bfloat16 *>(a.out)[i] = __float2bfloat16_rn(v);
}

// 1 / sum of a row; a row that sees nothing has sum 0 and stays 0, NaN stays NaN.
__device__ __forceinline__ float attn_inverse(float sum) { return sum == 0.0f ? 0.0f : 1.0f / sum; }

// The power of two that brings a row's largest magnitude into [2^13, 2^14), as an exponent.
__device__ __forceinline__ int attn_q_shift(float amax) {
    const int e = int(__float_as_uint(amax) >> 23) - 127;  // amax >= 0; zero and subnormal: -127
    if (e == 128) return 0;                                // infinity or NaN: left as it is
    return 13 - max(e, -100);
}
__device__ __forceinline__ float attn_exp2i(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127

// Adds four accumulators to the workspace, or puts them there (a unit's first time). The additions of one thread to
// one address come in its order: results repeat.
__device__ __forceinline__ void attn_flush4(float4 *to, bool first, float a, float b, float c, float d) {
    if (first) __stcg(to, make_float4(a, b, c, d));
    else asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(to), "f"(a), "f"(b), "f"(c), "f"(d) : "memory");
}
// Scales what is there; reads it.
__device__ __forceinline__ void attn_scale4(float4 *at, float f, float g) {
    const float4 v = __ldcg(at);
    __stcg(at, make_float4(v.x * f, v.y * f, v.z * g, v.w * g));
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

constexpr float kAttnRefDrop = 5.0f;    // a row's largest contribution is 2^5 .. 2^6 when its reference is set
constexpr float kAttnRefMove = 15.0f;   // and the reference moves when one would pass 2^15
constexpr float kAttnVLow = -64.0f;     // scales under 2^-64 units count as 2^-64 for the reference (row sums stay under 2^110)
constexpr float kAttnVHigh = 0x1p90f;   // scales above this many units change the unit
constexpr float kLn2 = 0.69314718055994531f;

// 1 / unit for pages with scales up to vmax: a power of two, 0 while all are 0.
__device__ __forceinline__ float attn_v_unit(float vmax) {
    const int e = int(__float_as_uint(vmax) >> 23) - 127;
    return vmax > 0.0f ? attn_exp2i(-min(max(e, -126), 126)) : 0.0f;
}
// The unit again.
__device__ __forceinline__ float attn_v_scale(float vinv) { return vinv > 0.0f ? 1.0f / vinv : 0.0f; }
// log2 of a page's scale in units, as the reference counts it.
__device__ __forceinline__ float attn_v_log(float r) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(r));
    return fmaxf(y, kAttnVLow);
}

// lse of a row from its reference (log2, whole) and sum, whose exponent is taken apart: the logarithm of a large sum
// has a large rounding error.
__device__ __forceinline__ float attn_lse(float ref, float sum) {
    if (sum == 0.0f) return __int_as_float(0xff800000);
    const int bits = __float_as_int(sum), e = (bits >> 23) - 127;
    if (bits < 0 || e == 128) return ref + sum;  // NaN, infinity
    return ((ref + float(e)) + __log2f(__int_as_float((bits & 0x7fffff) | 0x3f800000))) * kLn2;
}

// ---- few query rows: mma.sync tiles, one key tile per warp -------------------------
//
// Decode reads the cache once and does little with it. One CTA per SM; each of
// its warps takes every kWarps-th 32-key tile with its own softmax state, output
// accumulators and copies (K two tiles ahead, V one, TMA boxes of 128 bytes x
// up to 32 keys, 128-byte swizzle), so that nothing but the end of a unit makes
// warps wait for one another. m16n8k16 fp16 MMAs: 16 rows of 16-bit q, or 8 rows
// of fp32 q with the first terms in rows 0-7 and the second terms in rows 8-15
// of the same MMA (they meet in one thread, lanes of row g hold both), so fp32
// costs no extra MMA. A warp copies for itself because a ninth warp would cost
// the others a quarter of their registers (warps are allotted in fours): with
// one, the accumulators of D = 256 spilled.
//
// Measured (24 heads over 4 of 256): 1 request over 100003 keys, fp32, 54.1 us
// (3.8 TB/s of codes, 0.58 of a measured copy; 37 % of issue slots, 25 % of the
// tensor pipe: a warp's tile is a chain of loads, conversions and MMAs, two warps a
// scheduler cannot hide all of it, and registers allow no third); 32
// ragged bf16 requests of up to 16000 keys 133 us (4.35 TB/s, 0.67); 1 request over
// 1000 keys 13.9, most of it beginning and joining.
//
// Operand order. A key tile's codes go from shared memory to the MMA's B
// registers without a transpose:
//   K: lane (g, t) takes chunks 2t, 2t + 1 (16 bytes each) of key g's 128-byte
//      half row: 32 dims 32 t + 4 j + i, MMA j of 8 taking i = 0..3 as k =
//      2t, 2t + 1, 2t + 8, 2t + 9 (q is stored in that order).
//   V: lane (g, t) takes chunk g of keys 2t, 2t + 1, 2t + 8, 2t + 9: n-tile b
//      of 16 then has column n = dim 16 n + b, its k the four keys, paired
//      from two keys' words by byte permutes.
// With the 128-byte swizzle (chunk ^ (key & 7)) each quarter warp's 16-byte
// loads touch eight different bank groups in both.

constexpr int kAttnTile = 32;

template <int D, bool SPLIT> struct DecCfg {
    static constexpr int kRows = SPLIT ? 8 : 16;
    static constexpr int kWarps = 8;                             // 255 registers (12 warps of 168: D = 128 spills, 10 % slower)
    static constexpr bool kEarlyQ = D == 128;                    // room to hold the next unit's q while one ends
    static constexpr int kThreads = 32 * kWarps;
    // tiles (two accumulation steps each) between flushes; 16-bit outputs need none (what fits the memory: 2.6e-4 off)
    static constexpr int kFlush = 64;
    static constexpr int kStart = 32;                            // beginning a unit takes about as long as this many tiles (4 to 32 tried)
    static constexpr int kCodes = kAttnTile * D;                 // K or V codes of a tile
    static constexpr int kVOff = kWarps * 2 * kCodes;            // K: two slots per warp; V: one
    static constexpr int kQOff = kVOff + kWarps * kCodes;
    static constexpr int kRedBytes = 4 * kRows * D * 4;          // four warps' accumulators, in V's place
    static constexpr int kBarOff = kQOff + D / 16 * 512;
    // stats (reference, sum) per warp and row, row factors
    static constexpr int kStatOff = kBarOff + kWarps * 3 * 8;
    static constexpr int kRowOff = kStatOff + kWarps * 16 * 8;
    static constexpr int kPlanOff = kRowOff + 16 * 4;
    static constexpr int kSmem = kPlanOff + int(sizeof(AttnPlan)) + 1024;
    static_assert(kRedBytes <= kWarps * kCodes, "the accumulators fit in V's place");
    static_assert(kVOff >= (kAttnMaxSeqs + 1) * 4, "the plan's scratch lies in K's place");
    static_assert(kSmem <= 227 * 1024, "shared memory");
};

// 3-D tiled TMA load (no multicast) completing as transaction bytes on `bar`.
__device__ __forceinline__ void tma_load_3d(void *dst, const CUtensorMap *map, int x, int y, int z, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_addr(dst)),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_addr(bar))
        : "memory");
}

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack_h2(float a, float b) { return h2u(__floats2half2_rn(a, b)); }

// Pages and scales of up to 32 of a warp's tiles, one per lane (two pages with
// 16-token pages); a page that is not there is -1.
struct DecInfo {
    int page[2];
    float ks[2], vs[2];
};

template <int D, int FMT, bool SPLIT>
__global__ void __launch_bounds__(DecCfg<D, SPLIT>::kThreads, 1) attn_decode_kernel(const __grid_constant__ AttnArgs a) {
    using C = DecCfg<D, SPLIT>;
    constexpr int kRows = C::kRows, NA = D / 128, W = C::kWarps;  // NA: 128-byte atoms per key
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint4 *sq = reinterpret_cast<uint4 *>(smem + C::kQOff);
    float *red = reinterpret_cast<float *>(smem + C::kVOff);
    float2 *stat = reinterpret_cast<float2 *>(smem + C::kStatOff);  // [warp][16 rows]: reference, sum
    float *rowf = reinterpret_cast<float *>(smem + C::kRowOff);     // [row]: 2^-shift of its q
    AttnPlan &plan = *reinterpret_cast<AttnPlan *>(smem + C::kPlanOff);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint8_t *const my_k = smem + warp * 2 * C::kCodes, *const my_v = smem + C::kVOff + warp * C::kCodes;
    uint64_t *const k_bar = reinterpret_cast<uint64_t *>(smem + C::kBarOff) + 3 * warp, *const v_bar = k_bar + 2;

    if (lane == 0) {
        for (int i = 0; i < 3; i++) mbar_init(&k_bar[i], 1);
        fence_mbar_init();
    }
    pdl_wait();
    pdl_launch_dependents();
    attn_make_plan<kRows, kAttnTile, C::kStart>(a, plan, reinterpret_cast<int *>(smem));
    fence_proxy_async_smem();  // the plan's scratch before the copies into its place
    AttnWalk<kRows, kAttnTile, C::kStart> walk(a, plan);
    AttnUnit u;
    const int lb = a.block == 16 ? 4 : a.block == 32 ? 5 : a.block == 64 ? 6 : 7;
    const int pages = a.block == 16 ? 2 : 1, box = a.block < kAttnTile ? a.block : kAttnTile;

    // This warp's tiles of a unit: its i-th is unit tile t_first + W i (tile x of the CTA, counted over
    // units, goes to warp x % W).
    int t_first = 0, n_own = 0;
    // lanes 0..31: tiles 32 b .. 32 b + 31 of the warp
    auto look = [&](int b) {
        DecInfo f;
        const int key = (t_first + W * (32 * b + lane)) * kAttnTile;
#pragma unroll
        for (int j = 0; j < 2; j++) {
            f.page[j] = -1;
            f.ks[j] = f.vs[j] = 0.0f;
            if (32 * b + lane < n_own && key + 16 * j < u.kv_end && j < pages) f.page[j] = attn_page(a, u.s, (key + 16 * j) >> lb);
            if (f.page[j] >= 0) {
                f.ks[j] = a.k_scale[int64_t(f.page[j]) * a.hkv + u.h];
                f.vs[j] = a.v_scale[int64_t(f.page[j]) * a.hkv + u.h];
            }
        }
        if (pages == 1) f.page[1] = f.page[0], f.ks[1] = f.ks[0], f.vs[1] = f.vs[0];
        return f;
    };
    // copies the codes of the warp's tile i (whose info is lane i % 32's of f)
    auto copy = [&](const DecInfo &f, int i, const CUtensorMap *map, uint8_t *dst, uint64_t *bar) {
        const int p0 = __shfl_sync(0xffffffffu, f.page[0], i & 31), p1 = __shfl_sync(0xffffffffu, f.page[1], i & 31);
        if (lane == 0) {
            const int have = (p0 >= 0) + (pages == 2 && p1 >= 0);
            mbar_arrive_expect_tx(bar, uint32_t(have * box * D));
            const int in = pages == 2 ? 0 : ((t_first + W * i) * kAttnTile) & (a.block - 1);  // the tile's first key in its page
            if (p0 >= 0) tma_load_3d(dst, map, 0, (p0 * a.hkv + u.h) * a.block + in, 0, bar);
            if (pages == 2 && p1 >= 0) tma_load_3d(dst + NA * 16 * 128, map, 0, (p1 * a.hkv + u.h) * a.block, 0, bar);
        }
    };
    // the byte offset of a key's 128-byte atom in a tile: [atom][key], or with 16-token pages [page][atom][key]
    const int at_stride = box * 128, half_skip = pages == 2 ? (NA - 1) * 16 * 128 : 0;

    DecInfo cur, nxt;   // the current and the next 32 tiles
    int kc = 0, vc = 0; // tiles consumed over units: slots and parities
    int base = 0;       // the CTA's tiles of the units before
    bool dead = false;  // a wait has given up: take part in barriers only
    // the unit's first copies of K (V's place may still hold accumulators)
    auto begin = [&]() {
        const int x = ((warp - base) % W + W) % W, n = u.t1 - u.t0;
        t_first = u.t0 + x;
        n_own = x < n ? (n - x + W - 1) / W : 0;
        base += n;
        cur = look(0);
        nxt = cur;
        if (n_own > 0) copy(cur, 0, &a.tmap_k, my_k + (kc & 1) * C::kCodes, &k_bar[kc & 1]);
        if (n_own > 1) copy(cur, 1, &a.tmap_k, my_k + ((kc + 1) & 1) * C::kCodes, &k_bar[(kc + 1) & 1]);
    };
    // the unit's q rows of this warp, E elements per lane, in flight while the unit before ends
    constexpr int E = D / 32, QR = (kRows + W - 1) / W;
    float qx[QR][E];
    auto load_q = [&]() {
#pragma unroll
        for (int k = 0; k < QR; k++) {
            const int rr = warp + W * k, row = u.r * kRows + rr;
            const bool there = rr < kRows && row < u.seq.q * a.group;
            const int tok = u.seq.row0 + row / a.group, head = u.h * a.group + row % a.group;
            const int64_t at = tok * a.qs_tok + head * a.qs_head + lane * E;
#pragma unroll
            for (int e = 0; e < E; e++) qx[k][e] = there ? attn_q_at(a, at + e) : 0.0f;
        }
    };
    const int gq = lane >> 2, tq = lane & 3;
    bool more = walk.next(u);
    if (more) {
        if (C::kEarlyQ) load_q();
        begin();
    }
    auto flushed = [&]() {  // this lane's place for them (from special registers: none held meanwhile)
        uint32_t cta, thread;
        asm volatile("mov.u32 %0, %%ctaid.x;" : "=r"(cta));
        asm volatile("mov.u32 %0, %%tid.x;" : "=r"(thread));
        return a.acc + (int64_t(cta) * W + (thread >> 5)) * (D / 8 * 32) + (thread & 31);
    };
    bool gave_up = false;
    while (more && !gave_up) {
        if (n_own > 0) copy(cur, 0, &a.tmap_v, my_v, v_bar);
        // q of the unit's rows, as A fragments in the K order above
        if (!C::kEarlyQ) load_q();
#pragma unroll
        for (int k = 0; k < QR; k++) {
            const int rr = warp + W * k;
            if (rr >= kRows) break;
            float m = 0.0f;
#pragma unroll
            for (int e = 0; e < E; e++) m = fmaxf(m, fabsf(qx[k][e]));
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            const int sh = attn_q_shift(m);
            if (lane == 0) rowf[rr] = attn_exp2i(-sh);
            const float f = attn_exp2i(sh);
#pragma unroll
            for (int e = 0; e < E; e += 4) {
                const int d = lane * E + e;  // a group of four dims: one MMA's share of lane t
                uint32_t *to = reinterpret_cast<uint32_t *>(sq + ((d >> 7) * 8 + ((d >> 2) & 7)) * 32 + (rr & 7) * 4 + ((d >> 5) & 3));
                float hi[4], lo[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    hi[i] = __half2float(__float2half_rn(qx[k][e + i] * f));
                    lo[i] = qx[k][e + i] * f - hi[i];
                }
                to[rr >> 3] = pack_h2(hi[0], hi[1]);
                to[2 + (rr >> 3)] = pack_h2(hi[2], hi[3]);
                if constexpr (SPLIT) {
                    to[1] = pack_h2(lo[0], lo[1]);
                    to[3] = pack_h2(lo[2], lo[3]);
                }
            }
        }
        __syncthreads();

        constexpr int NR = SPLIT ? 1 : 2;  // real rows per lane: gq (and gq + 8)
        float o[D / 8][4];
#pragma unroll
        for (int i = 0; i < D / 8; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
        const float ninf = __int_as_float(0xff800000);
        float ref[NR], sum[NR], qf[NR];
        int lim[NR];
#pragma unroll
        for (int k = 0; k < NR; k++) {
            ref[k] = ninf;
            sum[k] = 0.0f;
            const int row = u.r * kRows + gq + 8 * k;
            qf[k] = rowf[gq + 8 * k] * a.scale_log2;
            lim[k] = a.causal ? min(u.seq.kv, u.seq.kv - u.seq.q + row / a.group + 1) : u.seq.kv;
        }
        float vinv = 0.0f;  // 1 / unit
        for (int i = 0;;) {
            const int stop = SPLIT ? min(n_own, i + C::kFlush) : n_own;
            for (; i < stop; i++, kc++, vc++) {
                if ((i & 31) == 0) {  // lanes look at the warp's next 32 tiles, long before they are needed
                    cur = nxt;
                    if (i + 32 < n_own) nxt = look(i / 32 + 1);
                }
                const int key0 = (t_first + W * i) * kAttnTile;
                const bool in0 = __shfl_sync(0xffffffffu, cur.page[0], i & 31) >= 0, in1 = __shfl_sync(0xffffffffu, cur.page[1], i & 31) >= 0;
                const float ks0 = __shfl_sync(0xffffffffu, cur.ks[0], i & 31), ks1 = __shfl_sync(0xffffffffu, cur.ks[1], i & 31);
                const float vs0 = __shfl_sync(0xffffffffu, cur.vs[0], i & 31), vs1 = __shfl_sync(0xffffffffu, cur.vs[1], i & 31);
                const int st = kc & 1;
                if (!dead && !mbar_wait_bounded(&k_bar[st], uint32_t(kc >> 1) & 1u)) dead = true;
                dead = __any_sync(0xffffffffu, dead);
                if (dead) break;
                const uint8_t *const sk = my_k + st * C::kCodes;
                float s[4][4];
#pragma unroll
                for (int nt = 0; nt < 4; nt++) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.0f;
#pragma unroll 1
                for (int at = 0; at < NA; at++) {
                    uint4 kw[4][2];
#pragma unroll
                    for (int nt = 0; nt < 4; nt++)
#pragma unroll
                        for (int c = 0; c < 2; c++)
                            kw[nt][c] = *reinterpret_cast<const uint4 *>(sk + at * at_stride + (nt >> 1) * half_skip + (8 * nt + gq) * 128 +
                                                                         (((2 * tq + c) ^ gq) << 4));
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const uint4 qw = sq[(at * 8 + j) * 32 + lane];
                        const uint32_t qa[4] = {qw.x, qw.y, qw.z, qw.w};
#pragma unroll
                        for (int nt = 0; nt < 4; nt++) {
                            const uint4 w = kw[nt][j >> 2];
                            const uint32_t word = (j & 3) == 0 ? w.x : (j & 3) == 1 ? w.y : (j & 3) == 2 ? w.z : w.w;
                            uint32_t b0, b1;
                            codes_h2<FMT>(word, b0, b1);
                            mma_f16(s[nt], qa, b0, b1);
                        }
                    }
                }
                __syncwarp();
                if (i + 2 < n_own) copy((i + 2) / 32 == i / 32 ? cur : nxt, i + 2, &a.tmap_k, my_k + st * C::kCodes, &k_bar[st]);
                float vf = 1.0f;  // old unit / new unit
                const float vmax = fmaxf(vs0, vs1);  // 0 where there is no page
                if (vinv == 0.0f || vmax * vinv > kAttnVHigh) {
                    const float old = vinv;
                    vinv = attn_v_unit(vmax);
                    if (old > 0.0f) vf = vinv / old;
                }
                const float l0 = attn_v_log(vs0 * vinv), l1 = attn_v_log(vs1 * vinv);
                // scores in log2, masked; the largest contribution
                float p[NR][8];
                float top[NR];
#pragma unroll
                for (int k = 0; k < NR; k++) {
                    float mx[2] = {ninf, ninf};
#pragma unroll
                    for (int nt = 0; nt < 4; nt++) {
                        const float f = qf[k] * (nt < 2 ? ks0 : ks1);
                        const bool in = nt < 2 ? in0 : in1;
#pragma unroll
                        for (int c = 0; c < 2; c++) {
                            const int key = key0 + 8 * nt + 2 * tq + c;
                            const float z = SPLIT ? s[nt][c] + s[nt][c + 2] : s[nt][2 * k + c];
                            p[k][2 * nt + c] = in && key < lim[k] ? z * f : ninf;
                            mx[nt >> 1] = fmaxf(mx[nt >> 1], p[k][2 * nt + c]);
                        }
                    }
                    top[k] = fmaxf(mx[0] + l0, mx[1] + l1);
                    top[k] = fmaxf(top[k], __shfl_xor_sync(0xffffffffu, top[k], 1));
                    top[k] = fmaxf(top[k], __shfl_xor_sync(0xffffffffu, top[k], 2));
                }
                // references: moved for the whole warp at once, seldom
                bool move = vf != 1.0f;
#pragma unroll
                for (int k = 0; k < NR; k++) move |= top[k] - ref[k] > kAttnRefMove;  // (exact for scores of any size; NaN before the first)
                if (__any_sync(0xffffffffu, move)) {
                    float of[NR];
#pragma unroll
                    for (int k = 0; k < NR; k++) {
                        float f = 1.0f;
                        if (top[k] - ref[k] > kAttnRefMove) {
                            const float to = floorf(top[k]) - kAttnRefDrop;
                            f = ex2(ref[k] - to);  // 0 for the first scores (ref = -inf)
                            ref[k] = to;
                        }
                        sum[k] *= f;
                        of[k] = f * vf;
                    }
#pragma unroll
                    for (int n = 0; n < D / 8; n++) {
                        o[n][0] *= of[0], o[n][1] *= of[0];
                        o[n][2] *= of[NR - 1], o[n][3] *= of[NR - 1];
                    }
                    if (SPLIT && i >= C::kFlush) {
                        float4 *const acc = flushed();
#pragma unroll 1
                        for (int n = 0; n < D / 8; n++) attn_scale4(acc + 32 * n, of[0], of[NR - 1]);
                    }
                }
                const float r0 = vs0 * vinv, r1 = vs1 * vinv;
#pragma unroll
                for (int k = 0; k < NR; k++) {
                    const float base_ref = ref[k] == ninf ? 0.0f : ref[k];
#pragma unroll
                    for (int n = 0; n < 8; n++) {
                        const float e = ex2(p[k][n] - base_ref);
                        sum[k] += e;
                        p[k][n] = e * (n < 4 ? r0 : r1);
                    }
                }
                uint32_t pa[2][4];
#pragma unroll
                for (int ks = 0; ks < 2; ks++) {
                    if constexpr (SPLIT) {
                        const float *pp = &p[0][4 * ks];
                        const __half2 h0 = __floats2half2_rn(pp[0], pp[1]), h1 = __floats2half2_rn(pp[2], pp[3]);
                        pa[ks][0] = h2u(h0);
                        pa[ks][2] = h2u(h1);
                        pa[ks][1] = pack_h2(pp[0] - __low2float(h0), pp[1] - __high2float(h0));
                        pa[ks][3] = pack_h2(pp[2] - __low2float(h1), pp[3] - __high2float(h1));
                    } else {
#pragma unroll
                        for (int k = 0; k < 2; k++) {
                            pa[ks][k] = pack_h2(p[k][4 * ks], p[k][4 * ks + 1]);
                            pa[ks][k + 2] = pack_h2(p[k][4 * ks + 2], p[k][4 * ks + 3]);
                        }
                    }
                }
                if (!mbar_wait_bounded(v_bar, uint32_t(vc) & 1u)) dead = true;
                dead = __any_sync(0xffffffffu, dead);
                if (dead) break;
                // O += P V
#pragma unroll
                for (int ks = 0; ks < 2; ks++) {
                    // e4m3: bytes of keys that are not there may be NaN, which 0 * NaN would keep
                    uint32_t keep[4] = {~0u, ~0u, ~0u, ~0u};
                    if constexpr (FMT != CPQ_KV_INT8) {
#pragma unroll
                        for (int n = 0; n < 4; n++)
                            keep[n] = (ks ? in1 : in0) && key0 + 16 * ks + 2 * tq + (n & 1) + 8 * (n >> 1) < u.seq.kv ? ~0u : 0u;
                    }
#pragma unroll
                    for (int at = 0; at < NA; at++) {
                        uint4 vw[4];
#pragma unroll
                        for (int n = 0; n < 4; n++) {
                            const int key = 16 * ks + 2 * tq + (n & 1) + 8 * (n >> 1);
                            vw[n] = *reinterpret_cast<const uint4 *>(my_v + at * at_stride + ks * half_skip + key * 128 + ((gq ^ (key & 7)) << 4));
                        }
#pragma unroll
                        for (int wi = 0; wi < 4; wi++) {
                            uint32_t w[4];
#pragma unroll
                            for (int n = 0; n < 4; n++) {
                                w[n] = wi == 0 ? vw[n].x : wi == 1 ? vw[n].y : wi == 2 ? vw[n].z : vw[n].w;
                                if constexpr (FMT != CPQ_KV_INT8) w[n] &= keep[n];
                            }
                            uint32_t b[4][2];
                            codes_h2<FMT>(__byte_perm(w[0], w[1], 0x5140), b[0][0], b[1][0]);
                            codes_h2<FMT>(__byte_perm(w[0], w[1], 0x7362), b[2][0], b[3][0]);
                            codes_h2<FMT>(__byte_perm(w[2], w[3], 0x5140), b[0][1], b[1][1]);
                            codes_h2<FMT>(__byte_perm(w[2], w[3], 0x7362), b[2][1], b[3][1]);
#pragma unroll
                            for (int n = 0; n < 4; n++) mma_f16(o[at * 16 + wi * 4 + n], pa[ks], b[n][0], b[n][1]);
                        }
                    }
                }
                __syncwarp();
                if (i + 1 < n_own) copy((i + 1) / 32 == i / 32 ? cur : nxt, i + 1, &a.tmap_v, my_v, v_bar);
            }
            if (!SPLIT || dead || i == n_own) break;
            if constexpr (SPLIT) {
                float4 *const acc = flushed();
#pragma unroll
                for (int n = 0; n < D / 8; n++) {
                    attn_flush4(acc + 32 * n, i == C::kFlush, o[n][0], o[n][1], o[n][2], o[n][3]);
                    o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
                }
            }
        }
        if (SPLIT && n_own > C::kFlush) {
            const float4 *const acc = flushed();
#pragma unroll
            for (int n = 0; n < D / 8; n++) {
                const float4 v = __ldcg(acc + 32 * n);
                o[n][0] += v.x, o[n][1] += v.y, o[n][2] += v.z, o[n][3] += v.w;
                if (n % 4 == 3) asm volatile("" ::: "memory");  // four loads in flight: no registers for more
            }
        }
        // join the warps: stats first, then the accumulators at the common reference. The next unit's first
        // copies of K go out meanwhile.
        const AttnUnit done = u;
        more = walk.next(u);
        if (more) {
            if (C::kEarlyQ) load_q();
            begin();
        }
#pragma unroll
        for (int k = 0; k < NR; k++) {
            sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], 1);
            sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], 2);
            if (tq == 0) stat[warp * 16 + gq + 8 * k] = make_float2(ref[k], sum[k]);
        }
        __syncthreads();
        float top[NR], all[NR];
#pragma unroll
        for (int k = 0; k < NR; k++) {
            top[k] = ninf;
            all[k] = 0.0f;
#pragma unroll
            for (int w = 0; w < W; w++) top[k] = fmaxf(top[k], stat[w * 16 + gq + 8 * k].x);
            const float b = top[k] == ninf ? 0.0f : top[k];
#pragma unroll
            for (int w = 0; w < W; w++) {
                const float2 x = stat[w * 16 + gq + 8 * k];
                all[k] += x.y * ex2(x.x - b);
            }
        }
        // fragment order: [16 at + b][row][n], dim 128 at + 16 n + b
        float *mine = red + (warp & 3) * (kRows * D);
#pragma unroll 1
        for (int r = W / 4 - 1; r >= 0; r--) {  // four warps at a time
            if ((warp >> 2) == r) {
#pragma unroll
                for (int k = 0; k < NR; k++) {
                    const float f = ex2(ref[k] - (top[k] == ninf ? 0.0f : top[k])) * attn_v_scale(vinv);
#pragma unroll
                    for (int i = 0; i < D / 8; i++) {
                        float2 *to = reinterpret_cast<float2 *>(mine + (i * kRows + gq + 8 * k) * 8 + 2 * tq);
                        float2 v = SPLIT ? make_float2((o[i][0] + o[i][2]) * f, (o[i][1] + o[i][3]) * f)
                                         : make_float2(o[i][2 * k] * f, o[i][2 * k + 1] * f);
                        if (r != W / 4 - 1) {
                            const float2 w = *to;
                            v.x += w.x, v.y += w.y;
                        }
                        *to = v;
                    }
                }
            }
            __syncthreads();
        }
        const bool whole = done.t0 == 0 && done.t1 == done.n;
        const int slot = attn_slot(done);
        for (int i = threadIdx.x; i < kRows * (D / 16); i += C::kThreads) {
            const int n = i & 7, rr = (i >> 3) % kRows, at = (i >> 3) / kRows;
            const int row = done.r * kRows + rr;
            const bool there = row < done.seq.q * a.group;
            float2 ml = make_float2(ninf, 0.0f);  // the row's statistics, as above
#pragma unroll
            for (int w = 0; w < W; w++) ml.x = fmaxf(ml.x, stat[w * 16 + rr].x);
#pragma unroll
            for (int w = 0; w < W; w++) ml.y += stat[w * 16 + rr].y * ex2(stat[w * 16 + rr].x - (ml.x == ninf ? 0.0f : ml.x));
            float v[16];
#pragma unroll
            for (int b = 0; b < 16; b++) {
                const int e = ((at * 16 + b) * kRows + rr) * 8 + n;
                v[b] = (red[e] + red[kRows * D + e]) + (red[2 * kRows * D + e] + red[3 * kRows * D + e]);
            }
            const int d0 = at * 128 + n * 16;
            if (whole) {
                if (there) {
                    const float f = attn_inverse(ml.y);
                    const int tok = done.seq.row0 + row / a.group, head = done.h * a.group + row % a.group;
                    const int64_t to = tok * a.os_tok + head * a.os_head + d0;
#pragma unroll
                    for (int b = 0; b < 16; b++) attn_out_at(a, to + b, v[b] * f);
                    if (d0 == 0 && a.lse) a.lse[int64_t(tok) * (a.hkv * a.group) + head] = attn_lse(ml.x, ml.y);
                }
            } else {
                float4 *to = reinterpret_cast<float4 *>(a.part_o + (int64_t(slot) * kRows + rr) * D + d0);
#pragma unroll
                for (int b = 0; b < 4; b++) to[b] = make_float4(v[4 * b], v[4 * b + 1], v[4 * b + 2], v[4 * b + 3]);
                if (d0 == 0) a.part_ml[slot * kRows + rr] = ml;
                if (i == 0) a.part_hdr[slot] = make_int4(done.s, done.r, done.h, done.t1 == done.n ? 2 : 1);
            }
        }
        gave_up = __syncthreads_or(dead) != 0;  // one warp's for all; q, stats and V's place are free again
        fence_proxy_async_smem();               // the accumulators before the copies into their place
    }
    // no copy may land after the CTA has left: one that gave up may have some under way
    if (gave_up) {
        for (int i = 0; i < 2; i++) mbar_wait_bounded(&k_bar[i], uint32_t((kc + i) >> 1) & 1u);
        mbar_wait_bounded(v_bar, uint32_t(vc) & 1u);
    }
}

// ---- joining a cut unit ------------------------------------------------------------
//
// grid (CTAs of the attention grid, rows / ROWS_HERE): block (c, y) joins rows
// of the unit that begins in CTA c and goes on in c + 1, ...: sum over the parts
// of part * 2^(reference - largest reference). D / 4 threads across a row; with
// few rows the parts are dealt out over the rest of the block and added in a
// fixed order. Latency: some 3 us of a decode step (its reads come from L2).

constexpr int kCombineThreads = 256;

template <int D, int ROWS> struct CombineCfg {
    static constexpr int kAcross = D / 4, kSets = kCombineThreads / kAcross;
    static constexpr int kRowsHere = ROWS > 16 ? kSets : 1;  // rows of a block
    static constexpr int kDeal = kSets / kRowsHere;          // sets that share a row's parts
};

template <int D, int ROWS>
__global__ void __launch_bounds__(kCombineThreads) attn_combine_kernel(const __grid_constant__ AttnArgs a) {
    using C = CombineCfg<D, ROWS>;
    __shared__ float4 s_o[C::kSets][C::kAcross];
    __shared__ float s_l[C::kSets];
    __shared__ int s_n;
    const int c = blockIdx.x;
    const int x = threadIdx.x % C::kAcross, set = threadIdx.x / C::kAcross;
    const int rr = blockIdx.y * C::kRowsHere + set / C::kDeal, z = set % C::kDeal;
    pdl_wait();
    pdl_launch_dependents();
    const int4 hdr = a.part_hdr[2 * c + 1];
    if (hdr.w == 0) return;
    const AttnSeq seq = attn_seq(a, hdr.x);
    if (hdr.y * ROWS + int(blockIdx.y) * C::kRowsHere >= seq.q * a.group) return;
    // parts: slot 2c + 1, then 2(c + 1), 2(c + 2), ... up to the one that ends the unit
    if (threadIdx.x == 0) s_n = int(gridDim.x) - c;
    __syncthreads();
    for (int i = threadIdx.x; i < int(gridDim.x) - c; i += kCombineThreads) {
        const int w = i == 0 ? hdr.w : a.part_hdr[2 * (c + i)].w;
        if (w != 1) atomicMin(&s_n, i + 1);
    }
    __syncthreads();
    const int n = s_n;
    auto slot = [&](int i) { return int64_t(i == 0 ? 2 * c + 1 : 2 * (c + i)); };
    float m = __int_as_float(0xff800000);
    for (int i = threadIdx.x & 31; i < n; i += 32) m = fmaxf(m, a.part_ml[slot(i) * ROWS + rr].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float b = m == __int_as_float(0xff800000) ? 0.0f : m;
    float4 acc = make_float4(0, 0, 0, 0);
    float l = 0.0f;
#pragma unroll 4
    for (int i = z; i < n; i += C::kDeal) {
        const float2 ml = a.part_ml[slot(i) * ROWS + rr];
        const float4 v = *reinterpret_cast<const float4 *>(a.part_o + (slot(i) * ROWS + rr) * D + 4 * x);
        const float f = ex2(ml.x - b);
        acc.x += v.x * f, acc.y += v.y * f, acc.z += v.z * f, acc.w += v.w * f;
        l += ml.y * f;
    }
    if constexpr (C::kDeal > 1) {
        s_o[set][x] = acc;
        if (x == 0) s_l[set] = l;
        __syncthreads();
        if (z) return;
        l = 0.0f;
        acc = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < C::kDeal; i++) {
            const float4 v = s_o[set + i][x];
            acc.x += v.x, acc.y += v.y, acc.z += v.z, acc.w += v.w;
            l += s_l[set + i];
        }
    }
    const int row = hdr.y * ROWS + rr;
    if (row >= seq.q * a.group) return;
    const float f = attn_inverse(l);
    const int tok = seq.row0 + row / a.group, head = hdr.z * a.group + row % a.group;
    const int64_t to = tok * a.os_tok + head * a.os_head + 4 * x;
    attn_out_at(a, to, acc.x * f);
    attn_out_at(a, to + 1, acc.y * f);
    attn_out_at(a, to + 2, acc.z * f);
    attn_out_at(a, to + 3, acc.w * f);
    if (x == 0 && a.lse) a.lse[int64_t(tok) * (a.hkv * a.group) + head] = attn_lse(m, l);
}

}  // namespace cpq
