// paged_attn_tc.cuh — attention over the paged 8-bit cache for many query rows
// (verify, chunked prefill) on tcgen05 tensor cores. Mathematics, numbers and
// split as in paged_attn.cuh; a row tile is 128 rows, a key tile 128 keys.
//
// Per key tile the tensor core does S[128 x 128] = Q K^T and O[128 x D] += P V
// (fp32 q: twice each, the two fp16 terms of Q and of P). At D = 256 these are
// 2048 (4096) tensor cycles; what the design has to hide behind them is the
// softmax of 128 x 128 scores (1024 cycles of ex2 per SM sub-partition) and
// turning 64 KB of codes into 128 KB of fp16 operands.
//
// The MMAs are issued by an elected lane with descriptors as 32-bit words that
// differ by constants. Issued under `lane == 0` with 64-bit descriptors they
// took 95 to 110 cycles of instructions each, whatever the shape, where N = 128
// needs 64 (a 1024-token chunk behind 16k keys: 715 us).
//
// Tensor memory (512 columns): O, fp32 [128][D]; two buffers of S, fp32
// [128][128], in which P takes its scores' place (per 16 keys 8 columns of first
// fp16 terms, 8 of second ones). Shared memory, all with the 128-byte
// swizzle: Q [128][D] (first, then second terms) as D / 64 blocks of 128 rows x
// 128 bytes; K [128 keys][D] in the same blocks, each filled and released on its
// own (a whole K at a time left the conversion idle during the first product and
// the tensor core during the conversion: 5700 cycles per key tile); V in stages of 32
// keys (four; two beside fp32 q) as D / 64 blocks of 32 rows x 128 bytes. K is the
// K-major operand of the first product (N = keys, K = dims), V the MN-major
// operand of the second (N = dims, K = keys): the same row layout, so both come
// from the same conversion.
//
//   warp 0       one lane issues the MMAs: per tile i S(i + 1), then P(i) V. S(i + 1)
//                waits for P(i - 1) V, whose P lies in its buffer, and is made while
//                the softmax of tile i runs
//   warp 1       the key tiles' cache rows and page scales, some tiles ahead
//   warps 4-11   softmax: a query row is a lane of tensor memory, its first 64 keys
//                belong to a thread of warps 4-7, the others to one of warps 8-11,
//                which exchange their maxima through shared memory. Scores are read
//                twice, 32 and then 16 at a time (maxima, exponentials), which keeps 28
//                warps within the register file. They also load Q, rescale O when a
//                reference moves, and write the unit's rows out, half of the columns
//                each
//   warps 12-19  conversion of K, in jobs of a 64-dim block, warps 20-27 of V, in jobs
//                of 32 keys, the same code, two sets of four warps that take turns
//                (a job takes some 1200 cycles, half of them latency): 16 bytes of codes
//                per load, two jobs in registers; keys that are not there become zeros
//
// The roles' inner loops are kept short: unrolled all the way, with variants for
// masked tiles and K and V apart, the warps waited for instructions more than
// for anything else (6 of 15 cycles per instruction; 8000 cycles per key tile).
// Masked tiles therefore get their -inf written into S beforehand.
//
// Measured (24 heads over 4 of 256): 1024 bf16 tokens behind 16384 keys 522 us
// (765 TFLOP/s, 0.47 of a measured GEMM; 491 us at a cool clock: 69 % of issue
// slots, 43 % of the tensor pipe; 547 in a long loop, at the power cap), three fp32
// chunks of up to 700 over up to 9000 keys, twice the products, 618 us (940 TFLOP/s
// of fp16 products, 0.57).
// Following each row's contributions instead of its scores cost 2 % of the first. Issue slots
// bound it, conversion and softmax together; S and P V as pairs of SMs would halve
// the conversions, which all CTAs of a head's row tiles repeat.
//
// Waits are bounded as everywhere (a timeout sets the device error word and an
// abort flag; MMAs in flight are waited for before tensor memory is released).
#pragma once

#include "paged_attn.cuh"

namespace cpq {

constexpr int kTaRows = 128;
constexpr int kTaTile = 128;
constexpr int kTaHalf = 64;       // keys of a conversion job, a softmax thread
constexpr int kTaQuarter = 32;    // keys of a V stage
constexpr int kTaThreads = 896;
constexpr int kTaConvWarps = 16;
constexpr int kTaSoftWarps = 8;
constexpr int kTaStart = 2;       // beginning a unit takes about as long as this many tiles
constexpr int kTaInfo = 4;        // key tiles looked up ahead
static_assert(kTaInfo == 4, "warp 1 looks up four tiles at a time");

struct TaInfo {
    int row[8];                   // cache row of each 16 keys' first one, -1: no such keys
    float ks[8], vs[8];
    int keys;                     // keys of the tile that the sequence has
    int pad;
};

template <int D, bool SPLIT> struct TaCfg {
    static constexpr int kVStages = SPLIT ? 2 : 4;
    static constexpr int kFlush = SPLIT ? 6 : 32;         // tiles (16, 8 accumulation steps each) between flushes of O
    static constexpr int kBlock = kTaTile * 128;          // a 64-dim block of Q or K
    static constexpr int kVBlock = kTaQuarter * 128;      // of a V stage
    static constexpr int kK = kTaTile * D * 2, kV = kTaQuarter * D * 2, kQ = kTaRows * D * 2;
    static constexpr int kVOff = kK;
    static constexpr int kQOff = kVOff + kVStages * kV;
    static constexpr int kMaxOff = kQOff + (SPLIT ? 2 : 1) * kQ;   // float [2][2][128], used in turns
    static constexpr int kInfoOff = kMaxOff + 4 * kTaRows * 4;
    static constexpr int kBarOff = kInfoOff + kTaInfo * int(sizeof(TaInfo));
    static constexpr int kBars = 2 * kTaInfo + 16 + 7;
    static constexpr int kPlanOff = kBarOff + kBars * 8;
    static constexpr int kSmem = kPlanOff + int(sizeof(AttnPlan)) + 12;
    // tensor memory columns
    static constexpr uint32_t kColO = 0, kColS = D;
    static_assert(kColS + 2 * kTaTile <= 512, "TMEM columns");
    static_assert(kSmem <= 227 * 1024, "shared memory");
    static_assert(kK >= (kAttnMaxSeqs + 1) * 4, "the plan's scratch lies in K's stage");
};

__device__ __forceinline__ void soft_sync() { asm volatile("bar.sync 1, %0;" ::"n"(32 * kTaSoftWarps) : "memory"); }

// The same barrier, with whether any thread passed true: all softmax warps go on or stop together.
__device__ __forceinline__ bool soft_any(bool x) {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, 1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(r)
                 : "r"(x ? 1u : 0u), "n"(32 * kTaSoftWarps)
                 : "memory");
    return r != 0;
}

// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}

// Shared-memory descriptors of SWIZZLE_128B operands (see smem_desc_sw128) as two
// words: the high one (stride byte offset 1024, version, layout) is the same
// for all; the low one holds the address and the leading byte offset, unused
// for a K-major operand. A MN-major operand has rows of 64 elements (128 bytes)
// along N, one per k, 8-row groups 1024 bytes apart, the next 64 elements of N
// `lbo` bytes on.
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_lo(uint32_t saddr, uint32_t lbo) { return ((saddr >> 4) & 0x3fffu) | ((lbo >> 4) << 16); }

// One-SM MMAs: D (TMEM) (+)= A x B, A in shared memory or TMEM, accumulating or not.
template <bool ACC>
__device__ __forceinline__ void tc_mma1_ss(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
        "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\tsetp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n\t}" ::"r"(d_tmem),
        "r"(a_lo), "r"(b_lo), "n"(kDescHi), "r"(idesc), "n"(ACC ? 1 : 0)
        : "memory");
}
template <bool ACC>
__device__ __forceinline__ void tc_mma1_ts(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
        "mov.b64 b, {%2, %3};\n\tsetp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "r"(b_lo), "n"(kDescHi), "r"(idesc), "n"(ACC ? 1 : 0)
        : "memory");
}
__device__ __forceinline__ void tc_commit1(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}

// 8 columns of this thread's lane, without waiting for completion.
__device__ __forceinline__ void tmem_st8_async(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
                 "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}

// 16 columns, load and wait in one statement.
__device__ __forceinline__ void tmem_ld16_wait(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}

// 32 consecutive fp32 columns of this thread's lane, load and wait in one
// statement: a use of the values cannot be moved between the two.
__device__ __forceinline__ void tmem_ld32_wait(uint32_t taddr, float (&v)[32]) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,"
        "%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 32; i++) v[i] = __uint_as_float(r[i]);
}

// 16 consecutive 32-bit TMEM columns of this thread's lane, without waiting for completion.
__device__ __forceinline__ void tmem_st16_async(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

// Two fp32 values at a time.
__device__ __forceinline__ uint64_t f2_pack(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void f2_unpack(uint64_t v, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t f2_mul(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// 16 bytes of codes, or zeros; the load stays in flight (selecting its result
// afterwards would wait for it). Not a non-coherent load: the append before may
// still be writing when this kernel begins.
__device__ __forceinline__ uint4 ldg_codes(const uint8_t *p, bool there) {
    uint4 r = make_uint4(0, 0, 0, 0);
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %5, 0;\n\t"
        "@p ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
        : "+r"(r.x), "+r"(r.y), "+r"(r.z), "+r"(r.w)
        : "l"(p), "r"(there ? 1u : 0u)
        : "memory");
    return r;
}

// A score's factor; never 0, so that a masked score of -inf stays one (others
// then vanish beside 1, as they should).
__device__ __forceinline__ float ta_factor(float f) { return f == 0.0f ? 1e-30f : f; }

// Eight elements of q from element i on.
__device__ __forceinline__ void attn_q8(const AttnArgs &a, int64_t i, float (&x)[8]) {
    if (!a.wide) {
#pragma unroll
        for (int k = 0; k < 8; k++) x[k] = attn_q_at(a, i + k);
    } else if (a.type == CPQ_TYPE_F32) {
        float lo[4], hi[4];
        Vec<float, 4> u;
        u.load(static_cast<const float *>(a.q) + i);
        u.get(lo);
        u.load(static_cast<const float *>(a.q) + i + 4);
        u.get(hi);
#pragma unroll
        for (int k = 0; k < 4; k++) x[k] = lo[k], x[k + 4] = hi[k];
    } else if (a.type == CPQ_TYPE_F16) {
        Vec<__half, 8> u;
        u.load(static_cast<const __half *>(a.q) + i);
        u.get(x);
    } else {
        Vec<__nv_bfloat16, 8> u;
        u.load(static_cast<const __nv_bfloat16 *>(a.q) + i);
        u.get(x);
    }
}

// 32 elements of the output from element i on.
__device__ __forceinline__ void attn_out32(const AttnArgs &a, int64_t i, const float (&x)[32]) {
#pragma unroll
    for (int k = 0; k < 32; k += 8) {
        const float f[8] = {x[k], x[k + 1], x[k + 2], x[k + 3], x[k + 4], x[k + 5], x[k + 6], x[k + 7]};
        if (!a.wide) {
#pragma unroll
            for (int j = 0; j < 8; j++) attn_out_at(a, i + k + j, f[j]);
        } else if (a.type == CPQ_TYPE_F32) {
            float *o = static_cast<float *>(a.out) + i + k;
            *reinterpret_cast<float4 *>(o) = make_float4(f[0], f[1], f[2], f[3]);
            *reinterpret_cast<float4 *>(o + 4) = make_float4(f[4], f[5], f[6], f[7]);
        } else if (a.type == CPQ_TYPE_F16) {
            Vec<__half, 8> u;
            u.set(f);
            u.store(static_cast<__half *>(a.out) + i + k);
        } else {
            Vec<__nv_bfloat16, 8> u;
            u.set(f);
            u.store(static_cast<__nv_bfloat16 *>(a.out) + i + k);
        }
    }
}

template <int D, int FMT, bool SPLIT>
__global__ void __launch_bounds__(kTaThreads, 1) attn_tc_kernel(const __grid_constant__ AttnArgs a) {
    using C = TaCfg<D, SPLIT>;
    extern __shared__ __align__(1024) uint8_t smem_tc[];  // the swizzle goes by address bits: 1024-byte aligned
    uint8_t *const smem = smem_tc;
    if (smem_addr(smem) & 1023u) {  // (dynamic shared memory begins on such a boundary; there is no room to align it here)
        if (threadIdx.x == 0) atomicOr(&g_dev_error, kDevErrBadLaunch);
        return;
    }
    uint8_t *sK = smem, *sV = smem + C::kVOff, *sQ = smem + C::kQOff;
    float(*s_max)[2][kTaRows] = reinterpret_cast<float(*)[2][kTaRows]>(smem + C::kMaxOff);
    TaInfo *info = reinterpret_cast<TaInfo *>(smem + C::kInfoOff);
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + C::kBarOff);
    uint64_t *info_full = bars, *info_empty = bars + kTaInfo;
    uint64_t *k_full = bars + 2 * kTaInfo, *k_empty = k_full + 4, *v_full = k_full + 8, *v_empty = k_full + 12;
    uint64_t *q_full = k_full + 16, *s_full = q_full + 1, *p_full = q_full + 3, *pv_done = q_full + 5, *stopped = q_full + 6;
    AttnPlan &plan = *reinterpret_cast<AttnPlan *>(smem + C::kPlanOff);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + C::kPlanOff + sizeof(AttnPlan));
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kTaInfo; i++) {
            mbar_init(&info_full[i], 1);
            mbar_init(&info_empty[i], kTaConvWarps + kTaSoftWarps);
        }
        for (int i = 0; i < 4; i++) {
            mbar_init(&k_full[i], kTaConvWarps / 4);  // the warps of a set
            mbar_init(&k_empty[i], 1);
            mbar_init(&v_full[i], kTaConvWarps / 4);
            mbar_init(&v_empty[i], 1);
        }
        mbar_init(q_full, kTaSoftWarps);
        for (int i = 0; i < 2; i++) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], kTaSoftWarps);
        }
        mbar_init(pv_done, 1);
        mbar_init(stopped, 1);
        // a wait on this device has already timed out: do no work (the error stays reported)
        *abort_flag = (*reinterpret_cast<volatile uint32_t *>(&g_dev_error) & kDevErrWaitTimeout) ? 1 : 0;
        fence_mbar_init();
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pdl_wait();
    pdl_launch_dependents();
    tc_fence_before();
    attn_make_plan<kTaRows, kTaTile, kTaStart>(a, plan, reinterpret_cast<int *>(sK));  // (its barriers also publish the TMEM address)
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    // g: key tiles of this CTA so far, over units; parities and the info slot follow from it

    if (warp < 4) {
        if (warp == 0 && elect_one()) {
            // ---- MMA issue ----
            AttnWalk<kTaRows, kTaTile, kTaStart> walk(a, plan);
            AttnUnit u;
            constexpr uint32_t idesc_s = tc_idesc_f16(kTaRows, kTaTile);
            constexpr uint32_t idesc_o = tc_idesc_f16(kTaRows, D) | (1u << 16);  // B is MN-major
            int g = 0, n_units = 0;
            bool ok = true, issued = false;
            const uint32_t q_lo = desc_lo(smem_addr(sQ), 16), k_lo = desc_lo(smem_addr(sK), 16);
            const uint32_t v_lo = desc_lo(smem_addr(sV), C::kVBlock);
            // S = Q K(gi)^T; fresh: the unit's first tile, or its second (the buffer's last P V has been waited for)
            auto scores = [&](int gi, bool fresh) {
                if (!fresh && !tc_wait(pv_done, uint32_t(gi - 2) & 1u, abort_flag)) return false;
                const uint32_t s = tmem + C::kColS + uint32_t(kTaTile) * uint32_t(gi & 1);
                // fp32 q: the second terms come first, while the sums are small and lose next to nothing
#pragma unroll
                for (int term = SPLIT ? 1 : 0; term >= 0; term--) {
#pragma unroll
                    for (int b = 0; b < D / 64; b++) {
                        if ((term || !SPLIT) && !tc_wait(&k_full[b], uint32_t(gi) & 1u, abort_flag)) return false;
                        tc_fence_after();
#pragma unroll
                        for (int x = 0; x < 4; x++) {
                            const uint32_t at = uint32_t(b * (C::kBlock / 16) + 2 * x), q = q_lo + uint32_t(term * (C::kQ / 16)) + at;
                            if (b == 0 && x == 0 && term == (SPLIT ? 1 : 0)) tc_mma1_ss<false>(s, q, k_lo + at, idesc_s);
                            else tc_mma1_ss<true>(s, q, k_lo + at, idesc_s);
                        }
                        issued = true;
                        if (term == 0) tc_commit1(&k_empty[b]);
                    }
                }
                tc_commit1(&s_full[gi & 1]);
                return true;
            };
            // O (+)= P(g) V for 32 keys
            auto values = [&](int quarter, bool fresh) {
                const int job = 4 * g + quarter, st = job % C::kVStages;
                if (!tc_wait(&v_full[st], uint32_t(job / C::kVStages) & 1u, abort_flag)) return false;
                tc_fence_after();
                const uint32_t v = v_lo + uint32_t(st * (C::kV / 16));
                const uint32_t p = tmem + C::kColS + uint32_t(kTaTile) * uint32_t(g & 1) + 32u * uint32_t(quarter);
                constexpr uint32_t first = SPLIT ? 8u : 0u;  // (second terms first here too)
                if (fresh) tc_mma1_ts<false>(tmem + C::kColO, p + first, v, idesc_o);
                else tc_mma1_ts<true>(tmem + C::kColO, p + first, v, idesc_o);
#pragma unroll
                for (int x = 1; x < (SPLIT ? 4 : 2); x++)
                    tc_mma1_ts<true>(tmem + C::kColO, p + (x < 2 ? first : 0u) + 16u * uint32_t(x & 1), v + 128u * uint32_t(x & 1), idesc_o);
                tc_commit1(&v_empty[st]);
                return true;
            };
            while (ok && walk.next(u)) {
                const int n = u.t1 - u.t0;
                ok = tc_wait(q_full, uint32_t(n_units) & 1u, abort_flag) && scores(g, true);
                n_units++;
                for (int j = 0; ok && j < n; j++, g++) {
                    ok = (j + 1 == n || scores(g + 1, j == 0)) && tc_wait(&p_full[g & 1], uint32_t(g >> 1) & 1u, abort_flag);
                    for (int x = 0; ok && x < 4; x++) ok = values(x, (j % C::kFlush | x) == 0);
                    if (!ok) break;
                    tc_commit1(pv_done);
                }
            }
            // MMAs in flight end before tensor memory is released: normally the softmax warps have waited for the
            // last of them; after an early stop one more commit tracks what was issued
            if (!ok && issued) {
                tc_commit1(stopped);
                mbar_wait_bounded(stopped, 0);
            }
        } else if (warp == 1) {
            // ---- cache rows and scales of the key tiles: lane = (tile of four, 16 keys of eight) ----
            AttnWalk<kTaRows, kTaTile, kTaStart> walk(a, plan);
            AttnUnit u;
            const int lb = a.block == 16 ? 4 : a.block == 32 ? 5 : a.block == 64 ? 6 : 7;
            int g = 0;
            bool ok = true;
            while (ok && walk.next(u)) {
                for (int b0 = u.t0; ok && b0 < u.t1; b0 += 4) {
                    const int key = (b0 + (lane >> 3)) * kTaTile + 16 * (lane & 7);
                    int row = -1;
                    float ks = 0.0f, vs = 0.0f;
                    if (b0 + (lane >> 3) < u.t1 && key < u.kv_end) {
                        const int page = attn_page(a, u.s, key >> lb);
                        if (page >= 0) {
                            row = (page * a.hkv + u.h) * a.block + (key & (a.block - 1));
                            ks = a.k_scale[int64_t(page) * a.hkv + u.h];
                            vs = a.v_scale[int64_t(page) * a.hkv + u.h];
                        }
                    }
                    const int n = min(4, u.t1 - b0);
                    for (int i = 0; i < n; i++, g++) {
                        const int slot = g % kTaInfo;
                        if (!__all_sync(0xffffffffu, tc_wait(&info_empty[slot], (uint32_t(g / kTaInfo) & 1u) ^ 1u, abort_flag))) {
                            ok = false;
                            break;
                        }
                        if ((lane >> 3) == i) {
                            info[slot].row[lane & 7] = row;
                            info[slot].ks[lane & 7] = ks;
                            info[slot].vs[lane & 7] = vs;
                            if ((lane & 7) == 0) info[slot].keys = u.seq.kv - (b0 + i) * kTaTile;
                        }
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&info_full[slot]);
                    }
                }
            }
        }
        __syncwarp();
    } else if (warp >= 12) {
        // ---- conversion ----
        // V: job j is the keys 32 (j & 3) .. of tile j / 4, a warp's part 8 keys, all dims.
        // K: job j is the 64-dim block j % (D / 64) of tile j / (D / 64), a warp's part 32 keys.
        // Load i of a lane: 16 dims of key key_in + step * i.
        const int w = warp & 3;
        const int set = (warp >> 2) - 3 & 1;
        const bool is_v = warp >= 20;
        constexpr int kLoads = 4, kLanes = D / 16, kVLoads = kLanes / 4;  // (V has two loads at D = 128)
        const int per_tile = is_v ? 4 : D / 64, step = is_v ? 32 / kLanes : 8;
        const int key_in = is_v ? 8 * w + lane / kLanes : 32 * w + (lane >> 2);
        const int d0 = is_v ? (lane % kLanes) * 16 : (lane & 3) * 16;
        // where the lane's 16 values go: two 16-byte units of a 64-dim block. Odd blocks store their second
        // unit first, so that a quarter warp's eight stores fall into eight bank groups.
        const int blk = d0 >> 6, unit = (d0 & 63) >> 3, swap = blk & 1;
        const uint8_t *const codes = (is_v ? a.v : a.k) + (key_in & 15) * D + d0;
        uint8_t *const dst0 = (is_v ? sV + blk * C::kVBlock : sK) + key_in * 128;
        int n_tiles = 0;
        {
            AttnWalk<kTaRows, kTaTile, kTaStart> walk(a, plan);
            AttnUnit u;
            while (walk.next(u)) n_tiles += u.t1 - u.t0;
        }
        const int n_jobs = per_tile * n_tiles;
        auto load = [&](int j, uint4 (&x)[kLoads]) {
            if (j >= n_jobs) return true;
            const int tile = j / per_tile, part = j - tile * per_tile, slot = tile % kTaInfo;
            if (!tc_wait(&info_full[slot], uint32_t(tile / kTaInfo) & 1u, abort_flag)) return false;
            const int keys = info[slot].keys - (is_v ? kTaQuarter * part : 0) - key_in;
            // the lane's keys lie in one group of 16 (V), or two (K)
            const int grp = is_v ? 2 * part + (w >> 1) : 2 * w;
            const int row0 = info[slot].row[grp], row1 = is_v ? row0 : info[slot].row[grp + 1] - 16;
            const uint8_t *at = codes + (is_v ? 0 : 64 * part);
#pragma unroll
            for (int i = 0; i < kLoads; i++) {
                const int row = i < 2 ? row0 : row1;
                const bool there = row >= (i < 2 || is_v ? 0 : -16) && step * i < keys && (i < kVLoads || !is_v);
                x[i] = ldg_codes(at + (int64_t(row) + step * i) * D, there);
            }
            if (part + 2 >= per_tile) {  // the set's last job of the tile
                __syncwarp();
                if (lane == 0) mbar_arrive(&info_empty[slot]);
            }
            return true;
        };
        auto run = [&](int j, uint4 (&x)[kLoads]) {  // job j, whose codes are in x
            if (j >= n_jobs) return true;
            const int st = is_v ? j % C::kVStages : j % (D / 64), use = is_v ? j / C::kVStages : j / (D / 64);
            if (!tc_wait((is_v ? v_empty : k_empty) + st, (uint32_t(use) & 1u) ^ 1u, abort_flag)) return false;
            uint8_t *const dst = dst0 + st * (is_v ? C::kV : C::kBlock);
#pragma unroll
            for (int i = 0; i < kLoads; i++) {
                if (i >= kVLoads && is_v) break;
                uint32_t h[8];
                codes_h2<FMT>(x[i].x, h[0], h[1]);
                codes_h2<FMT>(x[i].y, h[2], h[3]);
                codes_h2<FMT>(x[i].z, h[4], h[5]);
                codes_h2<FMT>(x[i].w, h[6], h[7]);
                const uint4 lo = make_uint4(h[0], h[1], h[2], h[3]), hi = make_uint4(h[4], h[5], h[6], h[7]);
                const int k7 = (key_in + step * i) & 7;
                uint8_t *at = dst + step * i * 128;
                *reinterpret_cast<uint4 *>(at + (((unit + swap) ^ k7) << 4)) = swap ? hi : lo;
                *reinterpret_cast<uint4 *>(at + (((unit + (swap ^ 1)) ^ k7) << 4)) = swap ? lo : hi;
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive((is_v ? v_full : k_full) + st);
            return load(j + 4, x);
        };
        uint4 x0[kLoads], x1[kLoads];
        bool ok = load(set, x0) && load(set + 2, x1);
#pragma unroll 1
        for (int j = set; ok && j < n_jobs; j += 4) ok = run(j, x0) && run(j + 2, x1);
        __syncwarp();
    } else {
        // ---- softmax: row = lane of tensor memory, 64 of the tile's keys per thread ----
        AttnWalk<kTaRows, kTaTile, kTaStart> walk(a, plan);
        AttnUnit u;
        const int hf = (warp - 4) >> 2;                     // which half of the keys, and of D
        const int rr = 32 * (warp & 3) + lane;
        const uint32_t tq = tmem + (uint32_t(32 * (warp & 3)) << 16);  // this warp's lanes
        const float ninf = __int_as_float(0xff800000);
        int g = 0;
        int turn = 0;  // of s_max: written again only two barriers later
        bool ok = true;
        while (ok && walk.next(u)) {
            const int row = u.r * kTaRows + rr;
            const bool there = row < u.seq.q * a.group;
            const int i_tok = there ? row / a.group : 0;
            const int tok = u.seq.row0 + i_tok, head = u.h * a.group + (there ? row % a.group : 0);
            // Q of the row, half of the dims (the previous unit's MMAs are done: their last commit was waited for)
            float qf;
            {
                const int64_t q0 = tok * a.qs_tok + head * a.qs_head + hf * (D / 2);
                float m = 0.0f;
                if (there)
                    for (int d = 0; d < D / 2; d += 8) {
                        float x[8];
                        attn_q8(a, q0 + d, x);
#pragma unroll
                        for (int k = 0; k < 8; k++) m = fmaxf(m, fabsf(x[k]));
                    }
                s_max[turn][hf][rr] = m;
                soft_sync();
                m = fmaxf(m, s_max[turn][hf ^ 1][rr]);
                turn ^= 1;
                const int sh = attn_q_shift(m);
                const float f = a.scale_log2 < 0.0f ? -attn_exp2i(sh) : attn_exp2i(sh);
                qf = attn_exp2i(-sh) * fabsf(a.scale_log2);  // (a negative scale turns q's sign: factors are positive)
#pragma unroll 2
                for (int j = 0; j < D / 16; j++) {  // 16-byte units
                    float x[8] = {};
                    uint32_t hi[4], lo[4];
                    if (there) attn_q8(a, q0 + 8 * j, x);
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const float x0 = x[2 * k] * f, x1 = x[2 * k + 1] * f;
                        const __half2 h = __floats2half2_rn(x0, x1);
                        hi[k] = half2_u32(h);
                        if constexpr (SPLIT) lo[k] = pack_h2(x0 - __low2float(h), x1 - __high2float(h));
                    }
                    const int d8 = hf * (D / 16) + j;
                    uint8_t *at = sQ + (d8 >> 3) * C::kBlock + rr * 128 + (((d8 & 7) ^ (rr & 7)) << 4);
                    *reinterpret_cast<uint4 *>(at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    if constexpr (SPLIT) *reinterpret_cast<uint4 *>(at + C::kQ) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                }
                fence_proxy_async_smem();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(q_full);
            }
            const int lim = !there ? 0 : a.causal ? min(u.seq.kv, u.seq.kv - u.seq.q + i_tok + 1) : u.seq.kv;
            float ref = ninf, sum = 0.0f, vinv = 0.0f;  // (1 / unit)
            const int n = u.t1 - u.t0;
            // half of the row's columns, by fours
            auto flushed = [&]() {  // (from special registers: none held meanwhile)
                uint32_t cta, thread;
                asm volatile("mov.u32 %0, %%ctaid.x;" : "=r"(cta));
                asm volatile("mov.u32 %0, %%tid.x;" : "=r"(thread));
                return a.acc + int64_t(cta) * (D / 4 * kTaRows) + ((thread - 128) >> 7) * (D / 8 * kTaRows) + (thread & 127);
            };
            for (int j = 0; j < n; j++, g++) {
                const int slot = g % kTaInfo;
                const int key0 = (u.t0 + j) * kTaTile + kTaHalf * hf;
                if (!__all_sync(0xffffffffu, tc_wait(&info_full[slot], uint32_t(g / kTaInfo) & 1u, abort_flag) &&
                                                 tc_wait(&s_full[g & 1], uint32_t(g >> 1) & 1u, abort_flag)))
                    ok = false;
                tc_fence_after();
                const uint32_t ts = tq + C::kColS + uint32_t(kTaTile) * uint32_t(g & 1) + uint32_t(kTaHalf * hf);
                const TaInfo &in = info[slot];
                float vmax = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; i++) vmax = fmaxf(vmax, in.vs[i]);  // 0 where there is no page
                float vf = 1.0f;  // old unit / new unit, the same for all rows
                if (vinv == 0.0f || vmax * vinv > kAttnVHigh) {
                    const float old = vinv;
                    vinv = attn_v_unit(vmax);
                    if (old > 0.0f) vf = vinv / old;
                }
                // keys past the row's limit or without a page: -inf in S
                const bool clear = key0 + kTaHalf <= lim && min(min(in.row[4 * hf], in.row[4 * hf + 1]), min(in.row[4 * hf + 2], in.row[4 * hf + 3])) >= 0;
                if (!__all_sync(0xffffffffu, clear)) {
#pragma unroll 1
                    for (int c = 0; c < 4; c++) {
                        uint32_t z[16];
                        tmem_ld16_wait(ts + 16u * uint32_t(c), z);
                        const int n_in = in.row[4 * hf + c] >= 0 ? lim - (key0 + 16 * c) : 0;
#pragma unroll
                        for (int i = 0; i < 16; i++) z[i] = i < n_in ? z[i] : 0xff800000u;
                        tmem_st16_async(ts + 16u * uint32_t(c), z);
                    }
                    tmem_wait_st();
                }
                // the largest contribution (log2, from the reference on, rounded as P's exponents below)
                float base = ref == ninf ? 0.0f : ref;
                const float limit = ref == ninf ? ninf : kAttnRefMove;
                float top = ninf;
#pragma unroll 1
                for (int c = 0; c < 2; c++) {
                    float z[32];
                    tmem_ld32_wait(ts + 32u * uint32_t(c), z);
                    float m[4];
#pragma unroll
                    for (int i = 0; i < 32; i++) m[i >> 3] = (i & 7) == 0 ? z[i] : fmaxf(m[i >> 3], z[i]);
                    const int i = 4 * hf + 2 * c;
                    top = fmaxf(top, fmaxf(__fmaf_rn(fmaxf(m[0], m[1]), ta_factor(in.ks[i] * qf), -base) + attn_v_log(in.vs[i] * vinv),
                                           __fmaf_rn(fmaxf(m[2], m[3]), ta_factor(in.ks[i + 1] * qf), -base) + attn_v_log(in.vs[i + 1] * vinv)));
                }
                s_max[turn][hf][rr] = top;
                soft_sync();
                top = fmaxf(top, s_max[turn][hf ^ 1][rr]);
                turn ^= 1;
                if (j > 0 && j % C::kFlush == 0) {  // half of O's columns to the workspace; P(j) V begins a new O
                    if (!__all_sync(0xffffffffu, tc_wait(pv_done, uint32_t(g - 1) & 1u, abort_flag))) ok = false;
                    tc_fence_after();
                    float4 *const acc = flushed();
#pragma unroll 1
                    for (int c = 0; c < D / 32; c++) {
                        uint32_t o[16];
                        tmem_ld16_wait(tq + C::kColO + uint32_t(hf * (D / 2) + 16 * c), o);
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            attn_flush4(acc + (4 * c + i) * kTaRows, j == C::kFlush, __uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]),
                                        __uint_as_float(o[4 * i + 2]), __uint_as_float(o[4 * i + 3]));
                    }
                }
                if (__any_sync(0xffffffffu, top > limit || vf != 1.0f)) {
                    float f = vf;
                    if (top > limit) {
                        const float to = base + (floorf(top) - kAttnRefDrop), e = ex2(ref - to);
                        ref = base = to;
                        sum *= e;
                        f *= e;
                    }
                    if (j >= C::kFlush) {
                        float4 *const acc = flushed();
#pragma unroll 1
                        for (int c = 0; c < D / 8; c++) attn_scale4(acc + c * kTaRows, f, f);
                    }
                    if (j % C::kFlush) {  // half of O's columns, once P(j - 1) V has been added
                        if (!__all_sync(0xffffffffu, tc_wait(pv_done, uint32_t(g - 1) & 1u, abort_flag))) ok = false;
                        tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < D / 64; c++) {
                            float o[32];
                            uint32_t b[32];
                            const uint32_t col = C::kColO + uint32_t(hf * (D / 2) + 32 * c);
                            tmem_ld32_wait(tq + col, o);
#pragma unroll
                            for (int i = 0; i < 32; i++) b[i] = __float_as_uint(o[i] * f);
                            tmem_st32_async(tq + col, b);
                        }
                    }
                }
                const uint64_t nbase = f2_pack(-base, -base);
                uint64_t part[2] = {0, 0};  // (two zeros each)
#pragma unroll 1
                for (int c = 0; c < 4; c++) {
                    uint32_t z[16], hi[8], lo[8];
                    tmem_ld16_wait(ts + 16u * uint32_t(c), z);
                    const float kf = ta_factor(in.ks[4 * hf + c] * qf), r = in.vs[4 * hf + c] * vinv;
                    const uint64_t kf2 = f2_pack(kf, kf), r2 = f2_pack(r, r);
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        float p0, p1;
                        f2_unpack(f2_fma(f2_pack(__uint_as_float(z[2 * i]), __uint_as_float(z[2 * i + 1])), kf2, nbase), p0, p1);
                        const uint64_t p = f2_pack(ex2(p0), ex2(p1));
                        part[i & 1] = f2_add(part[i & 1], p);
                        f2_unpack(f2_mul(p, r2), p0, p1);
                        hi[i] = pack_h2(p0, p1);
                        if constexpr (SPLIT) {
                            const float2 f = __half22float2(u32_half2(hi[i]));
                            lo[i] = pack_h2(p0 - f.x, p1 - f.y);
                        }
                    }
                    tmem_st8_async(ts + 16u * uint32_t(c), hi);
                    if constexpr (SPLIT) tmem_st8_async(ts + 16u * uint32_t(c) + 8u, lo);
                }
                {
                    float s0, s1;
                    f2_unpack(f2_add(part[0], part[1]), s0, s1);
                    sum += s0 + s1;
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&p_full[g & 1]);
                    mbar_arrive(&info_empty[slot]);
                }
            }
            // the unit's rows, half of the columns: O / sum to the output, or O and its statistics to the workspace
            // (the last two P V may both be under way: the barrier's phases are waited for one by one)
            if (n > 1 && !__all_sync(0xffffffffu, tc_wait(pv_done, uint32_t(g - 2) & 1u, abort_flag))) ok = false;
            if (!__all_sync(0xffffffffu, tc_wait(pv_done, uint32_t(g - 1) & 1u, abort_flag))) ok = false;
            tc_fence_after();
            if (n > C::kFlush) {  // what O held before
                const float4 *const acc = flushed();
#pragma unroll 1
                for (int c = 0; c < D / 32; c++) {
                    uint32_t o[16];
                    const uint32_t at = tq + C::kColO + uint32_t(hf * (D / 2) + 16 * c);
                    tmem_ld16_wait(at, o);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float4 v = __ldcg(acc + (4 * c + i) * kTaRows);
                        o[4 * i] = __float_as_uint(__uint_as_float(o[4 * i]) + v.x);
                        o[4 * i + 1] = __float_as_uint(__uint_as_float(o[4 * i + 1]) + v.y);
                        o[4 * i + 2] = __float_as_uint(__uint_as_float(o[4 * i + 2]) + v.z);
                        o[4 * i + 3] = __float_as_uint(__uint_as_float(o[4 * i + 3]) + v.w);
                    }
                    tmem_st16_async(at, o);
                }
                tmem_wait_st();
            }
            s_max[turn][hf][rr] = sum;
            ok = !soft_any(!ok || *abort_flag);
            sum += s_max[turn][hf ^ 1][rr];
            turn ^= 1;
            const bool whole = u.t0 == 0 && u.t1 == u.n;
            const int slot = attn_slot(u);
            const float f = whole ? attn_v_scale(vinv) * attn_inverse(sum) : attn_v_scale(vinv);
#pragma unroll 1
            for (int c = 0; c < D / 64; c++) {
                float o[32];
                const int d = hf * (D / 2) + 32 * c;
                tmem_ld32_wait(tq + C::kColO + uint32_t(d), o);
#pragma unroll
                for (int i = 0; i < 32; i++) o[i] *= f;
                if (whole) {
                    if (there) attn_out32(a, tok * a.os_tok + head * a.os_head + d, o);
                } else {
                    float4 *to = reinterpret_cast<float4 *>(a.part_o + (int64_t(slot) * kTaRows + rr) * D + d);
#pragma unroll
                    for (int i = 0; i < 8; i++) to[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                }
            }
            if (hf == 0) {
                if (whole) {
                    if (there && a.lse) a.lse[int64_t(tok) * (a.hkv * a.group) + head] = attn_lse(ref, sum);
                } else {
                    a.part_ml[slot * kTaRows + rr] = make_float2(ref, sum);
                    if (rr == 0) a.part_hdr[slot] = make_int4(u.s, u.r, u.h, u.t1 == u.n ? 2 : 1);
                }
            }
            tc_fence_before();  // the reads of O come before the next unit's MMAs (ordered by q_full)
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

}  // namespace cpq
