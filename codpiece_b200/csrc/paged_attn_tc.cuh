// paged_attn_tc.cuh — attention over the paged 8-bit cache for many query rows
// (verify, chunked prefill) on tcgen05 tensor cores. Mathematics, numbers and
// split as in paged_attn.cuh; a row tile is 128 rows, a key tile 64 keys.
//
// Per key tile the tensor core does S[128 x 64] = Q K^T and O[128 x D] += P V
// (fp32 q: twice each, the two fp16 terms of Q and of P). At D = 256 these are
// 1024 (2048) tensor cycles, against 32 KB of codes from L2 or HBM; what the
// design has to hide behind them is the softmax of 128 x 64 scores (512 cycles
// of ex2 alone per SM sub-partition) and turning 32 KB of codes into 64 KB of
// fp16 operands.
//
// Tensor memory (512 columns): O, fp32 [128][D]; Q, fp16 [128][D] (first
// terms; A operand, so Q costs no shared-memory reads); S, fp32 [128][64]; P,
// fp16 [128][64] first and second terms. Shared memory: two stages each of K
// [64 keys][D] and V [64 keys][D] in fp16, both as D / 64 blocks of 64 rows x
// 128 bytes with the 128-byte swizzle: the K-major operand of the first product
// (N = keys, K = dims) and the MN-major operand of the second (N = dims, K =
// keys) are the same bytes, so both come from the same conversion; fp32 q's
// second terms.
//
//   warp 0       one lane issues the MMAs: S(i + 1) as soon as the softmax has
//                read S(i), then O += P(i) V(i); so S(i + 1) is made during
//                softmax(i) and P(i) V(i) runs during softmax(i + 1)
//   warp 1       the key tiles' cache rows and page scales, eight tiles ahead
//   warps 4-7    softmax, one query row per thread: S to registers, reference
//                and sums as in paged_attn.cuh, P back to tensor memory; they
//                also load Q, rescale O when a reference moves, and write the
//                unit's rows out
//   warps 8-15   conversion: 16 bytes of codes per load, kept one tile ahead in
//                registers; keys that are not there become zeros
//
// Waits are bounded as everywhere (a timeout sets the device error word and an
// abort flag; MMAs in flight are waited for before tensor memory is released).
#pragma once

#include "paged_attn.cuh"

namespace cpq {

constexpr int kTaRows = 128;
constexpr int kTaTile = 64;
constexpr int kTaThreads = 512;
constexpr int kTaConvWarps = 8;
constexpr int kTaInfo = 8;  // key tiles looked up ahead

struct TaInfo {
    int row[4];     // cache row of each 16 keys' first one, -1: no such keys
    float ks[4], vs[4];
};

template <int D, bool SPLIT> struct TaCfg {
    static constexpr int kOperand = kTaTile * D * 2;     // a stage of K or V
    static constexpr int kQlOff = 4 * kOperand;
    static constexpr int kPlanOff = kQlOff + (SPLIT ? kTaRows * D * 2 : 0);
    static constexpr int kInfoOff = (kPlanOff + int(sizeof(AttnPlan)) + 15) / 16 * 16;
    static constexpr int kBarOff = (kInfoOff + kTaInfo * int(sizeof(TaInfo)) + 15) / 16 * 16;
    static constexpr int kBars = 2 * kTaInfo + 8 + 6;
    static constexpr int kSmem = kBarOff + kBars * 8 + 16 + 1024;
    // tensor memory columns
    static constexpr uint32_t kColO = 0, kColQ = D, kColS = D + D / 2, kColP = kColS + kTaTile;
    static_assert(kColP + kTaTile <= 512, "TMEM columns");
    static_assert(kSmem <= 227 * 1024, "shared memory");
};

// MN-major SWIZZLE_128B operand: rows of 64 elements (128 bytes) along N, one
// per k; 8-row groups 1024 bytes apart (stride byte offset), the next 64 elements
// of N `lbo` bytes on (leading byte offset).
__device__ __forceinline__ uint64_t smem_desc_sw128_mn(uint32_t saddr, uint32_t lbo) {
    return uint64_t((saddr >> 4) & 0x3fffu) | (uint64_t(lbo >> 4) << 16) | (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) |
           (uint64_t(2) << 61);
}

// One-SM MMAs: D (TMEM) (+)= A x B with A in TMEM or shared memory.
__device__ __forceinline__ void tc_mma1_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tc_mma1_f16_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tc_commit1(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}

__device__ __forceinline__ uint4 ldg_codes(const uint8_t *p) {
    uint4 r;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
    return r;
}

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
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *sK = smem, *sV = smem + 2 * C::kOperand, *sQl = smem + C::kQlOff;
    AttnPlan &plan = *reinterpret_cast<AttnPlan *>(smem + C::kPlanOff);
    TaInfo *info = reinterpret_cast<TaInfo *>(smem + C::kInfoOff);
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + C::kBarOff);
    uint64_t *info_full = bars, *info_empty = bars + kTaInfo;
    uint64_t *k_full = bars + 2 * kTaInfo, *k_empty = k_full + 2, *v_full = k_full + 4, *v_empty = k_full + 6;
    uint64_t *q_full = k_full + 8, *s_full = q_full + 1, *s_empty = q_full + 2, *p_full = q_full + 3, *pv_done = q_full + 4,
             *stopped = q_full + 5;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + C::kBars);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kTaInfo; i++) {
            mbar_init(&info_full[i], 1);
            mbar_init(&info_empty[i], kTaConvWarps + 4);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&k_full[i], kTaConvWarps);
            mbar_init(&k_empty[i], 1);
            mbar_init(&v_full[i], kTaConvWarps);
            mbar_init(&v_empty[i], 1);
        }
        mbar_init(q_full, 4);
        mbar_init(s_full, 1);
        mbar_init(s_empty, 4);
        mbar_init(p_full, 4);
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
    attn_make_plan<kTaRows, kTaTile>(a, plan);  // (its barriers also publish the TMEM address)
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    AttnWalk<kTaRows, kTaTile> walk(a, plan);
    AttnUnit u;
    // g: key tiles of this CTA so far, over units; a stage, its parities and the info slot follow from it

    if (warp == 0) {
        // ---- MMA issue ----
        if (lane == 0) {
            constexpr uint32_t idesc_s = tc_idesc_f16(kTaRows, kTaTile);
            constexpr uint32_t idesc_o = tc_idesc_f16(kTaRows, D) | (1u << 16);  // B is MN-major
            int g = 0, n_units = 0;
            bool ok = true, issued = false;
            // S = Q K(gi)^T
            auto scores = [&](int gi) {
                const int st = gi & 1;
                if (!tc_wait(&k_full[st], uint32_t(gi >> 1) & 1u, abort_flag)) return false;
                if (gi > 0 && !tc_wait(s_empty, uint32_t(gi - 1) & 1u, abort_flag)) return false;
                tc_fence_after();
                const uint64_t bd = smem_desc_sw128(smem_addr(sK + st * C::kOperand));
#pragma unroll
                for (int ks = 0; ks < D / 16; ks++)
                    tc_mma1_f16_ts(tmem + C::kColS, tmem + C::kColQ + 8u * uint32_t(ks), bd + uint64_t((ks >> 2) * (kTaTile * 128 / 16) + 2 * (ks & 3)),
                                   idesc_s, ks ? 1u : 0u);
                if constexpr (SPLIT) {
                    const uint64_t ad = smem_desc_sw128(smem_addr(sQl));
#pragma unroll
                    for (int ks = 0; ks < D / 16; ks++)
                        tc_mma1_f16_ss(tmem + C::kColS, ad + uint64_t((ks >> 2) * (kTaRows * 128 / 16) + 2 * (ks & 3)),
                                       bd + uint64_t((ks >> 2) * (kTaTile * 128 / 16) + 2 * (ks & 3)), idesc_s, 1u);
                }
                tc_commit1(&k_empty[st]);
                tc_commit1(s_full);
                issued = true;
                return true;
            };
            while (ok && walk.next(u)) {
                const int n = u.t1 - u.t0;
                ok = tc_wait(q_full, uint32_t(n_units) & 1u, abort_flag);
                n_units++;
                ok = ok && scores(g);
                for (int j = 0; ok && j < n; j++, g++) {
                    if (j + 1 < n && !scores(g + 1)) {
                        ok = false;
                        break;
                    }
                    const int st = g & 1;
                    if (!tc_wait(&v_full[st], uint32_t(g >> 1) & 1u, abort_flag) || !tc_wait(p_full, uint32_t(g) & 1u, abort_flag)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t sv = smem_addr(sV + st * C::kOperand);
#pragma unroll
                    for (int t = 0; t < (SPLIT ? 2 : 1); t++)
#pragma unroll
                        for (int ks = 0; ks < kTaTile / 16; ks++)
                            tc_mma1_f16_ts(tmem + C::kColO, tmem + C::kColP + 32u * uint32_t(t) + 8u * uint32_t(ks),
                                           smem_desc_sw128_mn(sv + 2048u * uint32_t(ks), kTaTile * 128), idesc_o, (j | t | ks) ? 1u : 0u);
                    tc_commit1(&v_empty[st]);
                    tc_commit1(pv_done);
                }
            }
            // MMAs in flight end before tensor memory is released: normally the softmax warps have waited for the
            // last of them; after an early stop one more commit tracks what was issued
            if (!ok && issued) {
                tc_commit1(stopped);
                mbar_wait_bounded(stopped, 0);
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ---- cache rows and scales of the key tiles: lane = (tile of eight, 16 keys of four) ----
        const int lb = a.block == 16 ? 4 : a.block == 32 ? 5 : a.block == 64 ? 6 : 7;
        int g = 0;
        bool ok = true;
        while (ok && walk.next(u)) {
            for (int b0 = u.t0; ok && b0 < u.t1; b0 += 8) {
                const int key = (b0 + (lane >> 2)) * kTaTile + 16 * (lane & 3);
                int row = -1;
                float ks = 0.0f, vs = 0.0f;
                if (b0 + (lane >> 2) < u.t1 && key < u.kv_end) {
                    const int page = attn_page(a, u.s, key >> lb);
                    if (page >= 0) {
                        row = (page * a.hkv + u.h) * a.block + (key & (a.block - 1));
                        ks = a.k_scale[int64_t(page) * a.hkv + u.h];
                        vs = a.v_scale[int64_t(page) * a.hkv + u.h];
                    }
                }
                const int n = min(8, u.t1 - b0);
                for (int i = 0; i < n; i++, g++) {
                    const int slot = g % kTaInfo;
                    if (!__all_sync(0xffffffffu, tc_wait(&info_empty[slot], (uint32_t(g / kTaInfo) & 1u) ^ 1u, abort_flag))) {
                        ok = false;
                        break;
                    }
                    if ((lane >> 2) == i) {
                        info[slot].row[lane & 3] = row;
                        info[slot].ks[lane & 3] = ks;
                        info[slot].vs[lane & 3] = vs;
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&info_full[slot]);
                }
            }
        }
    } else if (warp >= 8) {
        // ---- conversion: rows 8 w .. 8 w + 7 of every tile ----
        const int w = warp - 8;
        constexpr int kLanes = D / 16, kPer = 32 / kLanes, kLoads = 8 / kPer;  // lanes per key, keys per load, loads
        const int key_in = 8 * w + lane / kLanes, d0 = (lane % kLanes) * 16;   // of load 0; load i: + kPer i keys
        // where the lane's 16 values go: two 16-byte units of its 64-dim block. Odd blocks store their second
        // unit first, so that a quarter warp's eight stores fall into eight bank groups.
        const int blk = d0 >> 6, unit = (d0 & 63) >> 3, swap = blk & 1;
        // row: the cache row of the warp's 16 keys' first one; keys past kv or without a page read as code 0, zero in
        // both formats
        auto rows_of = [&](const uint8_t *base, int row, int key0, int kv, uint4 (&x)[kLoads]) {
#pragma unroll
            for (int i = 0; i < kLoads; i++) {
                const int k = key_in + kPer * i;
                x[i] = make_uint4(0, 0, 0, 0);
                if (row >= 0 && key0 + k < kv) x[i] = ldg_codes(base + (int64_t(row) + (k & 15)) * D + d0);
            }
        };
        auto store = [&](uint8_t *dst, const uint4 (&x)[kLoads]) {
#pragma unroll
            for (int i = 0; i < kLoads; i++) {
                const int k = key_in + kPer * i;
                uint32_t h[8];
                codes_h2<FMT>(x[i].x, h[0], h[1]);
                codes_h2<FMT>(x[i].y, h[2], h[3]);
                codes_h2<FMT>(x[i].z, h[4], h[5]);
                codes_h2<FMT>(x[i].w, h[6], h[7]);
                const uint4 lo = make_uint4(h[0], h[1], h[2], h[3]), hi = make_uint4(h[4], h[5], h[6], h[7]);
                uint8_t *at = dst + blk * (kTaTile * 128) + k * 128;
                *reinterpret_cast<uint4 *>(at + (((unit + swap) ^ (k & 7)) << 4)) = swap ? hi : lo;
                *reinterpret_cast<uint4 *>(at + (((unit + (swap ^ 1)) ^ (k & 7)) << 4)) = swap ? lo : hi;
            }
        };
        // tiles in order over units: cur is being converted, the walk stands at the next
        AttnUnit nu;
        int nt = 0;
        bool more = walk.next(nu);
        if (more) nt = nu.t0;
        uint4 xk[kLoads], xv[kLoads];
        bool ok = true;
        int in_row = -1, in_key0 = 0, in_kv = 0;
        auto look = [&](int gi) {  // the info of tile gi, the walk's next
            if (!__all_sync(0xffffffffu, tc_wait(&info_full[gi % kTaInfo], uint32_t(gi / kTaInfo) & 1u, abort_flag))) return false;
            in_row = info[gi % kTaInfo].row[w >> 1];  // a warp's eight keys lie in one group of 16
            in_key0 = nt * kTaTile;
            in_kv = nu.seq.kv;
            __syncwarp();
            if (lane == 0) mbar_arrive(&info_empty[gi % kTaInfo]);
            if (++nt == nu.t1) {
                more = walk.next(nu);
                nt = more ? nu.t0 : 0;
            }
            return true;
        };
        if (more) {
            ok = look(0);
            if (ok) {
                rows_of(a.k, in_row, in_key0, in_kv, xk);
                rows_of(a.v, in_row, in_key0, in_kv, xv);
            }
            for (int g = 0; ok; g++) {
                const int st = g & 1;
                const uint32_t ph = (uint32_t(g >> 1) & 1u) ^ 1u;
                const bool next = more;
                if (!__all_sync(0xffffffffu, tc_wait(&k_empty[st], ph, abort_flag))) break;
                store(sK + st * C::kOperand, xk);
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&k_full[st]);
                if (next) {
                    if (!look(g + 1)) break;
                    rows_of(a.k, in_row, in_key0, in_kv, xk);
                }
                if (!__all_sync(0xffffffffu, tc_wait(&v_empty[st], ph, abort_flag))) break;
                store(sV + st * C::kOperand, xv);
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&v_full[st]);
                if (!next) break;
                rows_of(a.v, in_row, in_key0, in_kv, xv);
            }
        }
    } else if (warp >= 4) {
        // ---- softmax: thread = row ----
        const int rr = 32 * (warp - 4) + lane;
        const uint32_t tq = tmem + (uint32_t(32 * (warp - 4)) << 16);  // this warp's lanes
        const float ninf = __int_as_float(0xff800000);
        int g = 0;
        bool ok = true;
        while (ok && walk.next(u)) {
            const int row = u.r * kTaRows + rr;
            const bool there = row < u.seq.q * a.group;
            const int i_tok = there ? row / a.group : 0;
            const int tok = u.seq.row0 + i_tok, head = u.h * a.group + (there ? row % a.group : 0);
            // Q of the row (the previous unit's MMAs are done: their last commit was waited for)
            float qf;
            {
                const int64_t q0 = tok * a.qs_tok + head * a.qs_head;
                float m = 0.0f;
                if (there)
                    for (int d = 0; d < D; d += 8) {
                        float x[8];
                        attn_q8(a, q0 + d, x);
#pragma unroll
                        for (int k = 0; k < 8; k++) m = fmaxf(m, fabsf(x[k]));
                    }
                const int sh = attn_q_shift(m);
                const float f = attn_exp2i(sh);
                qf = attn_exp2i(-sh) * a.scale_log2;
#pragma unroll 1
                for (int c = 0; c < D / 64; c++) {
                    uint32_t hi[32], lo[32];
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        float x[8] = {};
                        if (there) attn_q8(a, q0 + 64 * c + 8 * j, x);
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            const float x0 = x[2 * k] * f, x1 = x[2 * k + 1] * f;
                            const __half2 h = __floats2half2_rn(x0, x1);
                            hi[4 * j + k] = half2_u32(h);
                            if constexpr (SPLIT) lo[4 * j + k] = pack_h2(x0 - __low2float(h), x1 - __high2float(h));
                        }
                    }
                    tmem_st32_async(tq + C::kColQ + 32u * uint32_t(c), hi);
                    if constexpr (SPLIT) {
#pragma unroll
                        for (int j = 0; j < 8; j++)
                            *reinterpret_cast<uint4 *>(sQl + c * (kTaRows * 128) + rr * 128 + ((j ^ (rr & 7)) << 4)) =
                                make_uint4(lo[4 * j], lo[4 * j + 1], lo[4 * j + 2], lo[4 * j + 3]);
                    }
                }
                tmem_wait_st();
                if constexpr (SPLIT) fence_proxy_async_smem();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(q_full);
            }
            const int lim = !there ? 0 : a.causal ? min(u.seq.kv, u.seq.kv - u.seq.q + i_tok + 1) : u.seq.kv;
            float ref = ninf, sum = 0.0f, vref = 0.0f;
            const int n = u.t1 - u.t0;
            for (int j = 0; j < n; j++, g++) {
                const int slot = g % kTaInfo;
                const int key0 = (u.t0 + j) * kTaTile;
                if (!__all_sync(0xffffffffu, tc_wait(&info_full[slot], uint32_t(g / kTaInfo) & 1u, abort_flag) &&
                                                 tc_wait(s_full, uint32_t(g) & 1u, abort_flag))) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                float ks[4], vs[4];
                bool in[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    ks[i] = info[slot].ks[i] * qf;
                    vs[i] = info[slot].vs[i];
                    in[i] = info[slot].row[i] >= 0;
                }
                float z[2][32];
                tmem_ld32(tq + C::kColS, z[0]);
                tmem_ld32(tq + C::kColS + 32u, z[1]);
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(s_empty);
                    mbar_arrive(&info_empty[slot]);
                }
                // scores in log2; keys past the row's limit or without a page count as -inf
                float mx = ninf;
                const bool clear = key0 + kTaTile <= lim && in[0] && in[1] && in[2] && in[3];
                if (__all_sync(0xffffffffu, clear)) {
#pragma unroll
                    for (int i = 0; i < 64; i++) {
                        z[i >> 5][i & 31] *= ks[i >> 4];
                        mx = fmaxf(mx, z[i >> 5][i & 31]);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 64; i++) {
                        z[i >> 5][i & 31] = in[i >> 4] && key0 + i < lim ? z[i >> 5][i & 31] * ks[i >> 4] : ninf;
                        mx = fmaxf(mx, z[i >> 5][i & 31]);
                    }
                }
                // P(j - 1) V has been added: P and O are free
                if (j > 0) {
                    if (!__all_sync(0xffffffffu, tc_wait(pv_done, uint32_t(g - 1) & 1u, abort_flag))) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                }
                const float vmax = fmaxf(fmaxf(in[0] ? vs[0] : 0.0f, in[1] ? vs[1] : 0.0f), fmaxf(in[2] ? vs[2] : 0.0f, in[3] ? vs[3] : 0.0f));
                if (__any_sync(0xffffffffu, mx > ref + kAttnRefMove || vmax > kAttnVRatio * vref)) {
                    const float vnew = vmax > kAttnVRatio * vref ? vmax : vref;
                    float f = vnew > 0.0f ? vref / vnew : 0.0f;
                    vref = vnew;
                    if (mx > ref + kAttnRefMove) {
                        const float to = mx - kAttnRefDrop, e = ex2(ref - to);
                        ref = to;
                        sum *= e;
                        f *= e;
                    }
                    if (j > 0) {
#pragma unroll 1
                        for (int c = 0; c < D / 32; c++) {
                            float o[32];
                            uint32_t b[32];
                            tmem_ld32(tq + C::kColO + 32u * uint32_t(c), o);
#pragma unroll
                            for (int i = 0; i < 32; i++) b[i] = __float_as_uint(o[i] * f);
                            tmem_st32_async(tq + C::kColO + 32u * uint32_t(c), b);
                        }
                    }
                }
                const float base = ref == ninf ? 0.0f : ref;
                float ratio[4];
#pragma unroll
                for (int i = 0; i < 4; i++) ratio[i] = in[i] && vref > 0.0f ? vs[i] / vref : 0.0f;
                uint32_t hi[32];
#pragma unroll
                for (int i = 0; i < 32; i++) {
                    float &p0 = z[i >> 4][(2 * i) & 31], &p1 = z[i >> 4][(2 * i + 1) & 31];
                    p0 = ex2(p0 - base);
                    p1 = ex2(p1 - base);
                    sum += p0 + p1;
                    p0 *= ratio[i >> 3];
                    p1 *= ratio[i >> 3];
                    hi[i] = pack_h2(p0, p1);
                }
                tmem_st32_async(tq + C::kColP, hi);
                if constexpr (SPLIT) {
#pragma unroll
                    for (int i = 0; i < 32; i++) {
                        const float2 h = __half22float2(u32_half2(hi[i]));
                        hi[i] = pack_h2(z[i >> 4][(2 * i) & 31] - h.x, z[i >> 4][(2 * i + 1) & 31] - h.y);
                    }
                    tmem_st32_async(tq + C::kColP + 32u, hi);
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full);
            }
            if (!ok) break;
            // the unit's rows: O / sum to the output, or O and its statistics to the workspace
            if (!__all_sync(0xffffffffu, tc_wait(pv_done, uint32_t(g - 1) & 1u, abort_flag))) break;
            tc_fence_after();
            const bool whole = u.t0 == 0 && u.t1 == u.n;
            const int slot = attn_slot(u);
            const float f = whole ? vref * attn_inverse(sum) : vref;
#pragma unroll 1
            for (int c = 0; c < D / 32; c++) {
                float o[32];
                tmem_ld32(tq + C::kColO + 32u * uint32_t(c), o);
#pragma unroll
                for (int i = 0; i < 32; i++) o[i] *= f;
                if (whole) {
                    if (there) attn_out32(a, tok * a.os_tok + head * a.os_head + 32 * c, o);
                } else {
                    float4 *to = reinterpret_cast<float4 *>(a.part_o + (int64_t(slot) * kTaRows + rr) * D + 32 * c);
#pragma unroll
                    for (int i = 0; i < 8; i++) to[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                }
            }
            if (whole) {
                if (there && a.lse) a.lse[int64_t(tok) * (a.hkv * a.group) + head] = attn_lse(ref, sum);
            } else {
                a.part_ml[slot * kTaRows + rr] = make_float2(ref, sum);
                if (rr == 0) a.part_hdr[slot] = make_int4(u.s, u.r, u.h, u.t1 == u.n ? 2 : 1);
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
