// rope.cuh — rotary positions: ggml_rope_multi / ggml_rope_ext as the attention
// layers apply them to q and k (crates/codpiece-model/src/qwen35.rs:3000-3197),
// for text positions (one position per token).
//
// Pair i of the n_dims / 2 rotated pairs turns by pos * w_i, where w_i is the
// pair's frequency after scaling (rope.inl). Elements from n_dims on are
// copied. The pairs are (2i, 2i + 1) or (i, i + n_dims / 2).
//
// The angle. pos * w_i in fp32 is wrong in the second digit at position 10^6
// (an ulp of 10^6 rad is 0.06). The table holds w_i / 2 pi, the turns per
// position, as a 64-bit fixed-point fraction of a turn; pos times it modulo
// 2^64 is then exactly the fraction of a turn for every int32 position, and
// one conversion to fp32 leaves a relative error of 2^-24 for sincospif.
#pragma once

#include <cuda_bf16.h>

#include <type_traits>

#include "common.cuh"

namespace cpq {

constexpr int kRopeMaxPairs = 128;
constexpr int kRopeMaxTensors = 4;
constexpr int kRopeThreads = 256;
constexpr int kRopeMaxTok = 8;  // tokens of a CTA

// Division of n < 2^31 by a divisor known on the host (round-up method:
// q = (umulhi(n, m) + n) >> s).
struct FastDiv {
    uint32_t d, m, s;
    FastDiv() = default;
    explicit FastDiv(uint32_t div) : d(div), s(0) {
        while ((uint64_t(1) << s) < div) s++;
        m = uint32_t((((uint64_t(1) << s) - div) << 32) / div + 1);
    }
    __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(n, m) + n) >> s; }
};

struct RopeArgs {
    const void *x[kRopeMaxTensors];
    void *y[kRopeMaxTensors];
    int64_t xs_tok[kRopeMaxTensors], xs_head[kRopeMaxTensors];  // elements
    int64_t ys_tok[kRopeMaxTensors], ys_head[kRopeMaxTensors];
    int head0[kRopeMaxTensors + 1];  // first head of each tensor among all
    const int32_t *pos;
    int64_t t;
    int d, n_dims, n_tensors, heads_per_cta, tok_per_cta;
    int pair_items, items;           // a head's items: rotated ones, all
    int step;                        // heads side by side in a CTA
    FastDiv by_items, by_pairs;      // items, n_dims / 2
    float m;                         // magnitude of the rotation
    uint64_t turns[kRopeMaxPairs];
};

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// VEC elements of an activation row: one 16-byte word where they fill one (the
// caller has checked the alignment), else elements loaded and stored one by
// one. (A struct of eight bf16 objects is copied in eight 2-byte accesses.)
template <typename T, int VEC, bool WIDE = (sizeof(T) * VEC == 16)> struct Vec;

template <typename T, int VEC> struct Vec<T, VEC, true> {
    uint4 w;
    __device__ __forceinline__ void load(const T *p) { w = *reinterpret_cast<const uint4 *>(p); }
    __device__ __forceinline__ void store(T *p) const { *reinterpret_cast<uint4 *>(p) = w; }
    __device__ __forceinline__ void get(float (&f)[VEC]) const {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int k = 0; k < 4; k++) {
            if constexpr (sizeof(T) == 4) f[k] = __uint_as_float(u[k]);
            else if constexpr (std::is_same<T, __half>::value) {
                const float2 p = __half22float2(*reinterpret_cast<const __half2 *>(&u[k]));
                f[2 * k] = p.x, f[2 * k + 1] = p.y;
            } else {
                f[2 * k] = __uint_as_float(u[k] << 16);
                f[2 * k + 1] = __uint_as_float(u[k] & 0xffff0000u);
            }
        }
    }
    // the first n elements (n even); the others stay
    __device__ __forceinline__ void set(const float (&f)[VEC], int n = VEC) {
        uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int k = 0; k < 4; k++) {
            if (k * (VEC / 4) >= n) break;
            if constexpr (sizeof(T) == 4) u[k] = __float_as_uint(f[k]);
            else if constexpr (std::is_same<T, __half>::value) {
                const __half2 p = __floats2half2_rn(f[2 * k], f[2 * k + 1]);
                u[k] = *reinterpret_cast<const uint32_t *>(&p);
            } else {
                const __nv_bfloat162 p = __floats2bfloat162_rn(f[2 * k], f[2 * k + 1]);
                u[k] = *reinterpret_cast<const uint32_t *>(&p);
            }
        }
        w = make_uint4(u[0], u[1], u[2], u[3]);
    }
};

template <typename T, int VEC> struct Vec<T, VEC, false> {
    T v[VEC];
    __device__ __forceinline__ void load(const T *p) {
#pragma unroll
        for (int k = 0; k < VEC; k++) v[k] = p[k];
    }
    __device__ __forceinline__ void store(T *p) const {
#pragma unroll
        for (int k = 0; k < VEC; k++) p[k] = v[k];
    }
    __device__ __forceinline__ void get(float (&f)[VEC]) const {
#pragma unroll
        for (int k = 0; k < VEC; k++) f[k] = to_f32(v[k]);
    }
    __device__ __forceinline__ void set(const float (&f)[VEC], int n = VEC) {
#pragma unroll
        for (int k = 0; k < VEC; k++)
            if (k < n) v[k] = from_f32<T>(f[k]);
    }
};

// grid (token groups, head groups). An item is VEC pairs of one head (HALF:
// VEC elements of each half; else the pairs in VEC elements) or VEC elements of
// the tail. A thread keeps its place in the head and steps over heads and
// tokens, so an item costs little more than its loads, its rotation and its
// stores (finding each item by division took more instructions than the rest:
// 8191 tokens x 40 heads of 128, bf16, 58 us). The first items' loads are
// issued before the CTA makes its tokens' cos/sin table in shared memory.
// (Four items in flight instead of two: interleaved fp32 88 us instead of 69, bf16
// 36.6 instead of 38.7.)
// Bounded by HBM, one read and one write of each element, and each CTA's
// beginning: that case takes 36.6 us, 4.6 TB/s (0.7 of a measured copy), with
// halves in fp32 58.7 us, 5.7 TB/s; 8 tokens x 28 heads 2.3 us, a launch.
template <typename T, int VEC, bool HALF>
__global__ void __launch_bounds__(kRopeThreads, 4) rope_kernel(const __grid_constant__ RopeArgs a) {
    __shared__ __align__(16) float2 cs[kRopeMaxTok * kRopeMaxPairs];
    using V = Vec<T, VEC>;
    constexpr int NV = HALF ? 2 : 1, kBatch = HALF || sizeof(T) == 4 ? 2 : 4;  // items of a thread in flight
    constexpr int kPairs = HALF ? VEC : VEC / 2;  // of an item
    const int half_n = a.n_dims / 2, row = (half_n + 1) & ~1;
    const int64_t tok0 = int64_t(blockIdx.x) * a.tok_per_cta;
    const int n_tok = int(min(int64_t(a.tok_per_cta), a.t - tok0));
    const int h0 = blockIdx.y * a.heads_per_cta, h_end = min(h0 + a.heads_per_cta, a.head0[a.n_tensors]);
    const int tail0 = HALF ? a.n_dims : a.pair_items * VEC;  // first element that only tail items cover
    const int sub = int(a.by_items.div(threadIdx.x));         // which of `step` heads at a time
    const int step = a.step;

    pdl_wait();
    pdl_launch_dependents();
    bool table = false;
    for (int ten = 0; ten < a.n_tensors; ten++) {
        const int first = max(h0 - a.head0[ten], 0), heads = min(h_end, a.head0[ten + 1]) - a.head0[ten] - first;
        if (heads <= 0) continue;
        const T *const xb = static_cast<const T *>(a.x[ten]) + tok0 * a.xs_tok[ten] + first * a.xs_head[ten];
        T *const yb = static_cast<T *>(a.y[ten]) + tok0 * a.ys_tok[ten] + first * a.ys_head[ten];
        const int64_t xt = a.xs_tok[ten], xh = a.xs_head[ten], yt = a.ys_tok[ten], yh = a.ys_head[ten];
        for (int it = int(threadIdx.x) - sub * a.items; it < a.items || !table; it += kRopeThreads) {
            const bool turn = it < a.pair_items;
            const int e = turn ? it * VEC : tail0 + (it - a.pair_items) * VEC;
            V u[kBatch][NV];
            T *to[kBatch];
            int at[kBatch];                   // the items' tokens, n_tok: none
            int h = sub, tk = it < a.items && sub < step ? 0 : n_tok;  // the next item
            auto load = [&](int b) {
                while (h >= heads && tk < n_tok) h -= heads, tk++;
                at[b] = tk;
                if (tk >= n_tok) return;
                const T *x = xb + tk * xt + h * xh + e;
                to[b] = yb + tk * yt + h * yh + e;
                u[b][0].load(x);
                if constexpr (HALF)
                    if (turn) u[b][1].load(x + half_n);
                h += step;
            };
            auto finish = [&](int b) {
                if (at[b] >= n_tok) return;
                if (turn) {
                    float2 r[kPairs];
                    const float2 *c = cs + at[b] * row + it * kPairs;
                    if constexpr (kPairs >= 2) {
#pragma unroll
                        for (int k = 0; k < kPairs; k += 2) {
                            const float4 f = *reinterpret_cast<const float4 *>(c + k);
                            r[k] = make_float2(f.x, f.y), r[k + 1] = make_float2(f.z, f.w);
                        }
                    } else r[0] = c[0];
                    float f[VEC];
                    u[b][0].get(f);
                    if constexpr (HALF) {
                        float g[VEC];
                        u[b][1].get(g);
#pragma unroll
                        for (int k = 0; k < VEC; k++) {
                            const float p = f[k], q = g[k];
                            f[k] = p * r[k].x - q * r[k].y;
                            g[k] = p * r[k].y + q * r[k].x;
                        }
                        u[b][1].set(g);
                        u[b][1].store(to[b] + half_n);
                        u[b][0].set(f);
                    } else {
#pragma unroll
                        for (int k = 0; k < VEC; k += 2) {
                            const float p = f[k], q = f[k + 1];
                            f[k] = p * r[k / 2].x - q * r[k / 2].y;
                            f[k + 1] = p * r[k / 2].y + q * r[k / 2].x;
                        }
                        u[b][0].set(f, a.n_dims - e);
                    }
                }
                u[b][0].store(to[b]);
            };
#pragma unroll
            for (int b = 0; b < kBatch; b++) load(b);
            if (!table) {
                for (int i = threadIdx.x; i < n_tok * half_n; i += kRopeThreads) {
                    const int t = int(a.by_pairs.div(uint32_t(i))), p = i - t * half_n;
                    const int64_t phase = int64_t(uint64_t(int64_t(a.pos[tok0 + t])) * a.turns[p]);
                    float s, c;
                    sincospif(__ll2float_rn(phase) * 0x1p-63f, &s, &c);
                    cs[t * row + p] = make_float2(a.m * c, a.m * s);
                }
                __syncthreads();
                table = true;
            }
            while (at[0] < n_tok) {
#pragma unroll
                for (int b = 0; b < kBatch; b++) {
                    finish(b);
                    load(b);
                }
            }
        }
    }
}

}  // namespace cpq
