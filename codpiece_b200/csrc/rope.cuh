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

#include "common.cuh"

namespace cpq {

constexpr int kRopeMaxPairs = 128;
constexpr int kRopeMaxTensors = 4;
constexpr int kRopeThreads = 256;

struct RopeArgs {
    const void *x[kRopeMaxTensors];
    void *y[kRopeMaxTensors];
    int64_t xs_tok[kRopeMaxTensors], xs_head[kRopeMaxTensors];  // elements
    int64_t ys_tok[kRopeMaxTensors], ys_head[kRopeMaxTensors];
    int head0[kRopeMaxTensors + 1];  // first head of each tensor among all
    const int32_t *pos;
    int64_t t;
    int d, n_dims, n_tensors;
    int tok_per_cta, heads_per_cta;
    int copy_tail;  // elements from n_dims on are written too (y is not x)
    float m;        // magnitude of the rotation
    uint64_t turns[kRopeMaxPairs];
};

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// VEC elements; loaded and stored as one 16-byte word where they fill one (the
// caller has checked the alignment), element by element otherwise.
template <typename T, int VEC> struct alignas(sizeof(T) * VEC == 16 ? 16 : alignof(T)) Vec { T v[VEC]; };

// grid (token groups, head groups). A CTA makes its tokens' cos/sin once in
// shared memory and applies them to its heads. An item is VEC pairs of one
// head (HALF: VEC elements of each half; else 2 pairs or more in VEC
// elements), then VEC elements of the tail.
template <typename T, int VEC, bool HALF>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const __grid_constant__ RopeArgs a) {
    extern __shared__ float2 cs[];  // [tok_per_cta][n_dims / 2]
    const int half_n = a.n_dims / 2;
    const int64_t t0 = int64_t(blockIdx.x) * a.tok_per_cta;
    const int n_tok = int(min(int64_t(a.tok_per_cta), a.t - t0));
    const int h_all = a.head0[a.n_tensors];
    const int h0 = blockIdx.y * a.heads_per_cta, n_heads = min(a.heads_per_cta, h_all - h0);
    pdl_wait();
    pdl_launch_dependents();
    for (int i = threadIdx.x; i < n_tok * half_n; i += kRopeThreads) {
        const int tok = i / half_n, p = i - tok * half_n;
        const int64_t phase = int64_t(uint64_t(int64_t(a.pos[t0 + tok])) * a.turns[p]);
        float s, c;
        sincospif(__ll2float_rn(phase) * 0x1p-63f, &s, &c);
        cs[i] = make_float2(a.m * c, a.m * s);
    }
    __syncthreads();

    using V = Vec<T, VEC>;
    const int pair_items = HALF ? half_n / VEC : (a.n_dims + VEC - 1) / VEC;
    const int tail0 = HALF ? a.n_dims : pair_items * VEC;  // first element that only tail items cover
    const int tail_items = a.copy_tail ? (a.d - tail0) / VEC : 0;
    const int items = pair_items + tail_items;
    const int per_tok = items * n_heads;
    for (int i = threadIdx.x; i < n_tok * per_tok; i += kRopeThreads) {
        const int tok = i / per_tok, rest = i - tok * per_tok;
        const int hh = rest / items, it = rest - hh * items;
        int ten = 0;
#pragma unroll
        for (int k = 1; k < kRopeMaxTensors; k++)
            if (k < a.n_tensors && h0 + hh >= a.head0[k]) ten = k;
        const int head = h0 + hh - a.head0[ten];
        const T *x = static_cast<const T *>(a.x[ten]) + (t0 + tok) * a.xs_tok[ten] + head * a.xs_head[ten];
        T *y = static_cast<T *>(a.y[ten]) + (t0 + tok) * a.ys_tok[ten] + head * a.ys_head[ten];
        const float2 *c = cs + tok * half_n;
        if (it >= pair_items) {
            const int e = tail0 + (it - pair_items) * VEC;
            *reinterpret_cast<V *>(y + e) = *reinterpret_cast<const V *>(x + e);
        } else if constexpr (HALF) {
            const int e = it * VEC;
            V u = *reinterpret_cast<const V *>(x + e), w = *reinterpret_cast<const V *>(x + half_n + e);
#pragma unroll
            for (int k = 0; k < VEC; k++) {
                const float p = to_f32(u.v[k]), q = to_f32(w.v[k]);
                const float2 r = c[e + k];
                u.v[k] = from_f32<T>(p * r.x - q * r.y);
                w.v[k] = from_f32<T>(p * r.y + q * r.x);
            }
            *reinterpret_cast<V *>(y + e) = u;
            *reinterpret_cast<V *>(y + half_n + e) = w;
        } else {
            const int e = it * VEC;
            V u = *reinterpret_cast<const V *>(x + e);
#pragma unroll
            for (int k = 0; k < VEC; k += 2) {
                if (e + k < a.n_dims) {
                    const float p = to_f32(u.v[k]), q = to_f32(u.v[k + 1]);
                    const float2 r = c[(e + k) >> 1];
                    u.v[k] = from_f32<T>(p * r.x - q * r.y);
                    u.v[k + 1] = from_f32<T>(p * r.y + q * r.x);
                }
            }
            *reinterpret_cast<V *>(y + e) = u;
        }
    }
}

}  // namespace cpq
