// kv_cache.cuh — the paged 8-bit key/value cache: slot maps, append, gather.
//
// The cache is a pool of pages of `block` tokens. A page holds, per kv head,
// block x D codes (int8 or e4m3) and one fp32 scale for K and one for V:
//   codes [n_pages][n_head_kv][block][D], scales [n_pages][n_head_kv]
// and a code c stands for c * scale. A token's slot is page * block + place.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "common.cuh"
#include "rope.cuh"  // to_f32 / from_f32 / Vec

namespace cpq {

// ---- slot maps ---------------------------------------------------------------

constexpr int kSlotThreads = 1024;

struct SlotArgs {
    const int32_t *ctx, *add;  // [n] tokens cached before, tokens added
    int64_t n;
    int32_t *table;            // [n][table_stride]
    int64_t table_stride;
    int max_blocks, block;
    const int32_t *free_pages;
    int64_t n_free;
    const int32_t *taken;      // pages of free_pages in use before the call
    int32_t *taken_out;
    int32_t *seq_start, *kv_len, *pos;
    int64_t *slot;
    int64_t n_rows;
};

// Inclusive sums of two 64-bit values over the CTA (kSlotThreads threads).
__device__ __forceinline__ void slot_scan(int64_t &a, int64_t &b, int64_t (*part)[2]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t ua = __shfl_up_sync(0xffffffffu, a, o), ub = __shfl_up_sync(0xffffffffu, b, o);
        if (lane >= o) a += ua, b += ub;
    }
    if (lane == 31) part[warp][0] = a, part[warp][1] = b;
    __syncthreads();
    if (warp == 0) {
        int64_t x = part[lane][0], y = part[lane][1];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t ux = __shfl_up_sync(0xffffffffu, x, o), uy = __shfl_up_sync(0xffffffffu, y, o);
            if (lane >= o) x += ux, y += uy;
        }
        part[lane][0] = x, part[lane][1] = y;
    }
    __syncthreads();
    if (warp > 0) a += part[warp - 1][0], b += part[warp - 1][1];
}

// Every CTA scans the requests in chunks of kSlotThreads (a few KB from L2:
// cheaper than a second launch that would read the sums) and then writes its
// share of the rows; CTA 0 also writes the per-request outputs, the requests'
// new table entries are shared out over the CTAs. A row takes its page from
// the table where the request held that block before, from the free list
// otherwise, so no CTA reads what another writes. `taken` is read by every CTA
// and written by CTA 0, hence one CTA when taken_out is taken (the host's
// choice).
__global__ void __launch_bounds__(kSlotThreads) kv_slots_kernel(const SlotArgs a) {
    __shared__ int64_t part[32][2];
    __shared__ int s_start[kSlotThreads + 1];  // the chunk's first rows (clipped to n_rows)
    __shared__ int s_ctx[kSlotThreads];        // tokens before, -1: not served
    __shared__ int s_held[kSlotThreads];       // blocks held before
    __shared__ int64_t s_first[kSlotThreads];  // free-list place of the request's first new page
    __shared__ int64_t s_need[kSlotThreads];
    pdl_wait();
    pdl_launch_dependents();
    const int64_t taken = min(max(int64_t(*a.taken), int64_t(0)), a.n_free);
    const int64_t avail = a.n_free - taken;
    const int64_t row_lo = a.n_rows * blockIdx.x / gridDim.x, row_hi = a.n_rows * (blockIdx.x + 1) / gridDim.x;
    int64_t rows = 0, pages = 0, used = 0;  // sums over the chunks before
    for (int64_t c0 = 0; c0 < a.n; c0 += kSlotThreads) {
        const int64_t r = c0 + threadIdx.x;
        const int n_c = int(min(int64_t(kSlotThreads), a.n - c0));
        int64_t ctx = 0, add = 0, held = 0, need = 0;
        bool good = false;
        if (r < a.n) {
            ctx = a.ctx[r];
            add = max(a.add[r], 0);
            held = (ctx + a.block - 1) / a.block;
            const int64_t total = (ctx + add + a.block - 1) / a.block;
            good = ctx >= 0 && a.add[r] >= 0 && total <= a.max_blocks && ctx + add <= 0x7fffffff;
            need = good ? total - held : 0;
        }
        int64_t end = add, through = need;
        slot_scan(end, through, part);
        __syncthreads();  // part is written again below
        const int64_t start = rows + end - add, first = pages + through - need;
        const bool served = good && (need == 0 || first + need <= avail) && start + add <= a.n_rows;
        if (r < a.n) {
            s_start[threadIdx.x] = int(min(start, a.n_rows));
            s_ctx[threadIdx.x] = served ? int(ctx) : -1;
            s_held[threadIdx.x] = int(held);
            s_first[threadIdx.x] = taken + first;
            s_need[threadIdx.x] = served ? need : 0;
            if (blockIdx.x == 0) {
                a.seq_start[r] = int(min(start, a.n_rows));
                a.kv_len[r] = served ? int(ctx + add) : 0;
            }
        }
        // the last thread's sums are the chunk's
        if (threadIdx.x == kSlotThreads - 1) part[0][0] = end, part[0][1] = through;
        // pages given away: they are a prefix of the pages asked for
        int64_t mine = served && need > 0 ? first + need : 0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, o));
        __syncthreads();
        const int64_t c_rows = part[0][0], c_pages = part[0][1];
        __syncthreads();
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5][0] = mine;
        if (threadIdx.x == 0) s_start[n_c] = int(min(rows + c_rows, a.n_rows));
        __syncthreads();
        for (int w = 0; w < 32; w++) used = max(used, part[w][0]);
        rows += c_rows;
        pages += c_pages;
        // new table entries: a warp per request
        for (int i = int(blockIdx.x) * 32 + int(threadIdx.x >> 5); i < n_c; i += 32 * gridDim.x)
            for (int64_t j = threadIdx.x & 31; j < s_need[i]; j += 32)
                a.table[(c0 + i) * a.table_stride + s_held[i] + j] = a.free_pages[s_first[i] + j];
        // this CTA's rows among the chunk's
        const int64_t lo = max(row_lo, int64_t(s_start[0])), hi = min(row_hi, int64_t(s_start[n_c]));
        for (int64_t row = lo + threadIdx.x; row < hi; row += kSlotThreads) {
            int i = 0, top = n_c;  // the last request that starts at or before the row
            while (top - i > 1) {
                const int mid = (i + top) / 2;
                if (s_start[mid] <= row) i = mid;
                else top = mid;
            }
            int pos = 0;
            int64_t slot = -1;
            if (s_ctx[i] >= 0) {
                const int p = s_ctx[i] + int(row - s_start[i]);
                const int b = p / a.block;
                const int64_t page = b < s_held[i] ? a.table[(c0 + i) * a.table_stride + b]
                                                   : a.free_pages[s_first[i] + b - s_held[i]];
                pos = p;
                if (page >= 0) slot = page * a.block + (p - b * a.block);
            }
            a.pos[row] = pos;
            a.slot[row] = slot;
        }
        __syncthreads();
    }
    for (int64_t row = max(row_lo, min(rows, a.n_rows)) + threadIdx.x; row < row_hi; row += kSlotThreads) {
        a.pos[row] = 0;
        a.slot[row] = -1;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        a.seq_start[a.n] = int(min(rows, a.n_rows));
        *a.taken_out = int(taken + used);
    }
}

// ---- codes ----------------------------------------------------------------------

// The largest code, and scales below this are taken as zero (a block of
// values under about 1e-28 in magnitude: their quotients would underflow).
template <int FMT> __host__ __device__ constexpr float kv_top() { return FMT == CPQ_KV_INT8 ? 127.0f : 448.0f; }
constexpr float kKvMinScale = 0x1p-100f;

__device__ __forceinline__ float kv_finite_abs(float x) {
    const float m = fabsf(x);
    return m <= 3.402823466e38f ? m : 0.0f;  // infinities and NaN do not set a scale
}

// fp32 -> e4m3, nearest, ties to even, saturating.
__device__ __forceinline__ uint32_t e4m3_of(float x) {
    return uint32_t(__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3));
}
__device__ __forceinline__ float e4m3_to_f32(uint32_t c) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(c & 0xffu), __NV_E4M3)));
}

// The code nearest to the real quotient x / s, ties to even (not nearest to an
// fp32 quotient: a rounding before the rounding moves values at the borders).
//   int8: the fp32 estimate is off by one step at most; x - q s is exact in one
//         FMA for a q this near, so comparing it with s / 2 settles it.
//   e4m3: the fp32 quotient made odd-rounded (truncated, last bit set when
//         inexact) keeps on which side of a border the real one lies.
// NaN is stored as 0; infinities saturate.
template <int FMT>
__device__ __forceinline__ uint32_t kv_code(float x, float s, float inv) {
    if (!(x == x) || s == 0.0f) return 0u;
    if constexpr (FMT == CPQ_KV_INT8) {
        float q = rintf(fminf(fmaxf(x * inv, -127.0f), 127.0f));
        const float r = __fmaf_rn(-q, s, x), h = 0.5f * s;
        const bool odd = (int(q) & 1) != 0;
        if (r > h || (r == h && odd)) q += 1.0f;
        else if (r < -h || (r == -h && odd)) q -= 1.0f;
        return uint32_t(int(fminf(fmaxf(q, -127.0f), 127.0f))) & 0xffu;
    } else {
        float t = __fdiv_rn(x, s);
        if (fabsf(t) < 1024.0f) {
            const float r = __fmaf_rn(-t, s, x);
            if (r != 0.0f) {
                int b = __float_as_int(t);
                if ((r < 0.0f) != (x < 0.0f)) b -= 1;  // the quotient was rounded away from zero
                t = __int_as_float(b | 1);
            }
        }
        return e4m3_of(t);
    }
}

// The code of the real number c * s0 / s for a code c that was made at scale s0 <= s.
template <int FMT>
__device__ __forceinline__ uint32_t kv_recode(uint32_t c, float s0, float s) {
    if constexpr (FMT == CPQ_KV_INT8) {
        // c * s0 and q * s are exact in 64 bits (8 + 24), so their difference is too
        const double v = double(int(int8_t(c))) * double(s0), d = double(s), h = 0.5 * d;
        double q = rint(v / d);
        const double r = v - q * d;
        const bool odd = (int(q) & 1) != 0;
        if (r > h || (r == h && odd)) q += 1.0;
        else if (r < -h || (r == -h && odd)) q -= 1.0;
        return uint32_t(int(q)) & 0xffu;
    } else {
        const double v = double(e4m3_to_f32(c)) * double(s0);
        const double t = v / double(s);
        float f = __double2float_rz(t);
        if (double(f) != t) f = __int_as_float(__float_as_int(f) | 1);  // odd: on its side of every border
        return e4m3_of(f);
    }
}

template <int FMT>
__device__ __forceinline__ float kv_value(uint32_t c) {
    if constexpr (FMT == CPQ_KV_INT8) return float(int(int8_t(c)));
    else return e4m3_to_f32(c);
}

// ---- append ---------------------------------------------------------------------

constexpr int kAppendThreads = 256;

struct AppendArgs {
    const void *x[2];          // k, v
    int64_t xs_tok[2], xs_head[2];
    uint8_t *codes[2];
    float *scale[2];
    const int64_t *slot;
    int64_t t, n_slots;
    int n_head, d, block;
    int group;                 // rows whose runs one CTA looks after
};

// grid (row groups, kv heads, K or V). A run is a maximal stretch of rows with
// consecutive slots of one page; the CTA of its first row's group writes it,
// so a page's scale has one writer. Per run: the new rows' largest magnitude,
// the page's scale (kept, or raised when the new rows need it; a run at the
// page's start begins a new page), the rows held before coded again if the
// scale rose, the new rows' codes.
template <typename T, int VEC, int FMT>
__global__ void __launch_bounds__(kAppendThreads) kv_append_kernel(const AppendArgs a) {
    __shared__ float s_max[kAppendThreads / 32];
    __shared__ int s_len;
    const int h = blockIdx.y, z = blockIdx.z;
    const T *x = static_cast<const T *>(a.x[z]) + h * a.xs_head[z];
    const int64_t xs = a.xs_tok[z];
    const int d = a.d, per_row = d / VEC;
    pdl_wait();
    pdl_launch_dependents();
    const int64_t t_end = min(int64_t(blockIdx.x + 1) * a.group, a.t);
    for (int64_t t = int64_t(blockIdx.x) * a.group; t < t_end; t++) {
        const int64_t slot = a.slot[t];
        if (slot < 0 || slot >= a.n_slots) continue;
        const int64_t page = slot / a.block;
        const int off = int(slot - page * a.block);
        if (off != 0 && t > 0 && a.slot[t - 1] == slot - 1) continue;  // inside another row's run
        // the run's length: rows t + i with slot + i, up to the page's end
        __syncthreads();
        if (threadIdx.x == 0) s_len = a.block - off;
        __syncthreads();
        if (int(threadIdx.x) < a.block - off && (t + threadIdx.x >= a.t || a.slot[t + threadIdx.x] != slot + threadIdx.x))
            atomicMin(&s_len, int(threadIdx.x));
        __syncthreads();
        const int len = s_len;
        float m = 0.0f;
        for (int i = threadIdx.x; i < len * per_row; i += kAppendThreads) {
            const int r = i / per_row, e = (i - r * per_row) * VEC;
            const Vec<T, VEC> v = *reinterpret_cast<const Vec<T, VEC> *>(x + (t + r) * xs + e);
#pragma unroll
            for (int k = 0; k < VEC; k++) m = fmaxf(m, kv_finite_abs(to_f32(v.v[k])));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = m;
        __syncthreads();
        m = s_max[0];
#pragma unroll
        for (int w = 1; w < kAppendThreads / 32; w++) m = fmaxf(m, s_max[w]);
        float s = __fdiv_rn(m, kv_top<FMT>());
        if (s < kKvMinScale) s = 0.0f;
        float *const scale = a.scale[z] + page * a.n_head + h;
        uint8_t *const codes = a.codes[z] + (page * a.n_head + h) * int64_t(a.block) * d;
        const float s0 = off ? *scale : 0.0f;
        __syncthreads();  // every thread has read the scale
        if (off) {
            s = fmaxf(s, s0);
            if (s != s0)
                for (int i = threadIdx.x; i < off * d / 4; i += kAppendThreads) {
                    const uint32_t w = reinterpret_cast<const uint32_t *>(codes)[i];
                    uint32_t u = 0;
#pragma unroll
                    for (int k = 0; k < 4; k++) u |= kv_recode<FMT>((w >> (8 * k)) & 0xffu, s0, s) << (8 * k);
                    reinterpret_cast<uint32_t *>(codes)[i] = u;
                }
        }
        if (threadIdx.x == 0) *scale = s;
        const float inv = s > 0.0f ? __fdiv_rn(1.0f, s) : 0.0f;
        uint8_t *const to = codes + int64_t(off) * d;
        for (int i = threadIdx.x; i < len * per_row; i += kAppendThreads) {
            const int r = i / per_row, e = (i - r * per_row) * VEC;
            const Vec<T, VEC> v = *reinterpret_cast<const Vec<T, VEC> *>(x + (t + r) * xs + e);
            Vec<uint8_t, VEC> c;
#pragma unroll
            for (int k = 0; k < VEC; k++) c.v[k] = uint8_t(kv_code<FMT>(to_f32(v.v[k]), s, inv));
            if constexpr (VEC == 1) to[int64_t(r) * d + e] = c.v[0];
            else if constexpr (VEC == 4) *reinterpret_cast<uint32_t *>(to + int64_t(r) * d + e) =
                uint32_t(c.v[0]) | uint32_t(c.v[1]) << 8 | uint32_t(c.v[2]) << 16 | uint32_t(c.v[3]) << 24;
            else *reinterpret_cast<uint2 *>(to + int64_t(r) * d + e) =
                make_uint2(uint32_t(c.v[0]) | uint32_t(c.v[1]) << 8 | uint32_t(c.v[2]) << 16 | uint32_t(c.v[3]) << 24,
                           uint32_t(c.v[4]) | uint32_t(c.v[5]) << 8 | uint32_t(c.v[6]) << 16 | uint32_t(c.v[7]) << 24);
        }
    }
}

// ---- gather ---------------------------------------------------------------------

constexpr int kGatherThreads = 256;

struct GatherArgs {
    const uint8_t *codes[2];
    const float *scale[2];
    const int64_t *slot;
    void *y[2];
    int64_t ys_tok[2], ys_head[2];
    int64_t t, n_slots;
    int n_head, d, block;
};

// grid (items / threads, K or V): a thread turns 16 codes of a row's head into
// values; rows without a slot become zeros.
template <typename T, bool WIDE, int FMT>
__global__ void __launch_bounds__(kGatherThreads) kv_gather_kernel(const GatherArgs a) {
    const int z = blockIdx.y, per_head = a.d / 16, per_row = per_head * a.n_head;
    pdl_wait();
    pdl_launch_dependents();
    for (int64_t i = int64_t(blockIdx.x) * kGatherThreads + threadIdx.x; i < a.t * per_row;
         i += int64_t(gridDim.x) * kGatherThreads) {
        const int64_t row = i / per_row;
        const int rest = int(i - row * per_row), h = rest / per_head, e = (rest - h * per_head) * 16;
        const int64_t slot = a.slot[row];
        float v[16] = {};
        if (slot >= 0 && slot < a.n_slots) {
            const int64_t page = slot / a.block;
            const int64_t at = (page * a.n_head + h) * a.block + (slot - page * a.block);
            const uint4 c = *reinterpret_cast<const uint4 *>(a.codes[z] + at * a.d + e);
            const float s = a.scale[z][page * a.n_head + h];
            const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
            for (int k = 0; k < 16; k++) v[k] = kv_value<FMT>((w[k >> 2] >> (8 * (k & 3))) & 0xffu) * s;
        }
        T *y = static_cast<T *>(a.y[z]) + row * a.ys_tok[z] + h * a.ys_head[z] + e;
        constexpr int W = WIDE ? 16 / int(sizeof(T)) : 1;
#pragma unroll
        for (int k = 0; k < 16; k += W) {
            Vec<T, W> o;
#pragma unroll
            for (int j = 0; j < W; j++) o.v[j] = from_f32<T>(v[k + j]);
            *reinterpret_cast<Vec<T, W> *>(y + k) = o;
        }
    }
}

}  // namespace cpq
