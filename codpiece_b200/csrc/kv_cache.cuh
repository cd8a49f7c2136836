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
#include "rope.cuh"  // to_f32, from_f32, FastDiv

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
// choice). Latency: 16 decode requests 5.2 us, 300 requests with 60000 rows 6.4 (72 with one CTA).
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

// The larger of m and the values' magnitudes. An infinity makes it infinite; a
// NaN does not show (the codes' own check finds it).
template <typename T, int VEC, bool WIDE>
__device__ __forceinline__ float kv_top_of(float m, const Vec<T, VEC, WIDE> &u) {
    float f[VEC];
    u.get(f);
#pragma unroll
    for (int k = 0; k < VEC; k++) m = fmaxf(m, fabsf(f[k]));
    return m;
}
// The same over the finite values only.
template <typename T, int VEC, bool WIDE>
__device__ __forceinline__ float kv_top_finite(float m, const Vec<T, VEC, WIDE> &u) {
    float f[VEC];
    u.get(f);
#pragma unroll
    for (int k = 0; k < VEC; k++) m = fabsf(f[k]) < __int_as_float(0x7f800000) ? fmaxf(m, fabsf(f[k])) : m;
    return m;
}

// fp32 -> e4m3, nearest, ties to even, saturating.
__device__ __forceinline__ uint32_t e4m3_of(float x) {
    return uint32_t(__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3));
}
__device__ __forceinline__ float e4m3_to_f32(uint32_t c) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(c & 0xffu), __NV_E4M3)));
}

__device__ __forceinline__ __half2 u32_half2(uint32_t u) { return *reinterpret_cast<const __half2 *>(&u); }
__device__ __forceinline__ uint32_t half2_u32(__half2 h) { return *reinterpret_cast<const uint32_t *>(&h); }

// Codes (bytes 0, 1) and (bytes 2, 3) of w as fp16 pairs, exact. int8: 0x6400 |
// (code + 128) is the fp16 number 1152 + code.
template <int FMT>
__device__ __forceinline__ void codes_h2(uint32_t w, uint32_t &lo, uint32_t &hi) {
    if constexpr (FMT == CPQ_KV_INT8) {
        w ^= 0x80808080u;
        const __half2 k1152 = __float2half2_rn(1152.0f);
        lo = half2_u32(__hsub2(u32_half2(__byte_perm(w, 0x64646464u, 0x4140)), k1152));
        hi = half2_u32(__hsub2(u32_half2(__byte_perm(w, 0x64646464u, 0x4342)), k1152));
    } else {
        asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
            "cvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
            : "=r"(lo), "=r"(hi)
            : "r"(w));
    }
}

// The code nearest to the real quotient x / s, ties to even (not nearest to an
// fp32 quotient: a rounding before the rounding moves values at the borders),
// inv = 1 / s rounded.
//   int8: the fp32 estimate is off by one step at most; x - q s is exact in one
//         FMA for a q this near, so comparing it with s / 2 settles it.
//   e4m3: t + (x - t s) inv is within one ulp of the quotient, and its residue
//         (exact in one FMA) says on which side; made odd on that side
//         (truncated, last bit set), it stands where the quotient stands with
//         respect to every border, whose last bit is 0.
// NaN is stored as 0; infinities saturate.
template <int FMT>
__device__ __forceinline__ float kv_quotient(float x, float s, float inv) {
    if constexpr (FMT == CPQ_KV_INT8) {
        float q = rintf(fminf(fmaxf(x * inv, -127.0f), 127.0f));
        const float r = __fmaf_rn(-q, s, x), h = 0.5f * s;
        const bool odd = (int(q) & 1) != 0;
        if (r > h || (r == h && odd)) q += 1.0f;
        else if (r < -h || (r == -h && odd)) q -= 1.0f;
        return fminf(fmaxf(q, -127.0f), 127.0f);
    } else {
        float t = x * inv;
        if (fabsf(t) < 1024.0f) {
            t = __fmaf_rn(__fmaf_rn(-t, s, x), inv, t);
            const float r = __fmaf_rn(-t, s, x);
            if (r != 0.0f) t = __int_as_float((__float_as_int(t) - ((r < 0.0f) != (x < 0.0f) ? 1 : 0)) | 1);
        }
        return t;
    }
}

template <int FMT>
__device__ __forceinline__ uint32_t kv_pack4(const float (&q)[4]) {
    if constexpr (FMT == CPQ_KV_INT8) {
        uint32_t w = 0;
#pragma unroll
        for (int k = 0; k < 4; k++) w |= (uint32_t(int(q[k])) & 0xffu) << (8 * k);
        return w;
    } else {
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(q[0], q[1]), __NV_SATFINITE, __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(q[2], q[3]), __NV_SATFINITE, __NV_E4M3);
        return lo | hi << 16;
    }
}

// Four codes as a word, the exact way.
template <int FMT>
__device__ __forceinline__ uint32_t kv_codes4_exact(const float (&x)[4], float s, float inv) {
    float q[4];
#pragma unroll
    for (int k = 0; k < 4; k++) q[k] = x[k] == x[k] && s > 0.0f ? kv_quotient<FMT>(x[k], s, inv) : 0.0f;
    return kv_pack4<FMT>(q);
}

// Four codes as a word, from the fp32 product t = x * inv, which is within 2
// ulp of the quotient and gives the same code away from the borders between
// codes, and on them when it is the quotient itself (x - t s = 0: frequent with
// 16-bit x, whose quotients have few bits). `sure` is cleared for the others: a
// value within 4 ulp (e4m3; borders and codes have 19 zero bits at the end) or
// 2^-15 (int8) of a border, a few groups in 10^4, or a NaN or an infinity.
template <int FMT>
__device__ __forceinline__ uint32_t kv_codes4(const float (&x)[4], float s, float inv, bool &sure) {
    if constexpr (FMT == CPQ_KV_INT8) {
        constexpr float kRound = 12582912.0f;  // 1.5 * 2^23: the low byte of t + kRound is t to nearest
        uint32_t b[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float t = x[k] * inv, u = t + kRound;
            sure &= fabsf(t - (u - kRound)) <= 0.5f - 0x1p-15f || __fmaf_rn(-t, s, x[k]) == 0.0f;
            b[k] = __float_as_uint(u);
        }
        return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    } else {
        float q[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            q[k] = x[k] * inv;
            sure &= __float_as_uint(q[k]) * 8192u + 4u * 8192u > 8u * 8192u || __fmaf_rn(-q[k], s, x[k]) == 0.0f;
        }
        return kv_pack4<FMT>(q);
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

// ---- append ---------------------------------------------------------------------

constexpr int kAppendThreads = 256;  // at most

struct AppendArgs {
    const void *x[2];          // k, v
    int64_t xs_tok[2], xs_head[2];
    uint8_t *codes[2];
    float *scale[2];
    const int64_t *slot;
    int64_t t, n_slots;
    int n_head, d, log_block;
    int group;                 // rows whose runs one CTA looks after
};

// grid (row groups, kv heads, K or V). A run is a maximal stretch of rows with
// consecutive slots of one page; the CTA of its first row's group writes it,
// so a page's scale has one writer. Per run: its rows into shared memory (one
// bulk copy per row, so an SM has all its CTAs' runs in flight; rows that are
// not 16-byte aligned by plain loads), the largest magnitude, the page's scale
// (kept, or raised when the new rows need it; a run at the page's start begins
// a new page), the rows held before coded again if the scale rose, the new
// rows' codes. Holding the rows in registers between the two passes instead
// spilled and left an SM too few runs in flight (14080 rows x 8 heads of 128,
// bf16, pages of 32: 42 us). That case takes 34 us now (2.5 TB/s), with fp32 rows
// 36 (4.0 TB/s, 0.6 of a measured copy): what a CTA does before its copies and the
// two passes over a run in shared memory bound it (68 % of issue slots), not its
// bytes. 64 threads per 8 KB: with twice as many 39 us, with half 36 (fp32 57, 34).
// 40 registers instead of 48 (a few spilled outside the loops): 3 to 9 % less.
// These are calls in which no scale grows; where one does, the page's rows are
// coded again, a 64-bit division per code (24 rows, fp32 to int8, pages of 64: 3.1
// us, 24 with an eighth of the pages growing, 31 with all of them).
constexpr int kAppendMaxGroup = 32;

template <typename T, bool WIDE, int FMT>
__global__ void __launch_bounds__(kAppendThreads, 6) kv_append_kernel(const __grid_constant__ AppendArgs a) {
    extern __shared__ __align__(128) uint8_t s_rows[];
    __shared__ float s_max[2][kAppendThreads / 32];
    __shared__ int64_t s_slot[1 + kAppendMaxGroup + 128];  // of the row before the group, the group, a page's rows behind it
    __shared__ uint64_t s_bar;
    constexpr int VEC = 16 / int(sizeof(T));
    using V = Vec<T, VEC, true>;
    T *const rows = reinterpret_cast<T *>(s_rows);
    const int h = blockIdx.y, z = blockIdx.z, lane = threadIdx.x & 31, nt = blockDim.x;
    const T *x = static_cast<const T *>(a.x[z]) + h * a.xs_head[z];
    const int d = a.d, block = 1 << a.log_block;
    if (threadIdx.x == 0) {
        mbar_init(&s_bar, 1);
        fence_mbar_init();
    }
    pdl_wait();
    pdl_launch_dependents();
    const int64_t t0 = int64_t(blockIdx.x) * a.group;
    for (int i = threadIdx.x; i < 1 + a.group + block; i += nt) {
        const int64_t r = t0 - 1 + i;
        const int64_t slot = r >= 0 && r < a.t ? a.slot[r] : -1;
        s_slot[i] = slot >= 0 && slot < a.n_slots ? slot : -1;
    }
    __syncthreads();
    // the group's rows that begin a run
    const int64_t here = lane < a.group ? s_slot[1 + lane] : -1;
    const bool first = here >= 0 && ((here & (block - 1)) == 0 || s_slot[lane] != here - 1);
    int odd = 0;          // s_max is used in turns
    uint32_t parity = 0;  // of s_bar, once per run
    for (unsigned todo = __ballot_sync(0xffffffffu, first); todo; todo &= todo - 1) {
        const int at = __ffs(int(todo)) - 1;
        const int64_t t = t0 + at, slot = s_slot[1 + at], page = slot >> a.log_block;
        const int off = int(slot & (block - 1));
        float *const scale = a.scale[z] + page * a.n_head + h;
        uint8_t *const codes = a.codes[z] + (page * a.n_head + h) * int64_t(block) * d;
        // the run's length: rows t + i with slot + i, up to the page's end
        int len = 0;
        for (int i = 0; i < block; i += 32) {
            const unsigned in = __ballot_sync(0xffffffffu, i + lane < block - off && s_slot[1 + at + i + lane] == slot + i + lane);
            len += in == ~0u ? 32 : __ffs(int(~in)) - 1;
            if (in != ~0u) break;
        }
        const T *const xp = x + t * a.xs_tok[z];
        if constexpr (WIDE) {
            const uint32_t bytes = uint32_t(d) * uint32_t(sizeof(T));
            if (threadIdx.x == 0) mbar_arrive_expect_tx(&s_bar, bytes * uint32_t(len));
            for (int r = threadIdx.x; r < len; r += nt) bulk_g2s(rows + r * d, xp + int64_t(r) * a.xs_tok[z], bytes, &s_bar);
        } else {
            for (int i = threadIdx.x; i < len * d; i += nt) rows[i] = xp[int64_t(i / d) * a.xs_tok[z] + i % d];
        }
        const float s0 = off ? *scale : 0.0f;
        if constexpr (WIDE) {
            if (!mbar_wait_bounded(&s_bar, parity)) {  // (reported in the device's error word)
                mbar_wait_bounded(&s_bar, parity);     // no copy may land after the CTA has left
                return;
            }
            parity ^= 1u;
        } else __syncthreads();
        const int n = len * d / VEC;
        const uint4 *const items = reinterpret_cast<const uint4 *>(s_rows);
        // a reduction over the run
        auto largest = [&](auto f) {
            float m = 0.0f;
#pragma unroll 4
            for (int i = threadIdx.x; i < n; i += nt) m = f(m, V{items[i]});
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            if (lane == 0) s_max[odd][threadIdx.x >> 5] = m;
            __syncthreads();
            for (int w = 0; w < nt / 32; w++) m = fmaxf(m, s_max[odd][w]);
            odd ^= 1;
            return m;
        };
        float top = largest([](float m, const V &u) { return kv_top_of(m, u); });
        if (top == __int_as_float(0x7f800000))  // infinities do not set a scale
            top = largest([](float m, const V &u) { return kv_top_finite(m, u); });
        float s = __fdiv_rn(top, kv_top<FMT>());
        if (s < kKvMinScale) s = 0.0f;
        s = fmaxf(s, s0);  // (every thread read the page's scale before the barrier above)
        if (off && s != s0)
            for (int i = threadIdx.x; i < off * d / 4; i += nt) {
                const uint32_t w = reinterpret_cast<const uint32_t *>(codes)[i];
                uint32_t u = 0;
#pragma unroll 1
                for (int k = 0; k < 4; k++) u |= kv_recode<FMT>((w >> (8 * k)) & 0xffu, s0, s) << (8 * k);
                reinterpret_cast<uint32_t *>(codes)[i] = u;
            }
        if (threadIdx.x == 0) *scale = s;
        const float inv = s > 0.0f ? __fdiv_rn(1.0f, s) : 0.0f;
        uint8_t *const to = codes + int64_t(off) * d;  // rows of codes are dense
        auto put = [&](int i, const uint32_t (&w)[VEC / 4]) {
            if constexpr (VEC == 4) *reinterpret_cast<uint32_t *>(to + i * 4) = w[0];
            else *reinterpret_cast<uint2 *>(to + i * 8) = make_uint2(w[0], w[1]);
        };
        auto redo = [&](int i) {
            float f[VEC];
            uint32_t w[VEC / 4];
            V{items[i]}.get(f);
#pragma unroll
            for (int j = 0; j < VEC; j += 4) {
                const float g[4] = {f[j], f[j + 1], f[j + 2], f[j + 3]};
                w[j / 4] = kv_codes4_exact<FMT>(g, s, inv);
            }
            put(i, w);
        };
        for (int i0 = threadIdx.x; i0 < n; i0 += 4 * nt) {
            uint32_t unsure = 0;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int i = i0 + k * nt;
                if (i >= n) break;
                bool sure = s > 0.0f;
                float f[VEC];
                uint32_t w[VEC / 4];
                V{items[i]}.get(f);
#pragma unroll
                for (int j = 0; j < VEC; j += 4) {
                    const float g[4] = {f[j], f[j + 1], f[j + 2], f[j + 3]};
                    w[j / 4] = kv_codes4<FMT>(g, s, inv, sure);
                }
                put(i, w);
                unsure |= sure ? 0u : 1u << k;
            }
            for (; unsure; unsure &= unsure - 1) redo(i0 + (__ffs(int(unsure)) - 1) * nt);  // rare
        }
        __syncthreads();  // the next run's rows take these rows' place
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
    int n_head, d, log_block;
    FastDiv by_row;            // items of a row
};

// grid (row groups, K or V): a thread turns VEC codes of a row's head into 16
// bytes of values (one by one where the outputs are not aligned), lanes side
// by side in both, and keeps its place in the row while it steps over rows;
// rows without a slot become zeros. Bounded by the stores: 14080 rows x 8 heads
// of 128 to fp32 25 us (5.8 TB/s, 0.89 of a measured copy), to bf16 17 (5.1).
constexpr int kGatherRows = 8;

template <typename T, bool WIDE, int FMT>
__global__ void __launch_bounds__(kGatherThreads) kv_gather_kernel(const __grid_constant__ GatherArgs a) {
    constexpr int VEC = 16 / int(sizeof(T)), kBatch = 4;  // items of a thread in flight
    using V = Vec<T, VEC, WIDE>;
    __shared__ longlong2 s_at[kGatherRows];  // the row's place among codes (head 0) and scales, or -1
    const int z = blockIdx.y, lg = (a.d == 256 ? 8 : 7) - (VEC == 8 ? 3 : 2);  // log2 of a head row's items
    const int per_row = a.n_head << lg;
    pdl_wait();
    pdl_launch_dependents();
    const int64_t row0 = int64_t(blockIdx.x) * kGatherRows;
    const int n_rows = int(min(int64_t(kGatherRows), a.t - row0));
    if (int(threadIdx.x) < n_rows) {
        const int64_t slot = a.slot[row0 + threadIdx.x], page = slot >> a.log_block;
        const int64_t place = slot & ((1 << a.log_block) - 1);
        s_at[threadIdx.x] = slot >= 0 && slot < a.n_slots
                                ? make_longlong2(((page * a.n_head << a.log_block) + place) * a.d, page * a.n_head)
                                : make_longlong2(-1, -1);
    }
    __syncthreads();
    const int sub = int(a.by_row.div(threadIdx.x)), step = max(1, kGatherThreads / per_row);
    if (sub >= step) return;
    for (int col = int(threadIdx.x) - sub * per_row; col < per_row; col += kGatherThreads) {
        const int h = col >> lg, e = (col & ((1 << lg) - 1)) * VEC;
        const uint8_t *const codes = a.codes[z] + (int64_t(h) << a.log_block) * a.d + e;
        const float *const scale = a.scale[z] + h;
        T *const y = static_cast<T *>(a.y[z]) + row0 * a.ys_tok[z] + h * a.ys_head[z] + e;
        for (int r0 = sub; r0 < n_rows; r0 += kBatch * step) {
            uint32_t w[kBatch][VEC / 4];
            float s[kBatch];
#pragma unroll
            for (int b = 0; b < kBatch; b++) {
                const int r = r0 + b * step;
                if (r >= n_rows) break;
                const longlong2 at = s_at[r];
#pragma unroll
                for (int j = 0; j < VEC / 4; j++) w[b][j] = 0;  // code 0 is zero in both formats
                s[b] = 0.0f;
                if (at.x >= 0) {
                    s[b] = scale[at.y];
                    if constexpr (VEC == 4) w[b][0] = *reinterpret_cast<const uint32_t *>(codes + at.x);
                    else {
                        const uint2 u = *reinterpret_cast<const uint2 *>(codes + at.x);
                        w[b][0] = u.x, w[b][1] = u.y;
                    }
                }
            }
#pragma unroll
            for (int b = 0; b < kBatch; b++) {
                const int r = r0 + b * step;
                if (r >= n_rows) break;
                float o[VEC];
#pragma unroll
                for (int j = 0; j < VEC / 4; j++) {
                    uint32_t lo, hi;
                    codes_h2<FMT>(w[b][j], lo, hi);
                    const float2 f = __half22float2(u32_half2(lo)), g = __half22float2(u32_half2(hi));
                    o[4 * j] = f.x * s[b], o[4 * j + 1] = f.y * s[b], o[4 * j + 2] = g.x * s[b], o[4 * j + 3] = g.y * s[b];
                }
                V u;
                u.set(o);
                u.store(y + r * a.ys_tok[z]);
            }
        }
    }
}

}  // namespace cpq
