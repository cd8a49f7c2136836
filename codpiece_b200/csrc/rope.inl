// rope.inl — cpq_rope_*: frequencies and host side of rope.cuh.
//
// The scaling rules and their parameters are ggml's (ggml_rope_ext: n_dims,
// mode, n_ctx_orig, freq_base, freq_scale, ext_factor, attn_factor, beta_fast,
// beta_slow, frequency factors), so a model's hyper-parameters carry over.

#include <cmath>

struct cpq_rope {
    int n_dims, mode;
    float m;
    uint64_t turns[cpq::kRopeMaxPairs];
};

namespace cpq {

// w (radians per position) as a 64-bit fraction of a turn. Whole turns per
// position drop out, positions being integers.
static uint64_t turns_fixed(long double w) {
    long double t = w / (2.0L * 3.14159265358979323846264338327950288L);
    t -= floorl(t);
    const long double f = t * 18446744073709551616.0L;  // 2^64
    return f >= 18446744073709551615.0L ? 0 : uint64_t(llrintl(f * 0.5L)) * 2u;
}

// Bytes of one element of an activation type, 0 for others.
static int act_bytes(int32_t t) {
    return t == CPQ_TYPE_F32 ? 4 : t == CPQ_TYPE_F16 || t == CPQ_TYPE_BF16 ? 2 : 0;
}

// ne = [D, heads, tokens, 1] with contiguous heads' rows and whole-element strides.
static bool head_rows(const cpq_tensor *t) {
    const int b = t ? act_bytes(t->type) : 0;
    return b && t->nb[0] == size_t(b) && t->nb[1] % size_t(b) == 0 && t->nb[2] % size_t(b) == 0 && t->ne[0] > 0 &&
           t->ne[1] > 0 && t->ne[2] >= 0 && t->ne[3] == 1 && (t->data || t->ne[2] == 0);
}

template <typename T, int VEC>
static cudaError_t launch_rope_v(const RopeArgs &a, bool half, dim3 grid, cudaStream_t st) {
    return half ? launch(rope_kernel<T, VEC, true>, grid, dim3(kRopeThreads), 0, st, a)
                : launch(rope_kernel<T, VEC < 2 ? 2 : VEC, false>, grid, dim3(kRopeThreads), 0, st, a);
}

template <typename T>
static cudaError_t launch_rope(const RopeArgs &a, bool half, bool wide, dim3 grid, cudaStream_t st) {
    return wide ? launch_rope_v<T, 16 / sizeof(T)>(a, half, grid, st) : launch_rope_v<T, 1>(a, half, grid, st);
}

}  // namespace cpq

extern "C" cpq_status cpq_rope_create(const cpq_rope_params *p, cpq_rope **rope) {
    using namespace cpq;
    if (!p || !rope) return fail(CPQ_ERR_INVALID_ARG, "rope: null argument");
    *rope = nullptr;
    if (p->n_dims < 2 || p->n_dims % 2) return fail(CPQ_ERR_INVALID_ARG, "rope: n_dims=%d is not a positive even number", p->n_dims);
    if (p->n_dims > 2 * kRopeMaxPairs) return fail(CPQ_ERR_UNSUPPORTED, "rope: n_dims=%d > %d", p->n_dims, 2 * kRopeMaxPairs);
    if (p->mode != CPQ_ROPE_INTERLEAVED && p->mode != CPQ_ROPE_HALF) return fail(CPQ_ERR_INVALID_ARG, "rope: mode %d", p->mode);
    if (!(p->base > 0) || !std::isfinite(p->base) || !(p->freq_scale > 0) || !std::isfinite(p->freq_scale) ||
        !std::isfinite(p->ext_factor) || !std::isfinite(p->attn_factor))
        return fail(CPQ_ERR_INVALID_ARG, "rope: base=%g freq_scale=%g ext_factor=%g attn_factor=%g", p->base, p->freq_scale,
                    p->ext_factor, p->attn_factor);
    const bool yarn = p->ext_factor != 0;
    if (yarn && (!(p->base > 1) || p->n_ctx_orig < 1 || !(p->beta_fast > 0) || !(p->beta_slow > 0)))
        return fail(CPQ_ERR_INVALID_ARG, "rope: YaRN needs base > 1, n_ctx_orig >= 1 and positive betas");
    std::unique_ptr<cpq_rope> r(new (std::nothrow) cpq_rope);
    if (!r) return fail(CPQ_ERR_INVALID_ARG, "rope: out of host memory");
    r->n_dims = p->n_dims;
    r->mode = p->mode;
    // the pair whose wavelength turns `beta` times within the original context
    auto pair_of = [&](double beta) {
        return p->n_dims * std::log(p->n_ctx_orig / (beta * 2.0 * M_PI)) / (2.0 * std::log(p->base));
    };
    const double low = yarn ? std::max(0.0, std::floor(pair_of(p->beta_fast))) : 0;
    const double high = yarn ? std::min(p->n_dims - 1.0, std::ceil(pair_of(p->beta_slow))) : 0;
    for (int i = 0; i < p->n_dims / 2; i++) {
        long double w = powl((long double)p->base, -2.0L * i / p->n_dims);
        if (p->freq_factors) {
            if (!(p->freq_factors[i] > 0) || !std::isfinite(p->freq_factors[i]))
                return fail(CPQ_ERR_INVALID_ARG, "rope: frequency factor %d is %g", i, p->freq_factors[i]);
            w /= p->freq_factors[i];
        }
        const long double mix =
            yarn ? p->ext_factor * (1.0 - std::min(1.0, std::max(0.0, (i - low) / std::max(0.001, high - low)))) : 0.0;
        r->turns[i] = turns_fixed(w * p->freq_scale * (1.0L - mix) + w * mix);
    }
    r->m = float(p->attn_factor * (yarn ? 1.0 + 0.1 * std::log(1.0 / p->freq_scale) : 1.0));
    *rope = r.release();
    return CPQ_SUCCESS;
}

extern "C" void cpq_rope_destroy(cpq_rope *rope) { delete rope; }

extern "C" cpq_status cpq_rope_apply(const cpq_rope *rope, const cpq_tensor *const *x, cpq_tensor *const *y, int n,
                                     const int32_t *pos, void *stream) {
    using namespace cpq;
    if (!rope || !x || !y) return fail(CPQ_ERR_INVALID_ARG, "rope: null argument");
    if (n < 1 || n > kRopeMaxTensors) return fail(CPQ_ERR_INVALID_ARG, "rope: n=%d tensors (1 to %d)", n, kRopeMaxTensors);
    RopeArgs a{};
    bool copy = false, wide = true;
    for (int i = 0; i < n; i++) {
        if (!head_rows(x[i]) || !head_rows(y[i]))
            return fail(CPQ_ERR_INVALID_ARG, "rope: tensor %d must be F32, F16 or BF16 with ne=[D, heads, tokens, 1] and contiguous rows", i);
        for (int d = 0; d < 3; d++)
            if (x[i]->ne[d] != y[i]->ne[d] || (d != 1 && x[i]->ne[d] != x[0]->ne[d]))
                return fail(CPQ_ERR_INVALID_ARG, "rope: tensor %d differs in shape", i);
        if (x[i]->type != x[0]->type || y[i]->type != x[0]->type)
            return fail(CPQ_ERR_INVALID_ARG, "rope: tensors of different types");
        const size_t b = size_t(act_bytes(x[i]->type));
        const bool same = x[i]->data == y[i]->data;
        if (same && (x[i]->nb[1] != y[i]->nb[1] || x[i]->nb[2] != y[i]->nb[2]))
            return fail(CPQ_ERR_INVALID_ARG, "rope: tensor %d is rotated in place with other strides", i);
        copy |= !same;
        for (const cpq_tensor *t : {x[i], static_cast<const cpq_tensor *>(y[i])})
            wide &= aligned(t->data, 16) && t->nb[1] % 16 == 0 && t->nb[2] % 16 == 0;
        a.x[i] = x[i]->data;
        a.y[i] = y[i]->data;
        a.xs_head[i] = int64_t(x[i]->nb[1] / b);
        a.xs_tok[i] = int64_t(x[i]->nb[2] / b);
        a.ys_head[i] = int64_t(y[i]->nb[1] / b);
        a.ys_tok[i] = int64_t(y[i]->nb[2] / b);
        if (x[i]->ne[1] > (1 << 20)) return fail(CPQ_ERR_UNSUPPORTED, "rope: %lld heads", (long long)x[i]->ne[1]);
        a.head0[i + 1] = a.head0[i] + int(x[i]->ne[1]);
    }
    const int64_t d = x[0]->ne[0], t = x[0]->ne[2];
    if (rope->n_dims > d) return fail(CPQ_ERR_INVALID_ARG, "rope: n_dims=%d > head size %lld", rope->n_dims, (long long)d);
    if (d > 4096) return fail(CPQ_ERR_UNSUPPORTED, "rope: head size %lld > 4096", (long long)d);
    if (t == 0) return CPQ_SUCCESS;
    for (int i = 0; i < n; i++)  // the tensors are rotated at once, by CTAs that do not wait for one another
        for (int j = 0; j < n; j++)
            if (i != j && (y[i]->data == y[j]->data || y[i]->data == x[j]->data))
                return fail(CPQ_ERR_INVALID_ARG, "rope: output %d is also tensor %d", i, j);
    if (!pos) return fail(CPQ_ERR_INVALID_ARG, "rope: null positions");
    const bool half = rope->mode == CPQ_ROPE_HALF;
    // 16-byte items want whole vectors: of each half and of the tail, or of the head
    const int vec = 16 / act_bytes(x[0]->type);
    wide &= d % vec == 0 && (!half || (rope->n_dims / 2) % vec == 0);
    if (!wide && !half && d % 2) {
        return fail(CPQ_ERR_UNSUPPORTED, "rope: interleaved pairs need an even head size (%lld)", (long long)d);
    }
    a.pos = pos;
    a.d = int(d);
    a.n_dims = rope->n_dims;
    a.n_tensors = n;
    a.m = rope->m;
    memcpy(a.turns, rope->turns, sizeof a.turns);
    const int width = wide ? vec : half ? 1 : 2;  // elements of an item
    a.pair_items = half ? rope->n_dims / 2 / width : (rope->n_dims + width - 1) / width;
    a.items = a.pair_items + (copy ? int(d - (half ? rope->n_dims : a.pair_items * width)) / width : 0);
    if (t > 2147483647) return fail(CPQ_ERR_UNSUPPORTED, "rope: %lld tokens", (long long)t);
    // a CTA takes as many tokens' heads (up to kRopeMaxTok) as make whole waves of four CTAs per SM (40 heads of 128,
    // bf16, us: 8191 tokens 36.6 with seven in two waves, 38.3 with four in 3.5, 54 with one; halves 34.5 : 38.3); few tokens
    // share their heads out over as many CTAs as fill the GPU, down to about one item per thread (8 tokens x 28 heads:
    // 2.4, a CTA per token 4.0)
    const int heads = a.head0[n], least = std::min(heads, (kRopeThreads + a.items - 1) / a.items);
    const int64_t sms = sm_count(std::max(current_device(), 0));
    const int64_t groups = std::max<int64_t>(1, std::min<int64_t>(heads / least, 2 * sms / t));
    a.heads_per_cta = int((heads + groups - 1) / groups);
    const int64_t waves = (t + kRopeMaxTok * 4 * sms - 1) / (kRopeMaxTok * 4 * sms);
    a.tok_per_cta = int((t + waves * 4 * sms - 1) / (waves * 4 * sms));
    a.t = t;
    a.by_items = FastDiv(uint32_t(a.items));
    a.step = std::max(1, kRopeThreads / a.items);
    a.by_pairs = FastDiv(uint32_t(rope->n_dims / 2));
    const dim3 grid(unsigned((t + a.tok_per_cta - 1) / a.tok_per_cta), unsigned((heads + a.heads_per_cta - 1) / a.heads_per_cta));
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e;
    if (x[0]->type == CPQ_TYPE_F32) e = launch_rope<float>(a, half, wide, grid, st);
    else if (x[0]->type == CPQ_TYPE_F16) e = launch_rope<__half>(a, half, wide, grid, st);
    else e = launch_rope<__nv_bfloat16>(a, half, wide, grid, st);
    return e == cudaSuccess ? CPQ_SUCCESS : cuda_fail(e, "rope launch");
}
