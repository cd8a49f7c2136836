// kv_cache.inl — cpq_kv_*: host side of kv_cache.cuh.

namespace cpq {

static bool kv_block_ok(int32_t b) { return b == 16 || b == 32 || b == 64 || b == 128; }

// Lets a kernel use `bytes` of dynamic shared memory, once per device.
template <auto KERNEL>
static cudaError_t raise_shared_limit(int bytes) {
    static std::atomic<uint64_t> done{0};  // bit per device
    const uint64_t bit = uint64_t(1) << (std::max(current_device(), 0) & 63);
    if (done.load() & bit) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) done.fetch_or(bit);
    return e;
}

static int log_block(int32_t b) { return b == 16 ? 4 : b == 32 ? 5 : b == 64 ? 6 : 7; }

// The cache's own fields; what: the caller's name in messages.
static cpq_status check_cache(const cpq_kv_cache *c, const char *what) {
    if (!c) return fail(CPQ_ERR_INVALID_ARG, "%s: null cache", what);
    if (c->format != CPQ_KV_INT8 && c->format != CPQ_KV_E4M3)
        return fail(CPQ_ERR_INVALID_ARG, "%s: cache format %d", what, c->format);
    if (c->head_dim != 128 && c->head_dim != 256)
        return fail(CPQ_ERR_UNSUPPORTED, "%s: head size %d (128 or 256)", what, c->head_dim);
    if (!kv_block_ok(c->block)) return fail(CPQ_ERR_UNSUPPORTED, "%s: %d tokens per page (16, 32, 64 or 128)", what, c->block);
    if (c->n_head_kv < 1 || c->n_head_kv > 65535 || c->n_pages < 1 || c->n_pages > 2147483647)
        return fail(CPQ_ERR_INVALID_ARG, "%s: cache of %lld pages, %d kv heads", what, (long long)c->n_pages, c->n_head_kv);
    if (!c->k || !c->v || !c->k_scale || !c->v_scale) return fail(CPQ_ERR_INVALID_ARG, "%s: null cache pointer", what);
    if (!aligned(c->k, 128) || !aligned(c->v, 128) || !aligned(c->k_scale, 4) || !aligned(c->v_scale, 4))
        return fail(CPQ_ERR_UNSUPPORTED, "%s: the cache's codes must be 128-byte aligned", what);
    return CPQ_SUCCESS;
}

// k and v (or k_out and v_out): [D, n_head_kv, rows, 1] beside a cache.
static cpq_status check_kv_rows(const cpq_kv_cache *c, const cpq_tensor *k, const cpq_tensor *v, const char *what) {
    if (!head_rows(k) || !head_rows(v))
        return fail(CPQ_ERR_INVALID_ARG, "%s: k and v must be F32, F16 or BF16 with ne=[D, heads, rows, 1] and contiguous rows", what);
    if (k->type != v->type) return fail(CPQ_ERR_INVALID_ARG, "%s: k and v of different types", what);
    for (const cpq_tensor *t : {k, v})
        if (t->ne[0] != c->head_dim || t->ne[1] != c->n_head_kv || t->ne[2] != k->ne[2])
            return fail(CPQ_ERR_INVALID_ARG, "%s: ne=[%lld, %lld, %lld] does not fit the cache's %d heads of %d", what,
                        (long long)t->ne[0], (long long)t->ne[1], (long long)t->ne[2], c->n_head_kv, c->head_dim);
    if (k->ne[2] > 2147483647) return fail(CPQ_ERR_UNSUPPORTED, "%s: %lld rows", what, (long long)k->ne[2]);
    return CPQ_SUCCESS;
}

static bool wide_rows(const cpq_tensor *t, size_t a) { return aligned(t->data, a) && t->nb[1] % a == 0 && t->nb[2] % a == 0; }

template <typename T, bool WIDE, int FMT>
static cudaError_t launch_append_k(const AppendArgs &a, dim3 grid, cudaStream_t st) {
    constexpr int kMax = 128 * 256 * int(sizeof(T));  // a run of the largest page
    const int bytes = (a.d << a.log_block) * int(sizeof(T));
    if (bytes > 48 * 1024) {
        const cudaError_t e = raise_shared_limit<kv_append_kernel<T, WIDE, FMT>>(kMax);
        if (e != cudaSuccess) return e;
    }
    const int items = bytes / 16;  // a thread has some items, a CTA not more threads than it needs
    const dim3 block(unsigned(std::min(kAppendThreads, std::max(64, items / 8))));
    return launch(kv_append_kernel<T, WIDE, FMT>, grid, block, size_t(bytes), st, a);
}

template <typename T>
static cudaError_t launch_append(const AppendArgs &a, bool wide, int fmt, dim3 grid, cudaStream_t st) {
    if (fmt == CPQ_KV_INT8)
        return wide ? launch_append_k<T, true, CPQ_KV_INT8>(a, grid, st) : launch_append_k<T, false, CPQ_KV_INT8>(a, grid, st);
    return wide ? launch_append_k<T, true, CPQ_KV_E4M3>(a, grid, st) : launch_append_k<T, false, CPQ_KV_E4M3>(a, grid, st);
}

template <typename T>
static cudaError_t launch_gather(const GatherArgs &a, bool wide, int fmt, dim3 grid, cudaStream_t st) {
    const dim3 block(kGatherThreads);
    if (fmt == CPQ_KV_INT8)
        return wide ? launch(kv_gather_kernel<T, true, CPQ_KV_INT8>, grid, block, 0, st, a)
                    : launch(kv_gather_kernel<T, false, CPQ_KV_INT8>, grid, block, 0, st, a);
    return wide ? launch(kv_gather_kernel<T, true, CPQ_KV_E4M3>, grid, block, 0, st, a)
                : launch(kv_gather_kernel<T, false, CPQ_KV_E4M3>, grid, block, 0, st, a);
}

}  // namespace cpq

extern "C" cpq_status cpq_kv_slots(const cpq_kv_slot_args *s, void *stream) {
    using namespace cpq;
    if (!s) return fail(CPQ_ERR_INVALID_ARG, "kv_slots: null argument");
    if (s->n_seqs < 0 || s->n_rows < 0 || s->n_free < 0 || s->max_blocks < 0 || s->n_seqs > 2147483647 ||
        s->n_rows > 2147483647 || s->n_free > 2147483647)
        return fail(CPQ_ERR_INVALID_ARG, "kv_slots: n_seqs=%lld n_rows=%lld n_free=%lld max_blocks=%d", (long long)s->n_seqs,
                    (long long)s->n_rows, (long long)s->n_free, s->max_blocks);
    if (!kv_block_ok(s->block)) return fail(CPQ_ERR_UNSUPPORTED, "kv_slots: %d tokens per page (16, 32, 64 or 128)", s->block);
    if (s->table_stride < s->max_blocks)
        return fail(CPQ_ERR_INVALID_ARG, "kv_slots: table stride %lld < max_blocks %d", (long long)s->table_stride, s->max_blocks);
    if (!s->seq_start || !s->taken || !s->taken_out)
        return fail(CPQ_ERR_INVALID_ARG, "kv_slots: null seq_start, taken or taken_out");
    if (s->n_seqs > 0 && (!s->ctx_len || !s->new_len || !s->kv_len || (!s->table && s->max_blocks > 0)))
        return fail(CPQ_ERR_INVALID_ARG, "kv_slots: null per-sequence pointer");
    if (s->n_rows > 0 && (!s->pos || !s->slot)) return fail(CPQ_ERR_INVALID_ARG, "kv_slots: null pos or slot");
    if (s->n_free > 0 && !s->free_pages) return fail(CPQ_ERR_INVALID_ARG, "kv_slots: null free_pages");
    // CTAs read the inputs while others write the outputs
    const void *const in[4] = {s->ctx_len, s->new_len, s->free_pages, s->taken};
    const void *const out[6] = {s->table, s->taken_out, s->seq_start, s->kv_len, s->pos, s->slot};
    for (int i = 0; i < 6; i++) {
        for (int j = 0; j < 4; j++)
            if (out[i] && out[i] == in[j] && !(i == 1 && j == 3))
                return fail(CPQ_ERR_INVALID_ARG, "kv_slots: an output is also an input (only taken_out may be taken)");
        for (int j = 0; j < i; j++)
            if (out[i] && out[i] == out[j]) return fail(CPQ_ERR_INVALID_ARG, "kv_slots: two outputs at one address");
    }
    SlotArgs a{s->ctx_len, s->new_len, s->n_seqs, s->table, s->table_stride, s->max_blocks, s->block,
               s->free_pages, s->n_free, s->taken, s->taken_out, s->seq_start, s->kv_len, s->pos, s->slot, s->n_rows};
    // a row per thread; the scan, which every CTA repeats, takes longer than that (300 requests, 60000 rows: 6.4 us,
    // one CTA 72, eight times as many 6.2)
    const int64_t per_cta = 1024;
    int64_t ctas = s->taken_out == s->taken ? 1 : (s->n_rows + per_cta - 1) / per_cta;
    ctas = std::min<int64_t>(std::max<int64_t>(ctas, 1), sm_count(std::max(current_device(), 0)));
    const cudaError_t e = launch(kv_slots_kernel, dim3(unsigned(ctas)), dim3(kSlotThreads), 0, static_cast<cudaStream_t>(stream), a);
    return e == cudaSuccess ? CPQ_SUCCESS : cuda_fail(e, "kv_slots launch");
}

extern "C" cpq_status cpq_kv_append(const cpq_kv_cache *c, const cpq_tensor *k, const cpq_tensor *v, const int64_t *slot,
                                    void *stream) {
    using namespace cpq;
    cpq_status st = check_cache(c, "kv_append");
    if (st == CPQ_SUCCESS) st = check_kv_rows(c, k, v, "kv_append");
    if (st != CPQ_SUCCESS) return st;
    const int64_t t = k->ne[2];
    if (t == 0) return CPQ_SUCCESS;
    if (!slot) return fail(CPQ_ERR_INVALID_ARG, "kv_append: null slots");
    const size_t b = size_t(act_bytes(k->type));
    AppendArgs a{};
    const cpq_tensor *const x[2] = {k, v};
    for (int z = 0; z < 2; z++) {
        a.x[z] = x[z]->data;
        a.xs_head[z] = int64_t(x[z]->nb[1] / b);
        a.xs_tok[z] = int64_t(x[z]->nb[2] / b);
    }
    a.codes[0] = static_cast<uint8_t *>(c->k);
    a.codes[1] = static_cast<uint8_t *>(c->v);
    a.scale[0] = c->k_scale;
    a.scale[1] = c->v_scale;
    a.slot = slot;
    a.t = t;
    a.n_slots = c->n_pages * c->block;
    a.n_head = c->n_head_kv;
    a.d = c->head_dim;
    a.log_block = log_block(c->block);
    // A group's runs are written one after another, so few rows get a CTA each (24 rows with the gather that follows:
    // 8.0 us, groups of 32: 33); many rows are mostly insides of runs, whose CTAs would only look and leave (14000 rows:
    // 60 us, groups of one: 260).
    const int64_t work = t * c->n_head_kv * 2, sms = sm_count(std::max(current_device(), 0));
    a.group = int(std::min<int64_t>(kAppendMaxGroup, std::max<int64_t>(1, work / (16 * sms))));
    const dim3 grid(unsigned((t + a.group - 1) / a.group), unsigned(c->n_head_kv), 2);
    const bool wide = wide_rows(k, 16) && wide_rows(v, 16);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e;
    if (k->type == CPQ_TYPE_F32) e = launch_append<float>(a, wide, c->format, grid, s);
    else if (k->type == CPQ_TYPE_F16) e = launch_append<__half>(a, wide, c->format, grid, s);
    else e = launch_append<__nv_bfloat16>(a, wide, c->format, grid, s);
    return e == cudaSuccess ? CPQ_SUCCESS : cuda_fail(e, "kv_append launch");
}

extern "C" cpq_status cpq_kv_gather(const cpq_kv_cache *c, const int64_t *slot, cpq_tensor *k, cpq_tensor *v, void *stream) {
    using namespace cpq;
    cpq_status st = check_cache(c, "kv_gather");
    if (st == CPQ_SUCCESS) st = check_kv_rows(c, k, v, "kv_gather");
    if (st != CPQ_SUCCESS) return st;
    const int64_t t = k->ne[2];
    if (t == 0) return CPQ_SUCCESS;
    if (!slot) return fail(CPQ_ERR_INVALID_ARG, "kv_gather: null slots");
    if (k->data == v->data) return fail(CPQ_ERR_INVALID_ARG, "kv_gather: k and v are one tensor");
    const size_t b = size_t(act_bytes(k->type));
    GatherArgs a{};
    cpq_tensor *const y[2] = {k, v};
    for (int z = 0; z < 2; z++) {
        a.y[z] = y[z]->data;
        a.ys_head[z] = int64_t(y[z]->nb[1] / b);
        a.ys_tok[z] = int64_t(y[z]->nb[2] / b);
    }
    a.codes[0] = static_cast<const uint8_t *>(c->k);
    a.codes[1] = static_cast<const uint8_t *>(c->v);
    a.scale[0] = c->k_scale;
    a.scale[1] = c->v_scale;
    a.slot = slot;
    a.t = t;
    a.n_slots = c->n_pages * c->block;
    a.n_head = c->n_head_kv;
    a.d = c->head_dim;
    a.log_block = log_block(c->block);
    a.by_row = FastDiv(uint32_t(c->n_head_kv) * uint32_t(c->head_dim) / uint32_t(16 / b));
    const dim3 grid(unsigned((t + kGatherRows - 1) / kGatherRows), 2);
    const bool wide = wide_rows(k, 16) && wide_rows(v, 16);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e;
    if (k->type == CPQ_TYPE_F32) e = launch_gather<float>(a, wide, c->format, grid, s);
    else if (k->type == CPQ_TYPE_F16) e = launch_gather<__half>(a, wide, c->format, grid, s);
    else e = launch_gather<__nv_bfloat16>(a, wide, c->format, grid, s);
    return e == cudaSuccess ? CPQ_SUCCESS : cuda_fail(e, "kv_gather launch");
}
