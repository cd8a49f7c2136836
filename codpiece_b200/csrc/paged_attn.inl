// paged_attn.inl — cpq_paged_attn: host side of paged_attn.cuh and paged_attn_tc.cuh.

namespace cpq {

// The cache's codes as [D / 128][head rows][128] bytes, box 128 bytes x up to 32 keys x all of D, 128-byte swizzle.
static cpq_status kv_tensor_map(const cpq_kv_cache *c, const void *codes, CUtensorMap *out) {
    EncodeTiledFn enc = encode_tiled();
    if (!enc) return fail(CPQ_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    const cuuint64_t rows = cuuint64_t(c->n_pages) * cuuint64_t(c->n_head_kv) * cuuint64_t(c->block);
    const cuuint64_t dims[3] = {128, rows, cuuint64_t(c->head_dim / 128)};
    const cuuint64_t strides[2] = {cuuint64_t(c->head_dim), 128};
    const cuuint32_t box[3] = {128, cuuint32_t(std::min(c->block, kAttnTile)), cuuint32_t(c->head_dim / 128)};
    const cuuint32_t estr[3] = {1, 1, 1};
    const CUresult r = enc(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void *>(codes), dims, strides, box, estr,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? CPQ_SUCCESS : fail(CPQ_ERR_CUDA, "cuTensorMapEncodeTiled (kv cache) failed (%d)", int(r));
}

// Workspace of a launch of `ctas` CTAs with `rows` rows per unit: partial accumulators, statistics, headers, flushed
// accumulators.
static size_t attn_ws_bytes(int ctas, int rows, int d) {
    const size_t slots = 2 * size_t(ctas);
    return align_up(slots * rows * d * 4, 256) + align_up(slots * rows * 8, 256) + align_up(slots * 16, 256) + size_t(ctas) * kAttnAcc * d;
}

static void attn_carve(AttnArgs &a, void *ws, int ctas, int rows, int d) {
    const size_t slots = 2 * size_t(ctas);
    uint8_t *p = static_cast<uint8_t *>(ws);
    a.part_o = reinterpret_cast<float *>(p);
    p += align_up(slots * rows * d * 4, 256);
    a.part_ml = reinterpret_cast<float2 *>(p);
    p += align_up(slots * rows * 8, 256);
    a.part_hdr = reinterpret_cast<int4 *>(p);
    p += align_up(slots * 16, 256);
    a.acc = reinterpret_cast<float4 *>(p);
}

template <int D, int ROWS>
static cudaError_t launch_attn_combine(const AttnArgs &a, int ctas, cudaStream_t st) {
    constexpr int y = ROWS / CombineCfg<D, ROWS>::kRowsHere;
    return launch(attn_combine_kernel<D, ROWS>, dim3(unsigned(ctas), unsigned(y)), dim3(kCombineThreads), 0, st, a);
}

template <int D, int FMT, bool SPLIT>
static cudaError_t launch_attn_decode(const AttnArgs &a, int ctas, cudaStream_t st) {
    using C = DecCfg<D, SPLIT>;
    cudaError_t e = raise_shared_limit<attn_decode_kernel<D, FMT, SPLIT>>(C::kSmem);
    if (e != cudaSuccess) return e;
    e = launch(attn_decode_kernel<D, FMT, SPLIT>, dim3(unsigned(ctas)), dim3(C::kThreads), C::kSmem, st, a);
    if (e != cudaSuccess) return e;
    return launch_attn_combine<D, C::kRows>(a, ctas, st);
}

template <int D, int FMT, bool SPLIT>
static cudaError_t launch_attn_tc(const AttnArgs &a, int ctas, cudaStream_t st) {
    using C = TaCfg<D, SPLIT>;
    cudaError_t e = raise_shared_limit<attn_tc_kernel<D, FMT, SPLIT>>(C::kSmem);
    if (e != cudaSuccess) return e;
    e = launch(attn_tc_kernel<D, FMT, SPLIT>, dim3(unsigned(ctas)), dim3(kTaThreads), C::kSmem, st, a);
    if (e != cudaSuccess) return e;
    return launch_attn_combine<D, kTaRows>(a, ctas, st);
}

template <int D, bool SPLIT>
static cudaError_t launch_attn(const AttnArgs &a, bool tc, int fmt, int ctas, cudaStream_t st) {
    if (fmt == CPQ_KV_INT8)
        return tc ? launch_attn_tc<D, CPQ_KV_INT8, SPLIT>(a, ctas, st) : launch_attn_decode<D, CPQ_KV_INT8, SPLIT>(a, ctas, st);
    return tc ? launch_attn_tc<D, CPQ_KV_E4M3, SPLIT>(a, ctas, st) : launch_attn_decode<D, CPQ_KV_E4M3, SPLIT>(a, ctas, st);
}

// The decode kernel or the tensor-core kernel. The first reads a sequence's keys
// once per 8 or 16 query rows, the second once per 128 but begins late (some 15
// us). Decode while sequences have at most two of its row tiles on average (24
// heads over 4 of 256, us, decode : tensor core; fp32 1 request of 1 x 1000 keys
// 13.6 : 27.5, 4 requests of 2 x 20000 73 : 99; bf16 16 of 4 x 4000 75 : 75, 4 of
// 5 x 20000 78 : 82), and with more while the tables, which bound the keys, leave
// at most 40 (row tile, 32 keys) per SM (1 request of 8 x 1000 16.9 : 29.7, 8 x
// 8000 31 : 38, 32 x 1000 26 : 37; beyond, the tensor cores win: fp32 16 of 4 x 4000
// 95 : 94, and 4 of 8 x 20001 81 where the other would read every key six times).
// 24 heads over 8 of 128 agree (fp32 1 of 8 x 1000 14.2 : 20.8, 32 x 1000 19.0 : 23.1;
// bf16 16 x 1000 16.5 : 19.8, 32 x 1000 19.0 : 21.5). The mean and the width
// stand for lengths that the host does not know: a batch that mixes single tokens
// with a long chunk, or a table far wider than its keys, may get the slower kernel.
static int attn_few(const cpq_tensor *q) { return q->type == CPQ_TYPE_F32 ? 8 : 16; }
static bool attn_is_decode(const cpq_tensor *q, const cpq_kv_cache *c, int64_t n_seqs) {
    return q->ne[2] * (q->ne[1] / c->n_head_kv) <= 2 * attn_few(q) * n_seqs;
}
static int attn_rows(const cpq_tensor *q, const cpq_kv_cache *c, int64_t n_seqs, int64_t keys, int sms) {
    if (attn_is_decode(q, c, n_seqs)) return attn_few(q);
    const int64_t tiles = q->ne[2] * (q->ne[1] / c->n_head_kv) / attn_few(q) + n_seqs, key_tiles = (keys + kAttnTile - 1) / kAttnTile;
    return tiles <= 40 * sms && tiles * c->n_head_kv * key_tiles <= 40 * sms ? attn_few(q) : kTaRows;
}

}  // namespace cpq

extern "C" size_t cpq_paged_attn_workspace_size(const cpq_kv_cache *c, const cpq_tensor *q, int64_t n_seqs) {
    using namespace cpq;
    if (!c || !q || c->n_head_kv < 1) return 0;
    return attn_ws_bytes(sm_count(std::max(current_device(), 0)), attn_is_decode(q, c, n_seqs) ? attn_few(q) : kTaRows, c->head_dim);
}

extern "C" cpq_status cpq_paged_attn(const cpq_tensor *q, const cpq_kv_cache *c, const cpq_attn_seqs *s, float scale,
                                     int32_t causal, cpq_tensor *out, float *lse, void *workspace, size_t workspace_bytes,
                                     void *stream) {
    using namespace cpq;
    cpq_status st = check_cache(c, "paged_attn");
    if (st != CPQ_SUCCESS) return st;
    if (!head_rows(q) || !head_rows(out))
        return fail(CPQ_ERR_INVALID_ARG, "paged_attn: q and out must be F32, F16 or BF16 with ne=[D, heads, tokens, 1] and contiguous rows");
    if (q->type != out->type || q->ne[0] != out->ne[0] || q->ne[1] != out->ne[1] || q->ne[2] != out->ne[2])
        return fail(CPQ_ERR_INVALID_ARG, "paged_attn: out differs from q in type or shape");
    if (q->ne[0] != c->head_dim || q->ne[1] % c->n_head_kv)
        return fail(CPQ_ERR_INVALID_ARG, "paged_attn: q ne=[%lld, %lld] does not fit %d kv heads of %d", (long long)q->ne[0],
                    (long long)q->ne[1], c->n_head_kv, c->head_dim);
    if (!s) return fail(CPQ_ERR_INVALID_ARG, "paged_attn: null sequences");
    if (s->n_seqs < 0 || s->max_blocks < 0 || s->table_stride < s->max_blocks)
        return fail(CPQ_ERR_INVALID_ARG, "paged_attn: n_seqs=%lld max_blocks=%d table stride %lld", (long long)s->n_seqs, s->max_blocks,
                    (long long)s->table_stride);
    if (s->n_seqs > kAttnMaxSeqs) return fail(CPQ_ERR_UNSUPPORTED, "paged_attn: %lld sequences (at most %d)", (long long)s->n_seqs, kAttnMaxSeqs);
    if (!std::isfinite(scale)) return fail(CPQ_ERR_INVALID_ARG, "paged_attn: scale %g", scale);
    if (q->ne[2] == 0 || s->n_seqs == 0) return CPQ_SUCCESS;
    if (!s->seq_start || !s->kv_len || (!s->table && s->max_blocks > 0)) return fail(CPQ_ERR_INVALID_ARG, "paged_attn: null sequence pointer");
    const int64_t rows = q->ne[2] * q->ne[1];
    if (rows > 2147483647 || c->n_pages * c->n_head_kv * c->block > 2147483647 || int64_t(s->max_blocks) * c->block > 2147483647)
        return fail(CPQ_ERR_UNSUPPORTED, "paged_attn: more than 2^31 - 1 rows, cache rows or keys");
    const bool split = q->type == CPQ_TYPE_F32;
    const int ctas = sm_count(std::max(current_device(), 0));
    const int unit_rows = attn_rows(q, c, s->n_seqs, int64_t(s->max_blocks) * c->block, ctas);
    const bool tc = unit_rows == kTaRows;
    // the units' places (tiles, and those for beginning one) are counted in 32 bits
    const int tile = tc ? kTaTile : kAttnTile, begin = tc ? kTaStart : DecCfg<128, true>::kStart;
    const int64_t tiles = begin + std::max<int64_t>(1, (int64_t(s->max_blocks) * c->block + tile - 1) / tile);
    if ((rows / unit_rows + s->n_seqs * c->n_head_kv) > 2147483647 / tiles)
        return fail(CPQ_ERR_UNSUPPORTED, "paged_attn: %lld rows over up to %lld keys are too many for one call", (long long)rows,
                    (long long)s->max_blocks * c->block);
    if (!workspace) return fail(CPQ_ERR_NOT_INITIALIZED, "paged_attn: no workspace");
    const size_t need = cpq_paged_attn_workspace_size(c, q, s->n_seqs);
    if (!aligned(workspace, 256) || workspace_bytes < need)
        return fail(CPQ_ERR_WORKSPACE, "paged_attn: workspace of %zu bytes, 256-byte aligned, needs %zu", workspace_bytes, need);
    if (q->data == out->data)
        return fail(CPQ_ERR_INVALID_ARG, "paged_attn: out overlaps q (rows are read after others have been written)");
    AttnArgs a{};
    st = kv_tensor_map(c, c->k, &a.tmap_k);
    if (st == CPQ_SUCCESS) st = kv_tensor_map(c, c->v, &a.tmap_v);
    if (st != CPQ_SUCCESS) return st;
    a.k = static_cast<const uint8_t *>(c->k);
    a.v = static_cast<const uint8_t *>(c->v);
    a.k_scale = c->k_scale;
    a.v_scale = c->v_scale;
    a.n_pages = c->n_pages;
    a.block = c->block;
    a.hkv = c->n_head_kv;
    const size_t b = size_t(act_bytes(q->type));
    a.q = q->data;
    a.qs_head = int64_t(q->nb[1] / b);
    a.qs_tok = int64_t(q->nb[2] / b);
    a.out = out->data;
    a.os_head = int64_t(out->nb[1] / b);
    a.os_tok = int64_t(out->nb[2] / b);
    a.lse = lse;
    a.type = q->type;
    a.t = int(q->ne[2]);
    a.group = int(q->ne[1] / c->n_head_kv);
    a.n_seqs = int(s->n_seqs);
    a.seq_start = s->seq_start;
    a.kv_len = s->kv_len;
    a.table = s->table;
    a.table_stride = s->table_stride;
    a.max_blocks = s->max_blocks;
    a.causal = causal ? 1 : 0;
    a.scale_log2 = float(double(scale) * 1.4426950408889634);
    a.wide = wide_rows(q, 16) && wide_rows(out, 16) ? 1 : 0;
    // Short requests are spread wide, latency counts (1 x 1000 keys: 13.3 us, 16.4 with shares of 16 places; 8 x 1000
    // on the tensor cores: 30, 56 with 6).
    a.min_share = tc ? 1 : 4;
    attn_carve(a, workspace, ctas, unit_rows, c->head_dim);
    const cudaStream_t cs = static_cast<cudaStream_t>(stream);
    cudaError_t e;
    if (c->head_dim == 256) e = split ? launch_attn<256, true>(a, tc, c->format, ctas, cs) : launch_attn<256, false>(a, tc, c->format, ctas, cs);
    else e = split ? launch_attn<128, true>(a, tc, c->format, ctas, cs) : launch_attn<128, false>(a, tc, c->format, ctas, cs);
    return e == cudaSuccess ? CPQ_SUCCESS : cuda_fail(e, "paged_attn launch");
}
