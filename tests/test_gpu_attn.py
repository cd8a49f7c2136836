"""GPU checks of the attention core (codpiece_b200/attn.py) against oracle/attn_ref.py in 64 bits.

Bounds, fixed before the first run:
  slots, codes, scales and gathered values are equal.
  rope: |dy| <= 2^-20 m (|a| + |b|) per pair (angle pi 2^-24, sincospif 2 ulp, three roundings),
    plus half an ulp of a 16-bit output.
  attention: a score errs by at most dz = size * (2^-22 + (D / 16 + 2) 2^-23), size the largest scale *
    sum |q_d k_d|: q in 22 bits, one fp32 rounding per 16-deep MMA step and two for the scales; ex2 and the
    second product's terms add 2^-20. A softmax average then moves by at most 2 (dz + 2^-20) max|v|. 16-bit
    outputs: 2^-11 max|v| for fp16 probabilities and half an ulp of the output. lse: dz + 2^-20 + 2^-22 |lse|.
"""
import numpy as np
import pytest

from oracle import attn_ref as R

pytestmark = pytest.mark.gpu

FMT = {"int8": 0, "e4m3": 1}


@pytest.fixture
def A(cuda):
    from codpiece_b200 import attn
    return attn


def _dtype(torch, name):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def _np(t):
    return t.detach().double().cpu().numpy()


def _pool(torch, A, pages, heads, block, d, fmt, seed=0, spread=1.0):
    """A pool with random codes and scales; returns (cache, K values, V values) as numbers."""
    g = torch.Generator().manual_seed(seed)
    c = A.KvCache.empty(pages, heads, d, block, FMT[fmt])
    vals = []
    for codes, scale in ((c.k, c.k_scale), (c.v, c.v_scale)):
        x = torch.randn(pages, heads, block, d, generator=g)
        x = x / x.abs().amax(dim=(2, 3), keepdim=True) * R.TOP[fmt]
        q = torch.round(x).to(torch.int8) if fmt == "int8" else x.to(torch.float8_e4m3fn)
        codes.copy_(q)
        scale.copy_((torch.rand(pages, heads, generator=g) * spread + 0.5) / R.TOP[fmt] * 3)
        vals.append(_np(codes.float()) * _np(scale)[:, :, None, None])
    return c, vals[0], vals[1]


# ---- rope ---------------------------------------------------------------------------------


@pytest.mark.parametrize("d,n_dims,half,typ,params", [
    (256, 64, True, "f32", {}),
    (256, 256, False, "f32", {"base": 1e6}),
    (128, 128, True, "bf16", {"freq_scale": 0.25}),
    (128, 64, False, "f16", {"freq_scale": 0.25, "ext_factor": 1.0, "n_ctx_orig": 32768, "base": 1e6}),
    (256, 64, True, "f32", {"freq_scale": 0.125, "ext_factor": 1.0, "n_ctx_orig": 4096, "attn_factor": 1.5}),
    (128, 70, True, "f32", {}),      # halves that fill no 16-byte item
    (128, 70, False, "bf16", {}),    # the rotated part ends inside an item
    (96, 2, True, "f16", {"freq_factors": [3.0]}),
    (66, 66, False, "f32", {}),
    (67, 30, True, "f32", {}),       # an odd head size
])
@pytest.mark.parametrize("t", [1, 7])
def test_rope(cuda, A, d, n_dims, half, typ, params, t):
    torch = cuda
    g = torch.Generator().manual_seed(d + n_dims + t)
    dt = _dtype(torch, typ)
    q = torch.randn(t, 5, d, generator=g).to(dt).cuda()
    k = torch.randn(t, 2, d, generator=g).to(dt).cuda()
    pos = torch.tensor([0, 1, 5, 999983, 2147483647, -3, 131071][:t] if t > 1 else [1000003], dtype=torch.int32).cuda()
    table = A.Rope(n_dims, A.ROPE_HALF if half else A.ROPE_INTERLEAVED, **params)
    outs = A.rope(table, [q, k], pos)
    _, m = R.rope_frequencies(n_dims, **params)
    for x, y in zip((q, k), outs):
        xn, pn = _np(x), pos.cpu().numpy()
        # the last positions are far enough for 64-bit angles to err themselves: p * 2^-53 rad
        ref = R.rope(xn, pn, n_dims, half, **params)
        h = n_dims // 2
        a, b = (slice(0, h), slice(h, n_dims)) if half else (slice(0, n_dims, 2), slice(1, n_dims, 2))
        size = np.zeros_like(xn)
        size[..., a] = size[..., b] = np.abs(xn[..., a]) + np.abs(xn[..., b])
        far = np.abs(pn.astype(np.float64))[:, None, None] * 2.0 ** -51
        bound = m * size * (2.0 ** -20 + far)
        if typ != "f32":
            bound = bound + np.abs(ref) * torch.finfo(dt).eps / 2 * 1.001
        bound[..., n_dims:] = 0.0  # copied
        assert (np.abs(_np(y) - ref) <= bound).all()


def test_rope_in_place_and_in_views(cuda, A):
    """q and k as views of one projection output, rotated where they lie; the rest of the buffer untouched."""
    torch = cuda
    buf = torch.randn(9, 4 * 256 + 2 * 256 + 8, device="cuda")
    before = buf.clone()
    q, k = buf[:, :1024].unflatten(-1, (4, 256)), buf[:, 1024:1536].unflatten(-1, (2, 256))
    pos = torch.arange(9, dtype=torch.int32, device="cuda") + 7
    table = A.Rope(64)
    want = A.rope(table, [q.clone(), k.clone()], pos)
    A.rope(table, [q, k], pos, [q, k])
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert torch.equal(buf[:, 1536:], before[:, 1536:])
    # unaligned views take the element path
    odd = torch.randn(9, 3 * 131 + 1, device="cuda")[:, 1:].unflatten(-1, (3, 131))[..., :128]
    got = A.rope(A.Rope(128, A.ROPE_INTERLEAVED), [odd], pos)[0]
    assert torch.equal(got, A.rope(A.Rope(128, A.ROPE_INTERLEAVED), [odd.contiguous()], pos)[0])


def test_rope_many_tokens(cuda, A):
    """More tokens than CTAs, against the same rows rotated one at a time."""
    torch = cuda
    x = torch.randn(3001, 3, 128, device="cuda").bfloat16()
    pos = torch.randint(0, 1 << 20, (3001,), dtype=torch.int32, device="cuda")
    table = A.Rope(128, A.ROPE_HALF, base=1e6)
    y = A.rope(table, [x], pos)[0]
    for i in (0, 1, 1500, 2999, 3000):
        assert torch.equal(y[i:i + 1], A.rope(table, [x[i:i + 1]], pos[i:i + 1])[0])


# ---- slots --------------------------------------------------------------------------------


def _slots_case(torch, A, ctx, new, block, width, n_free, n_rows, taken=0, in_place=True, seed=0):
    rng = np.random.default_rng(seed)
    n = len(ctx)
    ids = rng.permutation(10000).astype(np.int32)
    table = np.full((n, width), -1, np.int32)
    at = 0
    for r in range(n):
        held = min(-(-max(ctx[r], 0) // block), width)
        table[r, :held] = ids[at:at + held]
        at += held
    free = ids[at:at + n_free].copy()
    i32 = lambda v: torch.tensor(np.asarray(v, np.int32)).cuda()  # noqa: E731
    tab, tk = i32(table), i32([taken])
    tk_out = tk if in_place else i32([-7])
    s = A.kv_slots(i32(ctx), i32(new), tab, i32(free), tk, block=block, n_rows=n_rows, taken_out=tk_out)
    ref_tab = table.copy()
    ref = R.kv_slots(ctx, new, ref_tab, free, taken, block, n_rows)
    for name in ("seq_start", "kv_len", "pos", "slot"):
        assert np.array_equal(getattr(s, name).cpu().numpy(), ref[name]), name
    assert np.array_equal(tab.cpu().numpy(), ref_tab)
    assert int(tk_out[0]) == ref["taken"]


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("ctx,new,block,width,n_free,n_rows", [
    ([0], [1], 16, 1, 1, 1),
    ([0], [0], 16, 1, 0, 0),
    ([15, 16, 17], [1, 1, 1], 16, 4, 5, 3),
    ([0, 5, 64], [130, 0, 1], 64, 5, 9, 140),
    ([0, 0, 0, 16], [40, 40, 3, 0], 16, 4, 5, 100),     # the second does not get its pages, the fourth needs none
    ([0, 30, 0], [70, 3, 5], 16, 4, 20, 100),           # the first is longer than the table
    ([0, 30, 0], [20, 10, 5], 16, 4, 20, 32),           # the rows end before the last request does
    ([-1, 4, 4], [2, -3, 2], 16, 4, 20, 10),            # negative lengths
])
def test_slots(cuda, A, ctx, new, block, width, n_free, n_rows, in_place):
    _slots_case(cuda, A, ctx, new, block, width, n_free, n_rows, in_place=in_place)
    _slots_case(cuda, A, ctx, new, block, width, n_free + 3, n_rows, taken=3, in_place=in_place)


@pytest.mark.parametrize("n,new,in_place", [(31, 1, True), (700, 9, False), (2050, 7, True), (2050, 7, False)])
def test_slots_many_requests(cuda, A, n, new, in_place):
    """More requests than threads, more rows than one CTA's, some without any row."""
    rng = np.random.default_rng(n)
    ctx, add = rng.integers(0, 60, n), rng.integers(0, new + 1, n)
    _slots_case(cuda, A, ctx, add, 32, 4, int(add.sum()) // 32 + n // 2, int(add.sum()) + 11, in_place=in_place)


# ---- append and gather --------------------------------------------------------------------


def _append_both(torch, A, cache, fmt, k, v, slot):
    """Appends on the GPU and in the reference; returns nothing, compares everything."""
    state = []
    for codes, scale, x in ((cache.k, cache.k_scale, k), (cache.v, cache.v_scale, v)):
        c, s = _np(codes.float()), scale.cpu().numpy().copy()
        R.kv_append(c, s, _np(x), slot.cpu().numpy(), fmt)
        state.append((c, s))
    A.kv_append(cache, k, v, slot)
    for (c, s), codes, scale in ((state[0], cache.k, cache.k_scale), (state[1], cache.v, cache.v_scale)):
        assert np.array_equal(scale.cpu().numpy(), s)
        assert np.array_equal(_np(codes.float()), c, equal_nan=True)  # places nobody wrote may hold anything


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("block,d,heads", [(16, 128, 1), (32, 256, 3), (64, 256, 4), (128, 128, 2)])
def test_append(cuda, A, fmt, typ, block, d, heads):
    """Runs that begin, fill, end in and leave pages; later appends with larger and smaller values; skipped rows."""
    torch = cuda
    g = torch.Generator().manual_seed(block + d)
    cache, _, _ = _pool(torch, A, 9, heads, block, d, fmt, seed=3)
    dt = _dtype(torch, typ)

    def rows(n, gain):
        return [(torch.randn(n, heads, d, generator=g) * gain).to(dt).cuda() for _ in range(2)]

    def seq(pages, a, b):
        return [pages[p // block] * block + p % block for p in range(a, b)]

    one, two, three = [4, 0, 7], [2], [8, 1]
    steps = [
        (1.0, seq(one, 0, block + 3) + [-1] + seq(two, 0, 5) + seq(three, 0, block)),
        (4.0, seq(one, block + 3, block + 4) + seq(two, 5, 6) + seq(three, block, block + 1)),   # scales grow: coded again
        (0.1, seq(one, block + 4, block + 5) + [9 * block, 1 << 40] + seq(two, 6, 9)),           # scales stay
        (30.0, seq(one, block + 5, 2 * block) + seq(one, 2 * block, 3 * block)),                 # to the end of a page
    ]
    for gain, slots in steps:
        k, v = rows(len(slots), gain)
        _append_both(torch, A, cache, fmt, k, v, torch.tensor(slots, dtype=torch.int64).cuda())


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_append_borders(cuda, A, fmt):
    """Values on the borders between codes (ties to even), next to them, zeros, subnormals, infinities and NaN."""
    torch = cuda
    vals, _ = R.code_values(fmt)
    border = ((vals[1:] + vals[:-1]) / 2).astype(np.float32)
    for s in (1.0, 0.0123, 3.7e-20, 1e20):
        x = np.concatenate([border * np.float32(s), np.nextafter(border, np.float32(9e9)) * np.float32(s), [0.0, np.inf, -np.inf, np.nan]])
        x = np.concatenate([[R.TOP[fmt] * s], x]).astype(np.float32)
        x = np.resize(x, (16, 1, 128))
        x[0, 0, 0] = R.TOP[fmt] * s
        cache, _, _ = _pool(torch, A, 2, 1, 16, 128, fmt)
        _append_both(torch, A, cache, fmt, torch.from_numpy(x).cuda(), torch.from_numpy(-x).cuda(), torch.arange(16).cuda())
    for fill in (0.0, 1e-45, 3e-31, float("inf"), float("nan")):  # nothing to scale by
        x = torch.full((3, 1, 128), fill).cuda()
        cache, _, _ = _pool(torch, A, 2, 1, 16, 128, fmt)
        _append_both(torch, A, cache, fmt, x, x, torch.tensor([16, 17, 18]).cuda())
        _append_both(torch, A, cache, fmt, torch.randn(1, 1, 128).cuda(), x[:1], torch.tensor([19]).cuda())


def test_append_views_and_random_quotients(cuda, A):
    """k, v as views of a projection output (unaligned ones too), and many values for the rounding."""
    torch = cuda
    for fmt in ("int8", "e4m3"):
        for first in (0, 1):
            buf = torch.randn(64, 2 * 2 * 256 + 8, device="cuda")[:, first:]
            k, v = buf[:, :512].unflatten(-1, (2, 256)), buf[:, 512:1024].unflatten(-1, (2, 256))
            cache, _, _ = _pool(torch, A, 3, 2, 64, 256, fmt)
            _append_both(torch, A, cache, fmt, k, v, (torch.arange(64) + 64).cuda())
            grown = 1.7 * torch.randn(1, 2, 256, device="cuda")
            cache2 = A.KvCache.empty(1, 2, 256, 64, FMT[fmt])
            _append_both(torch, A, cache2, fmt, k[:50], v[:50], torch.arange(50).cuda())
            _append_both(torch, A, cache2, fmt, 3 * grown, 5 * grown, torch.tensor([50]).cuda())


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [128, 256])
def test_gather(cuda, A, fmt, typ, d):
    torch = cuda
    cache, _, _ = _pool(torch, A, 5, 3, 16, d, fmt)
    slot = torch.tensor([79, 0, 17, -1, 16, 80, 17, 1 << 50, 33]).cuda()
    dt = _dtype(torch, typ)
    k, v = A.kv_gather(cache, slot, dtype=dt)
    for got, codes, scale in ((k, cache.k, cache.k_scale), (v, cache.v, cache.v_scale)):
        vals = codes.float() * scale[:, :, None, None]
        want = torch.zeros(9, 3, d, device="cuda")
        for i, s in enumerate(slot.tolist()):
            if 0 <= s < 80:
                want[i] = vals[s // 16, :, s % 16]
        assert torch.equal(got, want.to(dt))
    # into views that are not 16-byte aligned
    out = torch.full((9, 3 * d + 3), 7.0, dtype=dt, device="cuda")
    view = out[:, 1:1 + 3 * d].unflatten(-1, (3, d))
    A.kv_gather(cache, slot, outs=(view, torch.empty(9, 3, d, dtype=dt, device="cuda")))
    assert torch.equal(view, k) and (out[:, 0] == 7).all() and (out[:, 3 * d + 1:] == 7).all()


# ---- attention ----------------------------------------------------------------------------


def _attn_case(torch, A, q_lens, kv_lens, heads, group, d, block, typ, fmt, causal=True, pad=0, seed=0, spread=1.0,
               bad_pages=False, scale=None, gain=1.0, garbage=True):
    rng = np.random.default_rng(seed)
    n = len(q_lens)
    dt = _dtype(torch, typ)
    need = [-(-kv // block) for kv in kv_lens]
    pages = sum(need) + 3
    cache, kv, vv = _pool(torch, A, pages, heads, block, d, fmt, seed=seed + 1, spread=spread)
    ids = rng.permutation(pages)
    width = max(need + [1]) + 1
    table = np.full((n, width), 2 ** 31 - 1, np.int32)  # entries behind the sequences are no pages
    at = 0
    for s in range(n):
        table[s, :need[s]] = ids[at:at + need[s]]
        at += need[s]
    if garbage:  # nothing outside the sequences is fit to be read as a number
        used = {(int(table[s, j // block]), j % block) for s in range(n) for j in range(kv_lens[s])}
        for codes, scales in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
            raw = codes.view(torch.uint8)
            for p in range(pages):
                for i in range(block):
                    if (p, i) not in used:
                        raw[p, :, i] = 0x7f
                if not any((p, i) in used for i in range(block)):
                    scales[p] = float("nan")
    if bad_pages:
        for s in range(n):
            if need[s] > 1:
                table[s, rng.integers(0, need[s])] = [-1, pages, 2 ** 31 - 1, -2 ** 31][s % 4]
    start = np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32)
    t, hq = int(start[-1]) + pad, heads * group
    g = torch.Generator().manual_seed(seed + 2)
    buf = (gain * torch.randn(t, hq * d + 8, generator=g)).to(dt).cuda()
    q = buf[:, :hq * d].unflatten(-1, (hq, d))
    out = torch.full((t, hq, d + 8), 5.0, dtype=dt, device="cuda")[..., :d]
    lse = torch.full((t, hq), 5.0, device="cuda")
    full = torch.tensor(np.concatenate([table, table], axis=1)).cuda()
    sc = d ** -0.5 if scale is None else scale
    ref_all = R.paged_attn(_np(q), kv, vv, table, start, kv_lens, sc, causal)
    # tables just wide enough, and so wide that more than a few rows go to the tensor-core kernel
    for tab in (full[:, :width], torch.cat([full[:, :width], _no_pages(torch, n)], 1)):
        out.fill_(5.0)
        lse.fill_(5.0)
        A.paged_attn(q, cache, tab, torch.tensor(start).cuda(), torch.tensor(np.asarray(kv_lens, np.int32)).cuda(),
                     causal=causal, out=out, lse=lse, scale=scale)
        _check_attn(torch, out, lse, ref_all, start, vv, d, typ)


def _no_pages(torch, n):
    return torch.full((n, 12000), -1, dtype=torch.int32, device="cuda")


def _check_attn(torch, out, lse, ref_all, start, vv, d, typ):
    (ref, ref_lse, size), dt = ref_all, out.dtype
    got, got_lse = _np(out), _np(lse)
    inside = int(start[-1])
    assert (got[inside:] == 5).all() and (got_lse[inside:] == 5).all(), "rows behind the last sequence"
    got, got_lse, ref, ref_lse = got[:inside], got_lse[:inside], ref[:inside], ref_lse[:inside]
    assert np.isfinite(got).all()
    dz = size * (2.0 ** -22 + (d / 16 + 2) * 2.0 ** -23)
    top = np.abs(vv).max()
    bound = 2 * (dz + 2.0 ** -20) * top
    if typ != "f32":
        bound = bound + 2.0 ** -11 * top + np.abs(ref) * torch.finfo(dt).eps / 2 * 1.001
    assert (np.abs(got - ref) <= bound).all(), float(np.abs(got - ref).max())
    empty = np.isneginf(ref_lse)
    assert np.array_equal(empty, np.isneginf(got_lse)) and (got[empty] == 0).all()
    d_lse = np.abs(got_lse[~empty] - ref_lse[~empty])
    assert (d_lse <= dz + 2.0 ** -20 + 2.0 ** -22 * np.abs(ref_lse[~empty])).all()


@pytest.mark.parametrize("typ,fmt", [("f32", "int8"), ("f32", "e4m3"), ("bf16", "int8"), ("f16", "e4m3")])
@pytest.mark.parametrize("q_lens,kv_lens,heads,group,d,block", [
    ([1], [1], 1, 1, 128, 16),
    ([1], [33], 4, 6, 256, 64),
    ([1, 1, 1], [31, 32, 129], 2, 4, 128, 32),
    ([1, 0, 1], [300, 40, 5], 1, 8, 256, 16),        # a sequence without rows
    ([3, 8], [3, 150], 2, 3, 256, 128),
    ([2, 1, 4], [0, 0, 2], 2, 2, 128, 16),           # rows that see nothing
    ([17], [90], 1, 16, 128, 64),
    ([5, 60], [64, 61], 1, 7, 256, 32),
])
def test_attention(cuda, A, q_lens, kv_lens, heads, group, d, block, typ, fmt):
    _attn_case(cuda, A, q_lens, kv_lens, heads, group, d, block, typ, fmt, pad=2)


@pytest.mark.parametrize("typ,fmt", [("f32", "e4m3"), ("bf16", "int8")])
@pytest.mark.parametrize("q_lens,kv_lens", [([4, 1], [70, 7]), ([40], [3]), ([1, 3], [0, 200])])
def test_attention_without_causal_limit(cuda, A, q_lens, kv_lens, typ, fmt):
    """Every row sees every key, whatever the lengths (cross attention)."""
    _attn_case(cuda, A, q_lens, kv_lens, 2, 3, 128, 16, typ, fmt, causal=False)


@pytest.mark.parametrize("typ,fmt,d", [("f32", "int8", 256), ("f16", "e4m3", 128)])
def test_attention_skips_pages_outside_the_pool(cuda, A, typ, fmt, d):
    _attn_case(cuda, A, [1, 2, 1, 30], [100, 64, 17, 90], 2, 2, d, 16, typ, fmt, bad_pages=True)
    _attn_case(cuda, A, [1, 2, 1, 30], [400, 164, 17, 190], 1, 2, d, 64, typ, fmt, bad_pages=True)


@pytest.mark.parametrize("typ,fmt", [("f32", "int8"), ("bf16", "e4m3")])
def test_attention_scales_and_scores_far_apart(cuda, A, typ, fmt):
    """Page scales that differ by a factor of 60, peaked scores, a negative and a zero scale."""
    _attn_case(cuda, A, [1, 3], [500, 333], 1, 4, 128, 16, typ, fmt, spread=30.0)
    _attn_case(cuda, A, [1, 3], [500, 333], 1, 4, 256, 32, typ, fmt, gain=12.0)
    _attn_case(cuda, A, [2], [100], 1, 4, 256, 32, typ, fmt, scale=-0.1)
    _attn_case(cuda, A, [2], [100], 1, 4, 256, 32, typ, fmt, scale=0.0)
    _attn_case(cuda, A, [2], [100], 1, 2, 128, 32, typ, fmt, gain=1e-30)
    if typ == "f32":
        _attn_case(cuda, A, [2], [100], 1, 2, 128, 32, typ, fmt, gain=1e30, scale=1e-31)


def _dense(torch, A, q, cache, table, start, kv_lens, causal):
    """64-bit attention on the GPU, for lengths the loops of the reference take too long for."""
    d, hkv = cache.head_dim, cache.n_head_kv
    group = q.shape[1] // hkv
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for s, kv in enumerate(kv_lens):
        a, b = int(start[s]), int(start[s + 1])
        pg = table[s, :-(-kv // cache.block)].long()
        for h in range(hkv):
            k = (cache.k[pg, h].double() * cache.k_scale[pg, h].double()[:, None, None]).reshape(-1, d)[:kv]
            v = (cache.v[pg, h].double() * cache.v_scale[pg, h].double()[:, None, None]).reshape(-1, d)[:kv]
            z = torch.einsum("igd,jd->igj", q[a:b, h * group:(h + 1) * group].double(), k) * d ** -0.5
            if causal:
                lim = kv - (b - a) + torch.arange(b - a, device="cuda")
                z = z.masked_fill(torch.arange(kv, device="cuda")[None, None, :] > lim[:, None, None], float("-inf"))
            out[a:b, h * group:(h + 1) * group] = torch.softmax(z, -1) @ v
    return out


@pytest.mark.parametrize("typ,fmt", [("f32", "int8"), ("bf16", "e4m3")])
@pytest.mark.parametrize("q_lens,kv_lens,heads,group,d,block", [
    ([1], [40001], 4, 6, 256, 64),                       # one unit over many CTAs
    ([1] * 40, [50 + 97 * i for i in range(40)], 2, 4, 128, 16),
    ([8, 8, 8], [5000, 77, 3001], 4, 6, 256, 64),
    ([700, 1, 129], [2500, 4000, 129], 2, 6, 256, 32),
    ([513], [513], 1, 5, 128, 128),
])
def test_attention_long(cuda, A, q_lens, kv_lens, heads, group, d, block, typ, fmt):
    torch = cuda
    need = [-(-kv // block) for kv in kv_lens]
    cache, kvals, vvals = _pool(torch, A, sum(need), heads, block, d, fmt, seed=sum(kv_lens))
    ids = torch.randperm(sum(need), generator=torch.Generator().manual_seed(1)).to(torch.int32)
    table = torch.zeros(len(need), max(need), dtype=torch.int32)
    at = 0
    for s, m in enumerate(need):
        table[s, :m] = ids[at:at + m]
        at += m
    table = table.cuda()
    start = np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32)
    dt = _dtype(torch, typ)
    q = torch.randn(int(start[-1]), heads * group, d, device="cuda", generator=torch.Generator("cuda").manual_seed(2)).to(dt)
    args = (q, cache, table, torch.tensor(start).cuda(), torch.tensor(kv_lens, dtype=torch.int32).cuda())
    got = A.paged_attn(*args)
    ref = _dense(torch, A, q, cache, table, start, kv_lens, True)
    size = float(q.double().abs().max() * np.abs(kvals).max()) * d ** 0.5  # scale * sum over d of the largest terms
    top = float(np.abs(vvals).max())
    bound = 2 * (size * (2.0 ** -22 + (d / 16 + 2) * 2.0 ** -23) + 2.0 ** -20) * top
    if typ != "f32":
        bound = bound + 2.0 ** -11 * top + ref.abs() * torch.finfo(dt).eps / 2 * 1.001
    assert ((got.double() - ref).abs() <= bound).all()
    # the typical error is far below the worst case: 2-norm of the type's own rounding
    rel = float((got.double() - ref).norm() / ref.norm())
    assert rel <= (1e-5 if typ == "f32" else 5e-3), rel
    # the same call gives the same bits, whatever ran before
    again = A.paged_attn(*args)
    assert torch.equal(got, again)


@pytest.mark.parametrize("typ,fmt", [("f32", "int8"), ("f32", "e4m3"), ("f16", "int8"), ("bf16", "e4m3")])
def test_attention_many_rows_scales_and_pages_far_apart(cuda, A, typ, fmt):
    """What test_attention_scales_and_scores_far_apart asks of few rows, with tiles of 128 rows."""
    _attn_case(cuda, A, [40, 33], [500, 333], 1, 4, 128, 16, typ, fmt, spread=30.0)
    _attn_case(cuda, A, [40, 33], [500, 333], 1, 4, 256, 32, typ, fmt, gain=12.0)
    _attn_case(cuda, A, [50], [100], 1, 4, 256, 32, typ, fmt, scale=-0.1)
    _attn_case(cuda, A, [50], [100], 1, 4, 128, 64, typ, fmt, scale=0.0)
    _attn_case(cuda, A, [50], [100], 1, 3, 256, 128, typ, fmt, gain=1e-30)
    _attn_case(cuda, A, [70, 1, 90], [1100, 700, 90], 1, 2, 256, 16, typ, fmt, bad_pages=True)
    if typ == "f32":
        _attn_case(cuda, A, [50], [100], 1, 2, 128, 32, typ, fmt, gain=1e30, scale=1e-31)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("typ,fmt,q_lens", [("f32", "int8", [1, 2]), ("bf16", "e4m3", [1, 2]), ("f32", "e4m3", [60, 30]), ("f16", "int8", [60, 30])])
def test_attention_with_tables_shorter_than_the_lengths(cuda, A, typ, fmt, q_lens, causal):
    """A row's limit goes by kv_len; keys in blocks that the table does not have are not seen."""
    torch = cuda
    dt = _dtype(torch, typ)
    for block, cols, heads in ((16, 5, 1), (32, 3, 2), (64, 1, 2)):
        cache, kv, vv = _pool(torch, A, 2 * cols, heads, block, 128, fmt, seed=8)
        table = torch.randperm(2 * cols, generator=torch.Generator().manual_seed(3)).to(torch.int32).view(2, cols)
        lens = [block * cols + 7, 2 ** 31 - 1]
        start = np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32)
        q = torch.randn(int(start[-1]), 3 * heads, 128, generator=torch.Generator().manual_seed(4)).to(dt).cuda()
        out, lse = torch.empty_like(q), torch.empty(q.shape[:2], device="cuda")
        A.paged_attn(q, cache, table.cuda(), torch.tensor(start).cuda(), torch.tensor(lens, dtype=torch.int32).cuda(),
                     causal=causal, out=out, lse=lse)
        ref = R.paged_attn(_np(q), kv, vv, table.numpy(), start, lens, 128 ** -0.5, causal)
        _check_attn(torch, out, lse, ref, start, vv, 128, typ)


@pytest.mark.parametrize("typ,fmt,d", [("f32", "int8", 256), ("f32", "e4m3", 128), ("bf16", "e4m3", 256)])
def test_attention_one_row_each_with_pages_outside_the_pool(cuda, A, typ, fmt, d):
    for block in (16, 32, 128):
        _attn_case(cuda, A, [1, 1, 1, 1], [400, 164, 17, 290], 1, 2, d, block, typ, fmt, bad_pages=True)


@pytest.mark.parametrize("typ,fmt,q_lens", [("f32", "int8", [1, 1]), ("bf16", "int8", [1, 1]), ("f32", "int8", [40, 9]), ("f16", "e4m3", [40, 9])])
def test_attention_of_unaligned_views(cuda, A, typ, fmt, q_lens):
    """Rows that begin off 16-byte boundaries give what aligned ones give."""
    torch = cuda
    dt = _dtype(torch, typ)
    cache, _, _ = _pool(torch, A, 12, 2, 32, 128, fmt, seed=3)
    table = torch.arange(12, dtype=torch.int32, device="cuda").view(2, 6)
    if max(q_lens) > 1:
        table = torch.cat([table, _no_pages(torch, 2)], 1)
    start = torch.tensor([0, q_lens[0], sum(q_lens)], dtype=torch.int32, device="cuda")
    kv = torch.tensor([190, 77], dtype=torch.int32, device="cuda")
    t = sum(q_lens)
    buf = torch.randn(t, 4 * 128 + 3, device="cuda").to(dt)
    view = buf[:, 1:1 + 512].unflatten(-1, (4, 128))
    to = torch.full((t, 4 * 128 + 3), 7.0, dtype=dt, device="cuda")
    A.paged_attn(view, cache, table, start, kv, out=to[:, 1:513].unflatten(-1, (4, 128)))
    want = A.paged_attn(view.contiguous(), cache, table, start, kv)
    assert torch.equal(to[:, 1:513].unflatten(-1, (4, 128)), want)
    assert (to[:, 0] == 7).all() and (to[:, 513:] == 7).all()


@pytest.mark.parametrize("q_len", [1, 24])
def test_attention_with_pages_of_scale_zero(cuda, A, q_len):
    """A page of zeros has scale 0: its keys score 0 and its values add nothing."""
    torch = cuda
    cache, kvals, vvals = _pool(torch, A, 4, 1, 32, 128, "int8", seed=9)
    cache.k_scale[2] = 0
    cache.v_scale[2] = 0
    q = torch.randn(q_len, 4, 128, device="cuda")
    for order in ([0, 1, 2, 3], [2, 0, 1, 3], [2]):
        table = torch.cat([torch.tensor([order], dtype=torch.int32, device="cuda"), _no_pages(torch, 1)], 1)
        kv = 32 * len(order) - 3
        args = (q, cache, table, torch.tensor([0, q_len], dtype=torch.int32).cuda(), torch.tensor([kv], dtype=torch.int32).cuda())
        got = A.paged_attn(*args)
        ref = _dense(torch, A, q, cache, table, [0, q_len], [kv], True)
        size = float(q.double().abs().max() * np.abs(kvals).max()) * 128 ** 0.5
        assert ((got.double() - ref).abs() <= 2 * (size * (2.0 ** -22 + 10 * 2.0 ** -23) + 2.0 ** -20) * np.abs(vvals).max()).all()


@pytest.mark.parametrize("q_len", [1, 8])
def test_attention_of_1024_requests(cuda, A, q_len):
    torch = cuda
    n = 1024
    cache, kvals, vvals = _pool(torch, A, 64, 2, 16, 128, "int8", seed=4)
    g = torch.Generator().manual_seed(5)
    kv = torch.randint(q_len, 100, (n,), generator=g).to(torch.int32)
    table = torch.randint(0, 64, (n, 7), generator=g).to(torch.int32).cuda()  # requests share pages
    start = torch.arange(n + 1, dtype=torch.int32, device="cuda") * q_len
    q = torch.randn(n * q_len, 6, 128, generator=g).cuda()
    got = A.paged_attn(q, cache, table, start, kv.cuda())
    ref = _dense(torch, A, q, cache, table, start.tolist(), kv.tolist(), True)
    size = float(q.double().abs().max() * np.abs(kvals).max()) * 128 ** 0.5
    assert ((got.double() - ref).abs() <= 2 * (size * (2.0 ** -22 + 10 * 2.0 ** -23) + 2.0 ** -20) * np.abs(vvals).max()).all()
    with pytest.raises(Exception):
        A.paged_attn(q, cache, torch.zeros(1025, 7, dtype=torch.int32, device="cuda"),
                     torch.zeros(1026, dtype=torch.int32, device="cuda"), torch.zeros(1025, dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("n,q_len,kv,d", [(60, 1, 60000, 128), (30, 1, 60000, 256), (40, 8, 20000, 128), (40, 8, 20000, 256)])
def test_long_sums_do_not_drift(cuda, A, fmt, n, q_len, kv, d):
    """All values positive: a sum that is cut off, not rounded, at each step falls short step by step. With V in
    [0.5, 1] and equal weights a sum grows steadily, a step of 16 keys cuts less than 2^-23 of it, and over the
    at most 128 steps between two flushes that is 128 * 2^-23 / 2 = 7.6e-6 of what the sum has become, plus 2^-20
    for exponentials, terms of P and joins: 8.6e-6 at most. Unflushed, the expected shortfall of a share of 750
    or 2500 steps is 1.6e-5 or 5e-5 (half of 2^-24 .. 2^-23 a step)."""
    torch = cuda
    block, heads, group = 64, 4, 6
    pages = -(-kv // block)
    cache = A.KvCache.empty(pages, heads, d, block, FMT[fmt])
    g = torch.Generator("cuda").manual_seed(6)
    x = torch.randint(64, 128, cache.v.shape, generator=g, device="cuda")
    cache.v.copy_(x if fmt == "int8" else (x // 8).float())  # (8 to 15 are e4m3 values)
    cache.v_scale.fill_(1.0 / 128 if fmt == "int8" else 1.0 / 16)
    cache.k.zero_()
    cache.k_scale.fill_(1.0)
    table = torch.arange(pages, dtype=torch.int32, device="cuda").repeat(n, 1)  # all read the same pages
    start = torch.arange(n + 1, dtype=torch.int32, device="cuda") * q_len
    lens = torch.full((n,), kv, dtype=torch.int32, device="cuda")
    q = torch.randn(n * q_len, heads * group, d, generator=g, device="cuda")
    got = A.paged_attn(q, cache, table, start, lens, causal=False)
    v = (cache.v.float() * cache.v_scale[0, 0]).double().transpose(0, 1).reshape(heads, -1, d)[:, :kv].mean(1)
    ref = v.repeat_interleave(group, 0)
    assert float((got.double() / ref - 1).abs().max()) <= 8.6e-6


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("q_len,wide", [(2, False), (60, True)])
def test_attention_rows_with_nan_and_infinity_spoil_no_others(cuda, A, typ, q_len, wide):
    torch = cuda
    dt = _dtype(torch, typ)
    cache, _, _ = _pool(torch, A, 40, 2, 32, 128, "int8", seed=7)
    table = torch.arange(40, dtype=torch.int32, device="cuda").view(1, 40)
    if wide:  # the kernel for many rows
        table = torch.cat([table, _no_pages(torch, 1)], 1)
    start, kv = torch.tensor([0, q_len], dtype=torch.int32).cuda(), torch.tensor([1270], dtype=torch.int32).cuda()
    q = torch.randn(q_len, 8, 128, device="cuda").to(dt)
    clean = A.paged_attn(q, cache, table, start, kv)
    bad = q.clone()
    bad[0, 1, 5] = float("nan")
    bad[1, 6, 7] = float("inf")
    got = A.paged_attn(bad, cache, table, start, kv)
    keep = torch.ones(q_len, 8, dtype=torch.bool, device="cuda")
    keep[0, 1] = keep[1, 6] = False
    assert torch.equal(got[keep], clean[keep])
    assert not torch.isfinite(got[0, 1]).any()


def test_attention_in_a_graph_and_on_another_stream(cuda, A):
    """Captured with its lengths on the device, replayed after they changed; two graphs replayed side by side."""
    torch = cuda
    cache, _, _ = _pool(torch, A, 40, 2, 32, 128, "int8")
    graphs, outs, lens, qs = [], [], [], []
    table = torch.randperm(40, generator=torch.Generator().manual_seed(0)).to(torch.int32).view(2, 20).cuda()
    for i in range(2):
        q = torch.randn(2, 8, 128, device="cuda")
        start, kv = torch.tensor([0, 1, 2], dtype=torch.int32).cuda(), torch.tensor([640, 100 + i], dtype=torch.int32).cuda()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            A.paged_attn(q, cache, table, start, kv)
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out = A.paged_attn(q, cache, table, start, kv)
        graphs.append((g, s, start)), outs.append(out), lens.append(kv), qs.append(q)
    for step in range(3):
        for i in range(2):
            lens[i].copy_(torch.tensor([640 - 200 * step, 30 + 100 * i], dtype=torch.int32))
        torch.cuda.synchronize()
        for _ in range(20):
            for g, s, _ in graphs:
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for i in range(2):
            want = A.paged_attn(qs[i], cache, table, graphs[i][2], lens[i])
            assert torch.equal(outs[i], want)
    del graphs


@pytest.mark.parametrize("fmt,typ,block", [("int8", "f32", 16), ("e4m3", "bf16", 32)])
def test_the_operators_together(cuda, A, fmt, typ, block):
    """Two requests prefilled and decoded through slots -> rope -> append -> attention, against dense attention over
    the cache's own values, with the keys checked against what was appended."""
    torch = cuda
    dt = _dtype(torch, typ)
    heads, group, d, width = 2, 3, 128, 8
    cache = A.KvCache.empty(20, heads, d, block, FMT[fmt])
    table = torch.full((2, width), -1, dtype=torch.int32, device="cuda")
    free = torch.randperm(20, generator=torch.Generator().manual_seed(5)).to(torch.int32).cuda()
    taken, ctx = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    freqs = A.Rope(64, A.ROPE_HALF, base=1e6)
    g = torch.Generator("cuda").manual_seed(1)
    kept = [torch.zeros(0, heads, d, device="cuda") for _ in range(2)]
    for new in ([37, 5], [1, 1], [1, 1], [4, 0], [1, 1], [2, 3]):
        t = sum(new) + 3  # a padded batch
        q, k, v = (torch.randn(t, h, d, device="cuda", generator=g).to(dt) for h in (heads * group, heads, heads))
        add = torch.tensor(new, dtype=torch.int32).cuda()
        s = A.kv_slots(ctx, add, table, free, taken, block=block, n_rows=t)
        q, k = A.rope(freqs, [q, k], s.pos)
        A.kv_append(cache, k, v, s.slot)
        out = A.paged_attn(q, cache, table, s.seq_start, s.kv_len)
        ctx.add_(add)
        start = np.concatenate([[0], np.cumsum(new)])
        for r in range(2):
            kept[r] = torch.cat([kept[r], k[start[r]:start[r + 1]].float()])
        lens = ctx.tolist()
        assert s.kv_len.tolist() == lens
        ref = _dense(torch, A, q, cache, table, start, lens, True)[:start[-1]]
        rel = float((out[:start[-1]].double() - ref).norm() / ref.norm())
        assert rel <= (1e-5 if typ == "f32" else 5e-3)
        for r in range(2):  # the cache holds the rotated keys to within a step per recoding
            slots = torch.tensor([int(table[r, p // block]) * block + p % block for p in range(lens[r])]).cuda()
            got = A.kv_gather(cache, slots)[0]
            # int8: half a step of the page's largest value per coding; e4m3: 2^-4 of the value; a few recodings
            step = kept[r].abs().max() / 127 if fmt == "int8" else kept[r].abs() / 16 + kept[r].abs().max() * 2.0 ** -16
            assert ((got - kept[r]).abs() <= 4 * step).all()
    assert int(taken[0]) == sum(-(-n // block) for n in ctx.tolist())
