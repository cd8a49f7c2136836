"""The range of the attention weights (paged_attn): rows whose keys' weights or pages' v_scales lie far apart.

Each row is held against its own terms, not against the pool's largest value. With p_j a row's softmax weights,
s_j its pages' v_scales and c_j the codes, an element of the output may be off by
  2 (dz + 2^-20) sum p_j s_j |c_j|     a relative error of at most dz + 2^-20 in each weight (dz: a score's error, as in
                                       test_gpu_attn.py; 2^-20: exponential and the weight's two fp16 terms)
  + steps 2^-23 sum p_j s_j |c_j|      sums that are cut off at each accumulation step of 16 keys, twice with two terms,
                                       and flushed after at most 128 (fp32)
  + 2^-30 max(p_j s_j) sum |c_j|       a weight is not held finer than that
  + 2^-11 sum p_j s_j |c_j| + eps/2    16-bit types: one fp16 term, and the output's rounding
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

FMT = {"int8": 0, "e4m3": 1}


@pytest.fixture
def A(cuda):
    from codpiece_b200 import attn
    return attn


def _cache(torch, A, pages, heads, block, d, fmt, seed):
    """Codes of any size (e4m3: 8-bit floats up to 240), one K scale; V scales to be set by the test."""
    g = torch.Generator("cuda").manual_seed(seed)
    c = A.KvCache.empty(pages, heads, d, block, FMT[fmt])
    for codes in (c.k, c.v):
        x = torch.randint(-100, 101, codes.shape, generator=g, device="cuda")
        codes.copy_(x if fmt == "int8" else x.float())
    c.k_scale.fill_(0.02)
    c.v_scale.fill_(0.02)
    return c


def _run(torch, A, q, cache, table, kv, wide, causal=True, times=1):
    """One sequence (the same several times) whose pages are table [n]; wide: the kernel for many rows."""
    n = q.shape[0]
    tab = table.view(1, -1).repeat(times, 1)
    if wide:
        tab = torch.cat([tab, torch.full((times, 12000), -1, dtype=torch.int32, device="cuda")], 1)
    out, lse = A.paged_attn(q.repeat(times, 1, 1), cache, tab, n * torch.arange(times + 1, dtype=torch.int32, device="cuda"),
                            torch.full((times,), kv, dtype=torch.int32, device="cuda"), causal=causal, return_lse=True)
    return out, lse


def _check(torch, q, cache, table, kv, got, lse, causal=True):
    n, hq, d = q.shape
    hkv, b = cache.n_head_kv, cache.block
    pg = table[:-(-kv // b)].long()
    worst = 0.0
    for h in range(hkv):
        flat = lambda t: t[pg, h].double().reshape(-1, d)[:kv]  # noqa: E731
        k = flat(cache.k) * float(cache.k_scale[0, 0])
        c = flat(cache.v)
        s = cache.v_scale[pg, h].double().repeat_interleave(b)[:kv]
        for i0 in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
            x = q[:, i0].double()
            z = (x @ k.T) * d ** -0.5
            size = float((x.abs() @ k.abs().T).max()) * d ** -0.5
            if causal:
                lim = kv - n + torch.arange(n, device="cuda")
                z = z.masked_fill(torch.arange(kv, device="cuda")[None, :] > lim[:, None], float("-inf"))
            w = torch.softmax(z, -1) * s[None, :]
            ref, terms = w @ c, w @ c.abs()
            dz = size * (2.0 ** -22 + (d / 16 + 2) * 2.0 ** -23)
            steps = min(128, -(-kv // 16) * 2) if q.dtype == torch.float32 else -(-kv // 16)
            bound = (2 * (dz + 2.0 ** -20) + steps * 2.0 ** -23) * terms
            bound = bound + 2.0 ** -30 * w.amax(-1, keepdim=True) * c.abs().sum(0)[None, :]
            if q.dtype != torch.float32:
                bound = bound + 2.0 ** -11 * terms + ref.abs() * torch.finfo(q.dtype).eps / 2 * 1.001
            if q.dtype == torch.float16:
                bound = bound + 2.0 ** -25  # half a step of its subnormal numbers
            err = (got[:, i0].double() - ref).abs()
            assert torch.isfinite(got[:, i0]).all()
            worst = max(worst, float((err / bound.clamp(min=1e-300)).nan_to_num(0.0).max()))
            assert (err <= bound).all(), (i0, float((err / bound).nan_to_num(0.0).max()))
            ref_lse = torch.logsumexp(z, -1)
            assert ((lse[:, i0].double() - ref_lse).abs() <= dz + 2.0 ** -20 + 2.0 ** -22 * ref_lse.abs()).all()
    return worst


@pytest.mark.parametrize("typ,fmt", [("f32", "int8"), ("f32", "e4m3"), ("bf16", "int8"), ("f16", "e4m3")])
@pytest.mark.parametrize("n,wide", [(1, False), (3, False), (40, True)])
@pytest.mark.parametrize("ratio", [1e-8, 1e-4, 1e4, 1e6, 1e8, 1e16])
def test_pages_of_other_scales_that_carry_no_weight(cuda, A, typ, fmt, n, wide, ratio):
    """One page (the first, a middle one, the last) has another v_scale than the rest, and scores so low that its keys
    weigh e^-60 of the others; the last page is also beyond the causal limit of some rows. What the others add keeps
    its bits."""
    torch = cuda
    if typ == "f16" and ratio > 1:
        ratio = 1 / ratio  # (its outputs end at 65504)
    dt = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[typ]
    for block, d in ((16, 128), (64, 256)):
        pages = 12 if block == 16 else 6
        kv = pages * block - 3
        for where in (0, pages // 2, pages - 1):
            cache = _cache(torch, A, pages, 2, block, d, fmt, seed=3)
            table = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).to(torch.int32).cuda()
            cache.k[..., 0] = 0
            cache.k[int(table[where]), :, :, 0] = -64
            cache.v_scale[int(table[where])] = 0.02 * ratio
            q = torch.randn(n, 4, d, generator=torch.Generator("cuda").manual_seed(2), device="cuda")
            q[..., 0] = 60 / (64 * 0.02 * d ** -0.5)
            q = q.to(dt)
            out, lse = _run(torch, A, q, cache, table, kv, wide)
            _check(torch, q, cache, table, kv, out, lse)


@pytest.mark.parametrize("typ,fmt", [("f32", "int8"), ("bf16", "e4m3")])
@pytest.mark.parametrize("n,wide", [(3, False), (40, True)])
@pytest.mark.parametrize("ratio", [2.0 ** 10, 2.0 ** 20, 2.0 ** 40])
def test_rows_next_to_a_page_they_do_not_see(cuda, A, typ, fmt, n, wide, ratio):
    """The last page's v_scale is far above the rest; the rows before it do not see it, the last ones do. No score is
    large here, so the bound is tight."""
    torch = cuda
    dt = {"f32": torch.float32, "bf16": torch.bfloat16}[typ]
    for d in (128, 256):
        kv = 16 * 6 + 2
        cache = _cache(torch, A, 7, 2, 16, d, fmt, seed=5)
        table = torch.tensor([3, 1, 0, 6, 2, 5, 4], dtype=torch.int32).cuda()
        cache.v_scale[4] = 0.02 * ratio
        q = (0.3 * torch.randn(n, 4, d, generator=torch.Generator("cuda").manual_seed(6), device="cuda")).to(dt)
        out, lse = _run(torch, A, q, cache, table, kv, wide)
        _check(torch, q, cache, table, kv, out, lse)


@pytest.mark.parametrize("typ,fmt", [("f32", "int8"), ("bf16", "e4m3")])
@pytest.mark.parametrize("n,wide", [(1, False), (20, True)])
def test_many_small_weights_beside_a_large_one(cuda, A, typ, fmt, n, wide):
    """The first key has nearly all of the weight and values of zero; the output is what 20000 equal small weights add,
    so that their rounding does not average out. Many sequences, so that one CTA takes a row's keys from the first on."""
    torch = cuda
    dt = {"f32": torch.float32, "bf16": torch.bfloat16}[typ]
    kv, block, d = 20000, 64, 128
    pages = -(-kv // block)
    for nats in (8.3, 11.1, 12.4, 13.7):
        cache = _cache(torch, A, pages, 1, block, d, fmt, seed=7)
        g = torch.Generator("cuda").manual_seed(8)
        x = torch.randint(4, 8, cache.v.shape, generator=g, device="cuda") * 8
        cache.v.copy_(x if fmt == "int8" else x.float())
        cache.k.zero_()
        cache.k[0, 0, 0, 0] = 64
        cache.v[0, 0, 0] = 0
        table = torch.arange(pages, dtype=torch.int32, device="cuda")
        q = torch.zeros(n, 2, d, device="cuda")
        q[..., 0] = nats / (64 * 0.02 * d ** -0.5)
        q = q.to(dt)
        out, lse = _run(torch, A, q, cache, table, kv, wide, causal=False, times=160)
        for i in (0, 1, 77, 159):
            _check(torch, q, cache, table, kv, out[i * n:(i + 1) * n], lse[i * n:(i + 1) * n], causal=False)


@pytest.mark.parametrize("n,wide", [(1, False), (40, True)])
def test_scales_at_the_ends_of_the_range_stay_finite(cuda, A, n, wide):
    """Pages of zeros first, then the smallest and the largest scales that values can have: no row overflows."""
    torch = cuda
    for order in ([0.0, 1e-30, 1e30], [1e30, 0.0, 1e-30], [1e-30, 1e30, 0.0], [0.0, 0.0, 1e-30], [0.0, 1.0, 1e34]):
        cache = _cache(torch, A, 6, 1, 32, 128, "int8", seed=9)
        for i in range(6):
            cache.v_scale[i] = order[i // 2]
        table = torch.arange(6, dtype=torch.int32, device="cuda")
        q = torch.randn(n, 2, 128, generator=torch.Generator("cuda").manual_seed(10), device="cuda")
        out, lse = _run(torch, A, q, cache, table, 190, wide)
        _check(torch, q, cache, table, 190, out, lse)  # (keys of all pages weigh alike)


@pytest.mark.parametrize("typ", ["f32", "bf16"])
@pytest.mark.parametrize("n,wide", [(2, False), (40, True)])
def test_scores_of_any_size(cuda, A, typ, n, wide):
    """Scores of some 10^8, whole numbers apart by thousands: each row's output is its best key's value."""
    torch = cuda
    dt = {"f32": torch.float32, "bf16": torch.bfloat16}[typ]
    cache = _cache(torch, A, 12, 1, 32, 128, "int8", seed=11)
    cache.k.zero_()
    g = torch.Generator("cuda").manual_seed(12)
    order = torch.randperm(32 * 12, generator=torch.Generator().manual_seed(13)).cuda()
    places = cache.k.view(12 * 32, 128)
    places[:, 0] = 100
    places[:, 1] = (order % 100).to(torch.int8)
    places[:, 2] = (order // 100).to(torch.int8)
    cache.k_scale.fill_(1.0)
    cache.v_scale.fill_(2.0 ** -6)
    table = torch.arange(12, dtype=torch.int32, device="cuda")
    q = torch.zeros(n, 2, 128, device="cuda")
    q[..., 0], q[..., 1], q[..., 2] = 2.0 ** 20, 2.0 ** 13, 100 * 2.0 ** 13
    q[:, 1] = -q[:, 1]
    kv = 380
    out, lse = A.paged_attn(q.to(dt), cache, torch.cat([table.view(1, -1), torch.full((1, 12000), -1, dtype=torch.int32, device="cuda")], 1) if wide else table.view(1, -1),
                            torch.tensor([0, n], dtype=torch.int32, device="cuda"),
                            torch.tensor([kv], dtype=torch.int32, device="cuda"), scale=1.0, causal=False, return_lse=True)
    v = cache.v.view(12 * 32, 128)[:kv].float() * 2.0 ** -6
    x = q.to(dt).double()
    z = torch.einsum("ihd,jd->ihj", x, cache.k.view(12 * 32, 128)[:kv].double())
    first, second = torch.topk(z, 2, dim=-1).values.unbind(-1)
    assert float((first - second).min()) > 2000 and float(z.abs().max()) > 1e8
    want = v[z.argmax(-1)]
    assert ((out.float() - want).abs() <= want.abs() * (2.0 ** -20 if typ == "f32" else 2.0 ** -8)).all()
    assert ((lse.double() - first).abs() <= first.abs() * 2.0 ** -21).all()
