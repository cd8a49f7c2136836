"""The attention core without a GPU: what cpq_rope_*, cpq_kv_* and cpq_paged_attn refuse before any device work,
and the 64-bit reference (oracle/attn_ref.py) against closed forms."""
import ctypes as C
import math

import numpy as np
import pytest

from oracle import attn_ref as R

F32, F16, BF16 = 0, 1, 30
OK, INVALID, UNSUPPORTED, NOT_INIT, WORKSPACE = 0, 1, 2, 3, 4


@pytest.fixture(scope="module")
def L():
    from codpiece_b200 import _lib, build
    build.build()
    return _lib.lib()


def tensor(d, heads, tokens, typ=F32, data=0x10000, row=None, tok=None):
    from codpiece_b200._lib import CpqTensor
    b = 4 if typ == F32 else 2
    t = CpqTensor()
    t.type = typ
    t.ne[:] = [d, heads, tokens, 1]
    row = d * b if row is None else row
    tok = heads * row if tok is None else tok
    t.nb[:] = [b, row, tok, tok * max(tokens, 1)]
    t.data = data
    return t


def cache(fmt=0, d=256, heads=4, block=64, pages=10, k=0x100000, v=0x200000, ks=0x300000, vs=0x400000):
    from codpiece_b200._lib import CpqKvCache
    return CpqKvCache(fmt, d, heads, block, pages, k, v, ks, vs)


def arr(*ts):
    from codpiece_b200._lib import CpqTensor
    return (C.POINTER(CpqTensor) * len(ts))(*[C.pointer(t) for t in ts])


def rope_params(n_dims=64, mode=1, base=1e4, freq_scale=1.0, ext=0.0, attn=1.0, bf=32.0, bs=1.0, n_ctx=0, ff=None):
    from codpiece_b200._lib import CpqRopeParams
    return CpqRopeParams(n_dims, mode, base, freq_scale, ext, attn, bf, bs, n_ctx, ff)


def test_rope_create_refuses(L):
    h = C.c_void_p()
    make = lambda **k: L.cpq_rope_create(C.byref(rope_params(**k)), C.byref(h))  # noqa: E731
    assert make() == OK and h.value
    L.cpq_rope_destroy(h)
    for bad in ({"n_dims": 0}, {"n_dims": 63}, {"n_dims": -2}, {"mode": 2}, {"base": 0.0}, {"base": float("nan")},
                {"base": float("inf")}, {"freq_scale": 0.0}, {"freq_scale": -1.0}, {"ext": float("nan")},
                {"attn": float("inf")}, {"ext": 1.0}, {"ext": 1.0, "n_ctx": 4096, "base": 1.0},
                {"ext": 1.0, "n_ctx": 4096, "bf": 0.0}, {"ff": (C.c_double * 32)(*([1.0] * 31 + [0.0]))}):
        assert make(**bad) == INVALID, bad
        assert not h.value
    assert make(n_dims=258) == UNSUPPORTED
    assert L.cpq_rope_create(None, C.byref(h)) == INVALID
    assert L.cpq_rope_create(C.byref(rope_params()), None) == INVALID
    L.cpq_rope_destroy(None)


def test_rope_apply_refuses(L):
    h = C.c_void_p()
    assert L.cpq_rope_create(C.byref(rope_params(n_dims=64)), C.byref(h)) == OK
    pos = C.c_void_p(0x9000)

    def call(x, y, n=1, p=pos, table=h):
        return L.cpq_rope_apply(table, arr(*x), arr(*y), n, p, None)

    a, b = tensor(128, 4, 3), tensor(128, 4, 3, data=0x20000)
    assert call([a], [b], table=None) == INVALID
    assert call([a], [b], n=0) == INVALID
    assert call([a] * 5, [b] * 5, n=5) == INVALID
    assert call([a], [b], p=None) == INVALID
    assert call([a], [tensor(128, 4, 2)]) == INVALID                      # shapes
    assert call([a], [tensor(128, 4, 3, BF16)]) == INVALID                # types
    assert call([tensor(128, 4, 3, 8)], [b]) == INVALID                   # Q8_0
    assert call([tensor(128, 4, 3, data=0)], [b]) == INVALID
    assert call([a, tensor(128, 4, 5)], [b, tensor(128, 4, 5)], n=2) == INVALID  # token counts
    assert call([tensor(32, 4, 3)], [tensor(32, 4, 3)]) == INVALID        # n_dims > D
    assert call([tensor(128, 4, 3, row=513)], [b]) == INVALID             # not whole elements
    assert call([a], [tensor(128, 4, 3, tok=4096)]) == INVALID            # in place, other strides
    assert call([tensor(8192, 1, 3)], [tensor(8192, 1, 3, data=0x90000)]) == UNSUPPORTED
    assert call([tensor(128, 4, 0)], [tensor(128, 4, 0)], p=None) == OK   # no tokens
    L.cpq_rope_destroy(h)
    assert L.cpq_rope_create(C.byref(rope_params(n_dims=64, mode=0)), C.byref(h)) == OK
    odd = tensor(67, 1, 3)
    assert call([odd], [odd], table=h) == UNSUPPORTED                     # interleaved pairs of an odd head
    L.cpq_rope_destroy(h)


def test_kv_slots_refuses(L):
    from codpiece_b200._lib import CpqKvSlotArgs

    def args(**k):
        f = dict(ctx_len=0x10, new_len=0x20, n_seqs=2, table=0x30, table_stride=4, max_blocks=4, block=16, free_pages=0x40,
                 n_free=3, taken=0x50, taken_out=0x60, seq_start=0x70, kv_len=0x80, pos=0x90, slot=0xa0, n_rows=5)
        f.update(k)
        a = CpqKvSlotArgs()
        for name, v in f.items():
            setattr(a, name, v)
        return L.cpq_kv_slots(C.byref(a), None)

    assert L.cpq_kv_slots(None, None) == INVALID
    for bad in ({"n_seqs": -1}, {"n_rows": -1}, {"n_free": -1}, {"max_blocks": -1}, {"table_stride": 3}, {"n_rows": 1 << 31}):
        assert args(**bad) == INVALID, bad
    for name in ("ctx_len", "new_len", "table", "free_pages", "taken", "taken_out", "seq_start", "kv_len", "pos", "slot"):
        assert args(**{name: None}) == INVALID, name
    for b in (0, 8, 48, 256):
        assert args(block=b) == UNSUPPORTED


def test_append_and_gather_refuse(L):
    slot = C.c_void_p(0x5000)

    def append(c=None, k=None, v=None, s=slot):
        c, k, v = c or cache(), k or tensor(256, 4, 3), v or tensor(256, 4, 3, data=0x20000)
        rc = L.cpq_kv_append(C.byref(c), C.byref(k), C.byref(v), s, None)
        assert L.cpq_kv_gather(C.byref(c), s, C.byref(k), C.byref(v), None) == rc
        return rc

    assert L.cpq_kv_append(None, C.byref(tensor(256, 4, 3)), C.byref(tensor(256, 4, 3)), slot, None) == INVALID
    for bad in ({"fmt": 2}, {"pages": 0}, {"heads": 0}, {"k": None}, {"v": None}, {"ks": None}, {"vs": None}):
        assert append(cache(**bad)) == INVALID, bad
    for bad in ({"d": 64}, {"d": 192}, {"block": 8}, {"block": 256}, {"k": 0x100040}):
        assert append(cache(**bad)) == UNSUPPORTED, bad
    assert append(k=tensor(128, 4, 3)) == INVALID
    assert append(k=tensor(256, 3, 3)) == INVALID
    assert append(v=tensor(256, 4, 4)) == INVALID
    assert append(v=tensor(256, 4, 3, F16)) == INVALID
    assert append(k=tensor(256, 4, 3, 8)) == INVALID
    assert append(s=None) == INVALID
    assert append(k=tensor(256, 4, 0), v=tensor(256, 4, 0), s=None) == OK


def test_paged_attn_refuses(L):
    from codpiece_b200._lib import CpqAttnSeqs
    big = 1 << 30

    def call(q=None, c=None, out=None, seqs=None, scale=0.1, ws=0x80000, n_ws=big, **k):
        q, c = q or tensor(256, 24, 3), c or cache()
        out = out or tensor(256, 24, 3, q.type, data=0x30000)
        f = dict(seq_start=0x10, kv_len=0x20, table=0x30, table_stride=8, n_seqs=2, max_blocks=8)
        f.update(k)
        s = CpqAttnSeqs()
        for name, v in f.items():
            setattr(s, name, v)
        return L.cpq_paged_attn(C.byref(q), C.byref(c), None if seqs == "none" else C.byref(s), scale, 1, C.byref(out), None,
                                ws, n_ws, None)

    assert call(seqs="none") == INVALID
    assert call(q=tensor(128, 24, 3), out=tensor(128, 24, 3)) == INVALID          # head size
    assert call(q=tensor(256, 23, 3), out=tensor(256, 23, 3)) == INVALID          # heads not a multiple
    assert call(out=tensor(256, 24, 4)) == INVALID
    assert call(out=tensor(256, 24, 3, BF16)) == INVALID
    assert call(q=tensor(256, 24, 3, 8)) == INVALID
    assert call(scale=float("nan")) == INVALID and call(scale=float("inf")) == INVALID
    assert call(n_seqs=-1) == INVALID and call(max_blocks=-1) == INVALID and call(table_stride=7) == INVALID
    assert call(n_seqs=1025) == UNSUPPORTED
    for name in ("seq_start", "kv_len", "table"):
        assert call(**{name: None}) == INVALID, name
    assert call(c=cache(block=12)) == UNSUPPORTED
    assert call(c=cache(pages=1 << 30)) == UNSUPPORTED                           # cache rows past 31 bits
    assert call(max_blocks=1 << 26, table_stride=1 << 26) == UNSUPPORTED          # keys past 31 bits
    assert call(q=tensor(256, 24, 1 << 20), out=tensor(256, 24, 1 << 20), max_blocks=1 << 20, table_stride=1 << 20) == UNSUPPORTED
    assert call(ws=None) == NOT_INIT
    assert call(n_ws=1000) == WORKSPACE and call(ws=0x80010) == WORKSPACE
    assert call(q=tensor(256, 24, 0), out=tensor(256, 24, 0)) == OK               # no tokens
    assert call(n_seqs=0) == OK
    assert L.cpq_paged_attn_workspace_size(None, None, 1) == 0


def test_python_surface_refuses_cpu_tensors():
    import torch

    from codpiece_b200 import attn
    with pytest.raises(TypeError):
        attn.KvCache.wrap(torch.zeros(1, 1, 16, 128, dtype=torch.int8), torch.zeros(1, 1, 16, 128, dtype=torch.int8),
                          torch.zeros(1, 1), torch.zeros(1, 1))
    with pytest.raises(ValueError):
        attn.Rope(64, freq_factors=[1.0] * 31)
    with pytest.raises(TypeError):
        attn.rope(attn.Rope(64), [torch.zeros(2, 1, 64)], torch.zeros(2, dtype=torch.int32))
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(TypeError):
        attn.kv_slots(i, i, torch.zeros(1, 1, dtype=torch.int32), i, i, block=16, n_rows=1)


# ---- the reference itself -------------------------------------------------------------------


def test_reference_rope_is_a_rotation_and_adds_up():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((4, 2, 16))
    for half in (False, True):
        y = R.rope(x, [0, 1, 2, 3], 12, half)
        assert np.allclose(y[0], x[0]) and np.array_equal(y[..., 12:], x[..., 12:])
        assert np.allclose(np.linalg.norm(y, axis=-1), np.linalg.norm(x, axis=-1))
        z = R.rope(R.rope(x, [3] * 4, 12, half), [4] * 4, 12, half)
        assert np.allclose(z, R.rope(x, [7] * 4, 12, half))
    w, m = R.rope_frequencies(64, base=1e4, freq_scale=0.25, ext_factor=1.0, n_ctx_orig=4096)
    plain, _ = R.rope_frequencies(64, base=1e4)
    assert math.isclose(m, 1 + 0.1 * math.log(4))
    assert math.isclose(w[0], plain[0]) and math.isclose(w[-1], plain[-1] / 4)  # fast pairs keep, slow pairs scale


def test_reference_codes():
    import torch
    v, even = R.code_values("e4m3")
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float().numpy()
    assert np.array_equal(np.unique(codes[np.isfinite(codes)]), v)
    assert R.nearest_code(np.array([0.5, 1.5, 2.5, -0.5, -200.0, np.nan, np.inf]), "int8").tolist() == [0, 2, 2, 0, -127, 0, 127]
    assert R.nearest_code(np.array([17.0, 19.0, 460.0, 2.0 ** -10, 3 * 2.0 ** -10]), "e4m3").tolist() == [16.0, 20.0, 448.0, 0.0, 2.0 ** -8]


def test_reference_slots_and_append_and_attention():
    table = np.full((2, 3), -1, np.int32)
    table[1, 0] = 9
    r = R.kv_slots([0, 15], [17, 2], table, np.array([4, 5, 6], np.int32), 0, 16, 20)
    assert table.tolist() == [[4, 5, -1], [9, 6, -1]] and r["taken"] == 3
    assert r["seq_start"].tolist() == [0, 17, 19] and r["kv_len"].tolist() == [17, 17]
    assert r["slot"].tolist() == list(range(64, 80)) + [80, 9 * 16 + 15, 96, -1] and r["pos"].tolist()[-4:] == [16, 15, 16, 0]
    codes, scale = np.zeros((1, 1, 16, 2)), np.ones((1, 1), np.float32)
    R.kv_append(codes, scale, np.array([[[127.0, -63.5]], [[1.0, 0.4]]]), [0, 1], "int8")
    assert scale[0, 0] == 1 and codes[0, 0, :2].tolist() == [[127, -64], [1, 0]]
    R.kv_append(codes, scale, np.array([[[254.0, 3.0]]]), [2], "int8")
    assert scale[0, 0] == 2 and codes[0, 0, :3].tolist() == [[64, -32], [0, 0], [127, 2]]
    q, k = np.array([[1.0, 0.0]]), np.array([[0.0, 5.0], [math.log(3.0), 2.0]])
    o, lse, _ = R.attention(q, k, np.array([[4.0, 0.0], [0.0, 8.0]]), 1.0, True)
    assert np.allclose(o, [[1.0, 6.0]]) and math.isclose(lse[0], math.log(4.0))
    o, lse, _ = R.attention(np.zeros((3, 2)), k[:1], k[:1], 1.0, True)
    assert np.isneginf(lse[:2]).all() and (o[:2] == 0).all() and lse[2] == 0


def test_paged_attn_refuses_out_in_place_of_q(L):
    from codpiece_b200._lib import CpqAttnSeqs
    q, c, s = tensor(256, 24, 3), cache(), CpqAttnSeqs()
    out = tensor(256, 24, 3)  # the same address
    for name, v in dict(seq_start=0x10, kv_len=0x20, table=0x30, table_stride=8, n_seqs=2, max_blocks=8).items():
        setattr(s, name, v)
    assert L.cpq_paged_attn(C.byref(q), C.byref(c), C.byref(s), 0.1, 1, C.byref(out), None, 0x80000, 1 << 30, None) == INVALID


def test_rope_refuses_the_same_output_twice(L):
    h = C.c_void_p()
    assert L.cpq_rope_create(C.byref(rope_params(n_dims=64)), C.byref(h)) == OK
    call = lambda x, y: L.cpq_rope_apply(h, arr(*x), arr(*y), len(x), C.c_void_p(0x9000), None)  # noqa: E731
    a, b, c = tensor(128, 4, 3), tensor(128, 2, 3, data=0x20000), tensor(128, 4, 3, data=0x30000)
    assert call([a, a], [a, a]) == INVALID                 # in place, twice
    assert call([a, a], [c, c]) == INVALID
    assert call([a, b], [c, tensor(128, 2, 3, data=0x30000)]) == INVALID
    d = tensor(128, 4, 3, data=0x40000)
    assert call([a, c], [c, d]) == INVALID                 # one tensor's output is the other's input
    none = [tensor(128, 4, 0), tensor(128, 4, 0)]
    assert call(none, none) == OK                          # no tokens: nothing overlaps
    L.cpq_rope_destroy(h)


def test_kv_slots_refuses_outputs_over_inputs(L):
    from codpiece_b200._lib import CpqKvSlotArgs
    base = dict(ctx_len=0x10, new_len=0x20, n_seqs=2, table=0x30, table_stride=4, max_blocks=4, block=16, free_pages=0x40,
                n_free=3, taken=0x50, taken_out=0x60, seq_start=0x70, kv_len=0x80, pos=0x90, slot=0xa0, n_rows=5)

    def args(**k):
        a = CpqKvSlotArgs()
        for name, v in {**base, **k}.items():
            setattr(a, name, v)
        return L.cpq_kv_slots(C.byref(a), None)

    outs = ("table", "taken_out", "seq_start", "kv_len", "pos", "slot")
    for out in outs:
        for other in ("ctx_len", "new_len", "free_pages", "taken", *outs):
            if other != out and (out, other) not in (("taken_out", "taken"), ("taken", "taken_out")):
                assert args(**{out: base[other]}) == INVALID, (out, other)  # lengths advanced in place, for one


def test_gather_refuses_one_tensor_for_keys_and_values(L):
    slot, c = C.c_void_p(0x5000), cache()
    k, v = tensor(256, 4, 3), tensor(256, 4, 3)
    assert L.cpq_kv_gather(C.byref(c), slot, C.byref(k), C.byref(v), None) == INVALID
    none = tensor(256, 4, 0)
    assert L.cpq_kv_gather(C.byref(c), slot, C.byref(none), C.byref(none), None) == OK


def test_attn_core_refuses_gated_queries():
    """With q_has_gate attn_q gives 2 x 256 rows a head; read as heads of 256 they would be other heads' and gates."""
    import dataclasses

    from codpiece_b200 import stack, tp
    with pytest.raises(ValueError, match="gate"):
        stack.AttnCore(tp.HP_QWEN35_27B, 1, max_ctx=64)
    with pytest.raises(ValueError, match="head size"):
        stack.AttnCore(dataclasses.replace(tp.HP_BENCH_27B, head_v=128), 1, max_ctx=64)
