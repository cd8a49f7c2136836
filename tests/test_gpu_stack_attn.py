"""The 27B-shaped stack with its attention core (stack.AttnCore): steps over a growing cache, eager and captured,
verify batches and rollback, against the operators called one by one and dense attention in 64 bits."""
import pytest

pytestmark = pytest.mark.gpu


def _core(stack, tp, attn, n_layer, **kw):
    return stack.AttnCore(tp.HP_BENCH_27B, n_layer, **kw)


def _dense(torch, attn, q, cache, core, kv):
    """Attention of rows q (the last of kv tokens) over the cache's own values, 64 bits."""
    d, hkv, b = cache.head_dim, cache.n_head_kv, cache.block
    slots = torch.tensor([int(core.table[0, p // b]) * b + p % b for p in range(kv)], device="cuda")
    k, v = (t.double() for t in attn.kv_gather(cache, slots))
    m, hq, _ = q.shape
    z = torch.einsum("ihgd,jhd->ihgj", q.double().view(m, hkv, hq // hkv, d), k) * d ** -0.5
    lim = kv - m + torch.arange(m, device="cuda")
    z = z.masked_fill(torch.arange(kv, device="cuda") > lim[:, None, None, None], float("-inf"))
    return torch.einsum("ihgj,jhd->ihgd", torch.softmax(z, -1), v).reshape(m, hq, d)


@pytest.mark.parametrize("m,fmt", [(1, 0), (8, 1)])
def test_stack_step_runs_the_attention_core(cuda, m, fmt):
    torch = cuda
    from codpiece_b200 import attn, stack, tp
    from codpiece_b200 import mul_mat as mm

    core = _core(stack, tp, attn, 1, max_ctx=200, fmt=fmt)
    s = stack.Stack(tp.HP_BENCH_27B, n_layer=1, m=m, seed=3, head=False, attn_core=core)
    g = torch.Generator("cuda").manual_seed(1)
    for step in range(3):
        s.h.copy_(torch.randn(m, 5120, device="cuda", generator=g))
        h0 = s.h.clone()
        s.step_body()
        kv = m * (step + 1)
        assert int(core.ctx[0]) == kv and int(s.slots.kv_len[0]) == kv and int(core.taken[0]) == -(-kv // 64)
        q = s.qb.view(m, 24, 256)
        ref = _dense(torch, attn, q, core.caches[0], core, kv)
        got = s.ab.view(m, 24, 256).double()
        assert float((got - ref).norm() / ref.norm()) <= 1e-5
        # the rotated keys are in the cache to half a step of its codes, one coding each. A step is the scale for int8;
        # e4m3 has three bits after the leading one, so a step is at most |x| / 8 from 2^-6 scales on, and below that
        # (subnormal codes) it is 2^-9 scales whatever the value: their sum bounds both
        slots = torch.tensor([int(core.table[0, p // 64]) * 64 + p % 64 for p in range(kv - m, kv)], device="cuda")
        k = s.kb.view(m, 4, 256)
        back = attn.kv_gather(core.caches[0], slots)[0]
        scale = core.caches[0].k_scale[core.table[0, (kv - 1) // 64].long()][None, :, None]
        code_step = scale if fmt == 0 else k.abs() / 8 + scale * 2.0 ** -9
        assert ((back - k).abs() <= 0.501 * code_step).all()
        # the rest of the layer: o of the attention, then the FFN, as single calls
        lw = s.layers[0]
        part = mm.mul_mat(lw.o, s.ab)
        h = h0 + part
        gate, up = mm.mul_mat_fused([lw.gate, lw.up], h, mode=mm.PRO_RMS)
        down = mm.mul_mat_fused([lw.down], gate, mode=mm.PRO_SWIGLU, r=up)[0]
        want = h + down
        assert float((s.h_final - want).abs().max() / want.abs().max()) <= 1e-3
    s.release()


def test_captured_decode_equals_eager_decode_and_rolls_back(cuda):
    torch = cuda
    from codpiece_b200 import attn, stack, tp

    outs = []
    xs = torch.randn(70, 1, 5120, device="cuda", generator=torch.Generator("cuda").manual_seed(2))
    for captured in (False, True):
        core = _core(stack, tp, attn, 2, max_ctx=256, block=32)
        s = stack.Stack(tp.HP_BENCH_27B, n_layer=2, m=1, seed=5, head=False, attn_core=core)
        if captured:
            s.h.copy_(xs[0])
            s.capture()             # one eager step; what is captured does not run
            core.ctx.zero_()
            core.taken.zero_()
        got = []
        for x in xs:
            s.h.copy_(x)
            s.replay() if captured else s.step_body()
            got.append(s.h_final.clone())
        outs.append(torch.cat(got))
        assert int(core.ctx[0]) == 70 and int(core.taken[0]) == 3
        core.rollback(10)           # ten tokens rejected, then the same ones again
        assert int(core.ctx[0]) == 60 and int(core.taken[0]) == 2
        for x in xs[60:]:
            s.h.copy_(x)
            s.replay() if captured else s.step_body()
        assert int(core.ctx[0]) == 70 and int(core.taken[0]) == 3
        err = float((s.h_final - outs[-1][-1:]).abs().max() / outs[-1][-1:].abs().max())
        assert err <= 2e-2  # page scales only grow, so the second pass codes some keys in coarser steps
        s.release()
    assert torch.equal(outs[0], outs[1])


def test_a_full_cache_stops_the_length(cuda):
    torch = cuda
    from codpiece_b200 import attn, stack, tp

    core = _core(stack, tp, attn, 1, max_ctx=30, block=32)  # one page
    s = stack.Stack(tp.HP_BENCH_27B, n_layer=1, m=12, head=False, attn_core=core)
    steps = []
    # first the zero h a new stack has (v = 0, so attention gives 0 as well), then a real one
    for x in (torch.zeros(12, 5120, device="cuda"), torch.randn(12, 5120, device="cuda")):
        for want in (12, 24, 24, 24):
            s.h.copy_(x)
            s.step_body()
            assert int(core.ctx[0]) == want and int(core.taken[0]) == 1
            served = bool((s.slots.slot >= 0).all())
            assert bool((s.ab == 0).all()) == (not served or not x.any())
            assert int(s.slots.kv_len[0]) == (want if served else 0)
            steps.append(served)
        core.rollback(24)
    assert steps == [True, True, False, False] * 2
    core.ctx.fill_(5)
    core.rollback(100)
    assert int(core.ctx[0]) == 0 and int(core.taken[0]) == 0
    s.release()


def test_stack_refuses_what_the_core_does_not_run(cuda):
    from codpiece_b200 import attn, stack, tp

    core = _core(stack, tp, attn, 1, max_ctx=64)
    with pytest.raises(ValueError):
        stack.Stack(tp.HP_BENCH_27B, n_layer=2, m=1, head=False, attn_core=core)
    with pytest.raises(ValueError):
        stack.Stack(tp.HP_BENCH_27B, n_layer=1, m=1, head=False, attn_core=core, use_trunk=True)


@pytest.mark.parametrize("m", [1, 4])
def test_capture_in_mid_sequence_caches_nothing(cuda, m):
    """What capture() runs to warm up is no token of the sequence: length, pages, codes and scales stay, and the replayed
    steps go on where the eager ones ended."""
    torch = cuda
    from codpiece_b200 import attn, stack, tp

    xs = torch.randn(5, m, 5120, device="cuda", generator=torch.Generator("cuda").manual_seed(4))
    outs = []
    for captured in (False, True):
        core = _core(stack, tp, attn, 1, max_ctx=64, block=16)
        s = stack.Stack(tp.HP_BENCH_27B, n_layer=1, m=m, seed=5, head=False, attn_core=core)
        for x in xs[:2]:
            s.h.copy_(x)
            s.step_body()
        if captured:
            c = core.caches[0]
            state = [core.ctx, core.taken, core.table, c.k, c.v, c.k_scale, c.v_scale]
            before = [t.clone() for t in state]
            s.h.copy_(100 * xs[2])
            s.capture()
            for t, b in zip(state, before):
                assert torch.equal(t.view(torch.uint8), b.view(torch.uint8))
        got = []
        for x in xs[2:]:
            s.h.copy_(x)
            s.replay() if captured else s.step_body()
            got.append(s.h_final.clone())
        assert int(core.ctx[0]) == 5 * m
        outs.append(torch.cat(got))
        s.release()
    assert torch.equal(outs[0], outs[1])


def test_stack_refuses_a_core_of_other_shapes(cuda):
    import dataclasses

    from codpiece_b200 import attn, stack, tp

    hp = tp.HP_BENCH_27B
    for other in (dataclasses.replace(hp, n_head_kv=2), dataclasses.replace(hp, head_k=128, head_v=128)):
        core = stack.AttnCore(other, 1, max_ctx=64, rope=attn.Rope(64))
        with pytest.raises(ValueError):
            stack.Stack(hp, n_layer=1, m=1, head=False, attn_core=core)
    core = _core(stack, tp, attn, 1, max_ctx=64)
    with pytest.raises(ValueError, match="gate"):
        stack.Stack(dataclasses.replace(hp, q_has_gate=True), n_layer=1, m=1, head=False, attn_core=core)
    with pytest.raises(ValueError):
        stack.AttnCore(dataclasses.replace(hp, q_has_gate=True), 1, max_ctx=64)


@pytest.mark.parametrize("fmt", [0, 1])
def test_after_a_rollback_attention_is_that_of_what_the_cache_holds(cuda, fmt):
    """Rejected tokens are forgotten: each step after a rollback equals 64-bit attention over the cache's values, and what
    the rejected tokens leave behind is at most a coarser scale in the last page kept. Its codes are made again once for
    each rejected token that raises the scale, off by half a step of the new scale each time (int8: the scale; e4m3: at
    most 2^-4 of the value, or 2^-10 scales for the subnormal codes)."""
    torch = cuda
    from codpiece_b200 import attn, stack, tp

    core = _core(stack, tp, attn, 1, max_ctx=128, block=32, fmt=fmt)
    s = stack.Stack(tp.HP_BENCH_27B, n_layer=1, m=1, seed=5, head=False, attn_core=core)
    cache = core.caches[0]
    xs = torch.randn(60, 1, 5120, device="cuda", generator=torch.Generator("cuda").manual_seed(7))

    def step(x):
        s.h.copy_(x)
        s.step_body()
        kv = int(core.ctx[0])
        ref = _dense(torch, attn, s.qb.view(1, 24, 256), cache, core, kv)
        assert float((s.ab.view(1, 24, 256).double() - ref).norm() / ref.norm()) <= 1e-5

    def held():
        slots = torch.tensor([int(core.table[0, p // 32]) * 32 + p % 32 for p in range(45)], device="cuda")
        return attn.kv_gather(cache, slots)

    for x in xs[:45]:
        step(x)
    before, rejected = held(), 8
    for x in xs[45:45 + rejected]:
        step(x)
    core.rollback(rejected)
    assert int(core.ctx[0]) == 45 and int(core.taken[0]) == 2
    last = int(core.table[0, 1])
    for now, was, scale in zip(held(), before, (cache.k_scale[last], cache.v_scale[last])):
        assert torch.equal(now[:32], was[:32])                     # full pages are not touched
        half = scale[None, :, None] / 2 if fmt == 0 else torch.maximum(was[32:].abs() / 16, scale[None, :, None] * 2.0 ** -10)
        assert ((now[32:] - was[32:]).abs() <= 1.1 * rejected * half).all()  # (1.1: e4m3's values drift between codings)
    for x in xs[45 + rejected:]:
        step(x)
    s.release()


def test_a_capture_that_fails_leaves_the_steps_their_tokens(cuda, monkeypatch):
    from codpiece_b200 import attn, stack, tp

    core = _core(stack, tp, attn, 1, max_ctx=64)
    s = stack.Stack(tp.HP_BENCH_27B, n_layer=1, m=2, head=False, attn_core=core)
    with monkeypatch.context() as mp:
        mp.setattr(attn, "rope", lambda *a, **k: (_ for _ in ()).throw(RuntimeError("on the host")))
        with pytest.raises(RuntimeError, match="on the host"):
            s.capture()
    assert int(core.ctx[0]) == 0
    s.step_body()
    assert int(core.ctx[0]) == 2
    s.release()
