"""The attention core around the quantized projections, measured: rotary positions, block tables and slot maps,
the 8-bit paged cache (append, gather) and attention over it.

Where ``own`` is false, ``run`` computes each operator from elementary torch operations; where it is true, it makes the
calls of codpiece_b200.attn that a user's program makes. ``exact`` computes the same results in 64 bits, by other steps.
"""
import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
TOP = {"int8": 127.0, "e4m3": 448.0}  # the largest code of a cache format


# ---- the cases -----------------------------------------------------------------------------------------------------------

# The heads of the 27B trunk: 24 query heads over 4 kv heads of 256.
_TRUNK = {"hkv": 4, "group": 6, "d": 256, "block": 64}


def listed():
    return [
        # one chat request, a short context, one token: latency
        {"name": "attn decode 1x1000", "op": "attn", "n": 1, "q": 1, "kv": 1000, "ragged": False, "causal": True,
         "type": "f32", "fmt": "int8", **_TRUNK},
        # one request deep in a long context, one token
        {"name": "attn decode 1x100003", "op": "attn", "n": 1, "q": 1, "kv": 100003, "ragged": False, "causal": True,
         "type": "f32", "fmt": "int8", **_TRUNK},
        # a server's decode batch: requests of every length
        {"name": "attn decode 32x<16000", "op": "attn", "n": 32, "q": 1, "kv": 16000, "ragged": True, "causal": True,
         "type": "bf16", "fmt": "e4m3", "hkv": 8, "group": 4, "d": 128, "block": 32},
        # speculative verify: 8 tokens of each of 4 requests
        {"name": "attn verify 4x8x20001", "op": "attn", "n": 4, "q": 8, "kv": 20001, "ragged": True, "causal": True,
         "type": "f32", "fmt": "int8", **_TRUNK},
        # a prefill chunk behind a long prompt, 16-bit activations
        {"name": "attn prefill 1x1024x16384", "op": "attn", "n": 1, "q": 1024, "kv": 16384, "ragged": False,
         "causal": True, "type": "bf16", "fmt": "int8", **_TRUNK},
        # prefill chunks of several requests, the trunk's F32 activations
        {"name": "attn prefill 3x<700x9000", "op": "attn", "n": 3, "q": 700, "kv": 9000, "ragged": True,
         "causal": True, "type": "f32", "fmt": "e4m3", **_TRUNK},
        # q and k of a verify step: a quarter of the head rotated, YaRN-scaled far positions
        {"name": "rope verify 8", "op": "rope", "t": 8, "hq": 24, "hk": 4, "d": 256, "dims": 64, "half": True,
         "scaled": "yarn", "type": "f32", "far": 1000000},
        # q and k of a long prefill chunk: the whole head, interleaved pairs
        {"name": "rope prefill 8191", "op": "rope", "t": 8191, "hq": 32, "hk": 8, "d": 128, "dims": 128, "half": False,
         "scaled": "none", "type": "bf16", "far": 100000},
        # one token of each of 24 requests into its partly filled page
        {"name": "append decode 24", "op": "append", "n": 24, "new": 1, "type": "f32", "fmt": "int8", "hkv": 4,
         "d": 256, "block": 64},
        # a long prompt and some shorter ones, written to new and half-filled pages
        {"name": "append prefill 5x<4000", "op": "append", "n": 5, "new": 4000, "type": "bf16", "fmt": "e4m3", "hkv": 8,
         "d": 128, "block": 32},
        # the tables of a decode step
        {"name": "slots decode 16", "op": "slots", "n": 16, "new": 1, "ctx": 30000, "block": 64},
        # the tables of a mixed batch: long prompts beside single tokens
        {"name": "slots mixed 300", "op": "slots", "n": 300, "new": 700, "ctx": 9000, "block": 16},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attn"] * 5 + ["rope", "append", "slots"])
    if op == "rope":
        d = rng.choice([128, 256])
        return {"op": "rope", "t": _log(rng, 1, 8000), "hq": rng.randint(1, 32), "hk": rng.randint(1, 8), "d": d,
                "dims": rng.choice([d, d // 2, d // 4, 2 * rng.randint(3, d // 2)]), "half": rng.random() < 0.5,
                "scaled": rng.choice(["none", "linear", "yarn", "factors"]), "type": rng.choice(list(TYPES)),
                "far": _log(rng, 100, 2000000)}
    if op == "append":
        return {"op": "append", "n": _log(rng, 1, 48), "new": _log(rng, 1, 2000) if rng.random() < 0.6 else 1,
                "type": rng.choice(list(TYPES)), "fmt": rng.choice(list(TOP)), "hkv": rng.randint(1, 4),
                "d": rng.choice([128, 256]), "block": rng.choice([16, 32, 64, 128])}
    if op == "slots":
        return {"op": "slots", "n": _log(rng, 1, 400), "new": _log(rng, 1, 400) if rng.random() < 0.6 else 1,
                "ctx": _log(rng, 10, 9000), "block": rng.choice([16, 32, 64, 128])}
    kind = rng.choice(["decode", "decode", "verify", "prefill"])
    n = _log(rng, 1, 32 if kind == "decode" else 6)
    q = 1 if kind == "decode" else rng.randint(2, 16) if kind == "verify" else _log(rng, 40, 1000)
    hkv, group = rng.choice([1, 2, 4]), rng.choice([1, 2, 3, 4, 6, 7, 8])
    # no more keys than the largest listed case has work for
    most = min(90000, int(200000 / n)) if kind != "prefill" else min(16000, int(1024 * 16384 * 24 / (n * q * hkv * group)))
    return {"op": "attn", "n": n, "q": q, "kv": max(q + 1, _log(rng, 30, max(64, most))), "ragged": rng.random() < 0.7,
            "causal": rng.random() < 0.8, "type": rng.choice(list(TYPES)), "fmt": rng.choice(list(TOP)), "hkv": hkv,
            "group": group, "d": rng.choice([128, 256]), "block": rng.choice([16, 32, 64, 128])}


def _lens(case):
    """The requests' lengths: (new tokens, tokens cached before), a function of the case alone."""
    r = random.Random(repr(sorted(case.items(), key=str)))
    n = case["n"]
    if case["op"] == "attn":
        ragged = case["ragged"]
        kv = [case["kv"]] + [r.randint(max(1, case["kv"] // 50), case["kv"]) if ragged else case["kv"] for _ in range(n - 1)]
        q = [case["q"]] + [r.randint(max(1, case["q"] // 2), case["q"]) if ragged else case["q"] for _ in range(n - 1)]
        return [min(a, b) for a, b in zip(q, kv)], [b - min(a, b) for a, b in zip(q, kv)]
    if case["op"] == "append":
        new = [case["new"]] + [r.randint(max(1, case["new"] // 20), case["new"]) for _ in range(n - 1)]
        return new, [r.randint(0, 2 * case["block"]) for _ in range(n)]
    new = [case["new"]] + [1 if r.random() < 0.5 else r.randint(1, case["new"]) for _ in range(n - 1)]
    return new, [r.randint(0, case["ctx"]) for _ in range(n)]


def _blocks(length, block):
    return -(-length // block)


# ---- inputs --------------------------------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEV)


def _values(g, shape, dtype):
    """Keys and values as a projection leaves them: Gaussian, some channels several times as large as others."""
    gain = torch.exp(0.5 * torch.randn(shape[-1], generator=g, device=DEV))
    return (torch.randn(shape, generator=g, device=DEV) * gain).to(dtype)


def _codes(g, case, pages):
    """A cache pool with content: codes [pages, hkv, block, d] and scales [pages, hkv]."""
    shape = (pages, case["hkv"], case["block"], case["d"])
    x = _values(g, shape, torch.float32)
    scale = (x.abs().amax(dim=(2, 3)) / TOP[case["fmt"]]).clone()
    x = x / scale[:, :, None, None]
    if case["fmt"] == "int8":
        return torch.round(x).to(torch.int8), scale
    return x.clamp(-448.0, 448.0).to(torch.float8_e4m3fn), scale


def _rope_params(case):
    p = {"n_dims": case["dims"], "base": 1000000.0 if case["scaled"] != "none" else 10000.0, "freq_scale": 1.0,
         "ext_factor": 0.0, "attn_factor": 1.0, "beta_fast": 32.0, "beta_slow": 1.0, "n_ctx_orig": 0, "freq_factors": None}
    if case["scaled"] == "linear":
        p["freq_scale"] = 0.25
    elif case["scaled"] == "yarn":
        p.update(freq_scale=0.25, ext_factor=1.0, n_ctx_orig=262144)
    elif case["scaled"] == "factors":
        p["freq_factors"] = [1.0 + 7.0 * i / case["dims"] for i in range(case["dims"] // 2)]
    return p


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    state = {"case": dict(case)}
    if op == "rope":
        t, d = case["t"], case["d"]
        state["q"] = torch.randn(t, case["hq"], d, generator=g, device=DEV).to(TYPES[case["type"]])
        state["k"] = torch.randn(t, case["hk"], d, generator=g, device=DEV).to(TYPES[case["type"]])
        start = torch.randint(0, case["far"], (1,), generator=g, device=DEV)
        state["pos"] = (start + torch.arange(t, device=DEV)).to(torch.int32)
        return state
    new, ctx = _lens(case)
    n, block = len(new), case["block"]
    held = [_blocks(c, block) for c in ctx]
    total = [_blocks(c + a, block) for c, a in zip(ctx, new)]
    width = max(total)
    start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    if op == "slots":
        pages = sum(total) + 64
        perm = torch.randperm(pages, generator=g, device=DEV).to(torch.int32).cpu().numpy()
        table = np.full((n, width), -1, dtype=np.int32)
        at = 0
        for r in range(n):  # the pages that the requests hold already
            table[r, :held[r]] = perm[at:at + held[r]]
            at += held[r]
        state.update(ctx=_ints(ctx), new=_ints(new), table=torch.from_numpy(table).to(DEV),
                     free=torch.from_numpy(perm[at:].copy()).to(DEV), taken=_ints([0]), rows=int(start[-1]) + 5,
                     taken_out=_ints([0]))
        return state
    pages = sum(total) + (0 if op == "append" else 3)
    perm = torch.randperm(pages, generator=g, device=DEV).to(torch.int32).cpu().numpy()
    table = np.zeros((n, width), dtype=np.int32)
    at = 0
    for r in range(n):
        table[r, :total[r]] = perm[at:at + total[r]]
        at += total[r]
    state["k_codes"], state["k_scale"] = _codes(g, case, pages)
    state["v_codes"], state["v_scale"] = _codes(g, case, pages)
    if op == "attn":
        hq = case["hkv"] * case["group"]
        state["q"] = (1.5 * torch.randn(int(start[-1]), hq, case["d"], generator=g, device=DEV)).to(TYPES[case["type"]])
        state.update(table=torch.from_numpy(table).to(DEV), start=_ints(start), kv_len=_ints([a + b for a, b in zip(ctx, new)]))
        state["max_q"] = max(new)
        return state
    slots = np.concatenate([table[r, (ctx[r] + np.arange(new[r])) // block].astype(np.int64) * block
                            + (ctx[r] + np.arange(new[r])) % block for r in range(n)])
    t, dtype = int(start[-1]), TYPES[case["type"]]
    state.update(k=_values(g, (t, case["hkv"], case["d"]), dtype), v=_values(g, (t, case["hkv"], case["d"]), dtype),
                 slot=torch.from_numpy(slots).to(DEV), every=torch.arange(pages * block, device=DEV))
    return state


# ---- the operators in their plain form -----------------------------------------------------------------------------------

def _plain_turns(case):
    """Radians per position of each pair, in 64 bits, and the magnitude's factor."""
    p = _rope_params(case)
    i = torch.arange(case["dims"] // 2, dtype=torch.float64, device=DEV)
    f = torch.pow(torch.tensor(p["base"], dtype=torch.float64, device=DEV), -2.0 * i / case["dims"])
    if p["freq_factors"] is not None:
        f = f / torch.tensor(p["freq_factors"], dtype=torch.float64, device=DEV)
    scaled, m = f * p["freq_scale"], p["attn_factor"]
    if p["ext_factor"]:
        at = [case["dims"] * math.log(p["n_ctx_orig"] / (b * 2 * math.pi)) / (2 * math.log(p["base"]))
              for b in (p["beta_fast"], p["beta_slow"])]
        low, high = max(0.0, math.floor(at[0])), min(case["dims"] - 1.0, math.ceil(at[1]))
        mix = p["ext_factor"] * (1.0 - ((i - low) / max(0.001, high - low)).clamp(0.0, 1.0))
        scaled = scaled * (1.0 - mix) + f * mix
        m *= 1.0 + 0.1 * math.log(1.0 / p["freq_scale"])
    return scaled, m


def _plain_rotate(x, cos, sin, dims, half):
    a, b = (x[..., :dims // 2], x[..., dims // 2:dims]) if half else (x[..., 0:dims:2], x[..., 1:dims:2])
    a, b = a.float(), b.float()
    u, w = a * cos - b * sin, a * sin + b * cos
    turned = torch.cat([u, w], dim=-1) if half else torch.stack([u, w], dim=-1).flatten(-2)
    return torch.cat([turned.to(x.dtype), x[..., dims:]], dim=-1)


def _plain_rope(s):
    case = s["case"]
    f, m = _plain_turns(case)
    angle = s["pos"].double()[:, None] * f[None, :]
    cos, sin = (m * torch.cos(angle)).float()[:, None, :], (m * torch.sin(angle)).float()[:, None, :]
    return {"q": _plain_rotate(s["q"], cos, sin, case["dims"], case["half"]),
            "k": _plain_rotate(s["k"], cos, sin, case["dims"], case["half"])}


def _plain_slots(s):
    block, rows = s["case"]["block"], s["rows"]
    ctx, new, table, free = s["ctx"].long(), s["new"].long(), s["table"].long(), s["free"].long()
    held, total = (ctx + block - 1) // block, (ctx + new + block - 1) // block
    need = total - held
    through = torch.cumsum(need, 0)
    served = ((need == 0) | (through <= free.numel() - s["taken"].long())) & (total <= table.shape[1])
    first = s["taken"].long() + through - need
    j = torch.arange(table.shape[1], device=table.device)[None, :]
    fresh = served[:, None] & (j >= held[:, None]) & (j < total[:, None])
    table = torch.where(fresh, free[(first[:, None] + j - held[:, None]).clamp(0, free.numel() - 1)], table)
    taken = s["taken"].long() + (need * served).sum()
    end = torch.cumsum(new, 0)
    start = torch.cat([end.new_zeros(1), end])
    row = torch.arange(rows, device=table.device)
    r = torch.searchsorted(end, row, right=True)
    valid, r = r < ctx.numel(), r.clamp(max=ctx.numel() - 1)
    pos = ctx[r] + row - start[r]
    page = table[r, (pos // block).clamp(0, table.shape[1] - 1)]
    valid = valid & served[r]
    slot = torch.where(valid & (page >= 0), page * block + pos % block, torch.full_like(pos, -1))
    return {"table": table.int(), "taken": taken.int().reshape(1), "seq_start": start.clamp(max=rows).int(),
            "kv_len": torch.where(served, ctx + new, torch.zeros_like(ctx)).int(),
            "pos": torch.where(valid, pos, torch.zeros_like(pos)).int(), "slot": slot}


def _plain_round(y, fmt):
    """The nearest code of y (64 bits), ties to even, as a number."""
    y = y.clamp(-TOP[fmt], TOP[fmt])
    if fmt == "int8":
        return torch.round(y)
    step = torch.exp2(torch.frexp(y).exponent.double().clamp(min=-5.0) - 4.0)  # 3 bits after the first, down to 2^-9
    return torch.round(y / step) * step


def _plain_append(codes, scale, x, slot, block, fmt):
    """The pool after rows x were written to their slots: codes as numbers, and the scales. A page whose scale grew has the
    rows that it held before coded again."""
    page, at = slot // block, slot % block
    pages, hkv = scale.shape
    low = torch.full((pages,), block, dtype=torch.int64, device=x.device).scatter_reduce(0, page, at, "amin")
    touched = low < block  # the rows before a page's first new row were there already
    top = torch.zeros(pages, hkv, device=x.device).index_reduce(0, page, x.float().abs().amax(dim=-1), "amax")
    fresh = (top.double() / TOP[fmt]).float()  # the quotient itself, rounded once
    grown = torch.where((touched & (low > 0))[:, None], torch.maximum(scale, fresh), torch.where(touched[:, None], fresh, scale))
    ratio = torch.where(grown > 0, scale.double() / grown.double(), torch.zeros_like(grown, dtype=torch.float64))
    again = (touched & (low > 0))[:, None] & (grown != scale)
    old = codes.double()
    before = torch.arange(block, device=x.device)[None, :] < low[:, None]
    again = again[:, :, None, None] & before[:, None, :, None]
    old = torch.where(again, _plain_round(old * ratio[:, :, None, None], fmt), old)
    put = _plain_round(x.double() / grown[page].double()[:, :, None], fmt)
    old[page, :, at, :] = put
    return old, grown


def _plain_gather(values, scale, slot, block):
    return values[slot // block, :, slot % block, :].float() * scale[slot // block][:, :, None]


def _plain_attn(s):
    case = s["case"]
    block, hkv, group, d = case["block"], case["hkv"], case["group"], case["d"]
    table, start, kv_len = s["table"].long(), s["start"].long(), s["kv_len"].long()
    n, width = table.shape
    k = (s["k_codes"][table].float() * s["k_scale"][table][..., None, None]).transpose(1, 2).reshape(n, hkv, width * block, d)
    q_len = start[1:] - start[:-1]
    i = torch.arange(s["max_q"], device=DEV)
    row = (start[:-1, None] + i[None, :]).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][row].float().reshape(n, -1, hkv, group, d).permute(0, 2, 1, 3, 4).reshape(n, hkv, -1, d)
    scores = torch.matmul(q, k.transpose(-1, -2)).reshape(n, hkv, -1, group, width * block) * (d ** -0.5)
    del k
    last = kv_len[:, None] - q_len[:, None] + i[None, :] + 1 if case["causal"] else kv_len[:, None].expand(n, s["max_q"])
    sees = torch.arange(width * block, device=DEV)[None, None, :] < torch.minimum(last, kv_len[:, None])[:, :, None]
    scores = scores.masked_fill(~sees[:, None, :, None, :], float("-inf"))
    top = scores.amax(dim=-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    del scores
    total = p.sum(dim=-1, keepdim=True)
    v = (s["v_codes"][table].float() * s["v_scale"][table][..., None, None]).transpose(1, 2).reshape(n, hkv, width * block, d)
    v = torch.where((torch.arange(width * block, device=DEV)[None, :] < kv_len[:, None])[:, None, :, None], v, torch.zeros_like(v))
    o = torch.matmul(p.reshape(n, hkv, -1, width * block), v).reshape(n, hkv, -1, group, d)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    lse = (top + torch.log(total)).squeeze(-1)
    out, lses = torch.zeros_like(s["q"]), torch.zeros(s["q"].shape[:2], device=DEV)
    valid = i[None, :] < q_len[:, None]
    out[row[valid]] = o.permute(0, 2, 1, 3, 4).reshape(n, -1, hkv * group, d)[valid].to(out.dtype)
    lses[row[valid]] = lse.permute(0, 2, 1, 3).reshape(n, -1, hkv * group)[valid]
    return {"out": out, "lse": lses}


# ---- a pass --------------------------------------------------------------------------------------------------------------

def _own_cache(s):
    if "cache" not in s:  # the pool's handle, which a program keeps
        from codpiece_b200 import attn
        s["cache"] = attn.KvCache.wrap(s["k_codes"], s["v_codes"], s["k_scale"], s["v_scale"])
    return s["cache"]


def run(state):
    s, case = state, state["case"]
    op = case["op"]
    if own:
        from codpiece_b200 import attn
        if op == "rope":
            if "rope" not in s:  # the frequencies, made once per model
                s["rope"] = attn.Rope(mode=attn.ROPE_HALF if case["half"] else attn.ROPE_INTERLEAVED, **_rope_params(case))
            q, k = attn.rope(s["rope"], [s["q"], s["k"]], s["pos"])
            return {"q": q, "k": k}
        if op == "slots":
            r = attn.kv_slots(s["ctx"], s["new"], s["table"], s["free"], s["taken"], block=case["block"], n_rows=s["rows"],
                              taken_out=s["taken_out"])
            return {"table": s["table"], "taken": s["taken_out"], "seq_start": r.seq_start, "kv_len": r.kv_len, "pos": r.pos,
                    "slot": r.slot}
        cache = _own_cache(s)
        if op == "append":
            attn.kv_append(cache, s["k"], s["v"], s["slot"])
            k, v = attn.kv_gather(cache, s["every"], dtype=torch.float32)
            return {"k": k, "v": v, "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
        out, lse = attn.paged_attn(s["q"], cache, s["table"], s["start"], s["kv_len"], causal=case["causal"], return_lse=True)
        return {"out": out, "lse": lse}
    if op == "rope":
        return _plain_rope(s)
    if op == "slots":
        return _plain_slots(s)
    if op == "append":
        got = {}
        for name in ("k", "v"):
            values, scale = _plain_append(s[name + "_codes"].float(), s[name + "_scale"], s[name], s["slot"], case["block"],
                                          case["fmt"])
            got[name], got[name + "_scale"] = _plain_gather(values, scale, s["every"], case["block"]), scale
        return got
    return _plain_attn(s)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------

def work(case):
    op = case["op"]
    if op == "rope":
        heads = case["hq"] + case["hk"]
        return {"bytes": 2 * case["t"] * heads * case["d"] * SIZE[case["type"]] + 4 * case["t"],
                "flops": 3 * case["t"] * heads * case["dims"]}
    new, ctx = _lens(case)
    n, block = len(new), case["block"]
    total = [_blocks(c + a, block) for c, a in zip(ctx, new)]
    if op == "slots":
        fresh = sum(t - _blocks(c, block) for t, c in zip(total, ctx))
        return {"bytes": 4 * (2 * n + 2 * n + 1) + 8 * fresh + 12 * (sum(new) + 5), "flops": 0}
    hkv, d = case["hkv"], case["d"]
    if op == "append":
        pages = sum(total)
        written = sum(new) * hkv * d * 2
        # the rows, their codes, and the read-back of the whole pool with its values
        return {"bytes": written * (SIZE[case["type"]] + 1) + pages * block * hkv * d * 2 * (1 + 4) + 8 * pages * block
                + 4 * 4 * pages * hkv, "flops": 4 * written}
    kv = [a + b for a, b in zip(new, ctx)]
    hq = hkv * case["group"]
    pairs = sum((q * k - q * (q - 1) // 2) if case["causal"] else q * k for q, k in zip(new, kv))
    return {"bytes": 2 * sum(kv) * hkv * d + 2 * sum(new) * hq * d * SIZE[case["type"]] + 4 * sum(new) * hq
            + 8 * sum(total) * hkv + 4 * sum(total), "flops": 4 * pairs * hq * d}


# ---- in 64 bits, by other steps ------------------------------------------------------------------------------------------

def _exact_rope(case, s):
    p = _rope_params(case)
    dims, h = case["dims"], case["dims"] // 2
    f = np.array([p["base"] ** (-(2.0 * i) / dims) for i in range(h)])
    if p["freq_factors"] is not None:
        f = f / np.array(p["freq_factors"])
    w = f * p["freq_scale"]
    m = p["attn_factor"]
    if p["ext_factor"]:
        dim_of = lambda beta: dims * math.log(p["n_ctx_orig"] / (beta * 2 * math.pi)) / (2 * math.log(p["base"]))  # noqa: E731
        low, high = max(0, math.floor(dim_of(p["beta_fast"]))), min(dims - 1, math.ceil(dim_of(p["beta_slow"])))
        keep = np.array([p["ext_factor"] * (1 - min(1.0, max(0.0, (i - low) / max(0.001, high - low)))) for i in range(h)])
        w = f * keep + w * (1 - keep)
        m *= 1 + 0.1 * math.log(1 / p["freq_scale"])
    turn = torch.polar(torch.full((1,), m, dtype=torch.float64, device=DEV),
                       s["pos"].double()[:, None] * torch.from_numpy(w).to(DEV)[None, :])[:, None, :]
    got = {}
    for name in ("q", "k"):
        x = s[name].double()
        z = torch.complex(x[..., :h], x[..., h:dims]) if case["half"] else torch.view_as_complex(
            x[..., :dims].reshape(*x.shape[:-1], h, 2).contiguous())
        z = z * turn
        y = x.clone()
        if case["half"]:
            y[..., :h], y[..., h:dims] = z.real, z.imag
        else:
            y[..., :dims] = torch.view_as_real(z).flatten(-2)
        got[name] = y
    return got


def _exact_codes(fmt):
    """Every value that a code stands for, ascending, and the borders between neighbours with the side a tie goes to."""
    if fmt == "int8":
        values = np.arange(-127, 128, dtype=np.float64)
        even = np.arange(-127, 128) % 2 == 0
    else:
        mags = [(j / 8) * 2.0 ** -6 for j in range(8)] + [(1 + j / 8) * 2.0 ** e for e in range(-6, 9) for j in range(8)]
        mags = np.array(mags[:-1])  # the last pattern is no number
        values = np.concatenate([-mags[:0:-1], mags])
        ranks = np.arange(len(mags))
        even = np.concatenate([ranks[:0:-1], ranks]) % 2 == 0
    return values, even


def _exact_nearest(y, fmt):
    values, even = _exact_codes(fmt)
    border = (values[1:] + values[:-1]) / 2
    vt, et, bt = (torch.from_numpy(a).to(DEV) for a in (values, even, border))
    y = y.contiguous()
    i = torch.searchsorted(bt, y, right=False)          # a tie falls below its border
    tie = (i < bt.numel()) & (bt[i.clamp(max=bt.numel() - 1)] == y) & ~et[i]
    return vt[i + tie.long()]


def _exact_append(case, s):
    block, fmt = case["block"], case["fmt"]
    slot = s["slot"].cpu().numpy()
    got = {}
    for name in ("k", "v"):
        codes, scale = s[name + "_codes"].double().clone(), s[name + "_scale"].clone()
        x = s[name].double()
        page = slot // block
        cuts = np.flatnonzero(np.concatenate([[True], page[1:] != page[:-1]]))
        edges = np.append(cuts, len(slot))
        for a, b in zip(edges[:-1], edges[1:]):
            pg, off = int(page[a]), int(slot[a] % block)
            part = x[a:b].transpose(0, 1)  # [hkv, rows, d]
            fresh = (part.abs().amax(dim=(1, 2)) / TOP[fmt]).float()
            new = torch.maximum(scale[pg], fresh) if off else fresh
            if off:
                back = codes[pg, :, :off] * scale[pg].double()[:, None, None] / new.double()[:, None, None]
                same = (new == scale[pg])[:, None, None]
                codes[pg, :, :off] = torch.where(same, codes[pg, :, :off], _exact_nearest(back, fmt))
            codes[pg, :, off:off + (b - a)] = _exact_nearest(part / new.double()[:, None, None], fmt)
            scale[pg] = new
        got[name] = (codes * scale.double()[:, :, None, None]).transpose(1, 2).reshape(-1, case["hkv"], case["d"])
        got[name + "_scale"] = scale.double()
    return got


def _exact_attn(case, s):
    block, hkv, group, d = case["block"], case["hkv"], case["group"], case["d"]
    new, ctx = _lens(case)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    lse = torch.zeros(s["q"].shape[:2], dtype=torch.float64, device=DEV)
    at = 0
    for r, (nq, c) in enumerate(zip(new, ctx)):
        kv = nq + c
        pages = s["table"][r, :_blocks(kv, block)].long()
        for h in range(hkv):
            k = (s["k_codes"][pages, h].double() * s["k_scale"][pages, h].double()[:, None, None]).reshape(-1, d)[:kv]
            v = (s["v_codes"][pages, h].double() * s["v_scale"][pages, h].double()[:, None, None]).reshape(-1, d)[:kv]
            j = torch.arange(kv, device=DEV)
            for gi in range(group):
                q = s["q"][at:at + nq, h * group + gi].double()
                z = (q @ k.T) / math.sqrt(d)
                if case["causal"]:
                    z = z.masked_fill(j[None, :] > c + torch.arange(nq, device=DEV)[:, None], float("-inf"))
                lse[at:at + nq, h * group + gi] = torch.logsumexp(z, dim=-1)
                out[at:at + nq, h * group + gi] = torch.softmax(z, dim=-1) @ v
        at += nq
    return {"out": out, "lse": lse}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        return _exact_rope(case, s)
    if case["op"] == "append":
        return _exact_append(case, s)
    if case["op"] == "attn":
        return _exact_attn(case, s)
    return None  # whole numbers: equal or not
