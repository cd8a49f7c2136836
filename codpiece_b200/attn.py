"""Host-side surface of the attention core over libcpq (include/cpq.h: cpq_rope_*,
cpq_kv_*, cpq_paged_attn): what stands between the q/k/v projections and
attn_output in an attention layer (crates/codpiece-model/src/qwen35.rs:3000-3197).

q, k and v are CUDA tensors [tokens, heads, D] of float32, float16 or bfloat16
whose rows of D are contiguous (any other strides: views into a projection's
output). Keys and values live in a :class:`KvCache`, a pool of pages of 8-bit
codes with one scale per page and kv head. A step over requests of different
lengths:

    s = kv_slots(ctx_len, new_len, table, free_pages, taken, block=cache.block, n_rows=T)
    rope(table_of_frequencies, [q, k], s.pos, [q, k])
    kv_append(cache, k, v, s.slot)
    out = paged_attn(q, cache, table, s.seq_start, s.kv_len)

Every call goes to the device of its tensors, on the given stream or that
device's current one. There is no CPU or PyTorch fallback.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

import torch

from . import _lib
from ._lib import CpqAttnSeqs, CpqKvCache, CpqKvSlotArgs, CpqRopeParams, CpqTensor, check, lib

ROPE_INTERLEAVED, ROPE_HALF = 0, 1
KV_INT8, KV_E4M3 = 0, 1

_ACT_TYPES = {torch.float32: _lib.TYPE_F32, torch.float16: _lib.TYPE_F16, torch.bfloat16: _lib.TYPE_BF16}
_KV_TYPES = {torch.int8: KV_INT8, torch.float8_e4m3fn: KV_E4M3}
_KV_DTYPES = {KV_INT8: torch.int8, KV_E4M3: torch.float8_e4m3fn}


def _desc(t: torch.Tensor, what: str) -> CpqTensor:
    """Descriptor of a [tokens, heads, D] activation tensor (ne = [D, heads, tokens, 1])."""
    if not t.is_cuda or t.dtype not in _ACT_TYPES or t.dim() != 3:
        raise TypeError(f"{what}: expected a CUDA tensor [tokens, heads, D] of float32, float16 or bfloat16")
    if t.stride(2) != 1 and t.shape[2] != 1:
        raise TypeError(f"{what}: rows must be contiguous (stride {t.stride(2)} along the last dimension)")
    if min(t.stride()) < 0:
        raise TypeError(f"{what}: negative stride")
    b = t.element_size()
    d = CpqTensor()
    d.type = _ACT_TYPES[t.dtype]
    d.ne[:] = [t.shape[2], t.shape[1], t.shape[0], 1]
    d.nb[:] = [b, t.stride(1) * b, t.stride(0) * b, t.stride(0) * b * t.shape[0]]
    d.data = t.data_ptr()
    return d


def _check_ints(t: torch.Tensor, what: str, dtype: torch.dtype, device: torch.device, numel: int | None = None) -> None:
    if t.dtype != dtype or t.device != device or not t.is_contiguous() or (numel is not None and t.numel() != numel):
        raise TypeError(f"{what}: expected a contiguous {dtype} tensor{'' if numel is None else f' of {numel} elements'} on {device}")


def _same_device(device: torch.device, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} is on {t.device}, expected {device}")


def _table(table: torch.Tensor, n: int, device: torch.device) -> int:
    """Row stride of a block table [n, max_blocks]."""
    if table.dtype != torch.int32 or table.dim() != 2 or table.shape[0] != n or table.device != device:
        raise TypeError(f"block table: expected an int32 tensor [{n}, blocks] on {device}")
    if table.shape[1] > 1 and table.stride(1) != 1:
        raise TypeError("block table: rows must be contiguous")
    stride = table.stride(0) if n > 1 else table.shape[1]
    if stride < table.shape[1]:
        raise TypeError("block table: rows overlap")
    return stride


def _stream(stream, device: torch.device) -> C.c_void_p:
    return C.c_void_p((stream if stream is not None else torch.cuda.current_stream(device)).cuda_stream)


def _ptr(t: torch.Tensor | None):
    return None if t is None else C.c_void_p(t.data_ptr())


# ---- rotary positions ----------------------------------------------------------------


class Rope:
    """A model's rotary frequencies (cpq_rope_params: ggml_rope_ext's parameters)."""

    def __init__(self, n_dims: int, mode: int = ROPE_HALF, base: float = 10000.0, freq_scale: float = 1.0,
                 ext_factor: float = 0.0, attn_factor: float = 1.0, beta_fast: float = 32.0, beta_slow: float = 1.0,
                 n_ctx_orig: int = 0, freq_factors=None):
        self.handle = C.c_void_p()
        self.n_dims, self.mode = n_dims, mode
        ff = None
        if freq_factors is not None:
            values = [float(f) for f in freq_factors]
            if len(values) != n_dims // 2:
                raise ValueError(f"{len(values)} frequency factors for {n_dims // 2} pairs")
            ff = (C.c_double * len(values))(*values)
        p = CpqRopeParams(n_dims, mode, base, freq_scale, ext_factor, attn_factor, beta_fast, beta_slow, n_ctx_orig, ff)
        check(lib().cpq_rope_create(C.byref(p), C.byref(self.handle)), "cpq_rope_create")

    def __del__(self):
        if getattr(self, "handle", None):
            lib().cpq_rope_destroy(self.handle)
            self.handle = C.c_void_p()


def rope(table: Rope, xs: list[torch.Tensor], pos: torch.Tensor, outs: list[torch.Tensor] | None = None,
         stream=None) -> list[torch.Tensor]:
    """xs (q and k, up to 4 tensors [T, heads, D] of one type) rotated to pos [T] (int32).
    outs may be xs itself: rotated in place."""
    if not 1 <= len(xs) <= 4:
        raise ValueError(f"{len(xs)} tensors (1 to 4)")
    dev = xs[0].device
    if outs is None:
        outs = [torch.empty_like(x, memory_format=torch.contiguous_format) for x in xs]
    if len(outs) != len(xs):
        raise ValueError(f"{len(outs)} outputs for {len(xs)} tensors")
    _check_ints(pos, "pos", torch.int32, dev, xs[0].shape[0])
    for t in [*xs, *outs]:
        _same_device(dev, tensor=t)
    n = len(xs)
    xd, yd = [_desc(t, "rope") for t in xs], [_desc(t, "rope out") for t in outs]
    xa = (C.POINTER(CpqTensor) * n)(*[C.pointer(d) for d in xd])
    ya = (C.POINTER(CpqTensor) * n)(*[C.pointer(d) for d in yd])
    with torch.cuda.device(dev):
        check(lib().cpq_rope_apply(table.handle, xa, ya, n, _ptr(pos), _stream(stream, dev)), "cpq_rope_apply")
    return outs


# ---- the cache -----------------------------------------------------------------------


@dataclass
class KvCache:
    """A pool of pages: k and v codes [n_pages, n_head_kv, block, D] (int8 or float8_e4m3fn),
    k_scale and v_scale [n_pages, n_head_kv] (float32)."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor

    def __post_init__(self):
        k = self.k
        if not k.is_cuda or k.dim() != 4 or k.dtype not in _KV_TYPES:
            raise TypeError("KvCache: codes must be a CUDA tensor [pages, heads, block, D] of int8 or float8_e4m3fn")
        for name, t, shape, dtype in (("k", k, k.shape, k.dtype), ("v", self.v, k.shape, k.dtype),
                                      ("k_scale", self.k_scale, k.shape[:2], torch.float32),
                                      ("v_scale", self.v_scale, k.shape[:2], torch.float32)):
            if t.shape != shape or t.dtype != dtype or t.device != k.device or not t.is_contiguous():
                raise TypeError(f"KvCache: {name} must be a contiguous {dtype} tensor {tuple(shape)} on {k.device}")

    @classmethod
    def empty(cls, n_pages: int, n_head_kv: int, head_dim: int, block: int = 64, fmt: int = KV_INT8,
              device="cuda") -> "KvCache":
        """A new pool (its contents are whatever the memory holds: no page needs initialising)."""
        shape = (n_pages, n_head_kv, block, head_dim)
        codes = [torch.empty(shape, dtype=torch.uint8, device=device).view(_KV_DTYPES[fmt]) for _ in range(2)]
        scales = [torch.empty(shape[:2], dtype=torch.float32, device=device) for _ in range(2)]
        return cls(codes[0], codes[1], scales[0], scales[1])

    @classmethod
    def wrap(cls, k, v, k_scale, v_scale) -> "KvCache":
        """A pool over tensors that exist already."""
        return cls(k, v, k_scale, v_scale)

    @property
    def n_pages(self) -> int:
        return self.k.shape[0]

    @property
    def n_head_kv(self) -> int:
        return self.k.shape[1]

    @property
    def block(self) -> int:
        return self.k.shape[2]

    @property
    def head_dim(self) -> int:
        return self.k.shape[3]

    @property
    def device(self) -> torch.device:
        return self.k.device

    def desc(self) -> CpqKvCache:
        return CpqKvCache(_KV_TYPES[self.k.dtype], self.head_dim, self.n_head_kv, self.block, self.n_pages,
                          self.k.data_ptr(), self.v.data_ptr(), self.k_scale.data_ptr(), self.v_scale.data_ptr())


@dataclass
class Slots:
    """Where a step's rows go (cpq_kv_slots)."""

    seq_start: torch.Tensor  # int32 [n + 1]
    kv_len: torch.Tensor     # int32 [n]; 0 for a request that could not be served
    pos: torch.Tensor        # int32 [n_rows]
    slot: torch.Tensor       # int64 [n_rows], -1 for rows without a place


def kv_slots(ctx_len: torch.Tensor, new_len: torch.Tensor, table: torch.Tensor, free_pages: torch.Tensor,
             taken: torch.Tensor, *, block: int, n_rows: int, taken_out: torch.Tensor | None = None,
             out: Slots | None = None, stream=None) -> Slots:
    """Gives the requests' new tokens their pages (into table, from free_pages[taken:]) and
    slots. taken_out (default: taken itself) receives the pages of free_pages now in use."""
    dev, n = ctx_len.device, ctx_len.numel()
    taken_out = taken if taken_out is None else taken_out
    if out is None:
        ints = lambda m, dt=torch.int32: torch.empty(m, dtype=dt, device=dev)  # noqa: E731
        out = Slots(ints(n + 1), ints(n), ints(n_rows), ints(n_rows, torch.int64))
    for name, t, dt, m in (("ctx_len", ctx_len, torch.int32, n), ("new_len", new_len, torch.int32, n),
                           ("free_pages", free_pages, torch.int32, None), ("taken", taken, torch.int32, 1),
                           ("taken_out", taken_out, torch.int32, 1), ("seq_start", out.seq_start, torch.int32, n + 1),
                           ("kv_len", out.kv_len, torch.int32, n), ("pos", out.pos, torch.int32, n_rows),
                           ("slot", out.slot, torch.int64, n_rows)):
        _check_ints(t, name, dt, dev, m)
    if not ctx_len.is_cuda:
        raise TypeError("kv_slots: expected CUDA tensors")
    stride = _table(table, n, dev)
    a = CpqKvSlotArgs(ctx_len.data_ptr(), new_len.data_ptr(), n, table.data_ptr(), stride, table.shape[1], block,
                      free_pages.data_ptr(), free_pages.numel(), taken.data_ptr(), taken_out.data_ptr(),
                      out.seq_start.data_ptr(), out.kv_len.data_ptr(), out.pos.data_ptr(), out.slot.data_ptr(), n_rows)
    with torch.cuda.device(dev):
        check(lib().cpq_kv_slots(C.byref(a), _stream(stream, dev)), "cpq_kv_slots")
    return out


def kv_append(cache: KvCache, k: torch.Tensor, v: torch.Tensor, slot: torch.Tensor, stream=None) -> None:
    """Writes rows k, v [T, n_head_kv, D] to their slots [T] (int64; rows outside the pool are
    skipped). The rows of a call that go to one page must be consecutive, with consecutive slots."""
    dev = cache.device
    _same_device(dev, k=k, v=v)
    _check_ints(slot, "slot", torch.int64, dev, k.shape[0])
    cd, kd, vd = cache.desc(), _desc(k, "k"), _desc(v, "v")
    with torch.cuda.device(dev):
        check(lib().cpq_kv_append(C.byref(cd), C.byref(kd), C.byref(vd), _ptr(slot), _stream(stream, dev)),
              "cpq_kv_append")


def kv_gather(cache: KvCache, slot: torch.Tensor, dtype: torch.dtype = torch.float32,
              outs: tuple[torch.Tensor, torch.Tensor] | None = None, stream=None) -> tuple[torch.Tensor, torch.Tensor]:
    """The values of slots [T] (int64) as k, v [T, n_head_kv, D]; rows outside the pool are zeros."""
    dev = cache.device
    _check_ints(slot, "slot", torch.int64, dev)
    if outs is None:
        shape = (slot.numel(), cache.n_head_kv, cache.head_dim)
        outs = (torch.empty(shape, dtype=dtype, device=dev), torch.empty(shape, dtype=dtype, device=dev))
    k, v = outs
    _same_device(dev, k=k, v=v)
    if k.shape[0] != slot.numel():
        raise ValueError(f"{k.shape[0]} rows for {slot.numel()} slots")
    cd, kd, vd = cache.desc(), _desc(k, "k"), _desc(v, "v")
    with torch.cuda.device(dev):
        check(lib().cpq_kv_gather(C.byref(cd), _ptr(slot), C.byref(kd), C.byref(vd), _stream(stream, dev)),
              "cpq_kv_gather")
    return k, v


# ---- attention -----------------------------------------------------------------------


def paged_attn(q: torch.Tensor, cache: KvCache, table: torch.Tensor, seq_start: torch.Tensor, kv_len: torch.Tensor, *,
               scale: float | None = None, causal: bool = True, out: torch.Tensor | None = None,
               return_lse: bool = False, lse: torch.Tensor | None = None, workspace: torch.Tensor | None = None,
               stream=None):
    """softmax(scale * q K^T) V of rows q [T, n_head, D] over the cached keys of their sequences
    (scale: 1 / sqrt(D) by default). Rows outside every sequence are left as they are in out
    (undefined when it is made here). Returns out, or (out, lse [T, n_head]).

    The workspace (uint8, cpq_paged_attn_workspace_size bytes) comes from torch's allocator on
    the call's stream unless one is given."""
    dev, n = cache.device, kv_len.numel()
    _same_device(dev, q=q)
    _check_ints(seq_start, "seq_start", torch.int32, dev, n + 1)
    _check_ints(kv_len, "kv_len", torch.int32, dev, n)
    stride = _table(table, n, dev)
    qd, cd = _desc(q, "q"), cache.desc()
    if scale is None:
        scale = cache.head_dim ** -0.5
    s = stream if stream is not None else torch.cuda.current_stream(dev)
    with torch.cuda.device(dev), torch.cuda.stream(s):
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=dev)
        if lse is None and return_lse:
            lse = torch.empty(q.shape[:2], dtype=torch.float32, device=dev)
        need = lib().cpq_paged_attn_workspace_size(C.byref(cd), C.byref(qd), n)
        if workspace is None:
            workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    _same_device(dev, out=out, lse=lse, workspace=workspace)
    if lse is not None and (lse.dtype != torch.float32 or lse.shape != q.shape[:2] or not lse.is_contiguous()):
        raise TypeError(f"lse: expected a contiguous float32 tensor {tuple(q.shape[:2])}")
    if workspace.dtype != torch.uint8 or not workspace.is_contiguous():
        raise TypeError("workspace: expected a contiguous uint8 tensor")
    od = _desc(out, "out")
    seqs = CpqAttnSeqs(seq_start.data_ptr(), kv_len.data_ptr(), table.data_ptr(), stride, n, table.shape[1])
    with torch.cuda.device(dev):
        check(lib().cpq_paged_attn(C.byref(qd), C.byref(cd), C.byref(seqs), scale, 1 if causal else 0, C.byref(od),
                                   _ptr(lse), _ptr(workspace), workspace.numel(), C.c_void_p(s.cuda_stream)),
              "cpq_paged_attn")
    return (out, lse) if return_lse else out
