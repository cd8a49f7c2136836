"""Host-side surface of the attention core over libcpq (include/cpq.h: cpq_rope_*,
cpq_kv_*, cpq_paged_attn): what stands between the q/k/v projections and
attn_output in an attention layer (crates/codpiece-model/src/qwen35.rs:3000-3197),
but for the norms of q and k and the gate beside q.

q, k and v are CUDA tensors [tokens, heads, D] of float32, float16 or bfloat16
whose rows of D are contiguous (any other strides: views into a projection's
output). Keys and values live in a :class:`KvCache`, a pool of pages of 8-bit
codes with one scale per page and kv head. A step over requests of different
lengths:

    s = kv_slots(ctx_len, new_len, table, free_pages, taken, block=cache.block, n_rows=T, taken_out=taken_next)
    rope(table_of_frequencies, [q, k], s.pos, [q, k])
    kv_append(cache, k, v, s.slot)
    out = paged_attn(q, cache, table, s.seq_start, s.kv_len)

Every call goes to the device of its tensors, on the given stream or that
device's current one. There is no CPU or PyTorch fallback.
"""
from __future__ import annotations

import ctypes as C
import struct
import threading
from contextlib import nullcontext
from dataclasses import dataclass

import torch

from . import _lib
from ._lib import CpqAttnSeqs, CpqKvCache, CpqKvSlotArgs, CpqRopeParams, CpqTensor, check, lib

ROPE_INTERLEAVED, ROPE_HALF = 0, 1
KV_INT8, KV_E4M3 = 0, 1

_ACT_TYPES = {torch.float32: _lib.TYPE_F32, torch.float16: _lib.TYPE_F16, torch.bfloat16: _lib.TYPE_BF16}
_KV_TYPES = {torch.int8: KV_INT8, torch.float8_e4m3fn: KV_E4M3}
_KV_DTYPES = {KV_INT8: torch.int8, KV_E4M3: torch.float8_e4m3fn}


# The calls of this module stand between kernels of a few microseconds, so they are kept cheap: descriptors are
# packed as bytes into a per-thread scratch (a thread's call has returned before its next one packs) and passed by
# address, and the device is switched only when the tensors' is not the current one.
_TENSOR = struct.Struct("i4x4q4QQ")      # cpq_tensor
_CACHE = struct.Struct("4iq4Q")          # cpq_kv_cache
_SEQS = struct.Struct("3Q2qi4x")         # cpq_attn_seqs
_SLOT_ARGS = struct.Struct("2QqQq2iQqQ5Qq")  # cpq_kv_slot_args
assert (_TENSOR.size, _CACHE.size, _SEQS.size, _SLOT_ARGS.size) == tuple(
    C.sizeof(t) for t in (CpqTensor, CpqKvCache, CpqAttnSeqs, CpqKvSlotArgs))
_SLOTS = 8  # tensor descriptors of a call at most


class _Scratch(threading.local):
    def __init__(self):
        self.buf = C.create_string_buffer(_SLOTS * _TENSOR.size + 3 * 128 + _SLOTS * 8)
        base = C.addressof(self.buf)
        self.tensor = [base + i * _TENSOR.size for i in range(_SLOTS)]
        self.at = _SLOTS * _TENSOR.size  # cache, sequences, slot arguments: 128 bytes each
        self.cache, self.seqs, self.slots = (base + self.at + 128 * i for i in range(3))
        # arrays of pointers to the descriptors: 0-3 inputs, 4-7 outputs
        struct.pack_into(f"{_SLOTS}Q", self.buf, self.at + 384, *self.tensor)
        self.inputs, self.outputs = base + self.at + 384, base + self.at + 384 + 32


_scratch = _Scratch()
_fast: C.CDLL | None = None


def _calls() -> C.CDLL:
    """The library with these entry points taking addresses as integers."""
    global _fast
    if _fast is None:
        lib()
        f = C.CDLL(str(_lib.LIB_PATH))
        vp = C.c_void_p
        for name, args in (("cpq_rope_apply", [vp, vp, vp, C.c_int, vp, vp]), ("cpq_kv_slots", [vp, vp]),
                           ("cpq_kv_append", [vp] * 5), ("cpq_kv_gather", [vp] * 5),
                           ("cpq_paged_attn", [vp, vp, vp, C.c_float, C.c_int32, vp, vp, vp, C.c_size_t, vp])):
            getattr(f, name).argtypes, getattr(f, name).restype = args, C.c_int
        f.cpq_paged_attn_workspace_size.argtypes, f.cpq_paged_attn_workspace_size.restype = [vp, vp, C.c_int64], C.c_size_t
        _fast = f
    return _fast


def _put(sc: _Scratch, i: int, t: torch.Tensor, what: str) -> int:
    """Packs descriptor i from a [tokens, heads, D] activation tensor (ne = [D, heads, tokens, 1]); its address."""
    typ = _ACT_TYPES.get(t.dtype)
    if typ is None or not t.is_cuda or t.dim() != 3:
        raise TypeError(f"{what}: expected a CUDA tensor [tokens, heads, D] of float32, float16 or bfloat16")
    n, h, d = t.shape
    sn, sh, sd = t.stride()
    if sd != 1 and d != 1:
        raise TypeError(f"{what}: rows must be contiguous (stride {sd} along the last dimension)")
    b = 4 if typ == _lib.TYPE_F32 else 2
    _TENSOR.pack_into(sc.buf, i * _TENSOR.size, typ, d, h, n, 1, b, sh * b, sn * b, sn * b * n, t.data_ptr())
    return sc.tensor[i]


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
    blocks = table.shape[1]
    row, col = table.stride()
    if blocks > 1 and col != 1:
        raise TypeError("block table: rows must be contiguous")
    stride = row if n > 1 else blocks
    if stride < blocks:
        raise TypeError("block table: rows overlap")
    return stride


_same = nullcontext()


def _on(device: torch.device):
    """The device's context, when it is not the current one."""
    return _same if torch.cuda.current_device() == device.index else torch.cuda.device(device)


# the device's current stream without the Stream object around it (2 us a call), where torch has the call
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(stream, device: torch.device) -> int:
    if stream is not None:
        return stream.cuda_stream
    return _raw_stream(device.index) if _raw_stream is not None else torch.cuda.current_stream(device).cuda_stream


def _allocating(stream):
    """Tensors made under this belong to the call's stream."""
    return _same if stream is None else torch.cuda.stream(stream)


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


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
        if getattr(self, "handle", None) and lib is not None:  # (None while the interpreter shuts down)
            lib().cpq_rope_destroy(self.handle)
            self.handle = C.c_void_p()


def rope(table: Rope, xs: list[torch.Tensor], pos: torch.Tensor, outs: list[torch.Tensor] | None = None,
         stream=None) -> list[torch.Tensor]:
    """xs (q and k, up to 4 tensors [T, heads, D] of one type) rotated to pos [T] (int32).
    outs may be xs itself: rotated in place. No tensor may be given twice."""
    n = len(xs)
    if not 1 <= n <= 4:
        raise ValueError(f"{n} tensors (1 to 4)")
    dev = xs[0].device
    if outs is None:
        with _allocating(stream):
            outs = [torch.empty_like(x) for x in xs]
    if len(outs) != n:
        raise ValueError(f"{len(outs)} outputs for {n} tensors")
    _check_ints(pos, "pos", torch.int32, dev, xs[0].shape[0])
    sc = _scratch
    for i in range(n):
        _put(sc, i, xs[i], "rope")
        _put(sc, 4 + i, outs[i], "rope out")
        if xs[i].device != dev or outs[i].device != dev:
            raise ValueError(f"rope: tensors on {dev} and another device")
    with _on(dev):
        check(_calls().cpq_rope_apply(table.handle, sc.inputs, sc.outputs, n, pos.data_ptr(), _stream(stream, dev)), "cpq_rope_apply")
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

    def _put(self, sc: _Scratch) -> int:
        p, h, b, d = self.k.shape
        _CACHE.pack_into(sc.buf, sc.at, _KV_TYPES[self.k.dtype], d, h, b, p, self.k.data_ptr(), self.v.data_ptr(),
                         self.k_scale.data_ptr(), self.v_scale.data_ptr())
        return sc.cache


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
    slots. taken_out (default: taken itself) receives the pages of free_pages now in use;
    a tensor of its own lets many rows (a long prompt) be placed by many CTAs instead of one
    (60000 rows: 6.4 us, 72 in place; a step of single tokens takes the same)."""
    dev, n = ctx_len.device, ctx_len.numel()
    taken_out = taken if taken_out is None else taken_out
    if out is None:
        with _allocating(stream):
            out = Slots(torch.empty(n + 1, dtype=torch.int32, device=dev), torch.empty(n, dtype=torch.int32, device=dev),
                        torch.empty(n_rows, dtype=torch.int32, device=dev), torch.empty(n_rows, dtype=torch.int64, device=dev))
    else:
        for name, t, dt, m in (("seq_start", out.seq_start, torch.int32, n + 1), ("kv_len", out.kv_len, torch.int32, n),
                               ("pos", out.pos, torch.int32, n_rows), ("slot", out.slot, torch.int64, n_rows)):
            _check_ints(t, name, dt, dev, m)
    for name, t, m in (("ctx_len", ctx_len, n), ("new_len", new_len, n), ("free_pages", free_pages, None), ("taken", taken, 1),
                       ("taken_out", taken_out, 1)):
        _check_ints(t, name, torch.int32, dev, m)
    if not ctx_len.is_cuda:
        raise TypeError("kv_slots: expected CUDA tensors")
    stride = _table(table, n, dev)
    sc = _scratch
    _SLOT_ARGS.pack_into(sc.buf, sc.at + 256, ctx_len.data_ptr(), new_len.data_ptr(), n, table.data_ptr(), stride,
                         table.shape[1], block, free_pages.data_ptr(), free_pages.numel(), taken.data_ptr(),
                         taken_out.data_ptr(), out.seq_start.data_ptr(), out.kv_len.data_ptr(), out.pos.data_ptr(),
                         out.slot.data_ptr(), n_rows)
    with _on(dev):
        check(_calls().cpq_kv_slots(sc.slots, _stream(stream, dev)), "cpq_kv_slots")
    return out


def kv_append(cache: KvCache, k: torch.Tensor, v: torch.Tensor, slot: torch.Tensor, stream=None) -> None:
    """Writes rows k, v [T, n_head_kv, D] to their slots [T] (int64; rows outside the pool are
    skipped). The rows of a call that go to one page must be consecutive, with consecutive slots;
    a page's first rows begin at its first place, and its scale only grows until they do again."""
    dev = cache.device
    _same_device(dev, k=k, v=v)
    _check_ints(slot, "slot", torch.int64, dev, k.shape[0])
    sc = _scratch
    with _on(dev):
        check(_calls().cpq_kv_append(cache._put(sc), _put(sc, 0, k, "k"), _put(sc, 1, v, "v"), slot.data_ptr(),
                                     _stream(stream, dev)), "cpq_kv_append")


def kv_gather(cache: KvCache, slot: torch.Tensor, dtype: torch.dtype = torch.float32,
              outs: tuple[torch.Tensor, torch.Tensor] | None = None, stream=None) -> tuple[torch.Tensor, torch.Tensor]:
    """The values of slots [T] (int64) as k, v [T, n_head_kv, D]; rows outside the pool are zeros."""
    dev = cache.device
    _check_ints(slot, "slot", torch.int64, dev)
    n = slot.numel()
    if outs is None:
        _, h, _, d = cache.k.shape
        with _allocating(stream):
            outs = (torch.empty(n, h, d, dtype=dtype, device=dev), torch.empty(n, h, d, dtype=dtype, device=dev))
    k, v = outs
    _same_device(dev, k=k, v=v)
    if k.shape[0] != n:
        raise ValueError(f"{k.shape[0]} rows for {n} slots")
    sc = _scratch
    with _on(dev):
        check(_calls().cpq_kv_gather(cache._put(sc), slot.data_ptr(), _put(sc, 0, k, "k"), _put(sc, 1, v, "v"),
                                     _stream(stream, dev)), "cpq_kv_gather")
    return k, v


# ---- attention -----------------------------------------------------------------------


def paged_attn(q: torch.Tensor, cache: KvCache, table: torch.Tensor, seq_start: torch.Tensor, kv_len: torch.Tensor, *,
               scale: float | None = None, causal: bool = True, out: torch.Tensor | None = None,
               return_lse: bool = False, lse: torch.Tensor | None = None, workspace: torch.Tensor | None = None,
               stream=None):
    """softmax(scale * q K^T) V of rows q [T, n_head, D] over the cached keys of their sequences
    (scale: 1 / sqrt(D) by default). Rows outside every sequence are left as they are in out
    (undefined when it is made here). Returns out, or (out, lse [T, n_head]). One kernel is chosen
    for the whole call by the mean rows per sequence (and, for a few, the table's width): batches of
    single tokens beside long chunks are faster in two calls.

    The workspace (uint8, cpq_paged_attn_workspace_size bytes) comes from torch's allocator on
    the call's stream unless one is given."""
    dev, n = cache.device, kv_len.numel()
    _same_device(dev, q=q)
    _check_ints(seq_start, "seq_start", torch.int32, dev, n + 1)
    _check_ints(kv_len, "kv_len", torch.int32, dev, n)
    stride = _table(table, n, dev)
    sc = _scratch
    qd, cd = _put(sc, 0, q, "q"), cache._put(sc)
    if scale is None:
        scale = cache.head_dim ** -0.5
    calls = _calls()
    with _on(dev):
        with _allocating(stream):
            if out is None:
                out = torch.empty_like(q)
            if lse is None and return_lse:
                lse = torch.empty(q.shape[0], q.shape[1], dtype=torch.float32, device=dev)
            if workspace is None:
                workspace = torch.empty(calls.cpq_paged_attn_workspace_size(cd, qd, n), dtype=torch.uint8, device=dev)
        _same_device(dev, out=out, lse=lse, workspace=workspace)
        if lse is not None and (lse.dtype != torch.float32 or lse.shape != q.shape[:2] or not lse.is_contiguous()):
            raise TypeError(f"lse: expected a contiguous float32 tensor {tuple(q.shape[:2])}")
        if workspace.dtype != torch.uint8 or not workspace.is_contiguous():
            raise TypeError("workspace: expected a contiguous uint8 tensor")
        od = _put(sc, 1, out, "out")
        _SEQS.pack_into(sc.buf, sc.at + 128, seq_start.data_ptr(), kv_len.data_ptr(), table.data_ptr(), stride, n, table.shape[1])
        check(calls.cpq_paged_attn(qd, cd, sc.seqs, scale, 1 if causal else 0, od, _ptr(lse), workspace.data_ptr(),
                                   workspace.numel(), _stream(stream, dev)), "cpq_paged_attn")
    return (out, lse) if return_lse else out
