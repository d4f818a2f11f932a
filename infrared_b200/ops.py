"""Tensor-level entry points over the C ABI (device memory and streams from PyTorch).

Every function takes CUDA tensors, checks shapes/dtypes/contiguity on the
host, and launches on ``torch.cuda.current_stream()`` without synchronising
or allocating anything but its outputs (which the caller may pass in), so
each one can run inside ``torch.cuda.graph`` capture. Device-side errors
(bad block ids, slots, metadata) are accumulated in a per-device int32 flag
word that :func:`check_device_errors` reads and clears.

There is no CPU path: CPU tensors raise ``ValueError``.
"""

from __future__ import annotations

import functools
import threading

import torch

from . import _lib
from ._lib import DEVERR_BITS, DecodeShape, check

_DTYPES = {
    torch.float32: _lib.IR_DTYPE_F32,
    torch.bfloat16: _lib.IR_DTYPE_BF16,
    torch.float16: _lib.IR_DTYPE_F16,
}

# element types of 8-bit pools
_KV_FORMATS = {
    torch.float8_e4m3fn: _lib.IR_KV_E4M3,
    torch.int8: _lib.IR_KV_INT8,
}


class DeviceError(RuntimeError):
    """Errors a kernel recorded on the device (see ``IR_DEVERR_*``)."""

    def __init__(self, bits: int):
        names = [n for b, n in DEVERR_BITS.items() if bits & b]
        super().__init__(f"infrared_b200 device error 0x{bits:x}: {', '.join(names)}")
        self.bits = bits


_state_lock = threading.Lock()
_err_flags: dict[int, torch.Tensor] = {}
_workspaces: dict[int, torch.Tensor] = {}


def _on_tensor_device(fn):
    """Run ``fn`` with its first tensor argument's device current.

    A kernel launch into a stream of a device other than the calling thread's
    current one fails, and callers such as infrared's engine run their loop
    in a worker thread whose current device is the process default (0);
    this switches to the tensors' device for the call when they differ."""

    @functools.wraps(fn)
    def wrapper(first, *args, **kwargs):
        idx = first.device.index if isinstance(first, torch.Tensor) and first.is_cuda else None
        if idx is not None and idx != torch.cuda.current_device():
            with torch.cuda.device(idx):
                return fn(first, *args, **kwargs)
        return fn(first, *args, **kwargs)

    return wrapper


def dtype_code(dtype: torch.dtype) -> int:
    try:
        return _DTYPES[dtype]
    except KeyError:
        raise _lib.UnsupportedShape(_lib.IR_ERR_UNSUPPORTED, f"dtype {dtype} not supported")


def _dev_index(t: torch.Tensor) -> int:
    if not t.is_cuda:
        raise ValueError("infrared_b200 kernels take CUDA tensors (no CPU path)")
    return t.device.index if t.device.index is not None else torch.cuda.current_device()


def _index_of(device) -> int:
    if device is None:
        return torch.cuda.current_device()
    if isinstance(device, int):
        return device
    d = torch.device(device)
    return d.index if d.index is not None else torch.cuda.current_device()


def error_flag(device: torch.device | int | None = None) -> torch.Tensor:
    """The per-device int32 error word the kernels OR their error bits into."""
    idx = _index_of(device)
    t = _err_flags.get(idx)
    if t is not None:
        return t
    with _state_lock:
        t = _err_flags.get(idx)
        if t is None:
            t = torch.zeros(1, dtype=torch.int32, device=torch.device("cuda", idx))
            _err_flags[idx] = t
    return t


def check_device_errors(device=None, clear: bool = True) -> None:
    """Synchronise on the flag word; raise :class:`DeviceError` if any bit is set."""
    flag = error_flag(device)
    bits = int(flag.item())
    if bits and clear:
        flag.zero_()
    if bits:
        raise DeviceError(bits)


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _stream(device_index: int) -> int:
    return torch.cuda.current_stream(device_index).cuda_stream


# What a zeroed decode workspace turns on by default (ir_decode_shape.flags).
# Both features are opt-in (decode_workspace(dynamic=..., inline_merge=...)):
# on B200 the static shares with the separate merge kernel measured faster
# on every benchmark shape.
DYNAMIC_TAIL_DEFAULT = False
INLINE_MERGE_DEFAULT = False


def _default_flags(dynamic: bool | None = None, inline_merge: bool | None = None) -> int:
    dyn = DYNAMIC_TAIL_DEFAULT if dynamic is None else dynamic
    inl = INLINE_MERGE_DEFAULT if inline_merge is None else inline_merge
    return (_lib.IR_DECODE_DYNAMIC_TAIL if dyn else 0) | \
        (_lib.IR_DECODE_INLINE_MERGE if inl else 0)


def decode_workspace(nbytes: int, device, dynamic: bool | None = None,
                     inline_merge: bool | None = None) -> torch.Tensor:
    """A decode workspace of ``nbytes`` (at least 1 MiB) on ``device``, zero
    filled, marked with the features the decode calls given it may use:
    ``dynamic`` (``IR_DECODE_DYNAMIC_TAIL``: the last part of the tiles handed
    out as claimed units) and ``inline_merge`` (``IR_DECODE_INLINE_MERGE``:
    rows of at most 4 pieces merged in the decode kernel); None takes the
    module defaults. The kernels leave the header they count in zero after
    every call. Any other tensor given as a workspace gets neither."""
    t = torch.zeros(max(int(nbytes), 1 << 20), dtype=torch.uint8,
                    device=torch.device("cuda", _index_of(device)))
    # allocated inside a graph capture the zeroing only runs at replay: such
    # a workspace uses neither feature
    t._irb_flags = 0 if torch.cuda.is_current_stream_capturing() else \
        _default_flags(dynamic, inline_merge)
    return t


def _flags_of(ws: torch.Tensor | None) -> int:
    """Flags a call may ask for with this workspace (None: the cached one's)."""
    if ws is None:
        return _default_flags()
    return int(getattr(ws, "_irb_flags", 0))


def workspace(nbytes: int, device_index: int) -> torch.Tensor:
    """A cached, growing per-device workspace buffer (256-byte aligned, header
    zeroed: see :func:`decode_workspace`)."""
    t = _workspaces.get(device_index)
    if t is not None and t.numel() >= nbytes:
        return t
    with _state_lock:
        t = _workspaces.get(device_index)
        if t is None or t.numel() < nbytes:
            t = decode_workspace(nbytes, device_index)
            _workspaces[device_index] = t
    return t


def set_decode_path(path: int) -> None:
    """0 = automatic kernel choice, 1 = CUDA-core kernel, 2 = TMA kernel,
    3 = TMA kernel with one copy per (kv head, column half)."""
    check(_lib.load().ir_set_decode_path(path))
    _plans.clear()   # cached workspace sizes depend on the kernel choice
    _decode_q8_plans.clear()


# --- pool scatter / gather ----------------------------------------------------


def _check_pool(pool: torch.Tensor, name: str) -> None:
    if pool.dim() != 3 or not pool.is_contiguous():
        raise ValueError(f"{name} must be a contiguous [num_slots, Hkv, D] tensor")


@_on_tensor_device
def cache_write(k: torch.Tensor, v: torch.Tensor, k_pool: torch.Tensor,
                v_pool: torch.Tensor, slot_mapping: torch.Tensor) -> None:
    """``k_pool[slot_mapping] = k; v_pool[slot_mapping] = v`` (one layer's pools)."""
    dev = _dev_index(k_pool)
    _check_pool(k_pool, "k_pool")
    _check_pool(v_pool, "v_pool")
    if k_pool.shape != v_pool.shape or k_pool.dtype != v_pool.dtype:
        raise ValueError("k_pool and v_pool differ")
    n = slot_mapping.numel()
    hkv, d = k_pool.shape[1], k_pool.shape[2]
    k = k.reshape(n, hkv, d)
    v = v.reshape(n, hkv, d)
    for t, nm in ((k, "k"), (v, "v")):
        if t.dtype != k_pool.dtype or t.device != k_pool.device:
            raise ValueError(f"{nm} must match the pool's dtype and device")
        if n and (t.stride(2) != 1 or t.stride(1) != d):
            raise ValueError(f"{nm} rows must be [Hkv, D] contiguous")
    slots = slot_mapping.reshape(-1)
    if slots.dtype != torch.int64 or not slots.is_contiguous() or slots.device != k_pool.device:
        raise ValueError("slot_mapping must be a contiguous int64 tensor on the pool's device")
    if n == 0:
        return
    lib = _lib.load()
    check(lib.ir_cache_write(
        k.data_ptr(), v.data_ptr(), k.stride(0), v.stride(0), k_pool.data_ptr(),
        v_pool.data_ptr(), slots.data_ptr(), n, hkv, d, k_pool.shape[0],
        dtype_code(k_pool.dtype), error_flag(dev).data_ptr(), _stream(dev)))


@_on_tensor_device
def cache_gather(pool: torch.Tensor, slots: torch.Tensor) -> torch.Tensor:
    """``pool[slots]`` for a 1-D or 2-D int64 slot tensor -> ``[*slots.shape, Hkv, D]``."""
    dev = _dev_index(pool)
    _check_pool(pool, "pool")
    flat = slots.reshape(-1)
    if flat.dtype != torch.int64 or flat.device != pool.device:
        raise ValueError("slots must be int64 on the pool's device")
    flat = flat.contiguous()
    out = torch.empty((flat.numel(), pool.shape[1], pool.shape[2]), dtype=pool.dtype,
                      device=pool.device)
    if flat.numel():
        check(_lib.load().ir_cache_gather(
            out.data_ptr(), pool.data_ptr(), flat.data_ptr(), flat.numel(), pool.shape[1],
            pool.shape[2], pool.shape[0], dtype_code(pool.dtype),
            error_flag(dev).data_ptr(), _stream(dev)))
    return out.reshape(*slots.shape, pool.shape[1], pool.shape[2])


@_on_tensor_device
def derive_block_metadata(gather_slots: torch.Tensor, mask: torch.Tensor, block_size: int,
                          block_tables: torch.Tensor | None = None,
                          context_lens: torch.Tensor | None = None):
    """``(gather_slots [B, T], decode mask [B, 1, 1, T]) -> (block_tables, context_lens)``.

    ``block_tables`` is int32 ``[B, ceil(T / block_size)]``, ``context_lens``
    int32 ``[B]``; both may be passed in (e.g. static graph buffers).
    """
    dev = _dev_index(gather_slots)
    if gather_slots.dim() != 2 or gather_slots.dtype != torch.int64:
        raise ValueError("gather_slots must be int64 [B, T]")
    b, t = gather_slots.shape
    if gather_slots.stride(1) != 1:
        gather_slots = gather_slots.contiguous()
    m2 = mask.reshape(b, t) if mask.numel() == b * t else None
    if m2 is None:
        raise ValueError("mask must have B*T elements ([B, 1, 1, T])")
    if m2.stride(1) != 1:
        m2 = m2.contiguous()
    nb = -(-t // block_size)
    if block_tables is None:
        block_tables = torch.empty((b, max(nb, 1)), dtype=torch.int32, device=gather_slots.device)
    if context_lens is None:
        context_lens = torch.empty((b,), dtype=torch.int32, device=gather_slots.device)
    if b:
        check(_lib.load().ir_derive_block_metadata(
            gather_slots.data_ptr(), gather_slots.stride(0), m2.data_ptr(), m2.stride(0),
            dtype_code(m2.dtype), b, t, block_size, block_tables.data_ptr(),
            block_tables.stride(0), context_lens.data_ptr(), error_flag(dev).data_ptr(),
            _stream(dev)))
    return block_tables, context_lens


# --- decode -------------------------------------------------------------------


def _shape(q: torch.Tensor, k_pool: torch.Tensor, block_tables: torch.Tensor,
           block_size: int, scale: float, out_stride: int,
           flags: int = 0) -> DecodeShape:
    b, h, d = q.shape
    hkv = k_pool.shape[1]
    s = DecodeShape()
    s.batch = b
    s.num_heads = h
    s.num_kv_heads = hkv
    s.head_dim = d
    s.block_size = block_size
    s.max_blocks = block_tables.shape[1]
    s.bt_stride = block_tables.stride(0) if block_tables.shape[0] else block_tables.shape[1]
    s.q_stride = q.stride(0)
    s.out_stride = out_stride
    s.num_slots = k_pool.shape[0]
    s.scale = float(scale)
    s.dtype = dtype_code(q.dtype)
    s.flags = flags
    return s


def _check_decode_inputs(q, k_pool, v_pool, block_tables, context_lens):
    _dev_index(q)
    if q.dim() != 3:
        raise ValueError("q must be [B, H, D]")
    if q.stride(2) != 1 or q.stride(1) != q.shape[2]:
        raise ValueError("q rows must be [H, D] contiguous")
    _check_pool(k_pool, "k_pool")
    _check_pool(v_pool, "v_pool")
    if k_pool.shape != v_pool.shape:
        raise ValueError("k_pool and v_pool shapes differ")
    if k_pool.dtype != q.dtype or v_pool.dtype != q.dtype:
        raise ValueError("q and the pools must share a dtype")
    if k_pool.shape[2] != q.shape[2]:
        raise ValueError("head_dim of q and pools differ")
    if block_tables.dtype != torch.int32 or block_tables.dim() != 2 or \
            (block_tables.numel() and block_tables.stride(1) != 1):
        raise ValueError("block_tables must be int32 [B, max_blocks] with unit column stride")
    if context_lens.dtype != torch.int32 or not context_lens.is_contiguous():
        raise ValueError("context_lens must be contiguous int32 [B]")
    if block_tables.shape[0] != q.shape[0] or context_lens.numel() != q.shape[0]:
        raise ValueError("batch sizes of q, block_tables and context_lens differ")
    for t in (k_pool, v_pool, block_tables, context_lens):
        if t.device != q.device:
            raise ValueError("all tensors must be on the same device")


def decode_plan(q, k_pool, block_tables, block_size, scale=1.0, dynamic=False,
                inline_merge=None):
    """``(path, ctas_per_kv_head, workspace_bytes)`` the library picks for this
    call with a workspace from ``decode_workspace(dynamic=..., inline_merge=...)``
    (None: the module default)."""
    s = _shape(q, k_pool, block_tables, block_size, scale, q.shape[1] * q.shape[2],
               _default_flags(dynamic, inline_merge))
    lib = _lib.load()
    path, g = _lib.c_int(), _lib.c_int()
    check(lib.ir_paged_decode_plan(s, path, g))
    return path.value, g.value, lib.ir_paged_decode_workspace_size(s)


def _size_of(s: DecodeShape) -> int:
    lib = _lib.load()
    nbytes = lib.ir_paged_decode_workspace_size(s)
    if nbytes == 0:
        check(lib.ir_paged_decode_plan(s, None, None))
    return nbytes


def _ws_and_shape(make_shape, dev: int, ws: torch.Tensor | None, sized=None):
    """``(shape, workspace)`` of a decode call: the shape asks for the features
    the workspace is marked with (:func:`decode_workspace`; the cached
    per-device workspace has the module defaults unless it was allocated
    inside a graph capture). ``make_shape(flags)`` builds the shape;
    ``sized(flags)`` may return a cached ``(shape, bytes)``."""
    sized = sized or (lambda fl: (make_shape(fl), None))
    if ws is not None:
        s, nbytes = sized(_flags_of(ws))
        nbytes = _size_of(s) if nbytes is None else nbytes
        if ws.numel() < nbytes:
            raise ValueError(f"workspace of {ws.numel()} bytes < {nbytes} needed")
        return s, ws
    want = _flags_of(None)
    s, nbytes = sized(want)
    nbytes = _size_of(s) if nbytes is None else nbytes
    ws = workspace(nbytes, dev)
    got = _flags_of(ws)
    if got != want:   # fewer features need no more bytes
        s, _ = sized(got)
    return s, ws


# Validated call plans of paged_decode, keyed by everything the checks look
# at (shapes, strides, dtypes, devices, block size, scale): a repeated call
# (every layer of every decode step) skips the checks and the shape build.
_plans: dict = {}


def _decode_key(q, k_pool, v_pool, block_tables, context_lens, out, block_size, scale):
    return (q.shape, q.stride(), q.dtype, q.device, k_pool.shape, k_pool.stride(),
            k_pool.dtype, k_pool.device, v_pool.shape, v_pool.stride(), v_pool.dtype,
            v_pool.device, block_tables.shape, block_tables.stride(), block_tables.dtype,
            block_tables.device, context_lens.shape, context_lens.stride(),
            context_lens.dtype, context_lens.device, out.shape, out.stride(), out.dtype,
            block_size, float(scale))


@_on_tensor_device
def paged_decode(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                 block_tables: torch.Tensor, context_lens: torch.Tensor, scale: float,
                 block_size: int, out: torch.Tensor | None = None,
                 ws: torch.Tensor | None = None) -> torch.Tensor:
    """Decode attention: ``q [B, H, D]`` over paged K/V -> ``[B, H, D]`` (q's dtype).

    ``k_pool``/``v_pool`` are one layer's ``[num_slots, Hkv, D]`` pools,
    ``block_tables`` int32 ``[B, max_blocks]`` of block ids, ``context_lens``
    int32 ``[B]``. GQA: query head h reads kv head ``h // (H // Hkv)``.
    """
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    base = _decode_key(q, k_pool, v_pool, block_tables, context_lens, out, block_size, scale)

    def sized(flags):
        key = (base, flags)
        plan = _plans.get(key)
        if plan is None:
            _check_decode_inputs(q, k_pool, v_pool, block_tables, context_lens)
            if out.shape != q.shape or out.dtype != q.dtype or out.stride(2) != 1 or \
                    out.stride(1) != q.shape[2] or out.device != q.device:
                raise ValueError("out must be [B, H, D] with [H, D] contiguous rows")
            sh = _shape(q, k_pool, block_tables, block_size, scale, out.stride(0), flags)
            plan = (sh, _size_of(sh))
            if len(_plans) > 512:
                _plans.clear()
            _plans[key] = plan
        return plan

    dev = _dev_index(q)
    s, ws = _ws_and_shape(None, dev, ws, sized)
    check(_lib.load().ir_paged_decode(
        out.data_ptr(), q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(),
        block_tables.data_ptr(), context_lens.data_ptr(), s, ws.data_ptr(), ws.numel(),
        error_flag(dev).data_ptr(), _stream(dev)))
    return out


@_on_tensor_device
def paged_decode_write(q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor,
                       k_pool: torch.Tensor, v_pool: torch.Tensor,
                       slot_mapping: torch.Tensor, block_tables: torch.Tensor,
                       context_lens: torch.Tensor, scale: float, block_size: int,
                       out: torch.Tensor | None = None,
                       ws: torch.Tensor | None = None) -> torch.Tensor:
    """Cache write of ``k_new/v_new [B, Hkv, D]`` at ``slot_mapping`` fused with decode.

    ``slot_mapping[b]`` must be the slot of position ``context_lens[b] - 1``
    (the new token), as in the engine's decode step; otherwise the device
    error ``WRITE_SLOT`` is raised by :func:`check_device_errors`.
    """
    _check_decode_inputs(q, k_pool, v_pool, block_tables, context_lens)
    dev = _dev_index(q)
    b, hkv, d = q.shape[0], k_pool.shape[1], k_pool.shape[2]
    k_new = k_new.reshape(b, hkv, d)
    v_new = v_new.reshape(b, hkv, d)
    if k_new.stride(0) != v_new.stride(0) or k_new.stride(2) != 1 or k_new.stride(1) != d \
            or v_new.stride(2) != 1 or v_new.stride(1) != d:
        k_new, v_new = k_new.contiguous(), v_new.contiguous()
    if k_new.dtype != q.dtype or v_new.dtype != q.dtype:
        raise ValueError("k_new/v_new must match q's dtype")
    slots = slot_mapping.reshape(-1)
    if slots.dtype != torch.int64 or not slots.is_contiguous() or slots.numel() != b:
        raise ValueError("slot_mapping must be contiguous int64 [B]")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    s, ws = _ws_and_shape(lambda fl: _shape(q, k_pool, block_tables, block_size, scale,
                                            out.stride(0), fl), dev, ws)
    check(_lib.load().ir_paged_decode_write(
        out.data_ptr(), q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(),
        k_new.data_ptr(), v_new.data_ptr(), k_new.stride(0) if b else hkv * d,
        slots.data_ptr(), block_tables.data_ptr(), context_lens.data_ptr(), s,
        ws.data_ptr(), ws.numel(), error_flag(dev).data_ptr(), _stream(dev)))
    return out


@_on_tensor_device
def paged_decode_rope_write(q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor,
                            k_pool: torch.Tensor, v_pool: torch.Tensor,
                            slot_mapping: torch.Tensor, block_tables: torch.Tensor,
                            context_lens: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                            scale: float, block_size: int, out: torch.Tensor | None = None,
                            ws: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`paged_decode_write` with RoPE applied in the kernel.

    ``q [B, H, D]`` and ``k_new [B, Hkv, D]`` are un-rotated (they may be
    row views of one QKV projection output); ``cos``/``sin`` are fp32
    ``[B, D]`` (or ``[B, 1, D]``) tables at the new token's position, as
    infrared's ``RotaryEmbedding`` returns them (layers.py:121-136). The pool
    and the output equal ``apply_rotary_pos_emb`` (layers.py:79-89) followed
    by :func:`paged_decode_write`, bit for bit.
    """
    _check_decode_inputs(q, k_pool, v_pool, block_tables, context_lens)
    dev = _dev_index(q)
    b, hkv, d = q.shape[0], k_pool.shape[1], k_pool.shape[2]
    k_new = k_new.reshape(b, hkv, d)
    v_new = v_new.reshape(b, hkv, d)
    if k_new.stride(0) != v_new.stride(0) or k_new.stride(2) != 1 or k_new.stride(1) != d \
            or v_new.stride(2) != 1 or v_new.stride(1) != d:
        k_new, v_new = k_new.contiguous(), v_new.contiguous()
    if k_new.dtype != q.dtype or v_new.dtype != q.dtype:
        raise ValueError("k_new/v_new must match q's dtype")
    cos = cos.reshape(b, d) if cos.dim() != 2 else cos
    sin = sin.reshape(b, d) if sin.dim() != 2 else sin
    for name, t in (("cos", cos), ("sin", sin)):
        if t.dtype != torch.float32 or t.device != q.device or t.shape != (b, d) \
                or t.stride(1) != 1:
            raise ValueError(f"{name} must be fp32 [B, D] rows on q's device")
    if cos.stride(0) != sin.stride(0):
        cos, sin = cos.contiguous(), sin.contiguous()
    slots = slot_mapping.reshape(-1)
    if slots.dtype != torch.int64 or not slots.is_contiguous() or slots.numel() != b:
        raise ValueError("slot_mapping must be contiguous int64 [B]")
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    s, ws = _ws_and_shape(lambda fl: _shape(q, k_pool, block_tables, block_size, scale,
                                            out.stride(0), fl), dev, ws)
    check(_lib.load().ir_paged_decode_rope_write(
        out.data_ptr(), q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(),
        k_new.data_ptr(), v_new.data_ptr(), k_new.stride(0) if b else hkv * d,
        slots.data_ptr(), cos.data_ptr(), sin.data_ptr(), cos.stride(0) if b else d,
        block_tables.data_ptr(), context_lens.data_ptr(), s, ws.data_ptr(), ws.numel(),
        error_flag(dev).data_ptr(), _stream(dev)))
    return out


def _rope_rows(cos, sin, b, d, device):
    cos = cos.reshape(b, d) if cos.dim() != 2 else cos
    sin = sin.reshape(b, d) if sin.dim() != 2 else sin
    for name, t in (("cos", cos), ("sin", sin)):
        if t.dtype != torch.float32 or t.device != device or tuple(t.shape) != (b, d) \
                or t.stride(1) != 1:
            raise ValueError(f"{name} must be fp32 [B, D] rows on the tensors' device")
    if cos.stride(0) != sin.stride(0):
        cos, sin = cos.contiguous(), sin.contiguous()
    return cos, sin


@_on_tensor_device
def paged_decode_rope(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                      block_tables: torch.Tensor, context_lens: torch.Tensor,
                      cos: torch.Tensor, sin: torch.Tensor, scale: float, block_size: int,
                      out: torch.Tensor | None = None,
                      ws: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`paged_decode` with RoPE applied to the un-rotated ``q`` in the
    kernel (``cos``/``sin`` fp32 ``[B, D]``): the step's K/V are already in the
    pool (:func:`kv_proj_rope_write`)."""
    _check_decode_inputs(q, k_pool, v_pool, block_tables, context_lens)
    dev = _dev_index(q)
    b, _, d = q.shape
    cos, sin = _rope_rows(cos, sin, b, d, q.device)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    s, ws = _ws_and_shape(lambda fl: _shape(q, k_pool, block_tables, block_size, scale,
                                            out.stride(0), fl), dev, ws)
    check(_lib.load().ir_paged_decode_rope(
        out.data_ptr(), q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), cos.data_ptr(),
        sin.data_ptr(), cos.stride(0) if b else d, block_tables.data_ptr(),
        context_lens.data_ptr(), s, ws.data_ptr(), ws.numel(), error_flag(dev).data_ptr(),
        _stream(dev)))
    return out


@_on_tensor_device
def kv_proj_rope_write(x: torch.Tensor, w_k: torch.Tensor, w_v: torch.Tensor,
                       b_k: torch.Tensor | None, b_v: torch.Tensor | None,
                       cos: torch.Tensor | None, sin: torch.Tensor | None,
                       slot_mapping: torch.Tensor, k_pool: torch.Tensor,
                       v_pool: torch.Tensor) -> None:
    """``k_pool[slot] = rope(x @ w_k^T + b_k)``, ``v_pool[slot] = x @ w_v^T + b_v``
    for every row of ``x [N, hidden]`` in one tensor-core kernel
    (``ir_kv_proj_rope_write``): ``w_k`` / ``w_v`` are the ``nn.Linear``
    weights ``[Hkv * D, hidden]``, ``b_k`` / ``b_v`` their biases (or None),
    ``cos`` / ``sin`` fp32 ``[N, D]`` RoPE rows (or None: no RoPE), the pools
    one layer's ``[num_slots, Hkv, D]``; bf16 / fp16."""
    dev = _dev_index(x)
    _check_pool(k_pool, "k_pool")
    _check_pool(v_pool, "v_pool")
    if k_pool.shape != v_pool.shape or k_pool.dtype != v_pool.dtype:
        raise ValueError("k_pool and v_pool differ")
    hkv, d = k_pool.shape[1], k_pool.shape[2]
    x = x.reshape(-1, x.shape[-1])
    n, hidden = x.shape
    if x.stride(1) != 1:
        x = x.contiguous()
    for name, w in (("w_k", w_k), ("w_v", w_v)):
        if tuple(w.shape) != (hkv * d, hidden) or not w.is_contiguous():
            raise ValueError(f"{name} must be a contiguous [Hkv*D, hidden] weight")
    for name, t in (("x", x), ("w_k", w_k), ("w_v", w_v)):
        if t.dtype != k_pool.dtype or t.device != k_pool.device:
            raise ValueError(f"{name} must match the pool's dtype and device")
    for name, t in (("b_k", b_k), ("b_v", b_v)):
        if t is not None and (t.numel() != hkv * d or t.dtype != k_pool.dtype
                              or not t.is_contiguous() or t.device != k_pool.device):
            raise ValueError(f"{name} must be a contiguous [Hkv*D] bias of the pool's dtype")
    slots = slot_mapping.reshape(-1)
    if slots.dtype != torch.int64 or not slots.is_contiguous() or slots.numel() != n:
        raise ValueError("slot_mapping must be contiguous int64 [N]")
    rs = d
    if cos is not None:
        cos, sin = _rope_rows(cos, sin, n, d, x.device)
        rs = cos.stride(0) if n else d
    check(_lib.load().ir_kv_proj_rope_write(
        x.data_ptr(), x.stride(0) if n else hidden, n, hidden, w_k.data_ptr(), w_v.data_ptr(),
        _ptr(b_k), _ptr(b_v), _ptr(cos), _ptr(sin), rs, slots.data_ptr(), k_pool.data_ptr(),
        v_pool.data_ptr(), k_pool.shape[0], hkv, d, dtype_code(k_pool.dtype),
        error_flag(dev).data_ptr(), _stream(dev)))


@_on_tensor_device
def paged_decode_lse(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                     block_tables: torch.Tensor, context_lens: torch.Tensor, scale: float,
                     block_size: int, o: torch.Tensor | None = None,
                     lse: torch.Tensor | None = None, ws: torch.Tensor | None = None):
    """Partial decode: ``(o [B, H, D] fp32 normalised, lse [B, H] fp32 natural log)``."""
    _check_decode_inputs(q, k_pool, v_pool, block_tables, context_lens)
    dev = _dev_index(q)
    b, h, d = q.shape
    if o is None:
        o = torch.empty((b, h, d), dtype=torch.float32, device=q.device)
    if lse is None:
        lse = torch.empty((b, h), dtype=torch.float32, device=q.device)
    if not (o.is_contiguous() and lse.is_contiguous() and o.dtype == torch.float32
            and lse.dtype == torch.float32):
        raise ValueError("o and lse must be contiguous fp32")
    s, ws = _ws_and_shape(lambda fl: _shape(q, k_pool, block_tables, block_size, scale,
                                            h * d, fl), dev, ws)
    check(_lib.load().ir_paged_decode_lse(
        o.data_ptr(), lse.data_ptr(), q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(),
        block_tables.data_ptr(), context_lens.data_ptr(), s, ws.data_ptr(), ws.numel(),
        error_flag(dev).data_ptr(), _stream(dev)))
    return o, lse


@_on_tensor_device
def lse_merge(o_parts: torch.Tensor, lse_parts: torch.Tensor,
              dtype: torch.dtype = torch.float32,
              out: torch.Tensor | None = None) -> torch.Tensor:
    """Combine ``o_parts [P, B, H, D]`` / ``lse_parts [P, B, H]`` (fp32) -> ``[B, H, D]``.

    Each part must be contiguous; the parts may sit at any stride (e.g. the
    rows of a packed all-gather buffer)."""
    dev = _dev_index(o_parts)
    if o_parts.dim() != 4 or lse_parts.shape != o_parts.shape[:3]:
        raise ValueError("o_parts must be [P, B, H, D] and lse_parts [P, B, H]")
    if o_parts.dtype != torch.float32 or lse_parts.dtype != torch.float32:
        raise ValueError("partials must be fp32")
    p, b, h, d = o_parts.shape
    if not (o_parts[0].is_contiguous() and lse_parts[0].is_contiguous()):
        o_parts, lse_parts = o_parts.contiguous(), lse_parts.contiguous()
    if out is None:
        out = torch.empty((b, h, d), dtype=dtype, device=o_parts.device)
    if out.stride(2) != 1 or out.stride(1) != d:
        raise ValueError("out rows must be [H, D] contiguous")
    check(_lib.load().ir_lse_merge(
        out.data_ptr(), out.stride(0), o_parts.data_ptr(), o_parts.stride(0),
        lse_parts.data_ptr(), lse_parts.stride(0), p, b, h, d, dtype_code(out.dtype),
        _stream(dev)))
    return out


# --- prefill / mixed varlen (Sq > 1) ----------------------------------------


def set_prefill_path(path: int) -> None:
    """0 auto, 1 rows as decode rows, 2 the tcgen05 tensor-core kernel, 3 its
    CTA-pair form (head_dim 128, cta_group::2; only on request)."""
    check(_lib.load().ir_set_prefill_path(int(path)))


def _prefill_shape(q, k_pool, block_tables, q_start, block_size, scale, out_stride):
    t, h, d = q.shape
    s = _lib.PrefillShape()
    s.num_seqs = q_start.numel() - 1
    s.total_q = t
    s.num_heads = h
    s.num_kv_heads = k_pool.shape[1]
    s.head_dim = d
    s.block_size = block_size
    s.max_blocks = block_tables.shape[1]
    s.bt_stride = block_tables.stride(0) if block_tables.shape[0] else block_tables.shape[1]
    s.q_stride = q.stride(0) if t else h * d
    s.out_stride = out_stride
    s.num_slots = k_pool.shape[0]
    s.scale = float(scale)
    s.dtype = dtype_code(q.dtype)
    return s


def prefill_plan(q, k_pool, block_tables, q_start, block_size, scale=1.0):
    """``(path, workspace_bytes)`` of :func:`paged_prefill` for these shapes."""
    s = _prefill_shape(q, k_pool, block_tables, q_start, block_size, scale,
                       q.shape[1] * q.shape[2])
    lib = _lib.load()
    path = _lib.c_int()
    check(lib.ir_paged_prefill_plan(s, path))
    return path.value, lib.ir_paged_prefill_workspace_size(s)


@_on_tensor_device
def paged_prefill(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                  block_tables: torch.Tensor, context_lens: torch.Tensor,
                  q_start: torch.Tensor, scale: float, block_size: int,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal paged attention of packed query rows ``q [total_q, H, D]``.

    Sequence ``s`` owns rows ``q_start[s] .. q_start[s+1]-1``, its last
    positions ``context_lens[s] - q_len .. context_lens[s] - 1`` (the pool
    already holds this step's K/V); each row attends its own sequence up to
    its position. ``block_tables`` int32 ``[S, max_blocks]``,
    ``context_lens`` int32 ``[S]``, ``q_start`` int32 ``[S + 1]``.
    """
    _dev_index(q)
    if q.dim() != 3 or q.stride(2) != 1 or q.stride(1) != q.shape[2]:
        raise ValueError("q must be [total_q, H, D] with [H, D] contiguous rows")
    _check_pool(k_pool, "k_pool")
    _check_pool(v_pool, "v_pool")
    if k_pool.shape != v_pool.shape or k_pool.dtype != q.dtype or v_pool.dtype != q.dtype:
        raise ValueError("pools must match each other and q's dtype")
    if k_pool.shape[2] != q.shape[2]:
        raise ValueError("head_dim of q and pools differ")
    for name, t, n in (("context_lens", context_lens, None), ("q_start", q_start, None)):
        if t.dtype != torch.int32 or not t.is_contiguous() or t.device != q.device:
            raise ValueError(f"{name} must be a contiguous int32 tensor on q's device")
    if block_tables.dtype != torch.int32 or block_tables.dim() != 2 or \
            (block_tables.numel() and block_tables.stride(1) != 1) or \
            block_tables.device != q.device:
        raise ValueError("block_tables must be int32 [S, max_blocks] with unit column stride")
    nseq = q_start.numel() - 1
    if nseq < 0 or block_tables.shape[0] != nseq or context_lens.numel() != nseq:
        raise ValueError("q_start must have one more entry than block_tables / context_lens")
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    elif out.shape != q.shape or out.dtype != q.dtype or out.stride(2) != 1 or \
            out.stride(1) != q.shape[2]:
        raise ValueError("out must be [total_q, H, D] of q's dtype with contiguous rows")
    dev = _dev_index(q)
    s = _prefill_shape(q, k_pool, block_tables, q_start, block_size, scale,
                       out.stride(0) if out.shape[0] else q.shape[1] * q.shape[2])
    lib = _lib.load()
    nbytes = lib.ir_paged_prefill_workspace_size(s)
    ws = workspace(max(nbytes, 256), dev)
    check(lib.ir_paged_prefill(out.data_ptr(), q.data_ptr(), k_pool.data_ptr(),
                               v_pool.data_ptr(), block_tables.data_ptr(),
                               context_lens.data_ptr(), q_start.data_ptr(), s, ws.data_ptr(),
                               ws.numel(), error_flag(dev).data_ptr(), _stream(dev)))
    return out


@_on_tensor_device
def derive_varlen_metadata(gather_slots: torch.Tensor, mask: torch.Tensor, block_size: int):
    """``(block_tables [S, max_blocks], context_lens [S], q_start [S + 1])`` of
    one packed frame in infrared's form (``gather_slots [1, K]`` int64 and
    the additive ``mask [1, 1, Q, K]`` of inputs.py:38-94), built on the
    device; reading the sequence count back is one small synchronising copy.
    Inconsistent frames set device error bits (``check_device_errors``).
    """
    _dev_index(mask)
    gs = gather_slots.reshape(-1)
    if gs.dtype != torch.int64 or not gs.is_contiguous():
        gs = gs.to(torch.int64).contiguous()
    q, k = mask.shape[-2], mask.shape[-1]
    m2 = mask.reshape(q, k)
    if m2.stride(1) != 1:
        m2 = m2.contiguous()
    dev = _dev_index(mask)
    max_blocks = max(1, -(-k // block_size))
    bt = torch.empty((max(q, 1), max_blocks), dtype=torch.int32, device=mask.device)
    ctx = torch.empty(max(q, 1), dtype=torch.int32, device=mask.device)
    q_start = torch.empty(q + 1, dtype=torch.int32, device=mask.device)
    nseq = torch.empty(1, dtype=torch.int32, device=mask.device)
    scratch = torch.empty(max(3 * q, 1), dtype=torch.int32, device=mask.device)
    check(_lib.load().ir_derive_varlen_metadata(
        gs.data_ptr(), k, m2.data_ptr(), m2.stride(0) if q else k, dtype_code(m2.dtype), q,
        block_size, max_blocks, bt.data_ptr(), ctx.data_ptr(), q_start.data_ptr(),
        nseq.data_ptr(), scratch.data_ptr(), error_flag(dev).data_ptr(), _stream(dev)))
    s = int(nseq.item())
    return bt[:s], ctx[:s], q_start[:s + 1]


# --- 8-bit K/V cache ----------------------------------------------------------
#
# A call's checks depend on its tensors' shapes, strides, types and devices
# alone, so each entry point keeps the outcome (the shape structs and sizes it
# passes on) under a key of these: a repeated call, such as every layer of
# every step makes, skips the checks. No plan holds a tensor or an address.


class _Plans(dict):
    """Validated call plans, bounded."""

    def keep(self, key, plan):
        if len(self) > 512:
            self.clear()
        self[key] = plan
        return plan


_write_plans, _gather_plans, _decode_q8_plans, _prefill_q8_plans, _norm_plans = \
    (_Plans() for _ in range(5))

_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or _stream


_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_err_ptrs: dict[int, int] = {}   # device -> address of its error word (allocated once)


def _on_device(dev: int, fn, *args):
    """A library call with device ``dev`` current: plans and workspace sizes
    depend on it, and launches need it."""
    if dev == _current_device():
        return fn(*args)
    with torch.cuda.device(dev):
        return fn(*args)


def _issue(dev: int, fn, args) -> None:
    """One library call on device ``dev``; ``args`` end with its stream."""
    rc = _on_device(dev, fn, *args)
    if rc:
        check(rc)


def _err_ptr(dev: int) -> int:
    p = _err_ptrs.get(dev)
    if p is None:
        p = _err_ptrs[dev] = error_flag(dev).data_ptr()
    return p


def kv_format(dtype: torch.dtype) -> int:
    """``IR_KV_*`` of an 8-bit pool's dtype."""
    try:
        return _KV_FORMATS[dtype]
    except KeyError:
        raise _lib.UnsupportedShape(
            _lib.IR_ERR_UNSUPPORTED, f"8-bit pools are float8_e4m3fn or int8, not {dtype}")


def _row_stride(t: torch.Tensor, row: int) -> int:
    """Stride between t's rows of ``row`` elements (one row or none: any stride
    that the tensor reports stands for nothing, so the row itself)."""
    return t.stride(0) if t.shape[0] > 1 else row


def _check_pool_q8(pool: torch.Tensor, scale: torch.Tensor, block_size: int, name: str) -> int:
    """Checks one side of an 8-bit cache; its format."""
    fmt = kv_format(pool.dtype)
    _check_pool(pool, name)
    if block_size <= 0 or pool.shape[0] % block_size:
        raise ValueError(f"{name} must hold whole blocks of block_size rows")
    if scale.dtype != torch.float32 or not scale.is_contiguous() or \
            tuple(scale.shape) != (pool.shape[0] // block_size, pool.shape[1]):
        raise ValueError(f"the scale of {name} must be contiguous fp32 [num_blocks, Hkv]")
    if scale.device != pool.device:
        raise ValueError("all tensors must be on the same device")
    return fmt


def _check_pools_q8(k_pool, v_pool, k_scale, v_scale, block_size) -> int:
    fmt = _check_pool_q8(k_pool, k_scale, block_size, "k_pool")
    if _check_pool_q8(v_pool, v_scale, block_size, "v_pool") != fmt or \
            v_pool.shape != k_pool.shape or v_pool.device != k_pool.device:
        raise ValueError("k_pool and v_pool differ")
    return fmt


def _pools_key(k_pool, v_pool, k_scale, v_scale, block_size):
    return (k_pool.shape, k_pool.dtype, k_pool.is_contiguous(), k_pool.get_device(),
            v_pool.shape, v_pool.dtype, v_pool.is_contiguous(), v_pool.get_device(),
            k_scale.shape, k_scale.dtype, k_scale.is_contiguous(), k_scale.get_device(),
            v_scale.shape, v_scale.dtype, v_scale.is_contiguous(), v_scale.get_device(),
            block_size)


def cache_write_q8(k: torch.Tensor, v: torch.Tensor, k_pool: torch.Tensor,
                   v_pool: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                   slot_mapping: torch.Tensor, block_size: int) -> None:
    """Quantise ``k, v [N, Hkv, D]`` into one layer's 8-bit pools at ``slot_mapping``.

    The pools are ``[num_slots, Hkv, D]`` codes (``float8_e4m3fn`` or
    ``int8``), the scales fp32 ``[num_blocks, Hkv]``: a row's value is
    code * scale. Every touched (block, head) keeps the larger of its scale and
    the smallest power of two that holds the new rows; codes of other rows are
    rescaled when it grows; a write that holds a block's first row begins the
    block afresh (``ir_cache_write_q8``). Negative slots skip their rows.
    """
    key = (k.shape, k.stride(), k.dtype, k.get_device(), v.shape, v.stride(), v.dtype,
           v.get_device(), slot_mapping.shape, slot_mapping.dtype,
           slot_mapping.is_contiguous(), slot_mapping.get_device(),
           _pools_key(k_pool, v_pool, k_scale, v_scale, block_size))
    plan = _write_plans.get(key)
    if plan is None:
        dev = _dev_index(k_pool)
        fmt = _check_pools_q8(k_pool, v_pool, k_scale, v_scale, block_size)
        n = slot_mapping.numel()
        hkv, d = k_pool.shape[1], k_pool.shape[2]
        if slot_mapping.dtype != torch.int64 or not slot_mapping.is_contiguous() or \
                slot_mapping.device != k_pool.device:
            raise ValueError("slot_mapping must be a contiguous int64 tensor on the pool's device")
        strides = []
        for t, nm in ((k, "k"), (v, "v")):
            if t.dtype != k.dtype or t.device != k_pool.device:
                raise ValueError(f"{nm} must match k's dtype and the pool's device")
            r = t.reshape(n, hkv, d)
            if n and (r.stride(2) != 1 or r.stride(1) != d or r.data_ptr() != t.data_ptr()):
                raise ValueError(f"{nm} rows must be [Hkv, D] contiguous")
            strides.append(_row_stride(r, hkv * d))
        code = dtype_code(k.dtype)
        lib = _lib.load()
        nbytes = lib.ir_cache_write_q8_workspace_size(n, k_pool.shape[0], block_size)
        plan = _write_plans.keep(key, (dev, lib.ir_cache_write_q8, *strides, n, hkv, d,
                                       k_pool.shape[0], code, fmt, nbytes))
    dev, fn, ks, vs, n, hkv, d, num_slots, code, fmt, nbytes = plan
    if n == 0:
        return
    # (of this call alone: PyTorch's allocator orders its reuse on the stream)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=k_pool.device) if nbytes else None
    _issue(dev, fn, (k.data_ptr(), v.data_ptr(), ks, vs, k_pool.data_ptr(), v_pool.data_ptr(),
                     k_scale.data_ptr(), v_scale.data_ptr(), slot_mapping.data_ptr(), n, hkv, d,
                     block_size, num_slots, code, fmt, _ptr(ws), nbytes, _err_ptr(dev),
                     _raw_stream(dev)))


def cache_gather_q8(pool: torch.Tensor, scale: torch.Tensor, slots: torch.Tensor,
                    block_size: int, dtype: torch.dtype) -> torch.Tensor:
    """Rows of an 8-bit pool as values of ``dtype``: a 1-D or 2-D int64 slot tensor
    -> ``[*slots.shape, Hkv, D]`` (finite values beyond the dtype saturate)."""
    key = (pool.shape, pool.dtype, pool.is_contiguous(), pool.get_device(), scale.shape,
           scale.dtype, scale.is_contiguous(), scale.get_device(), slots.shape, slots.dtype,
           slots.get_device(), block_size, dtype)
    plan = _gather_plans.get(key)
    if plan is None:
        dev = _dev_index(pool)
        fmt = _check_pool_q8(pool, scale, block_size, "pool")
        if slots.dtype != torch.int64 or slots.device != pool.device:
            raise ValueError("slots must be int64 on the pool's device")
        plan = _gather_plans.keep(key, (dev, _lib.load().ir_cache_gather_q8, slots.numel(),
                                        (*slots.shape, pool.shape[1], pool.shape[2]),
                                        pool.shape, dtype_code(dtype), fmt))
    dev, fn, n, shape, (num_slots, hkv, d), code, fmt = plan
    out = pool.new_empty(shape, dtype=dtype)
    if n:
        slots = slots if slots.is_contiguous() else slots.contiguous()
        _issue(dev, fn, (out.data_ptr(), pool.data_ptr(), scale.data_ptr(), slots.data_ptr(), n,
                         hkv, d, block_size, num_slots, code, fmt, _err_ptr(dev),
                         _raw_stream(dev)))
    return out


def _check_decode_q8(q, k_pool, v_pool, k_scale, v_scale, block_tables, context_lens, out,
                     block_size):
    _dev_index(q)
    fmt = _check_pools_q8(k_pool, v_pool, k_scale, v_scale, block_size)
    if q.dim() != 3 or q.stride(2) != 1 or q.stride(1) != q.shape[2]:
        raise ValueError("q must be [rows, H, D] with [H, D] contiguous rows")
    if k_pool.shape[2] != q.shape[2]:
        raise ValueError("head_dim of q and pools differ")
    if block_tables.dtype != torch.int32 or block_tables.dim() != 2 or \
            (block_tables.numel() and block_tables.stride(1) != 1):
        raise ValueError("block_tables must be int32 [B, max_blocks] with unit column stride")
    if context_lens.dtype != torch.int32 or not context_lens.is_contiguous():
        raise ValueError("context_lens must be contiguous int32 [B]")
    for t in (k_pool, block_tables, context_lens):
        if t.device != q.device:
            raise ValueError("all tensors must be on the same device")
    if out is not None and (out.shape != q.shape or out.dtype != q.dtype or out.stride(2) != 1 or
                            out.stride(1) != q.shape[2] or out.device != q.device):
        raise ValueError("out must be of q's shape, dtype and device with [H, D] contiguous rows")
    return fmt


def _decode_q8_key(q, k_pool, v_pool, k_scale, v_scale, block_tables, context_lens, out, scale,
                   block_size):
    return (q.shape, q.stride(), q.dtype, q.get_device(), block_tables.shape,
            block_tables.stride(), block_tables.dtype, block_tables.get_device(),
            context_lens.shape, context_lens.dtype, context_lens.is_contiguous(),
            context_lens.get_device(), scale,
            None if out is None else (out.shape, out.stride(), out.dtype, out.get_device()),
            _pools_key(k_pool, v_pool, k_scale, v_scale, block_size))


def _scratch(ws: torch.Tensor | None, nbytes: int, q: torch.Tensor) -> torch.Tensor:
    """The caller's workspace, or one of this call alone: it needs no initial
    state, and PyTorch's allocator orders its reuse on the current stream and
    inside a graph capture, so calls on other streams and replayed graphs
    never share it."""
    if ws is None:
        return torch.empty(nbytes, dtype=torch.uint8, device=q.device)
    if ws.numel() * ws.element_size() < nbytes or ws.device != q.device or not ws.is_contiguous():
        raise ValueError(f"workspace must be {nbytes} contiguous bytes on q's device")
    return ws


def _plan_device(q: torch.Tensor) -> int:
    """Device whose plan is meant: q's, or the current one (q's shape may be all
    there is)."""
    return _dev_index(q) if q.is_cuda else _current_device()


def decode_plan_q8(q, k_pool, block_tables, block_size, scale=1.0):
    """``(path, ctas_per_kv_head, workspace_bytes)`` of :func:`paged_decode_q8`."""
    s = _shape(q, k_pool, block_tables, block_size, scale, q.shape[1] * q.shape[2])
    fmt = kv_format(k_pool.dtype)
    lib = _lib.load()
    dev = _plan_device(q)
    path, g = _lib.c_int(), _lib.c_int()
    check(_on_device(dev, lib.ir_paged_decode_q8_plan, s, fmt, path, g))
    return path.value, g.value, _on_device(dev, lib.ir_paged_decode_q8_workspace_size, s, fmt)


def paged_decode_q8(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                    k_scale: torch.Tensor, v_scale: torch.Tensor, block_tables: torch.Tensor,
                    context_lens: torch.Tensor, scale: float, block_size: int,
                    out: torch.Tensor | None = None,
                    ws: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`paged_decode` over an 8-bit cache (:func:`cache_write_q8`):
    ``q [B, H, D]`` (any dtype of the framework) -> ``[B, H, D]``."""
    key = _decode_q8_key(q, k_pool, v_pool, k_scale, v_scale, block_tables, context_lens, out,
                         scale, block_size)
    plan = _decode_q8_plans.get(key)
    if plan is None:
        fmt = _check_decode_q8(q, k_pool, v_pool, k_scale, v_scale, block_tables, context_lens, out,
                               block_size)
        if block_tables.shape[0] != q.shape[0] or context_lens.numel() != q.shape[0]:
            raise ValueError("batch sizes of q, block_tables and context_lens differ")
        dev = _dev_index(q)
        row = q.shape[1] * q.shape[2]
        s = _shape(q, k_pool, block_tables, block_size, scale,
                   row if out is None else _row_stride(out, row))
        s.q_stride, s.bt_stride = _row_stride(q, row), _row_stride(block_tables, s.max_blocks)
        lib = _lib.load()
        nbytes = _on_device(dev, lib.ir_paged_decode_q8_workspace_size, s, fmt)
        if nbytes == 0:
            check(_on_device(dev, lib.ir_paged_decode_q8_plan, s, fmt, None, None))
        plan = _decode_q8_plans.keep(key, (dev, lib.ir_paged_decode_q8, s, fmt, nbytes))
    dev, fn, s, fmt, nbytes = plan
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    ws = _scratch(ws, nbytes, q)
    _issue(dev, fn, (out.data_ptr(), q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(),
                     k_scale.data_ptr(), v_scale.data_ptr(), fmt, block_tables.data_ptr(),
                     context_lens.data_ptr(), s, ws.data_ptr(), ws.numel() * ws.element_size(),
                     _err_ptr(dev), _raw_stream(dev)))
    return out


def prefill_plan_q8(q, k_pool, block_tables, q_start, block_size, scale=1.0):
    """``(path, workspace_bytes)`` of :func:`paged_prefill_q8` for these shapes."""
    s = _prefill_shape(q, k_pool, block_tables, q_start, block_size, scale,
                       q.shape[1] * q.shape[2])
    fmt = kv_format(k_pool.dtype)
    lib = _lib.load()
    dev = _plan_device(q)
    path = _lib.c_int()
    check(_on_device(dev, lib.ir_paged_prefill_q8_plan, s, fmt, path))
    return path.value, _on_device(dev, lib.ir_paged_prefill_q8_workspace_size, s, fmt)


def paged_prefill_q8(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                     k_scale: torch.Tensor, v_scale: torch.Tensor, block_tables: torch.Tensor,
                     context_lens: torch.Tensor, q_start: torch.Tensor, scale: float,
                     block_size: int, out: torch.Tensor | None = None,
                     ws: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`paged_prefill` over an 8-bit cache (:func:`cache_write_q8`). With
    16-bit q its workspace holds the histories, or the pool, in q's dtype
    (``ir_paged_prefill_q8``)."""
    key = (_decode_q8_key(q, k_pool, v_pool, k_scale, v_scale, block_tables, context_lens, out,
                          scale, block_size),
           q_start.shape, q_start.dtype, q_start.is_contiguous(), q_start.get_device())
    plan = _prefill_q8_plans.get(key)
    if plan is None:
        fmt = _check_decode_q8(q, k_pool, v_pool, k_scale, v_scale, block_tables, context_lens, out,
                               block_size)
        if q_start.dtype != torch.int32 or not q_start.is_contiguous() or \
                q_start.device != q.device:
            raise ValueError("q_start must be a contiguous int32 tensor on q's device")
        nseq = q_start.numel() - 1
        if nseq < 0 or block_tables.shape[0] != nseq or context_lens.numel() != nseq:
            raise ValueError("q_start must have one more entry than block_tables / context_lens")
        row = q.shape[1] * q.shape[2]
        s = _prefill_shape(q, k_pool, block_tables, q_start, block_size, scale,
                           row if out is None else _row_stride(out, row))
        s.q_stride, s.bt_stride = _row_stride(q, row), _row_stride(block_tables, s.max_blocks)
        plan = _prefill_q8_plans.keep(key, (_dev_index(q), _lib.load(), s, fmt))
    dev, lib, s, fmt = plan
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    # (asked each time: it depends on the path chosen by set_prefill_path)
    nbytes = _on_device(dev, lib.ir_paged_prefill_q8_workspace_size, s, fmt)
    if nbytes == 0:
        check(_on_device(dev, lib.ir_paged_prefill_q8_plan, s, fmt, None))
    ws = _scratch(ws, max(nbytes, 256), q)
    _issue(dev, lib.ir_paged_prefill_q8,
           (out.data_ptr(), q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(),
            k_scale.data_ptr(), v_scale.data_ptr(), fmt, block_tables.data_ptr(),
            context_lens.data_ptr(), q_start.data_ptr(), s, ws.data_ptr(),
            ws.numel() * ws.element_size(), _err_ptr(dev), _raw_stream(dev)))
    return out


# --- q/k norm with rotation ---------------------------------------------------


def _like(t):
    return (t.shape, t.stride(), t.dtype, t.get_device())


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, w_q: torch.Tensor | None,
                 w_k: torch.Tensor | None, cos: torch.Tensor, sin: torch.Tensor, eps: float,
                 q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None):
    """RMS norm of every head of ``q [N, H, D]`` and ``k [N, Hkv, D]`` over D, times
    ``w_q`` / ``w_k [D]`` (None: one), and the rotary embedding with fp32
    ``cos`` / ``sin [N, D]``, in one kernel; returns ``(q_out, k_out)``.

    Computed in fp32 and rounded once. ``q`` and ``k`` may be row views of one
    QKV projection; ``q_out`` / ``k_out`` may be ``q`` / ``k`` themselves, but
    no other memory that overlaps them.
    """
    key = (q.shape, q.stride(), q.dtype, q.get_device(), k.shape, k.stride(), k.dtype,
           k.get_device(), cos.shape, cos.stride(), cos.dtype, cos.get_device(), sin.shape,
           sin.stride(), sin.dtype, sin.get_device(), w_q is None or _like(w_q),
           w_k is None or _like(w_k), q_out is None or _like(q_out),
           k_out is None or _like(k_out))
    plan = _norm_plans.get(key)
    if plan is None:
        dev = _dev_index(q)
        if q.dim() != 3 or k.dim() != 3 or q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2]:
            raise ValueError("q must be [N, H, D] and k [N, Hkv, D]")
        n, h, d = q.shape
        hkv = k.shape[1]
        strides = []
        for name, t, like in (("q", q, q), ("k", k, k), ("q_out", q_out, q), ("k_out", k_out, k)):
            row = like.shape[1] * d
            if t is None:
                strides.append(row)
                continue
            if t.dtype != q.dtype or t.device != q.device or t.shape != like.shape:
                raise ValueError(f"{name} must match q's dtype and device and its input's shape")
            if t.numel() and (t.stride(2) != 1 or t.stride(1) != d):
                raise ValueError(f"{name} rows must be [heads, D] contiguous")
            strides.append(_row_stride(t, row))
        for name, t in (("w_q", w_q), ("w_k", w_k)):
            if t is not None and (t.numel() != d or t.dtype != q.dtype or not t.is_contiguous()
                                  or t.device != q.device):
                raise ValueError(f"{name} must be a contiguous [D] weight of q's dtype")
        for name, t in (("cos", cos), ("sin", sin)):
            if t.dtype != torch.float32 or t.device != q.device or tuple(t.shape) != (n, d) or \
                    (n and t.stride(1) != 1):
                raise ValueError(f"{name} must be fp32 [N, D] rows on q's device")
        if _row_stride(cos, d) != _row_stride(sin, d):
            raise ValueError("cos and sin must have the same row stride")
        plan = _norm_plans.keep(key, (dev, _lib.load().ir_qk_norm_rope, strides,
                                      _row_stride(cos, d), n, h, hkv, d, dtype_code(q.dtype)))
    dev, fn, strides, rs, n, h, hkv, d, code = plan
    if q_out is None:
        q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if k_out is None:
        k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
    _issue(dev, fn, (q.data_ptr(), k.data_ptr(), q_out.data_ptr(), k_out.data_ptr(), *strides,
                     _ptr(w_q), _ptr(w_k), cos.data_ptr(), sin.data_ptr(), rs, eps, n, h, hkv, d,
                     code, _raw_stream(dev)))
    return q_out, k_out
