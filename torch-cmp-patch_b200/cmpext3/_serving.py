"""The step of a served transformer, bound to the C-ABI library: rotary positions, the append to a
paged key-value cache, the attention of one new token over that cache, and linear layers with 4-bit
weights.  ``cmpext3.ops`` offers them beside ``attention`` and ``linear``:

    qkv   = ops.linear_w4(x, w, scales, zeros)
    query = ops.kv_append(key, value, k_cache, v_cache, page_table, lengths, query=query, freqs=freqs)
    out   = ops.paged_attention(query, k_cache, v_cache, page_table, lengths)

    q, k  = ops.rope(q, positions, freqs, sections), ops.rope(k, positions, freqs, sections)
    out   = F.scaled_dot_product_attention(q, k, v)

As in the rest of the binding: arguments are checked here, outputs and scratch come from torch's
caching allocator, work goes to the current stream of the tensors' device, and what the kernels do not
cover raises ``RuntimeError`` / ``TypeError``.  ``rope`` has a gradient; the others are for inference
and refuse tensors that autograd is recording.  All refuse dual tensors (forward-mode derivatives).
"""
from __future__ import annotations

import ctypes
import math
import struct

import torch
from torch.autograd import forward_ad as _forward

from ._native import _CHECK, _DTYPE, OK, CmpxError, _post_check, _stream_handle, _traced, lib

_MAX_AXES = 4
_POS_KIND = {torch.int32: 1, torch.int64: 2, torch.float32: 3}

_I64x2, _I64x3, _I32x4 = ctypes.c_int64 * 2, ctypes.c_int64 * 3, ctypes.c_int32 * _MAX_AXES


class Rotation(ctypes.Structure):
    _fields_ = [("positions", ctypes.c_void_p), ("freqs", ctypes.c_void_p), ("pos_stride", _I64x3),
                ("pos_kind", ctypes.c_int32), ("pairs", ctypes.c_int32), ("axes", ctypes.c_int32),
                ("interleaved", ctypes.c_int32), ("section_end", _I32x4)]


class RopeDesc(ctypes.Structure):
    _fields_ = [("x", ctypes.c_void_p), ("y", ctypes.c_void_p), ("rot", Rotation),
                ("batch", ctypes.c_int64), ("heads", ctypes.c_int64), ("len", ctypes.c_int64),
                ("head_dim", ctypes.c_int64), ("x_stride", _I64x3), ("y_stride", _I64x3),
                ("dtype", ctypes.c_int32), ("inverse", ctypes.c_int32)]


class PagedCache(ctypes.Structure):
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("table", ctypes.c_void_p),
                ("lengths", ctypes.c_void_p), ("num_pages", ctypes.c_int64), ("page_size", ctypes.c_int64),
                ("heads_kv", ctypes.c_int64), ("head_dim", ctypes.c_int64), ("k_stride", _I64x3),
                ("v_stride", _I64x3), ("table_width", ctypes.c_int64), ("table_stride", ctypes.c_int64)]


class KvAppendDesc(ctypes.Structure):
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("q", ctypes.c_void_p), ("q_out", ctypes.c_void_p),
                ("new_lengths", ctypes.c_void_p), ("cache", PagedCache), ("rot", Rotation),
                ("batch", ctypes.c_int64), ("heads", ctypes.c_int64), ("len", ctypes.c_int64),
                ("k_in_stride", _I64x3), ("v_in_stride", _I64x3), ("q_stride", _I64x3), ("q_out_stride", _I64x3),
                ("dtype", ctypes.c_int32), ("reserved", ctypes.c_int32)]


class PagedAttnDesc(ctypes.Structure):
    _fields_ = [("q", ctypes.c_void_p), ("o", ctypes.c_void_p), ("workspace", ctypes.c_void_p), ("cache", PagedCache),
                ("workspace_bytes", ctypes.c_size_t), ("batch", ctypes.c_int64), ("heads", ctypes.c_int64),
                ("q_stride", _I64x2), ("o_stride", _I64x2), ("scale", ctypes.c_double),
                ("dtype", ctypes.c_int32), ("reserved", ctypes.c_int32)]


class LinearW4Desc(ctypes.Structure):
    _fields_ = [("x", ctypes.c_void_p), ("w", ctypes.c_void_p), ("scales", ctypes.c_void_p),
                ("zeros", ctypes.c_void_p), ("bias", ctypes.c_void_p), ("y", ctypes.c_void_p),
                ("m", ctypes.c_int64), ("n", ctypes.c_int64), ("k", ctypes.c_int64), ("group", ctypes.c_int64),
                ("x_row_stride", ctypes.c_int64), ("y_row_stride", ctypes.c_int64),
                ("w_row_stride", ctypes.c_int64), ("scales_row_stride", ctypes.c_int64),
                ("zeros_row_stride", ctypes.c_int64), ("dtype", ctypes.c_int32), ("reserved", ctypes.c_int32)]


for _name, _desc in (("rope", RopeDesc), ("kv_append", KvAppendDesc), ("paged_attn", PagedAttnDesc),
                     ("linear_w4", LinearW4Desc)):
    _fn = getattr(lib, f"cmpx_{_name}")
    _fn.argtypes, _fn.restype = [ctypes.POINTER(_desc), ctypes.c_void_p], ctypes.c_int
    _fn = getattr(lib, f"cmpx_{_name}_plan")
    _fn.argtypes, _fn.restype = [ctypes.POINTER(_desc), ctypes.c_char_p, ctypes.c_size_t], ctypes.c_int
lib.cmpx_paged_attn_workspace_size.argtypes = [ctypes.POINTER(PagedAttnDesc)]
lib.cmpx_paged_attn_workspace_size.restype = ctypes.c_size_t


# The checks, the descriptor and the output's layout of a call depend on its arguments' shapes, strides, types
# and devices alone; only the pointers differ from call to call.  What a signature came to the first time
# (the descriptor's bytes behind its pointers) is kept, so that a decoding loop's calls cost a lookup instead
# of the checks.  A call whose pointers the kernel declines (misaligned ones) goes the long way again.
_SIGNATURES: dict = {}
_SIGNATURES_MOST = 4096


def _from_bytes(name: str):
    """The entry point, taking its descriptor as bytes."""
    fn = lib[name]
    fn.argtypes, fn.restype = [ctypes.c_char_p, ctypes.c_void_p], ctypes.c_int
    return fn


_ROPE, _KV_APPEND, _PAGED_ATTN, _LINEAR_W4 = map(_from_bytes, ("cmpx_rope", "cmpx_kv_append", "cmpx_paged_attn",
                                                              "cmpx_linear_w4"))
_pack2, _pack4, _pack6, _pack7, _pack9 = (struct.Struct(f"={n}Q").pack for n in (2, 4, 6, 7, 9))


def _keep(key, value) -> None:
    if len(_SIGNATURES) >= _SIGNATURES_MOST:
        _SIGNATURES.clear()
    _SIGNATURES[key] = value


# One value per device and type, expanded to the shapes of outputs and workspaces: torch.empty_like of such a
# tensor costs half of what torch.empty with a type and a device does.  Never read.
_ONES: dict = {}


def _alike(shape, dtype, device) -> torch.Tensor:
    one = _ONES.get((dtype, device))
    if one is None:
        one = _ONES[dtype, device] = torch.empty((), dtype=dtype, device=device)
    return one.expand(shape)


_grad_on, _like_of = torch.is_grad_enabled, torch.empty_like
_device_now, _raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


def _direct(fn, data: bytes, index: int) -> int:
    if index == _device_now():
        st = fn(data, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            st = fn(data, _raw_stream(index))
    if st == OK and _CHECK:
        _post_check()
    return st


def _run(what: str, fn, desc, device: torch.device) -> None:
    if device.index == torch.cuda.current_device():
        st = fn(ctypes.byref(desc), _stream_handle(device))
    else:
        with torch.cuda.device(device):
            st = fn(ctypes.byref(desc), _stream_handle(device))
    if st != OK:
        raise CmpxError(what, st)
    _post_check()


def _plan(what: str, fn, desc) -> str:
    buf = ctypes.create_string_buffer(128)
    st = fn(ctypes.byref(desc), buf, 128)
    if st != OK:
        raise CmpxError(f"{what} plan", st)
    return buf.value.decode()


def _tensor(name: str, t, dim: int, dtype, device) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a Tensor")
    if t.dim() != dim:
        raise RuntimeError(f"{name} must be {dim}D")
    if t.dtype != dtype:
        raise RuntimeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.device != device:
        raise RuntimeError(f"{name} must be on {device}, got {t.device}")


def _rows(name: str, t) -> torch.device:
    """Checks a [batch, heads, tokens, head_dim] tensor that sets the call's dtype and device."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a Tensor")
    if t.dim() != 4:
        raise RuntimeError(f"{name} must be 4D (batch, heads, tokens, head_dim)")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor")
    if t.dtype not in _DTYPE:
        raise RuntimeError(f"{name} must be float32/float16/bfloat16")
    return t.device


def _no_grad_only(what: str, *tensors) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if isinstance(t, torch.Tensor) and t.requires_grad:
                raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad() or on detached tensors")


def _no_tangent(what: str, *tensors) -> None:
    """Refuses dual tensors, whose tangents the kernels would drop; only called within a dual level."""
    if torch._C._is_fwd_grad_enabled():
        for t in tensors:
            if isinstance(t, torch.Tensor) and _forward.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"{what} has no forward-mode derivative: call it on detached tensors")


def _unit(t: torch.Tensor) -> torch.Tensor:
    """t with a contiguous last dimension (a copy where it has none)."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _like(t: torch.Tensor) -> tuple[torch.Tensor, tuple]:
    """An output laid out as t, contiguous along the last dimension, and its strides."""
    out = torch.empty_like(t)
    if out.stride(-1) != 1 and t.shape[-1] != 1:  # (rows of t overlap in some odd way)
        out = torch.empty_like(t, memory_format=torch.contiguous_format)
    return out, out.stride()


def _is_like(out: torch.Tensor, t: torch.Tensor) -> bool:
    """True if torch.empty_like(t), which depends on t's shape and strides, is laid out as out."""
    return out.stride() == torch.empty_like(t).stride()


# ---------------------------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------------------------

def _whole(sections) -> tuple:
    # before a kept signature is looked up, where 8.0 would pass for 8
    sections = tuple(sections)
    if not all(type(n) is int for n in sections):
        raise TypeError("sections must be whole numbers")
    return sections


def _rotation(positions, freqs, sections, interleaved, batch: int, tokens: int, head_dim: int,
              device: torch.device) -> tuple[Rotation, tuple]:
    """The descriptor of a rotation, and the tensors it points into."""
    _tensor("freqs", freqs, 1, torch.float32, device)
    pairs = freqs.shape[0]
    if not 1 <= pairs <= head_dim // 2:
        raise RuntimeError(f"freqs must have 1 to head_dim // 2 = {head_dim // 2} values, got {pairs}")
    freqs = _unit(freqs)
    axes = 1
    ends = (pairs, 0, 0, 0)
    if sections is not None:
        sections = _whole(sections)
        axes = len(sections)
        if not 1 <= axes <= _MAX_AXES or min(sections) < 0 or sum(sections) != pairs:
            raise RuntimeError(f"sections must be 1 to {_MAX_AXES} counts of pairs that add up to {pairs}, got {sections}")
        at, out = 0, []
        for n in sections:
            at += n
            out.append(at)
        ends = tuple(out) + (0,) * (_MAX_AXES - axes)
    if positions is None:
        return Rotation(None, freqs.data_ptr(), _I64x3(0, 0, 0), 0, pairs, 1, 1 if interleaved else 0,
                        _I32x4(*ends)), (freqs,)
    if not isinstance(positions, torch.Tensor):
        raise TypeError("positions must be a Tensor")
    kind = _POS_KIND.get(positions.dtype)
    if kind is None:
        raise RuntimeError("positions must be int32, int64 or float32")
    if positions.device != device:
        raise RuntimeError(f"positions must be on {device}, got {positions.device}")
    shape, stride = tuple(positions.shape), positions.stride()
    lead = 0 if sections is None else 1
    if lead:
        if not shape or shape[0] != axes:
            raise RuntimeError(f"positions {shape} must begin with the {axes} axes of sections")
    rest = shape[lead:]
    if rest == (tokens,):
        strides = (stride[0] if lead else 0, 0, stride[-1])
    elif len(rest) == 2 and rest[1] == tokens and rest[0] in (1, batch):
        strides = (stride[0] if lead else 0, stride[-2] if rest[0] != 1 else 0, stride[-1])
    else:
        want = "[axes, tokens] or [axes, batch, tokens]" if lead else "[tokens] or [batch, tokens]"
        raise RuntimeError(f"positions {shape} must be {want} with batch {batch} and {tokens} tokens")
    return Rotation(positions.data_ptr(), freqs.data_ptr(), _I64x3(*strides), kind, pairs, axes,
                    1 if interleaved else 0, _I32x4(*ends)), (positions, freqs)


def _rope_desc(x, positions, freqs, sections, interleaved, inverse):
    device = _rows("input", x)
    if positions is None:
        raise TypeError("positions must be a Tensor")
    b, h, n, d = x.shape
    rot, keep = _rotation(positions, freqs, sections, interleaved, b, n, d, device)
    x = _unit(x)
    y, ys = _like(x)
    desc = RopeDesc(x.data_ptr(), y.data_ptr(), rot, b, h, n, d, _I64x3(*x.stride()[:3]), _I64x3(*ys[:3]),
                    _DTYPE[x.dtype], 1 if inverse else 0)
    return desc, y, (x, keep)


def _rope_call(x, positions, freqs, sections, interleaved, inverse):
    try:
        key = ("rope", x.shape, x.stride(), x.dtype, x.device, positions.shape, positions.stride(), positions.dtype,
               positions.device, freqs.shape, freqs.stride(), freqs.dtype, freqs.device, sections, interleaved, inverse)
        how = _SIGNATURES.get(key)
    except (AttributeError, TypeError):  # no tensors: the checks below name them
        key = how = None
    if how is not None:
        tail, index = how
        y = _like_of(x)
        if _direct(_ROPE, _pack4(x.data_ptr(), y.data_ptr(), positions.data_ptr(), freqs.data_ptr()) + tail, index) == OK:
            return y
    desc, y, used = _rope_desc(x, positions, freqs, sections, interleaved, inverse)
    if y.numel():
        _run("rope", lib.cmpx_rope, desc, y.device)
        if key is not None and used[0] is x and used[1][1] is freqs and _is_like(y, x):
            _keep(key, (bytes(desc)[32:], y.device.index))
    return y


_STREAM_NOTE = "cmpext3.rope stream"


def _check_leaf(x: torch.Tensor) -> None:
    """In a graph capture: refuses a leaf of which rope has recorded an eager graph on the default stream that is
    alive.  The captured backward pass would make that stream, which the leaf's autograd node belongs to and
    which cannot be captured, wait for the capturing one, an error in autograd's thread that ends the process (a
    graph recorded on a side stream, as in a warm-up, does no harm).  The note is on the node, which lives as long
    as the graphs that use it."""
    if torch.autograd.graph.get_gradient_edge(x).node.metadata.get(_STREAM_NOTE) == 0:
        raise RuntimeError("rope: an eager graph of this leaf from the default stream is alive; drop its outputs "
                           "before the capture")


def _note_leaf(y: torch.Tensor, device: torch.device) -> None:
    """Notes on the node of the leaf that y was computed from the stream on which that was recorded."""
    notes = y.grad_fn.next_functions[0][0].metadata
    notes.setdefault(_STREAM_NOTE, torch._C._cuda_getCurrentRawStream(device.index))


class _Rope(torch.autograd.Function):
    """The rotation's gradient is the rotation by the negative angles (which has one, too)."""

    @staticmethod
    def forward(ctx, x, positions, freqs, sections, interleaved, inverse):
        ctx.save_for_backward(positions, freqs)
        ctx.how = (sections, interleaved, inverse)
        return _rope_call(x, positions, freqs, sections, interleaved, inverse)

    @staticmethod
    def backward(ctx, grad):
        positions, freqs = ctx.saved_tensors
        sections, interleaved, inverse = ctx.how
        if _forward._current_level >= 0:
            _no_tangent("rope's gradient", grad)
        if torch.is_grad_enabled() and grad.requires_grad:
            gx = _Rope.apply(grad, positions, freqs, sections, interleaved, not inverse)
        else:
            gx = _rope_call(grad, positions, freqs, sections, interleaved, not inverse)
        return gx, None, None, None, None, None


@_traced("rope")
def rope(input, positions, freqs, sections=None, interleaved=False):
    """Rotary positions: pair j of every row of ``input`` [batch, heads, tokens, head_dim] turns by
    position * freqs[j] radians, (a, b) -> (a cos - b sin, a sin + b cos).

    ``freqs`` [pairs] fp32, 1 <= pairs <= head_dim // 2; the pair is (x[j], x[j + pairs]), or
    (x[2j], x[2j + 1]) with ``interleaved``; values behind the first 2 * pairs pass through.
    ``positions`` (int32, int64 or float32) is [tokens] or [batch, tokens].  With ``sections``, up to
    four counts that add up to pairs, positions has a leading axis of that many (time, height, width,
    ...): the first sections[0] pairs turn by positions[0], the next by positions[1], and so on.
    Angles are exact to fp32 below 2^50 radians (positions of up to 2^53); the result, a new tensor laid out
    as input, is rounded once.
    Differentiable in ``input`` (backward passes; forward mode is refused); positions and freqs have no gradient.
    A capture of forward and backward pass into a CUDA graph needs its leaves free of eager graphs from the
    default stream: RuntimeError where rope recorded them; those of other ops are not seen here, and end the
    process in autograd's thread as they do with any op.
    head_dim <= 256."""
    sections, interleaved = None if sections is None else _whole(sections), bool(interleaved)
    if _forward._current_level >= 0:
        _no_tangent("rope", input, positions, freqs)
    if torch.is_grad_enabled():
        _no_grad_only("rope in positions and freqs", positions, freqs)
        if isinstance(input, torch.Tensor) and input.requires_grad:
            leaf = input.is_leaf and input.is_cuda
            if leaf and torch.cuda.is_current_stream_capturing():
                _check_leaf(input)
            y = _Rope.apply(input, positions, freqs, sections, interleaved, False)
            if leaf:
                _note_leaf(y, input.device)
            return y
    return _rope_call(input, positions, freqs, sections, interleaved, False)


def rope_plan(input, positions, freqs, sections=None, interleaved=False) -> str:
    """Name of the kernel ``rope`` runs for these arguments."""
    desc, _y, _used = _rope_desc(input, positions, freqs, sections, interleaved, False)
    return _plan("rope", lib.cmpx_rope_plan, desc)


# ---------------------------------------------------------------------------------------------
# the paged cache
# ---------------------------------------------------------------------------------------------

def _paged(k_cache, v_cache, page_table, lengths, batch: int, dtype, device) -> PagedCache:
    _tensor("k_cache", k_cache, 4, dtype, device)
    _tensor("v_cache", v_cache, 4, dtype, device)
    _tensor("page_table", page_table, 2, torch.int32, device)
    _tensor("lengths", lengths, 1, torch.int32, device)
    shape = k_cache.shape
    if v_cache.shape != shape:
        raise RuntimeError(f"v_cache {tuple(v_cache.shape)} does not match k_cache {tuple(shape)}")
    pages, heads_kv, page_size, head_dim = shape
    if page_size < 1 or heads_kv < 1 or head_dim < 1:
        raise RuntimeError(f"k_cache {tuple(shape)} must be (pages, heads_kv, page_size, head_dim), none of the last three 0")
    if page_table.shape[0] != batch or lengths.shape[0] != batch:
        raise RuntimeError(f"page_table {tuple(page_table.shape)} and lengths {tuple(lengths.shape)} must have "
                           f"batch {batch} rows")
    ks, vs = k_cache.stride(), v_cache.stride()
    if (ks[3] != 1 or vs[3] != 1) and head_dim != 1:
        raise RuntimeError("k_cache and v_cache must be contiguous along head_dim")
    ts = page_table.stride()
    if ts[1] != 1 and page_table.shape[1] > 1 or lengths.stride(0) != 1 and batch > 1:
        raise RuntimeError("page_table's rows and lengths must be contiguous")
    return PagedCache(k_cache.data_ptr(), v_cache.data_ptr(), page_table.data_ptr(), lengths.data_ptr(), pages,
                      page_size, heads_kv, head_dim, _I64x3(ks[0], ks[1], ks[2]), _I64x3(vs[0], vs[1], vs[2]),
                      page_table.shape[1], ts[0])


def _append_desc(key, value, k_cache, v_cache, page_table, lengths, new_lengths, query, positions, freqs, sections,
                 interleaved):
    device = _rows("key", key)
    b, heads_kv, n, d = key.shape
    _tensor("value", value, 4, key.dtype, device)
    if value.shape != key.shape:
        raise RuntimeError(f"value {tuple(value.shape)} does not match key {tuple(key.shape)}")
    cache = _paged(k_cache, v_cache, page_table, lengths, b, key.dtype, device)
    if cache.heads_kv != heads_kv or cache.head_dim != d:
        raise RuntimeError(f"k_cache {tuple(k_cache.shape)} does not hold key {tuple(key.shape)}")
    for t in (k_cache, v_cache):
        if any(st == 0 and size > 1 for st, size in zip(t.stride(), t.shape)):
            raise RuntimeError("k_cache and v_cache must not be expanded tensors")
    if new_lengths is not None:
        _tensor("new_lengths", new_lengths, 1, torch.int32, device)
        if new_lengths.shape[0] != b or new_lengths.stride(0) != 1 and b > 1:
            raise RuntimeError(f"new_lengths must be {b} contiguous values")
    key, value = _unit(key), _unit(value)
    out, heads, qp, qs, op, os_ = None, 0, None, (0, 0, 0), None, (0, 0, 0)
    if query is not None:
        _tensor("query", query, 4, key.dtype, device)
        heads = query.shape[1]
        if query.shape[0] != b or query.shape[2] != n or query.shape[3] != d:
            raise RuntimeError(f"query {tuple(query.shape)} does not match key {tuple(key.shape)}")
        query = _unit(query)
        out, os_ = _like(query)
        qp, qs, op, os_ = query.data_ptr(), query.stride()[:3], out.data_ptr(), os_[:3]
    keep = ()
    if freqs is None:
        if positions is not None or sections is not None:
            raise RuntimeError("positions and sections need freqs")
        rot = Rotation()
    else:
        if positions is None and sections is not None:
            raise RuntimeError("sections need positions")
        rot, keep = _rotation(positions, freqs, sections, interleaved, b, n, d, device)
    desc = KvAppendDesc(key.data_ptr(), value.data_ptr(), qp, op,
                        None if new_lengths is None else new_lengths.data_ptr(), cache, rot, b, heads, n,
                        _I64x3(*key.stride()[:3]), _I64x3(*value.stride()[:3]), _I64x3(*qs), _I64x3(*os_),
                        _DTYPE[key.dtype], 0)
    return desc, out, (key, value, query, keep)


@_traced("kv_append")
def kv_append(key, value, k_cache, v_cache, page_table, lengths, new_lengths=None, query=None, positions=None,
              freqs=None, sections=None, interleaved=False):
    """Stores new keys and values in a paged cache, in place; with ``freqs`` the keys, and ``query`` if
    given, are turned on the way (``rope``).  Returns the turned query, or None.

    key, value [batch, heads_kv, tokens, head_dim]; query [batch, heads, tokens, head_dim];
    k_cache, v_cache [pages, heads_kv, page_size, head_dim] in the same dtype, any strides (a
    transposed view of [pages, page_size, heads_kv, head_dim] memory, too) with head_dim contiguous
    and rows on 16-byte boundaries; page_table [batch, width] and lengths [batch] int32.  Token t of
    sequence b lies in page page_table[b, t // page_size], row t % page_size.

    ``lengths`` count the new tokens: sequence b's new_lengths[b] tokens (all of them when None) go to
    the places up to lengths[b] - 1, so the same tensor serves this call and ``paged_attention`` after
    it.  Rows behind new_lengths[b] are padding: they are not stored, and their query comes back as it
    was.  A token's position is its place in its sequence unless ``positions`` says otherwise.

    A token whose place is negative, behind the table or in a page that does not exist is not stored and
    sets a bit of ``device_status()``.  Which of two tokens that share a slot stays is not defined; key and
    value must not lie in the caches' memory."""
    sections, interleaved = None if sections is None else _whole(sections), bool(interleaved)
    if torch.is_grad_enabled():
        _no_grad_only("kv_append", key, value, k_cache, v_cache, query, positions, freqs)
    if _forward._current_level >= 0:
        _no_tangent("kv_append", key, value, k_cache, v_cache, query, positions, freqs)
    try:
        sig = ("kv_append", key.shape, key.stride(), key.dtype, key.device, value.shape, value.stride(), value.dtype,
               value.device, k_cache.shape, k_cache.stride(), k_cache.dtype, k_cache.device, v_cache.shape,
               v_cache.stride(), v_cache.dtype, v_cache.device, page_table.shape, page_table.stride(), page_table.dtype,
               page_table.device, lengths.shape, lengths.stride(), lengths.dtype, lengths.device, sections, interleaved)
        for t in (new_lengths, query, positions, freqs):
            sig += (None,) if t is None else (t.shape, t.stride(), t.dtype, t.device)
        how = _SIGNATURES.get(sig)
    except (AttributeError, TypeError):
        sig = how = None
    if how is not None:
        middle, tail, index = how
        out = None if query is None else _like_of(query)
        data = b"".join((
            _pack9(key.data_ptr(), value.data_ptr(), 0 if out is None else query.data_ptr(),
                   0 if out is None else out.data_ptr(), 0 if new_lengths is None else new_lengths.data_ptr(),
                   k_cache.data_ptr(), v_cache.data_ptr(), page_table.data_ptr(), lengths.data_ptr()),
            middle, _pack2(0 if positions is None else positions.data_ptr(), 0 if freqs is None else freqs.data_ptr()),
            tail))
        if _direct(_KV_APPEND, data, index) == OK:
            _changed(k_cache, v_cache)
            return out
    desc, out, used = _append_desc(key, value, k_cache, v_cache, page_table, lengths, new_lengths, query, positions,
                                   freqs, sections, interleaved)
    if desc.batch and desc.len:
        _run("kv_append", lib.cmpx_kv_append, desc, key.device)
        _changed(k_cache, v_cache)
        if (sig is not None and used[0] is key and used[1] is value and used[2] is query
                and (out is None or _is_like(out, query)) and (freqs is None or used[3][-1] is freqs)):
            data, at = bytes(desc), KvAppendDesc.rot.offset
            _keep(sig, (data[72:at], data[at + 16:], key.device.index))
    return out


def _changed(*caches) -> None:
    """Counts the caches as written in place, for autograd's check of saved tensors."""
    for t in caches:
        if not t.is_inference():
            torch.autograd.graph.increment_version(t)


def kv_append_plan(key, value, k_cache, v_cache, page_table, lengths, new_lengths=None, query=None, positions=None,
                   freqs=None, sections=None, interleaved=False) -> str:
    """Name of the kernel ``kv_append`` runs for these arguments."""
    desc, _out, _used = _append_desc(key, value, k_cache, v_cache, page_table, lengths, new_lengths, query, positions,
                                     freqs, sections, interleaved)
    return _plan("kv_append", lib.cmpx_kv_append_plan, desc)


def _paged_attn_desc(query, k_cache, v_cache, page_table, lengths, scale):
    device = _rows("query", query)
    b, heads, n, d = query.shape
    if n != 1:
        raise RuntimeError(f"query must have one token per sequence, got {n}")
    cache = _paged(k_cache, v_cache, page_table, lengths, b, query.dtype, device)
    if cache.head_dim != d or heads % cache.heads_kv:
        raise RuntimeError(f"k_cache {tuple(k_cache.shape)} does not match query {tuple(query.shape)}")
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if not abs(scale) * math.log2(math.e) <= torch.finfo(torch.float32).max:  # the kernels' factor, of scores in log2 units
        raise RuntimeError("scale must be finite (in fp32)")
    st = query.stride()
    unit = 16 // query.element_size()
    if st[3] != 1 or b > 1 and st[0] % unit or heads > 1 and st[1] % unit or query.data_ptr() % 16:
        query = query.contiguous()
        if query.data_ptr() % 16:
            query = query.clone()
        st = query.stride()
    out, os_ = _like(query)  # whose rows are on 16-byte boundaries
    desc = PagedAttnDesc(query.data_ptr(), out.data_ptr(), None, cache, 0, b, heads, _I64x2(st[0], st[1]),
                         _I64x2(os_[0], os_[1]), scale, _DTYPE[query.dtype], 0)
    return desc, out, query


@_traced("paged_attention")
def paged_attention(query, k_cache, v_cache, page_table, lengths, scale=None):
    """Attention of one new token per sequence, query [batch, heads, 1, head_dim], over the first
    lengths[b] tokens of a paged cache (laid out as for ``kv_append``); heads is a multiple of heads_kv
    and query head h reads key head h // (heads // heads_kv).  scale defaults to 1 / sqrt(head_dim);
    head_dim <= 256, a multiple of 8 (fp32: of 4).  Returns [batch, heads, 1, head_dim].

    A sequence of length 0 gets zeros.  A length beyond the table, or a page that does not exist among a
    sequence's pages, makes that sequence's rows NaN and sets a bit of ``device_status()``.  The lengths
    are read on the device: a captured call can be replayed with other ones.  The schedule goes by the
    table's width: a table much wider than the sequences are long costs a few microseconds."""
    scale = None if scale is None else float(scale)
    if torch.is_grad_enabled():
        _no_grad_only("paged_attention", query, k_cache, v_cache)
    if _forward._current_level >= 0:
        _no_tangent("paged_attention", query, k_cache, v_cache)
    try:
        sig = ("paged_attention", query.shape, query.stride(), query.dtype, query.device, k_cache.shape, k_cache.stride(),
               k_cache.dtype, k_cache.device, v_cache.shape, v_cache.stride(), v_cache.dtype, v_cache.device,
               page_table.shape, page_table.stride(), page_table.dtype, page_table.device, lengths.shape,
               lengths.stride(), lengths.dtype, lengths.device, scale)
        how = _SIGNATURES.get(sig)
    except (AttributeError, TypeError):
        sig = how = None
    if how is not None:
        tail, scratch, index = how
        out = _like_of(query)
        ws = None if scratch is None else _like_of(scratch)
        data = _pack7(query.data_ptr(), out.data_ptr(), 0 if ws is None else ws.data_ptr(), k_cache.data_ptr(),
                      v_cache.data_ptr(), page_table.data_ptr(), lengths.data_ptr()) + tail
        if _direct(_PAGED_ATTN, data, index) == OK:
            return out
    desc, out, used = _paged_attn_desc(query, k_cache, v_cache, page_table, lengths, scale)
    if out.numel():
        dev = out.device
        with torch.cuda.device(dev):
            nbytes = lib.cmpx_paged_attn_workspace_size(ctypes.byref(desc))
        if nbytes:  # this call's own: concurrent calls and captured graphs share none
            ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
            desc.workspace, desc.workspace_bytes = ws.data_ptr(), nbytes
        _run("paged_attention", lib.cmpx_paged_attn, desc, dev)
        if sig is not None and used is query and _is_like(out, query):
            _keep(sig, (bytes(desc)[56:], _alike((nbytes,), torch.uint8, dev) if nbytes else None, dev.index))
    return out


def paged_attention_plan(query, k_cache, v_cache, page_table, lengths, scale=None) -> str:
    """Name of the schedule ``paged_attention`` runs for these arguments."""
    desc, _out, _used = _paged_attn_desc(query, k_cache, v_cache, page_table, lengths, scale)
    return _plan("paged_attention", lib.cmpx_paged_attn_plan, desc)


# ---------------------------------------------------------------------------------------------
# linear with 4-bit weights
# ---------------------------------------------------------------------------------------------

def _aligned_rows(t: torch.Tensor) -> torch.Tensor:
    """A 2-D operand with contiguous rows on 16-byte boundaries (a copy where it has none)."""
    row = t.stride(0) * t.element_size()
    if t.stride(1) == 1 and t.data_ptr() % 16 == 0 and (t.shape[0] == 1 or row % 16 == 0 and row <= 1 << 27):
        return t
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def _linear_w4_desc(input, weight, scales, zeros, bias):
    if not isinstance(input, torch.Tensor):
        raise TypeError("input must be a Tensor")
    if not input.is_cuda or input.dtype not in _DTYPE:
        raise RuntimeError("input must be a CUDA float32/float16/bfloat16 tensor")
    if input.dim() < 1:
        raise RuntimeError("input must have at least one dimension")
    device, dtype = input.device, input.dtype
    _tensor("weight", weight, 2, torch.uint8, device)
    _tensor("scales", scales, 2, dtype, device)
    n, k = weight.shape[0], 2 * weight.shape[1]
    groups = scales.shape[1]
    if input.shape[-1] != k:
        raise RuntimeError(f"input {tuple(input.shape)} does not match weight [{n}, {k} / 2]")
    if scales.shape[0] != n or groups < 1 or k % groups or (k // groups) % 32 or k == 0:
        raise RuntimeError(f"scales {tuple(scales.shape)} must be [{n}, {k} / group] with a group that is a multiple of 32")
    if zeros is not None:
        _tensor("zeros", zeros, 2, torch.uint8, device)
        if zeros.shape != scales.shape:
            raise RuntimeError(f"zeros {tuple(zeros.shape)} does not match scales {tuple(scales.shape)}")
        zeros = _unit(zeros)
    if bias is not None:
        _tensor("bias", bias, 1, dtype, device)
        if bias.shape[0] != n:
            raise RuntimeError(f"bias must have {n} values")
        bias = _unit(bias)
    x, w, scales = _aligned_rows(input.reshape(-1, k)), _aligned_rows(weight), _unit(scales)
    y = torch.empty((x.shape[0], n), dtype=dtype, device=device)
    desc = LinearW4Desc(x.data_ptr(), w.data_ptr(), scales.data_ptr(), None if zeros is None else zeros.data_ptr(),
                        None if bias is None else bias.data_ptr(), y.data_ptr(), x.shape[0], n, k, k // groups,
                        x.stride(0), n, w.stride(0), scales.stride(0), 0 if zeros is None else zeros.stride(0),
                        _DTYPE[dtype], 0)
    return desc, y, (x, w, scales, zeros, bias)


@_traced("linear_w4")
def linear_w4(input, weight, scales, zeros=None, bias=None):
    """Linear layer with 4-bit weights, for a few tokens:  y = input W^T (+ bias) with
    W[n, k] = (code[n, k] - zero[n, k // group]) * scale[n, k // group].

    input [..., K]; weight [N, K // 2] uint8, two codes (0..15) a byte, the even k in the low half;
    scales [N, K // group] in input's dtype; zeros [N, K // group] uint8 (0..15), 8 everywhere when
    None; bias [N] in input's dtype.  group, a multiple of 32 that divides K, follows from scales.  The
    weights are not rounded (whole-number differences, fp32 sums, one product with the scale a group)
    and the result is rounded once.  The weights are read once per 16 tokens: with many tokens a
    dequantised weight and ``linear`` are the faster way."""
    if torch.is_grad_enabled():
        _no_grad_only("linear_w4", input, scales, bias)
    if _forward._current_level >= 0:
        _no_tangent("linear_w4", input, scales, bias)
    try:
        sig = ("linear_w4", input.shape, input.stride(), input.dtype, input.device, weight.shape, weight.stride(),
               weight.dtype, weight.device, scales.shape, scales.stride(), scales.dtype, scales.device)
        for t in (zeros, bias):
            sig += (None,) if t is None else (t.shape, t.stride(), t.dtype, t.device)
        how = _SIGNATURES.get(sig)
    except (AttributeError, TypeError):
        sig = how = None
    if how is not None:
        tail, like, index = how
        y = _like_of(like)
        data = _pack6(input.data_ptr(), weight.data_ptr(), scales.data_ptr(), 0 if zeros is None else zeros.data_ptr(),
                      0 if bias is None else bias.data_ptr(), y.data_ptr()) + tail
        if _direct(_LINEAR_W4, data, index) == OK:
            return y
    desc, y, used = _linear_w4_desc(input, weight, scales, zeros, bias)
    shape = tuple(input.shape[:-1]) + (y.shape[1],)
    if y.numel():
        _run("linear_w4", lib.cmpx_linear_w4, desc, y.device)
        if (sig is not None and used[0].data_ptr() == input.data_ptr()
                and all(a is b for a, b in zip(used[1:], (weight, scales, zeros, bias)))):
            _keep(sig, (bytes(desc)[48:], _alike(shape, y.dtype, y.device), y.device.index))
    return y.view(shape)


def linear_w4_plan(input, weight, scales, zeros=None, bias=None) -> str:
    """Name of the kernel ``linear_w4`` runs for these arguments."""
    desc, _y, _used = _linear_w4_desc(input, weight, scales, zeros, bias)
    return _plan("linear_w4", lib.cmpx_linear_w4_plan, desc)
