"""Attention over a paged cache whose page table is CSR: rotary positions, appending to the
cache, and attention of a batch whose sequences share a prefix.

``sddmm`` and ``spmm`` are the two products of attention over a CSR pattern; a served model's
pattern is its page table.  Sequence b's pages are ``indices[indptr[b]:indptr[b + 1]]``, int64
as everywhere in this package, each a page of ``[pages, page, kv_heads, dim]`` caches; its
token at position p stands in slot ``p % page`` of its page ``p // page``.  Pages that a whole
batch shares are a list of their own and are read once for the batch.

Operands are torch tensors on one HIP device, bfloat16 or float16 (``rope`` and
``paged_append`` float32 too); any strides whose heads are contiguous.  Kernels are enqueued on
torch's current stream of that device and nothing waits for them.  Calls that the kernels
cannot serve raise ``ValueError`` before anything is enqueued, ones that autograd would have to
follow among them (``rope`` and ``rope_backward`` alone have a backward pass); HIP's own failures
raise ``TileGenHipError``.  The C ABI below is ``include/tilegen_attention.h`` (``libtgattn.so``); it
allocates nothing, and may be captured into a graph like the calls here.

    frequency, magnitude = rope_frequencies(128, scaling="yarn", factor=32, trained=4096)
    lengths += 1                              # of each sequence's own pages, new token included
    q = paged_append(k, v, key_cache, value_cache, indptr, indices, lengths, frequency,
                     query=q, offset=prefix_length, magnitude=magnitude)
    o = prefix_attention(q, key_cache, value_cache, prefix, prefix_length, indptr, indices,
                         lengths, max_length=1024)
"""

from __future__ import annotations

import ctypes
import math
import os
import struct
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad as _forward

from . import runtime as _rt

__all__ = ["rope_frequencies", "rope", "rope_backward", "paged_append", "prefix_attention"]

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_LAYOUTS = {"half": 0, "interleaved": 1}

# include/tilegen_attention.h: tg_rope, tg_paged_append, tg_prefix_attention
_ROPE = struct.Struct("4P10qdq")
_APPEND = struct.Struct("11P26qd")
_ATTENTION = struct.Struct("11P24qd")


def _unfit(e: struct.error) -> ValueError:
    return ValueError("a size, bound or offset that is no 64-bit whole number, or a factor that is "
                      "no number: %s" % e)


_LIB = None


def _lib():
    global _LIB
    if _LIB is None:
        _rt.lib()  # the runtime first, RTLD_GLOBAL
        path = os.path.join(_rt.lib_dir(), "libtgattn.so")
        if not os.path.exists(path):
            raise _rt.TileGenHipError("libtgattn.so is not built (%s); run "
                                      "__graft_entry__.build()" % path)
        L = ctypes.CDLL(path)
        for name in ("launch_rope", "launch_paged_append", "launch_prefix_attention"):
            getattr(L, name).argtypes = [ctypes.c_char_p, ctypes.c_void_p]
            getattr(L, name).restype = ctypes.c_int
        L.prefix_attention_workspace.argtypes = [ctypes.c_char_p]
        L.prefix_attention_workspace.restype = ctypes.c_int64
        _LIB = L
    return _LIB


# --------------------------------------------------------------------------- #
# checks
# --------------------------------------------------------------------------- #
# The checks are most of what a small call costs the host, so each asks the common case in one
# condition and works out what is wrong only when it fails.
def _heads(name: str, t: torch.Tensor, device: int, dtype: torch.dtype, dims: int,
           write: bool = False):
    """(shape, strides) of an operand whose last axis is a head."""
    shape, strides = t.shape, t.stride()
    if not (t.get_device() == device and t.dtype is dtype and len(shape) == dims
            and (strides[-1] == 1 or shape[-1] <= 1)):
        _refuse_heads(name, t, device, dtype, dims)
    if write and 0 in strides and any(s == 0 and n > 1 for s, n in zip(strides, shape)):
        raise ValueError("%s is written, but its elements share memory (strides %s)"
                         % (name, strides))
    return shape, strides


def _refuse_heads(name, t, device, dtype, dims):
    if t.get_device() != device or t.dtype != dtype:
        raise ValueError("%s is %s on %s, expected %s on device %d" % (name, t.dtype, t.device,
                                                                       dtype, device))
    if t.dim() != dims:
        raise ValueError("%s has %d axes, expected %d" % (name, t.dim(), dims))
    raise ValueError("%s: the elements of a head are not contiguous (strides %s)"
                     % (name, t.stride()))


def _list(name: str, t: torch.Tensor, device: int, n: Optional[int] = None,
          dtype: torch.dtype = torch.int64) -> int:
    """The address of a one-dimensional contiguous array (of n entries)."""
    if not (t.get_device() == device and t.dtype is dtype and t.dim() == 1
            and t.is_contiguous()):
        raise ValueError("%s is %s %s on %s, expected a contiguous list of %s on device %d" % (
            name, t.dtype, tuple(t.shape), t.device, dtype, device))
    if n is not None and t.shape[0] != n:
        raise ValueError("%s has %d entries, expected %d" % (name, t.shape[0], n))
    return t.data_ptr()


def _operand(name: str, t: torch.Tensor, dtypes) -> Tuple[int, torch.dtype]:
    """(device, type) that a call goes by."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError("%s is not a tensor on a HIP device" % name)
    if t.dtype not in dtypes:
        raise ValueError("%s is %s, expected one of %s" % (name, t.dtype,
                                                           ", ".join(map(str, dtypes))))
    return t.get_device(), t.dtype


def _like(x: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(x, memory_format=torch.contiguous_format)


def _layout(layout: str) -> int:
    if layout not in _LAYOUTS:
        raise ValueError("layout is %r, expected 'half' or 'interleaved'" % (layout,))
    return _LAYOUTS[layout]


# torch's current stream as a handle, without the object that current_stream() builds (2.7 us)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda device: torch.cuda.current_stream(device).cuda_stream)


def _on(device: int, entry, *args) -> int:
    """A C entry with the operands' device current: it launches there, and plans for its units."""
    if device == torch.cuda.current_device():
        return entry(*args)
    with torch.cuda.device(device):
        return entry(*args)


def _call(entry, packed: bytes, device: int, what: str) -> None:
    rc = _on(device, entry, packed, _raw_stream(device))
    if rc:
        _raise(rc, what)


# Tells autograd that the kernels write over tensors that it may have saved.
_written = torch.autograd.graph.increment_version


def _raise(rc: int, what: str) -> None:
    if rc < 0:  # an argument the library refused
        raise ValueError(_rt.last_error())
    _rt.check(rc, what)


# --------------------------------------------------------------------------- #
# rotary positions
# --------------------------------------------------------------------------- #
def rope_frequencies(rotary: int, base: float = 10000.0, scaling: Optional[str] = None,
                     factor: float = 1.0, trained: int = 0, beta_fast: float = 32.0,
                     beta_slow: float = 1.0, device="cuda") -> Tuple[torch.Tensor, float]:
    """(frequency, magnitude) for ``rope``: radians per position of each of the rotary / 2
    pairs, in 64 bits, base^(-2 i / rotary) scaled for contexts ``factor`` times as long:

    None       as it is
    "linear"   positions divided by factor
    "ntk"      base raised to base * factor^(rotary / (rotary - 2)): the lowest frequency is
               divided by factor, the highest kept
    "yarn"     by parts: pairs that turn at least beta_fast times over the ``trained``
               positions are kept, those that turn at most beta_slow times divided by factor,
               a ramp between; magnitude 0.1 ln(factor) + 1
    """
    if rotary < 0 or rotary % 2:
        raise ValueError("rotary is %d, expected an even number" % rotary)
    if not base > 0 or not factor >= 1:
        raise ValueError("base must be positive and factor at least 1")
    if scaling == "ntk" and rotary > 2:
        base = base * factor ** (rotary / (rotary - 2))
    f = [base ** (-i / rotary) for i in range(0, rotary, 2)]
    magnitude = 1.0
    if scaling == "linear":
        f = [x / factor for x in f]
    elif scaling == "yarn":
        if trained < 1 or not beta_fast > beta_slow:
            raise ValueError("yarn needs the trained length, and beta_fast over beta_slow")
        for i, x in enumerate(f):
            turns = trained * x / (2 * math.pi)
            keep = min(1.0, max(0.0, (turns - beta_slow) / (beta_fast - beta_slow)))
            f[i] = x * keep + x / factor * (1 - keep)
        magnitude = 0.1 * math.log(factor) + 1.0
    elif scaling not in (None, "ntk"):
        raise ValueError("scaling is %r, expected None, 'linear', 'ntk' or 'yarn'" % (scaling,))
    return torch.tensor(f, dtype=torch.float64, device=device), magnitude


def _turn(x, positions, frequency, layout, magnitude, out, sign, what):
    device, dtype = _operand("x", x, _DTYPES)
    shape, xs = _heads("x", x, device, dtype, 3)
    given = out is not None
    if not given:
        out = _like(x)
    oshape, ys = _heads("out", out, device, dtype, 3, write=True)
    if oshape != shape:
        raise ValueError("out is %s, expected %s" % (tuple(oshape), tuple(shape)))
    tokens, heads, dim = shape
    try:
        packed = _ROPE.pack(
            x.data_ptr(), out.data_ptr(), _list("positions", positions, device, tokens),
            _list("frequency", frequency, device, dtype=torch.float64), _DTYPES[dtype], tokens,
            heads, dim, 2 * frequency.shape[0], _layout(layout), xs[0], xs[1], ys[0], ys[1],
            magnitude, sign)
    except struct.error as e:
        raise _unfit(e) from None
    _call(_lib().launch_rope, packed, device, what)
    if given:
        _written(out)
    return out


def _tangent(t) -> bool:
    return _forward._current_level >= 0 and _forward.unpack_dual(t).tangent is not None


def _followed(t: torch.Tensor) -> bool:
    """Whether autograd follows t, backward or forward."""
    return (t.requires_grad and torch.is_grad_enabled()) or _tangent(t)


def _no_gradient(what: str, *operands: Optional[torch.Tensor]) -> None:
    """Refuses what autograd would follow: its results would have no gradient, silently.  An output
    that it follows would lose its own."""
    lost = False
    if torch.is_grad_enabled():
        for t in operands:
            if t is not None and t.requires_grad:
                lost = True
    if _forward._current_level >= 0:
        lost = lost or any(_tangent(t) for t in operands if t is not None)
    if lost:
        raise ValueError("%s has no backward pass for these operands: call it under "
                         "torch.no_grad(), or with detached operands" % what)


class _Rope(torch.autograd.Function):
    """The map is linear in x: its derivative along a tangent is the same map, its gradient the
    transposed one, and either is a call that autograd may follow again."""

    @staticmethod
    def forward(ctx, x, positions, frequency, layout, magnitude, sign):
        ctx.save_for_backward(positions, frequency)
        ctx.save_for_forward(positions, frequency)
        ctx.how = layout, magnitude, sign
        return _turn(x, positions, frequency, layout, magnitude, None, sign, "rope")

    @staticmethod
    def _again(ctx, x, flip):
        if x is None:
            return None
        positions, frequency = ctx.saved_tensors
        layout, magnitude, sign = ctx.how
        if x.stride(-1) != 1:       # a broadcast gradient, of a sum for example
            x = x.contiguous()
        return _linear(x, positions, frequency, layout, magnitude, None, flip * sign, "rope")

    @staticmethod
    def backward(ctx, grad):
        return _Rope._again(ctx, grad, -1), None, None, None, None, None

    @staticmethod
    def jvp(ctx, tangent, *_):
        return _Rope._again(ctx, tangent, 1)


def _linear(x, positions, frequency, layout, magnitude, out, sign, what):
    forward = _forward._current_level >= 0
    if getattr(x, "requires_grad", False) or forward:
        if _followed(x):
            if out is not None:
                raise ValueError("out cannot be given where x needs a gradient")
            _no_gradient(what, frequency)
            return _Rope.apply(x, positions, frequency, layout, magnitude, sign)
    if frequency.requires_grad or out is not None or forward:
        _no_gradient(what, frequency, out)
    return _turn(x, positions, frequency, layout, magnitude, out, sign, what)


def rope(x: torch.Tensor, positions: torch.Tensor, frequency: torch.Tensor, *,
         layout: str = "half", magnitude: float = 1.0,
         out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x [tokens, heads, dim] with its pairs turned by ``positions[t] * frequency[i]`` and
    multiplied by ``magnitude``: (a, b) becomes (a cos - b sin, b cos + a sin).

    A pair is elements (i, i + n) (layout "half") or (2 i, 2 i + 1) ("interleaved") of the
    first 2 n elements of each head, n = len(frequency); the others are copied.  Angles are
    taken in 64 bits, so positions may be as large as they come; the turn is made in 32 bits
    and rounded once.  ``out`` may be x itself, and share no other memory with it.  Heads may be
    those of a packed projection (``qkv[:, :heads + kv_heads]``), queries and keys in one call.
    Differentiable in x, as often as need be, backward and forward."""
    return _linear(x, positions, frequency, layout, magnitude, out, 1, "rope")


def rope_backward(grad: torch.Tensor, positions: torch.Tensor, frequency: torch.Tensor, *,
                  layout: str = "half", magnitude: float = 1.0,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The gradient of ``rope`` by x: the transposed map, which turns the other way.
    Differentiable in grad."""
    return _linear(grad, positions, frequency, layout, magnitude, out, -1, "rope_backward")


# --------------------------------------------------------------------------- #
# the cache
# --------------------------------------------------------------------------- #
def _caches(key_cache, value_cache, device, dtype, write):
    kshape, ks = _heads("key_cache", key_cache, device, dtype, 4, write)
    vshape, vs = _heads("value_cache", value_cache, device, dtype, 4, write)
    if kshape != vshape:
        raise ValueError("key_cache is %s and value_cache %s" % (tuple(kshape), tuple(vshape)))
    return kshape, ks, vs


def _table(indptr, indices, lengths, query_indptr, tokens, device):
    """(addresses, sequences) of a page table and what goes with it."""
    sequences = lengths.shape[0] if lengths.dim() == 1 else -1
    at = (_list("indptr", indptr, device, sequences + 1), _list("indices", indices, device),
          _list("lengths", lengths, device), 0 if query_indptr is None else
          _list("query_indptr", query_indptr, device, sequences + 1))
    if query_indptr is None and tokens != sequences:
        raise ValueError("%d tokens for %d sequences: query_indptr says whose they are"
                         % (tokens, sequences))
    return at, sequences


def paged_append(key: torch.Tensor, value: torch.Tensor, key_cache: torch.Tensor,
                 value_cache: torch.Tensor, indptr: torch.Tensor, indices: torch.Tensor,
                 lengths: torch.Tensor, frequency: Optional[torch.Tensor] = None, *,
                 query: Optional[torch.Tensor] = None,
                 query_out: Optional[torch.Tensor] = None,
                 query_indptr: Optional[torch.Tensor] = None, offset: int = 0,
                 layout: str = "half", magnitude: float = 1.0) -> Optional[torch.Tensor]:
    """Writes the new tokens' key and value [tokens, kv_heads, dim] into the caches, keys
    turned as ``rope`` does (``frequency=None``: as they are), and returns the same tokens'
    ``query`` [tokens, heads, dim] turned with them, in one launch.

    ``lengths[b]`` counts the tokens of sequence b's own pages, the new ones included: its n new
    tokens, rows query_indptr[b] to query_indptr[b + 1] (one each where that is None), go to
    positions lengths[b] - n and on, and are turned at ``offset`` (the shared prefix's length)
    more.  A token whose page is not on its list, or not in the cache, is left out.  Rows before
    query_indptr[0] (slices of a larger batch's row pointers) and from query_indptr[-1] on (a
    batch padded for a graph) belong to no sequence: nothing is written for them and their
    queries come back zero.  ``query_out`` may be ``query`` itself, and share no other memory
    with the operands."""
    device, dtype = _operand("key", key, _DTYPES)
    _no_gradient("paged_append", key, value, query, key_cache, value_cache, frequency, query_out)
    shape, ks = _heads("key", key, device, dtype, 3)
    vshape, vs = _heads("value", value, device, dtype, 3)
    cache, kcs, vcs = _caches(key_cache, value_cache, device, dtype, True)
    tokens, kv_heads, dim = shape
    if vshape != shape or cache[2:] != shape[1:]:
        raise ValueError("key is %s, value %s and the caches %s" % (tuple(shape), tuple(vshape),
                                                                    tuple(cache)))
    (p_indptr, p_indices, p_lengths, p_ends), sequences = _table(
        indptr, indices, lengths, query_indptr, tokens, device)
    heads, q, out, qs, os_ = 0, 0, 0, (0, 0), (0, 0)
    written = (key_cache, value_cache)
    if query is not None:
        qshape, qs = _heads("query", query, device, dtype, 3)
        if qshape[0] != tokens or qshape[2] != dim:
            raise ValueError("query is %s, key %s" % (tuple(qshape), tuple(shape)))
        if query_out is None:
            query_out = _like(query)
        else:
            written += (query_out,)
        oshape, os_ = _heads("query_out", query_out, device, dtype, 3, write=True)
        if oshape != qshape:
            raise ValueError("query_out is %s, expected %s" % (tuple(oshape), tuple(qshape)))
        heads, q, out = qshape[1], query.data_ptr(), query_out.data_ptr()
    elif query_out is not None:
        raise ValueError("query_out without query")
    p_frequency, rotary = 0, 0
    if frequency is not None:
        p_frequency = _list("frequency", frequency, device, dtype=torch.float64)
        rotary = 2 * frequency.shape[0]
    try:
        packed = _APPEND.pack(
            key.data_ptr(), value.data_ptr(), q, key_cache.data_ptr(), value_cache.data_ptr(), out,
            p_indptr, p_indices, p_lengths, p_ends, p_frequency, _DTYPES[dtype], tokens, sequences,
            heads, kv_heads, dim, rotary, _layout(layout), cache[0], cache[1], indices.shape[0],
            offset, ks[0], ks[1], vs[0], vs[1], qs[0], qs[1], os_[0], os_[1], kcs[0], kcs[1],
            kcs[2], vcs[0], vcs[1], vcs[2], magnitude)
    except struct.error as e:
        raise _unfit(e) from None
    _call(_lib().launch_paged_append, packed, device, "paged_append")
    _written(written)
    return query_out


# --------------------------------------------------------------------------- #
# attention
# --------------------------------------------------------------------------- #
_CACHED = (torch.bfloat16, torch.float16)


def _attend(query, fields, packed: bytes, device: int) -> int:
    """Plans and launches with the device current, the workspace from torch."""
    L = _lib()
    n = L.prefix_attention_workspace(packed)
    if n < 0:
        return n
    if n:
        workspace = query.new_empty(n, dtype=torch.uint8)
        fields[10], fields[11] = workspace.data_ptr(), n
        packed = _ATTENTION.pack(*fields)
    return L.launch_prefix_attention(packed, _raw_stream(device))


def prefix_attention(query: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                     prefix: torch.Tensor, prefix_length: int, indptr: torch.Tensor,
                     indices: torch.Tensor, lengths: torch.Tensor, *, max_length: int,
                     query_indptr: Optional[torch.Tensor] = None, max_query: int = 1,
                     scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                     return_lse: bool = False):
    """softmax(scale q.k) v of each new token's query [tokens, heads, dim] over the first
    ``prefix_length`` keys of the pages ``prefix``, which all sequences share, and the keys of
    its sequence's own pages up to its own position (``paged_append`` has written them:
    ``lengths`` and ``query_indptr`` are the same).

    Query head h reads kv head h // (heads // kv_heads); dim is a multiple of 8 up to 256;
    ``scale`` is 1 / sqrt(dim) by default.  ``max_query`` and ``max_length`` bound the new tokens
    and the length of a sequence: they size the launch (larger ones on the device are still
    right, only slower).  A row that sees no key (or scores of -inf alone), or belongs to no
    sequence, gives 0; what hidden keys and values hold does not matter.  With ``return_lse``
    also each row's logarithm of the sum of its exponentials, float32 [tokens, heads] (-inf for
    such a row), by which results over disjoint keys can be joined.  ``out`` may be the query,
    and share no other memory with the operands.

    Scores, probabilities and sums are held in 32 bits; probabilities are rounded to the
    caches' type for the matrix instructions that weigh the values.  Results do not depend on
    the order in which workgroups run."""
    device, dtype = _operand("query", query, _CACHED)
    _no_gradient("prefix_attention", query, key_cache, value_cache, out)
    shape, qs = _heads("query", query, device, dtype, 3)
    cache, kcs, vcs = _caches(key_cache, value_cache, device, dtype, False)
    tokens, heads, dim = shape
    if cache[3] != dim or not cache[2] or heads % cache[2]:
        raise ValueError("query is %s, the caches %s" % (tuple(shape), tuple(cache)))
    (p_indptr, p_indices, p_lengths, p_ends), sequences = _table(
        indptr, indices, lengths, query_indptr, tokens, device)
    given = out is not None
    if not given:
        out = _like(query)
    oshape, os_ = _heads("out", out, device, dtype, 3, write=True)
    if oshape != shape:
        raise ValueError("out is %s, expected %s" % (tuple(oshape), tuple(shape)))
    lse = query.new_empty(shape[:2], dtype=torch.float32) if return_lse else None
    fields = [query.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(),
              _list("prefix", prefix, device), p_indptr, p_indices, p_lengths, p_ends,
              out.data_ptr(), lse.data_ptr() if return_lse else 0, 0, 0, _DTYPES[dtype], tokens,
              sequences, heads, cache[2], dim, cache[0], cache[1], prefix.shape[0],
              prefix_length, indices.shape[0], max_query, max_length, qs[0], qs[1], os_[0],
              os_[1], kcs[0], kcs[1], kcs[2], vcs[0], vcs[1], vcs[2],
              dim ** -0.5 if scale is None else scale]
    try:
        packed = _ATTENTION.pack(*fields)
    except struct.error as e:
        raise _unfit(e) from None
    rc = _on(device, _attend, query, fields, packed, device)
    if rc:
        _raise(rc, "prefix_attention")
    if given:
        _written(out)
    return (out, lse) if return_lse else out
