"""K/V caches in 8 bits, and attention over cached keys.

Three operators over the C ABI (include/dh_b200.h):

* :func:`write_kv` -- K and V rows into an int8 cache as they are produced, a
  scale for each position and head (:class:`KVCacheI8`).
* :func:`read_kv` -- positions of such a cache back in floating point.
* :func:`attend` -- attention over the keys of a cache (int8, or 16-bit tensors)
  with a number of keys for each sequence, and behind a prefix that a batch
  shares and that is held and read once (prefix_drift._cached_suffix_forward,
  prefix_drift.py:155-238, keeps one for each sequence).

Every call runs on the current stream of its tensors' device, returns without
waiting for it, and can be captured in a CUDA graph.  Arguments are checked
before anything is launched; starts, counts and lengths that lie on the device
are not, but are kept inside the cache.  Results carry no gradients, and an
`out` tensor must not overlap the inputs.
"""

from __future__ import annotations

import functools
import operator
import struct
from typing import Any, NamedTuple, Optional, Tuple, Union

import torch

from . import _lib
from .scoring import _TYPES, _current_device, _ptr, _raw_stream

HEAD_DIM = 64
CAPACITY_STEP = 64
_TYPE_I8 = 3
# Work and workspace go by the capacity of a view.  Of caches with more positions than
# this, a call whose length the host knows shows only as many keys as that (8 x 512
# queries, 12 heads, over 500 of 32768 int8 keys: 49.2 us and 19 MB, whole 54.8 and 851;
# one over 33 of 2048 4.4 and 7.0 us).  In smaller ones lengths on the host and on the
# device give the same bits.
_WHOLE_KEYS = 512

Lengths = Union[int, torch.Tensor, None]


class KVCacheI8(NamedTuple):
    """Int8 K and V of ``entries`` sequences: position p of a head holds the row
    ``codes[p] * scale[p]``.  Build one with :meth:`empty`, or from tensors of
    these shapes, contiguous, with a capacity that is a multiple of 64."""

    k: torch.Tensor        # int8 [entries, heads, capacity, 64]
    k_scale: torch.Tensor  # fp32 [entries, heads, capacity]
    v: torch.Tensor
    v_scale: torch.Tensor

    @classmethod
    def empty(cls, entries: int, heads: int, capacity: int, device: Any = "cuda") -> "KVCacheI8":
        """Room for `capacity` positions (rounded up to a multiple of 64); what
        it holds is undefined until it is written."""
        if entries <= 0 or heads <= 0 or capacity <= 0:
            raise ValueError("entries, heads and capacity must be positive")
        capacity = -(-capacity // CAPACITY_STEP) * CAPACITY_STEP
        codes = [torch.empty((entries, heads, capacity, HEAD_DIM), dtype=torch.int8, device=device) for _ in range(2)]
        scales = [torch.empty((entries, heads, capacity), dtype=torch.float32, device=device) for _ in range(2)]
        return cls(codes[0], scales[0], codes[1], scales[1])

    @property
    def capacity(self) -> int:
        return self.k.shape[2]

    def nbytes(self, positions: Optional[int] = None) -> int:
        """Bytes that `positions` positions of every entry take (default: all)."""
        n, h, c, d = self.k.shape
        return n * h * (c if positions is None else positions) * 2 * (d + 4)


# Calls take a few microseconds of the host and the smallest of them little more of
# the GPU: a call that is as it should be passes few checks, and what it passes to C
# is packed in one go.
_pack4 = struct.Struct("=4Q").pack
_pack_view = struct.Struct("=5Q8Q4I").pack  # dh_kv_view of include/dh_b200.h


def _check_cache(name: str, c: KVCacheI8, index: int) -> tuple:
    """Shape of the codes of a cache that is all on GPU `index` (-1: the host)."""
    k, k_scale, v, v_scale = c
    shape = k.shape
    if index < 0 or not (k.get_device() == v.get_device() == k_scale.get_device() == v_scale.get_device() == index):
        if k.is_cuda:
            raise ValueError(f"all of {name} and the other tensors must be on one device")
        raise ValueError(f"{name} must hold CUDA tensors")
    if len(shape) != 4 or shape[3] != HEAD_DIM or shape[2] == 0 or shape[2] % CAPACITY_STEP:
        raise ValueError(f"{name} must hold int8 codes [entries, heads, capacity, 64], its capacity a multiple of 64")
    if not (v.shape == shape and k_scale.shape == v_scale.shape == shape[:3]):
        raise ValueError(f"the codes and scales of {name} must have one shape")
    if not (k.dtype is v.dtype is torch.int8 and k_scale.dtype is v_scale.dtype is torch.float32):
        raise ValueError(f"{name} must hold int8 codes and float32 scales")
    if not (k.is_contiguous() and v.is_contiguous() and k_scale.is_contiguous() and v_scale.is_contiguous()):
        raise ValueError(f"the tensors of {name} must be contiguous")
    if (k.data_ptr() | v.data_ptr() | k_scale.data_ptr() | v_scale.data_ptr()) & 15:
        raise ValueError(f"the tensors of {name} must start at 16-byte boundaries")
    return shape


def _on(name: str, t: torch.Tensor, index: int) -> torch.Tensor:
    if t.get_device() != index:
        raise ValueError(f"{name} must be a CUDA tensor on the device of the others")
    return t


def _ints(name: str, t: torch.Tensor, n: int, index: int) -> torch.Tensor:
    _on(name, t, index)
    if t.dtype is not torch.int32 or t.shape != (n,):
        raise ValueError(f"{name} must be an int32 vector of {n}")
    return t if t.is_contiguous() else t.contiguous()


def _strides(t: torch.Tensor) -> Tuple[int, ...]:
    """Element strides; 64 where a dimension holds one element and any will do."""
    a, b, c, d = t.stride()
    n, h, rows, _ = t.shape
    return (a if n > 1 else HEAD_DIM, b if h > 1 else HEAD_DIM, c if rows > 1 else HEAD_DIM, d)


def _run_rows(run_rows: Optional[torch.Tensor], index: int) -> Optional[int]:
    if run_rows is None:
        return None
    _on("run_rows", run_rows, index)
    if run_rows.dtype not in (torch.int32, torch.uint32) or run_rows.numel() != 1:
        raise ValueError("run_rows must be one int32 word")
    return run_rows.data_ptr()


def _call_on(name: str, index: int, *args: Any) -> None:
    """An entry point on the current stream of GPU `index`, its last argument."""
    if _current_device() == index:
        status = getattr(_lib.lib(), name)(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = getattr(_lib.lib(), name)(*args, _raw_stream(index))
    if status:
        raise _lib.DHStatusError(name, int(status))


def write_kv(cache: KVCacheI8, k: torch.Tensor, v: torch.Tensor, start: Union[int, torch.Tensor] = 0,
             counts: Optional[torch.Tensor] = None, *, run_rows: Optional[torch.Tensor] = None) -> None:
    """Quantise rows ``k`` and ``v`` [entries, heads, n, 64] (fp32, bf16 or f16,
    each its own, any strides: a transposed V as the QKV product leaves it is
    ``vt.transpose(2, 3)``) into positions ``start``, ``start`` + 1, ... of
    `cache` (dh_kv_write_i8).

    ``start``: an int, or int32 [entries] on the device; ``counts``: int32
    [entries] on the device, the rows of each sequence to write (default: all,
    which must fit behind an int ``start``).  Positions that lie outside the
    cache by a device ``start`` are not written, and all others stay as they
    were.  The scale of a row is its largest magnitude / 127; a row below 2^-100
    counts as zero, one with an infinity or NaN gets the scale NaN.
    ``run_rows``: one device word, only the sequences within its first rows of
    [entries * n] are written."""
    index = cache.k.get_device()
    shape = _check_cache("cache", cache, index)
    entries, heads, capacity, _ = shape
    rows = k.shape[2] if k.dim() == 4 else -1
    if k.shape != (entries, heads, rows, HEAD_DIM) or v.shape != k.shape:
        raise ValueError(f"k and v must be [{entries}, {heads}, n, {HEAD_DIM}]")
    k_type, v_type = _TYPES.get(k.dtype), _TYPES.get(v.dtype)
    if k_type is None or v_type is None:
        raise ValueError("k and v must be float32, bfloat16 or float16")
    if not k.get_device() == v.get_device() == index:
        raise ValueError("k and v must be CUDA tensors on the device of the cache")
    starts = None
    if isinstance(start, torch.Tensor):
        starts, start = _ints("start", start, entries, index), 0
    elif start < 0 or start > capacity or (counts is None and start + rows > capacity):
        raise ValueError(f"{rows} rows from {start} on do not fit the capacity of {capacity}")
    if counts is not None:
        counts = _ints("counts", counts, entries, index)
    run = _run_rows(run_rows, index)
    if rows == 0 or entries == 0 or heads == 0:
        return
    _call_on("dh_kv_write_i8", index, k.data_ptr(), k_type, _pack4(*k.stride()), v.data_ptr(), v_type,
             _pack4(*v.stride()), entries, heads, rows, _ptr(starts), start, _ptr(counts), cache.k.data_ptr(),
             cache.k_scale.data_ptr(), cache.v.data_ptr(), cache.v_scale.data_ptr(), capacity, run)


def read_kv(cache: KVCacheI8, start: int = 0, rows: Optional[int] = None, *,
            dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
    """K and V [entries, heads, rows, 64] of positions [start, start + rows)
    (default: to the end of the capacity) of every entry: codes * scales, rounded
    to `dtype` (fp32, bf16 or f16; dh_kv_read_i8)."""
    index = cache.k.get_device()
    entries, heads, capacity, _ = _check_cache("cache", cache, index)
    rows = capacity - start if rows is None else rows
    if start < 0 or rows < 0 or start + rows > capacity:
        raise ValueError(f"positions [{start}, {start + rows}) lie outside the capacity of {capacity}")
    out_type = _TYPES.get(dtype)
    if out_type is None:
        raise ValueError("dtype must be float32, bfloat16 or float16")
    k = cache.k.new_empty((entries, heads, rows, HEAD_DIM), dtype=dtype)
    v = torch.empty_like(k)
    if rows and entries and heads:
        _call_on("dh_kv_read_i8", index, cache.k.data_ptr(), cache.k_scale.data_ptr(), cache.v.data_ptr(),
                 cache.v_scale.data_ptr(), entries, heads, capacity, start, rows, k.data_ptr(), v.data_ptr(), out_type)
    return k, v


class _Keys(NamedTuple):
    view: bytes          # dh_kv_view
    entries: int
    heads: int
    capacity: int        # as in the view
    v_type: int          # with `turned`: what a prefix must have alike
    turned: bool         # V's columns are contiguous
    held: Any            # a tensor the view points into


def _shown(capacity: int, length: int, int8: bool) -> int:
    """The capacity that a call shows of a cache with `length` keys."""
    if capacity <= _WHOLE_KEYS:
        return capacity
    step = CAPACITY_STEP if int8 else 1
    return max(-(-length // step), 1) * step


def _view(name: str, kv: Any, lengths: Lengths, q: torch.Tensor, index: int) -> _Keys:
    turned = False
    if isinstance(kv, KVCacheI8):
        k, k_scale, v, v_scale = kv
        entries, heads, capacity, _ = _check_cache(name, kv, index)
        kt = vt = _TYPE_I8
        ks = vs = (0, capacity * HEAD_DIM, 0, 0)
        pointers = (k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr())
    else:
        k, v = kv
        if not k.get_device() == v.get_device() == index:
            raise ValueError(f"{name} must be CUDA tensors on the device of the others")
        if k.dim() != 4 or k.shape[3] != HEAD_DIM or v.shape != k.shape or k.shape[2] == 0:
            raise ValueError(f"k and v of {name} must be [entries, heads, n, {HEAD_DIM}] with n > 0")
        if k.dtype is not q.dtype or (v.dtype is not torch.bfloat16 and v.dtype is not torch.float16):
            raise ValueError(f"k of {name} must be of q's type, v bfloat16 or float16")
        entries, heads, capacity, _ = k.shape
        kt, vt = _TYPES[k.dtype], _TYPES[v.dtype]
        ks, vs = _strides(k), _strides(v)
        if vs[3] == 1:
            aligned = vs[0] | vs[1] | vs[2]
        elif capacity == 1 or vs[2] == 1:  # its columns are contiguous
            turned = True
            vs = (vs[0], vs[1], 1, vs[3])
            aligned = vs[0] | vs[1] | vs[3]
        else:
            raise ValueError(f"v of {name} must have contiguous rows or contiguous columns")
        if ks[3] != 1:
            raise ValueError(f"k of {name} must have contiguous rows")
        pointers = (k.data_ptr(), v.data_ptr(), 0, 0)
        if (aligned | ks[0] | ks[1] | ks[2]) % 8 or (pointers[0] | pointers[1]) & 15:
            raise ValueError(f"k and v of {name} must start at 16-byte boundaries, as must their rows and heads")
    held = None
    length = capacity
    if lengths is None:
        pass
    elif isinstance(lengths, torch.Tensor):
        held = _ints(f"lengths of {name}", lengths, entries, index)
    else:
        length = operator.index(lengths)
        if not 0 <= length <= capacity:
            raise ValueError(f"{length} keys of {name} do not lie within its capacity of {capacity}")
        capacity = _shown(capacity, length, kt == _TYPE_I8)
    view = _pack_view(*pointers, 0 if held is None else held.data_ptr(), *ks, *vs, kt, vt, capacity, length)
    return _Keys(view, entries, heads, capacity, vt, turned, held)


def attend(q: torch.Tensor, kv: Any, lengths: Lengths = None, *, prefix: Any = None, prefix_lengths: Lengths = None,
           scale: Optional[float] = None, return_lse: bool = False, out: Optional[torch.Tensor] = None,
           run_rows: Optional[torch.Tensor] = None) -> Any:
    """``softmax(scale q k^T) v`` of queries ``q`` [batch, heads, n, 64] (bf16 or
    f16) over cached keys (dh_kv_attention).  Returns [batch, n, heads, 64] of
    q's type: rows of a token together, as the attention-out product reads them.

    ``kv``: a :class:`KVCacheI8` with an entry for each sequence, or a pair of
    16-bit tensors k, v [batch, kv_heads, capacity, 64]: k of q's type, v bf16 or
    f16, its rows or its columns contiguous (``vt.transpose(2, 3)``), rows and
    heads at 16-byte boundaries.  ``heads`` is a multiple of ``kv_heads``; query
    head h reads K/V head ``h * kv_heads // heads``.
    ``lengths``: how many of the keys each sequence has, an int or int32 [batch]
    on the device (default: all); what lies behind them is not used, whatever it
    holds.

    ``prefix``: keys before those, of the same kind and layout as `kv`, with an
    entry for each group of consecutive sequences (their number divides the
    batch: 1 for a prefix of the whole batch), ``prefix_lengths`` as `lengths`
    for them.

    ``scale`` (2^-126 to 2^127) defaults to 1/8.  A query without keys gives 0.  With
    ``return_lse`` also the log of the sum of exponentials, fp32 [batch, n, heads]
    (-inf without keys), to join results over disjoint keys.  ``run_rows``: one
    device word, only the sequences within its first rows of [batch * n] are computed.

    Scores and sums are fp32; the weights enter the product with V rounded to 16
    bits (f16; bf16 for V in bf16).  Scores beyond 1.8e8 (2^28 log 2) count to 2^-21
    of their size.  V, and K in 8 bits, may be up to 2^90 in magnitude.
    Over int8 keys, where a K/V head has at most 16 query rows, a query is held in 15
    bits: an element is off by up to 1/32512 of its row's largest (all of a row
    below 2^-100 counts as zero).  With more rows a query is f16 relative to its
    row's largest value, and K and V are rounded to f16, factor and product, 2^-11 of
    themselves each (f16 queries: two f16, 2^-15), but not below 2^-19 of the largest
    value that the keys of the sequence and its prefix hold at this head.

    Calls that split the keys take 264 bytes of workspace for each query, head and
    part (at most 64 of the prefix and 64 of the rest); calls whose queries visit
    int8 keys many times hold those as f16, 256 bytes (f16 queries: 512) for each
    position and K/V head.  Parts and positions are those of the capacity or, for
    caches of more than 512 positions, of `lengths` as an int."""
    index = q.get_device()
    q_type = _TYPES.get(q.dtype)
    if index < 0:
        raise ValueError("q must be a CUDA tensor")
    if q.dim() != 4 or q.shape[3] != HEAD_DIM or not q_type:
        raise ValueError(f"q must be [batch, heads, n, {HEAD_DIM}] of bfloat16 or float16")
    batch, heads, n, _ = q.shape
    qs = _strides(q)
    if qs[3] != 1 or (qs[0] | qs[1] | qs[2]) % 8 or q.data_ptr() & 15:
        q = q.clone(memory_format=torch.contiguous_format)
        qs = _strides(q)
    keys = _view("kv", kv, lengths, q, index)
    kv_heads = keys.heads
    if keys.entries != batch:
        raise ValueError(f"kv has {keys.entries} entries for {batch} sequences")
    if kv_heads == 0 or heads % kv_heads:
        raise ValueError(f"{heads} query heads are no multiple of {kv_heads} K/V heads")
    prefixes, prefix_capacity, prefix_view = 0, 0, None
    if prefix is not None:
        if isinstance(prefix, KVCacheI8) != isinstance(kv, KVCacheI8):
            raise ValueError("prefix must be of the same kind as kv")
        before = _view("prefix", prefix, prefix_lengths, q, index)
        prefixes = before.entries
        if before.heads != kv_heads:
            raise ValueError(f"prefix has {before.heads} heads and kv {kv_heads}")
        if prefixes == 0 or batch % prefixes:
            raise ValueError(f"{prefixes} prefixes do not divide {batch} sequences")
        if before.v_type != keys.v_type or before.turned != keys.turned:
            raise ValueError("v of prefix must have the type and layout of v of kv")
        prefix_capacity, prefix_view = before.capacity, before.view
    elif prefix_lengths is not None:
        raise ValueError("prefix_lengths without a prefix")
    if scale is None:
        scale = 0.125
    elif not 2.0 ** -126 <= scale <= 2.0 ** 127:
        raise ValueError("scale must be positive and finite (2^-126 to 2^127)")
    if out is None:
        out = q.new_empty((batch, n, heads, HEAD_DIM))
    elif _on("out", out, index).numel() != batch * n * heads * HEAD_DIM or out.dtype is not q.dtype \
            or not out.is_contiguous() or out.data_ptr() & 15:
        raise ValueError(f"out must hold [{batch}, {n}, {heads}, {HEAD_DIM}] of q's type, contiguous and 16-byte aligned")
    lse = q.new_empty((batch, n, heads), dtype=torch.float32) if return_lse else None
    run = _run_rows(run_rows, index)
    if batch and n and heads:
        size = _workspace_bytes(batch, n, heads, kv_heads, prefixes, -(-prefix_capacity // CAPACITY_STEP),
                                -(-keys.capacity // CAPACITY_STEP), keys.v_type == _TYPE_I8, q_type, index)
        # (goes back to the allocator's pool of the current stream, which the
        # kernels that use it are on)
        ws = q.new_empty((size,), dtype=torch.uint8) if size else None
        _call_on("dh_kv_attention", index, q.data_ptr(), q_type, _pack4(*qs), batch, n, heads, kv_heads, keys.view,
                 prefix_view, prefixes, scale, out.data_ptr(), _ptr(lse), run, _ptr(ws), size)
    return (out, lse) if return_lse else out


def attend_launches(batch: int, n: int, heads: int, kv_heads: int, capacity: int, length: int, *, int8: bool,
                    prefixes: int = 0, prefix_capacity: int = 0, prefix_length: int = 0, device: Any = "cuda") -> int:
    """Kernels that :func:`attend` launches for queries [batch, heads, n, 64] over
    `length` keys (an int) of a cache, behind `prefix_length` keys of `prefixes` others."""
    with torch.cuda.device(device):
        return int(_lib.lib().dh_kv_attention_launches(
            batch, n, heads, kv_heads, prefixes, _shown(prefix_capacity, prefix_length, int8) if prefixes else 0,
            _shown(capacity, length, int8), _TYPE_I8 if int8 else _TYPES[torch.bfloat16]))


@functools.lru_cache(maxsize=256)
def _workspace_bytes(batch: int, n: int, heads: int, kv_heads: int, prefixes: int, prefix_tiles: int,
                     tiles: int, int8: bool, q_type: int, index: int) -> int:
    # (the same for all capacities of a number of tiles)
    with torch.cuda.device(index):
        return int(_lib.lib().dh_kv_attention_workspace_size(
            batch, n, heads, kv_heads, prefixes, prefix_tiles * CAPACITY_STEP, tiles * CAPACITY_STEP,
            _TYPE_I8 if int8 else q_type, q_type))
