"""Scores of tokens: how probable they are, and what else was likely.

Three operators over the C ABI (include/dh_b200.h):

* :func:`linear_i8` -- the W8A8 linear of any width, the reference's
  ``fixed_mlp.quantized_linear`` (fixed_mlp.py:65-136): an int8 matrix product
  with a scale for each token and each channel.
* :func:`token_logprobs` -- log probabilities of given tokens, entropy,
  logsumexp and the best alternatives of rows of logits
  (``mdlm._mdlm_log_probabilities``, mdlm.py:851-858, which excludes the mask
  token).
* :func:`head_logprobs` -- the same scores straight from the int8 output head;
  its logits never reach memory.

Every call runs on the current stream of its tensors' device, returns without
waiting for it, and can be captured in a CUDA graph.  Arguments are checked
before anything is launched; token ids are not (see each function for ids
outside the vocabulary).  Results carry no gradients, and an `out` tensor must
not overlap the inputs.
"""

from __future__ import annotations

import functools
from typing import Any, NamedTuple, Optional

import torch

from . import _lib

MAX_TOP_K = 32
NO_TOKEN = 0xFFFFFFFF
_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


class TokenScores(NamedTuple):
    """Scores of rows; ``logprobs`` has the shape of the given tokens and is
    None without them, the alternatives are None for ``top_k=0``."""

    logprobs: Optional[torch.Tensor]      # fp32
    entropy: torch.Tensor                 # fp32 [rows], nats
    logsumexp: torch.Tensor               # fp32 [rows]
    top_ids: Optional[torch.Tensor]       # int32 [rows, top_k], -1: none left
    top_logprobs: Optional[torch.Tensor]  # fp32 [rows, top_k]


# A call of these functions takes a few microseconds of the host, and the smallest
# of them as little of the GPU: the checks below are ordered so that a call that
# is as it should be passes few of them.
_current_device = torch.cuda.current_device
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(name: str, device: torch.device, *args: Any) -> None:
    """An entry point on the current stream of `device`, its last argument."""
    index = device.index
    if _current_device() == index:
        status = getattr(_lib.lib(), name)(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = getattr(_lib.lib(), name)(*args, _raw_stream(index))
    if status:
        raise _lib.DHStatusError(name, int(status))


def _cuda(name: str, t: torch.Tensor, device: Optional[torch.device] = None) -> torch.Tensor:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if device is not None and t.device != device:
        raise ValueError(f"{name} must be on {device}")
    return t


def _vector(name: str, t: torch.Tensor, n: int, device: torch.device) -> torch.Tensor:
    if t.dtype is torch.float32 and t.device == device and t.shape == (n,):
        return t if t.is_contiguous() else t.contiguous()
    _cuda(name, t, device)
    raise ValueError(f"{name} must be a float32 vector of {n}")


def _rows_i8(name: str, t: torch.Tensor, device: Optional[torch.device] = None) -> torch.Tensor:
    """int8 rows that start at 16-byte boundaries: `t`, or a copy with padded
    rows (store weights that way once: torch.nn.functional.pad)."""
    _cuda(name, t, device)
    if t.dtype is not torch.int8 or t.dim() != 2 or t.shape[1] == 0:
        raise ValueError(f"{name} must be a two-dimensional int8 tensor with columns")
    pitch, inner = t.stride()
    if inner == 1 and pitch >= t.shape[1] and not (pitch | t.data_ptr()) & 15:
        return t
    rows, cols = t.shape
    padded = torch.empty((rows, (cols + 15) // 16 * 16), dtype=torch.int8, device=t.device)
    padded[:, :cols].copy_(t)
    return padded[:, :cols]


def _empty(shape: tuple, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    # (empty_strided parses its arguments in half the time of empty)
    return torch.empty_strided(shape, (shape[1], 1) if len(shape) == 2 else (1,), dtype=dtype, device=device)


def linear_i8(a: torch.Tensor, a_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
              bias: Optional[torch.Tensor] = None, *, out_dtype: Optional[torch.dtype] = None,
              out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``(a @ w.T) * (a_scale[:, None] * w_scale) + bias`` of int8 ``a`` [m, k]
    and ``w`` [n, k] (dh_gemm_i8_scaled); ``a_scale`` [m], ``w_scale`` [n] and
    ``bias`` [n] fp32.  Returns [m, n] of ``out_dtype``: fp32 (default), bf16
    or f16; ``out`` of that shape and type, its rows contiguous, receives the
    result instead.  fp32 results equal the reference's float64 evaluation bit
    for bit.  Rows of ``a`` and ``w`` that do not start at 16-byte boundaries
    are copied first."""
    a = _rows_i8("a", a)
    dev = a.device
    w = _rows_i8("w", w, dev)
    m, k = a.shape
    n = w.shape[0]
    if w.shape[1] != k:
        raise ValueError(f"a has {k} columns and w {w.shape[1]}")
    a_scale, w_scale = _vector("a_scale", a_scale, m, dev), _vector("w_scale", w_scale, n, dev)
    if bias is not None:
        bias = _vector("bias", bias, n, dev)
    if out is None:
        if out_dtype is None:
            out_dtype = torch.float32
        elif out_dtype not in _TYPES:
            raise ValueError("out_dtype must be float32, bfloat16 or float16")
        out = _empty((m, n), out_dtype, dev)
        pitch = n
    else:
        _cuda("out", out, dev)
        if out.shape != (m, n) or out.dtype not in _TYPES or (out_dtype or out.dtype) != out.dtype:
            raise ValueError(f"out must be [{m}, {n}] of float32, bfloat16 or float16 and of out_dtype")
        if (n > 1 and out.stride(1) != 1) or (m > 1 and out.stride(0) < n):
            raise ValueError("out must have contiguous rows that do not overlap")
        pitch = out.stride(0) if m > 1 else n
    if m == 0 or n == 0:
        return out
    _call("dh_gemm_i8_scaled", dev, a.data_ptr(), a.stride(0), a_scale.data_ptr(), w.data_ptr(), w.stride(0),
          w_scale.data_ptr(), None if bias is None else bias.data_ptr(), out.data_ptr(), pitch, _TYPES[out.dtype],
          m, n, k)
    return out


def _targets(targets: Optional[torch.Tensor], rows: int, device: torch.device) -> tuple:
    """(contiguous tensor or None, tokens per row, bytes of an id)."""
    if targets is None:
        return None, 0, 0
    _cuda("targets", targets, device)
    if targets.dtype is torch.int64:
        size = 8
    elif targets.dtype is torch.int32:
        size = 4
    else:
        raise ValueError("targets must be int32 or int64")
    shape = targets.shape
    if len(shape) not in (1, 2) or shape[0] != rows:
        raise ValueError(f"targets must be [{rows}] or [{rows}, tokens]")
    return (targets if targets.is_contiguous() else targets.contiguous()), 1 if len(shape) == 1 else shape[1], size


def _excluded(mask_token_id: Optional[int], vocab: int) -> int:
    if mask_token_id is None:
        return NO_TOKEN
    if not 0 <= mask_token_id < vocab:
        raise ValueError("mask_token_id lies outside the vocabulary")
    return int(mask_token_id)


def _outputs(targets: Optional[torch.Tensor], rows: int, top_k: int, device: torch.device) -> TokenScores:
    if not 0 <= top_k <= MAX_TOP_K:
        raise ValueError(f"top_k must be in [0, {MAX_TOP_K}]")
    f32 = torch.float32
    entropy = _empty((rows,), f32, device)
    return TokenScores(
        None if targets is None else torch.empty_like(targets, dtype=f32), entropy, torch.empty_like(entropy),
        _empty((rows, top_k), torch.int32, device) if top_k else None,
        _empty((rows, top_k), f32, device) if top_k else None)


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def token_logprobs(logits: torch.Tensor, targets: Optional[torch.Tensor] = None, *, top_k: int = 0,
                   mask_token_id: Optional[int] = None) -> TokenScores:
    """Scores of logits [rows, vocab] (fp32, bf16 or f16; the vocabulary
    contiguous, any row stride) in one pass (dh_token_logprobs).

    ``targets``: int32 or int64 ids [rows] or [rows, tokens]; a negative id
    stands for "no token" and scores 0, one past the vocabulary scores NaN.
    ``mask_token_id``: this token's logit counts as -inf.  ``top_k`` (at most
    32): the tokens of largest logit, the lower id first among equals.  A row
    with nothing left has log probabilities -inf and entropy 0; one with a NaN
    or +inf scores NaN."""
    _cuda("logits", logits)
    if logits.dim() != 2 or logits.dtype not in _TYPES or logits.shape[1] == 0:
        raise ValueError("logits must be [rows, vocab] of float32, bfloat16 or float16")
    rows, vocab = logits.shape
    if vocab > 1 and logits.stride(1) != 1:
        raise ValueError("the logits of a row must be contiguous")
    dev = logits.device
    mask = _excluded(mask_token_id, vocab)
    targets, per_row, id_bytes = _targets(targets, rows, dev)
    out = _outputs(targets, rows, top_k, dev)
    if rows == 0:
        return out
    _call("dh_token_logprobs", dev, logits.data_ptr(), _TYPES[logits.dtype], logits.stride(0), rows, vocab, mask,
          _ptr(targets) if per_row else None, id_bytes, per_row, top_k, _ptr(out.logprobs) if per_row else None,
          out.entropy.data_ptr(), out.logsumexp.data_ptr(), _ptr(out.top_ids), _ptr(out.top_logprobs))
    return out


def head_logprobs(hidden: torch.Tensor, hidden_scale: torch.Tensor, weight: torch.Tensor, w_scale: torch.Tensor,
                  bias: Optional[torch.Tensor] = None, targets: Optional[torch.Tensor] = None, *, top_k: int = 0,
                  mask_token_id: Optional[int] = None) -> TokenScores:
    """:func:`token_logprobs` of ``linear_i8(hidden, hidden_scale, weight,
    w_scale, bias)`` without its logits ever reaching memory
    (dh_head_logprobs_i8): int8 ``hidden`` [rows, hidden_size] with a scale per
    row, int8 ``weight`` [vocab, hidden_size] with a scale per token.  The logits
    are those of ``linear_i8`` up to the rounding of a last bit.

    With ``top_k`` a call takes 10 bytes of workspace for each row and 64 tokens
    of the vocabulary (257 MB for 32768 x 50258).  Alternatives cost more time
    where many parts of 64 logits come close to a row's k-th best: within 2^-10 of
    its size where that lies between 6e-5 and 65504, within 6e-8 below, and at any
    distance above."""
    hidden = _rows_i8("hidden", hidden)
    dev = hidden.device
    weight = _rows_i8("weight", weight, dev)
    rows, size = hidden.shape
    vocab = weight.shape[0]
    if weight.shape[1] != size:
        raise ValueError(f"hidden has {size} columns and weight {weight.shape[1]}")
    if vocab == 0:
        raise ValueError("weight must have rows")
    hidden_scale = _vector("hidden_scale", hidden_scale, rows, dev)
    w_scale = _vector("w_scale", w_scale, vocab, dev)
    if bias is not None:
        bias = _vector("bias", bias, vocab, dev)
    mask = _excluded(mask_token_id, vocab)
    targets, per_row, id_bytes = _targets(targets, rows, dev)
    out = _outputs(targets, rows, top_k, dev)
    if rows == 0:
        return out
    # (the workspace goes back to the allocator's pool of the current stream,
    # which the kernels that use it are on)
    size_bytes = _workspace_bytes(rows, vocab, top_k > 0, dev.index)
    ws = _empty((size_bytes,), torch.uint8, dev)
    _call("dh_head_logprobs_i8", dev, hidden.data_ptr(), hidden.stride(0), hidden_scale.data_ptr(), weight.data_ptr(),
          weight.stride(0), w_scale.data_ptr(), _ptr(bias), rows, size, vocab, mask,
          _ptr(targets) if per_row else None, id_bytes, per_row, top_k, _ptr(out.logprobs) if per_row else None,
          out.entropy.data_ptr(), out.logsumexp.data_ptr(), _ptr(out.top_ids), _ptr(out.top_logprobs), ws.data_ptr(),
          size_bytes)
    return out


@functools.lru_cache(maxsize=256)
def _workspace_bytes(rows: int, vocab: int, top: bool, index: int) -> int:
    with torch.cuda.device(index):
        return int(_lib.lib().dh_head_logprobs_workspace_size(rows, vocab, 1 if top else 0))
