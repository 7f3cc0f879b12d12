"""Argument checks of the scoring entry points and functions (no device work)."""

import types

import pytest
import torch

from diffusionhard_b200 import _lib, api, scoring

P = 4096  # a non-null, 256-byte aligned address that no refused call touches
NULL, ALIGN, WORKSPACE, SHAPE, ARG = 100, 101, 102, 103, 105


def _gemm(**kw):
    a = dict(a=P, lda=64, a_scale=P, w=P, ldw=64, w_scale=P, bias=None, out=P, ldo=8, out_type=0, m=4, n=8, k=64)
    a.update(kw)
    return _lib.raw("dh_gemm_i8_scaled", *a.values(), None)


@pytest.mark.parametrize("change, status", [
    (dict(a=None), NULL), (dict(w=None), NULL), (dict(a_scale=None), NULL), (dict(w_scale=None), NULL),
    (dict(out=None), NULL), (dict(out_type=3), ARG), (dict(m=0), ARG), (dict(n=0), ARG), (dict(k=0), ARG),
    (dict(ldo=7), ARG), (dict(lda=48), ARG), (dict(ldw=48), ARG), (dict(a=P + 8), ALIGN), (dict(lda=72), ALIGN),
    (dict(w=P + 1), ALIGN), (dict(ldw=68), ALIGN), (dict(out=P + 2), ALIGN), (dict(out=P + 1, out_type=1), ALIGN),
    (dict(a_scale=P + 2), ALIGN), (dict(bias=P + 1), ALIGN), (dict(k=131072, lda=131072, ldw=131072), SHAPE),
    (dict(m=1 << 31), SHAPE), (dict(n=(1 << 32) - 1, ldo=1 << 33), SHAPE),
])
def test_gemm_scaled_refuses(change, status):
    assert _gemm(**change) == status


def _logits(**kw):
    a = dict(logits=P, type=0, stride=100, rows=2, vocab=100, mask=0, targets=P, target_bytes=8, per_row=1, top_k=4,
             logprobs=P, entropy=P, logsumexp=P, top_ids=P, top_logprobs=P)
    a.update(kw)
    return _lib.raw("dh_token_logprobs", *a.values(), None)


OUTPUT_CHANGES = [
    (dict(targets=None), NULL), (dict(logprobs=None), NULL), (dict(top_ids=None), NULL),
    (dict(top_logprobs=None), NULL), (dict(per_row=0, top_k=0, entropy=None, logsumexp=None), NULL),
    (dict(target_bytes=2), ARG), (dict(top_k=33), SHAPE), (dict(targets=P + 4), ALIGN), (dict(entropy=P + 2), ALIGN),
    (dict(top_ids=P + 1), ALIGN),
]


@pytest.mark.parametrize("change, status", OUTPUT_CHANGES + [
    (dict(logits=None), NULL), (dict(type=3), ARG), (dict(rows=0), ARG), (dict(vocab=0), ARG), (dict(mask=100), ARG),
    (dict(rows=(1 << 27) + 1), SHAPE), (dict(vocab=(1 << 30) + 1), SHAPE), (dict(logits=P + 2), ALIGN),
    (dict(logits=P + 1, type=2), ALIGN),
])
def test_token_logprobs_refuses(change, status):
    assert _logits(**change) == status


def _head(**kw):
    a = dict(hidden=P, ldh=64, a_scale=P, w=P, ldw=64, w_scale=P, bias=P, rows=2, size=64, vocab=100, mask=0,
             targets=P, target_bytes=8, per_row=1, top_k=4, logprobs=P, entropy=P, logsumexp=P, top_ids=P,
             top_logprobs=P, ws=P, ws_bytes=1 << 40)
    a.update(kw)
    return _lib.raw("dh_head_logprobs_i8", *a.values(), None)


@pytest.mark.parametrize("change, status", OUTPUT_CHANGES + [
    (dict(rows=0), 1), (dict(size=0), 2), (dict(vocab=0), 3), (dict(mask=100), 4), (dict(hidden=None), NULL),
    (dict(a_scale=None), NULL), (dict(w=None), NULL), (dict(w_scale=None), NULL), (dict(ws=None), NULL),
    (dict(ws=P + 128), ALIGN), (dict(w_scale=P + 2), ALIGN), (dict(hidden=P + 4), ALIGN), (dict(ldw=72), ALIGN),
    (dict(ldh=48), ARG), (dict(ws_bytes=64), WORKSPACE), (dict(size=131072, ldh=131072, ldw=131072), SHAPE),
    (dict(rows=(1 << 24) + 1), SHAPE), (dict(vocab=(1 << 24) + 1), SHAPE),
])
def test_head_logprobs_refuses(change, status):
    assert _head(**change) == status


def test_head_workspace_query():
    f = _lib.lib().dh_head_logprobs_workspace_size
    assert f(0, 100, 1) == 0 and f(1, 0, 1) == 0
    assert 0 < f(1, 100, 0) < f(1, 100, 1) <= f(300, 100, 1)
    assert f(32, 50258, 8) == f(32, 50258, 1)


def test_functions_refuse_host_tensors():
    i8, f = torch.zeros((2, 16), dtype=torch.int8), torch.zeros(2)
    with pytest.raises(ValueError, match="CUDA"):
        scoring.linear_i8(i8, f, i8, f)
    with pytest.raises(ValueError, match="CUDA"):
        scoring.token_logprobs(torch.zeros(2, 10))
    with pytest.raises(ValueError, match="CUDA"):
        scoring.head_logprobs(i8, f, i8, f)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bool, torch.complex64])
def test_score_tokens_wants_integers(dtype):
    model = types.SimpleNamespace(cfg=types.SimpleNamespace(mask_token_id=9, vocab_size=10), B=1, L=4, device="cuda:0")
    ids, other = torch.zeros((1, 4), dtype=torch.int64), torch.zeros((1, 4), dtype=dtype)
    with pytest.raises(ValueError, match="input_ids must be integers"):
        api.score_tokens(model, other, ids, mask_token_id=9)
    with pytest.raises(ValueError, match="target_ids must be integers"):
        api.score_tokens(model, ids, other, mask_token_id=9)


def test_head_shapes_without_a_workspace():
    """Where the query has no size, the call says that it is for the shape."""
    f = _lib.lib().dh_head_logprobs_workspace_size
    assert f(1 << 24, 1 << 24, 1) == 0
    assert _head(rows=1 << 24, vocab=1 << 24, ws=None, ws_bytes=0) == SHAPE
    assert _head(rows=(1 << 24) + 1, ws=None, ws_bytes=0) == SHAPE
