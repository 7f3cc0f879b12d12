"""Argument checks of the K/V cache entry points and functions (no device work)."""

import ctypes

import pytest
import torch

from diffusionhard_b200 import _lib, kvcache

P = 4096  # a non-null, 256-byte aligned address that no refused call touches
NULL, ALIGN, WORKSPACE, SHAPE, ARG = 100, 101, 102, 103, 105
U64x4 = ctypes.c_uint64 * 4
BIG = 1 << 31


def _write(**kw):
    a = dict(k=P, kt=1, ks=U64x4(4096, 1024, 64, 1), v=P, vt=2, vs=U64x4(4096, 1024, 1, 16), n=2, heads=4, rows=16,
             starts=None, start=0, counts=None, kc=P, ksc=P, vc=P, vsc=P, capacity=64, run=None)
    a.update(kw)
    return _lib.raw("dh_kv_write_i8", *a.values(), None)


@pytest.mark.parametrize("change, status", [
    (dict(k=None), NULL), (dict(v=None), NULL), (dict(ks=None), NULL), (dict(vs=None), NULL), (dict(kc=None), NULL),
    (dict(ksc=None), NULL), (dict(vc=None), NULL), (dict(vsc=None), NULL), (dict(kt=3), ARG), (dict(vt=4), ARG),
    (dict(n=0), ARG), (dict(heads=0), ARG), (dict(rows=0), ARG), (dict(capacity=0), ARG), (dict(start=65), ARG),
    (dict(start=49), ARG), (dict(rows=65), ARG), (dict(start=65, counts=P), ARG), (dict(k=P + 1), ALIGN),
    (dict(kt=0, k=P + 2), ALIGN), (dict(v=P + 1), ALIGN), (dict(kc=P + 4), ALIGN), (dict(vc=P + 1), ALIGN),
    (dict(ksc=P + 2), ALIGN), (dict(vsc=P + 1), ALIGN), (dict(starts=P + 2), ALIGN), (dict(counts=P + 2), ALIGN),
    (dict(run=P + 2), ALIGN), (dict(rows=BIG, capacity=BIG), SHAPE), (dict(n=1 << 30, heads=4), SHAPE),
    (dict(n=(1 << 32) - 1, heads=(1 << 32) - 1), SHAPE),
])
def test_write_refuses(change, status):
    assert _write(**change) == status


def _read(**kw):
    a = dict(kc=P, ksc=P, vc=P, vsc=P, n=2, heads=4, capacity=64, start=0, rows=64, k=P, v=P, t=1)
    a.update(kw)
    return _lib.raw("dh_kv_read_i8", *a.values(), None)


@pytest.mark.parametrize("change, status", [
    (dict(kc=None), NULL), (dict(ksc=None), NULL), (dict(vc=None), NULL), (dict(vsc=None), NULL), (dict(k=None), NULL),
    (dict(v=None), NULL), (dict(t=3), ARG), (dict(n=0), ARG), (dict(heads=0), ARG), (dict(rows=0), ARG),
    (dict(start=1), ARG), (dict(start=65, rows=1), ARG), (dict(rows=(1 << 32) - 1, start=2), ARG),
    (dict(kc=P + 4), ALIGN), (dict(vsc=P + 2), ALIGN), (dict(k=P + 8), ALIGN), (dict(v=P + 2), ALIGN),
    (dict(n=1 << 30, heads=4), SHAPE), (dict(n=(1 << 32) - 1, heads=(1 << 32) - 1), SHAPE),
])
def test_read_refuses(change, status):
    assert _read(**change) == status


def _view(**kw):
    a = dict(k=P, v=P, k_scale=P, v_scale=P, lengths=None, k_strides=U64x4(65536, 4096, 64, 1),
             v_strides=U64x4(65536, 4096, 64, 1), k_type=1, v_type=1, capacity=64, length=64)
    a.update(kw)
    return kvcache._pack_view(*(a[n] or 0 for n in ("k", "v", "k_scale", "v_scale", "lengths")), *a["k_strides"],
                              *a["v_strides"], a["k_type"], a["v_type"], a["capacity"], a["length"])


def _attend(own=None, prefix=None, **kw):
    own = _view() if own is None else own
    a = dict(q=P, qt=1, qs=U64x4(4096, 1024, 64), n=2, queries=16, heads=4, kv_heads=4, own=own, prefix=prefix, prefixes=0 if prefix is None else 1,
             scale=0.125, out=P, lse=None, run=None, ws=P, size=1 << 30)
    a.update(kw)
    return _lib.raw("dh_kv_attention", *a.values(), None)


@pytest.mark.parametrize("change, status", [
    (dict(q=None), NULL), (dict(qs=None), NULL), (dict(out=None), NULL), (dict(prefixes=1), NULL),
    (dict(qt=0), ARG), (dict(qt=3), ARG), (dict(n=0), ARG), (dict(queries=0), ARG), (dict(heads=0), ARG),
    (dict(kv_heads=0), ARG), (dict(kv_heads=3), ARG), (dict(scale=0.0), ARG), (dict(scale=-1.0), ARG),
    (dict(scale=float("inf")), ARG), (dict(scale=float("nan")), ARG), (dict(qt=2), ARG), (dict(q=P + 8), ALIGN),
    (dict(qs=U64x4(4096, 1020, 64)), ALIGN), (dict(out=P + 2), ALIGN), (dict(lse=P + 2), ALIGN),
    (dict(run=P + 1), ALIGN), (dict(n=BIG), SHAPE), (dict(heads=1 << 27, kv_heads=1 << 27), SHAPE),
    (dict(queries=(1 << 32) - 1), SHAPE),
])
def test_attention_refuses(change, status):
    assert _attend(**change) == status


I8 = dict(k_type=3, v_type=3)
TURNED = U64x4(65536, 4096, 1, 64)


@pytest.mark.parametrize("change, status", [
    (dict(k=None), NULL), (dict(v=None), NULL), (dict(capacity=0), ARG), (dict(length=65), ARG),
    (dict(capacity=BIG), ARG), (dict(k_type=0), ARG), (dict(v_type=0), ARG), (dict(v_type=3), ARG),
    (dict(k_type=3), ARG), (dict(k=P + 8), ALIGN), (dict(v=P + 8), ALIGN),
    (dict(k_strides=U64x4(65536, 4096, 60, 1)), ALIGN), (dict(v_strides=U64x4(65536, 4100, 64, 1)), ALIGN),
    (dict(v_strides=U64x4(65536, 4096, 1, 60)), ALIGN), (dict(k_strides=U64x4(65536, 4096, 1, 64)), SHAPE),
    (dict(v_strides=U64x4(65536, 4096, 128, 2)), SHAPE), (dict(k_strides=U64x4(1 << 40, 4096, 64, 1)), SHAPE),
    (dict(lengths=P + 2), ALIGN), (dict(I8, k_scale=None), NULL), (dict(I8, v_scale=None), NULL),
    (dict(I8, capacity=65, length=1), SHAPE), (dict(I8, k_scale=P + 4), ALIGN), (dict(I8, v=P + 8), ALIGN),
])
def test_keys_refused(change, status):
    assert _attend(_view(**change)) == status
    if "k_type" not in change and "v_type" not in change:
        assert _attend(prefix=_view(**change)) == status


def test_prefixes_refused():
    assert _attend(_view(**I8), _view()) == ARG
    assert _attend(_view(), _view(v_type=2)) == ARG
    assert _attend(_view(), _view(v_strides=TURNED)) == ARG
    assert _attend(prefix=_view(), n=3, prefixes=2) == ARG
    assert _attend(prefix=_view(), n=2, prefixes=3) == ARG


def test_workspace():
    f = _lib.lib().dh_kv_attention_workspace_size
    assert f(0, 1, 4, 4, 0, 0, 64, 1, 1) == 0 and f(1, 1, 4, 3, 0, 0, 64, 1, 1) == 0 and f(3, 1, 4, 4, 2, 64, 64, 1, 1) == 0
    size = f(1, 1, 4, 4, 0, 0, 1 << 16, 1, 1)
    assert 0 < size <= 64 * 4 * 264 + 256
    long = _view(capacity=1 << 16, length=1)
    args = dict(n=1, queries=1)
    assert _attend(long, ws=None, size=0, **args) == NULL
    assert _attend(long, ws=P + 128, size=size, **args) == ALIGN
    assert _attend(long, size=size - 1, **args) == WORKSPACE


def test_functions_refuse_host_tensors():
    c = kvcache.KVCacheI8.empty(1, 2, 100, device="cpu")
    assert c.capacity == 128 and c.nbytes(1) == 2 * 136 and c.nbytes() == 128 * 2 * 136
    x = torch.zeros(1, 2, 4, 64, dtype=torch.bfloat16)
    for call in (lambda: kvcache.write_kv(c, x, x), lambda: kvcache.read_kv(c), lambda: kvcache.attend(x, c),
                 lambda: kvcache.attend(x, (x, x))):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    for bad in ((0, 1, 1), (1, 0, 1), (1, 1, 0), (1, 1, -64)):
        with pytest.raises(ValueError, match="positive"):
            kvcache.KVCacheI8.empty(*bad, device="cpu")


@pytest.mark.parametrize("strides", [(4096, 8192), (0, 4096), (4032, 4032), (2048, 2048), (1 << 37, 1 << 37),
                                     (4097, 4097)])
def test_int8_pitch_refused(strides):
    """Heads of int8 keys that lie closer than their capacity, not in whole tiles, or
    differently for K and V."""
    k, v = (U64x4(0, s, 0, 0) for s in strides)
    bad = dict(I8, k_strides=k, v_strides=v)
    assert _attend(_view(**bad)) == SHAPE
    good = dict(I8, k_strides=U64x4(0, 8192, 0, 0), v_strides=U64x4(0, 8192, 0, 0))
    assert _attend(_view(**good), prefix=_view(**bad)) == SHAPE


def test_launches():
    f = _lib.lib().dh_kv_attention_launches
    assert f(0, 1, 4, 4, 0, 0, 64, 1) == 0 and f(1, 1, 4, 3, 0, 0, 64, 1) == 0 and f(3, 1, 4, 4, 2, 64, 64, 1) == 0
    assert f(1, 1, 12, 12, 0, 0, 64, 3) == 1  # one kernel, no parts
    assert f(32, 1024, 12, 12, 0, 0, 1024, 3) == 2  # keys turned into f16 first
    assert 2 <= f(128, 1, 12, 12, 1, 8192, 320, 1) <= 3


@pytest.mark.parametrize("scale", [3e38, 2.0 ** 127.9, 1e-39, 1e-45, -0.0])
def test_scales_out_of_range(scale):
    """Whose factor of scores, scale * log2(e), overflows, or lies below the normal floats."""
    assert _attend(scale=scale) == ARG
