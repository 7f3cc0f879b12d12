"""The K/V cache operators against plain float64 implementations.

Codes and scales are compared bit for bit.  Attention: with weights w_j = p_j /
sum p, relative errors e_j of the p_j move a result by sum_j w_j e_j (v_j - out) in
first order, so by at most sum_j w_j |e_j| (|v_j| + |out|).  The e_j are counted
below in `attention_bound` from the roundings of each step.
"""

import math

import pytest
import torch

from diffusionhard_b200 import _lib, kvcache
from diffusionhard_b200.kvcache import KVCacheI8, attend, read_kv, write_kv

pytestmark = pytest.mark.gpu
DIM = 64
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


# ------------------------------------------------------------ references

def ref_codes(x):
    """Codes and scales of rows of x, quotients in float64 rounded to fp32."""
    x = x.double().cpu()
    peak = x.abs().amax(-1)
    live = (peak >= 2.0 ** -100) & torch.isfinite(peak)
    scale = torch.where(live, (peak / 127).float(), torch.zeros(()))
    scale = torch.where(torch.isfinite(peak), scale, torch.full_like(scale, math.nan))
    code = (x / torch.where(live, scale, torch.ones(()))[..., None].double()).float()
    code = torch.where(live[..., None], code.round().clamp(-127, 127), torch.zeros(()))
    return code.to(torch.int8), scale


def values(shape, seed, dtype=BF16, spread=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g)
    if spread:
        x = x * (torch.rand(shape[:3], generator=g) * 2 + 0.2)[..., None]
    return x.to(dtype).cuda()


def cache_of(k, v, capacity=None):
    """A cache that holds k and v from position 0 on, NaN scales behind them."""
    n, h, rows, _ = k.shape
    c = KVCacheI8.empty(n, h, max(capacity or rows, 1))
    c.k.fill_(-128), c.v.fill_(-128)
    c.k_scale.fill_(math.nan), c.v_scale.fill_(math.nan)
    if rows:
        write_kv(c, k, v)
    return c


def dense(kv, entry, count):
    """float64 k, v [heads, count, 64] of an entry."""
    if isinstance(kv, KVCacheI8):
        return [c[entry, :, :count].double().cpu() * s[entry, :, :count, None].double().cpu()
                for c, s in ((kv.k, kv.k_scale), (kv.v, kv.v_scale))]
    return [t[entry, :, :count].double().cpu() for t in kv]


def ref_attend(q, kv, lengths, prefix=None, prefix_lengths=None, scale=0.125):
    """(out, lse, bound) in float64: out [batch, n, heads, 64]."""
    batch, heads, n, _ = q.shape
    out = torch.zeros(batch, n, heads, DIM, dtype=torch.float64)
    lse = torch.full((batch, n, heads), -math.inf, dtype=torch.float64)
    bound = torch.zeros_like(out)
    lse_bound = torch.zeros_like(lse)
    int8 = isinstance(kv, KVCacheI8)
    fine = int8 and q.dtype is F16
    # (half a step of 16 bits, relative: eps / 2)
    p_round = 2.0 ** -8 if not int8 and kv[1].dtype is BF16 else 2.0 ** -11
    for b in range(batch):
        k, v = dense(kv, b, lengths[b])
        if prefix is not None:
            groups = prefix[0].shape[0]
            pk, pv = dense(prefix, b * groups // batch, prefix_lengths[b * groups // batch])
            k, v = torch.cat([pk, k], 1), torch.cat([pv, v], 1)
        if k.shape[1] == 0:
            continue
        for h in range(heads):
            kh, vh = k[h * k.shape[0] // heads], v[h * k.shape[0] // heads]
            x = q[b, h].double().cpu()
            s = scale * (x @ kh.T)
            m = s.amax(-1, keepdim=True)
            p = torch.exp(s - m)
            total = p.sum(-1, keepdim=True)
            w = p / total
            o = w @ vh
            # a score: fp32 sums of 64 products; int8 rows are rounded to f16 twice
            # (factor and product), for f16 queries as two f16 (2^-15 each time), with
            # a floor of 2^-19 of the largest row
            ks = (64 * 2.0 ** -24 + (0 if not int8 else 2.0 ** -14 if fine else 2.0 ** -10)) * scale * (x.abs() @ kh.abs().T)
            if int8:
                ks = ks + 2.0 ** -19 * scale * x.abs().sum(-1, keepdim=True) * kh.abs().max()
                # (a query value below 2^-14 of its row's largest is rounded to 2^-25 of that)
                # (of few rows it has 15 bits)
                ks = ks + 2.0 ** (-15 if fine else -24) * scale * x.abs().amax(-1, keepdim=True) * kh.abs().sum(-1)[None, :]
            # a weight: its score, s c - m in fp32, the cubic for 2^x (7.8e-5), rounding
            # to 16 bits, whose smallest step is 2^-25 of a weight of 1
            e = ks + 2.0 ** -22 * ((s - m).abs().clamp(max=200) + s.abs()) + 8e-5 + p_round
            floor = (2.0 ** -25 / total).expand_as(w) if p_round < 2.0 ** -8 else torch.zeros_like(w)
            we = w * e + floor
            err = we @ vh.abs() + we.sum(-1, keepdim=True) * o.abs()
            # V: rounded to f16 twice, or to two f16, with a floor; fp32 sums of the products
            err = err + (k.shape[1] * 2.0 ** -24 + (0 if not int8 else 2.0 ** -14 if fine else 2.0 ** -10)) * (w @ vh.abs())
            if int8:
                err = err + 2.0 ** -19 * vh.abs().max()
            out[b, :, h], lse[b, :, h] = o, (m + torch.log(total))[:, 0]
            bound[b, :, h] = 1.05 * err + o.abs() * torch.finfo(q.dtype).eps / 2 + 1e-30
            if q.dtype is F16:
                bound[b, :, h] += 2.0 ** -25
            lse_bound[b, :, h] = 1.05 * (we.sum(-1) + 2.0 ** -22 * (1 + lse[b, :, h].abs()))
    return out, lse, bound, lse_bound


def check(q, kv, lengths=None, prefix=None, prefix_lengths=None, scale=None, **kw):
    cap = kv.capacity if isinstance(kv, KVCacheI8) else kv[0].shape[2]
    as_list = lambda n, count, most: [most if n is None else n] * count if not torch.is_tensor(n) else n.clamp(0, most).tolist()  # noqa: E731
    groups = prefix[0].shape[0] if prefix is not None else 0
    pcap = 0 if prefix is None else prefix[0].shape[2]
    ref = ref_attend(q, kv, as_list(lengths, q.shape[0], cap), prefix, as_list(prefix_lengths, groups, pcap),
                     0.125 if scale is None else scale)
    out, lse = attend(q, kv, lengths, prefix=prefix, prefix_lengths=prefix_lengths, scale=scale, return_lse=True, **kw)
    assert out.dtype is q.dtype and out.shape == (q.shape[0], q.shape[2], q.shape[1], DIM)
    diff = (out.double().cpu() - ref[0]).abs()
    assert torch.isfinite(out).all()
    assert (diff <= ref[2]).all(), float((diff / ref[2]).max())
    lse = lse.double().cpu()
    empty = torch.isinf(ref[1])
    assert torch.equal(torch.isinf(lse), empty) and (out.cpu()[empty] == 0).all()
    ldiff = (lse - ref[1]).abs()[~empty]
    assert (ldiff <= ref[3][~empty]).all(), float((ldiff / ref[3][~empty]).max())
    _lib.check_device_error()
    return out


def dev_ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ------------------------------------------------------ write and read back

@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows, start, capacity", [(1, 0, 1), (1, 63, 64), (7, 3, 64), (64, 0, 64), (65, 62, 192),
                                                   (333, 5, 384)])
@pytest.mark.parametrize("layout", ["heads", "tokens", "turned", "odd"])
def test_write(cuda, dtype, rows, start, capacity, layout):
    k, v = values((3, 2, rows, DIM), rows, dtype), values((3, 2, rows, DIM), rows + 1, dtype)

    def lay(x):
        if layout == "tokens":
            return x.transpose(1, 2).contiguous().transpose(1, 2)
        if layout == "turned":
            return x.transpose(2, 3).contiguous().transpose(2, 3)
        if layout == "odd":  # neither dimension contiguous, and no alignment
            wide = torch.zeros(3, 2, rows + 1, 2 * DIM + 3, dtype=dtype, device="cuda")
            wide[:, :, 1:, 1:2 * DIM + 1:2] = x
            return wide[:, :, 1:, 1:2 * DIM + 1:2]
        return x

    c = KVCacheI8.empty(3, 2, capacity)
    for t in c:
        t.fill_(77)
    write_kv(c, lay(k), lay(v), start)
    for x, codes, scale in ((k, c.k, c.k_scale), (v, c.v, c.v_scale)):
        want, want_scale = ref_codes(x)
        at = slice(start, start + rows)
        assert torch.equal(codes[:, :, at].cpu(), want) and torch.equal(scale[:, :, at].cpu(), want_scale)
        codes, scale = codes.clone(), scale.clone()
        codes[:, :, at], scale[:, :, at] = 77, 77
        assert (codes == 77).all() and (scale == 77).all()  # all others as they were


def test_write_values(cuda):
    """Rows of zeros, next to zero, next to the largest float, with values that
    are not finite, and quotients halfway between codes."""
    rows = torch.randn(12, DIM, generator=torch.Generator().manual_seed(0))
    rows[0] = 0
    rows[1] *= 1e-31 / rows[1].abs().max()   # below 2^-100
    rows[2] *= 1e-29 / rows[2].abs().max()
    rows[3] *= 3.4e38 / rows[3].abs().max()
    rows[4, 5] = math.inf
    rows[5, 63] = -math.inf
    rows[6, 0] = math.nan
    rows[7] = (torch.arange(DIM) - 31.5) / 127  # x / scale halfway or next to it
    rows[7, 0] = 1
    rows[8] = torch.arange(DIM) * 1e-42        # subnormal
    rows[9] = 0
    rows[9, 40] = -5
    rows[10, 3], rows[10, 4] = math.nan, math.inf
    for dtype in (F32, BF16):
        x = rows.to(dtype).view(1, 1, 12, DIM).cuda()
        c = KVCacheI8.empty(1, 1, 64)
        write_kv(c, x, x)
        want, scale = ref_codes(x)
        for codes, got in ((c.k, c.k_scale), (c.v, c.v_scale)):
            assert torch.equal(codes[:, :, :12].cpu(), want)
            assert torch.equal(torch.nan_to_num(got[:, :, :12].cpu(), nan=-1), torch.nan_to_num(scale, nan=-1))
        k, v = read_kv(c, 0, 12, dtype=F32)
        bad = torch.isnan(scale)[..., None].expand_as(want)
        assert torch.isnan(k.cpu()[bad]).all() and torch.isfinite(k.cpu()[~bad]).all() and torch.equal(v[0, 0, 9], k[0, 0, 9])
        assert float(k[0, 0, 9, 40]) == float(scale[0, 0, 9] * -127)  # (in fp32)


def test_write_ragged(cuda):
    """Starts and counts on the device, partly outside the cache or negative."""
    k, v = values((6, 3, 70, DIM), 1), values((6, 3, 70, DIM), 2, F16).transpose(2, 3).contiguous().transpose(2, 3)
    starts, counts = [0, 100, 60, -3, 127, 200], [70, 0, 70, 5, 1, 70]
    c = KVCacheI8.empty(6, 3, 128)
    for t in c:
        t.fill_(55)
    write_kv(c, k, v, dev_ints(starts), dev_ints(counts))
    for x, codes, scale in ((k, c.k, c.k_scale), (v, c.v, c.v_scale)):
        want = [torch.full(codes.shape, 55, dtype=torch.int8), torch.full(scale.shape, 55.0)]
        rc, rs = ref_codes(x)
        for b in range(6):
            for i in range(min(counts[b], 70)):
                p = starts[b] + i
                if 0 <= p < 128:
                    want[0][b, :, p], want[1][b, :, p] = rc[b, :, i], rs[b, :, i]
        assert torch.equal(codes.cpu(), want[0]) and torch.equal(scale.cpu(), want[1])
    # counts beyond the rows and negative ones are kept to [0, rows]
    write_kv(c, k[:, :, :4], v[:, :, :4], dev_ints([0] * 6), dev_ints([9, -2, 4, 0, 1, 2]))
    assert torch.equal(c.k[0, :, 4:60].cpu(), ref_codes(k)[0][0, :, 4:60])
    assert (c.k[1] == 55).all() and (c.k[3, :, 5:] == 55).all()


def test_write_run_rows(cuda):
    k, v = values((4, 2, 33, DIM), 3), values((4, 2, 33, DIM), 4)
    for run, live in ((0, 0), (33, 1), (70, 2), (132, 4)):
        c = KVCacheI8.empty(4, 2, 64)
        c.k.fill_(9)
        write_kv(c, k, v, 0, run_rows=dev_ints([run]))
        assert torch.equal(c.k[:live, :, :33].cpu(), ref_codes(k)[0][:live]) and (c.k[live:] == 9).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("start, rows", [(0, 1), (0, 192), (5, 63), (130, 62), (191, 1), (64, 0)])
def test_read(cuda, dtype, start, rows):
    c = cache_of(values((2, 3, 192, DIM), 5), values((2, 3, 192, DIM), 6))
    k, v = read_kv(c, start, rows, dtype=dtype)
    for got, codes, scale in ((k, c.k, c.k_scale), (v, c.v, c.v_scale)):
        want = (codes.double() * scale.double()[..., None]).to(F32).to(dtype)[:, :, start:start + rows]
        assert got.dtype is dtype and torch.equal(got, want)


# ------------------------------------------------------------- attention

LENGTHS = [1, 2, 31, 63, 64, 65, 127, 128, 129, 200, 1001, 3000]


@pytest.mark.parametrize("length", LENGTHS)
@pytest.mark.parametrize("kind", ["int8", "bf16", "f16", "turned"])
def test_one_token(cuda, length, kind):
    check(*case(2, 3, 3, 1, length, kind, length))


def case(batch, heads, kv_heads, n, length, kind, seed, capacity=None):
    """(q, kv): keys of a capacity (default: the length) behind which lies NaN."""
    dtype = F16 if kind == "f16" else BF16
    q = values((batch, heads, n, DIM), seed + 1000, dtype)
    k, v = values((batch, kv_heads, length, DIM), seed, dtype), values((batch, kv_heads, length, DIM), seed + 1, dtype)
    if kind == "int8":
        return (q, cache_of(k, v, capacity), length)
    cap = max(capacity or length, 1)
    kk = torch.full((batch, kv_heads, cap, DIM), math.nan, dtype=dtype, device="cuda")
    kk[:, :, :length] = k
    if kind == "turned":
        vv = torch.full((batch, kv_heads, DIM, (cap + 7) // 8 * 8), math.nan, dtype=F16, device="cuda")
        vv[:, :, :, :length] = v.transpose(2, 3).half()
        return q, (kk, vv.transpose(2, 3)[:, :, :cap]), length
    vv = torch.full_like(kk, math.nan)
    vv[:, :, :length] = v
    return q, (kk, vv), length


@pytest.mark.parametrize("n", [2, 8, 9, 16, 17, 64, 127, 128, 129, 300, 513])
@pytest.mark.parametrize("kind", ["int8", "bf16", "f16", "turned"])
def test_queries(cuda, n, kind):
    q, kv, length = case(2, 2, 2, n, 150, kind, n, capacity=200)
    check(q, kv, length)


@pytest.mark.parametrize("n, batch, length, prefix", [(1, 2, 700, 0), (16, 2, 130, 0), (17, 2, 1, 0), (40, 3, 3000, 0),
                                                      (129, 2, 65, 200), (600, 2, 1000, 0), (520, 4, 333, 130)])
def test_f16_queries_over_int8(cuda, n, batch, length, prefix):
    """Whose rounding shows more than bf16's: keys and values as two f16."""
    q, kv, _ = case(batch, 4, 2, n, length, "int8", n, capacity=length + 70)
    pre, pre_length = None, None
    if prefix:
        _, pre, pre_length = case(batch // 2, 4, 2, 1, prefix, "int8", 9, capacity=prefix + 60)
    check(q.half(), kv, length, pre, pre_length)
    got = attend(q.half(), kv, length, prefix=pre, prefix_lengths=pre_length)
    ref = ref_attend(q.half(), kv, [length] * batch, pre, [pre_length] * (batch // 2))[0]
    # at random: the output and a weight each 2^-11 / sqrt(3) at most, and scores 2^-14 of
    # a few units
    assert float((got.double().cpu() - ref).norm() / ref.norm()) < 2.0 ** -11


@pytest.mark.parametrize("heads, kv_heads", [(4, 1), (6, 2), (7, 7), (16, 4), (5, 1), (200, 1)])
@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("kind", ["int8", "bf16"])
def test_grouped_heads(cuda, heads, kv_heads, n, kind):
    check(*case(2, heads, kv_heads, n, 111, kind, heads))


@pytest.mark.parametrize("kind", ["int8", "bf16", "turned"])
@pytest.mark.parametrize("n", [1, 12, 33, 140, 600])
def test_ragged(cuda, kind, n):
    """A length for each sequence, none, all and beyond all among them."""
    q, kv, _ = case(8, 2, 2, n, 700, kind, n, capacity=720)
    lengths = dev_ints([700, 0, 1, 64, 65, -5, 333, 699])
    check(q, kv, lengths)
    q, kv, _ = case(2, 2, 2, n, 640, kind, n)
    check(q, kv, dev_ints([10 ** 9, 640]))


@pytest.mark.parametrize("kind", ["int8", "bf16", "f16", "turned"])
@pytest.mark.parametrize("groups, batch, n, prefix, own", [
    (1, 5, 1, 300, 70), (1, 130, 1, 257, 9), (2, 6, 3, 1000, 64), (3, 3, 2, 100, 100), (1, 4, 200, 130, 65),
    (2, 4, 128, 64, 64), (1, 9, 40, 1, 1), (1, 3, 1, 5000, 2), (2, 4, 600, 130, 65), (1, 700, 1, 70, 65),
    (1, 7, 2, 3000, 64), (1, 24, 20, 1500, 64), (2, 8, 40, 2500, 130), (1, 40, 2, 900, 300),
])
def test_prefix(cuda, kind, groups, batch, n, prefix, own):
    q, kv, length = case(batch, 4, 2, n, own, kind, prefix, capacity=own + 5)
    _, pre, pre_length = case(groups, 4, 2, 1, prefix, kind, prefix + 7, capacity=prefix + 3)
    check(q, kv, length, pre, pre_length)


@pytest.mark.parametrize("v_dtype", [BF16, F16])
@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("n", [1, 12, 40, 300])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_types_of_v(cuda, dtype, v_dtype, turned, n):
    """V in either 16-bit type by rows or columns, for queries and keys of either type,
    alone and behind a prefix, with NaN behind the last key."""

    def keys(entries, length, seed):
        cap = length + 11
        k = torch.full((entries, 2, cap, DIM), math.nan, dtype=dtype, device="cuda")
        k[:, :, :length] = values((entries, 2, length, DIM), seed, dtype)
        v = torch.full((entries, 2, (cap + 7) // 8 * 8, DIM), math.nan, dtype=v_dtype, device="cuda")
        v[:, :, :length] = values((entries, 2, length, DIM), seed + 1, v_dtype)
        if turned:
            v = v.transpose(2, 3).contiguous().transpose(2, 3)
        return k, v[:, :, :cap]

    q = values((4, 4, n, DIM), n, dtype)
    own, prefix = keys(4, 150, 21), keys(2, 333, 31)
    check(q, own, 150)
    check(q, own, dev_ints([150, 0, 65, 1]))
    check(q, own, 150, prefix, 333)
    check(q, own, dev_ints([150, 0, 65, 1]), prefix, dev_ints([333, 64]))


@pytest.mark.parametrize("kind", ["int8", "bf16", "turned"])
@pytest.mark.parametrize("n", [1, 150, 520])
def test_prefix_ragged(cuda, kind, n):
    """Lengths on the device for both parts; a sequence without keys of its own,
    a group without a prefix, and both together."""
    q, kv, _ = case(6, 2, 2, n, 90, kind, n, capacity=100)
    _, pre, _ = case(3, 2, 2, 1, 200, kind, n + 1, capacity=210)
    check(q, kv, dev_ints([0, 90, 0, 64, 1, 89]), pre, dev_ints([200, 0, 65]))


@pytest.mark.parametrize("kind", ["int8", "bf16"])
@pytest.mark.parametrize("n", [1, 70, 520])
def test_peaked_and_far_scores(cuda, kind, n):
    """Scores of hundreds whose maximum keeps growing along the keys, so that the
    sums are rescaled, and rows of V whose size grows and falls by 2^30."""
    q, kv, length = case(2, 2, 2, n, 640, kind, 3)
    if kind == "int8":
        ramp = torch.linspace(0.1, 12, 640, device="cuda").sqrt()
        kv.k_scale.mul_(ramp)
        kv.v_scale.mul_(torch.exp2((torch.arange(640, device="cuda") * 7919 % 61 - 30).float()))
    else:
        kv[0].mul_(torch.linspace(0.1, 12, 640, device="cuda").sqrt()[:, None].to(BF16))
    check(q * 4, kv, length)


@pytest.mark.parametrize("kind", ["int8", "bf16", "f16", "turned"])
@pytest.mark.parametrize("n", [1, 12, 40, 520])
def test_scores_beyond_the_steps_of_fp32(cuda, kind, n):
    """Scores up to 10^9 and more, of either sign, where fp32 holds no fractions: the
    key with the largest one has all the weight."""
    dtype = F16 if kind == "f16" else BF16
    q, k = values((2, 2, n, DIM), 5, dtype) * 100, values((2, 2, 300, DIM), 6, dtype) * 4000
    v = values((2, 2, 300, DIM), 7, F16 if kind == "turned" else dtype)
    kv = cache_of(k, v) if kind == "int8" else (k, v)
    if kind == "turned":
        wide = torch.zeros(2, 2, DIM, 304, dtype=F16, device="cuda")
        wide[..., :300] = v.transpose(2, 3)
        kv = (k, wide.transpose(2, 3)[:, :, :300])
    # roundings: the key's weight in the product, not in the divisor where rows are few
    # (bf16 2^-8, f16 2^-11; it is a power of two only if the score's rounding is none),
    # an int8 row twice, the output half a step
    p_round = {"bf16": 2.0 ** -8, "int8": 2.0 ** -11 + 2.0 ** -10}.get(kind, 2.0 ** -11)
    for scale in (1.0, 300.0):
        out, lse = attend(q, kv, 300, scale=scale, return_lse=True)
        out, lse = out.double().cpu(), lse.double().cpu()
        assert torch.isfinite(out).all()
        seen = 0
        for b in range(2):
            kk, vv = dense(kv, b, 300)
            for h in range(2):
                s = scale * (q[b, h].double().cpu() @ kk[h].T)
                top2 = s.topk(2).values
                # (int8 rows are rounded to f16 twice: 2^-10 of sum |q k|, 2^-7 of the largest score)
                sure = (top2[:, 0] - top2[:, 1]) > 2.0 ** -6 * top2[:, 0].abs() + 100
                seen += int(sure.sum())
                want = vv[h][s.argmax(-1)]
                err = (out[b, :, h] - want).abs()
                limit = want.abs() * (torch.finfo(dtype).eps / 2 + p_round) + 2.0 ** -18 * vv[h].abs().max()
                assert (err[sure] <= limit[sure]).all()
                assert ((lse[b, :, h] - top2[:, 0]).abs() <= 2.0 ** -7 * top2[:, 0].abs()).all()
        assert seen > 2 * n
    _lib.check_device_error()


def far_keys(kind, keys, power, sign, leads):
    """Keys whose score is sign 2^power for the best (in the middle) and `lead` fp32 steps
    less for six others, in its tile and in tiles before and behind it; all others lie far
    below.  V of each of them has a column of its own.  (q, kv, places, scores)"""
    dtype = F16 if kind == "f16" else BF16
    best = keys // 2
    places = [best, best - 1, best + 2, keys - 1, 0, best + 75, best - 75][:1 + len(leads)]
    half = power // 2
    k = torch.zeros(1, 1, keys, DIM, dtype=torch.float64)
    k[..., 0] = 0 if sign > 0 else -1.5 * 2.0 ** (power - half)
    v = torch.zeros(1, 1, keys, DIM, dtype=torch.float64)
    for i, p in enumerate(places):
        k[0, 0, p, 0], k[0, 0, p, 1] = sign * 2.0 ** (power - half), -([0] + leads)[i] * 2.0 ** (power - 23)
        v[0, 0, p, i] = 1024
    q = torch.zeros(1, 1, 1, DIM, dtype=torch.float64)
    q[..., 0], q[..., 1] = 2.0 ** half, 1
    s = (q @ k.transpose(2, 3))[0, 0, 0]
    assert torch.equal(s.float().double(), s) and all(torch.equal(t.to(dtype).double(), t) for t in (q, k, v))
    q, k, v = (t.to(dtype).cuda() for t in (q, k, v))
    if kind == "turned":
        wide = torch.zeros(1, 1, DIM, (keys + 7) // 8 * 8, dtype=F16, device="cuda")
        wide[..., :keys] = v.transpose(2, 3)
        v = wide.transpose(2, 3)[:, :, :keys]
    return q, (k, v), places, s


@pytest.mark.parametrize("kind", ["bf16", "f16", "turned"])
@pytest.mark.parametrize("n", [1, 12, 40, 520])
@pytest.mark.parametrize("keys", [300, 4000])
def test_far_scores_in_steps(cuda, kind, n, keys):
    """Keys a few steps of fp32 below the best one, at scores where a step is half a unit
    and more: their weights are those of the difference, in whichever tile or part."""
    p_round = 2.0 ** -8 if kind == "bf16" else 2.0 ** -11
    scale = math.log(2.0)
    leads = [1, 2, 4, 8, 16, 64]
    for power, sign in ((22, 1), (23, -1), (24, 1), (24, -1), (26, 1), (27, -1)):
        q, kv, places, s = far_keys(kind, keys, power, sign, leads)
        out, lse = attend(q.expand(1, 1, n, DIM), kv, scale=scale, return_lse=True)
        got = out[0, :, 0].double().cpu() / 1024
        want = torch.zeros(DIM, dtype=torch.float64)
        # (scale is a float, and its product with log2(e) another: 2^-23 of a difference)
        weights = torch.exp2(s - s.max())
        want[:len(places)] = (weights / weights.sum())[places]
        gap = torch.zeros(DIM, dtype=torch.float64)
        gap[:len(places)] = (s.max() - s)[places]
        # roundings: a weight, the sum of weights and the output to 16 bits, 2^x by a cubic
        # (8e-5 of a weight and of the sum), the difference in fp32; the largest weight is
        # 2^-8 at least, so the smallest step is 2^-17 of it (f16)
        limit = want * (2 * p_round + torch.finfo(q.dtype).eps / 2 + 2e-4 + gap.clamp(max=200) * 2.0 ** -22)
        limit += 0 if kind == "bf16" else 2.0 ** -17
        limit += 1e-30 if q.dtype is BF16 else 2.0 ** -35
        assert ((got - want).abs() <= limit).all(), (power, sign, float(((got - want).abs() / limit).max()))
        want_lse = float(torch.logsumexp(s * scale, 0))
        assert ((lse.double().cpu() - want_lse).abs() <= 2.0 ** -22 * abs(want_lse)).all()
    # from 2^28 on a score counts to 2^-21 of its size: what lies further below has no weight
    for power, sign in ((28, 1), (30, -1), (30, 1)):
        q, kv, places, s = far_keys(kind, keys, power, sign, [8, 16, 64])
        got = attend(q.expand(1, 1, n, DIM), kv, scale=scale)[0, :, 0].double().cpu() / 1024
        assert ((got[:, 0] - 1).abs() <= 2 * p_round).all() and (got[:, 1:] <= 2.0 ** -17).all(), (power, sign)
    _lib.check_device_error()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("n", [1, 12])
def test_far_scores_over_int8(cuda, dtype, n):
    """The same over int8 keys with few rows, whose scores are fp32: a score of 127 2^17 is
    off by half a step, half a unit, in the best key and in another."""
    c = KVCacheI8.empty(1, 1, 320)
    for t in c:
        t.zero_()
    c.k[0, 0, [150, 151, 20], 0] = 127
    c.k_scale[0, 0, [150, 151, 20]] = torch.tensor([2.0 ** 5, 2.0 ** 5 * (1 - 2.0 ** -21), 2.0 ** 5 * (1 - 2.0 ** -20)],
                                                   device="cuda")
    for i, p in enumerate((150, 151, 20)):
        c.v[0, 0, p, i], c.v_scale[0, 0, p] = 127, 1
    q = torch.zeros(1, 1, n, DIM, dtype=dtype, device="cuda")
    q[..., 0] = 2.0 ** 12
    got = attend(q, c, 320, scale=math.log(2.0))[0, :, 0].double().cpu() / 127
    # differences of 127 2^-4 and 127 2^-3; the second weight is 2^-16, small for f16
    assert ((torch.log2(got[:, 1] / got[:, 0]) + 127 / 16).abs() <= 1 + 2.0 ** -6).all()
    assert ((got[:, 0] - 1).abs() < 2.0 ** -6).all() and (got[:, 2] <= 2.0 ** -14).all()
    _lib.check_device_error()


@pytest.mark.parametrize("kind", ["int8", "f16"])
@pytest.mark.parametrize("batch, n, keys", [(1200, 1, 2048), (592, 20, 20000), (74, 1000, 20000)])
def test_many_light_keys(cuda, kind, batch, n, keys):
    """One key with almost all the weight, and thousands with 2^-25.25 of it each, which
    f16 relative to the largest weight would lose."""
    k = torch.zeros(1, 1, keys, DIM, dtype=F16, device="cuda")
    v = torch.full((1, 1, keys, DIM), 1024.0, dtype=F16, device="cuda")
    k[0, 0, 5, 3], v[0, 0, 5] = 25.25, 0
    q = torch.zeros(batch, 1, n, DIM, dtype=F16, device="cuda")
    q[..., 3] = 1
    k, v = k.expand(batch, 1, keys, DIM), v.expand(batch, 1, keys, DIM)
    out = attend(q, cache_of(k, v) if kind == "int8" else (k, v), keys, scale=math.log(2.0)).double().cpu()
    tail = (keys - 1) * 2.0 ** -25.25
    # weights relative to 2^-8 of the largest, where half a step of f16 is 2^-25: 2^-33 of
    # it, 0.47% of 2^-25.25; int8 rows of more than 16 query rows are rounded twice:
    # 25.25 ln 2 2^-10 = 1.71%; output 2^-11
    limit = 0.0047 + (0.0172 if kind == "int8" and n > 16 else 0) + 2.0 ** -11 + 1e-4
    assert ((out / (1024 * tail / (1 + tail)) - 1).abs() <= limit).all()
    _lib.check_device_error()


@pytest.mark.parametrize("n", [5, 50, 520])
def test_scales(cuda, n):
    q, kv, length = case(1, 2, 2, n, 100, "int8", 9)
    for scale in (1e-3, 0.125, 1.0, 3.0):
        check(q, kv, length, scale=scale)
    # queries and keys far from 1: the scores stay the same
    for by in (2.0 ** 40, 2.0 ** -40):
        far = KVCacheI8(kv.k, kv.k_scale / by, kv.v, kv.v_scale * by)
        a, b = attend(q, kv, length), attend((q.float() * by).to(BF16), far, length)
        assert torch.equal((a.double() * by).to(BF16), b)


@pytest.mark.parametrize("n", [3, 50, 520])
def test_zero_rows(cuda, n):
    """All-zero keys and values (scale 0) among others, and queries of zeros."""
    q, kv, length = case(1, 2, 2, n, 130, "int8", 10)
    kv.k[:, :, ::3], kv.k_scale[:, :, ::3] = 0, 0
    kv.v[:, :, 1::3], kv.v_scale[:, :, 1::3] = 0, 0
    q[:, :, 1] = 0
    check(q, kv, length)
    kv.k_scale.zero_(), kv.v_scale.zero_()
    assert (check(q, kv, length) == 0).all()


@pytest.mark.parametrize("kind", ["int8", "bf16", "turned"])
@pytest.mark.parametrize("at", [0, 1, 8, 9, 63, 64, 100, 129])
@pytest.mark.parametrize("n", [3, 40, 520])
def test_not_finite(cuda, kind, at, n):
    """A key or value that is not finite shows in every row that uses it, and
    in no other."""
    for which in (0, 1):
        q, kv, length = case(2, 2, 2, n, 130, kind, 11)
        clean = attend(q, kv, length)
        if kind == "int8":
            (kv.k_scale if which == 0 else kv.v_scale)[0, 1, at] = math.nan
        else:
            kv[which][0, 1, at, 7] = math.nan
        got = attend(q, kv, length)
        bad = torch.isnan(got)
        assert bad[0, :, 1, 7].all() and not bad[1].any() and not bad[0, :, 0].any()
        assert torch.equal(got[1], clean[1]) and torch.equal(got[0, :, 0], clean[0, :, 0])
        if kind != "int8":
            kv[0][0, 1, at] = math.inf
            assert torch.isnan(attend(q, kv, length)[0, :, 1]).all()
        # behind the last key it is not looked at
        assert not torch.isnan(attend(q, kv, at if at else 1)[0, :, 1]).any() or at == 0
    _lib.check_device_error()


@pytest.mark.parametrize("n", [5, 50, 520])
def test_queries_not_finite(cuda, n):
    for kind in ("int8", "bf16"):
        q, kv, length = case(1, 2, 2, n, 90, kind, 12)
        clean = attend(q, kv, length)
        q[0, 1, 2, 9], q[0, 0, 4, 0] = math.nan, math.inf
        got = attend(q, kv, length)
        assert torch.isnan(got[0, 2, 1]).all() and torch.isnan(got[0, 4, 0]).all()
        keep = torch.ones(1, n, 2, dtype=torch.bool, device="cuda")
        keep[0, 2, 1] = keep[0, 4, 0] = False
        assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("kind", ["int8", "bf16", "turned"])
def test_layouts(cuda, kind):
    """Strided queries, keys inside wider buffers, an `out` of the caller's own."""
    q, kv, length = case(3, 4, 2, 6, 100, kind, 13)
    want = attend(q, kv, length)
    tokens = q.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(attend(tokens, kv, length), want)
    wide = torch.zeros(3, 4, 6, 70, dtype=BF16, device="cuda")  # rows that start anywhere are copied
    wide[..., 3:67] = q
    assert torch.equal(attend(wide[..., 3:67], kv, length), want)
    out = torch.empty(18, 256, dtype=BF16, device="cuda")
    assert attend(q, kv, length, out=out) is out and torch.equal(out.view(3, 6, 4, DIM), want)
    if kind == "bf16":
        k, v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in kv)
        assert torch.equal(attend(q, (k, v), length), want)
        # one sequence's or one head's keys for all, never copied
        for dims in (0, 1):
            alike = [t.narrow(dims, 0, 1) for t in kv]
            a = attend(q, tuple(t.expand(3, 2, -1, -1) for t in alike), length)
            assert torch.equal(a, attend(q, tuple(t.expand(3, 2, -1, -1).contiguous() for t in alike), length))
        buf = torch.full((3, 2, 130, 128), math.nan, dtype=BF16, device="cuda")
        buf[:, :, 20:120, :64], buf[:, :, 20:120, 64:] = kv[0], kv[1]
        assert torch.equal(attend(q, (buf[:, :, 20:120, :64], buf[:, :, 20:120, 64:])), want)
    if kind == "int8":  # entries of a wider cache
        pick = KVCacheI8(*(torch.cat([t[:1], t])[1:] for t in kv))
        assert pick.k.data_ptr() != kv.k.data_ptr() and torch.equal(attend(q, pick, length), want)


@pytest.mark.parametrize("kind", ["int8", "bf16"])
@pytest.mark.parametrize("at", [1, 4])
def test_queries_that_start_anywhere(cuda, kind, at):
    """Contiguous queries whose first element lies at no 16-byte boundary."""
    q, kv, length = case(2, 2, 2, 6, 100, kind, 13)
    flat = torch.zeros(q.numel() + 8, dtype=BF16, device="cuda")
    flat[at:at + q.numel()] = q.reshape(-1)
    moved = flat[at:at + q.numel()].view(q.shape)
    assert moved.is_contiguous() and moved.data_ptr() % 16
    assert torch.equal(attend(moved, kv, length), attend(q, kv, length))


@pytest.mark.parametrize("kind", ["int8", "bf16"])
@pytest.mark.parametrize("n", [1, 130, 520])
def test_run_rows(cuda, kind, n):
    q, kv, length = case(4, 2, 2, n, 333, kind, 14)
    _, pre, pre_length = case(1, 2, 2, 1, 500, kind, 15)
    for kw in ({}, {"prefix": pre, "prefix_lengths": pre_length}):
        want = attend(q, kv, length, **kw)
        for run, live in ((0, 0), (n, 1), (3 * n + n - 1, 3), (4 * n, 4), (100 * n, 4)):
            out = torch.full((4, n, 2, DIM), 5.0, dtype=BF16, device="cuda")
            attend(q, kv, length, out=out, run_rows=dev_ints([run]), **kw)
            assert torch.equal(out[:live], want[:live]) and (out[live:] == 5).all()


def test_split_and_whole_agree(cuda):
    """Single tokens over long keys (many parts) against the same rows inside a
    batch that needs no split, and lse joins disjoint keys."""
    q, kv, _ = case(2, 2, 2, 1, 5000, "bf16", 16)
    out, lse = attend(q, kv, return_lse=True)
    parts = [attend(q, (kv[0][:, :, a:b], kv[1][:, :, a:b]), return_lse=True) for a, b in ((0, 1111), (1111, 5000))]
    total = torch.logaddexp(parts[0][1], parts[1][1])
    joined = sum(o.float() * torch.exp(l - total)[..., None] for o, l in parts)
    # both are within their bounds of the exact result
    ref = ref_attend(q, kv, [5000, 5000])
    assert ((joined.double().cpu() - ref[0]).abs() <= 3 * ref[2]).all()
    assert ((total - lse).abs().cpu() <= 3 * ref[3]).all()
    check(q, kv)


@pytest.mark.parametrize("kind", ["int8", "bf16", "turned"])
@pytest.mark.parametrize("n", [1, 32, 300])
def test_length_known_to_the_host(cuda, kind, n):
    """Keys that are a small part of a cache cost what they cost in a small one: the same
    bits, so the same parts, and no more memory."""
    torch = cuda

    def peak(call):
        out = call()
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        again = call()
        torch.cuda.synchronize()
        used = torch.cuda.max_memory_allocated() - before
        assert torch.equal(out, again)
        return out, used

    for length, prefix_length in ((600, None), (150, None), (1, None), (64, 600), (0, 128), (700, 0), (0, 0)):
        q, small, _ = case(4, 4, 2, n, max(length, 1), kind, n)
        _, large, _ = case(4, 4, 2, n, max(length, 1), kind, n, capacity=8000)
        kws = [{}, {}]
        if prefix_length is not None:
            kws = [dict(prefix=case(2, 4, 2, 1, max(prefix_length, 1), kind, n + 5, capacity=cap)[1],
                        prefix_lengths=prefix_length) for cap in (None, 9000)]
        a, used = peak(lambda: attend(q, small, length, **kws[0]))
        b, most = peak(lambda: attend(q, large, length, **kws[1]))
        assert torch.equal(a, b) and most <= used
        check(q, large, length, kws[1].get("prefix"), kws[1].get("prefix_lengths"))
    _lib.check_device_error()


def test_same_bits(cuda):
    """The same call gives the same bits, alone or beside others on two streams."""
    for kind in ("int8", "bf16"):
        q, kv, length = case(6, 4, 4, 1, 3000, kind, 17)
        _, pre, pre_length = case(2, 4, 4, 1, 2000, kind, 18)
        want = attend(q, kv, length, prefix=pre, prefix_lengths=pre_length)
        other, streams = [], [torch.cuda.Stream() for _ in range(2)]
        torch.cuda.synchronize()
        for i in range(10):
            with torch.cuda.stream(streams[i % 2]):
                other.append(attend(q, kv, length, prefix=pre, prefix_lengths=pre_length))
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in other)


def test_graphs(cuda):
    """Write, attend and read captured once and replayed on new rows; two graphs
    whose workspaces come from one pool."""
    c = KVCacheI8.empty(2, 3, 512)
    c.k_scale.fill_(math.nan), c.v_scale.fill_(math.nan)
    k, v, q = values((2, 3, 40, DIM), 1), values((2, 3, 40, DIM), 2), values((2, 3, 40, DIM), 3)
    at, lengths = dev_ints([0, 0]), dev_ints([0, 0])

    def step():
        write_kv(c, k, v, at)
        lengths.copy_(at + 40)
        a = attend(q, c, lengths)
        return a, attend(q[:, :, :1], c, lengths), read_kv(c, 0, 40)[0]

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    g, h = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        first = step()
    with torch.cuda.graph(h, pool=g.pool()):
        second = attend(q, c, lengths, return_lse=True)
    rows = []
    for i in range(8):
        k.copy_(values((2, 3, 40, DIM), 10 + i)), v.copy_(values((2, 3, 40, DIM), 20 + i))
        q.copy_(values((2, 3, 40, DIM), 30 + i))
        at.fill_(40 * i)
        rows.append((k.clone(), v.clone()))
        g.replay()
        got = [t.clone() for t in first]
        h.replay()
        torch.cuda.synchronize()
        whole = cache_of(torch.cat([r[0] for r in rows], 2), torch.cat([r[1] for r in rows], 2), 512)
        want = attend(q, whole, 40 * (i + 1))
        assert torch.equal(got[0], want) and torch.equal(second[0], want)
        assert torch.equal(got[1], attend(q[:, :, :1], whole, 40 * (i + 1)))
        assert torch.equal(got[2], read_kv(whole, 0, 40)[0])
    _lib.check_device_error()


@pytest.mark.parametrize("kind", ["int8", "bf16"])
def test_offsets_past_32_bits(cuda, kind):
    """Entries that lie past 2^32 bytes and elements: the last of a large cache."""
    free, _ = torch.cuda.mem_get_info()
    entries, capacity = 35, 2 ** 21
    if free < 24e9:
        pytest.skip("needs 24 GB")
    n = 300
    k, v, q = values((1, 1, n, DIM), 1), values((1, 1, n, DIM), 2), values((entries, 1, 2, DIM), 3)
    if kind == "int8":
        c = KVCacheI8.empty(entries, 1, capacity)
        lengths = torch.zeros(entries, dtype=torch.int32, device="cuda")
        lengths[-1] = n
        counts, starts = lengths.clone(), torch.zeros_like(lengths)
        write_kv(c, k.expand(entries, -1, -1, -1), v.expand(entries, -1, -1, -1), starts, counts)
        small = cache_of(k, v)
        assert torch.equal(c.k[-1, :, :n], small.k[0, :, :n]) and torch.equal(c.v_scale[-1, :, :n], small.v_scale[0, :, :n])
        got = attend(q, c, lengths)
        ref = ref_attend(q[-1:], small, [n])
        assert ((got[-1:].double().cpu() - ref[0]).abs() <= ref[2]).all() and (got[:-1] == 0).all()
        assert torch.equal(read_kv(KVCacheI8(*(t[-1:] for t in c)), 0, n)[0], read_kv(small, 0, n)[0])
        # the last positions of the last entry
        write_kv(c, k.expand(entries, -1, -1, -1), v.expand(entries, -1, -1, -1), starts + capacity - n, counts)
        assert torch.equal(c.k[-1, :, -n:], small.k[0, :, :n])
    else:
        big = torch.zeros(entries, 1, capacity, DIM, dtype=BF16, device="cuda")
        big[-1, :, :n] = k[0]
        lengths = torch.zeros(entries, dtype=torch.int32, device="cuda")
        lengths[-1] = n
        got = attend(q, (big, big), lengths)
        ref = ref_attend(q[-1:], (k, k), [n])
        assert ((got[-1:].double().cpu() - ref[0]).abs() <= ref[2]).all() and (got[:-1] == 0).all()
    _lib.check_device_error()
