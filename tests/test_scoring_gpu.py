"""The scoring operators against plain float64 implementations.

Tolerances come from the rounding of each step (u = 2^-24, half an fp32 step):
an exponential e^(x - m) is off by 2 u |x - m| (the difference and its product
with log2 e) and by 2^-22 (the hardware exponential), and a sum of positive
terms by u for each addition on its longest chain.  The softmax mean of
|x - m|, `spread` below, weighs the first of these.
"""

import math

import pytest
import torch

from diffusionhard_b200 import _lib, scoring

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


# ------------------------------------------------------------ references

def ref_scores(x, targets, top_k, mask=None):
    """Scores of float64 logits x [rows, vocab] on the CPU, row by row."""
    out = {"logprobs": [], "entropy": [], "logsumexp": [], "top_ids": [], "top_logprobs": [], "tol": []}
    for r in range(x.shape[0]):
        row = x[r].clone()
        if mask is not None:
            row[mask] = -math.inf
        t = targets[r].reshape(-1).tolist()
        if bool(torch.isnan(row).any()) or bool((row == math.inf).any()):
            nan = math.nan
            out["logprobs"].append([0.0 if i < 0 else nan for i in t])
            out["entropy"].append(nan)
            out["logsumexp"].append(nan)
            out["top_ids"].append([-1] * top_k)
            out["top_logprobs"].append([nan] * top_k)
            out["tol"].append(0.0)
            continue
        finite = row[row > -math.inf]
        if finite.numel() == 0:
            out["entropy"].append(0.0)
            out["logsumexp"].append(-math.inf)
            lp = torch.full_like(row, -math.inf)
            spread = 0.0
        else:
            # relative to the maximum: next to -3e38 even float64 holds no log of a sum
            d = row - finite.max()
            log_s = torch.log(torch.exp(d).sum())
            lp = d - log_s
            p = torch.exp(lp)
            out["entropy"].append(float(torch.special.entr(p).sum()))
            out["logsumexp"].append(float(finite.max() + log_s))
            spread = -float((p * d.clamp(min=-1e30)).sum())
        out["logprobs"].append([0.0 if i < 0 else (float(lp[i]) if i < row.numel() else math.nan) for i in t])
        ids = torch.sort(row, descending=True, stable=True).indices[:top_k].tolist()
        ids = [i for i in ids if row[i] > -math.inf]
        out["top_logprobs"].append([float(lp[i]) for i in ids] + [-math.inf] * (top_k - len(ids)))
        out["top_ids"].append(ids + [-1] * (top_k - len(ids)))
        # relative error of the sums: chains of at most V / 64 additions (a
        # quarter of a row's logits in pairs at the least), 64 joins and
        # rescalings, and the exponentials
        out["tol"].append((x.shape[1] / 64 + 64 + 4 * (spread + 4)) * U)
    return out


def check_scores(got, x, targets, top_k, mask=None):
    ref = ref_scores(x.cpu(), targets.cpu(), top_k, mask)
    g = {k: v.cpu() for k, v in got._asdict().items() if v is not None}
    rows = x.shape[0]
    if top_k:
        assert g["top_ids"].tolist() == ref["top_ids"]
    else:
        assert got.top_ids is None and got.top_logprobs is None
    for r in range(rows):
        tol = ref["tol"][r]
        pairs = [("entropy", [float(g["entropy"][r])], [ref["entropy"][r]]),
                 ("logsumexp", [float(g["logsumexp"][r])], [ref["logsumexp"][r]]),
                 ("logprobs", g["logprobs"][r].reshape(-1).tolist(), ref["logprobs"][r])]
        if top_k:
            pairs.append(("top", g["top_logprobs"][r].tolist(), ref["top_logprobs"][r]))
        for name, a, b in pairs:
            assert len(a) == len(b)
            for p, q in zip(a, b):
                if math.isnan(q) or math.isinf(q):
                    assert (math.isnan(p) and math.isnan(q)) or p == q, (name, r, p, q)
                else:
                    # t / s of the entropy carries the relative error of two sums
                    scale = 2 * (1 + abs(ref["entropy"][r]) + 4) if name == "entropy" else 1.0
                    assert abs(p - q) <= tol * scale + 4 * U * (abs(q) + 16), (name, r, p, q)


def logits_case(rows, vocab, dtype, seed, scale=3.0, pad=0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, vocab + pad, generator=g) * scale).to(dtype)
    t = torch.randint(0, vocab, (rows,), generator=g)
    return x, t


DTYPES = [torch.float32, torch.bfloat16, torch.float16]


# ------------------------------------------------------- token_logprobs

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, vocab, top_k", [
    (1, 1, 1), (3, 2, 2), (2, 7, 8), (4, 31, 32), (5, 257, 5), (2, 1000, 0), (3, 4099, 32), (1, 50258, 8),
    (7, 50258, 20), (200, 2049, 3), (2, 131072, 8),
])
def test_token_logprobs(cuda, dtype, rows, vocab, top_k):
    x, t = logits_case(rows, vocab, dtype, rows * vocab)
    got = scoring.token_logprobs(x.cuda(), t.cuda(), top_k=top_k)
    check_scores(got, x.double(), t, top_k)


@pytest.mark.parametrize("rows", [1, 2, 5, 17, 37, 74, 148, 297, 600, 1300])
def test_token_logprobs_row_counts(cuda, rows):
    """Every way the row count splits rows over the GPU."""
    x, t = logits_case(rows, 5003, torch.float32, rows)
    check_scores(scoring.token_logprobs(x.cuda(), t.cuda(), top_k=4), x.double(), t, 4)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("start", [1, 2, 3, 5, 7])
def test_token_logprobs_alignment(cuda, dtype, start):
    """Rows that start anywhere, inside a wider buffer whose other values would show."""
    x, t = logits_case(6, 3001, dtype, start, pad=16)
    x[:, :start] = 1000.0
    x[:, start + 3001:] = 1000.0
    got = scoring.token_logprobs(x.cuda()[:, start:start + 3001], t.cuda(), top_k=6)
    check_scores(got, x[:, start:start + 3001].double(), t, 6)


@pytest.mark.parametrize("dtype", DTYPES)
def test_token_logprobs_mask_token(cuda, dtype):
    for mask in (0, 1, 6, 7, 8, 2500, 4999, 5000):
        x, t = logits_case(3, 5001, dtype, mask)
        x[:, mask] = math.inf if mask % 2 else math.nan  # excluded, whatever it holds
        t[0] = mask
        check_scores(scoring.token_logprobs(x.cuda(), t.cuda(), top_k=5, mask_token_id=mask), x.double(), t, 5, mask)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows_more", [0, 900])
def test_token_logprobs_odd_rows(cuda, dtype, rows_more):
    """Banned tokens, empty rows, lowest finite values, infinities, NaN, ties."""
    low = torch.finfo(dtype).min
    x, _ = logits_case(14 + rows_more, 2500, dtype, 5)
    x[0, ::3] = -math.inf
    x[1] = -math.inf
    x[2] = -math.inf
    x[2, 77] = -5.0
    x[3] = low
    x[4] = low
    x[4, 2499] = 1.0
    x[5, 1200] = math.nan
    x[6, 3] = math.inf
    x[7] = -math.inf
    x[7, 9] = math.nan
    x[8] = 0.25
    x[9, ::2] = -0.0
    x[9, 1::2] = 0.0
    x[10] = torch.arange(2500).to(dtype) / 100
    x[11] = torch.arange(2500, 0, -1).to(dtype) / 100
    x[12] = -math.inf
    x[12, 2490:] = 3.0
    x[13, 5] = torch.finfo(dtype).max
    t = torch.tensor([[0, 77, -1, 2499, 2500]] * x.shape[0])
    for k in (0, 1, 8, 32):
        check_scores(scoring.token_logprobs(x.cuda(), t.cuda(), top_k=k), x.double(), t, k)


def test_token_logprobs_targets(cuda):
    x, _ = logits_case(4, 300, torch.float32, 0)
    xs = x.cuda()
    t = torch.randint(-2, 310, (4, 45), generator=torch.Generator().manual_seed(1))
    for tt in (t, t.to(torch.int32)):
        check_scores(scoring.token_logprobs(xs, tt.cuda()), x.double(), t, 0)
    wide = torch.stack([t, t + 1], 2).cuda()[:, :, 0]  # not contiguous
    check_scores(scoring.token_logprobs(xs, wide), x.double(), t, 0)
    big = torch.tensor([2 ** 40, -2 ** 40, 2 ** 32, 299])
    check_scores(scoring.token_logprobs(xs, big.cuda()), x.double(), big, 0)
    none = scoring.token_logprobs(xs)
    assert none.logprobs is None
    torch.testing.assert_close(none.entropy, scoring.token_logprobs(xs, t.cuda()).entropy, rtol=0, atol=0)
    assert scoring.token_logprobs(xs, t.cuda()[:, :0]).logprobs.shape == (4, 0)
    assert scoring.token_logprobs(xs[:0], t.cuda()[:0], top_k=2).top_ids.shape == (0, 2)


def test_token_logprobs_broadcast_row(cuda):
    """A row stride of 0 (one row of logits, many targets)."""
    x, _ = logits_case(1, 4000, torch.bfloat16, 3)
    t = torch.arange(0, 4000, 97)
    check_scores(scoring.token_logprobs(x.cuda().expand(t.numel(), -1), t.cuda(), top_k=2),
                 x.double().expand(t.numel(), -1), t, 2)


def test_token_logprobs_far_rows(cuda):
    """Row offsets past 2^32 bytes and 2^31 elements."""
    buf = torch.empty(2 ** 31 + 4096, dtype=torch.bfloat16, device="cuda")
    x = buf.as_strided((3, 1001), (2 ** 30 + 1, 1))
    src, t = logits_case(3, 1001, torch.bfloat16, 9)
    x.copy_(src)
    check_scores(scoring.token_logprobs(x, t.cuda(), top_k=3), src.double(), t, 3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shift, scale", [(1e4, 1.0), (-1e6, 1.0), (3e8, 1.0), (-1e10, 1.0), (3e38, 1.0), (0.0, 1e3),
                                          (0.0, 1e7), (-1e5, 1e9), (0.0, 1e12), (0.0, 1e37)])
def test_token_logprobs_magnitudes(cuda, dtype, shift, scale):
    """Logits around any value, and as far apart, with giants among usual ones."""
    x, t = logits_case(8, 30011, torch.float32, 17, scale=scale)
    x += shift
    x[3] = logits_case(1, 30011, torch.float32, 18)[0][0]
    x[4] = x[3]
    x[5] = x[3]
    x[3, 7000], x[4, 29000], x[5, 3] = 3e38, -3e38, 1.1e9
    lim = torch.finfo(dtype).max
    x = x.clamp(-lim, lim).to(dtype)
    for k in (0, 5):
        check_scores(scoring.token_logprobs(x.cuda(), t.cuda(), top_k=k), x.double(), t, k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [20001, 50258])
def test_token_logprobs_many_equal_or_ordered(cuda, dtype, vocab):
    """Rows most of whose logits reach the bound of the k best: all equal, rising, falling, in steps."""
    i = torch.arange(vocab, dtype=torch.float64)
    x = torch.stack([torch.full_like(i, -2.5), i / 4000, -i / 4000, (i / 1000).floor(), -(i / 1000).floor(),
                     i % 7, torch.where(i % 4096 == 5, 3.0, 1.0)]).to(dtype)
    t = torch.tensor([[0, vocab - 1, 4096]] * x.shape[0])
    for k in (1, 7, 9, 32):
        check_scores(scoring.token_logprobs(x.cuda(), t.cuda(), top_k=k, mask_token_id=vocab - 2), x.double(), t, k,
                     vocab - 2)


# ------------------------------------------------------------ linear_i8

def linear_case(m, n, k, seed, bias=True):
    g = torch.Generator().manual_seed(seed)
    a = torch.randint(-127, 128, (m, k), generator=g, dtype=torch.int32).to(torch.int8)
    w = torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int32).to(torch.int8)
    return (a, torch.rand(m, generator=g) * 0.05 + 1e-3, w, torch.rand(n, generator=g) * 0.01 + 1e-4,
            torch.randn(n, generator=g) if bias else None)


def ref_linear(a, a_scale, w, w_scale, bias):
    acc = (a.double() @ w.double().T)
    y = acc * (a_scale[:, None] * w_scale[None, :]).double()
    return acc, (y if bias is None else y + bias.double())


def cu(args):
    return [None if x is None else x.cuda() for x in args]


LINEAR = [(1, 1, 1), (1, 64, 16), (3, 5, 48), (2, 2304, 768), (9, 130, 784), (16, 768, 3072), (17, 100, 64),
          (32, 769, 1040), (33, 1000, 128), (65, 257, 272), (128, 256, 768), (129, 4097, 256), (300, 2304, 96),
          (1024, 768, 4096), (1, 50258, 768), (40, 50258, 768)]


@pytest.mark.parametrize("m, n, k", LINEAR)
def test_linear_i8(cuda, m, n, k):
    args = linear_case(m, n, k, m * n + k, bias=(m + n) % 3 != 0)
    acc, y = ref_linear(*args)
    dev = cu(args)
    got = scoring.linear_i8(*dev)
    assert got.dtype == torch.float32
    assert torch.equal(got.cpu(), y.float())  # one rounding, the reference's own
    for dtype in (torch.bfloat16, torch.float16):
        got = scoring.linear_i8(*dev, out_dtype=dtype).cpu().double()
        lim = torch.finfo(dtype)
        # fp32: the sum past 2^24 and the FMA; then half a step of the type
        # (of its smallest normal number below it)
        prod = y if args[4] is None else y - args[4].double()
        tol = U * (prod.abs() + y.abs()) * 1.01 + lim.eps / 2 * 1.01 * y.abs().clamp(min=lim.tiny)
        assert bool(((got - y).abs() <= tol).all()), float(((got - y).abs() - tol).max())


def test_linear_i8_strides(cuda):
    """Row pitches and starts that the kernel takes as they are, and those it copies."""
    a, sa, w, sw, b = linear_case(50, 70, 200, 1)
    _, y = ref_linear(a, sa, w, sw, b)
    y = y.float()
    sa, sw, b = sa.cuda(), sw.cuda(), b.cuda()
    wide = torch.full((50, 272), 99, dtype=torch.int8, device="cuda")
    for start in (0, 16, 3):
        av = wide[:, start:start + 200]
        av.copy_(a)
        assert torch.equal(scoring.linear_i8(av, sa, w.cuda(), sw, b).cpu(), y)
    assert torch.equal(scoring.linear_i8(a.cuda().T.contiguous().T, sa, w.cuda(), sw, b).cpu(), y)
    assert torch.equal(scoring.linear_i8(a.cuda(), torch.stack([sa, sa], 1)[:, 0], w.cuda(), sw, b).cpu(), y)


@pytest.mark.parametrize("m", [3, 60])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pitch, start", [(80, 0), (73, 0), (96, 16), (81, 1), (70, 0)])
def test_linear_i8_out(cuda, dtype, pitch, start, m):
    """Only the given rows and columns of `out` are written."""
    args = linear_case(m, 70, 64, 2)
    dev = cu(args)
    buf = torch.full((m + 5, pitch), 7.0, dtype=dtype, device="cuda")
    flat = buf.view(-1)[start:start + m * pitch]
    out = flat.as_strided((m, 70), (pitch, 1), flat.storage_offset())
    ret = scoring.linear_i8(*dev, out=out)
    assert ret is out
    assert torch.equal(out, scoring.linear_i8(*dev, out_dtype=dtype))
    out.fill_(7.0)
    assert bool((buf == 7.0).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n, pitch, start", [
    (5008, 5008, 0), (5008, 5024, 16), (5003, 5008, 0), (5002, 5002, 0), (5002, 5004, 2), (5001, 5001, 0),
    (5001, 5010, 1), (5000, 5004, 4), (4900, 4902, 6),
])
def test_linear_i8_out_large(cuda, dtype, n, pitch, start):
    """The large tiles: outputs of every alignment, ragged in rows and columns, and nothing beside them."""
    m = 390
    args = linear_case(m, n, 80, n + pitch)
    dev = cu(args)
    buf = torch.full((m + 2, pitch), 7.0, dtype=dtype, device="cuda")
    flat = buf.view(-1)[start:start + m * pitch]
    out = flat.as_strided((m, n), (pitch, 1), flat.storage_offset())
    scoring.linear_i8(*dev, out=out)
    y = ref_linear(*args)[1]
    if dtype == torch.float32:
        assert torch.equal(out.cpu(), y.float())
    else:
        prod = y - args[4].double()
        lim = torch.finfo(dtype)
        tol = U * (prod.abs() + y.abs()) * 1.01 + lim.eps / 2 * 1.01 * y.abs().clamp(min=lim.tiny)
        assert bool(((out.cpu().double() - y).abs() <= tol).all())
    out.fill_(7.0)
    assert bool((buf == 7.0).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m, n, k, pitch", [(19001, 64, 96, 64), (32768, 50, 64, 53), (38000, 1, 128, 1), (20000, 61, 144, 64)])
def test_linear_i8_tall(cuda, dtype, m, n, k, pitch):
    """Many rows and few columns: several narrow tiles to a multiprocessor."""
    args = linear_case(m, n, k, m + n)
    buf = torch.full((m + 1, pitch), 7.0, dtype=dtype, device="cuda")
    out = buf[:m, :n]
    scoring.linear_i8(*cu(args), out=out)
    y = ref_linear(*args)[1]
    if dtype == torch.float32:
        assert torch.equal(out.cpu(), y.float())
    else:
        prod = y - args[4].double()
        lim = torch.finfo(dtype)
        tol = U * (prod.abs() + y.abs()) * 1.01 + lim.eps / 2 * 1.01 * y.abs().clamp(min=lim.tiny)
        assert bool(((out.cpu().double() - y).abs() <= tol).all())
    out.fill_(7.0)
    assert bool((buf == 7.0).all())


def test_linear_i8_odd_scales_large(cuda):
    """Scales of 0, infinity, NaN, negative, tiny and huge, and odd biases, in the large tiles."""
    a, sa, w, sw, b = linear_case(300, 5000, 64, 12)
    sa[::7] = torch.tensor([0.0, math.inf, math.nan, -0.5, 1e-38, 1e30, 1e-45] * 7)[:sa[::7].numel()]
    sw[::11] = torch.tensor([0.0, math.inf, math.nan, -0.5, 1e-38, 1e30, 1e-45] * 66)[:sw[::11].numel()]
    b[::13] = torch.tensor([math.inf, -math.inf, math.nan, 3e38, 1e-45] * 78)[:b[::13].numel()]
    for rows in (300, 100):  # and the small tiles'
        y = ref_linear(a[:rows], sa[:rows], w, sw, b)[1].float()
        got = scoring.linear_i8(*cu((a[:rows], sa[:rows], w, sw, b))).cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(y))
        assert torch.equal(got.nan_to_num(0.5), y.nan_to_num(0.5))


def test_linear_i8_far_out(cuda):
    args = linear_case(3, 100, 64, 4)
    dev = cu(args)
    buf = torch.empty(2 ** 31 + 4096, dtype=torch.bfloat16, device="cuda")
    out = buf.as_strided((3, 100), (2 ** 30 + 8, 1))
    scoring.linear_i8(*dev, out=out)
    assert torch.equal(out, scoring.linear_i8(*dev, out_dtype=torch.bfloat16))


def test_linear_i8_extremes(cuda):
    """The largest sums, -128, scales of 0, infinity and NaN."""
    k = 131056
    a = torch.full((2, k), -128, dtype=torch.int8)
    w = torch.full((3, k), -128, dtype=torch.int8)
    w[1] = 127
    sa = torch.tensor([1.0, 0.0])
    sw = torch.tensor([1.0, 1.0, math.inf])
    y = (a.long() @ w.long().T).double() * (sa[:, None] * sw).double()
    got = scoring.linear_i8(a.cuda(), sa.cuda(), w.cuda(), sw.cuda()).cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(y)) and bool(torch.isnan(got[1, 2]))
    assert torch.equal(got.nan_to_num(0.5), y.float().nan_to_num(0.5))


# --------------------------------------------------------- head_logprobs

def head_case(rows, vocab, size, seed, bias=True):
    g = torch.Generator().manual_seed(seed)
    a = (torch.randn(rows, size, generator=g) * 38).round().clamp(-127, 127).to(torch.int8)
    w = (torch.randn(vocab, size, generator=g) * 40).round().clamp(-127, 127).to(torch.int8)
    sa = (torch.rand(rows, generator=g) * 1.5 + 0.5) * 0.02
    sw = (torch.rand(vocab, generator=g) * 0.7 + 0.7) * (0.03 / math.sqrt(size))
    b = torch.randn(vocab, generator=g) * 0.5 if bias else None
    return (a, sa, w, sw, b), torch.randint(0, vocab, (rows,), generator=g)


HEAD = [(1, 1, 16, 1), (2, 15, 16, 4), (1, 16, 32, 8), (3, 17, 48, 32), (5, 257, 64, 5), (1, 50258, 768, 8),
        (33, 5001, 768, 8), (128, 2000, 256, 1), (129, 2000, 272, 0), (130, 700, 1040, 8), (40, 3000, 1536, 32),
        (257, 9001, 128, 3), (1500, 1000, 64, 2), (20, 40000, 64, 20)]


@pytest.mark.parametrize("rows, vocab, size, top_k", HEAD)
def test_head_logprobs(cuda, rows, vocab, size, top_k):
    args, t = head_case(rows, vocab, size, rows + vocab, bias=vocab % 2 == 0)
    x = ref_linear(*args)[1].float().double()
    mask = None if rows % 2 else vocab // 3
    got = scoring.head_logprobs(*cu(args), t.cuda(), top_k=top_k, mask_token_id=mask)
    check_scores(got, x, t, top_k, mask)


@pytest.mark.parametrize("size", [784, 800, 1024])
@pytest.mark.parametrize("rows, top_k", [(3, 8), (300, 0), (300, 5)])
def test_head_logprobs_streamed(cuda, rows, top_k, size):
    """Hidden sizes past those whose rows stay in shared memory."""
    args, t = head_case(rows, 3001, size, size)
    x = ref_linear(*args)[1].float().double()
    check_scores(scoring.head_logprobs(*cu(args), t.cuda(), top_k=top_k), x, t, top_k)


@pytest.mark.parametrize("size", [64, 800, 1040])
@pytest.mark.parametrize("rows, vocab, top_k", [(300, 20000, 0), (300, 20000, 9), (900, 9001, 32), (128, 37888, 4)])
def test_head_logprobs_many_tiles(cuda, rows, vocab, top_k, size):
    """Enough tiles for several to a multiprocessor, of either width."""
    (a, sa, w, sw, b), t = head_case(rows, vocab, size, size + top_k)
    got = scoring.head_logprobs(*cu((a, sa, w, sw, b)), t.cuda(), top_k=top_k, mask_token_id=7)
    pick = torch.tensor([0, 1, 8, 17, 63, 64, 126, 127] + ([128, 255, 256, 299] if rows > 128 else []))
    x = ref_linear(a[pick], sa[pick], w, sw, b)[1].float().double()
    some = got._replace(**{f: v[pick.cuda()] for f, v in got._asdict().items() if v is not None})
    check_scores(some, x, t[pick], top_k, 7)


@pytest.mark.parametrize("rows", [3, 800])
@pytest.mark.parametrize("size", [64, 1040])
def test_head_logprobs_many_equal(cuda, rows, size):
    """Rows whose every logit, or every bias of many, is equal: more groups reach the bound than are kept."""
    (a, sa, w, sw, b), t = head_case(rows, 6001, size, rows, bias=True)
    sa[::2] = 0.0
    b[:] = 1.5
    b[4000:] = 0.25
    pick = torch.tensor([0, 1, 2] if rows == 3 else [0, 1, 2, 7, 128, 511, 798, 799])
    x = ref_linear(a[pick], sa[pick], w, sw, b)[1].float().double()
    for k in (1, 8, 32):
        got = scoring.head_logprobs(*cu((a, sa, w, sw, b)), t.cuda(), top_k=k, mask_token_id=2)
        some = got._replace(**{f: v[pick.cuda()] for f, v in got._asdict().items()})
        check_scores(some, x, t[pick], k, 2)


def test_head_logprobs_far_weights(cuda):
    """Row offsets past 2^32 bytes in the weights and the hidden rows."""
    (a, sa, w, sw, b), t = head_case(5, 40, 48, 6)
    buf = torch.empty(2 ** 27 * 40 + 4096, dtype=torch.int8, device="cuda")
    wv = buf.as_strided((40, 48), (2 ** 27 + 16, 1))
    av = buf.as_strided((5, 48), (2 ** 30 + 64, 1), 1024)
    wv.copy_(w)
    av.copy_(a)
    assert torch.equal(wv.cpu(), w)
    x = ref_linear(a, sa, w, sw, b)[1].float().double()
    check_scores(scoring.head_logprobs(av, sa.cuda(), wv, sw.cuda(), b.cuda(), t.cuda(), top_k=4), x, t, 4)
    assert torch.equal(scoring.linear_i8(av, sa.cuda(), wv, sw.cuda(), b.cuda()).cpu(), x.float())


def test_head_logprobs_matches_two_steps(cuda):
    """The fused head, and the product followed by the scores of its logits."""
    args, t = head_case(70, 50258, 768, 0)
    dev = cu(args)
    x = scoring.linear_i8(*dev)
    a = scoring.head_logprobs(*dev, t.cuda(), top_k=32, mask_token_id=50257)
    b = scoring.token_logprobs(x, t.cuda(), top_k=32, mask_token_id=50257)
    assert torch.equal(a.top_ids, b.top_ids)
    for p, q in ((a.logprobs, b.logprobs), (a.entropy, b.entropy), (a.logsumexp, b.logsumexp),
                 (a.top_logprobs, b.top_logprobs)):
        torch.testing.assert_close(p, q, rtol=0, atol=2 * (50258 / 64 + 128) * U)


def test_head_logprobs_odd_rows(cuda):
    """Bans through the bias, equal logits, scales of 0, infinity and NaN."""
    (a, sa, w, sw, b), _ = head_case(9, 3000, 64, 1)
    b[::3] = -math.inf
    w[100:120] = w[100]
    sw[100:120] = sw[100]
    b[100:120] = 30.0
    sa[1] = 0.0   # every logit its bias
    sa[2] = math.nan
    sa[3] = math.inf
    sa[4] = 1e30
    t = torch.tensor([[0, 1, -1, 101, 3000]] * 9)
    x = ref_linear(a, sa, w, sw, b)[1].float().double()
    for k in (0, 4, 32):
        got = scoring.head_logprobs(*cu((a, sa, w, sw, b)), t.cuda(), top_k=k, mask_token_id=110)
        check_scores(got, x, t, k, 110)
    b[:] = -math.inf
    got = scoring.head_logprobs(*cu((a[:2], sa[:2], w, sw, b)), t[:2].cuda(), top_k=3)
    assert bool((got.top_ids == -1).all()) and bool((got.logsumexp == -math.inf).all())
    assert got.entropy.tolist() == [0.0, 0.0]
    b[:] = torch.finfo(torch.float32).min
    b[7] = 2.0
    x = ref_linear(a[:2], sa[:2], w, sw, b)[1].float().double()
    got = scoring.head_logprobs(*cu((a[:2], sa[:2], w, sw, b)), t[:2].cuda(), top_k=1)
    assert got.top_ids.tolist() == [[7], [7]]
    check_scores(got._replace(top_ids=None, top_logprobs=None), x, t[:2], 0)


@pytest.mark.parametrize("vocab", [75776, 75777, 80000, 81665, 90001, 131072, 131073])
def test_head_logprobs_large_vocabularies(cuda, vocab):
    """As many rows as get a warp each, around the vocabularies whose maxima shared memory holds."""
    (a, sa, w, sw, b), t = head_case(770, vocab, 16, vocab)
    got = scoring.head_logprobs(*cu((a, sa, w, sw, b)), t.cuda(), top_k=8, mask_token_id=vocab - 1)
    pick = torch.tensor([0, 1, 127, 128, 400, 767, 768, 769])
    x = ref_linear(a[pick], sa[pick], w, sw, b)[1].float().double()
    some = got._replace(**{f: v[pick.cuda()] for f, v in got._asdict().items()})
    check_scores(some, x, t[pick], 8, vocab - 1)


@pytest.mark.parametrize("size", [64, 1040])
@pytest.mark.parametrize("shift", [0.0, 1e4, -1e6, 3e8, -5e8, 1e10, 1e30])
def test_head_logprobs_far_from_zero(cuda, size, shift):
    """Logits of any magnitude, about 0 or around a common value."""
    (a, sa, w, sw, b), t = head_case(9, 3000, size, 7)
    sa *= torch.tensor([1.0, 1e3, 1e6, 1e8, 1e9, 1e11, 1e14, 1e30, 0.0])
    b += shift
    b[2000:2100] -= abs(shift)  # one block of columns lies elsewhere
    x = ref_linear(a, sa, w, sw, b)[1].float().double()
    for k in (0, 5):
        check_scores(scoring.head_logprobs(*cu((a, sa, w, sw, b)), t.cuda(), top_k=k), x, t, k)


@pytest.mark.parametrize("size", [64, 1040])
@pytest.mark.parametrize("shift, scale", [(1e4, 1.0), (-1e6, 1.0), (3e8, 1.0), (-1e10, 1.0), (0.0, 1e4), (0.0, 1e7),
                                          (-1e5, 1e9), (0.0, 1e12)])
def test_head_logprobs_same_magnitude(cuda, size, shift, scale):
    """All rows' logits around the same large value, or as far apart."""
    (a, sa, w, sw, b), t = head_case(9, 3000, size, 9)
    b += shift
    x = ref_linear(a, sa * scale, w, sw, b)[1].float().double()
    for k in (0, 5):
        check_scores(scoring.head_logprobs(*cu((a, sa * scale, w, sw, b)), t.cuda(), top_k=k), x, t, k)


@pytest.mark.parametrize("at", [5, 600, 2999])
def test_head_logprobs_lone_giants(cuda, at):
    """One logit near the largest or the lowest number among usual ones."""
    (a, sa, w, sw, b), t = head_case(5, 3000, 64, 8)
    for value in (3e38, 2e38, 1.1e9, -3e38):
        b[at] = value
        x = ref_linear(a, sa, w, sw, b)[1].float().double()
        for k in (0, 3):
            check_scores(scoring.head_logprobs(*cu((a, sa, w, sw, b)), t.cuda(), top_k=k), x, t, k)


def test_head_logprobs_padded_rows(cuda):
    (a, sa, w, sw, b), t = head_case(21, 333, 100, 2)
    x = ref_linear(a, sa, w, sw, b)[1].float().double()
    wide = torch.full((333, 160), 77, dtype=torch.int8, device="cuda")
    for start in (0, 16, 5):  # the last is copied, and so are the 100-byte rows of `a`
        wv = wide[:, start:start + 100]
        wv.copy_(w)
        got = scoring.head_logprobs(a.cuda(), sa.cuda(), wv, sw.cuda(), b.cuda(), t.cuda(), top_k=7)
        check_scores(got, x, t, 7)


@pytest.mark.parametrize("size", [64, 1040])
@pytest.mark.parametrize("rows", [5, 800])
@pytest.mark.parametrize("kind", ["one zero", "few above", "both signs", "subnormal"])
def test_head_logprobs_near_zero(cuda, kind, rows, size):
    """Logits next to zero on either side, far below what a half float tells from it."""
    (a, sa, w, sw, b), t = head_case(rows, 1000, size, 11)
    g = torch.Generator().manual_seed(12)
    b[:] = -1e-8
    if kind == "one zero":
        b[200] = 0.0
    elif kind == "few above":
        b[[40, 200, 777]] = torch.tensor([1e-9, 3e-8, 5e-8])
    else:
        b[:] = torch.randn(1000, generator=g) * (1e-8 if kind == "both signs" else 1e-40)
    sa[:] = 0.0  # every logit its bias
    sa[1::2] = 1e-9 if kind != "subnormal" else 1e-39
    pick = torch.tensor([0, 1, 2, 3, 4] if rows == 5 else [0, 1, 127, 128, 513, 798, 799])
    x = ref_linear(a[pick], sa[pick], w, sw, b)[1].float().double()
    for k in (1, 2, 3, 5, 8, 9, 32):
        got = scoring.head_logprobs(*cu((a, sa, w, sw, b)), t.cuda(), top_k=k, mask_token_id=3)
        some = got._replace(**{f: v[pick.cuda()] for f, v in got._asdict().items()})
        check_scores(some, x, t[pick], k, 3)


@pytest.mark.parametrize("size", [64, 784, 1040])
@pytest.mark.parametrize("rows, vocab", [(6, 1000), (6, 1536), (6, 50), (800, 1536), (800, 1111)])
def test_head_logprobs_infinite_scales(cuda, rows, vocab, size):
    """Columns that are no token, or the excluded one, make no row NaN whose own logits are all -inf."""
    (a, sa, w, sw, b), _ = head_case(rows, vocab, size, 13)
    a = a.abs().clamp(min=1)
    w = -w.abs().clamp(min=1)
    a[5] = -a[5]
    sa[0] = math.inf    # every logit -inf
    sa[1] = 3e38        # the products finite, or past the largest float
    sa[2] = math.nan
    sa[4] = -math.inf   # every logit +inf
    sa[5] = -math.inf   # -inf again
    sw[7::50] = 1e30
    t = torch.tensor([[0, 8, -1, vocab - 1, vocab]] * rows)
    pick = torch.tensor([0, 1, 2, 3, 4, 5] + ([127, 128, 799] if rows > 6 else []))
    for mask in (None, 8):
        # an excluded logit is taken out before NaN or infinity can come of it
        x = ref_linear(a[pick], sa[pick], w, sw, b)[1].float().double()
        for k in (0, 5, 32):
            got = scoring.head_logprobs(*cu((a, sa, w, sw, b)), t.cuda(), top_k=k, mask_token_id=mask)
            some = got._replace(**{f: v[pick.cuda()] for f, v in got._asdict().items() if v is not None})
            check_scores(some, x, t[pick], k, mask)


@pytest.mark.parametrize("size", [64, 1040])
def test_head_logprobs_nothing_left(cuda, size):
    """The only token excluded: a row is empty, whatever its scale."""
    (a, sa, w, sw, b), _ = head_case(5, 1, size, 14)
    sa[:] = torch.tensor([1.0, 0.0, math.inf, -math.inf, math.nan])
    t = torch.zeros((5, 1), dtype=torch.int64)
    x = ref_linear(a, sa, w, sw, b)[1].float().double()
    got = scoring.head_logprobs(*cu((a, sa, w, sw, b)), t.cuda(), top_k=2, mask_token_id=0)
    check_scores(got, x, t, 2, 0)


@pytest.mark.parametrize("bits", [-1, 0x7FFFFFFF, 0x7FC00000, -0x400000, 0x7F800001])
@pytest.mark.parametrize("size", [64, 1040])
def test_head_logprobs_nan_bias(cuda, size, bits):
    """A token's NaN bias makes every row NaN, whatever its bits; the excluded token's none."""
    (a, sa, w, sw, b), t = head_case(5, 700, size, 15)
    b[33] = torch.tensor([bits], dtype=torch.int32).view(torch.float32)[0]
    x = ref_linear(a, sa, w, sw, b)[1].float().double()
    assert bool(torch.isnan(x[:, 33]).all())
    dev = cu((a, sa, w, sw, b))
    dev[4].view(torch.int32)[33] = bits  # as given, not as the host rounds it
    for mask in (None, 32, 33):
        check_scores(scoring.head_logprobs(*dev, t.cuda(), top_k=3, mask_token_id=mask), x, t, 3, mask)


@pytest.mark.parametrize("size", [752, 768, 769, 896, 1023])
@pytest.mark.parametrize("rows, vocab, top_k", [(3, 3001, 8), (300, 20000, 5), (128, 37888, 0)])
def test_head_logprobs_around_residency(cuda, rows, vocab, top_k, size):
    """Hidden sizes on both sides of the largest whose rows stay in shared memory, in tiles of either width."""
    (a, sa, w, sw, b), t = head_case(rows, vocab, size, size + rows)
    got = scoring.head_logprobs(*cu((a, sa, w, sw, b)), t.cuda(), top_k=top_k, mask_token_id=9)
    pick = torch.tensor([0, 1, 2] if rows == 3 else [0, 1, 63, 64, 127] + ([128, 299] if rows > 128 else []))
    x = ref_linear(a[pick], sa[pick], w, sw, b)[1].float().double()
    some = got._replace(**{f: v[pick.cuda()] for f, v in got._asdict().items() if v is not None})
    check_scores(some, x, t[pick], top_k, 9)


def test_head_logprobs_rounds_once(cuda):
    """Up to hidden 1024 a logit is its exact value rounded once, where float64 would be halfway."""
    # 13325 * 80581 = 2^30 + 1, so that token 1's logit is 1 + 2^-24 + 2^-54
    a, w = torch.zeros((1, 128), dtype=torch.int8), torch.zeros((2, 128), dtype=torch.int8)
    a[0, :104], a[0, 104] = 127, 117
    w[1, :105] = 1
    assert int(a[0].long() @ w[1].long()) == 13325
    sa, sw, b = torch.tensor([80581 * 2.0 ** -54]), torch.ones(2), torch.ones(2)
    dev = cu((a, sa, w, sw, b))
    got = scoring.head_logprobs(*dev, top_k=2)
    assert got.top_ids.tolist() == [[1, 0]]
    assert scoring.linear_i8(*dev).tolist() == [[1.0, 1.0]]  # as the reference rounds it


# ------------------------------------------------------- use of the calls

def _calls():
    x, t = logits_case(37, 5003, torch.bfloat16, 0)
    x, t = x.cuda(), t.cuda()
    lin = cu(linear_case(45, 500, 256, 0))
    head, ht = head_case(45, 6000, 256, 0)
    head, ht = cu(head), ht.cuda()
    return [lambda: scoring.token_logprobs(x, t, top_k=6, mask_token_id=1),
            lambda: (scoring.linear_i8(*lin), scoring.linear_i8(*lin, out_dtype=torch.bfloat16)),
            lambda: scoring.head_logprobs(*head, ht, top_k=6, mask_token_id=5)]


def _flat(out):
    return [o.clone() for o in out if o is not None]


def _same(a, b):
    return all(torch.equal(p, q) for p, q in zip(a, b)) and len(a) == len(b)


def test_repeatable_across_streams(cuda):
    """The same bits every time, on several streams at once."""
    calls = _calls()
    first = [_flat(c()) for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for i in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append([_flat(c()) for c in calls])
    torch.cuda.synchronize()
    for g in got:
        assert all(_same(a, b) for a, b in zip(first, g))
    _lib.check_device_error()


def test_captured_graphs(cuda):
    """Two captured graphs of the calls, replayed in turn and together, follow their inputs."""
    x, t = logits_case(9, 5003, torch.float32, 1)
    x, t = x.cuda(), t.cuda()
    head, ht = head_case(45, 6000, 256, 3)
    head, ht = cu(head), ht.cuda()

    def both():
        return (*_flat(scoring.token_logprobs(x, t, top_k=3)), *_flat(scoring.head_logprobs(*head, ht, top_k=3)),
                scoring.linear_i8(*head))

    both()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = both()
        graphs.append((g, out))
    for i in range(3):
        x.copy_(logits_case(9, 5003, torch.float32, 10 + i)[0])
        head[0].copy_(head_case(45, 6000, 256, 20 + i)[0][0])
        torch.cuda.synchronize()
        want = [o.clone() for o in both()]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graphs[0][0].replay()
        with torch.cuda.stream(side):
            graphs[1][0].replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert _same(want, list(out))


def test_outputs_stay_in_bounds(cuda):
    """The C entry points write their outputs' own elements only."""
    x, t = logits_case(5, 777, torch.float32, 2)
    head, ht = head_case(5, 777, 64, 2)
    a, sa, w, sw, b = cu(head)
    x, t = x.cuda(), t.cuda()
    size = _lib.lib().dh_head_logprobs_workspace_size(5, 777, 3)
    ws = torch.full((size + 512,), 171, dtype=torch.uint8, device="cuda")
    for fused in (False, True):
        bufs = [torch.full((64,), 9.0, device="cuda") for _ in range(4)]
        ids = torch.full((64,), 9, dtype=torch.int32, device="cuda")
        lp, en, ls, tl = (v[16:] for v in bufs)
        tail = (t.data_ptr(), 8, 1, 3, lp.data_ptr(), en.data_ptr(), ls.data_ptr(), ids[16:].data_ptr(),
                tl.data_ptr())
        if fused:
            _lib.call("dh_head_logprobs_i8", a.data_ptr(), 64, sa.data_ptr(), w.data_ptr(), 64, sw.data_ptr(),
                      b.data_ptr(), 5, 64, 777, 3, *tail, ws.data_ptr(), size, _lib.stream_handle())
        else:
            _lib.call("dh_token_logprobs", x.data_ptr(), 0, 777, 5, 777, 3, *tail, _lib.stream_handle())
        for v, n in ((bufs[0], 5), (bufs[1], 5), (bufs[2], 5), (bufs[3], 15), (ids.float(), 15)):
            assert bool((v[:16] == 9).all()) and bool((v[16 + n:] == 9).all())
            assert bool((v[16:16 + n] != 9).all())
    assert bool((ws[size:] == 171).all())


def test_refusals(cuda):
    x, t = logits_case(4, 50, torch.float32, 0)
    x, t = x.cuda(), t.cuda()
    a, sa, w, sw, b = cu(linear_case(4, 50, 32, 0))
    bad = [
        lambda: scoring.token_logprobs(x.double(), t), lambda: scoring.token_logprobs(x[0], t),
        lambda: scoring.token_logprobs(x.T.contiguous().T, t), lambda: scoring.token_logprobs(x[:, :0], t),
        lambda: scoring.token_logprobs(x, t[:3]), lambda: scoring.token_logprobs(x, t.float()),
        lambda: scoring.token_logprobs(x, t.cpu()), lambda: scoring.token_logprobs(x, t, top_k=33),
        lambda: scoring.token_logprobs(x, t, top_k=-1), lambda: scoring.token_logprobs(x, t, mask_token_id=50),
        lambda: scoring.token_logprobs(x, t, mask_token_id=-1), lambda: scoring.token_logprobs(x, t[None, :, None]),
        lambda: scoring.linear_i8(a.float(), sa, w, sw), lambda: scoring.linear_i8(a, sa[:3], w, sw),
        lambda: scoring.linear_i8(a, sa, w[:, :16], sw), lambda: scoring.linear_i8(a, sa.double(), w, sw),
        lambda: scoring.linear_i8(a, sa, w, sw, b[:3]), lambda: scoring.linear_i8(a, sa, w, sw.cpu()),
        lambda: scoring.linear_i8(a, sa, w, sw, out_dtype=torch.float64),
        lambda: scoring.linear_i8(a, sa, w, sw, out=torch.empty(4, 51, device="cuda")),
        lambda: scoring.linear_i8(a, sa, w, sw, out=torch.empty(50, 4, device="cuda").T),
        lambda: scoring.linear_i8(a, sa, w, sw, out=torch.empty(1, 50, device="cuda").expand(4, 50)),
        lambda: scoring.linear_i8(a, sa, w, sw, out=torch.empty(4, 50, device="cuda"), out_dtype=torch.float16),
        lambda: scoring.linear_i8(a, sa, w, sw, out=torch.empty(4, 50)),
        lambda: scoring.linear_i8(a[:, :0], sa, w[:, :0], sw),
        lambda: scoring.head_logprobs(a, sa, w, sw, b, t, top_k=40),
        lambda: scoring.head_logprobs(a, sa, w, sw, b, t, mask_token_id=50),
        lambda: scoring.head_logprobs(a, sa, w[:0], sw[:0]), lambda: scoring.head_logprobs(a, sa, w[:, :16], sw),
    ]
    for f in bad:
        with pytest.raises(ValueError):
            f()
