"""Cases of the scoring operators: the scaled int8 matrix product, the log
probabilities of tokens over given logits, and the output head fused with
them.

``run`` computes an operator in its plain form (elementary torch operations)
while ``own`` is false and through ``diffusionhard_b200.scoring`` while it is
true; ``exact`` is the same result from the definitions in 64 bits.

Definitions.  Rows r, columns (tokens) c, sums over k:
  linear   y[r, c] = (sum_k a[r, k] w[c, k]) (a_scale[r] w_scale[c]) + bias[c]
  scores   of a row of logits x with the excluded token's logit -inf:
           logsumexp = log sum_c e^x[c],  p[c] = e^(x[c] - logsumexp),
           logprobs[t] = x[t] - logsumexp for each given token t (0 for a
           negative t, which stands for "no token"), entropy =
           -sum_c p[c] log p[c], and the top_k tokens of largest x, the lower
           id first among equals, with their log probabilities.  A row with
           nothing left: logsumexp and logprobs -inf, entropy 0, and -1 for
           every alternative that does not exist.
  head     the scores of the rows of linear(hidden, weight), whose logits are
           rounded to fp32 before they are ranked.
"""

import math

import torch

own = False

VOCAB, MASK = 50258, 50257
_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _linear(name, m, n, k, out, bias=True):
    return {"name": name, "op": "linear", "m": m, "n": n, "k": k, "out": out, "bias": bias}


def _logits(name, rows, vocab, dtype, targets, top_k, banned=False, pad=0, mask=MASK):
    return {"name": name, "op": "logits", "rows": rows, "vocab": vocab, "dtype": dtype, "targets": targets,
            "top_k": top_k, "banned": banned, "pad": pad, "mask": mask}


def _head(name, rows, vocab, hidden, targets, top_k, mask=MASK):
    return {"name": name, "op": "head", "rows": rows, "vocab": vocab, "hidden": hidden, "targets": targets,
            "top_k": top_k, "mask": mask}


def listed():
    return [
        # the QKV projection of one position: latency alone
        _linear("linear one row", 1, 2304, 768, "f32"),
        # MLP-down of one active 32-position block of a session
        _linear("linear block", 32, 768, 3072, "bf16", bias=False),
        # fp32 logits of the selected rows of a canvas (row pitch not a multiple of 16 bytes)
        _linear("linear selected logits", 512, VOCAB, 768, "f32"),
        # MLP-up of a batch of 32 canvases of 1024 positions
        _linear("linear batch", 32768, 3072, 768, "bf16"),
        # one position's logits, with alternatives for a confidence display
        _logits("logits one row", 1, VOCAB, "f32", 1, 8),
        # the rows revealed at one transition of a batch
        _logits("logits selected", 512, VOCAB, "f32", 1, 5),
        # bf16 logits of another model's four canvases, where equal values abound
        _logits("logits bf16", 4096, VOCAB, "bf16", 1, 8),
        # answer choices under a grammar that bans tokens, rows inside a wider buffer
        _logits("logits choices banned", 333, 32001, "f16", 4, 20, banned=True, pad=7, mask=-1),
        # perplexity of a whole batch: no alternatives
        _logits("logits canvas", 16384, VOCAB, "f32", 1, 0),
        # confidence of one active block, logits never stored
        _head("head block", 32, VOCAB, 768, 1, 8),
        # an odd number of selected rows
        _head("head selected", 1001, VOCAB, 768, 1, 1),
        # every position of a batch of 32 canvases of 1024 positions
        _head("head canvas", 32768, VOCAB, 768, 1, 5),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["linear", "logits", "head"])
    if op == "linear":
        while True:
            m, n, k = _log_int(rng, 1, 32768), _log_int(rng, 64, 51000), 16 * _log_int(rng, 4, 256)
            if 2 * m * n * k <= 1.5e11 and m * n <= 1e8:
                break
        c = _linear("", m, n, k, rng.choice(["f32", "bf16", "f16"]), rng.random() < 0.7)
    elif op == "logits":
        while True:
            rows, vocab = _log_int(rng, 1, 16384), _log_int(rng, 500, 131072)
            if rows * vocab <= 8e8:
                break
        c = _logits("", rows, vocab, rng.choice(["f32", "bf16", "f16"]), rng.choice([1, 1, 1, 4, 7]),
                    rng.choice([0, 1, 5, 8, 20, 32]), rng.random() < 0.3, rng.choice([0, 0, 1, 7, 64]),
                    rng.choice([-1, vocab - 1, rng.randrange(vocab)]))
    else:
        rows, vocab = _log_int(rng, 1, 8192), _log_int(rng, 2000, 65536)
        c = _head("", rows, vocab, 16 * _log_int(rng, 8, 96), rng.choice([1, 1, 4]), rng.choice([0, 1, 3, 5, 8]),
                  rng.choice([-1, vocab - 1, rng.randrange(vocab)]))
    del c["name"]
    return c


def _int8(shape, sigma, gen):
    # quantised rows: a bell with its largest values at the ends of the range
    return (torch.randn(shape, generator=gen, device="cuda") * sigma).round_().clamp_(-127, 127).to(torch.int8)


def _tokens(rows, count, vocab, gen):
    # one token in 16 is absent (a position that is not scored)
    t = torch.randint(0, vocab, (rows, count), generator=gen, device="cuda")
    return torch.where(torch.rand(rows, count, generator=gen, device="cuda") < 1 / 16, torch.full_like(t, -1), t)


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)

    def uniform(n, low, high):
        return torch.rand(n, generator=gen, device="cuda") * (high - low) + low

    s = dict(case)
    if case["op"] in ("linear", "head"):
        if case["op"] == "linear":
            rows, n, k, bias = case["m"], case["n"], case["k"], case["bias"]
        else:
            rows, n, k, bias = case["rows"], case["vocab"], case["hidden"], True
        s["a"], s["w"] = _int8((rows, k), 38, gen), _int8((n, k), 40, gen)
        # products of about 1 (a linear layer's output) to 4 (peaked logits)
        s["a_scale"] = uniform(rows, 0.5, 2.0) * 0.02
        s["w_scale"] = uniform(n, 0.7, 1.4) * (0.03 / math.sqrt(k))
        s["bias"] = torch.randn(n, generator=gen, device="cuda") * 0.5 if bias else None
    else:
        rows, vocab, pad = case["rows"], case["vocab"], case["pad"]
        x = torch.empty(rows, vocab + pad, device="cuda")
        x.normal_(generator=gen)
        x.mul_(uniform(rows, 0.5, 3.0)[:, None])
        if case["banned"]:
            # a third of the tokens, all of them in one row and all but one in another
            x.masked_fill_(torch.rand(rows, vocab + pad, generator=gen, device="cuda") < 1 / 3, -math.inf)
            x[rows // 2] = -math.inf
            x[0, 1:] = -math.inf
        s["x"] = x.to(_TYPES[case["dtype"]])[:, :vocab]
    if case["op"] != "linear":
        t = _tokens(rows, case["targets"], case["vocab"], gen)
        s["t"] = t[:, 0].contiguous() if case["targets"] == 1 else t
    return s


def _product(a, w):
    # integer sums below 2^24 are exact in fp32; longer ones take 64 bits
    t = torch.float32 if a.shape[1] * 127 * 127 < 2 ** 24 else torch.float64
    return (a.to(t) @ w.to(t).T).double()


def _plain_linear(a, a_scale, w, w_scale, bias):
    y = _product(a, w) * (a_scale[:, None] * w_scale[None, :]).double()
    return (y if bias is None else y + bias.double()).float()


def _plain_scores(x, t, mask, top_k):
    """Scores of fp32 logits x [rows, vocab], which it may write."""
    if mask >= 0:
        x[:, mask] = -math.inf
    vocab = x.shape[1]
    top = x.amax(1, keepdim=True)
    empty = top == -math.inf
    base = torch.where(empty, torch.zeros_like(top), top)
    d = x - base
    e = torch.exp(d)
    s = e.sum(1, keepdim=True)
    log_s = torch.log(s)
    entropy = log_s - torch.where(e > 0, e * d, torch.zeros_like(e)).sum(1, keepdim=True) / s
    at = t if t.dim() == 2 else t[:, None]
    lp = (x.gather(1, at.clamp(0, vocab - 1)) - base) - log_s
    lp = torch.where(empty, torch.full_like(lp, -math.inf), lp)
    lp = torch.where(at < 0, torch.zeros_like(lp), lp)
    out = {"logprobs": lp.reshape(t.shape), "entropy": torch.where(empty, torch.zeros_like(s), entropy)[:, 0],
           "logsumexp": (base + log_s)[:, 0]}
    if top_k:
        # one 64-bit key a token, (logit, lower id first), so that no two are equal
        bits = (x + 0.0).view(torch.int32).long()
        key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits) * (1 << 32)
        key += vocab - 1 - torch.arange(vocab, device=x.device)
        ids = torch.topk(key, min(top_k, vocab), dim=1).indices
        v = x.gather(1, ids)
        gone = v == -math.inf
        out["top_ids"] = torch.where(gone, torch.full_like(ids, -1), ids).int()
        out["top_logprobs"] = torch.where(gone, v, (v - base) - log_s)
    return out


def run(state):
    s = state
    if own:
        from diffusionhard_b200 import scoring

        if s["op"] == "linear":
            return scoring.linear_i8(s["a"], s["a_scale"], s["w"], s["w_scale"], s["bias"],
                                     out_dtype=_TYPES[s["out"]])
        mask = None if s["mask"] < 0 else s["mask"]
        if s["op"] == "logits":
            r = scoring.token_logprobs(s["x"], s["t"], top_k=s["top_k"], mask_token_id=mask)
        else:
            r = scoring.head_logprobs(s["a"], s["a_scale"], s["w"], s["w_scale"], s["bias"], s["t"],
                                      top_k=s["top_k"], mask_token_id=mask)
        out = {"logprobs": r.logprobs, "entropy": r.entropy, "logsumexp": r.logsumexp}
        if s["top_k"]:
            out["top_ids"], out["top_logprobs"] = r.top_ids, r.top_logprobs
        return out
    if s["op"] == "linear":
        return _plain_linear(s["a"], s["a_scale"], s["w"], s["w_scale"], s["bias"]).to(_TYPES[s["out"]])
    if s["op"] == "logits":
        x = s["x"].to(torch.float32, copy=True)
    else:
        x = _plain_linear(s["a"], s["a_scale"], s["w"], s["w_scale"], s["bias"])
    return _plain_scores(x, s["t"], s["mask"], s["top_k"])


def work(case):
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        out = m * n * (4 if case["out"] == "f32" else 2)
        return {"bytes": m * k + n * k + 4 * (m + n) + (4 * n if case["bias"] else 0) + out, "flops": 2 * m * n * k}
    rows, vocab = case["rows"], case["vocab"]
    small = rows * (case["targets"] * (8 + 4) + 4 + 4 + case["top_k"] * 8)
    if case["op"] == "logits":
        # subtraction, exponential, two sums and the product of the entropy
        return {"bytes": rows * vocab * (4 if case["dtype"] == "f32" else 2) + small, "flops": 5 * rows * vocab}
    k = case["hidden"]
    return {"bytes": rows * k + vocab * k + 4 * rows + 8 * vocab + small, "flops": 2 * rows * vocab * k}


def _exact_scores(x, t, mask, top_k):
    """Scores of logits x [rows, vocab] in 64 bits, ranked as rounded to fp32."""
    if mask >= 0:
        x = x.index_fill(1, torch.tensor([mask], device=x.device), -math.inf)
    empty = torch.isinf(x).all(1) & (x < 0).all(1)
    lse = torch.logsumexp(x, 1)
    logp = x - torch.where(empty, torch.zeros_like(lse), lse)[:, None]
    out = {"logprobs": torch.where(t < 0, torch.zeros((), device=x.device, dtype=x.dtype),
                                   logp.gather(1, t.reshape(len(t), -1).clamp(min=0)).reshape(t.shape)),
           "logsumexp": lse}
    if top_k:
        ids = torch.sort(x.float(), dim=1, descending=True, stable=True).indices[:, :top_k]
        out["top_logprobs"] = logp.gather(1, ids)
        out["top_ids"] = ids.masked_fill(out["top_logprobs"] == -math.inf, -1).int()
    out["entropy"] = torch.special.entr(logp.exp()).sum(1)
    return out


def exact(case, seed):
    s = prepare(case, seed)

    def product(rows):
        y = torch.einsum("rk,ck->rc", s["a"][rows].double(), s["w"].double())
        y *= s["a_scale"][rows].double()[:, None]
        y *= s["w_scale"].double()[None, :]
        return y if s["bias"] is None else y + s["bias"].double()

    if case["op"] == "linear":
        return product(slice(None))
    parts = []
    for at in range(0, case["rows"], 2048):  # 64-bit rows of a part at a time
        rows = slice(at, min(case["rows"], at + 2048))
        x = s["x"][rows].double() if case["op"] == "logits" else product(rows)
        parts.append(_exact_scores(x, s["t"][rows], case["mask"], case["top_k"]))
    return {k: torch.cat([p[k] for p in parts]) for k in parts[0]}
