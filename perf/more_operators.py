"""Cases of the K/V cache operators: storing K and V in 8 bits, reading them
back, attention over such a cache, and attention of a batch whose sequences
share a long prefix that is held once.

``run`` computes an operator in its plain form (elementary torch operations)
while ``own`` is false and through ``diffusionhard_b200.kvcache`` while it is
true; ``exact`` is the same result from the definitions in 64 bits.

Definitions, for the 64 values x of a position and head:
  store    scale = amax / 127 with amax = max |x| (0 below 2^-100, NaN if a
           value is not finite), code = rint(x / scale) within +-127 (0 where
           the scale is 0 or NaN); both quotients are rounded to fp32.
  read     x = code * scale, rounded to the type asked for.
  attend   s[i, j] = (q_i . k_j) / 8 over the keys j of the sequence: those of
           its group's prefix, if there is one, then its own; p = exp(s - max);
           o_i = sum_j p[i, j] v_j / sum_j p[i, j]; 0 where there is no key.
"""

import math

import torch

own = False

HEADS, DIM = 12, 64
_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _store(name, batch, rows, capacity, dtype="bf16", layout="heads", ragged=False, heads=HEADS):
    return {"name": name, "op": "store", "batch": batch, "rows": rows, "capacity": capacity, "dtype": dtype,
            "layout": layout, "ragged": ragged, "heads": heads}


def _read(name, batch, rows, start, capacity, dtype="bf16", heads=HEADS):
    return {"name": name, "op": "read", "batch": batch, "rows": rows, "start": start, "capacity": capacity,
            "dtype": dtype, "heads": heads}


def _attend(name, batch, queries, keys, kind="int8", heads=HEADS, kv_heads=HEADS, ragged=True, groups=0, prefix=0,
            dtype="bf16", layout="heads"):
    return {"name": name, "op": "attend", "batch": batch, "queries": queries, "keys": keys, "kind": kind,
            "heads": heads, "kv_heads": kv_heads, "ragged": ragged, "groups": groups, "prefix": prefix,
            "dtype": dtype, "layout": layout}


def listed():
    return [
        # one new position of one sequence: latency alone
        _store("store one position", 1, 1, 1024),
        # a block of every sequence of a serving batch, as its projection lays it
        # out (positions before heads), of ragged lengths at ragged places
        _store("store ragged blocks", 61, 129, 1024, dtype="f32", layout="tokens", ragged=True),
        # 32 canvases of 1024 positions, K and the transposed V of the QKV product
        _store("store canvases", 32, 1024, 1024, layout="engine"),
        # an odd piece of one sequence's cache, to extend or inspect it
        _read("read a piece", 1, 333, 101, 1024),
        # the caches of 32 canvases
        _read("read canvases", 32, 1024, 0, 1024),
        # one query over one sequence's canvas: latency alone
        _attend("attend one token", 1, 1, 1001),
        # the active 32-position block of 8 sessions over their retained keys
        _attend("attend active blocks", 8, 32, 1024),
        # single tokens over long caches of different lengths
        _attend("attend long caches", 16, 1, 32768),
        # every query of 32 canvases
        _attend("attend canvases", 32, 1024, 1024, ragged=False),
        # single tokens of 128 sequences behind one long prompt, 16-bit
        _attend("prefix single tokens", 128, 1, 320, kind="16-bit", groups=1, prefix=8191),
        # blocks behind two prompts, 8-bit, several query heads for each K/V head
        _attend("prefix grouped blocks", 24, 32, 1000, heads=16, kv_heads=4, groups=2, prefix=4000),
        # 128 generated halves of canvases behind one prompt, as the QKV product lays K and V out
        _attend("prefix canvases", 128, 512, 512, kind="16-bit", ragged=False, groups=1, prefix=512,
                layout="engine"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["store", "read", "attend", "attend", "attend"])
    if op in ("store", "read"):
        while True:
            batch, rows, heads = _log_int(rng, 1, 64), _log_int(rng, 1, 2000), rng.choice([1, 4, 12, 16])
            start = _log_int(rng, 1, 500) - 1
            capacity = rows + start + rng.choice([0, 1, 30, 100])
            if batch * capacity * heads <= 400000:
                break
        dtype = rng.choice(["bf16", "f16", "f32"])
        c = (_store("", batch, rows, capacity, dtype, rng.choice(["heads", "tokens", "engine"]), rng.random() < 0.5,
                    heads) if op == "store" else _read("", batch, rows, start, capacity, dtype, heads))
    else:
        while True:
            kv_heads, ratio = rng.choice([(12, 1), (12, 1), (4, 4), (2, 7), (1, 8), (3, 2)])
            heads = kv_heads * ratio
            batch, queries, keys = _log_int(rng, 1, 128), _log_int(rng, 1, 1024), _log_int(rng, 1, 32768)
            groups = rng.choice([0, 1, 1, 2, 4])
            prefix = _log_int(rng, 1, 16384) if groups else 0
            if groups:
                batch = -(-batch // groups) * groups
            pairs = batch * heads * queries * (keys + prefix)
            if pairs <= 4e8 and batch * kv_heads * keys <= 6.5e6 and groups * kv_heads * prefix <= 6.5e6:
                break
        kind = rng.choice(["int8", "16-bit"])
        c = _attend("", batch, queries, keys, kind, heads, kv_heads, rng.random() < 0.7, groups, prefix,
                    rng.choice(["bf16", "bf16", "f16"]),
                    rng.choice(["heads", "tokens", "engine"]) if kind == "16-bit" else "heads")
    del c["name"]
    return c


def _lengths(case):
    """Keys of each sequence: all of them, or from none to all."""
    n, most = case["batch"], case["keys"] if case["op"] == "attend" else case["rows"]
    if not case["ragged"]:
        return [most] * n
    return [0 if i % 7 == 3 else most - (i * 7919) % (most // 2 + 1) for i in range(n)]


def _starts(case):
    room = case["capacity"] - case["rows"]
    return [(i * 613) % (room + 1) if case["ragged"] else room // 2 for i in range(case["batch"])]


def _values(shape, gen, channels=False):
    """[n, heads, rows, 64] of a projection's output: rows of different sizes;
    for keys some channels stand out."""
    x = torch.randn(shape, generator=gen, device="cuda")
    x.mul_(torch.rand(shape[:3], generator=gen, device="cuda").mul_(1.5).add_(0.5)[..., None])
    if channels:
        wide = torch.rand((1, shape[1], 1, DIM), generator=gen, device="cuda") < 0.05
        x.mul_(torch.where(wide, 3.0, 1.0))
    return x


def _laid_out(x, layout):
    """The same values with the memory layout asked for."""
    if layout == "tokens":     # positions before heads
        return x.transpose(1, 2).contiguous().transpose(1, 2)
    if layout == "engine":     # positions contiguous: a transposed V
        return x.transpose(2, 3).contiguous().transpose(2, 3)
    return x.contiguous()


def _quantise(x):
    x = x.float()
    amax = x.abs().amax(-1)
    scale = torch.where(amax < 2.0 ** -100, torch.zeros_like(amax), amax / torch.full_like(amax, 127.0))
    scale = torch.where(torch.isfinite(amax), scale, torch.full_like(scale, math.nan))
    step = torch.where(scale > 0, scale, torch.ones_like(scale))[..., None].expand_as(x)
    code = torch.round(x / step).clamp(-127, 127)
    return torch.where((scale > 0)[..., None], code, torch.zeros_like(code)).to(torch.int8), scale


def _cache(n, heads, rows, gen):
    """An 8-bit cache as earlier calls have left it; its capacity is a multiple of 64."""
    capacity = (rows + 63) // 64 * 64
    c = {}
    for name in ("k", "v"):
        codes, scale = _quantise(_values((n, heads, capacity, DIM), gen, name == "k").bfloat16())
        c[name], c[name + "_scale"] = codes, scale
    return c


def _kv16(n, heads, rows, case, gen):
    t = _TYPES[case["dtype"]]
    k, v = (_values((n, heads, rows, DIM), gen, i == 0) for i in range(2))
    if case["layout"] == "engine":
        # (a row of the transposed V starts at a 16-byte boundary)
        padded = torch.zeros(n, heads, DIM, (rows + 7) // 8 * 8, dtype=torch.float16, device="cuda")
        padded[..., :rows] = v.transpose(2, 3)
        return k.to(t), padded.transpose(2, 3)[:, :, :rows]
    return _laid_out(k.to(t), case["layout"]), _laid_out(v.to(t), case["layout"])


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    s = dict(case)
    if case["op"] in ("store", "read"):
        s["cache"] = _cache(case["batch"], case["heads"], case["capacity"], gen)
        if case["op"] == "store":
            shape, t, layout = (case["batch"], case["heads"], case["rows"], DIM), _TYPES[case["dtype"]], case["layout"]
            x = [_values(shape, gen, True), _values(shape, gen)]
            # a position of zeros, as padding gives it
            x[0][:, :, case["rows"] // 2] = 0
            x[1][:, :, case["rows"] // 2] = 0
            s["k"] = _laid_out(x[0].to(t), "heads" if layout == "engine" else layout)
            s["v"] = _laid_out(x[1].to(torch.float16 if layout == "engine" else t), layout)
            s["start"] = torch.tensor(_starts(case), dtype=torch.int32, device="cuda")
            s["counts"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
        return s
    n, heads = case["batch"], case["heads"]
    q = _values((n, heads, case["queries"], DIM), gen)
    s["q"] = q.to(_TYPES[case["dtype"]])
    s["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
    if case["kind"] == "int8":
        s["own"] = _cache(n, case["kv_heads"], case["keys"], gen)
        s["prefix_kv"] = _cache(case["groups"], case["kv_heads"], case["prefix"], gen) if case["groups"] else None
    else:
        s["own"] = _kv16(n, case["kv_heads"], case["keys"], case, gen)
        s["prefix_kv"] = _kv16(case["groups"], case["kv_heads"], case["prefix"], case, gen) if case["groups"] else None
    return s


def _own_cache(kvcache, c):
    return kvcache.KVCacheI8(c["k"], c["k_scale"], c["v"], c["v_scale"])


def _run_own(s):
    from diffusionhard_b200 import kvcache

    if s["op"] == "store":
        cache = _own_cache(kvcache, s["cache"])
        if s["ragged"]:
            kvcache.write_kv(cache, s["k"], s["v"], s["start"], s["counts"])
        else:
            kvcache.write_kv(cache, s["k"], s["v"], (s["capacity"] - s["rows"]) // 2)
        return s["cache"]
    if s["op"] == "read":
        return kvcache.read_kv(_own_cache(kvcache, s["cache"]), s["start"], s["rows"], dtype=_TYPES[s["dtype"]])
    if s["kind"] == "int8":
        keys = _own_cache(kvcache, s["own"])
        prefix = _own_cache(kvcache, s["prefix_kv"]) if s["groups"] else None
    else:
        keys, prefix = s["own"], s["prefix_kv"]
    return kvcache.attend(s["q"], keys, s["lengths"] if s["ragged"] else s["keys"], prefix=prefix,
                          prefix_lengths=s["prefix"] if s["groups"] else None)


def _plain_store(s):
    c = s["cache"]
    at = torch.arange(c["k"].shape[2], device="cuda")[None, :] - s["start"][:, None].long()
    live = (at >= 0) & (at < s["counts"][:, None])  # [batch, capacity]
    at = at.clamp(0, s["rows"] - 1)[:, None, :].expand(-1, s["heads"], -1)
    live = live[:, None, :]
    for name in ("k", "v"):
        codes, scale = _quantise(s[name])
        codes = codes.gather(2, at[..., None].expand(-1, -1, -1, DIM))
        c[name].copy_(torch.where(live[..., None], codes, c[name]))
        c[name + "_scale"].copy_(torch.where(live, scale.gather(2, at), c[name + "_scale"]))
    return c


def _plain_kv(kv, kind, rows):
    if kind == "int8":
        k, v = (kv[n][:, :, :rows].float() * kv[n + "_scale"][:, :, :rows, None] for n in ("k", "v"))
        return k, v
    return kv[0].float(), kv[1].float()


def _plain_attend(s):
    n, kv_heads, queries = s["batch"], s["kv_heads"], s["queries"]
    rows = s["heads"] // kv_heads * queries
    q = s["q"].float().reshape(n, kv_heads, rows, DIM) * 0.125
    k, v = _plain_kv(s["own"], s["kind"], s["keys"])
    x = q @ k.transpose(2, 3)
    gone = torch.arange(s["keys"], device="cuda") >= s["lengths"][:, None]
    x.masked_fill_(gone[:, None, None, :], -math.inf)
    top = x.amax(-1, keepdim=True)
    if s["groups"]:
        # the queries of a group side by side over the one copy of its prefix
        g = s["groups"]
        pk, pv = _plain_kv(s["prefix_kv"], s["kind"], s["prefix"])
        side = q.reshape(g, n // g, kv_heads, rows, DIM).transpose(1, 2).reshape(g, kv_heads, n // g * rows, DIM)
        y = side @ pk.transpose(2, 3)
        back = lambda t: t.reshape(g, kv_heads, n // g, rows, -1).transpose(1, 2).reshape(n, kv_heads, rows, -1)  # noqa: E731
        there = lambda t: t.reshape(g, n // g, kv_heads, rows, 1).transpose(1, 2).reshape(g, kv_heads, -1, 1)  # noqa: E731
        top = torch.maximum(top, back(y.amax(-1, keepdim=True)))
        y = torch.exp(y - there(top))
    base = torch.where(top == -math.inf, torch.zeros_like(top), top)
    x = torch.exp(x - base)
    total, out = x.sum(-1, keepdim=True), x @ v
    if s["groups"]:
        total, out = total + back(y.sum(-1, keepdim=True)), out + back(y @ pv)
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    out = out.reshape(n, s["heads"], queries, DIM).transpose(1, 2).contiguous()
    return out.to(_TYPES[s["dtype"]])


def run(state):
    s = state
    if own:
        return _run_own(s)
    if s["op"] == "store":
        return _plain_store(s)
    if s["op"] == "read":
        at = slice(s["start"], s["start"] + s["rows"])
        c = s["cache"]
        return tuple((c[n][:, :, at].float() * c[n + "_scale"][:, :, at, None]).to(_TYPES[s["dtype"]])
                     for n in ("k", "v"))
    return _plain_attend(s)


def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2}[case["dtype"]]
    if case["op"] == "store":
        live = sum(_lengths(case)) * case["heads"]
        v_size = 2 if case["layout"] == "engine" else size
        # largest magnitude, quotient, rounding and bounds of each value
        return {"bytes": live * (DIM * (size + v_size) + 2 * (DIM + 4)), "flops": live * 2 * DIM * 5}
    if case["op"] == "read":
        live = case["batch"] * case["rows"] * case["heads"]
        return {"bytes": live * 2 * (DIM + 4 + DIM * size), "flops": live * 2 * DIM}
    lengths = _lengths(case)
    key_bytes = 2 * (DIM + 4) if case["kind"] == "int8" else 2 * DIM * 2
    keys = case["kv_heads"] * (sum(lengths) + case["groups"] * case["prefix"])
    pairs = case["heads"] * case["queries"] * sum(n + case["prefix"] for n in lengths)
    return {"bytes": 2 * case["batch"] * case["queries"] * case["heads"] * DIM * size + keys * key_bytes,
            "flops": 4 * DIM * pairs}


def _exact_rows(x):
    """Codes and scales of rows, each quotient in 64 bits and then rounded to
    fp32, as the definition has it."""
    x = x.double()
    peak = x.abs().max(-1).values
    scale = (peak / 127).float()
    scale[peak < 2.0 ** -100] = 0
    scale[~torch.isfinite(peak)] = math.nan
    code = (x / scale.double().unsqueeze(-1)).float().round().clamp(-127, 127)
    code[~(scale > 0)] = 0
    return code.to(torch.int8), scale


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "store":
        c, starts, counts = s["cache"], _starts(case), _lengths(case)
        for b in range(case["batch"]):
            to = slice(starts[b], starts[b] + counts[b])
            for n in ("k", "v"):
                c[n][b, :, to], c[n + "_scale"][b, :, to] = _exact_rows(s[n][b, :, :counts[b]])
        return {n: t.double() if n.endswith("scale") else t for n, t in c.items()}
    if case["op"] == "read":
        at = slice(s["start"], s["start"] + s["rows"])
        return tuple(torch.mul(s["cache"][n][:, :, at].double(),
                               s["cache"][n + "_scale"][:, :, at].double().unsqueeze(-1)) for n in ("k", "v"))

    def keys_of(kv, i, count):
        if case["kind"] == "int8":
            return [torch.mul(kv[n][i, :, :count].double(), kv[n + "_scale"][i, :, :count].double().unsqueeze(-1))
                    for n in ("k", "v")]
        return [t[i, :, :count].double() for t in kv]

    out = torch.zeros(case["batch"], case["queries"], case["heads"], DIM, dtype=torch.float64, device="cuda")
    ratio = case["heads"] // case["kv_heads"]
    for b, count in enumerate(_lengths(case)):
        k, v = keys_of(s["own"], b, count)
        if case["groups"]:
            pk, pv = keys_of(s["prefix_kv"], b * case["groups"] // case["batch"], case["prefix"])
            k, v = torch.cat([pk, k], 1), torch.cat([pv, v], 1)
        if k.shape[1] == 0:
            continue
        for h in range(case["heads"]):
            logits = torch.einsum("qd,kd->qk", s["q"][b, h].double(), k[h // ratio]) / math.sqrt(DIM)
            out[b, :, h] = torch.softmax(logits, -1) @ v[h // ratio]
    return out
