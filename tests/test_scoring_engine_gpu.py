"""The scoring operators as the engine uses them: logits, scores of a forward,
and the scores of a canvas."""

import math

import pytest
import torch

from diffusionhard_b200 import _lib, api, scoring
from diffusionhard_b200.engine import MDLMEngine
from diffusionhard_b200.model import MDLMConfig, build_quantized

pytestmark = pytest.mark.gpu
VOCAB, MASK = 1003, 1002
U = 2.0 ** -24


@pytest.fixture(scope="module")
def engine(cuda):
    eng = MDLMEngine(build_quantized(MDLMConfig(vocab_size=VOCAB, mask_token_id=MASK, blocks=2), seed=0), 3, 64, "cuda")
    g = torch.Generator().manual_seed(3)
    ids = torch.randint(0, MASK, (3, 64), generator=g)
    ids[torch.rand(3, 64, generator=g) < 0.4] = MASK
    eng.forward(ids.view(-1).to("cuda", torch.int32))
    eng.ids = ids
    return eng


def reference(engine):
    """fp32 logits by the int32 accumulators and float64, and their log-softmax in float64."""
    hq, hs = engine.final_hidden_q()
    h = engine.head
    acc = torch.empty((engine.M, VOCAB), dtype=torch.int32, device="cuda")
    _lib.call("dh_gemm_i8_s32", hq.data_ptr(), 768, h.w.data_ptr(), 768, acc.data_ptr(), VOCAB, engine.M, VOCAB, 768,
              _lib.stream_handle())
    logits = (acc.double() * (hs[:, None] * h.w_scale[None, :]).double() + h.bias.double()).float()
    x = logits.double()
    x[:, MASK] = -math.inf
    return logits, torch.log_softmax(x, 1)


def close(got, want):
    # 1003 logits of magnitude below 16: chains of 1003 / 64 + 64 additions, twice
    # the softmax mean of |x - m| (below 16), then fp32 values of magnitude below 16
    # (the mask token's are -inf on both sides)
    return bool(((got.double() == want) | ((got.double() - want).abs() <= (16 + 64 + 64 + 64) * U)).all())


def test_logits_keep_their_bits(engine):
    logits, _ = reference(engine)
    assert torch.equal(engine.logits().view(-1, VOCAB), logits)


def test_selected_logits_keep_their_bits(cuda):
    eng = MDLMEngine(build_quantized(MDLMConfig(vocab_size=VOCAB, mask_token_id=MASK, blocks=1), seed=1), 1, 32, "cuda")
    ids = torch.randint(0, VOCAB, (1, 32), generator=torch.Generator().manual_seed(0))
    rows = torch.tensor([31, 0, 7, 7])
    got = eng.selected_logits(ids, rows)
    assert torch.equal(got, eng.logits().view(32, VOCAB)[rows.cuda()])


def test_score_of_a_forward(engine):
    _, lp = reference(engine)
    t = torch.randint(0, VOCAB, (engine.M, 2), generator=torch.Generator().manual_seed(4)).cuda()
    t[5, 1] = MASK
    t[6, 0] = -1
    r = engine.score(t, top_k=4)
    want = lp.gather(1, t.clamp(min=0))
    assert float(r.logprobs[5, 1]) == -math.inf and float(r.logprobs[6, 0]) == 0.0
    keep = torch.ones_like(t, dtype=torch.bool)
    keep[5, 1] = keep[6, 0] = False
    assert close(r.logprobs[keep], want[keep])
    top, ids = torch.sort(lp, dim=1, descending=True, stable=True)
    assert torch.equal(r.top_ids.long(), ids[:, :4])
    assert close(r.top_logprobs, top[:, :4])
    p = lp.exp()
    ent = torch.special.entr(p).sum(1)
    assert bool(((r.entropy.double() - ent).abs() <= 2 * (1 + 7 + 4) * 208 * U).all())
    # selected rows in any order, twice the same, none
    rows = torch.tensor([100, 3, 3, 191, 0])
    s = engine.score(t[rows.cuda()], rows=rows, top_k=4)
    for a, b in zip(s, r):
        assert torch.equal(a, b[rows.cuda()])
    assert engine.score(rows=torch.tensor([], dtype=torch.int64), top_k=2).top_ids.shape == (0, 2)


def test_scores_and_their_two_steps(engine):
    """Forward, logits and their scores, and the fused head agree."""
    x = engine.logits().view(-1, VOCAB)
    t = x.argmax(1)
    a = engine.score(t, top_k=8)
    b = scoring.token_logprobs(x, t, top_k=8, mask_token_id=MASK)
    assert torch.equal(a.top_ids, b.top_ids)
    for p, q in ((a.logprobs, b.logprobs), (a.entropy, b.entropy), (a.logsumexp, b.logsumexp),
                 (a.top_logprobs, b.top_logprobs)):
        torch.testing.assert_close(p, q, rtol=0, atol=24 * 208 * U)


def test_score_captured(engine):
    """A captured forward and score follow the canvas."""
    tokens = engine.ids.view(-1).to("cuda", torch.int32)
    t = torch.zeros(engine.M, dtype=torch.int64, device="cuda")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        engine.forward(tokens)
        engine.score(t, top_k=3)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        engine.forward(tokens)
        out = engine.score(t, top_k=3)
    for seed in (0, 1):
        tokens.copy_(torch.randint(0, VOCAB, (engine.M,), generator=torch.Generator().manual_seed(seed)))
        g.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in out]
        engine.forward(tokens)
        assert all(torch.equal(p, q) for p, q in zip(got, engine.score(t, top_k=3)))
    engine.forward(engine.ids.view(-1).to("cuda", torch.int32))
    _lib.check_device_error()


def test_score_tokens(engine):
    targets = torch.randint(0, MASK, (3, 64), generator=torch.Generator().manual_seed(5))
    r = api.score_tokens(engine, engine.ids, targets, mask_token_id=MASK, top_k=2)
    assert r["logprobs"].device == engine.ids.device
    masked = engine.ids == MASK
    assert torch.equal(r["scored"], masked)
    _, lp = reference(engine)
    want = lp.cpu().view(3, 64, VOCAB).gather(2, targets[..., None])[..., 0]
    assert close(r["logprobs"][masked], want[masked])
    assert bool((r["logprobs"][~masked] == 0).all()) and bool((r["entropy"][~masked] == 0).all())
    assert bool((r["top_ids"][~masked] == -1).all()) and bool((r["top_ids"][masked] >= 0).all())
    assert torch.equal(r["sequence_logprobs"], r["logprobs"].sum(1))
    full = api.score_tokens(engine, engine.ids, targets, mask_token_id=MASK, every_position=True)
    assert bool(full["scored"].all()) and torch.equal(full["logprobs"][masked], r["logprobs"][masked])
    none = api.score_tokens(engine, targets, targets, mask_token_id=MASK, top_k=1)
    assert not bool(none["scored"].any()) and none["sequence_logprobs"].tolist() == [0.0] * 3
    engine.forward(engine.ids.view(-1).to("cuda", torch.int32))


def test_refusals(engine):
    t = torch.zeros(3, 64, dtype=torch.int64)
    with pytest.raises(ValueError, match="mask_token_id"):
        api.score_tokens(engine, t, t, mask_token_id=5)
    with pytest.raises(ValueError, match="must be"):
        api.score_tokens(engine, t[:2], t, mask_token_id=MASK)
    with pytest.raises(ValueError, match="rows"):
        engine.score(rows=torch.tensor([192]))
    with pytest.raises(ValueError, match="rows"):
        engine.score(rows=torch.zeros(193, dtype=torch.int64))
    sharded = MDLMEngine(engine.qm, 1, 32, "cuda")
    sharded.shard_head(0, 500)
    with pytest.raises(ValueError, match="sharded"):
        sharded.score()
    assert sharded.logits().shape == (1, 32, 500)


def test_rows_of_other_types(engine):
    """Rows are checked as they are given, not after they were narrowed."""
    for bad in (torch.tensor([2 ** 32]), torch.tensor([-2 ** 32 + 1]), torch.tensor([0.5]), torch.tensor([True])):
        with pytest.raises(ValueError, match="rows"):
            engine.score(rows=bad)
    a = engine.score(rows=torch.tensor([3, 5], dtype=torch.int32), top_k=2)
    assert torch.equal(a.top_ids, engine.score(rows=torch.tensor([3, 5]).cuda(), top_k=2).top_ids)


def test_score_wants_a_whole_forward(cuda):
    """Nothing is scored from a residual stream that no forward of the whole canvas left."""
    eng = MDLMEngine(build_quantized(MDLMConfig(vocab_size=VOCAB, mask_token_id=MASK, blocks=2), seed=0), 2, 32, "cuda")
    ids = torch.full((2, 32), MASK)
    tokens = ids.view(-1).to("cuda", torch.int32)
    t = torch.arange(64, device="cuda")

    def refused():
        for rows in (None, torch.tensor([1])):
            with pytest.raises(RuntimeError, match="forward"):
                eng.score(rows=rows)

    refused()
    eng.forward(tokens)
    want = eng.score(t, top_k=3)

    def generations():
        for native in (True, False):
            for compact in (True, False):
                for graph in (False, True):
                    eng.compact = compact
                    yield lambda: eng.generate(ids, steps=4, native=native, graph=graph)
        for graph in (False, True, True):
            yield lambda: api.run_event_driven_candidate_sampler(eng, ids, mask_token_id=MASK, steps=4, reveal_seed=1,
                                                                 graph=graph)
        yield lambda: eng.forward(tokens, run_rows=eng.fwd_rows.fill_(32))

    for generation in generations():
        generation()
        refused()
        eng.forward(tokens)
        assert all(torch.equal(p, q) for p, q in zip(want, eng.score(t, top_k=3)))
    eng.generate(ids, steps=4)
    generated = eng.tokens.view(2, 32).long()
    r = api.score_tokens(eng, generated, generated, mask_token_id=MASK, every_position=True)
    eng.forward(generated.view(-1).to(torch.int32))
    _, lp = reference_of(eng)
    assert close(r["logprobs"].view(-1), lp.gather(1, generated.view(-1, 1))[:, 0])
    with pytest.raises(ValueError, match="input_ids"):
        eng.generate(ids[:1], steps=4)
    eng.score(t)  # the refused generation ran nothing
    _lib.check_device_error()


def reference_of(eng):
    logits = eng.logits().view(-1, VOCAB)
    x = logits.double()
    x[:, MASK] = -math.inf
    return logits, torch.log_softmax(x, 1)


def test_score_tokens_far_ids(engine):
    """Ids past 32 bits are not taken for the tokens that their low bits spell."""
    targets = torch.randint(0, MASK, (3, 64), generator=torch.Generator().manual_seed(6))
    ids = engine.ids.clone()
    ids[0, :4] = torch.tensor([2 ** 32 + MASK, 2 ** 32 + 5, -2 ** 32 + 7, -1])
    r = api.score_tokens(engine, ids, targets, mask_token_id=MASK, top_k=1)
    assert torch.equal(r["scored"], ids == MASK)
    last = ids.clone()
    last[0, :4] = VOCAB - 1  # what an id outside the vocabulary is embedded as
    full = api.score_tokens(engine, ids, targets, mask_token_id=MASK, every_position=True)
    want = api.score_tokens(engine, last, targets, mask_token_id=MASK, every_position=True)
    assert torch.equal(full["logprobs"], want["logprobs"])
    far = targets.clone()
    far[0, 0], far[1, 1] = 2 ** 40, -2 ** 40
    r = api.score_tokens(engine, ids, far, mask_token_id=MASK, every_position=True)
    assert bool(torch.isnan(r["logprobs"][0, 0])) and float(r["logprobs"][1, 1]) == 0.0
    for dtype in (torch.uint8, torch.int16, torch.int32):
        small = engine.ids.clamp(max=200 if dtype == torch.uint8 else MASK)
        a = api.score_tokens(engine, small.to(dtype), targets, mask_token_id=MASK, every_position=True)
        b = api.score_tokens(engine, small, targets, mask_token_id=MASK, every_position=True)
        assert torch.equal(a["logprobs"], b["logprobs"])
    engine.forward(engine.ids.view(-1).to("cuda", torch.int32))
