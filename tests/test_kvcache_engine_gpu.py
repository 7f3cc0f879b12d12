"""8-bit and shared K/V inside the engine: sessions, prefix-conditioned generation."""

import pytest

from diffusionhard_b200 import _lib
from diffusionhard_b200.engine import MDLMEngine
from diffusionhard_b200.model import MDLMConfig, build_quantized
from diffusionhard_b200.prefix import PrefixConditionedGenerator
from diffusionhard_b200.session import BlockCausalSession, evaluate_two_turn_mdlm_session

pytestmark = pytest.mark.gpu

SMALL = MDLMConfig(vocab_size=1000, mask_token_id=999, blocks=2)


@pytest.fixture(scope="module")
def model():
    return build_quantized(SMALL, seed=0)


def _ids(torch, rows, n, seed):
    return torch.randint(0, 999, (rows, n), generator=torch.Generator().manual_seed(seed))


def _off(a, b):
    return float((a - b).norm() / b.norm())


@pytest.mark.parametrize("sizes", [[64, 32], [32, 32, 96], [256, 32, 224]])
def test_session_in_8_bits(cuda, model, sizes):
    """Block forwards over 8-bit K/V against 16-bit ones: a code is off by at most
    1/254 of its row's largest value, so the residual stream by a few thousandths."""
    torch = cuda
    total = sum(sizes)
    ids = _ids(torch, 3, total, 1)
    sessions = [BlockCausalSession(model, 3, total, int8_kv=i8) for i8 in (False, True)]
    at = 0
    for n in sizes:
        x = [s.append(ids[:, at:at + n]).x.clone() for s in sessions]
        assert _off(x[1], x[0]) < 1e-2 and not torch.equal(x[0], x[1])
        at += n
    assert sessions[1].kv_bytes() == SMALL.blocks * 3 * total * 12 * 136
    _lib.check_device_error()


def test_session_generation_in_8_bits(cuda, model):
    """Over retained K/V and with every block recomputed: the same tokens."""
    torch = cuda
    for batch in (1, 2):
        s = BlockCausalSession(model, batch, 160, int8_kv=True)
        s.append(_ids(torch, batch, 64, 2))
        a, meta, _, _ = s.generate(32, steps=16, seed=5, recompute=True)
        b, meta_b, _, _ = s.generate(32, steps=16, seed=5)
        assert torch.equal(a, b) and meta == meta_b
        assert not (b == SMALL.mask_token_id).any()
        s.append(b)
        s.truncate(64)
        s.append(b)
        c, _, _, _ = s.generate(64, steps=8, seed=6)
        assert not (c == SMALL.mask_token_id).any()
    _lib.check_device_error()


def test_session_generation_in_a_large_cache(cuda, model):
    """The same where lengths are a small part of the cache, of which calls show no more,
    and as in a cache that has no more."""
    torch = cuda
    outs = []
    for capacity in (1024, 640):
        s = BlockCausalSession(model, 2, capacity, int8_kv=True)
        s.append(_ids(torch, 2, 64, 2))
        for n in (32, 480):
            a, _, _, _ = s.generate(n, steps=8, seed=5, recompute=True)
            b, _, _, _ = s.generate(n, steps=8, seed=5)
            assert torch.equal(a, b)
            s.append(b)
            outs.append(b)
    assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[3])
    _lib.check_device_error()


def test_two_turns_in_8_bits(cuda, model):
    r = evaluate_two_turn_mdlm_session(quantized=model, samples=2, steps=16, int8_kv=True)
    assert r["aggregate"]["exact_turn_1_sequences"] == r["aggregate"]["exact_turn_2_sequences"] == 2
    assert r["kv_cache"] == "int8"
    other = evaluate_two_turn_mdlm_session(quantized=model, samples=1, steps=16)
    assert r["aggregate"]["final_session_kv_mib"] * 256 == other["aggregate"]["final_session_kv_mib"] * 136


@pytest.mark.parametrize("int8_kv", [False, True])
@pytest.mark.parametrize("batch, prefixes, P, S", [(4, 1, 64, 32), (4, 2, 96, 160), (3, 3, 32, 64), (2, 1, 512, 512)])
def test_shared_prefix_forward(cuda, model, int8_kv, batch, prefixes, P, S):
    """A suffix forward behind prefixes held once against one behind a copy of its
    prefix for each sequence."""
    torch = cuda
    prefix, suffix = _ids(torch, prefixes, P, 3), _ids(torch, batch, S, 4)
    suffix[:, ::3] = SMALL.mask_token_id
    plain = PrefixConditionedGenerator(model, batch, P, S)
    shared = PrefixConditionedGenerator(model, batch, P, S, prefixes=prefixes, int8_kv=int8_kv)
    plain.set_prefix(prefix.repeat_interleave(batch // prefixes, 0))
    shared.set_prefix(prefix)
    for g in (plain, shared):
        g.suffix.tokens.copy_(suffix.reshape(-1).to(torch.int32))
        g.suffix.forward()
    assert _off(shared.suffix.x, plain.suffix.x) < 1e-2
    # the 16-bit prefixes are the same numbers, held once
    if not int8_kv:
        for (k, vt), (pk, pvt) in zip(shared.kv, plain.kv):
            assert torch.equal(k, pk[::batch // prefixes, :, :P]) and torch.equal(vt, pvt[::batch // prefixes, :, :, :P])
    _lib.check_device_error()


@pytest.mark.parametrize("int8_kv", [False, True])
@pytest.mark.parametrize("steps, graph", [(8, False), (40, True)])
def test_shared_prefix_generation(cuda, model, int8_kv, steps, graph):
    """One prefix for four sequences gives the tokens that four copies of it give;
    packed forwards (steps = 40, one prefix) and graphs among them.  With 128 rows a
    sequence both walk the same keys in the same tiles."""
    torch = cuda
    prefix, masked = _ids(torch, 1, 64, 5), torch.full((4, 128), SMALL.mask_token_id)
    outs = []
    for prefixes in (1, 4):
        gen = PrefixConditionedGenerator(model, 4, 64, 128, prefixes=prefixes, int8_kv=int8_kv)
        for _ in range(2):
            out, meta = gen.generate(prefix.expand(prefixes, -1), masked, steps=steps, seed=7, graph=graph)
        assert meta["all_tokens_committed"] and meta["prefix_forwards"] == 2
        outs.append(out.clone())
    assert torch.equal(outs[0], outs[1])
    _lib.check_device_error()


def test_refusals(cuda, model):
    with pytest.raises(ValueError, match="do not divide"):
        PrefixConditionedGenerator(model, 4, 32, 32, prefixes=3)
    with pytest.raises(ValueError, match="number of prefixes"):
        PrefixConditionedGenerator(model, 4, 32, 32, int8_kv=True)
    gen = PrefixConditionedGenerator(model, 4, 32, 32, prefixes=2)
    with pytest.raises(ValueError, match="prefix_ids"):
        gen.set_prefix(_ids(cuda, 4, 32, 1))
    with pytest.raises(ValueError, match="drift"):
        gen.drift_report(_ids(cuda, 2, 32, 1), _ids(cuda, 4, 32, 1))
    for int8_kv in (False, True):
        gen = PrefixConditionedGenerator(model, 4, 32, 32, prefixes=2, int8_kv=int8_kv)
        with pytest.raises(ValueError, match="dh_sample_loop"):
            gen.suffix.generate(cuda.full((4, 32), SMALL.mask_token_id), steps=4, native=True)
    gen = PrefixConditionedGenerator(model, 4, 32, 32, prefixes=2)
    with pytest.raises(ValueError, match="int8_kv"):
        MDLMEngine(model, 1, 64, int8_kv=[])
    with pytest.raises(ValueError, match="prefix_kv"):
        MDLMEngine(model, 1, 64, prefix_kv=gen.kv)


def _captured_kernels(torch, enqueue):
    from cuda.bindings import runtime as rt

    g = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(g):
        enqueue()
    graph = rt.cudaGraph_t(init_value=g.raw_cuda_graph())
    err, _, count = rt.cudaGraphGetNodes(graph, 0)
    assert err == rt.cudaError_t.cudaSuccess
    err, nodes, count = rt.cudaGraphGetNodes(graph, count)
    assert err == rt.cudaError_t.cudaSuccess
    kinds = [rt.cudaGraphNodeGetType(node)[1] for node in nodes[:count]]
    return sum(kind == rt.cudaGraphNodeType.cudaGraphNodeTypeKernel for kind in kinds)


@pytest.mark.parametrize("make", [
    lambda m: BlockCausalSession(m, 8, 1024, int8_kv=True).engine(960, 32),
    lambda m: BlockCausalSession(m, 1, 1024, int8_kv=True).engine(0, 64),
    lambda m: BlockCausalSession(m, 32, 1024, int8_kv=True).engine(0, 1024),
    lambda m: BlockCausalSession(m, 2, 256).engine(128, 32),
    lambda m: PrefixConditionedGenerator(m, 4, 512, 32, prefixes=1).suffix,
    lambda m: PrefixConditionedGenerator(m, 4, 512, 512, prefixes=2, int8_kv=True).suffix,
    lambda m: PrefixConditionedGenerator(m, 4, 512, 512, prefixes=4).suffix,
    lambda m: PrefixConditionedGenerator(m, 4, 512, 512).suffix,
])
def test_launch_count_is_the_captured_kernel_count(cuda, model, make):
    """launches_per_forward against the kernel nodes of a captured forward."""
    eng = make(model)
    eng.tokens.zero_()
    eng.forward()
    cuda.cuda.synchronize()
    assert _captured_kernels(cuda, eng.forward) == eng.launches_per_forward
    _lib.check_device_error()
