"""Several answers to one prompt: the forked cache, attention over the shared prompt and the draw, as the
model runs them and in captured graphs and streams."""
import pytest
import torch

from leanselect_amd import minicpm
from leanselect_amd.ops import (dense_attention_kvcache, kvcache_append, sample_logits,
                                shared_prefix_attention)

pytestmark = pytest.mark.gpu
DEV = "cuda"
D = 128


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _model(seed=3, **kw):
    cfg = minicpm.MiniCPMConfig(hidden_size=1024, num_hidden_layers=2, num_attention_heads=8, num_key_value_heads=2,
                                intermediate_size=2048, vocab_size=1000)
    return minicpm.MiniCPMLeanSelect(cfg, device=DEV, seed=seed, weight_std=0.05, **kw)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,length", [(1, 70), (5, 700), (20, 33)])
def test_answers_equal_prefills_of_the_same_tokens(dtype, n, length):
    """Each step's logits are those of prefilling the prompt and the answer so far (whose page budget holds
    every page), up to the model's 16-bit roundings, and the tokens are drawn from them."""
    model = _model(dtype=dtype)
    gen = torch.Generator(device=DEV).manual_seed(n)
    prompt = torch.randint(0, 1000, (length,), generator=gen, device=DEV, dtype=torch.int32)
    u = torch.rand(4, n, generator=gen, device=DEV)
    sampling = dict(temperature=0.8, top_k=100, top_p=0.95)
    tokens = model.generate(prompt, u, **sampling)
    assert tokens.shape == (n, 4) and tokens.dtype == torch.int32
    cache = model.new_cache(1, length)
    logits = model.prefill(prompt, cache=cache)
    before = cache.k.view(torch.int16).clone()
    fork = cache.fork(n, 3)
    assert torch.equal(tokens[:, 0], sample_logits(logits.expand(n, -1), u[0], **sampling))
    for step in range(1, 4):
        logits = model.decode_step(tokens[:, step - 1], fork)
        assert torch.equal(tokens[:, step], sample_logits(logits, u[step], **sampling))
        for b in {0, n // 2, n - 1}:
            want = model.prefill(torch.cat((prompt, tokens[b, :step])))[0].double()
            off = (logits[b].double() - want).norm() / want.norm()
            assert float(off) < 0.02, (step, b, float(off))
    assert torch.equal(cache.k.view(torch.int16), before) and fork.positions == [length + 3] * n


def test_answers_go_their_own_ways():
    model = _model()
    prompt = torch.arange(50, device=DEV, dtype=torch.int32)
    u = torch.rand(6, 8, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV)
    tokens = model.generate(prompt, u, temperature=1.5)
    assert len({tuple(t) for t in tokens.tolist()}) == 8
    again = model.generate(prompt, u[:, :1].contiguous(), temperature=1.5)
    assert torch.equal(tokens[0, :1], again[0, :1])
    greedy = model.generate(prompt, u, temperature=0.0)
    assert bool((greedy == greedy[0]).all())
    assert torch.equal(model.generate(prompt, u[:1], temperature=1.5), tokens[:, :1])
    with pytest.raises(ValueError, match="u must"):
        model.generate(prompt, u[0])


def test_quantized_weights_generate():
    model = _model().quantize_weights()
    prompt = torch.arange(90, device=DEV, dtype=torch.int32)
    tokens = model.generate(prompt, torch.rand(3, 4, device=DEV), top_k=20)
    assert tokens.shape == (4, 3) and bool(((tokens >= 0) & (tokens < 1000)).all())


def _step_state(B, P, capacity, seed, dtype=torch.bfloat16, H=8, G=2, vocab=5000):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def r(*shape):
        return torch.randn(*shape, generator=g, device=DEV).to(dtype)

    return dict(q=r(B, H, D), kp=r(P, G, D), vp=r(P, G, D), k=r(B, capacity, G, D), v=r(B, capacity, G, D),
                kn=r(B, G, D), vn=r(B, G, D), lens=_i32([3 + b for b in range(B)]), cu=_i32(list(range(B + 1))),
                logits=3 * r(B, vocab).float(), u=torch.rand(B, generator=g, device=DEV))


def _step(st, longest):
    B = st["q"].shape[0]
    host = [3 + b for b in range(B)]  # only checked
    kvcache_append(st["k"], st["v"], st["lens"], st["kn"], st["vn"], st["cu"], cache_seqlens_host=host,
                   cu_seqlens_new_host=list(range(B + 1)))
    after = st["lens"] + 1
    out = shared_prefix_attention(st["q"], st["kp"], st["vp"], st["k"], st["v"], after, st["cu"], longest, causal=True)
    own, lse = dense_attention_kvcache(st["q"], st["k"], st["v"], after, st["cu"], longest, softcap=20.0,
                                       window=(30, -1), return_lse=True)
    token, lp = sample_logits(st["logits"], st["u"], temperature=0.7, top_p=0.9, return_logprob=True)
    return out, own, lse, token, lp


def test_two_captured_steps_replayed():
    """Two graphs over states of their own, replayed in turn with lengths advanced on the device and eager
    calls in between, against eager runs on copies."""
    longest = 64
    states = [_step_state(5, 900, 64, 1), _step_state(9, 333, 64, 2)]
    copies = [{n: t.clone() for n, t in st.items()} for st in states]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for st in copies:  # warm up on copies
            _step({n: t.clone() for n, t in st.items()}, longest)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for st in states:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_step(st, longest))
        graphs.append(graph)
    gen = torch.Generator(device=DEV).manual_seed(4)
    for replay in range(4):
        for i in (0, 1) if replay % 2 else (1, 0):
            for st in (states[i], copies[i]):
                if st is states[i]:
                    new = {n: torch.randn(st[n].shape, generator=gen, device=DEV).to(st[n].dtype) for n in ("q", "kn", "vn")}
                    u = torch.rand(st["u"].shape, generator=gen, device=DEV)
                for n, t in new.items():
                    st[n].copy_(t)
                st["u"].copy_(u)
            graphs[i].replay()
            want = _step(copies[i], longest)
            torch.cuda.synchronize()
            for a, b in zip(outs[i], want):
                assert torch.equal(a, b), (replay, i)
            assert torch.equal(states[i]["k"], copies[i]["k"])
            states[i]["lens"].add_(1)
            copies[i]["lens"].add_(1)


def test_two_streams_at_once():
    """Calls on two streams, whose workspaces are their own, give what they give one after the other."""
    states = [_step_state(16, 4000, 64, 5), _step_state(3, 2000, 64, 6)]
    want = [_step({n: t.clone() for n, t in st.items()}, 64) for st in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    copies = [[{n: t.clone() for n, t in st.items()} for _ in range(5)] for st in states]
    torch.cuda.synchronize()
    got = [[], []]
    for k in range(5):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(_step(copies[i][k], 64))
    torch.cuda.synchronize()
    for i in range(2):
        for run in got[i]:
            for a, b in zip(run, want[i]):
                assert torch.equal(a, b)
