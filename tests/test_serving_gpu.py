"""The serving path: ragged batches over a paged cache against the framework's
own contiguous cache and full Forward, query/key norms through inference,
stepping and training.

Tolerances: both sides compute the same layers in fp32 (split-bf16 projections
and prefill, about 2^-16 relative), so outputs agree to 1e-4 at activations of a few
units; in bf16 each rounds its activations, 2e-2 as the layers' bf16 bar.
"""
import numpy as np
import pytest

import enilnets_b200 as enl
from enilnets_b200 import generation, serving, training
from oracle import attention_ref as aref
from oracle import serving_ref as sref
from tests.textgen_util import PROMPTS, load

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["fp32", "bf16"])
def precision(request):
    enl.set_precision(request.param)
    yield request.param
    enl.set_precision("fp32")


def _model(seed=3, layers=2, **kw):
    enl.set_seed(seed)
    net = enl.AttentionNet()
    net.add_embedding(50, 64)
    if kw.get("positional_scheme", "absolute") == "absolute":
        net.add_positional_encoding(200, 64, learnable=False)
    for _ in range(layers):
        net.add_transformer_block(64, 4, causal=True, **kw)
    net.add_layernorm()
    net.add_dense(None, 50, activation="softmax")
    rs = np.random.RandomState(seed)
    for layer in net.layers:
        for name in ("q_norm", "k_norm"):
            if name in layer:
                layer[name] = (1 + 0.3 * rs.standard_normal(layer[name].shape)).astype(np.float32)
    return net


CONFIGS = [dict(), dict(positional_scheme="rope", num_kv_heads=2),
           dict(positional_scheme="alibi"), dict(positional_scheme="rope", qk_norm=True),
           dict(qk_norm=True, num_kv_heads=1), dict(window_size=7, positional_scheme="rope")]


@pytest.mark.parametrize("kw", CONFIGS)
def test_ragged_steps_equal_full_forward(cuda, precision, kw):
    """Prompts of unequal lengths, single tokens, a chunk in the middle and a
    sequence that joins late: each step's newest logits are the full Forward's."""
    tol = 1e-4 if precision == "fp32" else 2e-2
    net = _model(**kw)
    cache = serving.PagedKVCache(40, 8, 200)
    rs = np.random.RandomState(1)
    ids = [list(rs.randint(0, 50, n)) for n in (37, 5, 16)]
    seqs = [cache.add(), cache.add()]

    def check(logits, prefixes):
        p = np.exp(logits.double().cpu().numpy())
        p /= p.sum(-1, keepdims=True)
        for row, prefix in zip(p, prefixes):
            want = net.Forward(np.array([prefix]))[0, -1]
            assert np.abs(row - want).max() <= tol, kw

    check(serving.paged_forward_step(net, [ids[0][:20], ids[1][:1]], cache, seqs),
          [ids[0][:20], ids[1][:1]])
    check(serving.paged_forward_step(net, [[ids[0][20]], [ids[1][1]]], cache, seqs),
          [ids[0][:21], ids[1][:2]])
    check(serving.paged_forward_step(net, [ids[0][21:35], [ids[1][2]]], cache, seqs),
          [ids[0][:35], ids[1][:3]])
    late = cache.add()
    check(serving.paged_forward_step(net, [[ids[0][35]], ids[2][:15]], cache, [seqs[0], late]),
          [ids[0][:36], ids[2][:15]])
    check(serving.paged_forward_step(net, [[ids[2][15]], [ids[0][36]], [ids[1][3]]], cache,
                                     [late, seqs[0], seqs[1]]),
          [ids[2], ids[0], ids[1][:4]])
    used = 40 - cache.free_pages
    assert used == 5 + 2 + 1
    cache.release(late)
    assert cache.free_pages == 40 - 6


@pytest.mark.parametrize("kw", [dict(qk_norm=True), dict(positional_scheme="rope", qk_norm=True),
                                dict(attention_kernel="linear", qk_norm=True)])
def test_normed_layers_step_as_they_forward(cuda, kw):
    """The contiguous cache's steps equal the full Forward for layers with norms."""
    net = _model(**kw)
    ids = np.random.RandomState(2).randint(0, 50, (2, 12))
    full = net.Forward(ids)
    cache = enl.KVCache()
    got = [enl.cached_forward_step(net, ids[:, :7], cache)]
    got += [enl.cached_forward_step(net, ids[:, i:i + 1], cache) for i in range(7, 12)]
    assert np.abs(np.concatenate(got, axis=1) - full).max() <= 1e-4


def test_norm_of_a_layer_matches_the_oracle(cuda):
    """One layer with norms and rotation against float64."""
    enl.set_seed(5)
    net = enl.AttentionNet()
    net.add_multihead_attention(embed_dim=64, num_heads=4, causal=True, positional_scheme="rope",
                                qk_norm=True, num_kv_heads=2)
    layer = net.layers[0]
    rs = np.random.RandomState(6)
    layer["q_norm"], layer["k_norm"] = (1 + 0.3 * rs.standard_normal((2, 16))).astype(np.float32)
    x = rs.standard_normal((2, 30, 64))
    W = {k: np.asarray(layer[k], np.float64) for k in ("Wq", "Wk", "Wv", "Wo")}
    cos, sin = aref.rope_tables(30, 16)
    q = (x @ W["Wq"].T).reshape(2, 30, 4, 16)
    k, v = ((x @ W[n].T).reshape(2, 30, 2, 16) for n in ("Wk", "Wv"))
    q = sref.norm_rope(q, layer["q_norm"], 1e-6, cos[:, None], sin[:, None])
    k = sref.norm_rope(k, layer["k_norm"], 1e-6, cos[:, None], sin[:, None])
    o, _ = aref.attention_ref(q, k, v, causal=True)
    assert np.abs(net.Forward(x) - o.reshape(2, 30, 64) @ W["Wo"].T).max() <= 1e-3


def test_training_gradients_of_norms_match_differences(cuda):
    """d_q_norm, d_k_norm, d_Wq and dx of a layer with norms against central
    differences of its fp32 forward. The loss sums 2*20*64 products of unit size;
    the forward's relative error of 2^-16 gives it about 1e-3, over 2 h = 0.1:
    1e-2, checked at 5e-2 with the h^2 term."""
    enl.set_seed(8)
    net = enl.AttentionNet()
    net.add_multihead_attention(embed_dim=64, num_heads=4, causal=True, positional_scheme="rope",
                                qk_norm=True)
    layer = net.layers[0]
    rs = np.random.RandomState(9)
    layer["q_norm"], layer["k_norm"] = (1 + 0.2 * rs.standard_normal((2, 16))).astype(np.float32)
    x = rs.standard_normal((2, 20, 64)).astype(np.float32)
    dout = rs.standard_normal((2, 20, 64)).astype(np.float32)
    y, cache = training.multihead_attention_forward_train(layer, x)
    assert np.abs(y - net.Forward(x)).max() <= 1e-3
    dx = training.multihead_attention_backward(dout, layer, cache)
    loss = lambda lay, a: float(np.sum(  # noqa: E731
        training.multihead_attention_forward_train(lay, a)[0].astype(np.float64) * dout))
    h = 0.05
    for name in ("q_norm", "k_norm", "Wq"):
        d = rs.standard_normal(layer[name].shape).astype(np.float32)
        d *= 1.0 if name != "Wq" else 0.1
        hi, lo = dict(layer), dict(layer)
        hi[name], lo[name] = layer[name] + h * d, layer[name] - h * d
        slope = (loss(hi, x) - loss(lo, x)) / (2 * h)
        want = float(np.sum(layer["d_" + name] * d))
        assert abs(slope - want) <= 5e-2 + 5 * h * h * max(1.0, abs(want)), (name, slope, want)
    d = 0.1 * rs.standard_normal(x.shape).astype(np.float32)
    slope = (loss(layer, x + h * d) - loss(layer, x - h * d)) / (2 * h)
    want = float(np.sum(dx * d))
    assert abs(slope - want) <= 5e-2 + 5 * h * h * max(1.0, abs(want))


@pytest.fixture
def gen(golden_dir):
    _, tok = load(golden_dir)
    enl.set_precision("fp32")
    enl.set_seed(42)
    return generation.TextGenerator(tok, embed_dim=32, num_heads=4, num_layers=2, max_seq_len=48)


def test_serve_equals_one_by_one_generation(cuda, gen):
    """Greedy texts of a ragged batch are those of generate for each prompt."""
    want = [gen.generate(p, max_new_tokens=12, greedy=True) for p in PROMPTS]
    assert gen.serve(PROMPTS, max_new_tokens=12, greedy=True) == want
    assert gen.serve(PROMPTS, max_new_tokens=12, greedy=True, page_size=3) == want
    assert gen.serve([], greedy=True) == []


def test_serve_samples_as_generate_does(cuda, gen):
    """One prompt, same seed: the device draws what numpy.random.choice drew."""
    for i in range(4):
        kw = dict(max_new_tokens=10, temperature=0.8, top_k=5, top_p=0.9)
        np.random.seed(i)
        want = gen.generate_ids("keys", **kw)
        np.random.seed(i)
        assert gen.serve_ids(["keys"], **kw) == [want]


def test_serve_with_a_window_holds_its_pages_only(cuda, gen, monkeypatch):
    """serve with a window: the tokens of the same steps on a roomy cache, from a
    pool that does not hold every position."""
    made = []

    class Cache(serving.PagedKVCache):
        def __init__(self, pages, *args, **kw):
            made.append(pages)
            super().__init__(pages, *args, **kw)

    kw = dict(window=7, sinks=2)
    want = []
    for ids in (gen._prompt_ids("the cache keeps keys"), gen._prompt_ids("a")):
        cache = serving.PagedKVCache(100, 2, gen.max_seq_len, **kw)
        seq, ids = cache.add(), list(ids)
        logits = serving.paged_forward_step(gen.network, [ids], cache, [seq])
        for _ in range(40):
            tok = serving.sample(logits, [0.0], greedy=True)[0]
            if tok == gen._id(gen.tokenizer.end_token):
                break
            ids.append(tok)
            if cache.length[seq] >= gen.max_seq_len:
                break
            logits = serving.paged_forward_step(gen.network, [[tok]], cache, [seq])
        want.append(ids)
    monkeypatch.setattr(serving, "PagedKVCache", Cache)
    got = gen.serve_ids(["the cache keeps keys", "a"], max_new_tokens=40, greedy=True, page_size=2,
                        **kw)
    assert got == want
    prompt = -(-len(gen._prompt_ids("the cache keeps keys")) // 2)
    assert made == [max(prompt, 6) + 6]


@pytest.mark.parametrize("kw", [dict(), dict(greedy=True), dict(top_k=3, temperature=0.5)])
def test_rows_without_a_logit_are_refused(cuda, gen, kw):
    """A row of NaN and -inf has no token: the draw raises, and so does serve on a
    model that gives such rows, instead of feeding a token number -1 on."""
    import torch
    nan, inf = float("nan"), float("inf")
    x = torch.tensor([[0.0, 1.0, -inf], [nan, -inf, nan], [1.0, nan, -inf], [-inf] * 3],
                     device="cuda")
    with pytest.raises(ValueError, match=r"rows \[1, 3\]"):
        serving.sample(x, [0.5] * 4, **kw)
    assert serving.sample(x[::2].contiguous(), [0.999, 0.5], **kw) == [1, 0]
    head = gen.network.layers[-1]
    head["bias"] = np.full_like(head["bias"], nan)
    with pytest.raises(ValueError, match="every logit is NaN or -inf"):
        gen.serve_ids(["keys", "a"], max_new_tokens=3, **kw)


def test_serve_stops_at_the_model_length(cuda, gen):
    ids = gen.serve_ids(["the cache keeps keys", "a"], max_new_tokens=60, greedy=True)
    want = [gen.generate_ids(p, max_new_tokens=60, greedy=True)
            for p in ("the cache keeps keys", "a")]
    assert ids == want


def test_streaming_cache_gives_pages_back(cuda):
    """A windowed cache holds a bounded number of pages, and its steps equal the
    oracle's visible set: first tokens and the last ones."""
    import torch
    from enilnets_b200 import kernels
    net = _model(layers=1, positional_scheme="rope", num_kv_heads=2)
    cache = serving.PagedKVCache(9, 4, 200, window=15, sinks=3)
    s = cache.add()
    rs = np.random.RandomState(4)
    serving.paged_forward_step(net, [list(rs.randint(0, 50, 6))], cache, [s])
    for i in range(60):
        logits = serving.paged_forward_step(net, [[int(rs.randint(0, 50))]], cache, [s])
        assert torch.isfinite(logits).all()
    assert cache.length[s] == 66 and cache.free_pages >= 9 - 6
    idx = next(i for i, lay in enumerate(net.layers) if lay["type"] == "multihead_attention")
    kp, vp = cache.pools[idx]
    q = torch.randn((1, 4, 16), device="cuda")
    table, lens = cache.table([s]), torch.tensor([66], dtype=torch.int32, device="cuda")
    o = kernels.attention_decode_paged(q, kp, vp, table, lens, window=15, sinks=3)
    ref, _ = sref.paged_decode(q.double().cpu().numpy(), kp.double().cpu().numpy(),
                               vp.double().cpu().numpy(), table.cpu().numpy(), [66], window=15,
                               sinks=3)
    assert np.abs(o.cpu().numpy() - ref).max() <= 1e-5


def test_paged_step_refusals(cuda):
    net = _model(layers=1)
    cache = serving.PagedKVCache(2, 4, 10)
    s = cache.add()
    cases = [(lambda: serving.paged_forward_step(net, [[1]], cache, [7]), "not in this cache"),
             (lambda: serving.paged_forward_step(net, [[]], cache, [s]), "one or more tokens"),
             (lambda: serving.paged_forward_step(net, [[1], [2]], cache, [s, s]), "different"),
             (lambda: serving.paged_forward_step(net, [[1] * 9], cache, [s]), "more pages"),
             (lambda: serving.paged_forward_step(net, [[1] * 11], cache, [s]), "max_seq_len=10"),
             (lambda: cache.release(99), "not in this cache")]
    for call, message in cases:
        with pytest.raises(ValueError, match=message):
            call()
    assert cache.free_pages == 2 and cache.length[s] == 0
    other = enl.AttentionNet()
    other.add_embedding(50, 64)
    other.add_multihead_attention(64, 4, causal=True, attention_kernel="linear")
    with pytest.raises(ValueError, match="softmax layers"):
        serving.paged_forward_step(other, [[1]], cache, [s])
