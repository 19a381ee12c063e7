"""Serving operators without a GPU: the oracle's own consistency, the ABI's
struct layouts, and the refusals that come before any launch."""
import ctypes

import numpy as np
import pytest

from enilnets_b200 import _native
from oracle import attention_ref
from oracle import serving_ref as ref
from tests.test_abi import _c_offsets


@pytest.mark.parametrize("cls,cname", [
    (_native.QkNormRopeArgs, "enl_qk_norm_rope_args"),
    (_native.QkNormRopeBackwardArgs, "enl_qk_norm_rope_backward_args"),
    (_native.PagedDecodeArgs, "enl_paged_decode_args"),
    (_native.SampleArgs, "enl_sample_args")])
def test_ctypes_struct_layout_matches_c(cls, cname):
    fields = [f for f, _ in cls._fields_]
    size, offsets = _c_offsets(cname, fields)
    assert ctypes.sizeof(cls) == size
    for f, off in zip(fields, offsets):
        assert getattr(cls, f).offset == off, f


def _rope_args():
    a = _native.QkNormRopeArgs()
    a.q = a.k = a.q_out = a.k_out = a.q_weight = a.k_weight = 256
    a.batch = a.seq = 1
    a.num_heads, a.num_kv_heads, a.head_dim = 4, 2, 64
    return a


def _call(name, a):
    lib = _native.load()
    _native.check(getattr(lib, name)(ctypes.byref(a), None), name)


@pytest.mark.parametrize("change,message", [
    (dict(num_kv_heads=3), "must divide"), (dict(head_dim=100), "head_dim=100"),
    (dict(head_dim=136), "head_dim=136"), (dict(in_dtype=5), "in_dtype=5"),
    (dict(out_dtype=-1), "out_dtype=-1"), (dict(k_weight=None), "come in pairs"),
    (dict(rope_cos=256), "come in pairs"), (dict(rope_cos=256, rope_sin=256), "rope_rows=0"),
    (dict(q_weight=None, k_weight=None), "norm weights, rotation tables or both"),
    (dict(q=None), "q must be non-NULL"), (dict(k_out=8), "k_out must be 16-byte"),
    (dict(q_stride_s=-64), "multiples of 16 bytes"), (dict(k_stride_h=20), "multiples of 16 bytes"),
    (dict(n_new=256), "n_new needs k_pages"), (dict(batch=-1), "batch=-1"),
    (dict(k_pages=256), "v must be non-NULL"),
    (dict(k_pages=256, v=256), "block_table must be non-NULL"),
    (dict(k_pages=256, v_pages=256, v=256, block_table=256), "num_pages=0"),
    (dict(k_pages=256, v_pages=256, v=256, block_table=256, num_pages=1, page_size=1 << 20,
          max_pages=1 << 11), "below 2\\^31"),
    (dict(k_pages=256, v_pages=256, v=256, block_table=256, num_pages=1, page_size=16,
          max_pages=1), "start must be non-NULL"),
    (dict(k_pages=256, v_pages=256, v=256, block_table=256, num_pages=1, page_size=16,
          max_pages=1, start=256, out_dtype=1), "must be equal"),
    (dict(k_pages=256, v_pages=256, v=256, block_table=256, num_pages=1, page_size=16,
          max_pages=1, start=256, pos0=4), "pos0 must be 0"),
])
def test_norm_rope_refusals(change, message):
    a = _rope_args()
    for name, value in change.items():
        setattr(a, name, value)
    with pytest.raises(ValueError, match=message):
        _call("enl_qk_norm_rope", a)


@pytest.mark.parametrize("seq,heads", [((1 << 31) - 1, 1), ((1 << 31) - 256, 1), (1 << 28, 8)])
def test_norm_rope_refuses_more_pairs_than_it_numbers(seq, heads):
    a = _rope_args()
    a.seq, a.num_heads, a.num_kv_heads = seq, heads, 1
    with pytest.raises(ValueError, match="exceeds 2\\^31 - 257"):
        _call("enl_qk_norm_rope", a)
    b = _native.QkNormRopeBackwardArgs()
    b.batch, b.seq, b.num_heads, b.num_kv_heads, b.head_dim = 1, seq, heads, 1, 64
    b.rope_cos = b.rope_sin = 256
    b.rope_rows = 4
    with pytest.raises(ValueError, match="exceeds 2\\^31 - 257"):
        _call("enl_qk_norm_rope_backward", b)


def test_norm_rope_empty_calls_launch_nothing():
    a = _rope_args()
    a.seq = 0
    _call("enl_qk_norm_rope", a)
    a.seq, a.batch = 1, 0
    _call("enl_qk_norm_rope", a)


@pytest.mark.parametrize("change,message", [
    (dict(seq=0), "seq=0"), (dict(num_heads=5), "must divide"), (dict(grad_dtype=9), "grad_dtype=9"),
    (dict(q_weight=256), "come in pairs"), (dict(rope_sin=256), "come in pairs"),
    (dict(), "norm weights, rotation tables or both"),
    (dict(rope_cos=256, rope_sin=256, rope_rows=4), "dq_out must be non-NULL"),
])
def test_norm_rope_backward_refusals(change, message):
    a = _native.QkNormRopeBackwardArgs()
    a.batch = a.seq = 1
    a.num_heads, a.num_kv_heads, a.head_dim = 4, 2, 64
    for name, value in change.items():
        setattr(a, name, value)
    with pytest.raises(ValueError, match=message):
        _call("enl_qk_norm_rope_backward", a)


@pytest.mark.parametrize("change,message", [
    (dict(num_heads=3), "must divide"), (dict(head_dim=12), "head_dim=12"),
    (dict(sinks=-1), "sinks=-1"), (dict(seq_lens=None), "seq_lens must be non-NULL"),
    (dict(q=None), "q must be non-NULL"), (dict(o=4), "o must be 16-byte"),
    (dict(page_stride_s=4), "multiples of 16 bytes"), (dict(max_pages=0), "max_pages=0"),
    (dict(in_dtype=2), "in_dtype=2"), (dict(batch=-3), "batch=-3"),
])
def test_paged_decode_refusals(change, message):
    a = _native.PagedDecodeArgs()
    a.q = a.k_pages = a.v_pages = a.block_table = a.seq_lens = a.o = 256
    a.batch, a.num_heads, a.num_kv_heads, a.head_dim = 1, 4, 2, 64
    a.num_pages = a.max_pages = 2
    a.page_size = 16
    for name, value in change.items():
        setattr(a, name, value)
    with pytest.raises(ValueError, match=message):
        _call("enl_attn_decode_paged", a)


@pytest.mark.parametrize("change,message", [
    (dict(vocab=0), "vocab=0"), (dict(vocab=(1 << 22) + 1), "2\\^22"), (dict(dtype=3), "dtype=3"),
    (dict(logits=None), "non-NULL"), (dict(u=None), "non-NULL"), (dict(stride_b=10), "stride_b=10"),
    (dict(logits=257), "aligned"), (dict(batch=-1), "batch=-1"),
])
def test_sample_refusals(change, message):
    a = _native.SampleArgs()
    a.logits = a.u = a.tokens = 256
    a.batch, a.vocab, a.stride_b = 2, 100, 100
    for name, value in change.items():
        setattr(a, name, value)
    with pytest.raises(ValueError, match=message):
        _call("enl_sample_tokens", a)


def test_oracle_norm_rope_gradient_matches_differences():
    rng = np.random.RandomState(3)
    x, w = rng.standard_normal((2, 3, 2, 16)), 1 + 0.3 * rng.standard_normal(16)
    cos, sin = attention_ref.rope_tables(5, 16)
    cos, sin = cos[2:5, None], sin[2:5, None]
    dy = rng.standard_normal(x.shape)
    dx, dw = ref.norm_rope_backward(dy, x, w, 1e-6, cos, sin)
    f = lambda a, b: np.sum(dy * ref.norm_rope(a, b, 1e-6, cos, sin))  # noqa: E731
    vx, vw = rng.standard_normal(x.shape), rng.standard_normal(16)
    h = 1e-5
    assert abs((f(x + h * vx, w) - f(x - h * vx, w)) / (2 * h) - np.sum(dx * vx)) < 1e-7
    assert abs((f(x, w + h * vw) - f(x, w - h * vw)) / (2 * h) - np.sum(dw * vw)) < 1e-7


def test_oracle_paged_decode_equals_contiguous_oracle():
    rng = np.random.RandomState(4)
    B, H, Hkv, D, n, page = 2, 4, 2, 8, 37, 5
    K, V = rng.standard_normal((2, B, Hkv, n, D))
    q = rng.standard_normal((B, H, D))
    table = rng.permutation(B * 8).reshape(B, 8)
    kp, vp = np.full((2, B * 8, Hkv, page, D), np.nan)
    for b in range(B):
        for j in range(n):
            kp[table[b, j // page], :, j % page] = K[b, :, j]
            vp[table[b, j // page], :, j % page] = V[b, :, j]
    for window in (None, 0, 6):
        o, lse = ref.paged_decode(q, kp, vp, table, [n, n], window=window)
        oref, lref = attention_ref.decode_ref(q, K, V, slot_begin=0, slot_end=n, pos_slot0=0,
                                              q_pos=n - 1, window=window)
        np.testing.assert_allclose(o, oref, atol=1e-12)
        np.testing.assert_allclose(lse, lref, atol=1e-12)


def test_oracle_sampling_follows_the_host_sampler():
    """The draw of one uniform number equals the host path's temperature ->
    top-k -> top-p -> numpy.random.choice (which inverts the running sum with one
    random_sample) where the filters keep distinct probabilities."""
    from enilnets_b200 import generation
    rng = np.random.RandomState(5)
    for i in range(50):
        logits = rng.standard_normal(60) * 3
        probs = np.exp(logits - logits.max())
        probs /= probs.sum()
        T, k, p = (1.0, 0.7, 1.4)[i % 3], (None, 10)[i % 2], (None, 0.8)[i // 2 % 2]
        np.random.seed(i)
        u = np.random.random_sample()
        np.random.seed(i)
        token = generation.sample_token(probs, T, p, k)
        assert token in ref.sample_answers(logits, u, T, k or 0, p or 1.0)


def test_oracle_sampling_edges():
    nan, inf = np.nan, np.inf
    assert ref.sample([-inf, -inf], 0.5) == -1
    assert ref.sample([nan, 1.0], 0.5) == 1
    assert ref.sample([2.0, inf, inf], 0.75) == 2
    assert ref.sample([1.0, 1.0, 1.0], 0.99, top_k=2) == 1   # ties: lowest indices first
    assert ref.sample([0.0, 1.0, 1.0], 0.9, temperature=0.0) == 1
    assert ref.sample([0.0, 5.0], 0.999999, top_p=0.0) == 1


def test_page_bookkeeping():
    """Pages are handed out as sequences grow and come back when they end or
    leave the window; a refused request takes none."""
    from enilnets_b200.serving import PagedKVCache
    c = PagedKVCache(6, 4, 100)
    a, b = c.add(), c.add()
    c.reserve([a, b], [5, 1])
    c.advance([a, b], [5, 1])
    assert c.free_pages == 3 and c.length == {a: 5, b: 1}
    c.reserve([a], [3])
    assert c.free_pages == 3
    with pytest.raises(ValueError, match="more pages"):
        c.reserve([a, b], [12, 9])
    assert c.free_pages == 3
    c.release(b)
    assert c.free_pages == 4
    with pytest.raises(ValueError, match="not in this cache"):
        c.release(b)
    with pytest.raises(ValueError, match="max_seq_len=100"):
        c.reserve([a], [96])
    for kw in (dict(num_pages=0), dict(num_pages=1, page_size=0), dict(num_pages=1, sinks=2),
               dict(num_pages=1, window=-1), dict(num_pages=1, max_seq_len=0)):
        with pytest.raises(ValueError):
            PagedKVCache(**kw)


def test_windowed_cache_keeps_first_and_last_pages():
    from enilnets_b200.serving import PagedKVCache
    c = PagedKVCache(20, 4, 1000, window=9, sinks=5)
    s = c.add()
    for n in range(1, 200):
        c.reserve([s], [1])
        # every position that the query at n - 1 sees has its page
        seen = [j for j in range(n) if n - 1 - j <= 9 or j < 5]
        assert all(c._pages[s][j // 4] >= 0 for j in seen), n
        c.advance([s], [1])
    assert 20 - c.free_pages <= 2 + 4


def test_pages_held_is_enough_and_bounded():
    """A pool of pages_held pages serves a sequence from its prompt to its end; a
    windowed one's does not grow with the end."""
    from enilnets_b200.serving import PagedKVCache
    rng = np.random.RandomState(0)
    for _ in range(300):
        prompt, page = int(rng.randint(1, 60)), int(rng.randint(1, 20))
        total = prompt + int(rng.randint(0, 200))
        window = None if rng.rand() < 0.2 else int(rng.randint(0, 60))
        sinks = 0 if window is None else int(rng.randint(0, 12))
        n = PagedKVCache.pages_held(prompt, total, page, window, sinks)
        c = PagedKVCache(n, page, 1000, window=window, sinks=sinks)
        s = c.add()
        c.reserve([s], [prompt])
        c.advance([s], [prompt])
        while c.length[s] < total:
            c.reserve([s], [1])
            c.advance([s], [1])
    held = [PagedKVCache.pages_held(20, total, 16, 100, 4) for total in (1000, 100000)]
    assert held[0] == held[1] == 1 + 7 + 1
    assert PagedKVCache.pages_held(20, 1000, 16) == 63


def test_qk_norm_builder_keeps_the_default_contract():
    """qk_norm adds weights without drawing random numbers; without it the layer
    dict is what it was."""
    import enilnets_b200 as enl
    layers = []
    for kw in (dict(), dict(qk_norm=True)):
        enl.set_seed(1)
        net = enl.AttentionNet()
        net.add_multihead_attention(64, 4, **kw)
        layers.append(net.layers[0])
    plain, normed = layers
    assert "q_norm" not in plain and set(normed) - set(plain) == {"q_norm", "k_norm", "qk_norm_eps"}
    assert np.array_equal(plain["Wo"], normed["Wo"]) and np.array_equal(normed["q_norm"], np.ones(16))


def test_package_imports_with_a_torch_built_without_cuda():
    """Building networks, tokenizing and the CPU paths need no CUDA torch, whose
    bindings such a build lacks."""
    import subprocess
    import sys
    from pathlib import Path
    code = ("import torch\n"
            "for n in [n for n in dir(torch._C) if n.startswith('_cuda_')]:\n"
            "    delattr(torch._C, n)\n"
            "import enilnets_b200 as enl\n"
            "net = enl.AttentionNet()\n"
            "net.add_multihead_attention(64, 4, qk_norm=True)\n"
            "print(len(net.layers))\n")
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True,
                         cwd=Path(__file__).resolve().parent.parent)
    assert out.returncode == 0 and out.stdout.strip() == "1", out.stderr


@pytest.mark.parametrize("ids", [[[50]], [[3, 1 << 40]], [[-51, 0]]])
def test_token_ids_outside_the_embedding_are_refused_on_the_host(ids):
    from enilnets_b200 import network
    with pytest.raises(IndexError, match="50 rows"):
        network.embed(ids, {"weights": np.zeros((50, 8), np.float32)})
