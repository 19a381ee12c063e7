"""Sampling against the float64 oracle.

A weight's relative error: the argument (l - max) / T carries two fp32
roundings, 2^-23 of at most 28 (smaller weights round to zero), and the
exponential two units in the last place: 4e-6 together. Moving the draw and the
thresholds by 1e-5 either way therefore gives every token a right computation
may return; nearly always that is one token, which the tests count.
"""
import numpy as np
import pytest

from oracle import serving_ref as ref

pytestmark = pytest.mark.gpu


def _dev(x, dtype="fp32"):
    import torch
    t = torch.from_numpy(np.asarray(x, dtype=np.float32)).cuda()
    return t.to(torch.bfloat16) if dtype == "bf16" else t


def _rows(seed, B, V, flat=0.0):
    rng = np.random.RandomState(seed)
    x = 2.0 * rng.standard_normal((B, V))
    n = min(V, 40)
    for b in range(B):
        x[b, rng.permutation(V)[:n]] += 6 + 3 * rng.standard_normal(n)
    return x * (1.0 - flat)


SETTINGS = [dict(), dict(temperature=0.0), dict(temperature=0.7), dict(top_k=1), dict(top_k=7),
            dict(top_k=300), dict(top_k=5000, temperature=1.5), dict(top_p=0.9), dict(top_p=0.3),
            dict(top_p=0.0), dict(top_p=0.999, temperature=1.3), dict(min_p=0.1),
            dict(min_p=1.0), dict(temperature=0.8, top_k=50, top_p=0.95),
            dict(temperature=1.2, top_k=900, top_p=0.7, min_p=0.02)]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("V", [1, 2, 31, 1000, 1025, 8191, 50001, 131072])
def test_settings(cuda, dtype, V):
    """Every setting, as numbers for all rows and as per-row tensors."""
    import torch
    from enilnets_b200 import kernels
    B = 3
    x = _dev(np.concatenate([_rows(V, B - 1, V), _rows(V + 1, 1, V, flat=0.9)]), dtype)
    host = x.double().cpu().numpy()
    single = total = 0
    for i, kw in enumerate(SETTINGS):
        u = np.random.RandomState(i).random_sample(B).astype(np.float32)
        tokens = kernels.sample_tokens(x, _dev(u), **kw).cpu().numpy()
        tensors = {k: torch.full((B,), v, dtype=torch.int32 if k == "top_k" else torch.float32,
                                 device="cuda") for k, v in kw.items()}
        again = kernels.sample_tokens(x, _dev(u), **tensors).cpu().numpy()
        assert (tokens == again).all(), kw
        for b in range(B):
            answers = ref.sample_answers(host[b], float(u[b]), **kw)
            assert tokens[b] in answers, (kw, b, tokens[b], answers)
            single += len(answers) == 1
            total += 1
    assert single >= 0.8 * total


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_draws_cover_the_distribution(cuda, dtype):
    """A grid of draws over one row: each token comes out in proportion to its
    probability, to within the two grid cells at its ends."""
    import torch
    from enilnets_b200 import kernels
    N, V = 4096, 97
    row = _dev(_rows(3, 1, V) * 0.5, dtype)
    u = (torch.arange(N, device="cuda") + 0.5) / N
    for kw in (dict(), dict(top_k=9), dict(top_p=0.6), dict(min_p=0.2), dict(temperature=2.0)):
        tokens = kernels.sample_tokens(row.expand(N, V).contiguous(), u.float(), **kw)
        count = torch.bincount(tokens, minlength=V).double().cpu().numpy()
        want = np.zeros(V)
        host = row[0].double().cpu().numpy()
        for i in range(N):
            want[ref.sample(host, (i + 0.5) / N, **kw)] += 1
        assert np.abs(count - want).max() <= 2, kw


def test_ties_take_the_lowest_indices(cuda):
    import torch
    from enilnets_b200 import kernels
    for V in (5, 3000, 40000):
        x = torch.zeros((4, V), device="cuda")
        u = torch.tensor([0.0, 0.34, 0.67, 0.9999], device="cuda")
        assert kernels.sample_tokens(x, u, top_k=3).tolist() == [0, 1, 2, 2]
        assert kernels.sample_tokens(x, u, temperature=0).tolist() == [0, 0, 0, 0]
        # 1.5 of V equal tokens: the leading set that reaches the mass has two
        assert kernels.sample_tokens(x, u, top_p=1.5 / V).tolist() == [0, 0, 1, 1]
        want = [min(V - 1, int(V * v)) for v in u.tolist()]
        got = kernels.sample_tokens(x, u).tolist()
        assert all(abs(a - b) <= 1 for a, b in zip(got, want))
        x[:, 1::2] = 1.0
        assert kernels.sample_tokens(x, u, top_k=2).tolist() == [1, 1, 3, 3]
    # half of a wide row ties at the threshold
    x = torch.zeros((1, 60000), device="cuda", dtype=torch.bfloat16)
    x[0, 30000:] = 2.0
    u = torch.tensor([0.9999], device="cuda")
    assert kernels.sample_tokens(x, u, top_k=29000).tolist()[0] in range(58995, 59000)
    assert kernels.sample_tokens(x, u, top_k=5).tolist() == [30004]


def test_not_a_number_and_infinities(cuda):
    import torch
    from enilnets_b200 import kernels
    inf, nan = float("inf"), float("nan")
    x = torch.full((6, 2000), -inf, device="cuda")
    x[0, 1999] = -1e30                      # one live logit
    x[1, 7], x[1, 8] = nan, 0.0
    x[2, 5], x[2, 1500] = inf, inf          # two infinite logits share the row
    # row 3: nothing live
    x[4] = nan
    x[5] = torch.finfo(torch.float32).min   # the lowest value everywhere is a flat row
    u = torch.full((6,), 0.75, device="cuda")
    for kw in (dict(), dict(top_k=4, top_p=0.999), dict(temperature=0.3), dict(min_p=0.5)):
        got = kernels.sample_tokens(x, u, **kw).tolist()
        assert got[:5] == [1999, 8, 1500, -1, -1], (kw, got)
        assert got[5] == (3 if "top_k" in kw else 1500), kw  # first sum above 0.75 of 4 or 2000
    assert kernels.sample_tokens(x, u, temperature=0).tolist() == [1999, 8, 5, -1, -1, 0]


def test_minus_zero_ties_with_zero(cuda):
    import torch
    from enilnets_b200 import kernels
    x = torch.tensor([[0.0, -0.0, 0.0, -0.0]], device="cuda")
    u = torch.tensor([0.99], device="cuda")
    assert kernels.sample_tokens(x, u, top_k=2).tolist() == [1]
    assert kernels.sample_tokens(x.bfloat16(), u, top_k=2).tolist() == [1]


def test_draw_ends(cuda):
    """u = 0 is the first kept token, the largest u below 1 the last one."""
    import torch
    from enilnets_b200 import kernels
    x = torch.tensor([[-30.0, 1.0, 2.0, -30.0, 1.5, -40.0]], device="cuda").repeat(3, 1)
    u = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0], device="cuda")
    assert kernels.sample_tokens(x, u, min_p=0.01).tolist() == [1, 4, 4]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_row_does_not_depend_on_the_batch(cuda, dtype):
    """A row alone, in a batch, in a strided view and at another alignment gives
    the same token."""
    import torch
    from enilnets_b200 import kernels
    V = 33333
    x = _dev(_rows(5, 40, V), dtype)
    g = torch.Generator(device="cuda").manual_seed(1)
    u = torch.rand((40,), device="cuda", generator=g)
    kw = [dict(), dict(top_k=50, top_p=0.9), dict(top_p=0.95, temperature=1.2)]
    for k in kw:
        want = kernels.sample_tokens(x, u, **k)
        for b in (0, 17, 39):
            assert kernels.sample_tokens(x[b:b + 1], u[b:b + 1], **k).tolist() == [want[b].item()]
        for off in (1, 2, 3, 5):
            wide = torch.full((40, V + 9), float("inf"), device="cuda", dtype=x.dtype)
            wide[:, off:off + V] = x
            assert torch.equal(kernels.sample_tokens(wide[:, off:off + V], u, **k), want), off


def test_mixed_settings_per_row(cuda):
    import torch
    from enilnets_b200 import kernels
    rng = np.random.RandomState(8)
    B, V = 64, 20001
    x = _dev(_rows(8, B, V), "bf16")
    host = x.double().cpu().numpy()
    t = rng.choice([0.0, 0.5, 1.0, 1.7], B).astype(np.float32)
    k = rng.choice([0, 1, 40, 1000, 5000, V + 5], B).astype(np.int32)
    p = rng.choice([1.0, 0.5, 0.95, 2.0], B).astype(np.float32)
    m = rng.choice([0.0, 0.05, 0.5], B).astype(np.float32)
    u = rng.random_sample(B).astype(np.float32)
    got = kernels.sample_tokens(x, _dev(u), temperature=_dev(t),
                                top_k=torch.from_numpy(k).cuda(), top_p=_dev(p), min_p=_dev(m))
    for b, token in enumerate(got.tolist()):
        assert token in ref.sample_answers(host[b], float(u[b]), float(t[b]), int(k[b]),
                                           float(p[b]), float(m[b])), b


@pytest.mark.parametrize("dtype,V", [("fp32", 2049), ("fp32", 4097), ("fp32", 8200),
                                     ("bf16", 4097), ("bf16", 8195), ("bf16", 16401)])
def test_rows_just_long_enough_for_several_blocks(cuda, dtype, V):
    """Vocabularies one vector past the size that gives a row another block: the
    last block has next to nothing to read and reaches the exchange of the row's
    extremes at once. The same tokens every time, and the definition's."""
    from enilnets_b200 import kernels
    B = 6
    x = _dev(_rows(V, B, V), dtype)
    host = x.double().cpu().numpy()
    u = np.random.RandomState(V).random_sample(B).astype(np.float32)
    for kw in (dict(temperature=0.0), dict(), dict(top_k=20, top_p=0.9), dict(top_p=0.8),
               dict(min_p=0.1)):
        first = kernels.sample_tokens(x, _dev(u), **kw).cpu().numpy()
        for b in range(B):
            assert first[b] in ref.sample_answers(host[b], float(u[b]), **kw), (kw, b)
        again = [kernels.sample_tokens(x, _dev(u), **kw) for _ in range(50)]
        assert all((t.cpu().numpy() == first).all() for t in again), kw


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("V", [3, 40, 515, 2047, 4095])
def test_top_p_of_rows_with_a_block_each(cuda, dtype, V):
    """More rows than SMs and small vocabularies, so that a row has one block and
    some of its warps have nothing to read: the estimate of the total follows the
    extremes at once. The same tokens every time, and the definition's."""
    from enilnets_b200 import kernels
    B = 300
    x = _dev(np.concatenate([_rows(V, B // 2, V), _rows(V + 1, B // 2, V, flat=0.8)]), dtype)
    host = x.double().cpu().numpy()
    u = np.random.RandomState(V).random_sample(B).astype(np.float32)
    for kw in (dict(top_p=0.5), dict(top_p=0.9), dict(top_p=0.99, temperature=1.4)):
        first = kernels.sample_tokens(x, _dev(u), **kw).cpu().numpy()
        for b in range(B):
            assert first[b] in ref.sample_answers(host[b], float(u[b]), **kw), (kw, b)
        again = [kernels.sample_tokens(x, _dev(u), **kw) for _ in range(50)]
        assert all((t.cpu().numpy() == first).all() for t in again), kw


@pytest.mark.parametrize("B", [3, 200])
@pytest.mark.parametrize("top", [1.0, 3e4, 1e30])
def test_logits_that_share_their_distance_from_the_largest(cuda, B, top):
    """One logit above many unequal ones that are all the same fp32 distance below
    it: their order is still theirs, not their indices'. Temperatures that keep
    their weights well above zero."""
    from enilnets_b200 import kernels
    rng = np.random.RandomState(3)
    for V, k in ((1000, 300), (1500, 1000), (9000, 700), (9000, 5000)):
        x = (1e-9 * top * rng.standard_normal((B, V))).astype(np.float32)
        x[:, V // 3] = top
        u = rng.random_sample(B).astype(np.float32)
        for kw in (dict(top_k=k), dict(top_k=k, top_p=0.9), dict(top_p=0.4),
                   dict(top_k=k, top_p=0.7, min_p=0.3)):
            kw["temperature"] = top
            got = kernels.sample_tokens(_dev(x), _dev(u), **kw).tolist()
            for b in range(0, B, max(1, B // 8)):
                answers = ref.sample_answers(x[b].astype(np.float64), float(u[b]), **kw)
                assert got[b] in answers, (V, kw, b, got[b], answers)


def _hard_rows(rng, V):
    """Rows whose cuts a histogram of a quarter of the logits guesses badly: flat
    ones, narrow clusters with thousands of tokens a bin, steps, a heavy tail, whole
    numbers (long ties) and one that is flat but for a single far token."""
    flat = rng.standard_normal(V)
    step = np.where(np.arange(V) % 7 == 0, 2.0, 0.0) + 1e-4 * rng.standard_normal(V)
    far = 1e-3 * rng.standard_normal(V)
    far[V // 2] = 12.0
    return [flat, 0.1 * flat, 3.0 + 1e-5 * flat, step, -rng.exponential(4.0, V),
            np.round(2.0 * flat), far, np.where(np.arange(V) < V // 3, flat, -1e30)]


def _may_draw(row, order, u, token, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, eps=1e-5):
    """Whether the draw u may give the token where weights are right to eps: with each
    threshold where it is or eps to a side, u is within eps of its stretch of the
    running sum."""
    w = np.exp((row - row[order[0]]) / temperature)
    for p in {top_p, *((top_p - eps, top_p + eps) if top_p < 1.0 else ())}:
        ws = w[order]
        if top_k > 0:
            ws[top_k:] = 0.0
        if p < 1.0:
            before = np.cumsum(ws) - ws
            ws[1:][before[1:] >= p * ws.sum()] = 0.0
        for m in {min_p, min_p * (1 - eps), min_p * (1 + eps)}:
            kept = np.zeros_like(w)
            kept[order] = np.where(ws < m, 0.0, ws)
            end = np.cumsum(kept) / kept.sum()
            start = end[token - 1] if token else 0.0
            if kept[token] > 0 and start - eps <= u <= end[token] + eps:
                return True
    return False


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("V,repeat", [(40009, 1), (20001, 20), (131072, 2)])
def test_rows_that_defeat_the_guesses(cuda, dtype, V, repeat):
    """Large top-k and flat nuclei over such rows, one block and several a row."""
    from enilnets_b200 import kernels
    rng = np.random.RandomState(V)
    rows = _hard_rows(rng, V)
    n = len(rows)
    x = _dev(np.stack(rows * repeat), dtype)
    host = x[:n].double().cpu().numpy()
    orders = [np.argsort(-r, kind="stable") for r in host]
    for kw in (dict(top_k=2500), dict(top_k=V // 3), dict(top_p=0.5), dict(top_p=0.99),
               dict(top_k=V // 5, top_p=0.7), dict(top_k=6000, top_p=0.9, min_p=0.3),
               dict(top_p=0.95, temperature=3.0)):
        u = rng.random_sample(len(x)).astype(np.float32)
        got = kernels.sample_tokens(x, _dev(u), **kw).tolist()
        for b in sorted({*range(n), *range(len(x) - n, len(x))}):
            assert _may_draw(host[b % n], orders[b % n], float(u[b]), got[b], **kw), (kw, b, got[b])


@pytest.mark.parametrize("T", [1e-45, 1e-40, 1e-38, 1e-30])
def test_lowest_temperatures(cuda, T):
    """A temperature whose reciprocal passes fp32 leaves the largest logit alone,
    under any setting; equal ones share the draw."""
    import torch
    from enilnets_b200 import kernels
    rng = np.random.RandomState(2)
    for B, V in ((3, 9), (3, 5000), (3, 70000), (200, 5000)):
        x = _dev(rng.standard_normal((B, V)))
        want = x.argmax(-1)
        u = _dev(rng.random_sample(B))
        tie = torch.zeros((B, V), device="cuda")
        tie[:, V // 2:V // 2 + 4] = 3.0
        for kw in (dict(), dict(min_p=0.1), dict(top_k=5), dict(top_k=2000), dict(top_p=0.5),
                   dict(top_k=50, top_p=1.0 - 2.0 ** -10, min_p=0.5)):
            out = torch.full((B,), -77, dtype=torch.int64, device="cuda")
            t = torch.full((B,), T, device="cuda")
            assert torch.equal(kernels.sample_tokens(x, u, temperature=T, out=out, **kw), want), kw
            assert torch.equal(kernels.sample_tokens(x, u, temperature=t, **kw), want), kw
            if "top_p" not in kw:
                got = kernels.sample_tokens(tie, u, temperature=T, **kw)
                assert torch.equal(got, V // 2 + (u * 4).long()), kw


def test_weights_equal_the_elementary_form(cuda):
    """The kernel's weights are those of elementary fp32 operations bit for bit:
    the draw, exact in whole numbers, equals one computed from exp() of torch."""
    import torch
    from enilnets_b200 import kernels
    g = torch.Generator(device="cuda").manual_seed(4)
    B, V = 256, 5003
    x = 3 * torch.randn((B, V), device="cuda", generator=g)
    u = torch.rand((B,), device="cuda", generator=g)
    inv = 1.0 / torch.full((B, 1), 0.9, device="cuda")
    top = x.amax(-1, keepdim=True)
    q = (torch.exp((x - top) * inv) * 2.0 ** 40).long()
    run = q.cumsum(-1)
    total = run[:, -1:]
    part = (u * 2.0 ** 24).long()[:, None]
    target = (total >> 24) * part + (((total & 0xFFFFFF) * part) >> 24)
    want = (run <= target).sum(-1)
    assert torch.equal(kernels.sample_tokens(x, u, temperature=0.9), want)


def test_refusals(cuda):
    import torch
    from enilnets_b200 import kernels
    x, u = torch.zeros((2, 10), device="cuda"), torch.zeros((2,), device="cuda")
    f = kernels.sample_tokens
    cases = [
        (lambda: f(x[0], u), "logits must"), (lambda: f(x.cpu(), u), "logits must"),
        (lambda: f(x.half(), u), "logits must"), (lambda: f(x.T, u), "logits must"),
        (lambda: f(x, u[:1]), "u must"), (lambda: f(x, u.double()), "u must"),
        (lambda: f(x, u, temperature=-1.0), "temperature=-1"),
        (lambda: f(x, u, top_k=-2), "top_k=-2"), (lambda: f(x, u, min_p=1.5), "min_p=1.5"),
        (lambda: f(x, u, top_p=float("nan")), "top_p=nan"),
        (lambda: f(x, u, top_k=u), "top_k must"), (lambda: f(x, u, temperature=u[:1]), "temperature"),
        (lambda: f(x[:, :0], u), "vocab=0"),
        (lambda: f(x, u, out=torch.zeros(2, device="cuda")), "out must"),
    ]
    for call, message in cases:
        with pytest.raises(ValueError, match=message):
            call()
    assert f(x[:0], u[:0]).shape == (0,)
