"""Per-head norm with rotation: forward, backward and the paged append, against
the float64 oracle on the values the kernels read.

Tolerances. fp32: about a dozen fp32 operations per element, the longest a sum
of D <= 128 squares: a relative error below 20 * 2^-24 = 1.2e-6 of values of
a few units, checked at 1e-5 absolute. bf16 outputs add one rounding, at most
2^-9 of the value: 2^-8 |y| + 1e-5. Weight gradients sum N products of unit
size in fp32, in partial sums of N / 64 or fewer: sqrt(N) 1e-5 + 1e-5.
"""
import numpy as np
import pytest

from oracle import attention_ref as aref
from oracle import serving_ref as ref

pytestmark = pytest.mark.gpu
EPS = 1e-6


def _t(x, dtype="fp32"):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).cuda()
    return t.to(torch.bfloat16) if dtype == "bf16" else t


def _np(t):
    return t.detach().double().cpu().numpy()


def _close(got, want, dtype):
    tol = 1e-5 + (2.0 ** -8 * np.abs(want) if dtype == "bf16" else 0.0)
    assert got.shape == want.shape
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), f"{bad.sum()} values off, worst {np.abs(got - want)[bad].max():.3e}"


def _inputs(seed, B, S, H, Hkv, D, dtype):
    """q, k, v head views of one fused tensor, and norm weights."""
    rng = np.random.RandomState(seed)
    qkv = _t(rng.standard_normal((B, S, (H + 2 * Hkv) * D)), dtype)
    q = qkv[..., :H * D].unflatten(-1, (H, D))
    k = qkv[..., H * D:(H + Hkv) * D].unflatten(-1, (Hkv, D))
    v = qkv[..., (H + Hkv) * D:].unflatten(-1, (Hkv, D))
    return q, k, v, 1 + 0.3 * rng.standard_normal(D), 1 + 0.3 * rng.standard_normal(D)


def _tables(rows, D):
    cos, sin = aref.rope_tables(rows, D)
    return cos.astype(np.float32), sin.astype(np.float32)


SHAPES = [(1, 1, 1, 1, 8), (2, 5, 3, 1, 24), (1, 7, 4, 4, 32), (3, 33, 6, 2, 40), (2, 17, 5, 5, 64),
          (1, 129, 9, 3, 80), (2, 31, 16, 2, 96), (4, 50, 20, 4, 128), (65, 1, 32, 8, 128)]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("B,S,H,Hkv,D", SHAPES)
@pytest.mark.parametrize("norm,rope", [(True, True), (True, False), (False, True)])
def test_forward(cuda, B, S, H, Hkv, D, dtype, norm, rope):
    import torch
    from enilnets_b200 import _native, kernels
    q, k, _, wq, wk = _inputs(B + S + D, B, S, H, Hkv, D, dtype)
    wq, wk = (wq.astype(np.float32), wk.astype(np.float32)) if norm else (None, None)
    cos, sin = _tables(S + 11, D)
    tables = (_t(cos), _t(sin)) if rope else None
    start = np.random.RandomState(1).randint(0, 9, B).astype(np.int32)
    qo, ko = kernels.qk_norm_rope(q, k, None if wq is None else _t(wq),
                                  None if wk is None else _t(wk), eps=EPS, rope=tables, pos0=2,
                                  start=torch.from_numpy(start).cuda())
    torch.cuda.synchronize()
    assert _native.device_error() == (0, 0)
    pos = 2 + start[:, None] + np.arange(S)
    c, s = (cos[pos][:, :, None], sin[pos][:, :, None]) if rope else (None, None)
    assert qo.dtype == q.dtype
    _close(_np(qo), ref.norm_rope(_np(q), wq, EPS, c, s), dtype)
    _close(_np(ko), ref.norm_rope(_np(k), wk, EPS, c, s), dtype)


def test_forward_in_place_and_mixed_types(cuda):
    """Outputs over the inputs; bf16 in and fp32 out, and the other way."""
    import torch
    from enilnets_b200 import kernels
    q, k, _, wq, wk = _inputs(7, 2, 9, 4, 2, 64, "bf16")
    wq, wk = _t(wq), _t(wk)
    tables = tuple(map(_t, _tables(9, 64)))
    qo, ko = kernels.qk_norm_rope(q, k, wq, wk, rope=tables, out_dtype=torch.float32)
    want = ref.norm_rope(_np(q), _np(wq), EPS, _np(tables[0])[:, None], _np(tables[1])[:, None])
    _close(_np(qo), want, "fp32")
    q2, _ = kernels.qk_norm_rope(q.float(), k.float(), wq, wk, rope=tables,
                                 out_dtype=torch.bfloat16)
    _close(_np(q2), want, "bf16")
    kernels.qk_norm_rope(q, k, wq, wk, rope=tables, out=(q, k))
    assert torch.equal(q, qo.bfloat16()) and torch.equal(k, ko.bfloat16())


def test_zero_rows_and_large_values(cuda):
    """A zero head stays zero (eps keeps its norm finite); heads of 1e15 and
    1e-15 normalise without overflow or loss; an infinite or NaN head stays in
    its own row."""
    import torch
    from enilnets_b200 import kernels
    x = torch.randn((1, 6, 2, 64), device="cuda")
    x[0, 1] = 0
    x[0, 2] *= 1e15
    x[0, 3] *= 1e-15
    x[0, 4, 0, 3] = float("inf")
    x[0, 4, 1, 5] = float("nan")
    w = torch.ones(64, device="cuda")
    q, _ = kernels.qk_norm_rope(x, x[:, :, :1], w, w, eps=1e-30)
    torch.cuda.synchronize()
    assert torch.count_nonzero(q[0, 1]) == 0
    _close(_np(q[0, [0, 2, 3, 5]]), ref.norm_rope(_np(x[0, [0, 2, 3, 5]]), _np(w), 1e-30, None, None),
           "fp32")


@pytest.mark.parametrize("in_dtype,grad_dtype", [("fp32", "fp32"), ("bf16", "fp32"),
                                                 ("bf16", "bf16"), ("fp32", "bf16")])
@pytest.mark.parametrize("B,S,H,Hkv,D", SHAPES + [(2, 700, 16, 4, 128)])
@pytest.mark.parametrize("norm,rope", [(True, True), (True, False), (False, True)])
def test_backward(cuda, B, S, H, Hkv, D, in_dtype, grad_dtype, norm, rope):
    import torch
    from enilnets_b200 import _native, kernels
    rng = np.random.RandomState(B * S + D)
    q, k, _, wq, wk = _inputs(B + S + D, B, S, H, Hkv, D, in_dtype)
    wq, wk = (wq.astype(np.float32), wk.astype(np.float32)) if norm else (None, None)
    dq, dk = _t(rng.standard_normal(q.shape), grad_dtype), _t(rng.standard_normal(k.shape),
                                                              grad_dtype)
    cos, sin = _tables(S + 3, D)
    tables = (_t(cos), _t(sin)) if rope else None
    tw = [None if w is None else _t(w) for w in (wq, wk)]
    gq, gk, gwq, gwk = kernels.qk_norm_rope_backward(
        dq, dk, q if norm else None, k if norm else None, *tw, eps=EPS, rope=tables, pos0=3,
        out_dtype=torch.float32)
    again = kernels.qk_norm_rope_backward(
        dq, dk, q if norm else None, k if norm else None, *tw, eps=EPS, rope=tables, pos0=3,
        out_dtype=torch.float32)
    torch.cuda.synchronize()
    assert _native.device_error() == (0, 0)
    c, s = (cos[3:, None], sin[3:, None]) if rope else (None, None)
    for got, dw, x, dy, w in ((gq, gwq, q, dq, wq), (gk, gwk, k, dk, wk)):
        want, wantw = ref.norm_rope_backward(_np(dy), _np(x), w, EPS, c, s)
        _close(_np(got), want, "fp32")
        if norm:
            n = x[..., 0].numel()
            assert np.abs(_np(dw) - wantw).max() <= 1e-5 * np.sqrt(n) + 1e-5
        else:
            assert dw is None
    for a, b in zip((gq, gk, gwq, gwk), again):
        assert a is None or torch.equal(a, b)  # the sums' order is fixed


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("B,S,H,Hkv,D", [(1, 1, 1, 1, 64), (2, 7, 4, 1, 64), (2, 7, 4, 2, 40),
                                         (3, 5, 3, 3, 128), (1, 33, 5, 5, 24), (2, 9, 8, 4, 128)])
def test_backward_without_eps(cuda, B, S, H, Hkv, D, dtype):
    """eps = 0 over heads that are not zero: heads and tokens that only fill up a
    block's share, and tokens outside the tables, add nothing to the weights'
    gradients."""
    import torch
    from enilnets_b200 import _native, kernels
    rng = np.random.RandomState(S + D)
    q, k, _, wq, wk = _inputs(S + D, B, S, H, Hkv, D, dtype)
    wq, wk = wq.astype(np.float32), wk.astype(np.float32)
    dq, dk = _t(rng.standard_normal(q.shape)), _t(rng.standard_normal(k.shape))
    cos, sin = _tables(S + 1, D)
    for rows in (S + 1, S):  # all tokens have angles; all but the last one
        _native.device_error(clear=True)
        gq, gk, gwq, gwk = kernels.qk_norm_rope_backward(
            dq, dk, q, k, _t(wq), _t(wk), eps=0.0, rope=(_t(cos[:rows]), _t(sin[:rows])), pos0=1,
            out_dtype=torch.float32)
        assert _native.device_error(clear=True)[0] == (0 if rows > S else 2)
        n = rows - 1
        c, s = cos[1:rows, None], sin[1:rows, None]
        for got, dw, x, dy, w in ((gq, gwq, q, dq, wq), (gk, gwk, k, dk, wk)):
            want, wantw = ref.norm_rope_backward(_np(dy)[:, :n], _np(x)[:, :n], w, 0.0, c, s)
            _close(_np(got)[:, :n], want, "fp32")
            assert torch.count_nonzero(got[:, n:]) == 0
            assert np.abs(_np(dw) - wantw).max() <= 1e-5 * np.sqrt(x[..., 0].numel()) + 1e-5


def test_backward_matches_differences_of_the_forward(cuda):
    """<gradient, direction> against central differences of the fp32 forward.
    The loss sums N = 2*40*6*64 products; fp32 rounding of the forward gives it
    an error of about 1e-7 sqrt(N) = 2e-5, over 2 h = 0.02: 1e-3, checked at
    2e-2 plus the h^2 term."""
    import torch
    from enilnets_b200 import kernels
    g = torch.Generator(device="cuda").manual_seed(2)
    r = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    q, k, wq, wk = r(2, 40, 4, 64), r(2, 40, 2, 64), 1 + 0.2 * r(64), 1 + 0.2 * r(64)
    cq, ck = r(2, 40, 4, 64), r(2, 40, 2, 64)
    tables = tuple(map(_t, _tables(40, 64)))

    def loss(q, k, wq, wk):
        a, b = kernels.qk_norm_rope(q, k, wq, wk, rope=tables)
        return float((a.double() * cq).sum() + (b.double() * ck).sum())

    grads = kernels.qk_norm_rope_backward(cq, ck, q, k, wq, wk, rope=tables)
    at = [q, k, wq, wk]
    h = 1e-2
    for i in range(4):
        d = r(*at[i].shape)
        hi, lo = [t.clone() for t in at], [t.clone() for t in at]
        hi[i] = at[i] + h * d
        lo[i] = at[i] - h * d
        slope = (loss(*hi) - loss(*lo)) / (2 * h)
        want = float((grads[i].double() * d).sum())
        assert abs(slope - want) <= 2e-2 + 5 * h * h * max(1.0, abs(want)), (i, slope, want)


def test_backward_in_place(cuda):
    import torch
    from enilnets_b200 import kernels
    dy, dk = torch.randn((2, 5, 4, 64), device="cuda"), torch.randn((2, 5, 2, 64), device="cuda")
    tables = tuple(map(_t, _tables(5, 64)))
    want = kernels.qk_norm_rope_backward(dy, dk, None, None, rope=tables)
    kernels.qk_norm_rope_backward(dy, dk, None, None, rope=tables, out=(dy, dk))
    assert torch.equal(dy, want[0]) and torch.equal(dk, want[1])


# ------------------------------------------------------------ paged append
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("B,S,H,Hkv,D,page", [(1, 1, 1, 1, 8, 1), (3, 1, 6, 2, 64, 16),
                                              (5, 1, 32, 8, 128, 24), (2, 37, 4, 4, 40, 7),
                                              (3, 100, 5, 1, 96, 64)])
@pytest.mark.parametrize("norm,rope", [(True, True), (False, True), (False, False)])
def test_append(cuda, B, S, H, Hkv, D, page, dtype, norm, rope):
    import torch
    from enilnets_b200 import _native, kernels
    rng = np.random.RandomState(S + D)
    q, k, v, wq, wk = _inputs(S + D, B, S, H, Hkv, D, dtype)
    wq, wk = (wq.astype(np.float32), wk.astype(np.float32)) if norm else (None, None)
    start = rng.randint(0, 40, B).astype(np.int32)
    n_new = rng.randint(0, S + 1, B).astype(np.int32)
    cols = -(-(int(start.max()) + S) // page)
    table = rng.permutation(B * cols + 2)[:B * cols].reshape(B, cols).astype(np.int32)
    kp = torch.full((B * cols + 2, Hkv, page, D), -7.0, dtype=q.dtype, device="cuda")
    vp = kp.clone()
    cos, sin = _tables(int(start.max()) + S, D)
    out = kernels.qk_norm_rope_append(
        q, k, v, kp, vp, torch.from_numpy(table).cuda(), torch.from_numpy(start).cuda(),
        n_new=torch.from_numpy(n_new).cuda(), q_weight=None if wq is None else _t(wq),
        k_weight=None if wk is None else _t(wk), eps=EPS, rope=(_t(cos), _t(sin)) if rope else None)
    torch.cuda.synchronize()
    assert _native.device_error() == (0, 0)
    pos = start[:, None] + np.arange(S)
    c, s = (cos[pos][:, :, None], sin[pos][:, :, None]) if rope else (None, None)
    wantq = ref.norm_rope(_np(q), wq, EPS, c, s)
    wantk = ref.norm_rope(_np(k), wk, EPS, c, s)
    kept = np.full(kp.shape, -7.0)
    keptv = kept.copy()
    for b in range(B):
        wantq[b, n_new[b]:] = 0
        for t in range(n_new[b]):
            at = table[b, pos[b, t] // page], slice(None), pos[b, t] % page
            kept[at] = wantk[b, t]
            keptv[at] = _np(v)[b, t]
    _close(_np(out), wantq, dtype)
    _close(_np(kp), kept, dtype)
    np.testing.assert_array_equal(_np(vp), keptv)  # values are copied, not computed


def test_append_slot_major_pool_and_far_pages(cuda):
    """A pool laid out (page, slot, head), and one whose last page starts past
    2^31 elements."""
    import torch
    from enilnets_b200 import kernels
    B, H, Hkv, D, page = 2, 4, 2, 128, 16
    q, k, v, _, _ = _inputs(1, B, 1, H, Hkv, D, "bf16")
    pages = (1 << 31) // (Hkv * page * D) + 3
    kp = torch.zeros((pages, page, Hkv, D), dtype=torch.bfloat16, device="cuda").permute(0, 2, 1, 3)
    vp = torch.zeros((pages, page, Hkv, D), dtype=torch.bfloat16, device="cuda").permute(0, 2, 1, 3)
    table = torch.tensor([[pages - 1, 5], [3, pages - 2]], dtype=torch.int32, device="cuda")
    start = torch.tensor([3, 16], dtype=torch.int32, device="cuda")
    kernels.qk_norm_rope_append(q, k, v, kp, vp, table, start)
    assert torch.equal(kp[pages - 1, :, 3], k[0, 0]) and torch.equal(vp[pages - 2, :, 0], v[1, 0])
    assert torch.count_nonzero(kp[5]) == 0 and torch.count_nonzero(kp[0]) == 0


@pytest.mark.parametrize("table,start", [([[9]], [0]), ([[-1]], [0]), ([[0]], [16]), ([[0]], [-1])])
def test_append_bad_page_sets_the_device_error(cuda, table, start):
    """A page outside the pool, or a position outside the table: the token is
    not cached, its query is zero, and the device error word says so."""
    import torch
    from enilnets_b200 import _native, kernels
    _native.device_error(clear=True)
    q, k, v, _, _ = _inputs(1, 1, 1, 2, 1, 64, "fp32")
    kp = torch.zeros((4, 1, 16, 64), device="cuda")
    vp = torch.zeros_like(kp)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    out = kernels.qk_norm_rope_append(q, k, v, kp, vp, i32(table), i32(start))
    assert _native.device_error(clear=True)[0] == 2
    assert torch.count_nonzero(out) == 0 and torch.count_nonzero(kp) == 0
    assert torch.count_nonzero(vp) == 0


def test_rotation_outside_the_tables_sets_the_device_error(cuda):
    import torch
    from enilnets_b200 import _native, kernels
    _native.device_error(clear=True)
    q, k, _, _, _ = _inputs(1, 1, 3, 2, 1, 64, "fp32")
    tables = tuple(map(_t, _tables(4, 64)))
    qo, _ = kernels.qk_norm_rope(q, k, rope=tables, pos0=2)
    assert _native.device_error(clear=True) == (2, 2)
    assert torch.count_nonzero(qo[:, 2]) == 0 and torch.count_nonzero(qo[:, :2]) > 0


def test_refusals(cuda):
    import torch
    from enilnets_b200 import kernels
    q, k, v, _, _ = _inputs(1, 2, 3, 4, 2, 64, "fp32")
    w = torch.ones(64, device="cuda")
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    kp = torch.zeros((4, 2, 16, 64), device="cuda")
    tab, st = i32([[0], [1]]), i32([0, 0])
    cases = [
        (lambda: kernels.qk_norm_rope(q, k), "norm weights, rotation tables or both"),
        (lambda: kernels.qk_norm_rope(q, k, w), "come in pairs"),
        (lambda: kernels.qk_norm_rope(q, k, w[:32], w), "q_weight must be"),
        (lambda: kernels.qk_norm_rope(q, k.bfloat16(), w, w), "k must be"),
        (lambda: kernels.qk_norm_rope(q.cpu(), k, w, w), "q must be"),
        (lambda: kernels.qk_norm_rope(q, k[:, :2], w, w), "k must be"),
        (lambda: kernels.qk_norm_rope(q.half(), k.half(), w, w), "q must be"),
        (lambda: kernels.qk_norm_rope(q, k, w, w, rope=(w, w)), "rope cos"),
        (lambda: kernels.qk_norm_rope(q, k, w, w, start=st.long()), "start must be"),
        (lambda: kernels.qk_norm_rope(q[..., 1:], k[..., 1:], w[1:], w[1:]), "head_dim=63"),
        (lambda: kernels.qk_norm_rope_append(q, k, v, kp, kp[:2], tab, st), "must share shape"),
        (lambda: kernels.qk_norm_rope_append(q, k, v, kp.bfloat16(), kp, tab, st), "k_pages must"),
        (lambda: kernels.qk_norm_rope_append(q, k, v, kp, kp, tab.long(), st), "block_table must"),
        (lambda: kernels.qk_norm_rope_append(q, k, v, kp, kp, tab[:1], st), "block_table must"),
        (lambda: kernels.qk_norm_rope_append(q, k, v, kp, kp, tab, st[:1]), "start must be"),
        (lambda: kernels.qk_norm_rope_append(q, k, v[..., :32], kp, kp, tab, st), "v must be"),
        (lambda: kernels.qk_norm_rope_backward(q, k, None, None, w, w), "q must be"),
        (lambda: kernels.qk_norm_rope_backward(q, k, q, k), "norm weights, rotation tables"),
    ]
    for call, message in cases:
        with pytest.raises(ValueError, match=message):
            call()


def test_backward_refuses_inputs_of_other_types(cuda):
    """Without weights the inputs are not read, but their type names the
    gradients'."""
    import torch
    from enilnets_b200 import kernels
    dq, dk = torch.ones((1, 3, 2, 64), device="cuda"), torch.ones((1, 3, 1, 64), device="cuda")
    tables = tuple(map(_t, _tables(3, 64)))
    for out in (None, (torch.empty_like(dq), torch.empty_like(dk))):
        with pytest.raises(ValueError, match="q must be"):
            kernels.qk_norm_rope_backward(dq, dk, dq.half(), dk.half(), rope=tables, out=out)


def test_counts_past_32_bits_are_refused(cuda):
    """A broadcast view of 2^32 + 1 tokens is no call for one token."""
    import torch
    from enilnets_b200 import kernels
    S = (1 << 32) + 1
    q, k = (torch.ones((1, 1, h, 64), device="cuda") for h in (2, 1))
    far = [t.expand(1, S, -1, -1) for t in (q, k)]
    w = torch.full((64,), 2.0, device="cuda")
    with pytest.raises(ValueError, match="below 2\\^31"):
        kernels.qk_norm_rope(*far, w, w, out=tuple(far))
    with pytest.raises(ValueError, match="below 2\\^31"):
        kernels.qk_norm_rope_backward(*far, *far, w, w, out=tuple(far))
    assert (q == 1).all() and (k == 1).all()


def test_empty_batches(cuda):
    import torch
    from enilnets_b200 import kernels
    w = torch.ones(64, device="cuda")
    q, k = torch.empty((0, 3, 4, 64), device="cuda"), torch.empty((0, 3, 2, 64), device="cuda")
    qo, ko = kernels.qk_norm_rope(q, k, w, w)
    assert qo.shape == q.shape and ko.shape == k.shape
    _, _, dw, _ = kernels.qk_norm_rope_backward(q, k, q, k, w, w)
    assert torch.count_nonzero(dw) == 0


def test_other_stream(cuda):
    """A call on a side stream sees what that stream computed before it."""
    import torch
    from enilnets_b200 import kernels
    w = torch.ones(128, device="cuda")
    x = torch.randn((4, 512, 8, 128), device="cuda")
    want, _ = kernels.qk_norm_rope(x * 3, x, w, w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = x * 3
        got, _ = kernels.qk_norm_rope(y, x, w, w)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
