"""Paged attention of one new token against the float64 oracle on the values
the kernel reads.

Tolerances, for unit-variance values and outputs below 5 in size. fp32: scores
and sums in fp32 (or products split into parts that carry 21 bits or more), so
an error below 1e-5. bf16 inputs are exact in the oracle too; a bf16 output is
rounded once, at most 2^-9 of it: 2^-8 |o| + 1e-5. LSE: 1e-5 absolute at values
up to about 15.
"""
import numpy as np
import pytest

from oracle import attention_ref as aref
from oracle import serving_ref as ref

pytestmark = pytest.mark.gpu


def _np(t):
    return t.detach().double().cpu().numpy()


def _i32(x):
    import torch
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def _case(seed, lens, H, Hkv, D, page, dtype, slot_major=False, spare=2):
    """q, pools and a shuffled block table; unused slots and pages hold NaN."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    B = len(lens)
    cols = max(1, max(-(-n // page) for n in lens))
    total = B * cols + spare
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    table = torch.randperm(total, device="cuda", generator=g)[:B * cols].reshape(B, cols).int()
    shape = (total, page, Hkv, D) if slot_major else (total, Hkv, page, D)
    pools = [torch.full(shape, float("nan"), device="cuda", dtype=dt) for _ in range(2)]
    if slot_major:
        pools = [p.permute(0, 2, 1, 3) for p in pools]
    for p in pools:
        for b, n in enumerate(lens):
            j = torch.arange(n, device="cuda")
            p[table[b].long()[j // page], :, j % page] = torch.randn(
                (n, Hkv, D), device="cuda", generator=g).to(dt)
    q = torch.randn((B, H, D), device="cuda", generator=g).to(dt)
    return q, pools[0], pools[1], table, _i32(lens)


def _check(q, kp, vp, table, lens, out, lse, **kw):
    import torch
    from enilnets_b200 import _native
    torch.cuda.synchronize()
    assert _native.device_error() == (0, 0)
    oref, lref = ref.paged_decode(_np(q), _np(kp), _np(vp), table.cpu().numpy(),
                                  lens.cpu().numpy(), **kw)
    o = _np(out)
    tol = 1e-5 + (2.0 ** -8 * np.abs(oref) if out.dtype == torch.bfloat16 else 0.0)
    assert np.isfinite(o).all()
    bad = ~(np.abs(o - oref) <= tol)
    assert not bad.any(), f"{bad.sum()} off, worst {np.abs(o - oref).max():.3e}"
    got = _np(lse)
    empty = np.isneginf(lref)
    assert np.isneginf(got[empty]).all()
    assert np.abs(got[~empty] - lref[~empty]).max(initial=0) <= 1e-5


def _run(case, out_dtype=None, **kw):
    from enilnets_b200 import kernels
    return kernels.attention_decode_paged(*case, out_dtype=out_dtype, return_lse=True, **kw)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("D", [8, 40, 64, 80, 128])
@pytest.mark.parametrize("Hkv,G", [(1, 1), (2, 2), (2, 3), (1, 5), (3, 8), (1, 16), (2, 20)])
def test_heads_and_dims(cuda, dtype, D, Hkv, G):
    case = _case(D + G, [1, 100, 0, 333], Hkv * G, Hkv, D, 16, dtype)
    import torch
    out, lse = _run(case, out_dtype=torch.float32)
    _check(*case, out, lse)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("page", [1, 7, 8, 16, 24, 64, 128, 300])
def test_pages_and_lengths(cuda, dtype, page):
    """Lengths on and around page, tile and split ends, and empty rows."""
    lens = [0, 1, page - 1, page, page + 1, 63, 64, 65, 127, 128, 129, 255, 257, 513, 1000, 0]
    case = _case(page, lens, 8, 2, 64, page, dtype)
    out, lse = _run(case)
    _check(*case, out, lse)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (0, 3), (1, 1), (15, 0), (16, 4), (100, 37),
                                          (499, 64), (5000, 4)])
def test_window_and_sinks(cuda, dtype, window, sinks):
    case = _case(window + sinks, [1, 2, 17, 130, 500, 900, 0, 64], 6, 2, 64, 24, dtype)
    out, lse = _run(case, window=window, sinks=sinks)
    _check(*case, out, lse, window=window, sinks=sinks)


def test_windows_past_32_bits(cuda):
    """A window of 2^32 sees everything, 2^32 first tokens are all of them."""
    import torch
    case = _case(4, [1, 300, 77], 8, 4, 64, 16, "bf16")
    want, lse = _run(case)
    for kw in (dict(window=1 << 32), dict(window=(1 << 32) + 3, sinks=1),
               dict(window=2, sinks=1 << 32)):
        out, got = _run(case, **kw)
        assert torch.equal(out, want) and torch.equal(got, lse), kw


def test_alibi_scale_and_window(cuda):
    import torch
    case = _case(3, [400, 31, 1], 8, 4, 128, 16, "fp32")
    slopes = aref.alibi_slopes(8).astype(np.float32)
    t = torch.from_numpy(slopes).cuda()
    for kw in (dict(), dict(window=50, sinks=2), dict(scale=0.3)):
        out, lse = _run(case, alibi_slopes=t, **kw)
        _check(*case, out, lse, slopes=slopes.astype(np.float64), **kw)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_long_uneven_batch(cuda, dtype):
    """One long sequence beside short ones: the long one is shared by many
    blocks, whose parts are joined."""
    case = _case(11, [9001, 3, 0, 700, 4096], 8, 2, 128, 16, dtype)
    out, lse = _run(case)
    _check(*case, out, lse)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("D", [64, 128])
def test_long_sums_are_not_cut(cuda, dtype, D):
    """Equal values of one sign over a long sequence: the output is that value.
    Sums that were cut towards zero instead of rounded would fall short by the
    number of additions times 2^-24; rounded ones stay within sqrt of it, checked
    at 1e-6 (bf16 inputs included: the output is fp32)."""
    import torch
    from enilnets_b200 import kernels
    q, kp, vp, table, lens = _case(40, [16000], 64, 64, D, 16, dtype)  # long runs per block
    kp = torch.where(torch.isnan(kp), kp, 0.01 * kp)
    value = 1.0 + torch.rand((D,), device="cuda").to(vp.dtype)
    vp = torch.where(torch.isnan(vp), vp, value)
    out = kernels.attention_decode_paged(q, kp, vp, table, lens, out_dtype=torch.float32)
    want = value.double()
    assert ((out[0].double() - want).abs() / want).max() <= 1e-6


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("G", [2, 4, 8])
def test_long_sums_are_not_cut_in_groups(cuda, D, G):
    """The same in fp32 for groups of query heads, whose products take other
    pipes than single heads'; the bound's reason is the same."""
    import torch
    from enilnets_b200 import kernels
    q, kp, vp, table, lens = _case(41, [16000], 64 * G, 64, D, 16, "fp32")
    kp = torch.where(torch.isnan(kp), kp, 0.01 * kp)
    value = 1.0 + torch.rand((D,), device="cuda").to(vp.dtype)
    vp = torch.where(torch.isnan(vp), vp, value)
    out = kernels.attention_decode_paged(q, kp, vp, table, lens, out_dtype=torch.float32)
    want = value.double()
    assert ((out[0].double() - want).abs() / want).max() <= 1e-6


def test_many_sequences(cuda):
    """More (sequence, head) pairs than blocks: several whole ones each."""
    lens = list(np.random.RandomState(0).randint(0, 90, 300))
    case = _case(12, lens, 8, 4, 64, 8, "bf16")
    out, lse = _run(case)
    _check(*case, out, lse)


def test_slot_major_pool_and_strided_tensors(cuda):
    """A (page, slot, head) pool; q and out as views of wider tensors; block
    table rows inside a wider table."""
    import torch
    q, kp, vp, table, lens = _case(13, [77, 300], 4, 2, 64, 16, "bf16", slot_major=True)
    wide = torch.randn((2, 3, 4, 64), device="cuda").bfloat16()
    wide[:, 1] = q
    big = torch.full((2, table.shape[1] + 5), -1, dtype=torch.int32, device="cuda")
    big[:, :table.shape[1]] = table
    out = torch.zeros((2, 2, 4, 64), device="cuda", dtype=torch.bfloat16)
    from enilnets_b200 import kernels
    _, lse = kernels.attention_decode_paged(wide[:, 1], kp, vp, big, lens, out=out[:, 1],
                                            return_lse=True)
    _check(q, kp, vp, table, lens, out[:, 1], lse)
    assert torch.count_nonzero(out[:, 0]) == 0


def test_offsets_past_32_bits(cuda):
    """Pages that start past 2^31 elements (and 2^32 bytes) of the pool."""
    import torch
    from enilnets_b200 import kernels
    q, kp, vp, table, lens = _case(14, [40, 33], 4, 2, 128, 16, "bf16", spare=0)
    pages = (1 << 31) // (2 * 16 * 128) + 8
    far_k = torch.empty((pages, 2, 16, 128), dtype=torch.bfloat16, device="cuda")
    far_v = torch.empty_like(far_k)
    n = kp.shape[0]
    far_k[pages - n:], far_v[pages - n:] = kp, vp
    out, lse = kernels.attention_decode_paged(q, far_k, far_v, table + (pages - n), lens,
                                              return_lse=True)
    _check(q, kp, vp, table, lens, out, lse)


@pytest.mark.parametrize("dtype,short", [("bf16", 0), ("bf16", 60), ("fp32", 0)])
def test_lengths_up_to_the_last_positions(cuda, dtype, short):
    """A sequence that ends within a tile of 2^31 positions, all of them one page:
    the output is that page's (short: of the page without its last slots, in all but
    a 42966th of the weight). Each of some 10^5 additions rounds by 2^-24: 1e-4
    covers them with the short page's 3e-5."""
    import torch
    from enilnets_b200 import kernels
    page, pages = 49981, 42966  # 2^31 - 2
    q, kp, vp, _, _ = _case(80, [page], 2, 1, 8, page, dtype, spare=0)
    table = torch.zeros((1, pages), dtype=torch.int32, device="cuda")
    out, lse = kernels.attention_decode_paged(q, kp, vp, table, _i32([page * pages - short]),
                                              out_dtype=torch.float32, return_lse=True)
    want, one = ref.paged_decode(_np(q), _np(kp), _np(vp), np.zeros((1, 1), int), [page])
    assert np.abs(_np(out) - want).max() <= 1e-4
    assert np.abs(_np(lse) - one - np.log(pages)).max() <= 1e-4


def test_extreme_scores(cuda):
    """Scores far apart: the largest takes all, nothing overflows; equal
    scores average; -inf and +inf keys in masked slots do not leak."""
    import torch
    from enilnets_b200 import kernels
    q, kp, vp, table, lens = _case(15, [200], 1, 1, 64, 16, "fp32")
    q[:] = 100.0
    kp[torch.isfinite(kp)] = 0.0
    kp[table[0, 5], 0, 2] = 10.0    # position 82 scores 8000 above the others
    kp[table[0, 12], 0, 9] = float("inf")   # past the end (200 = 12 * 16 + 8)
    vp[table[0, 12], 0, 9] = float("-inf")
    out, lse = kernels.attention_decode_paged(q, kp, vp, table, lens, return_lse=True)
    torch.cuda.synchronize()
    assert torch.equal(out[0, 0], vp[table[0, 5], 0, 2])
    assert abs(float(lse) - 8000.0) <= 8000 * 2.0 ** -20
    kp[table[0, 5], 0, 2] = 0.0
    out, _ = kernels.attention_decode_paged(q, kp, vp, table, lens, return_lse=True)
    _check(q, torch.where(torch.isfinite(kp), kp, 0 * q[0, 0]), vp, table, lens, out,
           torch.log(torch.tensor([[200.0]], device="cuda")))


def _check_infinite_value(dtype, D, G, window=None):
    """One infinite value among visible keys: that dim of the output is infinite
    for every query head of the key head, the other dims are the oracle's; a
    second one of the other sign makes it NaN; outside the window it changes
    nothing. A key whose score is minus infinity has no weight."""
    import torch
    from enilnets_b200 import kernels
    H, inf = 2 * G, float("inf")
    q, kp, vp, table, lens = _case(D + G, [200, 37], H, 2, D, 16, dtype)
    kw = dict(out_dtype=torch.float32, return_lse=True, window=window)
    plain, _ = kernels.attention_decode_paged(q, kp, vp, table, lens, **kw)
    at = (table[0, 11].long(), 1, 9)  # position 185 of the first sequence, its second key head
    for value in (inf, -inf):
        v = vp.clone()
        v[at][5] = value
        out, lse = kernels.attention_decode_paged(q, kp, v, table, lens, **kw)
        assert (out[0, G:, 5] == value).all()
        out[0, G:, 5] = plain[0, G:, 5]
        _check(q, kp, vp, table, lens, out, lse, window=window)
        v[table[0, 10].long(), 1, 3, 5] = -value
        out, _ = kernels.attention_decode_paged(q, kp, v, table, lens, **kw)
        assert torch.isnan(out[0, G:, 5]).all()
        assert torch.isfinite(out).sum() == out.numel() - G
        if window is not None:
            v = vp.clone()
            v[table[0, 1].long(), 1, 3, 5] = value
            out, _ = kernels.attention_decode_paged(q, kp, v, table, lens, **kw)
            assert torch.equal(out, plain)
        k, qq = kp.clone(), q.clone()
        k[at][7] = value
        qq[0, :, 7] = -np.sign(value) * (qq[0, :, 7].abs() + 0.1)
        qq[0, G, 7] = -np.sign(value)  # a power of two
        out, lse = kernels.attention_decode_paged(qq, k, vp, table, lens, **kw)
        _check(qq, k, vp, table, lens, out, lse, window=window)


@pytest.mark.parametrize("D", [40, 64, 128])
@pytest.mark.parametrize("G", [1, 4, 8, 16, 20])
@pytest.mark.parametrize("window", [None, 50])
def test_infinite_values_in_bf16(cuda, D, G, window):
    _check_infinite_value("bf16", D, G, window)


@pytest.mark.parametrize("D", [40, 64, 128])
@pytest.mark.parametrize("G", [1, 2, 4, 5, 8, 16])
@pytest.mark.parametrize("window", [None, 50])
def test_infinite_values_in_fp32(cuda, D, G, window):
    _check_infinite_value("fp32", D, G, window)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("G", [1, 4, 8, 16])
def test_bf16_probabilities_keep_their_bits(cuda, D, G):
    """An fp32 output from bf16 keys and values. A score below 16 in base 2 has
    an error of at most 2^-20, a weight 2^-20 ln 2 and the exponential's 2^-22: 9e-7
    at most, and the sum's roundings less."""
    import torch
    from enilnets_b200 import kernels
    q, kp, vp, table, lens = _case(70, [4000], G, 1, D, 16, "bf16")
    out = kernels.attention_decode_paged(q, kp, vp, table, lens, out_dtype=torch.float32)
    k, v = (p[table[0].long(), 0].reshape(-1, D)[:4000].double() for p in (kp, vp))
    want = torch.softmax(q[0].double() @ k.T / D ** 0.5, -1) @ v
    assert float((out[0].double() - want).norm() / want.norm()) <= 9e-7


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hkv", [8, 64])
def test_long_sums_are_not_cut_in_wide_groups(cuda, D, Hkv):
    """As test_long_sums_are_not_cut, for bf16 groups of 16 query heads."""
    import torch
    from enilnets_b200 import kernels
    q, kp, vp, table, lens = _case(42, [16000], 16 * Hkv, Hkv, D, 16, "bf16")
    kp = torch.where(torch.isnan(kp), kp, 0.01 * kp)
    value = 1.0 + torch.rand((D,), device="cuda").to(vp.dtype)
    vp = torch.where(torch.isnan(vp), vp, value)
    out = kernels.attention_decode_paged(q, kp, vp, table, lens, out_dtype=torch.float32)
    want = value.double()
    assert ((out[0].double() - want).abs() / want).max() <= 1e-6


@pytest.mark.parametrize("bad", [-1, 99])
def test_bad_page_counts_as_masked(cuda, bad):
    import torch
    from enilnets_b200 import _native, kernels
    q, kp, vp, table, lens = _case(16, [40], 2, 1, 64, 16, "bf16")
    _native.device_error(clear=True)
    table[0, 1] = bad  # positions 16..31
    out = kernels.attention_decode_paged(q, kp, vp, table, lens, out_dtype=torch.float32)
    assert _native.device_error(clear=True)[0] == 2
    K, V = _np(kp), _np(vp)
    rows = [(int(table[0, j // 16]), j % 16) for j in list(range(16)) + list(range(32, 40))]
    k = np.stack([K[p, 0, s] for p, s in rows])
    v = np.stack([V[p, 0, s] for p, s in rows])
    s = _np(q)[0] @ k.T / 8.0
    w = np.exp(s - s.max(-1, keepdims=True))
    assert np.abs(_np(out)[0] - w @ v / w.sum(-1, keepdims=True)).max() <= 1e-5


def test_length_past_the_table_is_cut(cuda):
    import torch
    from enilnets_b200 import _native, kernels
    q, kp, vp, table, lens = _case(17, [48], 2, 1, 64, 16, "fp32")
    want = kernels.attention_decode_paged(q, kp, vp, table, lens)
    _native.device_error(clear=True)
    got = kernels.attention_decode_paged(q, kp, vp, table, _i32([1000]))
    assert _native.device_error(clear=True)[0] == 2
    assert torch.equal(got, want)
    got = kernels.attention_decode_paged(q, kp, vp, table, _i32([-5]))
    assert torch.count_nonzero(got) == 0 and _native.device_error() == (0, 0)


def test_repeats_and_other_shapes_on_one_workspace(cuda):
    """The same bits every time, whatever ran on the workspace in between."""
    import torch
    from enilnets_b200 import kernels
    a = _case(18, [5000, 17, 900], 8, 2, 128, 16, "bf16")
    b = _case(19, list(range(64)), 40, 8, 64, 8, "fp32")
    first = kernels.attention_decode_paged(*a), kernels.attention_decode_paged(*b)
    for _ in range(20):
        again = kernels.attention_decode_paged(*a), kernels.attention_decode_paged(*b)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_streams_have_their_own_workspace(cuda):
    import torch
    from enilnets_b200 import kernels
    cases = [_case(20 + i, [6000 - 900 * i, 40], 8, 2, 128, 16, "bf16") for i in range(3)]
    want = [kernels.attention_decode_paged(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(10):
        got = []
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(kernels.attention_decode_paged(*c))
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_graph_replay_with_growing_lengths(cuda):
    """One captured call serves every step: lengths and pages are read on the
    device."""
    import torch
    from enilnets_b200 import kernels
    q, kp, vp, table, full = _case(30, [700, 300], 8, 2, 64, 16, "bf16")
    lens = _i32([1, 1])
    ws = torch.zeros(kernels.paged_decode_workspace_bytes(2, 8, 2, 64), dtype=torch.uint8,
                     device="cuda")
    out = torch.empty_like(q)
    kernels.attention_decode_paged(q, kp, vp, table, lens, out=out, workspace=ws)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kernels.attention_decode_paged(q, kp, vp, table, lens, out=out, workspace=ws)
    for step in ([700, 300], [5, 299], [0, 64], [1, 1]):
        lens.copy_(_i32(step))
        g.replay()
        assert torch.equal(out, kernels.attention_decode_paged(q, kp, vp, table, lens)), step


def _captured(case, stream):
    """(graph, its output) of one call with the default workspace."""
    import torch
    from enilnets_b200 import kernels
    out = torch.zeros_like(case[0])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        kernels.attention_decode_paged(*case, out=out)
    return g, out


def test_graphs_do_not_share_the_streams_workspace(cuda):
    """Graphs captured on one stream with the default workspace, from the largest
    batch down and replayed in the other order, with the stream's own calls in
    between and whatever the memory held before."""
    import torch
    from enilnets_b200 import kernels
    cases = [_case(50 + n, [900 + 10 * i for i in range(n)], 8, 2, 64, 16, "bf16")
             for n in (40, 8, 2)]
    want = [kernels.attention_decode_paged(*c) for c in cases]
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    graphs = [_captured(c, stream) for c in cases]
    kept = kernels._zeroed.get((torch.cuda.current_device(), stream.cuda_stream))
    if kept is not None:  # made under capture, not zeroed before the first graph replays
        kept.fill_(255)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        for _ in range(3):
            for (g, out), w, c in zip(graphs[::-1], want[::-1], cases[::-1]):
                out.zero_()
                g.replay()
                eager = kernels.attention_decode_paged(*c)
                stream.synchronize()
                assert torch.equal(out, w) and torch.equal(eager, w)


@pytest.mark.parametrize("B,H,Hkv", [(2, 8, 2), (3, 40, 2), (65, 9, 1), (20, 16, 16)])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_only_the_counters_need_zeros(cuda, dtype, B, H, Hkv):
    import torch
    from enilnets_b200 import kernels
    case = _case(B, [2000 + 7 * i for i in range(B)], H, Hkv, 64, 16, dtype)
    n = kernels.paged_decode_workspace_bytes(B, H, Hkv, 64)
    ws = torch.full((n,), 255, dtype=torch.uint8, device="cuda")
    ws[n - kernels._paged_counter_bytes(B, H, Hkv):] = 0
    want = kernels.attention_decode_paged(*case)
    for _ in range(2):
        assert torch.equal(kernels.attention_decode_paged(*case, workspace=ws), want)


def test_graph_keeps_its_workspace_when_the_streams_grows(cuda):
    """A graph captured after a small eager call; a larger one then replaces the
    stream's workspace, whose memory goes to the next tensor of its size."""
    import torch
    from enilnets_b200 import kernels
    small = _case(60, [700, 300], 8, 2, 64, 16, "bf16")
    large = _case(61, [300] * 64, 8, 2, 64, 16, "bf16")
    want = kernels.attention_decode_paged(*small)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        kernels.attention_decode_paged(*small)
        stream.synchronize()
        g, out = _captured(small, stream)
        n = kernels.paged_decode_workspace_bytes(2, 8, 2, 64)
        kernels.attention_decode_paged(*large)
        others = [torch.full((n,), 255, dtype=torch.uint8, device="cuda") for _ in range(4)]
        g.replay()
        stream.synchronize()
        assert torch.equal(out, want)
        assert all((t == 255).all() for t in others)


def test_refusals(cuda):
    import torch
    from enilnets_b200 import kernels
    q, kp, vp, table, lens = _case(31, [20, 30], 4, 2, 64, 16, "bf16")
    f = kernels.attention_decode_paged
    cases = [
        (lambda: f(q.float(), kp, vp, table, lens), "k_pages must"),
        (lambda: f(q[0], kp, vp, table, lens), "q must be"),
        (lambda: f(q.cpu(), kp, vp, table, lens), "q must be"),
        (lambda: f(q.half(), kp, vp, table, lens), "q must be"),
        (lambda: f(q, kp, vp[:1], table, lens), "must share shape"),
        (lambda: f(q, kp, vp.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3), table, lens),
         "strides"),
        (lambda: f(q, kp, vp, table.long(), lens), "block_table must"),
        (lambda: f(q, kp, vp, table[:1], lens), "block_table must"),
        (lambda: f(q, kp, vp, table, lens.long()), "seq_lens must"),
        (lambda: f(q, kp, vp, table, lens[:1]), "seq_lens must"),
        (lambda: f(q, kp, vp, table, lens, window=-1), "window must"),
        (lambda: f(q, kp, vp, table, lens, sinks=2), "needs a window"),
        (lambda: f(q, kp, vp, table, lens, window=3, sinks=-2), "sinks=-2"),
        (lambda: f(q[:, :3], kp, vp, table, lens), "must divide"),
        (lambda: f(q, kp, vp, table, lens, alibi_slopes=torch.ones(3, device="cuda")),
         "alibi_slopes must"),
        (lambda: f(q, kp, vp, table, lens, out=torch.empty((2, 4, 32), device="cuda")), "out must"),
        (lambda: f(q, kp, vp, table, lens,
                   workspace=torch.zeros(16, dtype=torch.uint8, device="cuda")), "workspace"),
    ]
    for call, message in cases:
        with pytest.raises(ValueError, match=message):
            call()
    assert f(q[:0], kp, vp, table[:0], lens[:0]).shape == (0, 4, 64)
