"""GPU: linear_cross_entropy (ceeg_linear_ce_fwd / _bwd) against its formula in 64 bits.

Bounds, with u = 2^-24 and S = sum_k |h_k w_k|: a logit is off by at most H u S (fp32 sums of exact bf16 products; fp32 inputs are three bf16
pieces with six products: 6 H u S, which covers the 2^-24 S that the dropped products are worth), an exponential by |x| 2^-23 + 2^-22 of itself.
dl adds half a step of bf16 (2^-8 of it) for bf16 inputs and three pieces' 2^-24 for fp32; a sum of n terms n u of their magnitudes (6 n u for
fp32); the store half a step of the output's type."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _inputs(T, H, V, dtype, seed=0, ignored=0.3, scale=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + T * 31 + H * 17 + V)
    h = torch.randn(T, H, generator=g, device="cuda").to(dtype)
    w = (torch.randn(V, H, generator=g, device="cuda") * (scale / H ** 0.5)).to(dtype)
    y = torch.randint(0, V, (T,), generator=g, device="cuda")
    y[torch.rand(T, generator=g, device="cuda") < ignored] = -100
    return h, w, y


def _check(h, w, y, loss, dh, dw, reduction, g, ignore=-100):
    """loss, dh and dw against the formula, element by element."""
    f32 = h.dtype == torch.float32
    keep = y != ignore
    hd, wd = torch.where(keep[:, None], h.double(), torch.zeros((), dtype=torch.float64, device="cuda")), w.double()
    (T, H), V = hd.shape, wd.shape[0]
    z = hd @ wd.t()
    lse = torch.logsumexp(z, 1)
    at = torch.where(keep, y, torch.zeros_like(y))
    rows = torch.where(keep, lse - z.gather(1, at[:, None])[:, 0], torch.zeros_like(lse))
    n = max(int(keep.sum()), 1)
    terms = (6 if f32 else 1) * H
    e_z = terms * U * float((hd.abs() @ wd.abs().t()).max())
    e_exp = float((z - lse[:, None]).abs().max() + 40) * 2 ** -23 + 2 ** -22   # the sum is rescaled when pieces are joined: once more |x| <= 40
    e_loss = 2 * e_z + e_exp + V * U
    if reduction == "none":
        assert bool(((loss.double() - rows).abs() <= e_loss + 2 * U * rows.abs() + U * (lse.abs() + z.abs().amax(1))).all())
        assert bool((loss[~keep] == 0).all())
    else:
        want = rows.sum() / (n if reduction == "mean" else 1)
        share = 1 if reduction == "mean" else int(keep.sum())
        assert abs(float(loss.double() - want)) <= share * (e_loss + U * float(lse.abs().max() + z.abs().max())) + 2 * U * abs(float(want))
    if dh is None and dw is None:
        return
    up = torch.where(keep, g.double().expand(T) / (n if reduction == "mean" else 1), torch.zeros((), dtype=torch.float64, device="cuda"))
    p = torch.exp(z - lse[:, None])
    hot = torch.zeros_like(p).scatter_(1, at[:, None], 1.0)
    dl = up[:, None] * (p - hot)
    size = up.abs()[:, None] * (p + hot)
    e_dl = 2 * e_z + 2 * e_exp + V * U + (4 * U if f32 else 2 ** -8)
    for got, want, bound, n_sum in ((dh, dl @ wd, size @ wd.abs(), V), (dw, dl.t() @ hd, size.t() @ hd.abs(), T)):
        if got is None:
            continue
        tol = (e_dl + (6 if f32 else 1) * n_sum * U + 8 * U) * bound + torch.finfo(got.dtype).eps / 2 * want.abs() + 1e-38
        assert bool(torch.isfinite(got).all())
        off = (got.double() - want).abs() - tol
        assert float(off.max()) <= 0, f"off by {float(off.max())} more than {float(tol.flatten()[off.argmax()])}"


def _run(h, w, y, reduction="mean", g=None, ignore=-100):
    from causal_eeg_vae_amd import linear_cross_entropy
    a, b = h.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss = linear_cross_entropy(a, b, y, ignore_index=ignore, reduction=reduction)
    g = torch.ones_like(loss) if g is None else g
    dh, dw = torch.autograd.grad(loss, (a, b), g)
    return loss.detach(), dh, dw, g


SIZES = [(1, 64, 512), (1, 8, 1), (2, 1, 3), (63, 65, 127), (64, 64, 128), (97, 64, 512), (130, 77, 1000), (257, 128, 129), (128, 192, 4096), (300, 96, 20001),
         (1000, 40, 257)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("T,H,V", SIZES)
def test_mean_and_its_gradients(T, H, V, dtype):
    h, w, y = _inputs(T, H, V, dtype)
    y[0] = V - 1
    loss, dh, dw, g = _run(h, w, y)
    _check(h, w, y, loss, dh, dw, "mean", g)
    assert loss.dtype == torch.float32 and dh.dtype == dtype and dw.dtype == dtype
    assert bool((dh[y == -100] == 0).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("T,H,V", [(2100, 576, 25701), (700, 640, 9001), (3001, 129, 5003)])
def test_every_tile_shape(T, H, V, dtype):
    """Grids large enough for the larger tiles in each of the four products, with edges inside the last tile on every side."""
    h, w, y = _inputs(T, H, V, dtype, ignored=0.1)
    loss, dh, dw, g = _run(h, w, y)
    _check(h, w, y, loss, dh, dw, "mean", g)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("T,H,V", [(3, 32768, 5), (70000, 5, 3), (2, 16, 1200000)])
def test_one_long_side(T, H, V, dtype):
    """The widest rows there may be, many tokens of few classes, more classes than a piece holds."""
    h, w, y = _inputs(T, H, V, dtype)
    loss, dh, dw, g = _run(h, w, y)
    _check(h, w, y, loss, dh, dw, "mean", g)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_reductions_and_upstream_gradients(reduction, dtype):
    h, w, y = _inputs(200, 72, 777, dtype, seed=3)
    gen = torch.Generator(device="cuda").manual_seed(5)
    g = torch.randn(200, generator=gen, device="cuda") * 3 if reduction == "none" else torch.tensor(-0.37, device="cuda")
    loss, dh, dw, g = _run(h, w, y, reduction, g)
    _check(h, w, y, loss, dh, dw, reduction, g)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("T,H,V", [(1, 129, 65), (2, 64, 4097), (3, 77, 63), (4, 768, 1030), (5, 8, 128), (7, 1538, 100), (8, 192, 5003), (9, 192, 5003), (1, 12352, 70), (6, 2100, 257)])
def test_few_tokens(T, H, V, reduction, dtype):
    """Up to eight tokens, where the vocabulary's rows are read as they are, and its edges; the last token is ignored, so that a single one leaves none."""
    h, w, y = _inputs(T, H, V, dtype, ignored=0.0)
    y[-1] = -100
    h[-1] = float("nan")
    g = torch.linspace(-1.5, 2.0, T, device="cuda") if reduction == "none" else torch.tensor(0.7, device="cuda")
    loss, dh, dw, g = _run(h, w, y, reduction, g)
    _check(h, w, y, loss, dh, dw, reduction, g)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_few_tokens_strided_and_out_of_range(dtype):
    from causal_eeg_vae_amd import linear_cross_entropy
    h, w, y = _inputs(6, 192, 1000, dtype, ignored=0.0)
    want = _run(h, w, y)
    wide = torch.full((6, 201), 9.0, dtype=dtype, device="cuda")
    wide[:, 3:195] = h
    base = torch.zeros(1000 * 192 + 1, dtype=dtype, device="cuda")
    base[1:] = w.reshape(-1)
    loose = torch.full((1000, 195), float("inf"), dtype=dtype, device="cuda")
    loose[:, :192] = w
    for a in (wide[:, 3:195], h):
        for b in (base[1:].view(1000, 192), loose[:, :192], w):
            for x, z in zip(_run(a, b, y), want):
                assert torch.equal(x, z)
    rows = linear_cross_entropy(h, w, y, reduction="none")
    y[2], y[4] = 1000, -1
    bad = linear_cross_entropy(h, w, y, reduction="none")
    odd = torch.tensor([False, False, True, False, True, False], device="cuda")
    assert torch.equal(bad.isnan(), odd) and torch.equal(bad[~odd], rows[~odd])


def test_no_upstream_gradient_is_zero():
    h, w, y = _inputs(50, 64, 300, torch.bfloat16)
    for reduction, g in (("none", torch.zeros(50, device="cuda")), ("sum", torch.zeros((), device="cuda"))):
        _, dh, dw, _ = _run(h, w, y, reduction, g)
        assert not bool(dh.any()) and not bool(dw.any())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_pieces_of_the_vocabulary(dtype):
    """More columns than one piece of the backward holds (its workspace is capped): 1 GiB / (planes * 4 bytes * tokens) columns."""
    from causal_eeg_vae_amd import _lib
    T, H, V = (4096, 16, 30001) if dtype == torch.float32 else (16384, 64, 20003)
    code = _lib.CEEG_F32 if dtype == torch.float32 else _lib.CEEG_BF16
    assert _lib.lib().ceeg_linear_ce_bwd_ws_bytes(T, H, 2 * V, code) < 1.5 * _lib.lib().ceeg_linear_ce_bwd_ws_bytes(T, H, V, code)
    h, w, y = _inputs(T, H, V, dtype, ignored=0.05)
    loss, dh, dw, g = _run(h, w, y)
    _check(h, w, y, loss, dh, dw, "mean", g)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_every_token_ignored(reduction):
    h, w, y = _inputs(70, 64, 300, torch.bfloat16)
    y.fill_(-100)
    loss, dh, dw, _ = _run(h, w, y, reduction)
    assert not bool(loss.any()) and not bool(dh.any()) and not bool(dw.any())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_ignored_rows_may_hold_anything(dtype):
    h, w, y = _inputs(150, 64, 300, dtype)
    clean = _run(h, w, y)
    dirty = h.clone()
    dirty[y == -100] = float("nan")
    dirty[(y == -100).nonzero()[0]] = float("inf")
    for a, b in zip(clean, _run(dirty, w, y)):
        assert torch.equal(a, b)


def test_another_ignore_index_and_ranked_inputs():
    """A batch of padded sequences, shifted by one as a language model's loss is: hidden[:, :-1] against target[:, 1:], both strided views."""
    from causal_eeg_vae_amd import linear_cross_entropy
    B, L, H, V = 5, 33, 96, 1003
    g = torch.Generator(device="cuda").manual_seed(1)
    hidden = torch.randn(B, L, H, generator=g, device="cuda").bfloat16().requires_grad_(True)
    w = (torch.randn(V, H, generator=g, device="cuda") / H ** 0.5).bfloat16().requires_grad_(True)
    ids = torch.randint(1, V, (B, L), generator=g, device="cuda")
    ids[:, 25:] = 0
    loss = linear_cross_entropy(hidden[:, :-1], w, ids[:, 1:], ignore_index=0)
    dh, dw = torch.autograd.grad(loss, (hidden, w))
    assert dh.shape == hidden.shape and not bool(dh[:, -1].any())
    _check(hidden.detach()[:, :-1].reshape(-1, H), w.detach(), ids[:, 1:].reshape(-1), loss.detach(), dh[:, :-1].reshape(-1, H), dw, "mean", torch.ones((), device="cuda"), ignore=0)
    rows = linear_cross_entropy(hidden.detach()[:, :-1], w.detach(), ids[:, 1:], ignore_index=0, reduction="none")
    assert rows.shape == (B, L - 1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_strides_and_alignment(dtype):
    """Rows of a wider buffer, a base that is not 16-byte aligned, a transposed weight: the same numbers as the contiguous call's."""
    h, w, y = _inputs(77, 64, 333, dtype)
    want = _run(h, w, y)
    wide = torch.full((77, 71), 9.0, dtype=dtype, device="cuda")
    wide[:, 1:65] = h
    base = torch.zeros(333 * 64 + 1, dtype=dtype, device="cuda")
    base[1:] = w.reshape(-1)
    tall = torch.empty(64, 333, dtype=dtype, device="cuda")
    tall.copy_(w.t())
    loose = torch.zeros(333, 67, dtype=dtype, device="cuda")
    loose[:, :64] = w
    for a in (wide[:, 1:65], h.t().contiguous().t()):
        for b in (base[1:].view(333, 64), tall.t(), loose[:, :64]):
            for x, z in zip(_run(a, b, y), want):
                assert torch.equal(x, z)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_large_logits_stay_finite(dtype):
    h, w, y = _inputs(64, 64, 500, dtype, scale=60.0)
    loss, dh, dw, g = _run(h, w, y)
    _check(h, w, y, loss, dh, dw, "mean", g)


def test_fp32_values_that_bf16_cannot_hold():
    """The largest fp32 numbers round to infinity in bf16, small ones below its grid: products stay those of fp32."""
    h = torch.tensor([[3.0e38, 1e-30, 1.0 + 2 ** -23, 0.0]], device="cuda")
    w = torch.tensor([[1e-38, 1.0, 1.0, 2.0], [0.0, 1e30, -1.0, 0.0], [1e-38, 0.0, 2.0, 1.0]], device="cuda")
    y = torch.tensor([1], device="cuda")
    loss, dh, dw, g = _run(h, w, y)
    _check(h, w, y, loss, dh, dw, "mean", g)


def test_a_class_out_of_range_is_loud():
    for bad in (300, -1, 1 << 40):
        h, w, y = _inputs(40, 64, 300, torch.bfloat16, ignored=0.0)
        clean = _run(h, w, y, "none")
        y[7] = bad
        loss, dh, dw, _ = _run(h, w, y, "none")
        assert bool(torch.isnan(loss[7])) and bool(torch.isnan(dh[7]).all()) and bool(torch.isnan(dw).any())
        keep = torch.arange(40, device="cuda") != 7
        assert torch.equal(loss[keep], clean[0][keep]) and torch.equal(dh[keep], clean[1][keep])
        assert bool(torch.isnan(_run(h, w, y)[0]))


def test_only_one_gradient_and_none():
    from causal_eeg_vae_amd import linear_cross_entropy
    h, w, y = _inputs(90, 64, 400, torch.bfloat16)
    loss, dh, dw, _ = _run(h, w, y)
    a = h.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(a, w, y), a)[0], dh)
    b = w.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(h, b, y), b)[0], dw)
    with torch.no_grad():
        assert torch.equal(linear_cross_entropy(h, w, y), loss)


def test_gradient_against_differences():
    """Along its own direction d = grad / |grad| the loss changes by |grad| per unit: central differences of step e are off by e^2 / 6 of the third
    derivative (below 30 here: |d| = 1, logits move by at most |w| e) and 2^-21 of the loss (about 6) over 2 e."""
    from causal_eeg_vae_amd import linear_cross_entropy
    h, w, y = _inputs(16, 32, 100, torch.float32, ignored=0.2)
    _, dh, dw, _ = _run(h, w, y, "sum")
    for x, dx, f in ((h, dh, lambda v: linear_cross_entropy(v, w, y, reduction="none")), (w, dw, lambda v: linear_cross_entropy(h, v, y, reduction="none"))):
        norm = dx.double().norm()
        d = (dx.double() / norm).float()
        e = 2.0 ** -6
        slope = (f(x + e * d).double().sum() - f(x - e * d).double().sum()) / (2 * e)
        assert abs(float(slope - norm)) <= 30 * e * e / 6 * 16 + 16 * 6 * 2.0 ** -21 / (2 * e)


def test_streams_and_repeats_are_bitwise():
    h, w, y = _inputs(333, 128, 5001, torch.bfloat16)
    want = _run(h, w, y)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for s in (s1, s2, s1):   # two streams at once, each with its own workspace
        with torch.cuda.stream(s):
            got.append(_run(h, w, y))
    torch.cuda.synchronize()
    for r in got:
        for a, b in zip(r, want):
            assert torch.equal(a, b)


def test_captured_into_a_graph():
    from causal_eeg_vae_amd import linear_cross_entropy
    h, w, y = _inputs(200, 64, 1000, torch.bfloat16)
    a, b = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(linear_cross_entropy(a, b, y), (a, b))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = linear_cross_entropy(a, b, y)
        dh, dw = torch.autograd.grad(loss, (a, b))
    for k in range(4):
        h2, w2, y2 = _inputs(200, 64, 1000, torch.bfloat16, seed=k + 1, ignored=0.2 * k)   # another number of tokens that count
        with torch.no_grad():
            a.copy_(h2), b.copy_(w2), y.copy_(y2)
        graph.replay()
        torch.cuda.synchronize()
        want = _run(h2, w2, y2)
        for x, z in zip((loss.detach(), dh, dw), want):
            assert torch.equal(x, z)


def test_no_token_at_all():
    from causal_eeg_vae_amd import linear_cross_entropy
    h = torch.zeros(0, 64, device="cuda", requires_grad=True)
    w = torch.randn(10, 64, device="cuda", requires_grad=True)
    y = torch.zeros(0, dtype=torch.int64, device="cuda")
    for reduction in ("mean", "sum"):
        loss = linear_cross_entropy(h, w, y, reduction=reduction)
        dh, dw = torch.autograd.grad(loss, (h, w))
        assert float(loss) == 0 and dh.shape == h.shape and dw.shape == w.shape and not bool(dw.any())
    assert linear_cross_entropy(h, w, y, reduction="none").shape == (0,)


def test_no_token_and_a_weight_that_is_not_finite():
    from causal_eeg_vae_amd import linear_cross_entropy
    h = torch.zeros(2, 0, 64, device="cuda", requires_grad=True)
    w = torch.full((10, 64), float("nan"), device="cuda", requires_grad=True)
    y = torch.zeros(2, 0, dtype=torch.int64, device="cuda")
    for reduction in ("mean", "sum", "none"):
        loss = linear_cross_entropy(h, w, y, reduction=reduction)
        dh, dw = torch.autograd.grad(loss.sum(), (h, w))
        assert loss.shape == (y.shape if reduction == "none" else ()) and not bool(loss.sum()) and dh.shape == h.shape and not bool(dw.any())


def test_a_weight_of_very_distant_rows():
    h, w, y = _inputs(5, 8, 3, torch.float32)
    far = torch.zeros(3, (1 << 22) + 9, device="cuda")
    far[:, :8] = w
    for x, z in zip(_run(h, far[:, :8], y), _run(h, w, y)):
        assert torch.equal(x, z)
