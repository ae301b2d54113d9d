"""GPU: linear_cross_entropy at values that are not finite, in forward mode and where saved tensors come back as other tensors."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BOTH = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])


def _inputs(T, H, V, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + T * 31 + H * 17 + V)
    h = torch.randn(T, H, generator=g, device="cuda").to(dtype)
    w = (torch.randn(V, H, generator=g, device="cuda") * (2 / H ** 0.5)).to(dtype)
    return h, w, torch.randint(0, V, (T,), generator=g, device="cuda")


def _run(h, w, y, reduction="mean", g=None):
    from causal_eeg_vae_amd import linear_cross_entropy
    a, b = h.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss = linear_cross_entropy(a, b, y, reduction=reduction)
    return (loss.detach(),) + torch.autograd.grad(loss, (a, b), torch.ones_like(loss) if g is None else g)


@BOTH
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("T", [3, 70])
def test_an_upstream_value_that_is_not_finite_stays_with_its_token(T, bad, dtype):
    h, w, y = _inputs(T, 72, 300, dtype)
    g = torch.linspace(-1.5, 2.0, T, device="cuda")
    g[1] = 0.0
    _, clean, _ = _run(h, w, y, "none", g)
    g[1] = bad
    _, dh, dw = _run(h, w, y, "none", g)
    others = torch.arange(T, device="cuda") != 1
    assert torch.equal(dh[others], clean[others]) and not bool(torch.isfinite(dh[1]).any()) and not bool(torch.isfinite(dw).any())
    g[:] = bad
    assert not bool(torch.isfinite(_run(h, w, y, "none", g)[1]).any())


@BOTH
@pytest.mark.parametrize("T,H,V", [(3, 40, 200), (8, 40, 200), (9, 40, 200), (70, 40, 200), (700, 64, 6001), (2100, 320, 25701)])
def test_a_class_of_minus_infinity_is_not_there(T, H, V, dtype):
    """A weight of -inf where every hidden state is positive gives the class no probability, whatever the number of tokens: loss and gradients are those of the
    vocabulary without it, its own gradient is zero, and only the column of the -inf is lost in dh (0 * inf).  Against 64 bits: every sum here has the same
    magnitudes as in the other parity tests of the package, rtol 1e-5 of a tensor's largest in float32; in bf16 dl and the gradient are rounded, 2^-8 each."""
    h, w, y = _inputs(T, H, V, dtype)
    h[:, 5] = h[:, 5].abs() + 0.25
    dead = V // 2
    y[y == dead] = 0
    w[dead, 5] = float("-inf")
    loss, dh, dw = _run(h, w, y)
    alive = torch.arange(V, device="cuda") != dead
    columns = torch.arange(H, device="cuda") != 5
    hd, wd = h.double(), w[alive].double()
    z = hd @ wd.t()
    lse = torch.logsumexp(z, 1)
    at, own = torch.arange(T, device="cuda"), torch.where(y > dead, y - 1, y)
    want = (lse - z[at, own]).mean()
    d = torch.exp(z - lse[:, None])
    d[at, own] -= 1
    d /= T
    assert abs(float(loss) - float(want)) <= 1e-5 * float(want)
    tol = 1e-5 if dtype == torch.float32 else 2.0 ** -7
    for got, ref in ((dh[:, columns], (d @ wd)[:, columns]), (dw[alive], d.t().contiguous() @ hd)):
        assert float((got.double() - ref).abs().max()) <= tol * float(ref.abs().max())
    assert not bool(torch.isfinite(dh[:, 5]).any()) and bool((dw[dead] == 0).all())


@BOTH
@pytest.mark.parametrize("T", [3, 9, 200])
def test_a_hidden_state_that_is_not_finite_is_one_tokens(T, dtype):
    from causal_eeg_vae_amd import linear_cross_entropy
    h, w, y = _inputs(T, 72, 700, dtype)
    clean, dh, _ = _run(h, w, y, "none")
    h[1, 3] = float("inf")
    rows, dh1, _ = _run(h, w, y, "none")
    others = torch.arange(T, device="cuda") != 1
    assert torch.equal(rows[others], clean[others]) and torch.equal(dh1[others], dh[others]) and not bool(torch.isfinite(rows[1]))
    assert torch.equal(linear_cross_entropy(h, w, y, reduction="none")[others], clean[others])


@BOTH
@pytest.mark.parametrize("T,H,V", [(1, 64, 200), (2, 64, 200), (9, 40, 200), (70, 64, 3000), (700, 64, 6001), (2100, 320, 25701)])
def test_the_largest_logits_there_are(T, H, V, dtype):
    """One class with a logit near the largest float32 takes all the probability: a token's loss is that logit (its own is gone in the rounding: 2^-24 of it, four of them), 0 where it is
    the target, and the gradient of the logits the difference of two ones.  Every product is a bf16 or float32 number times 1, but for the store (eps / 2) and 2^-22 of fp32 sums
    of up to T terms.  Logits that are all near the least one give losses from 0 to log V."""
    h, w, y = _inputs(T, H, V, dtype)
    h[:, 0] = 1.0
    top = V - 2
    w[top, 0] = 3e38
    y[T // 2:] = 1
    y[0] = top
    rows, _, _ = _run(h, w, y, "none")
    big = w[top, 0].double()
    want = torch.where(y == top, torch.zeros_like(big), big)
    assert bool(((rows.double() - want).abs() <= 2.0 ** -22 * big * (y != top)).all())
    loss, dh, dw = _run(h, w, y)
    assert abs(float(loss) - float(want.mean())) <= 2.0 ** -21 * float(big)
    d = torch.zeros(T, V, dtype=torch.float64, device="cuda")
    d[:, top] = 1
    d[torch.arange(T, device="cuda"), y] -= 1
    d /= T
    for got, ref, size in ((dh, d @ w.double(), d.abs() @ w.double().abs()), (dw, d.t().contiguous() @ h.double(), d.abs().t().contiguous() @ h.double().abs())):
        assert bool(((got.double() - ref).abs() <= (2.0 ** -22 + T * 2.0 ** -24) * size + torch.finfo(dtype).eps / 2 * ref.abs()).all())
    w[:, 0] = -3e38
    rows = _run(h, w, y, "none")[0]
    assert bool(((rows >= 0) & (rows <= torch.log(torch.tensor(float(V))) * 1.001)).all())


def test_forward_mode_is_refused():
    """A tangent that would be dropped is an error, with and without anything that asks for a gradient."""
    import torch.autograd.forward_ad as fwd
    from causal_eeg_vae_amd import linear_cross_entropy
    h, w, y = _inputs(20, 64, 100, torch.float32)
    with fwd.dual_level():
        for a, b in ((fwd.make_dual(h, torch.ones_like(h)), w), (h, fwd.make_dual(w, torch.ones_like(w)))):
            with pytest.raises(NotImplementedError):
                linear_cross_entropy(a, b, y)
            with torch.no_grad(), pytest.raises(NotImplementedError):
                linear_cross_entropy(a, b, y, reduction="none")
        linear_cross_entropy(h, w, y)       # no tangent: nothing to refuse


def _moved(x):
    """The values of x in a tensor of other strides and alignment."""
    if x.dim() < 2:
        return torch.cat((x.new_zeros(3), x))[3:]
    return torch.cat((x.new_zeros(x.shape[0], 3), x, x.new_zeros(x.shape[0], 2)), 1)[:, 3:3 + x.shape[1]]


@BOTH
@pytest.mark.parametrize("T,H,V", [(5, 64, 300), (60, 64, 333), (60, 70, 333), (1, 64, 1)])
def test_saved_tensors_that_come_back_as_others(T, H, V, dtype):
    """What a hook hands back holds the same values, not the same strides or alignment."""
    h, w, y = _inputs(T, H, V, dtype)
    wide = torch.full((V, H + 11), 9.0, dtype=dtype, device="cuda")
    wide[:, :H] = w
    want = _run(h, w, y)
    for weight in (w, wide[:, :H]):
        for unpack in (lambda x: x.clone(memory_format=torch.contiguous_format), _moved, lambda x: x.clone() if x.dim() < 2 else x.t().contiguous().t()):
            with torch.autograd.graph.saved_tensors_hooks(lambda x: x, unpack):
                got = _run(h, weight, y)
            for a, b in zip(got, want):
                assert torch.equal(a, b)
        with torch.autograd.graph.save_on_cpu():
            got = _run(h, weight, y)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
