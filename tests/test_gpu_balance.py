"""GPU: balance_loss (ceeg_balance_fwd / _bwd) against its formula in 64 bits.

Bounds, with u = 2^-24: a probability is off by at most c = (|x| 2^-23 + 2^-21 + E u) of itself, |x| <= the row's range of scores; the mean of it
adds T u at most, the loss is a sum of non-negative terms.  ds = E g / n p (f - d): p's error twice over |f| + d, and half a step of the output's type."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _reference(s, i, m, g):
    x = s.detach().double()
    (T, E), K = x.shape, i.shape[1]
    keep = torch.ones(T, dtype=torch.bool, device=x.device) if m is None else m
    n = max(int(keep.sum()), 1)
    given = i.long()[keep].reshape(-1)
    counts = torch.bincount(given[given >= 0], minlength=E)
    top = x.amax(1, keepdim=True)
    p = torch.exp(x - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(1, keepdim=True)
    p = torch.where(keep[:, None] & (total > 0), p / total, torch.zeros_like(p))
    f = counts.double() / (n * K)
    d = (p * f).sum(1, keepdim=True)
    loss = E * float((f * p.sum(0) / n).sum())
    ds = g * E / n * p * (f - d)
    size = abs(g) * E / n * p * (f + d)
    finite = x[keep][torch.isfinite(x[keep])]
    spread = min(float(finite.max() - finite.min()) if finite.numel() else 0.0, 104.0)   # below e^-104 a probability is 0 in fp32 either way
    return loss, counts, ds, size, spread * 2 ** -23 + 2 ** -21 + E * U


def _check(s, i, m=None, g=1.0):
    from causal_eeg_vae_amd import balance_loss
    a = s.detach().requires_grad_(True)
    loss, counts = balance_loss(a, i, mask=m)
    (ds,) = torch.autograd.grad(loss, a, torch.tensor(g, device="cuda"))
    want, w_counts, w_ds, size, c = _reference(s, i if i.dim() == 2 else i[:, None], m, g)
    assert torch.equal(counts, w_counts)
    assert loss.dtype == torch.float32 and ds.dtype == s.dtype and ds.shape == s.shape
    assert abs(float(loss.detach()) - want) <= (c + min(s.shape[0], 1 << 16) * U + 4 * U) * abs(want) + 1e-30
    tol = 4 * (c + 4 * U) * size + torch.finfo(s.dtype).eps / 2 * w_ds.abs() + 1e-36
    assert bool(((ds.double() - w_ds).abs() <= tol).all())
    return loss, counts, ds


def _inputs(T, E, K, dtype, seed=0, spread=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed + 13 * T + E)
    s = (torch.randn(T, E, generator=g, device="cuda") * spread).to(dtype)
    i = torch.rand(T, E, generator=g, device="cuda").topk(K, dim=1).indices
    i[torch.rand(T, K, generator=g, device="cuda") < 0.1] = -1
    m = torch.rand(T, generator=g, device="cuda") < 0.7
    return s, i.contiguous(), m


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("T,E,K", [(1, 1, 1), (1, 2, 1), (3, 3, 2), (61, 16, 2), (130, 8, 8), (257, 61, 3), (64, 64, 1), (500, 97, 4), (300, 256, 1), (70, 260, 5),
                                   (1000, 512, 1), (33, 520, 2), (90, 1000, 3), (50, 1028, 1), (40, 2048, 2), (9, 4095, 1), (21, 4096, 8), (70001, 24, 2)])
def test_loss_counts_and_gradient(T, E, K, dtype):
    s, i, m = _inputs(T, E, K, dtype)
    _check(s, i)
    _check(s, i.int(), m, g=-2.5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("E", [16, 64, 256, 512, 4096])
def test_strides_and_alignment(E, dtype):
    s, i, m = _inputs(45, E, 1, dtype)
    want = _check(s, i, m)
    for off, ld in ((1, E + 3), (8, E + 16), (0, E + 1)):
        wide = torch.full((45, ld + off), 77.0, dtype=dtype, device="cuda")
        wide[:, off:off + E] = s
        got = _check(wide[:, off:off + E], i[:, 0], m)     # indices [T]
        assert torch.equal(got[1], want[1])
    _check(s.t().contiguous().t(), i, m)


def test_rows_that_do_not_count():
    s, i, m = _inputs(100, 32, 2, torch.float32)
    want = _check(s, i, m)
    s2, i2 = s.clone(), i.clone()
    s2[~m], i2[~m] = float("nan"), 10 ** 6        # whatever masked rows hold
    for a, b in zip(_check_same(s2, i2, m), want):
        assert torch.equal(a, b)
    none = torch.zeros(100, dtype=torch.bool, device="cuda")
    from causal_eeg_vae_amd import balance_loss
    a = s2.requires_grad_(True)
    loss, counts = balance_loss(a, i2, none)
    (ds,) = torch.autograd.grad(loss, a)
    assert float(loss) == 0 and not bool(counts.any()) and not bool(ds.any())


def _check_same(s, i, m):
    from causal_eeg_vae_amd import balance_loss
    a = s.detach().requires_grad_(True)
    loss, counts = balance_loss(a, i, mask=m)
    return loss, counts, torch.autograd.grad(loss, a)[0]


@pytest.mark.parametrize("low", [float("-inf"), torch.finfo(torch.float32).min, -1e30])
def test_masked_codes(low):
    """Codes masked by -inf or by a type's lowest value, and a row that has none left."""
    s, i, m = _inputs(60, 40, 1, torch.float32)
    s[:, 30:] = low
    s[5] = low
    _check(s, i)


def test_a_code_out_of_range_is_loud():
    for bad in (40, -2):
        s, i, m = _inputs(60, 40, 1, torch.float32)
        i[3, 0] = bad
        loss, counts, ds = _check_same(s, i, None)
        assert bool(torch.isnan(loss)) and bool(torch.isnan(ds).all())


def test_even_use_gives_one_and_the_same_code_counts_twice():
    from causal_eeg_vae_amd import balance_loss
    loss, counts = balance_loss(torch.zeros(64, 16, device="cuda"), torch.arange(64, device="cuda") % 16)
    assert abs(float(loss) - 1) <= 4 * U * 16 and counts.tolist() == [4] * 16
    _, counts = balance_loss(torch.zeros(2, 4, device="cuda"), torch.tensor([[1, 1], [2, 1]], device="cuda"))
    assert counts.tolist() == [0, 3, 1, 0]


def test_gradient_against_differences():
    """Along its direction; third derivative of a mean of probabilities times E f below 8 E per row, fp32 loss off by 2^-20 of itself."""
    from causal_eeg_vae_amd import balance_loss
    s, i, m = _inputs(40, 12, 2, torch.float32, spread=1.0)
    a = s.clone().requires_grad_(True)
    (ds,) = torch.autograd.grad(balance_loss(a, i, m)[0], a)
    norm, e = float(ds.double().norm()), 2.0 ** -4
    d = (ds.double() / norm).float()
    slope = (float(balance_loss(s + e * d, i, m)[0]) - float(balance_loss(s - e * d, i, m)[0])) / (2 * e)
    assert abs(slope - norm) <= 8 * 12 / 40 * e * e / 6 + 2.0 ** -19 / (2 * e)


def test_captured_into_a_graph_and_on_streams():
    from causal_eeg_vae_amd import balance_loss
    s, i, m = _inputs(300, 96, 2, torch.bfloat16)
    a = s.clone().requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(balance_loss(a, i, m)[0], a)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, counts = balance_loss(a, i, m)
        (ds,) = torch.autograd.grad(loss, a)
    for k in range(4):
        s2, i2, m2 = _inputs(300, 96, 2, torch.bfloat16, seed=k + 1)
        with torch.no_grad():
            a.copy_(s2)
        i.copy_(i2), m.copy_(m2)
        graph.replay()
        torch.cuda.synchronize()
        for x, z in zip((loss, counts, ds), _check_same(s2, i2, m2)):
            assert torch.equal(x, z)


def test_no_row_at_all():
    from causal_eeg_vae_amd import balance_loss
    a = torch.zeros(0, 8, device="cuda", requires_grad=True)
    loss, counts = balance_loss(a, torch.zeros(0, 1, dtype=torch.int64, device="cuda"))
    assert float(loss) == 0 and counts.tolist() == [0] * 8 and torch.autograd.grad(loss, a)[0].shape == (0, 8)
