"""How far linear_cross_entropy in float32 may be from its formula in 64 bits, as root mean squares, and on the CPU that the bounds tell three bf16 planes of an
operand from two and from one, in each of the four products.

With u = 2^-24, a rounding's rms at most 0.41 u of a number and sums taken 32 terms a step: a sum of n terms has n / 32 roundings of partial sums, half the
result's square on average, 0.41 u sqrt(n / 64) of it (7.3 u for n = 20001).  LOW: logits of deviation 1/2, so that |l - lse| <= 13: its rounding is worth 5 u of an
exponential, lse's own (8 u at most, 0.41 of that) 4 u of all of them, dropped products and the store 1 u: 10 u of a gradient; the loss, below 16, 4 u in lse, 2 u in its
own store and 0.41 u sqrt(300 / 64) of a logit.  The bound is 2^-20, 16 u.  HIGH: logits of deviation 8, |l - lse| <= 64: 26 u of an exponential and 13 u for lse, and as much for the loss, with 8 times
the logits' error (8 u sqrt(300 / 64) 0.41 = 7 u): 31 u, bound 2^-18, 64 u.
Two planes leave 2^-17 of an operand out, 0.41 of that in the mean and from both sides 2^-17.8 of a product; in HIGH a logit is off by 8 times that."""
import pytest
import torch

LOW, HIGH = (0.5, 2.0 ** -20), (8.0, 2.0 ** -18)


def inputs(T, H, V, scale):
    g = torch.Generator().manual_seed(T * 31 + H * 17 + V)
    return torch.randn(T, H, generator=g), torch.randn(V, H, generator=g) * (scale / H ** 0.5), torch.randint(0, V, (T,), generator=g)


def reference(h, w, y):
    """Losses of the tokens, and the gradients of their mean."""
    h, w, T = h.double(), w.double(), y.numel()
    z = h @ w.t()
    lse = torch.logsumexp(z, 1)
    at = torch.arange(T, device=h.device)
    loss = lse - z[at, y]
    d = z.sub_(lse[:, None]).exp_()
    d[at, y] -= 1
    d /= T
    return loss, d @ w, d.t() @ h


def offsets(got, want):
    """rms of the losses' errors, and of the gradients' relative to their own rms."""
    rms = lambda x: float(x.double().pow(2).mean().sqrt())  # noqa: E731
    return [rms(got[0].double() - want[0])] + [rms(a.double() - b) / rms(b) for a, b in zip(got[1:], want[1:])]


def _product(a, b, planes):
    """a @ b of the leading bf16 planes of both, the products whose terms reach the last plane, in float32."""
    parts = []
    for x in (a, b):
        left, p = x.clone(), []
        for _ in range(planes):
            p.append(left.to(torch.bfloat16).float())
            left -= p[-1]
        parts.append(p)
    out = 0
    for t in reversed(range(planes)):
        for i in range(t + 1):
            out = out + parts[0][i] @ parts[1][t - i]
    return out


def _emulated(h, w, y, planes):
    """planes: of the operands of the forward's logits, of the backward's, of dh and of dW."""
    T = y.numel()
    at = torch.arange(T)
    z = _product(h, w.t().contiguous(), planes[0])
    lse = torch.logsumexp(z.double(), 1).float()
    loss = lse - z[at, y]
    if planes[1] != planes[0]:
        z = _product(h, w.t().contiguous(), planes[1])
    d = (z - lse[:, None]).exp_()
    d[at, y] -= 1
    return loss, _product(d, w, planes[2]) / T, _product(d.t().contiguous(), h, planes[3]) / T


@pytest.mark.parametrize("T,H,V", [(97, 64, 512), (1100, 64, 300), (400, 200, 6001)])
def test_the_bounds_tell_three_planes_from_two(T, H, V):
    for scale, bound in (LOW, HIGH):
        x = inputs(T, H, V, scale)
        want = reference(*x)
        holds = [offsets(_emulated(*x, planes), want) for planes in ((3, 3, 3, 3), (2, 3, 3, 3), (3, 2, 3, 3), (3, 3, 2, 3), (3, 3, 3, 2), (2, 2, 2, 2), (1, 1, 1, 1))]
        assert max(holds[0]) <= bound
        assert holds[1][0] > bound                                      # the forward's logits: the loss
        if scale == HIGH[0]:
            assert holds[2][1] > bound and holds[2][2] > bound          # the backward's: both gradients
        else:
            assert holds[3][1] > bound and holds[4][2] > bound          # dh, dW
        for off in holds[5:]:
            assert min(off) > bound
