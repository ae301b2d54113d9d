"""GPU: linear_cross_entropy where a lost plane of float32, or a lost piece of the vocabulary, would show."""
import pytest
import torch

from test_linear_ce_precision_cpu import HIGH, LOW, inputs, offsets, reference

pytestmark = pytest.mark.gpu


def _run(h, w, y):
    from causal_eeg_vae_amd import linear_cross_entropy
    a, b = h.detach().requires_grad_(True), w.detach().requires_grad_(True)
    rows = linear_cross_entropy(h, w, y, reduction="none")
    loss = linear_cross_entropy(a, b, y)
    return (rows,) + torch.autograd.grad(loss, (a, b))


@pytest.mark.parametrize("T,H,V", [(97, 64, 512), (1100, 64, 300), (400, 200, 6001), (700, 300, 20001), (8, 64, 3000)])
@pytest.mark.parametrize("scale,bound", [LOW, HIGH], ids=["low", "high"])
def test_float32_keeps_three_planes(T, H, V, scale, bound):
    """Tiles of 64 in every product (97, 8), slots of dW (1100), tiles of 128 in dh and dW (400) and in all four (700)."""
    h, w, y = (x.cuda() for x in inputs(T, H, V, scale))
    off = offsets(_run(h, w, y), reference(h, w, y))
    assert max(off) <= bound, off


@pytest.mark.parametrize("T,H,V,dtype", [(16384, 64, 40003, torch.bfloat16), (16380, 72, 40003, torch.bfloat16), (4096, 16, 50001, torch.float32)],
                         ids=["bf16", "bf16-packed", "f32"])
def test_two_pieces_of_the_vocabulary(T, H, V, dtype):
    """The backward holds dl of a piece of the vocabulary at a time; here it takes two, of which the last is shorter and odd.  float32: the bound of LOW.  bf16: dl and the
    gradients are rounded to bf16, 2^-8 each at most.  A dh without the first piece, or a dW whose pieces are exchanged, is not within it."""
    from causal_eeg_vae_amd import _lib
    f32 = dtype == torch.float32
    whole = (3 if f32 else 1) * 2 * T * V
    assert whole / 4 < _lib.lib().ceeg_linear_ce_bwd_ws_bytes(T, H, V, _lib.CEEG_F32 if f32 else _lib.CEEG_BF16) < whole * 0.9
    h, w, y = (x.cuda() for x in inputs(T, H, V, LOW[0]))
    h, w = h.to(dtype), w.to(dtype)
    rows, dh, dw = _run(h, w, y)
    want, dh64, dw64 = [], [], 0
    late = []                                       # dh of the second half of the vocabulary alone
    for at in torch.arange(T, device="cuda").split(2048):
        x, z = h[at].double(), None
        z = x @ w.double().t()
        lse = torch.logsumexp(z, 1)
        here = torch.arange(at.numel(), device="cuda")
        want.append(lse - z[here, y[at]])
        d = z.sub_(lse[:, None]).exp_()
        d[here, y[at]] -= 1
        d /= T
        dh64.append(d @ w.double())
        late.append(d[:, V // 2:].contiguous() @ w[V // 2:].double())
        dw64 = dw64 + d.t().contiguous() @ x
    want, dh64, late = torch.cat(want), torch.cat(dh64), torch.cat(late)
    bound = LOW[1] if f32 else 2.0 ** -7
    off = offsets((rows, dh, dw), (want, dh64, dw64))
    assert off[0] <= LOW[1] and max(off[1:]) <= bound, off
    assert min(offsets((rows, dh, dw), (want, late, torch.roll(dw64, V // 2, 0)))[1:]) > 10 * bound
