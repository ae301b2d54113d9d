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
