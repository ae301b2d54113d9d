"""GPU: the balance loss where saved tensors come back as other tensors."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _moved(x):
    """The values of x in a tensor of other strides and alignment."""
    if x.dim() < 2:
        return torch.cat((x.new_zeros(3), x))[3:]
    return torch.cat((x.new_zeros(x.shape[0], 3), x, x.new_zeros(x.shape[0], 2)), 1)[:, 3:3 + x.shape[1]]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("T,E,K", [(1, 5, 1), (60, 64, 2), (60, 61, 1), (300, 512, 1)])
def test_saved_tensors_that_come_back_as_others(T, E, K, dtype):
    """What a hook hands back holds the same values, not the same strides or alignment.  The probabilities are summed in another order where the row is read in
    pieces of another width: 2^-20 of the largest gradient, and a step of bf16 (2^-7) where that turns a rounding."""
    from causal_eeg_vae_amd import balance_loss
    g = torch.Generator(device="cuda").manual_seed(T + E)
    scores = torch.randn(T, E, generator=g, device="cuda").to(dtype)
    idx = torch.rand(T, E, generator=g, device="cuda").topk(K, dim=1).indices
    mask = torch.rand(T, generator=g, device="cuda") < 0.7
    wide = torch.full((T, E + 16), 9.0, dtype=dtype, device="cuda")
    wide[:, :E] = scores
    away = lambda x: x.clone(memory_format=torch.contiguous_format)  # noqa: E731

    def run(s):
        a = s.detach().requires_grad_(True)
        loss, counts = balance_loss(a, idx, mask)
        return loss.detach(), counts, torch.autograd.grad(loss, a)[0]

    want = run(scores)
    for s in (scores, wide[:, :E]):
        for hooks in (torch.autograd.graph.saved_tensors_hooks(lambda x: x, away), torch.autograd.graph.saved_tensors_hooks(lambda x: x, _moved),
                      torch.autograd.graph.saved_tensors_hooks(lambda x: x, lambda x: away(x) if x.dim() < 2 else x.t().contiguous().t()),
                      torch.autograd.graph.save_on_cpu()):
            with hooks:
                loss, counts, ds = run(s)
            assert torch.equal(counts, want[1]) and torch.equal(loss, want[0])
            off = (ds.double() - want[2].double()).abs()
            assert bool((off <= 2.0 ** -20 * float(want[2].abs().max()) + (2.0 ** -7 * want[2].double().abs() if dtype == torch.bfloat16 else 0)).all())
