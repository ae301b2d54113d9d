"""CPU: what the backward of linear_cross_entropy and of balance_loss hands to the library where saved tensors come back with other strides, as
torch.autograd.graph.save_on_cpu gives them: rows that a stride walks have to lie inside the tensor.  The library is replaced by one that only records."""
import contextlib

import pytest
import torch


class _Recorder:
    def __init__(self):
        self.calls = {}

    def __getattr__(self, name):
        def call(*args):
            self.calls[name] = args
            return 4096 if name.endswith("bytes") else 0
        return call


@pytest.fixture
def library(monkeypatch):
    from causal_eeg_vae_amd import _lib
    rec = _Recorder()
    monkeypatch.setattr(_lib, "lib", lambda: rec)
    monkeypatch.setattr(_lib, "require_cuda", lambda *t: None)
    monkeypatch.setattr(_lib, "on", lambda dev: contextlib.nullcontext())
    monkeypatch.setattr(_lib, "stream", lambda: None)
    return rec


def _hooks(back):
    """Saved tensors go away as copies and come back as `back` makes them; the last matrix that did."""
    seen = []

    def unpack(x):
        y = back(x)
        if y.dim() == 2:
            seen.append(y)
        return y

    return torch.autograd.graph.saved_tensors_hooks(lambda x: x, unpack), seen


BACK = {"packed": lambda x: x.clone(memory_format=torch.contiguous_format), "transposed": lambda x: x.t().contiguous().t() if x.dim() == 2 else x.clone(),
        "wider": lambda x: torch.cat((x, x), 1)[:, :x.shape[1]] if x.dim() == 2 else x.clone()}


def _inside(pointer, ld, rows, cols, given):
    """`rows` rows of `cols`, `ld` apart, from `pointer` on: inside the tensor that was given back, or packed rows of a copy."""
    if pointer != given.data_ptr():
        return ld == cols
    size = given.untyped_storage().nbytes() // given.element_size() - given.storage_offset()
    return ld >= cols and (rows - 1) * ld + cols <= size and (rows == 1 or ld == given.stride(0)) and given.stride(1) == 1


@pytest.mark.parametrize("back", list(BACK))
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_linear_cross_entropy(library, back, dtype):
    from causal_eeg_vae_amd import linear_cross_entropy
    V, H, T = 50, 8, 7
    w = torch.zeros(V, H + 3, dtype=dtype)[:, :H].requires_grad_(True)
    hooks, seen = _hooks(BACK[back])
    with hooks:
        loss = linear_cross_entropy(torch.zeros(T, H, dtype=dtype), w, torch.zeros(T, dtype=torch.int64))
        torch.autograd.grad(loss, w)
    packed, weight, ldw = library.calls["ceeg_linear_ce_bwd"][:3]
    assert _inside(weight, ldw, V, H, seen[-1])


@pytest.mark.parametrize("back", list(BACK))
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_balance_loss(library, back, dtype):
    from causal_eeg_vae_amd import balance_loss
    T, E = 50, 8
    s = torch.zeros(T, E + 3, dtype=dtype)[:, :E].requires_grad_(True)
    hooks, seen = _hooks(BACK[back])
    with hooks:
        loss, _ = balance_loss(s, torch.zeros(T, dtype=torch.int64))
        torch.autograd.grad(loss, s)
    scores, ld = library.calls["ceeg_balance_bwd"][:2]
    assert _inside(scores, ld, T, E, seen[-1])


@pytest.mark.parametrize("back", [lambda x: x.half(), lambda x: x[:-1].clone(), lambda x: x.reshape(-1, 1).clone()], ids=["type", "short", "shape"])
@pytest.mark.parametrize("which", [0, 1])
def test_another_tensor_is_refused(library, back, which):
    """`which`: of the saved tensors, in their order.  Nothing is launched on what is not the saved tensor."""
    from causal_eeg_vae_amd import balance_loss, linear_cross_entropy
    x = torch.zeros(50, 8, requires_grad=True)
    for entry, loss in (("ceeg_linear_ce_bwd", lambda: linear_cross_entropy(torch.zeros(7, 8), x, torch.zeros(7, dtype=torch.int64))),
                        ("ceeg_balance_bwd", lambda: balance_loss(x, torch.zeros(50, dtype=torch.int64), torch.ones(50, dtype=torch.bool))[0])):
        seen = []

        def pack(t):
            seen.append(t)
            return len(seen) - 1

        with torch.autograd.graph.saved_tensors_hooks(pack, lambda k: back(seen[k]) if k == which else seen[k]):
            out = loss()
        with pytest.raises(ValueError, match="came back"):
            torch.autograd.grad(out, x)
        assert entry not in library.calls
