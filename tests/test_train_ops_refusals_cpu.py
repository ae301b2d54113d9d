"""CPU: further calls that the operators of a training step refuse."""
import pytest
import torch


def test_adamw_step_refuses_a_gradient_of_another_shape():
    """As many elements in another order would be another update."""
    from causal_eeg_vae_amd import CeegError, adamw_step_
    t = lambda *s: torch.zeros(*s)  # noqa: E731
    for p, g in ((t(4, 6), t(6, 4)), (t(24), t(4, 6)), (t(4, 6), t(24)), (t(2, 3, 4), t(3, 2, 4))):
        with pytest.raises(ValueError, match="grads"):
            adamw_step_([t(3), p], [t(3), g], [t(3), t(24)], [t(3), t(24)], step=1)
    with pytest.raises(CeegError):      # the right shape gets as far as the device; moments may lie flat
        adamw_step_([t(3), t(4, 6)], [t(3), t(4, 6)], [t(3), t(24)], [t(3), t(24)], step=1)


def test_8_bit_moments_need_adamw():
    """They were asked for and not taken."""
    from causal_eeg_vae_amd.trainer import Trainer
    for bits in (8, 16):
        with pytest.raises(ValueError, match="adamw"):
            Trainer(torch.nn.Linear(2, 2), state_bits=bits)
    Trainer(torch.nn.Linear(2, 2), state_bits=32)
