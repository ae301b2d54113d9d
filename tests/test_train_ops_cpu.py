"""CPU: what linear_cross_entropy, balance_loss, adamw_step_ and AdamW refuse, in Python and at the C entries.  Every refusal comes before a launch, so
none of these calls needs a GPU; the pointers handed to the C entries are never read."""
import ctypes as C

import pytest
import torch

P = 0x10000   # an aligned address that nothing reads


def _lib():
    from causal_eeg_vae_amd import _lib
    return _lib.lib()


def test_linear_cross_entropy_refuses():
    from causal_eeg_vae_amd import CeegError, linear_cross_entropy as f
    h, w, y = torch.zeros(4, 8), torch.zeros(5, 8), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(CeegError):
        f(h, w, y)                                   # no CPU path
    for bad in ((h, torch.zeros(5, 7), y), (h, w, y[:3]), (h, w[0], y), (h, torch.zeros(0, 8), y), (torch.zeros(4, 0), torch.zeros(5, 0), y),
                (torch.tensor(1.0), w, y), (h, w, y[:, None])):
        with pytest.raises(ValueError):
            f(*bad)
    for bad in ((h.half(), w.half(), y), (h, w.bfloat16(), y), (h, w, y.int()), (h.long(), w, y), (h, w, [0] * 4)):
        with pytest.raises(TypeError):
            f(*bad)
    with pytest.raises(ValueError):
        f(h, w, y, reduction="batchmean")


def test_linear_cross_entropy_entries_refuse():
    L = _lib()
    fwd = [P, 64, P, 64, P, 10, 64, 100, 1, -100, 1, P, P, P, P, P, L.ceeg_linear_ce_fwd_ws_bytes(10, 64, 100, 1), None]
    bwd = [P, P, 64, 10, 64, 100, 1, 1, P, P, P, P, P, P, L.ceeg_linear_ce_bwd_ws_bytes(10, 64, 100, 1), None]
    for entry, good, cases in (
            (L.ceeg_linear_ce_fwd, fwd, [(0, None, -1), (2, None, -1), (4, None, -1), (11, None, -1), (12, None, -1), (13, None, -1), (14, None, -1), (14, P + 16, -1),
                                         (15, None, -3), (15, P + 1, -3), (16, 16, -3), (5, 0, -1), (6, 0, -1), (7, 0, -1), (1, 63, -1), (3, 63, -1), (8, 2, -2), (10, 3, -1),
                                         (10, -1, -1), (5, (1 << 22) + 1, -2), (7, (1 << 28) + 1, -2), (3, 1 << 23, -2), (2, P + 2, -1), (3, 72, -1), (4, P + 4, -1)]),
            (L.ceeg_linear_ce_bwd, bwd, [(0, None, -1), (0, P + 16, -1), (1, None, -1), (8, None, -1), (9, None, -1), (10, None, -1), (13, None, -3), (14, 16, -3), (6, 5, -2),
                                         (7, 3, -1), (3, 0, -1), (1, P + 8, -1), (2, 72, -1)])):
        for at, value, code in cases:
            args = list(good)
            args[at] = value
            assert entry(*args) == code, (entry.__name__, at, value)
    args = list(bwd)
    args[11] = args[12] = None                        # neither gradient wanted
    assert L.ceeg_linear_ce_bwd(*args) == -1
    for sizes in ((0, 8, 8, 0), (8, 0, 8, 0), (8, 8, 0, 0), (8, 1 << 16, 8, 0)):
        assert L.ceeg_linear_ce_fwd_ws_bytes(*sizes) == 0 and L.ceeg_linear_ce_bwd_ws_bytes(*sizes) == 0


def test_workspaces_stay_bounded():
    """The pieces of the backward are capped: its workspace does not grow with the vocabulary beyond that, and never holds the logits.  n pieces are
    made equally large, so that each is down to 1 - 1 / n of the cap: with the 4 pieces at least of 2^17 columns here, 4 / 3 between the two."""
    L = _lib()
    for dtype in (0, 1):
        for T, H in ((8192, 1024), (65536, 256)):
            a, b = (L.ceeg_linear_ce_bwd_ws_bytes(T, H, v, dtype) for v in (1 << 17, 1 << 20))
            assert b <= a * 4 / 3 and b < T * (1 << 20) * 4 / 4
            assert L.ceeg_linear_ce_fwd_ws_bytes(T, H, 1 << 17, dtype) < T * (1 << 17) * 4 / 4


def test_balance_loss_refuses():
    from causal_eeg_vae_amd import CeegError, VectorQuantizer, balance_loss as f
    s, i = torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int64)
    with pytest.raises(CeegError):
        f(s, i)
    for bad in ((s, i[:3]), (s[0], i), (s, i[:, :, None]), (torch.zeros(4, 1), i), (torch.zeros(4, 4097), i), (torch.zeros(4, 0), i), (s, i[:, :0])):
        with pytest.raises(ValueError):
            f(*bad)
    for bad in ((s.half(), i), (s, i.short()), (s, i.float()), (s, None)):
        with pytest.raises(TypeError):
            f(*bad)
    for m in (torch.ones(4), torch.ones(3, dtype=torch.bool), torch.ones(4, 1, dtype=torch.bool)):
        with pytest.raises(ValueError):
            f(s, i, mask=m)
    with pytest.raises(CeegError):
        VectorQuantizer(8, 4, 0.25).balance(torch.zeros(3, 4), torch.zeros(3, 1, dtype=torch.int64))


def test_balance_entries_refuse():
    L = _lib()
    fwd = [P, 64, 0, P, 8, 100, 64, 2, None, P, P, P, P, L.ceeg_balance_ws_bytes(100, 64), None]
    for at, value, code in ((0, None, -1), (1, 63, -1), (2, 3, -2), (3, None, -1), (3, P + 4, -1), (4, 2, -1), (5, 0, -1), (5, 1 << 31, -1), (6, 0, -1), (6, 4097, -1),
                            (7, 0, -1), (7, 65, -1), (9, None, -1), (10, None, -1), (11, None, -1), (12, None, -3), (12, P + 16, -3), (13, 8, -3), (0, P + 2, -1)):
        args = list(fwd)
        args[at] = value
        assert L.ceeg_balance_fwd(*args) == code, (at, value)
    args = list(fwd)
    args[1] = args[6] = 4097
    assert L.ceeg_balance_fwd(*args) == -2
    bwd = [P, 64, 1, 100, 64, None, P, P, P, None]
    for at, value, code in ((0, None, -1), (1, 1, -1), (2, 2, -2), (3, 0, -1), (4, 0, -1), (6, None, -1), (7, None, -1), (8, None, -1), (8, P + 8, -1)):
        args = list(bwd)
        args[at] = value
        assert L.ceeg_balance_bwd(*args) == code, (at, value)
    assert L.ceeg_balance_ws_bytes(0, 8) == 0 and L.ceeg_balance_ws_bytes(8, 0) == 0 and L.ceeg_balance_ws_bytes(8, 4097) == 0


def test_adamw_step_refuses():
    from causal_eeg_vae_amd import CeegError, adamw_step_ as f
    from causal_eeg_vae_amd.optim import block_state
    t = lambda n=6, d=torch.float32: torch.zeros(n, dtype=d)  # noqa: E731
    assert f([], [], [], [], step=1) is None
    with pytest.raises(CeegError):
        f([t()], [t()], [t()], [t()], step=1)
    for bad in (([t()], [], [t()], [t()]), ([t()], [t(5)], [t()], [t()]), ([t()], [t(6, torch.bfloat16)], [t()], [t()]), ([t()], [t()], [t(6, torch.bfloat16)], [t()]),
                ([t(), t(6, torch.bfloat16)], [t(), t()], [t(), t()], [t(), t()]), ([torch.zeros(4, 6).t()], [t(24)], [t(24)], [t(24)]), ([t()], [None], [t()], [t()]),
                ([t()], [t()], [block_state(t())], [(t(), t())]), ([t(300)], [t(300)], [block_state(t(300))], [(block_state(t(300))[0], t(1))])):
        with pytest.raises(ValueError):
            f(*bad, step=1)
    for bad in (([t(6, torch.half)], [t(6, torch.half)], [t()], [t()]), ([t()], [t()], [block_state(t())], [t()]), ([t()], [t()], [(t(), 1.0)], [(t(), 1.0)])):
        with pytest.raises(TypeError):
            f(*bad, step=1)


def test_adamw_entry_refuses():
    L = _lib()
    one = lambda x: (C.c_void_p * 1)(x)  # noqa: E731
    good = [1, (C.c_int64 * 1)(10), one(P), one(P), one(P), one(P), one(P), one(P), 0, 8, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, None, None, 0, None]
    for at, value, code in ((0, -1, -1), (1, None, -1), (1, (C.c_int64 * 1)(-1), -1), (2, None, -1), (2, one(None), -1), (2, one(P + 2), -1), (3, one(None), -1), (4, one(None), -1),
                            (5, one(None), -1), (6, None, -1), (6, one(None), -1), (7, one(P + 1), -1), (8, 2, -2), (9, 16, -2), (11, 1.0, -1), (12, -0.1, -1), (13, -1.0, -1),
                            (15, 0, -1), (11, float("nan"), -1)):
        args = list(good)
        args[at] = value
        assert L.ceeg_adamw_step(*args) == code, (at, value)
    assert L.ceeg_adamw_step(*([0] + [None] * 7 + good[8:])) == 0     # an empty list is nothing to do
    args = list(good)
    args[1] = (C.c_int64 * 1)(0)
    assert L.ceeg_adamw_step(*args) == 0
    from causal_eeg_vae_amd import optim
    assert L.ceeg_adamw_block() == optim.BLOCK


def test_adamw_class_refuses():
    from causal_eeg_vae_amd import AdamW
    from causal_eeg_vae_amd.trainer import Trainer
    p = [torch.nn.Parameter(torch.zeros(3))]
    for kw in (dict(state_bits=16), dict(betas=(1.0, 0.9)), dict(eps=-1.0), dict(weight_decay=-1.0), dict(lr=-1.0)):
        with pytest.raises(ValueError):
            AdamW(p, **kw)
    with pytest.raises(ValueError):
        Trainer(torch.nn.Linear(2, 2), optimizer="sgd")
    AdamW(p).step()                                    # no gradient: nothing to do
    with pytest.raises(ValueError):
        AdamW(p).load_state_dict(torch.optim.AdamW(p).state_dict())


def test_block_state_values():
    from causal_eeg_vae_amd.optim import block_state, block_values
    q, s = block_state(torch.zeros(3, 100))
    assert q.shape == (3, 100) and q.dtype == torch.float8_e4m3fn and s.shape == (2,)
    q.view(-1)[:] = torch.tensor(2.0).to(torch.float8_e4m3fn)
    s[:] = torch.tensor([0.5, 3.0])
    v = block_values((q, s)).view(-1)
    assert bool((v[:256] == 1).all()) and bool((v[256:] == 6).all())
    assert bool((block_values((q, s), square=True).view(-1)[256:] == 36).all())
    assert block_state(torch.zeros(0))[1].shape == (0,)
