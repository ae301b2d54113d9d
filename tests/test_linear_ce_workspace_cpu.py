"""CPU: the workspaces of the cross entropy stay within what include/ceeg.h says of them, up to the largest number of tokens."""
import itertools

import pytest

GIB, MIB = 1 << 30, 1 << 20


def _up(x, a):
    return -(-x // a) * a


@pytest.mark.parametrize("dtype", [0, 1], ids=["f32", "bf16"])
def test_workspaces_are_what_the_header_says(dtype):
    from causal_eeg_vae_amd import _lib
    L = _lib.lib()
    planes = 3 if dtype == 0 else 1
    for T, H, V in itertools.product((1, 9, 700, 8192, 65536, 1 << 20, 1 << 22), (1, 64, 72, 1024, 32768), (1, 100, 512, 50257, 1 << 17, 1 << 22, 1 << 28)):
        in_place = dtype == 1 and H % 64 == 0
        column = planes * 2 * (_up(T, 64) + (0 if in_place else _up(H, 64)))
        rest = max(4 * T * H, 64 * MIB) + 128 * MIB + 4 * T + 2 * 64 * _up(H, 64) + 4096
        assert L.ceeg_linear_ce_bwd_ws_bytes(T, H, V, dtype) <= max(GIB, 256 * column) + 256 * column + rest, (T, H, V)
        packed = 0 if in_place else planes * 2 * _up(H, 64)
        assert L.ceeg_linear_ce_fwd_ws_bytes(T, H, V, dtype) <= 8 * T * -(-V // 64) + min(max(GIB, 256 * packed) + 256 * packed, packed * _up(V, 256)) + 8 * T + 4096, (T, H, V)


def test_many_tokens_take_what_256_columns_take():
    from causal_eeg_vae_amd import _lib
    L = _lib.lib()
    for dtype, planes in ((0, 3), (1, 1)):
        dl = planes * 2 * 256 * (1 << 22)
        assert dl > GIB and dl <= L.ceeg_linear_ce_bwd_ws_bytes(1 << 22, 64, 1 << 17, dtype) <= 1.02 * dl + 4 * 64 * (1 << 22) + 192 * MIB
