"""The 8-bit linear layer on tensors without rows: they have no memory, so that their addresses are null.  Arguments are checked before a device is
looked for: without one these calls get as far as that."""
import pytest

from nncv_b200._lib import BF16, E4M3, F32, lib

EINVAL = 1
P = 1 << 20


@pytest.fixture
def done():
    import torch
    return 0 if torch.cuda.is_available() else 3


@pytest.mark.parametrize("at", [0, P])
def test_no_rows(done, at):
    L, a = lib(), at or None
    assert L.nncv_b200_rmsnorm(a, 0, a, P, 1e-6, a, a, BF16, None, BF16, 0, 256, None) == done
    assert L.nncv_b200_rmsnorm(a, 0, None, None, 1e-6, None, a, E4M3, a, BF16, 0, 256, None) == done
    assert L.nncv_b200_rmsnorm(a, 300, None, None, 1e-6, None, a, F32, None, F32, 0, 256, None) == done
    assert L.nncv_b200_gated_activation(a, a, 0, a, BF16, None, BF16, 0, 256, 5, None) == done
    assert L.nncv_b200_gated_activation(a, None, 512, a, E4M3, a, F32, 0, 256, 1, None) == done
    for rows in (1, 128):
        assert L.nncv_b200_quantize_e4m3(a, 0, F32, a, a, 0, 256, rows, None) == done
    assert L.nncv_b200_matmul_e4m3(a, a, P, 2 * P, a, 0, 8, 256, F32, None, 0, None) == done


def test_no_rows_and_a_wrong_argument():
    L = lib()
    assert L.nncv_b200_rmsnorm(None, 0, None, None, -1.0, None, None, BF16, None, BF16, 0, 256, None) == EINVAL
    assert L.nncv_b200_rmsnorm(None, 0, None, None, 1e-6, None, None, F32, None, BF16, 0, 256, None) == EINVAL
    assert L.nncv_b200_rmsnorm(None, 255, None, None, 1e-6, None, None, BF16, None, BF16, 0, 256, None) == EINVAL
    assert L.nncv_b200_gated_activation(None, None, 0, None, BF16, None, BF16, 0, 256, 6, None) == EINVAL
    assert L.nncv_b200_quantize_e4m3(None, 0, F32, None, None, 0, 256, 64, None) == EINVAL
    assert L.nncv_b200_matmul_e4m3(None, None, None, P, None, 0, 8, 256, F32, None, 0, None) == EINVAL
    assert L.nncv_b200_matmul_e4m3(None, None, P, P, None, 0, 8, 250, F32, None, 0, None) == EINVAL


def test_rows_need_addresses():
    L = lib()
    assert L.nncv_b200_rmsnorm(None, 0, None, None, 1e-6, None, P, BF16, None, BF16, 1, 256, None) == EINVAL
    assert L.nncv_b200_gated_activation(P, None, 0, None, BF16, None, BF16, 1, 256, 5, None) == EINVAL
    assert L.nncv_b200_quantize_e4m3(P, 0, F32, 2 * P, None, 1, 256, 1, None) == EINVAL
    for nulls in range(3):
        a = [P, 2 * P, 3 * P]
        a[nulls] = None
        assert L.nncv_b200_matmul_e4m3(a[0], a[1], 4 * P, 5 * P, a[2], 1, 8, 256, F32, None, 0, None) == EINVAL
