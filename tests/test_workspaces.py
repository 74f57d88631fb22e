"""Which tensors lend their bytes as a workspace (CPU)."""
import pytest
import torch

from femtochat_amd.kernels import _check_workspace

CPU = torch.device("cpu")


@pytest.mark.parametrize("make", [
    lambda: torch.empty(4096, dtype=torch.uint8), lambda: torch.empty(8, 4, 32, dtype=torch.float32),
    lambda: torch.empty(64, 64, dtype=torch.uint8).t(), lambda: torch.empty(8, 4, 16, 8, dtype=torch.uint8).permute(2, 0, 3, 1),
    lambda: torch.empty(4, 32, 32, dtype=torch.uint8).transpose(0, 2)[:, :, :, None], lambda: torch.empty(8000, dtype=torch.uint8)[100:4196],
])
def test_dense_memory_in_any_order(make):
    _check_workspace(make(), 4096, CPU)


@pytest.mark.parametrize("make", [
    lambda: torch.empty(4095, dtype=torch.uint8), lambda: torch.empty(1, dtype=torch.uint8).expand(4096),
    lambda: torch.empty(8192, dtype=torch.uint8)[::2], lambda: torch.empty(64, 128, dtype=torch.uint8)[:, :64],
    lambda: torch.empty(64, 1, dtype=torch.uint8).expand(64, 64), lambda: torch.empty(64, 128, dtype=torch.uint8)[:, :64].t(),
    lambda: torch.empty(4096, dtype=torch.uint8, device="meta"),
    lambda: torch.empty(127, dtype=torch.uint8).as_strided((64, 64), (1, 1)),
])
def test_repeated_missing_or_foreign_memory(make):
    with pytest.raises(ValueError, match="workspace"):
        _check_workspace(make(), 4096, CPU)
