"""State space operators at the sizes where another kernel, or another turn of a kernel's loop, takes over:
many rows and channels, few steps, so that the float64 reference stays quick."""
import pytest
import torch

import test_state_space_gpu as base
from test_state_space_gpu import BF16, F16, F32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("T,N,D,S,G,opt", [
    (9, 128, 1001, 4, 1, dict(state=True)), (17, 128, 1001, 3, 1, dict(lengths=torch.int64, z=False)),
    (11, 128, 1280, 4, 1, dict(lengths=torch.int64, state=True)), (9, 128, 1280, 2, 1, dict(half=True, z=False)),
    (10, 64, 1538, 1, 2, dict(lengths=torch.int32, batch_first=True)),
])
def test_selective_scan_of_many_channels_with_few_states(T, N, D, S, G, opt, dtype):
    """One lane a channel: blocks of 128 and 256 channels, staged one by one or in fours."""
    base.test_selective_scan(T, N, D, S, G, opt, dtype)
