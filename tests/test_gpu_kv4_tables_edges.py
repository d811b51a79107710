"""The tables of steps that bring nothing (csrc/kv4.cu)."""
import pytest
import torch

from braidinfer_b200.csrc.api import KernelError
from test_gpu_kv4 import DEV, K, dev  # noqa: F401 (K is a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 5, 3000])
def test_no_requests_and_rows_of_padding(K, rows):
    place, pos, seq = (torch.full((rows + 1,), 77, dtype=torch.int32, device=DEV) for _ in range(3))
    for _ in range(3):
        K.step_tables(dev([]), dev([]), dev([]), torch.empty(0, 4, dtype=torch.int32, device=DEV), place[:rows], num_pages=3, positions=pos[:rows],
                      token_seq=seq[:rows], q_start=dev([]))
    K.check_device_errors()
    assert (place[:rows] == -1).all() and (pos[:rows] == 0).all() and (seq[:rows] == -1).all()
    assert place[rows] == pos[rows] == seq[rows] == 77
