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


def test_requests_without_rows_and_blocks(K):
    start = torch.full((3,), 77, dtype=torch.int32, device=DEV)
    table = torch.empty(2, 0, dtype=torch.int32, device=DEV)
    K.step_tables(dev([0, 0]), dev([0, 0]), dev([]), table, dev([]), num_pages=3, q_start=start[:2])
    K.check_device_errors()
    assert start.tolist() == [0, 0, 77]
    K.step_tables(dev([0, 0]), dev([0, 9]), dev([]), table, dev([]), num_pages=3)
    with pytest.raises(KernelError, match="lengths of a step's requests"):
        K.check_device_errors()


def test_reading_back_past_the_table(K):
    """A sequence that is longer than its row of the page table is flagged, and what the table holds is read."""
    cache = torch.zeros(3, 2, K.kv4_page_bytes(64), dtype=torch.uint8, device=DEV)
    x = torch.randn(64, 128, generator=torch.Generator().manual_seed(1)).to(DEV)
    K.kv4_store(x, x, dev(torch.arange(64) + 64), cache, 64)
    out, want = torch.zeros(3, 2, 2, 64, 64, device=DEV), torch.zeros(3, 2, 2, 64, 64, device=DEV)
    K.kv4_expand(cache, want, dev([[1]]), dev([1]), dev([63]))
    K.check_device_errors()
    for before in (64, 5000, 2 ** 31 - 2):
        K.kv4_expand(cache, out.zero_(), dev([[1]]), dev([1]), dev([before]))
        with pytest.raises(KernelError, match="visible position"):
            K.check_device_errors()
        assert torch.equal(out, want)
    launched = K.launches
    for bad in (dict(page_table=dev([1])), dict(out=out.half())):
        with pytest.raises(KernelError):
            K.kv4_expand(**{**dict(cache=cache, out=out, page_table=dev([[1]]), q_len=dev([1]), kv_before=dev([5])), **bad})
    assert K.launches == launched
