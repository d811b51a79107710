"""The 4-bit cache without a GPU: steps that fail or bring nothing, the largest sizes."""
import torch

from braidinfer_b200.cache import CacheManager
from braidinfer_b200.parts.spec import CacheRequest


def test_page_lists_after_a_step_that_failed():
    """A step that fails after its pages were reserved leaves a sequence more blocks than its length wants; a list of pages has the step's, for
    the lists of all sequences lie end on end and are told apart by the lengths."""
    c = CacheManager([(CacheRequest("full", 2, 64, four_bit=True), None, 0), (CacheRequest("window", 2, 64, 70, four_bit=True), None, 0)],
                     64 * 9, 3, torch.bfloat16, "cpu")
    a, b = c.alloc_slot(), c.alloc_slot()
    c.begin_step([a, b], [200, 3], lists=True)                # (never ended)
    for full in c.begin_step([a, b], [1, 65], lists=True):
        assert [len(x) for x in full] == [1, 2]
    c.end_step([a, b], [1, 65])
    for full, g in zip(c.begin_step([b, a], [63, 128], lists=True), c.groups):
        assert full == [g.pages.blocks[b][:2], g.pages.blocks[a][:3]]
