"""The 4-bit cache without a GPU: steps that fail or bring nothing, the largest sizes."""
import ctypes

import pytest
import torch

from braidinfer_b200.cache import CacheManager
from braidinfer_b200.csrc import build
from braidinfer_b200.csrc.api import Kernels
from braidinfer_b200.engine.step import StepPacker
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


@pytest.mark.parametrize("stages", [2, 3])
def test_the_last_copies_of_a_ring(stages):
    """What a warp of attn_kv4_kernel waits for before it gives up: the last use of every stage, over both walks of a context (the second
    begins where the ring stands, after what the first had asked for and not walked)."""
    lib = ctypes.CDLL(str(build.kv4_attention_library(64, verbose=False)))
    for n in range(1, 9):
        for walked in range(n + 1):                           # units of the first walk
            phases = [0] * stages                             # copies that each stage has been given
            uses = 0
            asked = min(n, walked + stages)
            for k in range(asked):
                phases[uses % stages] += 1
                uses += 1
            for k in range(min(stages, n) + 1):               # and of the second, before one does not come
                for s in range(stages):
                    if phases[s]:                             # a barrier's phase of parity p is over when its copy has come: the last one's
                        assert lib.braid_attn_kv4_last_parity(uses, s, stages) == (phases[s] - 1) % 2
                phases[uses % stages] += 1
                uses += 1


def test_prompts_past_a_grids_depth_of_the_older_kernel():
    """The kernel for ordinary pages refuses more than 65,535 tiles of 64 columns of queries; the others take a grid's tiles in parts."""
    def over_pages(tokens, heads, tc):
        x = torch.empty(1, heads * 32, dtype=torch.bfloat16).expand(tokens, heads * 32)
        return Kernels._kv4_as_pages(x, x, tokens, tokens, 1, heads, 1, 32, tc)
    for heads, most in ((128, 65535), (64, 65535), (16, 4 * 65535), (1, 64 * 65535)):
        assert over_pages(most, heads, False) and not over_pages(most + 1, heads, False) and over_pages(2 * most + 1, heads, True)


@pytest.mark.parametrize("rows", [[], [0], [0, 1, 2]])
def test_rows_of_device_tokens_are_counted(rows):
    packer = StepPacker("cpu", 1)
    with pytest.raises(ValueError, match="rows of tokens"):
        packer.pack_lengths([0, 1], [[5], [6]], [3, 4], [[0], [0]], [[[0], [1]]], [4], token_source_rows=rows)
