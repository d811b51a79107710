"""The engine with a 4-bit cache where steps fail, and where its prompts go over pages that are read back."""
import pytest
import torch

from gpu_util import engine
from test_gpu_kv4_engine import folder_of
from tiny import config_of, random_prompts

pytestmark = pytest.mark.gpu


def test_a_step_that_failed_leaves_the_next_ones_right(tmp_path):
    folder = folder_of(tmp_path, "A64")
    prompts = random_prompts(config_of(folder).vocab_size, [40, 90], seed=3)
    logits = []
    for fails in (False, True):
        eng = engine(folder, "float32", max_tokens=64 * 12, cache_format="int4")
        a, b = eng.open(), eng.open()
        if fails:                                             # (its pages are taken by then)
            with pytest.raises(IndexError):
                eng.step([(a, [1] * 200), (b, [2])], want=[[200], [0]])
        out = [eng.step([(a, prompts[0]), (b, prompts[1])])]
        out.append(eng.step([(a, prompts[1][:60]), (b, [7])]))   # (a's second block)
        for i in range(5):
            out.append(eng.step([(a, [3 + i]), (b, [9 - i])]))
        eng.check()
        logits.append(torch.cat(out))
    assert torch.equal(*logits)
