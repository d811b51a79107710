"""The engine with a 4-bit cache where steps fail, and where its prompts go over pages that are read back."""
import inspect

import pytest
import torch

import plain_kv4
from braidinfer_b200.csrc.api import Kernels
from gpu_util import engine
from test_gpu_kv4 import U
from test_gpu_kv4_engine import MODELS, folder_of
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


@pytest.fixture(params=["auto", "pages"])
def route(request, monkeypatch):
    """Prompts as the sizes have it (here: over 4 bits), and over pages read back."""
    if request.param == "pages":
        monkeypatch.setattr(Kernels, "KV4_PAGES_FROM", 0)
    return request.param


STEPS = [[100, 60], [1, 1], [70, 3], [1, 90], [1, 5], [1, 1]]     # tokens of two sequences, step by step


def run_steps(eng, vocab):
    a, b = eng.open(), eng.open()
    other = eng.open()                                        # (pages of a third one lie between theirs)
    out = []
    for i, (m, n) in enumerate(STEPS):
        x, y = random_prompts(vocab, [m, n], seed=10 + i)
        out.append(eng.step([(a, x), (other, [i + 1]), (b, y)], want="all"))
    eng.check()
    return torch.cat(out)


@pytest.mark.parametrize("name", MODELS)
def test_attention_of_bfloat16_runs(tmp_path, monkeypatch, name, route):
    """Every layer's attention in every step, as the engine calls it, against the formula over the cache as it stands: prompts alone and
    beside single tokens, steps of padded rows, a sliding window.  (The bound: 2^-12 of a score's products twice, of a probability and of a value,
    and the result's bfloat16, as of prompts alone.)"""
    folder = folder_of(tmp_path, name)
    eng = engine(folder, "bfloat16", max_tokens=64 * 16, cache_format="int4", use_graphs=False)
    K, seen = eng.kernels, []
    attn, pages, signature = K.attn_kv4, K._attn_kv4_pages, inspect.signature(K.attn_kv4)

    def checked(*args, **kw):
        attn(*args, **kw)
        a = signature.bind(*args, **kw).arguments
        q_len, before = a["q_len"].tolist(), a["kv_before"].tolist()
        n, nqh, hd = sum(q_len), a["nqh"], a["hd"]
        assert a["settled"] and (a["token_seq"][n:] == -1).all()
        want, mag, smag = plain_kv4.attend(a["q"][:n, :nqh * hd].double().view(n, nqh, hd), a["cache"], a["page_table"].cpu(), q_len, before, a["scale"],
                                           a["window"])
        part = 2 * (2 * 2.0 ** -12 * smag[1] + 32 * U * smag[0])[..., None] + 2 * 2.0 ** -12 + 2.0 ** -18
        assert ((a["out"][:n].double().view(want.shape) - want).abs() <= mag * part + 2.0 ** -8 * want.abs() + 1e-30).all()
        seen.append(q_len)
    monkeypatch.setattr(K, "attn_kv4", checked)
    over_pages = []
    monkeypatch.setattr(K, "_attn_kv4_pages", lambda *a: (over_pages.append(a[-1]), pages(*a)))
    run_steps(eng, config_of(folder).vocab_size)
    assert len(seen) == len(STEPS) * len(eng.spec.schedule)
    assert (len(set(over_pages)) > 0) == (route == "pages")


@pytest.mark.parametrize("name", MODELS)
def test_replayed_prompts_over_pages_give_the_same_bits(tmp_path, monkeypatch, name):
    monkeypatch.setattr(Kernels, "KV4_PAGES_FROM", 0)
    folder = folder_of(tmp_path, name)
    logits = []
    for graphs in (True, False):
        eng = engine(folder, "bfloat16", max_tokens=64 * 40, cache_format="int4", use_graphs=graphs)
        out = []
        for _ in range(4):                                    # (each with other pages)
            out.append(run_steps(eng, config_of(folder).vocab_size))
        assert (eng.graph_replays > 0) == graphs
        logits.append(out)
    for a, b in zip(*logits):
        assert torch.equal(a, b) and torch.equal(a, logits[0][0])
