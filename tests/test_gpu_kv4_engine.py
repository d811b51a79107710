"""The engine with a cache held in 4 bits.

In float32 its logits are compared with the plain model whose keys and values are quantised (plain_kv4.py).  The codes hang on
roundings: keys and values that differ by float32's errors fall on another side of a border with a chance of some 3e-5 a number, and
one that does moves a number of one token by a bfloat16 step.  In a bfloat16 run all of them move so, within TOL_BF16 on the logits; one
of the thousands of a test moves them by less than a thirtieth of that.  In bfloat16 runs codes differ from the plain model's everywhere, so
there the first layer's pages are compared, byte for byte, with those made of an ordinary run's cache, whose keys and values are the
same numbers."""
import pytest
import torch

import braidinfer_b200 as lib
import plain_kv4
import plain_mistral as P
from gpu_util import engine, max_err, sharpen
from tiny import TOL_BF16, TOL_F32, config_of, make_folder, random_prompts, read_weights
from braidinfer_b200.engine.step import StepPacker

pytestmark = pytest.mark.gpu
DEV = "cuda"
TOL = 2 * TOL_F32 + TOL_BF16 / 30
MODELS = {"B": dict(), "A64": dict(head_dim=64), "C96": dict(head_dim=96, num_attention_heads=6, num_key_value_heads=2), "A128": dict(head_dim=128)}


def folder_of(tmp_path, name):
    return sharpen(make_folder(tmp_path, name[0], **MODELS[name]), 3.0)


@pytest.fixture
def quantised(monkeypatch):
    plain = P.attention

    def attention(q, k, v, window):
        k, v = (plain_kv4.numbers(*plain_kv4.quantise(x)).to(x.dtype) for x in (k, v))
        return plain(q, k, v, window)
    monkeypatch.setattr(P, "attention", attention)


@pytest.mark.parametrize("name", MODELS)
def test_logits_are_those_of_quantised_keys_and_values(tmp_path, request, name):
    folder = folder_of(tmp_path, name)
    cfg, w = config_of(folder), read_weights(folder)
    seqs = random_prompts(cfg.vocab_size, [75, 7, 140, 30], seed=4)
    full = [P.forward_logits(w, cfg, s, torch.float64) for s in seqs]
    request.getfixturevalue("quantised")
    want = [P.forward_logits(w, cfg, s, torch.float64) for s in seqs]
    eng = engine(folder, "float32", max_tokens=64 * 12, cache_format="int4")
    assert max(max_err(a, b) for a, b in zip(want, full)) > 3 * TOL           # (else nothing would be compared)
    slots = [eng.open() for _ in seqs]
    heads = [69, 1, 134, 24]
    got = eng.step([(s, t[:n]) for s, t, n in zip(slots, seqs, heads)], want="all")
    assert max_err(got, torch.cat([x[:n] for x, n in zip(want, heads)])) < TOL
    for i in range(6):                                        # replayed from the third on
        got = eng.step([(s, [t[n + i]]) for s, t, n in zip(slots, seqs, heads)])
        assert max_err(got, torch.stack([x[n + i] for x, n in zip(want, heads)])) < TOL
    eng.check()
    assert eng.graph_replays > 0


@pytest.mark.parametrize("name", ["B", "A64", "A128"])
def test_first_layers_pages(tmp_path, name):
    folder = folder_of(tmp_path, name)
    cfg = config_of(folder)
    prompts = random_prompts(cfg.vocab_size, [70, 3, 129], seed=2)
    runs = [engine(folder, "bfloat16", max_tokens=64 * 8, cache_format=f, use_graphs=False) for f in ("full", "int4")]
    for e in runs:
        slots = [e.open() for _ in prompts]
        e.step(list(zip(slots, prompts)), want=None)
        for i in range(3):
            e.step([(s, [5 + i]) for s in slots])
        e.check()
    full, four = (e.cache.groups[0].storage[0].cpu() for e in runs)
    kv, hd = full.shape[2], full.shape[4]
    assert runs[1].cache.nbytes() * 16 == runs[0].cache.nbytes() * 5          # 1.25 bytes for 4
    code, step, lo = plain_kv4.read(four, hd)
    live = torch.zeros(full.shape[0], 64, dtype=torch.bool)
    for s in slots:
        for c, page in enumerate(runs[1].cache.groups[0].pages.blocks[s]):
            assert page == runs[0].cache.groups[0].pages.blocks[s][c]
            if page >= 0:
                live[page, :max(0, min(64, runs[1].length(s) - 64 * c))] = True
    c, st, low = plain_kv4.quantise(full.double())
    at = live[:, None, None, :].expand(code.shape[:4])
    assert at.any() and torch.equal(code[at], c[at]) and torch.equal(step[at], st[at]) and torch.equal(lo[at], low[at])
    if cfg.sliding_window is None:                            # (a window gives pages back, with what was written)
        assert (code[~at] == 0).all()                         # nothing was written anywhere else


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["B", "A64"])
def test_replayed_steps_give_the_same_bits(tmp_path, name, dtype):
    """Sequences that come and go, so that pages lie in any order: graphs against kernel by kernel, and the plain kernels near both."""
    folder = folder_of(tmp_path, name)
    cfg = config_of(folder)
    seqs = random_prompts(cfg.vocab_size, [40, 90, 9, 130, 66, 20], seed=6)
    logits = []
    for kw in (dict(), dict(use_graphs=False)):
        eng = engine(folder, dtype, max_tokens=64 * 10, cache_format="int4", **kw)
        out, slots = [], []
        for r in range(3):
            slots = [eng.open() for _ in range(2)]
            out.append(eng.step([(s, seqs[2 * r + i]) for i, s in enumerate(slots)]))
            for i in range(5):
                out.append(eng.step([(s, [7 * i + r]) for s in slots]))
            out.append(eng.step([(slots[0], [1, 2, 3]), (slots[1], [4])], want="all"))
            eng.close(slots[r % 2])
            extra = eng.open()
            out.append(eng.step([(extra, seqs[r]), (slots[1 - r % 2], [3])]))
            eng.close(extra)
            eng.close(slots[1 - r % 2])
        eng.check()
        logits.append(torch.cat(out))
        assert (eng.graph_replays > 0) == (not kw) and eng.cache.pages_in_use() == [0] * len(eng.cache.groups)
    assert torch.equal(*logits)


def test_tables_built_on_the_device_are_the_hosts(tmp_path):
    folder = folder_of(tmp_path, "B")
    eng = engine(folder, "float32", max_tokens=64 * 12, cache_format="int4")
    K = eng.kernels
    host, here = StepPacker(DEV, 4), StepPacker(DEV, 4)
    lists = [[[3, 5], [-1, -1, 7], [0]], [[1, 2], [3, 4, 6], [8]]]
    for tokens, before in (([[1], [2], [3]], [70, 140, 0]), ([[1, 2, 3], [4], [5, 6]], [100, 150, 9])):
        for bucket in (False, True):
            want = [[len(t) - 1] for t in tokens]
            tables = [torch.tensor([b + [-1] * (3 - len(b)) for b in ls], dtype=torch.int32).numpy() for ls in lists]
            a = host.pack([4, 2, 9], tokens, before, want, tables, bucket_tables=bucket)
            for replayed in (False, True):
                b = here.pack_lengths([4, 2, 9], tokens, before, want, lists, [10, 10], bucket_tables=bucket)
                here.upload_lengths(b, K, replayed)
                K.check_device_errors()
                for name in ("token_ids", "positions", "token_seq", "q_start", "q_len", "kv_before", "slot_ids", "want_rows"):
                    assert getattr(a, name).tolist() == getattr(b, name).tolist(), name
                for name in ("rows", "n_tokens", "n_seqs", "n_want", "max_q_len", "max_kv_len", "all_decode"):
                    assert getattr(a, name) == getattr(b, name), name
                for x, y in zip(a.page_tables, b.page_tables):
                    assert torch.equal(x, y)
                for ls, place in zip(lists, b.places):
                    at = [ls[i][(p + j) // 64] * 64 + (p + j) % 64 for i, (t, p) in enumerate(zip(tokens, before)) for j in range(len(t))]
                    assert place.tolist() == at + [-1] * (b.rows - len(at))
                assert not bucket or here.token_source_view.tolist() == [0, 1, 2]


def test_generation_and_full_cache(tmp_path):
    folder = folder_of(tmp_path, "A64")
    m = lib.load(folder, dtype="bfloat16", max_seq_len=128, max_batch=3, verbose=False, cache_format="int4")
    prompts = random_prompts(256, [20, 3, 50], seed=1)
    a = [o.tokens for o in m.generate(prompts, lib.SamplingParams.greedy(), [], 20)]
    b = [o.tokens for o in m.generate(prompts, lib.SamplingParams.greedy(), [], 20)]
    assert a == b and [len(t) for t in a] == [20] * 3
    s = m.open()
    with pytest.raises(lib.CacheError if hasattr(lib, "CacheError") else RuntimeError, match="cache is full"):
        m.step([(s, [1] * 400)])
    m.close(s)
    assert [o.tokens for o in m.generate(prompts, lib.SamplingParams.greedy(), [], 20)] == a


def test_refusals(tmp_path):
    folder = make_folder(tmp_path, "A")                       # heads of 16
    with pytest.raises(ValueError, match="heads of 32"):
        engine(folder, "bfloat16", cache_format="int4")
    with pytest.raises(ValueError, match="cache format"):
        engine(folder, "bfloat16", cache_format="int3")
    from bidinex_tiny import BX_A                             # latent attention
    from braidinfer_b200.engine import Engine
    with pytest.raises(ValueError, match="not held in 4 bits"):
        Engine.from_random(BX_A, 0, dtype="bfloat16", max_tokens=128, verbose=False, cache_format="int4")
