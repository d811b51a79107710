"""The 4-bit cache on the GPU where its kernels meet others: what follows them in the stream, steps that leave them nothing to do."""
import pytest
import torch

from braidinfer_b200.csrc.api import Kernels
from test_gpu_kv4 import BF, DEV, F32, K, U, Case, dev  # noqa: F401 (K is a fixture)

pytestmark = pytest.mark.gpu


def arguments(c, out, max_q=None, window=None):
    return (c.q, out, c.cache, c.table.to(DEV), c.start.to(DEV), dev(c.q_len), dev(c.before), c.seq.to(DEV), len(c.q_len), max_q or max(c.q_len),
            max(n + b for n, b in zip(c.q_len, c.before)), c.nqh, c.nkh, c.hd, window, c.hd ** -0.5)


@pytest.mark.parametrize("slices", [None, 3])
@pytest.mark.parametrize("seqs", [[(60, 0), (60, 40)], [(300, 3000), (200, 2500), (9, 4000)]], ids=["short", "long"])
def test_what_follows_prompts_without_short_sequences(K, monkeypatch, seqs, slices):
    """A settled step whose bound on the tokens a sequence is its rows: the kernel for sequences of few tokens runs behind the prompts', and
    finds none.  What comes next in the stream starts as soon as that one has ended, and has to see the prompts' results."""
    if slices:
        monkeypatch.setattr(Kernels, "_kv4_prompt_slices", lambda *a: slices)
    c = Case(K, seqs, 32, 8, 128, BF, pad=8)
    ran, mma = [], K._attn_kv4_mma
    monkeypatch.setattr(K, "_attn_kv4_mma", lambda *a: (ran.append(a[-2:]), mma(*a)))
    out, next_to = torch.empty(c.rows, 32 * 128, dtype=BF, device=DEV), torch.empty(c.rows, 32 * 128, device=DEV)
    args = arguments(c, out, max_q=c.rows)
    K.attn_kv4(*args)                                         # (every kernel waits for the one ahead of it from its start)
    torch.cuda.synchronize()
    want = out.float()
    want[sum(c.q_len):] = 9.0
    ran.clear()
    for _ in range(30):
        out.fill_(9.0)
        K.attn_kv4(*args, settled=True)
        K.cast(out, next_to)
        assert torch.equal(next_to, want)
    K.check_device_errors()
    assert ran == [(True, 2)] * 30                            # (settled, sequences of up to two tokens)


# ------------------------------------------------------------------ warps that walk many units
HEADS = [64, 128, 160, 256]                                   # units of 64 tokens, and of 32 above 128


def one_slice(K, monkeypatch, hd):
    """A context is not sliced: four warps walk all of it, a unit each in turn."""
    monkeypatch.setitem(K.kv4_attention_library(hd).plans, 0, (1, [0] * 5))
    monkeypatch.setitem(K.kv4_attention_library(hd).plans, 1, (1, [0] * 5))


def refill(K, c, keys=None, values=None, seed=5):
    """The sequences' keys and values anew: functions of (numbers [tokens, kv heads, head], positions [tokens, 1, 1], length)."""
    x = torch.randn(2, c.num * 64, c.nkh, c.hd, generator=torch.Generator().manual_seed(seed))
    for i, (n, b) in enumerate(zip(c.q_len, c.before)):
        t = torch.arange(n + b)
        at = c.table[i].long()[t // 64] * 64 + t % 64
        for plane, f in enumerate((keys, values)):
            if f is not None:
                x[plane, at] = f(x[plane, at], t[:, None, None], n + b)
    K.kv4_store(x[0].flatten(1).to(DEV), x[1].flatten(1).to(DEV), dev(torch.arange(c.num * 64)), c.cache, c.hd)


@pytest.mark.parametrize("hd", HEADS)
@pytest.mark.parametrize("first, later", [(None, 1e10), (1e-18, 1e21), (1e-24, 1e30)])
def test_steps_far_above_the_first_units(K, monkeypatch, hd, first, later):
    """A group's scale comes from the first unit that a warp walks: later steps that pass float32's range times that scale are not lost."""
    one_slice(K, monkeypatch, hd)
    c = Case(K, [(1, 700), (3, 600)], 8, 2, hd, BF)
    refill(K, c, values=lambda x, t, n: torch.where(t < 256, x * first if first else torch.full_like(x, 3.0), x * later))
    c.check(K)


@pytest.mark.parametrize("seqs", [[(1, 700), (2, 600)], [(130, 600), (40, 500)]], ids=["few", "prompts"])
@pytest.mark.parametrize("hd", HEADS)
@pytest.mark.parametrize("power", [12, 20, 30, 40, 60])
def test_large_values_without_probability(K, monkeypatch, hd, power, seqs):
    """The first tokens' values are 2^power times the others', and their scores 50 lower: the result is all the others', whose products with
    their probabilities must keep their bits."""
    one_slice(K, monkeypatch, hd)
    monkeypatch.setattr(Kernels, "KV4_PAGES_FROM", 0)
    c = Case(K, seqs, 8, 2, hd, BF)
    c.q = c.q.clone()
    c.q[:, ::hd] = 8.0

    def keys(x, t, n):
        x[..., :1] = torch.where(t < 256, -50.0 / 8 * hd ** 0.5, 0.0)
        return x
    refill(K, c, keys=keys, values=lambda x, t, n: torch.where(t < 256, x, x * 2.0 ** -power))
    out = c.check(K)
    # prompts' float16 operands: half a step of 2^-12 for a key, a query, a value and a probability, and the result's bfloat16
    want, mag, smag = c.want()
    most = mag * (2 * (2 * 2.0 ** -12 * smag[1] + 32 * U * smag[0])[..., None] + 2 * 2.0 ** -12 + 2.0 ** -18) + 2.0 ** -8 * want.abs()
    assert ((out.double().view(want.shape) - want).abs() <= most)[:sum(c.q_len)].all()


@pytest.mark.parametrize("dt", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("hd", HEADS)
@pytest.mark.parametrize("rise", [0.0, 3.0, -3.0])
def test_many_units_a_warp(K, monkeypatch, hd, rise, dt):
    """Rings that are filled again and again, and maxima that rise all along the context (or fall: the first keeps to the end)."""
    one_slice(K, monkeypatch, hd)
    c = Case(K, [(1, 3000), (4, 2111), (2, 0), (3, 1300)], 8, 2, hd, dt)
    c.q = c.q.clone()
    c.q[:, ::hd] = 8.0

    def keys(x, t, n):
        x[..., :1] = rise * t / n * hd ** 0.5
        return x
    refill(K, c, keys=keys)
    out = c.check(K)
    assert torch.equal(c.run(K), out)
    c.check(K, window=1500, head_sinks=torch.linspace(-3, 3, 8, device=DEV))
    c.check(K, window=700, keep_first=500)


@pytest.mark.parametrize("hd", HEADS)
@pytest.mark.parametrize("at", [0.3, 0.97])
@pytest.mark.parametrize("factor", [1e6, 1e-12])
def test_second_walks_after_many_units(K, monkeypatch, hd, at, factor):
    """The values' sizes change where a warp has walked many units: it begins again, with its ring as it then stands."""
    one_slice(K, monkeypatch, hd)
    c = Case(K, [(1, 3000), (4, 2111), (1, 100), (3, 1300)], 8, 2, hd, BF)
    refill(K, c, values=lambda x, t, n: torch.where(t < at * n, x, x * factor))
    out = c.check(K)
    assert torch.equal(c.run(K), out)
    c.check(K, window=1500)


@pytest.mark.parametrize("hd, tokens", [(32, 131075), (160, 65539)])
def test_more_tiles_of_prompts_than_a_grid_is_deep(K, hd, tokens):
    """128 heads a kv head: a CTA takes 2 tokens, one of heads above 128, and the two here are more than 65,535.  Plain attention is within their
    roundings."""
    assert -(-tokens // (2 if hd <= 128 else 1)) > 65535
    g, nqh, window, blocks = torch.Generator(device=DEV).manual_seed(hd), 128, 24, -(-tokens // 64)
    x = torch.randn(2, 64 * blocks, hd, generator=g, device=DEV).to(BF)
    cache = torch.zeros(blocks, 1, K.kv4_page_bytes(hd), dtype=torch.uint8, device=DEV)
    every = torch.arange(64 * blocks, dtype=torch.int32, device=DEV)
    K.kv4_store(x[0], x[1], every, cache, hd)
    q = torch.randn(tokens + 3, nqh * hd, generator=g, device=DEV).to(BF)
    seq = torch.zeros(tokens + 3, dtype=torch.int32, device=DEV)
    seq[tokens:] = -1
    assert K._kv4_as_pages(q, q, tokens, tokens, 1, nqh, 1, hd, True)
    out = []
    for backend in ("auto", "plain"):
        out.append(torch.full((tokens + 3, nqh * hd), 9.0, dtype=BF, device=DEV))
        K.attn_kv4(q, out[-1], cache, every[None, :blocks].contiguous(), dev([0]), dev([tokens]), dev([0]), seq, 1, tokens, tokens, nqh, 1, hd, window, hd ** -0.5,
                   backend=backend)
    K.check_device_errors()
    a, b = out
    assert (a[tokens:] == 9).all() and (b[tokens:] == 9).all()
    # a score is off by 2^-12 of its products twice (|q| |k| hd^-1/2 of them: 1.2 hd^1/2), a probability by twice that; these are independent of the values, as
    # the values are of one another, so that a row of thousands of numbers is off by as much of its length
    most = 2 * 2 * 2.0 ** -12 * 1.2 * hd ** 0.5 + 2 * 2.0 ** -12 + 2 * 2.0 ** -9
    for i in range(0, tokens, 8192):
        x, y = (t[i:min(i + 8192, tokens)].float() for t in out)
        assert ((x - y).norm(dim=1) <= most * y.norm(dim=1)).all()


@pytest.mark.parametrize("far", [2 ** 31 - 65, 2 ** 31 - 1, 2 ** 31, 2 ** 40])
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("dt", [BF, F32], ids=["bf16", "f32"])
def test_windows_and_kept_tokens_of_any_size(K, monkeypatch, dt, new, far):
    """A window, or kept first tokens, past all there is (and past 32 bits) hide nothing."""
    monkeypatch.setattr(Kernels, "KV4_PAGES_FROM", 0)
    c = Case(K, [(new, 500), (new, 0)], 4, 2, 64, dt)
    for kw in (dict(window=far), dict(window=7, keep_first=far), dict(window=far, keep_first=far)):
        for backend in ("auto", "plain"):
            c.check(K, backend=backend, **kw)
    table = dev(torch.arange(8)[None])
    pages, want = (torch.zeros(c.num, 2, 2, 64, 64, device=DEV) for _ in range(2))
    K.kv4_expand(c.cache, pages, table[:, :8].contiguous(), dev([1]), dev([500]), window=3, keep_first=far)
    K.kv4_expand(c.cache, want, table[:, :8].contiguous(), dev([1]), dev([500]))
    K.check_device_errors()
    assert torch.equal(pages, want)
