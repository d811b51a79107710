"""The 4-bit cache on the GPU (csrc/kv4.cu, csrc/attn_kv4.cu) against the plain form in 64 bits (plain_kv4.py).

Tolerances.  The codes are exact, so pages have to be equal byte for byte, and read-back values to a float32 or bfloat16 rounding.
Attention: a score is a sum of 32-bit products.  The tensor cores take the codes 128 higher; with smag[0] a score's products so, and
U = 2^-24 a unit of float32, a group's sum is cut off twice (4 U each), the queries' own sum is rounded 5 times, and two
multiply-adds a group join them: 16 U smag[0], which moves every probability by twice that and the exponentials' 2^-21.  In bfloat16 runs each probability times a group's
step is rounded by 2^-8 of itself, and so is the result; prompts read keys and values as bfloat16 numbers: 2^-8 of a score's
products and of a value.  Sums over the keys lose 2 U a tile of 16."""
import math

import pytest
import torch

import plain_kv4 as P
from braidinfer_b200.csrc.api import KernelError, Kernels, get_kernels

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24


@pytest.fixture(scope="module")
def K():
    return get_kernels(verbose=False)


@pytest.fixture(params=["auto", "pages"])
def route(request, monkeypatch):
    """Prompts as the sizes have it (here: over 4 bits), and over pages read back."""
    if request.param == "pages":
        monkeypatch.setattr(Kernels, "KV4_PAGES_FROM", 0)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def dev(x, dt=torch.int32):
    return torch.as_tensor(x).to(dt).to(DEV)


# ------------------------------------------------------------------ tables
@pytest.mark.parametrize("q_len, before, pad, extra_cols", [
    ([1], [0], 0, 0), ([1], [63], 0, 0), ([1], [64], 3, 2), ([3, 0, 5], [0, 0, 128], 0, 0), ([0, 0], [0, 130], 4, 1), ([64, 65, 1], [64, 0, 127], 31, 5),
    ([1] * 300, [i * 7 for i in range(300)], 0, 0), ([2] * 5000, [i % 70 for i in range(5000)], 9, 0), ([40000], [100000], 1, 0)])
def test_tables(K, q_len, before, pad, extra_cols):
    blocks = [-(-(q + b) // 64) for q, b in zip(q_len, before)]
    num, rows, cols = sum(blocks) + 3, sum(q_len) + pad, max(blocks) + extra_cols
    pages = torch.randperm(num, generator=gen(len(q_len)))[:sum(blocks)].tolist()
    at = 0
    for q, b, n in zip(q_len, before, blocks):               # blocks that a window has given back
        if b > 200:
            pages[at] = -1
        at += n
    want = P.tables(q_len, before, pages, rows, cols)
    n = len(q_len)
    table, place, pos, seq, start = (torch.full(s, 77, dtype=torch.int32, device=DEV) for s in ((n, cols), (rows + 1,), (rows + 1,), (rows + 1,), (n + 1,)))
    K.step_tables(dev(q_len), dev(before), dev(pages), table, place[:rows], num_pages=num, positions=pos[:rows], token_seq=seq[:rows], q_start=start[:n])
    K.check_device_errors()
    for got, w in zip((table, place[:rows], pos[:rows], seq[:rows], start[:n]), want):
        assert got.tolist() == w
    assert place[rows] == pos[rows] == seq[rows] == start[n] == 77
    again, place2 = torch.empty_like(table), torch.empty_like(place[:rows])
    K.step_tables(dev(q_len), dev(before), dev(pages), again, place2, num_pages=num)     # the others are not asked for
    assert torch.equal(again, table) and torch.equal(place2, place[:rows])


@pytest.mark.parametrize("q_len, before, listed, rows, cols, num", [
    ([3, 4], [0, 0], [0, 1], 6, 1, 9),             # more tokens than rows
    ([3, 4], [0, 61], [0, 1], 7, 2, 9),            # fewer pages than blocks
    ([3, 4], [0, 61], [0, 1, 2], 7, 1, 9),         # a request of more blocks than the table has columns
    ([3, 4], [0, 0], [0, 9], 7, 1, 9),             # a page outside the cache
    ([3, 4], [0, 0], [-5, 0], 7, 1, 9),
    ([3, 4], [0, 0], [0, -1], 7, 1, 9),            # a new token's block was given back
    ([-3, 4], [0, 0], [0, 1], 7, 1, 9), ([3, 4], [0, -64], [0, 1], 7, 1, 9),
    ([2 ** 31 - 1, 4], [2 ** 31 - 1, 0], [0, 1], 7, 1, 9), ([2, 4], [2 ** 31 - 2, 0], [0, 1], 7, 1, 9)])
def test_tables_flag_what_does_not_fit(K, q_len, before, listed, rows, cols, num):
    table, place, pos, seq = (torch.full((s + 8,), 77, dtype=torch.int32, device=DEV) for s in (2 * cols, rows, rows, rows))
    K.step_tables(dev(q_len), dev(before), dev(listed), table[:2 * cols].view(2, cols), place[:rows], num_pages=num, positions=pos[:rows], token_seq=seq[:rows])
    with pytest.raises(KernelError, match="lengths of a step's requests"):
        K.check_device_errors()
    assert all((t[-8:] == 77).all() for t in (table, place, pos, seq))
    assert ((table[:-8] >= -1) & (table[:-8] < num)).all() and ((place[:-8] >= -1) & (place[:-8] < 64 * num)).all()


# ------------------------------------------------------------------ write, read back
def odd_rows(rows, kv, hd, g):
    x = torch.randn(rows, kv, hd, generator=g, dtype=torch.float64) * torch.rand(rows, 1, 1, generator=g) * 4
    x[0] = 3.0                                                # a group without a range
    x[1, 0, :32] = torch.arange(32) * 0.5                     # ties
    if rows > 8:
        x[2, -1, 5] = math.nan
        x[3, -1, 31] = -math.inf
        x[4, 0, :2] = torch.tensor([3e38, -3e38])             # a range past float32
        x[5, 0] = torch.randn(hd, generator=g) * 1e-39        # numbers below float32's normal ones
        x[6, 0] = 1000 + torch.arange(hd)
        x[7, 0, 1:32] = 0
    return x


@pytest.mark.parametrize("hd", range(32, 257, 32))
@pytest.mark.parametrize("dt, kv, shift", [(BF, 1, 0), (BF, 2, 8), (F32, 3, 0), (BF, 3, 1), (F32, 2, 3)])
def test_store_and_read_back(K, hd, dt, kv, shift):
    g = gen(hd + kv)
    rows, pages = 37, 4
    wide = torch.zeros(rows, 2 * kv * hd + shift + 8)
    k, v = odd_rows(rows, kv, hd, g), odd_rows(rows, kv, hd, g).flip(0)
    wide[:, shift:shift + kv * hd], wide[:, shift + kv * hd:shift + 2 * kv * hd] = k.flatten(1), v.flatten(1)
    wide = wide.to(dt)
    x = [wide[:, shift + i * kv * hd:shift + (i + 1) * kv * hd] for i in (0, 1)]
    place = torch.randperm(64 * pages, generator=g)[:rows]
    place[[9, 20]] = -1
    cache = torch.randint(0, 256, (pages, kv, K.kv4_page_bytes(hd)), generator=g, dtype=torch.uint8)
    want = cache.clone()
    for plane in (0, 1):
        P.write(want, place, plane, x[plane].double().view(rows, kv, hd))
    got, w = cache.to(DEV), wide.to(DEV)
    K.kv4_store(w[:, shift:shift + kv * hd], w[:, shift + kv * hd:shift + 2 * kv * hd], dev(place), got, hd)
    K.check_device_errors()
    assert_pages_equal(got.cpu(), want, hd)
    # all of it read back, but the last page: 20 of its places
    vals = P.numbers(*P.read(got, hd))
    for ot in (F32, BF):
        out = torch.full((pages + 1, 2, kv, 64, hd), 5.0, dtype=ot, device=DEV)[:pages]
        K.kv4_expand(got, out, dev([[2, 0, 3]]), dev([9]), dev([64 * 2 + 11]))
        K.check_device_errors()
        o = out.cpu().double()
        assert (o[1] == 5).all() and (o[3, :, :, 20:] == 0).all()
        for p, n in ((2, 64), (0, 64), (3, 20)):
            a, b = o[p, :, :, :n], vals[p, :, :, :n]
            assert torch.equal(a.isnan(), b.isnan())
            # (the random bytes hold infinities, numbers past the type's largest, and ones below its normal ones: half a step of those)
            inside = b.abs() < 3.3e38
            step, least = (U, 2.0 ** -150) if ot == F32 else (2.0 ** -8 + U, 2.0 ** -134 + 2.0 ** -150)
            assert ((a - b).abs() <= step * b.abs() + least)[inside].all() and (a[b.abs() > 3.42e38].isinf()).all()


def assert_pages_equal(got, want, hd):
    """Equal bytes; the bits of a NaN are whatever they are."""
    a, b = P.read(got, hd), P.read(want, hd)
    assert torch.equal(a[0], b[0])
    for x, y in zip(a[1:], b[1:]):
        assert torch.equal(x.isnan(), y.isnan()) and torch.equal(x.nan_to_num(0), y.nan_to_num(0))


def test_store_outside_and_expand_of_absent_pages(K):
    hd, kv = 64, 2
    cache = torch.zeros(4, kv, K.kv4_page_bytes(hd), dtype=torch.uint8, device=DEV)
    x = torch.randn(3, kv * hd, device=DEV)
    K.kv4_store(x, x, dev([5, 3 * 64, 64]), cache[:2], hd)
    with pytest.raises(KernelError, match="cache write outside"):
        K.check_device_errors()
    assert (cache[2:] == 0).all() and (cache[0] != 0).any() and (cache[1] != 0).any()
    out = torch.zeros(2, 2, kv, 64, hd, device=DEV)
    for page in (-1, 2, 1 << 30):
        K.kv4_expand(cache[:2], out, dev([[0, page]]), dev([1]), dev([70]))
        with pytest.raises(KernelError, match="visible position"):
            K.check_device_errors()
    # blocks behind the window may be absent; kept first ones may not
    K.kv4_expand(cache[:2], out, dev([[-1, -1, 1]]), dev([2]), dev([140]), window=13)
    K.check_device_errors()
    K.kv4_expand(cache[:2], out, dev([[-1, -1, 1]]), dev([2]), dev([140]), window=14)
    with pytest.raises(KernelError, match="visible position"):
        K.check_device_errors()
    K.kv4_expand(cache[:2], out, dev([[0, -1, 1]]), dev([2]), dev([140]), window=13, keep_first=3)
    K.check_device_errors()
    K.kv4_expand(cache[:2], out, dev([[-1, -1, 1]]), dev([2]), dev([140]), window=13, keep_first=3)
    with pytest.raises(KernelError, match="visible position"):
        K.check_device_errors()


# ------------------------------------------------------------------ attention
class Case:
    """Sequences over pages in any order, with rows of padding at the end."""

    def __init__(self, K, seqs, nqh, nkh, hd, dt, seed=0, pad=2, spread=1.0, lowest=None):
        g = gen(seed + hd + nqh)
        self.q_len, self.before = [n for n, _ in seqs], [b for _, b in seqs]
        blocks = [-(-(n + b) // 64) for n, b in seqs]
        self.num, self.rows, self.cols = sum(blocks) + 2, sum(self.q_len) + pad, max(blocks) + 1
        order = torch.randperm(self.num, generator=g)[:sum(blocks)].tolist()
        table, place, _, seq, start = P.tables(self.q_len, self.before, order, self.rows, self.cols)
        self.table, self.seq, self.start = (torch.tensor(x, dtype=torch.int32) for x in (table, seq, start))
        x = torch.randn(2, self.num * 64, nkh, hd, generator=g) * spread
        x[0] += torch.randn(1, nkh, hd, generator=g) * (torch.rand(1, nkh, hd, generator=g) < 0.1) * 3
        self.cache = torch.zeros(self.num, nkh, K.kv4_page_bytes(hd), dtype=torch.uint8, device=DEV)
        every = dev(torch.arange(self.num * 64))
        K.kv4_store(x[0].flatten(1).to(DEV), x[1].flatten(1).to(DEV), every, self.cache, hd)
        self.q = (torch.randn(self.rows, (nqh + 1) * hd, generator=g)).to(dt).to(DEV)[:, :nqh * hd]     # rows wider than the heads
        self.nqh, self.nkh, self.hd, self.dt = nqh, nkh, hd, dt

    def run(self, K, window=None, scale=None, backend="auto", max_kv=None, max_q=None, out=None, **kw):
        out = torch.full((self.rows, self.nqh * self.hd), 9.0, dtype=self.dt, device=DEV) if out is None else out
        K.attn_kv4(self.q, out, self.cache, self.table.to(DEV), self.start.to(DEV), dev(self.q_len), dev(self.before), self.seq.to(DEV), len(self.q_len),
                   max_q or max(self.q_len), max_kv or max(n + b for n, b in zip(self.q_len, self.before)), self.nqh, self.nkh, self.hd, window,
                   scale or self.hd ** -0.5, backend=backend, **kw)
        K.check_device_errors()
        return out

    def want(self, window=None, scale=None, sink=None, out_scale=1.0, head_sinks=None, head_gate=None, keep_first=0, head_scale=None, distance_bias=None,
             softcap=None):
        s = head_sinks if head_sinks is not None else torch.full((self.nqh,), sink) if sink is not None else None
        return P.attend(self.q.double().view(self.rows, self.nqh, self.hd), self.cache, self.table, self.q_len, self.before, scale or self.hd ** -0.5, window,
                        keep_first, s, head_gate.double() if head_gate is not None else None, out_scale, head_scale, distance_bias, softcap)

    def check(self, K, **kw):
        run_only = {k: kw.pop(k) for k in ("backend", "max_kv", "max_q") if k in kw}
        out = self.run(K, **kw, **run_only)
        want, mag, smag = self.want(**kw)
        total = sum(self.q_len)
        assert (out[total:] == 9.0).all()                    # rows of padding stay as they were
        off = (out.double().view(want.shape) - want).abs()[:total]
        score = 16 * U * smag[0]
        prompt = max(self.q_len) > 8 and self.dt == BF
        if prompt:
            score = score + 2.0 ** -8 * smag[1]
        if kw.get("distance_bias") is not None or kw.get("softcap"):
            score = score + 2.0 ** -18 * 60                  # their own float32 forms: a part in 2^18 of up to 60
        keys = max(n + b for n, b in zip(self.q_len, self.before))
        part = 2 * score[..., None] + 2.0 ** -19 + 4 * U * (keys / 16 + 8)
        if self.dt == BF:
            part = part + (2 if prompt else 1) * 2.0 ** -8
        most = mag * part + (2.0 ** -8 if self.dt == BF else 4 * U) * want.abs() + 1e-30
        bad = off > most[:total]
        assert not bad.any(), (bad.sum().item(), off.max().item(), most[:total][bad].min().item())
        return out


SHAPES = [  # sequences (new, before), heads, kv heads, head size
    ([(1, 0)], 1, 1, 32), ([(1, 62), (1, 63), (1, 64), (1, 700)], 4, 1, 64), ([(1, 15), (1, 16), (1, 2000)], 8, 2, 128), ([(1, 333)], 16, 1, 96),
    ([(3, 70), (8, 0), (1, 129)], 6, 2, 64), ([(8, 500)], 32, 4, 128), ([(5, 100), (0, 50), (2, 64)], 5, 5, 160), ([(1, 90), (4, 3)], 24, 1, 32),
    ([(1, 1000)], 40, 2, 192), ([(2, 40), (7, 300)], 9, 3, 224), ([(1, 127), (6, 128)], 8, 1, 256), ([(1, 17)], 66, 1, 64)]


@pytest.mark.parametrize("backend", ["plain", "auto"])
@pytest.mark.parametrize("dt", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("seqs, nqh, nkh, hd", SHAPES)
def test_few_tokens(K, seqs, nqh, nkh, hd, dt, backend):
    Case(K, seqs, nqh, nkh, hd, dt).check(K, backend=backend)


def test_nothing_to_do(K):
    c = Case(K, [(1, 5)], 2, 1, 64, BF)
    K.attn_kv4(c.q[:0], c.q[:0], c.cache, c.table.to(DEV), dev([0]), dev([0]), dev([5]), dev([]), 1, 1, 6, 2, 1, 64, None, 0.1)
    K.kv4_store(torch.zeros(0, 64, device=DEV), torch.zeros(0, 64, device=DEV), dev([]), c.cache, 64)
    K.step_tables(dev([]), dev([]), dev([]), torch.empty(0, 4, dtype=torch.int32, device=DEV), dev([]), num_pages=3)
    K.check_device_errors()


OPTIONS = {
    "window": dict(window=50), "window 1": dict(window=1), "kept": dict(window=40, keep_first=70), "sink": dict(sink=1.5), "low sink": dict(sink=-1e4),
    "high sink": dict(sink=90.0), "sinks": dict(head_sinks=True, out_scale=0.25), "gate": dict(head_gate=True, window=100), "scaled": dict(head_scale=True, scale=0.3),
    "bias": dict(distance_bias=True, window=130), "cap": dict(softcap=3.0, scale=0.5), "negative": dict(scale=-0.2, window=33, keep_first=5)}


def options(name, rows, nqh, dt, seed=3):
    g = gen(seed)
    kw = dict(OPTIONS[name])
    rnd = lambda *s: torch.randn(*s, generator=g)
    for key, make in (("head_sinks", lambda: rnd(nqh).to(DEV)), ("head_gate", lambda: rnd(rows, nqh + 3).to(dt).to(DEV)[:, 1:nqh + 1]),
                      ("head_scale", lambda: rnd(nqh).to(DEV)), ("distance_bias", lambda: (rnd(nqh).abs().to(DEV), rnd(nqh).abs().to(DEV)))):
        if kw.get(key) is True:
            kw[key] = make()
    return kw


@pytest.mark.parametrize("backend", ["plain", "auto"])
@pytest.mark.parametrize("dt", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("name", OPTIONS)
def test_options(K, name, dt, backend):
    c = Case(K, [(1, 200), (4, 130), (2, 0), (1, 63)], 10, 2, 64, dt)
    c.check(K, backend=backend, **options(name, c.rows, c.nqh, dt))


@pytest.mark.parametrize("dt", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("seqs, nqh, nkh, hd", [
    ([(9, 0)], 4, 2, 64), ([(130, 0), (17, 200)], 8, 2, 128), ([(64, 64), (1, 500), (0, 9), (33, 31)], 3, 1, 32), ([(70, 5)], 20, 1, 96), ([(40, 100)], 2, 2, 256),
    ([(12, 1000)], 6, 1, 160)])
def test_prompts(K, route, seqs, nqh, nkh, hd, dt):
    Case(K, seqs, nqh, nkh, hd, dt).check(K)


@pytest.mark.parametrize("slices", [2, 3, 8])
@pytest.mark.parametrize("name, hd", [("window", 64), ("sink", 128), ("sinks", 64), ("gate", 128), ("bias", 64), ("cap", 128), ("window", 96), ("gate", 32),
                                      ("window", 256), ("sinks", 160)])
def test_prompts_in_slices(K, monkeypatch, name, hd, slices):
    """The context cut into slices, some of them without a key that a row sees, or without any."""
    monkeypatch.setattr(Kernels, "KV4_PAGES_FROM", 0)
    monkeypatch.setattr(Kernels, "_kv4_prompt_slices", lambda *a: slices)
    c = Case(K, [(70, 900), (150, 0), (1, 100), (9, 333)], 8, 2, hd, BF)
    c.check(K, **options(name, c.rows, c.nqh, BF))


@pytest.mark.parametrize("slices", [None, 3])
@pytest.mark.parametrize("room", [1 << 30, 1])
@pytest.mark.parametrize("name, hd", [("window", 128), ("sinks", 64)])
def test_prompts_beside_single_tokens(K, monkeypatch, name, hd, room, slices):
    """Sequences of up to 2 tokens (8 columns of queries) are computed over 4 bits, the others over pages, a few sequences at a time."""
    monkeypatch.setattr(Kernels, "KV4_PAGES_FROM", 0)
    monkeypatch.setattr(Kernels, "KV4_PAGES_BYTES", room)
    if slices:
        monkeypatch.setattr(Kernels, "_kv4_prompt_slices", lambda *a: slices)
    c = Case(K, [(1, 3000), (200, 100), (8, 64), (9, 10), (0, 5), (1, 0), (3, 700), (1, 500), (20, 0)], 8, 2, hd, BF)
    ran = []
    mma = K._attn_kv4_mma
    monkeypatch.setattr(K, "_attn_kv4_mma", lambda *a: (ran.append(a[-1]), mma(*a)))
    c.check(K, **options(name, c.rows, c.nqh, BF))
    assert ran == [2]
    # one prompt of many tokens beside another: all of them over pages
    c = Case(K, [(200, 100), (150, 30), (1, 64)], 8, 2, hd, BF)
    c.check(K, **options(name, c.rows, c.nqh, BF))
    assert ran == [2]


@pytest.mark.parametrize("dt", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("name", OPTIONS)
def test_options_of_prompts(K, route, name, dt):
    c = Case(K, [(50, 100), (90, 0), (1, 300)], 4, 2, 64, dt)
    c.check(K, **options(name, c.rows, c.nqh, dt))


@pytest.mark.parametrize("new", [1, 6, 40])
@pytest.mark.parametrize("dt", [BF, F32], ids=["bf16", "f32"])
def test_what_is_not_seen_does_not_count(K, route, dt, new):
    """NaN in places behind the sequence's end and before its window, and in pages that no sequence holds; the values of a sequence
    whose own keys hold a NaN are NaN, and its neighbour's are not."""
    c = Case(K, [(new, 150), (new, 90)], 4, 2, 64, dt)
    clean = c.run(K, window=20)
    _, mag, smag = c.want(window=20)
    L = [n + b for n, b in zip(c.q_len, c.before)]
    held = {}
    for i in (0, 1):
        for blk in range(-(-L[i] // 64)):
            held[int(c.table[i, blk])] = (i, blk)
    bad = []
    for p in range(c.num):
        for t in range(64):
            i, blk = held.get(p, (None, 0))
            at = blk * 64 + t
            if i is None or at >= L[i] or at <= c.before[i] - 20:
                bad.append(p * 64 + t)
    nan = torch.full((len(bad), 2 * 64), math.nan, device=DEV)
    K.kv4_store(nan, nan, dev(bad), c.cache, 64)
    assert torch.equal(c.run(K, window=20), clean)
    # the second sequence's own last key
    last = int(c.table[1, (L[1] - 1) // 64]) * 64 + (L[1] - 1) % 64
    K.kv4_store(nan[:1], nan[:1], dev([last]), c.cache, 64)
    out = c.run(K, window=20)
    # (tokens that share a product's columns with the NaN may be computed in the kernel's other form: each is within its roundings of
    # the exact result, 2^-8 twice a bfloat16 number and prompts 2^-8 a key and value more, so they are within twice that of one another)
    n = 2 * new - 1
    part = 2 * 16 * U * smag[0] + (2 * 2.0 ** -8 * smag[1] if dt == BF and new > 8 else 0)
    most = 2 * (mag * (part[..., None] + 2.0 ** -18 + (2 * 2.0 ** -8 if dt == BF else 0)) + (2.0 ** -8 if dt == BF else 4 * U) * clean.double().view(mag.shape).abs())
    assert ((out.double() - clean.double()).view(mag.shape).abs() <= most)[:n].all() and out[n].isnan().all() and (out[n + 1:] == 9).all()
    assert torch.equal(out[:new], clean[:new])               # the other sequence is not touched at all


@pytest.mark.parametrize("backend", ["plain", "auto"])
@pytest.mark.parametrize("new", [1, 30])
def test_absent_pages_are_flagged(K, route, new, backend):
    c = Case(K, [(new, 100)], 4, 2, 64, BF)
    for page in (-1, c.num, 1 << 30):
        c.table[0, 0] = page
        with pytest.raises(KernelError, match="visible position"):
            c.run(K, backend=backend)
    c.table[0, 0] = -1
    c.run(K, backend=backend, window=30)                      # behind the window: nobody asks for it


def test_large_scores_and_small_ones(K):
    for spread, scale in ((100.0, 1.0), (1e-3, 1.0), (1e4, 1e-9), (1.0, 0.0)):
        c = Case(K, [(1, 300), (3, 64)], 8, 2, 128, F32, spread=spread)
        for dt in (F32, BF):
            c.dt, c.q = dt, c.q.to(dt)
            out = c.run(K, scale=scale or 1e-30)
            plain = c.run(K, scale=scale or 1e-30, backend="plain")
            want, mag, smag = c.want(scale=scale or 1e-30)
            n = 4
            smag = smag[0]
            rows = (smag[:n] < 2.0 ** 10)[..., None]          # rows whose scores are not all rounding
            for o in (out, plain):
                off = (o.double().view(want.shape) - want).abs()[:n]
                most = mag[:n] * (32 * U * smag[:n][..., None] + 2.0 ** -18 + (2.0 ** -8 if dt == BF else 0)) + (2.0 ** -8 if dt == BF else 4 * U) * want[:n].abs()
                assert o[:n].isfinite().all() and (off <= most)[rows.expand_as(off)].all()


SIZES = {  # factors on the values by position, on the keys, on the queries
    "grow": (lambda t: 10.0 ** (60.0 * t - 30), 1.0, 1.0), "shrink": (lambda t: 10.0 ** (30 - 60.0 * t), 1.0, 1.0), "tiny": (lambda t: 1e-30 + 0 * t, 1.0, 1.0),
    "huge": (lambda t: 1e30 + 0 * t, 1.0, 1.0), "one step up": (lambda t: 1 + 1e25 * (t > 0.5), 1.0, 1.0), "small queries": (lambda t: 1 + 0 * t, 1e15, 1e-15),
    "small keys": (lambda t: 1 + 0 * t, 1e-20, 1e20), "constant": (lambda t: 0 * t, 1.0, 1.0)}


@pytest.mark.parametrize("seqs", [[(1, 700), (3, 90)], [(200, 500), (60, 0)]], ids=["few", "prompts"])
@pytest.mark.parametrize("dt", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("name", SIZES)
def test_values_of_all_sizes(K, monkeypatch, name, dt, seqs):
    """Values whose sizes lie far apart within a sequence, and keys and queries that make up for each other: what is scaled on the way
    must not leave its range.  (Values grow before they shrink: a result then hangs on the largest ones that its probabilities keep.)"""
    monkeypatch.setattr(Kernels, "KV4_PAGES_FROM", 0)
    grow, fk, fq = SIZES[name]
    c = Case(K, seqs, 8, 2, 128, dt)
    g = gen(5)
    x = torch.randn(2, c.num * 64, 2, 128, generator=g)
    for i in (0, 1):
        L = c.q_len[i] + c.before[i]
        t = torch.arange(L)
        at = c.table[i].long()[t // 64] * 64 + t % 64
        x[1, at] = x[1, at] * grow(t / L)[:, None, None].float() + (3e4 if name == "constant" else 0.0)
    K.kv4_store((x[0] * fk).flatten(1).to(DEV), x[1].flatten(1).to(DEV), dev(torch.arange(c.num * 64)), c.cache, 128)
    c.q = (c.q.float() * fq).to(dt)
    c.check(K)
    c.check(K, backend="plain")


@pytest.mark.parametrize("hd", [64, 128, 224])
def test_a_bad_query_spoils_its_row_alone(K, monkeypatch, hd):
    monkeypatch.setattr(Kernels, "KV4_PAGES_FROM", 0)
    c = Case(K, [(150, 100), (30, 0)], 4, 2, hd, BF)
    clean = c.run(K).view(c.rows, 4, hd)
    c.q = c.q.clone()
    c.q[5, 3], c.q[140, hd + 1], c.q[160, 2 * hd:3 * hd] = math.nan, math.inf, 0.0
    out = c.run(K).view(c.rows, 4, hd)
    assert out[5, 0].isnan().all() and out[140, 1].isnan().all() and out[160, 2].isfinite().all()
    spoilt = torch.zeros(c.rows, 4, dtype=torch.bool, device=DEV)
    spoilt[5, 0] = spoilt[140, 1] = spoilt[160, 2] = True
    assert torch.equal(out[~spoilt], clean[~spoilt])


def test_long_float32_sums_have_no_bias(K, monkeypatch):
    """One slice of 40,000 tokens in float32.  Keys' and probabilities' errors are independent, as the values are, so that their share of the
    result is at most a probability's largest error: 16 2^-24 of a score's products and 8 2^-24.  Sums that are cut off at every 16 tokens, 625 times a
    warp and three times each, would be off by up to 1,875 2^-24."""
    monkeypatch.setitem(K.kv4_attention_library(32).plans, 1, (1, [0] * 5))
    c = Case(K, [(1, 40000)], 8, 4, 32, F32)
    out = c.run(K)[:1].double()
    want, _, smag = c.want()
    want = want[:1].flatten(1)
    assert (out - want).norm() <= (16 * smag[0].max() + 8) * U * want.norm()


def test_more_tiles_than_a_grid_is_deep(K):
    """A token a tile, 70,001 of them (a window keeps the plain kernel's share small): both are within their roundings of the exact result."""
    c = Case(K, [(70001, 30)], 8, 1, 32, F32)
    out, plain = c.run(K, window=40), c.run(K, window=40, backend="plain")
    n = 70001
    assert (out[n:] == 9).all()
    # scores of 32 numbers below 2^6, sums of 40: 16 2^-24 of the scores' products and some 2^-19 of the weights, of values up to 8
    assert (out[:n] - plain[:n]).abs().max() <= 2 * 8 * (2 * 16 * U * 64 + 2.0 ** -19)


@pytest.mark.parametrize("slices", [1, 3])
@pytest.mark.parametrize("hd", range(32, 257, 32))
def test_prompts_keep_the_bits_of_the_codes(K, monkeypatch, hd, slices):
    """Queries, keys, values and probabilities of prompts are float16 numbers of 11 bits: half a step is 2^-12 of each (and what lies far below
    the largest of its row or page is off by 2^-25 of that, here less than 2^-11 of a part in 2^12)."""
    monkeypatch.setattr(Kernels, "KV4_PAGES_FROM", 0)
    monkeypatch.setattr(Kernels, "_kv4_prompt_slices", lambda *a: slices)
    c = Case(K, [(150, 1000), (70, 0)], 8, 2, hd, BF)
    out = c.run(K)
    want, mag, smag = c.want()
    n = sum(c.q_len)
    score = 2 * 2.0 ** -12 * smag[1] + 32 * U * smag[0]
    most = mag * (2 * score[..., None] + 2 * 2.0 ** -12 + 2.0 ** -18) + 2.0 ** -8 * want.abs() + 1e-30
    assert ((out.double().view(want.shape) - want).abs() <= most)[:n].all()
    # rows of the result that start on 16 bytes, not on 32
    wide = torch.full((c.rows, c.nqh * hd + 8), 9.0, dtype=BF, device=DEV)
    again = c.run(K, out=wide[:, 8:])
    assert torch.equal(again, out) and (wide[:, :8] == 9).all()


@pytest.mark.parametrize("seqs", [[(1, 9000), (1, 10), (1, 4000)], [(4, 5000)], [(33, 3000)]])
@pytest.mark.parametrize("dt", [BF, F32], ids=["bf16", "f32"])
def test_long_contexts_slices_and_repeats(K, route, seqs, dt):
    c = Case(K, seqs, 8, 2, 64, dt)
    out = c.check(K)
    assert torch.equal(c.run(K), out)
    # bounds above the true lengths only change the slices
    wide = c.run(K, max_kv=20000)
    assert (wide.double() - out.double()).abs().max() <= 2.0 ** -6 * out[:-2].double().abs().max()


def test_run_of_all_of_them(K):
    """A batch as it is served: tables, write and attention step by step, prompts first and then a token each, against one pass
    over whole sequences."""
    hd, nqh, nkh, num = 64, 8, 2, 40
    g = gen(8)
    lens = [70, 1, 129]
    cache = torch.zeros(num, nkh, K.kv4_page_bytes(hd), dtype=torch.uint8, device=DEV)
    free = torch.randperm(num, generator=g).tolist()
    held = [[], [], []]
    before = [0, 0, 0]
    mirror = torch.zeros(num, nkh, K.kv4_page_bytes(hd), dtype=torch.uint8)
    for step in range(4):
        new = lens if step == 0 else [1, 1, 1] if step < 3 else [2, 65, 1]
        rows, pad = sum(new), 5
        for h, n, b in zip(held, new, before):
            while len(h) * 64 < n + b:
                h.append(free.pop())
        qkv = torch.randn(rows + pad, (nqh + 2 * nkh) * hd, generator=g).to(BF).to(DEV)
        table, place = torch.empty(3, 8, dtype=torch.int32, device=DEV), torch.empty(rows + pad, dtype=torch.int32, device=DEV)
        pos, seq, start = torch.empty_like(place), torch.empty_like(place), torch.empty(3, dtype=torch.int32, device=DEV)
        q_len, kvb = dev(new), dev(before)
        K.step_tables(q_len, kvb, dev(sum(held, [])), table, place, num_pages=num, positions=pos, token_seq=seq, q_start=start)
        k, v = qkv[:, nqh * hd:(nqh + nkh) * hd], qkv[:, (nqh + nkh) * hd:]
        K.kv4_store(k, v, place, cache, hd)
        out = torch.zeros(rows + pad, nqh * hd, dtype=BF, device=DEV)
        longest = max(n + b for n, b in zip(new, before))
        K.attn_kv4(qkv, out, cache, table, start, q_len, kvb, seq, 3, max(new), longest, nqh, nkh, hd, None, hd ** -0.5)
        K.check_device_errors()
        for plane, x in ((0, k), (1, v)):
            P.write(mirror, place.cpu(), plane, x.cpu().double().view(-1, nkh, hd))
        want, mag, smag = P.attend(qkv[:, :nqh * hd].double().view(-1, nqh, hd).cpu(), mirror, table.cpu(), new, before, hd ** -0.5)
        off = (out.cpu().double().view(want.shape) - want).abs()
        assert (off <= mag * (2.0 ** -7 + 2 * (2.0 ** -8 * smag[1] + 16 * U * smag[0])[..., None]) + 2.0 ** -8 * want.abs()).all()
        before = [n + b for n, b in zip(new, before)]


KINDS = {"few": ([(1, 300), (2, 64)], 8, 2, 64), "slices": ([(1, 20000)], 4, 1, 128), "prompts": ([(130, 200), (90, 0)], 8, 4, 128),
         "prompts of other heads": ([(130, 200), (90, 0)], 8, 4, 160)}


@pytest.mark.parametrize("kind", KINDS)
def test_graphs_and_streams_keep_apart(K, monkeypatch, kind):
    """The same call on two inputs, captured into graphs that replay at the same time, and on two streams at once."""
    if "prompts" in kind:
        monkeypatch.setattr(Kernels, "KV4_PAGES_FROM", 0)
    seqs, nqh, nkh, hd = KINDS[kind]
    cases = [Case(K, seqs, nqh, nkh, hd, BF, seed=s) for s in (1, 2)]
    want = [c.run(K) for c in cases]
    assert not torch.equal(*want)
    args, outs = [], [torch.empty_like(w) for w in want]
    for c, o in zip(cases, outs):
        args.append((c.q, o, c.cache, c.table.to(DEV), c.start.to(DEV), dev(c.q_len), dev(c.before), c.seq.to(DEV), len(seqs), max(c.q_len),
                     max(n + b for n, b in seqs), nqh, nkh, hd, None, hd ** -0.5))
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    graphs = []
    for a, s in zip(args, streams):
        with torch.cuda.stream(s):
            K.attn_kv4(*a)                                    # (libraries and attributes are set up outside of a capture)
            s.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                K.attn_kv4(*a)
            graphs.append(g)
    for how in ("graphs", "streams"):
        for _ in range(20):
            for o in outs:
                o.fill_(9.0)
            torch.cuda.synchronize()
            for _ in range(3):
                for a, s, g in zip(args, streams, graphs):
                    with torch.cuda.stream(s):
                        g.replay() if how == "graphs" else K.attn_kv4(*a)
            torch.cuda.synchronize()
            for o, w in zip(outs, want):
                assert torch.equal(o, w)
    K.check_device_errors()


@pytest.mark.parametrize("dt", [BF, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("seqs", [[(1, 100)], [(3, 9000)], [(140, 30)]])
def test_rows_that_start_anywhere(K, route, seqs, dt):
    c = Case(K, seqs, 6, 2, 64, dt)
    want = c.run(K)
    wide = torch.zeros(c.rows, 6 * 64 + 5, dtype=dt, device=DEV)
    wide[:, 3:3 + 6 * 64] = c.q
    c.q = wide[:, 3:3 + 6 * 64]
    out = torch.full((c.rows, 6 * 64 + 7), 9.0, dtype=dt, device=DEV)
    c.run(K, out=out[:, 1:1 + 6 * 64])
    off = (out[:, 1:1 + 6 * 64].double() - want.double()).abs().max()
    # (prompts that start on no 16 bytes go over 4 bits, where keys and values are not rounded: two roundings of 2^-8, and the results')
    assert (out[:, 0] == 9).all() and (out[:, 1 + 6 * 64:] == 9).all() and off <= (2.0 ** -6 if dt == BF else 2.0 ** -20) * want.abs().max()


def test_places_of_one_step_in_any_order(K):
    """Rows whose places are neighbours go through many threads at once: every byte is one row's."""
    hd, kv, rows = 128, 4, 6000
    g = gen(3)
    x = torch.randn(2, rows, kv * hd, generator=g).to(BF)
    place = torch.randperm(64 * 100, generator=g)[:rows]
    cache = torch.zeros(100, kv, K.kv4_page_bytes(hd), dtype=torch.uint8, device=DEV)
    K.kv4_store(x[0].to(DEV), x[1].to(DEV), dev(place), cache, hd)
    K.check_device_errors()
    code, step, lo = P.read(cache, hd)
    for plane in (0, 1):
        c, s, l = P.quantise(x[plane].double().view(rows, kv, hd))
        p, t = place // 64, place % 64
        assert torch.equal(code[p, plane, :, t], c) and torch.equal(step[p, plane, :, t], s) and torch.equal(lo[p, plane, :, t], l)
