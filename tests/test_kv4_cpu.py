"""The 4-bit cache without a GPU: the oracle's format, and what the entry points refuse."""
import ctypes
import math

import pytest
import torch

import plain_kv4 as P
from braidinfer_b200.csrc import api, build
from braidinfer_b200.csrc.api import KernelError, Kernels


def test_format_of_the_oracle():
    hd = 64
    x = torch.arange(2 * hd, dtype=torch.float64).view(1, 2, hd) * 0.5 - 3.0
    pages = torch.zeros(2, 2, P.PAGE * (hd + hd // 4), dtype=torch.uint8)
    P.write(pages, torch.tensor([64 + 17]), 1, x)
    code, step, lo = P.read(pages, hd)
    got = P.numbers(code, step, lo)[1, 1, :, 17]
    assert ((got - x[0]).abs() <= step[1, 1, :, 17].repeat_interleave(32, -1) / 2 + 2.0 ** -8 * x[0].abs()).all()
    # token 17 of the page is token 1 of record 1; number 0 of a head is the lowest (code 0), number 31 the highest of its group
    at = 20 * hd + 8 * hd + hd // 2
    assert code[1, 1, 0, 17, 31] == 15 and (pages[1, 0, at + 2 * 7 * 2 + 1] >> 4) == 15       # 16-bit word 7 * 2 + 0, bits 12..15
    assert (pages[0] == 0).all()
    # every bit of a token's codes belongs to one number
    for hd in range(32, 257, 32):
        for b in P.bits(hd):
            assert sorted((b // 4).tolist()) == list(range(hd)) and (b % 4 == 0).all()


def test_groups_of_the_oracle():
    x = torch.zeros(5, 32, dtype=torch.float64)
    x[0] = 7.0                                                # no range
    x[1, 3] = math.inf
    x[2, 4] = math.nan
    x[3, :2] = torch.tensor([3e38, -3e38])                    # a range past float32
    x[4] = torch.arange(32) * 0.5                             # ties: step 15.5 / 15 rounded to bfloat16
    code, step, lo = P.quantise(x)
    assert (code[:4] == 0).all() and step[0] == 0 and lo[0] == 7 and step[1:4].isnan().all() and lo[1:4].isnan().all()
    assert step[4] == 1.03125 and code[4].max() == 15 and code[4, 0] == 0


@pytest.fixture
def K():
    """The bindings without a device: refusals come before any launch, and the fake device index refuses the rest."""
    k = object.__new__(Kernels)
    k._part_libs, k._attn_libs, k._verbose, k._device_index, k.launches = {}, {}, False, 0, 0
    k._error_flag = torch.zeros(8, dtype=torch.int32)
    k._stream = lambda: None
    return k


def i32(*s):
    return torch.zeros(*s, dtype=torch.int32)


def attend_args(hd=64, nqh=4, nkh=2, rows=3, n=2, dt=torch.bfloat16):
    return dict(q=torch.zeros(rows, nqh * hd, dtype=dt), out=torch.zeros(rows, nqh * hd, dtype=dt),
                cache=torch.zeros(5, nkh, 64 * (hd + hd // 4), dtype=torch.uint8), page_table=i32(n, 3), q_start=i32(n), q_len=i32(n),
                kv_before=i32(n), token_seq=i32(rows), n_seqs=n, max_q_len=2, max_kv_len=100, nqh=nqh, nkh=nkh, hd=hd, window=None, scale=0.1)


BAD_ATTENTION = [
    dict(cache=torch.zeros(5, 2, 64 * 80, dtype=torch.int8)), dict(cache=torch.zeros(5, 2, 64 * 64, dtype=torch.uint8)),
    dict(cache=torch.zeros(5, 3, 64 * 80, dtype=torch.uint8)), dict(hd=48), dict(hd=288), dict(nqh=3), dict(nqh=0),
    dict(q=torch.zeros(3, 255, dtype=torch.bfloat16)), dict(q=torch.zeros(2, 256, dtype=torch.bfloat16)), dict(q=torch.zeros(3, 256)),
    dict(q=torch.zeros(256, 3, dtype=torch.bfloat16).T), dict(q=torch.zeros(3, 256, dtype=torch.float16), out=torch.zeros(3, 256, dtype=torch.float16)),
    dict(token_seq=i32(2)), dict(q_len=i32(1)), dict(q_start=torch.zeros(2, dtype=torch.int64)), dict(page_table=i32(1, 3)), dict(page_table=i32(6)),
    dict(page_table=i32(2, 6)[:, ::2]), dict(softcap=-1.0), dict(softcap=0.0), dict(softcap=1.0, distance_bias=(torch.zeros(4), torch.zeros(4))),
    dict(head_sinks=torch.zeros(3)), dict(head_scale=torch.zeros(4, dtype=torch.float64)), dict(head_gate=torch.zeros(3, 3, dtype=torch.bfloat16)),
    dict(head_gate=torch.zeros(2, 4, dtype=torch.bfloat16)), dict(keep_first=-1, window=4), dict(window=-1), dict(backend="other"), {},
]


@pytest.mark.parametrize("change", BAD_ATTENTION, ids=lambda c: "-".join(c) or "cpu")
def test_attention_refuses(K, change):
    with pytest.raises(KernelError):
        K.attn_kv4(**{**attend_args(), **change})             # (the last is whole, and refused for lying on the CPU)
    assert K.launches == 0


def test_others_refuse(K):
    cache = torch.zeros(5, 2, 64 * 80, dtype=torch.uint8)
    kv, place = torch.zeros(3, 128), i32(3)
    for bad in (dict(k=kv[:, :127]), dict(v=kv[:2]), dict(k=kv.bfloat16()), dict(place=i32(2)), dict(place=place.long()), dict(cache=cache[:, :1]), dict(hd=32),
                dict(cache=cache.float()), dict(k=kv.half(), v=kv.half()), {}):
        with pytest.raises(KernelError):
            K.kv4_store(**{**dict(k=kv, v=kv, place=place, cache=cache, hd=64), **bad})
    out = torch.zeros(5, 2, 2, 64, 64)
    for bad in (dict(out=out[:4]), dict(out=out[:, :1]), dict(out=torch.zeros(5, 2, 3, 64, 64)), dict(out=torch.zeros(5, 2, 2, 64, 96)), dict(out=out.half()),
                dict(q_len=i32(1)), dict(page_table=i32(2, 3).long()), dict(out=torch.zeros(5, 2, 2, 32, 64)), {}):
        with pytest.raises(KernelError):
            K.kv4_expand(**{**dict(cache=cache, out=out, page_table=i32(2, 3), q_len=i32(2), kv_before=i32(2)), **bad})
    for bad in (dict(q_len=i32(3)), dict(kv_before=i32(1)), dict(pages=i32(4).long()), dict(positions=i32(3)), dict(token_seq=i32(4).float()), dict(q_start=i32(1)),
                dict(page_table=i32(6)), {}):
        with pytest.raises(KernelError):
            K.step_tables(**{**dict(q_len=i32(2), kv_before=i32(2), pages=i32(4), page_table=i32(2, 3), place=i32(4), num_pages=9), **bad})
    assert K.launches == 0
    for hd in (0, 16, 48, 100, 288):
        assert not Kernels.kv4_supports(hd)
        with pytest.raises(KernelError):
            Kernels.kv4_page_bytes(hd)
    assert Kernels.kv4_page_bytes(128) == 64 * 160 and Kernels.kv4_page_bytes(32) == 64 * 40


def test_entry_points_refuse(K):
    """The C entry points themselves, with sizes that the Python side lets through."""
    lib = K.part_library("kv4")
    b = (ctypes.c_int * 64)()
    p = ctypes.addressof(b)
    even = p - p % 16
    tables = lambda n=2, listed=4, rows=4, cols=4, pages=9: lib.braid_step_tables(api._TABLES_ARGS.pack(*[p] * 5, 0, 0, 0, n, listed, rows, cols, pages, p), None)
    # more requests than the tables' shared memory holds; places past 32 bits
    assert tables(n=20000) == tables(pages=1 << 26) == tables(rows=-1) == -1
    store = lambda at=even, rows=3, kind=0, hd=64, kv=2: lib.braid_kv4_store(api._STORE_ARGS.pack(p, p, p, at, p, 128, 128, rows, kv, hd, 5, kind), None)
    assert store(at=even + 4) == store(kind=7) == store(hd=48) == store(hd=288) == store(kv=0) == -1
    expand = lambda at=even, n=2, kind=0: lib.braid_kv4_expand(api._EXPAND_ARGS.pack(even, at, p, p, p, p, 0, 0, 0, 0, n, 2, 64, 3, 5, 0, 0, 0, 0, kind, 0), None)
    assert expand(at=even + 8) == expand(kind=5) == -1 and expand(n=70000) == -1
    assert b"grid" in lib.braid_last_error()
    # nothing to do is no error
    assert tables(n=0, listed=0, rows=0) == store(rows=0) == expand(n=0) == 0
    assert build.page_size() == P.PAGE


def test_mixers_that_a_4_bit_cache_does_not_go_with():
    from braidinfer_b200.cache import CacheError, CacheManager
    from braidinfer_b200.engine.engine import parse_cache_format
    from braidinfer_b200.parts.attention import GQAAttention
    from braidinfer_b200.parts.runtime import Runtime
    from braidinfer_b200.parts.spec import CacheRequest, PartSpec

    def mixer(pe="rope", fmt="int4", **kw):
        rope = PartSpec(pe, {"head_dim": kw.get("head_dim", 64), "theta": 1e4})
        params = dict(hidden_size=64, num_heads=4, num_kv_heads=2, head_dim=64, position_encoding=rope)
        return GQAAttention({**params, **kw}, "l.", Runtime(torch.bfloat16, torch.device("cpu"), None, cache_format=fmt))

    req = mixer().cache_request()
    assert req.four_bit and not mixer(fmt="full").cache_request().four_bit and req.group_key() != mixer(fmt="full").cache_request().group_key()
    assert mixer(qk_norm={"eps": 1e-5, "q_name": "q", "k_name": "k"}).cache_request().four_bit and mixer("none").cache_request().four_bit
    for bad in (dict(head_dim=48), dict(head_dim=288), dict(conv=4), dict(talk="t"), dict(value_from_key=True), dict(pe="none", unit_qk_eps=1e-5)):
        with pytest.raises(ValueError):
            mixer(**bad)
        if "head_dim" not in bad:
            assert mixer(fmt="full", **bad) is not None
    with pytest.raises(ValueError):
        parse_cache_format("int8")
    assert parse_cache_format("int4") == "int4"
    c = CacheManager([(req, None, 0), (req, 0, 0)], 64 * 5, 3, torch.bfloat16, "cpu")
    assert c.four_bit and tuple(c.groups[0].storage.shape) == (1, 5, 2, 64 * 80) and c.groups[0].storage.dtype == torch.uint8
    assert c.layer_view(1).four_bit and c.layer_view(1).read_only
    a, b = c.alloc_slot(), c.alloc_slot()
    assert c.begin_step([b, a], [65, 1], lists=True) == [[[0, 1], [2]]]
    with pytest.raises(CacheError, match="in 4 bits"):
        CacheManager([(req, None, 0), (CacheRequest("full", 2, 64), 0, 0)], 64, 1, torch.bfloat16, "cpu")
