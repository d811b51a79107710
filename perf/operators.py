"""What a step does with a cache held in 4 bits, operator by operator, as cases that can be timed and compared.

tables   the page tables, positions and cache places of a step's rows, from the lengths of its requests
store    keys and values of new rows into pages of 4-bit numbers, and the pages read back as a chunked prompt reads them
attend   attention over such pages: one or a few tokens a request (decoding, drafts), and prompts

The format, per token and kv head: groups of 32 neighbouring numbers of the head share a step and a lowest value, both
bfloat16; a number is lowest + step * code, code 0 .. 15.  With x the number rounded to bfloat16 and lo, hi a group's lowest and
highest, step = bfloat16((hi - lo) / 15) and code = round((x - lo) / step), ties to even, kept within 0 .. 15 (0 where the step
is 0); a group whose range is not finite reads as NaN.  A page holds 64 tokens of every kv head as four records of 16
tokens: the key codes, the value codes, the keys' groups, the values' groups (uint8 [pages, kv heads, 64 (head + head / 4)]).
Key codes: 32-bit word j head/32 + w of a token holds numbers 32 w + 8 j + 2 n + b in bits 16 b + 4 n (j, n 0 .. 3; b 0, 1);
value codes: 16-bit word i head/32 + w holds numbers 32 w + 4 i + n in bits 4 n (i 0 .. 7); a group's 32-bit word holds its step
below its lowest value.

`own` False: elementary torch operations in float32.  `own` True: the library's kernels.  `exact`: 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
PAGE = 64
LOG2E = 1.4426950408889634


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # a decoding step of a small batch: the tables of 8 requests that bring a token each
        dict(name="tables of 8 decoding requests", op="tables", requests=8, before=4096, new=1, pad=0),
        # a busy server's step: chunks of prompts beside decoding requests, long contexts
        dict(name="tables of 200 mixed requests", op="tables", requests=200, before=32000, new=160, pad=37),
        # the cache write of a decoding step, sizes of the 7B preset
        dict(name="store 8 decoded rows", op="store", requests=8, before=1500, new=1, kv=8, dim=128, heads=32, f32=False),
        # the cache write of a step of prompts
        dict(name="store 5 prompts", op="store", requests=5, before=0, new=1600, kv=8, dim=128, heads=32, f32=False),
        # the same in a float32 run, small heads, chunks behind a cached start
        dict(name="store chunks float32", op="store", requests=3, before=700, new=500, kv=2, dim=64, heads=8, f32=True),
        # decoding: a small batch with short contexts (latency counts)
        dict(name="decode 8 at 1k", op="attend", requests=8, before=1100, new=1, kv=8, dim=128, heads=32, window=0, sinks=False, f32=False),
        # decoding: a large batch with contexts of all lengths (bytes count)
        dict(name="decode 64 at 8k", op="attend", requests=64, before=8190, new=1, kv=8, dim=128, heads=32, window=0, sinks=False, f32=False),
        # decoding: one request at the longest context that a preset allows
        dict(name="decode 1 at 128k", op="attend", requests=1, before=131071, new=1, kv=8, dim=128, heads=32, window=0, sinks=False,
             f32=False),
        # a few tokens a request (a checked draft) with the sliding window of the 7B preset and sinks
        dict(name="drafts of 5 in a window", op="attend", requests=6, before=9000, new=5, kv=8, dim=128, heads=32, window=4096, sinks=True,
             f32=False),
        # decoding in a float32 run
        dict(name="decode float32", op="attend", requests=4, before=3001, new=1, kv=2, dim=64, heads=8, window=0, sinks=False, f32=True),
        # prompts of several lengths together
        dict(name="3 prompts", op="attend", requests=3, before=0, new=1800, kv=8, dim=128, heads=32, window=0, sinks=False, f32=False),
        # a chunk of a prompt behind a long cached start
        dict(name="chunk behind 16k", op="attend", requests=1, before=16500, new=700, kv=8, dim=128, heads=32, window=0, sinks=False,
             f32=False),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tables", "store", "attend", "attend"])
    if op == "tables":
        n = _spread(rng, 1, 500)
        return dict(op=op, requests=n, before=_spread(rng, 1, 32000), new=_spread(rng, 1, max(2, 30000 // n)), pad=rng.randrange(64))
    kv = rng.choice([1, 2, 4, 8])
    dim = rng.choice([32, 64, 96, 128, 128, 256])
    shape = dict(kv=kv, dim=dim, heads=kv * rng.choice([1, 2, 3, 4, 5, 8]))
    if op == "store":
        n = _spread(rng, 1, 40)
        return dict(op=op, requests=n, before=rng.choice([0, _spread(rng, 1, 3000)]), new=_spread(rng, 1, max(2, 6000 // n)), f32=rng.random() < 0.3,
                    **shape)
    f32 = rng.random() < 0.25
    window = rng.choice([0, 0, _spread(rng, 50, 5000)])
    sinks = rng.random() < 0.3
    if f32 or rng.random() < 0.6:
        n = _spread(rng, 1, 64)
        return dict(op=op, requests=n, before=_spread(rng, 1, min(131071, 400000 // n)), new=rng.choice([1, 1, 1, rng.randrange(2, 9)]), window=window, sinks=sinks,
                    f32=f32, **shape)
    n = _spread(rng, 1, 12)
    return dict(op=op, requests=n, before=rng.choice([0, _spread(rng, 1, 16000)]), new=_spread(rng, 9, max(10, 2400 // n)), window=window, sinks=sinks, f32=False,
                **shape)


def _lengths(case):
    """(tokens that the requests bring, tokens cached before), part of the case: the first request has the most of both, the
    others any number."""
    g = torch.Generator().manual_seed(5)
    n, before, new = case["requests"], case["before"], case["new"]
    b = torch.randint(before // 2, before + 1, (n,), generator=g)
    b[0] = before
    if case["op"] == "tables" and new > 1:
        q = torch.randint(1, new + 1, (n,), generator=g)
        q[torch.rand(n, generator=g) < 0.4] = 1              # some requests decode
    elif new <= 8:
        q = torch.full((n,), new)
    else:
        q = torch.randint(new // 3, new + 1, (n,), generator=g)
    q[0] = new
    return q, b


# ------------------------------------------------------------------------------------------------ inputs
def _groups(x):
    """x [..., head] float32, numbers of bfloat16 -> codes uint8 [..., head], steps and lowest values bfloat16 [..., head / 32]."""
    x = x.unflatten(-1, (-1, 32))
    lo, hi = x.amin(-1), x.amax(-1)
    span = hi - lo
    fifteen = torch.full((), 15.0, device=x.device)
    step = (span / fifteen).to(torch.bfloat16)
    bad = ~torch.isfinite(span)
    step, lo = step.masked_fill(bad, math.nan), lo.masked_fill(bad, math.nan)
    s = step.float()[..., None]
    code = torch.where(s > 0, (x - lo[..., None]) / s, 0.0).round().clamp(0, 15)
    return torch.where(bad[..., None], 0.0, code).to(torch.uint8).flatten(-2), step, lo.to(torch.bfloat16)


def _words(step, lo):
    """Steps and lowest values [..., groups] -> bytes [..., 4 groups]."""
    return torch.stack([step, lo], -1).contiguous().view(torch.uint8).flatten(-2)


def _pages(k, v):
    """Keys and values of whole pages [pages, kv, 64, head] (numbers of bfloat16, float32) -> uint8 [pages, kv, bytes]."""
    p, kv, _, dim = k.shape
    w = dim // 32
    kc, ks, kl = _groups(k)
    c = kc.view(p, kv, 4, 16, w, 4, 2, 2, 2)                                       # group, j, upper half of n, lower half of n, b
    kb = (c[..., 0, :] | (c[..., 1, :] << 4)).permute(0, 1, 2, 3, 5, 4, 7, 6).reshape(p, kv, 4, -1)
    vc, vs, vl = _groups(v)
    c = vc.view(p, kv, 4, 16, w, 8, 2, 2)                                          # group, i, upper half of n, lower half of n
    vb = (c[..., 0] | (c[..., 1] << 4)).permute(0, 1, 2, 3, 5, 4, 6).reshape(p, kv, 4, -1)
    kw, vw = (_words(s, l).view(p, kv, 4, -1) for s, l in ((ks, kl), (vs, vl)))
    return torch.cat([kb, vb, kw, vw], -1).view(p, kv, -1)


def _random_pages(pages, kv, dim, g):
    """Pages of keys (some channels far from zero, as trained keys have them) and values."""
    out = torch.empty(pages, kv, PAGE * (dim + dim // 4), dtype=torch.uint8, device=DEVICE)
    shift = torch.randn(kv, 1, dim, generator=g, device=DEVICE) * (torch.rand(kv, 1, dim, generator=g, device=DEVICE) < 0.1) * 3
    some = max(1, (1 << 26) // (kv * PAGE * dim))
    for p in range(0, pages, some):
        n = min(some, pages - p)
        k = (torch.randn(n, kv, PAGE, dim, generator=g, device=DEVICE) + shift).to(torch.bfloat16).float()
        v = torch.randn(n, kv, PAGE, dim, generator=g, device=DEVICE).to(torch.bfloat16).float()
        out[p:p + n] = _pages(k, v)
    return out


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    q_len, before = _lengths(case)
    n = len(q_len)
    total = int(q_len.sum())
    rows = total + case.get("pad", 0)
    blocks = (q_len + before + PAGE - 1) // PAGE
    cols = int(blocks.max())
    spare = 1000 if case["op"] == "tables" else 3             # pages that no request holds
    pages = int(blocks.sum()) + spare
    at = torch.randperm(pages, generator=torch.Generator().manual_seed(seed + 1))
    i32 = dict(dtype=torch.int32, device=DEVICE)
    st = dict(case=case, rows=rows, total=total, n=n, cols=cols, pages=pages, max_q=int(q_len.max()), max_kv=int((q_len + before).max()),
              q_len=q_len.to(**i32), before=before.to(**i32), held=at[:pages - spare].to(**i32))
    table = torch.full((n, cols), -1, dtype=torch.int64)
    start, row0, seq = 0, [], torch.full((rows,), -1, dtype=torch.int64)
    place, r = torch.full((rows,), -1, dtype=torch.int64), 0
    for i in range(n):
        table[i, :blocks[i]] = at[start:start + int(blocks[i])]
        start += int(blocks[i])
        row0.append(r)
        t = int(q_len[i])
        pos = int(before[i]) + torch.arange(t)
        seq[r:r + t] = i
        place[r:r + t] = table[i, pos // PAGE] * PAGE + pos % PAGE
        r += t
    if case["op"] == "tables":
        st.update(table=torch.empty(n, cols, **i32), place=torch.empty(rows, **i32), positions=torch.empty(rows, **i32), seq=torch.empty(rows, **i32),
                  q_start=torch.empty(n, **i32))
        return st
    st.update(table=table.to(**i32), q_start=torch.tensor(row0).to(**i32), seq=seq.to(**i32), place=place.to(**i32))
    kv, dim, heads = case["kv"], case["dim"], case["heads"]
    dt = torch.float32 if case["f32"] else torch.bfloat16
    st["cache"] = _random_pages(pages, kv, dim, g)
    # a step's rows: query heads, key heads, value heads side by side, as the projection leaves them
    qkv = torch.randn(rows, (heads + 2 * kv) * dim, generator=g, device=DEVICE).to(dt)
    st["q"], st["k"], st["v"] = qkv[:, :heads * dim], qkv[:, heads * dim:(heads + kv) * dim], qkv[:, (heads + kv) * dim:]
    if case["op"] == "store":
        st["out"] = torch.zeros(pages, 2, kv, PAGE, dim, dtype=dt, device=DEVICE)
    else:
        st["out"] = torch.zeros(rows, heads * dim, dtype=dt, device=DEVICE)
        st["sinks"] = torch.randn(heads, generator=g, device=DEVICE) if case["sinks"] else None
    return st


# ------------------------------------------------------------------------------------------------ the library's calls
_kernels = None


def _own(st):
    global _kernels
    if _kernels is None:
        from braidinfer_b200.csrc.api import get_kernels
        _kernels = get_kernels(verbose=False)
    K, case = _kernels, st["case"]
    if case["op"] == "tables":
        K.step_tables(st["q_len"], st["before"], st["held"], st["table"], st["place"], num_pages=st["pages"], positions=st["positions"],
                      token_seq=st["seq"], q_start=st["q_start"])
        return dict(table=st["table"], place=st["place"], positions=st["positions"], seq=st["seq"], q_start=st["q_start"])
    if case["op"] == "store":
        K.kv4_store(st["k"], st["v"], st["place"], st["cache"], case["dim"])
        K.kv4_expand(st["cache"], st["out"], st["table"], st["q_len"], st["before"])
        return st["out"]
    K.attn_kv4(st["q"], st["out"], st["cache"], st["table"], st["q_start"], st["q_len"], st["before"], st["seq"], st["n"], st["max_q"],
               st["max_kv"], case["heads"], case["kv"], case["dim"], case["window"] or None, case["dim"] ** -0.5, head_sinks=st["sinks"])
    return st["out"]


# ------------------------------------------------------------------------------------------------ the plain form
def _values(pages, dim):
    """Bytes [..., kv, bytes of a page] -> keys and values [..., kv, 64, head], float32."""
    lead, w = pages.shape[:-1], dim // 32
    r = pages.unflatten(-1, (4, -1))
    kb, vb, kw, vw = r.split([8 * dim, 8 * dim, 2 * dim, 2 * dim], -1)
    c = kb.reshape(*lead, 4, 16, 4, w, 2, 2).transpose(-1, -2)                     # j, group, upper n, b
    c = torch.stack([c & 15, c >> 4], -2)                                          # ..., upper n, lower n, b
    k = c.flatten(-3).transpose(-2, -3).flatten(-3).flatten(-3, -2).unflatten(-1, (w, 32))
    c = vb.reshape(*lead, 4, 16, 8, w, 2)
    c = torch.stack([c & 15, c >> 4], -1).flatten(-2)
    v = c.transpose(-2, -3).flatten(-3).flatten(-3, -2).unflatten(-1, (w, 32))
    found = []
    for code, word in ((k, kw), (v, vw)):
        p = word.contiguous().view(torch.bfloat16).reshape(*lead, PAGE, w, 2).float()
        found.append((p[..., 1:] + p[..., :1] * code).flatten(-2))
    return found


def _plain_tables(st):
    q, before, dev = st["q_len"].long(), st["before"].long(), DEVICE
    blocks = (q + before + PAGE - 1) // PAGE
    ends, b_ends = q.cumsum(0), blocks.cumsum(0)
    c = torch.arange(st["cols"], device=dev)
    table = torch.where(c < blocks[:, None], st["held"].long()[((b_ends - blocks)[:, None] + c).clamp(max=len(st["held"]) - 1)], -1)
    r = torch.arange(st["rows"], device=dev)
    seq = torch.searchsorted(ends, r, right=True)
    live = r < ends[-1]
    seq = torch.where(live, seq, 0)
    pos = torch.where(live, before[seq] + r - (ends - q)[seq], 0)
    place = torch.where(live, table[seq, pos // PAGE] * PAGE + pos % PAGE, -1)
    i = torch.int32
    return dict(table=table.to(i), place=place.to(i), positions=pos.to(i), seq=torch.where(live, seq, -1).to(i), q_start=(ends - q).to(i))


def _plain_store(st):
    case = st["case"]
    kv, dim, pages = case["kv"], case["dim"], st["pages"]
    k, v = _values(st["cache"], dim)
    both = torch.stack([k, v], 1)                                                   # pages, 2, kv, 64, head
    place = st["place"].long()
    new = []
    for x in (st["k"], st["v"]):
        x = x.reshape(-1, kv, dim).to(torch.bfloat16).float()
        code, step, lo = _groups(x)
        new.append((lo.float()[..., None] + step.float()[..., None] * code.unflatten(-1, (-1, 32))).flatten(-2))
    both[place // PAGE, :, :, place % PAGE] = torch.stack(new, 1)
    # the requests' tokens only; what no request holds is not asked for
    end = (st["q_len"] + st["before"]).long()
    c = torch.arange(st["cols"], device=DEVICE)
    there = torch.zeros(pages + 1, dtype=torch.int64, device=DEVICE)
    there[st["table"].long()] = (end[:, None] - c * PAGE).clamp(0, PAGE)            # (-1: the last, which no page is)
    seen = torch.arange(PAGE, device=DEVICE) < there[:pages, None]
    return torch.where(seen[:, None, None, :, None], both, 0.0).to(st["out"].dtype)


def _plain_attend(st):
    case = st["case"]
    kv, dim, heads, n, t = case["kv"], case["dim"], case["heads"], st["n"], st["max_q"]
    k, v = _values(st["cache"][st["table"].long().clamp(min=0)], dim)               # n, cols, kv, 64, head
    k, v = (x.transpose(1, 2).flatten(2, 3) for x in (k, v))                        # n, kv, keys, head
    i = torch.arange(t, device=DEVICE)
    q_len, before = st["q_len"].long()[:, None], st["before"].long()[:, None]
    live = i < q_len
    row = torch.where(live, st["q_start"].long()[:, None] + i, 0)
    q = st["q"][row].float().view(n, t, kv, heads // kv, dim).permute(0, 2, 3, 1, 4).flatten(2, 3)
    s = (q @ k.transpose(-1, -2)) * dim ** -0.5
    pos = before + i
    key = torch.arange(k.shape[2], device=DEVICE)
    ok = key <= pos[..., None]
    if case["window"]:
        ok &= pos[..., None] - key < case["window"]
    s = s.view(n, kv, heads // kv, t, -1).masked_fill_(~ok[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    p = (s - m).exp_()
    total = p.sum(-1, keepdim=True)
    if st["sinks"] is not None:
        total = total + (st["sinks"].view(1, kv, -1, 1, 1) - m).exp()
    o = (p.flatten(2, 3) @ v).view(n, kv, heads // kv, t, dim) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(n, t, heads * dim).to(st["out"].dtype)
    out = torch.zeros_like(st["out"])
    out[row[live]] = o[live]
    return out


def run(st):
    if own:
        return _own(st)
    return {"tables": _plain_tables, "store": _plain_store, "attend": _plain_attend}[st["case"]["op"]](st)


# ------------------------------------------------------------------------------------------------ work, 64 bits
def work(case):
    q, before = _lengths(case)
    n, total = len(q), int(q.sum())
    blocks = int(((q + before + PAGE - 1) // PAGE).sum())
    if case["op"] == "tables":
        cols = -(-(case["before"] + case["new"]) // PAGE)
        return {"bytes": 4 * (3 * n + blocks + n * cols + 3 * (total + case["pad"])), "flops": 0}
    kv, dim, heads, size = case["kv"], case["dim"], case["heads"], 4 if case["f32"] else 2
    token = kv * (dim + dim // 4)                                                    # a cached token: codes and groups of key and value
    if case["op"] == "store":
        kept = int((q + before).sum())
        return {"bytes": total * (2 * kv * dim * size + token) + kept * token + blocks * PAGE * 2 * kv * dim * size + 4 * total, "flops": 0}
    pairs = seen = 0
    for a, b in zip(q.tolist(), before.tolist()):
        w = case["window"] or a + b
        seen += min(a + b, w + a - 1)
        full = max(0, min(a, b + a - w + 1 if b + a >= w else 0))                     # tokens that see a whole window
        part = a - full
        pairs += full * w + part * b + part * (part + 1) // 2
    return {"bytes": seen * token + 2 * total * heads * dim * size, "flops": 4 * pairs * heads * dim}


def _numbers(pages, dim):
    """The two planes of `pages`' bytes as float64 numbers, by where each number of a head lies."""
    d = torch.arange(dim, device=DEVICE)
    grp, low = d // 32, d % 32
    # bit of the number within a token's codes
    kbit = 32 * ((low // 8) * (dim // 32) + grp) + 16 * (low % 2) + 4 * ((low % 8) // 2)
    vbit = 16 * ((low // 4) * (dim // 32) + grp) + 4 * (low % 4)
    tok = torch.arange(PAGE, device=DEVICE)[:, None]
    rec, t = (tok // 16) * (20 * dim), tok % 16
    b = pages.to(torch.int32)

    def number(code0, bit, word0):
        code = (b[..., rec + code0 + t * (dim // 2) + bit // 8] >> (bit % 8)) & 15
        w = rec + word0 + (t * (dim // 32) + grp) * 4
        step, lo = ((((b[..., w + o] | (b[..., w + o + 1] << 8)) << 16).view(torch.float32)).double() for o in (0, 2))
        return lo + step * code

    return number(0, kbit, 16 * dim), number(8 * dim, vbit, 18 * dim)


def _exact_store(st, case):
    kv, dim = case["kv"], case["dim"]
    out = torch.zeros(st["pages"], 2, kv, PAGE, dim, dtype=torch.float64, device=DEVICE)
    k, v = _numbers(st["cache"], dim)
    for i in range(st["n"]):
        end = int(st["q_len"][i] + st["before"][i])
        for c in range(-(-end // PAGE)):
            p, m = int(st["table"][i, c]), min(PAGE, end - c * PAGE)
            out[p, 0, :, :m], out[p, 1, :, :m] = k[p, :, :m], v[p, :, :m]
    for plane, rows in enumerate((st["k"], st["v"])):
        x = rows.to(torch.bfloat16).double().reshape(-1, kv, dim // 32, 32)
        lo, hi = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
        step = ((hi - lo) / 15).to(torch.bfloat16).double()
        code = torch.round((x - lo) / torch.where(step > 0, step, 1.0)).clamp(0, 15) * (step > 0)
        place = st["place"].long()
        out[place // PAGE, plane, :, place % PAGE] = (lo + step * code).reshape(-1, kv, dim)
    return out


def exact(case, seed):
    if case["op"] == "tables":
        return None
    st = prepare(case, seed)
    if case["op"] == "store":
        return _exact_store(st, case)
    w = work(case)
    if w["flops"] > 1e13:
        return None
    kv, dim, heads = case["kv"], case["dim"], case["heads"]
    g = heads // kv
    out = torch.zeros(st["rows"], heads, dim, dtype=torch.float64, device=DEVICE)
    for i in range(st["n"]):
        a, b, r = int(st["q_len"][i]), int(st["before"][i]), int(st["q_start"][i])
        k, v = _numbers(st["cache"][st["table"][i, :-(-(a + b) // PAGE)].long()], dim)
        q = st["q"][r:r + a].double().view(a, heads, dim)
        for h in range(heads):
            keys, vals = (x[:, h // g].reshape(-1, dim)[:a + b] for x in (k, v))
            j = torch.arange(a + b, device=DEVICE)
            p = torch.arange(b, a + b, device=DEVICE)[:, None]
            s = q[:, h] @ keys.T / math.sqrt(dim)
            hidden = (j > p) | ((p - j >= case["window"]) if case["window"] else torch.zeros_like(j > p))
            s[hidden] = -math.inf
            if st["sinks"] is not None:
                s = torch.cat([s, st["sinks"][h].double().expand(a, 1)], 1)
            out[r:r + a, h] = torch.softmax(s, -1)[:, :a + b] @ vals
    return out.view(st["rows"], -1)
