"""A cache held in 4 bits and the attention that reads it, from the format's words and the attention's formula, in 64 bits.

Groups of 32 neighbouring numbers of a head share a step and a lowest value (bfloat16 both); a number is lowest + step * code.
`bits(hd)` says where in a token's codes each number lies; pages are [pages, kv heads, 64 (hd + hd / 4)] bytes, four records of
16 tokens: key codes, value codes, key groups, value groups."""
import math

import torch

PAGE, REC, GROUP = 64, 16, 32


def bf16(x):
    return x.to(torch.float32).to(torch.bfloat16).double()


def quantise(x):
    """x [..., hd] -> (code int64 [..., hd], step, lowest float64 [..., hd / 32])."""
    x = bf16(x).unflatten(-1, (-1, GROUP))
    lo, hi = x.min(-1).values, x.max(-1).values
    span = (hi.float() - lo.float()).double()                 # a range past float32 is infinite
    bad = ~torch.isfinite(span)
    step = bf16(span / 15)
    s = torch.where(bad | (step == 0), 1.0, step)[..., None]
    code = torch.round((x - lo[..., None]) / s).clamp(0, 15)
    code = torch.where((bad | (step == 0))[..., None], 0.0, code)
    nan = torch.full_like(step, math.nan)
    return code.long().flatten(-2), torch.where(bad, nan, step), torch.where(bad, nan, lo)


def numbers(code, step, lo):
    return (lo[..., None] + step[..., None] * code.unflatten(-1, (-1, GROUP))).flatten(-2)


def bits(hd):
    """The bit of every number within its token's key codes and value codes."""
    d = torch.arange(hd)
    w, r, W = d // GROUP, d % GROUP, hd // GROUP
    return 32 * ((r // 8) * W + w) + 16 * (r % 2) + 4 * (r % 8 // 2), 16 * ((r // 4) * W + w) + 4 * (r % 4)


def offsets(plane, hd):
    """Where a plane's codes and groups of the 64 tokens of a page begin: two [64] tensors."""
    t = torch.arange(PAGE)
    rec = t // REC * 20 * hd
    return rec + plane * 8 * hd + t % REC * (hd // 2), rec + (16 + 2 * plane) * hd + t % REC * (hd // 8)


def write(pages, place, plane, x):
    """Rows x [rows, kv, hd] into `pages` (uint8, on the CPU) at their places (-1: nowhere)."""
    kv, hd = x.shape[1:]
    code, step, lo = quantise(x)
    codes = torch.zeros(*code.shape[:-1], hd // 2, dtype=torch.uint8)
    at = bits(hd)[plane]
    for half in (0, 1):                                       # the two codes of every byte
        d = torch.nonzero(at % 8 == 4 * half).flatten()
        codes[..., at[d] // 8] |= (code[..., d] << (4 * half)).to(torch.uint8)
    words = torch.stack([step, lo], -1).to(torch.bfloat16).contiguous().view(torch.uint8).flatten(-2)
    c0, g0 = offsets(plane, hd)
    for r, p in enumerate(place.tolist()):
        if p >= 0:
            page, t = p // PAGE, p % PAGE
            pages[page, :, c0[t]:c0[t] + hd // 2] = codes[r]
            pages[page, :, g0[t]:g0[t] + hd // 8] = words[r]


def read(pages, hd):
    """(code, step, lowest) of both planes: [pages, 2, kv, 64, ...]."""
    b, found = pages.cpu().long(), []
    for plane in (0, 1):
        c0, g0 = offsets(plane, hd)
        at = bits(hd)[plane]
        code = (b[..., c0[:, None] + at // 8] >> (at % 8)) & 15
        g = g0[:, None] + 4 * torch.arange(hd // GROUP)
        step, lo = (((b[..., g + o] | (b[..., g + o + 1] << 8)) << 16).to(torch.int32).view(torch.float32).double() for o in (0, 2))
        found.append((code, step, lo))
    return tuple(torch.stack([f[i] for f in found], 1) for i in range(3))


def tables(q_len, before, pages, rows, cols):
    """(page_table, place, positions, token_seq, q_start), as lists."""
    table, place, positions, seqs, q_start, at = [], [], [], [], [], 0
    for i, (q, b) in enumerate(zip(q_len, before)):
        own = pages[at:at + -(-(q + b) // PAGE)]
        at += len(own)
        table.append(own + [-1] * (cols - len(own)))
        q_start.append(len(place))
        for p in range(b, b + q):
            place.append(own[p // PAGE] * PAGE + p % PAGE)
            positions.append(p)
            seqs.append(i)
    pad = rows - len(place)
    return table, place + [-1] * pad, positions + [0] * pad, seqs + [-1] * pad, q_start


def attend(q, pages, table, q_len, before, scale, window=None, keep_first=0, sinks=None, gate=None, out_scale=1.0, head_scale=None, bias=None,
           cap=None):
    """q [rows, nqh, hd] float64, `pages` bytes -> (result [rows, nqh, hd], for every row and head the sum of p (|step code| + |lowest|)
    of its values [rows, nqh, hd], the most that a score's products sum up to [2, rows, nqh]: with codes 128 higher, and as they are);
    all on q's device."""
    dev, nqh, hd = q.device, q.shape[1], q.shape[2]
    code, step, lo = (x.to(dev) for x in read(pages, hd))
    wide = lambda x: x.repeat_interleave(GROUP, -1)
    low, sc = wide(lo), wide(step)
    val = low + sc * code
    kv = pages.shape[1]
    out, mag, smag = torch.zeros_like(q), torch.zeros_like(q), torch.zeros(2, *q.shape[:2], dtype=torch.float64, device=dev)
    r = 0
    for i, (n, b) in enumerate(zip(q_len, before)):
        if n == 0:
            continue
        L = n + b
        own = table[i][:-(-L // PAGE)].clamp(min=0).long().to(dev)   # (blocks given back are behind every window)
        j = torch.arange(L, device=dev)
        p = torch.arange(b, L, device=dev)[:, None]
        see = j <= p
        if window:
            see &= (p - j < window) | (j < keep_first)
        for h in range(nqh):
            get = lambda x, plane: x[own, plane, h // (nqh // kv)].reshape(-1, hd)[:L]
            f = scale * (float(head_scale[h]) if head_scale is not None else 1.0)
            used = see.any(0)
            k = torch.where(used[:, None], get(val, 0), 0.0)
            v, vm = (torch.where(used[:, None], x, 0.0) for x in (get(val, 1), (get(sc, 1) * get(code, 1)).abs() + get(low, 1).abs()))
            s = q[r:r + n, h] @ k.T * f
            for c, more in enumerate((256, 0)):
                km = torch.where(used[:, None], get(sc, 0) * (more + get(code, 0)) + get(low, 0).abs(), 0.0)
                smag[c, r:r + n, h] = ((q[r:r + n, h].abs() @ km.T) * abs(f)).masked_fill(~see, 0.0).max(1).values
            if cap:
                s = cap * torch.tanh(s / cap)
            if bias is not None:
                s = s - float(bias[0][h]) * torch.log1p(float(bias[1][h]) * (p - j).clamp(min=0))
            s = s.masked_fill(~see, -math.inf)
            if sinks is not None:
                s = torch.cat([s, torch.full((n, 1), float(sinks[h]), dtype=s.dtype, device=dev)], 1)
            w = torch.softmax(s, 1)[:, :L]
            f = out_scale * (torch.sigmoid(gate[r:r + n, h])[:, None] if gate is not None else 1.0)
            out[r:r + n, h], mag[r:r + n, h] = (w @ v) * f, (w @ vm) * abs(f)
        r += n
    return out, mag, smag
