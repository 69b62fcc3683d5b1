"""More operators of the paged cache: cases over their real range, their plain forms, and the calls a user makes of them.

A paged cache keeps each sequence in a row of a block table: whole groups of 64 tokens in pages of 4-bit codes that rows may share, the newest
``residual`` to ``residual + 63`` tokens (all of a short sequence) in 16 bits in the row's ring, token t at place t mod ring.

Page, per kv head: key codes [D][32 bytes], key words [D] of 32 bits, value codes [64 tokens][D/64][32 bytes], value words [64][D/64].  A row of 64
values (a channel's 64 tokens; a token's 64 channels) has a scale T and a zero level z in 0..127: code e stands for
A + T * (book[z][e] - z) / 32.  The row's word holds T (f16) in its lower half and in its upper half z, or A (f16) where the row does not
straddle zero (then z is 0 above zero and 127 below).  book[z] are the levels of the zero-anchored log compander (alpha 2) in 127ths.

Three kinds of call:

  shared   attention of the newest ``q_len`` tokens of each row, rows in groups that share the pages of a common prefix, which is read once for a group
  window   attention of the newest ``q_len`` tokens of each row over the ``window`` newest tokens and the ``sinks`` first ones
  read     tokens of rows back as ordinary keys and values
"""
import math
import random

import torch

own = False

PAGE = 64
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---- cases

_SHAPE = {"kv_heads": 8, "head_dim": 128, "residual": 128, "dtype": "bf16"}


def _shared(name, groups, each, prefix, own_most, **kw):
    return {"name": name, "kind": "shared", "groups": groups, "each": each, "most": prefix, "least": prefix, "own": own_most, "q_heads": 32, "q_len": 1,
            **_SHAPE, **kw}


def _window(name, batch, most, least, window, sinks, **kw):
    return {"name": name, "kind": "window", "batch": batch, "most": most, "least": least, "window": window, "sinks": sinks, "q_heads": 32, "q_len": 1,
            **_SHAPE, **kw}


def _read(name, batch, most, least, **kw):
    return {"name": name, "kind": "read", "batch": batch, "most": most, "least": least, "first": 0, **_SHAPE, **kw}


def listed():
    return [
        # four beams over one prompt: launches and latency are most of it
        _shared("shared_beams", 1, 4, 1000, 40),
        # the benchmark's batch of 64 sequences, their 4096 tokens a common instruction; own tokens as far as they got
        _shared("shared_batch", 1, 64, 4224, 700),
        # 32 questions about one long document
        _shared("shared_long", 1, 32, 131072, 300),
        # prompts of unlike lengths, four samples of each, 8 query heads per kv head, half precision
        _shared("shared_samples", 12, 4, 16001, 515, least=500, q_heads=64, dtype="fp16"),
        # four drafted tokens a row are verified at once behind a common prefix, head_dim 64
        _shared("shared_verify", 1, 16, 8192, 300, head_dim=64, q_len=4),
        # one user's long chat under a window of 1024 and four sinks
        _window("window_single", 1, 20000, 20000, 1024, 4),
        # a batch of unlike lengths, some shorter than the window
        _window("window_batch", 64, 16001, 1, 4096, 4),
        # drafted tokens under a short window that ends inside a page, half precision, head_dim 64; the sinks fill more than a page
        _window("window_verify", 16, 2050, 700, 500, 100, head_dim=64, q_len=4, dtype="fp16"),
        # two long documents under a window of a quarter of them
        _window("window_long", 2, 131072, 100003, 32768, 64),
        # a short prompt's cache, for the dense attention of the next chunk
        _read("read_single", 1, 1000, 1000),
        # a batch of prompts of unlike lengths
        _read("read_batch", 16, 4224, 1777),
        # two long documents' later halves on a small half-precision model
        _read("read_long", 2, 131072, 100003, first=65000, head_dim=64, dtype="fp16"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choices(["shared", "window", "read"], [3, 2, 1])[0]
    c = {"kind": kind, "kv_heads": rng.choice([1, 2, 4, 8, 8]), "head_dim": rng.choices([128, 64], [4, 1])[0],
         "residual": rng.choices([128, 64, 0], [5, 1, 1])[0], "dtype": rng.choices(["bf16", "fp16"], [3, 1])[0]}
    if kind != "read":
        c["q_heads"] = c["kv_heads"] * rng.choices([1, 2, 4, 8, 5], [1, 2, 5, 3, 1])[0]
        c["q_len"] = rng.choices([1, 2, 3, 5, 8], [8, 1, 1, 1, 1])[0]
    if kind == "shared":
        c["groups"] = _log_uniform(rng, 1, 16)
        c["each"] = _log_uniform(rng, 1, 64 // c["groups"])
        rows = c["groups"] * c["each"]
        # logits of all rows, and pages of all groups, within the largest listed case's
        cap = min(32 * 32 * 131072 // (rows * c["q_heads"] * c["q_len"]), 8 * 131072 // (c["groups"] * c["kv_heads"]))
        c["most"] = _log_uniform(rng, 100, max(200, min(cap, 131072)))
        c["least"] = rng.choice([0, c["most"] // 3, c["most"]])
        c["own"] = rng.choice([0, rng.randint(1, 1000)])
    elif kind == "window":
        c["batch"] = _log_uniform(rng, 1, 64)
        cap = 64 * 8 * 16001 // (c["batch"] * c["kv_heads"])
        c["most"] = _log_uniform(rng, 40, min(cap, 131072))
        c["least"] = rng.choice([0, 1, c["most"] // 2, c["most"]])
        c["window"] = _log_uniform(rng, 1, min(64 * 8 * 4096 // (c["batch"] * c["kv_heads"]), 32768))
        c["sinks"] = rng.choice([0, 1, 4, 4, 64, rng.randint(1, 300)])
    else:
        c["batch"] = _log_uniform(rng, 1, 64)
        c["most"] = _log_uniform(rng, 40, min(16 * 8 * 4224 // (c["batch"] * c["kv_heads"]), 131072))
        c["least"] = rng.choice([0, 1, c["most"] // 2, c["most"]])
        c["first"] = rng.choice([0, 0, rng.randint(0, c["most"])])
    return c


def _quantized(c, length):
    """Tokens of a row of this length that stand in pages."""
    return max(0, (length - c["residual"]) // PAGE) * PAGE


def _spread(most, least, n, salt):
    """n lengths: the longest first, the others spread evenly from the least to the most (the same ones for every seed)."""
    rng = random.Random(7919 * most + 13 * n + least + 31 * salt)
    return [most] + [rng.randint(least, most) for _ in range(n - 1)]


def _lengths(c):
    """Tokens that each row of the batch holds."""
    if c["kind"] != "shared":
        return _spread(c["most"], c["least"], c["batch"], 0)
    own_tokens = _spread(c["own"], 0, c["groups"] * c["each"], 1)
    return [p + own_tokens[g * c["each"] + i] for g, p in enumerate(_spread(c["most"], c["least"], c["groups"], 0)) for i in range(c["each"])]


def _common(c):
    """Pages that each group's rows share: those of the sequence that they were forked from, of ``most`` tokens or fewer."""
    return [_quantized(c, p) // PAGE for p in _spread(c["most"], c["least"], c["groups"], 0)]


def _counts(c):
    """Tokens that a read brings from each row: all from the first one on."""
    return [max(0, n - c["first"]) for n in _lengths(c)]


def _page_bytes(c):
    return 72 * c["head_dim"]


# ---- the codec in elementary operations

_tables = {}


def _books(device):
    """(levels [128, 16], code of the nearest level [128, 128]) as small whole numbers; ties go to the lower code."""
    if device not in _tables:
        z = torch.arange(128, dtype=torch.float64).view(128, 1)
        e = torch.arange(16, dtype=torch.float64).view(1, 16)
        zc = (15 * z / 127).round()
        up = (127 - z) * (3.0 ** ((e - zc) / (15 - zc).clamp_min(1)) - 1) / 2
        dn = z * (3.0 ** ((zc - e) / zc.clamp_min(1)) - 1) / 2
        book = torch.where(e >= zc, z + up.round(), z - dn.round())
        r = torch.arange(128, dtype=torch.float64).view(1, 128, 1)
        _tables[device] = (book.to(torch.uint8).to(device), (book.view(128, 1, 16) - r).abs().argmin(-1).to(torch.uint8).to(device))
    return _tables[device]


def _quantize(x):
    """[..., 64] -> (codes [..., 32] uint8, two to a byte, the earlier one lower; words [...] int32)."""
    nearest = _books(x.device)[1]
    x = x.float().clamp(-65504.0, 65504.0)
    lo, hi = x.amin(-1), x.amax(-1)
    zero = torch.zeros_like(lo)
    a = torch.where(lo > 0, lo, torch.where(hi < 0, hi, zero)).half()
    bits = a.view(torch.int16).int() & 0xFFFF
    off = (bits & 0x7FFF) >= 128
    a = torch.where(off, a.float(), zero)
    dn = torch.where(a > 0, zero, (a - lo).clamp_min(0.0))
    up = torch.where(a < 0, zero, (hi - a).clamp_min(0.0))
    extent = dn + up
    some = extent > 0
    z = torch.where(some, (127.0 * dn / torch.where(some, extent, zero + 1)).round(), zero)
    z = torch.where(a < 0, zero + 127, z)
    t = (extent * (32.0 / 127.0)).half()
    inverse = torch.where(t > 0, 32.0 / t.float(), zero)
    r = ((x - a.unsqueeze(-1)) * inverse.unsqueeze(-1) + z.unsqueeze(-1)).round().clamp(0.0, 127.0)
    codes = nearest.view(-1)[z.long().unsqueeze(-1) * 128 + r.long()]
    word = (t.view(torch.int16).int() & 0xFFFF) | (torch.where(off, bits, z.int()) << 16)
    return codes[..., 0::2] | (codes[..., 1::2] << 4), word


def _dequantize(codes, word):
    """Codes and words -> values, in 32 bits."""
    book = _books(codes.device)[0]
    t = (word & 0xFFFF).short().view(torch.float16).float()
    field = (word >> 16) & 0xFFFF
    off = (field & 0x7FFF) >= 128
    a = torch.where(off, field.short().view(torch.float16).float(), torch.zeros_like(t))
    z = torch.where(off, torch.where(a < 0, 127, 0), field)
    e = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2)
    u = book.view(-1)[z.unsqueeze(-1) * 16 + e.int()].float()
    return a.unsqueeze(-1) + t.unsqueeze(-1) * (u - z.unsqueeze(-1).float()) / 32.0


def _pack(k, v):
    """Whole pages' keys and values [N, KVH, 64, D] -> bytes [N, KVH, page bytes]."""
    n, h, _, d = k.shape
    kc, kw = _quantize(k.transpose(2, 3))
    vc, vw = _quantize(v.reshape(n, h, PAGE, d // 64, 64))
    return torch.cat([p.contiguous().view(torch.uint8).reshape(n, h, -1) for p in (kc, kw, vc, vw)], dim=-1)


def _unpack(pages, d):
    """Bytes [..., page bytes] -> keys and values [..., 64, D] in 32 bits."""
    lead = pages.shape[:-1]
    kc, kw, vc, vw = pages.split([32 * d, 4 * d, 32 * d, 4 * d], dim=-1)
    k = _dequantize(kc.reshape(*lead, d, 32), kw.contiguous().view(torch.int32))
    v = _dequantize(vc.reshape(*lead, PAGE, d // 64, 32), vw.contiguous().view(torch.int32).reshape(*lead, PAGE, d // 64))
    return k.transpose(-1, -2), v.flatten(-2)


# ---- inputs

def _cache(c, lengths, gen):
    """A layer's cache whose row i holds lengths[i] tokens, its pages in no order; rows of a group share their first pages."""
    dev = torch.device("cuda")
    dt, h, d, res, rows = _DTYPES[c["dtype"]], c["kv_heads"], c["head_dim"], c["residual"], len(lengths)
    counts = [_quantized(c, n) // PAGE for n in lengths]
    width = max(max(counts), 1) + 2
    table = torch.full((rows, width), -1, dtype=torch.int64)
    common, each = (_common(c), c["each"]) if c["kind"] == "shared" else ([0], rows)
    at = 0
    for g, n in enumerate(common):
        table[g * each:(g + 1) * each, :n] = torch.arange(at, at + n)
        at += n
    for i, n in enumerate(counts):
        m = common[i // each]
        table[i, m:n] = torch.arange(at, at + n - m)
        at += n - m
    pages = at + 3
    order = torch.randperm(pages, device=dev, generator=gen).int()
    table = table.to(dev)
    table = torch.where(table >= 0, order[table.clamp_min(0)], -1).int().contiguous()
    store = torch.zeros((1, pages, h, _page_bytes(c)), dtype=torch.uint8, device=dev)
    # keys ~ N(0,1) with log-normal channel scales, values ~ N(0,1)
    chan = torch.exp(torch.randn(d, device=dev, generator=gen)).to(dt)
    for first in range(0, at, 512):              # as many pages at a time as the intermediates fit easily
        n = min(512, at - first)
        k, v = (torch.randn((n, h, PAGE, d), device=dev, generator=gen, dtype=dt) for _ in range(2))
        store[0, order[first:first + n].long()] = _pack(k * chan, v)
    tail = torch.randn((1, rows, 2, h, res + 2 * PAGE, d), device=dev, generator=gen, dtype=dt)
    tail[:, :, 0] *= chan
    refs = torch.zeros(pages, dtype=torch.int32, device=dev)
    used = table.flatten().long()
    refs.index_add_(0, used.clamp_min(0), (used >= 0).int())
    return {"store": store, "tail": tail, "block_table": table, "lengths": torch.tensor(lengths, dtype=torch.int32, device=dev), "page_refs": refs,
            "status": torch.zeros(1, dtype=torch.int32, device=dev)}


def prepare(case, seed):
    c = case
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    lengths = _lengths(c)
    n = len(lengths)
    s = {"case": c, "longest": max(lengths)}
    t = _cache(c, lengths, gen)
    if c["kind"] == "shared":
        # groups come in any order, a group's rows one after the other
        order = list(range(c["groups"]))
        random.Random(seed).shuffle(order)
        rows = [g * c["each"] + i for g in order for i in range(c["each"])]
        s["common"] = [_common(c)[g] for g in order]
        s["groups"] = torch.arange(0, n + 1, c["each"], dtype=torch.int32, device=dev)
    else:
        rows = list(range(n))
        random.Random(seed).shuffle(rows)        # a batch need not come in the order of the table
    s["rows"] = torch.tensor(rows, dtype=torch.int32, device=dev)
    if c["kind"] == "read":
        counts = _counts(c)
        offsets = [0]
        for r in rows:
            offsets.append(offsets[-1] + counts[r])
        s["offsets"] = torch.tensor(offsets, dtype=torch.int32, device=dev)
        s["first"] = torch.full((n,), c["first"], dtype=torch.int32, device=dev)
        s["tokens"] = offsets[-1]
    else:
        s["query"] = torch.randn((n, c["q_len"], c["q_heads"], c["head_dim"]), device=dev, generator=gen, dtype=_DTYPES[c["dtype"]])
    s["tensors"] = t
    if own:
        # the handle that a program keeps around these tensors
        from muzero_b200 import MuZeroPagedCache
        s["cache"] = MuZeroPagedCache(**t, residual_length=c["residual"])
    return s


# ---- one pass

def _ring(s, rows, packed):
    """The rows' ring tokens in their order: keys and values [b, h, span, d], positions [b, span] (from ``packed`` on; those at or beyond the length are not there)."""
    t, res = s["tensors"], s["case"]["residual"]
    b, h, ring, d = rows.numel(), t["tail"].shape[3], t["tail"].shape[4], t["tail"].shape[5]
    span = res + PAGE - 1
    pos = packed.view(b, 1) + torch.arange(span, device=rows.device)
    tail = t["tail"][0][rows].float()
    at = (pos % ring).view(b, 1, span, 1).expand(b, h, span, d)
    return tail[:, 0].gather(2, at), tail[:, 1].gather(2, at), pos


def _paged(s, rows, pages):
    """Keys and values [b, h, tokens, d] and positions [b, tokens] of the pages [b, n] of rows."""
    c, t = s["case"], s["tensors"]
    b, n = pages.shape
    ids = t["block_table"][rows].gather(1, pages.clamp(0, t["block_table"].shape[1] - 1)).long().clamp_min(0)
    k, v = (x.transpose(1, 2).reshape(b, c["kv_heads"], n * PAGE, c["head_dim"]) for x in _unpack(t["store"][0][ids], c["head_dim"]))
    return k, v, (pages.unsqueeze(-1) * PAGE + torch.arange(PAGE, device=rows.device)).view(b, n * PAGE)


def _softmax_sums(logits):
    """exp(logits - their maximum) and its sum; rows without a finite logit give zeros and 1."""
    top = logits.amax(-1, keepdim=True)
    p = torch.exp(logits - torch.where(top > -math.inf, top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    return p, torch.where(total > 0, total, torch.ones_like(total))


def _plain_shared(s):
    c, t = s["case"], s["tensors"]
    h, d, lq, each = c["kv_heads"], c["head_dim"], c["q_len"], c["each"]
    g = c["q_heads"] // h
    out = torch.empty_like(s["query"])
    for i, common in enumerate(s["common"]):
        rows = s["rows"][i * each:(i + 1) * each].long()
        n = t["lengths"][rows].long()
        packed = (n - c["residual"]).clamp_min(0) // PAGE * PAGE
        # [b, h, lq * g, d], and the same with the group's rows next to one another
        q = s["query"][i * each:(i + 1) * each].float().view(each, lq, h, g, d).permute(0, 2, 1, 3, 4).reshape(each, h, lq * g, d) * d ** -0.5
        qpos = (n.view(each, 1) - lq + torch.arange(lq, device=n.device)).repeat_interleave(g, dim=1).view(each, 1, -1, 1)
        ks, vs, ps = _paged(s, rows[:1], torch.arange(common, device=n.device).view(1, -1))
        width = max(1, _quantized(c, s["longest"]) // PAGE - common)       # pages that a row may have of its own
        own_pages = common + torch.arange(min(width, -(-c["own"] // PAGE) + 1), device=n.device).expand(each, -1)
        kp, vp, pp = _paged(s, rows, own_pages)
        pp = torch.where(pp < packed.view(each, 1), pp, pp.new_full((), 1 << 40))
        kr, vr, pr = _ring(s, rows, packed)
        k, v, place = torch.cat([kp, kr], 2), torch.cat([vp, vr], 2), torch.cat([pp, pr], 1).view(each, 1, 1, -1)
        seen = (place <= qpos) & (place < n.view(each, 1, 1, 1))
        mine = torch.where(seen, q @ k.transpose(2, 3), torch.full((), -math.inf, device=n.device))
        m = common * PAGE
        common_logits = (q.transpose(0, 1).reshape(h, each * lq * g, d) @ ks[0].transpose(1, 2)).view(h, each, lq * g, m).transpose(0, 1)
        common_logits = torch.where(ps.view(1, 1, 1, -1) <= qpos, common_logits, torch.full((), -math.inf, device=n.device))
        p, total = _softmax_sums(torch.cat([common_logits, mine], -1))
        o = (p[..., :m].transpose(0, 1).reshape(h, each * lq * g, m) @ vs[0]).view(h, each, lq * g, d).transpose(0, 1)
        o = (o + p[..., m:] @ torch.where(seen.any(2).unsqueeze(-1), v, torch.zeros_like(v))) / total
        out[i * each:(i + 1) * each] = o.view(each, h, lq, g, d).permute(0, 2, 1, 3, 4).reshape(each, lq, h * g, d).to(out.dtype)
    return out


def _plain_window(s):
    c, t = s["case"], s["tensors"]
    h, d, lq, window, sinks = c["kv_heads"], c["head_dim"], c["q_len"], c["window"], c["sinks"]
    g, rows = c["q_heads"] // h, s["rows"].long()
    b, n = rows.numel(), t["lengths"][rows].long()
    packed = (n - c["residual"]).clamp_min(0) // PAGE * PAGE
    # the sinks' pages, and those from the first query's window on
    heads = min(-(-sinks // PAGE), _quantized(c, s["longest"]) // PAGE)
    first = ((n - lq + 1 - window).clamp_min(0) // PAGE).clamp_min(heads)
    width = min((window + lq - 2) // PAGE + 2, max(0, _quantized(c, s["longest"]) // PAGE - heads))
    pages = torch.cat([torch.arange(heads, device=n.device).expand(b, -1), first.view(b, 1) + torch.arange(width, device=n.device)], 1)
    k, v, place = _paged(s, rows, pages)
    place = torch.where(place < packed.view(b, 1), place, place.new_full((), 1 << 40))
    kr, vr, pr = _ring(s, rows, packed)
    k, v, place = torch.cat([k, kr], 2), torch.cat([v, vr], 2), torch.cat([place, pr], 1).view(b, 1, 1, -1)
    q = s["query"].float().view(b, lq, h, g, d).permute(0, 2, 1, 3, 4).reshape(b, h, lq * g, d)
    qpos = (n.view(b, 1) - lq + torch.arange(lq, device=n.device)).repeat_interleave(g, dim=1).view(b, 1, -1, 1)
    seen = (place <= qpos) & (place < n.view(b, 1, 1, 1)) & ((place > qpos - window) | (place < sinks))
    p, total = _softmax_sums(torch.where(seen, (q @ k.transpose(2, 3)) * d ** -0.5, torch.full((), -math.inf, device=n.device)))
    out = (p @ torch.where(seen.any(2).unsqueeze(-1), v, torch.zeros_like(v))) / total
    return out.view(b, h, lq, g, d).permute(0, 2, 1, 3, 4).reshape(b, lq, h * g, d).to(s["query"].dtype)


def _plain_read(s):
    c, t = s["case"], s["tensors"]
    rows = s["rows"].long()
    packed = (t["lengths"][rows].long() - c["residual"]).clamp_min(0) // PAGE * PAGE
    width = _quantized(c, s["longest"]) // PAGE
    kp, vp, _ = _paged(s, rows, torch.arange(width, device=rows.device).expand(rows.numel(), -1))
    kr, vr, _ = _ring(s, rows, packed)
    token = torch.arange(s["tokens"], device=rows.device)
    entry = torch.searchsorted(s["offsets"][1:].long(), token, right=True)
    pos = token - s["offsets"].long()[entry] + s["first"].long()[entry]
    at = torch.where(pos < packed[entry], pos, width * PAGE + pos - packed[entry])
    dt = t["tail"].dtype
    top = torch.finfo(dt).max                    # a code may stand for a little more than the type's largest number
    return tuple(torch.cat(x, 2)[entry, :, at].clamp(-top, top).to(dt) for x in ((kp, kr), (vp, vr)))


def run(state):
    s = state
    c = s["case"]
    if not own:
        return {"shared": _plain_shared, "window": _plain_window, "read": _plain_read}[c["kind"]](s)
    if c["kind"] == "shared":
        return s["cache"].attend(0, s["query"], rows=s["rows"], groups=s["groups"])
    if c["kind"] == "window":
        return s["cache"].attend(0, s["query"], rows=s["rows"], window=c["window"], sinks=c["sinks"])
    return s["cache"].read(0, rows=s["rows"], offsets=s["offsets"], first=s["first"], tokens=s["tokens"])


def _visible(c, n):
    """(query, token) pairs of a row of n tokens, its tokens in pages, and its ring's, that any of its queries sees."""
    w, k = c["window"], c["sinks"]
    qs = [q for q in range(n - c["q_len"], n) if q >= 0]
    pairs = sum(min(q + 1, w + min(k, max(0, q + 1 - w))) for q in qs)
    packed = _quantized(c, n)
    lo = max(0, n - c["q_len"] + 1 - w)          # the first query's window begins here
    in_pages = max(0, packed - max(lo, min(k, packed))) + min(k, packed)
    return pairs, in_pages, n - max(packed, min(lo, n)) + max(0, min(k, lo, n) - packed)


def work(case):
    c = case
    h, d = c["kv_heads"], c["head_dim"]
    token, coded = h * d * 4, h * _page_bytes(c) / PAGE      # a token's keys and values in 16 bits and in a page
    n = _lengths(c)
    if c["kind"] == "read":
        counts = _counts(c)
        paged = sum(max(0, _quantized(c, x) - c["first"]) for x in n)
        return {"bytes": paged * coded + (sum(counts) - paged) * token + sum(counts) * token, "flops": 0}
    queries = len(n) * c["q_len"] * c["q_heads"] * d * 4     # read, and the output written
    if c["kind"] == "shared":
        common = sum(_common(c)) * PAGE
        mine = sum(_quantized(c, x) for x in n) - common * c["each"]
        ring = sum(x - _quantized(c, x) for x in n)
        return {"bytes": (common + mine) * coded + ring * token + queries, "flops": 4 * sum(n) * c["q_len"] * c["q_heads"] * d}
    seen = [_visible(c, x) for x in n]
    return {"bytes": sum(x[1] for x in seen) * coded + sum(x[2] for x in seen) * token + queries, "flops": 4 * sum(x[0] for x in seen) * c["q_heads"] * d}


# ---- the same from the definitions, in 64 bits

def _exact_page(raw, d, z_book):
    """One kv head's pages [N, page bytes] -> keys [N*64, D], values [N*64, D] in 64 bits."""
    n = raw.shape[0]

    def side(codes, words):
        t = (words % 65536).to(torch.int32).to(torch.int16).view(torch.float16).double()
        f = words // 65536 % 65536
        signed = f.to(torch.int32).to(torch.int16).view(torch.float16).double()
        straddles = f % 32768 < 128
        z = torch.where(straddles, f, torch.where(signed < 0, torch.full_like(f, 127), torch.zeros_like(f)))
        anchor = torch.where(straddles, torch.zeros_like(t), signed)
        e = torch.empty((*codes.shape[:-1], 64), dtype=torch.int64, device=raw.device)
        e[..., 0::2], e[..., 1::2] = codes.long() % 16, codes.long() // 16
        u = z_book[z[..., None], e]
        return anchor[..., None] + t[..., None] * (u - z[..., None].double()) / 32

    def words(lo, hi):
        b = raw[:, lo:hi].long().view(n, -1, 4)
        return b[..., 0] + 256 * b[..., 1] + 65536 * b[..., 2] + 16777216 * b[..., 3]

    k = side(raw[:, :32 * d].reshape(n, d, 32), words(32 * d, 36 * d)).transpose(1, 2).reshape(n * PAGE, d)
    v = side(raw[:, 36 * d:68 * d].reshape(n, PAGE * (d // 64), 32), words(68 * d, 72 * d)).reshape(n * PAGE, d)
    return k, v


def _level_book(device):
    book = torch.zeros((128, 16), dtype=torch.float64)
    for z in range(128):
        zc = round(15 * z / 127)
        for e in range(16):
            if e >= zc:
                book[z, e] = z + round((127 - z) * math.expm1(math.log(3) * (e - zc) / max(15 - zc, 1)) / 2)
            else:
                book[z, e] = z - round(z * math.expm1(math.log(3) * (zc - e) / zc) / 2)
    return book.to(device)


def exact(case, seed):
    c = case
    global own
    was, own = own, False
    try:
        s = prepare(c, seed)
    finally:
        own = was
    t = s["tensors"]
    h, d, ring = c["kv_heads"], c["head_dim"], t["tail"].shape[4]
    book = _level_book(t["store"].device)
    lengths, rows = t["lengths"].tolist(), s["rows"].tolist()
    held = {}                                    # pages are looked at in pieces that neighbouring rows may share

    def piece(row, head, lo, hi):
        ids = t["block_table"][row, lo:hi]
        key = (head, lo, hi)
        if key not in held or not torch.equal(held[key][0], ids):
            held[key] = (ids, *_exact_page(t["store"][0, ids.long(), head], d, book))
        return held[key][1:]

    def row_tokens(row, head):
        n = lengths[row]
        np_ = _quantized(c, n) // PAGE
        places = [p % ring for p in range(np_ * PAGE, n)]
        m = _quantized(c, c["most"]) // PAGE if c["kind"] == "shared" else 0
        parts = [piece(row, head, lo, hi) for lo, hi in ((0, min(m, np_)), (min(m, np_), np_)) if hi > lo]
        parts.append(tuple(t["tail"][0, row, i, head, places].double() for i in range(2)))
        return tuple(torch.cat([p[i] for p in parts]) for i in range(2))

    if c["kind"] == "read":
        top = float(torch.finfo(t["tail"].dtype).max)
        out = tuple(torch.empty((s["tokens"], h, d), dtype=torch.float64, device=t["store"].device) for _ in range(2))
        for i, row in enumerate(rows):
            lo, hi = s["offsets"][i:i + 2].tolist()
            for head in range(h):
                for o, x in zip(out, row_tokens(row, head)):
                    o[lo:hi, head] = x[c["first"]:].clamp(-top, top)
            held.clear()
        return out
    q = s["query"].double()
    b, lq, hq, _ = q.shape
    g = hq // h
    out = torch.zeros_like(q)
    for head in range(h):
        for i, row in enumerate(rows):
            n = lengths[row]
            k, v = row_tokens(row, head)
            for j in range(lq):
                m = n - lq + j + 1               # tokens up to the query's own
                if m <= 0:
                    continue
                at = q[i, j, head * g:(head + 1) * g]
                kk, vv = k[:m], v[:m]
                if c["kind"] == "window" and m > c["window"]:
                    first = max(m - c["window"], min(c["sinks"], m))
                    keep = min(c["sinks"], m)
                    kk, vv = torch.cat([k[:keep], k[first:m]]), torch.cat([v[:keep], v[first:m]])
                out[i, j, head * g:(head + 1) * g] = torch.softmax(at @ kk.T / math.sqrt(d), dim=-1) @ vv
        held.clear()
    return out
