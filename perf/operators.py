"""The paged cache's operators: cases over their real range, their plain forms, and the calls a user makes of them.

A paged cache keeps each sequence in a row of a block table: whole groups of 64 tokens in pages of 4-bit codes that rows may share, the newest
``residual`` to ``residual + 63`` tokens (all of a short sequence) in 16 bits in the row's ring, token t at place t mod ring.

Page, per kv head: key codes [D][32 bytes], key words [D] of 32 bits, value codes [64 tokens][D/64][32 bytes], value words [64][D/64].  A row of 64
values (a channel's 64 tokens; a token's 64 channels) has a scale T and a zero level z in 0..127: code e stands for
A + T * (book[z][e] - z) / 32.  The row's word holds T (f16) in its lower half and in its upper half z, or A (f16) where the row does not
straddle zero (then z is 0 above zero and 127 below).  book[z] are the levels of the zero-anchored log compander (alpha 2) in 127ths.

Four kinds of call:

  attend   attention of the newest ``q_len`` tokens of each row over its pages and ring
  append   new tokens' keys and values into pages (quantized) and ring
  fork     rows become children of others: pages are shared and counted, live ring places are copied, for all layers
  retire   rows end: their pages are freed, and the pool is compacted (live pages move into the lowest places), for all layers
"""
import math
import random

import torch

own = False

PAGE = 64
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---- cases

def _attend(name, batch, most, least, **kw):
    c = {"name": name, "kind": "attend", "batch": batch, "most": most, "least": least, "kv_heads": 8, "q_heads": 32, "head_dim": 128,
         "q_len": 1, "residual": 128, "dtype": "bf16"}
    c.update(kw)
    return c


def _append(name, batch, most, least, **kw):
    c = {"name": name, "kind": "append", "batch": batch, "most": most, "least": least, "before": 0, "kv_heads": 8, "head_dim": 128,
         "residual": 128, "dtype": "bf16"}
    c.update(kw)
    return c


def _pages(name, kind, rows, most, least, touched, layers, **kw):
    c = {"name": name, "kind": kind, "rows": rows, "most": most, "least": least, "touched": touched, "layers": layers, "kv_heads": 8,
         "head_dim": 128, "residual": 128, "dtype": "bf16"}
    c.update(kw)
    return c


def listed():
    return [
        # a chat turn of one user: launches and host work are all there is
        _attend("attend_single", 1, 500, 500),
        # the benchmark's batch: 64 sequences of 4096 tokens and the residual window
        _attend("attend_batch", 64, 4224, 4224),
        # requests of unlike lengths in one batch, 8 query heads per kv head, half precision
        _attend("attend_ragged", 24, 16001, 1, q_heads=64, dtype="fp16"),
        # two long documents
        _attend("attend_long", 2, 131072, 100003),
        # four drafted tokens a row are verified at once, head_dim 64
        _attend("attend_verify", 16, 2050, 700, head_dim=64, q_len=4),
        # a decode step's write: one token a row; every 64th row or so fills a page
        _append("append_step", 64, 1, 1, before=4224),
        # prompts of unlike lengths into an empty cache
        _append("append_prompts", 16, 4096, 1777),
        # the next chunk of a long prompt on a small half-precision model
        _append("append_chunk", 3, 1111, 515, before=2050, head_dim=64, dtype="fp16"),
        # one prompt sampled four ways
        _pages("fork_one", "fork", 5, 1000, 1000, 4, 4),
        # a beam search of width 4 over 16 prompts: every beam's row is renewed
        _pages("fork_beams", "fork", 64, 4224, 2100, 48, 4),
        # a few sequences of a small pool end
        _pages("retire_few", "retire", 8, 1500, 300, 2, 2, head_dim=64),
        # a third of a full pool's sequences end
        _pages("retire_pool", "retire", 48, 4224, 1000, 16, 4),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choices(["attend", "append", "fork", "retire"], [5, 3, 1, 1])[0]
    c = {"kind": kind, "kv_heads": rng.choice([1, 2, 4, 8, 8]), "head_dim": rng.choices([128, 64], [4, 1])[0],
         "residual": rng.choices([128, 64, 0], [5, 1, 1])[0], "dtype": rng.choices(["bf16", "fp16"], [3, 1])[0]}
    if kind == "attend":
        c["q_heads"] = c["kv_heads"] * rng.choices([1, 2, 4, 8, 5], [1, 2, 5, 3, 1])[0]
        c["q_len"] = rng.choices([1, 2, 3, 5, 8], [8, 1, 1, 1, 1])[0]
        c["batch"] = _log_uniform(rng, 1, 64)
        cap = 64 * 8 * 4224 // (c["batch"] * c["kv_heads"])
        c["most"] = _log_uniform(rng, 40, max(80, min(cap, 131072)))
        c["least"] = rng.choice([0, 1, c["most"] // 2, c["most"]])
    elif kind == "append":
        c["batch"] = _log_uniform(rng, 1, 64)
        cap = 16 * 8 * 4096 // (c["batch"] * c["kv_heads"])
        c["most"] = rng.choice([1, _log_uniform(rng, 2, max(4, min(cap, 16384)))])
        c["least"] = rng.choice([0, 1, c["most"]])
        c["before"] = rng.choice([0, rng.randint(1, 5000)])
    else:
        c["rows"] = _log_uniform(rng, 4, 64)
        c["touched"] = rng.randint(1, max(1, c["rows"] - 2 if kind == "fork" else c["rows"] // 2))
        c["layers"] = rng.randint(1, 4)
        c["most"] = _log_uniform(rng, 300, min(16384, 48 * 4 * 8 * 4224 // (c["rows"] * c["layers"] * c["kv_heads"])))
        c["least"] = rng.choice([0, c["most"] // 3])
    return c


def _quantized(c, length):
    """Tokens of a row of this length that stand in pages."""
    return max(0, (length - c["residual"]) // PAGE) * PAGE


def _lengths(c, n):
    """A case's lengths: the longest first, the others spread evenly from the least to the most (the same ones for every seed)."""
    rng = random.Random(7919 * c["most"] + 13 * n + c["least"])
    return [c["most"]] + [rng.randint(c["least"], c["most"]) for _ in range(n - 1)]


def _before(c, n):
    """Tokens that a row holds before an append."""
    rng = random.Random(104729 * c["before"] + n)
    return [c["before"] + rng.randint(0, 63) if c["before"] else 0 for _ in range(n)]


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
    x = x.float()
    x = torch.where(x != x, torch.zeros_like(x), x).clamp(-65504.0, 65504.0)
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
    """Inverse of _quantize, in 32 bits."""
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

def _synthetic(c, tokens, gen, chan):
    """Keys ~ N(0,1) with log-normal channel scales and values ~ N(0,1), [tokens, KVH, D] in the model's type."""
    shape, dt = (tokens, c["kv_heads"], c["head_dim"]), _DTYPES[c["dtype"]]
    k = torch.randn(shape, device="cuda", generator=gen, dtype=dt).mul_(chan.to(dt))
    return k, torch.randn(shape, device="cuda", generator=gen, dtype=dt)


def _cache(c, rows, lengths, layers, spare_pages, gen, fill=True):
    """A cache whose row i holds lengths[i] tokens, its pages in no order; as a dict of tensors, and the rows' page lists on the host."""
    dev = torch.device("cuda")
    dt, h, d, res = _DTYPES[c["dtype"]], c["kv_heads"], c["head_dim"], c["residual"]
    counts = [_quantized(c, n) // PAGE for n in lengths]
    pages = sum(counts) + spare_pages
    order = torch.randperm(pages, device=dev, generator=gen).int()
    width = max(max(counts), 1) + 2
    table = torch.full((rows, width), -1, dtype=torch.int32)
    at = 0
    place = torch.zeros((rows, width), dtype=torch.int64)
    for i, n in enumerate(counts):
        place[i, :n] = torch.arange(at, at + n)
        table[i, :n] = 0
        at += n
    table = torch.where(table.to(dev) >= 0, order[place.to(dev)], table.to(dev)).contiguous()
    store = torch.zeros((layers, pages, h, _page_bytes(c)), dtype=torch.uint8, device=dev)
    chan = torch.exp(torch.randn(d, device=dev, generator=gen))
    for layer in range(layers if fill else 0):
        for first in range(0, at, 512):          # as many pages at a time as the inputs' intermediates fit easily
            n = min(512, at - first)
            k, v = (x.view(n, PAGE, h, d).transpose(1, 2) for x in _synthetic(c, n * PAGE, gen, chan))
            store[layer, order[first:first + n].long()] = _pack(k, v)
    ring = res + 2 * PAGE
    tail = torch.zeros((layers, rows, 2, h, ring, d), dtype=dt, device=dev)
    tail.normal_(generator=gen)
    tail[:, :, 0] *= chan.to(dt)
    refs = torch.zeros(pages, dtype=torch.int32, device=dev)
    refs[order[:at].long()] = 1
    return {"store": store, "tail": tail, "block_table": table, "lengths": torch.tensor(lengths + [0] * (rows - len(lengths)), dtype=torch.int32, device=dev),
            "page_refs": refs, "status": torch.zeros(1, dtype=torch.int32, device=dev)}, chan


def prepare(case, seed):
    c = case
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    rng = random.Random(seed)
    s = {"case": c}
    if c["kind"] == "attend":
        lengths = _lengths(c, c["batch"])
        t, _ = _cache(c, c["batch"], lengths, 1, 3, gen)
        rows = list(range(c["batch"]))
        rng.shuffle(rows)                        # a batch need not come in the order of the table
        s["rows"] = torch.tensor(rows, dtype=torch.int32, device=dev)
        s["query"] = torch.randn((c["batch"], c["q_len"], c["q_heads"], c["head_dim"]), device=dev, generator=gen, dtype=_DTYPES[c["dtype"]])
        s["longest"] = max(lengths)
    elif c["kind"] == "append":
        new = _lengths(c, c["batch"])
        before = _before(c, c["batch"])
        after = [a + b for a, b in zip(before, new)]
        t, chan = _cache(c, c["batch"], after, 1, 3, gen, fill=False)      # the pages stand in the table; this call writes them
        offsets = [0]
        for n in new:
            offsets.append(offsets[-1] + n)
        s["offsets"] = torch.tensor(offsets, dtype=torch.int32, device=dev)
        s["key"], s["value"] = _synthetic(c, offsets[-1], gen, chan)
        s["most"] = max(new)
        # what the plain form goes through: (row, page) to be quantized, (row, token) to stay in the ring
        filled = [(i, p) for i in range(len(new)) for p in range(_quantized(c, before[i]) // PAGE, _quantized(c, after[i]) // PAGE)]
        kept = [(i, p) for i in range(len(new)) for p in range(max(_quantized(c, after[i]), before[i]), after[i])]
        s["filled"] = torch.tensor(filled, dtype=torch.int64, device=dev).view(-1, 2)
        s["kept"] = torch.tensor(kept, dtype=torch.int64, device=dev).view(-1, 2)
        s["before"] = torch.tensor(before, dtype=torch.int64, device=dev)
    else:
        rows, touched = c["rows"], c["touched"]
        lengths = _lengths(c, rows)
        if c["kind"] == "fork":
            # parents come first; children take their places in rows that hold older sequences
            parents = [rng.randrange(rows - touched) for _ in range(touched)]
            s["source"] = torch.tensor(parents, dtype=torch.int32, device=dev)
            s["target"] = torch.tensor(list(range(rows - touched, rows)), dtype=torch.int32, device=dev)
        else:
            s["ended"] = torch.tensor(sorted(rng.sample(range(rows), touched)), dtype=torch.int32, device=dev)
        t, _ = _cache(c, rows, lengths, c["layers"], 3, gen)
        # a pass changes the tables: it starts from these
        s["start"] = {k: t[k].clone() for k in ("block_table", "lengths", "page_refs")}
    s["tensors"] = t
    if own:
        # the handle that a program keeps around these tensors
        from muzero_b200 import MuZeroPagedCache
        s["cache"] = MuZeroPagedCache(**t, residual_length=c["residual"])
    return s


# ---- one pass

def _plain_attend(s):
    c, t = s["case"], s["tensors"]
    b, lq, hq, d = s["query"].shape
    h, res = c["kv_heads"], c["residual"]
    rows = s["rows"].long()
    n = t["lengths"][rows].long()
    packed = (n - res).clamp_min(0) // PAGE * PAGE
    width = max(1, _quantized(c, s["longest"]) // PAGE)
    k, v = _unpack(t["store"][0][t["block_table"][rows, :width].long().clamp_min(0)], d)               # [b, page, h, 64, d]
    k, v = (x.transpose(1, 2).reshape(b, h, width * PAGE, d) for x in (k, v))
    ring = t["tail"].shape[4]
    span = min(ring, res + PAGE - 1) if res + PAGE > 1 else 1
    pos = packed.view(b, 1) + torch.arange(span, device=n.device)                               # the ring's tokens in their order
    tail = t["tail"][0][rows].float()
    at = (pos % ring).view(b, 1, span, 1).expand(b, h, span, d)
    k = torch.cat([k, tail[:, 0].gather(2, at)], dim=2)
    v = torch.cat([v, tail[:, 1].gather(2, at)], dim=2)
    place = torch.arange(width * PAGE, device=n.device).expand(b, -1)
    place = torch.cat([torch.where(place < packed.view(b, 1), place, place.new_full((), 1 << 40)), pos], dim=1)        # a token's position
    q = s["query"].float().view(b, lq, h, hq // h, d).permute(0, 2, 1, 3, 4).reshape(b, h, lq * (hq // h), d)
    qpos = (n.view(b, 1) - lq + torch.arange(lq, device=n.device)).repeat_interleave(hq // h, dim=1)
    logits = (q @ k.transpose(2, 3)) * d ** -0.5
    seen = (place.view(b, 1, 1, -1) <= qpos.view(b, 1, -1, 1)) & (place < n.view(b, 1)).view(b, 1, 1, -1)
    logits = torch.where(seen, logits, torch.full_like(logits, -math.inf))
    top = logits.amax(-1, keepdim=True)
    p = torch.exp(logits - torch.where(top > -math.inf, top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    out = (p @ torch.where(seen.any(2).unsqueeze(-1), v, torch.zeros_like(v))) / torch.where(total > 0, total, torch.ones_like(total))
    return out.view(b, h, lq, hq // h, d).permute(0, 2, 1, 3, 4).reshape(b, lq, hq, d).to(s["query"].dtype)


def _plain_append(s):
    t = s["tensors"]
    ring = t["tail"].shape[4]
    first = s["offsets"][:-1].long()
    row, page = s["filled"].unbind(1)
    if row.numel():
        pos = page.view(-1, 1) * PAGE + torch.arange(PAGE, device=page.device)                   # [N, 64] tokens of the pages to fill
        old = pos < s["before"][row].view(-1, 1)
        fresh = (first[row].view(-1, 1) + pos - s["before"][row].view(-1, 1)).clamp(0, s["key"].shape[0] - 1)
        blocks = []
        for side, x in ((0, s["key"]), (1, s["value"])):
            held = t["tail"][0, row.view(-1, 1), side, :, pos % ring]                            # [N, 64, h, d]
            blocks.append(torch.where(old.view(*old.shape, 1, 1), held, x[fresh]).transpose(1, 2))
        t["store"][0, t["block_table"][row, page].long()] = _pack(*blocks)
    row, pos = s["kept"].unbind(1)
    fresh = first[row] + pos - s["before"][row]
    t["tail"][0, row, 0, :, pos % ring] = s["key"][fresh]
    t["tail"][0, row, 1, :, pos % ring] = s["value"][fresh]
    return {"store": t["store"], "tail": t["tail"]}


def _count(refs, table, by):
    pages = table.flatten().long()
    refs.index_add_(0, pages.clamp_min(0), (pages >= 0).int() * by)


def _plain_fork(s):
    t, src, dst = s["tensors"], s["source"].long(), s["target"].long()
    res, ring = s["case"]["residual"], t["tail"].shape[4]
    _count(t["page_refs"], t["block_table"][dst], -1)
    _count(t["page_refs"], t["block_table"][src], 1)
    t["block_table"][dst] = t["block_table"][src]
    t["lengths"][dst] = t["lengths"][src]
    n = t["lengths"][dst].long().view(-1, 1)
    packed = (n - res).clamp_min(0) // PAGE * PAGE
    live = (torch.arange(ring, device=n.device) - packed) % ring < n - packed
    t["tail"][:, dst] = torch.where(live.view(1, -1, 1, 1, ring, 1), t["tail"][:, src], t["tail"][:, dst])
    return t


def _plain_retire(s):
    t, ended = s["tensors"], s["ended"].long()
    _count(t["page_refs"], t["block_table"][ended], -1)
    t["block_table"][ended] = -1
    t["lengths"][ended] = 0
    live = t["page_refs"] > 0
    place = torch.arange(live.numel(), device=live.device)
    below = place < live.sum()
    src, dst = (live & ~below).nonzero().view(-1), (~live & below).nonzero().view(-1)
    t["store"][:, dst] = t["store"][:, src]
    moved = place.int()
    moved[src] = dst.int()
    table = t["block_table"]
    t["block_table"].copy_(torch.where(table >= 0, moved[table.long().clamp_min(0)], table))
    t["page_refs"][dst] = t["page_refs"][src]
    t["page_refs"][src] = 0
    return t


def run(state):
    s = state
    kind = s["case"]["kind"]
    if kind in ("fork", "retire"):
        for k, v in s["start"].items():
            s["tensors"][k].copy_(v)
    if not own:
        out = {"attend": _plain_attend, "append": _plain_append, "fork": _plain_fork, "retire": _plain_retire}[kind](s)
    elif kind == "attend":
        out = s["cache"].attend(0, s["query"], rows=s["rows"])
    elif kind == "append":
        s["cache"].append(0, s["key"], s["value"], offsets=s["offsets"], max_new=s["most"])
        out = {"store": s["tensors"]["store"], "tail": s["tensors"]["tail"]}
    elif kind == "fork":
        s["cache"].fork(s["source"], s["target"])
        out = s["tensors"]
    else:
        s["cache"].free(s["ended"])
        s["cache"].compact()
        out = s["tensors"]
    if kind in ("fork", "retire"):
        # a fork leaves the pages as they are, a retirement the rings
        out = {k: out[k] for k in ("block_table", "lengths", "page_refs", "tail" if kind == "fork" else "store")}
    return out


def work(case):
    c = case
    h, d, layers = c["kv_heads"], c["head_dim"], c.get("layers", 1)
    token = h * d * 4                            # a token's 16-bit keys and values
    if c["kind"] == "attend":
        n = _lengths(c, c["batch"])
        packed = sum(_quantized(c, x) for x in n)
        rows = c["batch"] * c["q_len"] * c["q_heads"]
        return {"bytes": packed // PAGE * (h * _page_bytes(c) + 4) + (sum(n) - packed) * token + rows * d * 4,
                "flops": 4 * sum(n) * c["q_len"] * c["q_heads"] * d}
    if c["kind"] == "append":
        total = 0
        for x, old in zip(_lengths(c, c["batch"]), _before(c, c["batch"])):
            first, last = _quantized(c, old), _quantized(c, old + x)
            # new tokens are read, and written to the ring where they stay; pages take old tokens from the ring
            total += x * token + (old + x - max(last, old)) * token + max(0, min(last, old) - first) * token + (last - first) // PAGE * h * _page_bytes(c)
        return {"bytes": total, "flops": 0}
    n = _lengths(c, c["rows"])
    packed = [_quantized(c, x) for x in n]
    if c["kind"] == "fork":
        live = (sum(n) - sum(packed)) / len(n)   # of a parent, on average
        return {"bytes": c["touched"] * (2 * live * token * layers + sum(packed) / len(n) / PAGE * 16), "flops": 0}
    pages = sum(packed) // PAGE
    left = pages * (c["rows"] - c["touched"]) / c["rows"]
    moved = left * (1 - left / (pages + 3))      # the live pages of the upper places
    return {"bytes": 2 * moved * layers * h * _page_bytes(c) + pages * 8, "flops": 0}


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


def exact(case, seed):
    if case["kind"] != "attend":
        return None                              # bytes of pages (codes and words are whole numbers) and copies: equal or wrong
    c = case
    global own
    was, own = own, False
    try:
        s = prepare(c, seed)
    finally:
        own = was
    t, q = s["tensors"], s["query"].double()
    b, lq, hq, d = q.shape
    h, g, ring = c["kv_heads"], c["q_heads"] // c["kv_heads"], t["tail"].shape[4]
    book = torch.zeros((128, 16), dtype=torch.float64)
    for z in range(128):
        zc = round(15 * z / 127)
        for e in range(16):
            if e >= zc:
                book[z, e] = z + round((127 - z) * math.expm1(math.log(3) * (e - zc) / max(15 - zc, 1)) / 2)
            else:
                book[z, e] = z - round(z * math.expm1(math.log(3) * (zc - e) / zc) / 2)
    book = book.to(q.device)
    out = torch.zeros_like(q)
    lengths = t["lengths"].tolist()
    for i, row in enumerate(s["rows"].tolist()):
        n = lengths[row]
        if n == 0:
            continue
        np_ = _quantized(c, n) // PAGE
        ids = t["block_table"][row, :np_].long()
        places = [p % ring for p in range(np_ * PAGE, n)]
        for head in range(h):
            k, v = _exact_page(t["store"][0, ids, head], d, book) if np_ else (q.new_zeros((0, d)), q.new_zeros((0, d)))
            k = torch.cat([k, t["tail"][0, row, 0, head, places].double()])
            v = torch.cat([v, t["tail"][0, row, 1, head, places].double()])
            for j in range(lq):
                m = n - lq + j + 1               # tokens that this query sees
                if m > 0:
                    w = torch.softmax(q[i, j, head * g:(head + 1) * g] @ k[:m].T / math.sqrt(d), dim=-1)
                    out[i, j, head * g:(head + 1) * g] = w @ v[:m]
    return out
