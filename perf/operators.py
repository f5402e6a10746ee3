"""The 8-bit paged KV cache and the attention that reads it: what is measured.

A cache holds 8-bit codes (int8 or e4m3) in pages of `page` tokens, one FP32 scale
for each page, head and K or V: value = scale * code.  Its tensors:

    k, v             [layers, pages, kv_heads, page, d]   codes
    k_scale, v_scale [layers, pages, kv_heads]            FP32
    table            [slots, max_pages] int32             page of each block of positions, -1 unused
    length           [slots] int32                        tokens of each sequence
    ref              [pages] int32                        sequences that use a page, 0 = free

The operators (`op` of a case):

    write    rows of new keys and values quantised into the pages of their positions
    decode   attention of one query position per sequence over its pages
    prefill  causal attention of the last tokens of each sequence over its pages
    pages    free, fork and extend sequences (bookkeeping, and the copy of the partly
             filled page of each fork in all layers)
    compact  the pages in use moved to the front of the pool, the table following
"""
import math

import torch

own = False

QMAX = {"i8": 127.0, "e4m3": 448.0}
DTYPE = {"i8": torch.int8, "e4m3": torch.float8_e4m3fn}
I32 = torch.int32


def _pkg():
    """This repository's package (its folder's name is not an identifier)."""
    import importlib.util
    import sys
    from pathlib import Path

    if "bmle_b200" not in sys.modules:
        d = Path(__file__).resolve().parent.parent / "bare-metal-llm-engine_b200"
        if not d.is_dir():
            d = Path.cwd() / "bare-metal-llm-engine_b200"
        spec = importlib.util.spec_from_file_location("bmle_b200", d / "__init__.py", submodule_search_locations=[str(d)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["bmle_b200"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["bmle_b200"]


# ------------------------------------------------------------------------ cases


def listed():
    h8 = {"heads": 32, "kv_heads": 8, "d": 128}  # the heads of the repository's attention and layer benchmarks
    return [
        # one generated token of each of 64 sequences goes into its page: latency, mostly partly filled pages
        {"name": "write one token x64, i8", "op": "write", "kv": "i8", "batch": 64, "low": 100, "high": 4000, "new": 1, "page": 64, **h8},
        # prompts of uneven lengths enter the cache
        {"name": "write prompts 8 x ~1500, e4m3", "op": "write", "kv": "e4m3", "batch": 8, "low": 301, "high": 4096, "new": 0, "page": 32, **h8},
        # a few users of a small model with short contexts: latency; heads without sharing, small pages, odd lengths
        {"name": "decode 4 x 33-577, d64 e4m3", "op": "decode", "kv": "e4m3", "batch": 4, "low": 33, "high": 577, "page": 16, "heads": 16, "kv_heads": 16, "d": 64},
        # one user, a long context
        {"name": "decode 1 x 131072, e4m3", "op": "decode", "kv": "e4m3", "batch": 1, "low": 131072, "high": 131072, "page": 128, **h8},
        # a serving batch of uneven contexts
        {"name": "decode 48 x 200-16384, i8", "op": "decode", "kv": "i8", "batch": 48, "low": 200, "high": 16384, "page": 64, **h8},
        # a few draft tokens of each sequence are verified against its context
        {"name": "prefill verify 16 x 4 of ~4000", "op": "prefill", "kv": "i8", "batch": 16, "low": 1000, "high": 8000, "new": 4, "page": 64, **h8},
        # a chunk of a long prompt: the cached part is longer than the chunk
        {"name": "prefill chunk 512 of 8704, e4m3", "op": "prefill", "kv": "e4m3", "batch": 1, "low": 8704, "high": 8704, "new": 512, "page": 64, **h8},
        # whole prompts of uneven lengths
        {"name": "prefill prompts 4 x 700-5000", "op": "prefill", "kv": "i8", "batch": 4, "low": 700, "high": 5000, "new": 0, "page": 32, **h8},
        # one step of a scheduler: a few sequences end, fork and grow; a small model
        {"name": "pages 4 forks, 4 layers", "op": "pages", "kv": "i8", "batch": 16, "low": 50, "high": 700, "forks": 4, "new": 3, "layers": 4, "page": 16, "heads": 8, "kv_heads": 2, "d": 64},
        # many samples of some prompts: the partly filled pages of 32 layers are copied
        {"name": "pages 48 forks, 32 layers", "op": "pages", "kv": "e4m3", "batch": 12, "low": 100, "high": 1500, "forks": 48, "new": 40, "layers": 32, "page": 64, **h8},
        # a pool in which every other page is in use is compacted
        {"name": "compact 640 pages, 32 layers", "op": "compact", "kv": "i8", "batch": 20, "low": 500, "high": 1800, "layers": 32, "page": 32, **h8},
        # the same in the small pool of a small model: latency
        {"name": "compact 30 pages, 2 layers", "op": "compact", "kv": "e4m3", "batch": 6, "low": 20, "high": 150, "layers": 2, "page": 16, "heads": 8, "kv_heads": 2, "d": 64},
    ]


def _between(rng, a, b):
    """A whole number of [a, b], spread over its logarithm."""
    return max(a, min(b, int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))))


def draw(rng):
    heads, kv_heads, d = rng.choice([(32, 8, 128), (32, 8, 128), (16, 16, 64), (16, 2, 128), (8, 1, 128), (12, 4, 64), (20, 4, 128)])
    c = {"op": rng.choice(["write", "decode", "decode", "prefill", "prefill", "pages", "compact"]), "kv": rng.choice(["i8", "e4m3"]),
         "page": rng.choice([16, 32, 64, 128]), "heads": heads, "kv_heads": kv_heads, "d": d}
    c["batch"] = _between(rng, 1, 64)
    if c["op"] == "write":
        c["new"] = rng.choice([0, 1, 1, _between(rng, 2, 40)])
        c["high"] = _between(rng, 41, 20000 // c["batch"] if c["new"] == 0 and c["batch"] < 200 else 5000)
    elif c["op"] == "decode":
        c["high"] = _between(rng, 1, min(131072, 150000 // c["batch"]))
    elif c["op"] == "prefill":
        if rng.random() < 0.4:  # whole prompts
            c["new"], c["batch"] = 0, _between(rng, 1, 8)
            c["high"] = _between(rng, 2, 5500 // c["batch"])
        else:
            c["new"] = _between(rng, 1, 600)
            c["batch"] = max(1, min(c["batch"], 1200 // c["new"]))
            c["high"] = c["new"] + _between(rng, 1, 24000 // max(c["batch"], c["new"] // 32))
    else:
        c["layers"] = _between(rng, 1, 32)
        c["batch"] = _between(rng, 1, 24)
        c["high"] = _between(rng, 20, 1500)
        if c["op"] == "pages":
            c["forks"] = _between(rng, 1, 48)
            c["new"] = _between(rng, 1, 100)
    c["low"] = _between(rng, max(1, c.get("new", 1) if c["op"] in ("write", "prefill") else 1), c["high"])
    return c


def _lengths(c):
    """The sequences' lengths: from low to high, evenly over the logarithm."""
    n = c["batch"]
    if n == 1:
        return [c["high"]]
    return [max(1, int(round(c["low"] * (c["high"] / c["low"]) ** (i / (n - 1))))) for i in range(n)]


def _new(c):
    """New tokens of each sequence: `new`, or all of them where that is 0."""
    return [min(c["new"], n) if c["new"] else n for n in _lengths(c)]


def work(c):
    L, H, Hk, d, page = _lengths(c), c["heads"], c["kv_heads"], c["d"], c["page"]
    pages = sum(-(-n // page) for n in L)
    if c["op"] == "write":
        t = sum(_new(c))
        return {"bytes": t * Hk * d * 2 * 3, "flops": t * Hk * d * 2 * 2}
    if c["op"] == "decode":
        return {"bytes": sum(L) * Hk * d * 2 + pages * Hk * 8 + len(L) * H * d * 4, "flops": 4 * sum(L) * H * d}
    if c["op"] == "prefill":
        t = _new(c)
        pairs = sum(m * n - m * (m - 1) // 2 for m, n in zip(t, L))
        return {"bytes": sum(L) * Hk * d * 2 + pages * Hk * 8 + sum(t) * H * d * 4, "flops": 4 * pairs * H * d}
    one = 2 * c["layers"] * Hk * (page * d + 4)
    if c["op"] == "pages":
        copied = sum(L[i % len(L)] % page != 0 for i in range(c["forks"]))
        return {"bytes": 2 * copied * one + 4 * c["forks"] * max(-(-n // page) for n in L), "flops": 0}
    moved = _moved(c)
    return {"bytes": 2 * moved * one + 8 * pages + 16 * pages, "flops": 0}


def _moved(c):
    """Pages that a compaction of a pool with every other page in use moves."""
    pages = sum(-(-n // c["page"]) for n in _lengths(c))
    return (pages + 1) // 2


# ----------------------------------------------------------------------- inputs


def _quantised(x, kv):
    """Codes and scales of x [..., page, d]: one scale for each page and head."""
    s = x.abs().amax((-2, -1)) / QMAX[kv]
    q = x / s[..., None, None]
    return (q.round().to(torch.int8) if kv == "i8" else q.to(torch.float8_e4m3fn)), s


def _keys(shape, g, dev):
    """Keys and values as projections make them: a few channels are larger."""
    x = torch.randn(shape, generator=g, device=dev)
    return x * (1 + 3 * (torch.arange(shape[-1], device=dev) % 29 == 5))


def _cache(c, g, dev, layers, n_pages, slots, max_pages):
    shape = (layers, n_pages, c["kv_heads"], c["page"], c["d"])
    s = {}
    for n in ("k", "v"):
        s[n] = torch.empty(shape, dtype=DTYPE[c["kv"]], device=dev)
        s[n + "_scale"] = torch.empty(shape[:3], device=dev)
        for i in range(layers):
            s[n][i], s[n + "_scale"][i] = _quantised(_keys(shape[1:], g, dev) * (0.5 + torch.rand(shape[1:3], generator=g, device=dev))[..., None, None], c["kv"])
    s["table"] = torch.full((slots, max_pages), -1, dtype=I32, device=dev)
    s["length"] = torch.zeros(slots, dtype=I32, device=dev)
    s["ref"] = torch.zeros(n_pages, dtype=I32, device=dev)
    return s


def prepare(c, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    h = torch.Generator()
    h.manual_seed(seed)
    L = _lengths(c)
    order = torch.randperm(len(L), generator=h).tolist()
    L = [L[i] for i in order]
    page, Hk, d = c["page"], c["kv_heads"], c["d"]
    need = [-(-n // page) for n in L]
    used = sum(need)
    layers = c.get("layers", 1)
    forks = c.get("forks", 0)
    grown = -(-(c["high"] + c.get("new", 0)) // page) + 1 if c["op"] == "pages" else max(need)
    if c["op"] == "pages":  # parents, then the forks' slots; pages for the forks' own ends
        n_pages = used + forks * (2 + -(-c["new"] // page)) + 5
        s = _cache(c, g, dev, layers, n_pages, len(L) + forks, grown)
        ids = torch.randperm(n_pages, generator=h)[:used].to(I32)
    elif c["op"] == "compact":  # every other page is in use
        n_pages = 2 * used
        s = _cache(c, g, dev, layers, n_pages, len(L), grown)
        ids = (torch.randperm(used, generator=h) * 2 + 1).to(I32)
    else:
        n_pages = used + 3
        s = _cache(c, g, dev, layers, n_pages, len(L), grown)
        ids = torch.randperm(n_pages, generator=h)[:used].to(I32)
    table = torch.full(tuple(s["table"].shape), -1, dtype=I32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = ids[at:at + n]
        at += n
    s["table"].copy_(table)
    s["length"][: len(L)] = torch.tensor(L, dtype=I32)
    s["ref"][ids.long().to(dev)] = 1
    s["slots"] = torch.arange(len(L), dtype=I32, device=dev)
    if c["op"] in ("write", "prefill"):
        new = [_new(c)[i] for i in order]
        s["cu"] = torch.tensor([0] + new, device=dev).cumsum(0).to(I32)
        s["most"], s["tokens"] = max(new), sum(new)
        s["one"] = c["op"] == "write" and c["new"] == 1
    if c["op"] == "write":  # the keys and values of a fused projection's rows
        rows = torch.cat([torch.randn(s["tokens"], c["heads"] * d, generator=g, device=dev), _keys((s["tokens"], 2 * Hk, d), g, dev).flatten(1)], 1).half()
        s["k_rows"] = rows[:, c["heads"] * d: (c["heads"] + Hk) * d]
        s["v_rows"] = rows[:, (c["heads"] + Hk) * d:]
    if c["op"] == "decode":
        s["q"] = torch.randn(len(L), c["heads"], d, generator=g, device=dev).half()
    if c["op"] == "prefill":
        s["q"] = torch.randn(s["tokens"], c["heads"], d, generator=g, device=dev).half()
    if c["op"] == "pages":
        s["parents"] = (torch.arange(forks, device=dev) % len(L)).to(I32)
        s["children"] = (len(L) + torch.arange(forks, device=dev)).to(I32)
        s["n_new"] = torch.full((forks,), c["new"], dtype=I32, device=dev)
    if c["op"] == "compact":
        s["table0"], s["ref0"] = s["table"].clone(), s["ref"].clone()
    s["op"], s["kind"], s["scale"] = c["op"], c["kv"], d ** -0.5
    s["handle"] = None
    return s


# ------------------------------------------------------------------------- runs


def run(s):
    if own:
        return _run_own(s)
    return {"write": _write, "decode": _decode, "prefill": _prefill, "pages": _pages, "compact": _compact}[s["op"]](s)


def _run_own(s):
    ops = _pkg().ops
    if s["handle"] is None:  # the program's cache object: made once, of its tensors
        s["handle"] = ops.PagedKV(s["k"], s["v"], s["k_scale"], s["v_scale"], s["table"], s["length"], s["ref"])
    kv = s["handle"]
    if s["op"] == "write":
        ops.kv_pages_write(kv, 0, s["k_rows"], s["v_rows"], s["slots"], None if s["one"] else s["cu"])
        return [s["k"], s["v"], s["k_scale"], s["v_scale"]]
    if s["op"] == "decode":
        return ops.attention_paged_decode(kv, 0, s["q"], s["slots"], s["scale"])
    if s["op"] == "prefill":
        return ops.attention_paged_prefill(kv, 0, s["q"], s["slots"], s["cu"], s["scale"])
    if s["op"] == "pages":
        ops.kv_pages_free(kv, s["children"])
        a = ops.kv_pages_fork(kv, s["parents"], s["children"])
        b = ops.kv_pages_extend(kv, s["children"], s["n_new"])
        return [s["k"], s["v"], s["k_scale"], s["v_scale"], s["table"], s["length"], s["ref"], a, b]
    s["table"].copy_(s["table0"])
    s["ref"].copy_(s["ref0"])
    remap = ops.kv_pages_compact(kv)
    return [s["k"], s["v"], s["k_scale"], s["v_scale"], s["table"], s["ref"], remap]


def _store(s, n, rows):
    """Rows [tokens, kv_heads * d] of the last tokens of each sequence into the pages of `n`."""
    codes, scales = s[n][0], s[n + "_scale"][0]
    pages, Hk, page, d = codes.shape
    Q = QMAX[s["kind"]]
    cu, L = s["cu"].long(), s["length"].long()
    t = torch.arange(rows.shape[0], device=rows.device)
    b = torch.searchsorted(cu, t, right=True) - 1
    pos = L[b] - (cu[b + 1] - t)
    first = L[b] - (cu[b + 1] - cu[b])  # the position of the sequence's first new row
    at = s["table"].long()[s["slots"].long()[b], pos // page]
    x = rows.float().view(-1, Hk, d)
    most = torch.zeros_like(scales).scatter_reduce_(0, at[:, None].expand(-1, Hk), x.abs().amax(-1), "amax")
    hit = torch.zeros(pages, dtype=torch.bool, device=rows.device)
    hit[at] = True
    kept = torch.zeros(pages, dtype=torch.bool, device=rows.device)  # pages that hold earlier rows
    kept[at] = first - pos // page * page > 0
    old = torch.where(kept[:, None], scales, 0.0)
    new = torch.maximum(old, most * (1.0 / Q))
    grown = (hit & kept)[:, None] & (new > old)
    ratio = torch.where(grown, old / new, 1.0)
    inv = torch.where(new > 0, 1.0 / new, 0.0)
    again = codes.float() * ratio[..., None, None]
    y = x * inv[at][..., None]
    if s["kind"] == "i8":
        again, y = again.round(), y.round().clamp(-Q, Q)
    codes.copy_(torch.where(grown[..., None, None], again, codes.float()).to(codes.dtype))
    place = (at[:, None] * Hk + torch.arange(Hk, device=rows.device)) * page + (pos % page)[:, None]
    codes.view(torch.uint8).view(-1, d)[place.reshape(-1)] = y.to(codes.dtype).view(torch.uint8).view(-1, d)
    scales.copy_(torch.where(hit[:, None], new, scales))


def _write(s):
    _store(s, "k", s["k_rows"])
    _store(s, "v", s["v_rows"])
    return [s["k"], s["v"], s["k_scale"], s["v_scale"]]


def _values(s, n):
    """The values of the sequences' pages: [batch, kv_heads, positions, d], FP32."""
    at = s["table"][s["slots"].long()].long().clamp(min=0)
    x = s[n][0][at].float() * s[n + "_scale"][0][at][..., None, None]  # [batch, pages, kv_heads, page, d]
    return x.transpose(1, 2).flatten(2, 3)


def _attend(q, k, v, seen, scale):
    """q [batch, kv_heads, rows, d] over k / v [batch, kv_heads, keys, d]; seen [batch, 1, rows, keys]."""
    x = (q @ k.transpose(-1, -2)) * scale
    x = torch.where(seen, x, -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    return (p @ v) / p.sum(-1, keepdim=True)


def _decode(s):
    k, v = _values(s, "k"), _values(s, "v")
    B, H, d = s["q"].shape
    q = s["q"].float().view(B, k.shape[1], -1, d)
    seen = torch.arange(k.shape[2], device=q.device) < s["length"][:, None, None, None]
    return _attend(q, k, v, seen, s["scale"]).reshape(B, H, d).half()


def _prefill(s):
    k, v = _values(s, "k"), _values(s, "v")
    B, Hk, keys, d = k.shape
    T, H, _ = s["q"].shape
    G, M = H // Hk, s["most"]
    cu, L = s["cu"].long(), s["length"].long()
    i = torch.arange(M, device=k.device)
    n = cu[1:] - cu[:-1]
    rows = (cu[:-1, None] + i).clamp(max=T - 1)  # [batch, M]; past a sequence's own: not read again
    q = s["q"].float()[rows].view(B, M, Hk, G, d).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * M, d)
    last = (L - n)[:, None] + i  # the last key that a row sees
    seen = torch.arange(keys, device=k.device) <= last[:, :, None]
    seen = seen[:, None].expand(B, G, M, keys).reshape(B, 1, G * M, keys)
    o = _attend(q, k, v, seen, s["scale"]).view(B, Hk, G, M, d).permute(0, 3, 1, 2, 4).reshape(B, M, H, d)
    t = torch.arange(T, device=k.device)
    b = torch.searchsorted(cu, t, right=True) - 1
    return o[b, t - cu[b]].half()


def _free_pages(ref):
    """The free pages, lowest first, before those in use."""
    return torch.argsort((ref > 0).to(torch.int8), stable=True).to(I32)


def _pages(s):
    table, length, ref = s["table"], s["length"], s["ref"]
    page, width = s["k"].shape[3], table.shape[1]
    par, chi = s["parents"].long(), s["children"].long()
    j = torch.arange(width, device=table.device)
    # free
    mine = j < -(-length[chi] // page)[:, None]
    ref.scatter_add_(0, torch.where(mine, table[chi], 0).long().flatten(), -mine.to(I32).flatten())
    table[chi] = -1
    length[chi] = 0
    # fork: full pages are shared, the partly filled one is copied in all layers
    full, part = length[par] // page, length[par] % page != 0
    room = _free_pages(ref)
    new = room[(part.cumsum(0) - 1).clamp(min=0)]
    src = table[par].gather(1, full.long().clamp(max=width - 1)[:, None])[:, 0]  # the partly filled page
    rows = torch.where(j < full[:, None], table[par], -1)
    rows = torch.where((j == full[:, None]) & part[:, None], new[:, None], rows)
    shared = j < full[:, None]
    ref.scatter_add_(0, torch.where(shared, rows, 0).long().flatten(), shared.to(I32).flatten())
    ref.scatter_add_(0, torch.where(part, new, 0).long(), part.to(I32))
    table[chi], length[chi] = rows, length[par]
    to, of = torch.where(part, new, table[par][:, 0]).long(), torch.where(part, src, table[par][:, 0]).long()
    for x in (s["k"].view(torch.uint8), s["v"].view(torch.uint8), s["k_scale"], s["v_scale"]):
        x[:, to] = x[:, of]
    a = torch.zeros(1, dtype=I32, device=table.device)
    # extend
    before = -(-length[chi] // page)
    after = -(-(length[chi] + s["n_new"]) // page)
    room = _free_pages(ref)
    start = (after - before).cumsum(0) - (after - before)
    fresh = (j >= before[:, None]) & (j < after[:, None])
    ids = room[(start[:, None] + j - before[:, None]).clamp(0, room.numel() - 1)]
    table[chi] = torch.where(fresh, ids, table[chi])
    ref.scatter_add_(0, torch.where(fresh, ids, 0).long().flatten(), fresh.to(I32).flatten())
    length[chi] = length[chi] + s["n_new"]
    return [s["k"], s["v"], s["k_scale"], s["v_scale"], table, length, ref, a, torch.zeros_like(a)]


def _compact(s):
    s["table"].copy_(s["table0"])
    s["ref"].copy_(s["ref0"])
    table, ref = s["table"], s["ref"]
    n = ref.numel()
    j = torch.arange(n, device=ref.device)
    live = ref > 0
    count = live.sum()
    hole, mover = ~live & (j < count), live & (j >= count)
    # the k-th hole gets the k-th live page at or past `count`
    holes = torch.argsort((~hole).to(torch.int8), stable=True)
    k = (mover.cumsum(0) - 1).clamp(min=0)
    remap = torch.where(live, torch.where(mover, holes[k], j), -1)
    src = torch.argsort((~mover).to(torch.int8), stable=True)
    moved = j < mover.sum()
    half = n // 2  # at most half of the pages move
    of, to = torch.where(moved, src, holes)[:half], holes[:half]
    for x in (s["k"].view(torch.uint8), s["v"].view(torch.uint8), s["k_scale"], s["v_scale"]):
        x[:, to] = x[:, of]
    ref.copy_(torch.zeros_like(ref).scatter_add_(0, remap.clamp(min=0), torch.where(live, ref, 0)))
    table.copy_(torch.where(table >= 0, remap[table.long().clamp(min=0)].to(I32), table))
    return [s["k"], s["v"], s["k_scale"], s["v_scale"], table, ref, remap.to(I32)]


# ------------------------------------------------------------------------ exact


def exact(c, seed):
    """From the definitions, in 64 bits, one sequence (and head) at a time."""
    if c["op"] in ("pages", "compact"):
        return None  # whole numbers and copies
    s = prepare(c, seed)
    page, Hk, d = c["page"], c["kv_heads"], c["d"]
    G = c["heads"] // Hk
    table, L = s["table"].cpu().tolist(), s["length"].cpu().tolist()
    if c["op"] == "write":
        cu, Q = s["cu"].cpu().tolist(), QMAX[c["kv"]]
        got = []
        for n in ("k", "v"):
            code, scale = s[n].double(), s[n + "_scale"].double()
            rows = s[n + "_rows"].double().view(-1, Hk, d)
            for b in range(len(L)):
                m = cu[b + 1] - cu[b]
                p = L[b] - m
                while p < L[b]:  # page by page
                    end = min(L[b], (p // page + 1) * page)
                    x = rows[cu[b] + p - (L[b] - m): cu[b] + end - (L[b] - m)].transpose(0, 1)  # [kv_heads, rows, d]
                    w, off = table[b][p // page], p % page
                    before = scale[0, w].clone()
                    after = x.abs().amax((1, 2)) / Q
                    if off:
                        after = torch.maximum(before, after)
                        code[0, w] = _round64(code[0, w] * (before / after)[:, None, None], c["kv"])
                    code[0, w, :, off: off + end - p] = _round64(x / after[:, None, None], c["kv"])
                    scale[0, w] = after
                    p = end
            got.append((code if c["kv"] == "e4m3" else None, scale))
        return [got[0][0], got[1][0], got[0][1], got[1][1]]
    new = s["cu"].cpu().tolist() if c["op"] == "prefill" else list(range(len(L) + 1))
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for b, n in enumerate(L):
        ids = torch.tensor(table[b][: -(-n // page)], device=out.device)
        q = s["q"][new[b]: new[b + 1]].double()
        m = q.shape[0]
        for h in range(Hk):
            k, v = ((s[x][0, ids, h].double() * s[x + "_scale"][0, ids, h].double()[:, None, None]).reshape(-1, d)[:n] for x in ("k", "v"))
            for a in range(0, m, 2048):  # some rows at a time
                rows = q[a: a + 2048, h * G: (h + 1) * G]
                x = torch.einsum("rgd,kd->rgk", rows, k) * s["scale"]
                last = torch.arange(a, a + rows.shape[0], device=out.device) + (n - m)
                x.masked_fill_((torch.arange(n, device=out.device) > last[:, None])[:, None], -math.inf)
                out[new[b] + a: new[b] + a + rows.shape[0], h * G: (h + 1) * G] = torch.einsum("rgk,kd->rgd", torch.softmax(x, -1), v)
    return out


def _round64(x, kv):
    """The nearest code, ties to even."""
    if kv == "i8":
        return x.round().clamp(-127, 127)
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -40))).clamp(min=-6)
    step = torch.exp2(e - 3)
    return ((x / step).round() * step).clamp(-448, 448)
