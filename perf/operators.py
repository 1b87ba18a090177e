"""Performance cases of the paged cache's sharing: the operations on its pages
and the decode of sequences that share a prefix, through their public entry
points (``own`` true) or in their plain form (elementary torch operations).

A case is a dict of plain values.  ``listed()`` names twelve; ``draw(rng)``
gives others of the same ranges.  ``kind`` says which operator a case runs:

``copy``     ``copy_pages``: pages of the pool copied to others, with their 8-bit
             copy and its scales where the cache has one
``fork``     ``fork_sequences``: empty batch rows become forks of others; whole
             pages are shared, a partly filled last page is copied
``free``     ``free_sequences``: batch rows are emptied, and the pool's pages
             that no row holds any more are listed
``compact``  ``compact_pages``: the pages in use move to the front of the pool
``shared``   ``paged_decode_attention_shared``: decode of groups of sequences,
             the keys that a group shares read once for all of its queries

Lengths are spread over [lo, hi] evenly in their logarithm; lo = hi is a
uniform batch.  Values are N(0, 1), pages are scattered over the pool by a
random permutation.
"""

import math

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    gqa = {"heads": 32, "kv_heads": 8, "dim": 128}
    pages = {"kv_heads": 8, "dim": 128}
    return [
        # The last pages of a few beams, as an engine that keeps its tables on the host copies them: latency.
        {"name": "copy_small", "kind": "copy", "dtype": "fp16", "pairs": 16, "pool": 256, "page": 16,
         "mirror": False, **pages},
        # A pool rearranged by its engine: a quarter of the pages, with their 8-bit copy.
        {"name": "copy_large", "kind": "copy", "dtype": "bf16", "pairs": 8192, "pool": 32768, "page": 16,
         "mirror": True, **pages},
        # One prompt, four samples.
        {"name": "fork_small", "kind": "fork", "dtype": "fp16", "parents": 1, "each": 4, "lo": 700, "hi": 700,
         "page": 16, "mirror": False, **pages},
        # Sixteen prompts, fifteen samples of each, on a cache with an 8-bit copy and pages of 64 tokens.
        {"name": "fork_large", "kind": "fork", "dtype": "bf16", "parents": 16, "each": 15, "lo": 200, "hi": 8000,
         "page": 64, "mirror": True, **pages},
        # Four requests of a small batch end.
        {"name": "free_small", "kind": "free", "batch": 32, "rows": 4, "lo": 64, "hi": 4096, "page": 16},
        # A large batch on pages of one token, an eighth of it ends.
        {"name": "free_large", "kind": "free", "batch": 512, "rows": 64, "lo": 200, "hi": 8000, "page": 1},
        # A small pool packed after a few requests ended.
        {"name": "compact_small", "kind": "compact", "dtype": "fp16", "batch": 8, "lo": 64, "hi": 2048, "spare": 0.5,
         "prefix": 0, "page": 16, "mirror": False, **pages},
        # A pool of gigabytes packed before its end is given back, prompts shared among its sequences.
        {"name": "compact_large", "kind": "compact", "dtype": "bf16", "batch": 128, "lo": 500, "hi": 8000,
         "spare": 0.5, "prefix": 1024, "page": 16, "mirror": False, **pages},
        # Four samples of one short prompt, the next token of each: latency and launches.
        {"name": "shared_small", "kind": "shared", "dtype": "fp16", "kv": "same", "groups": 1, "each": 4,
         "plo": 512, "phi": 512, "lo": 4, "hi": 64, "tokens": 1, "page": 16, **gqa},
        # The benchmark's batch and context as a system prompt, chats of different lengths behind it.
        {"name": "shared_batch", "kind": "shared", "dtype": "fp16", "kv": "same", "groups": 1, "each": 32,
         "plo": 4096, "phi": 4096, "lo": 64, "hi": 1024, "tokens": 1, "page": 16, **gqa},
        # A long document that many requests ask about, on an fp8 cache.
        {"name": "shared_large", "kind": "shared", "dtype": "bf16", "kv": "fp8", "groups": 1, "each": 128,
         "plo": 32768, "phi": 32768, "lo": 100, "hi": 2000, "tokens": 1, "page": 16, **gqa},
        # Eight prompts, six samples of each, four drafted tokens verified per sample.
        {"name": "shared_verify", "kind": "shared", "dtype": "bf16", "kv": "same", "groups": 8, "each": 6,
         "plo": 1000, "phi": 8000, "lo": 40, "hi": 900, "tokens": 4, "page": 16, **gqa},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["copy", "fork", "free", "compact", "shared", "shared", "shared", "shared"])
    heads, kv_heads = rng.choice([(32, 8), (32, 8), (16, 8), (8, 8), (16, 2), (64, 8), (32, 1), (28, 4)])
    case = {"kind": kind, "dtype": rng.choice(["fp16", "bf16"]), "kv_heads": kv_heads,
            "dim": rng.choice([128, 128, 64]), "page": rng.choice([16, 16, 32, 64, 1])}
    if kind == "free":
        case = {"kind": kind, "batch": _log(rng, 2, 512), "page": case["page"], "hi": _log(rng, 16, 8000)}
        case["lo"] = max(1, int(case["hi"] * rng.choice([1.0, rng.uniform(0.03, 1.0)])))
        case["rows"] = max(1, int(case["batch"] * rng.uniform(0.02, 0.7)))
        return case
    if kind == "copy":
        case.update(pairs=_log(rng, 1, 8192), mirror=rng.random() < 0.4, dtype=rng.choice(["fp16", "bf16", "fp32"]))
        case["mirror"] = case["mirror"] and case["dtype"] != "fp32"
        case["pool"] = 2 * case["pairs"] + _log(rng, 1, 4096)
        while work(case)["bytes"] > 1.5e9:
            case["pairs"] = case["pairs"] // 2 + 1
        return case
    if kind == "fork":
        case.update(parents=_log(rng, 1, 32), each=_log(rng, 1, 32), hi=_log(rng, 2, 8000),
                    mirror=rng.random() < 0.4)
        case["lo"] = max(1, int(case["hi"] * rng.choice([1.0, rng.uniform(0.03, 1.0)])))
        while case["parents"] * case["each"] > 240:
            case["each"] = case["each"] // 2 + 1
            case["parents"] = case["parents"] * 2 // 3 + 1
        return case
    if kind == "compact":
        case.update(batch=_log(rng, 1, 128), hi=_log(rng, 16, 8000), spare=round(rng.uniform(0.05, 2.0), 2),
                    prefix=rng.choice([0, 0, _log(rng, 16, 2048)]), mirror=rng.random() < 0.3)
        case["lo"] = max(1, int(case["hi"] * rng.choice([1.0, rng.uniform(0.03, 1.0)])))
        while sum(_lens(case["batch"], case["lo"], case["hi"])) * case["kv_heads"] * case["dim"] > 3.2e8 or \
                work(case)["bytes"] > 1.5e9:
            case["hi"] = case["hi"] // 2 + 8
            case["lo"] = case["lo"] // 2 + 1
        return case
    case.update(heads=heads, kv=rng.choice(["same", "same", "int8", "fp8"]), tokens=rng.choice([1, 1, 1, 1, 2, 4]))
    case["groups"] = rng.choice([1, 1, _log(rng, 1, 16)])
    case["each"] = _log(rng, 1, 128 // case["groups"] + 1)
    case["phi"] = _log(rng, 64, 32768)
    case["plo"] = max(1, int(case["phi"] * rng.choice([1.0, rng.uniform(0.03, 1.0)])))
    case["hi"] = _log(rng, 2, 2000)
    case["lo"] = max(1, int(case["hi"] * rng.choice([1.0, rng.uniform(0.03, 1.0)])))
    while work(case)["flops"] > 8e10 or work(case)["bytes"] > 6e8:
        case["phi"], case["plo"] = case["phi"] // 2 + 1, case["plo"] // 2 + 1
        case["hi"], case["lo"] = case["hi"] // 2 + 1, case["lo"] // 2 + 1
    return case


def _lens(n, lo, hi):
    """``n`` lengths over [lo, hi], evenly spread in their logarithm."""
    return [int(round(lo * (hi / lo) ** ((0.5 + 0.6180339887 * i) % 1.0))) for i in range(n)]


def _prefixes(case):
    """Tokens that each group shares: whole pages."""
    return [n // case["page"] * case["page"] for n in _lens(case["groups"], case["plo"], case["phi"])]


def _tails(case):
    """Tokens behind the prefix of each sequence of a ``shared`` case, its new ones among them."""
    return [n + case["tokens"] for n in _lens(case["groups"] * case["each"], case["lo"], case["hi"])]


def work(case):
    kind, page = case["kind"], case["page"]
    if kind == "free":
        lens = _lens(case["batch"], case["lo"], case["hi"])
        pool = _pool_pages(sum(-(-n // page) for n in lens), 0.25)
        kept = sum(-(-n // page) for n in lens[case["rows"]:])
        return {"bytes": 4 * (kept + 2 * case["batch"] + case["rows"] + pool), "flops": 0}
    row = case["kv_heads"] * case["dim"]
    elem = 4 if case["dtype"] == "fp32" else 2
    if kind != "shared":
        # one page of K and V, and of their 8-bit copy with its scales
        block = 2 * page * row * elem + (2 * page * row + 8 * case["kv_heads"] if case["mirror"] else 0)
    if kind == "copy":
        return {"bytes": case["pairs"] * (2 * block + 8), "flops": 0}
    if kind == "fork":
        total = 0
        for n in _lens(case["parents"], case["lo"], case["hi"]):
            used = -(-n // page)
            total += 4 * used + case["each"] * (4 * used + 16)
            if n % page:
                total += block + case["each"] * block
        return {"bytes": total, "flops": 0}
    if kind == "compact":
        used, entries = _compact_pages_of(case)
        pool = _pool_pages(used, case["spare"])
        moved = used * (pool - used) / pool  # of pages scattered at random, those behind the first `used`
        return {"bytes": int(2 * moved * block + 8 * entries + 4 * pool), "flops": 0}
    prefixes, tails = _prefixes(case), _tails(case)
    kv = "same" if case["kv"] == "same" else "8bit"
    rows = len(tails) * case["tokens"]
    keys = sum(prefixes) + sum(tails)
    held = sum(p // page for p in prefixes) + sum(-(-n // page) for n in tails)
    pairs = sum(case["tokens"] * (prefixes[i // case["each"]] + n) for i, n in enumerate(tails))
    return {"bytes": 2 * rows * case["heads"] * case["dim"] * 2 + 2 * keys * row * (2 if kv == "same" else 1)
            + (8 * case["kv_heads"] * held if kv != "same" else 0) + 4 * held,
            "flops": 4 * case["heads"] * case["dim"] * pairs}


def _pool_pages(used, spare):
    return used + max(3, int(used * spare))


def _compact_pages_of(case):
    """Pages in use and table entries of a ``compact`` case."""
    page, shared = case["page"], case["prefix"] // case["page"]
    per = [-(-n // page) + shared for n in _lens(case["batch"], case["lo"], case["hi"])]
    groups = -(-case["batch"] // 4)
    return sum(per) - shared * (case["batch"] - groups), sum(per)


# ---------------------------------------------------------------------------
# What a user's program has in hand
# ---------------------------------------------------------------------------
def _tables(g, shared, own_pages, leaders, pool):
    """Table [batch, widest] of distinct random pages: row b has ``shared[b]`` pages of row ``leaders[b]``, then
    ``own_pages[b]`` of its own (a leader's shared ones are its own)."""
    widest = max(s + o for s, o in zip(shared, own_pages))
    perm = torch.randperm(pool, generator=g, device=g.device).to(torch.int32)
    table = torch.zeros(len(shared), max(1, widest), dtype=torch.int32, device=g.device)
    at = 0
    for b, (s, o) in enumerate(zip(shared, own_pages)):
        if leaders[b] == b:
            table[b, :s] = perm[at:at + s]
            at += s
        else:
            table[b, :s] = table[leaders[b], :s]
        table[b, s:s + o] = perm[at:at + o]
        at += o
    return table, at


def _mirror(k, v):
    """An int8 copy of float pages and its scales [pages, kv_heads] (absmax over a page's slots and dims)."""
    out = {}
    for name, x in (("k", k), ("v", v)):
        out["q" + name], out["s" + name] = _codes(x, "int8")
    return out


def _codes(pages, mode):
    top = 127.0 if mode == "int8" else 448.0
    codes = torch.empty(pages.shape, dtype=torch.int8 if mode == "int8" else torch.float8_e4m3fn, device=pages.device)
    scale = torch.empty(pages.shape[0], pages.shape[2], device=pages.device)
    for lo in range(0, pages.shape[0], 8192):
        x = pages[lo:lo + 8192].float()
        s = (x.abs().amax(dim=(1, 3)) / top).clamp_min(1e-8)
        y = x / s[:, None, :, None]
        codes[lo:lo + 8192] = (y.round() if mode == "int8" else y).clamp(-top, top).to(codes.dtype)
        scale[lo:lo + 8192] = s
    return codes, scale


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    kind, page = case["kind"], case["page"]

    def randn(*shape, dtype):
        return torch.randn(shape, generator=g, device=g.device, dtype=dtype)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device=g.device)

    state = {"kind": kind, "page": page}
    if kind == "free":
        lens = _lens(case["batch"], case["lo"], case["hi"])
        per = [-(-n // page) for n in lens]
        pool = _pool_pages(sum(per), 0.25)
        table, _ = _tables(g, [0] * len(lens), per, list(range(len(lens))), pool)
        # The pool's values play no part; its shape says how many pages there are.
        pages = torch.zeros(pool, page, 1, 32, dtype=torch.float16, device=g.device)
        state.update(k=pages, v=pages, table=table, lens=ints(lens),
                     rows=torch.arange(case["rows"], dtype=torch.int32, device=g.device))
        state["before"] = state["lens"].clone()
        return state
    dtype = _DTYPES[case["dtype"]]
    kv_heads, dim = case["kv_heads"], case["dim"]
    if kind == "copy":
        pool, n = case["pool"], case["pairs"]
        perm = torch.randperm(pool, generator=g, device=g.device).to(torch.int32)
        state.update(src=perm[:n].contiguous(), dst=perm[n:2 * n].contiguous(),
                     table=torch.zeros(1, 1, dtype=torch.int32, device=g.device), lens=ints([0]))
    elif kind == "fork":
        lens = _lens(case["parents"], case["lo"], case["hi"])
        per = [-(-n // page) for n in lens]
        children = case["parents"] * case["each"]
        pool = sum(per) + children + 3
        table, used = _tables(g, [0] * len(per), per, list(range(len(per))), pool)
        width = max(per) + 4  # room to grow
        wide = torch.zeros(case["parents"] + children, width, dtype=torch.int32, device=g.device)
        wide[:case["parents"], :table.shape[1]] = table
        free = torch.ones(pool, dtype=torch.bool, device=g.device)
        for b, n in enumerate(per):
            free[table[b, :n].long()] = False
        ids = free.nonzero()[:, 0].to(torch.int32)
        state.update(table=wide, lens=ints(lens + [0] * children),
                     parents=ints([i // case["each"] for i in range(children)]),
                     children=ints([case["parents"] + i for i in range(children)]), pages=ids[:children].contiguous())
        state["before"] = state["lens"].clone()
    elif kind == "compact":
        lens = _lens(case["batch"], case["lo"], case["hi"])
        shared = case["prefix"] // page
        per = [-(-n // page) for n in lens]
        used, _ = _compact_pages_of(case)
        pool = _pool_pages(used, case["spare"])
        leaders = [b - b % 4 for b in range(len(lens))]
        table, _ = _tables(g, [shared] * len(lens), per, leaders, pool)
        state.update(table=table, lens=ints([shared * page + n for n in lens]), before=table.clone())
    else:
        prefixes, tails = _prefixes(case), _tails(case)
        each = case["each"]
        shared = [prefixes[b // each] // page for b in range(len(tails))]
        per = [-(-n // page) for n in tails]
        pool = sum(p // page for p in prefixes) + sum(per) + 3
        table, _ = _tables(g, shared, per, [b - b % each for b in range(len(tails))], pool)
        shape = (len(tails), case["heads"], dim) if case["tokens"] == 1 else (len(tails), case["tokens"],
                                                                             case["heads"], dim)
        state.update(table=table, lens=ints([prefixes[b // each] + n for b, n in enumerate(tails)]),
                     cu_groups=ints([each * i for i in range(case["groups"] + 1)]), prefix_lens=ints(prefixes),
                     prefixes=prefixes, each=each, tails=tails, q=randn(*shape, dtype=dtype))
    state["k"] = randn(pool, page, kv_heads, dim, dtype=dtype)
    state["v"] = randn(pool, page, kv_heads, dim, dtype=dtype)
    if kind == "shared":
        state["scales"] = None
        if case["kv"] != "same":
            (state["k"], sk), (state["v"], sv) = _codes(state["k"], case["kv"]), _codes(state["v"], case["kv"])
            state["scales"] = {"k": sk, "v": sv}
    elif case["mirror"]:
        state.update(_mirror(state["k"], state["v"]))
    return state


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
_POOLS = ("k", "v", "qk", "qv", "sk", "sv")


def run(state):
    kind = state["kind"]
    # The engine's scheduler owns the lengths and tables: as they were before the operation.
    if kind in ("fork", "free"):
        state["lens"].copy_(state["before"])
    elif kind == "compact":
        state["table"].copy_(state["before"])
    return (_run_own if own else _run_plain)(state)


def _outputs(state, **more):
    return {**{name: state[name] for name in _POOLS if name in state}, **more}


def _run_own(state):
    import flashattntile_amd as fat

    kind = state["kind"]
    cache = fat.PagedKVCache(state["k"], state["v"], state["table"], state["lens"], state["page"])
    if kind == "shared":
        return fat.paged_decode_attention_shared(state["q"], cache, state["cu_groups"], state["prefix_lens"],
                                                 scales=state["scales"])
    if kind == "free":
        pages, count = fat.free_sequences(cache, state["rows"])
        return {"seq_lens": state["lens"], "pages": pages, "count": count}
    quantized = None
    if "qk" in state:
        quantized = (fat.PagedKVCache(state["qk"], state["qv"], state["table"], state["lens"], state["page"]),
                     {"k": state["sk"], "v": state["sv"]})
    if kind == "copy":
        fat.copy_pages(cache, state["src"], state["dst"], quantized=quantized)
        return _outputs(state)
    if kind == "fork":
        fat.fork_sequences(cache, state["parents"], state["children"], state["pages"], quantized=quantized)
        return _outputs(state, page_table=state["table"], seq_lens=state["lens"])
    remap, count = fat.compact_pages(cache, quantized=quantized)
    return _outputs(state, page_table=state["table"], remap=remap, count=count)


def _used(table, lens, page, pool):
    """Columns [batch, widest] that the lengths use, and whether a page is in one of them."""
    columns = torch.arange(table.shape[1], device=table.device) < ((lens + page - 1) // page)[:, None]
    used = torch.zeros(pool, dtype=torch.bool, device=table.device)
    used[table[columns].long()] = True
    return columns, used


def _run_plain(state):
    kind = state["kind"]
    if kind == "shared":
        return _attend_plain(state)
    table, lens, page, pool = state["table"], state["lens"], state["page"], state["k"].shape[0]
    if kind == "copy":
        src, dst = state["src"].long(), state["dst"].long()
        for name in _POOLS:
            if name in state:
                state[name][dst] = state[name][src]
        return _outputs(state)
    if kind == "fork":
        parents, children = state["parents"].long(), state["children"].long()
        n = lens[parents]
        full, used = n // page, (n + page - 1) // page
        rows = table[parents]
        column = torch.arange(table.shape[1], device=table.device)
        partial = (n % page != 0)[:, None] & (column == full[:, None])
        rows = torch.where(partial, state["pages"][:, None], rows)
        table[children] = torch.where(column < used[:, None], rows, table[children])
        lens[children] = n
        part = (n % page).nonzero()[:, 0]
        src, dst = table[parents[part], full[part].long()].long(), state["pages"][part].long()
        for name in _POOLS:
            if name in state:
                state[name][dst] = state[name][src]
        return _outputs(state, page_table=table, seq_lens=lens)
    if kind == "free":
        lens[state["rows"].long()] = 0
        _, used = _used(table, lens, page, pool)
        free = (~used).nonzero()[:, 0].to(torch.int32)
        pages = torch.full((pool,), -1, dtype=torch.int32, device=table.device)
        pages[:free.shape[0]] = free
        return {"seq_lens": lens, "pages": pages, "count": pool - used.sum(dtype=torch.int32)}
    columns, used = _used(table, lens, page, pool)
    count = used.sum(dtype=torch.int32)
    ids = torch.arange(pool, device=table.device)
    src = (used & (ids >= count)).nonzero()[:, 0]
    dst = (~used & (ids < count)).nonzero()[:, 0]
    remap = torch.where(used, ids, -1).to(torch.int32)
    remap[src] = dst.to(torch.int32)
    for name in _POOLS:
        if name in state:
            state[name][dst] = state[name][src]
    table.copy_(torch.where(columns, remap[table.long()], table))
    return _outputs(state, page_table=table, remap=remap, count=count)


def _attend_plain(state):
    """Scores of the shared keys once for all of a group's rows, of the others in one padded batch; their softmax is
    joined by the larger maximum.  In 32 bits, rounded once."""
    q, page, table, each = state["q"], state["page"], state["table"], state["each"]
    k, v, scales = state["k"], state["v"], state["scales"]
    kv_heads, dim = k.shape[2], k.shape[3]
    q4 = (q if q.dim() == 4 else q[:, None]).float() * dim ** -0.5
    batch, tokens, heads = q4.shape[:3]
    # [batch, kv_heads, rows, dim], rows = tokens x heads of one KV head
    rows = q4.view(batch, tokens, kv_heads, heads // kv_heads, dim).permute(0, 2, 1, 3, 4).reshape(
        batch, kv_heads, -1, dim)

    def keys(ids):
        """K and V of the pages ``ids`` [..., pages], as [..., kv_heads, tokens, dim]."""
        out = []
        for x, name in ((k, "k"), (v, "v")):
            x = x[ids].float()
            if scales is not None:
                x = x * scales[name][ids][..., None, :, None]
            x = x.flatten(-4, -3)  # pages x slots
            out.append(x.transpose(-3, -2).contiguous())
        return out

    def attend(r, kk, vv, mask=None):
        s = r @ kk.transpose(-1, -2).contiguous()
        if mask is not None:
            s = s.masked_fill(mask, -math.inf)
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - top)
        return p @ vv, top, p.sum(-1, keepdim=True)

    device = q.device
    prefixes, tails = state["prefixes"], state["tails"]
    acc = torch.zeros(rows.shape, device=device)
    top = torch.full((*rows.shape[:3], 1), -math.inf, device=device)
    total = torch.zeros((*rows.shape[:3], 1), device=device)
    for i, n in enumerate(prefixes):
        if n:
            lo, hi = i * each, (i + 1) * each
            r = rows[lo:hi].transpose(0, 1).reshape(kv_heads, -1, dim)
            kk, vv = keys(table[lo, :n // page].long())
            a, m, t = attend(r, kk, vv)
            for to, x in ((acc, a), (top, m), (total, t)):
                to[lo:hi] = x.view(kv_heads, each, -1, x.shape[-1]).transpose(0, 1)
    # The other keys: each row's pages behind its prefix, padded to the widest.
    first = torch.tensor([p // page for p in prefixes], device=device).repeat_interleave(each)
    left = torch.tensor(tails, device=device)
    column = first[:, None] + torch.arange(-(-max(tails) // page), device=device)
    kk, vv = keys(table.gather(1, column.clamp_max(table.shape[1] - 1)).long())
    key = torch.arange(kk.shape[-2], device=device)
    token = torch.arange(tokens, device=device).repeat_interleave(heads // kv_heads)
    mask = key >= (left[:, None] - tokens + 1 + token)[:, None, :, None]
    a, m, t = attend(rows, kk, vv, mask)
    both = torch.maximum(top, m)
    w0, w1 = torch.exp(top - both), torch.exp(m - both)
    out = (acc * w0 + a * w1) / (total * w0 + t * w1)
    out = out.view(batch, kv_heads, tokens, heads // kv_heads, dim).permute(0, 2, 1, 3, 4).reshape(q4.shape)
    return out.reshape(q.shape).to(q.dtype)


# ---------------------------------------------------------------------------
# The same in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    """Attention only: the other operators move bits and whole numbers."""
    if case["kind"] != "shared":
        return None
    state = prepare(case, seed)
    q, page, scales = state["q"], state["page"], state["scales"]
    q = q.double() if q.dim() == 4 else q.double()[:, None]
    heads, dim = q.shape[2:]
    kv_heads = case["kv_heads"]
    group = heads // kv_heads
    out = torch.empty_like(q)
    for b, n in enumerate(state["lens"].tolist()):
        ids = state["table"][b, :-(-n // page)].long()
        kv = []
        for name in ("k", "v"):
            x = state[name][ids].double()
            if scales is not None:
                x = x * scales[name][ids].double()[:, None, :, None]
            kv.append(x.reshape(-1, kv_heads, dim)[:n])
        for t in range(q.shape[1]):
            seen = n - q.shape[1] + 1 + t
            for j in range(kv_heads):
                s = q[b, t, j * group:(j + 1) * group] @ kv[0][:seen, j].t().contiguous() * dim ** -0.5
                p = torch.exp(s - s.amax(dim=1, keepdim=True))
                out[b, t, j * group:(j + 1) * group] = (p / p.sum(dim=1, keepdim=True)) @ kv[1][:seen, j].contiguous()
    return out if state["q"].dim() == 4 else out[:, 0]
