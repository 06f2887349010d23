"""The paged key-value cache and the attention that reads it, as cases that can
be timed and compared.

A cache holds the keys and values of every layer in pages of ``page`` positions
([layers, pages, kv_heads, page, head_dim]); each sequence has a row of a table
naming its pages, a length, and every page a count of the rows that name it.

- ``decode``   one new token of each sequence against its pages, all of them or
               a sliding window and a few first tokens (sinks): PagedAttention;
- ``prompt``   the tokens of prompts or chunks of prompts, ragged, against the
               pages of what came before and of themselves: PagedPrefill;
- ``append``   rows of new keys and values into the pages a sequence grows by:
               KVReserve and KVAppend, for a decode step and for prompts;
- ``fork``     sequences branched from others (beams, shared prefixes): whole
               pages shared, a last page that is partly full copied: KVFree of
               the branches that lost and KVFork of those that go on;
- ``compact``  a fragmented pool's pages moved to its lowest numbers, so that
               the rest can be given back: KVCompact.

With ``own`` false every pass is elementary torch in 32 bits on the same
tensors; with ``own`` true it is the package's operators.  An append and a
compaction start from the bookkeeping they found (a copy of it is laid over it
first), so that they can be repeated; branching anew repeats itself.

Sizes are those of the repository's benchmark layer (4096 wide: 32 query heads
and 8 key-value heads of 128) and generic odd ones.
"""
import math

import torch

own = False

NONE = -1      # a table entry without a page (0xffffffff as the cache's unsigned words)


# ---- the cases ---------------------------------------------------------------

def listed():
    return [
        # one sequence early in a chat: the smallest call, where latency counts
        dict(name="decode_short", op="decode", B=1, lo=200, hi=200, q="bf16", kv="bf16",
             heads=32, kv_heads=8, dim=128, page=16, window=0, sinks=0),
        # one long context in the framework's f32 activations: the split over
        # its length and the join are all the parallelism there is
        dict(name="decode_long_f32", op="decode", B=1, lo=32768, hi=32768, q="f32", kv="bf16",
             heads=32, kv_heads=8, dim=128, page=16, window=0, sinks=0),
        # a serving batch of very different lengths: the bytes
        dict(name="decode_batch", op="decode", B=64, lo=1, hi=8192, q="bf16", kv="bf16",
             heads=32, kv_heads=8, dim=128, page=16, window=0, sinks=0),
        # streaming generation: a window and four sinks, pages behind it given back
        dict(name="decode_window", op="decode", B=33, lo=500, hi=16000, q="f16", kv="f16",
             heads=16, kv_heads=4, dim=64, page=32, window=1000, sinks=4),
        # a prompt of the benchmark's length
        dict(name="prompt_bf16", op="prompt", B=1, lo=2048, hi=2048, prefix=0, q="bf16",
             kv="bf16", heads=32, kv_heads=8, dim=128, page=16, window=0, sinks=0),
        # a long prompt through a sliding window with sinks: the largest
        dict(name="prompt_window", op="prompt", B=1, lo=8192, hi=8192, prefix=0, q="bf16",
             kv="bf16", heads=32, kv_heads=8, dim=128, page=16, window=1024, sinks=4),
        # chunks of several prompts, of odd lengths, after cached prefixes, head
        # and page sizes off the tiles
        dict(name="chunks_ragged", op="prompt", B=5, lo=3, hi=700, prefix=1500, q="f16",
             kv="f16", heads=12, kv_heads=4, dim=80, page=8, window=333, sinks=5),
        # a prompt in f32 activations, to f32 accuracy
        dict(name="prompt_f32", op="prompt", B=1, lo=333, hi=333, prefix=100, q="f32",
             kv="bf16", heads=32, kv_heads=8, dim=128, page=64, window=0, sinks=0),
        # a decode step's new keys and values in f32, one layer, with the pages they need
        dict(name="append_step", op="append", B=64, n=1, lo=1, hi=4096, q="f32", kv="bf16",
             layers=2, kv_heads=8, dim=128, page=16),
        # a batch of prompts' keys and values
        dict(name="append_prompts", op="append", B=7, n=1000, lo=0, hi=500, q="bf16", kv="bf16",
             layers=2, kv_heads=8, dim=128, page=16),
        # four requests of eight beams each: seven lose and branch off again
        dict(name="fork_beams", op="fork", B=4, beams=8, lo=100, hi=2000, kv="bf16", layers=32,
             kv_heads=8, dim=128, page=16),
        # a pool of 16 layers, seven pages in ten live, a quarter of those out of place
        dict(name="compact_pool", op="compact", B=24, pages=2000, live=1400, moved=350,
             kv="bf16", layers=16, kv_heads=8, dim=128, page=16),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 2, 3, 4, 4, 7, 8])
    while kv_heads * group > 32:
        group = max(1, group // 2)
    dim = rng.choice([64, 64, 80, 96, 128, 128, 128, 256])
    return dict(heads=kv_heads * group, kv_heads=kv_heads, dim=dim)


def _types(rng):
    q, kv = rng.choice([("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16"), ("f32", "f16")])
    return dict(q=q, kv=kv)


def _window(rng):
    if rng.random() < 0.5:
        return dict(window=0, sinks=0)
    return dict(window=_log(rng, 16, 2000), sinks=rng.choice([0, 1, 4, 13, 64]))


def draw(rng):
    op = rng.choice(["decode", "decode", "prompt", "prompt", "append", "fork", "compact"])
    page = rng.choice([8, 16, 16, 32, 64])
    if op == "decode":
        h = _heads(rng)
        B, hi = _log(rng, 1, 128), _log(rng, 30, 40000)
        # no more keys and values than the largest listed batch
        while B * hi * h["kv_heads"] * h["dim"] > 64 * 8192 * 1024:
            B, hi = max(1, B // 2), max(30, hi * 3 // 4)
        return dict(op="decode", B=B, lo=rng.randint(1, hi), hi=hi, page=page, **h,
                    **_types(rng), **_window(rng))
    if op == "prompt":
        h, t, w = _heads(rng), _types(rng), _window(rng)
        B, hi, prefix = rng.choice([1, 1, 2, 3, 6]), _log(rng, 2, 4000), 0
        if rng.random() < 0.5:
            prefix = _log(rng, 1, 3000)
        cost = 3 if t["q"] == "f32" else 1
        while B * hi * (hi + prefix) * h["heads"] * h["dim"] * cost > 2048 * 2048 * 4096 * 4:
            hi, prefix = max(2, hi * 3 // 4), prefix * 3 // 4
        return dict(op="prompt", B=B, lo=max(1, hi // 3), hi=hi, prefix=prefix, page=page, **h,
                    **t, **w)
    h = _heads(rng)
    shape = dict(kv_heads=h["kv_heads"], dim=h["dim"], page=page)
    if op == "append":
        B = _log(rng, 1, 128)
        return dict(op="append", B=B, n=1 if rng.random() < 0.5 else _log(rng, 2, 4000 // B + 3),
                    lo=0, hi=_log(rng, 1, 2000), layers=rng.choice([1, 2, 3]), **shape,
                    **_types(rng))
    if op == "fork":
        return dict(op="fork", B=_log(rng, 1, 8), beams=rng.randint(2, 8), lo=1,
                    hi=_log(rng, 10, 2000), layers=_log(rng, 1, 16),
                    kv=rng.choice(["bf16", "f16"]), **shape)
    pages = _log(rng, 10, 2000)
    live = rng.randint(pages // 3, pages - 1)
    return dict(op="compact", B=_log(rng, 1, 30), pages=pages, live=live,
                moved=rng.randint(0, min(live, pages - live)), layers=_log(rng, 1, 8),
                kv=rng.choice(["bf16", "f16"]), **shape)


# ---- inputs --------------------------------------------------------------------

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _spread(B, lo, hi):
    """B whole numbers evenly from hi down to lo, in a mixed order that is the
    same for every seed (outputs of one case have one shape)."""
    n = [hi - (hi - lo) * i // max(1, B - 1) for i in range(B)]
    return [n[i] for i in torch.randperm(B, generator=torch.Generator().manual_seed(B)).tolist()]


def _lengths(case):
    """Each sequence's length (decode), new tokens (prompt) or tokens before
    the call (append, fork)."""
    return _spread(case["B"], case["lo"], case["hi"])


def _new(case):
    """The tokens each sequence brings or grows by."""
    if case["op"] == "append":
        return _spread(case["B"], max(1, case["n"] // 2), case["n"])
    return _lengths(case) if case["op"] == "prompt" else [1] * case["B"]


def _total(case):
    """Each sequence's length with what it brings (decode, prompt)."""
    if case["op"] == "decode":
        return _lengths(case)
    before = _spread(case["B"], 0, case["prefix"])
    return [a + b for a, b in zip(before[::-1], _new(case))]


def _table(case, held, pages, slots, cpu):
    """Rows of `held[i]` pages out of a shuffled pool, and the pages' counts."""
    order = torch.randperm(pages, generator=cpu)
    table = torch.full((len(held), slots), NONE, dtype=torch.int32)
    refs = torch.zeros(pages, dtype=torch.int32)
    at = 0
    for i, n in enumerate(held):
        table[i, :n] = order[at:at + n].int()
        refs[order[at:at + n]] = 1
        at += n
    return table, refs


def _behind(case, total, new, s):
    """The table slots of a sequence whose positions no query sees any more."""
    if not case.get("window"):
        return range(0)
    first = -(-case["sinks"] // case["page"])
    return range(first, max(first, (total - new - case["window"] + 1) // case["page"]))


def _cache(case, layers, pages, g):
    shape = (layers, pages, case["kv_heads"], case["page"], case["dim"])
    return (torch.randn(shape, generator=g, device="cuda", dtype=_TYPES[case["kv"]]),
            torch.randn(shape, generator=g, device="cuda", dtype=_TYPES[case["kv"]]))


def _inputs(case, seed):
    """Everything drawn for a case, from the seed alone.  The bookkeeping is one
    tensor, its views the pages' counts, the tables and the lengths."""
    cpu = torch.Generator().manual_seed(int(seed))
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    op, page = case["op"], case["page"]
    up = lambda n: -(-n // page)  # noqa: E731
    r = dict(op=op)
    if op in ("decode", "prompt"):
        new, total = _new(case), _total(case)
        slots = up(max(total)) + 2
        held = [up(n) for n in total]
        gone = [_behind(case, t, n, s) for s, (t, n) in enumerate(zip(total, new))]
        pages = max(1, sum(held) - sum(len(x) for x in gone)) + 5
        full, _ = _table(case, held, sum(held), slots, cpu)
        order = torch.randperm(pages, generator=cpu).int()
        table, at = torch.full_like(full, NONE), 0
        for i, x in enumerate(gone):
            keep = [j for j in range(held[i]) if j not in x]
            table[i, keep] = order[at:at + len(keep)]
            at += len(keep)
        refs = torch.zeros(pages, dtype=torch.int32)
        refs[order[:at].long()] = 1
        lens = torch.tensor(total, dtype=torch.int32)
        r["keys"], r["values"] = _cache(case, 1, pages, g)
        # scores spread as trained heads' are: a few keys weigh most
        r["q"] = (2 * torch.randn(sum(new), case["heads"], case["dim"], generator=g,
                                  device="cuda")).to(_TYPES[case["q"]])
        r["new"], r["total"] = new, total
    elif op == "append":
        before, new = _lengths(case), _new(case)
        held, most = [up(n) for n in before], [up(a + b) for a, b in zip(before, new)]
        slots, pages = max(most) + 1, sum(most) + 9
        table, refs = _table(case, held, pages, slots, cpu)
        lens = torch.tensor(before, dtype=torch.int32)
        r["keys"], r["values"] = _cache(case, case["layers"], pages, g)
        for x in ("k", "v"):
            r[x] = torch.randn(sum(new), case["kv_heads"], case["dim"], generator=g,
                               device="cuda").to(_TYPES[case["q"]])
        r["new"], r["layer"] = new, case["layers"] - 1
    elif op == "fork":
        n = _lengths(case)
        held = [up(x) for x in n]
        rows = case["B"] * case["beams"]
        slots, pages = max(held) + 1, sum(held) + rows + 3
        full, refs = _table(case, held, pages, slots, cpu)
        table = torch.full((rows, slots), NONE, dtype=torch.int32)
        lens = torch.zeros(rows, dtype=torch.int32)
        table[::case["beams"]] = full
        lens[::case["beams"]] = torch.tensor(n, dtype=torch.int32)
        r["keys"], r["values"] = _cache(case, case["layers"], pages, g)
        r["parents"] = [b * case["beams"] for b in range(case["B"])
                        for _ in range(1, case["beams"])]
        r["children"] = [b * case["beams"] + i for b in range(case["B"])
                         for i in range(1, case["beams"])]
    else:
        pages, live, moved = case["pages"], case["live"], case["moved"]
        refs = torch.zeros(pages, dtype=torch.int32)
        refs[torch.randperm(live, generator=cpu)[:live - moved]] = 1
        refs[live + torch.randperm(pages - live, generator=cpu)[:moved]] = 1
        named = refs.nonzero().flatten()
        named = named[torch.randperm(live, generator=cpu)]
        # every row as many pages as the next, and the first pages of row 0 in
        # all rows, as branches of one prompt have
        per = -(-live // case["B"])
        shared = min(4, per)
        slots = per + shared
        table = torch.full((case["B"], slots), NONE, dtype=torch.int32)
        lens = torch.zeros(case["B"], dtype=torch.int32)
        for i in range(case["B"]):
            mine = named[i * per:(i + 1) * per]
            if i and len(mine):
                mine = torch.cat([named[:shared], mine])
                refs[named[:shared]] += 1
            table[i, :len(mine)] = mine.int()
            lens[i] = len(mine) * page
        r["keys"], r["values"] = _cache(case, case["layers"], pages, g)
    parts = [refs, table.flatten(), lens]
    r["book"] = torch.cat(parts).cuda()
    r["refs"], flat, r["lens"] = r["book"].split([len(p) for p in parts])
    r["table"] = flat.view(table.shape)
    r["case"] = case
    return r


def prepare(case, seed):
    s = _inputs(case, seed)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    if case["op"] == "fork":
        # the branches of the step before: a pass frees them and branches anew
        s["parent_rows"], s["child_rows"] = ints(s["parents"]), ints(s["children"])
        _fork(s)
    s["saved"] = s["book"].clone()
    if "new" in s:
        s["grow"] = ints(s["new"])
        s["offsets"] = torch.nn.functional.pad(s["grow"].cumsum(0), (1, 0)).int()
    if "q" in s:
        s["out"] = torch.empty_like(s["q"])
    if case["op"] == "compact":
        s["live"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    if own:
        _bind(s)
    torch.cuda.synchronize()
    return s


# ---- one pass through the package's operators --------------------------------------

_device = None


def _bind(s):
    """The state's tensors as buffers of the package, and its cache."""
    global _device
    import accel_amd
    if _device is None:
        _device = accel_amd.Device(0)
    codes = {torch.float32: accel_amd.F32, torch.float16: accel_amd.F16,
             torch.bfloat16: accel_amd.BF16, torch.int32: accel_amd.U32}
    b = {k: accel_amd.Buffer(_device, t.data_ptr(), t.numel() * t.element_size(),
                             codes[t.dtype], tuple(t.shape))
         for k, t in s.items() if isinstance(t, torch.Tensor)}
    s["dev"], s["b"] = _device, b
    s["cache"] = accel_amd.KVCache(_device, b["keys"], b["values"], b["refs"], b["table"],
                                   b["lens"])


def _run_own(s):
    dev, b, cache, case = s["dev"], s["b"], s["cache"], s["case"]
    st = torch.cuda.current_stream().cuda_stream
    op = s["op"]
    if op == "decode":
        dev.PagedAttention(b["q"], cache, b["out"], window=case["window"],
                           sinks=case["sinks"], stream=st)
        return s["out"]
    if op == "prompt":
        dev.PagedPrefill(b["q"], b["offsets"], cache, b["out"], window=case["window"],
                         sinks=case["sinks"], stream=st)
        return s["out"]
    if op != "fork":
        s["book"].copy_(s["saved"])
    if op == "append":
        dev.KVReserve(cache, b["grow"], stream=st)
        dev.KVAppend(cache, s["layer"], b["k"], b["v"], offsets=b["offsets"], stream=st)
    elif op == "fork":
        dev.KVFree(cache, b["child_rows"], stream=st)
        dev.KVFork(cache, b["parent_rows"], b["child_rows"], stream=st)
    else:
        dev.KVCompact(cache, b["live"], stream=st)
        return [s[k] for k in ("keys", "values", "refs", "table", "lens", "live")]
    return [s[k] for k in ("keys", "values", "refs", "table", "lens")]


# ---- one pass in plain torch -------------------------------------------------------

def _attend(s):
    """Each sequence's queries against the keys they see: gather, product,
    mask, softmax, product, one key-value head at a time."""
    case = s["case"]
    page, w, sinks = case["page"], case["window"], case["sinks"]
    G = case["heads"] // case["kv_heads"]
    scale = 1 / math.sqrt(case["dim"])
    at = 0
    for i, (n, total) in enumerate(zip(s["new"], s["total"])):
        lo = max(0, total - n - w + 1) if w else 0
        first = min(sinks, lo) if w else 0
        pos = torch.cat([torch.arange(first, device="cuda"),
                         torch.arange(lo, total, device="cuda")])
        where = s["table"][i].long()[pos // page]
        at_q = torch.arange(total - n, total, device="cuda")[:, None]
        seen = pos <= at_q
        if w:
            seen &= (at_q - pos < w) | (pos < sinks)
        for h in range(case["kv_heads"]):
            k = s["keys"][0, where, h, pos % page].float()
            v = s["values"][0, where, h, pos % page].float()
            q = s["q"][at:at + n, h * G:(h + 1) * G].float()
            score = (q @ k.t().contiguous()) * scale
            score = score.masked_fill(~seen[:, None], -math.inf)
            p = torch.exp(score - score.amax(-1, keepdim=True))
            s["out"][at:at + n, h * G:(h + 1) * G] = (p @ v) / p.sum(-1, keepdim=True)
        at += n
    return s["out"]


def _reserve(s):
    """Pages for the positions each sequence grows by: the lowest free ones,
    sequence by sequence."""
    page, slots = s["case"]["page"], s["table"].shape[1]
    have = (s["lens"] + page - 1) // page
    want = (s["lens"] + s["grow"] + page - 1) // page
    slot = torch.arange(slots, device="cuda")
    fresh = (slot >= have[:, None]) & (slot < want[:, None])
    rows, cols = fresh.nonzero(as_tuple=True)
    free = (s["refs"] == 0).nonzero().flatten()[:len(rows)]
    s["table"][rows, cols] = free.int()
    s["refs"][free] = 1
    s["lens"] += s["grow"]


def _append(s):
    page = s["case"]["page"]
    T = s["k"].shape[0]
    row = torch.arange(T, device="cuda")
    seq = torch.searchsorted(s["offsets"][1:].contiguous(), row.int(), right=True)
    pos = s["lens"][seq].long() - s["offsets"][seq + 1].long() + row
    where = s["table"][seq, pos // page].long()
    s["keys"][s["layer"]][where, :, pos % page] = s["k"].to(s["keys"].dtype)
    s["values"][s["layer"]][where, :, pos % page] = s["v"].to(s["values"].dtype)


def _free(s):
    rows = s["child_rows"].long()
    named = s["table"][rows].flatten()
    named = named[named >= 0].long()
    s["refs"].index_add_(0, named, torch.full_like(named, -1, dtype=torch.int32))
    s["table"][rows] = NONE
    s["lens"][rows] = 0


def _fork(s):
    page = s["case"]["page"]
    parent, child = s["parent_rows"].long(), s["child_rows"].long()
    n = s["lens"][parent]
    table = s["table"][parent]
    # the last page, where it is partly full, is the child's own copy
    part = (n % page != 0).nonzero().flatten()
    last = (n[part] // page).long()
    src = table[part, last].long()
    dst = (s["refs"] == 0).nonzero().flatten()[:len(part)]
    whole = torch.arange(table.shape[1], device="cuda") < (n // page)[:, None]
    shared = table[whole].long()
    s["refs"].index_add_(0, shared, torch.ones_like(shared, dtype=torch.int32))
    table = torch.where(whole, table, torch.full_like(table, NONE))
    table[part, last] = dst.int()
    s["refs"][dst] = 1
    s["table"][child] = table
    s["lens"][child] = n
    s["keys"][:, dst] = s["keys"][:, src]
    s["values"][:, dst] = s["values"][:, src]


def _compact(s):
    live = s["refs"] > 0
    count = live.sum()
    page = torch.arange(len(live), device="cuda")
    dst = ((page < count) & ~live).nonzero().flatten()
    src = ((page >= count) & live).nonzero().flatten()
    remap = page.clone()
    remap[src] = dst
    t = s["table"]
    s["table"].copy_(torch.where(t >= 0, remap[t.clamp_min(0).long()].int(), t))
    s["refs"][dst] = s["refs"][src]
    s["refs"][src] = 0
    s["keys"][:, dst] = s["keys"][:, src]
    s["values"][:, dst] = s["values"][:, src]
    s["live"].copy_(count)


def run(s):
    if own:
        return _run_own(s)
    op = s["op"]
    if op in ("decode", "prompt"):
        return _attend(s)
    if op != "fork":
        s["book"].copy_(s["saved"])
    if op == "append":
        _reserve(s)
        _append(s)
    elif op == "fork":
        _free(s)
        _fork(s)
    else:
        _compact(s)
        return [s[k] for k in ("keys", "values", "refs", "table", "lens", "live")]
    return [s[k] for k in ("keys", "values", "refs", "table", "lens")]


# ---- what a pass cannot do without ---------------------------------------------------

def _pairs(case, new, total):
    """Query and key pairs that see each other, and keys that some query sees."""
    w, sinks = case["window"], case["sinks"]
    before = total - new
    if not w:
        return new * before + new * (new + 1) / 2, total
    pairs = 0.0
    # in at most 64 strips of queries, each at its middle
    for i in range(64):
        p = before + (i + 0.5) * new / 64
        near = min(p + 0.5, w)
        pairs += new / 64 * (near + min(sinks, max(0, p + 0.5 - w)))
    lo = max(0, before - w + 1)
    return pairs, total - lo + min(sinks, lo)


def work(case):
    op = case["op"]
    wide = 4 if case.get("q") == "f32" else 2
    row = case["kv_heads"] * case["dim"]
    if op in ("decode", "prompt"):
        d = case["heads"] * case["dim"]
        size = flops = 0
        for new, total in zip(_new(case), _total(case)):
            pairs, keys = _pairs(case, new, total)
            size += keys * row * 4 + 2 * wide * new * d
            flops += pairs * 4 * d
        return {"bytes": size, "flops": flops}
    if op == "append":
        return {"bytes": sum(_new(case)) * row * 2 * (wide + 2), "flops": 0}
    page = 2 * 2 * row * case["page"] * case["layers"]
    if op == "fork":
        # a partly full page a branch, its row of the table read and written
        part = sum(1 for n in _lengths(case) if n % case["page"])
        slots = sum(-(-n // case["page"]) for n in _lengths(case))
        return {"bytes": (case["beams"] - 1) * (2 * part * page + 8 * slots), "flops": 0}
    return {"bytes": 2 * case["moved"] * page + 8 * case["live"] + 8 * case["pages"],
            "flops": 0}


# ---- the same in 64 bits ---------------------------------------------------------------

def exact(case, seed):
    """Attention by its definition, query by query in blocks: every key of the
    sequence with its weight exp(q.k / sqrt(dim)) or 0.  Rows put into pages are
    themselves; what only moves has no such value."""
    op = case["op"]
    if op in ("fork", "compact"):
        return None
    r = _inputs(case, seed)
    page, table = case["page"], r["table"].long()
    if op == "append":
        keys, values = r["keys"].double(), r["values"].double()
        return [*_exact_append(case, r, keys, values), None, None, None]
    out = torch.zeros(r["q"].shape, dtype=torch.float64, device="cuda")
    at = 0
    G = case["heads"] // case["kv_heads"]
    for b, (n, total) in enumerate(zip(r["new"], r["total"])):
        ids = table[b, :-(-total // page)].clamp_min(0)
        # [kv_heads, total, dim]; what no query sees is there with weight 0
        K = r["keys"][0, ids].double().transpose(0, 1).reshape(
            case["kv_heads"], -1, case["dim"])[:, :total]
        V = r["values"][0, ids].double().transpose(0, 1).reshape(
            case["kv_heads"], -1, case["dim"])[:, :total]
        j = torch.arange(total, device="cuda")
        for i0 in range(0, n, 512):
            i = torch.arange(i0, min(n, i0 + 512), device="cuda") + (total - n)
            ok = j[None, :] <= i[:, None]
            if case["window"]:
                ok &= (j[None, :] > i[:, None] - case["window"]) | (j < case["sinks"])[None, :]
            for head in range(case["heads"]):
                q = r["q"][at + i0:at + i0 + len(i), head].double()
                x = torch.mm(q, K[head // G].t().contiguous()).div_(math.sqrt(case["dim"]))
                top = torch.where(ok, x, x.new_full((), -math.inf)).max(1, keepdim=True).values
                e = torch.where(ok, (x - top).exp(), x.new_zeros(()))
                out[at + i0:at + i0 + len(i), head] = torch.mm(e / e.sum(1, keepdim=True),
                                                              V[head // G])
        at += n
    return out


def _exact_append(case, r, keys, values):
    """The caches after a reservation and an append, from lists."""
    page, layer = case["page"], r["layer"]
    free = [p for p, c in enumerate(r["refs"].tolist()) if c == 0]
    tables, lens = r["table"].tolist(), r["lens"].tolist()
    where, slot = [], []
    for b, n in enumerate(r["new"]):
        for pos in range(lens[b], lens[b] + n):
            if tables[b][pos // page] == NONE:
                tables[b][pos // page] = free.pop(0)
            where.append(tables[b][pos // page])
            slot.append(pos % page)
    where = torch.tensor(where, device="cuda")
    slot = torch.tensor(slot, device="cuda")
    keys[layer][where, :, slot] = r["k"].double()
    values[layer][where, :, slot] = r["v"].double()
    return keys, values
