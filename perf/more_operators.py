"""A step of decoding that checks a tree of drafted tokens, as cases that can be
timed and compared.

A draft of a sequence is a tree: node 0 is the newest token, every other node a
guess for the token after its parent.  The nodes' keys and values lie in the
paged cache behind the sequence's context, in the nodes' order.

- ``tree``    attention of every node over the context and the nodes on its own
              path: PagedTreeAttention;
- ``sample``  a token of each row of logits by temperature, top-k, top-p and
              min-p from a given random number, and the logarithm of the chance
              it had: Sample;
- ``accept``  the walk from node 0 down the nodes whose tokens were sampled:
              TreeAccept;
- ``keep``    the accepted nodes' keys and values moved up behind the context in
              every layer, the rest's pages given back: KVKeep.

With ``own`` false every pass is elementary torch on the same tensors (32 bits;
the weights that choose tokens in 64); with ``own`` true it is the package's
operators.  A ``keep`` starts from the bookkeeping it found (a copy of it is laid
over it first), and its nodes that move come from places that no node moves to,
so that it can be repeated.

Sizes are those of the repository's benchmark layer (4096 wide: 32 query heads
and 8 key-value heads of 128) and generic odd ones.
"""
import math

import torch

own = False

NONE = -1      # 0xffffffff as the package's unsigned words: no page, no parent, no token


# ---- the cases ---------------------------------------------------------------

def listed():
    return [
        # a short chat with a small tree: the smallest attention, where latency counts
        dict(name="tree_small", op="tree", B=1, lo=500, hi=500, few=8, most=8, q="bf16",
             kv="bf16", heads=32, kv_heads=8, dim=128, page=16, window=0, sinks=0),
        # a serving batch of different contexts and trees: the bytes
        dict(name="tree_batch", op="tree", B=32, lo=300, hi=8000, few=16, most=64, q="bf16",
             kv="bf16", heads=32, kv_heads=8, dim=128, page=16, window=0, sinks=0),
        # one long context in the framework's f32 activations
        dict(name="tree_long_f32", op="tree", B=1, lo=32768, hi=32768, few=48, most=48, q="f32",
             kv="bf16", heads=32, kv_heads=8, dim=128, page=16, window=0, sinks=0),
        # streaming generation, heads and pages off the tiles, trees of one node and of many
        dict(name="tree_window", op="tree", B=9, lo=0, hi=3000, few=1, most=100, q="f16",
             kv="f16", heads=12, kv_heads=4, dim=80, page=8, window=333, sinks=5),
        # one request's next token: the smallest call
        dict(name="sample_one", op="sample", R=1, V=128000, x="f32", std=3.0, T_lo=0.7, T_hi=0.7, k_lo=50,
             k_hi=50, p_lo=0.9, p_hi=0.9, m_lo=0, m_hi=0),
        # a decode step's batch in the head product's 16-bit results, each row's own settings
        dict(name="sample_batch", op="sample", R=64, V=100003, x="bf16", std=2.5, T_lo=0, T_hi=1.3,
             k_lo=0, k_hi=200, p_lo=0.5, p_hi=1, m_lo=0, m_hi=0.1),
        # an odd vocabulary, temperature and top-p alone over nearly flat logits
        dict(name="sample_flat", op="sample", R=17, V=32001, x="f16", std=0.5, T_lo=0.8, T_hi=1.5,
             k_lo=0, k_hi=0, p_lo=0.9, p_hi=1, m_lo=0, m_hi=0),
        # every node of eight trees of 64: the largest
        dict(name="sample_nodes", op="sample", R=512, V=128000, x="f32", std=3.0, T_lo=0.6, T_hi=1,
             k_lo=0, k_hi=64, p_lo=0.8, p_hi=0.95, m_lo=0, m_hi=0.05),
        # one sequence's small tree
        dict(name="accept_one", op="accept", B=1, few=8, most=8, width=8),
        # a large batch of trees of different sizes
        dict(name="accept_batch", op="accept", B=256, few=1, most=64, width=12),
        # one sequence, 32 layers, nearly all of a short draft accepted
        dict(name="keep_one", op="keep", B=1, lo=700, hi=700, few=12, most=12, width=6, kv="bf16",
             layers=32, kv_heads=8, dim=128, page=16),
        # a serving batch: up to eight accepted of up to 64
        dict(name="keep_batch", op="keep", B=48, lo=10, hi=900, few=20, most=64, width=8,
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


def draw(rng):
    op = rng.choice(["tree", "tree", "tree", "sample", "sample", "sample", "accept", "keep"])
    page = rng.choice([8, 16, 16, 32, 64])
    if op == "tree":
        h = _heads(rng)
        q, kv = rng.choice([("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16"), ("f32", "f16")])
        B, hi, most = _log(rng, 1, 64), _log(rng, 30, 32768), _log(rng, 1, 128)
        # no more keys, values and products than the largest listed calls
        while B * hi * h["kv_heads"] * h["dim"] > 32 * 4000 * 1024:
            B, hi = max(1, B // 2), max(30, hi * 3 // 4)
        while B * hi * h["heads"] * h["dim"] * most > 32768 * 4096 * 48:
            most = max(1, most // 2)
        window = 0 if rng.random() < 0.6 else _log(rng, 16, 2000)
        return dict(op=op, B=B, lo=rng.randint(0, hi), hi=hi, few=rng.randint(1, most), most=most,
                    q=q, kv=kv, page=page, window=window,
                    sinks=rng.choice([0, 1, 4, 13, 64]) if window else 0, **h)
    if op == "sample":
        R, V = _log(rng, 1, 512), _log(rng, 1000, 200000)
        while R * V > 512 * 128000:
            R //= 2
        T = round(rng.uniform(0.3, 1.5), 3)
        k = rng.choice([0, 0, 1, 20, 50, 200, 1000])
        return dict(op=op, R=R, V=V, x=rng.choice(["f32", "f32", "bf16", "f16"]),
                    std=round(rng.uniform(0.5, 4), 3), T_lo=rng.choice([0, T, T]), T_hi=T,
                    k_lo=rng.choice([0, k]), k_hi=k, p_lo=rng.choice([0.3, 0.7, 0.9, 1]), p_hi=1,
                    m_lo=0, m_hi=rng.choice([0, 0, 0.02, 0.1]))
    most = _log(rng, 1, 128)
    if op == "accept":
        return dict(op=op, B=_log(rng, 1, 512), few=rng.randint(1, most), most=most,
                    width=rng.randint(1, 16))
    most = max(2, most)
    h = _heads(rng)
    B, layers = _log(rng, 1, 48), _log(rng, 1, 32)
    while B * layers > 48 * 16:
        layers = max(1, layers // 2)
    few = rng.randint(1, most)
    return dict(op=op, B=B, lo=0, hi=_log(rng, 10, 900), few=few, most=most,
                width=rng.randint(1, 12), kv=rng.choice(["bf16", "f16"]), layers=layers,
                page=page, kv_heads=h["kv_heads"], dim=h["dim"])


# ---- inputs --------------------------------------------------------------------

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _spread(B, lo, hi):
    """B whole numbers evenly from hi down to lo, in a mixed order that is the
    same for every seed (outputs of one case have one shape)."""
    n = [hi - (hi - lo) * i // max(1, B - 1) for i in range(B)]
    return [n[i] for i in torch.randperm(B, generator=torch.Generator().manual_seed(B)).tolist()]


def _nodes(case):
    return _spread(case["B"], case["few"], case["most"])


def _context(case):
    """Positions before the nodes, in another order than their numbers."""
    return _spread(case["B"], case["lo"], case["hi"])[::-1]


def _kept(case):
    """(accepted, of them in place already) of each sequence of a keep."""
    r = []
    for i, m in enumerate(_nodes(case)):
        n = min(case["width"] - i % max(1, case["width"]), m)
        # those that move come from past all places they move to
        stay = max(1, n - max(0, m - n)) if n else 0
        r.append((n, min(n, stay + i % 2)))
    return r


def _parents(nodes, cpu):
    """Trees of two to four guesses a node, level by level, a few nodes of each
    hung elsewhere."""
    r = []
    for m in nodes:
        t = torch.arange(m)
        wide = int(torch.randint(2, 5, (1,), generator=cpu))
        up = (t - 1) // wide
        other = (torch.rand(m, generator=cpu) * t).long()
        up = torch.where(torch.rand(m, generator=cpu) < 0.2, other, up)
        up[0] = NONE
        r.append(up)
    return torch.cat(r).int()


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


def _between(lo, hi, n, g):
    """n settings from lo to hi, every fourth lo itself."""
    r = lo + (hi - lo) * torch.rand(n, generator=g, device="cuda")
    r[::4] = lo
    return r


def _inputs(case, seed):
    """Everything drawn for a case, from the seed alone."""
    cpu = torch.Generator().manual_seed(int(seed))
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    op = case["op"]
    r = dict(op=op, case=case)
    if op == "sample":
        R, V = case["R"], case["V"]
        x = torch.randn(R, V, generator=g, device="cuda").mul_(case["std"])
        # a head's logits: most rows have a few tokens that stand out
        hot = torch.randint(0, V, (R, 5), generator=g, device="cuda")
        x.scatter_add_(1, hot, case["std"] * 4 * torch.rand(R, 5, generator=g, device="cuda"))
        # and some have tokens that are not allowed
        x[::3, V // 2:V // 2 + V // 7] = -math.inf
        r["x"] = x.to(_TYPES[case["x"]])
        r["u"] = torch.rand(R, generator=g, device="cuda")
        # settings of requests, of two digits
        for name in ("T", "p", "m"):
            r[name] = _between(case[name + "_lo"], case[name + "_hi"], R, g)
            r[name] = r[name].mul(100).round().div(100)
        r["k"] = _between(case["k_lo"], case["k_hi"], R, g).round().int()
        return r
    nodes = _nodes(case)
    r["nodes"] = nodes
    r["parents"] = _parents(nodes, cpu).cuda()
    r["offsets"] = torch.nn.functional.pad(torch.tensor(nodes).cumsum(0), (1, 0)).int().cuda()
    if op == "accept":
        T, W = sum(nodes), 32000
        token = torch.randint(0, W, (T,), generator=cpu)
        sampled = torch.randint(0, W, (T,), generator=cpu)
        # seven of ten nodes that have a guess behind them drew one of its tokens
        up, at = r["parents"].cpu().long(), 0
        for m in nodes:
            hit = (torch.rand(m, generator=cpu) < 0.7).tolist()
            for t in torch.randperm(m, generator=cpu).tolist():
                if t and hit[t]:
                    sampled[at + up[at + t]] = token[at + t]
            at += m
        r["token"], r["sampled"] = token.int().cuda(), sampled.int().cuda()
        return r
    page = case["page"]
    total = [a + b for a, b in zip(_context(case), nodes)]
    held = [-(-n // page) for n in total]
    slots, pages, layers = max(held) + 1, sum(held) + 3, case.get("layers", 1)
    table, refs = _table(case, held, pages, slots, cpu)
    shape = (layers, pages, case["kv_heads"], page, case["dim"])
    for x in ("keys", "values"):
        r[x] = torch.randn(shape, generator=g, device="cuda", dtype=_TYPES[case["kv"]])
    lens = torch.tensor(total, dtype=torch.int32)
    parts = [refs, table.flatten(), lens]
    r["book"] = torch.cat(parts).cuda()
    r["refs"], flat, r["lens"] = r["book"].split([len(p) for p in parts])
    r["table"], r["total"] = flat.view(table.shape), total
    if op == "tree":
        # scores spread as trained heads' are: a few keys weigh most
        r["q"] = (2 * torch.randn(sum(nodes), case["heads"], case["dim"], generator=g,
                                  device="cuda")).to(_TYPES[case["q"]])
        return r
    path = torch.full((case["B"], case["width"]), NONE, dtype=torch.int32)
    for i, (m, (n, stay)) in enumerate(zip(nodes, _kept(case))):
        path[i, :stay] = torch.arange(stay)
        path[i, stay:n] = (n + torch.randperm(m - n, generator=cpu)[:n - stay]).sort().values
    r["path"] = path.cuda()
    r["count"] = torch.tensor([n for n, _ in _kept(case)], dtype=torch.int32, device="cuda")
    return r


def prepare(case, seed):
    s = _inputs(case, seed)
    empty = lambda *n: torch.zeros(n, dtype=torch.int32, device="cuda")  # noqa: E731
    if case["op"] == "tree":
        s["out"] = torch.empty_like(s["q"])
    elif case["op"] == "sample":
        s["out"], s["logprob"] = empty(case["R"]), torch.zeros(case["R"], device="cuda")
    elif case["op"] == "accept":
        s["path"], s["count"], s["next"] = (empty(case["B"], case["width"]), empty(case["B"]),
                                            empty(case["B"]))
    else:
        s["saved"] = s["book"].clone()
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
    if "keys" in b:
        s["cache"] = accel_amd.KVCache(_device, b["keys"], b["values"], b["refs"], b["table"],
                                       b["lens"])


def _run_own(s):
    dev, b, case = s["dev"], s["b"], s["case"]
    st = torch.cuda.current_stream().cuda_stream
    op = s["op"]
    if op == "tree":
        dev.PagedTreeAttention(b["q"], b["offsets"], b["parents"], s["cache"], b["out"],
                               window=case["window"], sinks=case["sinks"], stream=st)
        return s["out"]
    if op == "sample":
        dev.Sample(b["x"], b["u"], b["out"], b["logprob"], temperature=b["T"], top_k=b["k"],
                   top_p=b["p"], min_p=b["m"], stream=st)
        return [s["out"], s["logprob"]]
    if op == "accept":
        dev.TreeAccept(b["token"], b["parents"], b["offsets"], b["sampled"], b["path"],
                       b["count"], b["next"], stream=st)
        return [s[k] for k in ("path", "count", "next")]
    s["book"].copy_(s["saved"])
    dev.KVKeep(s["cache"], b["path"], b["count"], b["offsets"], stream=st)
    return [s[k] for k in ("keys", "values", "refs", "table", "lens")]


# ---- one pass in plain torch -------------------------------------------------------

def _lineage(up, m):
    """Which of a tree's m nodes lie on each one's path (itself among them), and
    how deep each is."""
    on = torch.eye(m, dtype=torch.bool, device="cuda")
    at = torch.arange(m, device="cuda")
    depth = torch.zeros(m, dtype=torch.long, device="cuda")
    while True:
        at = torch.where(at >= 0, up[at.clamp_min(0)], at)
        live = at >= 0
        if not bool(live.any()):
            break
        on[live, at[live]] = True
        depth += live
    return on, depth


def _attend(s):
    """Each tree's queries against its context and its nodes: gather, product,
    mask, softmax, product, one key-value head at a time."""
    case = s["case"]
    page, w, sinks = case["page"], case["window"], case["sinks"]
    G = case["heads"] // case["kv_heads"]
    scale = 1 / math.sqrt(case["dim"])
    at = 0
    for i, (m, total) in enumerate(zip(s["nodes"], s["total"])):
        on, depth = _lineage(s["parents"][at:at + m].long(), m)
        L = total - m
        pos = torch.arange(total, device="cuda")
        # the position a key stands for: a node's is its depth's
        stands = torch.where(pos < L, pos, L + depth[(pos - L).clamp_min(0)])
        seen = torch.cat([torch.ones(m, L, dtype=torch.bool, device="cuda"), on], 1)
        if w:
            seen &= ((L + depth)[:, None] - stands < w) | (stands < sinks)
        where = s["table"][i].long()[pos // page]
        for h in range(case["kv_heads"]):
            k = s["keys"][0, where, h, pos % page].float()
            v = s["values"][0, where, h, pos % page].float()
            q = s["q"][at:at + m, h * G:(h + 1) * G].float()
            score = (q @ k.t().contiguous()) * scale
            score = score.masked_fill(~seen[:, None], -math.inf)
            p = torch.exp(score - score.amax(-1, keepdim=True))
            s["out"][at:at + m, h * G:(h + 1) * G] = (p @ v) / p.sum(-1, keepdim=True)
        at += m
    return s["out"]


def _sample(s):
    """Sorted, weighed in 64 bits, cut by each rule, and drawn from what is left;
    64 rows at a time."""
    V = s["case"]["V"]
    rank = torch.arange(V, device="cuda")
    for i in range(0, s["case"]["R"], 64):
        T, k, p, m, u = (s[n][i:i + 64, None].double() for n in ("T", "k", "p", "m", "u"))
        x, order = s["x"][i:i + 64].float().sort(dim=1, descending=True, stable=True)
        w = ((x.double() - x[:, :1].double()) / torch.where(T > 0, T, 1.0)).exp()
        w = torch.where((rank < k) | (k == 0), w, 0.0)
        run = w.cumsum(1)
        kept = (run - w < p * run[:, -1:]) | (p >= 1)
        kept &= w >= m
        kept[:, 0] = True
        run = torch.where(kept, w, 0.0).cumsum(1)
        pick = (run <= u * run[:, -1:]).sum(1, keepdim=True)
        pick = torch.where(T > 0, pick, 0)
        s["out"][i:i + 64] = order.gather(1, pick)[:, 0].int()
        chance = w.gather(1, pick) / run[:, -1:]
        s["logprob"][i:i + 64] = torch.where(T > 0, chance.log(), 0.0)[:, 0].float()
    return [s["out"], s["logprob"]]


def _accept(s):
    """All trees a step down at a time."""
    start, width = s["offsets"][:-1].long(), s["case"]["width"]
    most = max(s["nodes"])
    t = torch.arange(most, device="cuda")
    there = start[:, None] + t
    real = there < s["offsets"][1:, None]
    there = torch.where(real, there, 0)
    up, token = s["parents"][there], s["token"][there]
    node = torch.zeros_like(start)
    going = torch.ones_like(start, dtype=torch.bool)
    s["path"].fill_(NONE)
    s["count"].zero_()
    for d in range(width):
        s["path"][:, d] = torch.where(going, node, NONE).int()
        s["count"] += going
        s["next"].copy_(s["sampled"][start + node])
        fits = real & (t > 0) & (up == node[:, None]) & (token == s["next"][:, None])
        fits &= going[:, None]
        going = fits.any(1)
        node = torch.where(going, fits.int().argmax(1), node)
    return [s[k] for k in ("path", "count", "next")]


def _keep(s):
    page = s["case"]["page"]
    nodes = torch.diff(s["offsets"])
    L = (s["lens"] - nodes).long()
    c = torch.arange(s["case"]["width"], device="cuda")
    seq, c = ((c < s["count"][:, None]) & (s["path"] != c)).nonzero(as_tuple=True)
    src, dst = L[seq] + s["path"][seq, c], L[seq] + c
    src_page, dst_page = (s["table"][seq, x // page].long() for x in (src, dst))
    for x in ("keys", "values"):
        s[x][:, dst_page, :, dst % page] = s[x][:, src_page, :, src % page]
    s["lens"].copy_(L + s["count"])
    slot = torch.arange(s["table"].shape[1], device="cuda")
    gone = (slot >= (s["lens"][:, None] + page - 1) // page) & (s["table"] >= 0)
    freed = s["table"][gone].long()
    s["refs"].index_add_(0, freed, torch.full_like(freed, -1, dtype=torch.int32))
    s["table"].masked_fill_(gone, NONE)


def run(s):
    if own:
        return _run_own(s)
    op = s["op"]
    if op == "tree":
        return _attend(s)
    if op == "sample":
        return _sample(s)
    if op == "accept":
        return _accept(s)
    s["book"].copy_(s["saved"])
    _keep(s)
    return [s[k] for k in ("keys", "values", "refs", "table", "lens")]


# ---- what a pass cannot do without ---------------------------------------------------

def work(case):
    op = case["op"]
    if op == "sample":
        wide = 4 if case["x"] == "f32" else 2
        return {"bytes": case["R"] * (case["V"] * wide + 28), "flops": 0}
    nodes = _nodes(case)
    if op == "accept":
        return {"bytes": 12 * sum(nodes) + case["B"] * (4 * case["width"] + 12), "flops": 0}
    row = case["kv_heads"] * case["dim"]
    if op == "keep":
        moved = sum(n - stay for n, stay in _kept(case))
        return {"bytes": moved * case["layers"] * row * 8, "flops": 0}
    wide, d = (4 if case["q"] == "f32" else 2), case["heads"] * case["dim"]
    size = flops = 0
    for L, m in zip(_context(case), nodes):
        w, sinks = case["window"] or L + m, case["sinks"]
        context = min(L, w - 1) + min(sinks, max(0, L - w + 1))
        # a node's path is the logarithm of its number long
        size += (context + m) * row * 4 + m * (2 * wide * d + 4)
        flops += m * (context + math.log2(m + 1)) * 4 * d
    return {"bytes": size, "flops": flops}


# ---- the same in 64 bits ---------------------------------------------------------------

def exact(case, seed):
    """Attention by its definition, node by node: the list of the positions it
    sees, a weight each.  Tokens by the definition too, row by row; rows that
    move are themselves, and whole numbers that are compared have no such value."""
    if case["op"] == "accept":
        return None
    r = _inputs(case, seed)
    if case["op"] == "keep":
        return [*_exact_moves(case, r), None, None, None]
    if case["op"] == "sample":
        return _exact_tokens(case, r)
    page, w, sinks = case["page"], case["window"], case["sinks"]
    G, KV, D = case["heads"] // case["kv_heads"], case["kv_heads"], case["dim"]
    out = torch.zeros(r["q"].shape, dtype=torch.float64, device="cuda")
    up, first = r["parents"].tolist(), 0
    for b, (m, total) in enumerate(zip(r["nodes"], r["total"])):
        L = total - m
        ids = r["table"][b, :-(-total // page)].long()
        K, V = (r[x][0, ids].double().transpose(0, 1).reshape(KV, -1, D)[:, :total]
                for x in ("keys", "values"))
        for t in range(m):
            line, a = [], t
            while a != NONE:
                line.append(a)
                a = up[first + a]
            depth = len(line) - 1
            # the k-th of the line, from the node up, stands k positions before it
            near = [L + a for k, a in enumerate(line) if not w or k < w or L + depth - k < sinks]
            low = max(0, L + depth - w + 1) if w else 0
            pos = list(range(min(sinks, low, L))) + list(range(low, L)) + near
            pos = torch.tensor(pos, device="cuda")
            q = r["q"][first + t].double().view(KV, G, D)
            x = torch.matmul(q, K[:, pos].transpose(1, 2).contiguous()) / math.sqrt(D)
            e = (x - x.amax(2, keepdim=True)).exp()
            o = torch.matmul(e / e.sum(2, keepdim=True), V[:, pos].contiguous())
            out[first + t] = o.reshape(KV * G, D)
        first += m
    return out


def _exact_moves(case, r):
    """The caches after a keep, from lists of where each row goes."""
    page, table = case["page"], r["table"].tolist()
    moves = []
    for b, (m, total) in enumerate(zip(r["nodes"], r["total"])):
        for c, t in enumerate(r["path"][b].tolist()):
            if t != NONE:
                moves.append([x for pos in (total - m + t, total - m + c)
                              for x in (table[b][pos // page], pos % page)])
    a, i, b, j = torch.tensor(moves, device="cuda").t()
    keys, values = r["keys"].double(), r["values"].double()
    for x in (keys, values):
        x[:, b, :, j] = x[:, a, :, i]
    return keys, values


def _exact_tokens(case, r):
    """No sorting: each rule's border is searched for among the logits' own
    values, and ties are counted from the lowest index."""
    if case["R"] * case["V"] > 1 << 23:
        return None
    tokens, chance = [], []
    cols = {n: r[n].tolist() for n in ("T", "k", "p", "m", "u")}
    for i in range(case["R"]):
        T, k, p, m, u = (cols[n][i] for n in ("T", "k", "p", "m", "u"))
        x = r["x"][i].double()
        if T <= 0:
            tokens.append(int((x == x.max()).nonzero()[0]))
            chance.append(0.0)
            continue
        # the distinct values from the largest down, and how often each is there
        value, often = x.unique(return_counts=True)
        value, often = value.flip(0), often.flip(0).double()
        w = ((value - value[0]) / T).exp()
        if k:
            often = torch.minimum(often, (k - (often.cumsum(0) - often)).clamp_min(0))
        mass = (often * w).cumsum(0)
        if p < 1:
            # of each value as many as still start below the border
            need = ((p * mass[-1] - (mass - often * w)) / w).ceil().clamp_min(0)
            often = torch.minimum(often, need)
        often = torch.where(w >= m, often, 0.0)
        often[0] = often[0].clamp_min(1)
        mass = (often * w).cumsum(0)
        target = u * mass[-1]
        j = min(int((mass <= target).sum()), len(w) - 1)
        nth = int(((target - (mass[j] - often[j] * w[j])) / w[j]).floor().clamp_min(0))
        tokens.append(int((x == value[j]).nonzero()[min(nth, int(often[j]) - 1)]))
        chance.append(float((w[j] / mass[-1]).log()))
    return [torch.tensor(tokens, dtype=torch.int32, device="cuda"),
            torch.tensor(chance, dtype=torch.float64, device="cuda")]
