"""The operators of sequences that share a cache, as they are timed: each case is one pass
through one of them, from what a serving program has in hand before the call.

  prefix   ``prefix.prepare_prefix_decode``: decode attention of groups of sequences whose
           first pages are the same ones (beams of a prompt, requests under one system
           prompt), those read once for the whole group;
  select   ``beams.beam_select``: the n best continuations of a request's beams over the
           vocabulary, from the step's logits;
  reorder  ``beams.beam_tables``: the beams' block tables after that choice, with the rows of
           part-filled pages that several beams go on from copied, in every layer's pool.

``run`` makes those calls where ``own`` is set; otherwise it computes the same in elementary
torch operations, in 32 bits (the selection in 64: its order is of unrounded sums).
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
Q_STD = 1.5                      # logits of standard deviation ~1.5 under 1 / sqrt(D)
LARGEST_FLOPS = 33 * 10 ** 9               # prefix: operations
LARGEST_READ = 22 * 10 ** 7                # prefix: bytes
LARGEST_LOGITS = 64 * 4 * 131072 * 2       # select: bytes of logits
LARGEST_POOLS = 40 * 600 * 16 * 8 * 128    # reorder: layers x slots x page x KV heads x head dim
LARGEST_MOVED = 2 * 10 ** 8                # reorder: bytes


def _log(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def _pages(t, page):
    return -(-t // page)


# A prefix case's groups, [(shared pages, [tokens behind them, ...]), ...], from the case's own
# `spread` (a request mix that stays the same from pass to pass).
def _groups(c):
    r = random.Random(c["spread"])
    return [(_log(r, c["shared_lo"] + 1, c["shared_hi"] + 1) - 1,
             [_log(r, c["own_lo"] + 1, c["own_hi"] + 1) - 1
              for _ in range(r.randint(c["n_lo"], c["n_hi"]))])
            for _ in range(c["groups"])]


# A reorder case's requests: (shared pages, tokens of each beam, parent of each beam).
def _requests(c):
    r = random.Random(c["spread"])
    K, P, out = c["K"], c["page"], []
    for _ in range(c["B"]):
        # the better a beam, the more of the next step's go on from it
        parents = [min(K - 1, int(r.expovariate(3.0 / K))) for _ in range(K)]
        shared = r.randint(c["shared_lo"], c["shared_hi"])
        out.append((shared, shared * P + r.randint(1, c["own_pages"] * P), parents))
    return out


def listed():
    return [
        # four beams over a short prompt of a small model: launches and latency
        {"name": "prefix-beams-2k", "kind": "prefix", "groups": 1, "n_lo": 4, "n_hi": 4,
         "shared_lo": 128, "shared_hi": 128, "own_lo": 40, "own_hi": 40, "Hq": 16, "Hkv": 8,
         "D": 128, "S": 1, "page": 16, "dtype": "f16", "spread": 1, "cap": 0.0, "window": 0},
        # chats under one system prompt
        {"name": "prefix-chats-8k", "kind": "prefix", "groups": 1, "n_lo": 24, "n_hi": 24,
         "shared_lo": 512, "shared_hi": 512, "own_lo": 20, "own_hi": 1500, "Hq": 32, "Hkv": 8,
         "D": 128, "S": 1, "page": 16, "dtype": "bf16", "spread": 2, "cap": 0.0, "window": 0},
        # beam search of 16 requests at once, each over its own prompt
        {"name": "prefix-beams-16x4", "kind": "prefix", "groups": 16, "n_lo": 4, "n_hi": 4,
         "shared_lo": 30, "shared_hi": 250, "own_lo": 16, "own_hi": 160, "Hq": 40, "Hkv": 8,
         "D": 128, "S": 1, "page": 16, "dtype": "bf16", "spread": 3, "cap": 0.0, "window": 0},
        # wide heads, soft-capped, each token seeing the last 4,096; four draft tokens at once
        {"name": "prefix-d256-window", "kind": "prefix", "groups": 3, "n_lo": 2, "n_hi": 6,
         "shared_lo": 16, "shared_hi": 90, "own_lo": 4, "own_hi": 700, "Hq": 16, "Hkv": 8,
         "D": 256, "S": 4, "page": 64, "dtype": "bf16", "spread": 4, "cap": 50.0, "window": 4096},
        # small heads, an odd head group, ragged groups; one of them may be alone
        {"name": "prefix-d64-ragged", "kind": "prefix", "groups": 9, "n_lo": 1, "n_hi": 9,
         "shared_lo": 0, "shared_hi": 120, "own_lo": 1, "own_hi": 900, "Hq": 14, "Hkv": 2,
         "D": 64, "S": 1, "page": 32, "dtype": "f16", "spread": 5, "cap": 0.0, "window": 0},
        # the largest: 64 questions about one document of 32 k tokens
        {"name": "prefix-32k-x64", "kind": "prefix", "groups": 1, "n_lo": 64, "n_hi": 64,
         "shared_lo": 2048, "shared_hi": 2048, "own_lo": 30, "own_hi": 1400, "Hq": 32, "Hkv": 8,
         "D": 128, "S": 1, "page": 16, "dtype": "bf16", "spread": 6, "cap": 0.0, "window": 0},
        # one request's four beams over a small vocabulary: latency
        {"name": "select-1x4", "kind": "select", "B": 1, "K": 4, "V": 32000, "n": 8,
         "dtype": "bf16", "first": False, "banned": 0.0},
        # the first step of eight requests (one beam each counts), an odd vocabulary, half banned
        {"name": "select-first-8x5", "kind": "select", "B": 8, "K": 5, "V": 100003, "n": 10,
         "dtype": "f16", "first": True, "banned": 0.5},
        # wide beams, 32-bit logits
        {"name": "select-4x16-f32", "kind": "select", "B": 4, "K": 16, "V": 131072, "n": 32,
         "dtype": "f32", "first": False, "banned": 0.0},
        # the largest: a full batch
        {"name": "select-64x4", "kind": "select", "B": 64, "K": 4, "V": 131072, "n": 8,
         "dtype": "bf16", "first": False, "banned": 0.0},
        # one request's four beams, 28 layers
        {"name": "reorder-1x4", "kind": "reorder", "B": 1, "K": 4, "page": 16, "layers": 28,
         "Hkv": 8, "D": 128, "dtype": "f16", "own_pages": 3, "shared_lo": 125, "shared_hi": 125,
         "spread": 1},
        # a batch of wide beams, 40 layers
        {"name": "reorder-16x8", "kind": "reorder", "B": 16, "K": 8, "page": 16, "layers": 40,
         "Hkv": 8, "D": 128, "dtype": "bf16", "own_pages": 5, "shared_lo": 4, "shared_hi": 30,
         "spread": 2},
    ]


# More of the same ranges: every head dim, type, page size, odd lengths and head groups.
def draw(rng):
    kind = rng.choice(["prefix", "prefix", "prefix", "select", "select", "reorder"])
    c = {"kind": kind}
    if kind == "select":
        c["dtype"] = rng.choice(["bf16", "bf16", "f16", "f32"])
        c["V"] = _log(rng, 100, 131072)
        c["K"] = _log(rng, 1, 32)
        most = LARGEST_LOGITS // (4 if c["dtype"] == "f32" else 2) // (c["K"] * c["V"])
        c["B"] = _log(rng, 1, max(1, min(256, most)))
        c["n"] = min(64, rng.choice([1, 2]) * c["K"])
        c["first"] = rng.random() < 0.25
        c["banned"] = rng.choice([0.0, 0.0, 0.5])
        return c
    c["spread"] = rng.randrange(1 << 20)
    D = c["D"] = rng.choice([64, 128, 256])
    P = c["page"] = rng.choice([16, 32, 64, 128, 256])
    Hkv = c["Hkv"] = rng.choice([1, 2, 4, 5, 8, 16])
    if kind == "reorder":
        c["dtype"] = rng.choice(["bf16", "f16", "f32"])
        c["K"] = _log(rng, 1, 32)
        c["layers"] = _log(rng, 1, 40)
        c["own_pages"] = rng.randint(1, 5)
        c["shared_lo"], c["shared_hi"] = 0, _log(rng, 1, 40)
        room = LARGEST_POOLS // (c["layers"] * P * Hkv * D) // (2 if c["dtype"] == "f32" else 1)
        while c["K"] * c["own_pages"] + c["shared_hi"] > room and c["K"] * c["shared_hi"] > 1:
            c["K"], c["shared_hi"] = max(1, c["K"] // 2), max(1, c["shared_hi"] // 2)
            c["own_pages"] = max(1, c["own_pages"] - 1)
        c["B"] = _log(rng, 1, max(1, min(64, room // (c["K"] * c["own_pages"] + c["shared_hi"]))))
        while work(c)["bytes"] > LARGEST_MOVED:
            c["layers"] = c["layers"] * 2 // 3
        return c
    c["dtype"] = rng.choice(["bf16", "bf16", "f16"])
    c["Hq"] = Hkv * rng.choice([1, 2, 4, 5, 7, 8])
    c["S"] = rng.choice([1, 1, 1, 2, 4])
    c["cap"] = 50.0 if rng.random() < 0.2 else 0.0
    c["window"] = rng.choice([0, 0, 0, 1024])
    c["groups"] = _log(rng, 1, 24)
    c["n_lo"], c["n_hi"] = 1, _log(rng, 1, 64)
    c["shared_lo"], c["shared_hi"] = 0, _log(rng, 1, 32768 // P)
    c["own_lo"], c["own_hi"] = c["S"], _log(rng, c["S"] + 8, 1500)
    for _ in range(40):
        w = work(dict(c, window=0))
        if w["flops"] <= LARGEST_FLOPS and w["bytes"] <= LARGEST_READ:
            break
        c["shared_hi"] = max(1, c["shared_hi"] * 2 // 3)
        c["groups"] = max(1, c["groups"] * 3 // 4)
        c["n_hi"] = max(1, c["n_hi"] * 3 // 4)
    return c


# ---- inputs --------------------------------------------------------------------------
def _randn(seed, shape, dtype, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _prefix_inputs(c, seed):
    P, dt, groups = c["page"], DTYPES[c["dtype"]], _groups(c)
    R = sum(len(n) for _, n in groups)
    owned = [_pages(t, P) for _, n in groups for t in n]
    shared = [s for s, n in groups for _ in n]
    n_slots = sum(s for s, _ in groups) + sum(owned) + 3
    perm = torch.randperm(n_slots, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.zeros((R, max(1, max(a + b for a, b in zip(shared, owned)))), dtype=torch.int32)
    at, r, starts = 0, 0, [0]
    for s, n in groups:
        table[r:r + len(n), :s] = perm[at:at + s]
        at += s
        for i in range(r, r + len(n)):
            table[i, s:s + owned[i]] = perm[at:at + owned[i]]
            at += owned[i]
        r += len(n)
        starts.append(r)
    lens = [s * P + t for s, n in groups for t in n]
    i32 = dict(dtype=torch.int32, device="cuda")
    return {"q": _randn(seed, (R, c["Hq"], c["S"], c["D"]), dt, Q_STD),
            "arena": _randn(seed + 1, (n_slots, 2, c["Hkv"], P, c["D"]), dt),
            "table": table.cuda(), "lens": lens, "len_t": torch.tensor(lens, **i32),
            "starts": starts, "start_t": torch.tensor(starts, **i32),
            "shared": [s for s, _ in groups],
            "shared_t": torch.tensor([s for s, _ in groups], **i32)}


def _select_inputs(c, seed):
    dt, shape = DTYPES[c["dtype"]], (c["B"], c["K"], c["V"])
    x = _randn(seed, shape, torch.float32, 2.5)
    if c["banned"]:
        g = torch.Generator(device="cuda").manual_seed(seed + 1)
        x.masked_fill_(torch.rand(c["V"], generator=g, device="cuda") < c["banned"], -math.inf)
    scores = -20 * torch.rand(shape[:2], generator=torch.Generator().manual_seed(seed + 2))
    if c["first"]:
        scores = torch.full(shape[:2], -math.inf)
        scores[:, 0] = 0.0
    return {"logits": x.to(dt), "scores": scores.sort(-1, descending=True).values.cuda()}


def _reorder_inputs(c, seed):
    B, K, P, reqs = c["B"], c["K"], c["page"], _requests(c)
    g = torch.Generator().manual_seed(seed)
    cols = [_pages(t, P) for _, t, _ in reqs]
    n_slots = sum(s + K * (n - s) for (s, _, _), n in zip(reqs, cols)) + 1
    perm = torch.randperm(n_slots, generator=g).to(torch.int32)
    table = torch.zeros((B * K, max(cols)), dtype=torch.int32)
    parents, at = [], 0
    for b, ((s, t, par), n) in enumerate(zip(reqs, cols)):
        rows = table[b * K:(b + 1) * K]
        rows[:, :s] = perm[at:at + s]
        at += s
        rows[:, s:n] = perm[at:at + K * (n - s)].reshape(K, n - s)
        at += K * (n - s)
        # the mix is the case's; the seed moves the beams about
        move = torch.randperm(K, generator=g)
        parents.append(move[torch.tensor(par)[torch.randperm(K, generator=g)]])
    i32 = dict(dtype=torch.int32, device="cuda")
    pools = _randn(seed, (c["layers"], n_slots, 2, c["Hkv"], P, c["D"]), DTYPES[c["dtype"]])
    return {"parents": torch.stack(parents).to(torch.int32).cuda(), "table": table.cuda(),
            "lens": torch.tensor([t for _, t, _ in reqs], **i32).repeat_interleave(K),
            "shared": torch.tensor([s for s, _, _ in reqs], **i32), "pools": pools,
            "new_table": torch.zeros_like(table, device="cuda"),
            "copies": torch.zeros((B * K, 2), **i32), "count": torch.zeros(1, **i32),
            "released": torch.full((table.numel(),), -1, **i32)}


def prepare(case, seed):
    c = case
    make = {"prefix": _prefix_inputs, "select": _select_inputs, "reorder": _reorder_inputs}
    st = {"c": c, **make[c["kind"]](c, seed)}
    if own and c["kind"] == "prefix":
        from helm_amd import prefix
        st["step"] = prefix.prepare_prefix_decode(
            st["q"], st["arena"][:, 0], st["arena"][:, 1], st["table"], st["len_t"], st["start_t"],
            st["shared_t"], softcap=c["cap"] or None, window=c["window"] or None)
    if own and c["kind"] == "reorder":
        from helm_amd import beams
        st["store"] = beams.PageStore(list(st["pools"].unbind(0)))
        st["out"] = beams.BeamTables(st["new_table"], st["copies"], st["released"], st["count"])
    return st


# ---- the plain forms ------------------------------------------------------------------
def _scores(q, k, c):
    x = torch.matmul(q, k.transpose(-1, -2).contiguous()) * (1.0 / math.sqrt(c["D"]))
    return torch.tanh(x / c["cap"]) * c["cap"] if c["cap"] else x


def _plain_prefix(st):
    """Group by group: its shared tokens under all of its rows at once, then each sequence's own,
    padded to the group's longest."""
    c, out = st["c"], torch.empty_like(st["q"])
    G, S, P, Hkv, D, dev = c["Hq"] // c["Hkv"], c["S"], c["page"], c["Hkv"], c["D"], out.device
    for a, e, s in zip(st["starts"], st["starts"][1:], st["shared"]):
        n, lens = e - a, st["len_t"][a:e].long()
        # [n, Hkv, G S, D], a row's position and the tokens that it sees
        q = st["q"][a:e].float().unflatten(1, (Hkv, G)).flatten(2, 3)
        p = (lens[:, None] - S + torch.arange(S, device=dev)).repeat(1, G)
        w = max(1, max(_pages(t, P) for t in st["lens"][a:e]) - s)
        own_t = torch.arange(w * P, device=dev) + s * P
        col = (own_t[::P] // P).clamp(max=st["table"].size(1) - 1)
        kv = st["arena"][st["table"][a:e][:, col].long()].float()      # [n, w, 2, Hkv, P, D]
        kv = kv.permute(2, 0, 3, 1, 4, 5).flatten(3, 4)                # [2, n, Hkv, w P, D]
        x = _scores(q, kv[0], c)
        hide = own_t > p[..., None]
        hide |= (own_t <= p[..., None] - c["window"]) if c["window"] else False
        x = x.masked_fill(hide[:, None], -math.inf)
        if s:
            pre = st["arena"][st["table"][a, :s].long()].float()
            pre = pre.permute(1, 2, 0, 3, 4).flatten(2, 3)             # [2, Hkv, s P, D]
            t = torch.arange(s * P, device=dev)
            y = _scores(q.transpose(0, 1).flatten(1, 2), pre[0], c)
            y = y.unflatten(1, (n, G * S)).transpose(0, 1)
            hide = t > p[..., None]
            hide |= (t <= p[..., None] - c["window"]) if c["window"] else False
            x = torch.cat([y.masked_fill(hide[:, None], -math.inf), x], -1)
        m = x.amax(-1, keepdim=True)
        x = torch.exp(x - torch.where(torch.isinf(m), torch.zeros_like(m), m))
        total = x.sum(-1, keepdim=True)
        x = x / torch.where(total > 0, total, torch.ones_like(total))
        o = torch.matmul(x[..., s * P:], torch.where(_past_end(own_t, lens), 0.0, kv[1]))
        if s:
            y = x[..., :s * P].transpose(0, 1).flatten(1, 2)
            o = o + torch.matmul(y, pre[1]).unflatten(1, (n, G * S)).transpose(0, 1)
        out[a:e] = o.unflatten(2, (G, S)).flatten(1, 2).to(out.dtype)
    return out


def _past_end(t, lens):
    """[n, 1, T, 1]: tokens past a sequence's end, whose rows hold anything."""
    return (t >= lens[:, None])[:, None, :, None]


def _plain_select(st):
    c, x, scores = st["c"], st["logits"].double(), st["scores"].double()
    x = (x - torch.logsumexp(x, -1, keepdim=True) + scores[..., None]).flatten(1)
    at = torch.arange(x.size(1), device=x.device)
    best, which = [], []
    for _ in range(c["n"]):
        m = x.amax(-1, keepdim=True)
        i = torch.where(x == m, at, x.size(1)).amin(-1, keepdim=True)   # ties: the lowest
        best.append(m)
        which.append(i)
        x.scatter_(1, i, -math.inf)
    best, which = torch.cat(best, 1), torch.cat(which, 1)
    none = best == -math.inf
    return [best.float(), torch.where(none, -1, which % c["V"]),
            torch.where(none, -1, which // c["V"]).int()]


def _plain_reorder(st):
    c, P = st["c"], st["c"]["page"]
    B, K, W, dev = c["B"], c["K"], st["table"].size(1), st["table"].device
    old, par = st["table"].view(B, K, W), st["parents"].long()
    j = torch.arange(K, device=dev)
    par = torch.where((par >= 0) & (par < K), par, j)
    child = par[:, None, :] == j[None, :, None]                      # [b, parent, child]
    has = child.any(-1)
    keeper = torch.where(child.diagonal(dim1=1, dim2=2), j, child.int().argmax(-1))
    extra = keeper.gather(1, par) != j
    # the e-th row that keeps no page takes that of the e-th row without a child
    rank_e, rank_d = extra.cumsum(1), (~has).cumsum(1)
    pair = (rank_e[:, :, None] == rank_d[:, None, :]) & extra[:, :, None] & (~has)[:, None, :]
    spare = pair.int().argmax(-1)
    lens = st["lens"].view(B, K)[:, :1].long()
    full, col = lens // P, torch.arange(W, device=dev)
    new = old.gather(1, par[..., None].expand(B, K, W))
    tail = old.gather(1, torch.where(extra, spare, par)[..., None].expand(B, K, W))
    part = lens % P != 0
    new = torch.where((col == full)[:, None] & part[:, None], tail, new)
    new = torch.where((col >= full + part)[:, None], old, new)
    st["new_table"].copy_(new.view(B * K, W))
    # the pages copied, (from, to) of each row, and their tokens in every layer
    at = full.clamp(max=W - 1)[:, None].expand(B, K, 1)
    src = old.gather(2, at)[..., 0].gather(1, par)
    dst = new.gather(2, at)[..., 0]
    moved = extra & part
    both = torch.where(moved[..., None], torch.stack([src, dst], -1), -1)
    st["copies"].copy_(both.view(B * K, 2))
    s, d = src[moved].long(), dst[moved].long()
    n = (lens % P).expand(B, K)[moved]
    keep = (torch.arange(P, device=dev) < n[:, None])[None, :, None, None, :, None]
    st["pools"][:, d] = torch.where(keep, st["pools"][:, s], st["pools"][:, d])
    # full pages behind the shared ones that no row holds any more, the first row's naming of each
    held = (old[:, :, None] == new[:, None]).any(2)
    twice = ((old[:, :, None] == old[:, None]) & (j[:, None] > j)[None, :, :, None]).any(2)
    gone = ~held & ~twice & (col >= st["shared"][:, None])[:, None] & (col < full)[:, None]
    gone = old.transpose(1, 2)[gone.transpose(1, 2)]                 # by request, column, row
    st["released"][:gone.numel()] = gone
    st["count"].fill_(gone.numel())
    return _reordered(st)


def _reordered(st):
    return [st["new_table"], st["copies"], st["released"], st["count"], st["pools"]]


def run(state):
    st, kind = state, state["c"]["kind"]
    if not own:
        plain = {"prefix": _plain_prefix, "select": _plain_select, "reorder": _plain_reorder}
        return plain[kind](st)
    if kind == "prefix":
        return st["step"].run()
    from helm_amd import beams
    if kind == "select":
        return list(beams.beam_select(st["logits"], st["scores"], n=st["c"]["n"]))
    beams.beam_tables(st["parents"], st["table"], st["lens"], st["c"]["page"],
                      shared_pages=st["shared"], pages=st["store"], out=st["out"])
    return _reordered(st)


# ---- what a pass cannot do without ----------------------------------------------------
def work(case):
    c = case
    es = 4 if c["dtype"] == "f32" else 2
    if c["kind"] == "select":
        R = c["B"] * c["K"]           # the logits once; a difference, an exponential, a sum each
        return {"bytes": R * c["V"] * es + 4 * R + 16 * c["B"] * c["n"], "flops": 3 * R * c["V"]}
    P, row = c["page"], c["Hkv"] * c["D"]
    if c["kind"] == "reorder":
        moved = cells = 0
        for s, t, parents in _requests(c):
            moved += (t % P) * (c["K"] - len(set(parents)))
            cells += c["K"] * (_pages(t, P) - s)
        # a copied token's K and V in and out, in every layer; the tables' own columns in and out
        return {"bytes": 2 * moved * 2 * row * es * c["layers"] + 8 * cells + 12 * c["B"] * c["K"],
                "flops": cells}
    G, S, w = c["Hq"] // c["Hkv"], c["S"], c["window"]
    seen = pairs = R = pages = 0
    for s, n in _groups(c):
        T = s * P
        first = [max(0, T + t - S + 1 - w) if w else 0 for t in n]     # a sequence's first seen
        seen += max(0, T - min(first)) + sum(t - max(0, f - T) for f, t in zip(first, n))
        pairs += sum(min(w or T + t, T + t - S + 1 + i) for t in n for i in range(S))
        R += len(n)
        pages += s + sum(_pages(t, P) for t in n)
    return {"bytes": 2 * seen * row * es + 2 * R * S * c["Hq"] * c["D"] * es + 4 * pages + 4 * R,
            "flops": 4 * pairs * c["Hq"] * c["D"]}


# ---- the same results in 64 bits ------------------------------------------------------
def exact(case, seed):
    c = case
    if c["kind"] == "reorder":
        return None          # whole numbers and copies: the plain form's are the definition's
    if c["kind"] == "select":
        x = _select_inputs(c, seed)
        p = torch.log(torch.softmax(x["logits"].double(), -1)) + x["scores"].double()[..., None]
        p = p.flatten(1)
        n = min(c["n"], p.size(1))
        best = torch.full((c["B"], c["n"]), -math.inf, dtype=torch.float64, device="cuda")
        best[:, :n] = torch.topk(p, n, -1).values
        return [best, None, None]
    x = _prefix_inputs(c, seed)
    P, S, G = c["page"], c["S"], c["Hq"] // c["Hkv"]
    outs = []
    for r, t in enumerate(x["lens"]):                 # each sequence by itself, head by head
        kv = x["arena"][x["table"][r, :_pages(t, P)].long()]
        pos = t - S + torch.arange(S, device="cuda")[:, None]
        j = torch.arange(t, device="cuda")[None, :]
        hidden = (j > pos) | (j <= pos - c["window"]) if c["window"] else j > pos
        heads = []
        for h in range(c["Hkv"]):
            k = kv[:, 0, h].flatten(0, 1)[:t].double()
            v = kv[:, 1, h].flatten(0, 1)[:t].double()
            q = x["q"][r, h * G:(h + 1) * G].double()
            z = torch.matmul(q, k.t().contiguous()) / math.sqrt(c["D"])
            if c["cap"]:
                z = c["cap"] * torch.tanh(z / c["cap"])
            z = torch.softmax(z.masked_fill(hidden, -math.inf), -1)
            heads.append(torch.matmul(z, v))
        outs.append(torch.cat(heads))
    return torch.stack(outs)
