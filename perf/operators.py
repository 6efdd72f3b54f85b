"""The serving operators over a pool of 4-bit pages, as they are timed: each case is one
pass through one of them, from what a serving program has in hand before the call.

  tables   ``paged.batch_tables``: a step's request lengths into block tables, slots,
           positions and offsets, on the GPU;
  write    ``pool4.Pool4.write`` and ``.read``: a step's K and V rows into 4-bit pages and
           the values they stand for back out (what a prompt over a cached prefix takes);
  attn4    ``pool4.prepare_pool4_decode``: attention of the newest tokens over the pages;
  prompt   ``prompt.prompt_attention``: causal attention over packed whole prompts.

``run`` makes those calls where ``own`` is set; otherwise it computes the same in elementary
torch operations in 32 bits.  A 4-bit page holds E2M1 codes (0, .5, 1, 1.5, 2, 3, 4, 6 and
their negatives) in groups of 32 dimensions under one power of two: the smallest 2^e,
-125 <= e <= 125, that brings the group's largest magnitude to 7 or less, each value
rounded to the nearest code, ties to the even one, above 6 to 6.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
Q_STD = 1.5                      # logits of standard deviation ~1.5 under 1 / sqrt(D)
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
LARGEST_CACHED = 4 * 65536 * 8 * 128        # attn4: cached tokens x KV heads x head dim
LARGEST_WRITTEN = 16384 * 8 * 128           # write: tokens x KV heads x head dim
LARGEST_PAIRS = 16384 * 16385 // 2 * 32 * 128   # prompt: visible pairs x heads x head dim
LARGEST_TOKENS = 65536                      # tables: new tokens of a step


# Lengths of a case's B sequences: `lo` to `hi`, spread over their logarithm, from the
# case's own `spread` (a request mix that stays the same from pass to pass).
def _lens(c, lo="lo", hi="hi"):
    r = random.Random(c["spread"])
    lo, hi = c[lo], c[hi]
    return [min(hi, max(lo, int(math.exp(r.uniform(math.log(lo + 1), math.log(hi + 2)))) - 1))
            for _ in range(c["B"])]


def listed():
    return [
        # a full decode batch at mixed depths: one token each
        {"name": "tables-step-256", "kind": "tables", "B": 256, "page": 16, "spread": 2,
         "cached_lo": 16, "cached_hi": 32768, "lo": 1, "hi": 1},
        # 48 prompts and prompt chunks entering together, ~50 k tokens
        {"name": "tables-prompts-48", "kind": "tables", "B": 48, "page": 64, "spread": 3,
         "cached_lo": 0, "cached_hi": 4096, "lo": 64, "hi": 8192},
        # the step's tokens of 8 sequences: latency
        {"name": "write-step-8", "kind": "write", "N": 8, "Hkv": 8, "D": 128, "page": 16,
         "dtype": "bf16"},
        # a large prompt batch of one layer
        {"name": "write-prompt-16k", "kind": "write", "N": 16384, "Hkv": 8, "D": 128, "page": 16,
         "dtype": "bf16"},
        # a short context of a small model: launch and latency
        {"name": "attn4-2k", "kind": "attn4", "B": 1, "lo": 2048, "hi": 2048, "Hq": 16, "Hkv": 8,
         "D": 128, "S": 1, "page": 16, "dtype": "f16", "spread": 1, "cap": 0.0, "mask": "none"},
        # the long single-request decode
        {"name": "attn4-32k", "kind": "attn4", "B": 1, "lo": 32768, "hi": 32768, "Hq": 32,
         "Hkv": 8, "D": 128, "S": 1, "page": 16, "dtype": "bf16", "spread": 1, "cap": 0.0,
         "mask": "none"},
        # wide heads, soft-capped, under a sliding-window mask; four draft tokens at once
        {"name": "attn4-d256-window", "kind": "attn4", "B": 3, "lo": 4000, "hi": 8000, "Hq": 16,
         "Hkv": 8, "D": 256, "S": 4, "page": 64, "dtype": "bf16", "spread": 5, "cap": 50.0,
         "mask": "window"},
        # the largest: four sequences of 64 k tokens
        {"name": "attn4-64k-b4", "kind": "attn4", "B": 4, "lo": 65536, "hi": 65536, "Hq": 40,
         "Hkv": 8, "D": 128, "S": 1, "page": 16, "dtype": "bf16", "spread": 1, "cap": 0.0,
         "mask": "none"},
        # short ragged prompts of a small model at head dim 64
        {"name": "prompt-short-d64", "kind": "prompt", "B": 7, "lo": 1, "hi": 300, "Hq": 14,
         "Hkv": 2, "D": 64, "dtype": "f16", "spread": 3, "cap": 0.0, "window": 0},
        # a batch of ragged prompts of a grouped-head model
        {"name": "prompt-ragged", "kind": "prompt", "B": 9, "lo": 200, "hi": 2500, "Hq": 40,
         "Hkv": 8, "D": 128, "dtype": "bf16", "spread": 4, "cap": 0.0, "window": 0},
        # wide heads, soft-capped, each token seeing the last 1,024
        {"name": "prompt-d256-window", "kind": "prompt", "B": 4, "lo": 700, "hi": 4700, "Hq": 16,
         "Hkv": 8, "D": 256, "dtype": "bf16", "spread": 2, "cap": 50.0, "window": 1024},
        # one long prompt: the largest
        {"name": "prompt-16k", "kind": "prompt", "B": 1, "lo": 16384, "hi": 16384, "Hq": 32,
         "Hkv": 8, "D": 128, "dtype": "bf16", "spread": 1, "cap": 0.0, "window": 0},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


# More of the same ranges: every head dim, type, page size, odd lengths and head groups.
def draw(rng):
    kind = rng.choice(["tables", "write", "attn4", "attn4", "prompt", "prompt"])
    c = {"kind": kind, "spread": rng.randrange(1 << 20)}
    if kind == "tables":
        c["page"] = rng.choice([16, 32, 64, 128, 256])
        c["B"] = _log(rng, 1, 1024)
        step = rng.random() < 0.5
        c["lo"] = 1 if step else rng.choice([0, 1, 16])
        c["hi"] = 1 if step else _log(rng, 2, max(2, min(8192, LARGEST_TOKENS // c["B"])))
        c["cached_lo"], c["cached_hi"] = rng.choice([0, 1, 100]), _log(rng, 128, 32768)
        return c
    D = c["D"] = rng.choice([64, 128, 256])
    Hkv = c["Hkv"] = rng.choice([1, 2, 4, 5, 8, 16])
    if kind == "write":
        del c["spread"]
        c["page"] = rng.choice([16, 32, 64, 128, 256])
        c["N"] = _log(rng, 1, LARGEST_WRITTEN // (Hkv * D))
        c["dtype"] = rng.choice(["bf16", "f16", "f32"])
        return c
    c["dtype"] = rng.choice(["bf16", "bf16", "f16"])
    G = rng.choice([1, 2, 4, 5, 7, 8])
    c["Hq"] = Hkv * G
    c["cap"] = 50.0 if rng.random() < 0.2 else 0.0
    c["B"] = _log(rng, 1, 16)
    if kind == "attn4":
        c["page"] = rng.choice([16, 32, 64, 128, 256])
        c["S"] = rng.choice([1, 1, 1, 2, 4, 7])
        c["mask"] = rng.choice(["none", "none", "none", "window"])
        c["hi"] = _log(rng, 64, min(65536, LARGEST_CACHED // (c["B"] * Hkv * D)))
        c["lo"] = max(c["S"], rng.choice([c["S"], c["hi"] // 3, c["hi"]]))
    else:
        c["hi"] = _log(rng, 32, 8192)
        c["lo"] = rng.choice([0, 1, c["hi"] // 2])
        c["window"] = rng.choice([0, 0, 0, 1024])
        while sum(t * (t + 1) // 2 for t in _lens(c)) * c["Hq"] * D > LARGEST_PAIRS:
            c["hi"] = c["hi"] * 2 // 3
            c["lo"] = min(c["lo"], c["hi"])
    return c


# ---- inputs --------------------------------------------------------------------------
def _randn(seed, shape, dtype, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _page_table(seed, pages, width):
    """Each row's pages from one shuffled pool; (table [B, width] int32, slots in all)."""
    g = torch.Generator().manual_seed(seed)
    perm = torch.randperm(max(1, sum(pages)), generator=g).to(torch.int32)
    table = torch.zeros((len(pages), max(1, width)), dtype=torch.int32)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = perm[at:at + n]
        at += n
    return table.cuda(), perm.numel()


def _pages(t, page):
    return -(-t // page)


def _table_inputs(c, seed):
    g = torch.Generator().manual_seed(seed)
    new = _lens(c)
    cached = _lens(c, "cached_lo", "cached_hi")
    P = c["page"]
    # the mix is the case's; the seed moves the requests about
    order = torch.randperm(c["B"], generator=g).tolist()
    new, cached = [new[i] for i in order], [cached[i] for i in order]
    # each request somewhere inside its last page, as steps leave them
    cached = [max(0, t - int(torch.randint(0, P, (1,), generator=g))) if t >= P else t
              for t in cached]
    old = [_pages(t, P) for t in cached]
    need = [_pages(t + n, P) - o for t, n, o in zip(cached, new, old)]
    perm = torch.randperm(sum(old) + sum(need) + 64, generator=g).to(torch.int32)
    table = torch.zeros((c["B"], max(1, max(o + n for o, n in zip(old, need)))),
                        dtype=torch.int32)
    at = 0
    for b, o in enumerate(old):
        table[b, :o] = perm[at:at + o]
        at += o
    return {"new": torch.tensor(new, dtype=torch.int32, device="cuda"),
            "cached": torch.tensor(cached, dtype=torch.int32, device="cuda"),
            "table": table.cuda(), "free": perm[at:].cuda(),
            "tokens": max(1, sum(new)), "page": P}


def _write_inputs(c, seed):
    N, P = c["N"], c["page"]
    n_slots = _pages(N, P) + 3
    g = torch.Generator().manual_seed(seed)
    pages = torch.randperm(n_slots, generator=g)
    first = int(torch.randint(0, P, (1,), generator=g))       # the run starts inside a page
    t = torch.arange(N) + first
    slots = (pages[t // P] * P + t % P).to(torch.int64)
    dt = DTYPES[c["dtype"]]
    # K's channels differ in size, as they do in trained models
    width = torch.exp(0.5 * _randn(seed + 2, (c["Hkv"], c["D"]), torch.float32))
    k = (_randn(seed, (N, c["Hkv"], c["D"]), torch.float32) * width).to(dt)
    return {"k": k, "v": _randn(seed + 1, (N, c["Hkv"], c["D"]), dt), "slots": slots.cuda(),
            "n_slots": n_slots}


def _attn_inputs(c, seed):
    lens, P, D, Hkv, S = _lens(c), c["page"], c["D"], c["Hkv"], c["S"]
    dt = DTYPES[c["dtype"]]
    pages = [_pages(t, P) for t in lens]
    table, n_slots = _page_table(seed, pages, max(pages))
    slots = torch.cat([(table[b, :pages[b]].long()[:, None] * P
                        + torch.arange(P, device="cuda")).reshape(-1)[:t]
                       for b, t in enumerate(lens)])
    n = sum(lens)
    x = {"q": _randn(seed, (c["B"], c["Hq"], S, D), dt, Q_STD),
         "k": _randn(seed + 1, (n, Hkv, D), dt), "v": _randn(seed + 2, (n, Hkv, D), dt),
         "slots": slots, "table": table, "n_slots": n_slots, "lens": lens, "mask": None,
         "len_t": torch.tensor(lens, dtype=torch.int32, device="cuda")}
    if c["mask"] == "window":
        # additive, of the model's type: the last half of the longest context and a left pad
        T = max(lens)
        m = torch.zeros((c["B"], 1, S, T), dtype=dt, device="cuda")
        for b, t in enumerate(lens):
            for s in range(S):
                m[b, 0, s, :max(0, t - S + s + 1 - T // 2)] = torch.finfo(dt).min
        x["mask"] = m
    return x


def _prompt_inputs(c, seed):
    lens = _lens(c)
    g = torch.Generator().manual_seed(seed)
    lens = [lens[i] for i in torch.randperm(c["B"], generator=g).tolist()]
    n, D, dt = max(1, sum(lens)), c["D"], DTYPES[c["dtype"]]
    # q, k and v are slices of one fused projection, as a model's layer hands them over
    qkv = _randn(seed, (n, c["Hq"] + 2 * c["Hkv"], D), torch.float32)
    qkv[:, :c["Hq"]] *= Q_STD
    qkv = qkv.to(dt)
    cu = torch.zeros(c["B"] + 1, dtype=torch.int32)
    cu[1:] = torch.cumsum(torch.tensor(lens), 0)
    return {"qkv": qkv, "q": qkv[:, :c["Hq"]], "k": qkv[:, c["Hq"]:c["Hq"] + c["Hkv"]],
            "v": qkv[:, c["Hq"] + c["Hkv"]:], "cu": cu.cuda(), "lens": lens}


def prepare(case, seed):
    c = case
    if c["kind"] == "tables":
        return {"c": c, **_table_inputs(c, seed)}
    if c["kind"] == "prompt":
        return {"c": c, **_prompt_inputs(c, seed)}
    x = _write_inputs(c, seed) if c["kind"] == "write" else _attn_inputs(c, seed)
    st = {"c": c, **x}
    if own:
        from helm_amd import pool4
        pool = pool4.Pool4(x["n_slots"], c["Hkv"], c["D"], page_size=c["page"], device="cuda")
        st["pool"] = pool
        if c["kind"] == "attn4":
            pool.write(x["k"], x["v"], x["slots"])
            st["step"] = pool4.prepare_pool4_decode(
                x["q"], pool, x["table"], x["len_t"], softcap=c["cap"] or None,
                attention_mask=x["mask"], causal=True)
    else:
        rows = x["n_slots"] * c["page"]
        st["codes"] = torch.zeros((rows, 2, c["Hkv"], c["D"] // 2), dtype=torch.uint8, device="cuda")
        st["exps"] = torch.zeros((rows, 2, c["Hkv"], c["D"] // 32), dtype=torch.uint8,
                                 device="cuda")
        if c["kind"] == "attn4":
            _plain_write(st)
    if c["kind"] == "attn4":
        del st["k"], st["v"]
    return st


# 2^e for whole e, from the number's bits (a device's pow may be a step off).
def _pow2(e):
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _pow2_64(e):
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


# ---- the plain forms ------------------------------------------------------------------
def _plain_codes(x):
    """Codes [..., D] and biased exponents [..., D / 32] of x's groups."""
    g = x.float().unflatten(-1, (-1, 32))
    m, k = torch.frexp(g.abs().amax(-1))           # largest = m 2^k, m in [0.5, 1)
    e = (k - 3 + (m > 0.875).to(k.dtype)).clamp(-125, 125)
    y = g * _pow2(-e)[..., None]
    a = y.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75).to(torch.uint8) + (a > 1.25).to(torch.uint8)
            + (a >= 1.75).to(torch.uint8) + (a > 2.5).to(torch.uint8) + (a >= 3.5).to(torch.uint8)
            + (a > 5.0).to(torch.uint8) + 8 * (y < 0).to(torch.uint8))
    return code.flatten(-2), (e + 127).to(torch.uint8)


def _plain_write(st):
    for i, x in enumerate((st["k"], st["v"])):
        code, e = _plain_codes(x)
        st["codes"][st["slots"], i] = code[..., 0::2] | (code[..., 1::2] << 4)
        st["exps"][st["slots"], i] = e


def _plain_read(st, slots):
    """[n, 2, Hkv, D] in 32 bits: the values of the rows `slots`."""
    p = st["codes"][slots]
    code = torch.stack([p & 15, p >> 4], -1).flatten(-2).long()
    grid = torch.tensor(GRID + tuple(-v for v in GRID), device=p.device)
    val = grid[code].unflatten(-1, (-1, 32))
    return (val * _pow2(st["exps"][slots].int() - 127)[..., None]).flatten(-2)


def _softmax(x):
    m = x.amax(-1, keepdim=True)
    w = torch.exp(x - torch.where(torch.isinf(m), torch.zeros_like(m), m))
    s = w.sum(-1, keepdim=True)
    return w / torch.where(s > 0, s, torch.ones_like(s))


def _plain_rows(q, k, v, scale, cap, hidden, mask=None):
    """q [G, S, D], k and v [T, D], hidden [S, T] (or None), mask [S, T]: [G, S, D]."""
    x = torch.matmul(q, k.t().contiguous()) * scale
    if cap:
        x = torch.tanh(x / cap) * cap
    if mask is not None:
        x = x + mask
    if hidden is not None:
        x = x.masked_fill(hidden, -math.inf)
    return torch.matmul(_softmax(x), v)


def _plain_tables(st):
    new, cached, table, free, P = st["new"].long(), st["cached"].long(), st["table"], st["free"], st["page"]
    B, N, dev = new.numel(), st["tokens"], new.device
    cu = torch.zeros(B + 1, dtype=torch.int64, device=dev)
    cu[1:] = torch.cumsum(new, 0)
    total = cached + new
    old = (cached + P - 1) // P
    need = (total + P - 1) // P - old
    first = torch.cumsum(need, 0) - need
    col = torch.arange(table.size(1), device=dev)[None, :]
    fresh = (col >= old[:, None]) & (col < (old + need)[:, None])
    src = (first[:, None] + col - old[:, None]).clamp(0, free.numel() - 1)
    table.copy_(torch.where(fresh, free[src], table))
    i = torch.arange(N, device=dev)
    b = (i[:, None] >= cu[None, 1:]).sum(1).clamp(max=B - 1)
    live = i < cu[B]
    pos = torch.where(live, cached[b] + i - cu[b], torch.zeros_like(i))
    slot = table[b, torch.where(live, pos // P, torch.zeros_like(pos))].long() * P + pos % P
    slot = torch.where(live, slot, torch.full_like(slot, -1))
    return [cu.int(), pos, slot, total.int(), need.sum().int().reshape(1), table]


def _plain_attn(st):
    c, q = st["c"], st["q"].float()
    G, S, out, at = c["Hq"] // c["Hkv"], c["S"], [], 0
    for b, t in enumerate(st["lens"]):
        kv = _plain_read(st, st["slots"][at:at + t])
        at += t
        pos = torch.arange(t, device=q.device)
        hidden = pos[None, :] > (t - S + torch.arange(S, device=q.device))[:, None] if S > 1 else None
        mask = None if st["mask"] is None else st["mask"][b, 0, :, :t].float()
        out.append(torch.cat([
            _plain_rows(q[b, h * G:(h + 1) * G], kv[:, 0, h].contiguous(), kv[:, 1, h].contiguous(),
                        1.0 / math.sqrt(c["D"]), c["cap"], hidden, mask)
            for h in range(c["Hkv"])]))
    return torch.stack(out).to(st["q"].dtype)


def _prompt_by_rows(c, q, k, v, lens, scale, rows, attend):
    """out [n, Hq, D] in q's type, `rows` query rows of a sequence and one KV head at a time."""
    G, out, at = c["Hq"] // c["Hkv"], torch.zeros_like(q), 0
    for t in lens:
        for r in range(0, t, rows):
            e = min(t, r + rows)
            lo = max(0, r - c["window"] + 1) if c["window"] else 0
            i = torch.arange(r, e, device=q.device)[:, None]
            j = torch.arange(lo, e, device=q.device)[None, :]
            hidden = (j > i) | (j <= i - c["window"]) if c["window"] else j > i
            for h in range(c["Hkv"]):
                o = attend(q[at + r:at + e, h * G:(h + 1) * G].transpose(0, 1).contiguous(),
                           k[at + lo:at + e, h].contiguous(), v[at + lo:at + e, h].contiguous(),
                           scale, c["cap"], hidden)
                out[at + r:at + e, h * G:(h + 1) * G] = o.transpose(0, 1)
        at += t
    return out


def run(state):
    st, c = state, state["c"]
    kind = c["kind"]
    if not own:
        if kind == "tables":
            return _plain_tables(st)
        if kind == "write":
            _plain_write(st)
            kv = _plain_read(st, st["slots"]).to(DTYPES[c["dtype"]])
            return [kv[:, 0], kv[:, 1]]
        if kind == "attn4":
            return _plain_attn(st)
        q, k, v = st["q"].float(), st["k"].float(), st["v"].float()
        return _prompt_by_rows(c, q, k, v, st["lens"], 1.0 / math.sqrt(c["D"]), 4096,
                               _plain_rows).to(st["q"].dtype)
    if kind == "tables":
        from helm_amd import paged
        t = paged.batch_tables(st["new"], st["cached"], st["table"], st["free"], st["page"],
                               max_tokens=st["tokens"])
        return [t.cu_seqlens, t.positions, t.slot_map, t.seq_lens, t.pages_taken, st["table"]]
    if kind == "write":
        st["pool"].write(st["k"], st["v"], st["slots"])
        return list(st["pool"].read(st["slots"], dtype=DTYPES[c["dtype"]]))
    if kind == "attn4":
        return st["step"].run()
    from helm_amd import prompt
    return prompt.prompt_attention(st["q"], st["k"], st["v"], st["cu"], softcap=c["cap"] or None,
                                   window=c["window"] or None)


# ---- what a pass cannot do without ----------------------------------------------------
def work(case):
    c = case
    if c["kind"] == "tables":
        new, cached = _lens(c), _lens(c, "cached_lo", "cached_hi")
        n = sum(new)
        fresh = sum(_pages(t + m, c["page"]) - _pages(t, c["page"]) for t, m in zip(cached, new))
        # lengths in; offsets, totals out; a position and a slot a token; each page
        # taken read and written, each part-filled page's entry read
        return {"bytes": 8 * c["B"] + 8 * c["B"] + 4 + 16 * n + 8 * fresh + 4 * c["B"],
                "flops": 4 * n + 4 * c["B"]}
    es = 4 if c["dtype"] == "f32" else 2
    row = c["Hkv"] * c["D"]
    if c["kind"] == "write":
        n = 2 * c["N"] * row           # K and V values: in, 4 bits and scales out and in, out
        return {"bytes": n * 2 * es + 2 * (n // 2 + n // 32) + 2 * 8 * c["N"], "flops": 6 * n}
    lens = _lens(c)
    if c["kind"] == "attn4":
        S = c["S"]
        T = max(lens)
        low = [max(0, t - S + 1 - T // 2) if c["mask"] == "window" else 0 for t in lens]
        seen = sum(t - lo for t, lo in zip(lens, low))
        pairs = sum(S * (t - lo) for t, lo in zip(lens, low))
        mask = c["B"] * S * T * es if c["mask"] == "window" else 0
        pages = sum(_pages(t, c["page"]) for t in lens)
        return {"bytes": seen * row * 17 // 16 + 2 * c["B"] * S * c["Hq"] * c["D"] * es
                + 4 * pages + 4 * c["B"] + mask,
                "flops": 4 * pairs * c["Hq"] * c["D"]}
    w = c["window"]
    pairs = sum(t * (t + 1) // 2 - (max(0, t - w) * (max(0, t - w) + 1) // 2 if w else 0)
                for t in lens)
    return {"bytes": sum(lens) * 2 * (c["Hq"] + c["Hkv"]) * c["D"] * es + 4 * (c["B"] + 1),
            "flops": 4 * pairs * c["Hq"] * c["D"]}


# ---- the same results in 64 bits ------------------------------------------------------
def _stored64(x):
    """The values that 4 bits keep of x, by distance to every code, in float64."""
    g = x.double().unflatten(-1, (-1, 32))
    a = g.abs().amax(-1)
    e = torch.ceil(torch.log2(a.clamp_min(1e-300) / 7))
    e = torch.where(a > 7 * _pow2_64(e), e + 1, e)
    e = torch.where(a <= 7 * _pow2_64(e - 1), e - 1, e).clamp(-125, 125)
    step = _pow2_64(e)[..., None]
    best = torch.full_like(g, math.inf)
    val = torch.zeros_like(g)
    for i in (0, 2, 4, 6, 1, 3, 5, 7):              # even codes first: they keep ties
        d = (g.abs() / step - GRID[i]).abs()
        val = torch.where(d < best, GRID[i] * step, val)
        best = torch.minimum(best, d)
    return (val * torch.sign(g)).flatten(-2)


def _attend64(q, k, v, scale, cap, hidden, mask=None):
    x = torch.matmul(q, k.t().contiguous()) * scale
    if cap:
        x = torch.tanh(x / cap) * cap
    if mask is not None:
        x = x + mask
    if hidden is not None:
        x = x.masked_fill(hidden, -math.inf)
    return torch.matmul(torch.softmax(x, -1), v)


def exact(case, seed):
    c = case
    if c["kind"] == "tables":
        return None          # whole numbers: the plain form's are the definition's
    if c["kind"] == "write":
        x = _write_inputs(c, seed)
        return [_stored64(x["k"]), _stored64(x["v"])]
    scale = 1.0 / math.sqrt(c["D"])
    if c["kind"] == "prompt":
        x = _prompt_inputs(c, seed)
        return _prompt_by_rows(c, x["q"].double(), x["k"].double(), x["v"].double(), x["lens"],
                               scale, 2048, _attend64)
    x = _attn_inputs(c, seed)
    G, S, at, outs = c["Hq"] // c["Hkv"], c["S"], 0, []
    for b, t in enumerate(x["lens"]):
        k, v = x["k"][at:at + t], x["v"][at:at + t]
        at += t
        last = t - S + torch.arange(S, device="cuda")[:, None]
        hidden = torch.arange(t, device="cuda")[None, :] > last
        mask = None if x["mask"] is None else x["mask"][b, 0, :, :t].double()
        outs.append(torch.cat([
            _attend64(x["q"][b, h * G:(h + 1) * G].double(), _stored64(k[:, h]), _stored64(v[:, h]),
                      scale, c["cap"], hidden, mask)
            for h in range(c["Hkv"])]))
    return torch.stack(outs)
