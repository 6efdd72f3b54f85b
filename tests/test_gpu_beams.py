"""Beam selection and beam tables against their restatements: ties, banned tokens, rows without
a distribution, odd sizes and strides; every shape of parents, page boundaries, pools."""
import math
import random

import pytest
import torch

from helm_amd import beams, pool4
from oracle import beams as R

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
I32 = dict(dtype=torch.int32, device=DEV)


def randn(seed, shape, dtype, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def check_select(logits, scores, n):
    got = beams.beam_select(logits, scores, n=n)
    want, tokens, parents = R.select(logits, scores, n)
    assert torch.equal(got.tokens.cpu(), tokens)
    assert torch.equal(got.parents.cpu().long(), parents)
    none = want == -math.inf
    assert torch.equal(got.scores.cpu() == -math.inf, none)
    # an exponential is off by 2^-23 and its row's sum by 2^-24 a term of 32, so log by less
    # than 2^-21; then half a step of fp32
    off = (got.scores.cpu().double() - want)[~none].abs()
    assert (off <= 2.0 ** -21 + 2.0 ** -24 * want[~none].abs()).all()
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,K,V,n", [
    (1, 1, 1, 1), (1, 1, 1, 4), (2, 3, 7, 3), (1, 4, 2048, 8), (3, 5, 2049, 10), (2, 2, 8191, 64),
    (1, 64, 1000, 64), (2, 1, 32003, 2), (7, 4, 40000, 8), (40, 4, 33000, 8)])
def test_select(B, K, V, n, dtype):
    logits = randn(V, (B, K, V), dtype, 3.0)
    scores = -10 * torch.rand((B, K), device=DEV)
    check_select(logits, scores, n)


@pytest.mark.parametrize("n", [1, 8, 64])
@pytest.mark.parametrize("make", ["equal", "few_values", "ascending", "descending", "one_run",
                                  "zeros_of_both_signs"])
def test_select_ties_and_orders(make, n):
    """Whole rows of equal logits, sorted rows: more near the top than a chunk's list holds."""
    B, K, V = 2, 3, 20000
    if make == "equal":
        x = torch.full((B, K, V), 1.5, device=DEV)
    elif make == "few_values":
        g = torch.Generator(device=DEV).manual_seed(n)
        x = torch.randint(0, 3, (B, K, V), generator=g, device=DEV).float()
    elif make == "ascending":
        x = (torch.arange(V, device=DEV) / V).expand(B, K, V).contiguous()
    elif make == "descending":
        x = (-torch.arange(V, device=DEV) / V).expand(B, K, V).contiguous()
    elif make == "one_run":
        x = torch.zeros((B, K, V), device=DEV)
        x[:, 1, 4096:4196] = 5.0
    else:
        x = torch.where(torch.arange(V, device=DEV) % 2 == 0, 0.0, -0.0)
        x = x.expand(B, K, V).contiguous()
    for scores in (torch.zeros((B, K), device=DEV),
                   torch.tensor([[0.0, -1.0, 0.5]] * B, device=DEV)):
        check_select(x, scores, n)
        check_select(x.bfloat16(), scores, n)


def test_select_first_step_banned_and_missing():
    B, K, V = 4, 4, 5000
    x = randn(1, (B, K, V), torch.float16, 2.0)
    x[:, :, ::2] = -math.inf
    scores = torch.full((B, K), -math.inf, device=DEV)
    scores[:, 0] = 0.0
    got = check_select(x, scores, 8)
    assert (got.parents == 0).all() and (got.tokens % 2 == 1).all()
    x[1] = -math.inf                                    # nothing allowed in one request
    x[2, :, :] = -math.inf
    x[2, 0, 4321] = -3.0                                # and a single token in another
    got = check_select(x, scores, 8)
    assert (got.tokens[1] == -1).all() and got.tokens[2, 0] == 4321 and got.scores[2, 0] == 0.0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_select_rows_without_a_distribution(bad, dtype):
    x = randn(2, (3, 3, 9000), dtype)
    x[0, 1, 8999] = bad
    x[1, :, 17] = bad                                   # every beam of a request
    x[2, 0] = bad                                       # a whole row
    scores = torch.tensor([[0.0, 5.0, -1.0]] * 3, device=DEV)
    got = check_select(x, scores, 4)
    assert (got.parents[0] != 1).all() and (got.tokens[1] == -1).all()
    scores = torch.tensor([[math.nan, math.inf, -math.inf], [0.0, math.nan, 1.0], [0.0, 0.0, 0.0]],
                          device=DEV)
    check_select(randn(3, (3, 3, 100), dtype), scores, 5)


def test_select_extreme_logits():
    x = torch.tensor([[[3.0e38, -3.0e38, 0.0, 1.0], [-3.0e38, -3.0e38, -3.0e38, -3.4e38]]],
                     device=DEV)
    check_select(x, torch.zeros((1, 2), device=DEV), 8)


def test_select_strides_alignment_and_out():
    B, K, V = 3, 2, 3001
    base = randn(4, (B, K + 1, V + 6), torch.bfloat16, 3.0)
    scores = -torch.rand((B, K), device=DEV)
    for off in range(4):                                # rows at any alignment, apart
        check_select(base[:, 1:, off:off + V], scores, 4)
    check_select(base[:, :1, :V].expand(B, K, V), scores, 4)        # one row for all beams
    check_select(base[:, :K, :V].transpose(1, 2).contiguous().transpose(1, 2), scores, 4)
    out = beams.beam_select(base[:, :K, :V], scores, n=4)
    again = beams.beam_select(base[:, 1:, :V], scores, n=4, out=out)
    assert again is out
    want = R.select(base[:, 1:, :V], scores, 4)
    assert torch.equal(out.tokens.cpu(), want[1])


def test_select_is_the_same_on_another_stream_and_in_a_graph():
    x = randn(5, (6, 4, 30000), torch.bfloat16, 3.0)
    scores = -10 * torch.rand((6, 4), device=DEV)
    want = beams.beam_select(x, scores, n=8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = beams.beam_select(x, scores, n=8)
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = beams.beam_select(x, scores, n=8)
    for seed in range(3):
        x.copy_(randn(6 + seed, x.shape, torch.float32, 3.0))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, beams.beam_select(x, scores, n=8)):
            assert torch.equal(a, b)


# ---- tables ----------------------------------------------------------------------------
def make_tables(r, B, K, page, width, lens, shared):
    """Rows whose shared columns are the same and whose others share pages here and there, the
    part-filled page each row's own."""
    table, at = [], 0
    for b in range(B):
        rows = [[0] * width for _ in range(K)]
        full = lens[b] // page
        for c in range(width):
            if c < shared[b]:
                names = [at] * K
            elif c < full:
                kinds = r.randint(1, K)
                names = [at + r.randrange(kinds) for _ in range(K)]
            else:
                names = [at + j for j in range(K)]
            for j in range(K):
                rows[j][c] = names[j]
            at = max(names) + 1
        table += rows
    return table, at


def parents_of(r, kind, K):
    return {"same": list(range(K)), "one": [r.randrange(K)] * K,
            "reverse": list(range(K))[::-1], "any": [r.randrange(K) for _ in range(K)],
            "none": [-1] * K, "outside": [r.choice([-1, K, 7 * K, -2 ** 31, r.randrange(K)])
                                         for _ in range(K)]}[kind]


@pytest.mark.parametrize("B,K,page,width", [
    (1, 1, 16, 1), (1, 4, 16, 9), (3, 2, 1, 5), (5, 3, 32, 130), (2, 64, 16, 20), (33, 8, 64, 257),
    (2, 5, 48, 300)])
@pytest.mark.parametrize("seed", range(4))
def test_tables(B, K, page, width, seed):
    r = random.Random(1000 * B + seed)
    lens, shared = [], []
    for b in range(B):
        full = r.choice([0, r.randrange(width + 1), width])
        lens.append(full * page + (r.choice([0, r.randrange(page)]) if full < width else 0))
        shared.append(r.randint(0, lens[-1] // page))
    table, n = make_tables(r, B, K, page, width, lens, shared)
    slots = list(range(n + 3))
    r.shuffle(slots)
    table = [[slots[s] for s in row] for row in table]
    kinds = ["same", "one", "reverse", "any", "none", "outside"]
    parents = [parents_of(r, kinds[(b + seed) % 6] if B > 1 else kinds[seed % 4], K)
               for b in range(B)]
    rows = [t for t in lens for _ in range(K)]
    want, copies, released = R.tables(parents, table, rows, page, shared)
    args = (torch.tensor(parents, **I32), torch.tensor(table, **I32), torch.tensor(rows, **I32))
    sh = torch.tensor(shared, **I32)
    pool = randn(seed, (n + 3, 2, 1, page, 8), torch.float16)
    moved = R.copy_pages(pool.cpu(), copies, rows, page, K)
    # a wider table's columns, out's own stride, and in place
    for form in ("new", "strided", "in_place"):
        store = beams.PageStore([pool.clone(), pool.clone()])
        par, tab, ln = (x.clone() for x in args)
        out = None
        if form == "strided":
            tab = torch.cat([tab, torch.full_like(tab, 12345)], 1)[:, :width]
            out = beams.BeamTables(torch.full((B * K, width + 3), 777, **I32)[:, :width],
                                   torch.empty((B * K, 2), **I32),
                                   torch.full((B * K * width,), -9, **I32), torch.empty(1, **I32))
        if form == "in_place":
            out = beams.BeamTables(tab, torch.empty((B * K, 2), **I32),
                                   torch.full((B * K * width,), -9, **I32), torch.empty(1, **I32))
        got = beams.beam_tables(par, tab, ln, page, shared_pages=sh, pages=store, out=out)
        assert got.page_table.cpu().tolist() == want
        assert [tuple(c) for c in got.copies.cpu().tolist()] == copies
        assert int(got.n_released) == len(released)
        assert got.released[:len(released)].cpu().tolist() == released
        if out is not None:
            assert (got.released[len(released):] == -9).all()
        for p in store.pools:
            assert torch.equal(p.cpu(), moved)
        if form != "in_place":
            assert torch.equal(tab, args[1])


def test_tables_no_page_is_shared_and_written():
    """Random steps of one request in place: part-filled pages stay each row's own, released
    pages are never named again, nothing is lost."""
    r = random.Random(3)
    K, page, width, n = 4, 16, 12, 200
    free = list(range(n))
    r.shuffle(free)
    table = torch.zeros((K, width), **I32)
    base = [free.pop() for _ in range(2)]
    length = 2 * page + 5
    for j in range(K):
        table[j, :2] = torch.tensor(base, **I32)
        table[j, 2] = free.pop()
    used = set(range(n)) - set(free)
    for _ in range(9 * page - 6):
        par = torch.tensor([parents_of(r, r.choice(["any", "one", "same", "reverse"]), K)], **I32)
        lens = torch.full((K,), length, **I32)
        t = beams.beam_tables(par, table, lens, page)
        table = t.page_table
        back = t.released[:int(t.n_released)].tolist()
        assert len(set(back)) == len(back) and set(back) <= used
        used -= set(back)
        free += back
        pages = -(-length // page)
        named = {int(s) for s in table[:, :pages].flatten()}
        assert named == used
        if length % page:
            assert len({int(s) for s in table[:, length // page]}) == K
        else:                                          # the next token's page, each row its own
            for j in range(K):
                table[j, length // page] = free.pop()
                used.add(int(table[j, length // page]))
        length += 1


@pytest.mark.parametrize("layout", ["arena", "k_and_v", "pool4", "odd_rows", "many", "transposed"])
def test_tables_pools(layout):
    r = random.Random(7)
    B, K, page, width, H, D, n = 2, 4, 32, 4, 3, 64, 40
    lens = [page + 19, 2 * page + 1]
    table, names = make_tables(r, B, K, page, width, lens, [0, 1])
    parents = [[0, 0, 0, 2], [3, 3, 1, 1]]
    rows = [t for t in lens for _ in range(K)]
    _, copies, _ = R.tables(parents, table, rows, page, [0, 1])
    assert sum(s >= 0 for s, _ in copies) == 4
    unit = 1
    if layout == "arena":
        pools = [randn(i, (n, 2, H, page, D), torch.bfloat16) for i in range(3)]
    elif layout == "k_and_v":
        arena = randn(0, (n, 2, H, page, D), torch.float32)
        pools = [arena[:, 0], arena[:, 1]]
    elif layout == "pool4":
        pools = [pool4.Pool4(n, H, D, page_size=page, device=DEV) for _ in range(2)]
        for i, p in enumerate(pools):
            p.data.copy_(torch.randint(0, 256, p.data.shape, device=DEV, dtype=torch.uint8))
        unit = 16
    elif layout == "odd_rows":
        pools = [randn(i, (n, H, page, 5), torch.float16) for i in range(2)]
    elif layout == "many":                              # more than one launch's
        pools = [randn(i, (n, page, 8), torch.float16) for i in range(131)]
    else:                                               # slots in the second dimension
        pools = [randn(i, (2, n, H, page, D), torch.float16)[i].transpose(0, 0) for i in range(2)]
    data = [p.data if layout == "pool4" else p for p in pools]
    want = [R.copy_pages(x.cpu(), copies, rows, page, K, unit) for x in data]
    store = beams.PageStore(pools)
    args = (torch.tensor(parents, **I32), torch.tensor(table, **I32), torch.tensor(rows, **I32))
    t = beams.beam_tables(*args, page, shared_pages=torch.tensor([0, 1], **I32), pages=store)
    for x, w in zip(data, want):
        assert torch.equal(x.cpu(), w)
    # pages outside the pool are left alone
    bad = args[1].clone()
    bad[:, 1] = torch.tensor([5, -1, n, 2 ** 31 - 1] * 2, **I32)
    before = [x.clone() for x in data]
    beams.beam_tables(args[0], bad, torch.full((8,), page + 3, **I32), page, pages=store)
    if layout == "arena":
        c = R.tables(parents, bad.tolist(), [page + 3] * 8, page)[1]
        for x, w in zip(data, before):
            assert torch.equal(x.cpu(), R.copy_pages(w.cpu(), c, [page + 3] * 8, page, K))
    assert int(t.n_released) >= 0


def test_tables_empty_and_long():
    t = beams.beam_tables(torch.zeros((0, 3), **I32), torch.zeros((0, 4), **I32),
                          torch.zeros(0, **I32), 16)
    assert int(t.n_released) == 0 and t.page_table.shape == (0, 4)
    # a length past the table's end, a negative one, a table without columns
    tab = torch.arange(8, **I32).view(4, 2)
    par = torch.tensor([[1, 1], [0, 0]], **I32)
    lens = [100, 100, -5, -5]
    t = beams.beam_tables(par, tab, torch.tensor(lens, **I32), 16)
    want, copies, released = R.tables(par.tolist(), tab.tolist(), lens, 16)
    assert t.page_table.tolist() == want and t.released[:int(t.n_released)].tolist() == released
    assert [tuple(c) for c in t.copies.tolist()] == copies
    t = beams.beam_tables(par, torch.zeros((4, 0), **I32), torch.tensor(lens, **I32), 16)
    assert int(t.n_released) == 0 and (t.copies == -1).all()


def test_tables_in_a_graph():
    r = random.Random(11)
    B, K, page, width = 3, 4, 16, 140
    par, lens = torch.zeros((B, K), **I32), torch.zeros(B * K, **I32)
    tab = torch.zeros((B * K, width), **I32)
    pool = randn(0, (B * K * width, 1, page, 8), torch.float16)
    first = pool.clone()
    store = beams.PageStore([pool])
    beams.beam_tables(par, tab, lens, page, pages=store)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = beams.beam_tables(par, tab, lens, page, pages=store)
    for _ in range(4):
        ln = [r.randrange(width * page) for _ in range(B)]
        t, n = make_tables(r, B, K, page, width, ln, [0] * B)
        p = [parents_of(r, "any", K) for _ in range(B)]
        rows = [x for x in ln for _ in range(K)]
        par.copy_(torch.tensor(p, **I32))
        tab.copy_(torch.tensor(t, **I32))
        lens.copy_(torch.tensor(rows, **I32))
        pool.copy_(first)
        graph.replay()
        torch.cuda.synchronize()
        want, copies, released = R.tables(p, t, rows, page)
        assert held.page_table.tolist() == want
        assert held.released[:int(held.n_released)].tolist() == released
        assert torch.equal(pool.cpu(), R.copy_pages(first.cpu(), copies, rows, page, K))
