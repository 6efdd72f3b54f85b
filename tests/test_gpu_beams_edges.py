"""Beam selection and beam tables at their edges: sums that 64 bits do not tell apart; pools with
heads outermost, pages outside the pool in every layout."""
import ctypes
import math
import random

import pytest
import torch

from helm_amd import _native, beams, pool4
from oracle import beams as R
from test_gpu_beams import DEV, I32, check_select, make_tables, randn

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 4, 40, 64])
@pytest.mark.parametrize("K,V", [(3, 20000), (40, 4001)])
def test_select_sums_that_round_alike(K, V, n, dtype):
    """A score so far out that no logit changes it: the lowest beam's lowest tokens, whatever
    their logits."""
    x = randn(n, (2, K, V), dtype, 3.0)
    x[0, 0, :V // 2] = -math.inf                       # the first allowed one lies far behind
    for far in (-1e30, 1e30):
        check_select(x, torch.full((2, K), far, device=DEV), n)
    # a beam that is not, with fewer tokens than are wanted: the rest from the others
    scores = torch.full((2, K), -1e30, device=DEV)
    scores[:, 1] = -5.0
    x[:, 1, 3:] = -math.inf
    got = check_select(x, scores, n)
    assert (got.parents[:, :3] == 1).all() and (got.parents[:, 3:] == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [1, 8, 64])
def test_select_logits_next_to_zero(n, dtype):
    """Logits that a score of ordinary size takes in whole."""
    B, K, V = 2, 4, 30000
    x = randn(n, (B, K, V), torch.float32, 1e-25).to(dtype)
    scores = torch.tensor([[-3.0, -1.0, -2.0, -1.5]] * B, device=DEV)
    x[1, 1, ::2] = -1.0
    x[1, 1, 20001] = 0.0
    check_select(x, scores, n)


@pytest.mark.parametrize("n", [1, 7, 64])
def test_select_groups_of_sums(n):
    """Logits 2^-22 apart, each in two forms 2^-24 apart, under a score of 2^30 whose sums are whole
    multiples of 2^-22: the forms tie, the steps do not."""
    g = torch.Generator(device=DEV).manual_seed(n)
    step = torch.randint(0, 50, (3, 2, 20000), generator=g, device=DEV)
    form = torch.randint(0, 2, step.shape, generator=g, device=DEV)
    x = 0.5 + step * 2.0 ** -22 + form * 2.0 ** -24
    scores = torch.tensor([[-2.0 ** 30, -2.0 ** 30 - 256]] * 3, device=DEV)
    check_select(x, scores, n)


@pytest.mark.parametrize("layout", ["heads_outermost", "k_and_v_heads_outermost", "arena",
                                    "k_and_v", "pool4", "odd_rows", "many"])
def test_tables_pools_and_pages_outside_them(layout):
    r = random.Random(9)
    B, K, page, width, H, D, n = 2, 4, 32, 4, 3, 64, 40
    lens, shared, unit = [page + 19, 2 * page + 1], [0, 1], 1
    table, _ = make_tables(r, B, K, page, width, lens, shared)
    parents = [[0, 0, 0, 2], [3, 3, 1, 1]]
    rows = [t for t in lens for _ in range(K)]
    if layout == "heads_outermost":
        pools = [randn(i, (H, n, page, D), torch.float16).transpose(0, 1) for i in range(2)]
    elif layout == "k_and_v_heads_outermost":
        pools = [randn(i, (2, H, n, page, D), torch.float32).permute(2, 0, 1, 3, 4)
                 for i in range(2)]
    elif layout == "arena":
        pools = [randn(i, (n, 2, H, page, D), torch.bfloat16) for i in range(3)]
    elif layout == "k_and_v":
        arena = randn(0, (n, 2, H, page, D), torch.float32)
        pools = [arena[:, 0], arena[:, 1]]
    elif layout == "pool4":
        pools, unit = [pool4.Pool4(n, H, D, page_size=page, device=DEV) for _ in range(2)], 16
        for p in pools:
            p.data.copy_(torch.randint(0, 256, p.data.shape, device=DEV, dtype=torch.uint8))
    elif layout == "odd_rows":
        pools = [randn(i, (n, H, page, 5), torch.float16) for i in range(2)]
    else:
        pools = [randn(i, (n, page, 8), torch.float16) for i in range(131)]
    data = [p.data if layout == "pool4" else p for p in pools]
    store = beams.PageStore(pools)
    outside = [list(x) for x in table]
    for j, x in enumerate([5, -1, n, 2 ** 31 - 1] * B):
        outside[j][lens[j // K] // page] = x
    outside[6][2], outside[7][2] = 7, 8
    for tab, sh in ((table, shared), (outside, None)):
        new, copies, released = R.tables(parents, tab, rows, page, sh)
        want = [R.copy_pages(x.cpu(), copies, rows, page, K, unit) for x in data]
        got = beams.beam_tables(torch.tensor(parents, **I32), torch.tensor(tab, **I32),
                                torch.tensor(rows, **I32), page, pages=store,
                                shared_pages=None if sh is None else torch.tensor(sh, **I32))
        for x, w in zip(data, want):
            assert torch.equal(x.cpu(), w)
        assert got.page_table.tolist() == new
        assert [tuple(c) for c in got.copies.tolist()] == copies
        assert got.released[:int(got.n_released)].tolist() == released


@pytest.mark.parametrize("n", [1, 128, 131])
def test_tables_of_no_request(n):
    """With pools, too, of more than one launch."""
    pools = [randn(i, (4, 16, 8), torch.float16) for i in range(n)]
    t = beams.beam_tables(torch.zeros((0, 3), **I32), torch.zeros((0, 4), **I32),
                          torch.zeros(0, **I32), 16, pages=beams.PageStore(pools))
    assert int(t.n_released) == 0 and t.page_table.shape == (0, 4) and t.copies.shape == (0, 2)
    for i, p in enumerate(pools):
        assert torch.equal(p, randn(i, (4, 16, 8), torch.float16))


def test_a_refused_call_leaves_the_table_as_it_was():
    """In place, with a pool that is null."""
    lib = _native.load()
    tab = torch.arange(24, **I32).view(6, 4)
    before = tab.clone()
    par, lens = torch.tensor([[1, 1, 0], [2, 0, 0]], **I32), torch.full((6,), 40, **I32)
    cop, rel, cnt = torch.zeros(12, **I32), torch.zeros(24, **I32), torch.zeros(1, **I32)
    pool = torch.zeros((24, 16, 8), dtype=torch.float16, device=DEV)
    need = lib.helm_beam_tables_workspace_bytes(2, 3, 4)
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)
    rc = lib.helm_beam_tables(par.data_ptr(), 2, 3, tab.data_ptr(), 4, 4, lens.data_ptr(), 16, None,
                              tab.data_ptr(), 4, cop.data_ptr(), rel.data_ptr(), cnt.data_ptr(),
                              (ctypes.c_void_p * 2)(pool.data_ptr(), None), 2, 24, 256, 1, 256, 1,
                              16, ws.data_ptr(), need, None)
    torch.cuda.synchronize()
    assert rc == _native.HELM_E_INVALID and torch.equal(tab, before)


def test_a_store_without_a_slot_copies_nothing():
    t = beams.beam_tables(torch.tensor([[1, 1]], **I32), torch.zeros((2, 2), **I32),
                          torch.full((2,), 5, **I32), 16,
                          pages=beams.PageStore([torch.zeros((0, 16, 8), device=DEV)]))
    assert t.copies.tolist() == [[0, 0], [-1, -1]]


def test_operands_between_a_pools_pages():
    """Memory between the pages is nobody's: outputs may lie there."""
    lib = _native.load()
    par, lens = torch.tensor([[1, 1, 0], [2, 0, 0]], **I32), torch.full((6,), 40, **I32)
    tab = torch.arange(24, **I32).view(6, 4)
    want, copies, released = R.tables(par.tolist(), tab.tolist(), [40] * 6, 16)
    buf = torch.arange(24 * 32, **I32)                 # pages of 16 tokens of 4 bytes, 128 apart
    pages = buf.view(24, 32)[:, :16].reshape(24, 16, 1).cpu()
    rel, new = torch.zeros(24, **I32), torch.zeros((6, 4), **I32)
    need = lib.helm_beam_tables_workspace_bytes(2, 3, 4)
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)
    at = buf.data_ptr()
    rc = lib.helm_beam_tables(par.data_ptr(), 2, 3, tab.data_ptr(), 4, 4, lens.data_ptr(), 16, None,
                              new.data_ptr(), 4, at + 64, rel.data_ptr(), at + 23 * 128 + 124,
                              (ctypes.c_void_p * 1)(at), 1, 24, 128, 1, 64, 1, 4, ws.data_ptr(),
                              need, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert rc == 0 and new.tolist() == want and int(buf[-1]) == len(released)
    assert [tuple(c) for c in buf[16:28].view(6, 2).tolist()] == copies
    assert torch.equal(buf.view(24, 32)[:, :16].reshape(24, 16, 1).cpu(),
                       R.copy_pages(pages, copies, [40] * 6, 16, 3))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("make", ["equal", "few_values", "one_run"])
@pytest.mark.parametrize("K,V,n", [(8, 20000, 64), (64, 20000, 64), (64, 2500, 40)])
def test_select_more_ties_than_the_joining_holds(K, V, n, make, dtype):
    """Rows alike, more of their lists' candidates at the bound than 2,048."""
    B = 2
    g = torch.Generator(device=DEV).manual_seed(K + V)
    if make == "equal":
        row = torch.full((B, 1, V), -2.5, device=DEV)
    elif make == "few_values":
        row = torch.randint(0, 3, (B, 1, V), generator=g, device=DEV).float()
    else:                                              # the largest at the row's end
        row = torch.zeros((B, 1, V), device=DEV)
        row[..., V - 100:] = 3.0
    x = row.expand(B, K, V).to(dtype).contiguous()
    check_select(x, torch.zeros((B, K), device=DEV), n)
    scores = -(torch.arange(K, device=DEV) % 3).float().expand(B, K).contiguous()
    check_select(x, scores.flip(1).contiguous(), n)
    x[:, K // 2] = -math.inf                           # one row offers nothing, one a single token
    x[:, K // 3, 1:] = -math.inf
    check_select(x, scores, n)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,K,V,n", [(1, 1, 152064, 8), (4, 4, 152064, 16), (1, 1, 200001, 64),
                                     (1, 1, 600001, 33), (1, 2, 300001, 1), (1, 64, 300001, 64)])
def test_select_many_chunks_a_row(B, K, V, n, dtype):
    """More chunks a row than the joining's lanes, more lists than one of its sweeps takes."""
    x = randn(V, (B, K, V), dtype, 3.0)
    check_select(x, -10 * torch.rand((B, K), generator=torch.Generator(device=DEV).manual_seed(V),
                                     device=DEV), n)
    if K * V < 2 * 10 ** 6:
        x = (x.float().clamp(min=4.0) * 2).round().to(dtype)        # a few values
        check_select(x, -32.0 * torch.arange(K, device=DEV).expand(B, K).contiguous(), n)
