"""batch_tables against the oracle's walk in Python: whole numbers, equal."""
import random

import pytest
import torch

from helm_amd import paged
from oracle import serving as R

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _check(new, cached, table, free, page, max_tokens, wide=0):
    """`wide`: the table is a slice of a wider one, whose other columns stay."""
    width = len(table[0]) if table else 0
    back = torch.full((len(new), width + wide), -7, dtype=torch.int32, device=DEV)
    t = back[:, :width]
    if width:
        t.copy_(_i32(table))
    got = paged.batch_tables(_i32(new), _i32(cached), t, _i32(free), page, max_tokens)
    want = R.tables(new, cached, table, free, page, max_tokens)
    for name, a, b in zip(paged.BatchTables._fields, got, want):
        assert a.tolist() == ([b] if name == "pages_taken" else b), name
    assert t.tolist() == want[5]
    assert (back[:, width:] == -7).all()
    return got


def _case(r, B, page, new_hi, cached_hi, short_free=0, narrow=0):
    new = [r.choice([0, 1, r.randint(0, new_hi)]) for _ in range(B)]
    cached = [r.choice([0, page - 1, page, r.randint(0, cached_hi)]) for _ in range(B)]
    need = [-(-(c + n) // page) for c, n in zip(cached, new)]
    have = [-(-c // page) for c in cached]
    width = max(1, max(need) - narrow)
    free = list(range(1000, 1000 + max(0, sum(need) - sum(have) - short_free)))
    r.shuffle(free)
    table = [[(100 * b + i if i < h else -3) for i in range(width)] for b, h in enumerate(have)]
    return new, cached, table, free


@pytest.mark.parametrize("B,page,new_hi,cached_hi", [
    (1, 16, 1, 40), (1, 16, 300, 0), (2, 64, 5, 200), (7, 16, 100, 300), (64, 16, 40, 100),
    (65, 32, 3, 70), (255, 16, 1, 50), (256, 128, 20, 400), (257, 1, 9, 9), (1000, 16, 30, 64),
    (4096, 48, 3, 100)])
@pytest.mark.parametrize("pad", [0, 13])
def test_tables(B, page, new_hi, cached_hi, pad):
    r = random.Random(B * 131 + page + pad)
    new, cached, table, free = _case(r, B, page, new_hi, cached_hi)
    _check(new, cached, table, free, page, sum(new) + pad, wide=pad)


def test_no_tokens_and_negative_lengths():
    _check([0, 0], [5, 0], [[3], [4]], [], 16, 0)
    _check([0], [0], [[9]], [], 16, 3)
    _check([-4, 2], [3, -1], [[3], [4]], [8], 16, 4)


def test_too_few_pages_tokens_or_columns():
    r = random.Random(3)
    new, cached, table, free = _case(r, 9, 16, 200, 100, short_free=5)
    got = _check(new, cached, table, free, 16, sum(new))
    assert int(got.pages_taken) > len(free)
    new, cached, table, free = _case(r, 9, 16, 200, 100, narrow=3)
    _check(new, cached, table, free, 16, sum(new) + 2)
    new, cached, table, free = _case(r, 9, 16, 200, 100)
    _check(new, cached, table, free, 16, sum(new) // 2)


def test_lengths_near_the_int32_range():
    top = 2 ** 31 - 1
    t = torch.full((2, 2), 5, dtype=torch.int32, device=DEV)
    got = paged.batch_tables(_i32([top, top]), _i32([0, top - 1]), t, _i32([]), 2 ** 30, 3)
    assert got.cu_seqlens.tolist() == [0, top, top] and got.seq_lens.tolist() == [top, top]
    assert got.slot_map.tolist() == [-1, -1, -1] and got.positions.tolist() == [0, 1, 2]
    assert t.tolist() == [[-1, -1], [5, 5]]


def test_results_written_again_and_replayed():
    """One set of outputs for every step, captured: each replay reads the lengths,
    table and free list as they are then."""
    r = random.Random(11)
    page, B, N = 16, 6, 64
    new, cached = _i32([0] * B), _i32([0] * B)
    table, free = torch.zeros((B, 40), dtype=torch.int32, device=DEV), _i32(list(range(200)))
    out = paged.batch_tables(new, cached, table, free, page, N)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        paged.batch_tables(new, cached, table, free, page, N, out=out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged.batch_tables(new, cached, table, free, page, N, out=out)
    for _ in range(4):
        nl = [r.randint(0, 10) for _ in range(B)]
        cl = [r.randint(0, 500) for _ in range(B)]
        tb = [[r.randint(0, 99) for _ in range(40)] for _ in range(B)]
        fl = [r.randint(100, 999) for _ in range(200)]
        new.copy_(_i32(nl)); cached.copy_(_i32(cl)); table.copy_(_i32(tb)); free.copy_(_i32(fl))
        graph.replay()
        torch.cuda.synchronize()
        want = R.tables(nl, cl, tb, fl, page, N)
        assert [out[i].tolist() for i in range(4)] == [list(w) for w in want[:4]]
        assert out.pages_taken.item() == want[4] and table.tolist() == want[5]


def _loop(r, B, N, top, captured):
    """Steps whose cached lengths are the outputs' seq_lens, kept in place: each step's tables
    are the oracle's, and the lengths after it the next step's."""
    page, width = 16, 60
    used = 0
    new, free = _i32([0] * B), _i32([0] * 400)
    table = torch.full((B, width), -3, dtype=torch.int32, device=DEV)
    out = paged.batch_tables(new, _i32([0] * B), table, free, page, N)
    cached, lens = out.seq_lens, [0] * B
    rows = table.tolist()
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            paged.batch_tables(new, cached, table, free, page, N, out=out)
        cached.zero_()
    for _ in range(5):
        nl = [r.randint(0, top) for _ in range(B)]
        fl = list(range(used, used + 400))
        new.copy_(_i32(nl))
        free.copy_(_i32(fl))
        if captured:
            graph.replay()
        else:
            assert paged.batch_tables(new, cached, table, free, page, N, out=out) is out
        torch.cuda.synchronize()
        want = R.tables(nl, lens, rows, fl, page, N)
        assert [out[i].tolist() for i in range(4)] == [list(w) for w in want[:4]]
        assert out.pages_taken.item() == want[4] and table.tolist() == want[5]
        lens, rows, used = want[3], want[5], used + want[4]


@pytest.mark.parametrize("B,N,top", [(1, 3, 1), (3, 16, 4), (70, 500, 6), (300, 12000, 30)])
@pytest.mark.parametrize("captured", [False, True])
def test_lengths_kept_in_place(B, N, top, captured):
    """One workgroup's steps and many workgroups'."""
    _loop(random.Random(B), B, N, top, captured)


def test_outputs_over_operands_are_refused():
    B, page, N = 4, 16, 20
    new, cached = _i32([3] * B), _i32([5] * B)
    back = torch.zeros((B, 40), dtype=torch.int32, device=DEV)
    table, free = back[:, :8], _i32(list(range(10, 40)))
    out = paged.batch_tables(new, cached, table, free, page, N)
    shifted = _i32([5] * (B + 1))
    wide = torch.zeros(40, dtype=torch.int64, device=DEV)
    for lens, o in ((cached, out._replace(seq_lens=new)), (shifted[:B], out._replace(seq_lens=shifted[1:])),
                    (cached, out._replace(positions=wide[:N], slot_map=wide[N - 1:2 * N - 1])),
                    (cached, out._replace(pages_taken=free[7:8])), (cached, out._replace(seq_lens=back[2, 6:10])),
                    (out.cu_seqlens[1:], out), (out.pages_taken.expand(B).contiguous()[:B], out._replace(
                        seq_lens=out.cu_seqlens[:B]))):
        with pytest.raises(ValueError, match="over another operand"):
            paged.batch_tables(new, lens, table, free, page, N, out=o)
    with pytest.raises(ValueError, match="over another operand"):
        paged.batch_tables(new, back[1, 4:8], table, free, page, N)
    # columns of the table's buffer that are not the table's are nobody else's either
    got = paged.batch_tables(new, back[1, 8:8 + B], table, free, page, N,
                             out=out._replace(seq_lens=back[2, 12:12 + B]))
    assert got.seq_lens.tolist() == [3] * B
