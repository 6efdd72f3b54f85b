"""prefix_decode_attention against 64 bits.

The bound per element, u the type's half step (bf16 2^-8, f16 2^-11): the output's rounding
u |o|; weights rounded to the type at worst, w' = w (1 + d), |d| <= u, with the sum over w', move
a mean by at most u / (1 - u) sum p |v - o| <= 1.01 u (sum p |v| + |o|); an fp32 logit is off by
(D + 4) 2^-24 L, L the largest sum of its terms' magnitudes, and 2^-22 (L + 8) for its scaling
and exponent, twice that times max|v|; f16 weights end at 2^-34 of the largest, and sums of
T terms in fp32, partial ones and their joining among them, add T 2^-24 max|v|."""
import math
import random

import pytest
import torch

from helm_amd import paged, prefix
from oracle import serving as R

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
I32 = dict(dtype=torch.int32, device=DEV)
BF, HF = torch.bfloat16, torch.float16


def _randn(seed, shape, dtype, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def make(groups, Hq, Hkv, D, page, dtype, S=1, seed=0, alone=(), extra=3):
    """groups: [(shared pages, [lengths])], alone: lengths of sequences outside them (behind)."""
    r = random.Random(seed)
    lens = [t for _, n in groups for t in n] + list(alone)
    shared = [s for s, n in groups for _ in n] + [0] * len(alone)
    need = [max(0, -(-t // page) - s) for t, s in zip(lens, shared)]
    n_slots = sum(s for s, _ in groups) + sum(need) + extra
    slots = list(range(n_slots))
    r.shuffle(slots)
    width = max([1] + [s + n for s, n in zip(shared, need)])
    rows, row = [], 0
    for s, n in groups:
        own = [slots.pop() for _ in range(s)]
        for _ in n:
            rows.append(own + [slots.pop() for _ in range(need[row])])
            row += 1
    for _ in alone:
        rows.append([slots.pop() for _ in range(need[row])])
        row += 1
    table = torch.tensor([x + [r.choice([-1, 0, 10 ** 9])] * (width - len(x)) for x in rows],
                         **I32).view(len(lens), width)
    starts = [0]
    for _, n in groups:
        starts.append(starts[-1] + len(n))
    return {"q": _randn(seed, (len(lens), Hq, S, D), dtype, 1.5),
            "arena": _randn(seed + 1, (n_slots, 2, Hkv, page, D), dtype), "table": table,
            "lens": lens, "len_t": torch.tensor(lens, **I32),
            "start_t": torch.tensor(starts, **I32),
            "shared_t": torch.tensor([s for s, _ in groups], **I32), "page": page}


def call(c, **kw):
    return prefix.prefix_decode_attention(c["q"], c["arena"][:, 0], c["arena"][:, 1], c["table"],
                                          c["len_t"], c["start_t"], c["shared_t"], **kw)


def check(c, out, scale=None, cap=0.0, window=0, rows=None, heads=None):
    q, arena, page = c["q"], c["arena"], c["page"]
    _, Hq, S, D = q.shape
    Hkv, n_slots = arena.size(2), arena.size(0)
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    u = HALF[out.dtype]
    for r in rows if rows is not None else range(q.size(0)):
        t = min(c["lens"][r], c["table"].size(1) * page)
        slots = c["table"][r, :-(-t // page)].long()
        there = (slots >= 0) & (slots < n_slots)
        kv = arena[torch.where(there, slots, torch.zeros_like(slots))]
        pos = t - S + torch.arange(S, device=DEV)[:, None]
        j = torch.arange(t, device=DEV)[None, :]
        hidden = (j > pos) | ~there.repeat_interleave(page)[:t][None, :]
        if window:
            hidden = hidden | (j <= pos - window)
        for h in heads or range(Hq):
            k = kv[:, 0, h // (Hq // Hkv)].reshape(-1, D)[:t]
            v = kv[:, 1, h // (Hq // Hkv)].reshape(-1, D)[:t]
            want, mag = R.attend(q[r, h][None], k, v, scale, cap, hidden)
            want, mag = want[0], mag[0]
            fin = torch.nan_to_num(k.double(), nan=0.0, posinf=0.0, neginf=0.0)
            size = R.logit_size(q[r, h], fin, scale)
            fine = v[torch.isfinite(v)]
            vmax = fine.abs().max().item() if fine.numel() else 0.0
            e = (D + 4) * 2.0 ** -24 * size + 2.0 ** -22 * (size + 8)
            tol = u * want.abs() + 1.01 * u * (mag + want.abs()) \
                + vmax * (2 * e + t * (2.0 ** -24 + 2.0 ** -34)) + 1e-30
            got = out[r, h].double()
            ok = ((got - want).abs() <= tol) | (got == want) | \
                (torch.isnan(got) & torch.isnan(want))
            assert ok.all(), (r, h, (got - want).abs().max().item(), tol.min().item())


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 48, 128])
def test_beams_of_a_prompt(dtype, D, page):
    c = make([(5, [5 * page + 3] * 4), (1, [page + 1, page + 17, 2 * page])], 8, 2, D, page, dtype,
             seed=D + page)
    check(c, call(c))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (7, 1), (14, 2), (40, 8), (16, 16), (33, 1)])
def test_head_groups(Hq, Hkv, dtype):
    c = make([(9, [9 * 16 + n for n in (1, 30, 200)]), (20, [20 * 16 + 64] * 2)], Hq, Hkv, 64, 16,
             dtype, seed=Hq, alone=[77])
    check(c, call(c), heads=[0, Hq // 2, Hq - 1])


@pytest.mark.parametrize("lens", [
    [(0, [1])], [(0, [0, 1, 2])], [(1, [16, 17])], [(2, [31, 32, 33, 5, 0, 1])], [(3, [])],
    [(0, [500, 3]), (4, []), (7, [112, 113]), (7, [0, 0])], [(64, [1024] * 3)],
    [(40, [700, 641, 639, 1, 640])]])
def test_lengths(lens):
    """From none to long: sequences that end within the shared pages, groups without a sequence,
    all pages shared, nothing shared."""
    c = make(lens, 4, 2, 128, 16, BF, seed=3, alone=[0, 1, 35])
    check(c, call(c))


@pytest.mark.parametrize("S", [1, 2, 4, 7])
@pytest.mark.parametrize("G", [1, 5])
@pytest.mark.parametrize("window", [0, 1, 40, 300])
def test_drafts_and_windows(S, G, window):
    """The last S tokens, each up to its own; rows before a sequence's first token see nothing."""
    c = make([(8, [8 * 16 + n for n in (0, 1, 3, 150)]), (3, [48, 20, 2, 400])], 2 * G, 2, 64, 16,
             HF, S=S, seed=10 * S + G, alone=[1, 0, 9, 333])
    out = call(c, window=window)
    check(c, out, window=window)
    for r, t in enumerate(c["lens"]):
        for s in range(S):
            if t - S + s < 0:
                assert (out[r, :, s] == 0).all()


@pytest.mark.parametrize("dtype,D", [(BF, 64), (HF, 128), (BF, 256)])
@pytest.mark.parametrize("cap,scale", [(50.0, None), (5.0, 0.3), (0.0, -0.2), (0.0, 0.0),
                                       (30.0, -1.0)])
def test_softcap_and_scale(dtype, D, cap, scale):
    c = make([(6, [120, 130, 99])], 4, 2, D, 16, dtype, seed=D, alone=[50])
    check(c, call(c, softcap=cap or None, scale=scale), scale=scale, cap=cap)


@pytest.mark.parametrize("dtype,D,Hkv,n", [(BF, 128, 2, 9), (HF, 64, 1, 40), (BF, 256, 1, 33),
                                           (HF, 128, 1, 70), (BF, 64, 3, 100)])
def test_many_rows_of_a_group(dtype, D, Hkv, n):
    """More rows than a walk has, split over many workgroups."""
    r = random.Random(n)
    c = make([(70, [70 * 16 + r.randint(0, 90) for _ in range(n)]), (3, [60] * 3)], 4 * Hkv, Hkv,
             D, 16, dtype, seed=n)
    check(c, call(c), rows=[0, 1, n // 2, n - 1, n], heads=[0, 4 * Hkv - 1])


def test_long_shared_document():
    c = make([(1250, [20000 + n for n in (0, 1, 37, 800)])], 8, 2, 128, 16, BF, seed=4)
    check(c, call(c))
    c = make([(500, [500 * 16 + 3] * 20)], 16, 2, 64, 16, HF, seed=5)
    check(c, call(c, window=5000), window=5000, rows=[0, 7, 19])


@pytest.mark.parametrize("R,n_groups", [(300, 100), (4096, 512), (1000, 3), (65, 1)])
def test_many_sequences(R, n_groups):
    r = random.Random(R)
    groups = []
    left = R
    for g in range(n_groups):
        n = left // (n_groups - g) if n_groups > 3 else r.randint(1, left - (n_groups - g - 1))
        groups.append((r.randint(0, 4), [r.randint(0, 90) for _ in range(n)]))
        left -= n
    c = make(groups, 2, 1, 64, 16, BF, seed=R, alone=[r.randint(0, 50) for _ in range(left)])
    out = call(c)
    check(c, out, rows=r.sample(range(R), 24) + [0, R - 1])
    # one by one, as sequences that share nothing
    none = dict(c, start_t=torch.zeros(1, **I32), shared_t=torch.zeros(0, **I32))
    solo = call(none)
    assert ((out.float() - solo.float()).abs() <= 4 * HALF[BF] * 4.5).all()


def test_hidden_rows_hold_anything():
    """NaN and infinities in pages' unused rows, in pages of no sequence, past a causal limit and
    out of the window; slots that the pool does not have."""
    for window in (0, 30):
        for S in (1, 3):
            c = make([(4, [64 + 5, 64 + 20, 64, 40, 3]), (2, [32, 33])], 4, 2, 128, 16, BF, S=S,
                     seed=6, alone=[18])
            clean = call(c, window=window)
            used = torch.zeros(c["arena"].size(0) * 16, dtype=torch.bool, device=DEV)
            for r, t in enumerate(c["lens"]):
                j = torch.arange(t, device=DEV)
                used[c["table"][r][j // 16].long() * 16 + j % 16] = True
            bad = torch.tensor([math.nan, math.inf, -math.inf, 3e38], device=DEV)
            noise = bad[torch.randint(0, 4, c["arena"].shape, device=DEV)].to(BF)
            keep = used.view(-1, 1, 1, 16, 1).expand_as(c["arena"])
            c["arena"] = torch.where(keep, c["arena"], noise)
            assert torch.equal(call(c, window=window), clean)
            c["table"][0, 1] = -1
            c["table"][1, 5] = c["arena"].size(0)
            c["table"][7, 0] = -2 ** 31
            c["table"][1:5, 1] = -1                        # (shared: as in the first row)
            check(c, call(c, window=window), window=window)


@pytest.mark.parametrize("dtype,D", [(BF, 64), (HF, 128), (BF, 256)])
@pytest.mark.parametrize("n", [3, 60])
def test_visible_infinities_and_nan(dtype, D, n):
    """They count at any weight in the rows that see them, and in no other."""
    S = 2
    c = make([(6, [96 + 40 + i for i in range(n)]), (2, [40, 41])], 2, 1, D, 16, dtype, S=S, seed=7)
    clean = call(c)
    shared, own = int(c["table"][0, 2]), int(c["table"][1, 6])
    a = c["arena"]
    a[shared, 1, 0, 3, 5] = math.inf
    a[shared, 1, 0, 9, 6] = -math.inf
    a[shared, 1, 0, 4, 7] = math.nan
    a[shared, 1, 0, 5, 8] = math.inf
    a[shared, 1, 0, 6, 8] = -math.inf
    a[own, 1, 0, 0, 9] = math.inf
    last = (c["lens"][1] - 1)
    a[int(c["table"][1, last // 16]), 1, 0, last % 16, 10] = math.nan   # its last row's alone
    out = call(c)
    assert (out[:n, :, :, 5] == math.inf).all() and (out[:n, :, :, 6] == -math.inf).all()
    assert torch.isnan(out[:n, :, :, 7]).all() and torch.isnan(out[:n, :, :, 8]).all()
    assert (out[1, :, :, 9] == math.inf).all()
    assert torch.isnan(out[1, :, 1, 10]).all() and not torch.isnan(out[1, :, 0, 10]).any()
    same = torch.ones_like(out, dtype=torch.bool)
    same[:n, :, :, 5:9] = False
    same[1, :, :, 9:11] = False
    u = HALF[dtype]
    assert ((out.float() - clean.float()).abs()[same] <= 2.1 * u * 5.0).all()
    assert torch.equal(out[n:], clean[n:])
    # a key of NaN takes the whole row
    a[own, 0, 0, 0, 0] = math.nan
    out = call(c)
    assert torch.isnan(out[1]).all() and not torch.isnan(out[0, :, :, :5]).any()


def test_far_apart_scores():
    """One part's weights far below the other's: the joined sums keep what is left of them."""
    c = make([(8, [8 * 16 + 20] * 3)], 2, 1, 128, 16, BF, seed=8)
    c["arena"][c["table"][0, :8].long(), 0] *= 40
    check(c, call(c))
    c["arena"][c["table"][0, :8].long(), 0] *= -1
    check(c, call(c))
    c["arena"][:, 0] = 0                                   # all weights alike
    check(c, call(c))


def test_layouts_of_the_pools_and_q():
    c = make([(4, [64 + 9, 64 + 30])], 4, 2, 64, 32, HF, seed=9)
    want = call(c)
    a = c["arena"]
    k, v = a[:, 0].contiguous(), a[:, 1].contiguous()
    args = (c["table"], c["len_t"], c["start_t"], c["shared_t"])
    assert torch.equal(prefix.prefix_decode_attention(c["q"], k, v, *args), want)
    wide = torch.zeros((a.size(0), 5, 2, 32, 64), dtype=HF, device=DEV)      # slots far apart
    wide[:, 1], wide[:, 3] = k, v
    assert torch.equal(prefix.prefix_decode_attention(c["q"], wide[:, 1], wide[:, 3], *args), want)
    heads = torch.zeros((2, 2, a.size(0), 32, 64), dtype=HF, device=DEV)     # heads outermost
    heads[0], heads[1] = k.transpose(0, 1), v.transpose(0, 1)
    assert torch.equal(prefix.prefix_decode_attention(
        c["q"], heads[0].transpose(0, 1), heads[1].transpose(0, 1), *args), want)
    q = c["q"].transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(prefix.prefix_decode_attention(q, k, v, *args), want)
    buf = torch.zeros(c["q"].numel() + 1, dtype=HF, device=DEV)
    odd = buf[1:].view(c["q"].shape)
    odd.copy_(c["q"])
    assert torch.equal(prefix.prefix_decode_attention(odd, k, v, *args), want)
    tab = torch.full((2, 40), 12345, **I32)
    tab[:, :c["table"].size(1)] = c["table"]
    assert torch.equal(prefix.prefix_decode_attention(c["q"], k, v, tab[:, :c["table"].size(1)],
                                                      *args[1:]), want)
    assert torch.equal(prefix.prefix_decode_attention(c["q"], k, v, tab, *args[1:],
                                                      max_pages=c["table"].size(1)), want)
    out = torch.empty_like(want)
    assert prefix.prefix_decode_attention(c["q"], k, v, *args, out=out) is out
    assert torch.equal(out, want)
    own = c["q"].clone()
    prefix.prefix_decode_attention(own, k, v, *args, out=own)                # out may be q
    assert torch.equal(own, want)


def test_max_pages_and_table_width_end_a_sequence():
    c = make([(4, [150, 64 + 9])], 2, 2, 64, 16, BF, seed=11)
    cut = dict(c, lens=[96, 73])
    check(cut, call(c, max_pages=6))
    wide = dict(c, len_t=torch.tensor([10 ** 6, -5], **I32))
    check(dict(c, lens=[c["table"].size(1) * 16, 0]), call(wide))


def test_groups_past_the_batch_and_counts_past_the_table():
    c = make([(3, [60, 70]), (2, [50, 40])], 2, 2, 64, 16, BF, seed=12)
    want = call(c)
    # starts outside 0 .. R are taken to its ends, shared columns to the table's
    got = call(dict(c, start_t=torch.tensor([-7, 2, 99], **I32)))
    assert torch.equal(got, want)
    c = make([(4, [64, 60])], 2, 2, 64, 16, BF, seed=13)
    assert torch.equal(call(dict(c, shared_t=torch.tensor([2 ** 31 - 1], **I32))), call(c))
    none = call(dict(c, shared_t=torch.tensor([-3], **I32)))
    check(c, none)


@pytest.mark.parametrize("starts", [[0, 5, 2, 7], [7, 0], [3, 2 ** 31 - 1, -2 ** 31, 1]])
def test_starts_that_do_not_ascend_share_nothing(starts):
    c = make([(6, [6 * 16 + 20 * i for i in range(7)])], 4, 2, 64, 16, BF, seed=21)
    n = len(starts) - 1
    got = call(dict(c, start_t=torch.tensor(starts, **I32), shared_t=torch.full((n,), 6, **I32)))
    check(c, got)
    none = dict(c, start_t=torch.zeros(1, **I32), shared_t=torch.zeros(0, **I32))
    check(c, call(none))


def test_the_most_sequences_of_the_widest_heads():
    r = random.Random(5)
    c = make([(1, [r.randint(16, 40) for _ in range(8)]) for _ in range(512)], 1, 1, 256, 16, BF,
             seed=22)
    check(c, call(c), rows=r.sample(range(4096), 40) + [0, 4095])


def test_the_same_as_paged_decode():
    """Whole tables: the answer of the operator that reads every sequence's pages by itself."""
    c = make([(30, [30 * 16 + n for n in (5, 60, 130, 700)])], 16, 4, 128, 16, BF, seed=14)
    got = call(c)
    tab = torch.where((c["table"] < 0) | (c["table"] >= c["arena"].size(0)), 0, c["table"])
    want = paged.paged_decode_attention(c["q"], c["arena"][:, 0], c["arena"][:, 1], tab, c["len_t"])
    assert ((got.float() - want.float()).abs()
            <= 2 * 2.0 ** -8 * want.float().abs() + 2.0 ** -10).all()


def test_prepared_runs_streams_and_graphs():
    c = make([(20, [20 * 16 + n for n in (5, 60, 130)]), (0, [40])], 8, 2, 128, 16, BF, seed=15)
    step = prefix.prepare_prefix_decode(c["q"], c["arena"][:, 0], c["arena"][:, 1], c["table"],
                                        c["len_t"], c["start_t"], c["shared_t"])
    want = call(c)
    assert torch.equal(step.run(), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call(c)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held, whole = step.run(), call(c)
    r = random.Random(1)
    for i in range(4):
        c["q"].copy_(_randn(40 + i, c["q"].shape, torch.float32, 1.5))
        c["len_t"].copy_(torch.tensor([r.randint(0, 20 * 16 + 5) for _ in range(4)], **I32))
        c["shared_t"][0] = r.randint(0, 20)
        graph.replay()
        torch.cuda.synchronize()
        again = call(c)
        assert torch.equal(held, again) and torch.equal(whole, again)


def test_two_calls_at_once():
    """Two streams, each with calls of its own: they share nothing."""
    a = make([(60, [60 * 16 + n for n in (5, 60, 130)])], 8, 2, 128, 16, BF, seed=16)
    b = make([(10, [10 * 16 + 40] * 30)], 4, 4, 64, 16, HF, seed=17)
    want_a, want_b = call(a), call(b)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(10):
        with torch.cuda.stream(s1):
            got.append((call(a), want_a))
        with torch.cuda.stream(s2):
            got.append((call(b), want_b))
    torch.cuda.synchronize()
    for x, y in got:
        assert torch.equal(x, y)


def test_no_sequence():
    c = make([], 2, 2, 64, 16, BF, seed=18)
    assert call(c).shape == (0, 2, 1, 64)
    e = torch.zeros((0, 2, 16, 64), dtype=BF, device=DEV)              # a pool without a slot
    out = prefix.prefix_decode_attention(_randn(0, (2, 2, 1, 64), BF), e, e,
                                         torch.zeros((2, 0), **I32), torch.tensor([5, 0], **I32),
                                         torch.tensor([0, 2], **I32), torch.zeros(1, **I32))
    assert (out == 0).all()
