"""The 4-bit pool against its definition (oracle/serving.py, 64 bits): what is written
and read back is equal; attention differs by roundings that each test counts.

Attention's bound per output element, u the half step of the output type: u |o| for the
output; weights enter as hi + lo bf16 parts, 2^-16 of each at most, and an fp32 logit is
off by at most (D + 4) 2^-24 L, L the largest sum of its terms' magnitudes (the products
are exact: bf16 codes and queries in parts), plus 2^-22 of the logit's size for its
scaling and exponent; a weight's relative error e moves the mean by at most 2 e max|v|;
sums of T terms in fp32 add T 2^-24 max|v| (far more than their trees do)."""
import copy
import math

import pytest
import torch

from helm_amd import pool4
from oracle import serving as R

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def _randn(seed, *shape):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(shape, generator=g, device=DEV)


def _slots(seed, n, n_slots, page):
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(n_slots * page, generator=g)[:n].to(DEV)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,Hkv,page,n", [
    (64, 1, 16, 1), (64, 2, 32, 777), (64, 5, 48, 33), (128, 8, 16, 40), (128, 1, 16, 1),
    (128, 3, 64, 1001), (256, 2, 16, 130), (256, 1, 256, 17)])
def test_written_values_read_back(dtype, D, Hkv, page, n):
    n_slots = n // page + 3
    pool = pool4.Pool4(n_slots, Hkv, D, page_size=page, device=DEV)
    slots = _slots(n, n, n_slots, page)
    spread = torch.exp(3 * _randn(5, n, Hkv, D // 32, 1)).expand(n, Hkv, D // 32, 32)
    k = (_randn(1, n, Hkv, D) * spread.reshape(n, Hkv, D)).clamp(-6e4, 6e4).to(dtype)
    v = _randn(2, n, Hkv, D).to(dtype)
    before = pool.data.clone()
    pool.write(k, v, slots)
    gk, gv = pool.read(slots, dtype=torch.float32)
    assert torch.equal(gk.double(), R.stored4(k)) and torch.equal(gv.double(), R.stored4(v))
    hk, hv = pool.read(slots, dtype=dtype)
    assert torch.equal(hk, gk.to(dtype)) and torch.equal(hv, gv.to(dtype))
    # the rows that no slot names stay
    rest = torch.ones(n_slots * page, dtype=torch.bool, device=DEV)
    rest[slots] = False
    if rest.any():
        rk, rv = pool.read(torch.nonzero(rest).flatten(), dtype=torch.float32)
        assert (rk == 0).all() and (rv == 0).all()
    pool.write(k[:0], v[:0], slots[:0])
    assert pool.data.shape == before.shape


def test_codes_ties_and_edges():
    """Every code's neighbourhood at many exponents, ties, zeros, subnormal and largest
    values, infinities and NaN, which stay in their group of 32 dims."""
    rows = []
    ys = torch.tensor([0, .2499, .25, .2501, .5, .7499, .75, .76, 1.25, 1.2501, 1.75, 2.5, 2.51, 3.5,
                       3.49, 5, 5.01, 6, 6.5, 7, -.25, -.75, -5, -6.9, -0.0, 1, 2, 3, 4, .3, .6, 1.4])
    for e in (-125, -124, -100, -20, 0, 3, 100, 124, 125):
        y = ys.clone()
        y[0] = 7.0                              # the group's largest: exponent e
        rows.append((y.double() * 2.0 ** e).float())
    rows.append(torch.zeros(32))
    rows.append(torch.full((32,), 1e-45))
    rows.append(torch.full((32,), 1.5 * 2.0 ** -126))
    rows.append(torch.full((32,), torch.finfo(torch.float32).max))
    for odd in (math.inf, -math.inf, math.nan):
        r = torch.ones(32)
        r[7] = odd
        rows.append(r)
    x = torch.stack(rows)
    n = x.size(0)
    x = torch.cat([x, x.flip(0)], 1).view(n, 1, 64).to(DEV)
    pool = pool4.Pool4(4, 1, 64, device=DEV)
    slots = torch.arange(n, device=DEV) + 3
    pool.write(x, -x, slots)
    k, v = pool.read(slots, dtype=torch.float32)
    want = R.stored4(x.cpu())
    assert torch.equal(torch.nan_to_num(k.double().cpu(), nan=12345.0),
                       torch.nan_to_num(want, nan=12345.0))
    assert torch.equal(torch.nan_to_num(v.double().cpu(), nan=12345.0),
                       torch.nan_to_num(-want, nan=12345.0))


def test_strides_and_rows_outside_the_pool():
    n, Hkv, D = 50, 2, 128
    qkv = _randn(3, n, 3 * Hkv * D + 8).to(torch.bfloat16)
    k = qkv[:, 8:8 + Hkv * D].view(n, Hkv, D)
    v = qkv[:, 8 + Hkv * D:8 + 2 * Hkv * D].view(n, Hkv, D)
    odd = _randn(4, n, Hkv, D + 1).to(torch.bfloat16)[..., 1:]     # rows that are not aligned
    turned = _randn(6, n, D, Hkv).to(torch.bfloat16).transpose(1, 2)
    one = _randn(7, 1, Hkv, D).to(torch.bfloat16).expand(n, Hkv, D)
    for a, b in ((k, v), (odd, k), (turned, odd), (one, turned)):
        pool = pool4.Pool4(5, Hkv, D, device=DEV)
        slots = torch.arange(n, device=DEV)
        slots[::7], slots[3] = -1, 5 * 16 + 2
        guard = pool.data.clone()
        pool.write(a, b, slots)
        gk, gv = pool.read(slots, dtype=torch.float32)
        live = (slots >= 0) & (slots < 80)
        for got, x in ((gk, a), (gv, b)):
            assert torch.equal(got[live].double(), R.stored4(x[live]))
            assert (got[~live] == 0).all()
        assert (pool.read(torch.arange(n, 80, device=DEV))[0] == 0).all() and guard.numel()


def test_slots_past_32_bits():
    """A pool of more than 2^31 bytes: the last page's rows."""
    pool = pool4.Pool4(2 ** 31 // (16 * 17 * 64) + 300, 2, 64, page_size=256, device=DEV)
    assert pool.data.numel() > 2 ** 31 * 1.9
    n = pool.n_slots * 256
    slots = torch.tensor([n - 1, 0, n - 256, 5], device=DEV)
    k, v = _randn(1, 4, 2, 64), _randn(2, 4, 2, 64)
    pool.write(k, v, slots)
    gk, gv = pool.read(slots, dtype=torch.float32)
    assert torch.equal(gk.double(), R.stored4(k)) and torch.equal(gv.double(), R.stored4(v))
    q = _randn(3, 1, 2, 1, 64).half()
    table = torch.tensor([[pool.n_slots - 1]], dtype=torch.int32, device=DEV)
    out = pool4.pool4_decode_attention(q, pool, table, torch.tensor([1], dtype=torch.int32, device=DEV))
    assert torch.equal(out[0, :, 0].double(), R.stored4(v[2]).half().double())


# ---- attention ---------------------------------------------------------------------------
def _case(seed, lens, Hq, Hkv, D, S, page, dtype, extra=2):
    pages = [-(-t // page) for t in lens]
    g = torch.Generator().manual_seed(seed)
    n_slots = sum(pages) + extra
    perm = torch.randperm(n_slots, generator=g).to(torch.int32)
    table = torch.full((len(lens), max(pages + [1]) + 1), -1, dtype=torch.int32)
    pool = pool4.Pool4(n_slots, Hkv, D, page_size=page, device=DEV)
    pool.data.random_(0, 256)                   # whatever a page held before
    at, ks, vs = 0, [], []
    for b, (t, p) in enumerate(zip(lens, pages)):
        table[b, :p] = perm[at:at + p]
        at += p
        k, v = _randn(seed + 2 * b, t, Hkv, D), _randn(seed + 2 * b + 1, t, Hkv, D)
        pos = torch.arange(t)
        slots = (table[b][pos // page].long() * page + pos % page).to(DEV)
        pool.write(k, v, slots)
        ks.append(R.stored4(k))
        vs.append(R.stored4(v))
    q = (1.5 * _randn(seed + 99, len(lens), Hq, S, D)).to(dtype)
    return dict(q=q, pool=pool, table=table.to(DEV), lens=torch.tensor(lens, dtype=torch.int32, device=DEV),
                ks=ks, vs=vs)


def _want(c, b, hq, causal, scale, cap=0.0, mask=None):
    q, k, v = c["q"], c["ks"][b], c["vs"][b]
    G, S, t = q.size(1) // k.size(1), q.size(2), k.size(0)
    k, v = k[:, hq // G], v[:, hq // G]
    hidden = None
    if causal:
        hidden = (torch.arange(t, device=DEV)[None, :]
                  > (t - S + torch.arange(S, device=DEV))[:, None])
    m = None
    if mask is not None:
        m = mask[b if mask.size(0) > 1 else 0, hq if mask.size(1) > 1 else 0, :, :t]
    out, _ = R.attend(q[b, hq:hq + 1], k, v, scale, cap, hidden, m)
    size = R.logit_size(q[b, hq], torch.nan_to_num(k, nan=0.0), scale)
    return out[0], size, (v[torch.isfinite(v)].abs().max().item() if t else 0.0)


def _assert_close(c, out, causal=False, scale=None, cap=0.0, mask=None, heads=None):
    B, Hq, S, D = c["q"].shape
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    for b in range(B):
        for hq in heads or range(Hq):
            want, size, vmax = _want(c, b, hq, causal, scale, cap, mask)
            got = out[b, hq].double()
            e = 2.0 ** -16 + (D + 4) * 2.0 ** -24 * size + 2.0 ** -22 * (size + 8)
            tol = HALF[out.dtype] * want.abs() + vmax * (2 * e + c["ks"][b].size(0) * 2.0 ** -24) + 1e-30
            ok = ((got - want).abs() <= tol) | (torch.isnan(got) & torch.isnan(want))
            assert ok.all(), (b, hq, (got - want).abs().max().item(), tol.min().item())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens,Hq,Hkv,D,S,page", [
    ([1], 1, 1, 64, 1, 16), ([17], 8, 8, 128, 1, 16), ([2048], 16, 8, 128, 1, 16),
    ([0, 1, 15, 16, 31, 33], 4, 2, 128, 1, 16), ([300, 0, 4097, 63], 14, 2, 64, 1, 64),
    ([513, 255], 16, 8, 256, 1, 32), ([130, 7], 10, 2, 256, 3, 48), ([1000, 5], 40, 8, 128, 1, 256),
    ([129, 2], 5, 1, 128, 7, 16), ([700], 56, 7, 64, 4, 16), ([9000, 100], 4, 4, 128, 2, 16)])
def test_attention(dtype, lens, Hq, Hkv, D, S, page):
    c = _case(sum(lens) + D, lens, Hq, Hkv, D, S, page, dtype)
    for causal in ((False, True) if S > 1 else (False,)):
        out = pool4.pool4_decode_attention(c["q"], c["pool"], c["table"], c["lens"], causal=causal)
        _assert_close(c, out, causal)


def test_long_context_and_splits():
    c = _case(5, [40000], 8, 2, 128, 1, 16, torch.bfloat16)
    out = pool4.pool4_decode_attention(c["q"], c["pool"], c["table"], c["lens"])
    _assert_close(c, out, heads=[0, 3, 7])


@pytest.mark.parametrize("B,D,t,S", [(16384, 64, 4400, 1), (16384, 256, 4400, 1), (8192, 128, 12350, 1)])
def test_many_sequences_of_long_contexts(B, D, t, S):
    """So many sequences that a split holds more blocks than a wave looks up at once; they
    share one context's pages (a table row expanded) and end at different tokens."""
    c = _case(D, [t], 1, 1, D, S, 16, torch.bfloat16)
    q = (1.5 * _randn(77, B, 1, S, D)).to(torch.bfloat16)
    table = c["table"].expand(B, -1)
    assert table.stride(0) == 0
    lens = (t - torch.arange(B, device=DEV) % 97).to(torch.int32)
    out = pool4.pool4_decode_attention(q, c["pool"], table, lens)
    for b in (0, 1, 50, B // 2, B - 1):
        n = int(lens[b])
        d = dict(q=q[b:b + 1], ks=[c["ks"][0][:n]], vs=[c["vs"][0][:n]])
        _assert_close(d, out[b:b + 1])


@pytest.mark.parametrize("mdt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,S,cap", [(64, 1, 0.0), (128, 1, 30.0), (256, 4, 50.0), (128, 3, 0.0)])
def test_masks_and_softcap(mdt, D, S, cap):
    """A per-head mask with -inf, the type's lowest value and moderate values; a row that
    -inf hides everywhere is zeros, one at the lowest value everywhere the mean of V."""
    lens, Hq, Hkv = [150, 37], 6, 3
    c = _case(D + S, lens, Hq, Hkv, D, S, 16, torch.float16)
    m = (2 * _randn(8, 2, Hq, S, 160)).to(mdt)
    m[:, :, :, 5:20] = -math.inf
    m[:, 1, :, 30:] = torch.finfo(mdt).min
    m[0, 2] = -math.inf
    # the lowest value everywhere (fp32's and bf16's absorb the logits; f16's -65504 does not)
    m[0, 3] = torch.finfo(mdt).min
    out = pool4.pool4_decode_attention(c["q"], c["pool"], c["table"], c["lens"], softcap=cap or None,
                                       attention_mask=m, causal=True)
    assert (out[0, 2] == 0).all()
    # logits are rounded beside the mask: half a step of |logit + mask| in fp32
    heads = [0, 1, 2, 4, 5] if mdt != torch.float16 else [0, 2, 4, 5]
    _assert_close(c, out, True, cap=cap, mask=m, heads=heads)
    if mdt != torch.float16:
        t = 150 - S + 1
        mean = c["vs"][0][:t, 3 // (Hq // Hkv)].mean(0)
        assert ((out[0, 3, 0].double() - mean).abs() <= 2.0 ** -11 * mean.abs() + 1e-5 * 6).all()


def test_mask_broadcasts_strides_and_width():
    c = _case(21, [70, 64], 4, 2, 64, 2, 16, torch.bfloat16)
    wide = _randn(3, 1, 1, 2, 200).float()
    for m in (wide[..., :70], wide[:, :, :1, 9:79], wide.expand(2, 4, 2, 200)[..., 100:170]):
        out = pool4.pool4_decode_attention(c["q"], c["pool"], c["table"], c["lens"], attention_mask=m)
        _assert_close(c, out, mask=m.expand(2, 4, 2, m.size(3)))
    # a mask of fewer columns hides what it does not cover
    out = pool4.pool4_decode_attention(c["q"], c["pool"], c["table"], c["lens"],
                                       attention_mask=wide[..., :33])
    full = torch.full((2, 4, 2, 70), -math.inf, device=DEV)
    full[..., :33] = wide[..., :33]
    _assert_close(c, out, mask=full)


def test_nan_groups_stay_where_they_are_seen():
    """Infinite rows are held as NaN: a visible one shows in the dims of its group (V) or in
    the row (K); hidden ones (mask, causal limit, past the end) show nowhere."""
    lens, S, D = [60], 2, 128
    c = _case(31, lens, 2, 1, D, S, 16, torch.float16)
    k, v = _randn(1, 60, 1, D), _randn(2, 60, 1, D)
    v[10, 0, 40], k[20, 0, 3], v[59, 0, 100], k[59, 0, 0] = math.inf, math.nan, -math.inf, math.inf
    pos = torch.arange(60)
    slots = (c["table"].cpu()[0][pos // 16].long() * 16 + pos % 16).to(DEV)
    c["pool"].write(k, v, slots)
    c["ks"], c["vs"] = [R.stored4(k)], [R.stored4(v)]
    m = torch.zeros(1, 1, 1, 60, device=DEV)
    m[..., 20] = -math.inf
    out = pool4.pool4_decode_attention(c["q"], c["pool"], c["table"], c["lens"], attention_mask=m,
                                       causal=True)
    assert torch.isnan(out[0, :, 0, 32:64]).all() and torch.isnan(out[0, :, 1]).all()
    assert torch.isfinite(out[0, :, 0, :32]).all() and torch.isfinite(out[0, :, 0, 64:]).all()
    m[..., 10] = -math.inf
    out = pool4.pool4_decode_attention(c["q"], c["pool"], c["table"], c["lens"], attention_mask=m,
                                       causal=True)
    want = R.attend(c["q"][0, :, 0:1], c["ks"][0][:59, 0], c["vs"][0][:59, 0], D ** -0.5, mask=m[0, 0, :, :59])[0]
    assert torch.isfinite(out[0, :, 0]).all()
    assert ((out[0, :, 0].double() - want[:, 0]).abs() <= 2.0 ** -11 * want[:, 0].abs() + 1e-3).all()


def test_bad_slots_and_narrow_tables_hide_tokens():
    c = _case(41, [100], 4, 2, 128, 1, 16, torch.bfloat16)
    c["table"][0, 2], c["table"][0, 4] = -1, c["pool"].n_slots
    m = torch.zeros(1, 1, 1, 100, device=DEV)
    m[..., 32:48] = -math.inf
    m[..., 64:80] = -math.inf
    out = pool4.pool4_decode_attention(c["q"], c["pool"], c["table"], c["lens"])
    _assert_close(c, out, mask=m)
    c = _case(42, [100], 4, 2, 128, 1, 16, torch.bfloat16)
    out = pool4.pool4_decode_attention(c["q"], c["pool"], c["table"], c["lens"], max_pages=3)
    c["ks"], c["vs"] = [c["ks"][0][:48]], [c["vs"][0][:48]]
    _assert_close(c, out)
    out = pool4.pool4_decode_attention(c["q"], c["pool"], c["table"], c["lens"], max_pages=0)
    assert (out == 0).all()
    none = pool4.pool4_decode_attention(c["q"][:0], c["pool"], c["table"][:0], c["lens"][:0])
    assert none.shape == (0, 4, 1, 128)


def test_prepared_step_follows_its_operands_and_replays():
    lens = [200, 31]
    c = _case(51, lens, 8, 2, 128, 1, 16, torch.bfloat16)
    step = pool4.prepare_pool4_decode(c["q"], c["pool"], c["table"], c["lens"])
    assert torch.equal(step.run(), pool4.pool4_decode_attention(c["q"], c["pool"], c["table"], c["lens"]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step.run()
    for i in range(3):
        c["q"].copy_((1.5 * _randn(60 + i, 2, 8, 1, 128)).to(torch.bfloat16))
        c["lens"].copy_(torch.tensor([200 - 37 * i, 31 - i], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got = step.out.clone()
        assert torch.equal(got, pool4.pool4_decode_attention(c["q"], c["pool"], c["table"], c["lens"]))
        d = dict(c, ks=[c["ks"][0][:200 - 37 * i], c["ks"][1][:31 - i]],
                 vs=[c["vs"][0][:200 - 37 * i], c["vs"][1][:31 - i]])
        _assert_close(d, got)


def test_calls_on_two_streams():
    """Calls that overlap take a workspace each."""
    a = _case(71, [5000], 8, 2, 128, 1, 16, torch.bfloat16)
    b = _case(72, [4000], 8, 2, 128, 1, 16, torch.bfloat16)
    want = [pool4.pool4_decode_attention(c["q"], c["pool"], c["table"], c["lens"]) for c in (a, b)]
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for _ in range(10):
        for s, c in ((s1, a), (s2, b)):
            with torch.cuda.stream(s):
                outs.append(pool4.pool4_decode_attention(c["q"], c["pool"], c["table"], c["lens"]))
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        assert torch.equal(o, want[i % 2])


def test_a_copied_pool_has_its_own_pages():
    pool = pool4.Pool4(3, 2, 64, device=DEV)
    slots = torch.arange(48, device=DEV)
    k, v = _randn(1, 48, 2, 64), _randn(2, 48, 2, 64)
    pool.write(k, v, slots)
    twin = copy.deepcopy(pool)
    twin.write(v, k, slots)
    for p, a, b in ((pool, k, v), (twin, v, k)):
        rk, rv = p.read(slots, dtype=torch.float32)
        assert torch.equal(rk.double(), R.stored4(a)) and torch.equal(rv.double(), R.stored4(b))


def test_a_prepared_step_dropped_while_it_runs_on_another_stream():
    """Its workspace and output are not handed out again before that stream is done."""
    c = _case(73, [5000], 8, 2, 128, 1, 16, torch.bfloat16)
    want = pool4.pool4_decode_attention(c["q"], c["pool"], c["table"], c["lens"])
    step = pool4.prepare_pool4_decode(c["q"], c["pool"], c["table"], c["lens"])
    ws, at = step._keep[-1].numel(), (step._keep[-1].data_ptr(), step.out.data_ptr())
    assert ws > 0
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        kept = step.run().clone()
    del step
    fresh = [torch.zeros(ws, dtype=torch.uint8, device=DEV), torch.zeros_like(c["q"])]
    running = not side.query()
    assert not running or not set(at) & {t.data_ptr() for t in fresh}
    torch.cuda.synchronize()
    assert torch.equal(kept, want)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("T", [60, 500, 1500])
@pytest.mark.parametrize("mdt", [None, torch.float32, torch.bfloat16])
def test_a_visible_nan_group_counts_however_small_its_weight(dtype, D, T, mdt):
    """One key 153.6 nats above the others (e^-153.6 is no fp32 number), a NaN group of V
    before it and one behind: the formula weighs both, in one split and in several.  A mask's
    lowest finite value hides nothing, -inf does."""
    c = _case(D + T, [T], 2, 1, D, 2, 16, dtype)
    q, k, v = c["q"].zero_(), torch.zeros(T, 1, D, device=DEV), _randn(9, T, 1, D)
    q[..., 0], k[40, 0, 0] = 8.0, 128.0                      # 8 * 128 * 0.15
    v[5, 0, 3], v[T - 8, 0, 40] = math.inf, math.nan         # groups 0 and 1
    v[T - 1, 0, D - 1] = math.nan                            # the last row's alone
    pos = torch.arange(T)
    slots = (c["table"].cpu()[0][pos // 16].long() * 16 + pos % 16).to(DEV)
    c["pool"].write(k, v, slots)
    c["ks"], c["vs"] = [R.stored4(k)], [R.stored4(v)]
    m = None
    if mdt is not None:
        m = torch.zeros(1, 1, 1, T, dtype=mdt, device=DEV)
        m[..., 5] = torch.finfo(mdt).min
    def attend():
        return pool4.pool4_decode_attention(c["q"], c["pool"], c["table"], c["lens"], scale=0.15,
                                            attention_mask=m, causal=True)
    out = attend()
    _assert_close(c, out, True, scale=0.15, mask=m)
    assert torch.isnan(out[..., :64]).all() and torch.isnan(out[0, :, 1, D - 32:]).all()
    if D > 64:
        assert torch.isfinite(out[0, :, 0, 64:]).all() and torch.isfinite(out[0, :, 1, 64:D - 32]).all()
    if m is not None:
        m[..., 5] = m[..., T - 8] = -math.inf
        out = attend()
        _assert_close(c, out, True, scale=0.15, mask=m)
        assert torch.isfinite(out[0, :, 0]).all()


@pytest.mark.parametrize("D,Hkv,page", [(64, 3, 16), (128, 2, 48), (256, 1, 32)])
def test_rows_that_no_slot_names_keep_k_and_v(D, Hkv, page):
    pool = pool4.Pool4(7, Hkv, D, page_size=page, device=DEV)
    rows = 7 * page
    every = torch.arange(rows, device=DEV)
    pool.write(_randn(1, rows, Hkv, D), _randn(2, rows, Hkv, D), every)
    k0, v0 = pool.read(every, dtype=torch.float32)
    before = pool.data.clone()
    slots = _slots(3, 33, 7, page)
    k, v = _randn(4, 33, Hkv, D), _randn(5, 33, Hkv, D)
    pool.write(k[:0], v[:0], slots[:0])
    pool.write(k, v, torch.full_like(slots, -1))
    assert torch.equal(pool.data, before)
    pool.write(k, v, slots)
    k1, v1 = pool.read(every, dtype=torch.float32)
    k0[slots], v0[slots] = R.stored4(k).float(), R.stored4(v).float()
    assert torch.equal(k1, k0) and torch.equal(v1, v0)


@pytest.mark.parametrize("lens,S", [([200, 31], 1), ([5000, 100], 4)])
def test_out_may_be_q(lens, S):
    c = _case(81, lens, 10, 2, 128, S, 16, torch.float16)
    want = pool4.pool4_decode_attention(c["q"], c["pool"], c["table"], c["lens"], causal=True)
    q = c["q"].clone()
    assert pool4.pool4_decode_attention(q, c["pool"], c["table"], c["lens"], causal=True, out=q) is q
    assert torch.equal(q, want)


@pytest.mark.parametrize("D,page", [(64, 2 ** 25), (128, 2 ** 24 + 48), (256, 2 ** 23 + 32)])
def test_one_page_past_32_bits(D, page):
    """A page of more than 2^31 bytes a head: rows before, at and behind that byte, and the last."""
    pool = pool4.Pool4(1, 1, D, page_size=page, device=DEV)
    assert pool.data.numel() > 2 ** 31
    edge = 2 ** 31 // (17 * D) * 16
    slots = torch.tensor([edge - 3, edge + 5, edge + 21, page - 1, 7], device=DEV)
    k, v = torch.zeros(5, 1, D, device=DEV), _randn(2, 5, 1, D)
    k[:, 0, 0] = 128.0
    pool.write(k, v, slots)
    rk, rv = pool.read(slots, dtype=torch.float32)
    assert torch.equal(rk, k) and torch.equal(rv.double(), R.stored4(v))
    # 102 nats above everything else, which holds zeros: its V
    q = torch.zeros(1, 2, 1, D, dtype=torch.bfloat16, device=DEV)
    q[..., 0] = 8.0
    table = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    for i in range(4):
        pool.data.zero_()
        pool.write(k[i:i + 1], v[i:i + 1], slots[i:i + 1])
        n = torch.tensor([int(slots[i]) + 1], dtype=torch.int32, device=DEV)
        out = pool4.pool4_decode_attention(q, pool, table, n, scale=0.1)
        assert torch.equal(out[0, :, 0].double(), R.stored4(v[i]).expand(2, D).bfloat16().double())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("T", [70, 1400])
def test_hidden_tokens_may_hold_any_bytes(dtype, D, T):
    """Tokens inside the sequence that were never written, under -inf or past a row's
    causal limit: any exponent byte, 253 and 254 among them."""
    c = _case(D + T, [T], 2, 1, D, 2, 16, dtype)
    g = torch.Generator(device=DEV).manual_seed(T)
    c["pool"].data.copy_(torch.randint(244, 256, c["pool"].data.shape, generator=g, device=DEV))
    live = torch.arange(3, T - 1, 2)                     # (the second row sees T - 1 under -inf)
    k, v = _randn(1, T, 1, D), _randn(2, T, 1, D)
    slots = (c["table"].cpu()[0][live // 16].long() * 16 + live % 16).to(DEV)
    live = live.to(DEV)
    c["pool"].write(k[live], v[live], slots)
    m = torch.full((1, 1, 2, T), -math.inf, device=DEV)
    m[..., live] = 0.0
    m[:, :, 0, T - 1] = 0.0                              # (hidden by the causal limit)
    c["ks"], c["vs"] = [R.stored4(k)], [R.stored4(v)]
    out = pool4.pool4_decode_attention(c["q"], c["pool"], c["table"], c["lens"], attention_mask=m,
                                       causal=True)
    _assert_close(c, out, True, mask=m)
    assert torch.isfinite(out).all()


def test_the_largest_groups_are_attended():
    """Exponents of 252, the largest that a write leaves, are values and no NaN."""
    c = _case(7, [40], 2, 1, 64, 1, 16, torch.bfloat16)
    k, v = 0 * _randn(1, 40, 1, 64), _randn(2, 40, 1, 64)
    v[17] *= 2.0 ** 126
    v[17, 0, 5], v[17, 0, 40] = 6 * 2.0 ** 125, -6 * 2.0 ** 125
    pos = torch.arange(40)
    slots = (c["table"].cpu()[0][pos // 16].long() * 16 + pos % 16).to(DEV)
    c["pool"].write(k, v, slots)
    out = pool4.pool4_decode_attention(c["q"], c["pool"], c["table"], c["lens"])
    want = R.stored4(v)[:, 0].mean(0)
    # (equal weights: the sum of 40 exact values in fp32, 1 / 40, the output's rounding)
    assert ((out[0, :, 0].double() - want).abs()
            <= 2.0 ** -8 * want.abs() + 45 * 2.0 ** -24 * R.stored4(v).abs().max() / 40).all()
