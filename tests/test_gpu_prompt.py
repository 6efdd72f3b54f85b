"""prompt_attention against 64 bits.

The bound per element, u the type's half step (bf16 2^-8, f16 2^-11): the output's rounding
u |o|; weights rounded to the type, w' = w (1 + d), |d| <= u, with the sum over w', move a
mean by at most u / (1 - u) sum p |v - o| <= 1.01 u (sum p |v| + |o|); an fp32 logit is off by
(D + 4) 2^-24 L, L the largest sum of its terms' magnitudes, and 2^-22 (L + 8) for its scaling
and exponent, twice that times max|v|; f16 weights end at 2^-34 of the largest, and sums of
T terms in fp32 add T 2^-24 max|v| (far more than their trees do)."""
import math

import pytest
import torch

from helm_amd import prompt
from oracle import serving as R

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _randn(seed, *shape):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(shape, generator=g, device=DEV)


def _cu(lens):
    return torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=DEV)


def _case(seed, n, Hq, Hkv, D, dtype):
    qkv = _randn(seed, n, Hq + 2 * Hkv, D)
    qkv[:, :Hq] *= 1.5
    qkv = qkv.to(dtype)
    return qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]


def _assert_close(out, q, k, v, lens, scale=None, cap=0.0, window=0, heads=None, first=0):
    D, G = q.size(2), q.size(1) // k.size(1)
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    u, at = HALF[out.dtype], first
    for t in lens:
        i = torch.arange(t, device=DEV)
        hidden = i[None, :] > i[:, None]
        if window:
            hidden = hidden | (i[None, :] <= i[:, None] - window)
        for h in heads or range(q.size(1)):
            if not t:
                continue
            qs, ks, vs = q[at:at + t, h], k[at:at + t, h // G], v[at:at + t, h // G]
            want, mag = R.attend(qs[None], ks, vs, scale, cap, hidden)
            want, mag = want[0], mag[0]
            fin = torch.nan_to_num(ks.double(), nan=0.0, posinf=0.0, neginf=0.0)
            size = R.logit_size(qs, fin, scale)
            vmax = vs[torch.isfinite(vs)].abs().max().item()
            e = (D + 4) * 2.0 ** -24 * size + 2.0 ** -22 * (size + 8)
            tol = u * want.abs() + 1.01 * u * (mag + want.abs()) \
                + vmax * (2 * e + t * (2.0 ** -24 + 2.0 ** -34)) + 1e-30
            got = out[at:at + t, h].double()
            ok = ((got - want).abs() <= tol) | (torch.isnan(got) & torch.isnan(want)) | (got == want)
            assert ok.all(), (t, h, (got - want).abs().max().item())
        at += t


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens,Hq,Hkv,D", [
    ([1], 1, 1, 64), ([1, 2, 3], 14, 2, 64), ([31, 32, 33], 4, 4, 128), ([127, 128, 129, 0, 1], 5, 1, 128),
    ([300, 0, 0, 65], 8, 2, 64), ([64, 63, 191], 8, 8, 256), ([257, 40], 6, 3, 256), ([700, 5], 40, 8, 128),
    ([1000], 4, 2, 128), ([0, 0], 2, 1, 64)])
def test_packed_prompts(dtype, lens, Hq, Hkv, D):
    n = sum(lens)
    q, k, v = _case(n + D, n, Hq, Hkv, D, dtype)
    out = prompt.prompt_attention(q, k, v, _cu(lens))
    _assert_close(out, q, k, v, lens)


@pytest.mark.parametrize("D,cap,window,scale", [
    (64, 0.0, 1, None), (64, 30.0, 0, None), (128, 0.0, 70, None), (128, 50.0, 33, 0.2),
    (256, 50.0, 128, None), (256, 0.0, 200, -0.05), (128, 0.0, 1000000, 0.0), (128, 5.0, 64, -0.3),
    (64, 0.0, 129, None), (128, 0.0, 0, -0.1)])
def test_softcap_window_and_scale(D, cap, window, scale):
    lens = [333, 1, 150]
    q, k, v = _case(D + window % 97, sum(lens), 4, 2, D, torch.bfloat16)
    out = prompt.prompt_attention(q, k, v, _cu(lens), scale=scale, softcap=cap or None,
                                  window=window or None)
    _assert_close(out, q, k, v, lens, scale, cap, window)


def test_many_sequences():
    lens = [(i * 37) % 23 for i in range(200)]
    q, k, v = _case(3, sum(lens), 2, 1, 64, torch.float16)
    _assert_close(prompt.prompt_attention(q, k, v, _cu(lens)), q, k, v, lens)


def test_long_prompt():
    q, k, v = _case(9, 9001, 4, 1, 128, torch.bfloat16)
    _assert_close(prompt.prompt_attention(q, k, v, _cu([9001])), q, k, v, [9001], heads=[0, 3])


def test_few_large_logits_against_many_small():
    """One key 17 nats above the others: together they are 2.7e-3 of the row at 65,536."""
    n = 4096
    q = torch.zeros(n, 1, 64, device=DEV).half()
    k = torch.zeros(n, 1, 64, device=DEV).half()
    q[:, 0, 0], k[0, 0, 0] = 8.0, 17.0            # 8 * 17 / 8 = 17
    v = torch.ones(n, 1, 64, device=DEV).half()
    v[0] = 0.0
    out = prompt.prompt_attention(q, k, v, _cu([n]))
    rest = torch.arange(n, device=DEV).double() * math.exp(-17.0)
    want = (rest / (1 + rest))[:, None]
    # (weights rounded to f16's half step, none lost)
    assert ((out[:, 0].double() - want).abs() <= 3 * 2.0 ** -11 * want + 2.0 ** -25).all()


def test_strides_and_rows_outside():
    lens, n = [40, 130], 200
    q, k, v = _case(4, n, 4, 2, 128, torch.bfloat16)
    cu = _cu(lens)
    want = prompt.prompt_attention(q.contiguous(), k.contiguous(), v.contiguous(), cu)
    assert (want[170:] == 0).all()
    _assert_close(want, q, k, v, lens)
    assert torch.equal(prompt.prompt_attention(q, k, v, cu), want)
    heads_first = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]
    assert torch.equal(prompt.prompt_attention(*heads_first, cu), want)
    odd = []
    for x in (q, k, v):                              # rows that are not aligned
        y = torch.zeros(n, x.size(1), 129, dtype=x.dtype, device=DEV)
        y[..., 1:] = x
        odd.append(y[..., 1:])
    assert torch.equal(prompt.prompt_attention(*odd, cu), want)
    assert torch.equal(prompt.prompt_attention(q, k[:, :1].expand(n, 2, 128), v, cu)[:170, :2],
                       want[:170, :2])
    out = torch.full((n, 4, 128), 3.0, dtype=torch.bfloat16, device=DEV)
    assert prompt.prompt_attention(q, k, v, cu, out=out) is out
    assert torch.equal(out[:170], want[:170]) and (out[170:] == 3).all()
    # rows before the first sequence, and no sequence at all
    off = prompt.prompt_attention(q, k, v, cu + 7)
    assert (off[:7] == 0).all() and (off[177:] == 0).all()
    _assert_close(off, q, k, v, lens, first=7)
    assert (prompt.prompt_attention(q, k, v, cu[:1]) == 0).all()
    assert prompt.prompt_attention(q[:0], k[:0], v[:0], cu[:1]).shape == (0, 4, 128)
    # offsets outside the rows are clamped to them
    wild = torch.tensor([0, 40, 10 ** 9], dtype=torch.int32, device=DEV)
    _assert_close(prompt.prompt_attention(q, k, v, wild), q, k, v, [40, 160])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("window", [0, 40])
def test_infinities_and_nan_where_they_are_hidden(dtype, D, window):
    """Every kind of value in K and V, seen by some rows and hidden from others, and in
    the next sequence's rows."""
    lens = [100, 70]
    q, k, v = (x.contiguous() for x in _case(D, 170, 2, 1, D, dtype))
    v[30, 0, 3], v[50, 0, 4], v[60, 0, 5] = math.inf, -math.inf, math.nan
    v[70, 0, 3], v[100, 0, 6] = -math.inf, math.nan
    k[80, 0, 1], q[20, 1, 0] = math.nan, math.inf
    out = prompt.prompt_attention(q, k, v, _cu(lens), window=window or None)
    _assert_close(out, q, k, v, lens, window=window)
    assert torch.isfinite(out[:20, 0]).all() and torch.isnan(out[20, 1]).all()
    assert torch.isfinite(out[30:49, 0, 7]).all() and (out[31, :, 3] == math.inf).all()


# Up to 512 or 640 tiles of 32 rows (times heads; 1,280 for long prompts) a workgroup's waves share a
# tile's keys, beyond each has rows of its own: the same edges on either side.
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens,Hq,Hkv,D,window,cap", [
    ([127, 128, 129, 0, 1, 33], 36, 4, 64, 0, 0.0), ([127, 128, 129, 0, 1, 33], 36, 4, 128, 0, 0.0),
    ([255, 256, 257, 1], 40, 8, 256, 0, 0.0), ([400, 31], 72, 8, 64, 129, 30.0),
    ([400, 31], 72, 8, 128, 33, 30.0), ([400, 31], 72, 8, 256, 97, 30.0),
    ([2500], 2, 1, 64, 0, 0.0), ([2049], 3, 1, 128, 1000, 0.0), ([1, 700, 64], 3, 1, 256, 0, 20.0),
    ([4100], 1, 1, 256, 4000, 0.0), ([97], 8, 2, 128, 96, 0.0)])
def test_either_form(dtype, lens, Hq, Hkv, D, window, cap):
    q, k, v = _case(len(lens) + D, sum(lens), Hq, Hkv, D, dtype)
    out = prompt.prompt_attention(q, k, v, _cu(lens), window=window or None, softcap=cap or None)
    _assert_close(out, q, k, v, lens, cap=cap, window=window, heads=[0, Hq // 2, Hq - 1])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("window", [0, 40])
def test_infinities_and_nan_with_many_heads(dtype, D, window):
    lens, H = [100, 70], 66
    q, k, v = (x.contiguous() for x in _case(D + 1, 170, H, H // 2, D, dtype))
    v[30, :, 3], v[50, :, 4], v[60, :, 5] = math.inf, -math.inf, math.nan
    v[70, :, 3], v[100, :, 6] = -math.inf, math.nan
    k[80, :, 1], q[20, 1, 0] = math.nan, math.inf
    out = prompt.prompt_attention(q, k, v, _cu(lens), window=window or None)
    _assert_close(out, q, k, v, lens, window=window, heads=[0, 1, H - 1])
    assert torch.isfinite(out[:20, 0]).all() and torch.isnan(out[20, 1]).all()
    assert (out[31, :, 3] == math.inf).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("H", [2, 66])
def test_a_visible_infinity_counts_however_small_its_weight(dtype, D, H):
    """One key 150 nats above the others (e^-150 is no fp32 number), an infinity before it
    and one behind it: the formula weighs both."""
    n = 200
    q, k, v = _case(5, n, H, 1, D, dtype)
    q, k, v = torch.zeros_like(q), torch.zeros_like(k), v.contiguous()
    q[:, :, 0], k[40, :, 0] = 8.0, 150.0
    v[5, :, 3], v[70, :, 4] = math.inf, -math.inf
    out = prompt.prompt_attention(q, k, v, _cu([n]), scale=0.125)
    _assert_close(out, q, k, v, [n], scale=0.125, heads=[0, H - 1])
    assert torch.isfinite(out[:5]).all() and (out[5:, :, 3] == math.inf).all()
    assert torch.isfinite(out[:70, :, 4]).all() and (out[70:, :, 4] == -math.inf).all()
    rest = [d for d in range(D) if d not in (3, 4)]
    assert torch.equal(out[40:, 0, rest], v[40, 0, rest].expand(n - 40, D - 2))


def test_captured_call_follows_its_operands():
    n = 160
    q, k, v = (x.contiguous() for x in _case(12, n, 4, 2, 128, torch.bfloat16))
    cu = _cu([90, 70])
    out = torch.zeros(n, 4, 128, dtype=torch.bfloat16, device=DEV)
    prompt.prompt_attention(q, k, v, cu, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        prompt.prompt_attention(q, k, v, cu, out=out)
    for i, lens in enumerate(([90, 70], [1, 159], [160, 0], [100, 33])):
        nq, nk, nv = _case(20 + i, n, 4, 2, 128, torch.bfloat16)
        q.copy_(nq); k.copy_(nk); v.copy_(nv); cu.copy_(_cu(lens))
        out.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[:sum(lens)], prompt.prompt_attention(q, k, v, cu)[:sum(lens)])
        assert (out[sum(lens):] == 7).all()
        _assert_close(out, q, k, v, lens)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("H", [2, 82])
@pytest.mark.parametrize("window", [0, 120])
def test_large_values_without_weight_add_nothing(D, H, window):
    """One key 150 nats above the others and finite values of 1e38 before it and behind: e^-150 of
    them is below half a step of any output.  A NaN that some rows of a tile do not see
    (which makes a workgroup walk twice) changes nothing for those."""
    n = 200
    q, k, v = (x.contiguous() for x in _case(6, n, H, 1, D, torch.bfloat16))
    q.zero_(), k.zero_()
    q[:, :, 0], k[40, :, 0] = 8.0, 150.0
    v[5, :, 3], v[20, :, 7], v[70, :, 4] = 1e38, -1e38, 1e38
    v[110, :, 9] = math.nan
    out = prompt.prompt_attention(q, k, v, _cu([n]), scale=0.125, window=window or None)
    seen = min(n, 40 + window) if window else n              # rows that see token 40
    assert torch.equal(out[40:110], v[40].expand(70, H, D))
    rest = [d for d in range(D) if d != 9]
    assert torch.equal(out[110:seen, :, rest], v[40, :, rest].expand(seen - 110, H, D - 1))
    assert torch.isnan(out[110:, :, 9]).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B", [255, 256, 257, 700])
@pytest.mark.parametrize("Hq,Hkv,D", [(1, 1, 128), (40, 4, 64), (6, 2, 256)])
def test_many_sequences_of_any_number(dtype, B, Hq, Hkv, D):
    """Up to 256 sequences the longest walks come first over the batch, beyond each sequence's
    in turn: empty sequences, one of several tiles in each window of 64, rows outside."""
    lens = [(i * 37) % 5 for i in range(B)]
    lens[3], lens[70], lens[140], lens[B - 1] = 300, 0, 129, 257
    n, first = sum(lens), 9
    q, k, v = _case(B + D, first + n + 70, Hq, Hkv, D, dtype)
    cu = _cu(lens) + first
    out = prompt.prompt_attention(q, k, v, cu)
    _assert_close(out, q, k, v, lens, first=first, heads=[0, Hq - 1])
    assert (out[:first] == 0).all() and (out[first + n:] == 0).all()
    kept = torch.full_like(out, 3.0)
    prompt.prompt_attention(q, k, v, cu, out=kept)
    assert torch.equal(kept[first:first + n], out[first:first + n])
    assert (kept[:first] == 3).all() and (kept[first + n:] == 3).all()


@pytest.mark.parametrize("heads", [2, 40])
def test_more_sequences_than_rows(heads):
    """300 empty sequences: every row is outside."""
    q, k, v = _case(1, 150, heads, 1, 64, torch.bfloat16)
    cu = torch.full((301,), 60, dtype=torch.int32, device=DEV)
    assert (prompt.prompt_attention(q, k, v, cu) == 0).all()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("lens,Hq,Hkv", [([333, 1, 150], 4, 2), ([700, 400], 40, 8)])
def test_out_may_be_q(D, lens, Hq, Hkv):
    n = sum(lens) + 5
    q, k, v = (x.contiguous() for x in _case(D, n, Hq, Hkv, D, torch.bfloat16))
    v[100, :, 3] = math.nan                     # (some workgroups walk twice)
    want, rest = prompt.prompt_attention(q, k, v, _cu(lens)), q[sum(lens):].clone()
    assert prompt.prompt_attention(q, k, v, _cu(lens), out=q) is q
    same = (q == want) | (torch.isnan(q) & torch.isnan(want))
    assert same[:sum(lens)].all() and torch.equal(q[sum(lens):], rest)
