"""prefix_decode_attention at its edges, against 64 bits: what its roundings are."""
import math

import pytest
import torch

from oracle import serving as R
from test_gpu_prefix import BF, DEV, HALF, HF, call, make

pytestmark = pytest.mark.gpu


def _attend(c, r, h):
    """Sequence r's row h in 64 bits, and the mean of |v| under its weights."""
    Hq, D = c["q"].size(1), c["q"].size(3)
    t, page = c["lens"][r], c["page"]
    kv = c["arena"][c["table"][r, :-(-t // page)].long(), :, h // (Hq // c["arena"].size(2))]
    k, v = (kv[:, i].reshape(-1, D)[:t] for i in (0, 1))
    want, mag = R.attend(c["q"][r, h][None], k, v, c["scale"])
    return want[0, 0], mag[0, 0]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_weights_are_held_in_two_parts(dtype, D):
    """An output is off by its own rounding and hardly more.  q and k of -1, 0, 1 and a scale that
    is a power of two: logits are exact.  Weights are off by at most w of themselves: u^2, their
    second part's rounding; 2^-24 3 L, L the largest logit, for log2(e) in fp32 and the exponent's
    rounding; 2^-24 16 for exponentials, the joining's among them.  The mean is then off by
    d <= 2 w (mean |v| + |o|); where that changes its rounding, the value was within d of the
    middle, so each error is at most its rounding's + 2 d, and so are their norms."""
    c = make([(1, [16 + n for n in range(1, 25)]), (2, [32 + n for n in range(8)])], 8, 2, D, 16,
             dtype, seed=D)
    g = torch.Generator(device=DEV).manual_seed(D + 1)
    for x in (c["q"], c["arena"][:, 0]):
        x.copy_(torch.randint(-1, 2, x.shape, generator=g, device=DEV).float())
    c["scale"] = 2.0 ** -round(math.log2(D) / 2 + 2)
    out = call(c, scale=c["scale"])
    rows = [(r, h) for r in range(out.size(0)) for h in range(8)]
    want, mag = (torch.stack(x) for x in zip(*(_attend(c, r, h) for r, h in rows)))
    got = torch.stack([out[r, h, 0] for r, h in rows]).double()
    largest = max(R.logit_size(c["q"][r], c["arena"][:, 0].reshape(-1, D), c["scale"])
                  for r in range(out.size(0)))
    u = HALF[dtype]
    d = 2 * (u * u + 2.0 ** -24 * (3 * largest + 16)) * (mag + want.abs())
    rounding = (want.to(dtype).double() - want).norm()
    assert (got - want).norm() <= rounding + 2 * d.norm()


def _tolerance(q, k, v, want, mag, scale, u):
    """Roundings of the output and the weights, of the logits' products in fp32 and of sums."""
    size = R.logit_size(q, k, scale)
    e = (q.size(-1) + 4) * 2.0 ** -24 * size + 2.0 ** -22 * (size + 8)
    return u * want.abs() + 2 * u * u * (mag + want.abs()) \
        + v.abs().max().item() * (2 * e + v.size(0) * (2.0 ** -24 + 2.0 ** -34)) + 1e-30


@pytest.mark.parametrize("dtype,D", [(BF, 128), (HF, 64)])
@pytest.mark.parametrize("S", [1, 4])
@pytest.mark.parametrize("window", [0, 20, 96])
def test_lengths_past_the_table_keep_their_rows_positions(dtype, D, S, window):
    """Row s stands at len - S + s though the table ends before: it sees the table's tokens up
    to there, and with a window only those that are not too far behind."""
    page, room = 16, 96
    c = make([(4, [150, 98, 97, 96, 96, 150]), (0, [150, 95])], 4, 2, D, page, dtype, S=S, seed=S)
    lens = [150, 98, 97, 96, 73, 2 ** 31 - 1, 96 + 19, 95]
    c["len_t"].copy_(torch.tensor(lens, dtype=torch.int32))
    out = call(c, max_pages=room // page, window=window)
    for r, t in enumerate(lens):
        kv = c["arena"][c["table"][r, :room // page].long()]
        pos = t - S + torch.arange(S, device=DEV)[:, None]
        j = torch.arange(room, device=DEV)[None, :]
        hidden = j > pos
        if window:
            hidden = hidden | (j <= pos - window)
        for h in range(4):
            k, v = (kv[:, i, h // 2].reshape(-1, D) for i in (0, 1))
            scale = D ** -0.5
            want, mag = (x[0] for x in R.attend(c["q"][r, h][None], k, v, scale, 0.0, hidden))
            tol = _tolerance(c["q"][r, h], k, v, want, mag, scale, HALF[dtype])
            assert ((out[r, h].double() - want).abs() <= tol).all(), (r, h)
            assert (out[r, h][hidden.all(-1)] == 0).all()


@pytest.mark.parametrize("window", [37, 100, 333])
@pytest.mark.parametrize("nothing", [0, -7, 3000])
def test_a_sequence_that_sees_nothing_leaves_its_groups_walk_alone(nothing, window):
    """Its group's others get the same answer, bit for bit, as without it: nothing in front of
    their windows, or behind them, is walked for its sake (its own window may lie past the table)."""
    c = make([(60, [960 + n for n in (5, 60, 130)])], 16, 8, 128, 16, HF, seed=31)
    c["len_t"][1:3] = torch.tensor([700, 650], dtype=torch.int32)
    want = call(c, window=window)
    d = dict(c, q=torch.cat([c["q"], c["q"][:1]]), table=torch.cat([c["table"], c["table"][:1]]),
             len_t=torch.cat([c["len_t"], torch.full_like(c["len_t"][:1], nothing)]),
             start_t=torch.tensor([0, 4], dtype=torch.int32, device=DEV))
    got = call(d, window=window)
    assert torch.equal(got[:3], want) and (got[3] == 0).all()
