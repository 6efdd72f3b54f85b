"""Beam selection and beam tables at their edges: sums that 64 bits do not tell apart."""
import math

import pytest
import torch

from test_gpu_beams import DEV, check_select, randn

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
