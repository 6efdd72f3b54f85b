"""A beam search as a program runs it, over two layers' paged arenas: prompts fanned out to beams,
beam_select, beam_tables with its copies, batch_tables for the next token's pages, K and V
written, prefix_decode_attention; every step against the beams' own histories in 64 bits.

Tolerances: those of one call of each operator (test_gpu_prefix.py, test_gpu_beams.py); a step's
operands are the same 16-bit rows on both sides, so nothing grows over the steps."""
import math
import random

import pytest
import torch

from helm_amd import beams, paged, pool4, prefix
from oracle import beams as RB
from oracle import serving as RS

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
I32 = dict(dtype=torch.int32, device=DEV)
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def randn(seed, shape, dtype=torch.float32):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(shape, generator=g, device=DEV).to(dtype)


@pytest.mark.parametrize("dtype,Hq,Hkv,D,page,K,window", [
    (torch.bfloat16, 4, 2, 64, 16, 4, None), (torch.float16, 8, 1, 128, 32, 3, None),
    (torch.bfloat16, 2, 2, 256, 16, 2, 30)])
def test_beam_search(dtype, Hq, Hkv, D, page, K, window):
    prompts, L, V, steps, n_slots = [5, 2 * page, 2 * page + 5], 2, 61, 2 * page + 3, 160
    B, R, u, scale = len(prompts), len(prompts) * K, HALF[dtype], 1.0 / math.sqrt(D)
    width = -(-(max(prompts) + steps + 1) // page)
    kv = [randn(i, (V, 2, Hkv, D), dtype) for i in range(L)]        # a token's K and V
    turn = [randn(10 + i, (256, Hkv, D), dtype) for i in range(L)]  # and its position's share of K
    embed, head = randn(20, (V, Hq, D), dtype), randn(21, (Hq * D, V)) / math.sqrt(Hq * D)

    def rows(layer, tokens, positions):
        x = kv[layer][tokens].clone()
        x[:, 0] += turn[layer][positions]
        return x
    free = list(range(n_slots))
    random.Random(0).shuffle(free)
    arenas = [torch.full((n_slots, 2, Hkv, page, D), math.nan, dtype=dtype, device=DEV)
              for _ in range(L)]
    store = beams.PageStore(arenas)

    def write(layer, slots, x):
        arenas[layer][slots // page, :, :, slots % page] = x
    # the prompts, cached by row 0 of each request; its beams name its full pages, and have a
    # free page each where the last one is part-filled
    r = random.Random(1)
    table, told = torch.zeros((R, width), **I32), []
    for b, n in enumerate(prompts):
        tokens = [r.randrange(V) for _ in range(n)]
        own = [free.pop() for _ in range(-(-n // page))]
        for j in range(K):
            told.append(list(tokens))
            names = list(own) if j == 0 or n % page == 0 else own[:-1] + [free.pop()]
            table[b * K + j, :len(names)] = torch.tensor(names, **I32)
        at = torch.arange(n, device=DEV)
        slots = torch.tensor(own, device=DEV)[at // page] * page + at % page
        for i in range(L):
            write(i, slots, rows(i, torch.tensor(tokens, device=DEV), at))
    shared = torch.tensor([n // page for n in prompts], **I32)
    starts = torch.arange(0, R + 1, K, **I32)
    lens = torch.tensor([n for n in prompts for _ in range(K)], **I32)
    ones = torch.ones(R, **I32)
    scores = torch.full((B, K), -math.inf, device=DEV)
    scores[:, 0] = 0.0
    logits = randn(30, (B, K, V))
    for i in range(steps):
        choice = beams.beam_select(logits, scores)
        want, tok, par = RB.select(logits, scores, K)
        assert torch.equal(choice.tokens.cpu(), tok)
        assert torch.equal(choice.parents.cpu().long(), par)
        assert ((choice.scores.cpu().double() - want).abs()
                <= 2.0 ** -21 + 2.0 ** -24 * want.abs()).all()
        scores = choice.scores
        t = beams.beam_tables(choice.parents, table, lens, page, shared_pages=shared, pages=store)
        free += t.released[:int(t.n_released)].tolist()
        assert len(set(free)) == len(free)
        table = t.page_table
        told = [told[b * K + int(par[b, j])] + [int(tok[b, j])]
                for b in range(B) for j in range(K)]
        s = paged.batch_tables(ones, lens, table, torch.tensor(free[::-1], **I32), page, R)
        taken = int(s.pages_taken)
        free = free[:len(free) - taken]
        lens = s.seq_lens
        new = choice.tokens.flatten()
        x = embed[new]
        for layer in range(L):
            write(layer, s.slot_map, rows(layer, new, s.positions))
            q = x[:, :, None].contiguous()
            k_pool, v_pool = arenas[layer][:, 0], arenas[layer][:, 1]
            out = prefix.prefix_decode_attention(q, k_pool, v_pool, table, lens, starts, shared,
                                                 window=window)
            if i in (0, 1, page, steps - 1):
                for row, tokens in enumerate(told):
                    n = len(tokens)
                    assert n == int(lens[row])
                    at = torch.arange(n, device=DEV)
                    own = rows(layer, torch.tensor(tokens, device=DEV), at)
                    hidden = (at <= n - 1 - window)[None] if window else None
                    for h in range(Hq):
                        k, v = own[:, 0, h // (Hq // Hkv)], own[:, 1, h // (Hq // Hkv)]
                        want, mag = RS.attend(q[row, h][None], k, v, scale, hidden=hidden)
                        size = RS.logit_size(q[row, h], k, scale)
                        e = (D + 4) * 2.0 ** -24 * size + 2.0 ** -22 * (size + 8)
                        tol = u * want.abs() + 1.01 * u * (mag + want.abs()) \
                            + v.abs().max().item() * (2 * e + n * (2.0 ** -24 + 2.0 ** -34))
                        off = (out[row, h].double() - want[0]).abs()
                        assert (off <= tol[0]).all(), (i, row, h)
            x = out[:, :, 0]
        logits = torch.matmul(x.flatten(1).float(), head).view(B, K, V) * 4
    # every page is free or named, once
    named = {int(p) for row in range(R) for p in table[row, :-(-int(lens[row]) // page)]}
    assert named | set(free) == set(range(n_slots)) and not named & set(free)


def test_a_step_in_a_graph():
    """Attention, choice, tables and copies of one step, captured and replayed over new states."""
    B, K, Hq, Hkv, D, page, V, n = 2, 4, 4, 2, 128, 16, 5000, 90
    R, width = B * K, 9
    head = randn(1, (Hq * D, V)) / math.sqrt(Hq * D)
    q = torch.zeros((R, Hq, 1, D), dtype=torch.bfloat16, device=DEV)
    arena = torch.zeros((n, 2, Hkv, page, D), dtype=torch.bfloat16, device=DEV)
    packed = pool4.Pool4(n, Hkv, D, page_size=page, device=DEV)
    table, lens = torch.zeros((R, width), **I32), torch.zeros(R, **I32)
    scores, shared = torch.zeros((B, K), device=DEV), torch.zeros(B, **I32)
    starts = torch.tensor([0, K, 2 * K], **I32)

    def fresh():
        return beams.BeamTables(torch.zeros((R, width), **I32), torch.zeros((R, 2), **I32),
                                torch.full((R * width,), -9, **I32), torch.zeros(1, **I32))

    def step(q, arena, packed, table, out, attend):
        x = attend()
        logits = torch.matmul(x.flatten(1).float(), head).view(B, K, V)
        choice = beams.beam_select(logits, scores)
        a = beams.beam_tables(choice.parents, table, lens, page, shared_pages=shared,
                              pages=beams.PageStore([arena]), out=out)
        # (the same copies again, in the 4-bit pool)
        b = beams.beam_tables(choice.parents, table, lens, page, shared_pages=shared,
                              pages=beams.PageStore([packed]))
        return x, *choice, *a, *b[:2]

    def state(seed):
        r = random.Random(seed)
        q.copy_(randn(seed, q.shape))
        arena.copy_(randn(seed + 1, arena.shape))
        packed.data.copy_(torch.randint(0, 128, packed.data.shape, device=DEV, dtype=torch.uint8))
        scores.copy_(-torch.rand((B, K), device=DEV))
        slots = list(range(n))
        r.shuffle(slots)
        lengths = [r.randint(1, (width - 1) * page), r.choice([0, page, 3 * page + 1])]
        lens.copy_(torch.tensor([t for t in lengths for _ in range(K)], **I32))
        for b, t in enumerate(lengths):
            same = r.randint(0, t // page)
            shared[b] = same
            own = [slots.pop() for _ in range(t // page)]
            for j in range(K):
                names = own + [slots.pop()] * (t % page != 0)
                table[b * K + j, :len(names)] = torch.tensor(names, **I32)

    prepared = prefix.prepare_prefix_decode(q, arena[:, 0], arena[:, 1], table, lens, starts,
                                            shared)
    held = fresh()
    state(100)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(q, arena.clone(), packed, table, fresh(), prepared.run)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(q, arena, packed, table, held, prepared.run)
    for seed in (200, 300, 400, 500):
        state(seed)
        pages, four = arena.clone(), pool4.Pool4(n, Hkv, D, page_size=page, device=DEV)
        four.data.copy_(packed.data)
        held.released.fill_(-9)
        want = step(q, pages, four, table, fresh(), lambda: prefix.prefix_decode_attention(
            q, pages[:, 0], pages[:, 1], table, lens, starts, shared))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        assert torch.equal(arena, pages) and torch.equal(packed.data, four.data)
