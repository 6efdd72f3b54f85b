"""The serving operators together, as a serving loop runs them: prompts enter, each step's
lengths become tables and slots on the GPU, K and V go into a 4-bit pool, prompts attend
over their own rows and later tokens over the pool."""
import math
import random

import pytest
import torch

from helm_amd import paged, pool4, prompt
from oracle import serving as R

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.mark.parametrize("dtype,D,page", [(torch.bfloat16, 128, 16), (torch.float16, 64, 32)])
def test_prompts_then_decode_steps(dtype, D, page):
    B, Hq, Hkv, width, steps = 5, 8, 2, 24, 6
    r = random.Random(D)
    prompts = [r.randint(1, 200) for _ in range(B)]
    prompts[2] = page                                  # a page filled to its end
    n_slots = 90
    order = list(range(n_slots))
    r.shuffle(order)
    free = torch.tensor(order, dtype=torch.int32, device=DEV)
    table = torch.zeros((B, width), dtype=torch.int32, device=DEV)
    pool = pool4.Pool4(n_slots, Hkv, D, page_size=page, device=DEV)
    cached = torch.zeros(B, dtype=torch.int32, device=DEV)
    ks, vs = [[] for _ in range(B)], [[] for _ in range(B)]
    u = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
    g = torch.Generator(device=DEV).manual_seed(D)

    def rows(n):
        x = torch.randn((n, Hq + 2 * Hkv, D), generator=g, device=DEV).to(dtype)
        return x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:]

    new = torch.tensor(prompts, dtype=torch.int32, device=DEV)
    n = sum(prompts)
    t = paged.batch_tables(new, cached, table, free, page, n + 3)
    q, k, v = rows(n + 3)                              # three rows of padding
    pool.write(k, v, t.slot_map)
    out = prompt.prompt_attention(q, k, v, t.cu_seqlens)
    assert (out[n:] == 0).all()
    at = 0
    for b, m in enumerate(prompts):
        hid = torch.ones(m, m, dtype=torch.bool, device=DEV).triu(1)
        for h in (0, Hq - 1):
            want, mag = R.attend(q[at:at + m, h][None], k[at:at + m, h // 4], v[at:at + m, h // 4],
                                 D ** -0.5, hidden=hid)
            err = (out[at:at + m, h].double() - want[0]).abs()
            assert (err <= 2.1 * u * (mag[0] + want[0].abs()) + 1e-3 * u).all()
        ks[b], vs[b] = R.stored4(k[at:at + m]), R.stored4(v[at:at + m])
        at += m
    cached = t.seq_lens.clone()

    one = torch.ones(B, dtype=torch.int32, device=DEV)
    for step in range(steps * page // 8):
        free = free[int(t.pages_taken):]
        t = paged.batch_tables(one, cached, table, free, page, B)
        q, k, v = rows(B)
        pool.write(k, v, t.slot_map)
        out = pool4.pool4_decode_attention(q.unsqueeze(2).contiguous(), pool, table, t.seq_lens)
        for b in range(B):
            ks[b], vs[b] = torch.cat([ks[b], R.stored4(k[b:b + 1])]), torch.cat([vs[b], R.stored4(v[b:b + 1])])
            assert int(t.positions[b]) == ks[b].size(0) - 1
            for h in (0, 5):
                want, mag = R.attend(q[b:b + 1, h][None], ks[b][:, h // 4], vs[b][:, h // 4], D ** -0.5)
                err = (out[b, h, 0].double() - want[0, 0]).abs()
                assert (err <= 1.1 * u * want[0, 0].abs() + 2.0 ** -13 * mag[0, 0]).all()
        cached = t.seq_lens.clone()
    # every sequence's rows, read back by the slots its table names
    for b in range(B):
        m = int(cached[b])
        pos = torch.arange(m, device=DEV)
        slots = table[b][pos // page].long() * page + pos % page
        rk, rv = pool.read(slots, dtype=torch.float32)
        assert torch.equal(rk.double(), ks[b]) and torch.equal(rv.double(), vs[b])
    assert math.isfinite(out.float().abs().max().item())


def test_a_captured_step():
    """A decode step of every operator in one graph, replayed with other lengths, tables, free
    slots and tokens: each replay equals the calls made one by one."""
    B, Hq, Hkv, D, page, width, n_slots = 4, 8, 2, 128, 16, 12, 64
    r = random.Random(5)
    g = torch.Generator(device=DEV).manual_seed(5)
    i32 = dict(dtype=torch.int32, device=DEV)
    one, cached = torch.ones(B, **i32), torch.zeros(B, **i32)
    table, free = torch.zeros((B, width), **i32), torch.zeros(n_slots, **i32)
    q = torch.zeros(B, Hq, 1, D, dtype=torch.bfloat16, device=DEV)
    kv = torch.zeros(2, B, Hkv, D, dtype=torch.bfloat16, device=DEV)
    pool = pool4.Pool4(n_slots, Hkv, D, page_size=page, device=DEV)
    t = paged.batch_tables(one, cached, table, free, page, B)
    res = {}

    def step(tables=None):
        tb = paged.batch_tables(one, cached, table, free, page, B, out=tables)
        pool.write(kv[0], kv[1], tb.slot_map)
        k, v = pool.read(tb.slot_map)
        own = prompt.prompt_attention(q[:, :, 0], k, v, tb.cu_seqlens)
        return tb, k, v, own, pool4.pool4_decode_attention(q, pool, table, tb.seq_lens)

    step(t)                                            # (libraries loaded before capture)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res["out"] = step(t)
    for i in range(4):
        slots = list(range(n_slots))
        r.shuffle(slots)
        lens = [r.randint(0, width * page - 1) for _ in range(B)]
        rows, at = [], 0
        for n in lens:
            have = -(-n // page)
            rows.append(slots[at:at + have] + [-1] * (width - have))
            at += have
        pool.data.copy_(torch.randint(0, 100, pool.data.shape, generator=g, device=DEV))
        q.copy_(torch.randn(q.shape, generator=g, device=DEV))
        kv.copy_(torch.randn(kv.shape, generator=g, device=DEV))
        rest = slots[at:] + [0] * at

        def inputs():
            cached.copy_(torch.tensor(lens, **i32))
            table.copy_(torch.tensor(rows, **i32))
            free.copy_(torch.tensor(rest, **i32))
        inputs()
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in (*res["out"][0], *res["out"][1:], table, pool.data)]
        inputs()
        eager = step()
        torch.cuda.synchronize()
        for a, b in zip(got, (*eager[0], *eager[1:], table, pool.data)):
            assert torch.equal(a, b)
        assert torch.equal(got[7], got[6].repeat_interleave(Hq // Hkv, 1))   # a row alone: its V
        assert torch.isfinite(got[8].float()).all()
