"""What the beam operators refuse: argument checks of the Python entry points and of the C-ABI
(which return before any device work), and the restatements' own properties."""
import ctypes
import math

import numpy as np
import pytest
import torch

from helm_amd import _native, beams, pool4
from helm_amd.runtime import engine
from oracle import beams as R

I32, I64, F32 = torch.int32, torch.int64, torch.float32


def _select(B=2, K=3, V=8, **kw):
    return dict(dict(logits=torch.zeros((B, K, V)), scores=torch.zeros((B, K))), **kw)


@pytest.mark.parametrize("bad,err", [
    (dict(logits=torch.zeros((6, 8))), ValueError),
    (dict(scores=torch.zeros((2, 4))), ValueError),
    (dict(logits=torch.zeros((2, 3, 8), dtype=torch.float64)), TypeError),
    (dict(logits=torch.zeros((2, 3, 8), dtype=I32)), TypeError),
    (dict(scores=torch.zeros((2, 3), dtype=torch.bfloat16)), TypeError),
    (dict(scores=torch.zeros((3, 2)).t()), ValueError),
    (dict(n=0), ValueError), (dict(n=65), ValueError),
    (dict(logits=torch.zeros((2, 65, 8)), scores=torch.zeros((2, 65))), ValueError),
    (dict(logits=torch.zeros((2, 3, 0))), ValueError),
    (dict(logits=torch.zeros((1, 1)).expand(65536, 1, 1), scores=torch.zeros((65536, 1))),
     ValueError),
    (dict(logits=torch.zeros((2, 3, 8), requires_grad=True)), RuntimeError),
    ({}, RuntimeError),            # CPU tensors
])
def test_select_refusals(bad, err):
    with pytest.raises(err):
        beams.beam_select(**_select(**bad))


def test_select_out_refusals(monkeypatch):
    good = beams.BeamChoice(torch.zeros((2, 3)), torch.zeros((2, 3), dtype=I64),
                            torch.zeros((2, 3), dtype=I32))
    for bad in (good._replace(scores=torch.zeros((2, 4))),
                good._replace(tokens=torch.zeros((2, 3), dtype=I32)),
                good._replace(parents=torch.zeros((3, 2), dtype=I32).t())):
        with pytest.raises(ValueError):
            beams.beam_select(**_select(), out=bad)
    monkeypatch.setattr(engine, "common_device", lambda *a: 0)
    a = _select()
    buf = torch.zeros(12)
    for bad in (good._replace(scores=a["scores"]),                  # read until the last row is
                good._replace(scores=a["logits"].view(-1)[40:46].view(2, 3)),
                good._replace(scores=buf[:6].view(2, 3), parents=buf.view(I32)[5:11].view(2, 3))):
        with pytest.raises(ValueError, match="lies over"):
            beams.beam_select(**a, out=bad)


def test_select_out_over_logits_that_are_copied_first(monkeypatch):
    """Their own memory is the operand, not the copy's."""
    monkeypatch.setattr(engine, "common_device", lambda *a: 0)
    buf = torch.zeros(48)
    out = beams.BeamChoice(buf[10:16].view(2, 3), torch.zeros((2, 3), dtype=I64),
                           torch.zeros((2, 3), dtype=I32))
    with pytest.raises(ValueError, match="lies over"):
        beams.beam_select(buf.view(2, 8, 3).transpose(1, 2), torch.zeros((2, 3)), out=out)


def _tables(B=2, K=3, W=4, **kw):
    return dict(dict(parents=torch.zeros((B, K), dtype=I32),
                     page_table=torch.zeros((B * K, W), dtype=I32),
                     seq_lens=torch.zeros(B * K, dtype=I32), page_size=16), **kw)


@pytest.mark.parametrize("bad,err", [
    (dict(parents=torch.zeros((2, 3), dtype=I64)), TypeError),
    (dict(page_table=torch.zeros((6, 4), dtype=I64)), TypeError),
    (dict(seq_lens=torch.zeros(6, dtype=I64)), TypeError),
    (dict(parents=torch.zeros(6, dtype=I32)), ValueError),
    (dict(parents=torch.zeros((3, 2), dtype=I32).t()), ValueError),
    (dict(page_table=torch.zeros((5, 4), dtype=I32)), ValueError),
    (dict(page_table=torch.zeros((4, 6), dtype=I32).t()), ValueError),
    (dict(page_table=torch.zeros((1, 4), dtype=I32).expand(6, 4)), ValueError),
    (dict(seq_lens=torch.zeros(2, dtype=I32)), ValueError),
    (dict(seq_lens=torch.zeros(12, dtype=I32)[::2]), ValueError),
    (dict(page_size=0), ValueError),
    (dict(shared_pages=torch.zeros(2, dtype=I64)), TypeError),
    (dict(shared_pages=torch.zeros(6, dtype=I32)), ValueError),
    (dict(parents=torch.zeros((1, 65), dtype=I32), page_table=torch.zeros((65, 4), dtype=I32),
          seq_lens=torch.zeros(65, dtype=I32)), ValueError),
    (dict(pages=beams.PageStore([torch.zeros(4, 2, 32, 8)])), ValueError),     # 32, not 16
    (dict(out=beams.BeamTables(torch.zeros((6, 4), dtype=I32), torch.zeros((6, 2), dtype=I32),
                               torch.zeros(23, dtype=I32), torch.zeros(1, dtype=I32))), ValueError),
    (dict(out=beams.BeamTables(torch.zeros((6, 4), dtype=I64), torch.zeros((6, 2), dtype=I32),
                               torch.zeros(24, dtype=I32), torch.zeros(1, dtype=I32))), ValueError),
    ({}, RuntimeError),            # CPU tensors
])
def test_tables_refusals(bad, err):
    with pytest.raises(err):
        beams.beam_tables(**_tables(**bad))


@pytest.mark.parametrize("bad", [
    [], [torch.zeros(4, 16)], [torch.zeros(4, 2, 16, 8), torch.zeros(4, 2, 16, 4)],
    [torch.zeros(4, 2, 16, 8), torch.zeros(4, 2, 16, 8).half()],
    [torch.zeros(4, 2, 16, 8), torch.zeros(8, 2, 16, 8)[::2]],
    [torch.zeros(4, 2, 8, 16).transpose(2, 3)], [torch.zeros(4, 2, 16, 16)[..., :8]],
    [torch.zeros(4, 3, 2, 16, 8)[:, :, :1].expand(4, 3, 2, 16, 8)],       # parts over each other
    [torch.zeros(4, 3, 5, 16, 8)[:, :, ::2]],                             # no one stride
    [torch.zeros(1, 2, 16, 8).expand(4, 2, 16, 8)],                       # pages over each other
    [torch.zeros(4, 2, 16, 0)],
    [pool4.Pool4(4, 2, 64, device="cpu"), pool4.Pool4(4, 2, 64, device="cpu").data],
])
def test_page_store_refusals(bad):
    with pytest.raises(ValueError):
        beams.PageStore(bad)


def test_page_store_layouts():
    """(slots, bytes between slots, segments, bytes between them, tokens and bytes of a unit)"""
    assert beams.PageStore([torch.zeros(5, 2, 3, 16, 8)])._shape == (5, 768 * 4, 6, 512, 1, 32)
    a = torch.zeros(5, 2, 3, 16, 8).half()
    assert beams.PageStore([a[:, 0], a[:, 1]])._shape == (5, 1536, 3, 256, 1, 16)
    assert beams.PageStore([torch.zeros(5, 16, 8).half()])._shape == (5, 256, 1, 256, 1, 16)
    p = pool4.Pool4(5, 2, 64, page_size=32, device="cpu")
    s = beams.PageStore([p])
    assert s._shape == (5, 2 * 2 * 17 * 64, 2, 2 * 17 * 64, 16, 17 * 64) and s.page_size == 32


def test_page_store_takes_every_layout_without_overlaps():
    """Slots, parts and strides: refused exactly where two parts share an element."""
    heads = torch.zeros(2, 3, 5, 16, 8).half()                  # [K and V, heads, slots, page, D]
    assert beams.PageStore([heads[0].transpose(0, 1)])._shape == (5, 256, 3, 1280, 1, 16)
    assert beams.PageStore([heads.permute(2, 0, 1, 3, 4)])._shape == (5, 256, 6, 1280, 1, 16)
    for n in (1, 2, 4):
        for segs in (1, 2, 3):
            for slot in range(0, 13):
                for step in range(0, 13):
                    t = torch.zeros(64).as_strided((n, segs, 1, 4), (slot, step, 4, 1))
                    at = [i * slot + j * step + d for i in range(n) for j in range(segs)
                          for d in range(4)]
                    if len(set(at)) == len(at):
                        beams.PageStore([t])
                    else:
                        with pytest.raises(ValueError):
                            beams.PageStore([t])


def _i32(n):
    a = np.zeros(max(1, n), dtype=np.int32)
    return a, a.ctypes.data


def test_c_entries_refuse_before_device_work():
    lib = _native.load()
    f = np.zeros(4096, dtype=np.float32)
    at, E = f.ctypes.data, (_native.HELM_E_INVALID, _native.HELM_E_UNSUPPORTED,
                            _native.HELM_E_WORKSPACE)

    def select(logits=at, bs=24, ks=8, dt=2, scores=at, B=2, K=3, V=8, n=3, o=at, ws=at, nb=4096):
        return lib.helm_beam_select(logits, bs, ks, dt, scores, B, K, V, n, o, o, o, ws, nb, None)
    assert select(dt=7) == E[1]
    for kw in (dict(K=0), dict(K=65), dict(n=0), dict(n=65), dict(V=0), dict(B=-1), dict(B=30000),
               dict(bs=-1), dict(logits=None), dict(scores=None), dict(o=None),
               dict(logits=at + 2)):
        assert select(**kw) == E[0], kw
    for kw in (dict(ws=None), dict(nb=8), dict(ws=at + 4)):
        assert select(**kw) == E[2], kw
    assert select(B=0) == 0
    assert lib.helm_beam_select_workspace_bytes(2, 3, 8, 3, 2) == 6 * (12 + 24)
    assert lib.helm_beam_select_workspace_bytes(2, 0, 8, 3, 2) == 0

    sizes = dict(par=6, tab=24, lens=6, new=24, cop=12, rel=24, cnt=1)
    arr = {k: _i32(n) for k, n in sizes.items()}
    ptr = {k: v[1] for k, v in arr.items()}
    need = lib.helm_beam_tables_workspace_bytes(2, 3, 4)
    ws = np.zeros(need // 4, dtype=np.int32)
    pool = (ctypes.c_void_p * 1)(at)

    def tables(B=2, K=3, W=4, ts=4, ns=4, page=16, pools=None, n=0, geo=(4, 64, 2, 32, 1, 2),
               wsp=ws.ctypes.data, nb=need, **kw):
        p = dict(ptr, **kw)
        return lib.helm_beam_tables(p["par"], B, K, p["tab"], ts, W, p["lens"], page, None,
                                    p["new"], ns, p["cop"], p["rel"], p["cnt"], pools, n, *geo,
                                    wsp, nb, None)
    for kw in (dict(K=0), dict(K=65), dict(B=-1), dict(W=-1), dict(ts=3), dict(ns=3), dict(page=0),
               dict(par=None), dict(tab=None), dict(lens=None), dict(new=None), dict(cop=None),
               dict(rel=None), dict(cnt=None), dict(n=-1), dict(n=1),
               dict(n=1, pools=pool, geo=(-1, 64, 2, 32, 1, 2)),
               dict(n=1, pools=pool, geo=(4, 64, 0, 32, 1, 2)),
               dict(n=1, pools=pool, geo=(4, 64, 2, 16, 1, 2)),        # segments over each other
               dict(n=1, pools=pool, geo=(4, 64, 2, 2 ** 31, 1, 2 ** 30))):
        assert tables(**kw) == E[0], kw
    for kw in (dict(wsp=None), dict(nb=need - 4)):
        assert tables(**kw) == E[2], kw
    # an output over an operand, byte by byte; the table may be its own
    tab = ptr["tab"]
    for kw in (dict(cop=tab), dict(rel=ptr["par"]), dict(new=tab + 4), dict(cnt=tab + 92),
               dict(cop=ptr["lens"]), dict(rel=ptr["cop"]), dict(cnt=ptr["new"] + 20),
               dict(new=tab, ns=5)):
        assert tables(**kw) == E[0], kw
        assert b"lies over" in lib.helm_last_error_string()


def _tables_call(pools, n_slots=4, slot=64, **kw):
    """helm_beam_tables of 2 x 3 beams with 4 columns over `pools`, of 2 segments of 16 tokens of 2
    bytes a page; kw: addresses to take instead of the operands' own."""
    lib = _native.load()
    sizes = dict(par=6, tab=24, lens=6, new=24, cop=12, rel=24, cnt=1, ws=0)
    sizes["ws"] = lib.helm_beam_tables_workspace_bytes(2, 3, 4) // 4
    arr = {k: np.zeros(n, dtype=np.int32) for k, n in sizes.items()}
    p = dict({k: a.ctypes.data for k, a in arr.items()}, **kw)
    return lib.helm_beam_tables(p["par"], 2, 3, p["tab"], 4, 4, p["lens"], 16, None, p["new"], 4,
                                p["cop"], p["rel"], p["cnt"],
                                (ctypes.c_void_p * len(pools))(*pools), len(pools), n_slots, slot, 2,
                                32, 1, 2, p["ws"], 4 * sizes["ws"], None)


def test_a_null_pool_is_refused_before_device_work():
    """With the other arguments (the workspace is looked at last)."""
    at = np.zeros(256, dtype=np.uint8)
    pools = [at.ctypes.data] * 130 + [None]
    assert _tables_call(pools, ws=None) == _native.HELM_E_INVALID
    assert b"null pool" in _native.load().helm_last_error_string()
    assert _tables_call(pools[:130], ws=None) == _native.HELM_E_WORKSPACE
    assert _tables_call([None], n_slots=0, ws=None) == _native.HELM_E_WORKSPACE


def test_sizes_past_32_bits_are_refused():
    """And not cut to what is left of them."""
    logits = torch.zeros((1, 1, 1)).expand(1, 1, 2 ** 32 + 5)
    for x in (logits, logits[..., :2 ** 31]):
        with pytest.raises(ValueError, match="logits"):
            beams.beam_select(x, torch.zeros((1, 1)))
    for shape in ((1, 2 ** 32 + 1, 1, 1), (2, 2 ** 20, 16, 128)):
        with pytest.raises(ValueError, match="2.31"):
            beams.PageStore([torch.zeros(shape, dtype=torch.uint8, device="meta")])
    lib = _native.load()
    for V, n in ((2 ** 31 - 1, 64), (2 ** 31 - 2048, 1)):
        chunks = -(-V // 8192)
        assert lib.helm_beam_select_workspace_bytes(1, 1, V, n, 1) == chunks * (12 + 8 * n)
    assert lib.helm_beam_select_workspace_bytes(1, 64, 2 ** 31 - 1, 64, 1) == 0


def test_operands_over_a_pool_are_refused():
    """Read or written, in any part of any page: pages of 64 bytes, 128 apart, from byte 1024 on."""
    buf = np.zeros(512, dtype=np.int32)
    at = buf.ctypes.data
    other = np.zeros(1024, dtype=np.uint8)
    lib, pools = _native.load(), [other.ctypes.data, at + 1024]
    for kw in (dict(new=at + 932), dict(new=at + 1024), dict(rel=at + 1264), dict(cnt=at + 1052),
               dict(cop=at + 980), dict(cnt=at + 1440), dict(par=at + 1024), dict(lens=at + 1080),
               dict(tab=at + 1216)):
        assert _tables_call(pools, slot=128, **kw) == _native.HELM_E_INVALID, kw
        assert b"lies over" in lib.helm_last_error_string()
    assert _tables_call(pools, slot=31) == _native.HELM_E_INVALID        # pages over each other


def test_the_restated_choice():
    """By hand: two beams of two tokens, and ties."""
    x = torch.tensor([[[0.0, 0.0], [0.0, 0.0]]])
    y, tok, par = R.select(x, torch.tensor([[0.0, 0.0]]), 5)
    assert tok.tolist() == [[0, 1, 0, 1, -1]] and par.tolist() == [[0, 0, 1, 1, -1]]
    assert torch.allclose(y[0, :4], torch.full((4,), -math.log(2.0), dtype=torch.float64))
    assert y[0, 4] == -math.inf


def test_the_restated_tables():
    """By hand: pages of 4, 6 tokens; beams 1 and 2 go on from 1, beam 0 from 2."""
    table = [[10, 20, 0], [11, 21, 0], [11, 22, 0]]
    new, copies, released = R.tables([[2, 1, 1]], table, [6] * 3, 4)
    # beam 2's page goes on under row 0, beam 1's under row 1; row 2 takes the page of beam 0
    assert new == [[11, 22, 0], [11, 21, 0], [11, 20, 0]]
    assert copies == [(-1, -1), (-1, -1), (21, 20)] and released == [10]
