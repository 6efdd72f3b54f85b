"""What shared-prefix decode refuses: argument checks of the Python entry points and of the
C-ABI, which return before any device work."""
import copy
import pickle

import numpy as np
import pytest
import torch

from helm_amd import _native, prefix
from helm_amd.runtime import engine

I32, BF, HF = torch.int32, torch.bfloat16, torch.float16


def _args(R=2, Hq=4, Hkv=2, S=1, D=64, page=16, slots=5, width=3, n=1, **kw):
    arena = torch.zeros((slots, 2, Hkv, page, D), dtype=BF)
    return dict(dict(q=torch.zeros((R, Hq, S, D), dtype=BF), k_pool=arena[:, 0],
                     v_pool=arena[:, 1], page_table=torch.zeros((R, width), dtype=I32),
                     seq_lens=torch.zeros(R, dtype=I32),
                     group_starts=torch.zeros(n + 1, dtype=I32),
                     shared_pages=torch.zeros(n, dtype=I32)), **kw)


def _pool(*shape, dtype=BF):
    return torch.zeros(shape, dtype=dtype)


def _both(k):
    return dict(k_pool=k, v_pool=k)


@pytest.mark.parametrize("bad,err", [
    (dict(q=_pool(2, 4, 64)), ValueError),
    (_both(_pool(5, 2, 64)), ValueError),
    (dict(q=_pool(2, 4, 1, 128)), ValueError),                 # heads of another length
    (dict(q=_pool(2, 3, 1, 64)), ValueError),                  # 3 heads over 2
    (dict(q=_pool(2, 4, 0, 64)), ValueError),
    (dict(v_pool=_pool(4, 2, 16, 64)), ValueError),
    (dict(q=_pool(2, 4, 1, 64, dtype=HF)), TypeError),
    (dict(q=torch.zeros((2, 4, 1, 64)), **_both(torch.zeros((5, 2, 16, 64)))), TypeError),
    (dict(q=_pool(2, 4, 1, 96), **_both(_pool(5, 2, 16, 96))), NotImplementedError),
    (_both(_pool(5, 2, 24, 64)), ValueError), (_both(_pool(5, 2, 8, 64)), ValueError),
    (dict(v_pool=_pool(5, 2, 16, 64)), ValueError),            # strides of its own
    (_both(_pool(5, 2, 16, 128)[..., :64]), ValueError),
    (_both(_pool(5, 2, 64, 16).transpose(2, 3)), ValueError),
    (_both(_pool(5 * 2 * 16 * 64 + 4)[4:].view(5, 2, 16, 64)), ValueError),    # 8 bytes off
    (_both(_pool(5 * 2060).as_strided((5, 2, 16, 64), (2052, 1024, 64, 1))), ValueError),
    (dict(page_table=torch.zeros((2, 3), dtype=torch.int64)), TypeError),
    (dict(seq_lens=torch.zeros(2, dtype=torch.int64)), TypeError),
    (dict(group_starts=torch.zeros(2, dtype=torch.int64)), TypeError),
    (dict(shared_pages=torch.zeros(1, dtype=torch.int64)), TypeError),
    (dict(page_table=torch.zeros((3, 3), dtype=I32)), ValueError),
    (dict(page_table=torch.zeros((3, 2), dtype=I32).t()), ValueError),
    (dict(seq_lens=torch.zeros(3, dtype=I32)), ValueError),
    (dict(seq_lens=torch.zeros(4, dtype=I32)[::2]), ValueError),
    (dict(group_starts=torch.zeros(1, dtype=I32)), ValueError),
    (dict(shared_pages=torch.zeros((1, 1), dtype=I32)), ValueError),
    (dict(max_pages=4), ValueError), (dict(max_pages=-1), ValueError),
    (dict(window=-1), ValueError),
    (dict(scale=float("nan")), ValueError), (dict(softcap=-1.0), ValueError),
    (dict(out=_pool(2, 4, 2, 64)), ValueError),
    (dict(out=_pool(2, 4, 1, 64, dtype=HF)), ValueError),
    (dict(out=_pool(4, 2, 1, 64).transpose(0, 1)), ValueError),
    (dict(q=torch.zeros((2, 4, 1, 64), dtype=BF, requires_grad=True)), RuntimeError),
    (_args(n=513), ValueError), (_args(R=4097), ValueError),
    ({}, RuntimeError),                                        # CPU tensors
])
def test_refusals(bad, err):
    for entry in (prefix.prefix_decode_attention, prefix.prepare_prefix_decode):
        with pytest.raises(err):
            entry(**_args(**bad))


def test_out_and_prepared_refusals(monkeypatch):
    monkeypatch.setattr(engine, "common_device", lambda *a: 0)
    a = _args()
    table = torch.zeros((2, 128), dtype=I32)
    arena = torch.zeros((5, 2, 2, 16, 64), dtype=BF)
    for bad in (dict(k_pool=arena[:, 0], v_pool=arena[:, 1],
                     out=arena.view(-1)[9728:10240].view(2, 4, 1, 64)),
                dict(page_table=table, out=table.view(BF).view(2, 4, 1, 64))):
        with pytest.raises(ValueError, match="lies over"):
            prefix.prefix_decode_attention(**dict(a, **bad))
    q = torch.zeros(2 * 4 * 64 + 8, dtype=BF)
    with pytest.raises(ValueError, match="lies over"):         # a part of q; the whole is allowed
        prefix.prefix_decode_attention(**dict(a, q=q[:512].view(2, 4, 1, 64),
                                              out=q[8:].view(2, 4, 1, 64)))
    with pytest.raises(ValueError, match="16-byte"):
        prefix.prefix_decode_attention(**dict(a, out=torch.zeros(513, dtype=BF)[1:]
                                              .view(2, 4, 1, 64)))
    with pytest.raises(ValueError, match="contiguous"):
        prefix.prepare_prefix_decode(**dict(a, q=_pool(4, 2, 1, 64).transpose(0, 1)))
    with pytest.raises(ValueError, match="16-byte"):
        prefix.prepare_prefix_decode(**dict(a, q=torch.zeros(513, dtype=BF)[1:].view(2, 4, 1, 64)))
    p = prefix.prepare_prefix_decode(**a)
    assert type(copy.copy(p)) is prefix.PreparedPrefixDecode
    for no in (lambda: pickle.dumps(p), lambda: copy.deepcopy(p)):
        with pytest.raises(TypeError):
            no()


def test_tables_past_32_bits_are_refused():
    for width, page in ((2 ** 32 + 3, 16), (2 ** 27, 16), (2 ** 20, 2048)):
        table = torch.zeros((2, width), dtype=I32, device="meta")
        with pytest.raises(ValueError, match="2.31"):
            prefix.prefix_decode_attention(**_args(page=page, page_table=table))


def test_c_entry_refuses_before_device_work():
    lib = _native.load()
    raw = np.zeros(1 << 16, dtype=np.uint8)
    at = (raw.ctypes.data + 15) // 16 * 16
    need = lib.helm_prefix_workspace_bytes(2, 4, 2, 1, 64, 1)
    E = _native.HELM_E_INVALID

    def run(q=at, out=at, k=at, v=at, slots=5, ss=4096, hs=1024, page=16, table=at, ts=3, mp=3,
            lens=at, starts=at, shared=at, n=1, R=2, Hq=4, Hkv=2, S=1, D=64, scale=0.125, cap=0.0,
            window=0, dt=1, ws=at, nb=need):
        return lib.helm_prefix_decode_attn(q, out, k, v, slots, ss, hs, page, table, ts, mp, lens,
                                           starts, shared, n, R, Hq, Hkv, S, D, scale, cap, window,
                                           dt, ws, nb, None)
    for kw in (dict(dt=2), dict(dt=9), dict(D=96), dict(D=0)):
        assert run(**kw) == _native.HELM_E_UNSUPPORTED, kw
    for kw in (dict(R=-1), dict(R=4097), dict(n=513), dict(n=-1), dict(Hq=5), dict(Hkv=0),
               dict(Hq=0), dict(S=0), dict(mp=-1), dict(page=8), dict(page=24), dict(slots=-1),
               dict(slots=2 ** 31), dict(ts=-1), dict(ss=-8), dict(hs=-8), dict(ss=4100),
               dict(hs=1028), dict(mp=2 ** 27), dict(mp=2 ** 26, R=4096, n=0),
               dict(scale=float("inf")), dict(scale=float("nan")), dict(cap=float("nan")),
               dict(q=None), dict(out=None), dict(k=None), dict(v=None), dict(table=None),
               dict(lens=None), dict(starts=None), dict(shared=None), dict(q=at + 2),
               dict(out=at + 8), dict(k=at + 4), dict(v=at + 4), dict(ws=at + 8)):
        assert run(**kw) == E, kw
    for kw in (dict(ws=None), dict(nb=need - 1), dict(nb=0)):
        assert run(**kw) == _native.HELM_E_WORKSPACE, kw
    assert run(R=0) == 0
    for bad in ((4097, 4, 2, 1, 64, 1), (2, 5, 2, 1, 64, 1), (2, 4, 2, 0, 64, 1),
                (2, 4, 2, 1, 64, 513)):
        assert lib.helm_prefix_workspace_bytes(*bad) == 0
