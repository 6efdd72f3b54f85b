"""What the serving operators refuse, and what they do not need a GPU for: argument
checks of the Python entry points and of the C-ABI (which return before any device
work), the oracle's own properties."""
import copy
import io
import math
import pickle

import pytest
import torch

from helm_amd import _native, paged, pool4, prompt
from oracle import serving as R

I32, I64 = torch.int32, torch.int64


def _tables(B=2, width=4, **kw):
    a = dict(new_lens=torch.ones(B, dtype=I32), cached_lens=torch.zeros(B, dtype=I32),
             page_table=torch.zeros((B, width), dtype=I32), free_slots=torch.arange(8, dtype=I32),
             page_size=16, max_tokens=4)
    a.update(kw)
    return a


@pytest.mark.parametrize("bad,err", [
    (dict(new_lens=torch.ones(2, dtype=I64)), TypeError),
    (dict(free_slots=torch.arange(8, dtype=I64)), TypeError),
    (dict(cached_lens=torch.zeros(3, dtype=I32)), ValueError),
    (dict(page_table=torch.zeros((3, 4), dtype=I32)), ValueError),
    (dict(page_table=torch.zeros((4, 2), dtype=I32).t()), ValueError),
    (dict(page_table=torch.zeros((1, 4), dtype=I32).expand(2, 4)), ValueError),
    (dict(new_lens=torch.ones(4, dtype=I32)[::2]), ValueError),
    (dict(page_size=0), ValueError),
    (dict(max_tokens=-1), ValueError),
    (dict(new_lens=torch.ones(4097, dtype=I32), cached_lens=torch.zeros(4097, dtype=I32),
          page_table=torch.zeros((4097, 1), dtype=I32)), ValueError),
    (dict(max_tokens=2 ** 31), ValueError), (dict(page_size=2 ** 31), ValueError),
    ({}, RuntimeError),            # CPU tensors
])
def test_batch_tables_refusals(bad, err):
    with pytest.raises(err):
        paged.batch_tables(**_tables(**bad))


def test_batch_tables_out_refusals():
    good = paged.BatchTables(torch.zeros(3, dtype=I32), torch.zeros(4, dtype=I64),
                             torch.zeros(4, dtype=I64), torch.zeros(2, dtype=I32),
                             torch.zeros(1, dtype=I32))
    with pytest.raises(ValueError):
        paged.batch_tables(**_tables(), out=good._replace(slot_map=torch.zeros(5, dtype=I64)))
    with pytest.raises(ValueError):
        paged.batch_tables(**_tables(), out=good._replace(positions=torch.zeros(4, dtype=I32)))


@pytest.mark.parametrize("kw,err", [
    (dict(head_dim=96), NotImplementedError), (dict(page_size=24), ValueError),
    (dict(page_size=0), ValueError), (dict(n_slots=-1), ValueError),
    (dict(num_kv_heads=0), ValueError)])
def test_pool4_refusals(kw, err):
    a = dict(n_slots=4, num_kv_heads=2, head_dim=64, page_size=16, device="cpu")
    a.update(kw)
    with pytest.raises(err):
        pool4.Pool4(**a)


@pytest.mark.parametrize("k,v,slots,err", [
    (torch.zeros(3, 2, 64), torch.zeros(3, 2, 64), torch.zeros(3, dtype=I32), TypeError),
    (torch.zeros(3, 2, 64), torch.zeros(3, 2, 64), torch.zeros(4, dtype=I64), ValueError),
    (torch.zeros(3, 1, 64), torch.zeros(3, 2, 64), torch.zeros(3, dtype=I64), ValueError),
    (torch.zeros(3, 2, 128), torch.zeros(3, 2, 128), torch.zeros(3, dtype=I64), ValueError),
    (torch.zeros(3, 2, 64), torch.zeros(3, 2, 64).half(), torch.zeros(3, dtype=I64), TypeError),
    (torch.zeros(3, 2, 64).double(), torch.zeros(3, 2, 64).double(), torch.zeros(3, dtype=I64),
     TypeError),
    (torch.zeros(3, 2, 64), torch.zeros(3, 2, 64), torch.zeros(6, dtype=I64)[::2], ValueError),
    (torch.zeros(3, 2, 64), torch.zeros(3, 2, 64), torch.zeros(3, dtype=I64), RuntimeError),
])
def test_pool4_write_refusals(k, v, slots, err):
    pool = pool4.Pool4(2, 2, 64, device="cpu")
    with pytest.raises(err):
        pool.write(k, v, slots)
    if err is RuntimeError:
        with pytest.raises(err):
            pool.read(slots)


def _saved(pool):
    f = io.BytesIO()
    torch.save(pool, f)
    f.seek(0)
    return torch.load(f, weights_only=False)


@pytest.mark.parametrize("twin", [copy.deepcopy, lambda p: pickle.loads(pickle.dumps(p)), _saved])
def test_a_copied_pool_is_written_and_read_in_its_own_storage(twin, monkeypatch):
    pool = pool4.Pool4(3, 2, 64, device="cpu")
    pool.data.random_(0, 256)
    other, calls = twin(pool), []
    assert torch.equal(other.data, pool.data) and other.data.data_ptr() != pool.data.data_ptr()
    monkeypatch.setattr(pool4._engine, "common_device", lambda what, *t: 0)
    monkeypatch.setattr(pool4._engine, "launch_on", lambda idx, fn, *args: calls.append((fn, args)))
    rows, slots = torch.zeros(3, 2, 64), torch.zeros(3, dtype=I64)
    for p in (pool, other):
        p.write(rows, rows, slots)
        p.read(slots)
        for fn, args in calls:
            assert args[:5] == (p.data.data_ptr(), 3, 16, 2, 64), fn
        assert [fn for fn, _ in calls] == ["helm_pool4_write", "helm_pool4_read"]
        calls.clear()


def _decode(**kw):
    a = dict(q=torch.zeros(2, 4, 1, 64, dtype=torch.bfloat16),
             pool=pool4.Pool4(4, 2, 64, device="cpu"), page_table=torch.zeros((2, 2), dtype=I32),
             seq_lens=torch.ones(2, dtype=I32))
    a.update(kw)
    return a


@pytest.mark.parametrize("bad,err", [
    (dict(q=torch.zeros(2, 4, 1, 64)), TypeError),
    (dict(q=torch.zeros(2, 3, 1, 64).bfloat16()), ValueError),
    (dict(q=torch.zeros(2, 4, 0, 64).bfloat16()), ValueError),
    (dict(q=torch.zeros(2, 4, 64).bfloat16()), ValueError),
    (dict(q=torch.zeros(2, 4, 1, 128).bfloat16()), ValueError),
    (dict(page_table=torch.zeros((2, 2), dtype=I64)), TypeError),
    (dict(page_table=torch.zeros((3, 2), dtype=I32)), ValueError),
    (dict(seq_lens=torch.ones(3, dtype=I32)), ValueError),
    (dict(max_pages=3), ValueError), (dict(max_pages=-1), ValueError),
    (dict(softcap=-1.0), ValueError), (dict(softcap=math.inf), ValueError),
    (dict(scale=math.nan), ValueError),
    (dict(attention_mask=torch.zeros(2, 4, 1, 32, dtype=torch.bool)), TypeError),
    (dict(attention_mask=torch.zeros(2, 3, 1, 32)), ValueError),
    (dict(attention_mask=torch.zeros(1, 32)), ValueError),
    (dict(attention_mask=torch.zeros(2, 1, 1, 0)), ValueError),
    (dict(out=torch.zeros(2, 4, 1, 64)), ValueError),
    ({}, RuntimeError)])
def test_pool4_decode_refusals(bad, err):
    with pytest.raises(err):
        pool4.pool4_decode_attention(**_decode(**bad))


def test_prepared_pool4_decode_reads_in_place():
    q = torch.zeros(2, 1, 4, 64, dtype=torch.bfloat16).transpose(1, 2)
    assert not q.is_contiguous() or q.shape[2] == 1
    q = torch.zeros(2, 4, 2, 128, dtype=torch.bfloat16)[..., :64]
    with pytest.raises(ValueError, match="in place"):
        pool4.prepare_pool4_decode(**_decode(q=q))
    with pytest.raises(ValueError, match="in place"):
        pool4.prepare_pool4_decode(**_decode(attention_mask=torch.zeros(2, 1, 1, 32).double()))


def test_a_prepared_call_is_not_copied_with_its_addresses():
    step = pool4.PreparedPool4Decode(0, (1, 2), torch.zeros(2), (torch.zeros(3),))
    for twin in (copy.deepcopy, pickle.dumps, lambda s: copy.deepcopy({"layer": [s]})):
        with pytest.raises(TypeError, match="prepare"):
            twin(step)
    same = copy.copy(step)                      # of the same operands
    assert same.out is step.out and same._args is step._args and same._keep is step._keep


def _prompt(**kw):
    a = dict(q=torch.zeros(5, 4, 64).half(), k=torch.zeros(5, 2, 64).half(),
             v=torch.zeros(5, 2, 64).half(), cu_seqlens=torch.tensor([0, 5], dtype=I32))
    a.update(kw)
    return a


@pytest.mark.parametrize("bad,err", [
    (dict(q=torch.zeros(5, 4, 64)), TypeError),
    (dict(v=torch.zeros(5, 2, 64).bfloat16()), TypeError),
    (dict(q=torch.zeros(5, 3, 64).half()), ValueError),
    (dict(q=torch.zeros(6, 4, 64).half()), ValueError),
    (dict(v=torch.zeros(5, 1, 64).half()), ValueError),
    (dict(q=torch.zeros(5, 4, 80).half(), k=torch.zeros(5, 2, 80).half(),
          v=torch.zeros(5, 2, 80).half()), NotImplementedError),
    (dict(cu_seqlens=torch.tensor([0, 5])), TypeError),
    (dict(cu_seqlens=torch.zeros((1, 2), dtype=I32)), ValueError),
    (dict(window=-1), ValueError), (dict(softcap=-2.0), ValueError),
    (dict(scale=math.inf), ValueError),
    (dict(out=torch.zeros(5, 4, 64)), ValueError),
    ({}, RuntimeError)])
def test_prompt_refusals(bad, err):
    with pytest.raises(err):
        prompt.prompt_attention(**_prompt(**bad))


def test_out_over_another_operand_is_refused(monkeypatch):
    monkeypatch.setattr(prompt._engine, "common_device", lambda what, *t: 0)
    monkeypatch.setattr(prompt._engine, "launch_on", lambda idx, fn, *args: 0)
    back = torch.zeros(16 * 4 * 64).half()
    qkv = torch.zeros(3, 5, 4, 64).half()

    def prom(out, **kw):
        a = dict(q=qkv[0], k=qkv[1, :, :2], v=qkv[2, :, :2], cu_seqlens=torch.tensor([0, 5], dtype=I32))
        return prompt.prompt_attention(**dict(a, **kw), out=out)
    for out in (qkv[1], qkv[2], qkv.view(-1)[256:256 + 1280].view(5, 4, 64),
                qkv.view(-1)[1280 - 8:2560 - 8].view(5, 4, 64)):
        with pytest.raises(ValueError, match="out lies over"):
            prom(out)
    with pytest.raises(ValueError, match="out lies over"):
        prom(back[:1280].view(5, 4, 64), cu_seqlens=back[1270:1274].view(I32))
    fused = torch.zeros(5, 8, 64).half()
    with pytest.raises(ValueError, match="out lies over"):           # q's rows, but not at q's strides
        prom(fused.view(-1)[:1280].view(5, 4, 64), q=fused[:, :4])
    for out in (qkv[0], torch.zeros(5, 4, 64).half(), back[:1280].view(5, 4, 64)):
        assert prom(out, cu_seqlens=back[1280:1284].view(I32)) is out
    turned = torch.zeros(4, 5, 64).half().transpose(0, 1)
    assert prom(torch.zeros(5, 4, 64).half(), q=turned).shape == (5, 4, 64)
    assert prom(torch.zeros(0, 4, 64).half(), q=qkv[0, :0], k=qkv[1, :0, :2], v=qkv[2, :0, :2]).numel() == 0

    d = _decode()
    mask = torch.zeros(2, 4, 1, 64).bfloat16()
    for out, kw in ((mask, dict(attention_mask=mask)),
                    (d["pool"].data.view(-1)[4096:4096 + 1024].view(torch.bfloat16).view(2, 4, 1, 64), {})):
        for call in (pool4.pool4_decode_attention, pool4.prepare_pool4_decode):
            with pytest.raises(ValueError, match="out lies over"):
                call(**dict(d, **kw), out=out)
    assert pool4.pool4_decode_attention(**d, out=d["q"]) is d["q"]


@pytest.mark.parametrize("bad", [
    dict(scale=1e300), dict(scale=-1e39), dict(softcap=1e39), dict(softcap=1e-60), dict(softcap=1e-39),
    dict(softcap=math.nan), dict(scale=1e20, softcap=1e-20), dict(scale=-3e38)])
def test_scores_out_of_fp32s_range_are_refused(bad):
    """1e-60 is 0 in fp32, which would turn the cap off; a factor of infinity makes NaN of
    zero scores."""
    with pytest.raises(ValueError, match="scale|softcap"):
        pool4.pool4_decode_attention(**_decode(**bad))
    with pytest.raises(ValueError, match="scale|softcap"):
        prompt.prompt_attention(**_prompt(**bad))
    lib, E, BF = _native.load(), _native.HELM_E_INVALID, _native.HELM_BF16
    scale, cap = bad.get("scale", 0.125), bad.get("softcap", 0.0)
    if cap != 1e-60:                           # (0 as the C entries get it: off)
        assert lib.helm_pool4_decode_attn(16, 16, 16, 1, 16, 16, 1, 1, 16, 1, 2, 1, 1, 64, scale, cap, None,
                                          0, 0, 0, 0, BF, 0, BF, None, 0, None) == E
        assert lib.helm_prompt_attn(16, 128, 64, 16, 64, 64, 16, 64, 64, 16, 128, 64, 16, 1, 1, 2, 1, 64,
                                    scale, cap, 0, 0, BF, None) == E
    for good in (dict(scale=0.0), dict(scale=2.0 ** 126), dict(softcap=2.0 ** -126),
                 dict(softcap=2.0 ** 126), dict(softcap=0.0)):
        with pytest.raises(RuntimeError, match="HIP tensors"):
            prompt.prompt_attention(**_prompt(**good))


def test_operands_that_ask_for_a_gradient_are_refused():
    a = _prompt()
    a["q"].requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient"):
        prompt.prompt_attention(**a)
    with torch.no_grad(), pytest.raises(RuntimeError, match="HIP tensors"):
        prompt.prompt_attention(**a)


@pytest.mark.parametrize("quiet", [False, True])
def test_operands_with_a_tangent_are_refused(quiet):
    from torch.autograd import forward_ad
    with forward_ad.dual_level(), torch.set_grad_enabled(not quiet):
        for name in "qkv":
            a = _prompt()
            a[name] = forward_ad.make_dual(a[name], torch.ones_like(a[name]))
            with pytest.raises(RuntimeError, match="tangent"):
                prompt.prompt_attention(**a)
            a = dict(q=torch.zeros(3, 2, 64), k=torch.zeros(3, 2, 64))
            a["k" if name == "k" else "q"] = forward_ad.make_dual(torch.zeros(3, 2, 64),
                                                                  torch.ones(3, 2, 64))
            with pytest.raises(RuntimeError, match="tangent"):
                pool4.Pool4(2, 2, 64, device="cpu").write(a["q"], a["k"], torch.zeros(3, dtype=I64))
        m = forward_ad.make_dual(torch.zeros(1, 1, 1, 9), torch.ones(1, 1, 1, 9))
        for call in (pool4.pool4_decode_attention, pool4.prepare_pool4_decode):
            with pytest.raises(RuntimeError, match="tangent"):
                call(**_decode(attention_mask=m))
        with pytest.raises(RuntimeError, match="HIP tensors"):
            prompt.prompt_attention(**_prompt())       # operands without one
    with pytest.raises(RuntimeError, match="tangent|functorch|storage"):
        torch.func.jvp(lambda q: prompt.prompt_attention(**_prompt(q=q)), (_prompt()["q"],),
                       (torch.ones(5, 4, 64).half(),))


def test_c_entries_refuse_before_device_work():
    lib = _native.load()
    E, U, W = _native.HELM_E_INVALID, _native.HELM_E_UNSUPPORTED, _native.HELM_E_WORKSPACE
    BF, F32 = _native.HELM_BF16, _native.HELM_F32

    def tables(B=1, page=16, width=1, stride=1, n=0, p=1):
        return lib.helm_batch_tables(p, p, B, p, stride, width, p, n, page, 1, p, p, p, p, p, None)
    assert tables(B=0) == E and tables(B=4097) == E and tables(page=0) == E
    assert tables(stride=0) == E and tables(n=-1) == E and tables(p=None) == E

    def write(D=64, page=16, n=1, dt=BF, p=16, ts=64):
        return lib.helm_pool4_write(p, 1, page, 1, D, p, n, p, ts, 64, p, ts, 64, dt, None)
    assert write(D=96) == U and write(page=8) == E and write(dt=9) == E and write(n=-1) == E
    assert write(p=None) == E and write(p=8) == E and write(ts=65) == E
    assert write(n=0) == 0

    def attn(D=64, page=16, dt=BF, p=16, B=1, Hq=2, Hkv=1, S=1, mp=1, ts=1, mask=None, ml=0, mdt=F32,
             ws=None, wb=0, q=16):
        return lib.helm_pool4_decode_attn(q, p, p, 1, page, p, ts, mp, p, B, Hq, Hkv, S, D, 1.0, 0.0,
                                          mask, 0, 0, 0, ml, mdt, 0, dt, ws, wb, None)
    assert attn(D=80) == U and attn(dt=F32) == U and attn(page=20) == E and attn(Hq=3, Hkv=2) == E
    assert attn(S=0) == E and attn(ts=-1) == E and attn(p=None) == E and attn(q=8) == E
    assert attn(mask=16, ml=0) == E and attn(mask=16, ml=4, mdt=7) == E
    assert attn(mp=4096, ts=4096) == W and attn(B=0) == 0
    assert lib.helm_pool4_workspace_bytes(1, 2, 1, 1, 64, 4096, 16) > 0
    assert lib.helm_pool4_workspace_bytes(1, 3, 2, 1, 64, 16, 16) == 0

    def prom(D=64, dt=BF, p=16, B=1, N=1, Hq=2, Hkv=1, scale=1.0, ts=64, kt=64):
        return lib.helm_prompt_attn(p, ts, 64, p, kt, 64, p, kt, 64, p, 128, 64, p, B, N, Hq, Hkv, D,
                                    scale, 0.0, 0, 0, dt, None)
    assert prom(D=96) == U and prom(dt=F32) == U and prom(Hq=3, Hkv=2) == E and prom(N=-1) == E
    assert prom(scale=math.nan) == E and prom(p=None) == E and prom(p=8) == E and prom(ts=4) == E
    assert prom(kt=1 << 26) == E and prom(N=0) == 0
    assert prom(N=0x7fffffff, Hq=64) == E


def test_batch_tables_c_entry_refuses_outputs_over_operands():
    lib, E = _native.load(), _native.HELM_E_INVALID
    # (addresses of nothing: the call ends at its checks)
    at = dict(new=0x1000, cached=0x2000, table=0x3000, free=0x4000, cu=0x5000, pos=0x6000,
              slot=0x7000, lens=0x8000, taken=0x9000)
    B, width, stride, n_free, N = 4, 8, 40, 30, 20

    def refused(**kw):
        a = dict(at, **kw)
        rc = lib.helm_batch_tables(a["new"], a["cached"], B, a["table"], stride, width, a["free"], n_free,
                                   16, N, a["cu"], a["pos"], a["slot"], a["lens"], a["taken"], None)
        return rc == E and b"over another operand" in lib.helm_last_error_string()

    t, row, used = at["table"], 4 * stride, 4 * width
    for lens in (at["new"], at["cached"] + 4, at["cached"] - 12, t, t + used - 4, t + row, t + row - 4,
                 t + 3 * row + used - 4, t - 12, t + 2 * row - 16 + 4, at["free"] + 4 * n_free - 4):
        assert refused(lens=lens)
    assert refused(pos=at["slot"] - 8 * N + 8) and refused(slot=at["pos"] + 8 * N - 8)
    assert refused(cu=at["taken"] - 4 * B) and refused(taken=at["pos"]) and refused(cu=at["cached"])
    assert refused(new=t + used - 4) and refused(cached=t + 3 * row) and refused(free=t - 4)


# ---- the oracle ------------------------------------------------------------------------
def test_stored_values_are_nearest_within_half_a_step():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(64, 64, generator=g) * torch.exp(4 * torch.randn(64, 1, generator=g))
    y = R.stored4(x)
    top = x.double().unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(top / 7))
    r = x.double().unflatten(-1, (-1, 32)).abs() / 2 ** e
    half = torch.where(r < 2, 0.25, torch.where(r < 4, 0.5, 1.0))
    err = (y.unflatten(-1, (-1, 32)) - x.double().unflatten(-1, (-1, 32))).abs() / 2 ** e
    assert (err <= half).all()
    assert (R.stored4(y) == y).all()           # what is held stays


def test_stored_edges():
    x = torch.zeros(8, 32)
    x[1, 3] = 7.0
    x[2, 3] = 7.0000005
    x[3, :2] = torch.tensor([6.0, 0.25])
    x[4, :3] = torch.tensor([6.0, 0.75, -2.5])
    x[5, 0], x[6, 0] = math.inf, math.nan
    x[7, 0] = 1e-45
    y = R.stored4(x)
    assert y[1, 3] == 6.0 and y[2, 3] == 8.0 and y[3, 1] == 0.0
    assert y[4, 1] == 1.0 and y[4, 2] == -2.0
    assert torch.isnan(y[5]).all() and torch.isnan(y[6]).all() and (y[7] == 0).all()
