"""The scaled 8-bit cache on the CPU: pins of the oracle by closed forms, and the
refusals of the Python entry points and the C ABI before any launch."""

import ctypes
import math

import pytest
import torch

from oracle import cache8_oracle as O
from srswa import UnsupportedShape, _lib, cache8
from srswa.unlimited_dash_ops import attend_triton

E4M3 = torch.float8_e4m3fn


def test_scale_is_the_smallest_power_of_two():
    for dt in (torch.int8, E4M3):
        q = O.QMAX[dt]
        assert O.scale_for(0.0, dt) == 2.0 ** -100
        for e in (-20, 0, 3):
            assert O.scale_for(q * 2.0 ** e, dt) == 2.0 ** e
            assert O.scale_for(q * 2.0 ** e * (1 + 1e-6), dt) == 2.0 ** (e + 1)


def test_append_rounds_once_and_keeps_what_it_does_not_write():
    g = torch.Generator().manual_seed(5)
    for dt in (torch.int8, E4M3):
        x = torch.randn(21, 2, 64, generator=g).to(torch.bfloat16)
        cache = torch.zeros(3, 16, 2, 64).to(dt)
        cache.view(torch.int8)[:] = 3
        scale = torch.ones(3, 2)
        c1, s1 = O.append(x[:9], cache, scale, [[2, 0]], [0], [9])
        c2, s2 = O.append(x[9:], c1, s1, [[2, 0]], [9], [12])
        got = torch.cat([c2[2], c2[0]])[:21].float() * torch.cat([s2[2][None].expand(16, 2), s2[0][None].expand(16, 2)])[
            :21, :, None]
        step = 0.5 * s2.max() if dt == torch.int8 else x.float().abs() * 2.0 ** -4 + s2.max() * 2.0 ** -10
        assert ((got - x.float()).abs() <= step * (2 if dt == torch.int8 else 1)).all()
        assert (c2.view(torch.int8)[0, 5:] == 3).all() and (c2.view(torch.int8)[1] == 3).all() and (s2[1] == 1).all()


def test_attend_is_a_softmax_of_the_visible_keys():
    g = torch.Generator().manual_seed(6)
    kc = torch.randn(4, 16, 1, 64, generator=g).to(E4M3)
    vc = torch.randn(4, 16, 1, 64, generator=g).to(E4M3)
    one = torch.ones(4, 1)
    q = torch.randn(2, 2, 64, generator=g).to(torch.bfloat16)
    o, lse, tol = O.attend(q, kc, vc, one, one, [[3, 1, 0]], [0, 2], [37], 0.125, window=9, sinks=2)
    k, v = (torch.cat([c[3], c[1], c[0]])[:37, 0].double() for c in (kc.float(), vc.float()))
    for i in range(2):
        p = 35 + i
        see = torch.tensor([j <= p and (j > p - 9 or j < 2) for j in range(37)])
        z = (q[i].double() @ k.T * 0.125).masked_fill(~see, -math.inf)
        assert torch.allclose(o[i], torch.softmax(z, -1) @ v, rtol=0, atol=1e-12)
        assert torch.allclose(lse[i], torch.logsumexp(z, -1), rtol=0, atol=1e-12)
    # every listed block and the window together are every key
    ids = torch.tensor([[[0, 1, 2, 1]]]).expand(1, 2, 4)
    a = O.attend(q, kc, vc, one, one, [[3, 1, 0]], [0, 2], [37], 0.125, window=16, topk=ids)[0]
    assert torch.allclose(a, O.attend(q, kc, vc, one, one, [[3, 1, 0]], [0, 2], [37], 0.125)[0], rtol=0, atol=1e-12)


# ------------------------------------------------------------------ refusals
@pytest.fixture
def host(monkeypatch):
    """Entry points that think the CPU a GPU and fail on any launch."""
    class Lib:
        def __getattr__(self, name):
            raise AssertionError(f"{name} reached")
    for mod in (cache8,):
        monkeypatch.setattr(mod, "_require_cuda", lambda *ts: None)
    monkeypatch.setattr(_lib, "lib", Lib)
    monkeypatch.setattr(_lib, "stream_ptr", lambda device: 0)


def _cache(dt=torch.int8, page=16, H=2, D=64, n=4):
    z = torch.zeros(n, page, H, D).to(dt)
    return [z, z.clone(), torch.ones(n, H), torch.ones(n, H)]


def test_host_tensors_are_refused():
    c, q = _cache(), torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    bt, one = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        cache8.cache8_decode(q, *c, bt, one, scale=1.0)
    with pytest.raises(RuntimeError, match="no CPU path"):
        cache8.cache8_append(q, q, *c, bt, one)
    with pytest.raises(RuntimeError, match="no CPU path"):
        cache8.cache8_prefill(q, *c, bt, torch.tensor([0, 1]), one, 1, scale=1.0)


def test_attend_refusals(host):
    bt, sl = torch.zeros(2, 3, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    run = lambda q=q, c=None, bt=bt, sl=sl, **k: cache8.cache8_decode(q, *(c or _cache()), bt, sl, scale=1.0, **k)  # noqa: E731
    with pytest.raises(UnsupportedShape, match="bf16 / fp16"):
        run(q=q.float())
    with pytest.raises(UnsupportedShape, match="float8_e4m3fn or int8"):
        run(c=_cache(torch.float8_e5m2))
    with pytest.raises(ValueError, match="rows"):
        run(decode_query_len=2)
    with pytest.raises(ValueError, match="rows"):
        run(decode_query_len=0)
    with pytest.raises(ValueError, match="window"):
        run(window=0)
    with pytest.raises(ValueError, match="sinks"):
        run(window=4, sinks=-1)
    with pytest.raises(ValueError, match="k_scale"):
        c = _cache()
        c[2] = torch.ones(4, 3)
        run(c=c)
    with pytest.raises(ValueError, match="v_scale"):
        c = _cache()
        c[3] = c[3].double()
        run(c=c)
    with pytest.raises(ValueError, match="one dtype"):
        c = _cache()
        c[1] = c[1].to(E4M3)
        run(c=c)
    with pytest.raises(ValueError, match="block_table"):
        run(bt=bt[:1])
    with pytest.raises(ValueError, match="total_q"):
        run(q=q[..., :32])
    with pytest.raises(UnsupportedShape, match="contiguous"):
        run(q=torch.zeros(2, 4, 128, dtype=torch.bfloat16)[..., ::2])
    with pytest.raises(ValueError, match="out"):
        run(out=torch.zeros(2, 4, 64))
    with pytest.raises(ValueError, match="cu_seqlens_q"):
        cache8.cache8_prefill(q, *_cache(), bt, torch.tensor([0, 2]), sl, 2, scale=1.0)
    with pytest.raises(ValueError, match="max_query_len"):
        cache8.cache8_prefill(q, *_cache(), bt, torch.tensor([0, 1, 2]), sl, -1, scale=1.0)


def test_append_refusals(host):
    bt, st = torch.zeros(2, 3, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    x = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    run = lambda k=x, v=x, **kw: cache8.cache8_append(k, v, *_cache(), bt, st, **kw)  # noqa: E731
    with pytest.raises(UnsupportedShape, match="bf16 / fp16"):
        run(x.float(), x.float())
    with pytest.raises(ValueError, match="total"):
        run(x, x[:1])
    with pytest.raises(ValueError, match="divide"):
        run(x[:1], x[:1])
    with pytest.raises(ValueError, match="max_new_len"):
        run(cu_seqlens=torch.tensor([0, 1, 2]))
    with pytest.raises(ValueError, match="max_new_len"):
        run(max_new_len=3)
    with pytest.raises(ValueError, match="cu_seqlens"):
        run(cu_seqlens=torch.tensor([0, 2]), max_new_len=2)


def test_selected_refusals(host):
    bt, sl = torch.zeros(2, 3, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    ids = torch.zeros(2, 2, 3, dtype=torch.int32)
    kc, vc, ks, vs = _cache()
    run = lambda i=ids, b=None, **kw: attend_triton.dash_sparse_attn_decode(  # noqa: E731
        q, kc, vc, i, b, bt, sl, 2, 1.0, torch.empty_like(q), 1, local_blocks=1, sparse_block_size=16, **kw)
    with pytest.raises(ValueError, match="both or neither"):
        run(k_scale=ks)
    with pytest.raises(ValueError, match="topk_idx"):
        run(ids[:1], k_scale=ks, v_scale=vs)
    with pytest.raises(ValueError, match="blk_bias"):
        run(b=torch.zeros(2, 2, 2), k_scale=ks, v_scale=vs)
    with pytest.raises(UnsupportedShape, match="1024"):
        run(torch.zeros(2, 2, 1025, dtype=torch.int32), k_scale=ks, v_scale=vs)


def _attend_struct(**over):
    a = _lib.Cache8AttendArgs()
    for i, n in enumerate(("q", "k_cache", "v_cache", "k_scale", "v_scale", "block_table", "seq_lens", "out")):
        setattr(a, n, 0x100000 * (i + 1))
    a.R, a.total_q, a.max_query_len, a.HQ, a.HKV, a.D = 2, 2, 1, 4, 2, 64
    a.max_blocks, a.num_pages, a.page_size, a.scale = 8, 16, 16, 1.0
    a.dtype, a.kv_dtype = _lib.SRSWA_BF16, _lib.SRSWA_I8
    a.q_sn = a.o_sn = 256
    a.q_sh = a.o_sh = 64
    a.k_sp = a.v_sp = 16 * 128
    a.k_st = a.v_st = 128
    a.k_sh = a.v_sh = 64
    for k, v in over.items():
        setattr(a, k, v)
    return a


def test_abi_refuses_before_any_launch():
    L = _lib.lib()
    U, I = _lib.SRSWA_UNSUPPORTED, _lib.SRSWA_INVALID
    for want, over in ((I, dict(q=None)), (I, dict(R=-1)), (I, dict(window=-1)), (I, dict(total_q=3)), (U, dict(HQ=3)),
                       (U, dict(D=96)), (U, dict(dtype=0)), (U, dict(kv_dtype=5)), (U, dict(page_size=24)),
                       (U, dict(page_size=2048)), (U, dict(q_sn=252)), (U, dict(k_st=120)), (U, dict(out=0x100008)),
                       (U, dict(max_blocks=1 << 27)), (U, dict(window=(1 << 30) + 1))):
        a = _attend_struct(**over)
        for fn in (L.srswa_cache8_decode, L.srswa_cache8_prefill):
            assert fn(ctypes.byref(a), None, 0, None) == want, over
    a = _attend_struct(max_blocks=4096)
    need = L.srswa_cache8_decode_workspace(ctypes.byref(a))
    assert need > 0
    assert L.srswa_cache8_decode(ctypes.byref(a), ctypes.c_void_p(0x9000000), need - 1, None) == _lib.SRSWA_WORKSPACE
    a = _attend_struct(topk=0x900000, topk_n=2, window=16)
    assert L.srswa_cache8_prefill(ctypes.byref(a), None, 0, None) == U
    for R, total in ((0, 0), (2, 0)):       # nothing to do is no error
        a = _attend_struct(R=R, total_q=total, max_query_len=0)
        assert L.srswa_cache8_decode(ctypes.byref(a), None, 0, None) == _lib.SRSWA_OK
    b = _lib.Cache8AppendArgs()
    assert L.srswa_cache8_append(ctypes.byref(b), None) == I


def test_abi_refuses_far_strides_and_large_grids():
    """Strides that 32-bit address parts cannot hold, and launches past the grid."""
    L = _lib.lib()
    U = _lib.SRSWA_UNSUPPORTED
    for over in (dict(k_sp=1 << 31), dict(v_sp=(1 << 31) + 16), dict(k_st=1 << 28), dict(v_st=1 << 31), dict(v_sh=1 << 31), dict(k_sp=-16),
                 dict(ks_sp=1 << 31), dict(vs_sp=-1)):
        a = _attend_struct(**over)
        for fn in (L.srswa_cache8_decode, L.srswa_cache8_prefill):
            assert fn(ctypes.byref(a), None, 0, None) == U, over
    a = _attend_struct(R=1 << 15, total_q=1 << 15, HQ=1 << 18, HKV=1 << 18, q_sn=1 << 24, o_sn=1 << 24)
    assert L.srswa_cache8_decode(ctypes.byref(a), None, 0, None) == U
    # a bound on the longest request that no table of items could hold: sized by the rows there are
    a = _attend_struct(R=4096, total_q=4096, max_query_len=1 << 30, cu_seqlens_q=0x900000)
    assert L.srswa_cache8_prefill_workspace(ctypes.byref(a)) < 1 << 32
