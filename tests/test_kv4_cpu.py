"""The 4-bit cache without a GPU: its reference quantiser, the constructor's contracts, and the C
ABI's rejections (nothing is launched)."""
import ctypes

import numpy as np
import pytest
import torch

from megaqwen_amd import _lib
from megaqwen_amd.kv4 import KV4Cache
from oracle.q4_ref import attend, kv4_quantize, kv4_values, round_bf16


def test_reference_quantizer():
    x = torch.randn(50, 128, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).double().numpy()
    x[7] = 0.0
    for g in (32, 64, 128):
        u, s = kv4_quantize(x, g)
        assert u.min() >= 1 and u.max() <= 15
        back = kv4_values(u, s)
        assert (back[7] == 0).all() and (u[7] == 8).all()
        # half a step; the largest value may be clipped by the scale's rounding (7 2^-8 of a step)
        assert (np.abs(back - x) <= (0.5 + 7 * 2.0 ** -8) * np.repeat(s, g, -1) + 1e-12).all()
        # rounding the values again changes nothing
        u2, s2 = kv4_quantize(back, g)
        ok = np.abs(back).reshape(50, -1, g).max(-1) == 7 * s
        assert (u2.reshape(50, -1, g)[ok] == u.reshape(50, -1, g)[ok]).all()
    assert (round_bf16(np.array([1.0, 1.00390625, 1.01171875])) == [1.0, 1.0, 1.015625]).all()


def test_reference_attention_empty_rows():
    g = np.random.default_rng(2)
    q, k, v = g.standard_normal((1, 3, 2, 64)), g.standard_normal((1, 1, 9, 64)), g.standard_normal((1, 1, 9, 64))
    out = attend(q, k, v, [2], 0.125)          # row 0 is before the first position
    assert (out[0, 0] == 0).all()
    np.testing.assert_allclose(out[0, 1], np.repeat(v[0, :, 0], 2, 0))
    assert (attend(q, k, v, [0], 0.125) == 0).all()


def test_constructor_contracts():
    for kw in (dict(batch=0), dict(head_dim=96), dict(group_size=16), dict(head_dim=64, group_size=128),
               dict(max_seq_len=0), dict(num_kv_heads=0), dict(device="cpu")):
        with pytest.raises(ValueError):
            KV4Cache(**{**dict(batch=1, num_kv_heads=2, max_seq_len=8), **kw})
    c, s = torch.zeros(1, 2, 8, 64, dtype=torch.uint8), torch.zeros(1, 2, 8, 2, 4, dtype=torch.bfloat16)
    for args in ((c, c, s), (c, c[:, :1], s), (c.int(), c, s), (c, c, s.float()), (c, c, s[..., :3]), (c[0], c[0], s)):
        with pytest.raises(ValueError):
            KV4Cache.from_tensors(*args)


def test_c_abi_rejections():
    lib, A = _lib.load(), 1 << 24
    ok = dict(k=A, v=2 * A, s=3 * A, b=2, h=4, n=100, d=128, g=32)

    def desc(**kw):
        a = {**ok, **kw}
        return ctypes.byref(_lib.Kv4Cache(a["k"], a["v"], a["s"], a["b"], a["h"], a["n"], a["d"], a["g"]))

    st = (ctypes.c_int64 * 3)(512, 512, 128)
    neg = (ctypes.c_int64 * 3)(512, -512, 128)
    bf, f32, bad = _lib.MQ_DTYPE_BF16, _lib.MQ_DTYPE_F32, _lib.MQ_ERR_INVALID_ARG
    append = lambda c, k=4 * A, ks=st, v=5 * A, vs=st, n=6 * A, t=1, ty=bf: lib.mq_kv4_append(c, k, ks, v, vs, n, t, ty, None)  # noqa: E731
    read = lambda c, n=6 * A, t=1, k=4 * A, v=5 * A, ty=bf: lib.mq_kv4_read(c, n, t, k, v, ty, None)  # noqa: E731

    def att(c, q=4 * A, qs=st, n=6 * A, t=1, hq=8, ml=100, ty=bf, o=5 * A, ws=7 * A, wb=A):
        return lib.mq_kv4_attend(c, q, qs, n, t, hq, ml, ty, 0.1, o, ws, wb, None)

    for kw in (dict(d=96), dict(g=16), dict(d=64, g=128), dict(h=0), dict(n=0), dict(b=-1), dict(k=None),
               dict(v=None), dict(s=None), dict(k=A + 8), dict(s=3 * A + 2), dict(b=70000)):
        for f in (append, read, att):
            assert f(desc(**kw)) == bad, kw
            assert lib.mq_last_error()
    for f in (append, read, att):
        assert f(None) == bad and f(desc(), t=-1) == bad and f(desc(), n=None) == bad and f(desc(), ty=9) == bad
        assert f(desc(), t=0) == _lib.MQ_OK and f(desc(b=0)) == _lib.MQ_OK
    for kw in (dict(k=None), dict(v=None), dict(ks=None), dict(vs=neg), dict(ty=f32)):
        assert append(desc(), **kw) == bad, kw
    for kw in (dict(k=None), dict(v=None), dict(k=4 * A + 2)):
        assert read(desc(), **kw) == bad, kw
    for kw in (dict(q=None), dict(o=None), dict(qs=neg), dict(hq=6), dict(hq=0), dict(ml=0), dict(ml=101),
               dict(ty=f32), dict(o=4 * A), dict(o=A + 16), dict(o=3 * A), dict(o=5 * A + 2)):
        assert att(desc(), **kw) == bad, kw
    need = lib.mq_kv4_attend_workspace_bytes(desc(b=1, n=32768), 1, 8, 32768)
    if need:
        assert att(desc(b=1, n=32768), ml=32768, wb=need - 1) == bad and b"workspace" in lib.mq_last_error()
        assert att(desc(b=1, n=32768), ml=32768, ws=None) == bad
    assert lib.mq_kv4_attend_workspace_bytes(None, 1, 8, 100) == 0
    assert lib.mq_kv4_attend_workspace_bytes(desc(), 1, 7, 100) == 0


def test_c_abi_attend_head_limits():
    lib, A = _lib.load(), 1 << 24
    st = (ctypes.c_int64 * 3)(1 << 20, 1 << 20, 128)
    for h, hq in ((1, 257), (257, 257), (2, 514), (300, 600)):
        c = ctypes.byref(_lib.Kv4Cache(A, 2 * A, 3 * A, 1, h, 100, 128, 32))
        assert lib.mq_kv4_attend(c, 4 * A, st, 6 * A, 1, hq, 100, _lib.MQ_DTYPE_BF16, 0.1, 5 * A, 7 * A, A,
                                 None) == _lib.MQ_ERR_INVALID_ARG
        assert b"256" in lib.mq_last_error()
        assert lib.mq_kv4_attend_workspace_bytes(c, 1, hq, 100) == 0


def test_at_most_256_kv_heads():
    with pytest.raises(ValueError, match="256"):
        KV4Cache(1, 257, 8)
    c, s = torch.zeros(1, 257, 1, 64, dtype=torch.uint8), torch.zeros(1, 257, 1, 2, 4, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="256"):
        KV4Cache.from_tensors(c, c, s)
    lib, A = _lib.load(), 1 << 24
    st = (ctypes.c_int64 * 3)(1 << 20, 1 << 20, 128)
    c = ctypes.byref(_lib.Kv4Cache(A, 2 * A, 3 * A, 1, 257, 100, 128, 32))
    assert lib.mq_kv4_append(c, 4 * A, st, 5 * A, st, 6 * A, 1, _lib.MQ_DTYPE_BF16, None) == _lib.MQ_ERR_INVALID_ARG
    assert b"256" in lib.mq_last_error()
    assert lib.mq_kv4_read(c, 6 * A, 1, 4 * A, 5 * A, _lib.MQ_DTYPE_BF16, None) == _lib.MQ_ERR_INVALID_ARG


def test_workspace_of_sizes_that_are_refused():
    """0, and no arithmetic on them."""
    lib, A = _lib.load(), 1 << 24
    for kw in (dict(g=0), dict(g=-32), dict(g=48), dict(d=64, g=128), dict(d=0), dict(d=96), dict(h=0), dict(h=257), dict(b=0),
               dict(b=70000), dict(n=0), dict(n=1 << 25)):
        a = {**dict(b=1, h=4, n=32768, d=128, g=32), **kw}
        c = ctypes.byref(_lib.Kv4Cache(A, 2 * A, 3 * A, a["b"], a["h"], a["n"], a["d"], a["g"]))
        for t in (1, 0, -1, 1 << 30):
            assert lib.mq_kv4_attend_workspace_bytes(c, t, 8, 32768) == 0, kw
