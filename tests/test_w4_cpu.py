"""w4_linear without a GPU: the quantiser against its definition, the argument contracts that precede
the launch, and the C ABI's rejections."""
import numpy as np
import pytest
import torch

from megaqwen_amd import _lib
from megaqwen_amd.w4 import quantize_w4, w4_linear
from oracle.q4_ref import w4_weight


def _np(t):
    return None if t is None else t.double().numpy() if t.dtype != torch.uint8 else t.numpy()


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("scale_dtype", [torch.bfloat16, torch.float16])
def test_quantize_is_nearest(group, symmetric, scale_dtype):
    w = torch.randn(9, 256, generator=torch.Generator().manual_seed(group)) * 0.02
    w[3] = 0.0
    w[4] = w[4].abs()                       # one-sided: the asymmetric range starts at 0
    q, s, z = quantize_w4(w, group, symmetric=symmetric, scale_dtype=scale_dtype)
    assert q.shape == (9, 128) and q.dtype == torch.uint8 and s.shape == (9, 256 // group)
    assert s.dtype == scale_dtype and (z is None) == symmetric
    back = w4_weight(q.numpy(), _np(s), _np(z))
    assert (back[3] == 0).all()
    step = np.repeat(_np(s), group, axis=1)
    # half a step of the codes; at the ends of the range the scale's rounding (and, asymmetric, the
    # zero point's) may clip up to 15 scale roundings and half a step more
    slack = 0.5 + 15 * torch.finfo(scale_dtype).eps + (0.0 if symmetric else 0.5)
    assert (np.abs(back - w.double().numpy()) <= slack * step + 1e-12).all()


def test_quantize_refusals():
    w = torch.zeros(4, 256)
    for bad in (lambda: quantize_w4(w, 48), lambda: quantize_w4(torch.zeros(4, 100), 32),
                lambda: quantize_w4(torch.zeros(256), 32), lambda: quantize_w4(w.int(), 32),
                lambda: quantize_w4(w, 32, scale_dtype=torch.float32)):
        with pytest.raises(ValueError):
            bad()


def test_front_end_on_cpu():
    q, s, _ = quantize_w4(torch.randn(8, 64), 32)
    with pytest.raises(ValueError, match="expects CUDA tensors"):
        w4_linear(torch.zeros(1, 64, dtype=torch.bfloat16), q, s)


def test_c_abi_rejections():
    f, A = _lib.load().mq_w4_linear, 1 << 20
    bf, f16, f32 = _lib.MQ_DTYPE_BF16, _lib.MQ_DTYPE_F16, _lib.MQ_DTYPE_F32
    ok = dict(x=A, q=2 * A, s=3 * A, z=None, r=None, o=4 * A, m=1, n=16, k=256, g=64, xt=bf, st=bf, ot=bf)

    def call(**kw):
        a = {**ok, **kw}
        return f(a["x"], a["q"], a["s"], a["z"], a["r"], a["o"], a["m"], a["n"], a["k"], a["g"],
                 a["xt"], a["st"], a["ot"], None)

    bad = [dict(x=None), dict(q=None), dict(s=None), dict(o=None), dict(m=-1), dict(n=-1), dict(k=0),
           dict(g=48), dict(g=0), dict(k=96), dict(xt=f32), dict(xt=9), dict(st=f32), dict(ot=f16),
           dict(ot=7), dict(x=A + 2), dict(q=2 * A + 8), dict(o=A + 16), dict(o=2 * A + 16),
           dict(o=3 * A), dict(z=4 * A), dict(r=4 * A + 2)]
    for kw in bad:
        assert call(**kw) == _lib.MQ_ERR_INVALID_ARG, kw
        assert _lib.load().mq_last_error()
    assert call(m=0) == _lib.MQ_OK and call(n=0) == _lib.MQ_OK      # nothing to launch
