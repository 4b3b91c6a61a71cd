"""w4_linear on the GPU against the float64 product (oracle/q4_ref.py), within the bounds of
tests/q4_tolerances.py; its refusals, and its behaviour under streams and HIP graphs."""
import numpy as np
import pytest
import torch

from oracle.q4_ref import w4_weight
from tests.q4_tolerances import w4_bound

pytestmark = pytest.mark.gpu


def _linear(*args, **kw):
    from megaqwen_amd.w4 import w4_linear
    return w4_linear(*args, **kw)


def _weight(n, k, group, dtype, zeros, seed):
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.int32).to(torch.uint8)
    s = (0.01 + 0.02 * torch.rand(n, k // group, generator=g)).to(dtype)
    s = s * torch.where(torch.rand(s.shape, generator=g) < 0.1, -1, 1).to(dtype)
    z = torch.randint(0, 16, (n, k // group), generator=g, dtype=torch.int32).to(torch.uint8) if zeros else None
    return q, s, z


def _cuda(t):
    return None if t is None else t.cuda()


def _np(t):
    return None if t is None else t.double().numpy()


def _check(y, x, q, s, z, r, group):
    w = w4_weight(q.numpy(), _np(s), None if z is None else z.numpy())
    xs = _np(x).reshape(-1, x.shape[-1])
    ref = xs @ w.T
    if r is not None:
        ref = ref + _np(r).reshape(ref.shape)
    got = y.double().cpu().numpy().reshape(ref.shape)
    err, bound = np.abs(got - ref), w4_bound(xs, _np(s), ref, x.shape[-1], group, y.dtype)
    at = np.unravel_index(np.argmax(err - bound), err.shape)
    assert (err <= bound).all(), f"{(err > bound).sum()} off, worst {at}: {got[at]} for {ref[at]}, bound {bound[at]}"


# rows of x around the tiles of 16 and the blocks of 64, output counts that end inside a tile of 16,
# inputs of one group to many
@pytest.mark.parametrize("m,n,k", [(1, 1, 128), (1, 16, 256), (1, 4096, 1024), (2, 17, 384), (3, 1000, 128),
                                   (1, 40, 11008), (7, 129, 3200), (15, 33, 640), (16, 64, 512), (17, 100, 1152),
                                   (31, 15, 256), (33, 260, 896), (48, 31, 1024), (64, 96, 2048),
                                   (65, 50, 512), (130, 70, 640), (1, 20011, 256), (5, 6000, 2944)])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_shapes(m, n, k, group, dtype):
    zeros, res = (m + n) % 2 == 0, k % 512 == 0
    out = torch.float32 if m in (1, 16, 33) else dtype
    q, s, z = _weight(n, k, group, dtype, zeros, seed=m + n + k)
    g = torch.Generator().manual_seed(1)
    x = torch.randn(m, k, generator=g).to(dtype)
    r = torch.randn(m, n, generator=g).to(out) if res else None
    y = _linear(x.cuda(), q.cuda(), s.cuda(), _cuda(z), residual=_cuda(r), out_dtype=out)
    assert y.shape == (m, n) and y.dtype == out
    _check(y, x, q, s, z, r, group)


@pytest.mark.parametrize("group", [32, 64, 128])
def test_one_group_and_odd_group_counts(group):
    """K of 1, 3 and 5 groups: scale rows that are not a multiple of 4 bytes."""
    for groups in (1, 3, 5):
        for m in (1, 20):
            q, s, z = _weight(37, groups * group, group, torch.bfloat16, True, seed=groups)
            x = torch.randn(m, groups * group, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
            _check(_linear(x.cuda(), q.cuda(), s.cuda(), z.cuda()), x, q, s, z, None, group)


@pytest.mark.parametrize("m", [1, 24])
def test_scale_and_input_types_mix(m):
    q, s, z = _weight(50, 512, 64, torch.float16, False, seed=9)
    x = torch.randn(m, 512, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    _check(_linear(x.cuda(), q.cuda(), s.cuda()), x, q, s, z, None, 64)
    s2 = s.to(torch.bfloat16)
    _check(_linear(x.half().cuda(), q.cuda(), s2.cuda()), x.half(), q, s2, z, None, 64)


def test_single_codes():
    """One input at a time is 1: the output is that column of weights, exactly (fp32 out, scales that
    are powers of two), so every code's place and value shows."""
    n, k, group = 32, 256, 32
    q, s, z = _weight(n, k, group, torch.bfloat16, True, seed=4)
    s = torch.exp2(torch.randint(-3, 3, s.shape, generator=torch.Generator().manual_seed(5)).float()).to(torch.bfloat16)
    w = w4_weight(q.numpy(), _np(s), z.numpy())
    eye = torch.eye(k, dtype=torch.bfloat16)
    for rows in (eye[:1], eye[77:78], eye[:16], eye[100:149], eye):
        at = rows.float().argmax(-1).numpy()
        y = _linear(rows.cuda(), q.cuda(), s.cuda(), z.cuda(), out_dtype=torch.float32)
        assert np.array_equal(y.double().cpu().numpy(), w[:, at].T)


def test_non_finite_inputs():
    """A NaN or an infinity reaches its own row of x (an infinite scale its own output) and no other."""
    q, s, z = _weight(40, 256, 64, torch.bfloat16, False, seed=6)
    x = torch.randn(20, 256, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16)
    want = _linear(x.cuda(), q.cuda(), s.cuda()).cpu()
    x2, s2 = x.clone(), s.clone()
    x2[3, 10], x2[18, 255] = float("nan"), float("inf")
    s2[7, 1] = float("inf")
    got = _linear(x2.cuda(), q.cuda(), s2.cuda()).cpu()
    assert not torch.isfinite(got[3]).any() and not torch.isfinite(got[18]).any() and not torch.isfinite(got[:, 7]).any()
    keep = torch.ones(20, 40, dtype=torch.bool)
    keep[3], keep[18], keep[:, 7] = False, False, False
    assert torch.equal(got[keep], want[keep])


def test_views_and_leading_dimensions():
    """x as [2, 3, K], a strided view of it, one row as [K], one that starts 2 bytes into memory;
    a slice of the weight's outputs; a strided residual."""
    q, s, z = (_cuda(t) for t in _weight(48, 256, 64, torch.bfloat16, True, seed=7))
    x = torch.randn(6, 512, generator=torch.Generator().manual_seed(5)).to(torch.bfloat16).cuda()
    half = x[:, :256]
    want = _linear(half.contiguous(), q, s, z)
    assert torch.equal(_linear(half, q, s, z), want)
    assert torch.equal(_linear(half.reshape(2, 3, 256), q, s, z), want.view(2, 3, 48))
    assert torch.equal(_linear(half[2], q, s, z), _linear(half[2:3].contiguous(), q, s, z)[0])
    odd = torch.empty(6 * 256 + 1, dtype=x.dtype, device="cuda")[1:].view(6, 256)
    odd.copy_(half)
    assert odd.data_ptr() % 4 == 2 and torch.equal(_linear(odd, q, s, z), want)
    assert torch.equal(_linear(half, q[16:40], s[16:40], z[16:40]), want[:, 16:40])
    r = torch.randn(6, 96, device="cuda").to(torch.bfloat16)[:, ::2]
    assert torch.equal(_linear(half, q, s, z, residual=r), _linear(half, q, s, z, residual=r.contiguous()))


def test_rows_do_not_depend_on_their_number_of_neighbours():
    """The same call twice gives the same bits."""
    q, s, _ = (_cuda(t) for t in _weight(1000, 1024, 128, torch.bfloat16, False, seed=8))
    x = torch.randn(40, 1024, generator=torch.Generator().manual_seed(6)).to(torch.bfloat16).cuda()
    for m in (1, 7, 40):
        assert torch.equal(_linear(x[:m], q, s), _linear(x[:m], q, s))


def test_empty():
    q, s, _ = (_cuda(t) for t in _weight(16, 128, 64, torch.bfloat16, False, seed=8))
    assert _linear(torch.empty(0, 128, dtype=torch.bfloat16, device="cuda"), q, s).shape == (0, 16)
    assert _linear(torch.empty(3, 128, dtype=torch.bfloat16, device="cuda"), q[:0], s[:0]).shape == (3, 0)


@pytest.mark.parametrize("m", [1, 30])
def test_side_stream_and_graph(m):
    q, s, z = (_cuda(t) for t in _weight(500, 1024, 128, torch.bfloat16, True, seed=10))
    xs = [torch.randn(m, 1024, generator=torch.Generator().manual_seed(i)).to(torch.bfloat16).cuda() for i in range(4)]
    want = [_linear(x, q, s, z) for x in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [_linear(x, q, s, z) for x in xs]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    x, graph = xs[0].clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = _linear(x, q, s, z)
    for i in (1, 2, 3, 0):
        x.copy_(xs[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[i])


def test_argument_contracts():
    q, s, z = (_cuda(t) for t in _weight(16, 256, 64, torch.bfloat16, True, seed=11))
    x = torch.zeros(2, 256, dtype=torch.bfloat16, device="cuda")
    bad = [((x.float(), q, s), "only supports"), ((x[:, :128], q, s), "K = 256"), ((x, q.int(), s), "uint8"),
           ((x, q, s[:, :3]), "do not fit"), ((x, q, s[:8]), "do not fit"), ((x, q, s.float()), "fp16/bf16"),
           ((x, q, s, z[:, :2]), "zeros"), ((x, q, s, z.int()), "zeros"), ((x, q.cpu(), s), "qweight is on"),
           ((x, q.t().contiguous().t(), s), "contiguous")]
    for args, match in bad:
        with pytest.raises(ValueError, match=match):
            _linear(*args)
    for kw, match in ((dict(out_dtype=torch.float16), "out_dtype"), (dict(residual=x), "residual"),
                      (dict(residual=torch.zeros(2, 16, device="cuda")), "residual")):
        with pytest.raises(ValueError, match=match):
            _linear(x, q, s, z, **kw)
    with pytest.raises(ValueError, match="no backward"):
        _linear(x.clone().requires_grad_(), q, s, z)
    with torch.no_grad():
        assert not _linear(x.clone().requires_grad_(), q, s, z).requires_grad


@pytest.mark.parametrize("m,n,k", [(1, 4500, 512), (9, 8300, 512), (20, 6200, 1024), (20, 6200, 1792), (40, 4200, 896),
                                   (64, 3100, 1536), (5, 8300, 6656), (100, 1800, 640), (65, 2600, 512), (33, 4200, 256),
                                   (200, 900, 1024)])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_many_outputs(m, n, k, group, dtype):
    """Outputs enough for every way the work is laid out, inputs that end inside a block of 128 (one
    group more than k), and row counts over several blocks of 64."""
    k += group
    zeros = (n // 100) % 2 == 0
    q, s, z = _weight(n, k, group, dtype, zeros, seed=m + n + k)
    x = torch.randn(m, k, generator=torch.Generator().manual_seed(7)).to(dtype)
    _check(_linear(x.cuda(), q.cuda(), s.cuda(), _cuda(z)), x, q, s, z, None, group)


@pytest.mark.parametrize("m,n,k", [(1, 40, 640), (1, 4500, 640), (9, 8300, 640), (20, 6200, 1920), (40, 4200, 640)])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_an_infinite_scale_stays_in_its_output(m, n, k, group):
    """Inputs that end inside the last turn of a workgroup: what is read for the rest is not the next
    output's scale."""
    q, s, z = _weight(n, k, group, torch.bfloat16, True, seed=11)
    x = torch.randn(m, k, generator=torch.Generator().manual_seed(8)).to(torch.bfloat16)
    want = _linear(x.cuda(), q.cuda(), s.cuda(), z.cuda()).cpu()
    s[1::2] = float("inf")
    got = _linear(x.cuda(), q.cuda(), s.cuda(), z.cuda()).cpu()
    assert torch.equal(got[:, ::2], want[:, ::2]) and not torch.isfinite(got[:, 1::2]).any()


@pytest.mark.parametrize("m,n", [(1, 100), (1, 5000), (12, 9000), (40, 5000), (40, 100)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_residual_in_place(m, n, dtype):
    """The C entry point adds into out itself."""
    from megaqwen_amd import _lib
    k = 1152
    q, s, z = (_cuda(t) for t in _weight(n, k, 64, torch.bfloat16, True, seed=12))
    x = torch.randn(m, k, generator=torch.Generator().manual_seed(9)).to(torch.bfloat16).cuda()
    r = torch.randn(m, n, generator=torch.Generator().manual_seed(10)).to(dtype).cuda()
    want = _linear(x, q, s, z, residual=r, out_dtype=dtype)
    _lib.check(_lib.load().mq_w4_linear(
        x.data_ptr(), q.data_ptr(), s.data_ptr(), z.data_ptr(), r.data_ptr(), r.data_ptr(), m, n, k, 64, _lib.MQ_DTYPE_BF16,
        _lib.MQ_DTYPE_BF16, _lib.MQ_DTYPE_BF16 if dtype == torch.bfloat16 else _lib.MQ_DTYPE_F32,
        torch.cuda.current_stream().cuda_stream))
    assert torch.equal(r, want)


@pytest.mark.parametrize("m,n,k", [(1, 5, 1024), (1, 70, 4096), (1, 1023, 8192), (2, 130, 2048), (3, 1030, 3072), (4, 9, 5120),
                                   (5, 2050, 1024), (7, 900, 3072), (8, 31, 2048), (9, 31, 2048)])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_few_outputs(m, n, k, group):
    """Inputs of few outputs in slices, whole and with one group more or less than the slices hold."""
    for k in (k, k + group, k - group):
        q, s, z = _weight(n, k, group, torch.bfloat16, True, seed=m + n + k)
        g = torch.Generator().manual_seed(12)
        x, r = torch.randn(m, k, generator=g).to(torch.bfloat16), torch.randn(m, n, generator=g).to(torch.bfloat16)
        _check(_linear(x.cuda(), q.cuda(), s.cuda(), z.cuda(), residual=r.cuda()), x, q, s, z, r, group)


def test_non_finite_inputs_in_slices():
    """As test_non_finite_inputs, where a product holds several slices of the inputs."""
    q, s, z = _weight(40, 4096, 64, torch.bfloat16, True, seed=13)
    x = torch.randn(4, 4096, generator=torch.Generator().manual_seed(13)).to(torch.bfloat16)
    want = _linear(x.cuda(), q.cuda(), s.cuda(), z.cuda()).cpu()
    x[2, 1500], s[7, 63], s[20, 0] = float("nan"), float("inf"), float("inf")
    got = _linear(x.cuda(), q.cuda(), s.cuda(), z.cuda()).cpu()
    keep = torch.ones(4, 40, dtype=torch.bool)
    keep[2], keep[:, 7], keep[:, 20] = False, False, False
    assert not torch.isfinite(got[~keep]).any() and torch.equal(got[keep], want[keep])
