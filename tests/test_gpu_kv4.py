"""The 4-bit cache on the GPU: append and read bit for bit against the float64 quantiser, attend
against the float64 attention over the values held (oracle/q4_ref.py), within half a step of the
output type plus ATTEND_ABS of the largest value (tests/q4_tolerances.py)."""
import numpy as np
import pytest
import torch

from oracle import q4_ref
from tests.q4_tolerances import ATTEND_ABS, half_step

pytestmark = pytest.mark.gpu


def _cache(b, h, s, d, g):
    from megaqwen_amd.kv4 import KV4Cache
    return KV4Cache(b, h, s, d, g)


def _np(t):
    return t.double().cpu().numpy()


def _randn(shape, seed, dtype=torch.bfloat16, std=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype).cuda()


def _lengths(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _state(c):
    return [t.clone() for t in (c.k_codes, c.v_codes, c.scales.view(torch.int16))]


def _fill(c, seed, std=(1.0, 0.64)):
    """Every position of the cache, quantised on the CPU by the reference."""
    g = np.random.default_rng(seed)
    for i, codes in enumerate((c.k_codes, c.v_codes)):
        u, s = q4_ref.kv4_quantize(g.standard_normal((*codes.shape[:3], c.head_dim)) * std[i], c.group_size)
        u = torch.from_numpy(u.astype(np.uint8)).cuda()
        codes.copy_(u[..., 0::2] | (u[..., 1::2] << 4))
        c.scales[:, :, :, i] = torch.from_numpy(s).to(torch.bfloat16).cuda()


def _held(c):
    return [q4_ref.kv4_values(q4_ref.unpack(x.cpu().numpy()), _np(c.scales[:, :, :, i]))
            for i, x in enumerate((c.k_codes, c.v_codes))]


# ------------------------------------------------------------------------- append and read
@pytest.mark.parametrize("d,g", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("b,t,h,s,lens", [(1, 1, 8, 16, [1]), (1, 1, 8, 16, [16]), (2, 7, 3, 40, [7, 33]),
                                          (3, 70, 2, 100, [100, 70, 12]), (4, 5, 1, 9, [0, 3, 9, 11]),
                                          (1, 33, 5, 33, [33])])
def test_append_and_read(b, t, h, s, lens, d, g, dtype):
    c = _cache(b, h, s, d, g)
    _fill(c, seed=s)
    before = _state(c)
    k, v = _randn((b, t, h, d), 1, dtype), _randn((b, t, h, d), 2, dtype, 30.0)
    k[:, 0, 0, :g] = 0.0
    c.append(k, v, _lengths(lens))
    after = _state(c)
    want = [torch.zeros(b, t, h, d, dtype=torch.float64) for _ in range(2)]
    for j in range(b):
        for i in range(t):
            p = lens[j] - t + i
            if 0 <= p < s:
                for which, (x, codes) in enumerate(((k, after[0]), (v, after[1]))):
                    u, sc = q4_ref.kv4_quantize(_np(x[j, i]), g)
                    packed = (u[..., 0::2] + 16 * u[..., 1::2]).astype(np.uint8)
                    assert np.array_equal(codes[j, :, p].cpu().numpy(), packed)
                    assert np.array_equal(_np(c.scales[j, :, p, which]), sc)
                    want[which][j, i] = torch.from_numpy(q4_ref.kv4_values(u, sc))
        rows = [p for p in range(s) if not max(0, lens[j] - t) <= p < lens[j]]      # left as they were
        for x, y in zip(before, after):
            assert torch.equal(x[j][:, rows], y[j][:, rows])
    for out in (torch.float32, torch.bfloat16, torch.float16):
        for got, w in zip(c.read(_lengths(lens), t, out), want):
            assert got.shape == (b, t, h, d) and torch.equal(got.cpu(), w.to(out))


def test_append_strided_rows():
    """Keys and values inside a fused q|k|v product [b, t, 4096], one that starts 2 bytes into memory,
    and heads ahead of positions."""
    b, t, h, d = 2, 5, 8, 128
    qkv = _randn((b, t, 4096), 3)
    k, v = qkv[..., 2048:3072].view(b, t, h, d), qkv[..., 3072:].view(b, t, h, d)
    odd = torch.empty(k.numel() + 1, dtype=k.dtype, device="cuda")[1:].view(k.shape)
    odd.copy_(k)
    flipped = k.transpose(1, 2).contiguous().transpose(1, 2)
    every = k.transpose(2, 3).contiguous().transpose(2, 3)          # the last dimension is not contiguous
    states = []
    for kk in (k.contiguous(), k, odd, flipped, every):
        c = _cache(b, h, 9, d, 32)
        c.append(kk, v if kk is k else v.contiguous(), _lengths([9, 6]))
        states.append(_state(c))
    for st in states[1:]:
        assert all(torch.equal(x, y) for x, y in zip(st, states[0]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_append_extreme_groups(dtype):
    """Largest, smallest and zero groups, values on a grid, infinities and NaN (their group reads as
    NaN, the others are untouched)."""
    big, tiny = torch.finfo(dtype).max, torch.finfo(dtype).tiny
    x = torch.zeros(1, 8, 1, 128, dtype=dtype)
    x[0, 0, 0, 5], x[0, 0, 0, 40] = big, -big
    x[0, 1, 0, 0], x[0, 1, 0, 64] = tiny, -tiny * 1.5
    x[0, 2, 0, :32] = torch.arange(32) * 0.5 - 7
    x[0, 3, 0, :] = -7.0
    x[0, 4, 0, 33], x[0, 5, 0, 97], x[0, 6, 0, 0] = float("inf"), float("nan"), -float("inf")
    x[0, 4, 0, :32] = x[0, 5, 0, :32] = 1.0
    x[0, 7, 0, :] = torch.linspace(-3, 3, 128).to(dtype)
    c = _cache(1, 1, 8, 128, 32)
    c.append(x.cuda(), x.cuda(), _lengths([8]))
    k, v = c.read(_lengths([8]), 8, torch.float32)
    u, s = q4_ref.kv4_quantize(x.double().numpy(), 32)
    want = torch.from_numpy(q4_ref.kv4_values(u, s)).float()
    assert torch.equal(k.isnan().cpu(), want.isnan()) and torch.equal(k.nan_to_num().cpu(), want.nan_to_num())
    assert torch.equal(k.nan_to_num(), v.nan_to_num())
    # 1 / 7 = 0.142857 is 0.142578125 in bf16 (steps of 2^-10 there), and 7 of them are 0.998046875
    assert k.isnan().sum() == 96 and (k[0, 4, 0, :32] == 0.998046875).all()


def test_lengths_outside_the_cache():
    """Whatever lengths holds, rows outside the cache are skipped, read as 0 and give no attention."""
    c = _cache(5, 2, 12, 128, 32)
    _fill(c, seed=5)
    before = _state(c)
    x, lens = _randn((5, 3, 2, 128), 6), _lengths([-4, 40, 2 ** 31 - 1, -2 ** 31, 0])
    c.append(x, x, lens)
    assert all(torch.equal(a, b) for a, b in zip(before, _state(c)))
    assert all((y == 0).all() for y in c.read(lens, 3))
    out = c.attend(_randn((5, 3, 4, 128), 7), lens)
    assert (out[[0, 3, 4]] == 0).all() and torch.isfinite(out).all()


# ---------------------------------------------------------------------------------- attend
def _check_attend(c, q, lens, out, scale=None, limit=None, held=None):
    k, v = _held(c) if held is None else held
    n = c.max_seq_len if limit is None else limit
    ref = q4_ref.attend(_np(q), k[:, :, :n], v[:, :, :n], lens, c.head_dim ** -0.5 if scale is None else scale)
    got = _np(out)
    assert out.dtype == q.dtype and out.shape == q.shape and np.isfinite(got).all()
    err, bound = np.abs(got - ref), half_step(ref, q.dtype) * 1.01 + ATTEND_ABS * np.nanmax(np.abs(v))
    at = np.unravel_index(np.argmax(err - bound), err.shape)
    assert (err <= bound).all(), f"{(err > bound).sum()} off, worst {at}: {got[at]} for {ref[at]}, bound {bound[at]}"


# (batch, t, kv heads, query heads per kv head, positions, lengths): single tokens, lengths at and
# around the tiles of 16 and 32, chunks, heads 1:1 to 16:1, empty sequences, padded fronts
CASES = [(1, 1, 8, 2, 16, [1]), (1, 1, 8, 2, 64, [31]), (1, 1, 2, 2, 64, [32]), (1, 1, 2, 1, 64, [33]),
         (1, 1, 1, 16, 200, [200]), (2, 1, 1, 7, 300, [129, 255]), (3, 1, 2, 4, 700, [0, 1, 700]),
         (1, 2, 2, 2, 90, [90]), (2, 5, 2, 3, 150, [3, 149]), (1, 16, 1, 8, 100, [100]), (1, 33, 2, 2, 400, [333]),
         (2, 100, 1, 2, 260, [57, 260]), (1, 1, 2, 2, 5000, [4999]), (1, 3, 1, 1, 3000, [2500])]


@pytest.mark.parametrize("case", CASES, ids=str)
@pytest.mark.parametrize("d,g", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attend(case, d, g, dtype):
    b, t, h, r, s, lens = case
    c = _cache(b, h, s, d, g)
    _fill(c, seed=s + t)
    q = _randn((b, t, h * r, d), 8, dtype)
    _check_attend(c, q, lens, c.attend(q, _lengths(lens)))


@pytest.mark.parametrize("scale", [0.0, -0.2, 1.5])
@pytest.mark.parametrize("t", [1, 20])
def test_attend_scales_and_peaked_rows(scale, t):
    """Scores from flat to hundreds wide: most weights vanish, the running maximum moves often."""
    c = _cache(1, 2, 600, 128, 32)
    _fill(c, seed=9)
    q = _randn((1, t, 4, 128), 10) * 2
    out, (k, v) = c.attend(q, _lengths([600]), scale=scale), _held(c)
    ref = q4_ref.attend(_np(q), k, v, [600], scale)
    # a score is off by up to 48 u sqrt(32) |scale| sum|q| s_k, s_k <= 0.7: the weights by that much
    off = 48 * 2.0 ** -24 * 32 ** 0.5 * abs(scale) * np.abs(_np(q)).sum(-1).max() * 0.7
    assert (np.abs(_np(out) - ref) <= half_step(ref, q.dtype) * 1.01 + (ATTEND_ABS + 2 * off) * np.abs(v).max()).all()


@pytest.mark.parametrize("t,n", [(1, 700), (1, 40), (9, 200)])
def test_attend_max_length_cuts(t, n):
    c = _cache(2, 2, 2000, 128, 64)
    _fill(c, seed=11)
    q, lens = _randn((2, t, 4, 128), 12), [n, n - 7]
    want = c.attend(q, _lengths(lens))
    _check_attend(c, q, lens, want)
    got = c.attend(q, _lengths(lens), max_length=n)
    _check_attend(c, q, lens, got)
    cut = c.attend(q, _lengths([2000, n]), max_length=n)       # positions from max_length on are not seen
    _check_attend(c, q, [2000, n], cut, limit=n)
    assert (c.attend(q, _lengths(lens), max_length=0) == 0).all()


@pytest.mark.parametrize("t", [1, 6, 40])
def test_rows_behind_the_length_do_not_matter(t):
    """Codes of any value and scales of NaN or infinity behind the last position, and behind a query's
    own position for the queries before it."""
    n = 83
    c = _cache(1, 2, 200, 128, 32)
    _fill(c, seed=13)
    q = _randn((1, t, 4, 128), 14)
    want = c.attend(q, _lengths([n]))
    held = _held(c)
    c.scales[:, :, n:] = float("nan")
    c.scales[:, :, n + 3::2] = float("inf")
    c.k_codes[:, :, n:] = 0
    assert torch.equal(c.attend(q, _lengths([n])), want)
    c.scales[:, :, n - 1] = float("nan")                       # the last query's own position
    got = c.attend(q, _lengths([n]))
    assert got[0, -1].isnan().all() and torch.equal(got[0, :-1], want[0, :-1])
    _check_attend(c, q[:, :-1], [n - 1], got[:, :-1], held=held) if t > 1 else None


def test_attend_strided_queries():
    c = _cache(2, 8, 50, 128, 32)
    _fill(c, seed=15)
    qkv = _randn((2, 3, 4096), 16)
    q = qkv[..., :2048].view(2, 3, 16, 128)
    want = c.attend(q.contiguous(), _lengths([50, 20]))
    odd = torch.empty(q.numel() + 1, dtype=q.dtype, device="cuda")[1:].view(q.shape)
    odd.copy_(q)
    for x in (q, odd, q.transpose(1, 2).contiguous().transpose(1, 2), q.transpose(2, 3).contiguous().transpose(2, 3)):
        assert torch.equal(c.attend(x, _lengths([50, 20])), want)


def test_long_cache_past_32_bit_offsets():
    """Codes of more than 2^32 bytes: the last sequence lies behind that offset."""
    b, h, s, d = 68, 8, 131072, 128                            # 4.56 GB of key codes
    c = _cache(b, h, s, d, 128)
    n, q = 300, _randn((b, 1, 8, d), 17)
    k, v = _randn((b, 200, h, d), 18), _randn((b, 200, h, d), 19)
    lens = torch.full((b,), n, dtype=torch.int32, device="cuda")
    c.append(k[:, :100], v[:, :100], lens - 200)
    c.append(k, v, lens)
    got = c.read(lens, 200, torch.float32)
    u, sc = q4_ref.kv4_quantize(_np(k[-1]), 128)
    assert torch.equal(got[0][-1].cpu().double(), torch.from_numpy(q4_ref.kv4_values(u, sc)))
    out = c.attend(q, lens, max_length=n)
    held = [q4_ref.kv4_values(q4_ref.unpack(x[-1:, :, :n].cpu().numpy()), _np(c.scales[-1:, :, :n, i]))
            for i, x in enumerate((c.k_codes, c.v_codes))]
    ref = q4_ref.attend(_np(q[-1:]), held[0], held[1], [n], d ** -0.5)
    bound = half_step(ref, torch.bfloat16) * 1.01 + ATTEND_ABS * np.abs(held[1]).max()
    assert (np.abs(_np(out[-1:]) - ref) <= bound).all()


def test_two_streams_and_two_graphs():
    """Calls on two streams at once, and two captured graphs replayed at once with lengths that move
    between replays, over one cache."""
    c = _cache(1, 8, 4096, 128, 32)
    _fill(c, seed=21)
    qs = [_randn((1, 1, 16, 128), 22 + i) for i in range(2)]
    lens = [_lengths([4000]), _lengths([3000])]
    want = [c.attend(q, n) for q, n in zip(qs, lens)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(c.attend(qs[i], lens[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i in range(2) for y in got[i])
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(c.attend(qs[i], lens[i]))
        graphs.append(g)
    for n in ([4000, 3000], [17, 4096], [0, 1], [4000, 3000]):
        for i in range(2):
            lens[i].fill_(n[i])
        torch.cuda.synchronize()
        for st, g in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i], c.attend(qs[i], lens[i]))


def test_captured_decode_loop():
    """append + attend captured once and replayed for token after token: the same as eager calls."""
    h, d, start = 2, 128, 60
    eager, cap = _cache(1, h, 80, d, 64), _cache(1, h, 80, d, 64)
    for c in (eager, cap):
        _fill(c, seed=23)
    k, v, q, n = _randn((1, 1, h, d), 1), _randn((1, 1, h, d), 2), _randn((1, 1, 4, d), 3), _lengths([start])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        n.add_(1)
        cap.append(k, v, n)
        out = cap.attend(q, n)
    n.fill_(start)
    for i in range(12):
        ki, vi, qi = (_randn(x.shape, 100 + 3 * i + j) for j, x in enumerate((k, v, q)))
        k.copy_(ki), v.copy_(vi), q.copy_(qi)
        g.replay()
        m = _lengths([start + i + 1])
        eager.append(ki, vi, m)
        assert torch.equal(out, eager.attend(qi, m))
    assert all(torch.equal(a, b) for a, b in zip(_state(eager), _state(cap)))


def test_argument_contracts():
    c = _cache(2, 4, 32, 128, 32)
    k, n = torch.zeros(2, 1, 4, 128, dtype=torch.bfloat16, device="cuda"), _lengths([1, 1])
    bad = [(lambda: c.append(k.float(), k.float(), n), "only supports"), (lambda: c.append(k, k.half(), n), "Shape mismatch"),
           (lambda: c.append(k[:1], k[:1], n), "must be"), (lambda: c.append(k, k[:, :, :, :64], n), "must be"),
           (lambda: c.append(k[:, :, :2], k[:, :, :2], n), "must be"), (lambda: c.append(k.cpu(), k, n), "is on"),
           (lambda: c.append(k, k, n.long()), "lengths"), (lambda: c.append(k, k, n[:1]), "lengths"),
           (lambda: c.append(k, k, n.cpu()), "lengths"), (lambda: c.read(n, -1), "negative"),
           (lambda: c.read(n, 1, torch.float64), "dtype"), (lambda: c.attend(k[:, :, :3], n), "not a multiple"),
           (lambda: c.attend(k, n, max_length=33), "max_length"), (lambda: c.attend(k, n, max_length=-1), "max_length"),
           (lambda: c.attend(k.requires_grad_(), n), "no backward")]
    for f, match in bad:
        with pytest.raises(ValueError, match=match):
            f()
    k = k.detach()
    assert c.attend(k[:, :0], n).shape == (2, 0, 4, 128) and c.read(n, 0)[0].shape == (2, 0, 4, 128)
    c.append(k[:, :0], k[:, :0], n)


@pytest.mark.parametrize("b,t,h,r,s", [(2, 5, 7, 3, 700), (1, 3, 1, 256, 40), (1, 1, 256, 2, 33), (3, 11, 5, 13, 90),
                                       (1, 2, 3, 255, 1100)])
def test_attend_odd_and_largest_head_counts(b, t, h, r, s):
    """Every query row finds its head and its position for head counts that are no power of two."""
    c = _cache(b, h, s, 128, 64)
    _fill(c, seed=31)
    q, lens = _randn((b, t, h * r, 128), 32), [s - 5 * i for i in range(b)]
    _check_attend(c, q, lens, c.attend(q, _lengths(lens)))


@pytest.mark.parametrize("dtype,top", [(torch.bfloat16, 0), (torch.bfloat16, -62), (torch.bfloat16, -60), (torch.bfloat16, 127),
                                       (torch.bfloat16, -126), (torch.float16, 0), (torch.float16, 15)])
def test_append_every_pair_of_mantissas(dtype, top):
    """Codes and scales are those of exact quotients: every mantissa as a group's maximum 2^top .. with
    every mantissa of the four binades up to it (every 7th for fp16), ties among them."""
    bits = 7 if dtype == torch.bfloat16 else 10
    mant = 1 + torch.arange(1 << bits, dtype=torch.float64) / (1 << bits)
    x = torch.cat([mant * 2.0 ** -e for e in range(4)])[::1 if bits == 7 else 7]
    x = torch.cat([x, torch.zeros(-x.numel() % 31, dtype=x.dtype)])
    rows = []
    for m in mant:
        y = torch.where(x <= m, x, x / 2).view(-1, 31)
        rows.append(torch.cat([m.expand(y.shape[0], 1), y * torch.where(torch.arange(31) % 2 == 0, 1.0, -1.0)], 1))
    y = (torch.cat(rows) * 2.0 ** top).to(dtype)                 # exact, but for bf16's smallest
    y = torch.cat([y, torch.zeros(-y.shape[0] % 4, 32, dtype=dtype)]).view(1, -1, 1, 128)
    t = y.shape[1]
    c = _cache(1, 1, t, 128, 32)
    c.append(y.cuda(), -y.cuda(), _lengths([t]))
    u, s = q4_ref.kv4_quantize(_np(y)[0, :, 0], 32)
    assert np.array_equal(c.scales[0, 0, :, 0].double().cpu().numpy(), s)
    assert np.array_equal(c.scales[0, 0, :, 1].double().cpu().numpy(), s)
    for codes, want in ((c.k_codes, u), (c.v_codes, 16 - u)):
        got = torch.stack([codes[0, 0] & 15, codes[0, 0] >> 4], -1).flatten(-2).cpu().numpy()
        assert np.array_equal(got, want)
