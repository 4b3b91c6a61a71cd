"""token_logprobs on the GPU against the float64 softmax (oracle/q4_ref.py): values within LOGPROB_ABS
(tests/q4_tolerances.py), tokens exactly; the decoder's and the quality harness's use of it."""
import math

import numpy as np
import pytest
import torch

from oracle import q4_ref
from tests.q4_tolerances import LOGPROB_ABS

pytestmark = pytest.mark.gpu


def _lp(*args, **kw):
    from megaqwen_amd.logprobs import token_logprobs
    return token_logprobs(*args, **kw)


def _close(got, want):
    got = got.double().cpu().numpy()
    # the results are fp32: the lowest less the largest of a type, -2 * 3.4e38, is -inf there
    want = np.where(want < -np.finfo(np.float32).max, -np.inf, want)
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got == -np.inf, want == -np.inf)
    assert not (got == np.inf).any()
    err = np.abs(got[fine] - want[fine])
    # fp32 results: half a step of the result itself on top
    assert (err <= LOGPROB_ABS + 2.0 ** -23 * np.abs(want[fine])).all(), err.max()


def _check(x, tok, k):
    """x: CPU tensor of the tested type."""
    r = _lp(x.cuda(), tok.cuda(), top_k=k)
    rows = x.reshape(-1, x.shape[-1]).double().numpy()
    lp, ent, top, at = q4_ref.token_logprobs(rows, tok.reshape(-1).numpy(), k)
    assert r.logprobs.shape == tok.shape and r.top_tokens.shape == tok.shape + (k,) and r.top_tokens.dtype == torch.int32
    assert np.array_equal(r.top_tokens.cpu().numpy().reshape(at.shape), at)
    _close(r.logprobs.reshape(-1), lp)
    _close(r.entropy.reshape(-1), ent)
    _close(r.top_logprobs.reshape(top.shape), top)
    return r


def _rand(rows, vocab, dtype, seed, std=2.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, vocab, generator=g) * std).to(dtype), torch.randint(0, vocab, (rows,), generator=g)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 2), (3, 7), (2, 63), (1, 64), (5, 65), (2, 1000), (1, 4097),
                                        (7, 32001), (1, 151936), (40, 50021), (300, 2050)])
@pytest.mark.parametrize("k", [0, 1, 5, 20, 32])
def test_shapes(rows, vocab, dtype, k):
    x, tok = _rand(rows, vocab, dtype, rows + vocab)
    _check(x, tok, min(k, vocab))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [1, 700])
def test_ties_take_the_lower_token(dtype, rows):
    """Few distinct values, equal everywhere, +0 against -0, and runs of equal values at the end."""
    g = torch.Generator().manual_seed(3)
    V = 5003
    x = torch.randint(0, 3, (rows, V), generator=g).to(dtype)
    x[0] = 1.5
    tok = torch.randint(0, V, (rows,), generator=g)
    if rows > 3:
        x[1] = 0.0
        x[1, ::2] = -0.0
        x[2] = -1.0
        x[2, V - 25:] = 2.0
        x[3] = torch.arange(V).to(dtype)
    _check(x, tok, 32)


@pytest.mark.parametrize("vocab", [40, 3000, 151936])
def test_top_tokens_close_together(vocab):
    """The largest values next to each other, and spread at strides that one thread or wave could
    hold alone."""
    g = torch.Generator().manual_seed(4)
    rows = []
    for step in (1, 2, 4, 8, 64, 256, 512, 1024, 2048, 4096):
        x = torch.randn(vocab, generator=g)
        at = (5 + torch.arange(60) * step) % vocab
        x[at] = 8.0 + torch.rand(60, generator=g)
        rows.append(x)
    x = torch.stack(rows)
    _check(x, torch.zeros(len(rows), dtype=torch.int64), 32)
    _check(x[3:4], torch.zeros(1, dtype=torch.int64), 32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [1, 600])
def test_masked_rows(dtype, rows):
    """-inf and the type's lowest value as masks: all but one, all but a few, all; infinities and NaN."""
    V = 9001
    x, tok = _rand(rows, V, dtype, 5)
    low = torch.finfo(dtype).min
    kinds = 9
    for i in range(min(rows, kinds)):
        j = i if rows > 1 else None
        for kind in ([i] if j is not None else range(kinds)):
            y = x[i].clone()
            keep = torch.zeros(V, dtype=torch.bool)
            if kind in (0, 3):
                keep[1234] = True
            elif kind in (1, 4):
                keep[torch.tensor([0, 17, V - 1])] = True
            if kind <= 2:
                y[~keep] = -math.inf
            elif kind <= 5:
                y[~keep] = low
            elif kind == 6:
                y[77] = math.nan
            elif kind == 7:
                y[4000] = math.inf
            else:
                y[::2] = low
                y[1::2] = torch.finfo(dtype).max
            if j is None:
                _check(y[None], tok, 6)
            else:
                x[i] = y
    _check(x, tok, 6)


def test_large_spread_and_flat_rows():
    V = 20000
    x = torch.stack([torch.linspace(-4e4, 4e4, V), torch.zeros(V), torch.full((V,), 30.0), torch.linspace(0, 1e-3, V)])
    x[1, 7] = 40.0
    _check(x, torch.tensor([V - 1, 7, 3, 0]), 8)


def test_tokens_outside_and_leading_dimensions():
    x, tok = _rand(12, 1001, torch.float32, 6)
    tok[3], tok[4], tok[5] = -1, 1001, 2 ** 40
    _check(x, tok, 2)
    tok32 = tok.clamp(-100, 2000).int()
    r = _check(x.view(3, 4, 1001), tok32.view(3, 4), 2)
    assert r.logprobs.shape == (3, 4)
    one = _lp(x[0].cuda(), tok32[0].cuda(), top_k=2)
    assert one.logprobs.shape == () and one.top_tokens.shape == (2,)
    assert torch.equal(one.top_tokens, r.top_tokens.view(12, 2)[0])
    assert _lp(x[:0].cuda(), tok[:0].cuda(), top_k=2).top_logprobs.shape == (0, 2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strided_and_unaligned_rows(dtype):
    """Rows inside a wider, odd-sized buffer (every alignment), one row expanded, transposed logits."""
    g = torch.Generator().manual_seed(7)
    wide = (torch.randn(9, 4111, generator=g) * 3).to(dtype)
    tok = torch.randint(0, 4000, (9,), generator=g)
    for off in (0, 1, 3, 7):
        view = wide.cuda()[:, off:off + 4000]
        got, want = _lp(view, tok.cuda(), top_k=4), _check(wide[:, off:off + 4000].contiguous(), tok, 4)
        for a, b in zip(got, want):
            assert torch.allclose(a.double(), b.double(), rtol=0, atol=2 * LOGPROB_ABS)
        assert torch.equal(got.top_tokens, want.top_tokens)
    row = wide[:1, :4000].cuda().contiguous()
    got, want = _lp(row.expand(9, 4000), tok.cuda(), top_k=4), _lp(row.repeat(9, 1), tok.cuda(), top_k=4)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    t = wide[:, :4000].cuda().t().contiguous().t()
    assert torch.equal(_lp(t, tok.cuda(), top_k=4).top_tokens, _lp(t.contiguous(), tok.cuda(), top_k=4).top_tokens)


@pytest.mark.parametrize("rows", [1, 33])
def test_streams_and_graph(rows):
    xs = [_rand(rows, 60000, torch.bfloat16, 10 + i) for i in range(3)]
    dev = [(x.cuda(), t.cuda()) for x, t in xs]
    want = [_lp(x, t, top_k=20) for x, t in dev]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for st, (x, t) in zip(streams, dev):
        with torch.cuda.stream(st):
            got.append(_lp(x, t, top_k=20))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    x, t, g = dev[0][0].clone(), dev[0][1].clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = _lp(x, t, top_k=20)
    for i in (1, 2, 0, 1):
        x.copy_(dev[i][0]), t.copy_(dev[i][1])
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want[i]))


def test_argument_contracts():
    x, t = torch.zeros(2, 40, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
    for f, match in ((lambda: _lp(x.double(), t), "only supports"), (lambda: _lp(x, t.float()), "int32 or int64"),
                     (lambda: _lp(x, t[:1]), "Shape mismatch"), (lambda: _lp(x, t.cpu()), "is on"),
                     (lambda: _lp(x, t, top_k=33), "top_k"), (lambda: _lp(x, t, top_k=-1), "top_k"),
                     (lambda: _lp(x[:, :3], t, top_k=4), "top_k"), (lambda: _lp(x[:, :0], t), "vocab"),
                     (lambda: _lp(x.requires_grad_(), t), "no backward")):
        with pytest.raises(ValueError, match=match):
            f()


def test_decoder_and_quality_harness():
    """decode_step_with_logprobs and decoder_logprobs agree with log_softmax of the decoder's logits."""
    from megaqwen_amd.quality import decoder_logprobs, decoder_perplexity, perplexity_from_logits
    from tests.helpers import build_pair
    dec, _, sp, _ = build_pair(1, 2000, 64, seed=3, norm_jitter=0.1, oracle=False)
    ids = [5, 1999, 0, 77, 3]
    dec.reset()
    steps = [dec.decode_step_with_logits(t) for t in ids]
    logits = torch.stack([s[1] for s in steps])
    lp = torch.log_softmax(logits.double(), -1)
    dec.reset()
    for i, t in enumerate(ids):
        nxt, r = dec.decode_step_with_logprobs(t, top_k=4)
        assert nxt == steps[i][0] and int(r.top_tokens[0]) == nxt
        assert torch.equal(r.top_tokens.long(), torch.topk(lp[i], 4).indices)
        assert abs(float(r.logprobs) - float(lp[i, nxt])) <= LOGPROB_ABS
        assert torch.equal(r.logprobs, r.top_logprobs[0])
    r = decoder_logprobs(dec, ids, top_k=2)
    want = lp[:-1].gather(1, torch.tensor(ids[1:], device="cuda")[:, None])[:, 0]
    assert (r.logprobs.double() - want).abs().max() <= LOGPROB_ABS and r.top_tokens.shape == (4, 2)
    assert decoder_perplexity(dec, ids) == pytest.approx(perplexity_from_logits(logits, torch.tensor(ids)), rel=1e-5)
    with pytest.raises(ValueError, match="top_k"):
        dec.decode_step_with_logprobs(5, top_k=33)
    assert dec.position() == 4                     # refused before the step
