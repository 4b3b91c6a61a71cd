"""token_logprobs without a GPU: its reference against torch's log_softmax and closed forms, the
argument contracts, the C ABI's rejections, and the scoring flow of the quality harness."""
import math

import numpy as np
import pytest
import torch

from megaqwen_amd import _lib, logprobs
from megaqwen_amd.logprobs import TokenLogprobs, token_logprobs
from megaqwen_amd.quality import decoder_logprobs, decoder_perplexity, perplexity_from_logits
from oracle import q4_ref


def test_reference_matches_torch():
    x = torch.randn(6, 501, generator=torch.Generator().manual_seed(0), dtype=torch.float64) * 4
    tok = torch.tensor([0, 500, 7, 7, 250, 3])
    lp, ent, top, at = q4_ref.token_logprobs(x.numpy(), tok.numpy(), 5)
    ref = torch.log_softmax(x, -1)
    np.testing.assert_allclose(lp, ref[torch.arange(6), tok].numpy(), rtol=1e-13)
    np.testing.assert_allclose(ent, torch.distributions.Categorical(logits=x).entropy().numpy(), rtol=1e-12)
    np.testing.assert_array_equal(at, torch.topk(x, 5).indices.numpy())
    np.testing.assert_allclose(top, torch.topk(ref, 5).values.numpy(), rtol=1e-13)


def test_reference_edges():
    x = np.full((3, 8), -np.inf)
    x[1, 5] = 2.0
    x[2] = 1.0
    lp, ent, top, at = q4_ref.token_logprobs(x, [1, 5, 9], 3)
    assert lp[0] == -np.inf and ent[0] == 0 and (at[0] == [0, 1, 2]).all() and (top[0] == -np.inf).all()
    assert lp[1] == 0 and ent[1] == 0 and (at[1] == [5, 0, 1]).all() and (top[1, 1:] == -np.inf).all()
    assert lp[2] == -np.inf and ent[2] == pytest.approx(math.log(8)) and (at[2] == [0, 1, 2]).all()


def test_front_end_on_cpu():
    with pytest.raises(ValueError, match="expects CUDA tensors"):
        token_logprobs(torch.zeros(2, 8), torch.zeros(2, dtype=torch.int64))


def test_c_abi_rejections():
    lib, A = _lib.load(), 1 << 24
    ok = dict(x=A, st=1000, t=2 * A, lp=3 * A, e=4 * A, tl=5 * A, tt=6 * A, r=2, v=1000, k=5, ty=2, ws=7 * A, wb=A)

    def call(**kw):
        a = {**ok, **kw}
        return lib.mq_token_logprobs(a["x"], a["st"], a["t"], 1, a["lp"], a["e"], a["tl"], a["tt"], a["r"],
                                     a["v"], a["k"], a["ty"], a["ws"], a["wb"], None)

    for kw in (dict(x=None), dict(t=None), dict(lp=None), dict(e=None), dict(tl=None), dict(tt=None),
               dict(r=-1), dict(v=0), dict(k=-1), dict(k=33), dict(v=4, k=5), dict(ty=3), dict(st=-1),
               dict(x=A + 2)):
        assert call(**kw) == _lib.MQ_ERR_INVALID_ARG, kw
        assert lib.mq_last_error()
    need = lib.mq_token_logprobs_workspace_bytes(1, 151936, 20)
    if need:
        assert call(r=1, v=151936, k=20, wb=need - 1) == _lib.MQ_ERR_INVALID_ARG
        assert call(r=1, v=151936, k=20, ws=None) == _lib.MQ_ERR_INVALID_ARG
    assert call(r=0) == _lib.MQ_OK
    assert lib.mq_token_logprobs_workspace_bytes(1, 10, 33) == 0


class _StubDecoder:
    """Row i of fixed logits for the i-th decoded token."""

    def __init__(self, logits):
        self.logits, self.fed = logits, []

    def reset(self):
        self.fed = []

    def decode_step_with_logits(self, t):
        self.fed.append(t)
        row = self.logits[len(self.fed) - 1]
        return int(row.argmax()), row


def test_scoring_flow(monkeypatch):
    """decoder_logprobs feeds every token but the last and scores the next one; its perplexity is
    perplexity_from_logits'."""
    def plain(logits, tokens, *, top_k=0):
        lp = torch.log_softmax(logits.double(), -1)
        top = torch.topk(lp, top_k)
        return TokenLogprobs(lp[tokens], -(lp.exp() * lp).sum(), top.values, top.indices.int())

    monkeypatch.setattr(logprobs, "token_logprobs", plain)
    x = torch.randn(5, 40, generator=torch.Generator().manual_seed(3))
    ids = [4, 9, 9, 30, 2]
    dec = _StubDecoder(x)
    r = decoder_logprobs(dec, ids, top_k=3)
    assert dec.fed == ids[:-1]
    assert r.logprobs.shape == (4,) and r.entropy.shape == (4,) and r.top_tokens.shape == (4, 3)
    assert torch.equal(r.top_tokens[:, 0].long(), x[:4].argmax(-1))
    assert decoder_perplexity(dec, ids) == pytest.approx(perplexity_from_logits(x, torch.tensor(ids)), rel=1e-6)
    with pytest.raises(ValueError):
        decoder_logprobs(dec, [4])
