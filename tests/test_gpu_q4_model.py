"""A token in 4 bits, end to end: a small decoder whose projections are w4_linear, whose cache is
KV4Cache and whose tokens are scored by token_logprobs, over a prompt, a padded batch and single tokens.
Every operator's result is checked in float64 on the inputs that it got."""
import numpy as np
import pytest
import torch

from oracle import q4_ref
from tests.q4_tolerances import ATTEND_ABS, LOGPROB_ABS, half_step, w4_bound

pytestmark = pytest.mark.gpu

H, INTER, HQ, HK, D, VOCAB, LAYERS, GROUP = 512, 768, 8, 4, 128, 3001, 2, 64


def _np(t):
    return t.double().cpu().numpy()


def _rms(x):
    return (x.float() * torch.rsqrt(x.float().pow(2).mean(-1, keepdim=True) + 1e-6)).to(x.dtype)


class _Model:
    def __init__(self, batch, max_seq):
        from megaqwen_amd.kv4 import KV4Cache
        from megaqwen_amd.w4 import quantize_w4
        g = torch.Generator().manual_seed(0)

        def w4(n, k, symmetric=True):
            w = torch.randn(n, k, generator=g) * k ** -0.5
            return [None if t is None else t.cuda() for t in quantize_w4(w, GROUP, symmetric=symmetric)]

        self.embed = torch.randn(VOCAB, H, generator=g).to(torch.bfloat16).cuda()
        self.layers = [{"qkv": w4((HQ + 2 * HK) * D, H), "o": w4(H, HQ * D), "gu": w4(2 * INTER, H, False),
                        "down": w4(H, INTER, False)} for _ in range(LAYERS)]
        self.head = w4(VOCAB, H)
        self.caches = [KV4Cache(batch, HK, max_seq, D, 32) for _ in range(LAYERS)]

    def linear(self, x, w, **kw):
        from megaqwen_amd.w4 import w4_linear
        y = w4_linear(x, *w, **kw)
        q, s, z = w
        xs = _np(x).reshape(-1, x.shape[-1])
        ref = xs @ q4_ref.w4_weight(q.cpu().numpy(), _np(s), None if z is None else z.cpu().numpy()).T
        if kw.get("residual") is not None:
            ref = ref + _np(kw["residual"]).reshape(ref.shape)
        bound = w4_bound(xs, _np(s), ref, x.shape[-1], GROUP, y.dtype)
        assert (np.abs(_np(y).reshape(ref.shape) - ref) <= bound).all()
        return y

    def step(self, tokens, lengths):
        """Logits (fp32) of [batch, t] tokens at the last t positions of every sequence."""
        x = self.embed[tokens]
        b, t = tokens.shape
        n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        for lay, cache in zip(self.layers, self.caches):
            qkv = self.linear(_rms(x), lay["qkv"])
            q, k, v = qkv.split([HQ * D, HK * D, HK * D], -1)
            q, k = (_rms(y.unflatten(-1, (-1, D))) for y in (q, k))
            v = v.unflatten(-1, (HK, D))
            cache.append(k, v, n)
            back = cache.read(n, t, torch.float32)
            for y, got in zip((k, v), back):
                u, s = q4_ref.kv4_quantize(_np(y), cache.group_size)
                want = q4_ref.kv4_values(u, s)
                for j, m in enumerate(lengths):
                    want[j, :max(0, t - m)] = 0
                assert np.array_equal(_np(got), want)
            att = cache.attend(q, n, max_length=max(lengths))
            held = [q4_ref.kv4_values(q4_ref.unpack(c.cpu().numpy()), _np(cache.scales[:, :, :, i]))
                    for i, c in enumerate((cache.k_codes, cache.v_codes))]
            ref = q4_ref.attend(_np(q), *held, lengths, D ** -0.5)
            assert (np.abs(_np(att) - ref) <= half_step(ref, att.dtype) * 1.01 + ATTEND_ABS * np.abs(held[1]).max()).all()
            x = self.linear(att.flatten(-2), lay["o"], residual=x)
            gate, up = self.linear(_rms(x), lay["gu"]).chunk(2, -1)
            x = self.linear(torch.nn.functional.silu(gate) * up, lay["down"], residual=x)
        return self.linear(_rms(x), self.head, out_dtype=torch.float32)


def test_prompt_then_tokens():
    from megaqwen_amd.logprobs import token_logprobs
    m = _Model(2, 40)
    prompt = torch.randint(0, VOCAB, (2, 21), generator=torch.Generator().manual_seed(1)).cuda()
    lengths = [21, 13]                                 # the second prompt is padded by 8 rows
    logits = m.step(prompt, lengths)
    # scoring the prompt: row i for token i + 1
    r = token_logprobs(logits[:, :-1], prompt[:, 1:], top_k=3)
    lp, ent, top, at = q4_ref.token_logprobs(_np(logits[:, :-1]).reshape(-1, VOCAB), prompt[:, 1:].cpu().numpy().ravel(), 3)
    assert np.array_equal(r.top_tokens.cpu().numpy().reshape(at.shape), at)
    for got, want in ((r.logprobs, lp), (r.entropy, ent), (r.top_logprobs, top)):
        assert (np.abs(_np(got).reshape(want.shape) - want) <= LOGPROB_ABS).all()
    nxt = token_logprobs(logits[:, -1], prompt[:, -1], top_k=1).top_tokens.long()
    single = []
    for i in range(5):                                 # greedy tokens, one at a time
        lengths = [n + 1 for n in lengths]
        logits = m.step(nxt, lengths)
        single.append(nxt)
        nxt = token_logprobs(logits[:, -1], nxt[:, 0], top_k=1).top_tokens.long()
        assert torch.equal(nxt, logits[:, -1].argmax(-1, keepdim=True))
    # the same five tokens as one chunk over a cache that went back to the prompt
    chunk = m.step(torch.cat(single, 1), lengths)
    assert torch.equal(chunk[:, -1].argmax(-1, keepdim=True), nxt) or \
        (chunk[:, -1] - logits[:, -1]).abs().max() < 0.1 * logits.abs().max()
