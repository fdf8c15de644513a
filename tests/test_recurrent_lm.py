"""A small recurrent language model made of the operators: scaled_embedding, rms_norm, two blocks of
gated_linear_recurrence (values, then logits) with residual_rms_norm behind each, and
fused_cross_entropy over the tied embedding.

Checked in fp32 against the same model in 64 bits on the CPU.  About twenty operators follow
one another, each within 100 * 2^-24 of its result's norm, and none is expected to magnify an
error by more than 4: 20 * 100 * 2^-24 * 4 = 5e-4 of the norm of what is compared.
"""
import math

import pytest
import torch
import torch.nn.functional as F

from operators.fused_cross_entropy import fused_cross_entropy
from operators.gated_linear_recurrence import (gated_linear_recurrence,
                                               gated_linear_recurrence_step)
from operators.residual_rms_norm import residual_rms_norm
from operators.rms_norm import rms_norm
from operators.scaled_embedding import scaled_embedding

pytestmark = pytest.mark.gpu
DEV = "cuda"
V, N, EPS, SCALE = 211, 96, 1e-5, 8.0
TOL = 5e-4


def _params(dtype=torch.float32):
    gen = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    p = {"emb": r(V, N) / math.sqrt(N), "w0": 1 + 0.1 * r(N)}
    for b in "ab":
        p["proj" + b] = r(N, 4 * N) / math.sqrt(N)
        p["post" + b], p["w" + b], p["s" + b] = 1 + 0.1 * r(N), 1 + 0.1 * r(N), 0.5 + 0.1 * r(N)
    p["decay"] = r(N) - 3
    return {k: t.to(dtype) for k, t in p.items()}


class Plain:
    """The operators' definitions, for any floating type."""

    def embed(self, ids, w):
        return F.embedding(ids, w) * math.sqrt(N)

    def norm(self, x, w):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w

    def scan(self, x, g, beta, decay, reset, h0):
        if decay is None:
            a, b = g, beta * x
        else:
            u = -SCALE * F.softplus(decay) * torch.sigmoid(g)
            a, m = u.exp(), torch.sqrt(-torch.expm1(2 * u))
            if reset is not None:
                a, m = a * ~reset[..., None], torch.where(reset[..., None], torch.ones_like(m), m)
            b = m * torch.sigmoid(beta) * x
        if decay is None and reset is not None:
            a = a * ~reset[..., None]
        h, out = h0 if h0 is not None else torch.zeros_like(x[:, 0]), []
        for t in range(x.shape[1]):
            h = a[:, t] * h + b[:, t]
            out.append(h)
        return torch.stack(out, 1), h

    def glue(self, y, r, w, post, gate, s):
        r = r + s * F.silu(gate) * self.norm(y, post)
        return self.norm(r, w), r

    def loss(self, logits, target):
        return F.cross_entropy(logits, target)


class Own:
    def embed(self, ids, w):
        return scaled_embedding(ids, w, math.sqrt(N))

    def norm(self, x, w):
        return rms_norm(x, (N,), w, EPS)

    def scan(self, x, g, beta, decay, reset, h0):
        return gated_linear_recurrence(x, g, beta, decay, decay_scale=SCALE, reset=reset,
                                       initial_state=h0, output_final_state=True)

    def glue(self, y, r, w, post, gate, s):
        return residual_rms_norm(y, r, w, post_weight=post, gate=gate, scale=s, eps=EPS)

    def loss(self, logits, target):
        return fused_cross_entropy(logits, target)


def _logits(ops, p, ids, reset=None, states=(None, None)):
    r = ops.embed(ids, p["emb"])
    x = ops.norm(r, p["w0"])
    last = []
    for b, h0 in zip("ab", states):
        v, g, beta, gate = (x @ p["proj" + b]).split(N, -1)
        if b == "a":
            g, beta = torch.sigmoid(g + 2), torch.sigmoid(beta)
        y, hT = ops.scan(v, g, beta, p["decay"] if b == "b" else None, reset, h0)
        last.append(hT)
        x, r = ops.glue(y, r, p["w" + b], p["post" + b], gate, p["s" + b])
    return x @ p["emb"].t(), last


def _near(got, ref, name):
    off = float((got.double().cpu() - ref).norm() / ref.norm())
    assert off <= TOL, (name, off)


def _batch(B, L):
    gen = torch.Generator().manual_seed(1)
    ids = torch.randint(0, V, (B, L + 1), generator=gen)
    reset = torch.rand(B, L, generator=gen) < 0.02
    return ids[:, :-1], ids[:, 1:], reset


def test_loss_and_gradients():
    ids, target, reset = _batch(3, 150)
    ref = {k: t.double().requires_grad_() for k, t in _params().items()}
    lr = Plain().loss(_logits(Plain(), ref, ids, reset)[0].reshape(-1, V), target.reshape(-1))
    lr.backward()
    p = {k: t.to(DEV).requires_grad_() for k, t in _params().items()}
    lo = Own().loss(_logits(Own(), p, ids.to(DEV), reset.to(DEV))[0].reshape(-1, V),
                    target.reshape(-1).to(DEV))
    lo.backward()
    assert abs(lo.item() - lr.item()) <= TOL * lr.item()
    for k in p:
        _near(p[k].grad, ref[k].grad, k)


def test_decoding_continues_the_prompt():
    """Logits of a whole sequence, and of a prompt followed by single tokens."""
    ids, _, _ = _batch(4, 40)
    p64 = {k: t.double() for k, t in _params().items()}
    want = _logits(Plain(), p64, ids)[0]
    p = {k: t.to(DEV) for k, t in _params().items()}
    ids = ids.to(DEV)
    got, _ = _logits(Own(), p, ids)
    _near(got, want, "whole")
    got, states = _logits(Own(), p, ids[:, :25])
    for t in range(25, 40):
        r = scaled_embedding(ids[:, t], p["emb"], math.sqrt(N))
        x = rms_norm(r, (N,), p["w0"], EPS)
        for b, state in zip("ab", states):
            v, g, beta, gate = (x @ p["proj" + b]).split(N, -1)
            if b == "a":
                g, beta = torch.sigmoid(g + 2), torch.sigmoid(beta)
            y = gated_linear_recurrence_step(v, g, beta, state, p["decay"] if b == "b" else None,
                                             decay_scale=SCALE)
            x, r = residual_rms_norm(y, r, p["w" + b], post_weight=p["post" + b], gate=gate,
                                     scale=p["s" + b], eps=EPS)
        _near(x @ p["emb"].t(), want[:, t], f"token {t}")


def test_captured_decode_step():
    """One token through the block as a CUDA graph: the states advance with every replay."""
    p = {k: t.to(DEV) for k, t in _params().items()}
    tok = torch.zeros(4, dtype=torch.int64, device=DEV)
    state = torch.zeros(4, N, device=DEV)

    def step():
        r = scaled_embedding(tok, p["emb"], math.sqrt(N))
        v, g, beta, gate = (rms_norm(r, (N,), p["w0"], EPS) @ p["projb"]).split(N, -1)
        y = gated_linear_recurrence_step(v, g, beta, state, p["decay"], decay_scale=SCALE)
        return residual_rms_norm(y, r, p["wb"], post_weight=p["postb"], gate=gate, scale=p["sb"], eps=EPS)[0]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    state.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    state.zero_()
    got = []
    for t in range(6):
        tok.fill_(t + 3)
        graph.replay()
        got.append(out.clone())
    after = state.clone()
    state.zero_()
    for t in range(6):
        tok.fill_(t + 3)
        assert torch.equal(step(), got[t])
    assert torch.equal(state, after)


@pytest.mark.parametrize("B,L", [(1, 1000), (64, 150)])
def test_two_calls_at_once(B, L):
    """The operators on two streams, interleaved: each bit for bit as alone (no library product among
    them; few rows take clusters, many take chains)."""
    ids, _, reset = _batch(B, L)
    ids, reset = ids.to(DEV), reset.to(DEV)
    sets = [{n: t.to(DEV).mul(1 + k / 8).requires_grad_() for n, t in _params().items()} for k in (0, 1)]

    def work(p):
        r = scaled_embedding(ids, p["emb"], math.sqrt(N))
        h = gated_linear_recurrence(r, r, r, p["decay"], decay_scale=SCALE, reset=reset)
        out, res = residual_rms_norm(h, r, p["wa"], post_weight=p["posta"], gate=r, scale=p["sa"], eps=EPS)
        used = [p[k] for k in ("emb", "decay", "wa", "posta", "sa")]
        return [out.detach(), res.detach(), *torch.autograd.grad((out, res), used, (out.detach(), r.detach()))]
    alone = [work(p) for p in sets]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(4):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((k, work(sets[k])))
    torch.cuda.synchronize()
    for k, out in got:
        for a, b in zip(out, alone[k]):
            assert torch.equal(a, b)
