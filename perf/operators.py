"""Timing cases of the layers around a recurrent language-model block.

Four operators, each in its plain form (elementary torch operations in 32 bits,
rounded once at the end) and through this package's public functions:

  recurrence  h_t = a_t h_{t-1} + b_t per channel over a long axis, forward and backward.
              gates "values": a_t = g_t, b_t = beta_t x_t.
              gates "logits": a_t = exp(-8 softplus(decay) sigmoid(g_t)),
                              b_t = sqrt(1 - a_t^2) sigmoid(beta_t) x_t.
              A step marked in `reset` takes a_t as 0.
  step        the same recurrence for one token of each sequence, the state updated in place.
  norm        r' = r + s * u,  out = rms_norm(r') w,  u = act(gate) rms_norm(y) w_post.
  embedding   out = scale * W[ids], and W's gradient.

`own` selects which of the two `run` computes.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
EPS = 1e-6
DECAY_SCALE = 8.0
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one new token of each of 64 sequences being decoded, 16 heads of 128 channels
        {"name": "step_64x2048_bf16", "op": "step", "B": 64, "C": 2048, "type": "bf16", "gates": "logits"},
        # one long prompt of one user; x and both gates are column blocks of one projection
        {"name": "recurrence_prompt_16384", "op": "recurrence", "B": 1, "L": 16384, "C": 2048, "type": "bf16", "gates": "logits",
         "train": False, "packed": True, "reset": False},
        # a training step of the layer at the delta rule's benchmark size
        {"name": "recurrence_train_8x8192", "op": "recurrence", "B": 8, "L": 8192, "C": 2048, "type": "bf16", "gates": "logits",
         "train": True, "packed": False, "reset": False},
        # fp32 fine-tuning on ragged sizes, with documents that end inside a sequence
        {"name": "recurrence_train_odd_fp32", "op": "recurrence", "B": 3, "L": 1021, "C": 1111, "type": "fp32", "gates": "values",
         "train": True, "packed": False, "reset": True},
        # the block's norms while 16 sequences are decoded
        {"name": "norm_16x4096_bf16", "op": "norm", "M": 16, "N": 4096, "type": "bf16", "act": "silu", "post": True, "train": False},
        # a training step's norms at the rms_norm benchmark sizes
        {"name": "norm_train_16384x8192", "op": "norm", "M": 16384, "N": 8192, "type": "bf16", "act": "silu", "post": True, "train": True},
        {"name": "norm_train_4096x4096_fp32", "op": "norm", "M": 4096, "N": 4096, "type": "fp32", "act": "none", "post": True, "train": True},
        # a narrow odd width, sigmoid gate, no norm behind the block
        {"name": "norm_train_odd_fp16", "op": "norm", "M": 5003, "N": 1001, "type": "fp16", "act": "sigmoid", "post": False, "train": True},
        # the tokens of 16 sequences being decoded, into the cross-entropy benchmark's vocabulary
        {"name": "embedding_16_bf16", "op": "embedding", "T": 16, "V": 128256, "N": 4096, "type": "bf16", "ids": "zipf", "train": False},
        # a training step's tokens, distributed as words are
        {"name": "embedding_train_16384", "op": "embedding", "T": 16384, "V": 128256, "N": 4096, "type": "bf16", "ids": "zipf", "train": True},
        # a small vocabulary of odd width in fp32, one token in three the same (padding)
        {"name": "embedding_train_odd_fp32", "op": "embedding", "T": 30011, "V": 5003, "N": 771, "type": "fp32", "ids": "pad", "train": True},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm; half of them multiples of 8 where that fits."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    n = max(lo, min(hi, n))
    if rng.random() < 0.5 and n >= 16:
        n -= n % 8
    return n


def draw(rng):
    op = rng.choice(["recurrence", "recurrence", "norm", "norm", "embedding", "embedding", "step"])
    kind = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    train = rng.random() < 0.6
    if op == "step":
        return {"op": op, "B": _spread(rng, 1, 512), "C": _spread(rng, 64, 8192), "type": kind, "gates": rng.choice(["logits", "values"])}
    if op == "recurrence":
        C, L = _spread(rng, 64, 4096), _spread(rng, 1, 32768)
        B = max(1, min(_spread(rng, 1, 16), (64 << 20) // (C * L)))
        return {"op": op, "B": B, "L": L, "C": C, "type": kind, "gates": rng.choice(["logits", "values"]), "train": train,
                "packed": not train and rng.random() < 0.5, "reset": rng.random() < 0.3}
    if op == "norm":
        N = _spread(rng, 64, 16384)
        M = _spread(rng, 1, max(2, min(32768, (64 << 20) // N)))
        return {"op": op, "M": M, "N": N, "type": kind, "act": rng.choice(["silu", "sigmoid", "none"]), "post": rng.random() < 0.7, "train": train}
    N, V = _spread(rng, 64, 8192), _spread(rng, 100, 131072)
    V = min(V, max(100, (256 << 20) // N))
    return {"op": op, "T": _spread(rng, 1, max(2, min(65536, (64 << 20) // N))), "V": V, "N": N, "type": kind,
            "ids": rng.choice(["zipf", "uniform", "pad"]), "train": train}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    t = TYPES[case["type"]]
    op = case["op"]
    train = case.get("train", False)

    def normal(*shape, mean=0.0, std=1.0):
        return torch.randn(*shape, generator=gen, device=DEV) * std + mean

    def uniform(*shape):
        return torch.rand(*shape, generator=gen, device=DEV)

    def leaf(v, kind=t):
        return v.to(kind).requires_grad_(train)

    s = {"case": case}
    if op in ("recurrence", "step"):
        B, C = case["B"], case["C"]
        shape = (B, case["L"], C) if op == "recurrence" else (B, C)
        x, g, beta = normal(*shape), normal(*shape), normal(*shape)
        if case["gates"] == "values":
            g, beta = torch.sigmoid(g + 3.0), torch.sigmoid(beta)
        else:
            # decays of 0.9 to 0.999 a step where the gate is fully open
            a = 0.9 + 0.099 * uniform(C)
            s["decay"] = leaf(torch.log(torch.expm1(-torch.log(a) / DECAY_SCALE)), torch.float32)
        if case.get("packed"):
            x, g, beta = torch.cat((x, g, beta), -1).to(t).split(C, -1)
        else:
            x, g, beta = leaf(x), leaf(g), leaf(beta)
        s.update(x=x, g=g, beta=beta, state=leaf(normal(B, C, std=0.5), torch.float32))
        if op == "recurrence":
            if case["reset"]:
                s["reset"] = uniform(B, case["L"]) < 0.004
            if train:
                s["dh"] = normal(*shape).to(t)
                s["dstate"] = normal(B, C)
    elif op == "norm":
        M, N = case["M"], case["N"]
        s.update(y=leaf(normal(M, N)), r=leaf(normal(M, N, std=2.0)), w=leaf(normal(N, mean=1.0, std=0.1)),
                 scale=leaf(normal(N, mean=0.5, std=0.1)))
        if case["act"] != "none":
            s["gate"] = leaf(normal(M, N))
        if case["post"]:
            s["w_post"] = leaf(normal(N, mean=1.0, std=0.1))
        if train:
            s.update(dout=normal(M, N).to(t), dr=normal(M, N).to(t))
    else:
        T, V, N = case["T"], case["V"], case["N"]
        u = uniform(T)
        if case["ids"] == "zipf":
            rank = torch.exp(u * math.log(V)).to(torch.int64) - 1
            ids = torch.randperm(V, generator=gen, device=DEV)[rank.clamp_(0, V - 1)]
        else:
            ids = (u * V).to(torch.int64).clamp_(0, V - 1)
            if case["ids"] == "pad":
                ids[uniform(T) < 1 / 3] = V // 2
        s.update(ids=ids, weight=leaf(normal(V, N, std=0.02)), scale=math.sqrt(N))
        if train:
            s["dout"] = normal(T, N).to(t)
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t along dim 1, by doubling."""
    n = 1
    while n < a.shape[1]:
        b = torch.cat((b[:, :n], b[:, n:] + a[:, n:] * b[:, :-n]), 1)
        a = torch.cat((a[:, :n], a[:, n:] * a[:, :-n]), 1)
        n *= 2
    return b


def _gates(s, kind):
    """(x, a, m, i, parts): the decay a, the input's factors m and i."""
    x, g, beta = s["x"].to(kind), s["g"].to(kind), s["beta"].to(kind)
    if s["case"]["gates"] == "values":
        a, m, i, parts = g, None, beta, None
    else:
        sp = torch.log1p(torch.exp(s["decay"].to(kind)))
        sg, i = 1 / (1 + torch.exp(-g)), 1 / (1 + torch.exp(-beta))
        u = -DECAY_SCALE * sp * sg
        a, parts = torch.exp(u), (u, sg)
    if "reset" in s:
        a = torch.where(s["reset"][:, :, None], torch.zeros_like(a), a)
    if parts is not None:
        m = torch.sqrt(-torch.expm1(2 * u))
        if "reset" in s:
            m = torch.where(s["reset"][:, :, None], torch.ones_like(m), m)
    return x, a, m, i, parts


def _plain_recurrence(s):
    c, f = s["case"], torch.float32
    t = TYPES[c["type"]]
    x, a, m, i, parts = _gates(s, f)
    b = i * x if m is None else m * i * x
    h0 = s["state"].detach()
    b[:, 0] += a[:, 0] * h0
    h = _scan(a, b)
    outs = [h.to(t), h[:, -1].clone()]
    if not c["train"]:
        return outs
    d = s["dh"].to(f, copy=True)
    d[:, -1] += s["dstate"]
    later = torch.cat((a[:, 1:], torch.zeros_like(a[:, :1])), 1)
    d = _scan(later.flip(1), d.flip(1)).flip(1)
    before = torch.cat((h0[:, None], h[:, :-1]), 1)
    if parts is None:
        dg = d * before
        if "reset" in s:
            dg = torch.where(s["reset"][:, :, None], torch.zeros_like(dg), dg)
        return outs + [(d * i).to(t), dg.to(t), (d * x).to(t), a[:, 0] * d[:, 0]]
    u, sg = parts
    du = d * (before * a - i * x * a * a / m)
    if "reset" in s:
        du = torch.where(s["reset"][:, :, None], torch.zeros_like(du), du)
    ddecay = (du * sg).sum((0, 1)) * (-DECAY_SCALE / (1 + torch.exp(-s["decay"])))
    return outs + [(d * m * i).to(t), (du * u * (1 - sg)).to(t), (d * m * x * i * (1 - i)).to(t), a[:, 0] * d[:, 0], ddecay]


def _plain_step(s):
    x, a, m, i, _ = _gates(s, torch.float32)
    h = a * s["state"] + (i * x if m is None else m * i * x)
    s["state"].copy_(h)
    return [h.to(TYPES[s["case"]["type"]]), s["state"]]


def _act(case, gate):
    """The gate's factor and its derivative."""
    sg = 1 / (1 + torch.exp(-gate))
    if case["act"] == "sigmoid":
        return sg, sg * (1 - sg)
    return gate * sg, sg * (1 + gate * (1 - sg))


def _plain_norm(s):
    c, f = s["case"], torch.float32
    t = TYPES[c["type"]]
    y, r, w, scale = (s[k].to(f) for k in ("y", "r", "w", "scale"))
    p = y
    if c["post"]:
        inv1 = 1 / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS)
        n, wp = y * inv1, s["w_post"].to(f)
        p = n * wp
    u = p
    if c["act"] != "none":
        act, slope = _act(c, s["gate"].to(f))
        u = p * act
    r2 = r + scale * u
    inv2 = 1 / torch.sqrt((r2 * r2).mean(-1, keepdim=True) + EPS)
    outs = [(r2 * inv2 * w).to(t), r2.to(t)]
    if not c["train"]:
        return outs
    do = s["dout"].to(f)
    e = do * w
    d = s["dr"].to(f) + inv2 * e - r2 * inv2 ** 3 * (e * r2).mean(-1, keepdim=True)
    dw, dscale, dp = (do * r2 * inv2).sum(0), (d * u).sum(0), d * scale
    more = []
    if c["act"] != "none":
        more.append((dp * p * slope).to(t))
        dp = dp * act
    dy = dp
    if c["post"]:
        more.append((dp * n).sum(0).to(t))
        k = dp * wp
        dy = inv1 * k - y * inv1 ** 3 * (k * y).mean(-1, keepdim=True)
    return outs + [dy.to(t), d.to(t), dw.to(t), dscale.to(t)] + more


def _plain_embedding(s):
    c, f = s["case"], torch.float32
    t = TYPES[c["type"]]
    outs = [(s["weight"][s["ids"]].to(f) * s["scale"]).to(t)]
    if c["train"]:
        dw = torch.zeros(c["V"], c["N"], dtype=f, device=DEV)
        dw.index_add_(0, s["ids"], s["dout"].to(f))
        outs.append((dw * s["scale"]).to(t))
    return outs


# ---------------------------------------------------------------------------
# this package's calls
# ---------------------------------------------------------------------------
def _package():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flag-operators_b200")
    if root not in sys.path:
        sys.path.insert(0, root)


def _own_recurrence(s):
    from operators.gated_linear_recurrence import gated_linear_recurrence
    h, last = gated_linear_recurrence(s["x"], s["g"], s["beta"], s.get("decay"), decay_scale=DECAY_SCALE, initial_state=s["state"],
                                      reset=s.get("reset"), output_final_state=True)
    if not s["case"]["train"]:
        return [h, last]
    leaves = [s["x"], s["g"], s["beta"], s["state"]] + ([s["decay"]] if "decay" in s else [])
    return [h.detach(), last.detach(), *torch.autograd.grad((h, last), leaves, (s["dh"], s["dstate"]))]


def _own_step(s):
    from operators.gated_linear_recurrence import gated_linear_recurrence_step
    return [gated_linear_recurrence_step(s["x"], s["g"], s["beta"], s["state"], s.get("decay"), decay_scale=DECAY_SCALE), s["state"]]


def _own_norm(s):
    from operators.residual_rms_norm import residual_rms_norm
    c = s["case"]
    out, r = residual_rms_norm(s["y"], s["r"], s["w"], post_weight=s.get("w_post"), gate=s.get("gate"), gate_activation=c["act"],
                               scale=s["scale"], eps=EPS)
    if not c["train"]:
        return [out, r]
    leaves = [s[k] for k in ("y", "r", "w", "scale", "gate", "w_post") if k in s]
    return [out.detach(), r.detach(), *torch.autograd.grad((out, r), leaves, (s["dout"], s["dr"]))]


def _own_embedding(s):
    from operators.scaled_embedding import scaled_embedding
    out = scaled_embedding(s["ids"], s["weight"], s["scale"])
    if not s["case"]["train"]:
        return [out]
    return [out.detach(), *torch.autograd.grad(out, [s["weight"]], s["dout"])]


_PLAIN = {"recurrence": _plain_recurrence, "step": _plain_step, "norm": _plain_norm, "embedding": _plain_embedding}
_OWN = {"recurrence": _own_recurrence, "step": _own_step, "norm": _own_norm, "embedding": _own_embedding}


def run(state):
    op = state["case"]["op"]
    if own:
        _package()
        return _OWN[op](state)
    with torch.no_grad():
        return _PLAIN[op](state)


# ---------------------------------------------------------------------------
# bytes and operations of one pass
# ---------------------------------------------------------------------------
def work(case):
    e = 4 if case["type"] == "fp32" else 2
    op, train = case["op"], case.get("train", False)
    logits = case.get("gates") == "logits"
    if op == "step":
        n = case["B"] * case["C"]
        return {"bytes": 4 * n * e + 8 * n + (4 * case["C"] if logits else 0), "flops": (16 if logits else 3) * n}
    if op == "recurrence":
        B, L, C = case["B"], case["L"], case["C"]
        n = B * L * C
        small = 8 * B * C + (4 * C if logits else 0) + (B * L if case["reset"] else 0)
        if not train:
            return {"bytes": 4 * n * e + small, "flops": (16 if logits else 3) * n}
        return {"bytes": 8 * n * e + 2 * small, "flops": (48 if logits else 9) * n}
    if op == "norm":
        M, N = case["M"], case["N"]
        gate, post = case["act"] != "none", case["post"]
        flops = (9 + 6 * gate + 3 * post) * M * N
        # y, gate, r in and out, r' out; with gradients two more in and those of y, gate and r out
        streams, vectors = 4 + gate, 2 + post
        if train:
            return {"bytes": (2 * streams * M * N + 2 * vectors * N) * e, "flops": 3 * flops}
        return {"bytes": (streams * M * N + vectors * N) * e, "flops": flops}
    T, V, N = case["T"], case["V"], case["N"]
    if case["ids"] == "zipf":
        # expected distinct ids of T draws of a log-uniform rank
        edges = [0] + [int(V ** (k / 256)) for k in range(1, 257)]
        rows = sum((hi - lo) * (1 - math.exp(-T / 256 / (hi - lo))) for lo, hi in zip(edges, edges[1:]) if hi > lo)
    else:
        rows = V * (1 - math.exp(-T * (2 / 3 if case["ids"] == "pad" else 1) / V)) + (case["ids"] == "pad")
    rows = min(rows, T, V)
    n = rows * N + T * N
    if train:
        n += T * N + V * N
    return {"bytes": n * e + 8 * T, "flops": T * N * (2 if train else 1)}


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    for k, v in s.items():
        if isinstance(v, torch.Tensor) and v.is_floating_point():
            s[k] = v.detach().double()
    return {"recurrence": _exact_recurrence, "step": _exact_step, "norm": _exact_norm, "embedding": _exact_embedding}[case["op"]](s)


def _exact_decay(s):
    """log a, a, 1 - a^2 under the square root, and the open input gate."""
    u = -DECAY_SCALE * torch.nn.functional.softplus(s["decay"]) * torch.sigmoid(s["g"])
    return u, u.exp(), (-(2 * u).expm1()).sqrt(), torch.sigmoid(s["beta"])


def _exact_step(s):
    if s["case"]["gates"] == "values":
        h = s["g"] * s["state"] + s["beta"] * s["x"]
    else:
        _, a, m, i = _exact_decay(s)
        h = a * s["state"] + m * i * s["x"]
    return [h, h]


def _exact_recurrence(s):
    c = s["case"]
    L, logits = c["L"], c["gates"] == "logits"
    keep = 1.0 if "reset" not in s else (~s["reset"]).double()[:, :, None]
    if logits:
        u, a, m, i = _exact_decay(s)
        a = a * keep
        m = m * keep + (1 - keep)
        b = m * i * s["x"]
    else:
        a, b = s["g"] * keep, s["beta"] * s["x"]
    h, now = torch.empty_like(b), s["state"]
    for t in range(L):
        now = torch.addcmul(b[:, t], a[:, t], now)
        h[:, t] = now
    outs = [h, now]
    if not c["train"]:
        return outs
    d, now = s["dh"], s["dstate"]
    for t in range(L - 1, -1, -1):
        now = d[:, t].add_(now)
        now = now * a[:, t]
    dstate = now
    before = torch.roll(h, 1, 1)
    before[:, 0] = s["state"]
    if not logits:
        return outs + [d * s["beta"], d * before * keep, d * s["x"], dstate]
    da = d * (before - i * s["x"] * a / m) * keep
    du = da * a
    sg = torch.sigmoid(s["g"])
    dg = du * u * (1 - sg)
    ddecay = (du * -DECAY_SCALE * sg).sum((0, 1)) * torch.sigmoid(s["decay"])
    return outs + [d * m * i, dg, d * m * s["x"] * i * (1 - i), dstate, ddecay]


def _exact_norm(s):
    c = s["case"]
    names = [k for k in ("y", "r", "w", "scale", "gate", "w_post") if k in s]
    v = {k: s[k].requires_grad_(c["train"]) for k in names}
    u = v["y"]
    if c["post"]:
        u = u * torch.rsqrt(u.square().mean(-1, keepdim=True) + EPS) * v["w_post"]
    if c["act"] == "silu":
        u = u * torch.nn.functional.silu(v["gate"])
    elif c["act"] == "sigmoid":
        u = u * torch.sigmoid(v["gate"])
    r = v["r"] + v["scale"] * u
    out = r * torch.rsqrt(r.square().mean(-1, keepdim=True) + EPS) * v["w"]
    if not c["train"]:
        return [out, r]
    return [out.detach(), r.detach(), *torch.autograd.grad((out, r), [v[k] for k in names], (s["dout"], s["dr"]))]


def _exact_embedding(s):
    c = s["case"]
    outs = [s["weight"][s["ids"]] * s["scale"]]
    if c["train"]:
        order = torch.argsort(s["ids"], stable=True)
        total = torch.cumsum(s["dout"][order], 0)
        which, count = torch.unique_consecutive(s["ids"][order], return_counts=True)
        total = total[torch.cumsum(count, 0) - 1]
        dw = torch.zeros(c["V"], c["N"], dtype=torch.float64, device=DEV)
        dw[which] = torch.diff(total, dim=0, prepend=torch.zeros_like(total[:1])) * s["scale"]
        outs.append(dw)
    return outs
