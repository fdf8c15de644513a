"""gated_linear_recurrence against its definition in 64 bits.

Tolerances are running error bounds, evaluated in 64 bits next to the values: with U = 2^-24,
  a = e^u: u = -scale softplus sigmoid carries about 11 U (softplus, product, ex2 and rcp of the
  sigmoid), so a is off by at most (4 + 11 |u|) a U <= 16 U; b = m i x carries at most 16 U;
  h:  E_t = a_t E_{t-1} + 20 U (H_{t-1} + |b_t|) + 2 U H_t, H the recurrence of absolute values
  D:  the same going backwards;
  du = D (a h' - a^2/m i x): E_du = E_D P + D (a E_h + (40 + 24 |u|) U P), P the bracket's
  absolute value; and what multiplies du or D carries at most 20 U more.
Sums add their depth (L + B) in U.  Each output adds half a step of its type.
"""
import pytest
import torch

from operators import _lib
from operators.gated_linear_recurrence import (gated_linear_recurrence,
                                               gated_linear_recurrence_step, timeouts)

DEV = "cuda"
U = 2.0 ** -24
gpu = pytest.mark.gpu


def _within(got, ref, tol, name):
    half = torch.finfo(got.dtype).eps / 2
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 1e-37
    err = (got.double().cpu() - ref).abs()
    lim = tol + half * (ref.abs() + tol) + tiny
    bad = ~(err <= lim)
    assert not bool(bad.any()), (
        f"{name}: {int(bad.sum())} of {bad.numel()} off, worst {float((err / lim).max()):.2f} of the bound")


def _inputs(B, L, C, dtype, gate_dtype, logits, seed=0, reset=0.0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    v = {"x": r(B, L, C).to(dtype)}
    if logits:
        v["g"], v["beta"] = (2 * r(B, L, C)).to(gate_dtype), r(B, L, C).to(gate_dtype)
        a = 0.9 + 0.0999 * torch.rand(C, generator=gen)
        v["decay"] = torch.log(torch.expm1(-torch.log(a) / 8))
    else:
        v["g"] = torch.sigmoid(r(B, L, C) + 2).to(gate_dtype)
        v["beta"] = torch.sigmoid(r(B, L, C)).to(gate_dtype)
    v["h0"] = 0.5 * r(B, C)
    v["dh"], v["dhT"] = r(B, L, C).to(dtype), r(B, C)
    v["reset"] = torch.rand(B, L, generator=gen) < reset if reset else None
    return v


def _reference(v, scale, state=True):
    """{name: (value, tolerance)} in 64 bits, step by step."""
    x, g, beta = v["x"].double(), v["g"].double(), v["beta"].double()
    B, L, C = x.shape
    keep = torch.ones(B, L, 1).double() if v["reset"] is None else (~v["reset"]).double()[..., None]
    logits = "decay" in v
    if logits:
        sp = torch.nn.functional.softplus(v["decay"].double())
        s, i = torch.sigmoid(g), torch.sigmoid(beta)
        u = -scale * sp * s
        a, m = torch.exp(u) * keep, torch.sqrt(-torch.expm1(2 * u))
        m = m * keep + (1 - keep)
        b = m * i * x
    else:
        a, b = g * keep, beta * x
    h0 = v["h0"].double() if state else torch.zeros(B, C).double()
    h, H, E = [h0], [h0.abs()], [torch.zeros(B, C).double()]
    for t in range(L):
        A = a[:, t].abs()
        h.append(a[:, t] * h[-1] + b[:, t])
        H.append(A * H[-1] + b[:, t].abs())
        # at a reset the old state is not looked at
        E.append(A * E[-1] + 20 * U * ((A > 0) * H[-2] + b[:, t].abs()) + 2 * U * H[-1])
    st = lambda z: torch.stack(z, 1)  # noqa: E731
    out = {"h": (st(h[1:]) if L else x, st(E[1:]) if L else x), "hT": (h[-1], E[-1])}
    d, ad, e = v["dhT"].double(), v["dhT"].double().abs(), torch.zeros(B, C).double()
    D, AD, ED = [], [], []
    for t in range(L - 1, -1, -1):
        dt = v["dh"][:, t].double()
        d, ad = d + dt, ad + dt.abs()
        e = e + 2 * U * ad
        D.append(d), AD.append(ad), ED.append(e)
        A = a[:, t].abs()
        d, ad, e = a[:, t] * d, A * ad, A * e + 20 * U * (A > 0) * ad
    out["dh0"] = (d, e)
    if L == 0:
        return out
    D, AD, ED = (torch.stack(z[::-1], 1) for z in (D, AD, ED))
    hb, Hb, Eb = st(h[:-1]), st(H[:-1]), st(E[:-1])

    def times(f, extra=0.0):
        return D * f, ED * f.abs() + AD * extra + 20 * U * (D * f).abs()
    if not logits:
        out["dx"], out["dbeta"] = times(beta), times(x)
        out["dg"] = tuple(z * keep for z in times(hb, Eb))
        return out
    am = torch.where(m > 0, a * a / m, torch.zeros_like(m))
    P = a * Hb + am * i * x.abs()
    du = D * (a * hb - am * i * x) * keep
    Edu = (ED * P + AD * (a * Eb + (40 + 24 * u.abs()) * U * P)) * keep
    f = u * (1 - s)
    out["dg"] = (du * f, Edu * f.abs() + 20 * U * (du * f).abs())
    q = -scale * torch.sigmoid(v["decay"].double())
    out["ddecay"] = ((du * s).sum((0, 1)) * q,
                     ((Edu * s).sum((0, 1)) + (L + B + 40) * U * (du * s).abs().sum((0, 1))) * q.abs())
    out["dx"] = times(m * i)
    out["dbeta"] = times(m * x * i * (1 - i))
    return out


def _leaf(t):
    return None if t is None else t.to(DEV).requires_grad_()


def _run(v, scale, state=True):
    leaves = {k: _leaf(v[k]) for k in ("x", "g", "beta", "decay") if k in v}
    h0 = _leaf(v["h0"]) if state else None
    reset = v["reset"].to(DEV) if v["reset"] is not None else None
    h, hT = gated_linear_recurrence(*leaves.values(), decay_scale=scale, initial_state=h0,
                                    reset=reset, output_final_state=True)
    grads = torch.autograd.grad((h, hT), [*leaves.values(), *([h0] if state else [])],
                                (v["dh"].to(DEV), v["dhT"].to(DEV)))
    out = {"h": h.detach(), "hT": hT.detach()}
    out.update(zip(["d" + k for k in leaves] + (["dh0"] if state else []), grads))
    return out


def _check(v, scale=8.0, state=True):
    ref = _reference(v, scale, state)
    got = _run(v, scale, state)
    for k, t in got.items():
        if t.numel():
            _within(t, *ref[k], k)
    return got


TYPES = [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
         (torch.float16, torch.float16), (torch.bfloat16, torch.float32),
         (torch.float16, torch.float32)]


@gpu
@pytest.mark.parametrize("logits", [False, True])
@pytest.mark.parametrize("dtype,gate_dtype", TYPES)
def test_types(dtype, gate_dtype, logits):
    _check(_inputs(2, 200, 96, dtype, gate_dtype, logits))


@gpu
@pytest.mark.parametrize("logits", [False, True])
@pytest.mark.parametrize("L", [1, 2, 7, 63, 64, 65, 127, 129, 512, 1000, 3001])
def test_lengths(L, logits):
    _check(_inputs(1, L, 64, torch.bfloat16, torch.bfloat16, logits, seed=L))


@gpu
@pytest.mark.parametrize("C", [1, 2, 3, 31, 33, 66, 130, 1111])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_widths(C, dtype):
    _check(_inputs(3, 90, C, dtype, dtype, True, seed=C))


@gpu
@pytest.mark.parametrize("B,L,C", [(5, 300, 128), (1, 9000, 64), (40, 33, 256), (2, 2100, 2048)])
def test_batches_and_long_axes(B, L, C):
    _check(_inputs(B, L, C, torch.bfloat16, torch.bfloat16, True, seed=B, reset=0.01))


@gpu
@pytest.mark.parametrize("logits", [False, True])
def test_reset_starts_again(logits):
    v = _inputs(2, 400, 64, torch.float32, torch.float32, logits, reset=0.05)
    v["reset"][0, 0] = v["reset"][1, 64] = v["reset"][1, 399] = True
    got = _check(v)
    # a reset step does not see what is before it, whatever that is
    v["x"][1, 63] = 3e38
    other = _run(v, 8.0)
    assert torch.equal(other["h"][1, 64:], got["h"][1, 64:])


@gpu
def test_step_marks_its_state_as_changed():
    """A graph that saved the state in front of a step raises instead of using the state behind it."""
    x, state = torch.rand(2, 8, device=DEV), torch.rand(2, 8, device=DEV)
    w = torch.rand(2, 8, device=DEV, requires_grad=True)
    y = (w * state).sum()
    with torch.no_grad():
        gated_linear_recurrence_step(x, x, x, state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        state = torch.zeros(2, 8, device=DEV)
        assert torch.equal(gated_linear_recurrence_step(x, x, x, state), state)


@gpu
@pytest.mark.parametrize("B,L", [(1, 700), (64, 300)])
@pytest.mark.parametrize("logits", [False, True])
def test_nothing_crosses_a_reset(logits, B, L):
    """NaN and infinity on one side of a reset (few slabs: clusters; many: chains): the other side is as
    it is without them, bit for bit, forward and backward."""
    v = _inputs(B, L, 256, torch.float32, torch.float32, logits)
    v["reset"] = torch.zeros(B, L, dtype=torch.bool)
    v["reset"][:, 130] = v["reset"][:, 0] = True
    clean = _run(v, 8.0)
    w = {k: (t.clone() if t is not None else None) for k, t in v.items()}
    w["x"][:, 100:130] = float("nan")
    w["h0"][:] = float("inf")
    got = _run(w, 8.0)
    for k in ("h", "dx", "dg", "dbeta"):
        assert torch.equal(got[k][:, 130:], clean[k][:, 130:]), k
    assert torch.equal(got["h"][:, :100], clean["h"][:, :100])
    assert torch.equal(got["hT"], clean["hT"])
    w = {k: (t.clone() if t is not None else None) for k, t in v.items()}
    w["dh"][:, 140:160] = float("nan")
    w["dhT"][:] = float("inf")
    got = _run(w, 8.0)
    for k in ("h", "dx", "dg", "dbeta"):
        assert torch.equal(got[k][:, :130], clean[k][:, :130]), k
    assert bool((got["dh0"] == 0).all()) and bool((clean["dh0"] == 0).all())


@gpu
def test_reset_everywhere_and_nowhere():
    v = _inputs(2, 130, 40, torch.float32, torch.float32, True)
    v["reset"] = torch.ones(2, 130, dtype=torch.bool)
    _check(v)
    a = _run(dict(v, reset=torch.zeros(2, 130, dtype=torch.bool)), 8.0)
    b = _run(dict(v, reset=None), 8.0)
    assert all(torch.equal(a[k], b[k]) for k in a)


@gpu
def test_no_initial_state_and_zero_gates():
    _check(_inputs(2, 150, 70, torch.float32, torch.float32, True), state=False)
    v = _inputs(2, 150, 70, torch.float32, torch.float32, False)
    v["g"][:, 50] = 0.0
    _check(v, state=False)


@gpu
def test_padded_steps_keep_the_state():
    """g = 1, beta = 0 as values and g = -inf as logits: the state passes through, and where a
    thread's 8 steps begin it is A s + H of the 8 before instead of their walk.  Both are within
    E of the exact state, so they are within 2 E of each other; between the
    places where maps are put together (80, and 128 where the next tile of 64 begins) nothing
    changes, and behind them nothing changes any more."""
    for logits in (False, True):
        v = _inputs(2, 200, 64, torch.float32, torch.float32, logits)
        v["g"][:, 77:] = float("-inf") if logits else 1.0
        if not logits:
            v["beta"][:, 77:] = 0.0
        got = _run(v, 8.0)
        ref = _reference(v, 8.0)["hT"]
        _within(got["hT"], got["h"][:, 76].double().cpu(), 2 * ref[1], "hT")
        assert torch.equal(got["hT"], got["h"][:, 199])
        for a, b in ((76, 80), (80, 128), (128, 200)):
            assert bool((got["h"][:, a:b] == got["h"][:, b - 1:b]).all())
        assert bool((got["dg"][:, 77:] == 0).all()) or not logits
        assert all(bool(torch.isfinite(t).all()) for t in got.values())
        short = {k: (t[:, :77] if k in ("x", "g", "beta", "dh") else t) for k, t in v.items()}
        v["dh"][:, 77:] = 0
        a, b = _run(v, 8.0), _run(short, 8.0)
        torch.testing.assert_close(a["dx"][:, :77], b["dx"], rtol=1e-5, atol=1e-6)


@gpu
def test_saturated_gates():
    """Logits of either sign far out: decays of exactly 1 and of 0, gradients finite."""
    v = _inputs(2, 130, 64, torch.float32, torch.float32, True)
    v["g"][:, ::5] = 200.0
    v["g"][:, 1::5] = -200.0
    v["beta"][:, 2::5] = -200.0
    v["beta"][:, 3::5] = 200.0
    v["decay"][:8] = 60.0
    v["decay"][8:16] = -60.0
    got = _run(v, 8.0)
    ref = _reference(v, 8.0)
    for k, t in got.items():
        assert bool(torch.isfinite(t).all()), k
    _within(got["h"], *ref["h"], "h")


@gpu
def test_growing_gates_over_a_zero_state():
    """Values above 1 whose product leaves the fp32 range: an empty state stays empty."""
    v = _inputs(1, 2000, 64, torch.float32, torch.float32, False)
    v["g"].fill_(2.0)
    v["x"].zero_()
    v["x"][0, 1990:] = 1.0
    v["dh"].zero_()
    v["dhT"].zero_()
    got = _run(v, 1.0, state=False)
    ref = _reference(v, 1.0, state=False)
    _within(got["h"], *ref["h"], "h")
    assert bool((got["dx"] == 0).all())


@gpu
def test_nan_stays_in_its_channel():
    v = _inputs(2, 300, 64, torch.bfloat16, torch.bfloat16, True)
    v["x"][1, 100, 5] = float("nan")
    got = _run(v, 8.0)
    bad = torch.isnan(got["h"])
    assert bool(bad[1, 100:, 5].all()) and int(bad.sum()) == 200
    assert int(torch.isnan(got["dx"]).sum()) <= 300  # nothing outside [1, :, 5]
    ok = torch.ones(64, dtype=torch.bool)
    ok[5] = False
    assert bool(torch.isfinite(got["dg"].cpu()[:, :, ok]).all())


@gpu
def test_strided_views_of_one_projection():
    v = _inputs(2, 140, 72, torch.bfloat16, torch.bfloat16, True)
    want = _run(v, 8.0)
    p = torch.cat((v["x"], v["g"], v["beta"]), -1).to(DEV).requires_grad_()
    x, g, beta = p.split(72, -1)
    assert not x.is_contiguous()
    dec, h0 = v["decay"].to(DEV), v["h0"].to(DEV)
    h, hT = gated_linear_recurrence(x, g, beta, dec, decay_scale=8.0, initial_state=h0,
                                    output_final_state=True)
    assert torch.equal(h, want["h"]) and torch.equal(hT, want["hT"])
    (dp,) = torch.autograd.grad((h, hT), [p], (v["dh"].to(DEV), v["dhT"].to(DEV)))
    assert torch.equal(dp, torch.cat((want["dx"], want["dg"], want["dbeta"]), -1))
    # an odd column offset (no vector alignment), transposed time, and a batch broadcast
    wide = torch.zeros(2, 140, 75, dtype=torch.bfloat16, device=DEV)
    wide[..., 1:73] = v["x"].to(DEV)
    h = gated_linear_recurrence(wide[..., 1:73], v["g"].to(DEV), v["beta"].to(DEV), dec,
                                decay_scale=8.0, initial_state=h0)
    assert torch.equal(h, want["h"])
    xt = v["x"].to(DEV).transpose(1, 2).contiguous().transpose(1, 2)
    h = gated_linear_recurrence(xt, v["g"].to(DEV), v["beta"].to(DEV), dec, decay_scale=8.0,
                                initial_state=h0)
    assert torch.equal(h, want["h"])


@gpu
def test_broadcast_gate_gradient_sums():
    v = _inputs(3, 80, 64, torch.float32, torch.float32, False)
    v["g"] = v["g"][:1].expand(3, -1, -1)
    ref = _reference(v, 1.0)
    g = v["g"][:1].to(DEV).requires_grad_()
    h, hT = gated_linear_recurrence(v["x"].to(DEV), g.expand(3, -1, -1), v["beta"].to(DEV),
                                    initial_state=v["h0"].to(DEV), output_final_state=True)
    (dg,) = torch.autograd.grad((h, hT), [g], (v["dh"].to(DEV), v["dhT"].to(DEV)))
    _within(dg, ref["dg"][0].sum(0, keepdim=True),
            ref["dg"][1].sum(0, keepdim=True) + 4 * U * ref["dg"][0].abs().sum(0, keepdim=True), "dg")


@gpu
def test_only_one_output_used():
    v = _inputs(2, 100, 64, torch.float32, torch.float32, True)
    for name, zero in (("h", "dhT"), ("hT", "dh")):
        w = dict(v, **{zero: torch.zeros_like(v[zero])})
        ref = _reference(w, 8.0)
        x = _leaf(v["x"])
        h, hT = gated_linear_recurrence(x, v["g"].to(DEV), v["beta"].to(DEV), v["decay"].to(DEV),
                                        decay_scale=8.0, initial_state=v["h0"].to(DEV),
                                        output_final_state=True)
        out, cot = (h, v["dh"]) if name == "h" else (hT, v["dhT"])
        (dx,) = torch.autograd.grad(out, [x], cot.to(DEV))
        _within(dx, *ref["dx"], "dx")


@gpu
def test_gradients_against_differences():
    """Central differences of the kernel's own forward in fp32.  With a step of 2^-6 the third
    derivative leaves at most 2^-12/6 times it and rounding about 2^-24 * 32 per output: 2e-3 of
    the gradient's scale covers both."""
    v = _inputs(1, 40, 8, torch.float32, torch.float32, True, seed=3)
    got = _run(v, 8.0)
    w, wT = v["dh"].double(), v["dhT"].double()

    def loss(k, t):
        u = {n: (t if n == k else v[n]).to(DEV) for n in ("x", "g", "beta", "decay", "h0")}
        h, hT = gated_linear_recurrence(u["x"], u["g"], u["beta"], u["decay"], decay_scale=8.0,
                                        initial_state=u["h0"], output_final_state=True)
        return float((h.double().cpu() * w).sum() + (hT.double().cpu() * wT).sum())
    gen = torch.Generator().manual_seed(1)
    for k in ("x", "g", "beta", "decay", "h0"):
        grad = got["d" + k].double().cpu()
        dirn = torch.randn(v[k].shape, generator=gen)
        dirn /= dirn.norm()
        e = 2.0 ** -6
        num = (loss(k, v[k] + e * dirn) - loss(k, v[k] - e * dirn)) / (2 * e)
        assert abs(num - float((grad * dirn.double()).sum())) <= 2e-3 * float(grad.norm()), k


@gpu
def test_step_equals_the_sequence():
    for dtype, gd, logits in ((torch.float32, torch.float32, True), (torch.bfloat16, torch.float32, False),
                              (torch.bfloat16, torch.bfloat16, True)):
        v = {k: (t.to(DEV) if t is not None else None)
             for k, t in _inputs(5, 20, 130, dtype, gd, logits).items()}
        h, hT = gated_linear_recurrence(v["x"], v["g"], v["beta"], v.get("decay"), decay_scale=8.0,
                                        initial_state=v["h0"], output_final_state=True)
        state = v["h0"].clone()
        for t in range(20):
            o = gated_linear_recurrence_step(v["x"][:, t], v["g"][:, t], v["beta"][:, t], state,
                                             v.get("decay"), decay_scale=8.0)
            torch.testing.assert_close(o, h[:, t], rtol=torch.finfo(dtype).eps, atol=1e-6)
        torch.testing.assert_close(state, hT, rtol=1e-6, atol=1e-6)


@gpu
@pytest.mark.parametrize("B,C", [(1, 64), (1, 1), (3, 65), (512, 2048), (70000, 8)])
def test_step_sizes(B, C):
    v = _inputs(B, 1, C, torch.bfloat16, torch.bfloat16, True)
    ref = _reference(v, 8.0)
    state = v["h0"].to(DEV)
    o = gated_linear_recurrence_step(v["x"][:, 0].to(DEV), v["g"][:, 0].to(DEV),
                                     v["beta"][:, 0].to(DEV), state, v["decay"].to(DEV),
                                     decay_scale=8.0)
    _within(o, ref["h"][0][:, 0], ref["h"][1][:, 0], "h")
    _within(state, *ref["hT"], "state")


@gpu
def test_empty():
    for shape in ((0, 5, 8), (2, 0, 8), (2, 5, 0)):
        x = torch.randn(*shape, device=DEV, requires_grad=True)
        g = torch.rand(*shape, device=DEV)
        dec = torch.randn(shape[2], device=DEV, requires_grad=True)
        h0 = torch.randn(shape[0], shape[2], device=DEV, requires_grad=True)
        h, hT = gated_linear_recurrence(x, g, g, dec, initial_state=h0, output_final_state=True)
        assert h.shape == shape and torch.equal(hT, h0)
        dx, dd, dh0 = torch.autograd.grad((h.sum(), hT.sum()), [x, dec, h0])
        assert dx.shape == shape and bool((dd == 0).all()) and bool((dh0 == 1).all())
    z = torch.zeros(0, 4, device=DEV)
    assert gated_linear_recurrence_step(z, z, z, z.clone()).shape == (0, 4)
    h, hT = gated_linear_recurrence(*[torch.zeros(2, 0, 8, device=DEV)] * 3, output_final_state=True)
    assert bool((hT == 0).all())


@gpu
def test_repeatable_and_on_another_stream():
    v = _inputs(4, 700, 256, torch.bfloat16, torch.bfloat16, True, reset=0.01)
    a = _run(v, 8.0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b = _run(v, 8.0)
    s.synchronize()
    assert all(torch.equal(a[k], b[k]) for k in a)


@gpu
def test_captured_forward_and_backward_replay():
    v = _inputs(2, 300, 128, torch.bfloat16, torch.bfloat16, True)
    want = _run(v, 8.0)
    ins = [v[k].to(DEV) for k in ("x", "g", "beta", "decay")]
    h0, dh, dhT = v["h0"].to(DEV), v["dh"].to(DEV), v["dhT"].to(DEV)

    def work():
        leaves = [t.detach().requires_grad_() for t in (*ins, h0)]
        h, hT = gated_linear_recurrence(*leaves[:4], decay_scale=8.0, initial_state=leaves[4],
                                        output_final_state=True)
        return (h.detach(), hT.detach(), *torch.autograd.grad((h, hT), leaves, (dh, dhT)))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        work()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    names = ["h", "hT", "dx", "dg", "dbeta", "ddecay", "dh0"]
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[k]) for k, o in zip(names, out))
    v2 = _inputs(2, 300, 128, torch.bfloat16, torch.bfloat16, True, seed=9)
    for t, k in zip((*ins, h0, dh, dhT), ("x", "g", "beta", "decay", "h0", "dh", "dhT")):
        t.copy_(v2[k])
    graph.replay()
    want = _run(v2, 8.0)
    assert all(torch.equal(o, want[k]) for k, o in zip(names, out))


@gpu
def test_offsets_over_32_bits():
    """2.2e9 elements: the last steps of the whole sequence, and of its tail from the state in front
    of it.  The tiles lie otherwise, so both carry the bound of their own way: E of h is at most
    20 U (H + 1) a step over the memory of the gates (values of at most 0.95: 20 steps), so they are
    within 2 * 20 * 20 U * 4 = 1e-4 of each other in fp32; h and the gradients add a step of bf16."""
    L, C, cut = (1 << 20) + 77, 2050, (1 << 20) - 200
    gen = torch.Generator(device=DEV).manual_seed(0)
    x = torch.randn(1, L, C, device=DEV, generator=gen, dtype=torch.bfloat16)
    g = torch.rand(1, L, C, device=DEV, generator=gen, dtype=torch.bfloat16).mul_(0.95)
    assert x.numel() > 1 << 31
    leaf = x.requires_grad_()
    h, hT = gated_linear_recurrence(leaf, g, g, output_final_state=True)
    with torch.no_grad():
        _, front = gated_linear_recurrence(leaf[:, :cut], g[:, :cut], g[:, :cut], output_final_state=True)
    tail = leaf.detach()[:, cut:].clone().requires_grad_()
    gt = g[:, cut:]
    ht, hTt = gated_linear_recurrence(tail, gt, gt, initial_state=front, output_final_state=True)
    torch.testing.assert_close(hT, hTt, rtol=0, atol=1e-4)
    torch.testing.assert_close(h[:, cut:], ht, rtol=2 ** -7, atol=1e-4)
    ones = torch.ones_like(hT)
    (dx,) = torch.autograd.grad((h, hT), [leaf], (x.detach(), ones))
    (dt,) = torch.autograd.grad((ht, hTt), [tail], (tail.detach(), ones))
    torch.testing.assert_close(dx[:, cut:], dt, rtol=2 ** -7, atol=1e-4)
    assert bool(torch.isfinite(dx[:, ::4099]).all())


@gpu
def test_no_wait_timed_out():
    _check(_inputs(1, 5000, 64, torch.bfloat16, torch.bfloat16, True, reset=0.01))
    assert timeouts() == 0


@gpu
def test_double_backward_is_refused():
    x = torch.randn(1, 8, 32, device=DEV, requires_grad=True)
    g = torch.rand(1, 8, 32, device=DEV)
    h = gated_linear_recurrence(x, g, g)
    (dx,) = torch.autograd.grad(h.sum(), [x], create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()


@gpu
@pytest.mark.parametrize("B,L", [(1, 700), (64, 300)])
@pytest.mark.parametrize("logits,bad", [(False, "nan"), (False, "inf"), (False, "growing"), (True, "nan")])
def test_bad_gates_do_not_cross_a_reset(logits, bad, B, L):
    """Gates that are NaN or infinite, or whose product leaves the fp32 range, among the steps that a
    warp has with the reset: the other document is as it is without them."""
    v = _inputs(B, L, 256, torch.float32, torch.float32, logits)
    v["reset"] = torch.zeros(B, L, dtype=torch.bool)
    v["reset"][:, 130] = True
    value = {"nan": float("nan"), "inf": float("inf"), "growing": 1e25}[bad]

    def with_gates(u, steps):
        u = dict(u, g=u["g"].clone())
        u["g"][:, steps] = value
        return u
    front = dict(v)
    if bad == "growing":
        front["x"], front["h0"] = v["x"].clone(), torch.zeros_like(v["h0"])
        front["x"][:, :130] = 0
        front["x"][:, 127] = 1e-30
    clean = _run(front, 8.0)
    for steps in ([128], [129], [128, 129], list(range(100, 130))):
        got = _run(with_gates(front, steps), 8.0)
        for k in ("h", "dx", "dg", "dbeta"):
            assert torch.equal(got[k][:, 130:], clean[k][:, 130:]), (k, steps)
        assert torch.equal(got["h"][:, :steps[0]], clean["h"][:, :steps[0]]), steps
        assert torch.equal(got["hT"], clean["hT"]), steps
    behind = dict(v)
    if bad == "growing":
        behind["dh"], behind["dhT"] = v["dh"].clone(), torch.zeros_like(v["dhT"])
        behind["dh"][:, 130:] = 0
        behind["dh"][:, 140] = 1e-30
    clean = _run(behind, 8.0)
    for steps in ([131], [133], [131, 132, 135], list(range(131, 160))):
        got = _run(with_gates(behind, steps), 8.0)
        for k in ("h", "dx", "dg", "dbeta"):
            assert torch.equal(got[k][:, :130], clean[k][:, :130]), (k, steps)
        assert torch.equal(got["dh0"], clean["dh0"]), steps


@gpu
@pytest.mark.parametrize("B", [1, 64])
@pytest.mark.parametrize("logits", [False, True])
def test_the_gate_of_a_reset_step_is_not_used(logits, B):
    """a_t is 0 there whatever g_t is, NaN and infinity included, and g_t's gradient is 0."""
    v = _inputs(B, 300, 256, torch.float32, torch.float32, logits)
    v["reset"] = torch.zeros(B, 300, dtype=torch.bool)
    v["reset"][:, 0] = v["reset"][:, 130] = v["reset"][:, 131] = True
    clean = _run(v, 8.0)
    for value in (float("nan"), float("inf"), float("-inf")):
        w = dict(v, g=v["g"].clone())
        w["g"][:, 0] = w["g"][:, 130] = w["g"][:, 131] = value
        got = _run(w, 8.0)
        assert bool((got["dg"][v["reset"]] == 0).all()), value
        for k in got:
            assert torch.equal(got[k], clean[k]), (k, value)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_closed_input_gates(dtype):
    """Input gates far closed, over an empty state, where h is b = m i x alone.  beta log2(e) is rounded
    twice, which is 2 |beta| U of its exponential, and the rest of b carries 16 U; forward and step are
    each within that of the formula.  What is below the smallest normal number may be 0, and -inf is 0."""
    beta = torch.tensor([-30., -41.5, -41.7, -44.5, -50., -64., -80., -87.2, -200., float("-inf")])
    B = len(beta)
    v = _inputs(B, 40, 64, dtype, dtype, True)
    v["beta"] = beta[:, None, None].expand(B, 40, 64).to(dtype).contiguous()
    v["h0"].zero_()
    i = torch.sigmoid(v["beta"].double())
    size = torch.where(torch.isinf(v["beta"]), torch.zeros(()), v["beta"].float()).abs().double()
    on = {k: t.to(DEV) for k, t in v.items() if t is not None}
    want = i * v["x"].double()  # m is 1 where every step starts again
    got = gated_linear_recurrence(on["x"], on["g"], on["beta"], on["decay"], decay_scale=8.0,
                                  reset=torch.ones(B, 40, dtype=torch.bool, device=DEV))
    _within(got, want, (2 * size + 16) * U * want.abs(), "h, every step a reset")
    assert bool((got[-1] == 0).all())
    u = -8 * torch.nn.functional.softplus(v["decay"].double()) * torch.sigmoid(v["g"].double())
    want = (torch.sqrt(-torch.expm1(2 * u)) * want)[:, 0]
    tol = (2 * size[:, 0] + 16) * U * want.abs()
    got = gated_linear_recurrence(on["x"][:, :1], on["g"][:, :1], on["beta"][:, :1], on["decay"],
                                  decay_scale=8.0)[:, 0]
    _within(got, want, tol, "h, one step")
    state = torch.zeros(B, 64, device=DEV)
    step = gated_linear_recurrence_step(on["x"][:, 0], on["g"][:, 0], on["beta"][:, 0], state, on["decay"],
                                        decay_scale=8.0)
    _within(step, want, tol, "step")
    assert bool((got[-1] == 0).all()) and bool((step[-1] == 0).all())
    # a NaN is no closed gate
    on["beta"][:, 7] = float("nan")
    got = gated_linear_recurrence(on["x"], on["g"], on["beta"], on["decay"], decay_scale=8.0)
    assert bool(torch.isnan(got[:, 7:]).all()) and bool(torch.isfinite(got[:, :7]).all())


@gpu
def test_rates_beyond_the_fp32_range():
    """decay or decay_scale times its softplus infinite in fp32: an open gate forgets all (a = 0, m = 1), a
    closed one nothing (a = 1, m = 0), and neither has a slope."""
    v = _inputs(2, 150, 64, torch.float32, torch.float32, True)
    v["g"][:, ::3] = float("-inf")
    i = torch.sigmoid(v["beta"].double())
    want, now = [], v["h0"].double()
    for t in range(150):
        now = now if t % 3 == 0 else i[:, t] * v["x"][:, t].double()
        want.append(now)
    want = torch.stack(want, 1)
    for scale, decay in ((8.0, float("inf")), (3e38, 5.0)):
        v["decay"].fill_(decay)
        got = _run(v, scale)
        _within(got["h"], want, 20 * U * want.abs(), "h")
        assert all(bool(torch.isfinite(t).all()) for t in got.values())
        assert bool((got["dg"] == 0).all()) and bool((got["ddecay"] == 0).all())
        state = v["h0"].to(DEV)
        for t in range(2):
            o = gated_linear_recurrence_step(*(v[k][:, t].to(DEV) for k in ("x", "g", "beta")), state,
                                             v["decay"].to(DEV), decay_scale=scale)
            _within(o, want[:, t], 20 * U * want[:, t].abs(), "step")


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gates_near_1(dtype):
    """a = e^{-y}, read as a single step's state from 1 without input, as the step's, and as the gradient
    of the state in front: a long memory gathers its errors, so it has to be little more than rounded.
    y = rate sigmoid(g) carries at most 20 U: 6 of softplus, 12 of the sigmoid with |g| <= 4, products.
    The polynomial of 1 - a^2 adds 1.7 U of its value 2 y at most, half of which reaches a, what it is
    subtracted from half a U of as much, and the exponential's own error (3 U) is left times y.
    With the rounding of a itself: half a U + 26 y U."""
    B, C = 64, 2048
    v = _inputs(B, 1, C, dtype, dtype, True)
    v["g"] = v["g"].clamp(-4, 4)
    v["x"].zero_(), v["dh"].zero_(), v["h0"].fill_(1), v["dhT"].fill_(1)
    v["decay"] = torch.log(torch.expm1(torch.logspace(-5, -0.7, C)))
    y = torch.nn.functional.softplus(v["decay"].double()) * torch.sigmoid(v["g"][:, 0].double())
    got = _run(v, 1.0)
    state = v["h0"].to(DEV)
    gated_linear_recurrence_step(*(v[k][:, 0].to(DEV) for k in ("x", "g", "beta")), state,
                                 v["decay"].to(DEV))
    for name, a in (("hT", got["hT"]), ("dh0", got["dh0"]), ("step", state)):
        off = (a.double().cpu() - torch.exp(-y)).abs() / ((0.5 + 26 * y) * U)
        assert float(off.max()) <= 1, (name, float(off.max()))


# ---------------------------------------------------------------------------
# refusals, on the CPU: nothing reaches the library
# ---------------------------------------------------------------------------
@pytest.fixture()
def host(monkeypatch):
    def call(name, *a):
        raise AssertionError(f"{name} was reached")
    monkeypatch.setattr(_lib, "call", call)
    monkeypatch.setattr(_lib, "require_cuda", lambda t, op: None)


def _z(*s, dtype=torch.float32):
    return torch.zeros(*s, dtype=dtype)


@pytest.mark.parametrize("err,args,kw", [
    (ValueError, (_z(2, 3), _z(2, 3), _z(2, 3)), {}),
    (ValueError, (_z(2, 3, 4), _z(2, 3, 5), _z(2, 3, 4)), {}),
    (ValueError, (_z(2, 3, 4), _z(2, 3, 4), _z(2, 3)), {}),
    (TypeError, (_z(2, 3, 4), _z(2, 3, 4), _z(2, 3, 4, dtype=torch.bfloat16)), {}),
    (TypeError, (_z(2, 3, 4), *[_z(2, 3, 4, dtype=torch.bfloat16)] * 2), {}),
    (TypeError, ([_z(2, 3, 4, dtype=torch.float64)] * 3), {}),
    (ValueError, ([_z(2, 3, 4)] * 3), {"decay": _z(5)}),
    (ValueError, ([_z(2, 3, 4)] * 3), {"initial_state": _z(2, 3)}),
    (ValueError, ([_z(2, 3, 4)] * 3), {"reset": _z(2, 3)}),
    (ValueError, ([_z(2, 3, 4)] * 3), {"reset": _z(3, 2, dtype=torch.bool)}),
])
def test_refusals(host, err, args, kw):
    with pytest.raises(err, match="gated_linear_recurrence"):
        gated_linear_recurrence(*args, **kw)


def test_step_refusals(host):
    x = _z(2, 4)
    for state in (_z(2, 5), _z(2, 4, dtype=torch.bfloat16), _z(4, 2).t()):
        with pytest.raises(ValueError, match="state must be"):
            gated_linear_recurrence_step(x, x, x, state)
    with pytest.raises(ValueError, match=r"\[B, C\]"):
        gated_linear_recurrence_step(_z(2, 1, 4), x, x, x)
    with pytest.raises(RuntimeError, match="not differentiable"):
        gated_linear_recurrence_step(x.clone().requires_grad_(), x, x, _z(2, 4))


@pytest.mark.parametrize("scale", [-1.0, float("nan"), float("inf")])
def test_decay_scale_refusals(host, scale):
    with pytest.raises(ValueError, match="decay_scale"):
        gated_linear_recurrence(*[_z(2, 3, 4)] * 3, _z(4), decay_scale=scale)
    with pytest.raises(ValueError, match="decay_scale"):
        gated_linear_recurrence_step(*[_z(2, 4)] * 4, _z(4), decay_scale=scale)


def test_tangents_are_refused(host):
    """A dual tensor would lose its tangent in a launch."""
    fw = torch.autograd.forward_ad
    with fw.dual_level():
        for k in range(5):
            a = [_z(2, 3, 4), _z(2, 3, 4), _z(2, 3, 4), _z(4), _z(2, 4)]
            a[k] = fw.make_dual(a[k], torch.ones_like(a[k]))
            with pytest.raises(RuntimeError, match="gated_linear_recurrence: has no forward-mode"):
                gated_linear_recurrence(*a[:4], initial_state=a[4])
            a = [_z(2, 4), _z(2, 4), _z(2, 4), _z(2, 4), _z(4)]
            a[k] = fw.make_dual(a[k], torch.ones_like(a[k]))
            with pytest.raises(RuntimeError, match="_step: has no forward-mode"):
                gated_linear_recurrence_step(*a)
        _lib.refuse_tangents("op", _z(2, 4), None)  # under a level, without a tangent


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        gated_linear_recurrence(*[_z(1, 2, 4)] * 3)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        gated_linear_recurrence_step(*[_z(2, 4)] * 4)


def test_c_entry_checks():
    f32, bf16 = 0, 2
    P = 0x1000
    nul = [None] * 9
    with pytest.raises(ValueError, match="negative size"):
        _lib.call("fo_glr_fwd", *nul, -1, 4, 4, None, 1.0, f32, f32, None)
    with pytest.raises(ValueError, match="over the grid's limit"):
        _lib.call("fo_glr_fwd", *nul, 1 << 31, 4, 4, None, 1.0, f32, f32, None)
    with pytest.raises(ValueError, match="null pointer"):
        _lib.call("fo_glr_fwd", *nul, 1, 4, 4, None, 1.0, f32, f32, None)
    st = _lib.i64_array([0] * 6)
    with pytest.raises(RuntimeError, match="gates of dtype code 2"):
        _lib.call("fo_glr_fwd", P, P, P, None, None, None, P, None, None, 1, 4, 4, st, 1.0, f32, bf16,
                  None)
    with pytest.raises(RuntimeError, match="unsupported dtype code 5"):
        _lib.call("fo_glr_fwd", P, P, P, None, None, None, P, None, None, 1, 4, 4, st, 1.0, 5, 5, None)
    with pytest.raises(ValueError, match="ddecay without decay"):
        _lib.call("fo_glr_bwd", P, P, P, None, *[P] * 9, 1, 4, 4, st, 1.0, f32, f32, P, 1 << 30, None)
    with pytest.raises(RuntimeError, match="workspace of"):
        _lib.call("fo_glr_bwd", *[P] * 13, 1, 4, 4, st, 1.0, f32, f32, None, 0, None)
    _lib.call("fo_glr_fwd", *nul, 0, 4, 4, None, 1.0, f32, f32, None)
    _lib.call("fo_glr_step", *[None] * 6, 4, 0, None, 1.0, f32, f32, None)
