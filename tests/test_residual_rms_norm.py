"""residual_rms_norm against its definition in 64 bits.

Tolerances: with U = 2^-24, a sum over N terms in the kernels' order carries at most
(N/256 + 10) U of the sum of the terms' magnitudes, an exponential at most (|z| + 6) U, a root,
quotient or product one or two U.  K = N/128 + 60 + 2 max|z| covers the factors of any one
quantity, and a quantity's bound is K U times the same formula over magnitudes (|r| + |s u| for
r', and so on: the difference matters where terms cancel).  The second norm divides by |r'|,
which magnifies by cond = max over rows of ||(|r| + |s u|)|| / ||r'||.  Gradients go through at most
four such quantities: 4 K U cond.  Sums over rows add M U.  Each output adds half a step of its type.
"""
import pytest
import torch

from operators import _lib
from operators.residual_rms_norm import _rows, residual_rms_norm
from operators.rms_norm import rms_norm

DEV = "cuda"
U = 2.0 ** -24
EPS = 1e-6
gpu = pytest.mark.gpu


def _within(got, ref, tol, name):
    half = torch.finfo(got.dtype).eps / 2
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 1e-37
    err = (got.double().cpu() - ref).abs()
    lim = tol + half * (ref.abs() + tol) + tiny
    bad = ~(err <= lim)
    assert not bool(bad.any()), (
        f"{name}: {int(bad.sum())} of {bad.numel()} off, worst {float((err / lim).max()):.2f} of the bound")


def _inputs(M, N, dtype, w_dtype=None, act="silu", post=True, scale="vec", seed=0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    wd = w_dtype or dtype
    v = {"y": r(M, N).to(dtype), "residual": (2 * r(M, N)).to(dtype), "weight": (1 + 0.2 * r(N)).to(wd)}
    if post:
        v["post_weight"] = (1 + 0.2 * r(N)).to(wd)
    if act != "none":
        v["gate"] = (1.5 * r(M, N)).to(dtype)
    v["scale"] = (0.5 + 0.2 * r(N)).to(wd) if scale == "vec" else scale
    cot = r(M, N).to(dtype), r(M, N).to(dtype)
    return v, cot


def _reference(v, act, cot):
    """{name: (value, tolerance)}."""
    f = {k: (t.double() if isinstance(t, torch.Tensor) else float(t)) for k, t in v.items()}
    y, r, w, s = f["y"], f["residual"], f["weight"], f["scale"]
    M, N = y.shape
    post = "post_weight" in f
    inv1 = 1 / torch.sqrt(y.square().mean(-1, keepdim=True) + EPS) if post else torch.ones(M, 1).double()
    wp = f["post_weight"] if post else torch.ones(N).double()
    z = f.get("gate")
    a, da = torch.ones_like(y), torch.zeros_like(y)
    if z is not None:
        sg = torch.sigmoid(z)
        a, da = (z * sg, sg * (1 + z * (1 - sg))) if act == "silu" else (sg, sg * (1 - sg))
    n = y * inv1
    p = n * wp
    u = a * p
    r2 = r + s * u
    r2a = r.abs() + (s * u).abs()
    inv2 = 1 / torch.sqrt(r2.square().mean(-1, keepdim=True) + EPS)
    K = N / 128 + 60 + (2 * float(z.abs().max()) if z is not None and z.numel() else 0)
    cond = float((r2a.square().mean(-1).sqrt() * inv2[:, 0]).max()) if M else 1.0
    k1, k2 = K * U, 4 * K * U * max(cond, 1.0)
    out = {"out": (r2 * inv2 * w, k2 * (r2a * inv2 * w).abs()), "res": (r2, k1 * r2a)}
    do, dr = (c.double() if c is not None else torch.zeros_like(y) for c in cot)
    e = do * w
    c2, c2a = ((x * inv2 ** 3).mean(-1, keepdim=True) for x in (e * r2, (e.abs() * r2a)))
    D = dr + inv2 * e - r2 * c2
    Da = dr.abs() + inv2 * e.abs() + r2a * c2a
    out["residual"] = D, k2 * Da
    if z is not None:
        # act'(z) of silu is a difference: its terms' magnitudes
        daa = sg * (1 + z.abs() * (1 - sg)) if act == "silu" else da
        out["gate"] = s * D * p * da, k2 * (s * Da * p * daa).abs()
    dp, dpa = s * D * a, (s * Da * a).abs()
    k, ka = dp * wp, dpa * wp.abs()
    if post:
        out["y"] = (inv1 * k - y * inv1 ** 3 * (k * y).mean(-1, keepdim=True),
                    k2 * (inv1 * ka + y.abs() * inv1 ** 3 * (ka * y.abs()).mean(-1, keepdim=True)))
        out["post_weight"] = ((dp * n).sum(0), (k2 + M * U) * (dpa * n.abs()).sum(0))
    else:
        out["y"] = k, k2 * ka
    out["weight"] = (do * r2 * inv2).sum(0), (k2 + M * U) * (do.abs() * r2a * inv2).sum(0)
    if isinstance(v["scale"], torch.Tensor):
        out["scale"] = (D * u).sum(0), (k2 + M * U) * (Da * u.abs()).sum(0)
    return out


def _run(v, act, cot, **kw):
    leaves = {k: t.to(DEV).requires_grad_() for k, t in v.items() if isinstance(t, torch.Tensor)}
    args = {**v, **leaves, **kw}
    out, res = residual_rms_norm(args.pop("y"), args.pop("residual"), args.pop("weight"),
                                 gate_activation=act, eps=EPS, **args)
    outs, cots = zip(*[(o, c.to(DEV)) for o, c in zip((out, res), cot) if c is not None])
    grads = torch.autograd.grad(outs, list(leaves.values()), cots)
    return {"out": out.detach(), "res": res.detach(), **dict(zip(leaves, grads))}


def _check(v, act, cot):
    got, ref = _run(v, act, cot), _reference(v, act, cot)
    for k, t in got.items():
        _within(t, *ref[k], k)
    return got


@gpu
@pytest.mark.parametrize("dtype,w_dtype", [(torch.float32, None), (torch.bfloat16, None),
                                           (torch.float16, None), (torch.bfloat16, torch.float32),
                                           (torch.float16, torch.float32)])
@pytest.mark.parametrize("act,post", [("silu", True), ("sigmoid", False), ("none", True), ("none", False)])
def test_types_and_parts(dtype, w_dtype, act, post):
    v, cot = _inputs(37, 512, dtype, w_dtype, act, post)
    _check(v, act, cot)


@gpu
@pytest.mark.parametrize("N", [1, 2, 7, 8, 33, 64, 100, 257, 1001, 1024, 2048, 2056, 4096, 5000,
                               8192, 8200, 16384, 20000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_widths(N, dtype):
    _check(*_with(_inputs(9, N, dtype, seed=N), "silu"))


def _with(vc, act):
    return vc[0], act, vc[1]


@gpu
@pytest.mark.parametrize("M", [1, 2, 16, 147, 149, 300, 1500, 20011])
def test_heights(M):
    _check(*_with(_inputs(M, 128, torch.bfloat16, seed=M), "silu"))
    _check(*_with(_inputs(M, 96, torch.float32, act="none", post=False, seed=M), "none"))


@gpu
def test_many_rows_of_a_wide_block():
    _check(*_with(_inputs(1200, 8192, torch.bfloat16), "silu"))
    _check(*_with(_inputs(1200, 4096, torch.float32, act="sigmoid"), "sigmoid"))


@gpu
def test_scale_as_a_number():
    for s in (1.0, -0.25, 0.0, 3):
        v, cot = _inputs(20, 320, torch.float32, scale=s)
        got = _check(v, "silu", cot)
        if s == 0.0:
            assert torch.equal(got["res"].cpu(), v["residual"]) and bool((got["y"] == 0).all())


@gpu
def test_one_gradient_only():
    v, (do, dr) = _inputs(33, 640, torch.float32)
    _check(v, "silu", (do, None))
    _check(v, "silu", (None, dr))


@gpu
def test_rows_of_zeros_and_large_values():
    v, cot = _inputs(8, 256, torch.float32)
    v["y"][2] = 0
    v["residual"][3] = 0
    v["y"][4] = 0
    v["residual"][4] = 0
    v["y"][5] *= 1e15
    v["residual"][6] *= 1e15
    got, ref = _run(v, "silu", cot), _reference(v, "silu", cot)
    for k, t in got.items():
        assert bool(torch.isfinite(t).all()), k
    for k in ("out", "res"):
        _within(got[k], *ref[k], k)


@gpu
def test_nan_and_inf_stay_in_their_row():
    v, cot = _inputs(6, 512, torch.bfloat16)
    want = _run(v, "silu", cot)
    v["y"][2, 7] = float("nan")
    v["residual"][4, 9] = float("inf")
    got = _run(v, "silu", cot)
    keep = torch.tensor([0, 1, 3, 5])
    for k in ("out", "res", "y", "residual", "gate"):
        assert torch.equal(got[k].cpu()[keep], want[k].cpu()[keep])
    assert bool(torch.isnan(got["out"][2]).all())


@gpu
def test_strided_rows_and_leading_dimensions():
    v, cot = _inputs(24, 320, torch.bfloat16)
    want = _run(v, "silu", cot)
    wide = torch.cat((v["y"], v["gate"], v["residual"]), -1).to(DEV).view(2, 3, 4, 960).requires_grad_()
    y, gate, r = wide.split(320, -1)
    sh = (2, 3, 4, 320)
    out, res = residual_rms_norm(y, r, v["weight"].to(DEV), post_weight=v["post_weight"].to(DEV),
                                 gate=gate, scale=v["scale"].to(DEV), eps=EPS)
    assert out.shape == sh and torch.equal(out.view(24, 320), want["out"])
    (dw,) = torch.autograd.grad((out, res), [wide], tuple(c.to(DEV).view(sh) for c in cot))
    assert torch.equal(dw.view(24, 960), torch.cat((want["y"], want["gate"], want["residual"]), -1))
    # one element off any vector alignment
    pad = torch.zeros(24, 322, dtype=torch.bfloat16, device=DEV)
    pad[:, 1:321] = v["y"].to(DEV)
    out2, _ = residual_rms_norm(pad[:, 1:321], v["residual"].to(DEV), v["weight"].to(DEV),
                                post_weight=v["post_weight"].to(DEV), gate=v["gate"].to(DEV),
                                scale=v["scale"].to(DEV), eps=EPS)
    # another order of the sums: one rounding step at most
    torch.testing.assert_close(out2, want["out"], rtol=2 ** -7, atol=1e-6)


@gpu
def test_gate_shared_by_rows():
    v, cot = _inputs(30, 256, torch.float32)
    v["gate"] = v["gate"].view(3, 10, 256)[:, :1].expand(3, 10, 256).reshape(30, 256)
    ref = _reference(v, "silu", cot)
    gate = v["gate"].view(3, 10, 256)[:, :1].to(DEV).requires_grad_()
    sh = (3, 10, 256)
    out, res = residual_rms_norm(v["y"].to(DEV).view(sh), v["residual"].to(DEV).view(sh),
                                 v["weight"].to(DEV), post_weight=v["post_weight"].to(DEV),
                                 gate=gate.expand(sh), scale=v["scale"].to(DEV), eps=EPS)
    (dg,) = torch.autograd.grad((out, res), [gate], tuple(c.to(DEV).view(sh) for c in cot))
    val, tol = (t.view(sh).sum(1, keepdim=True) for t in ref["gate"])
    _within(dg, val, tol + 10 * U * ref["gate"][0].view(sh).abs().sum(1, keepdim=True), "gate")


@gpu
def test_without_parts_it_is_add_then_rms_norm():
    v, _ = _inputs(64, 1024, torch.float32, act="none", post=False)
    y, r, w = (v[k].to(DEV) for k in ("y", "residual", "weight"))
    out, res = residual_rms_norm(y, r, w, eps=EPS)
    assert torch.equal(res, y + r)
    torch.testing.assert_close(out, rms_norm(y + r, (1024,), w, EPS), rtol=1e-6, atol=1e-6)


@gpu
def test_gradients_against_differences():
    """Central differences of the kernel's own fp32 forward along a unit direction, step 2^-6: the
    third derivative leaves 2^-12/6 of its size, rounding 2^-24 * 2^6 of the outputs; 2e-3 of the
    gradient's norm covers both."""
    v, cot = _inputs(4, 64, torch.float32, seed=5)
    got = _run(v, "silu", cot)
    gen = torch.Generator().manual_seed(2)

    def loss(k, t):
        a = {n: (t if n == k else x).to(DEV) for n, x in v.items()}
        o = residual_rms_norm(a.pop("y"), a.pop("residual"), a.pop("weight"), eps=EPS, **a)
        return sum(float((x.double().cpu() * c.double()).sum()) for x, c in zip(o, cot))
    for k in v:
        dirn = torch.randn(v[k].shape, generator=gen)
        dirn /= dirn.norm()
        e = 2.0 ** -6
        num = (loss(k, v[k] + e * dirn) - loss(k, v[k] - e * dirn)) / (2 * e)
        g = got[k].double().cpu()
        assert abs(num - float((g * dirn.double()).sum())) <= 2e-3 * float(g.norm()), k


@gpu
def test_empty_and_repeatable():
    w = torch.ones(64, device=DEV, requires_grad=True)
    y = torch.empty(0, 3, 64, device=DEV, requires_grad=True)
    out, res = residual_rms_norm(y, y, w, post_weight=w, scale=w)
    assert out.shape == y.shape
    dw, dy = torch.autograd.grad(out.sum() + res.sum(), [w, y])
    assert bool((dw == 0).all()) and dy.shape == y.shape
    v, cot = _inputs(700, 2048, torch.bfloat16)
    a, b = _run(v, "silu", cot), _run(v, "silu", cot)
    assert all(torch.equal(a[k], b[k]) for k in a)


@gpu
def test_offsets_over_32_bits():
    """2.2e9 elements: rows do not depend on one another, so the last ones equal those of a call of
    their own, bit for bit."""
    M, N = 262144 + 301, 8192
    gen = torch.Generator(device=DEV).manual_seed(0)
    r = lambda *s: torch.randn(*s, device=DEV, generator=gen, dtype=torch.bfloat16)  # noqa: E731
    y, w = r(M, N).requires_grad_(), r(N)
    assert y.numel() > 1 << 31
    out, res = residual_rms_norm(y, y.detach(), w, post_weight=w, gate=y.detach(), scale=w)
    (dy,) = torch.autograd.grad((out, res), [y], (y.detach(), y.detach()))
    t = y.detach()[-400:].clone().requires_grad_()
    o2, r2 = residual_rms_norm(t, t.detach(), w, post_weight=w, gate=t.detach(), scale=w)
    (dt,) = torch.autograd.grad((o2, r2), [t], (t.detach(), t.detach()))
    assert torch.equal(out[-400:], o2) and torch.equal(res[-400:], r2) and torch.equal(dy[-400:], dt)


@gpu
def test_captured_replay_and_other_stream():
    v, cot = _inputs(300, 1024, torch.bfloat16)
    want = _run(v, "silu", cot)
    ins = {k: t.to(DEV) for k, t in v.items()}
    dcot = [c.to(DEV) for c in cot]

    def work():
        lv = {k: t.detach().requires_grad_() for k, t in ins.items()}
        a = dict(lv)
        o = residual_rms_norm(a.pop("y"), a.pop("residual"), a.pop("weight"), eps=EPS, **a)
        return [*(x.detach() for x in o), *torch.autograd.grad(o, list(lv.values()), dcot)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = work()
    torch.cuda.current_stream().wait_stream(s)
    names = ["out", "res", *ins]
    assert all(torch.equal(o, want[k]) for k, o in zip(names, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    v2, _ = _inputs(300, 1024, torch.bfloat16, seed=4)
    for k, t in ins.items():
        t.copy_(v2[k])
    graph.replay()
    want = _run(v2, "silu", cot)
    assert all(torch.equal(o, want[k]) for k, o in zip(names, out))


@gpu
@pytest.mark.parametrize("N,dtype", [(256, torch.float32), (257, torch.float32), (8200, torch.float32),
                                     (512, torch.bfloat16), (16384, torch.bfloat16)])
@pytest.mark.parametrize("which", ["y", "residual"])
def test_gradients_of_large_and_small_rows(N, dtype, which, monkeypatch):
    """Rows whose norm's cube, or its reciprocal's, is outside the fp32 range.  Small ones want eps = 0:
    the formulas' gradients then grow as the rows shrink."""
    for size in (1e15, 1e-14):
        monkeypatch.setitem(globals(), "EPS", 1e-6 if size > 1 else 0.0)
        post = which == "y"
        v, (do, dr) = _inputs(6, N, dtype, post=post)
        v["y"][2] *= size
        if not post:
            v["residual"][2] *= size
        for cot in ((do, dr), (do, None)):
            _check(v, "silu", cot)


# ---------------------------------------------------------------------------
# on the CPU: the row view, refusals
# ---------------------------------------------------------------------------
def test_row_view_of_strided_tensors():
    base = torch.arange(2 * 3 * 4 * 10.).view(2, 3, 4, 10)
    cases = [base, base[..., 2:7], base[:, :, ::2, 2:7], base[:, 1:2, :, :5], base[:, :, 1:2, :5],
             base.transpose(1, 2), base[:1, ::2, 1, 3:], base[..., ::2], base[0, 0, 0], base[0, 0, 0, ::3],
             base[:, :, :1].expand(2, 3, 4, 10), torch.as_strided(base, (2, 1, 3, 4), (40, 40, 10, 1)),
             torch.as_strided(base, (3, 1, 4), (7, 99, 1)), base[..., :1]]
    for t in cases:
        N = t.shape[-1]
        rows, ld = _rows(t, N)
        M = t.numel() // N
        flat = torch.as_strided(rows, (M, N), (ld, 1), rows.storage_offset())
        assert torch.equal(flat, t.reshape(M, N)), (t.shape, t.stride())


@pytest.fixture()
def host(monkeypatch):
    def call(name, *a):
        raise AssertionError(f"{name} was reached")
    monkeypatch.setattr(_lib, "call", call)
    monkeypatch.setattr(_lib, "require_cuda", lambda t, op: None)


def _z(*s, dtype=torch.float32):
    return torch.zeros(*s, dtype=dtype)


@pytest.mark.parametrize("err,args,kw", [
    (ValueError, (_z(2, 4), _z(2, 5), _z(4)), {}),
    (ValueError, (_z(2, 4), _z(2, 4), _z(5)), {}),
    (ValueError, (_z(2, 4), _z(2, 4), _z(4)), {"post_weight": _z(1)}),
    (ValueError, (_z(2, 4), _z(2, 4), _z(4)), {"gate": _z(2, 1)}),
    (ValueError, (_z(2, 4), _z(2, 4), _z(4)), {"gate": _z(2, 4), "gate_activation": "none"}),
    (ValueError, (_z(2, 4), _z(2, 4), _z(4)), {"gate_activation": "relu"}),
    (ValueError, (_z(2, 4), _z(2, 4), _z(4)), {"scale": _z(())}),
    (ValueError, (_z(()), _z(()), _z(4)), {}),
    (ValueError, (_z(2, 0), _z(2, 0), _z(0)), {}),
    (TypeError, (_z(2, 4), _z(2, 4, dtype=torch.float16), _z(4)), {}),
    (TypeError, (_z(2, 4), _z(2, 4), _z(4, dtype=torch.float16)), {}),
    (TypeError, (_z(2, 4), _z(2, 4), _z(4)), {"scale": _z(4, dtype=torch.float16)}),
    (TypeError, (_z(2, 4), _z(2, 4), _z(4)), {"gate": _z(2, 4, dtype=torch.float16)}),
    (TypeError, [_z(2, 4, dtype=torch.float64)] * 2 + [_z(4)], {}),
])
def test_refusals(host, err, args, kw):
    with pytest.raises(err, match="residual_rms_norm"):
        residual_rms_norm(*args, **kw)


def test_tangents_are_refused(host):
    """A dual tensor would lose its tangent in a launch."""
    fw = torch.autograd.forward_ad
    with fw.dual_level():
        for k in range(6):
            a = [_z(2, 4), _z(2, 4), _z(4), _z(4), _z(2, 4), _z(4)]
            a[k] = fw.make_dual(a[k], torch.ones_like(a[k]))
            with pytest.raises(RuntimeError, match="residual_rms_norm: has no forward-mode"):
                residual_rms_norm(*a[:3], post_weight=a[3], gate=a[4], scale=a[5])


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        residual_rms_norm(_z(2, 4), _z(2, 4), _z(4))


def test_c_entry_checks():
    P, nul = 0x1000, None

    def fwd(M, N, act, gate, dtype=0, w_dtype=0, p=P):
        _lib.call("fo_residual_rms_norm_fwd", p, p, p, nul, gate, nul, 1.0, p, p, nul, nul, M, N, N, N, N,
                  1e-6, act, dtype, w_dtype, None)
    with pytest.raises(ValueError, match="bad size"):
        fwd(1, 0, 0, nul)
    with pytest.raises(ValueError, match="bad activation"):
        fwd(1, 4, 3, P)
    with pytest.raises(ValueError, match="a gate needs"):
        fwd(1, 4, 0, P)
    with pytest.raises(ValueError, match="a gate needs"):
        fwd(1, 4, 1, nul)
    with pytest.raises(ValueError, match="null pointer"):
        fwd(1, 4, 0, nul, p=nul)
    with pytest.raises(RuntimeError, match="weights of dtype code 1"):
        fwd(1, 4, 0, nul, dtype=0, w_dtype=1)
    with pytest.raises(RuntimeError, match="unsupported dtype code 4"):
        fwd(1, 4, 0, nul, dtype=4, w_dtype=4)
    fwd(0, 4, 0, nul, p=nul)
    with pytest.raises(RuntimeError, match="workspace of"):
        _lib.call("fo_residual_rms_norm_bwd", P, P, P, P, P, nul, nul, nul, 1.0, nul, P, P, P, nul, P, nul,
                  nul, 2, 8, 8, 8, 8, 0, 0, 0, nul, 0, None)
