"""scaled_embedding against its definition in 64 bits.

Tolerances, with U = 2^-24: the lookup is one fp32 product, U of its value, and half a step of
the output's type.  A gradient row of n terms carries at most (n + 1) U of the sum of their
magnitudes in any order, and half a step.
"""
import ctypes

import pytest
import torch

from operators import _lib
from operators.scaled_embedding import scaled_embedding, scaled_embedding_backward

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


def _ids(T, V, kind, gen, dtype=torch.int64):
    if kind == "same":
        ids = torch.full((T,), V - 1)
    elif kind == "zipf":
        ids = (torch.exp(torch.rand(T, generator=gen) * torch.log(torch.tensor(float(V)))) - 1).long().clamp(0, V - 1)
    elif kind == "descending":
        ids = (V - 1 - torch.arange(T)) % V
    else:
        ids = torch.randint(0, V, (T,), generator=gen)
    return ids.to(dtype)


def _check(T, V, N, dtype, kind="uniform", scale=1.5, index=torch.int64, padding_idx=None, ids=None):
    gen = torch.Generator().manual_seed(T + V + N)
    ids = _ids(T, V, kind, gen, index) if ids is None else ids
    w = (0.02 * torch.randn(V, N, generator=gen)).to(dtype)
    dout = torch.randn(T, N, generator=gen).to(dtype)
    wd = w.to(DEV).requires_grad_()
    out = scaled_embedding(ids.to(DEV), wd, scale, padding_idx=padding_idx)
    (dw,) = torch.autograd.grad(out, [wd], dout.to(DEV))
    inside = (ids >= 0) & (ids < V)
    look = ids.long().clamp(0, V - 1)
    ref = w.double()[look] * scale * inside[:, None]
    _within(out.detach(), ref, U * ref.abs(), "out")
    counted = inside.clone()
    if padding_idx is not None:
        counted &= ids != padding_idx % V
    terms = dout.double() * scale * counted[:, None]
    rw = torch.zeros(V, N, dtype=torch.float64).index_add_(0, look, terms)
    mag = torch.zeros(V, N, dtype=torch.float64).index_add_(0, look, terms.abs())
    n = torch.bincount(look[counted], minlength=V).double()[:, None]
    _within(dw, rw, (n + 1) * U * mag, "dw")
    # rows without a token are exactly zero
    assert bool((dw.cpu()[(n[:, 0] == 0)] == 0).all())
    return out.detach(), dw


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("index", [torch.int64, torch.int32])
@pytest.mark.parametrize("kind", ["uniform", "zipf", "same", "descending"])
def test_types_and_distributions(dtype, index, kind):
    _check(700, 300, 128, dtype, kind, index=index)


@gpu
@pytest.mark.parametrize("T", [1, 2, 31, 32, 33, 127, 128, 129, 1000, 1024, 1025, 4095, 4096, 4097,
                               8193, 20000])
def test_token_counts(T):
    _check(T, 517, 32, torch.float32, "zipf")


@gpu
@pytest.mark.parametrize("N", [1, 3, 8, 9, 64, 65, 771, 1000, 1024, 2048, 4096, 4100, 8192, 9001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_widths(N, dtype):
    _check(300, 40, N, dtype, "zipf")


@gpu
@pytest.mark.parametrize("V", [1, 2, 255, 256, 257, 511, 512, 513, 65535, 65536, 65537, 128256, 300007])
def test_vocabularies(V):
    _check(3000, V, 16, torch.bfloat16, "uniform")
    _check(9000, V, 8, torch.float32, "zipf")


@gpu
def test_many_equal_ids():
    _check(30000, 100, 72, torch.float32, "same")
    ids = torch.randint(0, 50, (30000,), generator=torch.Generator().manual_seed(0))
    ids[::3] = 7
    _check(30000, 50, 40, torch.bfloat16, ids=ids)


@gpu
def test_many_tokens():
    _check(200000, 1000, 8, torch.float32, "zipf")


@gpu
def test_padding_rows_get_no_gradient():
    ids = torch.randint(0, 64, (5000,), generator=torch.Generator().manual_seed(0))
    ids[::2] = 63
    for p in (63, -1, 0):
        _, dw = _check(5000, 64, 48, torch.float32, ids=ids, padding_idx=p)
        assert bool((dw[p] == 0).all())


@gpu
def test_ids_outside_are_zero_rows(monkeypatch):
    ids = torch.randint(0, 100, (2000,), generator=torch.Generator().manual_seed(0))
    ids[5::7] = -1
    ids[6::7] = 100
    ids[3] = 2 ** 40
    ids[4] = -2 ** 40
    out, _ = _check(2000, 100, 64, torch.float32, ids=ids)
    assert bool((out[5::7] == 0).all()) and bool((out[3:7] == 0).all())
    _check(500, 20, 8, torch.float32, ids=torch.full((500,), -100))
    monkeypatch.setenv("FLAGOPS_CHECK_INDEX", "1")
    with pytest.raises(IndexError, match="out of range"):
        scaled_embedding(ids.to(DEV), torch.zeros(100, 8, device=DEV))


@gpu
def test_nan_and_inf_stay_in_their_rows():
    ids = torch.tensor([3, 5, 3, 7, 5, 3] * 40)
    dout = torch.randn(240, 24, generator=torch.Generator().manual_seed(0))
    dout[1, 4] = float("nan")
    dout[3, 2] = float("inf")
    dw = scaled_embedding_backward(dout.to(DEV), ids.to(DEV), 9).cpu()
    assert bool(torch.isnan(dw[5, 4])) and bool(torch.isinf(dw[7, 2]))
    dw[5, 4] = dw[7, 2] = 0
    assert bool(torch.isfinite(dw).all())


@gpu
def test_strides_shapes_and_repeatability():
    gen = torch.Generator().manual_seed(0)
    wide = torch.randn(80, 200, generator=gen).to(DEV)
    ids = torch.randint(0, 80, (4, 6, 5), generator=gen).to(DEV)
    for w in (wide[:, 8:72], wide[:, 1:65], wide[::2, 8:72], wide.t()[:80, :64]):
        i = ids % w.shape[0]
        assert torch.equal(scaled_embedding(i, w, 2.0), 2 * w[i])
    t = ids.permute(2, 0, 1)
    assert torch.equal(scaled_embedding(t, wide, 2.0), 2 * wide[t])
    assert scaled_embedding(ids[0, 0, 0], wide, 2.0).shape == (200,)
    d = torch.randn(6, 4, 5, 200, generator=gen).to(DEV).transpose(0, 1)
    a = scaled_embedding_backward(d, ids, 80, 0.5)
    assert torch.equal(a, scaled_embedding_backward(d.contiguous(), ids, 80, 0.5))
    big = torch.randint(0, 50, (50000,), generator=gen).to(DEV)
    g = torch.randn(50000, 96, generator=gen).to(DEV).to(torch.bfloat16)
    first = scaled_embedding_backward(g, big, 50)
    for _ in range(3):
        assert torch.equal(first, scaled_embedding_backward(g, big, 50))


@gpu
def test_offsets_over_32_bits():
    """A table of 2.2e9 elements, and 2.2e9 elements looked up."""
    V, N = 270007, 8192
    w = torch.zeros(V, N, dtype=torch.bfloat16, device=DEV)
    w[-50:] = torch.randn(50, N, device=DEV).to(torch.bfloat16)
    ids = torch.randint(V - 50, V, (300,), generator=torch.Generator().manual_seed(0)).to(DEV)
    assert w.numel() > 1 << 31
    assert torch.equal(scaled_embedding(ids, w, 2.0), 2 * w[ids])
    d = torch.randn(300, N, device=DEV).to(torch.bfloat16)
    dw = scaled_embedding_backward(d, ids, V)
    small = scaled_embedding_backward(d, ids - (V - 50), 50)
    assert torch.equal(dw[-50:], small) and not bool(dw[:-50].any())
    del dw
    # ids of few rows, many tokens: the sums of the last tokens alone
    d = torch.zeros(V, N, dtype=torch.bfloat16, device=DEV)
    d[-30:] = 1
    many = torch.arange(V, device=DEV) % 7
    assert torch.equal(scaled_embedding(many, w[-7:], 1.0)[-20:], w[-7:][many[-20:]])
    dw = scaled_embedding_backward(d, many, 7)
    n = torch.bincount(many[-30:], minlength=7)
    assert torch.equal(dw.float(), n[:, None].float().expand(7, N))


@gpu
def test_empty():
    w = torch.randn(10, 16, device=DEV, requires_grad=True)
    out = scaled_embedding(torch.empty(0, 3, dtype=torch.int64, device=DEV), w)
    assert out.shape == (0, 3, 16)
    (dw,) = torch.autograd.grad(out.sum(), [w])
    assert bool((dw == 0).all())
    none = torch.empty(0, 16, device=DEV)
    assert bool((scaled_embedding(torch.tensor([0, 5], device=DEV), none) == 0).all())
    assert scaled_embedding(torch.tensor([0], device=DEV), torch.empty(4, 0, device=DEV)).shape == (1, 0)
    assert scaled_embedding_backward(torch.randn(2, 4, device=DEV), torch.tensor([0, 1], device=DEV),
                                     0).shape == (0, 4)


@gpu
def test_captured_replay_and_other_stream():
    gen = torch.Generator().manual_seed(0)
    ids = torch.randint(0, 400, (9000,), generator=gen).to(DEV)
    w = torch.randn(400, 64, generator=gen).to(DEV)
    d = torch.randn(9000, 64, generator=gen).to(DEV)

    def work():
        lw = w.detach().requires_grad_()
        out = scaled_embedding(ids, lw, 3.0)
        return out.detach(), *torch.autograd.grad(out, [lw], d)
    want = work()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = work()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    ids.copy_(torch.randint(0, 400, (9000,), generator=gen))
    d.copy_(torch.randn(9000, 64, generator=gen))
    for _ in range(2):
        graph.replay()
    want = work()
    assert all(torch.equal(a, b) for a, b in zip(want, out))


# ---------------------------------------------------------------------------
# refusals, on the CPU
# ---------------------------------------------------------------------------
@pytest.fixture()
def host(monkeypatch):
    def call(name, *a):
        raise AssertionError(f"{name} was reached")
    monkeypatch.setattr(_lib, "call", call)
    monkeypatch.setattr(_lib, "require_cuda", lambda t, op: None)


def test_refusals(host):
    i, w = torch.zeros(3, dtype=torch.int64), torch.zeros(4, 2)
    with pytest.raises(ValueError, match=r"\[V, N\]"):
        scaled_embedding(i, torch.zeros(4))
    with pytest.raises(TypeError, match="int64 or int32"):
        scaled_embedding(i.float(), w)
    with pytest.raises(TypeError, match="float64"):
        scaled_embedding(i, w.double())
    for p in (4, -5):
        with pytest.raises(ValueError, match="padding_idx"):
            scaled_embedding(i, w, padding_idx=p)
    with pytest.raises(ValueError, match="does not fit"):
        scaled_embedding_backward(torch.zeros(2, 2), i, 4)
    with pytest.raises(TypeError, match="float64"):
        scaled_embedding_backward(torch.zeros(3, 2).double(), i, 4)


def test_checked_ids_raise_before_the_library(host, monkeypatch):
    monkeypatch.setenv("FLAGOPS_CHECK_INDEX", "1")
    with pytest.raises(IndexError, match="out of range"):
        scaled_embedding(torch.tensor([0, 4]), torch.zeros(4, 2))
    with pytest.raises(IndexError, match="out of range"):
        scaled_embedding_backward(torch.zeros(1, 2), torch.tensor([-1]), 4)


def test_tangents_are_refused(host):
    """A dual tensor would lose its tangent in a launch."""
    fw = torch.autograd.forward_ad
    i, w, d = torch.zeros(3, dtype=torch.int64), torch.zeros(4, 2), torch.zeros(3, 2)
    with fw.dual_level():
        with pytest.raises(RuntimeError, match="scaled_embedding: has no forward-mode"):
            scaled_embedding(i, fw.make_dual(w, torch.ones_like(w)))
        with pytest.raises(RuntimeError, match="scaled_embedding_backward: has no forward-mode"):
            scaled_embedding_backward(fw.make_dual(d, torch.ones_like(d)), i, 4)


def test_cpu_tensors_are_refused():
    i, w = torch.zeros(3, dtype=torch.int64), torch.zeros(4, 2)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        scaled_embedding(i, w)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        scaled_embedding_backward(torch.zeros(3, 2), i, 4)


def test_c_entry_checks():
    P = 0x1000
    with pytest.raises(ValueError, match="negative size"):
        _lib.call("fo_embedding_fwd", P, P, P, -1, 4, 4, 4, 1.0, 0, 5, None)
    with pytest.raises(ValueError, match="over 2\\^30"):
        _lib.call("fo_embedding_fwd", P, P, P, 1 << 31, 4, 4, 4, 1.0, 0, 5, None)
    with pytest.raises(ValueError, match="null pointer"):
        _lib.call("fo_embedding_fwd", None, P, P, 1, 4, 4, 4, 1.0, 0, 5, None)
    with pytest.raises(ValueError, match="int64 or int32"):
        _lib.call("fo_embedding_fwd", P, P, P, 1, 4, 4, 4, 1.0, 0, 0, None)
    with pytest.raises(RuntimeError, match="unsupported dtype code 3"):
        _lib.call("fo_embedding_fwd", P, P, P, 1, 4, 4, 4, 1.0, 3, 5, None)
    with pytest.raises(ValueError, match="null pointer"):
        _lib.call("fo_embedding_bwd", None, None, P, 1, 4, 4, -1, 1.0, 0, 5, None, 0, None)
    _lib.call("fo_embedding_fwd", None, None, None, 0, 4, 4, 4, 1.0, 0, 5, None)
    n = ctypes.c_int64(-1)
    _lib.call("fo_embedding_bwd_workspace_bytes", 5, 4, 4, ctypes.byref(n))
    assert n.value >= 0
