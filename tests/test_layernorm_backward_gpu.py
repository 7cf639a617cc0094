"""GPU: LayerNorm backward against its formula in 64 bits and against central differences.

Tolerances.  u = 2^-24.  A sum whose longest chain of FP32 additions has k links is off by at most k u times the sum of
the terms' magnitudes (first order).  With A the largest |x| of a row, mean and deviations are off by at most
(k + 1) u A, rstd relatively by (k + 4) u plus twice that times rstd A (the deviations enter squared), so every product
in dx is off by at most 4 (k + 4) u (1 + rstd A) times its own magnitude; dx is then rounded once, by at most half a
step of its type.  k counts a thread's elements, the five lane steps, the warps and the partial rows; 64 covers them for
rows up to 20480 columns on at least 256 threads, 128 the column sums of up to 20000 rows."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _types(torch):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _inputs(torch, dtype, rows, cols, gamma=True, residual=False, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    x = (normal(rows, cols) * (0.25 + normal(rows, 1).abs()) + normal(rows, 1)).to(dtype)
    return dict(dy=normal(rows, cols).to(dtype), x=x, gamma=(1.0 + 0.2 * normal(cols)).to(dtype) if gamma else None,
                residual=normal(rows, cols).to(dtype) if residual else None)


def _reference(torch, dy, x, eps, gamma=None, ddof=0, residual=None):
    """(dx, dgamma, dbeta) in 64 bits and what their rounding errors scale with."""
    x64, dy64 = x.double(), dy.double()
    n = x.shape[1]
    d = n - ddof
    mean = x64.mean(1, keepdim=True)
    dev = x64 - mean
    var = (dev * dev).sum(1, keepdim=True) / d if d > 0 else torch.zeros_like(mean)
    rstd = (var + eps).rsqrt()
    xhat = dev * rstd
    w = dy64 * gamma.double() if gamma is not None else dy64
    c1 = w.mean(1, keepdim=True)
    c2 = (w * xhat).sum(1, keepdim=True) / d if d > 0 else torch.zeros_like(mean)
    dx = rstd * (w - c1 - xhat * c2)
    spread = 1.0 + rstd * x64.abs().amax(1, keepdim=True)
    absw = w.abs().mean(1, keepdim=True)
    dx_scale = rstd * spread * (w.abs() + absw + xhat.abs() * (w * xhat).abs().sum(1, keepdim=True) / max(d, 1) + absw * spread)
    if residual is not None:
        dx = dx + residual.double()
        dx_scale = dx_scale + residual.double().abs()
    return (dx, (dy64 * xhat).sum(0), dy64.sum(0)), (dx_scale, (dy64.abs() * (xhat.abs() + 1.0) * spread).sum(0), dy64.abs().sum(0))


def _check(torch, got, want, scale, dtype):
    half_step = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    smallest = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
    for name, g, w, s, step, tiny, k in (("dx", got[0], want[0], scale[0], half_step, smallest, 64),
                                         ("dgamma", got[1], want[1], scale[1], 0.0, 0.0, 128),
                                         ("dbeta", got[2], want[2], scale[2], 0.0, 0.0, 128)):
        tol = step * w.abs() * (1 + 2 * step) + tiny + 4 * (k + 4) * U * s
        worst = ((g.double() - w).abs() / tol).nan_to_num(nan=float("inf")).max().item() if g.numel() else 0.0
        assert worst <= 1.0, (name, worst)


SHAPES = [(1, 1), (1, 7), (3, 8), (2, 64), (5, 250), (7, 1001), (64, 256), (33, 512), (130, 768), (9, 1000), (300, 1024), (17, 2048), (12, 2056),
          (40, 4096), (5, 5120), (3, 8192), (4, 10240), (2, 16384), (3, 20480), (2, 20481), (1, 40000), (2000, 64), (20000, 24), (4099, 96)]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_matches_the_formula(cuda, lib, ko, kind, rows, cols):
    dtype = _types(cuda)[kind]
    for gamma, residual, ddof in ((True, False, 0), (False, True, 1), (True, True, 0)):
        a = _inputs(cuda, dtype, rows, cols, gamma, residual, seed=rows + cols)
        got = ko.layernorm_backward(a["dy"], a["x"], 1e-5, a["gamma"], ddof, residual=a["residual"])
        want, scale = _reference(cuda, a["dy"], a["x"], 1e-5, a["gamma"], ddof, a["residual"])
        _check(cuda, got, want, scale, dtype)
        again = ko.layernorm_backward(a["dy"], a["x"], 1e-5, a["gamma"], ddof, residual=a["residual"])
        assert all(cuda.equal(p, q) for p, q in zip(got, again)), "the same call gives the same bits"


@pytest.mark.parametrize("rows,cols", [(3, 40), (2, 513), (4, 1024)])
def test_matches_central_differences(cuda, ko, rows, cols):
    a = _inputs(cuda, cuda.float32, rows, cols, seed=5)
    eps, h = 1e-5, 1e-6
    beta = cuda.zeros(cols, device="cuda", dtype=cuda.float64)

    def loss(x, gamma, beta):
        dev = x - x.mean(1, keepdim=True)
        return (a["dy"].double() * (dev * ((dev * dev).mean(1, keepdim=True) + eps).rsqrt() * gamma + beta)).sum()

    grads = ko.layernorm_backward(a["dy"], a["x"], eps, a["gamma"])
    at = (a["x"].double(), a["gamma"].double(), beta)
    gen = cuda.Generator(device="cuda").manual_seed(1)
    for i, grad in enumerate(grads):
        for _ in range(4):
            v = cuda.randn(at[i].shape, generator=gen, device="cuda", dtype=cuda.float64)
            plus, minus = list(at), list(at)
            plus[i], minus[i] = at[i] + h * v, at[i] - h * v
            slope = (loss(*plus) - loss(*minus)).item() / (2 * h)
            # differences: third derivatives (O(1) here) times h^2, and 2^-53 |loss| / h of cancellation; the gradient's own FP32 error
            mine = (grad.double() * v).sum().item()
            assert abs(mine - slope) <= 1e-6 * (grad.double() * v).abs().sum().item() * 64 + 1e-5, (i, mine, slope)


def test_forward_and_backward_agree_on_eps_and_ddof(cuda, ko):
    """The forward pass's own output is the xhat that the backward pass differentiates: dgamma = sum(dy * y) without affine."""
    a = _inputs(cuda, cuda.float32, 50, 640, gamma=False)
    for eps, ddof in ((1e-12, 0), (0.5, 1)):
        y = ko.layernorm(a["x"], eps, ddof=ddof)
        dgamma = ko.layernorm_backward(a["dy"], a["x"], eps, ddof=ddof)[1].double()
        want = (a["dy"].double() * y.double()).sum(0)
        assert ((dgamma - want).abs() <= 200 * U * (a["dy"].double().abs() * (y.double().abs() + 4)).sum(0)).all()


@pytest.mark.parametrize("cols", [512, 771, 20480])
def test_dx_may_replace_any_input(cuda, ko, cols):
    a = _inputs(cuda, cuda.bfloat16, 77, cols, residual=True)
    want = ko.layernorm_backward(a["dy"], a["x"], 1e-5, a["gamma"], residual=a["residual"])
    for name in ("dy", "x", "residual"):
        b = {k: v.clone() for k, v in a.items()}
        got = ko.layernorm_backward(b["dy"], b["x"], 1e-5, b["gamma"], residual=b["residual"], dx=b[name])
        assert got[0] is b[name] and all(cuda.equal(p, q) for p, q in zip(got, want))


def test_constant_rows_and_a_single_column(cuda, ko):
    """No spread: rstd = eps^-1/2 and xhat = 0."""
    x = cuda.full((4, 96), 3.0, device="cuda")
    dy = cuda.randn(4, 96, device="cuda")
    dx, dgamma, dbeta = ko.layernorm_backward(dy, x, 0.25)
    want = 2.0 * (dy.double() - dy.double().mean(1, keepdim=True))
    assert ((dx.double() - want).abs() <= 2 * 70 * U * (dy.abs() + 1).double()).all()
    assert not dgamma.any() and ((dbeta.double() - dy.double().sum(0)).abs() <= 8 * U * dy.double().abs().sum(0)).all()
    for ddof in (0, 1):
        dx, dgamma, dbeta = ko.layernorm_backward(dy[:, :1].contiguous(), x[:, :1].contiguous(), 0.25, ddof=ddof)
        assert not dx.any() and not dgamma.any()


def test_no_eps(cuda, ko):
    """eps = 0, with every number of rows left over by the blocks."""
    for cols in (24, 64, 100, 200, 512, 1001):
        for rows in (1, 3, 31, 33):
            a = _inputs(cuda, cuda.float32, rows, cols, seed=rows)
            got = ko.layernorm_backward(a["dy"], a["x"], 0.0, a["gamma"])
            want, scale = _reference(cuda, a["dy"], a["x"], 0.0, a["gamma"])
            _check(cuda, got, want, scale, cuda.float32)


def test_a_bad_row_stays_in_its_row(cuda, ko):
    for cols in (256, 1001, 20480):
        a = _inputs(cuda, cuda.float16, 40, cols)
        want = ko.layernorm_backward(a["dy"], a["x"], 1e-5, a["gamma"])[0]
        a["x"][7, cols // 2] = float("inf")
        a["x"][21, 0] = float("nan")
        got, dgamma, dbeta = ko.layernorm_backward(a["dy"], a["x"], 1e-5, a["gamma"])
        good = [r for r in range(40) if r not in (7, 21)]
        assert cuda.equal(got[good], want[good]) and got[7].isnan().any() and got[21].isnan().all()
        assert dgamma.isnan().all() and dbeta.isfinite().all()


def test_no_rows_and_no_columns(cuda, ko):
    x = cuda.empty(0, 48, device="cuda")
    dx, dgamma, dbeta = ko.layernorm_backward(x, x, 1e-5)
    assert dx.shape == (0, 48) and not dgamma.any() and not dbeta.any()
    x = cuda.empty(5, 0, device="cuda")
    assert ko.layernorm_backward(x, x, 1e-5)[0].shape == (5, 0)


def test_unaligned_operands_and_guards(cuda, lib, ko):
    """Operands that start between vector boundaries, with guard bytes on both sides of every one of them."""
    import ctypes as C

    from test_guard_regions_gpu import Guarded

    for cols in (64, 250, 768, 1001, 4096, 20480):
        rows = 37
        a = _inputs(cuda, cuda.float32, rows, cols, residual=True, seed=cols)
        want, scale = _reference(cuda, a["dy"], a["x"], 1e-5, a["gamma"], 0, a["residual"])
        need = C.c_size_t()
        assert lib.ko_layernorm_backward_workspace(0, rows, cols, C.byref(need)) == 0
        for shift in (0, 4):   # bytes past a 16-byte boundary
            g = {k: Guarded.of(cuda, np.concatenate([np.zeros(shift // 4, np.float32), v.cpu().numpy().ravel()])) for k, v in a.items()}
            dx = Guarded(cuda, rows * cols * 4 + shift)
            dgamma, dbeta, ws = Guarded(cuda, cols * 4), Guarded(cuda, cols * 4), Guarded(cuda, need.value)
            rc = lib.ko_layernorm_backward_f32(g["dy"].ptr() + shift, g["x"].ptr() + shift, dx.ptr() + shift, rows, cols, 1e-5,
                                               g["gamma"].ptr() + shift, g["residual"].ptr() + shift, dgamma.ptr(), dbeta.ptr(), 0,
                                               ws.ptr(), need.value, cuda.cuda.current_stream().cuda_stream)
            assert rc == 0, lib.ko_last_error_string()
            cuda.cuda.synchronize()
            assert all(b.intact() for b in (*g.values(), dx, dgamma, dbeta, ws))
            got = [cuda.from_numpy(t.copy()).cuda() for t in (dx.numpy(np.float32, -1)[shift // 4:].reshape(rows, cols),
                                                              dgamma.numpy(np.float32, cols), dbeta.numpy(np.float32, cols))]
            _check(cuda, got, want, scale, cuda.float32)


def test_either_vector_may_be_left_out(cuda, lib):
    import ctypes as C

    a = _inputs(cuda, cuda.float32, 300, 640)
    need = C.c_size_t()
    assert lib.ko_layernorm_backward_workspace(0, 300, 640, C.byref(need)) == 0
    ws = cuda.empty(need.value, dtype=cuda.uint8, device="cuda")
    s = cuda.cuda.current_stream().cuda_stream
    outs = []
    for g_wanted, b_wanted in ((True, True), (True, False), (False, True), (False, False)):
        dx, dgamma, dbeta = cuda.empty_like(a["x"]), cuda.full((640,), -7.0, device="cuda"), cuda.full((640,), -7.0, device="cuda")
        assert lib.ko_layernorm_backward_f32(a["dy"].data_ptr(), a["x"].data_ptr(), dx.data_ptr(), 300, 640, 1e-5, a["gamma"].data_ptr(), None,
                                             dgamma.data_ptr() if g_wanted else None, dbeta.data_ptr() if b_wanted else None, 0,
                                             ws.data_ptr(), need.value, s) == 0
        outs.append((dx, dgamma, dbeta))
    for (dx, dgamma, dbeta), g_wanted, b_wanted in zip(outs, (True, True, False, False), (True, False, True, False)):
        assert cuda.equal(dx, outs[0][0])
        assert cuda.equal(dgamma, outs[0][1]) if g_wanted else bool((dgamma == -7).all())
        assert cuda.equal(dbeta, outs[0][2]) if b_wanted else bool((dbeta == -7).all())


@pytest.mark.parametrize("rows,cols", [(540_000, 4096), (540_000, 4097), (270_000, 8200)])
def test_offsets_past_32_bits(cuda, lib, ko, rows, cols):
    """More than 2^31 elements a tensor (one pass, single elements, two passes): zeros but for the last rows, which are checked."""
    a = _inputs(cuda, cuda.bfloat16, 70, cols, residual=True, seed=1)
    big = {name: cuda.zeros(rows, cols, dtype=cuda.bfloat16, device="cuda") for name in ("dy", "x", "residual")}
    for name, t in big.items():
        assert t.numel() > 2 ** 31
        t[-70:] = a[name]
    dx, dgamma, dbeta = ko.layernorm_backward(big["dy"], big["x"], 1e-5, a["gamma"], residual=big["residual"], dx=big["dy"])
    want, scale = _reference(cuda, a["dy"], a["x"], 1e-5, a["gamma"], residual=a["residual"])
    _check(cuda, (dx[-70:], dgamma, dbeta), want, scale, cuda.bfloat16)
    assert not dx[:-70].any() and lib.ko_poll_device_status() == 0


def test_streams_and_graphs(cuda, lib, ko):
    """On another stream by context and by handle; two graphs captured on one stream and replayed side by side."""
    a, b = _inputs(cuda, cuda.bfloat16, 900, 1024, seed=1), _inputs(cuda, cuda.bfloat16, 900, 1024, seed=2)
    want_a = ko.layernorm_backward(a["dy"], a["x"], 1e-5, a["gamma"])
    want_b = ko.layernorm_backward(b["dy"], b["x"], 1e-5, b["gamma"])
    side, other = cuda.cuda.Stream(), cuda.cuda.Stream()
    cuda.cuda.synchronize()
    with cuda.cuda.stream(side):
        got = ko.layernorm_backward(a["dy"], a["x"], 1e-5, a["gamma"])
    got2 = ko.layernorm_backward(a["dy"], a["x"], 1e-5, a["gamma"], stream=other.cuda_stream)
    cuda.cuda.synchronize()
    assert all(cuda.equal(p, q) and cuda.equal(r, q) for p, r, q in zip(got, got2, want_a))
    graphs, outs = [], []
    for t in (a, b):
        graph = cuda.cuda.CUDAGraph()
        with cuda.cuda.graph(graph, stream=side):
            outs.append(ko.layernorm_backward(t["dy"], t["x"], 1e-5, t["gamma"]))
        graphs.append(graph)
    for _ in range(5):
        with cuda.cuda.stream(side):
            graphs[0].replay()
        with cuda.cuda.stream(other):
            graphs[1].replay()
        cuda.cuda.synchronize()
        assert all(cuda.equal(p, q) for p, q in zip(outs[0], want_a)) and all(cuda.equal(p, q) for p, q in zip(outs[1], want_b))


def test_refusals_that_need_a_device(cuda, lib, ko):
    a = _inputs(cuda, cuda.float32, 16, 64)
    dx = cuda.empty_like(a["x"])
    ws = cuda.empty(64, dtype=cuda.uint8, device="cuda")
    call = lambda w, n: lib.ko_layernorm_backward_f32(a["dy"].data_ptr(), a["x"].data_ptr(), dx.data_ptr(), 16, 64, 1e-5, None, None, None,
                                                      None, 0, w, n, None)
    assert call(None, 1 << 20) == 1 and b"workspace" in lib.ko_last_error_string()
    assert call(ws.data_ptr(), 64) == 1
    assert call(ws.data_ptr() + 4, 1 << 20) == 2
    with pytest.raises(ValueError):
        ko.layernorm_backward(a["dy"].half(), a["x"], 1e-5)
    with pytest.raises(ValueError):
        ko.layernorm_backward(a["dy"].t(), a["x"].t(), 1e-5)
    with pytest.raises(ValueError):
        ko.layernorm_backward(a["dy"], a["x"], 1e-5, gamma=cuda.ones(63, device="cuda"))
    with pytest.raises(ValueError):
        ko.layernorm_backward(a["dy"].cpu(), a["x"], 1e-5)
