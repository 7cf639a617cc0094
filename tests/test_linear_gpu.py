"""GPU: the linear layer and its gradients against their formulas in 64 bits and against central differences.

Tolerances.  A product of K 16-bit terms is exact term by term and summed in FP32; tensor cores may cut every addition off
instead of rounding it, so an accumulator of K terms (K / 16 instructions deep, a few additions inside each) is off by at
most (K / 4 + 64) * 2^-23 times the sum of the terms' magnitudes -- a bound with a large margin: errors of either sign cancel.
act has a slope of at most 1.13 in magnitude (all five), so act(z) is off by 1.13 times z's error plus the activation's own:
2e-6 (1 + |z|) for 16-bit results, 8 * 2^-24 (1 + |z|) for FP32 ones.  Slopes have a slope of at most 1.1.  Every stored
value is then rounded once, by half a step of its type."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]


def _act(torch, z, kind):
    c = math.sqrt(2.0 / math.pi)
    return {"none": lambda: z, "relu": lambda: z.clamp(min=0), "gelu": lambda: 0.5 * z * torch.erfc(-z * math.sqrt(0.5)),
            "gelu_tanh": lambda: z * torch.sigmoid(2 * c * (z + 0.044715 * z ** 3)), "silu": lambda: z * torch.sigmoid(z)}[kind]()


def _slope(torch, z, kind):
    z = z.detach().clone().requires_grad_()
    if kind == "relu":
        return (z > 0).double()
    return torch.autograd.grad(_act(torch, z, kind).sum(), z)[0].detach() if kind != "none" else torch.ones_like(z)


def _dtype(torch, kind):
    return {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}[kind]


def _randn(torch, shape, dtype, seed, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)


def _close(torch, got, want, err, what):
    """|got - want| <= err + half a step of got's type (and half its smallest subnormal)."""
    info = torch.finfo(got.dtype)
    half, tiny = info.eps / 2, info.smallest_normal * info.eps / 2
    tol = (1 + 2 * half) * err + half * want.abs() + tiny
    worst = ((got.double() - want).abs() / tol).nan_to_num(nan=float("inf")).max().item() if got.numel() else 0.0
    assert worst <= 1.0, (what, worst)


def _sum_error(a, b, K):
    return (K / 4 + 64) * 2.0 ** -23 * (a.double().abs() @ b.double().abs())


def _own_error(z, exact):
    return (8 * 2.0 ** -24 if exact else 2e-6) * (1 + z.abs())


def _forward_case(cuda, ko, kind, out_kind, m, n, k, act, bias, residual, pre, seed=0):
    dtype, out = _dtype(cuda, kind), _dtype(cuda, out_kind)
    x, w = _randn(cuda, (m, k), dtype, seed), _randn(cuda, (n, k), dtype, seed + 1, k ** -0.5)
    b = _randn(cuda, (n,), dtype, seed + 2, 0.5) if bias else None
    r = _randn(cuda, (m, n), out, seed + 3) if residual else None
    nan = float("nan")
    y0 = cuda.full((m, n), nan, dtype=out, device="cuda")
    z0 = cuda.full((m, n), nan, dtype=dtype, device="cuda") if pre else None
    got = ko.linear(x, w, b, act, r, out=y0, pre=z0)
    z = x.double() @ w.double().t()
    if bias:
        z = z + b.double()
    err = _sum_error(x, w.t(), k) + 2.0 ** -24 * z.abs()
    y, y_err = _act(cuda, z, act), 1.13 * err + (0 if act in ("none", "relu") else _own_error(z, out_kind == "f32"))
    if residual:
        y = y + r.double()
        y_err = y_err + 2.0 ** -24 * y.abs()
    if pre:
        got, got_z = got
        assert got_z is z0
        _close(cuda, got_z, z, err, ("pre", m, n, k))
    assert got is y0
    _close(cuda, got, y, y_err, ("y", kind, out_kind, m, n, k, act))
    again = ko.linear(x, w, b, act, r, out_dtype=out)
    assert cuda.equal(again, got), "the same call gives the same bits"


SHAPES = [(1, 1, 8), (1, 4096, 512), (2, 33, 40), (7, 100, 1000), (8, 16, 264), (9, 250, 776), (16, 1000, 2048), (17, 64, 4096), (31, 31, 72),
          (32, 513, 128), (33, 1, 8), (33, 100, 64), (100, 2053, 1096), (128, 256, 64), (129, 130, 136), (300, 768, 8192), (257, 520, 200),
          (1000, 36, 56), (1021, 1004, 72), (2048, 2048, 264), (4096, 512, 1024)]


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_forward(cuda, lib, ko, kind, m, n, k):
    for i, (out, bias, residual, pre) in enumerate([(kind, True, False, True), (kind, True, True, False), ("f32", False, True, True),
                                                    ("f32", True, False, False), (kind, False, False, False)]):
        _forward_case(cuda, ko, kind, out, m, n, k, ACTS[(m + i) % 5], bias, residual, pre, seed=i)
    assert lib.ko_poll_device_status() == 0


@pytest.mark.parametrize("kind,out", [("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("act", ACTS)
def test_activations_over_their_range(cuda, ko, kind, out, act):
    """Pre-activations from -30 to 30 through an identity weight, in every kernel form; values of the stored Z are exact."""
    dtype = _dtype(cuda, kind)
    for m in (8, 64, 4096):
        x = cuda.linspace(-30, 30, m * 64, device="cuda").to(dtype).view(m, 64)
        eye = cuda.eye(64, device="cuda").to(dtype)
        y, pre = ko.linear(x, eye, activation=act, out_dtype=_dtype(cuda, out), return_pre=True)
        assert cuda.equal(pre, x)
        z = x.double()
        _close(cuda, y, _act(cuda, z, act), 0.0 * z.abs() if act in ("none", "relu") else _own_error(z, out == "f32"), (act, m))
        dx = ko.linear_backward_input(cuda.ones_like(x), eye, x, act, out_dtype=_dtype(cuda, out))
        _close(cuda, dx, _slope(cuda, z, act), 0.0 * z.abs() if act in ("none", "relu") else _own_error(z, out == "f32"), ("slope", act, m))


BACK_SHAPES = [(1, 8, 8), (3, 64, 40), (33, 1000, 776), (128, 128, 256), (129, 136, 264), (250, 4096, 96), (1000, 520, 1032), (2048, 256, 2048),
               (4099, 512, 768)]


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("m,n,k", BACK_SHAPES)
def test_input_gradient(cuda, lib, ko, kind, m, n, k):
    dtype = _dtype(cuda, kind)
    dy, w, z = _randn(cuda, (m, n), dtype, 1), _randn(cuda, (n, k), dtype, 2, n ** -0.5), _randn(cuda, (m, k), dtype, 3, 1.5)
    plain = dy.double() @ w.double()
    err = _sum_error(dy, w, n)
    for out in (kind, "f32"):
        for act in ACTS:
            dx = cuda.full((m, k), float("nan"), dtype=_dtype(cuda, out), device="cuda")
            assert ko.linear_backward_input(dy, w, None if act == "none" else z, act, out=dx) is dx
            slope = _slope(cuda, z.double(), act)
            own = 0.0 if act in ("none", "relu") else plain.abs() * _own_error(z.double(), out == "f32")
            _close(cuda, dx, plain * slope, 1.13 * err + own + 2.0 ** -24 * (plain * slope).abs(), (m, n, k, act, out))
    assert lib.ko_poll_device_status() == 0


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("m,n,k", BACK_SHAPES + [(8, 2048, 2048), (20000, 64, 128), (5, 4104, 8), (777, 1000, 520), (8195, 1024, 264)])
def test_weight_and_bias_gradients(cuda, lib, ko, kind, m, n, k):
    dtype = _dtype(cuda, kind)
    dy, x = _randn(cuda, (m, n), dtype, 1, 0.1), _randn(cuda, (m, k), dtype, 2)
    plain, err = dy.double().t() @ x.double(), _sum_error(dy.t(), x, m)
    for out, with_c in (("f32", False), ("f32", True), (kind, False), (kind, True)):
        c = _randn(cuda, (n, k), _dtype(cuda, out), 4) if with_c else None
        dw = cuda.full((n, k), float("nan"), dtype=_dtype(cuda, out), device="cuda")
        got, dbias = ko.linear_backward_weight(dy, x, c, out=dw)
        want = plain + c.double() if with_c else plain
        assert got is dw
        _close(cuda, got, want, err + 2.0 ** -24 * want.abs(), ("dw", m, n, k, out, with_c))
        _close(cuda, dbias, dy.double().sum(0), (m / 8 + 64) * 2.0 ** -24 * dy.double().abs().sum(0), ("dbias", m, n))
        if with_c:
            again = ko.linear_backward_weight(dy, x, c, out=c, return_bias=False)   # gathered in place
            assert again is c and cuda.equal(again, got)
    assert lib.ko_poll_device_status() == 0


@pytest.mark.parametrize("act", ACTS)
def test_gradients_match_central_differences(cuda, ko, act):
    """loss = sum(g * (act(x0 w0^T + b0) w1^T)): differences of the 64-bit loss against the chained calls with FP32 results.
    The calls round z and the hidden activation to 16 bits, so the loss takes the weights where they act: from there on."""
    m, k, h, n = 40, 64, 72, 48
    dt = cuda.bfloat16
    x, w0, b0 = _randn(cuda, (m, k), dt, 1), _randn(cuda, (h, k), dt, 2, 0.12), _randn(cuda, (h,), dt, 3, 0.3)
    w1, g = _randn(cuda, (n, h), dt, 4, 0.12), _randn(cuda, (m, n), dt, 5)
    _, z = ko.linear(x, w0, b0, act, return_pre=True)
    dz = ko.linear_backward_input(g, w1, z, act, out_dtype=cuda.float32)
    z64 = z.double()
    if act == "relu":
        z64 = cuda.where(z64.abs() < 1e-3, cuda.full_like(z64, 0.5), z64)   # differences do not see a kink
    step = 1e-5
    gen = cuda.Generator(device="cuda").manual_seed(9)
    for _ in range(3):
        v = cuda.randn(m, h, generator=gen, device="cuda", dtype=cuda.float64)
        if act == "relu":
            v = v * (z.double().abs() >= 1e-3)
        f = lambda t: (g.double() * (_act(cuda, t, act) @ w1.double().t())).sum().item()
        slope = (f(z64 + step * v) - f(z64 - step * v)) / (2 * step)
        mine = (dz.double() * v).sum().item()
        assert abs(mine - slope) <= 1e-5 * (dz.double() * v).abs().sum().item() + 1e-5, (act, mine, slope)
    dzb = dz.to(dt)
    dw, db = ko.linear_backward_weight(dzb, x)
    for _ in range(3):
        v = cuda.randn(h, k, generator=gen, device="cuda", dtype=cuda.float64)
        slope = (dzb.double() * (x.double() @ v.t())).sum().item()      # the loss is linear in w0 from here on
        assert abs((dw.double() * v).sum().item() - slope) <= 1e-5 * (dw.double() * v).abs().sum().item() + 1e-6
    assert ((db.double() - dzb.double().sum(0)).abs() <= 80 * 2.0 ** -24 * dzb.double().abs().sum(0)).all()


def test_outputs_over_their_inputs(cuda, ko):
    for m in (5, 200, 4096):
        dt = cuda.bfloat16
        x, w, r = _randn(cuda, (m, 256), dt, 1), _randn(cuda, (512, 256), dt, 2, 0.06), _randn(cuda, (m, 512), dt, 3)
        want = ko.linear(x, w, activation="gelu", residual=r)
        r2 = r.clone()
        assert ko.linear(x, w, activation="gelu", residual=r2, out=r2) is r2 and cuda.equal(r2, want)
        z = _randn(cuda, (m, 256), dt, 4)
        dy = _randn(cuda, (m, 512), dt, 5)
        want = ko.linear_backward_input(dy, w, z, "silu")
        z2 = z.clone()
        assert ko.linear_backward_input(dy, w, z2, "silu", out=z2) is z2 and cuda.equal(z2, want)


def test_bad_values_stay_in_their_row(cuda, ko):
    """An infinity or NaN in one token reaches that token only, tails included (what lies past K, M or N is not multiplied in)."""
    for m, n, k in ((20, 100, 1000), (200, 100, 1000), (4097, 520, 72)):
        dt = cuda.float16
        x, w = _randn(cuda, (m, k), dt, 1), _randn(cuda, (n, k), dt, 2, k ** -0.5)
        want = ko.linear(x, w, activation="silu")
        x[3, k - 1], x[m - 1, 0] = float("inf"), float("nan")
        got = ko.linear(x, w, activation="silu")
        good = [i for i in range(m) if i not in (3, m - 1)]
        assert cuda.equal(got[good], want[good]) and got[m - 1].isnan().all() and not got[3].isfinite().all()


def test_no_tokens(cuda, ko):
    x, w = cuda.empty(0, 64, device="cuda", dtype=cuda.float16), _randn(cuda, (32, 64), cuda.float16, 1)
    assert ko.linear(x, w).shape == (0, 32)
    assert ko.linear_backward_input(cuda.empty(0, 32, device="cuda", dtype=cuda.float16), w).shape == (0, 64)
    dy = cuda.empty(0, 32, device="cuda", dtype=cuda.float16)
    dw, db = ko.linear_backward_weight(dy, x)
    assert not dw.any() and not db.any() and dw.shape == (32, 64)
    c = cuda.randn(32, 64, device="cuda")
    assert cuda.equal(ko.linear_backward_weight(dy, x, c, return_bias=False), c)


@pytest.mark.parametrize("n,k", [(256, 512), (1032, 264), (2048, 2048)])
def test_fp32_results_of_long_sums(cuda, lib, ko, n, k):
    """Tensor cores cut an accumulator off at every addition: up to 2^-23 of it per instruction (16 terms), half of that on
    average, always towards zero.  Sums kept in FP32 are therefore taken in periods of at most 2048 terms, 128 instructions, and the
    periods' sums added with rounding: off by 128 * 2^-24 plus half a step per period, relative to the sums' size (2-norm over
    all results, whose partial sums are no larger than the results on the whole).  A single accumulator over all 16384 terms
    is off by 1.9e-5."""
    m = 16384
    bound = 128 * 2.0 ** -24 + m / 2048 * 2.0 ** -24

    def off(got, want):
        return ((got.double() - want).norm() / want.norm()).item()

    dt = cuda.bfloat16
    dy, x = _randn(cuda, (m, n), dt, 1), _randn(cuda, (m, k), dt, 2)
    c = _randn(cuda, (n, k), cuda.float32, 3)
    want = dy.double().t() @ x.double()
    dw, db = ko.linear_backward_weight(dy, x)
    assert off(dw, want) <= bound and off(db, dy.double().sum(0)) <= bound
    assert off(ko.linear_backward_weight(dy, x, c, return_bias=False), want + c.double()) <= bound
    a, w = dy.t().contiguous(), x.t().contiguous()      # the same sums as a forward product and as an input gradient
    assert off(ko.linear(a, w, out_dtype=cuda.float32), want) <= bound
    assert off(ko.linear_backward_input(a, x, out_dtype=cuda.float32), want) <= bound
    assert lib.ko_poll_device_status() == 0


@pytest.mark.parametrize("tile,slices", [(128, 0), (128, 3), (256, 0), (256, 2), (2048, 0), (2048, 3)])
def test_every_plan_of_the_three_products(cuda, lib, ko, tile, slices):
    """Pinned tiles and K slices, with short and long sums, FP32 and 16-bit results."""
    P = lambda t: None if t is None else t.data_ptr()
    dt, s = cuda.bfloat16, cuda.cuda.current_stream().cuda_stream
    ws = cuda.empty(1 << 27, dtype=cuda.uint8, device="cuda")
    for m, n, k in ((300, 264, 392), (520, 392, 4104), (4104, 520, 264)):
        x, w, z = _randn(cuda, (m, k), dt, 1), _randn(cuda, (n, k), dt, 2, k ** -0.5), _randn(cuda, (m, k), dt, 3, 1.5)
        dy, bias = _randn(cuda, (m, n), dt, 4), _randn(cuda, (n,), dt, 5)
        for odt, fmt in ((dt, 2), (cuda.float32, 0)):
            r, c = _randn(cuda, (m, n), odt, 6), _randn(cuda, (n, k), odt, 7)
            y, pre = cuda.full((m, n), float("nan"), dtype=odt, device="cuda"), cuda.empty(m, n, dtype=dt, device="cuda")
            dx, dw = cuda.full((m, k), float("nan"), dtype=odt, device="cuda"), cuda.full((n, k), float("nan"), dtype=odt, device="cuda")
            db = cuda.empty(n, device="cuda")
            assert lib.ko_linear_tuned(1, fmt, 4, m, n, k, P(x), P(w), P(bias), P(r), P(y), P(pre), P(ws), ws.numel(), tile, slices, s) == 0
            assert lib.ko_linear_backward_input_tuned(1, fmt, 2, m, n, k, P(dy), P(w), P(z), P(dx), P(ws), ws.numel(), tile, slices, s) == 0
            assert lib.ko_linear_backward_weight_tuned(1, fmt, m, n, k, P(dy), P(x), P(c), P(dw), P(db), P(ws), ws.numel(), tile, slices, s) == 0
            assert lib.ko_poll_device_status() == 0
            z0 = x.double() @ w.double().t() + bias.double()
            err = _sum_error(x, w.t(), k) + 2.0 ** -23 * z0.abs()
            _close(cuda, pre, z0, err, "pre")
            _close(cuda, y, _act(cuda, z0, "silu") + r.double(), 1.13 * err + _own_error(z0, not fmt) + 2.0 ** -23 * (z0.abs() + r.double().abs()), "y")
            plain = dy.double() @ w.double()
            _close(cuda, dx, plain * _slope(cuda, z.double(), "gelu"),
                   1.13 * _sum_error(dy, w, n) + plain.abs() * (_own_error(z.double(), not fmt) + 2.0 ** -23), "dx")
            want = dy.double().t() @ x.double() + c.double()
            _close(cuda, dw, want, _sum_error(dy.t(), x, m) + 2.0 ** -23 * want.abs(), "dw")
            _close(cuda, db, dy.double().sum(0), (m / 8 + 64) * 2.0 ** -24 * dy.double().abs().sum(0), "db")


def test_no_input_features(cuda, ko):
    """k = 0: dw is empty, the bias gradient is still the column sums."""
    for m, n in ((5, 64), (3000, 200)):
        dy, x = _randn(cuda, (m, n), cuda.bfloat16, 1), cuda.empty(m, 0, device="cuda", dtype=cuda.bfloat16)
        dw, db = ko.linear_backward_weight(dy, x)
        assert dw.shape == (n, 0) and ((db.double() - dy.double().sum(0)).abs() <= (m / 8 + 64) * 2.0 ** -24 * dy.double().abs().sum(0)).all()


def test_bias_gradient_of_a_large_batch(cuda, ko):
    """A dY of more than half the L2, and its column sums."""
    dy, x = _randn(cuda, (6500, 4104), cuda.float16, 1, 0.1), _randn(cuda, (6500, 72), cuda.float16, 2)
    dw, db = ko.linear_backward_weight(dy, x)
    _close(cuda, dw, dy.double().t() @ x.double(), _sum_error(dy.t(), x, 6500), "dw")
    _close(cuda, db, dy.double().sum(0), (6500 / 8 + 64) * 2.0 ** -24 * dy.double().abs().sum(0), "dbias")
    again = ko.linear_backward_weight(dy, x)
    assert cuda.equal(dw, again[0]) and cuda.equal(db, again[1])


@pytest.mark.parametrize("out", ["bf16", "f32"])
@pytest.mark.parametrize("act", ACTS)
def test_activations_of_huge_and_bad_values(cuda, ko, out, act):
    """Far out every activation is its argument or nothing, and its slope 1 or 0; a NaN stays a NaN and its neighbours are spared."""
    big = cuda.tensor([1e3, 1e10, 3e18, 1e30], device="cuda")
    row = cuda.cat([big, -big, cuda.tensor([float("nan"), 1.0, -1.0, float("nan"), 2.0, -60.0, 60.0, float("nan")], device="cuda")]).bfloat16()
    ok = ~row.isnan()
    eye = cuda.eye(16, device="cuda").bfloat16()
    for m in (4, 64, 4096):
        z = row.repeat(m, 1)
        clean = cuda.where(ok, z, cuda.zeros_like(z))
        bias = cuda.where(ok, cuda.zeros_like(row), row)                 # the NaNs arrive with the bias: a product would spread them
        y = ko.linear(clean, eye, bias, act, out_dtype=_dtype(cuda, out)).double()
        dx = ko.linear_backward_input(cuda.ones_like(z), eye, None if act == "none" else z, act, out_dtype=_dtype(cuda, out)).double()
        assert (y.isnan() == ~ok).all() and (act in ("none", "relu") or (dx.isnan() == ~ok).all())
        tame = z.double().clamp(-1e3, 1e3)                               # the formulas overflow beyond
        want, slope = _act(cuda, tame, act), _slope(cuda, tame, act)
        want = cuda.where((z.double().abs() > 1e3) & (z.double() > 0), z.double(), want)
        if act == "none":
            want = z.double()
        step = cuda.finfo(_dtype(cuda, out)).eps
        assert ((y - want).abs()[:, ok] <= (step * want.abs() + 2e-6 * 61)[:, ok]).all()
        assert ((dx - slope).abs()[:, ok] <= (step * slope.abs() + 2e-6 * 61)[:, ok]).all()


def _np16(cuda, t):
    return t.contiguous().view(cuda.int16).cpu().numpy()


def test_guards_and_unaligned_outputs(cuda, lib, ko):
    """Guard bytes around every operand; outputs, bias and residual also off the 16-byte grid, which takes the direct stores."""
    import ctypes as C

    from test_guard_regions_gpu import Guarded

    dt, s = cuda.bfloat16, cuda.cuda.current_stream().cuda_stream
    for m, n, k in ((3, 37, 72), (20, 250, 264), (33, 100, 64), (200, 131, 1096), (300, 264, 72), (4097, 520, 136)):
        x, w, b = _randn(cuda, (m, k), dt, 1), _randn(cuda, (n, k), dt, 2, k ** -0.5), _randn(cuda, (n,), dt, 3)
        need = C.c_size_t()
        assert lib.ko_linear_workspace(m, n, k, C.byref(need)) == 0
        for out_fmt in (0, 2):
            size, odt = (2, dt) if out_fmt else (4, cuda.float32)
            r = _randn(cuda, (m, n), odt, 4)
            want, want_z = ko.linear(x, w, b, "gelu", r, out_dtype=odt, return_pre=True)
            for shift in (0, size):
                def shifted(t):
                    raw = np.frombuffer(t.contiguous().view(cuda.uint8).cpu().numpy().tobytes(), np.uint8)
                    return Guarded.of(cuda, np.concatenate([np.zeros(shift, np.uint8), raw]))
                gx, gw, gb, gr = Guarded.of(cuda, _np16(cuda, x)), Guarded.of(cuda, _np16(cuda, w)), shifted(b), shifted(r)
                gy, gz, ws = Guarded(cuda, m * n * size + shift), Guarded(cuda, m * n * 2 + shift), Guarded(cuda, need.value)
                rc = lib.ko_linear(1, out_fmt, 2, m, n, k, gx.ptr(), gw.ptr(), gb.ptr() + shift, gr.ptr() + shift, gy.ptr() + shift, gz.ptr() + shift,
                                   ws.ptr(), need.value, s)
                assert rc == 0, lib.ko_last_error_string()
                cuda.cuda.synchronize()
                assert lib.ko_poll_device_status() == 0
                assert all(g.intact() for g in (gx, gw, gb, gr, gy, gz, ws))
                y = cuda.from_numpy(gy.bytes.cpu().numpy()[shift:].copy()).cuda().view(odt).view(m, n)
                z = cuda.from_numpy(gz.bytes.cpu().numpy()[shift:].copy()).cuda().view(dt).view(m, n)
                # K slices may be cut differently for the two kinds of stores: FP32 summation order, at most one step of the type apart
                for got, ref in ((y, want), (z, want_z)):
                    step = cuda.finfo(got.dtype).eps * ref.double().abs() + _sum_error(x, w.t(), k) * 1.13 + 2e-6
                    assert ((got.double() - ref.double()).abs() <= step).all(), (m, n, k, out_fmt, shift)
    for m, n, k in ((5, 64, 40), (200, 264, 136), (3000, 128, 264)):
        dy, x, w = _randn(cuda, (m, n), dt, 1), _randn(cuda, (m, k), dt, 2), _randn(cuda, (n, k), dt, 3)
        need = C.c_size_t()
        for out_fmt, shift in ((0, 0), (2, 0), (0, 4), (2, 2)):
            size, odt = (2, dt) if out_fmt else (4, cuda.float32)
            gdy, gx, gw = (Guarded.of(cuda, _np16(cuda, t)) for t in (dy, x, w))
            assert lib.ko_linear_backward_weight_workspace(m, n, k, C.byref(need)) == 0
            gd, gbias, ws = Guarded(cuda, n * k * size + shift), Guarded(cuda, n * 4), Guarded(cuda, need.value)
            assert lib.ko_linear_backward_weight(1, out_fmt, m, n, k, gdy.ptr(), gx.ptr(), None, gd.ptr() + shift, gbias.ptr(), ws.ptr(),
                                                 need.value, s) == 0, lib.ko_last_error_string()
            cuda.cuda.synchronize()
            assert all(g.intact() for g in (gdy, gx, gd, gbias, ws))
            dw = cuda.from_numpy(gd.bytes.cpu().numpy()[shift:].copy()).cuda().view(odt).view(n, k)
            _close(cuda, dw, dy.double().t() @ x.double(), _sum_error(dy.t(), x, m), ("dw", m, n, k))
            assert lib.ko_linear_backward_input_workspace(m, n, k, C.byref(need)) == 0
            gx2, ws = Guarded(cuda, m * k * size + shift), Guarded(cuda, need.value)
            assert lib.ko_linear_backward_input(1, out_fmt, 2, m, n, k, gdy.ptr(), gw.ptr(), gx.ptr(), gx2.ptr() + shift, ws.ptr(), need.value, s) == 0
            cuda.cuda.synchronize()
            assert all(g.intact() for g in (gdy, gw, gx, gx2, ws))
            dx = cuda.from_numpy(gx2.bytes.cpu().numpy()[shift:].copy()).cuda().view(odt).view(m, k)
            plain = dy.double() @ w.double()
            _close(cuda, dx, plain * _slope(cuda, x.double(), "gelu"), 1.13 * _sum_error(dy, w, n) + plain.abs() * _own_error(x.double(), not out_fmt), ("dx", m, n, k))
        assert lib.ko_poll_device_status() == 0


@pytest.mark.parametrize("m,n,k", [(700, 520, 1024), (700, 520, 1096), (2048, 4104, 2048), (2049, 4101, 4096), (130, 2056, 6904)])
def test_fp32_results_of_middling_sums(cuda, lib, ko, m, n, k):
    """As above: up to 1024 values of K in one accumulator (64 instructions), beyond that in periods of at most as many, in one tile a
    CTA and in several, stored by TMA and row by row.  One accumulator over 4096 values would be off by 4.5e-6."""
    bound = 64 * 2.0 ** -24 + (k / 896 + 1) * 2.0 ** -24
    x, w = _randn(cuda, (m, k), cuda.float16, 1), _randn(cuda, (n, k), cuda.float16, 2)
    want = x.double() @ w.double().t()
    got = ko.linear(x, w, out_dtype=cuda.float32)
    assert ((got.double() - want).norm() / want.norm()).item() <= bound
    if n % 8 == 0:
        got = ko.linear_backward_input(x, w.t().contiguous(), out_dtype=cuda.float32)
        assert ((got.double() - want).norm() / want.norm()).item() <= bound
    assert lib.ko_poll_device_status() == 0


@pytest.mark.parametrize("tile,slices", [(128, 0), (128, 2), (256, 0), (256, 2), (2048, 0), (2048, 2), (0, 0)])
@pytest.mark.parametrize("tokens", [130, 2100, 8200])
def test_bias_gradient_of_every_plan(cuda, lib, ko, tile, slices, tokens):
    """The column sums' way through every tile, alone or shared by tiles, with and without K slices; a workspace full of NaN."""
    import ctypes as C

    n, k, dt = 264, 1032, cuda.bfloat16
    dy, x = _randn(cuda, (tokens, n), dt, 1), _randn(cuda, (tokens, k), dt, 2)
    tiles = -(-n // 128) * -(-k // 128)
    need = C.c_size_t(max(slices, 1) * (tiles * 2 * 128 * 256 + 4 * n) * 4)
    if tile == 0:
        assert lib.ko_linear_backward_weight_workspace(tokens, n, k, C.byref(need)) == 0
    ws = cuda.full((need.value // 4,), float("nan"), device="cuda")
    for out_fmt, odt in ((0, cuda.float32), (2, dt)):
        dw, db = cuda.full((n, k), float("nan"), dtype=odt, device="cuda"), cuda.full((n,), float("nan"), device="cuda")
        assert lib.ko_linear_backward_weight_tuned(1, out_fmt, tokens, n, k, dy.data_ptr(), x.data_ptr(), None, dw.data_ptr(), db.data_ptr(), ws.data_ptr(),
                                                   ws.numel() * 4, tile, slices, cuda.cuda.current_stream().cuda_stream) == 0, lib.ko_last_error_string()
        _close(cuda, dw, dy.double().t() @ x.double(), _sum_error(dy.t(), x, tokens), "dw")
        # 16 rows added one by one, then a block's sums: at most 16 + tokens / 64 + 8 roundings on the way of a value
        _close(cuda, db, dy.double().sum(0), (tokens / 64 + 24) * 2.0 ** -24 * dy.double().abs().sum(0), "db")
    assert lib.ko_poll_device_status() == 0


@pytest.mark.parametrize("n", [4096, 4097])
def test_offsets_past_32_bits(cuda, lib, ko, n):
    """More than 2^31 elements of Y, Z and dX (stored by TMA, and row by row) and of dY: the last rows are checked."""
    m, k, dt = 540_000, 64, cuda.bfloat16
    x, w, b = _randn(cuda, (m, k), dt, 1), _randn(cuda, (n, k), dt, 2, k ** -0.5), _randn(cuda, (n,), dt, 3)
    y, z = ko.linear(x, w, b, "relu", return_pre=True)
    assert y.numel() > 2 ** 31
    for rows in (slice(0, 70), slice(m - 70, m)):
        want = x[rows].double() @ w.double().t() + b.double()
        err = _sum_error(x[rows], w.t(), k) + 2.0 ** -24 * want.abs()
        _close(cuda, z[rows], want, err, "z")
        _close(cuda, y[rows], want.clamp(min=0), err, "y")
    if n % 8 == 0:
        dx = ko.linear_backward_input(x, w.t().contiguous(), z, "relu", out=y)
        rows = slice(m - 70, m)
        _close(cuda, dx[rows], (x[rows].double() @ w.double().t()) * (z[rows] > 0), _sum_error(x[rows], w.t(), k), "dx")
        y[:-70].zero_()
        dw, db = ko.linear_backward_weight(y, x)
        _close(cuda, dw, y[rows].double().t() @ x[rows].double(), _sum_error(y[rows].t(), x[rows], m), "dw")
        _close(cuda, db, y[rows].double().sum(0), (m / 8 + 64) * 2.0 ** -24 * y[rows].double().abs().sum(0), "db")
    assert lib.ko_poll_device_status() == 0


def test_streams_and_graphs(cuda, lib, ko):
    """Other streams, and two graphs with K slices captured on one stream and replayed side by side."""
    dt = cuda.bfloat16
    sets = [(_randn(cuda, (128, 8192), dt, s), _randn(cuda, (256, 8192), dt, s + 1, 0.01), _randn(cuda, (256,), dt, s + 2)) for s in (1, 11)]
    dys = [_randn(cuda, (4096, 64), dt, s) for s in (21, 22)]
    xs = [_randn(cuda, (4096, 128), dt, s) for s in (31, 32)]

    def calls(i):
        return (ko.linear(*sets[i], activation="gelu"), ko.linear(sets[i][0][:4], *sets[i][1:]), *ko.linear_backward_weight(dys[i], xs[i]),
                ko.linear_backward_input(sets[i][0][:, :256].contiguous(), sets[i][1]))

    want = [calls(0), calls(1)]
    side, other = cuda.cuda.Stream(), cuda.cuda.Stream()
    cuda.cuda.synchronize()
    y = ko.linear(*sets[0], activation="gelu", stream=other.cuda_stream)
    with cuda.cuda.stream(side):
        got = calls(1)
    cuda.cuda.synchronize()
    assert cuda.equal(y, want[0][0]) and all(cuda.equal(p, q) for p, q in zip(got, want[1]))
    graphs, outs = [], []
    for i in (0, 1):
        graph = cuda.cuda.CUDAGraph()
        with cuda.cuda.graph(graph, stream=side):
            outs.append(calls(i))
        graphs.append(graph)
    for _ in range(5):
        with cuda.cuda.stream(side):
            graphs[0].replay()
        with cuda.cuda.stream(other):
            graphs[1].replay()
        cuda.cuda.synchronize()
        for i in (0, 1):
            assert all(cuda.equal(p, q) for p, q in zip(outs[i], want[i]))
    assert lib.ko_poll_device_status() == 0


def test_refusals_that_need_a_device(cuda, lib, ko):
    dt = cuda.bfloat16
    x, w = _randn(cuda, (128, 8192), dt, 1), _randn(cuda, (256, 8192), dt, 2)
    y = cuda.empty(128, 256, dtype=dt, device="cuda")
    assert lib.ko_linear(1, 2, 0, 128, 256, 8192, x.data_ptr(), w.data_ptr(), None, None, y.data_ptr(), None, None, 0, None) == 1
    assert b"workspace" in lib.ko_last_error_string()
    for bad in (lambda: ko.linear(x, w.half()), lambda: ko.linear(x, w[:, :64]), lambda: ko.linear(x, w, out_dtype=cuda.float16),
                lambda: ko.linear(x, w, bias=cuda.zeros(256, device="cuda")), lambda: ko.linear(x, w, activation="tanh"),
                lambda: ko.linear(x.float(), w.float()), lambda: ko.linear(x, w, residual=cuda.zeros(128, 255, device="cuda", dtype=dt)),
                lambda: ko.linear(x, w.cpu()), lambda: ko.linear(x[:, ::2], w[:, :4096].contiguous()),
                lambda: ko.linear_backward_weight(x, w), lambda: ko.linear_backward_input(x, w)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(ko.KoError):
        ko.linear(x[:, :12].contiguous(), w[:, :12].contiguous())       # K not a multiple of 8
    with pytest.raises(ko.KoError):
        ko.linear_backward_input(x, w.t().contiguous(), activation="gelu")   # no pre-activation
