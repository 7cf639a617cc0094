"""GPU: the activations of the linear layer and their slopes far out, at infinity, and in every form of the epilogue.

Through an identity weight a pre-activation reaches the epilogue exactly, whatever the form sums: few tokens (up to 32 rows), tiles
stored by TMA, tiles stored row by row (an output off the 16-byte grid), K slices."""
import pytest

pytestmark = pytest.mark.gpu

ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]
CODES = {name: i for i, name in enumerate(ACTS)}
FORMS = ["few", "tile", "rows", "slices"]


def _dtype(torch, kind):
    return {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}[kind]


def _places(torch, form, m, n, odt):
    """An output of m x n, off the 16-byte grid where the form wants it."""
    if form != "rows":
        return torch.full((m, n), float("nan"), dtype=odt, device="cuda")
    return torch.full((m * n + 1,), float("nan"), dtype=odt, device="cuda")[1:].view(m, n)


def _act(torch, lib, z, act, odt, form, bias=None):
    """act(z + bias) by ko_linear: z times the identity."""
    fmt = 1 if z.dtype == torch.bfloat16 else 0
    m, n = z.shape
    k = 128 if form == "slices" else n      # two slices of 64, the second over zeros
    x = torch.zeros(m, k, dtype=z.dtype, device="cuda")
    x[:, :n] = z
    w = torch.eye(n, k, device="cuda").to(z.dtype)
    y = _places(torch, form, m, n, odt)
    ws = torch.empty(1 << 24, dtype=torch.uint8, device="cuda")
    rows = range(0, m, 32) if form == "few" else (0,)
    size = y.element_size()
    for r in rows:
        part = min(32, m - r) if form == "few" else m
        status = lib.ko_linear_tuned(fmt, 0 if odt == torch.float32 else fmt + 1, CODES[act], part, n, k, x.data_ptr() + r * k * 2, w.data_ptr(),
                                     None if bias is None else bias.data_ptr(), None, y.data_ptr() + r * n * size, None, ws.data_ptr(), ws.numel(),
                                     0 if form == "few" else 128, 2 if form == "slices" else 0, torch.cuda.current_stream().cuda_stream)
        assert status == 0, lib.ko_last_error_string()
    return y


def _slope(torch, lib, z, act, odt, form):
    """act'(z) by ko_linear_backward_input: ones times the identity times the slope.  No form for few tokens: it takes the tiles."""
    fmt = 1 if z.dtype == torch.bfloat16 else 0
    m, n = z.shape
    k = 128 if form == "slices" else n
    dy = torch.zeros(m, k, dtype=z.dtype, device="cuda")
    dy[:, :n] = 1
    w = torch.eye(k, n, device="cuda").to(z.dtype)
    dx = _places(torch, form, m, n, odt)
    ws = torch.empty(1 << 24, dtype=torch.uint8, device="cuda")
    assert lib.ko_linear_backward_input_tuned(fmt, 0 if odt == torch.float32 else fmt + 1, CODES[act], m, k, n, dy.data_ptr(), w.data_ptr(), z.data_ptr(),
                                              dx.data_ptr(), ws.data_ptr(), ws.numel(), 128, 2 if form == "slices" else 0,
                                              torch.cuda.current_stream().cuda_stream) == 0, lib.ko_last_error_string()
    return dx


def _ordinary(torch, m, n, dtype, seed, scale=1.5):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(m, n, generator=gen, device="cuda") * scale).to(dtype)


@pytest.mark.parametrize("form", FORMS[1:])
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("kind,out", [("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32")])
def test_slopes_far_out_beside_ordinary_values(cuda, lib, kind, out, act, form):
    """Large z in even and odd columns and rows, whatever their neighbours hold: from 20 on every slope is 1 to within 5e-8, and below -30
    nothing.  What may be off: at most 20 times the logistic function's own error of 2^-22 (its reciprocal, two roundings), 4.8e-6,
    and half a step of the type."""
    dtype, odt = _dtype(cuda, kind), _dtype(cuda, out)
    far = cuda.tensor([20.0, 33.0, 1e2, 1e3, 2e4, 65504.0] + ([1e6, 1e10, 3e18, 1e30] if kind == "bf16" else []), device="cuda").to(dtype)
    for sign in (1, -1):
        if sign < 0:
            far = far[1:]
        for r0 in (0, 1):
            for c0 in (0, 1):
                z = _ordinary(cuda, 256, 64, dtype, 10 + r0 * 2 + c0)
                picked = z[r0::2, c0::2]
                picked.copy_((sign * far).repeat(-(-picked.numel() // len(far)))[:picked.numel()].view(picked.shape))
                got = _slope(cuda, lib, z, act, odt, form)[r0::2, c0::2].double()
                want = 1.0 if sign > 0 else 0.0
                worst = (got - want).abs().max().item()
                assert worst <= 6e-6 + want * cuda.finfo(odt).eps / 2, (sign, r0, c0, worst)
    assert lib.ko_poll_device_status() == 0


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("kind,out", [("f16", "f16"), ("bf16", "bf16"), ("f16", "f32"), ("bf16", "f32")])
def test_infinite_pre_activations(cuda, lib, kind, out, act, form):
    """The limits, for every type of result: act is inf and 0, its slope 1 and 0.  (FP16 pre-activations become infinite by overflow.)"""
    dtype, odt = _dtype(cuda, kind), _dtype(cuda, out)
    m, n = 64, 64
    inf = float("inf")
    bias = cuda.zeros(n, device="cuda", dtype=dtype)
    bias[5::9], bias[2::9] = inf, -inf
    z = _ordinary(cuda, m, n, dtype, 3)
    up, down = bias == inf, bias == -inf
    y = _act(cuda, lib, z, act, odt, form, bias)
    assert (y[:, up] == inf).all()
    assert (y[:, down] == (-inf if act == "none" else 0)).all()
    assert y[:, ~(up | down)].isfinite().all()
    if form != "few" and act != "none":
        z = z + bias
        dx = _slope(cuda, lib, z, act, odt, form)
        assert (dx[:, up] == 1).all() and (dx[:, down] == 0).all() and dx.isfinite().all()
    assert lib.ko_poll_device_status() == 0


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("kind,out", [("f16", "f16"), ("bf16", "bf16"), ("f16", "f32"), ("bf16", "f32")])
def test_every_form_gives_the_same_bits(cuda, lib, kind, out, act):
    """The same sums make the same results, wherever a value lies and whatever lies beside it."""
    dtype, odt = _dtype(cuda, kind), _dtype(cuda, out)
    m, n = 4096, 64
    z = _ordinary(cuda, m, n, dtype, 5, 4.0)
    bits = cuda.int32 if odt == cuda.float32 else cuda.int16
    y = _act(cuda, lib, z, act, odt, "tile")
    slope = None if act == "none" else _slope(cuda, lib, z, act, odt, "tile")
    for form in FORMS:
        got = _act(cuda, lib, z, act, odt, form)
        assert cuda.equal(got.view(bits) if form != "rows" else got.contiguous().view(bits), y.view(bits)), form
        if slope is not None and form != "few":
            assert cuda.equal(_slope(cuda, lib, z, act, odt, form), slope), form
    # other neighbours, in columns and in rows
    order = cuda.randperm(m * n, generator=cuda.Generator(device="cuda").manual_seed(1), device="cuda")
    mixed = z.view(-1)[order].view(m, n).contiguous()
    for form in FORMS:
        assert cuda.equal(_act(cuda, lib, mixed, act, odt, form).reshape(-1), y.view(-1)[order]), form
        if slope is not None and form != "few":
            assert cuda.equal(_slope(cuda, lib, mixed, act, odt, form).reshape(-1), slope.view(-1)[order]), form
    assert lib.ko_poll_device_status() == 0


@pytest.mark.parametrize("form", FORMS[1:])
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_small_slopes_keep_their_size(cuda, lib, kind, act, form):
    """Slopes of 16-bit gradients where they vanish: off by 8e-4 of themselves (GELU's fit 7.4e-4, its nine FP32 steps 2e-5, the rest of
    the arithmetic 2^-20) and half a step of the type -- not by a fixed amount that is more than the slope."""
    import math

    dtype = _dtype(cuda, kind)
    lowest = {"gelu": -5.5, "gelu_tanh": -6.0, "silu": -80.0}[act]
    if kind == "f16":       # the slope is to stay a normal FP16 number
        lowest = {"gelu": -4.5, "gelu_tanh": -4.0, "silu": -11.0}[act]
    z = cuda.linspace(lowest, -3.0, 256 * 64, device="cuda").to(dtype).view(256, 64)
    z = z.reshape(-1)[cuda.randperm(z.numel(), generator=cuda.Generator(device="cuda").manual_seed(2), device="cuda")].view(256, 64).contiguous()
    t = z.double()
    c = math.sqrt(2.0 / math.pi)
    if act == "gelu":
        want = 0.5 * cuda.special.erfc(-t * math.sqrt(0.5)) + t * cuda.exp(-t * t / 2) * (0.5 * c)
    else:
        u = 2 * c * (t + 0.044715 * t ** 3) if act == "gelu_tanh" else t
        du = 2 * c * (1 + 3 * 0.044715 * t ** 2) if act == "gelu_tanh" else 1.0
        s = cuda.sigmoid(u)
        want = s + t * s * cuda.sigmoid(-u) * du
    got = _slope(cuda, lib, z, act, dtype, form).double()
    half = cuda.finfo(dtype).eps / 2
    worst = ((got - want).abs() / want.abs()).max().item()
    assert worst <= 8e-4 + half * (1 + 8e-4), worst
