"""GPU: products over hundreds of thousands of terms of one sign, in every form.

The tensor cores cut an accumulator off at every addition, always towards zero: K / 16 instructions, each off by up to 2^-23 of what the
accumulator holds by then, half of that on average, which for terms of one sign grows evenly: K / 16 * 2^-25 of the result, 7.5e-4 at
K = 400000 -- more than half a step of FP16.  16-bit results of more than 16384
terms are therefore summed in periods of 8192 (FP32 ones of more than 1024 in periods of 896) whose sums are added with rounding: 512 * 2^-24
for a period's own cut (twice its average for terms of one sign) and half a step, 2^-24, for each addition, K / 896 of them at most."""
import pytest

pytestmark = pytest.mark.gpu

K = 400_000


def _positive(torch, shape, dtype, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.rand(*shape, generator=gen, device="cuda") * 0.5 + 0.5).mul_(2.0 ** -4).to(dtype)


def _close(torch, got, want, terms=K):
    err = 512 * 2.0 ** -24 + (terms / 896 + 8) * 2.0 ** -24
    half = torch.finfo(got.dtype).eps / 2
    worst = ((got.double() - want).abs() / want).max().item()
    assert worst <= err + half * (1 + err), (worst, err, half)


@pytest.mark.parametrize("tile,slices,shift", [(128, 0, 0), (128, 2, 0), (128, 0, 2), (256, 0, 0), (256, 2, 0), (2048, 0, 0), (2048, 2, 0)])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_16_bit_results_of_long_sums(cuda, lib, kind, tile, slices, shift):
    """All three products; shift: bytes of the outputs past a 16-byte boundary, for the tiles that are stored row by row."""
    dt = {"f16": cuda.float16, "bf16": cuda.bfloat16}[kind]
    fmt, s = (1 if kind == "bf16" else 0), cuda.cuda.current_stream().cuda_stream
    ws = cuda.empty(1 << 24, dtype=cuda.uint8, device="cuda")
    n, k = 264, 328
    P = lambda t: t.data_ptr()

    def out(rows, cols):
        return cuda.full((rows * cols + shift // 2,), float("nan"), dtype=dt, device="cuda")[shift // 2:].view(rows, cols)

    dy, x = _positive(cuda, (K, n), dt, 1), _positive(cuda, (K, k), dt, 2)
    want = dy.double().t() @ x.double()
    dw, db = out(n, k), cuda.empty(n, device="cuda")
    assert lib.ko_linear_backward_weight_tuned(fmt, fmt + 1, K, n, k, P(dy), P(x), None, P(dw), P(db), P(ws), ws.numel(), tile, slices, s) == 0
    _close(cuda, dw, want)
    assert ((db.double() - dy.double().sum(0)).abs() <= (K / 64 + 24) * 2.0 ** -24 * dy.double().sum(0)).all()
    a, w = dy.t().contiguous(), x.t().contiguous()
    y = out(n, k)
    assert lib.ko_linear_tuned(fmt, fmt + 1, 0, n, k, K, P(a), P(w), None, None, P(y), None, P(ws), ws.numel(), tile, slices, s) == 0, lib.ko_last_error_string()
    _close(cuda, y, want)
    dx = out(n, k)
    assert lib.ko_linear_backward_input_tuned(fmt, fmt + 1, 0, n, K, k, P(a), P(x), None, P(dx), P(ws), ws.numel(), tile, slices, s) == 0
    _close(cuda, dx, want)
    assert lib.ko_poll_device_status() == 0


@pytest.mark.parametrize("m", [1, 8, 13, 20, 32])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_few_tokens_of_many_features(cuda, lib, ko, kind, m):
    dt = {"f16": cuda.float16, "bf16": cuda.bfloat16}[kind]
    for n in (2500, 24):        # one block a stretch of W, and clusters
        x, w = _positive(cuda, (m, K), dt, 3), _positive(cuda, (n, K), cuda.float32, 4)
        w = (w * cuda.linspace(0.5, 1.0, n, device="cuda")[:, None]).to(dt)      # results spread over a factor of two
        want = x.double() @ w.double().t()
        y = ko.linear(x, w)
        _close(cuda, y, want)
        # roundings of the spread results average out (five deviations of a uniform error's mean), what is cut off does not
        if n < 1000:
            continue
        half = cuda.finfo(dt).eps / 2
        assert ((y.double() - want) / want).mean().abs().item() <= (32 + 8) * 2.0 ** -24 + 5 * half / (3 * y.numel()) ** 0.5
        _close(cuda, ko.linear(x, w, out_dtype=cuda.float32), want)


@pytest.mark.parametrize("m", [1, 8, 13, 20, 32])
@pytest.mark.parametrize("k", [4096, 16384, 131072])
def test_fp32_results_for_few_tokens(cuda, ko, m, k):
    """A warp takes an eighth or a quarter of K, in pieces of 128, and puts its accumulators aside every 1024 values (64 instructions):
    terms of one sign, so each is off by 2^-25 of the accumulator on average, 32 * 2^-24 of the result.  Of K / 4 values in one
    accumulator a result would be off by K / 128 * 2^-24."""
    x, w = _positive(cuda, (m, k), cuda.bfloat16, 5), _positive(cuda, (4000, k), cuda.bfloat16, 6)
    want = x.double() @ w.double().t()
    got = ko.linear(x, w, out_dtype=cuda.float32)
    off = ((got.double() - want) / want).abs().mean().item()
    assert off <= (32 + 8) * 2.0 ** -24, off * 2 ** 24


@pytest.mark.parametrize("n,k", [(256, 512), (1032, 264), (2048, 2048), (250, 1001)])
def test_fp32_results_take_short_periods(cuda, lib, ko, n, k):
    """Terms of either sign.  A cut takes 0.36 * 2^-23 of the accumulator on average (half a unit of the last place, over mantissas), the
    accumulator is two thirds of a period's sum in size (it grows with the root of the terms), and the cuts go against its sign: at most
    0.24 * 2^-23 of the sum for each instruction of a period, which does not average out over periods.  With 56 instructions, 896 terms,
    1.6e-6 of the result's 2-norm; the periods' additions are rounded, and 2^-24 of each averages out.  Periods of 2048 terms would be
    off by more than twice as much."""
    m = 16384
    bound = 0.24 * 56 * 2.0 ** -23 + (m / 896) ** 0.5 * 2.0 ** -24

    def off(got, want):
        return ((got.double() - want).norm() / want.norm()).item()

    gen = cuda.Generator(device="cuda").manual_seed(n + k)
    a = cuda.randn(n, m, generator=gen, device="cuda").bfloat16()
    w = cuda.randn(k, m, generator=gen, device="cuda").bfloat16()
    want = a.double() @ w.double().t()
    assert off(ko.linear(a, w, out_dtype=cuda.float32), want) <= bound
    if n % 8 == 0:
        assert off(ko.linear_backward_weight(a.t().contiguous(), w.t().contiguous(), return_bias=False), want) <= bound
        assert off(ko.linear_backward_input(a, w.t().contiguous(), out_dtype=cuda.float32), want) <= bound
    assert lib.ko_poll_device_status() == 0
