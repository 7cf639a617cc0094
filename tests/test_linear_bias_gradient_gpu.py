"""GPU: the bias gradient's way beside the weight gradient's product, by every plan of the pair of CTAs.

dY holds small whole numbers, so that its column sums are exact in FP32 in any order: a value taken too early from a stage of the
ring, twice or not at all shows as a difference."""
import ctypes as C

import pytest

pytestmark = pytest.mark.gpu


def _whole(torch, shape, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-8, 9, shape, generator=gen, device="cuda").to(torch.bfloat16)


@pytest.mark.parametrize("slices", [0, 2, 5])
@pytest.mark.parametrize("k", [264, 512, 520, 1024, 1032, 2056])
def test_sums_of_a_pair_are_exact(cuda, lib, ko, k, slices):
    """Two to nine columns of tiles, an odd number of them too, features that end inside either half of a tile, long and short."""
    stream = cuda.cuda.current_stream().cuda_stream
    for n, tokens in ((136, 700), (264, 130 * 64), (392, 8193), (1000, 4100)):
        tiles = -(-n // 256) * -(-k // 256)
        ws = cuda.full((max(slices, 1) * (tiles * 256 * 256 + 4 * n),), float("nan"), device="cuda")
        x = _whole(cuda, (tokens, k), 7)
        want_dw = None
        for seed in range(4):
            dy = _whole(cuda, (tokens, n), seed)
            want_dw = dy.float().t().double() @ x.double()
            dw, db = cuda.full((n, k), float("nan"), device="cuda"), cuda.full((n,), float("nan"), device="cuda")
            assert lib.ko_linear_backward_weight_tuned(1, 0, tokens, n, k, dy.data_ptr(), x.data_ptr(), None, dw.data_ptr(), db.data_ptr(), ws.data_ptr(),
                                                       ws.numel() * 4, 2048, slices, stream) == 0, lib.ko_last_error_string()
            assert cuda.equal(db.double(), dy.double().sum(0)), (n, tokens, seed)
            assert cuda.equal(dw.double(), want_dw), (n, tokens, seed)      # |sums| below 2^24: exact as well
    assert lib.ko_poll_device_status() == 0


@pytest.mark.parametrize("tokens,n,k", [(16384, 4096, 256), (16384, 1024, 512), (32768, 512, 2048), (8192, 768, 768), (70000, 256, 72)])
def test_sums_of_chosen_plans_are_exact(cuda, lib, ko, tokens, n, k):
    for seed in range(3):
        dy, x = _whole(cuda, (tokens, n), seed), _whole(cuda, (tokens, k), seed + 9)
        dw, db = ko.linear_backward_weight(dy, x)
        assert cuda.equal(db.double(), dy.double().sum(0))
        assert cuda.equal(ko.linear_backward_weight(dy, x, return_bias=False).double(), dy.double().t() @ x.double())
        assert cuda.equal(dw.double(), dy.double().t() @ x.double())
    assert lib.ko_poll_device_status() == 0


def test_a_pair_needs_two_columns_of_tiles_for_the_sums(cuda, lib, ko):
    tokens, n, k = 512, 256, 256
    dy, x = _whole(cuda, (tokens, n), 1), _whole(cuda, (tokens, k), 2)
    dw, db = cuda.empty(n, k, device="cuda"), cuda.empty(n, device="cuda")
    call = lambda bias: lib.ko_linear_backward_weight_tuned(1, 0, tokens, n, k, dy.data_ptr(), x.data_ptr(), None, dw.data_ptr(), bias, None, 0, 2048, 0,
                                                            cuda.cuda.current_stream().cuda_stream)
    assert call(db.data_ptr()) == 3 and b"pair" in lib.ko_last_error_string()
    assert call(None) == 0
    assert cuda.equal(dw.double(), dy.double().t() @ x.double())
