"""CPU: what the linear layer's entry points refuse before any CUDA call is made."""
import ctypes as C

import pytest

P = 1 << 20   # a made-up, aligned address: never dereferenced, every call below is refused or empty


def test_forward_arguments(lib):
    def call(fmt=1, out=2, act=0, m=64, n=64, k=64, x=P, w=2 * P, y=3 * P, z=None, bias=None, residual=None):
        return lib.ko_linear(fmt, out, act, m, n, k, x, w, bias, residual, y, z, None, 0, None)

    assert call(fmt=2) == 1 and call(out=1) == 1 and call(fmt=0, out=2) == 1 and call(out=3) == 1
    assert call(act=5) == 1 and call(act=-1) == 1 and b"activation" in lib.ko_last_error_string()
    assert call(m=-1) == 1 and call(n=1 << 31) == 3
    assert call(k=0) == 3 and call(k=12) == 3
    assert call(x=None) == 1 and call(w=None) == 1 and call(y=None) == 1
    assert call(x=P + 2) == 2 and call(w=P + 8) == 2 and call(y=3 * P + 1) == 2 and call(bias=P + 1) == 2 and call(out=0, residual=P + 2) == 2
    assert call(y=P) == 1 and call(y=2 * P) == 1 and call(z=3 * P) == 1 and call(z=P) == 1 and call(z=4 * P, residual=4 * P) == 1
    assert call(m=0) == 0 and call(n=0) == 0


def test_backward_arguments(lib):
    def dx(fmt=1, out=2, act=0, m=64, n=64, k=64, dy=P, w=2 * P, z=None, x=3 * P):
        return lib.ko_linear_backward_input(fmt, out, act, m, n, k, dy, w, z, x, None, 0, None)

    assert dx(fmt=-1) == 1 and dx(out=1) == 1 and dx(act=9) == 1 and dx(n=0) == 3 and dx(n=12) == 3 and dx(k=20) == 3 and dx(m=-2) == 1
    assert dx(act=2) == 1 and b"pre-activation" in lib.ko_last_error_string()
    assert dx(dy=None) == 1 and dx(w=P + 4) == 2 and dx(x=P) == 1 and dx(out=0, act=1, z=3 * P) == 1 and dx(act=1, z=P + 1) == 2
    assert dx(m=0) == 0 and dx(k=0) == 0

    def dw(fmt=1, out=0, m=64, n=64, k=64, dy=P, x=2 * P, c=None, w=3 * P, b=None):
        return lib.ko_linear_backward_weight(fmt, out, m, n, k, dy, x, c, w, b, None, 0, None)

    assert dw(fmt=3) == 1 and dw(out=1) == 1 and dw(n=4) == 3 and dw(k=4) == 3 and dw(m=-1) == 1
    assert dw(dy=None) == 1 and dw(x=None) == 1 and dw(w=None) == 1 and dw(dy=P + 2) == 2 and dw(w=3 * P + 2) == 2 and dw(c=3 * P + 2) == 2
    assert dw(w=P) == 1 and dw(w=2 * P) == 1 and dw(b=3 * P) == 1 and dw(b=P + 2) == 2
    assert dw(b=P) == 1 and dw(b=2 * P) == 1 and dw(c=4 * P, b=4 * P) == 1 and dw(k=0, b=P) == 1 and b"dbias" in lib.ko_last_error_string()
    assert dw(n=0) == 0


def test_workspace_queries(lib):
    n = C.c_size_t(7)
    for name in ("ko_linear_workspace", "ko_linear_backward_input_workspace", "ko_linear_backward_weight_workspace"):
        f = getattr(lib, name)
        assert f(4, 4, 4, None) == 1 and f(-1, 4, 4, C.byref(n)) == 1 and n.value == 0
        assert f(0, 64, 64, C.byref(n)) == 0 and n.value == 0
    assert lib.ko_linear_workspace(32, 4096, 4096, C.byref(n)) == 0 and n.value == 0   # few tokens need none


def test_wrappers_refuse_host_tensors(ko):
    import torch

    x, w = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(16, 8, dtype=torch.bfloat16)
    for call in (lambda: ko.linear(x, w), lambda: ko.linear_backward_input(x, w.t()), lambda: ko.linear_backward_weight(x, x),
                 lambda: ko.linear(x[0], w), lambda: ko.linear(x, w, activation="swish"), lambda: ko.linear(x.double(), w.double())):
        with pytest.raises(ValueError):
            call()


def test_pinned_plans(lib):
    """Slices without a tile are refused for any number of tokens, few ones included, which no plan would have used them for."""
    def call(m, tile, slices):
        return lib.ko_linear_tuned(1, 2, 0, m, 64, 256, P, 2 * P, None, None, 3 * P, None, None, 0, tile, slices, None)

    for m in (4, 64):
        assert call(m, 0, 2) == 1 and b"slices" in lib.ko_last_error_string()
        assert call(m, 64, 0) == 1 and b"tile code" in lib.ko_last_error_string()
    assert lib.ko_linear_backward_weight_tuned(1, 0, 64, 64, 64, P, 2 * P, None, 3 * P, None, None, 0, 0, 2, None) == 1
