"""CPU: what the LayerNorm backward entry points refuse before any CUDA call is made."""
import ctypes as C

import pytest


def test_argument_validation_needs_no_gpu(lib):
    def call(rows, cols, ddof=0, entry="f32"):
        return getattr(lib, f"ko_layernorm_backward_{entry}")(None, None, None, rows, cols, 1e-5, None, None, None, None, ddof, None, 0, None)

    for entry in ("f32", "f16", "bf16"):
        assert call(-1, 4, entry=entry) == 1 and b"negative" in lib.ko_last_error_string()
        assert call(4, -4, entry=entry) == 1
        assert call(4, 4, ddof=2, entry=entry) == 1 and b"ddof" in lib.ko_last_error_string()
        assert call(4, 4, entry=entry) == 1 and b"NULL" in lib.ko_last_error_string()
        assert call(4, (1 << 30) + 1, entry=entry) == 3
        assert call(0, 16, entry=entry) == 0 and call(16, 0, entry=entry) == 0   # empty problems are legal no-ops
    n = C.c_size_t(99)
    assert lib.ko_layernorm_backward_workspace(0, 4, 4, None) == 1
    assert lib.ko_layernorm_backward_workspace(7, 4, 4, C.byref(n)) == 1 and n.value == 0
    assert lib.ko_layernorm_backward_workspace(0, -4, 4, C.byref(n)) == 1
    assert lib.ko_layernorm_backward_workspace(0, 0, 4, C.byref(n)) == 0 and n.value == 0


def test_wrapper_refuses_host_tensors_and_wrong_ranks(ko):
    import torch

    x = torch.zeros(4, 8)
    with pytest.raises(ValueError):
        ko.layernorm_backward(x, x, 1e-5)
    with pytest.raises(ValueError):
        ko.layernorm_backward(x[0], x[0], 1e-5)
    with pytest.raises(ValueError):
        ko.layernorm_backward(x.double(), x.double(), 1e-5)


@pytest.mark.parametrize("entry,size", [("f32", 4), ("f16", 2), ("bf16", 2)])
def test_addresses_between_elements(lib, entry, size):
    """Refused before any CUDA call: the kernels would load and store across element boundaries, which the hardware does not do."""
    p = 1 << 20   # made-up addresses, never dereferenced

    def call(dy=p, x=2 * p, dx=3 * p, gamma=None, residual=None, dgamma=None, dbeta=None):
        return getattr(lib, f"ko_layernorm_backward_{entry}")(dy, x, dx, 4, 16, 1e-5, gamma, residual, dgamma, dbeta, 0, 4 * p, 1 << 20, None)

    for name, at in (("dy", p), ("x", 2 * p), ("dx", 3 * p), ("gamma", 5 * p), ("residual", 6 * p)):
        for off in range(1, size):
            assert call(**{name: at + off}) == 2 and b"aligned" in lib.ko_last_error_string(), (name, off)
    for off in (1, 2, 3):
        assert call(dgamma=7 * p + off) == 2 and call(dbeta=7 * p + off) == 2
