"""GPU: LayerNorm backward on 16-bit operands that start between vector boundaries, guard bytes around every one of them.

Tolerances as in test_layernorm_backward_gpu."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("cols", [8, 24, 64, 250, 501, 512, 1001, 2048, 3001, 4096, 8192, 8200])
def test_unaligned_16_bit_operands(cuda, lib, ko, kind, cols):
    """Widths that whole vectors would fit, and odd ones; rows left over by the blocks of every form; each operand shifted alone too."""
    from test_guard_regions_gpu import Guarded
    from test_layernorm_backward_gpu import _check, _inputs, _reference, _types

    dtype, code = _types(cuda)[kind], {"f16": 1, "bf16": 2}[kind]
    entry = getattr(lib, f"ko_layernorm_backward_{kind}")
    names = ("dy", "x", "gamma", "residual", "dx")
    for rows in (1, 37, 601):
        a = _inputs(cuda, dtype, rows, cols, residual=True, seed=cols + rows)
        want, scale = _reference(cuda, a["dy"], a["x"], 1e-5, a["gamma"], 0, a["residual"])
        need = C.c_size_t()
        assert lib.ko_layernorm_backward_workspace(code, rows, cols, C.byref(need)) == 0
        for moved in (names,) + tuple((n,) for n in names if rows == 37):
            shift = {n: 2 if n in moved else 0 for n in names}       # bytes past a 16-byte boundary
            bits = lambda n: a[n].contiguous().view(cuda.int16).cpu().numpy().ravel()
            g = {n: Guarded.of(cuda, np.concatenate([np.zeros(shift[n] // 2, np.int16), bits(n)])) for n in names[:4]}
            g["dx"] = Guarded(cuda, rows * cols * 2 + shift["dx"])
            dgamma, dbeta, ws = Guarded(cuda, cols * 4), Guarded(cuda, cols * 4), Guarded(cuda, need.value)
            at = {n: g[n].ptr() + shift[n] for n in names}
            assert entry(at["dy"], at["x"], at["dx"], rows, cols, 1e-5, at["gamma"], at["residual"], dgamma.ptr(), dbeta.ptr(), 0, ws.ptr(), need.value,
                         cuda.cuda.current_stream().cuda_stream) == 0, lib.ko_last_error_string()
            cuda.cuda.synchronize()
            assert all(b.intact() for b in (*g.values(), dgamma, dbeta, ws)), (rows, moved)
            dx = cuda.from_numpy(g["dx"].bytes.cpu().numpy()[shift["dx"]:].copy()).cuda().view(dtype).view(rows, cols)
            got = [dx] + [cuda.from_numpy(t.numpy(np.float32, cols).copy()).cuda() for t in (dgamma, dbeta)]
            _check(cuda, got, want, scale, dtype)
    assert lib.ko_poll_device_status() == 0
