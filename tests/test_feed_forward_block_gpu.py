"""GPU: the operators together, as one pre-norm feed-forward block is trained and served with them:

    h = layernorm(x);  a = gelu(h W1^T + b1), z kept;  y = a W2^T + b2 + x
    and back: dW2, db2, dz (through the GELU), dW1, db1, dh, dx (through the norm, plus the skip connection)

against the same block in 64 bits.  Every call hands on 16-bit tensors, so each step's inputs carry the rounding of the step
before, relative 2^-9 (BF16) or 2^-12 (FP16) each; a gradient passes at most six of them (h, a, z, dz, dh and its own result).
Roundings are independent and each product or norm at most doubles a relative 2-norm error, which bounds the 2-norm of every
result by 32 half steps of its type, FP32 sums by the same since their inputs are 16 bits."""
import pytest

pytestmark = pytest.mark.gpu


def _block(ko, p, x, eps=1e-5):
    h = ko.layernorm(x, eps, p["gamma"], p["beta"])
    a, z = ko.linear(h, p["w1"], p["b1"], activation="gelu", return_pre=True)
    return ko.linear(a, p["w2"], p["b2"], residual=x), (x, h, a, z)


def _block_backward(ko, p, dy, saved, eps=1e-5, into=None):
    x, h, a, z = saved
    into = into or {}
    dw2, db2 = ko.linear_backward_weight(dy, a, c=into.get("w2"), out=into.get("w2"))
    dz = ko.linear_backward_input(dy, p["w2"], z, activation="gelu")
    dw1, db1 = ko.linear_backward_weight(dz, h, c=into.get("w1"), out=into.get("w1"))
    dh = ko.linear_backward_input(dz, p["w1"])
    dx, dgamma, dbeta = ko.layernorm_backward(dh, x, eps, p["gamma"], residual=dy, dx=dh)
    return dict(x=dx, gamma=dgamma, beta=dbeta, w1=dw1, b1=db1, w2=dw2, b2=db2)


def _parameters(torch, dtype, width, inner, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s, scale=1.0, shift=0.0: (torch.randn(*s, generator=gen, device="cuda") * scale + shift).to(dtype)
    return dict(gamma=r(width, scale=0.2, shift=1.0), beta=r(width, scale=0.1), w1=r(inner, width, scale=width ** -0.5),
                b1=r(inner, scale=0.1), w2=r(width, inner, scale=inner ** -0.5), b2=r(width, scale=0.1))


def _reference(torch, p, x, dy, eps=1e-5):
    q = {k: v.double().requires_grad_() for k, v in {**p, "x": x}.items()}
    F = torch.nn.functional
    h = F.layer_norm(q["x"], (x.shape[1],), q["gamma"], q["beta"], eps)
    y = F.linear(F.gelu(F.linear(h, q["w1"], q["b1"])), q["w2"], q["b2"]) + q["x"]
    return y.detach(), dict(zip(q, torch.autograd.grad(y, list(q.values()), dy.double())))


def _off(got, want):
    return ((got.double() - want).norm() / want.norm()).item()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("tokens,width,inner", [(1, 64, 256), (20, 136, 520), (700, 768, 2048), (4099, 256, 1024)])
def test_training_step(cuda, lib, ko, kind, tokens, width, inner):
    dtype = cuda.float16 if kind == "f16" else cuda.bfloat16
    p = _parameters(cuda, dtype, width, inner, 1)
    gen = cuda.Generator(device="cuda").manual_seed(2)
    x, dy = (cuda.randn(tokens, width, generator=gen, device="cuda").to(dtype) for _ in range(2))
    want_y, want = _reference(cuda, p, x, dy)
    y, saved = _block(ko, p, x)
    bound = 32 * cuda.finfo(dtype).eps / 2
    assert _off(y, want_y) <= bound
    grads = _block_backward(ko, p, dy, saved)
    for name, w in want.items():
        assert _off(grads[name], w) <= bound, (name, _off(grads[name], w))
    # a second micro-batch gathered into the first one's weight gradients
    first = {n: grads[n].clone() for n in ("w1", "w2")}
    again = _block_backward(ko, p, dy, saved, into={n: grads[n] for n in ("w1", "w2")})
    for n in ("w1", "w2"):
        assert again[n] is grads[n] and _off(again[n], 2 * first[n].double()) <= 2.0 ** -20
    assert lib.ko_poll_device_status() == 0


def test_captured_training_step(cuda, lib, ko):
    """The whole step in one graph, captured without any call before it, replayed on other inputs; an eager step runs between."""
    p = _parameters(cuda, cuda.bfloat16, 512, 2048, 3)
    x, dy = (cuda.zeros(1000, 512, device="cuda", dtype=cuda.bfloat16) for _ in range(2))
    side = cuda.cuda.Stream()
    graph = cuda.cuda.CUDAGraph()
    with cuda.cuda.graph(graph, stream=side):
        y, saved = _block(ko, p, x)
        grads = _block_backward(ko, p, dy, saved)
    for seed in (1, 2):
        gen = cuda.Generator(device="cuda").manual_seed(seed)
        x.copy_(cuda.randn(1000, 512, generator=gen, device="cuda"))
        dy.copy_(cuda.randn(1000, 512, generator=gen, device="cuda"))
        eager_y, eager_saved = _block(ko, p, x)
        eager = _block_backward(ko, p, dy, eager_saved)
        graph.replay()
        cuda.cuda.synchronize()
        assert cuda.equal(y, eager_y) and all(cuda.equal(grads[n], eager[n]) for n in grads)
    assert lib.ko_poll_device_status() == 0


def test_first_calls_of_a_process_inside_a_capture():
    """Nothing has to be called once before: the first use of every kernel may be the captured one."""
    import os
    import subprocess
    import sys

    code = '''
import torch, kernel_optimization_b200 as ko
from test_feed_forward_block_gpu import _block, _block_backward, _parameters
p = _parameters(torch, torch.bfloat16, 512, 2048, 3)
x, dy = (torch.randn(1000, 512, device="cuda").bfloat16() for _ in range(2))
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y, saved = _block(ko, p, x)
    grads = _block_backward(ko, p, dy, saved)
    token = _block(ko, p, x[:1])[0]
graph.replay()
want, saved = _block(ko, p, x)
again = _block_backward(ko, p, dy, saved)
torch.cuda.synchronize()
assert torch.equal(y, want) and all(torch.equal(grads[n], again[n]) for n in grads) and torch.equal(token, _block(ko, p, x[:1])[0])
assert ko.lib().ko_poll_device_status() == 0
print("captured")
'''
    here = os.path.dirname(os.path.abspath(__file__))
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([os.path.dirname(here), here, os.environ.get("PYTHONPATH", "")]))
    out = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "captured" in out.stdout, out.stderr[-2000:]


def test_tokens_one_by_one(cuda, ko):
    """Serving: each token alone gives what it gives in a batch, to the rounding of the steps' results."""
    p = _parameters(cuda, cuda.float16, 768, 2048, 4)
    x = cuda.randn(40, 768, generator=cuda.Generator(device="cuda").manual_seed(5), device="cuda").half()
    batch, _ = _block(ko, p, x)
    alone = cuda.cat([_block(ko, p, x[i:i + 1])[0] for i in range(40)])
    assert _off(alone, batch.double()) <= 8 * cuda.finfo(cuda.float16).eps
