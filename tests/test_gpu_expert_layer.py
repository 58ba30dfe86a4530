"""examples/expert_layer.py: the layer's gradients and its 4-bit answers against
the same formulas in 64 bits, and its training."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

_path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples", "expert_layer.py")
_spec = importlib.util.spec_from_file_location("expert_layer", _path)
E = importlib.util.module_from_spec(_spec)
_spec.loader.exec_module(E)

EXPERTS, WIDTH, HIDDEN = 6, 64, 128
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


@pytest.fixture(params=[torch.bfloat16, torch.float16, torch.float32], ids=str)
def layer(request):
    layer = E.Experts(EXPERTS, WIDTH, HIDDEN, request.param, seed=3)
    layer.b1.normal_(generator=torch.Generator(device="cuda").manual_seed(4))
    yield layer
    torch.cuda.synchronize()
    layer.close()


def tokens(n):
    g = torch.Generator(device="cuda").manual_seed(n)
    x = torch.randn(n, WIDTH, generator=g, device="cuda")
    scores = torch.randn(n, EXPERTS, generator=g, device="cuda")
    scores[:, 4] = -100.0  # an expert that nobody goes to
    return x, E.Routing(scores, 2), torch.randn(2 * n, WIDTH, generator=g, device="cuda")


def close(got, want, unit, what):
    """Norms: a result has a rounding of its own and those of the up to 2 rounded values
    it is formed from (h or grad_h, and what these come from), each half a unit at most; a
    sign of h that a rounding changes is one near 0, whose share is of that size too.
    sqrt(depth) * 2^-24 of an fp32 sum is far below the factor of 8 that is given."""
    far = (got.double().cpu() - want).norm() / want.norm()
    print(what, "%.3g of %.3g" % (far, 8 * unit), flush=True)
    assert far <= 8 * unit


@pytest.mark.parametrize("n", [1, 37, 300])
def test_gradients(layer, n):
    x, routing, grad_y = tokens(n)
    unit = UNIT[layer.dtype]
    y, kept = layer.forward(x, routing)
    got = layer.backward(grad_y, kept, routing)
    offsets = routing.offsets.tolist()
    assert offsets[0] == 0 and offsets[-1] == 2 * n and offsets[4] == offsets[5]
    held = [t.to(layer.dtype).double().cpu() for t in (x, layer.w1, layer.w2)]
    chosen = held[0][routing.token.cpu()].requires_grad_()
    w1, w2 = held[1].requires_grad_(), held[2].requires_grad_()
    b1 = layer.b1.double().cpu().requires_grad_()
    want = torch.cat([torch.relu(chosen[b:e] @ w1[i].t() + b1[i]) @ w2[i].t()
                      for i, (b, e) in enumerate(zip(offsets, offsets[1:]))])
    want.backward(grad_y.to(layer.dtype).double().cpu())
    close(y, want.detach(), unit, "y")
    for name, g, w in zip(("x", "w1", "b1", "w2"), got, (chosen, w1, b1, w2)):
        close(g, w.grad, unit, name)


@pytest.mark.parametrize("n", [1, 4, 37])
def test_answers_in_4_bits(layer, n):
    x, routing, _ = tokens(n)
    server = E.Server(layer)
    got = server.answer(x, routing)
    offsets = routing.offsets.tolist()
    chosen = x.to(layer.dtype).double().cpu()[routing.token.cpu()]
    w1, w2, b1 = server.w1_values.double().cpu(), server.w2_values.double().cpu(), layer.b1.double().cpu()
    y = torch.cat([torch.relu(chosen[b:e] @ w1[i].t() + b1[i]) @ w2[i].t()
                   for i, (b, e) in enumerate(zip(offsets, offsets[1:]))])
    want = torch.zeros(n, WIDTH, dtype=torch.double).index_add_(0, routing.token.cpu(),
                                                                y * routing.gate.double().cpu()[:, None])
    close(got, want, UNIT[layer.dtype], "y")


def test_training_lowers_the_loss(layer):
    x, routing, _ = tokens(300)
    teacher = E.Experts(EXPERTS, WIDTH, HIDDEN, layer.dtype, seed=5)
    target = routing.join(teacher.forward(x, routing)[0], 300)
    losses = [layer.step(x, target, routing, 4.0).item() for _ in range(20)]
    teacher.close()
    print(losses, flush=True)
    assert all(b < a for a, b in zip(losses, losses[1:]))
