"""examples/expert_layer.py on another stream than the one its layer was made on:
all of a step is enqueued on torch's current stream."""
import pytest
import torch

from test_gpu_expert_steps import TOP, E, inputs, layer  # noqa: F401  (layer: a fixture)

pytestmark = pytest.mark.gpu


def step(layer, n):  # noqa: F811
    """Everything that a layer computes, trained and served."""
    x, scores, grad = inputs(n)
    routing = E.Routing(scores, TOP)
    y, kept = layer.forward(x, routing)
    out = routing.join(y, n)
    grad_y, grad_gates = routing.join_gradients(grad, y)
    gradients = layer.backward(grad_y, kept, routing)
    served = E.Server(layer, 32).answer(x, routing)
    floats = E.FloatServer(layer).answer(x, routing)
    return [out, grad_y, grad_gates, routing.dispatch_gradient(gradients[0]), *gradients, served, floats]


def test_a_step_on_another_stream_waits_for_nothing_on_the_first(layer):  # noqa: F811
    want = step(layer, 40)
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    with torch.cuda.stream(other):
        step(layer, 40)  # (what is made once to a stream, its contexts, is there)
    a, b = torch.randn(2, 8192, 8192, device="cuda").unbind()
    torch.cuda.synchronize()
    for _ in range(20):  # some hundred milliseconds on the layer's own stream
        torch.mm(a, b)
    with torch.cuda.stream(other):
        got = step(layer, 40)
    other.synchronize()
    # What the other stream has computed is there, whatever the first one is still at.
    with torch.cuda.stream(other):
        same = [bool(torch.equal(g, w)) for g, w in zip(got, want)]
    torch.cuda.synchronize()
    assert all(same), same
