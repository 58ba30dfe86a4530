"""The calls for layers of experts one after the other, as examples/expert_layer.py makes them: sorted,
dispatched, multiplied, combined, and back; and the same in 4-bit floats. Against the layer's formulas in
64 bits, and step by step against the oracle of 4-bit floats."""
import importlib.util
import os

import numpy as np
import pytest
import torch

import mxfp4_reference as Q
from ruy_amd import _structs as S
from ruy_amd import api

pytestmark = pytest.mark.gpu

_path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples", "expert_layer.py")
_spec = importlib.util.spec_from_file_location("expert_layer", _path)
E = importlib.util.module_from_spec(_spec)
_spec.loader.exec_module(E)

EXPERTS, WIDTH, HIDDEN, TOP = 6, 96, 160, 3
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


@pytest.fixture(params=[torch.bfloat16, torch.float16, torch.float32], ids=str)
def layer(request):
    layer = E.Experts(EXPERTS, WIDTH, HIDDEN, request.param, seed=3)
    layer.b1.normal_(generator=torch.Generator(device="cuda").manual_seed(4))
    yield layer
    torch.cuda.synchronize()
    layer.close()


def inputs(n):
    g = torch.Generator(device="cuda").manual_seed(n)
    x = torch.randn(n, WIDTH, generator=g, device="cuda")
    scores = torch.randn(n, EXPERTS, generator=g, device="cuda")
    scores[:, 4] = -100.0  # an expert that nobody goes to
    return x, scores, torch.randn(n, WIDTH, generator=g, device="cuda")


def close(got, want, unit, what):
    """Norms, as in test_gpu_expert_layer.py: a result has roundings of its own and of the up to 3 rounded values
    that it is formed from, each half a unit at most; a factor of 8 is given."""
    far = (got.double().cpu() - want).norm() / want.norm()
    print(what, "%.3g of %.3g" % (far, 8 * unit), flush=True)
    assert far <= 8 * unit


@pytest.mark.parametrize("n", [1, 37, 400])
def test_a_whole_step_and_its_gradients(layer, n):
    x, scores, grad = inputs(n)
    routing = E.Routing(scores, TOP)
    y, kept = layer.forward(x, routing)
    out = routing.join(y, n)
    grad_y, grad_gates = routing.join_gradients(grad, y)
    grad_chosen, grad_w1, grad_b1, grad_w2 = layer.backward(grad_y, kept, routing)
    grad_x = routing.dispatch_gradient(grad_chosen)
    # The formula, token by token and choice by choice.
    held = [t.to(layer.dtype).double().cpu().requires_grad_() for t in (x, layer.w1, layer.w2)]
    b1, gates = layer.b1.double().cpu().requires_grad_(), routing.gates.double().cpu().requires_grad_()
    choices = torch.topk(torch.softmax(scores.float(), dim=1), TOP, dim=1)[1].cpu()
    want = 0
    for j in range(TOP):
        w1, w2 = held[1][choices[:, j]], held[2][choices[:, j]]
        h = torch.relu((w1 @ held[0][:, :, None])[:, :, 0] + b1[choices[:, j]])
        want = want + gates[:, j:j + 1] * (w2 @ h[:, :, None])[:, :, 0]
    want.backward(grad.double().cpu())
    unit = UNIT[layer.dtype]
    close(out, want.detach(), unit, "y")
    for name, got, of in (("x", grad_x, held[0]), ("gates", grad_gates, gates), ("w1", grad_w1, held[1]), ("b1", grad_b1, b1),
                          ("w2", grad_w2, held[2])):
        close(got, of.grad, unit, name)


def quantized(rows):
    """The float64 values that rows of a device tensor are held as in 4 bits."""
    return torch.from_numpy(Q.values(*Q.quantize(rows.double().cpu().numpy())))


@pytest.mark.parametrize("n", [1, 4, 37, 400])
def test_answers_in_4_bit_floats(layer, n):
    x, scores, _ = inputs(n)
    routing = E.Routing(scores, TOP)
    server = E.FloatServer(layer)
    got = server.answer(x, routing)
    # Step by step on what the calls have to give: weights and tokens in 4 bits are the oracle's, bit for bit.
    w1, w2 = (quantized(w.reshape(-1, w.shape[2])).view(w.shape) for w in (layer.w1, layer.w2))
    assert torch.equal(server.values(server.w1).double().cpu(), w1) and torch.equal(server.values(server.w2).double().cpu(), w2)
    chosen = quantized(x.to(layer.dtype))[routing.token.cpu()]
    offsets = routing.offsets.tolist()
    # h is what the calls gave (a rounding of it that falls to the other side of a border of 4 bits is a step of them),
    held = server.tokens(x.to(layer.dtype).contiguous(), routing)
    h = torch.empty(TOP * n, HIDDEN, dtype=layer.dtype, device="cuda")
    api.mul_mxfp4(server.w1, held, E.params(layer.dtype, layer.b1, relu=True), layer.context, E.by_columns(h), routing.groups)
    b1 = layer.b1.double().cpu()
    want_h = torch.cat([torch.relu(chosen[b:e] @ w1[i].t() + b1[i]) for i, (b, e) in enumerate(zip(offsets, offsets[1:]))])
    close(h, want_h, UNIT[layer.dtype], "h")
    # and y that of the oracle's 4 bits of it.
    y = torch.cat([quantized(h)[b:e] @ w2[i].t() for i, (b, e) in enumerate(zip(offsets, offsets[1:]))])
    want = torch.zeros(n, WIDTH, dtype=torch.double).index_add_(0, routing.token.cpu(), y * routing.gate.double().cpu()[:, None])
    close(got, want, UNIT[layer.dtype], "y")


def test_padding_has_no_part_in_it():
    """A batch whose last tokens are padding (choices of -1): its answers are those without them, and padding's are zeros."""
    layer = E.Experts(EXPERTS, WIDTH, HIDDEN, torch.bfloat16, seed=3)
    x, scores, _ = inputs(50)
    routing = E.Routing(scores[:40], TOP)
    alone = routing.join(layer.forward(x[:40], routing)[0], 40)
    padded = E.Routing(scores, TOP)
    choices = torch.topk(torch.softmax(scores.float(), dim=1), TOP, dim=1)[1].contiguous()
    choices[40:] = -1
    api.sort_tokens(E.by_columns(choices), padded.routing, E.shared_context())
    assert padded.offsets[-1].item() == 40 * TOP and (padded.places[40:] == -1).all()
    x[40:] = float("nan")
    y, _ = layer.forward(x, padded)
    y[40 * TOP:] = float("nan")  # rows behind the last place
    joined = padded.join(y, 50)
    assert torch.equal(joined[:40], alone) and (joined[40:] == 0).all()
    layer.close()


def test_a_served_step_replayed_from_a_graph():
    """Sort, quantise into places, both products and the sum recorded once, replayed on other tokens and choices with eager
    work in between."""
    layer = E.Experts(EXPERTS, 512, 1024, torch.bfloat16, seed=3)
    server = E.FloatServer(layer)
    n, context = 24, api.Context()
    x = torch.zeros(n, 512, dtype=torch.bfloat16, device="cuda")
    choices = torch.zeros(n, 2, dtype=torch.int64, device="cuda")
    gates = torch.zeros(n, 2, device="cuda")

    def buffers():
        ints = dict(dtype=torch.int32, device="cuda")
        return dict(offsets=torch.zeros(EXPERTS + 1, **ints), places=torch.zeros(n, 2, **ints),
                    x4=server.empty(2 * n, 512), h=torch.zeros(2 * n, 1024, dtype=torch.bfloat16, device="cuda"),
                    h4=server.empty(2 * n, 1024), y=torch.zeros(2 * n, 512, dtype=torch.bfloat16, device="cuda"),
                    out=torch.zeros(n, 512, device="cuda"))

    def step(b):
        r = api.Routing(n, 2, EXPERTS, b["offsets"], b["places"])
        x4, h4 = api.MxFp4Matrix(2 * n, 512, *b["x4"]), api.MxFp4Matrix(2 * n, 1024, *b["h4"])
        api.sort_tokens(E.by_columns(choices), r, context)
        api.quantize_mxfp4(E.by_rows(x), context, x4, r)
        api.mul_mxfp4(server.w1, x4, E.params(x.dtype, layer.b1, relu=True), context, E.by_columns(b["h"]), r.groups())
        api.quantize_mxfp4(E.by_rows(b["h"]), context, h4)
        api.mul_mxfp4(server.w2, h4, E.params(x.dtype), context, E.by_columns(b["y"]), r.groups())
        api.combine_tokens(E.by_columns(b["y"]), r, E.by_columns(gates), context, E.by_columns(b["out"]))

    own, recorded = buffers(), buffers()
    torch.cuda.synchronize()
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    context.set_stream(stream.cuda_stream)
    with torch.cuda.graph(graph, stream=stream):
        step(recorded)
    context.set_stream(torch.cuda.current_stream().cuda_stream)
    rng = np.random.default_rng(0)
    for i in range(3):
        x.normal_()
        gates.uniform_()
        choices.copy_(torch.from_numpy(np.stack([rng.permutation(EXPERTS)[:2] for _ in range(n)])))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        step(own)
        torch.cuda.synchronize()
        assert own["out"].abs().sum() > 0 and torch.equal(own["out"], recorded["out"]), i
        assert torch.equal(own["offsets"], recorded["offsets"]) and torch.equal(own["places"], recorded["places"])
    context.close()
    layer.close()


def test_matrices_far_from_each_other():
    """Groups whose matrices and scales lie more than 2^32 bytes behind the first one's, on every kind of kernel."""
    context = api.Context()
    context.set_stream(torch.cuda.current_stream().cuda_stream)
    m, k, gap = 300, 512, (1 << 31) + 48
    rng = np.random.default_rng(0)
    data, scales = (torch.empty(2 * gap + m * k, dtype=torch.uint8, device="cuda") for _ in range(2))  # 4 GB each
    values = []
    for g in range(3):
        numbers = rng.integers(0, 16, (m, k), dtype=np.uint8)
        s = rng.integers(126, 129, (m, k // 32)).astype(np.uint8)
        data[g * gap:g * gap + m * k // 2] = torch.from_numpy(Q.pack(numbers)).flatten()
        scales[g * gap:g * gap + m * k // 32] = torch.from_numpy(s).flatten()
        values.append(torch.from_numpy(Q.values(numbers, s)).cuda())
    weights = api.MxFp4Matrix(m, k, data, scales, 0, 0, gap, gap)
    for n, tile in ((6, (16, 16)), (90, (64, 64)), (90, (64, 64, 1)), (300, (128, 128)), (700, (256, 256)), (6, None)):
        numbers = rng.integers(0, 16, (n, k), dtype=np.uint8)
        s = rng.integers(126, 129, (n, k // 32)).astype(np.uint8)
        x = api.MxFp4Matrix(n, k, torch.from_numpy(Q.pack(numbers)).cuda(), torch.from_numpy(s).cuda())
        offsets = torch.tensor([0, n // 3, n // 2, n], dtype=torch.int32, device="cuda")
        y = torch.zeros(n, m, device="cuda")
        context.force_tile(*(tile or (0, 0)))
        context.force_generic_kernel(tile is None)
        print("[case]", n, tile, flush=True)
        api.mul_mxfp4(weights, x, api.MulParams(S.F32, S.F32), context, api.Matrix(S.F32, y, api.Layout(m, n, m, api.Order.kColMajor)),
                      api.Groups(offsets, 3))
        xv = torch.from_numpy(Q.values(numbers, s)).cuda()
        for g, (b, e) in enumerate(((0, n // 3), (n // 3, n // 2), (n // 2, n))):
            assert torch.equal(y[b:e].double(), xv[b:e] @ values[g].t().contiguous())
    context.close()
