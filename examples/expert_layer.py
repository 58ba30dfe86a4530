"""A layer of experts, trained and then served, on the grouped and 4-bit products.

Every token goes to `top` of the experts, y = sum over them of gate * W2 relu(W1 x + b):

  python examples/expert_layer.py [--experts 16] [--width 512] [--hidden 1024] [--tokens 2048]

Training: the tokens are put in the order of their experts once a step; W1, W2 and both
gradients of either are then one product each (ruyamd_mul_grouped with the weights
as they lie, and transposed; ruyamd_mul_grouped_depth), whatever the experts' shares are.
The offsets stay on the device: nothing in a step waits for it. Serving: the weights
in 4 bits, a scale and a zero point to every 64 of a row (ruyamd_mul_int4), a few
tokens at a time.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
from ruy_amd import _structs as S  # noqa: E402
from ruy_amd import api  # noqa: E402

DTYPES = {torch.bfloat16: S.BF16, torch.float16: S.F16, torch.float32: S.F32}


def by_columns(t):
    """The tokens t[i] as the columns of a matrix."""
    return api.Matrix(DTYPES[t.dtype], t, api.make_simple_layout(t.shape[1], t.shape[0], api.Order.kColMajor))


def by_rows(t):
    return api.Matrix(DTYPES[t.dtype], t, api.make_simple_layout(t.shape[-2], t.shape[-1], api.Order.kRowMajor))


def params(dtype, bias=None, relu=False):
    p = api.MulParams(S.F32, DTYPES[dtype])
    p.set_bias(bias)
    if relu:
        p.set_clamp_min(0.0)
    return p


class Routing:
    """Which expert each of a batch's tokens goes to, in the order of the experts."""

    def __init__(self, scores, top):
        gate, expert = torch.topk(torch.softmax(scores.float(), dim=1), top, dim=1)
        experts = scores.shape[1]
        order = torch.argsort(expert.flatten(), stable=True)
        self.token = order // top
        self.gate = gate.flatten()[order]
        edges = torch.arange(experts + 1, device=scores.device)
        self.offsets = torch.searchsorted(expert.flatten()[order].contiguous(), edges).int()
        self.groups = api.Groups(self.offsets, experts)

    def join(self, y, count):
        """The experts' answers to each of `count` tokens, weighted and added up."""
        out = torch.zeros(count, y.shape[1], dtype=torch.float32, device=y.device)
        return out.index_add_(0, self.token, y.float() * self.gate[:, None])


class Experts:
    def __init__(self, experts, width, hidden, dtype=torch.bfloat16, seed=0):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        self.dtype = dtype
        self.w1 = torch.randn(experts, hidden, width, generator=g, device="cuda") * (2.0 / width) ** 0.5
        self.w2 = torch.randn(experts, width, hidden, generator=g, device="cuda") / hidden ** 0.5
        self.b1 = torch.zeros(experts, hidden, device="cuda")
        self.context = api.Context()
        self.context.set_stream(torch.cuda.current_stream().cuda_stream)
        self.context.set_synchronous(False)

    def close(self):
        self.context.close()

    def forward(self, x, routing):
        """The experts' answers, one row to each token and expert it goes to."""
        w1, w2 = self.w1.to(self.dtype), self.w2.to(self.dtype)
        chosen = x.to(self.dtype)[routing.token]
        n = chosen.shape[0]
        h = torch.empty(n, w1.shape[1], dtype=self.dtype, device="cuda")
        y = torch.empty(n, w2.shape[1], dtype=self.dtype, device="cuda")
        api.mul_grouped(by_rows(w1), by_columns(chosen), routing.groups, params(self.dtype, self.b1, relu=True),
                        self.context, by_columns(h))
        api.mul_grouped(by_rows(w2), by_columns(h), routing.groups, params(self.dtype), self.context, by_columns(y))
        return y, (chosen, h, w1, w2)

    def backward(self, grad_y, kept, routing):
        """From the gradient of the experts' answers those of chosen tokens, w1, b1 and w2."""
        chosen, h, w1, w2 = kept
        grad_y = grad_y.to(self.dtype)
        grad_h, grad_x = torch.empty_like(h), torch.empty_like(chosen)
        grad_w1 = torch.empty(w1.shape, device="cuda")
        grad_w2 = torch.empty(w2.shape, device="cuda")
        grad_b1 = torch.empty(w1.shape[0], w1.shape[1], 1, device="cuda")
        ones = torch.ones(chosen.shape[0], 1, dtype=self.dtype, device="cuda")

        def transposed(w):  # the same memory, read by columns
            return api.Matrix(DTYPES[w.dtype], w, api.make_simple_layout(w.shape[2], w.shape[1], api.Order.kColMajor))

        wide, plain = params(torch.float32), params(self.dtype)
        api.mul_grouped_depth(by_columns(grad_y), by_rows(h), routing.groups, wide, self.context, by_rows(grad_w2))
        api.mul_grouped(transposed(w2), by_columns(grad_y), routing.groups, plain, self.context, by_columns(grad_h))
        grad_h *= h > 0
        api.mul_grouped_depth(by_columns(grad_h), by_rows(chosen), routing.groups, wide, self.context, by_rows(grad_w1))
        api.mul_grouped_depth(by_columns(grad_h), by_rows(ones), routing.groups, wide, self.context, by_rows(grad_b1))
        api.mul_grouped(transposed(w1), by_columns(grad_h), routing.groups, plain, self.context, by_columns(grad_x))
        return grad_x, grad_w1, grad_b1[:, :, 0], grad_w2

    def step(self, x, target, routing, rate):
        """One step of gradient descent on the mean squared error; the loss before it."""
        y, kept = self.forward(x, routing)
        error = routing.join(y, x.shape[0]) - target
        grad_y = (error * (2.0 / error.numel()))[routing.token] * routing.gate[:, None]
        _, grad_w1, grad_b1, grad_w2 = self.backward(grad_y, kept, routing)
        self.w1 -= rate * grad_w1
        self.b1 -= rate * grad_b1
        self.w2 -= rate * grad_w2
        return error.square().mean()


def quantize(w, group_size=64):
    """4-bit weights (experts, rows, cols): an Int4Matrix, and the values it stands for."""
    experts, rows, cols = w.shape
    if cols % group_size:
        raise ValueError("the depth must be a multiple of the group size")
    parts = w.view(experts, rows, cols // group_size, group_size)
    low, high = parts.amin(3).clamp(max=0), parts.amax(3).clamp(min=0)
    scale = ((high - low) / 15).clamp(min=1e-8).to(torch.bfloat16)
    zero = torch.round(-low / scale.float()).clamp(0, 15)
    q = torch.round(parts / scale.float()[..., None] + zero[..., None]).clamp(0, 15)
    values = ((q - zero[..., None]) * scale.float()[..., None]).view(w.shape)
    q = q.to(torch.uint8).view(experts, rows, cols)
    data = q[..., 0::2] | q[..., 1::2] << 4
    return api.Int4Matrix(rows, cols, group_size, data, scale, S.BF16, zero.to(torch.uint8)), values


class Server:
    """The trained experts in 4 bits."""

    def __init__(self, trained, group_size=64):
        self.dtype, self.context, self.b1 = trained.dtype, trained.context, trained.b1
        self.w1, self.w1_values = quantize(trained.w1, group_size)
        self.w2, self.w2_values = quantize(trained.w2, group_size)

    def answer(self, x, routing):
        chosen = x.to(self.dtype)[routing.token]
        n = chosen.shape[0]
        h = torch.empty(n, self.w1.rows, dtype=self.dtype, device="cuda")
        y = torch.empty(n, self.w2.rows, dtype=self.dtype, device="cuda")
        api.mul_int4(self.w1, by_columns(chosen), params(self.dtype, self.b1, relu=True), self.context, by_columns(h),
                     routing.groups)
        api.mul_int4(self.w2, by_columns(h), params(self.dtype), self.context, by_columns(y), routing.groups)
        return routing.join(y, x.shape[0])


def main():
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--experts", type=int, default=16)
    parser.add_argument("--width", type=int, default=512)
    parser.add_argument("--hidden", type=int, default=1024)
    parser.add_argument("--tokens", type=int, default=2048)
    parser.add_argument("--top", type=int, default=2)
    parser.add_argument("--steps", type=int, default=30)
    args = parser.parse_args()
    torch.manual_seed(0)
    teacher = Experts(args.experts, args.width, args.hidden, seed=1)
    layer = Experts(args.experts, args.width, args.hidden, seed=2)
    router = torch.randn(args.width, args.experts, device="cuda") / args.width ** 0.5
    x = torch.randn(args.tokens, args.width, device="cuda")
    routing = Routing(x @ router, args.top)
    target = routing.join(teacher.forward(x, routing)[0], args.tokens)
    rate = 0.005 * args.width * args.experts
    for i in range(args.steps):
        loss = layer.step(x, target, routing, rate)
        if i % 10 == 0 or i == args.steps - 1:
            print("step %d: loss %.4f" % (i, loss.item()))
    server = Server(layer)
    few = x[:3]
    routing = Routing(few @ router, args.top)
    y, wanted = server.answer(few, routing), routing.join(layer.forward(few, routing)[0], 3)
    print("4 bits, 3 tokens: %.3f of the answers' norm away from those of 16 bits" % ((y - wanted).norm() / wanted.norm()))
    layer.close()
    teacher.close()


if __name__ == "__main__":
    main()
