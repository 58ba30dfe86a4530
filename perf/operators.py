"""The workloads by which the speed of the products for expert layers is judged.

Three kinds of pass, the ones that a mixture-of-experts layer is trained and
served with:

  grouped    every token against the weights of its own expert
             (`ruy_amd.api.mul_grouped`), with an optional bias and ReLU;
  gradients  that product's backward pass: the gradient of the tokens
             (`mul_grouped` with the weights transposed) and of every expert's
             weights (`mul_grouped_depth`);
  int4       a few tokens against weights of 4 bits with a scale, and where the
             case has them a zero point, to every group of depth positions
             (`mul_int4`), one weight matrix or one to each expert.

Tokens lie one behind the other, sorted by expert; the first token of each
expert is in device memory, as a router leaves it there. A weight matrix has a
row to each output. `listed()` names twelve passes and `draw()` gives more of
the same ranges.
"""
import functools
import math

import torch

own = False  # True: run() calls the library, False: the plain form

_TORCH = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}


def _case(name, op, type_, experts, m, k, tokens, **options):
    """m x k weights for each of `experts` (0: one matrix, no groups), `tokens`
    tokens in all. skew: expert number i gets tokens in proportion to
    1 / (i + 1) ** skew. pad: values between one token and the next."""
    case = {"op": op, "type": type_, "experts": experts, "m": m, "k": k, "tokens": tokens, "skew": 0.0, "pad": 0}
    if op == "grouped":
        case["relu"] = False  # with a bias
    elif op == "gradients":
        case["weights_f32"] = False  # the weights' gradients in 32 bits
    else:
        case.update(group=128, zeros=False)
    case.update(options)
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # One token, sent to two of a small layer's eight experts: latency.
        _case("grouped one token", "grouped", "bf16", 8, 1024, 1024, 2),
        # A decoding step: 16 requests, two experts each, most experts idle or with a token or two.
        _case("grouped decode", "grouped", "f16", 64, 2048, 2048, 32, skew=0.8),
        # A long prompt through a layer of eight large experts.
        _case("grouped prefill", "grouped", "bf16", 8, 4096, 2048, 8192, skew=0.5),
        # Sizes that nothing divides, a few crowded experts and many with hardly a token.
        _case("grouped ragged", "grouped", "f16", 20, 1000, 1111, 3001, skew=1.2, relu=True, pad=3),
        # The library's own floating type.
        _case("grouped f32", "grouped", "f32", 4, 1024, 1024, 1500, skew=0.5, relu=True),
        # A training step of a large layer; the optimizer adds the weights' gradients up in 32 bits.
        _case("gradients large", "gradients", "bf16", 8, 2048, 4096, 8192, skew=0.5, weights_f32=True),
        # Many small experts of odd sizes, some without a token.
        _case("gradients ragged", "gradients", "f16", 48, 515, 771, 2500, skew=1.2),
        # One token through the largest layer of this repository's benchmark, the weights in 4 bits.
        _case("int4 16384", "int4", "f16", 0, 16384, 16384, 1),
        # One token through a small layer: latency.
        _case("int4 2048", "int4", "bf16", 0, 2048, 2048, 1, group=64),
        # A batch of requests that each decode a token.
        _case("int4 batch", "int4", "bf16", 0, 8192, 4096, 48, zeros=True),
        # 32-bit tokens, odd sizes, a last group that is cut short.
        _case("int4 f32 ragged", "int4", "f32", 0, 1000, 2051, 3, group=32, zeros=True, pad=1),
        # The decoding step again, its experts in 4 bits.
        _case("int4 experts", "int4", "bf16", 64, 2048, 2048, 32, group=32, skew=0.8),
    ]


# No drawn pass computes or reads more than the largest listed ones do.
_MOST_FLOPS = {"grouped": 1.3e11, "gradients": 2.7e11, "int4": 1.5e10}
_MOST_WEIGHTS = {"grouped": 1 << 27, "gradients": 1 << 26, "int4": 1 << 28}


def _spread(rng, lo, hi):
    """A size spread over the logarithm of [lo, hi]; every other one is a
    multiple of 64 as layers mostly have them, the rest are as they fall."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5:
        v = (v + 63) // 64 * 64
    return max(lo, min(hi, v))


def draw(rng):
    op = rng.choice(["grouped", "grouped", "gradients", "int4", "int4"])
    type_ = rng.choice(["bf16", "bf16", "f16", "f16", "f32"])
    o = {"pad": rng.choice([0, 0, 0, 1, 8])}
    if op == "int4":
        experts = rng.choice([0, 0, 8, 64])
        m, k = _spread(rng, 256, 16384), _spread(rng, 256, 16384)
        tokens = 1 if rng.random() < 0.4 else _spread(rng, 1, 64)
        o.update(group=rng.choice([32, 64, 128]), zeros=rng.random() < 0.5)
    else:
        experts = rng.choice([1, 4, 8, 16, 33, 64])
        m, k = _spread(rng, 128, 4096), _spread(rng, 128, 4096)
        few = op == "grouped" and rng.random() < 0.4
        tokens = rng.randint(1, 64) if few else _spread(rng, 256, 8192)
        if op == "grouped":
            o["relu"] = rng.random() < 0.5
        else:
            o["weights_f32"] = rng.random() < 0.5
    if experts:
        o["skew"] = rng.choice([0.0, 0.5, 1.0, 1.5])
    while max(experts, 1) * m * k > _MOST_WEIGHTS[op]:
        m = (m + 1) // 2
    # (32-bit products run at a fraction of the others' rate.)
    most = _MOST_FLOPS[op] / (8 if type_ == "f32" and op != "int4" else 1)
    passes = 4 if op == "gradients" else 2
    while passes * m * k * tokens > most:
        tokens = (tokens + 1) // 2
    return _case("", op, type_, experts, m, k, tokens, **o)


def _counts(case):
    """Tokens to each expert, the most frequent first: token number i goes to
    the expert in which (i + 1/2) / tokens lies of the summed-up shares."""
    shares = [(i + 1.0) ** -case["skew"] for i in range(case["experts"])]
    total, at, sums = sum(shares), 0.0, []
    for s in shares:
        at += s / total
        sums.append(at)
    counts, expert = [0] * len(shares), 0
    for i in range(case["tokens"]):
        while expert + 1 < len(shares) and (i + 0.5) / case["tokens"] > sums[expert]:
            expert += 1
        counts[expert] += 1
    return counts


def _rows(g, rows, cols, pad, type_, scale):
    """rows x cols values of normal distribution, `pad` unused ones behind each row."""
    x = torch.randn(rows, cols + pad, generator=g, device=g.device).mul_(scale).to(_TORCH[type_])
    return x[:, :cols]


def prepare(case, seed):
    c, g = case, torch.Generator(device="cuda")
    g.manual_seed(seed)
    m, k, tokens, matrices = c["m"], c["k"], c["tokens"], max(c["experts"], 1)
    s = {"case": c}
    if c["experts"]:
        # (Which expert is the frequent one is another matter for each seed.)
        counts = _counts(c)
        order = torch.randperm(c["experts"], generator=torch.Generator().manual_seed(seed)).tolist()
        s["counts"] = [counts[i] for i in order]
        s["offsets"] = torch.tensor([0] + s["counts"], device="cuda").cumsum(0).to(torch.int32)
    s["x"] = _rows(g, tokens, k, c["pad"], c["type"], 1.0)
    # A few channels of a layer's input are much larger than the others.
    s["x"][:, torch.randint(k, (1 + k // 256,), generator=g, device="cuda")] *= 16
    if c["op"] == "int4":
        groups = -(-k // c["group"])
        s["w"] = torch.randint(256, (matrices, m, -(-k // 2)), generator=g, device="cuda", dtype=torch.uint8)
        scales = torch.rand(matrices, m, groups, generator=g, device="cuda").add_(0.5).mul_(0.2 / math.sqrt(k))
        s["scales"] = scales.to(_TORCH[c["type"]])
        s["zeros"] = None
        if c["zeros"]:
            s["zeros"] = torch.randint(5, 12, scales.shape, generator=g, device="cuda", dtype=torch.uint8)
        s["y"] = torch.zeros(tokens, m, device="cuda", dtype=_TORCH[c["type"]])
        return s
    s["w"] = _rows(g, matrices * m, k, 0, c["type"], 1 / math.sqrt(k)).view(matrices, m, k)
    if c["op"] == "grouped":
        s["bias"] = torch.randn(matrices, m, generator=g, device="cuda").mul_(0.2) if c["relu"] else None
        s["y"] = torch.zeros(tokens, m, device="cuda", dtype=_TORCH[c["type"]])
    else:
        s["dy"] = _rows(g, tokens, m, c["pad"], c["type"], 0.05)
        s["dx"] = torch.zeros(tokens, k, device="cuda", dtype=_TORCH[c["type"]])
        s["dw"] = torch.zeros(matrices, m, k, device="cuda",
                              dtype=torch.float32 if c["weights_f32"] else _TORCH[c["type"]])
    return s


# ---- The plain form: 32 bits throughout, rounded once at the end ----

def _values_of_int4(w, scales, zeros, k, group):
    """(q - zero point) * scale of matrices of 4-bit values, two to a byte."""
    q = torch.stack((w & 15, w >> 4), -1).flatten(-2)[..., :k].float()
    z = zeros.float().repeat_interleave(group, -1)[..., :k] if zeros is not None else 8.0
    return (q - z) * scales.float().repeat_interleave(group, -1)[..., :k]


def _plain_grouped(s):
    c = s["case"]
    parts = [x.float() @ s["w"][e].float().t() + (s["bias"][e] if c["relu"] else 0.0)
             for e, x in enumerate(s["x"].split(s["counts"])) if len(x)]
    y = torch.cat(parts)
    return (y.clamp_min_(0.0) if c["relu"] else y).to(s["y"].dtype)


def _plain_gradients(s):
    dys, xs = s["dy"].split(s["counts"]), s["x"].split(s["counts"])
    dx = torch.cat([dy.float() @ s["w"][e].float() for e, dy in enumerate(dys) if len(dy)])
    dw = torch.stack([dy.float().t() @ x.float() for dy, x in zip(dys, xs)])
    return {"dx": dx.to(s["dx"].dtype), "dw": dw.to(s["dw"].dtype)}


def _plain_int4(s):
    c = s["case"]
    parts = [x.float() @ _values_of_int4(s["w"][e], s["scales"][e], None if s["zeros"] is None else s["zeros"][e],
                                         c["k"], c["group"]).t()
             for e, x in enumerate(s["x"].split(s.get("counts", [c["tokens"]]))) if len(x)]
    return torch.cat(parts).to(s["y"].dtype)


# ---- The library's ----

@functools.lru_cache(None)
def _library():
    """The package and this program's context: it launches on torch's stream
    and its calls return once they are enqueued."""
    from ruy_amd import _structs, api
    context = api.Context()
    context.set_stream(torch.cuda.current_stream().cuda_stream)
    context.set_synchronous(False)
    return api, {"bf16": _structs.BF16, "f16": _structs.F16, "f32": _structs.F32}, context


def _calls(s):
    """The calls of a pass with their arguments: the descriptors of buffers that
    a program makes once and keeps with them."""
    api, types, context = _library()
    c, kinds = s["case"], {_TORCH[name]: types[name] for name in types}
    by_rows, by_cols = api.Order.kRowMajor, api.Order.kColMajor

    def matrix(t, rows, cols, order):
        """`t`: a tensor with a row (by_rows) or a column to each of its first index."""
        return api.Matrix(kinds[t.dtype], t, api.Layout(rows, cols, t.stride(-2), order))

    def params(t, relu=False):
        p = api.MulParams(types["f32"], kinds[t.dtype])
        if relu:
            p.set_bias(s["bias"])
            p.set_clamp_min(0.0)
        return p

    m, k, tokens = c["m"], c["k"], c["tokens"]
    groups = api.Groups(s["offsets"], c["experts"]) if c["experts"] else None
    if c["op"] == "int4":
        weights = api.Int4Matrix(m, k, c["group"], s["w"], s["scales"], kinds[s["scales"].dtype], s["zeros"])
        return [(api.mul_int4, (weights, matrix(s["x"], k, tokens, by_cols), params(s["y"]), context,
                                matrix(s["y"], m, tokens, by_cols), groups))], s["y"]
    if c["op"] == "grouped":
        return [(api.mul_grouped, (matrix(s["w"], m, k, by_rows), matrix(s["x"], k, tokens, by_cols), groups,
                                   params(s["y"], c["relu"]), context, matrix(s["y"], m, tokens, by_cols)))], s["y"]
    dy = matrix(s["dy"], m, tokens, by_cols)
    return [(api.mul_grouped, (matrix(s["w"], k, m, by_cols), dy, groups, params(s["dx"]), context,
                               matrix(s["dx"], k, tokens, by_cols))),
            (api.mul_grouped_depth, (dy, matrix(s["x"], tokens, k, by_rows), groups, params(s["dw"]), context,
                                     matrix(s["dw"], m, k, by_rows)))], {"dx": s["dx"], "dw": s["dw"]}


def run(state):
    if not own:
        return {"grouped": _plain_grouped, "gradients": _plain_gradients, "int4": _plain_int4}[state["case"]["op"]](state)
    if "calls" not in state:
        state["calls"] = _calls(state)
    calls, outputs = state["calls"]
    for call, arguments in calls:
        call(*arguments)
    return outputs


def work(case):
    c = case
    m, k, tokens, size = c["m"], c["k"], c["tokens"], _BYTES[c["type"]]
    reached = sum(n > 0 for n in _counts(c)) if c["experts"] else 1
    flops = 2.0 * tokens * m * k
    count = tokens * (k + m) * size
    if c["op"] == "int4":
        count += reached * m * (-(-k // 2) + -(-k // c["group"]) * (size + c["zeros"]))
    elif c["op"] == "grouped":
        count += reached * m * (k * size + 4 * c["relu"])
    else:
        flops *= 2
        count += tokens * k * size + reached * m * k * size
        count += c["experts"] * m * k * (4 if c["weights_f32"] else size)
    return {"bytes": float(count), "flops": flops}


def exact(case, seed):
    """From the definition, in 64 bits, expert by expert."""
    c, s = case, prepare(case, seed)
    bounds = [0, c["tokens"]] if not c["experts"] else s["offsets"].tolist()
    x = s["x"].double()
    if c["op"] == "gradients":
        dy = s["dy"].double()
        dx, dw = torch.zeros_like(s["dx"], dtype=torch.float64), torch.zeros_like(s["dw"], dtype=torch.float64)
        for e in range(c["experts"]):
            at = slice(bounds[e], bounds[e + 1])
            dx[at] = torch.matmul(dy[at], s["w"][e].double())
            dw[e] = torch.matmul(dy[at].t().contiguous(), x[at])
        return {"dx": dx, "dw": dw}
    y = torch.zeros_like(s["y"], dtype=torch.float64)
    for e in range(len(bounds) - 1):
        at = slice(bounds[e], bounds[e + 1])
        if at.start == at.stop:
            continue
        if c["op"] == "int4":
            k = torch.arange(c["k"], device="cuda")
            q = (s["w"][e][:, k // 2].int() >> (4 * (k % 2)).int()) & 15
            zero = 8 if s["zeros"] is None else s["zeros"][e][:, k // c["group"]].int()
            w = (q - zero).double() * s["scales"][e][:, k // c["group"]].double()
        else:
            w = s["w"][e].double()
        y[at] = torch.matmul(x[at], w.t())
        if c.get("relu"):
            y[at] = torch.clamp(y[at] + s["bias"][e].double(), min=0.0)
    return y
