"""The workloads by which the speed of what surrounds the experts' products is judged.

Five kinds of pass, the ones that a mixture-of-experts layer is trained and
served with beside the products of `operators.py`:

  route      the router's choices sorted by expert (`ruy_amd.api.sort_tokens`)
             and every token copied to its places (`dispatch_tokens`);
  combine    the experts' answers to each token, weighted and added up
             (`combine_tokens`);
  gradients  the backward pass of both: of the answers and the weights
             (`combine_tokens_gradients`), and of the tokens (`combine_tokens`);
  quantize   values to 4-bit floats with a power of two to every 32 of a row,
             each token to its places where the case has them
             (`quantize_mxfp4`), and what they stand for (`dequantize_mxfp4`);
  mxfp4      products of two such matrices (`mul_mxfp4`), one weight matrix or
             one to each expert.

Tokens are rows of tensors. A choice that is no expert, as of a batch's padding,
has no place; rows behind the last place stay as they are. `listed()` names
twelve passes and `draw()` gives more of the same ranges.
"""
import functools
import math

import numpy as np
import torch

own = False  # True: run() calls the library, False: the plain form

_TORCH = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}
_BLOCK = 32  # values to a power of two


def _case(name, op, type_, tokens, **options):
    """tokens: rows of the pass's input. experts, top: each token chooses `top`
    of them (top 0: none has a place). skew: expert number i is chosen in
    proportion to 1 / (i + 1) ** skew. drop: every so manieth token is padding.
    pad: values (bytes of 4-bit rows) between one row and the next."""
    case = {"op": op, "type": type_, "tokens": tokens, "experts": 0, "skew": 0.0, "pad": 0}
    if op == "mxfp4":
        case.update(m=0, k=0, relu=False)  # m x k weights to each expert (experts 0: one matrix); with a bias
    else:
        case.update(width=0, top=0, drop=0)
    case.update(options)
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # A decoding step: 16 requests, two experts each: latency.
        _case("route decode", "route", "f16", 16, width=2048, experts=64, top=2, skew=0.8),
        # Long prompts through a wide layer of many experts, some of the batch padding.
        _case("route prefill", "route", "bf16", 8192, width=4096, experts=64, top=4, skew=0.5, drop=16),
        # The decoding step's answers.
        _case("combine decode", "combine", "bf16", 16, width=2048, experts=64, top=2, skew=0.8),
        # A prompt's answers.
        _case("combine prefill", "combine", "f16", 8192, width=4096, experts=8, top=2, skew=0.5),
        # A training step of a large layer.
        _case("gradients large", "gradients", "bf16", 8192, width=4096, experts=8, top=2, skew=0.5),
        # Many small experts of an odd width, in 32 bits, with padding.
        _case("gradients ragged", "gradients", "f32", 2500, width=771, experts=48, top=6, skew=1.2, drop=7, pad=3),
        # A prompt's tokens on their way to the experts in 4 bits.
        _case("quantize prefill", "quantize", "bf16", 8192, width=4096, experts=8, top=2, skew=0.5),
        # A small layer's weights of odd sizes: a last block that is cut short.
        _case("quantize ragged", "quantize", "f32", 1000, width=1111, pad=1),
        # One token through the largest layer of this repository's benchmark.
        _case("mxfp4 16384", "mxfp4", "f16", 1, m=16384, k=16384),
        # The decoding step through experts in 4 bits.
        _case("mxfp4 decode", "mxfp4", "bf16", 32, m=2048, k=2048, experts=64, skew=0.8),
        # A long prompt through a layer of eight large experts.
        _case("mxfp4 prefill", "mxfp4", "bf16", 8192, m=4096, k=2048, experts=8, skew=0.5, relu=True),
        # The size of this repository's headline product.
        _case("mxfp4 8192", "mxfp4", "bf16", 8192, m=8192, k=8192),
    ]


# No drawn pass moves or computes more than the largest listed ones do.
_MOST_VALUES = 1 << 27
_MOST_WEIGHTS = 1 << 28
_MOST_FLOPS = 1.1e12


def _spread(rng, lo, hi):
    """A size spread over the logarithm of [lo, hi]; every other one is a
    multiple of 64 as layers mostly have them, the rest are as they fall."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5:
        v = (v + 63) // 64 * 64
    return max(lo, min(hi, v))


def draw(rng):
    op = rng.choice(["route", "combine", "gradients", "quantize", "mxfp4", "mxfp4"])
    type_ = rng.choice(["bf16", "bf16", "f16", "f16", "f32"])
    o = {"pad": rng.choice([0, 0, 0, 1, 8])}
    tokens = rng.randint(1, 64) if rng.random() < 0.4 else _spread(rng, 64, 16384)
    if op == "mxfp4":
        o["experts"] = rng.choice([0, 0, 8, 64])
        m, k = _spread(rng, 128, 16384), _spread(rng, 128, 16384)
        if rng.random() < 0.6:  # (layers have whole blocks, mostly)
            k = max(k // _BLOCK, 1) * _BLOCK
        while max(o["experts"], 1) * m * k > _MOST_WEIGHTS:
            m = (m + 1) // 2
        while 2.0 * m * k * tokens > _MOST_FLOPS or m * tokens > _MOST_VALUES:
            tokens = (tokens + 1) // 2
        o.update(m=m, k=k)
        if o["experts"]:
            o.update(skew=rng.choice([0.0, 0.5, 1.0, 1.5]), relu=rng.random() < 0.5)
        return _case("", op, type_, tokens, **o)
    o["width"] = _spread(rng, 64, 8192)
    if op != "quantize" or rng.random() < 0.5:
        o.update(experts=rng.choice([8, 16, 33, 64, 256]), top=rng.randint(1, 8), skew=rng.choice([0.0, 0.5, 1.0]),
                 drop=rng.choice([0, 0, 3, 16]))
    while tokens * max(o.get("top", 1), 1) * o["width"] > _MOST_VALUES:
        tokens = (tokens + 1) // 2
    return _case("", op, type_, tokens, **o)


def _counts(case):
    """Tokens to each expert of a product, the most frequent first: token number i
    goes to the expert in which (i + 1/2) / tokens lies of the summed-up shares."""
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


def _layer_input(g, rows, cols, pad, type_):
    """A layer's input: a few channels are much larger than the others."""
    x = _rows(g, rows, cols, pad, type_, 1.0)
    x[:, torch.randint(cols, (1 + cols // 256,), generator=g, device="cuda")] *= 16
    return x


def _choices(g, c):
    """What a router leaves: `top` different experts to each token, the likeliest
    first, their weights, and -1 for each choice of a token of padding."""
    likely = -torch.arange(1, c["experts"] + 1, device="cuda").double().log() * c["skew"]
    noise = torch.rand(c["tokens"], c["experts"], generator=g, device="cuda", dtype=torch.float64)
    scores = likely[torch.randperm(c["experts"], generator=g, device="cuda")] - (-noise.clamp_min(1e-300).log()).log()
    best, experts = scores.topk(c["top"], dim=1)
    if c["drop"]:
        experts[c["drop"] - 1::c["drop"]] = -1
    return experts.contiguous(), torch.softmax(best, dim=1).float().contiguous()


def _plain_sort(experts, count):
    """(offsets, places, sources) of int64 choices."""
    flat = experts.flatten()
    key = torch.where((flat >= 0) & (flat < count), flat, count)
    order = torch.argsort(key, stable=True)
    reached = torch.searchsorted(key[order], torch.arange(count + 1, device=flat.device))
    places = torch.empty_like(order)
    places[order] = torch.arange(len(order), device=flat.device)
    places = torch.where(key < count, places, -1)
    sources = torch.where(torch.arange(len(order), device=flat.device) < reached[-1], order, -1)
    return reached.int(), places.int().view_as(experts), sources.int()


# ---- 4-bit floats: eight magnitudes and a sign, a power of two to a block ----

def _in_blocks(x, fill=0):
    """rows x cols values as rows x blocks x 32."""
    short = -x.shape[1] % _BLOCK
    if short:
        x = torch.nn.functional.pad(x, (0, short), value=fill)
    return x.unflatten(1, (-1, _BLOCK))


def _power(exponent, type_=torch.float32):
    """2 ** exponent, exactly, of whole numbers -126 .. 127."""
    return ((exponent + 127) << 23).int().view(torch.float32).to(type_)


def _plain_quantize(x):
    """Numbers 0 .. 15 for the values of the rows x cols x, and a scale's exponent to each block."""
    blocks = _in_blocks(x.float())
    exponent = (torch.frexp(blocks.abs().amax(2))[1] - 3).clamp_(-127, 127)
    exponent = torch.where(blocks.abs().amax(2) > 0, exponent, -127).int()
    size = (blocks * _power(-exponent)[..., None]).abs()
    step = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0))
    size = (size / step).round_().mul_(step).clamp_(max=6)
    number = torch.where(size < 2, size * 2, torch.where(size < 4, size + 2, size / 2 + 4)).to(torch.uint8)
    number += torch.signbit(blocks).to(torch.uint8) * 8
    return number.flatten(1)[:, :x.shape[1]], exponent


def _packed(number):
    """Two numbers to a byte, the first one low."""
    if number.shape[1] % 2:
        number = torch.nn.functional.pad(number, (0, 1))
    return number[:, 0::2] | number[:, 1::2] << 4


@functools.lru_cache(None)
def _magnitudes():
    half = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device="cuda")
    return torch.cat((half, -half))


def _plain_values(number, exponent):
    """What rows x cols numbers and their blocks' exponents stand for, in 32 bits."""
    blocks = _in_blocks(_magnitudes()[number.int()])
    # (2 ** -127 has no exponent of its own in 32 bits.)
    low = exponent < -126
    values = blocks * _power(torch.where(low, exponent + 1, exponent))[..., None]
    return torch.where(low[..., None], values * 0.5, values).flatten(1)[:, :number.shape[1]]


def _unpacked(data, cols):
    return torch.stack((data & 15, data >> 4), -1).flatten(-2)[..., :cols]


def _four_bits(g, rows, cols, pad, x):
    """x (rows x cols) as a program keeps it: bytes of two values, `pad` unused ones
    behind each row, and bytes of scales."""
    number, exponent = _plain_quantize(x)
    data = torch.randint(256, (rows, (cols + 1) // 2 + pad), generator=g, device="cuda", dtype=torch.uint8)
    data[:, :(cols + 1) // 2] = _packed(number)
    return data, (exponent + 127).to(torch.uint8)


def prepare(case, seed):
    c, g = case, torch.Generator(device="cuda")
    g.manual_seed(seed)
    tokens, type_, s = c["tokens"], c["type"], {"case": case}
    if c["op"] == "mxfp4":
        m, k, matrices = c["m"], c["k"], max(c["experts"], 1)
        if c["experts"]:
            # (Which expert is the frequent one is another matter for each seed.)
            counts = _counts(c)
            order = torch.randperm(c["experts"], generator=torch.Generator().manual_seed(seed)).tolist()
            s["counts"] = [counts[i] for i in order]
            s["offsets"] = torch.tensor([0] + s["counts"], device="cuda").cumsum(0).to(torch.int32)
        s["w"], s["w_scales"] = _four_bits(g, matrices * m, k, c["pad"], _rows(g, matrices * m, k, 0, "f32", 1 / math.sqrt(k)))
        s["x"], s["x_scales"] = _four_bits(g, tokens, k, c["pad"], _layer_input(g, tokens, k, 0, "f32"))
        s["bias"] = torch.randn(matrices, m, generator=g, device="cuda").mul_(0.2) if c["relu"] else None
        s["y"] = torch.zeros(tokens, m, device="cuda", dtype=_TORCH[type_])
        return s
    width, top = c["width"], c["top"]
    rows = tokens * max(top, 1)
    if top:
        s["experts"], s["weights"] = _choices(g, c)
        s["offsets"], s["places"], s["sources"] = _plain_sort(s["experts"], c["experts"])
    if c["op"] in ("route", "quantize"):
        s["x"] = _layer_input(g, tokens, width, c["pad"], type_)
    if c["op"] in ("combine", "gradients"):
        s["answers"] = _rows(g, rows, width, c["pad"], type_, 1.0)
    if c["op"] == "route":
        # (What a sort leaves is its own.)
        s["offsets"], s["places"], s["sources"] = (torch.zeros_like(s[n]) for n in ("offsets", "places", "sources"))
        s["chosen"] = torch.zeros(rows, width, device="cuda", dtype=_TORCH[type_])
    elif c["op"] == "combine":
        s["y"] = torch.zeros(tokens, width, device="cuda", dtype=_TORCH[type_])
    elif c["op"] == "gradients":
        s["dy"] = _rows(g, tokens, width, c["pad"], type_, 0.05)
        s["dchosen"] = _rows(g, rows, width, c["pad"], type_, 0.05)
        s["danswers"] = torch.zeros(rows, width, device="cuda", dtype=_TORCH[type_])
        s["dweights"] = torch.zeros(tokens, top, device="cuda")
        s["dx"] = torch.zeros(tokens, width, device="cuda", dtype=_TORCH[type_])
    else:
        s["data"] = torch.zeros(rows, (width + 1) // 2, device="cuda", dtype=torch.uint8)
        s["scales"] = torch.zeros(rows, -(-width // _BLOCK), device="cuda", dtype=torch.uint8)
        s["values"] = torch.zeros(rows, width, device="cuda", dtype=_TORCH[type_])
    return s


# ---- The plain form: 32 bits throughout, rounded once at the end ----

def _plain_route(s):
    offsets, places, sources = _plain_sort(s["experts"], s["case"]["experts"])
    chosen = torch.zeros_like(s["chosen"])
    used = sources[:int(offsets[-1])].long() // s["case"]["top"]
    chosen[:len(used)] = s["x"][used]
    return {"offsets": offsets, "places": places, "sources": sources, "chosen": chosen}


def _plain_sum(rows, places, weights):
    """Of each token's rows, with weights: in 32 bits."""
    there = (places >= 0)[..., None]
    picked = rows[places.clamp_min(0).long()].float()
    return torch.where(there, picked * weights[..., None], 0.0).sum(1)


def _plain_combine(s):
    return _plain_sum(s["answers"], s["places"], s["weights"]).to(s["y"].dtype)


def _plain_gradients(s):
    places, there = s["places"].clamp_min(0).long(), s["places"] >= 0
    dy = s["dy"].float()
    dweights = torch.where(there, (s["answers"][places].float() * dy[:, None]).sum(2), 0.0)
    danswers = torch.zeros_like(s["danswers"])
    danswers[places[there]] = (dy[:, None] * s["weights"][..., None])[there].to(danswers.dtype)
    dx = _plain_sum(s["dchosen"], s["places"], torch.ones_like(s["weights"])).to(s["dx"].dtype)
    return {"danswers": danswers, "dweights": dweights, "dx": dx}


def _plain_quantized(s):
    number, exponent = _plain_quantize(s["x"])
    values = _plain_values(number, exponent).to(s["values"].dtype)
    if not s["case"]["top"]:
        return values
    out = torch.zeros_like(s["values"])
    there = s["places"] >= 0
    out[s["places"][there].long()] = values[:, None].expand(-1, s["case"]["top"], -1)[there]
    return out


def _plain_product(s):
    c = s["case"]
    m, k = c["m"], c["k"]

    def values(data, scales):
        return _plain_values(_unpacked(data[:, :(k + 1) // 2], k), scales.int() - 127)

    x = values(s["x"], s["x_scales"])
    at = lambda e: slice(e * m, (e + 1) * m)  # noqa: E731
    parts = [part @ values(s["w"][at(e)], s["w_scales"][at(e)]).t() + (s["bias"][e] if c["relu"] else 0.0)
             for e, part in enumerate(x.split(s.get("counts", [c["tokens"]]))) if len(part)]
    y = torch.cat(parts)
    return (y.clamp_min_(0.0) if c["relu"] else y).to(s["y"].dtype)


# ---- The library's ----

@functools.lru_cache(None)
def _library():
    """The package and this program's context: it launches on torch's stream
    and its calls return once they are enqueued."""
    from ruy_amd import _structs, api
    context = api.Context()
    context.set_stream(torch.cuda.current_stream().cuda_stream)
    context.set_synchronous(False)
    return api, {"bf16": _structs.BF16, "f16": _structs.F16, "f32": _structs.F32, "i64": _structs.I64}, context


def _calls(s):
    """The calls of a pass with their arguments, and its outputs: the descriptors of
    buffers that a program makes once and keeps with them."""
    api, types, context = _library()
    c, kinds = s["case"], {**{_TORCH[name]: types[name] for name in _TORCH}, torch.int64: types["i64"]}

    def by_columns(name):
        """The rows of a tensor as the columns of a matrix."""
        t = s[name]
        return api.Matrix(kinds[t.dtype], t, api.Layout(t.shape[1], t.shape[0], t.stride(0), api.Order.kColMajor))

    def by_rows(name):
        t = s[name]
        return api.Matrix(kinds[t.dtype], t, api.Layout(t.shape[0], t.shape[1], t.stride(0), api.Order.kRowMajor))

    if c["op"] == "mxfp4":
        p = api.MulParams(types["f32"], kinds[s["y"].dtype])
        if c["relu"]:
            p.set_bias(s["bias"])
            p.set_clamp_min(0.0)
        w = api.MxFp4Matrix(c["m"], c["k"], s["w"], s["w_scales"], s["w"].stride(0))
        x = api.MxFp4Matrix(c["tokens"], c["k"], s["x"], s["x_scales"], s["x"].stride(0))
        groups = api.Groups(s["offsets"], c["experts"]) if c["experts"] else None
        return [(api.mul_mxfp4, (w, x, p, context, by_columns("y"), groups))], s["y"]
    routing = None
    if c["top"]:
        routing = api.Routing(c["tokens"], c["top"], c["experts"], s["offsets"], s["places"], s["sources"])
    if c["op"] == "route":
        return ([(api.sort_tokens, (by_columns("experts"), routing, context)),
                 (api.dispatch_tokens, (by_columns("x"), routing, context, by_columns("chosen")))],
                {n: s[n] for n in ("offsets", "places", "sources", "chosen")})
    if c["op"] == "combine":
        return [(api.combine_tokens, (by_columns("answers"), routing, by_columns("weights"), context, by_columns("y")))], s["y"]
    if c["op"] == "gradients":
        return ([(api.combine_tokens_gradients, (by_columns("dy"), by_columns("answers"), routing, by_columns("weights"),
                                                 context, by_columns("danswers"), by_columns("dweights"))),
                 (api.combine_tokens, (by_columns("dchosen"), routing, None, context, by_columns("dx")))],
                {n: s[n] for n in ("danswers", "dweights", "dx")})
    # (Each token to its places: of all rows that there may be, those behind the last one stay zeros.)
    held = api.MxFp4Matrix(s["data"].shape[0], c["width"], s["data"], s["scales"])
    return [(api.quantize_mxfp4, (by_rows("x"), context, held, routing)),
            (api.dequantize_mxfp4, (held, context, by_rows("values")))], s["values"]


def run(state):
    if not own:
        return {"route": _plain_route, "combine": _plain_combine, "gradients": _plain_gradients,
                "quantize": _plain_quantized, "mxfp4": _plain_product}[state["case"]["op"]](state)
    if "calls" not in state:
        state["calls"] = _calls(state)
    calls, outputs = state["calls"]
    for call, arguments in calls:
        call(*arguments)
    return outputs


def work(case):
    c, size = case, _BYTES[case["type"]]
    tokens = c["tokens"]
    if c["op"] == "mxfp4":
        reached = sum(n > 0 for n in _counts(c)) if c["experts"] else 1
        row = (c["k"] + 1) // 2 + -(-c["k"] // _BLOCK)
        count = (reached * c["m"] + tokens) * row + tokens * c["m"] * size + 4 * reached * c["m"] * c["relu"]
        return {"bytes": float(count), "flops": 2.0 * tokens * c["m"] * c["k"]}
    wanted = tokens - (tokens // c["drop"] if c["drop"] else 0)  # tokens that are not padding
    rows, width = wanted * c["top"], c["width"]
    choices = tokens * c["top"]
    if c["op"] == "route":
        return {"bytes": float(choices * (8 + 4 + 4) + 4 * (c["experts"] + 1) + (wanted + rows) * width * size),
                "flops": 0.0}
    if c["op"] == "combine":
        return {"bytes": float(choices * 8 + (rows + tokens) * width * size), "flops": 2.0 * rows * width}
    if c["op"] == "gradients":
        return {"bytes": float(choices * (4 + 4 + 4) + (wanted + 3 * rows + tokens) * width * size),
                "flops": 4.0 * rows * width}
    row = (width + 1) // 2 + -(-width // _BLOCK)
    if not c["top"]:
        rows = wanted = tokens
    return {"bytes": float(4 * choices + wanted * width * size + rows * (2 * row + width * size)), "flops": 0.0}


def _exact_values(numbers, scales):
    """float64 of numbers 0 .. 15 and bytes of scales, from the formats' bits: a sign, two bits
    of exponent (bias 1; 0: no leading one), one of mantissa; a scale is 2 ** (byte - 127)."""
    numbers = numbers.cpu().numpy().astype(np.int64)
    sign, exponent, mantissa = numbers >> 3, numbers >> 1 & 3, numbers & 1
    values = np.where(exponent > 0, np.ldexp(1.0 + mantissa / 2.0, exponent - 1), mantissa / 2.0) * np.where(sign, -1.0, 1.0)
    scales = scales.cpu().numpy().astype(np.int64) - 127
    return np.ldexp(values, np.repeat(scales, _BLOCK, axis=1)[:, :values.shape[1]].astype(np.int32))


def _exact_quantized(x):
    """The float64 values that the rows of x are held as."""
    x = x.double().cpu().numpy()
    out = np.zeros_like(x)
    grid = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
    for at in range(0, x.shape[1], _BLOCK):
        block = x[:, at:at + _BLOCK]
        largest = np.abs(block).max(axis=1)
        with np.errstate(divide="ignore"):
            scale = np.where(largest > 0, np.exp2(np.maximum(np.floor(np.log2(largest)), -125.0) - 2.0), 2.0 ** -127)
        # (log2 may round up to a whole number just below a power of two.)
        scale = np.where(scale * 4 > np.maximum(largest, 2.0 ** -125), scale / 2, scale)
        size = np.abs(block) / scale[:, None]
        low = np.clip(np.searchsorted(grid, size, side="right") - 1, 0, 6)
        middle = (grid[low] + grid[low + 1]) / 2
        up = (size > middle) | ((size == middle) & (low % 2 == 1))
        out[:, at:at + _BLOCK] = np.copysign(grid[low + up], block) * scale[:, None]
    return out


def exact(case, seed):
    """From the definitions, in 64 bits, choice by choice and expert by expert."""
    c, s = case, prepare(case, seed)
    if c["op"] == "mxfp4":
        bounds = [0, c["tokens"]] if not c["experts"] else s["offsets"].tolist()
        k, m = c["k"], c["m"]
        unpack = lambda t: torch.stack((t % 16, t // 16), 2).view(t.shape[0], -1)[:, :k]  # noqa: E731

        def values(data, scales):
            if data.shape[0] * k <= 1 << 22:
                return torch.from_numpy(_exact_values(unpack(data[:, :(k + 1) // 2]), scales)).cuda()
            n = unpack(data[:, :(k + 1) // 2]).int()
            e, f = (n // 2) % 4, (n % 2).double()
            size = torch.where(e > 0, (1 + f / 2) * (1 << (e - 1).clamp_min(0)), f / 2)
            power = torch.pow(torch.tensor(2.0, dtype=torch.float64, device="cuda"), scales.double() - 127)
            return torch.where(n >= 8, -size, size) * power.repeat_interleave(_BLOCK, 1)[:, :k]

        y = torch.zeros_like(s["y"], dtype=torch.float64)
        for e in range(len(bounds) - 1):
            at = slice(bounds[e], bounds[e + 1])
            if at.start == at.stop:
                continue
            w = values(s["w"][e * m:(e + 1) * m], s["w_scales"][e * m:(e + 1) * m])
            y[at] = torch.matmul(values(s["x"][at], s["x_scales"][at]), w.t())
            if c["relu"]:
                y[at] = torch.clamp(y[at] + s["bias"][e].double(), min=0.0)
        return y
    if c["top"]:
        # Choice by choice: an expert's next place is behind its last one's.
        chosen = s["experts"].flatten().tolist()
        count = [0] * (c["experts"] + 1)
        for e in chosen:
            if 0 <= e < c["experts"]:
                count[e + 1] += 1
        offsets = np.cumsum(count).tolist()
        following, places, sources = list(offsets), [-1] * len(chosen), [-1] * len(chosen)
        for i, e in enumerate(chosen):
            if 0 <= e < c["experts"]:
                places[i] = following[e]
                sources[following[e]] = i
                following[e] += 1
        reached = torch.tensor([i for i in sources if i >= 0], device="cuda", dtype=torch.int64)  # of each row its choice
        token = reached // c["top"]
        n = len(reached)
        weights = s["weights"].double().flatten()
    if c["op"] == "route":
        rows = torch.zeros_like(s["chosen"], dtype=torch.float64)
        rows[:n] = s["x"].double()[token]
        whole = [torch.tensor(v, device="cuda", dtype=torch.int32) for v in (offsets, places, sources)]
        return {"offsets": whole[0], "places": whole[1].view_as(s["places"]), "sources": whole[2], "chosen": rows}
    if c["op"] == "combine":
        y = torch.zeros_like(s["y"], dtype=torch.float64)
        for j in range(c["top"]):  # (a token's rows of one j are of different tokens: no sum has another order)
            mine = (reached % c["top"] == j).nonzero()[:, 0]
            y[token[mine]] += s["answers"][mine].double() * weights[reached[mine]][:, None]
        return y
    if c["op"] == "gradients":
        danswers = torch.zeros_like(s["danswers"], dtype=torch.float64)
        dweights = torch.zeros(len(chosen), device="cuda", dtype=torch.float64)
        dx = torch.zeros_like(s["dx"], dtype=torch.float64)
        for j in range(c["top"]):
            mine = (reached % c["top"] == j).nonzero()[:, 0]
            dy = s["dy"][token[mine]].double()
            danswers[mine] = dy * weights[reached[mine]][:, None]
            dweights[reached[mine]] = (dy * s["answers"][mine].double()).sum(1)
            dx[token[mine]] += s["dchosen"][mine].double()
        return {"danswers": danswers, "dweights": dweights.view_as(s["dweights"]), "dx": dx}
    values = torch.from_numpy(_exact_quantized(s["x"])).cuda()
    if not c["top"]:
        return values
    out = torch.zeros_like(s["values"], dtype=torch.float64)
    out[:n] = values[token]
    return out
