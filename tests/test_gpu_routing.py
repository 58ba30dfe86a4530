"""Tokens to their experts and back (ruyamd_sort_tokens, ruyamd_dispatch_tokens,
ruyamd_combine_tokens, ruyamd_combine_tokens_gradients) against their definitions.

Sorting and copying are exact. Sums of small whole numbers are exact in fp32, and
the result must be the exact one, rounded once; sums of normally distributed values
are held to the bound of an fp32 sum (grouped_reference.error_bound).
"""
import ctypes as C

import numpy as np
import pytest
import torch

import grouped_reference as R
from grouped_reference import COL, ROW, Buffer
from ruy_amd import _structs as S
from ruy_amd import api
from ruy_amd._capi import lib

pytestmark = pytest.mark.gpu

TYPES = [S.BF16, S.F16, S.F32]
name_of = S.DTYPE_NAMES.get


def announce(*what):
    print("[case]", *what, flush=True)


@pytest.fixture(scope="module")
def context():
    ctx = api.Context()
    ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    yield ctx
    ctx.close()


@pytest.fixture(params=["generic", "chosen"])
def kernel(request, context):
    context.force_generic_kernel(request.param == "generic")
    yield request.param
    context.force_generic_kernel(False)


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def sorted_by_definition(experts, count):
    """(offsets, places, sources) of a tokens x top array."""
    flat = experts.reshape(-1).astype(np.int64)
    valid = (flat >= 0) & (flat < count)
    order = np.argsort(np.where(valid, flat, count), kind="stable")
    used = int(valid.sum())
    offsets = np.searchsorted(flat[order[:used]], np.arange(count + 1))
    places, sources = np.full(len(flat), -1), np.full(len(flat), -1)
    places[order[:used]] = np.arange(used)
    sources[:used] = order[:used]
    return offsets, places.reshape(experts.shape), sources


def choices(rng, tokens, top, count, invalid=0.1, skew=1.0):
    shares = (np.arange(count) + 1.0) ** -skew
    e = rng.choice(count, size=(tokens, top), p=shares / shares.sum())
    wrong = rng.random((tokens, top)) < invalid
    return np.where(wrong, rng.choice([-1, count, -2 ** 31, 2 ** 31 - 1], size=e.shape), e)


class Sorted:
    """A routing of device memory with guard words behind each part."""

    def __init__(self, tokens, top, count, sources=True):
        self.n, self.count = tokens * top, count
        self.parts = [torch.full((n + 5,), -99, dtype=torch.int32, device="cuda") for n in (count + 1, self.n, self.n)]
        self.routing = api.Routing(tokens, top, count, self.parts[0], self.parts[1], self.parts[2] if sources else None)

    def check(self, experts):
        want = sorted_by_definition(experts, self.count)
        for got, w, name in zip(self.parts, want, ("offsets", "places", "sources")):
            if name == "sources" and self.routing.sources is None:
                assert (got == -99).all()
                continue
            w = w.reshape(-1)
            got = got.cpu().numpy()
            assert (got[:len(w)] == w).all(), "%s: %d wrong" % (name, (got[:len(w)] != w).sum())
            assert (got[len(w):] == -99).all(), name


def experts_matrix(experts, wide, order=COL, pad=0):
    """The tokens x top choices as a top x tokens matrix in device memory."""
    tokens, top = experts.shape
    held = np.clip(experts, -2 ** 31, 2 ** 31 - 1)
    inner, outer = (top, tokens) if order == COL else (tokens, top)
    flat = torch.full((outer * (inner + pad) + 1,), 0, dtype=torch.int64 if wide else torch.int32, device="cuda")
    strides = (inner + pad, 1) if order == COL else (1, inner + pad)
    torch.as_strided(flat, (tokens, top), strides).copy_(torch.tensor(held))
    return api.Matrix(S.I64 if wide else S.I32, flat, api.Layout(top, tokens, inner + pad, order)), held


SORTS = [(0, 2, 4), (1, 1, 1), (1, 8, 8), (3, 0, 5), (16, 2, 64), (37, 3, 7), (64, 1, 65536), (255, 4, 33), (1000, 7, 256),
         (8192, 4, 64), (5000, 9, 100), (40000, 1, 3),
         # Enough choices and experts for three launches; a last part of any length.
         (16384, 8, 256), (9001, 7, 1000), (60000, 2, 257), (20011, 8, 4096), (300000, 1, 16), (70001, 3, 1024)]


@pytest.mark.parametrize("wide", [False, True], ids=["i32", "i64"])
@pytest.mark.parametrize("tokens,top,count", SORTS)
def test_sort(context, kernel, tokens, top, count, wide):
    if kernel == "generic" and tokens * top * count > 1 << 27:
        pytest.skip("the plain kernel reads all choices for every expert")
    announce("sort", tokens, top, count, wide)
    rng = np.random.default_rng(tokens + top)
    experts = choices(rng, tokens, top, count)
    for order, pad, sources in [(COL, 0, True), (ROW, 0, False), (COL, 3, True), (ROW, 2, True)]:
        matrix, held = experts_matrix(experts, wide, order, pad)
        s = Sorted(tokens, top, count, sources)
        api.sort_tokens(matrix, s.routing, context)
        s.check(held)


@pytest.mark.parametrize("tokens,top,count", [(50, 2, 8), (20000, 8, 128)])
@pytest.mark.parametrize("kind", ["none", "one", "last", "same"])
def test_sort_with_empty_experts(context, tokens, top, count, kind):
    experts = {"none": lambda: np.full((tokens, top), -1), "one": lambda: np.full((tokens, top), 3),
               "last": lambda: np.full((tokens, top), count - 1),
               "same": lambda: np.repeat(np.arange(tokens)[:, None] % count, top, axis=1)}[kind]()
    matrix, held = experts_matrix(experts, True)
    s = Sorted(tokens, top, count)
    api.sort_tokens(matrix, s.routing, context)
    s.check(held)


def test_sort_of_wide_numbers_looks_at_all_bits(context):
    experts = torch.tensor([[1 << 32, 1], [(1 << 32) + 1, -(1 << 32)]], device="cuda")
    s = Sorted(2, 2, 2)
    api.sort_tokens(api.Matrix(S.I64, experts, api.Layout(2, 2, 2, COL)), s.routing, context)
    assert s.parts[1][:4].tolist() == [-1, 0, -1, -1] and s.parts[0][:3].tolist() == [0, 0, 1]


def test_sort_of_many_choices(context):
    """More than a part's 32 choices of a lane in one launch, and over a million in three."""
    for tokens, top, count in [(200000, 1, 4), (1 << 20, 2, 64)]:
        announce("sort", tokens, top, count)
        experts = choices(np.random.default_rng(1), tokens, top, count)
        matrix, held = experts_matrix(experts, False)
        s = Sorted(tokens, top, count)
        api.sort_tokens(matrix, s.routing, context)
        s.check(held)


# ---- Moving and adding up ----

def places_of(rng, tokens, top, spare=3, invalid=0.15):
    """Random places: (tokens x top array with some -1 or outside, number of columns). No place twice."""
    n = tokens * top
    columns = n + spare
    p = rng.permutation(columns)[:n].reshape(tokens, top)
    wrong = rng.random(p.shape) < invalid
    if tokens > 2:
        wrong[1] = True  # a token without any
    return np.where(wrong, rng.choice([-1, columns, -7, 2 ** 31 - 1], size=p.shape), p), columns


def routing_of(places):
    tokens, top = places.shape
    return api.Routing(tokens, top, 1, None, torch.tensor(places.astype(np.int32), device="cuda"))


def held_places(places, columns):
    return [[int(p) if 0 <= p < columns else -1 for p in row] for row in places]


# Widths: shorter than 16 bytes, one unit, overlapping units, several segments.
SHAPES = [(1, 1, 8), (1, 8, 2048), (5, 2, 1), (7, 3, 3), (16, 2, 64), (9, 5, 1111), (33, 9, 520), (300, 2, 4096), (40, 4, 8199),
          (2500, 2, 65),
          # Several tokens to a wave, and just not.
          (1000, 5, 24), (333, 9, 100), (2001, 1, 128), (777, 6, 130), (101, 4, 255), (403, 2, 256), (55, 3, 257)]
LAYOUTS = [((COL, 0, 0), (COL, 0, 0)), ((COL, 3, 1), (COL, 5, 1)), ((ROW, 0, 0), (COL, 1, 0)), ((COL, 0, 1), (ROW, 2, 0))]


@pytest.mark.parametrize("type_", TYPES, ids=name_of)
@pytest.mark.parametrize("tokens,top,width", SHAPES)
def test_dispatch(context, kernel, type_, tokens, top, width):
    announce("dispatch", name_of(type_), tokens, top, width)
    rng, g = np.random.default_rng(width), generator(tokens)
    places, columns = places_of(rng, tokens, top)
    for (order_s, pad_s, shift_s), (order_d, pad_d, shift_d) in LAYOUTS:
        src = Buffer(type_, width, tokens, order_s, pad_s, shift_s).set(torch.randn(width, tokens, generator=g, device="cuda"))
        dst = Buffer(type_, width, columns, order_d, pad_d, shift_d, fill=-77.0)
        before, want = dst.flat.clone(), dst.view().clone()
        for t, row in enumerate(held_places(places, columns)):
            for p in row:
                if p >= 0:
                    want[:, p] = src.view()[:, t]
        api.dispatch_tokens(src.matrix(), routing_of(places), context, dst.matrix())
        assert torch.equal(dst.view(), want)
        assert dst.untouched(before, lambda i: (slice(None), slice(None)))


def test_dispatch_copies_bits(context):
    """NaN of any payload, infinities and denormals arrive as they are."""
    bits = torch.arange(65536, dtype=torch.int32, device="cuda").to(torch.int16).view(64, 1024)
    src = api.Matrix(S.F16, bits, api.Layout(1024, 64, 1024, COL))
    out = torch.zeros(128, 1024, dtype=torch.int16, device="cuda")
    places = np.stack([np.arange(64), 127 - np.arange(64)], axis=1)
    api.dispatch_tokens(src, routing_of(places), context, api.Matrix(S.F16, out, api.Layout(1024, 128, 1024, COL)))
    assert torch.equal(out[:64], bits) and torch.equal(out[64:].flip(0), bits)


def weights_of(g, type_, tokens, top, order, whole):
    """(Buffer of top x tokens or None, float64 tokens x top)."""
    if type_ is None:
        return None, torch.ones(tokens, top, dtype=torch.float64, device="cuda")
    w = R.whole_numbers(g, (top, tokens), 3) if whole else torch.rand(top, tokens, generator=g, device="cuda").double()
    b = Buffer(type_, top, tokens, order, 2).set(w)
    return b, b.view().double().t()


def check(got, want, dst_type, bound=None):
    if bound is None:
        wrong = got != R.rounded(want, dst_type)
        assert not wrong.any().item(), "%d wrong, the first at %s" % (wrong.sum().item(), wrong.nonzero()[0].tolist())
    else:
        error = (got.double() - want).abs()
        assert (error <= bound).all(), "%.3g times the bound" % (error / bound).max().item()


@pytest.mark.parametrize("whole", [True, False], ids=["whole", "normal"])
@pytest.mark.parametrize("type_,dst_type", [(t, d) for t in TYPES for d in {t, S.F32}], ids=name_of)
@pytest.mark.parametrize("tokens,top,width", SHAPES)
def test_combine(context, kernel, type_, dst_type, tokens, top, width, whole):
    announce("combine", name_of(type_), name_of(dst_type), tokens, top, width)
    rng, g = np.random.default_rng(width), generator(tokens)
    places, columns = places_of(rng, tokens, top)
    for n, ((order_d, pad_d, shift_d), (order_s, pad_s, shift_s)) in enumerate(LAYOUTS):
        x = R.whole_numbers(g, (width, columns), 9) if whole else torch.randn(width, columns, generator=g, device="cuda").double()
        src = Buffer(type_, width, columns, order_s, pad_s, shift_s).set(x)
        weights, w = weights_of(g, [None, S.F32, S.BF16, S.F16][n], tokens, top, [COL, COL, ROW, COL][n], whole)
        used = {p for row in held_places(places, columns) for p in row if p >= 0}
        idle = [p for p in range(columns) if p not in used]
        src.view()[:, idle] = float("nan")  # what is no place has no influence,
        if weights:  # nor has the weight of a choice without one
            for t, row in enumerate(held_places(places, columns)):
                for j, p in enumerate(row):
                    if p < 0:
                        weights.view()[j, t] = float("inf")
        dst = Buffer(dst_type, width, tokens, order_d, pad_d, shift_d, fill=-77.0)
        before = dst.flat.clone()
        api.combine_tokens(src.matrix(), routing_of(places), weights.matrix() if weights else None, context, dst.matrix())
        want = torch.zeros(width, tokens, dtype=torch.float64, device="cuda")
        magnitude = torch.zeros_like(want)
        for j in range(top):
            at = torch.tensor([r[j] for r in held_places(places, columns)], device="cuda")
            there = at >= 0
            term = src.view()[:, at.clamp_min(0)].double() * torch.where(there, w[:, j], 0.0)
            term = torch.where(there, term, 0.0)
            want += term
            magnitude += term.abs()
        check(dst.view(), want, dst_type, None if whole else R.error_bound(magnitude, top, want, dst_type))
        assert dst.untouched(before, lambda i: (slice(None), slice(None)))


@pytest.mark.parametrize("whole", [True, False], ids=["whole", "normal"])
@pytest.mark.parametrize("type_,grad_type", [(t, d) for t in TYPES for d in {t, S.F32}], ids=name_of)
@pytest.mark.parametrize("tokens,top,width", SHAPES)
def test_gradients(context, kernel, type_, grad_type, tokens, top, width, whole):
    announce("gradients", name_of(type_), name_of(grad_type), tokens, top, width)
    rng, g = np.random.default_rng(width), generator(tokens)
    places, columns = places_of(rng, tokens, top)
    held = held_places(places, columns)
    for n, ((order_g, pad_g, shift_g), (order_s, pad_s, shift_s)) in enumerate(LAYOUTS):
        make = (lambda *s: R.whole_numbers(g, s, 3)) if whole else (lambda *s: torch.randn(*s, generator=g, device="cuda").double())
        grad = Buffer(grad_type, width, tokens, order_g, pad_g, shift_g).set(make(width, tokens))
        src = Buffer(type_, width, columns, order_s, pad_s, shift_s).set(make(width, columns))
        weights, w = weights_of(g, [S.F32, None, S.BF16, S.F16][n], tokens, top, [COL, COL, ROW, COL][n], whole)
        w_type = [S.F32, S.F32, S.BF16, S.F16][n]
        for want_rows, want_weights in [(True, True), (True, False), (False, True)]:
            grad_src = Buffer(type_, width, columns, order_s, pad_s + 1, shift_s, fill=-77.0)
            grad_weights = Buffer(w_type, top, tokens, [COL, ROW][n % 2], 1, fill=-77.0)
            before, before_w = grad_src.flat.clone(), grad_weights.flat.clone()
            rows = grad_src.view().clone()
            api.combine_tokens_gradients(grad.matrix(), src.matrix() if want_weights else None, routing_of(places),
                                         weights.matrix() if weights else None, context,
                                         grad_src.matrix() if want_rows else None,
                                         grad_weights.matrix() if want_weights else None)
            for j in range(top):
                at = torch.tensor([r[j] for r in held], device="cuda")
                there = (at >= 0).nonzero()[:, 0]
                gr = grad.view().double()[:, there]
                if want_rows:
                    # (One product in fp32, rounded, then rounded to the type.)
                    product = gr * w[there, j]
                    rows[:, at[there]] = R.rounded(product, type_)
                if want_weights:
                    terms = torch.zeros(width, tokens, dtype=torch.float64, device="cuda")
                    terms[:, there] = gr * src.view().double()[:, at[there]]
                    want = terms.sum(0)
                    bound = None if whole else R.error_bound(terms.abs().sum(0), width, want, w_type)
                    check(grad_weights.view()[j], want, w_type, bound)
            if want_rows:
                assert torch.equal(grad_src.view(), rows)
            assert grad_src.untouched(before, lambda i: (slice(None), slice(None)) if want_rows else None)
            assert grad_weights.untouched(before_w, lambda i: (slice(None), slice(None)) if want_weights else None)


@pytest.mark.parametrize("type_", TYPES, ids=name_of)
def test_gradients_are_those_of_the_sums_differences(context, type_):
    """The sum is linear in rows and in weights: with whole numbers its differences are exact, and
    <grad, difference> must be <gradient, step>."""
    tokens, top, width = 50, 3, 72
    rng, g = np.random.default_rng(0), generator(0)
    places, columns = places_of(rng, tokens, top)
    routing = routing_of(places)
    whole = lambda *s: R.whole_numbers(g, s, 2)  # noqa: E731
    src, step = Buffer(type_, width, columns, COL).set(whole(width, columns)), whole(width, columns)
    weights, w_step = Buffer(S.F32, top, tokens, COL).set(whole(top, tokens)), whole(top, tokens)
    grad = Buffer(type_, width, tokens, COL).set(whole(width, tokens))

    def combined(rows, w):
        dst = Buffer(S.F32, width, tokens, COL)
        api.combine_tokens(Buffer(type_, width, columns, COL).set(rows).matrix(), routing,
                           Buffer(S.F32, top, tokens, COL).set(w).matrix(), context, dst.matrix())
        return dst.view().double()

    grad_src = Buffer(type_, width, columns, COL, fill=0.0)
    grad_weights = Buffer(S.F32, top, tokens, COL, fill=0.0)
    api.combine_tokens_gradients(grad.matrix(), src.matrix(), routing, weights.matrix(), context, grad_src.matrix(),
                                 grad_weights.matrix())
    x, w, gr = src.view().double(), weights.view().double(), grad.view().double()
    at = combined(x, w)
    assert ((combined(x + step, w) - at) * gr).sum() == (grad_src.view().double() * step).sum()
    assert ((combined(x, w + w_step) - at) * gr).sum() == (grad_weights.view().double() * w_step).sum()
    # The gradient of dispatch_tokens is the sum without weights.
    d = Buffer(S.F32, width, tokens, COL)
    api.combine_tokens(src.matrix(), routing, None, context, d.matrix())
    moved = Buffer(type_, width, columns, COL, fill=0.0)
    api.dispatch_tokens(grad.matrix(), routing, context, moved.matrix())
    assert (moved.view().double() * x).sum() == (d.view().double() * gr).sum()


def test_special_values(context, kernel):
    """Infinities and NaN of a token's own rows arrive in its sum and gradients, and nowhere else."""
    inf, nan = float("inf"), float("nan")
    src = torch.ones(4, 16, device="cuda")  # rows of places 0 .. 3
    src[0, 3], src[1, 3], src[2, 5] = inf, -inf, nan
    places = np.array([[0, 1], [2, 3], [-1, 3]])
    y = torch.zeros(3, 16, device="cuda")
    col = lambda t: api.Matrix(S.F32, t, api.Layout(t.shape[1], t.shape[0], t.shape[1], COL))  # noqa: E731
    api.combine_tokens(col(src), routing_of(places), None, context, col(y))
    want = torch.full((3, 16), 2.0, device="cuda")
    want[0, 3], want[1, 5], want[2] = nan, nan, 1.0
    assert torch.equal(torch.isnan(y), torch.isnan(want)) and torch.equal(y.nan_to_num(9), want.nan_to_num(9))
    dw = torch.zeros(3, 2, device="cuda")
    grad = torch.ones(3, 16, device="cuda")
    api.combine_tokens_gradients(col(grad), col(src), routing_of(places), None, context, None, col(dw))
    assert dw.tolist()[0] == [inf, -inf] and np.isnan(dw.tolist()[1][0]) and dw.tolist()[1][1] == 16
    assert dw.tolist()[2] == [0.0, 16.0]


def test_empty_calls(context, kernel):
    none, some = Buffer(S.F32, 8, 0, COL), Buffer(S.F32, 8, 5, COL, fill=-3.0)
    empty = np.zeros((0, 2), int)
    # No tokens, or tokens that choose nothing: columns of dst stay; sums are zeros.
    api.dispatch_tokens(none.matrix(), routing_of(empty), context, some.matrix())
    assert (some.flat == -3).all()
    api.combine_tokens(some.matrix(), routing_of(empty), None, context, none.matrix())
    choiceless = api.Routing(5, 0, 1, None, None)
    api.combine_tokens(none.matrix(), choiceless, None, context, some.matrix())
    assert (some.view() == 0).all()
    api.dispatch_tokens(some.matrix(), choiceless, context, none.matrix())
    # Rows of no length: weights have gradients of zero.
    flat = Buffer(S.F32, 0, 5, COL)
    dw = Buffer(S.F32, 1, 5, COL, fill=-3.0)
    api.combine_tokens_gradients(flat.matrix(), flat.matrix(), routing_of(np.arange(5)[:, None]), None, context, flat.matrix(),
                                 dw.matrix())
    assert (dw.view() == 0).all()
    # No columns of places: none of the places is one.
    api.combine_tokens(none.matrix(), routing_of(np.arange(5)[:, None]), None, context, some.matrix())
    assert (some.view() == 0).all()
    assert context.last_kernel_name() in ("tokens", "generic")


def test_long_rows_and_far_columns(context):
    """Places whose columns lie more than 2^31 values, and 2^32 bytes, behind the first."""
    width, pad = 1000, (1 << 27) - 1000
    flat = torch.empty(20 * (width + pad) + width, dtype=torch.float16, device="cuda")  # 5 GB
    rows = torch.as_strided(flat, (21, width), (width + pad, 1))
    rows.fill_(0)
    x = torch.randn(3, width, device="cuda").half()
    far = api.Matrix(S.F16, flat, api.Layout(width, 21, width + pad, COL))
    places = np.array([[0, 20], [17, 3], [16, 19]])
    near = api.Matrix(S.F16, x, api.Layout(width, 3, width, COL))
    api.dispatch_tokens(near, routing_of(places), context, far)
    for t in range(3):
        for p in places[t]:
            assert torch.equal(rows[p], x[t])
    y = torch.zeros(3, width, device="cuda")
    api.combine_tokens(far, routing_of(places), None, context, api.Matrix(S.F32, y, api.Layout(width, 3, width, COL)))
    assert torch.equal(y, 2 * x.float())
    dw = torch.zeros(3, 2, device="cuda")
    api.combine_tokens_gradients(near, far, routing_of(places), None, context, None, api.Matrix(S.F32, dw, api.Layout(2, 3, 2, COL)))
    want = (x.double() ** 2).sum(1, keepdim=True).expand(3, 2)
    assert ((dw.double() - want).abs() <= R.error_bound(want, width, want, S.F32)).all()
    rows.fill_(0)
    api.combine_tokens_gradients(near, None, routing_of(places), None, context, far, None)
    for t in range(3):
        for p in places[t]:
            assert torch.equal(rows[p], x[t])


@pytest.mark.parametrize("width", [100, 250, 600])
def test_many_narrow_tokens(context, width):
    """More than the caches hold, several tokens to a wave and one. Small whole numbers: every sum is exact."""
    tokens, top = 100000, 2
    announce("many narrow tokens", width)
    g = generator(width)
    x = torch.randint(-3, 4, (tokens, width), generator=g, device="cuda").to(torch.bfloat16)
    rows = torch.randint(-3, 4, (tokens * top + 3, width), generator=g, device="cuda").to(torch.bfloat16)
    weights = torch.randint(-2, 3, (tokens, top), generator=g, device="cuda").float()
    places = torch.randperm(tokens * top + 3, generator=g, device="cuda")[:tokens * top].reshape(tokens, top).int()
    routing = api.Routing(tokens, top, 1, None, places)
    at = places.long()

    def col(t):
        return api.Matrix({torch.bfloat16: S.BF16, torch.float32: S.F32}[t.dtype], t, api.Layout(t.shape[1], t.shape[0], t.shape[1], COL))

    y, dw, moved, drows = torch.zeros(tokens, width, device="cuda"), torch.zeros_like(weights), torch.full_like(rows, 9), torch.full_like(rows, 9)
    api.dispatch_tokens(col(x), routing, context, col(moved))
    api.combine_tokens(col(rows), routing, col(weights), context, col(y))
    api.combine_tokens_gradients(col(x), col(rows), routing, col(weights), context, col(drows), col(dw))
    left = torch.ones(tokens * top + 3, dtype=torch.bool, device="cuda")
    left[at.flatten()] = False
    assert bool((moved[left] == 9).all()) and bool((drows[left] == 9).all())
    want = torch.zeros_like(y)
    for j in range(top):
        assert torch.equal(moved[at[:, j]], x)
        assert torch.equal(drows[at[:, j]], weights[:, j:j + 1].bfloat16() * x)
        want += weights[:, j:j + 1] * rows[at[:, j]].float()
        assert torch.equal(dw[:, j], (x.float() * rows[at[:, j]].float()).sum(1))
    assert torch.equal(y, want)


def test_the_most_tokens(context):
    """2^31 - 1 choices, one of each token: the last workgroup's waves have tokens up to the last number there is, and none behind."""
    tokens, width, columns, piece = 2 ** 31 - 1, 8, 5, 1 << 26
    announce("most tokens")
    places = torch.full((tokens,), -1, dtype=torch.int32, device="cuda")
    where = torch.tensor([0, 1 << 30, tokens - 2, tokens - 1], device="cuda")
    places[where] = torch.tensor([3, 0, 4, 1], dtype=torch.int32, device="cuda")
    routing = api.Routing(tokens, 1, 1, None, places)
    g = generator(5)
    src = torch.randint(-4, 5, (columns, width), generator=g, device="cuda").to(torch.bfloat16)
    grad = torch.ones(tokens, width, dtype=torch.bfloat16, device="cuda")
    grad[where] = torch.randint(-4, 5, (4, width), generator=g, device="cuda").to(torch.bfloat16)
    grad_src = torch.full((columns, width), -77.0, dtype=torch.bfloat16, device="cuda")
    grad_weights = torch.full((tokens,), -77.0, dtype=torch.bfloat16, device="cuda")
    api.combine_tokens_gradients(api.Matrix(S.BF16, grad, api.Layout(width, tokens, width, COL)),
                                 api.Matrix(S.BF16, src, api.Layout(width, columns, width, COL)), routing, None, context,
                                 api.Matrix(S.BF16, grad_src, api.Layout(width, columns, width, COL)),
                                 api.Matrix(S.BF16, grad_weights, api.Layout(1, tokens, 1, COL)))
    taken = places[where].long()
    assert torch.equal(grad_src[taken], grad[where]) and bool((grad_src[2] == -77).all())
    assert torch.equal(grad_weights[where], (grad[where].float() * src[taken].float()).sum(1).to(torch.bfloat16))
    grad_weights[where] = 0
    for at in range(0, tokens, piece):
        assert not grad_weights[at:at + piece].any().item()

    # grad's memory as the sums'.
    api.combine_tokens(api.Matrix(S.BF16, src, api.Layout(width, columns, width, COL)), routing, None, context,
                       api.Matrix(S.BF16, grad, api.Layout(width, tokens, width, COL)))
    assert torch.equal(grad[where], src[taken])
    grad[where] = 0
    for at in range(0, tokens, piece):
        assert not grad[at:at + piece].any().item()

    # And their places: token t chooses expert t % 64.
    del grad, grad_weights
    experts = torch.arange(tokens, dtype=torch.int32, device="cuda")
    experts &= 63
    offsets = torch.zeros(65, dtype=torch.int32, device="cuda")
    api.sort_tokens(api.Matrix(S.I32, experts, api.Layout(1, tokens, 1, COL)), api.Routing(tokens, 1, 64, offsets, places), context)
    begins = torch.arange(65, dtype=torch.int64) * (1 << 25)
    begins[64] = tokens  # (the last expert has one less)
    assert torch.equal(offsets.cpu().long(), begins)
    for at in range(0, tokens, piece):
        t = torch.arange(at, min(at + piece, tokens), dtype=torch.int64, device="cuda")
        assert torch.equal(places[at:at + piece].long(), (t & 63) * (1 << 25) + (t >> 6))


def test_results_do_not_change_from_call_to_call(context):
    rng, g = np.random.default_rng(0), generator(0)
    tokens, top, width = 500, 6, 1030
    places, columns = places_of(rng, tokens, top)
    src = Buffer(S.BF16, width, columns, COL).set(torch.randn(width, columns, generator=g, device="cuda"))
    grad = Buffer(S.BF16, width, tokens, COL).set(torch.randn(width, tokens, generator=g, device="cuda"))
    weights = Buffer(S.F32, top, tokens, COL).set(torch.rand(top, tokens, generator=g, device="cuda"))
    outs = []
    for _ in range(3):
        y, dw = Buffer(S.F32, width, tokens, COL, fill=0.0), Buffer(S.F32, top, tokens, COL, fill=0.0)
        api.combine_tokens(src.matrix(), routing_of(places), weights.matrix(), context, y.matrix())
        api.combine_tokens_gradients(grad.matrix(), src.matrix(), routing_of(places), None, context, None, dw.matrix())
        outs.append((y.flat, dw.flat))
    assert all(torch.equal(a, b) for o in outs[1:] for a, b in zip(outs[0], o))


def test_refusals(context):
    good = torch.zeros(64, device="cuda")
    ints = torch.zeros(64, dtype=torch.int32, device="cuda")
    host = torch.zeros(64)

    def mat(dtype=S.F32, data=good, rows=8, cols=4, stride=None, order=COL, zero_point=0):
        return api.Matrix(dtype, data, api.Layout(rows, cols, rows if stride is None else stride, order), zero_point)

    def routing(tokens=4, top=2, count=3, offsets=ints, places=ints, sources=None):
        return api.Routing(tokens, top, count, offsets, places, sources)

    def refused(code, f, *arguments):
        with pytest.raises(api.RuyAmdError) as e:
            f(*arguments)
        assert e.value.code == code and str(e.value)

    experts = mat(S.I32, ints, 2, 4)
    api.sort_tokens(experts, routing(), context)
    for bad in (routing(tokens=-1), routing(top=-2), routing(count=0), routing(count=65537), routing(offsets=None),
                routing(places=None), routing(tokens=5), routing(places=ints.data_ptr() + 2)):
        refused(S.E_INVALID, api.sort_tokens, experts, bad, context)
    for bad in (routing(tokens=1 << 20, top=1 << 11), routing(places=host), routing(offsets=host), routing(sources=host)):
        refused(S.E_UNSUPPORTED, api.sort_tokens, experts, bad, context)
    for bad in (mat(S.I32, ints, 3, 4), mat(S.I32, ints, 2, 4, 1), mat(S.I32, ints, 2, 4, order=2), mat(S.I32, None, 2, 4),
                mat(S.I32, ints, 2, 4, zero_point=1), mat(S.I64, ints.data_ptr() + 4, 2, 4)):
        refused(S.E_INVALID, api.sort_tokens, bad, routing(), context)
    for bad in (mat(S.F32, ints, 2, 4), mat(S.I16, ints, 2, 4), mat(S.I32, host, 2, 4)):
        refused(S.E_UNSUPPORTED, api.sort_tokens, bad, routing(), context)

    rows = mat(cols=6, data=torch.zeros(64, device="cuda"))
    api.dispatch_tokens(mat(), routing(), context, rows)
    api.combine_tokens(rows, routing(), None, context, mat())
    for bad in (mat(cols=5), mat(rows=7), mat(stride=7), mat(data=None), mat(zero_point=3)):
        refused(S.E_INVALID, api.dispatch_tokens, bad, routing(), context, rows)
        refused(S.E_INVALID, api.combine_tokens, rows, routing(), None, context, bad)
    for bad in (mat(S.F16), mat(S.F64), mat(S.I32), mat(data=host)):
        refused(S.E_UNSUPPORTED, api.dispatch_tokens, bad, routing(), context, rows)
        refused(S.E_UNSUPPORTED, api.combine_tokens, rows, routing(), None, context, bad)
    refused(S.E_INVALID, api.dispatch_tokens, mat(), routing(count=0), context, rows)
    weights = mat(rows=2, cols=4)
    for bad in (mat(rows=3, cols=4), mat(rows=2, cols=3), mat(rows=2, cols=4, data=None)):
        refused(S.E_INVALID, api.combine_tokens, rows, routing(), bad, context, mat())
        refused(S.E_INVALID, api.combine_tokens_gradients, mat(), rows, routing(), bad, context, rows, None)
        refused(S.E_INVALID, api.combine_tokens_gradients, mat(), rows, routing(), None, context, None, bad)
    refused(S.E_UNSUPPORTED, api.combine_tokens, rows, routing(), mat(S.I32, ints, 2, 4), context, mat())

    gradients = api.combine_tokens_gradients
    gradients(mat(), rows, routing(), weights, context, rows, weights)
    refused(S.E_INVALID, gradients, mat(), rows, routing(), weights, context, None, None)
    refused(S.E_INVALID, gradients, mat(), None, routing(), weights, context, None, weights)
    refused(S.E_INVALID, gradients, mat(), rows, routing(), weights, context, mat(S.F16, cols=6), weights)
    refused(S.E_INVALID, gradients, mat(), rows, routing(), weights, context, mat(cols=7), weights)
    refused(S.E_UNSUPPORTED, gradients, mat(S.F16), rows, routing(), weights, context, rows, weights)
    with pytest.raises(api.RuyAmdError):
        context._check(lib.ruyamd_sort_tokens(context._h, None, None))
    context.set_runtime_enabled_paths(S.PATH_STANDARD_CPP)
    refused(S.E_NO_PATH, api.sort_tokens, experts, routing(), context)
    context.set_runtime_enabled_paths(S.PATH_GFX950)
    # The context is as good as before.
    api.sort_tokens(experts, routing(), context)
    r = routing().to_struct()
    assert lib.ruyamd_sort_tokens(None, C.byref(experts.to_struct()), C.byref(r)) == S.E_INVALID


def test_replayed_from_a_graph(context):
    """A step of sort, dispatch, combine and gradients recorded once, replayed on other choices and values
    with eager work between the replays."""
    tokens, top, count, width = 4096, 8, 256, 264  # (three launches of the sort)
    rng, g = np.random.default_rng(5), generator(5)
    experts = torch.zeros(tokens, top, dtype=torch.int64, device="cuda")
    x = torch.zeros(tokens, width, dtype=torch.bfloat16, device="cuda")
    weights = torch.zeros(tokens, top, device="cuda")

    def buffers():
        s = Sorted(tokens, top, count)
        return s, [torch.zeros(tokens * top, width, dtype=x.dtype, device="cuda"), torch.zeros_like(x),
                   torch.zeros(tokens * top, width, dtype=x.dtype, device="cuda"), torch.zeros_like(weights)]

    kinds = {torch.bfloat16: S.BF16, torch.float32: S.F32, torch.int64: S.I64}

    def col(t):
        return api.Matrix(kinds[t.dtype], t, api.Layout(t.shape[1], t.shape[0], t.shape[1], COL))

    def step(s, b):
        api.sort_tokens(col(experts), s.routing, context)
        api.dispatch_tokens(col(x), s.routing, context, col(b[0]))
        api.combine_tokens(col(b[0]), s.routing, col(weights), context, col(b[1]))
        api.combine_tokens_gradients(col(x), col(b[0]), s.routing, col(weights), context, col(b[2]), col(b[3]))

    stream = torch.cuda.Stream()
    own, recorded = buffers(), buffers()
    graph = torch.cuda.CUDAGraph()
    context.set_stream(stream.cuda_stream)
    try:
        with torch.cuda.graph(graph, stream=stream):
            step(*recorded)
    finally:
        context.set_stream(torch.cuda.current_stream().cuda_stream)
    for i in range(3):
        e = choices(rng, tokens, top, count)
        experts.copy_(torch.tensor(np.clip(e, -2 ** 31, 2 ** 31 - 1)))
        x.normal_(generator=g)
        weights.uniform_(generator=g)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        step(*own)
        torch.cuda.synchronize()
        recorded[0].check(experts.cpu().numpy())
        used = int(own[0].parts[0][count])
        for a, b in zip(own[1], recorded[1]):
            n = used if a.shape[0] == tokens * top else len(a)
            assert torch.equal(a[:n], b[:n]), i


def test_two_contexts_on_their_own_streams():
    """Calls of two contexts overlap and do not disturb each other."""
    contexts = [api.Context() for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    sets = []
    for i, (ctx, stream) in enumerate(zip(contexts, streams)):
        ctx.set_stream(stream.cuda_stream)
        ctx.set_synchronous(False)
        experts = choices(np.random.default_rng(i), 9001, 7, 1000)
        matrix, held = experts_matrix(experts, False)
        sets.append((matrix, held, [Sorted(9001, 7, 1000) for _ in range(5)]))
    torch.cuda.synchronize()
    for k in range(5):
        for ctx, (matrix, _, out) in zip(contexts, sets):
            api.sort_tokens(matrix, out[k].routing, ctx)
    torch.cuda.synchronize()
    for _, held, out in sets:
        for s in out:
            s.check(held)
    for ctx in contexts:
        ctx.close()
