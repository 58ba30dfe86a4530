"""Sorting choices by expert in three launches (ruyamd_sort_tokens): recorded into
a graph, at the most experts that it takes, and next to the line of one launch.
"""
import numpy as np
import pytest
import torch

from test_gpu_routing import Sorted, announce, choices, context, experts_matrix  # noqa: F401  (context: a fixture)
from ruy_amd import _structs as S
from ruy_amd import api

pytestmark = pytest.mark.gpu

# tokens, top, count that take three launches; their counts lie in `places` from one to the next.
THREE_LAUNCHES = [(8192, 8, 256), (24577, 2, 5), (32769, 1, 16384)]


@pytest.mark.parametrize("tokens,top,count", THREE_LAUNCHES)
def test_three_launches_replayed_from_a_graph(context, tokens, top, count):  # noqa: F811
    """Recorded once, replayed on other choices, with eager calls and synchronizations in between."""
    announce("replayed sort", tokens, top, count)
    rng = np.random.default_rng(tokens)
    experts = torch.full((tokens, top), -1, dtype=torch.int64, device="cuda")
    matrix = api.Matrix(S.I64, experts, api.Layout(top, tokens, top, api.Order.kColMajor))
    own, recorded = Sorted(tokens, top, count), Sorted(tokens, top, count)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    context.set_stream(stream.cuda_stream)
    try:
        with torch.cuda.graph(graph, stream=stream):
            api.sort_tokens(matrix, recorded.routing, context)
    finally:
        context.set_stream(torch.cuda.current_stream().cuda_stream)
    # (Skewed, even, of padding alone, of one expert alone.)
    for make in (lambda: choices(rng, tokens, top, count), lambda: choices(rng, tokens, top, count, 0.5, 0.0),
                 lambda: np.full((tokens, top), -1), lambda: np.full((tokens, top), count - 1),
                 lambda: choices(rng, tokens, top, count, 0.0)):
        experts.copy_(torch.tensor(make()))
        for part in recorded.parts:
            part.fill_(-99)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        api.sort_tokens(matrix, own.routing, context)
        torch.cuda.synchronize()
        recorded.check(experts.cpu().numpy())
        own.check(experts.cpu().numpy())


# 16384 experts are the most of three launches: 64 KiB of LDS hold their counts.
@pytest.mark.parametrize("tokens,top,count", [(32768, 1, 16384), (50001, 1, 16384), (20000, 3, 16383), (40000, 2, 16000),
                                              (30001, 3, 8193), (2000, 3, 16385), (49152, 1, 4), (49153, 1, 4)])
@pytest.mark.parametrize("wide", [False, True], ids=["i32", "i64"])
def test_many_experts_and_the_line_between_one_launch_and_three(context, tokens, top, count, wide):  # noqa: F811
    announce("sort", tokens, top, count, wide)
    rng = np.random.default_rng(count)
    for skew in (0.0, 1.0):
        matrix, held = experts_matrix(choices(rng, tokens, top, count, 0.1, skew), wide)
        s = Sorted(tokens, top, count)
        api.sort_tokens(matrix, s.routing, context)
        s.check(held)
    # Numbers next to the ends: the first expert, the last, and what is just outside.
    held = np.resize(np.array([0, count - 1, count, -1, count - 1, 0, 1 % count]), (tokens, top))
    matrix, held = experts_matrix(held, wide)
    s = Sorted(tokens, top, count)
    api.sort_tokens(matrix, s.routing, context)
    s.check(held)
