"""Which kernels the calls for layers of experts run on, on a model of the HIP
runtime (tests/cpp/expert_routes_test.cc). No device is needed.

GPU tests that are named for a kernel say nothing when a rule for choosing
kernels has moved and they run on another one. Here the calls that these tests
make are recorded, without making them, and what each would launch is looked up.
"""
import itertools
import os
import re
import subprocess

import pytest

import test_gpu_mxfp4 as products
import test_gpu_routing as routing
import test_gpu_sort_launches as sort_tests
from ruy_amd import _structs as S
from ruy_amd import build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def launched(tmp_path_factory):
    """f(lines): of each the kernels' names."""
    exe = str(tmp_path_factory.mktemp("expert_routes") / "expert_routes_test")
    here = os.path.join(ROOT, "ruy_amd")
    rocm = os.path.dirname(os.path.dirname(build.HIPCC))
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-rdynamic", "-D__HIP_PLATFORM_AMD__",
                           "-I" + os.path.join(rocm, "include"), "-I" + os.path.join(ROOT, "include"),
                           "-I" + build.CSRC, os.path.join(ROOT, "tests", "cpp", "expert_routes_test.cc"),
                           "-L" + here, "-lruy_amd", "-Wl,-rpath," + here,
                           "-Wl,-rpath-link," + os.path.join(rocm, "lib"), "-o", exe])

    def run(lines):
        answers = subprocess.run([exe], input="\n".join(lines) + "\n", capture_output=True, text=True, check=True).stdout.splitlines()
        assert len(answers) == len(lines) and all(a.split()[0] == "0" for a in answers)
        return [a.split()[1:] for a in answers]
    return run


# ---- Sorting ----

SORT_NAMES = ("CountKernel", "AddUpKernel", "PlaceKernel")


def sort_launches(launched, shapes):
    """1 or 3 for each (tokens, top, count)."""
    out = []
    for type_ in (S.I32, S.I64):
        names = launched(["sort %d %d %d %d" % (type_, *s) for s in shapes])
        for one in names:
            assert [n for n in one if "SortByExpertKernel" in n] == one[:1] or all(x in n for x, n in zip(SORT_NAMES, one)) and len(one) == 3
        out.append([len(n) for n in names])
    assert out[0] == out[1]
    return out[0]


def test_both_ways_of_sorting_are_tested(launched):
    shapes = [s for s in routing.SORTS if s[0] * s[1]]
    taken = sort_launches(launched, shapes)
    assert taken == [3 if s in routing.SORTS[-6:] else 1 for s in shapes]
    # With empty experts, of two contexts at once, and of many choices.
    assert sort_launches(launched, [(50, 2, 8), (20000, 8, 128), (9001, 7, 1000), (200000, 1, 4), (1 << 20, 2, 64)]) == [1, 3, 3, 3, 3]


def test_sorts_in_three_launches_are_recorded(launched):
    assert set(sort_launches(launched, sort_tests.THREE_LAUNCHES)) == {3}
    marks = [m for m in sort_tests.test_many_experts_and_the_line_between_one_launch_and_three.pytestmark if m.name == "parametrize"]
    shapes = next(m.args[1] for m in marks if "tokens" in m.args[0])
    assert sort_launches(launched, shapes) == [1 if c > 16384 or (t, p, c) == (49152, 1, 4) else 3 for t, p, c in shapes]


# ---- Products of 4-bit floats ----

def tile_of(name):
    """The tile of a kernel, as the arguments that force it."""
    if "MxFp4StreamKernel" in name:
        return (16, 16, 0)
    if "MxFp4LargeKernel" in name:
        return (256, 256, 0)
    if "MxFp4WideKernel" in name:
        return (256, 128, 0)
    if "GenericMxFp4Kernel" in name:
        return None
    wm, wn, bm, bn, _, stages = map(int, re.search(r"MxFp4GemmKernelILi(\d+)ELi(\d+)ELi(\d+)ELi(\d+)ELb(\d)ELi(\d+)E", name).groups())
    return (wm * bm * 16, wn * bn * 16, int(stages == 4))


class Recorder:
    """Stands in for a context and, as run_mul, for a call's making."""

    def __init__(self):
        self.tile, self.lines, self.forced, self.usable = (0, 0, 0), [], [], []

    def force_tile(self, rows=0, cols=0, deep=0):
        self.tile = (rows, cols, deep)

    def last_kernel_name(self):
        return "mxfp4_stream" if self.tile == (16, 16, 0) else "mxfp4_mfma"

    def run_mul(self, context, dst_type, m, n, k, offsets=None, pads=(0, 0, 0, 0), shift=0, gap=0, dst_order=0, *rest, **more):
        assert context is self
        count = 0 if offsets is None else len(offsets) - 1
        row, blocks = (k + 1) // 2, -(-k // 32)
        lhs, rhs = (row + pads[0], blocks + pads[1]), (row + pads[2], blocks + pads[3])
        matrix = m * lhs[0] + gap
        self.lines.append("mxfp4 " + " ".join(str(int(v)) for v in (
            dst_type, dst_order, m, n, k, count, *lhs, matrix, m * lhs[1] + gap, *rhs, shift, *self.tile)))
        self.forced.append(self.tile)
        direct = k % 32 == 0 and all(v % 4 == 0 for v in (shift, lhs[0], rhs[0], matrix))
        self.usable.append({
            (16, 16, 0): k >= 32,
            (64, 64, 0): k >= 32,
            (128, 128, 0): k >= 32,
            # (Its scales of the whole depth are in LDS.)
            (64, 64, 1): direct and k >= 32 and 4 * 128 * 128 + -(-k // 512) * 2048 <= 156 << 10,
        }.get(self.tile, direct and k >= 512))


def recorded(monkeypatch, test):
    """The calls of a GPU test, over all of its parameters."""
    recorder = Recorder()
    monkeypatch.setattr(products, "run_mul", recorder.run_mul)
    marks = [m for m in test.pytestmark if m.name == "parametrize"]
    names = [[n.strip() for n in m.args[0].split(",")] for m in marks]
    for values in itertools.product(*(m.args[1] for m in marks)):
        arguments = {}
        for n, v in zip(names, values):
            arguments.update(zip(n, v if len(n) > 1 else (v,)))
        test(context=recorder, **arguments)
    return recorder


@pytest.mark.parametrize("test", [
    products.test_every_tile_at_every_end_of_the_depth, products.test_every_tile_at_every_alignment, products.test_streams,
    products.test_tiles_of_four_stages, products.test_tiles_of_steps_of_128, products.test_the_largest_tile,
    products.test_tiles_left_after_full_rounds], ids=lambda t: t.__name__)
def test_forced_tiles_run_where_they_can(launched, monkeypatch, test):
    calls = recorded(monkeypatch, test)
    names = launched(calls.lines)
    assert all(len(n) == 1 for n in names)
    ran = [tile_of(n[0]) for n in names]
    for line, tile, forced, usable in zip(calls.lines, ran, calls.forced, calls.usable):
        assert tile is not None and (tile == forced) == usable, (line, tile)
    # Every tile that the test is about runs: how many of its calls, of how many.
    counts = {f: (sum(t == f for t, g in zip(ran, calls.forced) if g == f), calls.forced.count(f)) for f in set(calls.forced)}
    print(counts)
    assert all(here >= 8 for here, _ in counts.values()), counts


def test_tiles_of_scales_at_any_address_run(launched):
    """The calls of the GPU test of that name: rows of data at multiples of 4 bytes, scales anywhere."""
    lines, forced = [], []
    marks = {m.args[0]: m.args[1] for m in products.test_scales_at_any_address.pytestmark if m.name == "parametrize"}
    for tile, k in itertools.product(marks["tile"], marks["k"]):
        for pad, shift in ((0, 0), (1, 4), (2, 12), (3, 4)):
            row, blocks = k // 2, k // 32
            lines.append("mxfp4 %d 0 300 140 %d 0 %d %d 0 0 %d %d %d %d %d %d" % (S.BF16, k, row, blocks + pad, row + 16, blocks, shift, *tile))
            lines.append("mxfp4 %d 0 70 300 %d 4 %d %d %d %d %d %d %d %d %d %d" % (
                S.F32, k, row + 4, blocks, 70 * (row + 4) + 4 * pad + 4, 70 * blocks + 4 * pad + 4, row, blocks + pad, shift, *tile))
            forced += [tile, tile]
    assert [tile_of(n[0]) for n in launched(lines)] == forced
