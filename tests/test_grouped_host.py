"""The calls for layers of experts on the host side: structs, defaults, the
native call path. No device is needed."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest
import torch

from ruy_amd import _structs as S
from ruy_amd import api
from ruy_amd._capi import lib, native

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_struct_layouts_match_the_header(tmp_path):
    fields = {"ruyamd_groups": S.Groups, "ruyamd_int4_mat": S.Int4Mat}
    lines = ['printf("%%zu\\n", sizeof(%s));' % name for name in fields]
    lines += ['printf("%%zu\\n", offsetof(%s, %s));' % (name, f) for name, t in fields.items() for f, _ in t._fields_]
    src = tmp_path / "probe.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "ruy_amd/c_api.h"\nint main(void) {\n%s\nreturn 0; }\n'
                   % "\n".join(lines))
    exe = str(tmp_path / "probe")
    subprocess.check_call(["gcc", "-I" + os.path.join(ROOT, "include"), str(src), "-o", exe])
    got = [int(x) for x in subprocess.check_output([exe]).split()]
    want = [C.sizeof(t) for t in fields.values()] + [getattr(t, f).offset for t in fields.values() for f, _ in t._fields_]
    assert got == want


def test_params_of_16_bit_floating_destinations():
    for dtype in (S.BF16, S.F16):
        p = api.MulParams(S.F32, dtype)
        assert (p.clamp_min, p.clamp_max) == (float("-inf"), float("inf"))
        with pytest.raises(ValueError):
            api.MulParams(S.I32, dtype)


def test_the_native_call_path_gathers_what_to_struct_does():
    if native is None:
        pytest.skip("no native call path for this interpreter")
    seen = []

    def copy(pointer, type_):
        return bytes(C.string_at(pointer, C.sizeof(type_))) if pointer else None

    def fake(which, first):
        def call(ctx, lhs, rhs, groups, params, dst):
            # (A struct's padding is not looked at.)
            seen.append((which, ctx, copy(lhs, first)[:first.reserved.offset + 1 if first is S.Mat else None], copy(rhs, S.Mat)[:27], copy(groups, S.Groups),
                         copy(params, S.MulParamsStruct)[:S.MulParamsStruct.reserved.offset + 1], copy(dst, S.Mat)[:27]))
            return 5
        return C.CFUNCTYPE(C.c_int, *[C.c_void_p] * 6)(call)

    callbacks = [fake(0, S.Mat), fake(1, S.Mat), fake(2, S.Int4Mat)]
    real = [C.cast(f, C.c_void_p).value for f in (lib.ruyamd_mul_grouped, lib.ruyamd_mul_grouped_depth, lib.ruyamd_mul_int4)]
    native.bind_with_groups([C.cast(f, C.c_void_p).value for f in callbacks], api.Groups, api.Int4Matrix)
    try:
        lhs = api.Matrix(S.BF16, 1 << 40, api.Layout(3, 5, 7, 1))
        rhs = api.Matrix(S.BF16, torch.zeros(8, dtype=torch.bfloat16), api.Layout(5, 2, 5, 0))
        dst = api.Matrix(S.F32, np.zeros(6, np.float32), api.Layout(3, 2, 3, 0))
        int4 = api.Int4Matrix(3, 5, 32, torch.zeros(9, dtype=torch.uint8), np.zeros(3), S.F16, 1 << 33, 11, 2, 1 << 35, 6)
        params = api.MulParams(S.F32, S.F32)
        params.set_bias(1 << 20)
        params.set_clamp_max(2.5)
        groups = api.Groups(np.zeros(4, np.int32), 3, 1 << 36, 9)
        for which, first, g in [(0, lhs, groups), (1, lhs, groups), (2, int4, groups), (2, int4, None)]:
            assert native.mul_with_groups(which, first, rhs, g, params, 77, dst) == 5
            got = seen.pop()
            assert got[:2] == (which, 77)
            assert got[2] == bytes(first.to_struct())[:len(got[2])]
            assert got[3] == bytes(rhs.to_struct())[:27] and got[6] == bytes(dst.to_struct())[:27]
            assert got[4] == (bytes(g.to_struct()) if g else None)
            assert got[5] == bytes(params.to_struct())[:S.MulParamsStruct.reserved.offset + 1]
        # What is left to the Python code: other classes, another destination type, values that are no integers.
        class Mine(api.Groups):
            pass
        assert native.mul_with_groups(0, lhs, rhs, Mine(None, 1), params, 77, dst) is None
        assert native.mul_with_groups(2, lhs, rhs, groups, params, 77, dst) is None
        assert native.mul_with_groups(0, int4, rhs, groups, params, 77, dst) is None
        assert native.mul_with_groups(0, lhs, rhs, api.Groups(None, 1.5), params, 77, dst) is None
        assert native.mul_with_groups(0, lhs, rhs, groups, api.MulParams(S.F32, S.BF16), 77, dst) is None
        for wrong in [(3, lhs, rhs, groups, params, 77, dst), (-1, lhs, rhs, groups, params, 77, dst), (0,)]:
            with pytest.raises(TypeError):
                native.mul_with_groups(*wrong)
        assert not seen
    finally:
        native.bind_with_groups(real, api.Groups, api.Int4Matrix)


def test_a_null_context_is_refused():
    for f in (lib.ruyamd_mul_grouped, lib.ruyamd_mul_grouped_depth, lib.ruyamd_mul_int4):
        assert f(None, None, None, None, None, None) == S.E_INVALID
