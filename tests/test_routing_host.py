"""The calls around the experts' products and for 4-bit floats on the host side:
structs, the native call path, the oracle of 4-bit floats. No device is needed."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest
import torch

import mxfp4_reference as Q
from ruy_amd import _structs as S
from ruy_amd import api
from ruy_amd._capi import lib, native

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_struct_layouts_match_the_header(tmp_path):
    fields = {"ruyamd_routing": S.Routing, "ruyamd_mxfp4_mat": S.MxFp4Mat}
    lines = ['printf("%%zu\\n", sizeof(%s));' % name for name in fields]
    lines += ['printf("%%zu\\n", offsetof(%s, %s));' % (name, f) for name, t in fields.items() for f, _ in t._fields_]
    lines += ['printf("%d\\n", RUYAMD_DTYPE_I64);']
    src = tmp_path / "probe.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "ruy_amd/c_api.h"\nint main(void) {\n%s\nreturn 0; }\n'
                   % "\n".join(lines))
    exe = str(tmp_path / "probe")
    subprocess.check_call(["gcc", "-I" + os.path.join(ROOT, "include"), str(src), "-o", exe])
    got = [int(x) for x in subprocess.check_output([exe]).split()]
    want = [C.sizeof(t) for t in fields.values()] + [getattr(t, f).offset for t in fields.values() for f, _ in t._fields_]
    assert got == want + [S.I64]


def matrix(rows, cols, dtype=S.F32, data=1 << 40):
    return api.Matrix(dtype, data, api.Layout(rows, cols, rows + 2, 0))


def test_the_native_call_path_gathers_what_to_struct_does():
    if native is None:
        pytest.skip("no native call path for this interpreter")
    seen = []

    def fake(types):
        def call(ctx, *pointers):
            seen.append((ctx, [C.string_at(p, C.sizeof(t)) if p else None for p, t in zip(pointers, types)]))
            return 5
        return C.CFUNCTYPE(C.c_int, *[C.c_void_p] * (1 + len(types)))(call)

    m, r, x, g, p = S.Mat, S.Routing, S.MxFp4Mat, S.Groups, S.MulParamsStruct
    types = [(m, r), (m, r, m), (m, r, m, m), (m, m, r, m, m, m), (m, r, x), (x, m), (x, x, g, p, m)]
    callbacks = [fake(t) for t in types]
    native.bind_calls([C.cast(f, C.c_void_p).value for f in callbacks], api.Routing, api.MxFp4Matrix)
    try:
        a, b, c = matrix(3, 5), matrix(8, 2, S.BF16, torch.zeros(20, dtype=torch.bfloat16)), matrix(1, 1, S.I64, np.zeros(3))
        routing = api.Routing(5, 2, 7, torch.zeros(8, dtype=torch.int32), 1 << 33, None)
        held = api.MxFp4Matrix(3, 64, torch.zeros(96, dtype=torch.uint8), 1 << 35, 33, 4, 1 << 36, 9)
        other = api.MxFp4Matrix(2, 64, 1 << 34, np.zeros(4, np.uint8))
        groups, params = api.Groups(np.zeros(4, np.int32), 3, 0, 9), api.MulParams(S.F32, S.F32)
        params.set_clamp_min(0.0)
        for which, objects in [(0, (c, routing)), (1, (a, routing, b)), (2, (a, routing, None, b)), (2, (a, routing, c, b)),
                               (3, (a, None, routing, None, b, None)), (3, (a, b, routing, c, b, c)), (4, (a, None, held)),
                               (4, (a, routing, held)), (5, (held, a)), (6, (held, other, None, params, a)),
                               (6, (held, other, groups, params, a))]:
            assert native.call(which, 77, *objects) == 5
            ctx, got = seen.pop()
            assert ctx == 77
            for o, bytes_, t in zip(objects, got, types[which]):
                if o is None:
                    assert bytes_ is None
                    continue
                # (A struct's padding is not looked at.)
                end = t.reserved.offset + t.reserved.size if hasattr(t, "reserved") else C.sizeof(t)
                assert bytes_[:end] == bytes(o.to_struct())[:end]

        # What is left to the Python code, and mistakes.
        class Mine(api.Routing):
            pass
        assert native.call(0, 77, c, Mine(1, 1, 1, None, None)) is None
        assert native.call(5, 77, a, held) is None
        assert native.call(1, 77, a, routing, None) is None
        assert native.call(0, 77, c, api.Routing(1.5, 1, 1, None, None)) is None
        for wrong in [(7, 77, a, b), (-1, 77, a, b), (0, 77, c), (0,), ()]:
            with pytest.raises(TypeError):
                native.call(*wrong)
        assert not seen
    finally:
        native.bind_calls([C.cast(f, C.c_void_p).value for f in api._CALLS], api.Routing, api.MxFp4Matrix)


def test_a_null_context_is_refused():
    for f in api._CALLS:
        assert f(None, *[None] * (len(f.argtypes) - 1)) == S.E_INVALID


def test_a_product_whose_parameters_are_of_another_type_is_refused():
    with pytest.raises(ValueError):
        api.mul_mxfp4(None, None, api.MulParams(S.F32, S.BF16), None, matrix(2, 2))


def test_the_oracle_of_4_bit_floats():
    x = np.array([[0, -0.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 7, -0.26, 0.74, 4, -6, 7.9, -5.1]])
    n, s = Q.quantize(x)
    # The largest is 7.9 = 1.975 * 2^2: the scale is 1.
    assert s.tolist() == [[127]]
    assert n[0].tolist() == [0, 8, 0, 2, 2, 4, 4, 6, 6, 7, 9, 1, 6, 15, 7, 15]
    assert Q.values(n, s)[0].tolist() == [0, 0, 0, 1, 1, 2, 2, 4, 4, 6, -0.5, 0.5, 4, -6, 6, -6]
    assert (Q.unpack(Q.pack(n), 16) == n).all()
    n, s = Q.quantize(np.array([[0.0] * 32 + [np.inf, 1.0] + [0.0] * 30 + [2.0 ** -149]]))
    assert s.tolist() == [[0, 255, 0]] and not n.any() and np.isnan(Q.values(n, s)[0, 32:64]).all()
    # A block's values come back where they are on its grid.
    y = Q.values(np.arange(16, dtype=np.uint8)[None], np.array([[130]], np.uint8))
    n, s = Q.quantize(y)
    assert (Q.values(n, s) == y).all()


def test_a_torch_tensor_of_places_keeps_its_groups():
    r = api.Routing(4, 2, 3, 1 << 30, 1 << 31)
    g = r.groups(7, 9).to_struct()
    assert (g.offsets, g.count, g.matrix_stride, g.bias_stride) == (1 << 30, 3, 7, 9)
    assert lib.ruyamd_version()
