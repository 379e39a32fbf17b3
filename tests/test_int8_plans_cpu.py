"""The int8 Linear's dispatch rules at sizes past what one launch takes, without a GPU: whether a product is taken goes by
its sizes alone, not by where its operands lie or how large a workspace is."""
import ctypes
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "cti-inference-optimization_amd", "csrc")

# threads of a workgroup of each form; the rows form by the steps of K (128 bytes) that it has
THREADS = {1: 256, 2: 256, 3: 512, 4: 512, 5: 512, 6: 512}


class _Part(ctypes.Structure):
    _fields_ = [("form", ctypes.c_int), ("splits", ctypes.c_int), ("steps", ctypes.c_int),
                ("n_begin", ctypes.c_int32), ("n_end", ctypes.c_int32)]


class _Plan(ctypes.Structure):
    _fields_ = [("parts", ctypes.c_int), ("part", _Part * 2), ("padded", ctypes.c_bool)]


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    work = tmp_path_factory.mktemp("plans8")
    (work / "rules.cpp").write_text(
        '#include "ebag_rules.h"\n'
        'extern "C" int64_t launch_rows(int32_t N, int gated) { return cti::linear8_launch_rows(N, gated != 0); }\n'
        'extern "C" void plan(int64_t M, int32_t N, int32_t K, int gated, int aligned, int64_t ws, cti::Linear8Plan* p,\n'
        "                     int64_t* tiles) {\n"
        "  *p = cti::linear8_plan(M, N, K, gated != 0, aligned != 0, ws);\n"
        "  for (int i = 0; i < p->parts; ++i)\n"
        "    tiles[i] = cti::linear8_tiles(p->part[i].form, M, p->part[i].n_end - p->part[i].n_begin, gated != 0);\n}\n")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{CSRC}",
                    str(work / "rules.cpp"), "-o", str(work / "rules.so")], check=True)
    lib = ctypes.CDLL(str(work / "rules.so"))
    I, P = ctypes.c_int64, ctypes.POINTER
    lib.plan.argtypes = [I, ctypes.c_int32, ctypes.c_int32, ctypes.c_int, ctypes.c_int, I, P(_Plan), P(I)]
    lib.plan.restype = None
    lib.launch_rows.argtypes = [ctypes.c_int32, ctypes.c_int]
    lib.launch_rows.restype = I

    class Rules:
        launch_rows = staticmethod(lib.launch_rows)

        @staticmethod
        def plan(M, N, K, gated, aligned, ws):
            p, tiles = _Plan(), (I * 2)()
            lib.plan(M, N, K, gated, aligned, ws, ctypes.byref(p), tiles)
            return p, tiles

    return Rules


@pytest.mark.parametrize("gated", [0, 1])
def test_every_plan_is_one_that_launches(rules, gated):
    """Fewer than 2^32 threads in a launch, for operands at any address and with any workspace, up to the largest outputs
    that are taken (2^22 - 1 tiles of 256 columns of the weight's rows)."""
    most = (2 ** 22 - 1) * (128 if gated else 256)
    for N in (1, 777, 4096, 32768, 65536, 2 ** 20, 2 ** 22 + 1, 2 ** 24, 2 ** 26, 2 ** 26 + 1, 2 ** 28, most - 1, most):
        step = rules.launch_rows(N, gated)
        assert 1 <= step <= 2 ** 20
        for M in {1, 5, 17, 100, 129, 3000, 2 ** 17, 2 ** 19 + 1, step}:
            if M > step:
                continue
            for K in (1, 16, 100, 1024, 4097, 131071):
                for aligned in (0, 1) if K % 16 == 0 else (0,):
                    for ws in (0, 1 << 62):
                        plan, tiles = rules.plan(M, N, K, gated, aligned, ws)
                        for i, part in enumerate(plan.part[:plan.parts]):
                            rows = 256 if part.steps <= 16 else 512 if part.steps <= 32 else 1024
                            threads = THREADS.get(part.form, rows)
                            assert tiles[i] * threads < 2 ** 32, (M, N, K, aligned, ws, part.form)
                            assert tiles[i] * part.splits * threads < 2 ** 32
                            assert tiles[i] < 2 ** 31


def test_launches_of_ordinary_products_have_as_many_rows_as_before(rules):
    assert all(rules.launch_rows(n, gated) == 2 ** 20 for n in (1, 777, 32768, 100000) for gated in (0, 1))


def test_outputs_are_refused_by_their_size_alone(pkg):
    """(The pointers are not real: nothing is launched.)"""
    c = pkg._capi

    def status(rows, cols, n, gate, q, work, nbytes):
        return c.lib().cti_ebag_linear_int8(q, 256, rows, cols, 256, 256, n, None, c.F32, gate, 256, c.BF16, work, nbytes, None)

    for gate, most in ((c.GATE_NONE, (2 ** 22 - 1) * 256), (c.GATE_SILU, (2 ** 22 - 1) * 128)):
        for rows in (1, 2 ** 20, 2 ** 31 - 1):
            for cols in (16, 100):
                for q, work, nbytes in ((256, None, 0), (257, None, 0), (256, 4096, 1 << 60)):
                    assert status(rows, cols, most + 1, gate, q, work, nbytes) == c.EUNSUPPORTED
                    assert "tiles" in c.last_error()
