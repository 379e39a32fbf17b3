"""The dispatch rules of the int8 operators without a GPU. At sizes past what one launch takes: whether a product is taken
goes by its sizes alone, not by where its operands lie or how large a workspace is. And that the GPU tests reach every form
that the rules can choose."""
import ctypes
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "cti-inference-optimization_amd", "csrc")

# threads of a workgroup of each form; the rows form by the steps of K (128 bytes) that it has
THREADS = {1: 256, 2: 256, 3: 512, 4: 512, 5: 512, 6: 512}


# What of the kernels a product reaches: bits of (form, gated, K split, second part, class of steps of the rows form, rest
# of K in the forms that load whole steps). ways() of one product, draw() of random ones.
WAYS = r"""
#include <cmath>
#include <random>
#include <set>
extern "C" int ways(int64_t M, int32_t N, int32_t K, int gated, int aligned, int workspace, int* out) {
  const int64_t ws = workspace ? cti::linear8_workspace_bytes(M, N, K, gated != 0, aligned != 0) : 0;
  const auto plan = cti::linear8_plan(M, N, K, gated != 0, aligned != 0 && K % 16 == 0, ws);
  for (int i = 0; i < plan.parts; ++i) {
    const cti::Linear8Part& p = plan.part[i];
    const bool rows = p.form == cti::kLinear8Rows, any = p.form == cti::kLinear8Any;
    const int steps = !rows ? 0 : p.steps <= 4 ? 1 : p.steps <= 8 ? 2 : p.steps <= 16 ? 3 : p.steps <= 32 ? 4 : 5;
    const int rest = !rows && !any && !plan.padded && K % cti::kLinear8Step != 0;
    out[i] = p.form * 1000 + steps * 100 + rest * 10 + (i * 4 + (p.splits > 1) * 2 + gated);
  }
  return plan.parts;
}
extern "C" int norm_form(int64_t rows, int64_t cols, int size) {
  const cti::Norm8Form f = cti::norm8_form(rows, cols, 16 / size);
  return f.vectors * 100 + f.waves;
}
extern "C" int draw(uint64_t seed, int count, int* out) {
  std::mt19937_64 g(seed);
  const auto size = [&](int least, int most) {
    return static_cast<int>(std::lround(std::exp(std::uniform_real_distribution<double>(std::log(least), std::log(most))(g))));
  };
  std::set<int> seen;
  for (int i = 0; i < count; ++i) {
    const int step[] = {1, 2, 16, 64, 128}, of = step[g() % 5], gated = g() % 2;
    int M = size(1, 16384), N = size(1, 16384);
    const int K = std::max(of, size(1, 16384) / of * of);
    if (g() % 2) {  // a few columns more than rounds of 256 x 256 tiles
      M = size(200, 16384);
      const int rows = (M + 255) / 256;
      N = std::min(16384, static_cast<int>(1 + g() % 3) * 256 / rows * (gated ? 128 : 256) + size(1, 300));
    }
    int w[2];
    const int n = ways(M, N, K, gated, K % 16 == 0 && g() % 4 != 0, g() % 4 != 0, w);
    seen.insert(w, w + n);
  }
  int n = 0;
  for (int w : seen) out[n++] = w;
  return n;
}
"""


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
        "    tiles[i] = cti::linear8_tiles(p->part[i].form, M, p->part[i].n_end - p->part[i].n_begin, gated != 0);\n}\n"
        + WAYS)
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
        def ways(M, N, K, gated, aligned, workspace):
            w = (ctypes.c_int * 2)()
            return set(w[:lib.ways(I(M), N, K, gated, aligned, workspace, w)])

        @staticmethod
        def norm_form(rows, cols, size):
            return lib.norm_form(I(rows), I(cols), size)

        @staticmethod
        def draw(seed, count):
            w = (ctypes.c_int * 10000)()
            return set(w[:lib.draw(ctypes.c_uint64(seed), count, w)])

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


def test_the_gpu_tests_reach_every_form_of_the_product(rules):
    """Whatever random products reach (of up to 16,384 rows, columns and outputs, plain and gated, at any address, with and
    without a workspace) is in the list of test_gpu_int8_forms.py."""
    import test_gpu_int8_forms as g

    reached = set()
    for rows, cols, n, aligned, workspace, gated in g.CASES:
        reached |= rules.ways(rows, n, cols, gated, aligned, workspace)
    drawn = rules.draw(1, 1000000)
    assert len(drawn) > 110
    assert drawn - reached == set()


@pytest.mark.parametrize("size", [2, 4])
def test_the_gpu_tests_reach_every_form_of_the_norms(rules, size):
    import test_gpu_int8_norm_forms as g

    rng = random.Random(0)
    reached = {rules.norm_form(r, c, size) for r, c in g.shapes(size)}
    drawn = {rules.norm_form(int(2 ** rng.uniform(0, 15)), int(2 ** rng.uniform(0, 16)), size) for _ in range(20000)}
    assert drawn == reached and len(drawn) == 11
