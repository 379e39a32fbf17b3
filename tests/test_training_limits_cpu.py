"""What a gradient cannot do is refused where the differentiable call is made, not in the backward pass."""
import ctypes
import importlib
import os
import subprocess

import pytest
import torch


@pytest.fixture
def training(pkg):
    return importlib.import_module(pkg.__name__ + ".training")


def wide(rows, dim):
    """A table of any shape that takes no memory."""
    return torch.zeros(1).expand(rows, dim).requires_grad_()


def test_limits_are_the_librarys(pkg, training):
    """Each limit passes, and one more does not, in Python as in C (ids, rows, columns; n = 0 launches nothing that matters here: the
    call ends at its NULL pointers or its workspace)."""
    c, lib = pkg._capi, pkg.load_library()

    def lookup(n, rows, dim):
        return lib.cti_ebag_lookup_backward(64, c.F32, 64, c.I64, n, rows, dim, 1.0, -1, 64, c.F32, None, None, 0, None, 0, None)

    ids, rows, dim = training._MOST_IDS, training._MOST_ROWS, training._MOST_COLUMNS
    for sizes in ((ids, 10, 8), (4, rows, 8), (4, 10, dim)):
        training._check_gradient(sizes[0], 0, *sizes[1:])
        assert lookup(*sizes) == c.EWORKSPACE, sizes
    for sizes in ((ids + 1, 10, 8), (4, rows + 1, 8), (4, 10, dim + 1)):
        with pytest.raises(pkg.EbagError):
            training._check_gradient(sizes[0], 0, *sizes[1:])
        assert lookup(*sizes) == c.EUNSUPPORTED, sizes
    with pytest.raises(pkg.EbagError):
        training._check_gradient(4, ids + 1, 10, 8)

    def fields(n):
        descs = (c.Table * n)()
        for f, d in enumerate(descs):
            d.data, d.rows, d.row_stride, d.dim, d.out_col = 4096 * (f + 1), 10, 8, 8, 8 * f
        return lib.cti_ebag_backward(64, c.F32, 8 * n, 64, c.I64, 4, 64, 2, n, descs, c.SUM, -1, c.F32, None, None, None, 0, None, 0, None)

    assert fields(training._MOST_FIELDS) == c.EWORKSPACE and fields(training._MOST_FIELDS + 1) == c.EUNSUPPORTED


def test_more_fields_than_a_gradient_has(pkg):
    values, offsets = torch.zeros(65, dtype=torch.int64), torch.arange(66)
    with pytest.raises(pkg.EbagError, match="65 fields"):
        pkg.embedding_bag_train(values, offsets, [torch.zeros(5, 8, requires_grad=True)] * 65)
    with pytest.raises(ValueError, match="GPU tensor"):  # without a gradient the limit is not there
        pkg.embedding_bag_train(values, offsets, [torch.zeros(5, 8)] * 65)
    with torch.no_grad(), pytest.raises(ValueError, match="GPU tensor"):
        pkg.embedding_bag_train(values, offsets, [torch.zeros(5, 8, requires_grad=True)] * 65)


@pytest.mark.parametrize("rows,dim", [(2 ** 31 - 1, 4), (5, 2 ** 22 + 1)])
def test_tables_past_the_limits(pkg, rows, dim):
    ids, offsets = torch.zeros(4, dtype=torch.int64), torch.tensor([0, 2, 4])
    for call in (lambda w: pkg.embedding_lookup(ids, w), lambda w: pkg.embedding_bag_train(ids, offsets, [w]),
                 lambda w: pkg.fused_embedding_train(ids, offsets[:1], offsets, w)):
        with pytest.raises(pkg.EbagError, match="no gradient"):
            call(wide(rows, dim))
    half = [wide(2 ** 30, 4), wide(2 ** 30, 4)]
    with pytest.raises(pkg.EbagError, match="no gradient"):  # rows of all tables that have a gradient count
        pkg.embedding_bag_train(ids, torch.arange(5), half)
    with pytest.raises(ValueError, match="GPU tensor"):
        pkg.embedding_bag_train(ids, torch.arange(5), [half[0], half[1].detach()])


def test_ids_and_bags_past_the_limits(pkg):
    def numbers(n):
        return torch.zeros(1, dtype=torch.int64).expand(n)

    few, w, most = numbers(4), torch.zeros(5, 8, requires_grad=True), 2 ** 30
    for call in (lambda k: pkg.embedding_lookup(numbers(most + k), w),
                 lambda k: pkg.embedding_bag_train(numbers(most + k), numbers(2), [w]),
                 lambda k: pkg.embedding_bag_train(few, numbers(most + 1 + k), [w]),
                 lambda k: pkg.fused_embedding_train(numbers(most + k), few[:1], few[:2], w),
                 lambda k: pkg.fused_embedding_train(few, few[:1], numbers(most + 1 + k), w)):
        with pytest.raises(pkg.EbagError, match="no gradient"):
            call(1)
    for call in (lambda: pkg.embedding_lookup(numbers(most), w), lambda: pkg.embedding_bag_train(few, numbers(most + 1), [w])):
        with pytest.raises(ValueError, match="GPU tensor"):  # the limits themselves pass
            call()


def operators(pkg):
    """name, call of one tensor, that tensor's shape: every input through which an operator is differentiable."""
    ids, offsets = torch.zeros(4, dtype=torch.int64), torch.tensor([0, 2, 4])
    x, one = torch.ones(4, 8), torch.ones(8)
    return [("lookup", lambda w: pkg.embedding_lookup(ids, w), (5, 8)), ("dropout", lambda t: pkg.dropout(t, 0.5, 1), (4, 8)),
            ("dropout residual", lambda t: pkg.dropout(x, 0.5, 1, residual=t), (4, 8)),
            ("norm", lambda t: pkg.dropout_add_layer_norm(t, one, one), (4, 8)),
            ("norm residual", lambda t: pkg.dropout_add_layer_norm(x, one, one, residual=t), (4, 8)),
            ("norm weight", lambda t: pkg.dropout_add_layer_norm(x, t, one), (8,)),
            ("norm bias", lambda t: pkg.dropout_add_layer_norm(x, one, t), (8,)),
            ("bags", lambda t: pkg.embedding_bag_train(ids, offsets, [t]), (5, 8)),
            ("second table", lambda t: pkg.embedding_bag_train(ids, torch.arange(5), [torch.zeros(5, 8), t]), (5, 8)),
            ("fused", lambda t: pkg.fused_embedding_train(ids, offsets[:1], offsets, t), (5, 8))]


@pytest.mark.parametrize("which", range(10))
@pytest.mark.parametrize("grad", [True, False])
def test_tangents_are_refused(pkg, which, grad):
    """A dual tensor's tangent is not dropped without a word; outside of it the operator goes its way (here to its refusal of a
    CPU tensor)."""
    name, call, shape = operators(pkg)[which]
    t = torch.ones(shape)
    with torch.set_grad_enabled(grad):
        with torch.autograd.forward_ad.dual_level():
            dual = torch.autograd.forward_ad.make_dual(t, torch.ones(shape))
            with pytest.raises(ValueError, match="tangent"):
                call(dual)
            with pytest.raises(ValueError, match="GPU tensor"):
                call(t)
        with pytest.raises(ValueError, match="tangent"):
            torch.func.jvp(call, (t,), (t,))
        with pytest.raises(ValueError, match="GPU tensor"):
            call(t)


def test_fill_beside_the_sort_stays_within_a_launch(pkg, tmp_path):
    """The most shares of the fill, with the most workgroups of each kind of launch that takes them, are fewer than 2^32 threads; the
    library refuses one share more."""
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cti-inference-optimization_amd", "csrc")
    (tmp_path / "rules.cpp").write_text(
        '#include "ebag_train_rules.h"\nusing namespace cti;\n'
        'extern "C" int64_t shares() { return kGradMostShares; }\n'
        'extern "C" int64_t share() { return kGradFillShare; }\n'
        'extern "C" int range_bits(int64_t n, int bits) { return grad_range_bits(n, bits); }\n'
        'extern "C" int64_t tiles(int64_t n) { return grad_plan(n, 0, 8, 2, 100, false).tiles; }\n')
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{csrc}", str(tmp_path / "rules.cpp"), "-o",
                    str(tmp_path / "rules.so")], check=True)
    lib = ctypes.CDLL(str(tmp_path / "rules.so"))
    for f in (lib.shares, lib.share, lib.tiles):
        f.restype = ctypes.c_int64
    lib.tiles.argtypes, lib.range_bits.argtypes = [ctypes.c_int64], [ctypes.c_int64, ctypes.c_int]
    ranges = max(1 << lib.range_bits(n, bits) for n in (1, 64, 128, 4096, 8193, 32768) for bits in range(1, 32))
    for groups, threads in ((1, 1024), (ranges, 1024), (2048 // 64, 1024), (lib.tiles(2 ** 30), 512)):
        assert (lib.shares() + groups) * threads < 2 ** 32, (groups, threads)
    c, row = pkg._capi, 2 ** 18  # bytes of a row of 2^16 fp32 columns, four shares
    rows = lib.shares() * lib.share() // row + 1
    # without ids: it ends at the limit, or at a launch
    status = pkg.load_library().cti_ebag_lookup_backward(None, c.F32, None, c.I64, 0, rows, 2 ** 16, 1.0, -1, 64, c.F32, None, None, 0, None, 0, None)
    assert status == c.EUNSUPPORTED and "2^38" in c.last_error()


def test_chunks_of_the_widest_rows(tmp_path):
    """A chunk's 8 columns lie within its row, also in rows of 2^31 - 1 columns; arithmetic that wraps ends the program."""
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cti-inference-optimization_amd", "csrc")
    (tmp_path / "chunks.cpp").write_text('''
#include "ebag_train_rules.h"
#include <cstdio>
int main() {
  for (int64_t cols : {8, 9, 15, 16, 1021, (1 << 28) - 1, (1 << 28), 2147483640, 2147483641, 2147483646, 2147483647})
    for (int64_t chunk = 0; chunk * 8 < cols; chunk = chunk == 2 && cols > 64 ? (cols - 1) / 8 - 2 : chunk + 1) {
      const int64_t at = cti::chunk_start(static_cast<int>(chunk * 8), static_cast<int>(cols));
      const int64_t want = chunk * 8 + 8 <= cols ? chunk * 8 : cols - 8;
      if (at != want || at < 0 || at + 8 > cols) return std::printf("%lld %lld: %lld", (long long)cols, (long long)chunk, (long long)at), 1;
    }
}''')
    subprocess.run(["g++", "-std=c++17", "-O1", "-ftrapv", f"-I{csrc}", str(tmp_path / "chunks.cpp"), "-o", str(tmp_path / "chunks")], check=True)
    subprocess.run([str(tmp_path / "chunks")], check=True)
    # and the lookup, which alone takes rows of more than 2^28 columns, goes by it
    text = open(os.path.join(csrc, "ebag_backward.hip")).read()
    assert "chunk_start(col[k], p.dim)" in text and "col[k] + 8" not in text


def test_malformed_calls_are_explained(pkg):
    """The package's errors, with or without a gradient, where an IndexError or a message of torch's stood, or nothing."""
    ids, offsets = torch.zeros(4, dtype=torch.int64), torch.tensor([0, 2, 4])
    table, flat = torch.zeros(5, 8), torch.zeros(8)
    for grad in (False, True):
        w, v, s = (t.clone().requires_grad_(grad) for t in (table, flat, torch.zeros(())))
        for bad in (-1, 5):
            for call in (lambda: pkg.embedding_lookup(ids, w, padding_idx=bad), lambda: pkg.embedding_bag_train(ids, offsets, [w], padding_idx=bad),
                         lambda: pkg.fused_embedding_train(ids, offsets[:1], offsets, w, padding_idx=bad)):
                with pytest.raises(ValueError, match="padding_idx"):
                    call()
        for t in (v, s):
            with pytest.raises(ValueError):
                pkg.embedding_lookup(ids, t)
            with pytest.raises(ValueError, match="2-D"):
                pkg.embedding_bag_train(ids, offsets, [w, t])
            with pytest.raises(ValueError, match="2-D"):
                pkg.fused_embedding_train(ids, offsets[:1], offsets, t)
        for call in (lambda: pkg.embedding_lookup([1, 2], w), lambda: pkg.embedding_bag_train([1, 2], offsets, [w]),
                     lambda: pkg.fused_embedding_train(ids, [0], offsets, w), lambda: pkg.fused_embedding_train(ids, offsets[:1], None, w)):
            with pytest.raises((TypeError, ValueError), match="must be a (torch.Tensor|GPU tensor)"):
                call()
        with pytest.raises(ValueError, match="entries for"):
            pkg.fused_embedding_train(ids, offsets[:1], offsets[:0], w)
    with pytest.raises(ValueError, match="at least one table"):
        pkg.embedding_bag_train(ids, offsets, [])


def test_single_launch_of_the_norm_covers_its_columns(tmp_path):
    """The kernel knows a form's columns a workgroup when it is built, the launch by its size: one rule, of whole chunks, that leaves a
    wavefront's threads a row's share each; the workgroups' sums fit their LDS."""
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cti-inference-optimization_amd", "csrc")
    (tmp_path / "rules.cpp").write_text(
        '#include "ebag_train_rules.h"\nusing namespace cti;\n'
        'extern "C" int lanes(int64_t cols) { return train_norm_back_form(cols).lanes; }\n'
        'extern "C" int columns(int lanes) { return train_norm_few_cols(lanes); }\n'
        'extern "C" int few(int64_t rows, int64_t cols) { return train_norm_few(rows, cols); }\n')
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{csrc}", str(tmp_path / "rules.cpp"), "-o",
                    str(tmp_path / "rules.so")], check=True)
    lib = ctypes.CDLL(str(tmp_path / "rules.so"))
    for f in (lib.lanes, lib.few):
        f.argtypes = [ctypes.c_int64] * (1 if f is lib.lanes else 2)
    for cols in [*range(1, 300), 511, 512, 513, 1024, 1025, 2047, 2048, 2049, 4096, 4097, 8191, 8192]:
        assert lib.few(256, cols) and not lib.few(257, cols)
        columns, threads = lib.columns(lib.lanes(cols)), max(256, lib.lanes(cols))
        assert columns == (64 if cols <= 2048 else 128)
        # chunks of 8 columns a thread; two of those rows of threads add up gamma's and beta's sums
        assert columns % 8 == 0 and threads % (columns // 8) == 0 and 2 * columns // 8 <= threads
    assert not lib.few(1, 8193)
