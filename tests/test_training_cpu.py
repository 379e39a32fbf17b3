"""Training operators without a GPU: the generator against its published vectors, the size rules against what the
kernels assume, and the refusals of the C ABI (no HIP call is reached)."""
import ctypes
import math
import os
import random
import subprocess

import numpy as np
import pytest
import torch

import _training as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "cti-inference-optimization_amd", "csrc")


@pytest.mark.parametrize("counter,key,want", [
    ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
     (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)),
])
def test_philox_gives_the_published_words(counter, key, want):
    assert tuple(int(w) for w in ref.philox(*counter, *key)) == want


@pytest.mark.parametrize("p", [0.1, 0.5, 0.9])
def test_mask_keeps_the_stated_share(p):
    rows, cols = 512, 1000
    keep = ref.keep_mask(rows, cols, p, seed=7, offset=3)
    share = 1 - ref.threshold(p) / 65536
    # six standard deviations of independent draws
    assert abs(float(keep.double().mean()) - share) < 6 * math.sqrt(share * (1 - share) / (rows * cols))
    # columns, rows, offsets and seeds are independent: agreement of two masks is that of two draws
    for other in (ref.keep_mask(rows, cols, p, 7, 4), ref.keep_mask(rows, cols, p, 8, 3), keep.roll(1, 0), keep.roll(1, 1)):
        agree = share ** 2 + (1 - share) ** 2
        assert abs(float((keep == other).double().mean()) - agree) < 6 * math.sqrt(agree * (1 - agree) / (rows * cols))


class Plan(ctypes.Structure):
    _fields_ = [("tiles", ctypes.c_int64), ("bits", ctypes.c_int), ("digit_bits", ctypes.c_int), ("walk", ctypes.c_bool),
                ("lane_cols", ctypes.c_int), ("log_lanes", ctypes.c_int), ("run", ctypes.c_int), ("blocks", ctypes.c_int), ("workgroups", ctypes.c_int64), ("ids", ctypes.c_int64 * 2),
                ("counts", ctypes.c_int64), ("totals", ctypes.c_int64), ("heads", ctypes.c_int64),
                ("last_rank", ctypes.c_int64), ("inv_len", ctypes.c_int64), ("partial", ctypes.c_int64), ("bytes", ctypes.c_int64)]


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    work = tmp_path_factory.mktemp("train_rules")
    (work / "rules.cpp").write_text(
        '#include "ebag_train_rules.h"\n'
        "using namespace cti;\n"
        'extern "C" uint32_t divide(uint32_t n, uint32_t d) { return ChunkDivide::by(d).quotient(n); }\n'
        'extern "C" void plan(int64_t n, int64_t bags, int64_t dim, int elem, uint32_t rows, int even, GradPlan* p) {\n'
        "  *p = grad_plan(n, bags, dim, elem, rows, even);\n}\n"
        'extern "C" int range_bits(int64_t n, int bits) { return grad_range_bits(n, bits); }\n'
        'extern "C" int form(int64_t cols, int elem, int* chunks) {\n'
        "  const TrainNormForm f = train_norm_form(cols, elem);\n  *chunks = f.chunks;\n  return f.lanes;\n}\n"
        'extern "C" int back_form(int64_t cols, int* chunks) {\n'
        "  const TrainNormForm f = train_norm_back_form(cols);\n  *chunks = f.chunks;\n  return f.lanes;\n}\n"
        'extern "C" int64_t norm_groups(int64_t rows, int64_t cols) { return train_norm_workgroups(rows, cols); }\n'
        'extern "C" int64_t norm_bytes(int64_t rows, int64_t cols) { return train_norm_workspace_bytes(rows, cols); }\n')
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{CSRC}", str(work / "rules.cpp"), "-o",
                    str(work / "rules.so")], check=True)
    lib = ctypes.CDLL(str(work / "rules.so"))
    lib.divide.argtypes, lib.divide.restype = [ctypes.c_uint32] * 2, ctypes.c_uint32
    lib.plan.argtypes = [ctypes.c_int64, ctypes.c_int64, ctypes.c_int64, ctypes.c_int, ctypes.c_uint32, ctypes.c_int,
                         ctypes.POINTER(Plan)]
    lib.form.argtypes = [ctypes.c_int64, ctypes.c_int, ctypes.POINTER(ctypes.c_int)]
    lib.back_form.argtypes = [ctypes.c_int64, ctypes.POINTER(ctypes.c_int)]
    for f in (lib.norm_groups, lib.norm_bytes):
        f.argtypes, f.restype = [ctypes.c_int64] * 2, ctypes.c_int64
    return lib


def test_division_of_chunk_numbers(rules):
    rng = random.Random(0)
    for _ in range(20000):
        d = rng.choice([1, 2, 3, 7, 2 ** 28, rng.randrange(1, 2 ** rng.randrange(1, 31)), 2 ** rng.randrange(31),
                        2 ** rng.randrange(1, 30) + 1, 2 ** rng.randrange(2, 31) - 1])
        top = 2 ** 31 - 1
        for n in (rng.randrange(2 ** 31), 0, top, top // d * d, max(0, top // d * d - 1), d, d - 1):
            assert rules.divide(n, d) == n // d, (n, d)


def test_gradient_plan_holds_what_the_kernels_assume(rules):
    rng = random.Random(1)
    p = Plan()
    for _ in range(4000):
        n, dim = int(2 ** rng.uniform(0, 30)), int(2 ** rng.uniform(0, 22))
        rows, elem = int(2 ** rng.uniform(0, 30.99)), rng.choice([2, 4])
        bags = rng.choice([0, int(2 ** rng.uniform(0, 30))])
        even = rng.random() < 0.5
        rules.plan(n, bags, dim, elem, rows, even, ctypes.byref(p))
        assert p.tiles == -(-n // 4096)
        # every key, the dropped ids' key `rows` too, has its bits; digits have 2 to 11
        assert rows < 2 ** p.bits and 2 <= p.digit_bits <= 11 and -(-p.bits // p.digit_bits) == -(-p.bits // 11)
        # lane groups cover a block of columns; blocks cover the row, and fit the grid
        assert p.log_lanes <= 6 and (1 << p.log_lanes) * p.lane_cols * p.blocks >= dim and p.blocks <= 65535
        assert p.blocks == 1 or p.log_lanes == 6
        assert p.lane_cols in (1, 2, 4, 8) and p.lane_cols * elem <= 16 and (p.blocks - 1) * 64 * p.lane_cols < dim
        if p.walk:
            assert even and dim >= 64 and p.log_lanes == 6 and p.run <= 128 and p.lane_cols <= dim
        else:
            assert p.lane_cols * elem == 16
        groups = 256 >> p.log_lanes
        assert groups * p.run <= 2048 and p.workgroups == -(-n // (groups * p.run))
        assert p.workgroups * 256 < 2 ** 32 and p.workgroups < 2 ** 31
        # parts of the workspace, in their order, neither overlap nor end before what is written there
        ends = [(p.ids[0], n * 8), (p.ids[1], n * 8), (p.counts, (p.tiles << p.digit_bits) * 4), (p.totals, 2048 * 4), (p.heads, (p.workgroups + 1) * 4), (p.last_rank, p.workgroups * 4), (p.inv_len, bags * 4),
                (p.partial, p.workgroups * p.blocks * 2 * (p.lane_cols << p.log_lanes) * 4), (p.bytes, 0)]
        for (a, size), (b, _) in zip(ends, ends[1:]):
            assert a % 256 == 0 and a + size <= b


def test_ranges_of_keys_leave_a_word_for_key_and_position(rules):
    rules.range_bits.argtypes = [ctypes.c_int64, ctypes.c_int]
    for n in [1, 2, 63, 64, 100, 127, 128, 129, 1000, 4096, 8191, 8193, 16384, 32767, 32768, 32769, 10 ** 6]:
        for bits in range(1, 32):
            r = rules.range_bits(n, bits)
            if n > 32768:
                assert r == 0
            if r:
                # positions have 15 bits, the rest of a key 17; a key keeps a bit outside its range's
                assert 1 <= r <= 8 and r < bits and bits - r <= 17 and n <= 2 ** 15


def test_norm_forms_cover_their_rows(rules):
    chunks = ctypes.c_int()
    for cols in [*range(1, 600), 1023, 1024, 1025, 2047, 2049, 4095, 4097, 8191, 8192, 8193, 16383, 16384]:
        for elem in (2, 4):
            lanes = rules.form(cols, elem, ctypes.byref(chunks))
            assert lanes * chunks.value * 8 >= cols and lanes in (8, 16, 32, 64, 128, 256, 512)
        lanes = rules.back_form(cols, ctypes.byref(chunks))
        assert lanes * chunks.value * 8 >= cols and lanes in (8, 16, 32, 64, 128, 256, 512, 1024)
        for rows in (1, 3, 100, 10 ** 6):
            groups = rules.norm_groups(rows, cols)
            assert 1 <= groups <= 1024
            few = rows <= 256 and cols <= 8192  # no second launch, no workspace
            assert rules.norm_bytes(rows, cols) == (0 if few else groups * 2 * -(-cols // 8) * 8 * 4)
    for cols in (16385, 10 ** 6):
        assert rules.form(cols, 2, ctypes.byref(chunks)) == 0 and rules.back_form(cols, ctypes.byref(chunks)) == 0 and 1 <= rules.norm_groups(1000, cols) <= 128 and rules.norm_groups(3, 2 ** 28 - 1) == 1


# ---------------------------------------------------------------------------------------------
# Refusals of the C ABI. Addresses are numbers that nothing reads.
# ---------------------------------------------------------------------------------------------
def test_lookup_refuses(pkg):
    c, f = pkg._capi, pkg.load_library().cti_ebag_lookup
    ok = dict(ids=64, it=c.I64, n=4, w=64, dt=c.BF16, rows=10, stride=8, dim=8, scale=1.0, out=64, odt=c.BF16)
    for change, needle in [(dict(dt=3), "table dtype"), (dict(odt=9), "output dtype"), (dict(it=2), "index type"), (dict(n=-1), "ids"),
                           (dict(dim=0), "dim"), (dict(rows=0), "rows"), (dict(stride=7), "row_stride"), (dict(ids=None), "NULL"),
                           (dict(w=None), "NULL"), (dict(out=None), "NULL")]:
        a = {**ok, **change}
        assert f(*a.values(), None) == c.EINVAL and needle in c.last_error(), change
    assert f(*{**ok, "n": 0, "ids": None, "out": None}.values(), None) == c.OK


def test_lookup_backward_refuses(pkg):
    c, lib = pkg._capi, pkg.load_library()
    size = lib.cti_ebag_backward_workspace_bytes(4, 4, 10, 8, c.SUM)
    ok = dict(grad=64, gdt=c.BF16, ids=64, it=c.I64, n=4, rows=10, dim=8, scale=1.0, pad=-1, out=64, odt=c.F32, rows_out=None,
              count=None, cap=0, ws=256, ws_bytes=size)
    for change, status, needle in [
            (dict(gdt=3), c.EINVAL, "gradient dtype"), (dict(odt=7), c.EINVAL, "output dtype"), (dict(it=5), c.EINVAL, "index type"),
            (dict(n=-1), c.EINVAL, "ids"), (dict(dim=0), c.EINVAL, "dim"), (dict(rows=0), c.EINVAL, "rows"),
            (dict(dim=2 ** 22 + 1), c.EUNSUPPORTED, "dim"), (dict(rows=2 ** 31 - 1), c.EUNSUPPORTED, "rows"),
            (dict(n=2 ** 30 + 1), c.EUNSUPPORTED, "ids"), (dict(pad=10), c.EINVAL, "padding"), (dict(pad=-2), c.EINVAL, "padding"),
            (dict(grad=None), c.EINVAL, "NULL"), (dict(ids=None), c.EINVAL, "NULL"), (dict(out=None), c.EINVAL, "NULL"),
            (dict(rows_out=64), c.EINVAL, "together"), (dict(count=64), c.EINVAL, "together"),
            (dict(rows_out=64, count=64, cap=3), c.EINVAL, "capacity"), (dict(ws=None), c.EWORKSPACE, "needed"),
            (dict(ws_bytes=size - 1), c.EWORKSPACE, "needed"), (dict(ws=264), c.EINVAL, "aligned")]:
        a = {**ok, **change}
        assert lib.cti_ebag_lookup_backward(*a.values(), None) == status and needle in c.last_error(), change
    assert size >= 4 * 4 * 4
    for bad in ((0, 4, 10, 8, 0), (4, -1, 10, 8, 0), (4, 4, 0, 8, 0), (4, 4, 10, 0, 0), (2 ** 30 + 1, 4, 10, 8, 0), (4, 4, 2 ** 31, 8, 0)):
        assert lib.cti_ebag_backward_workspace_bytes(*bad) == 0


def test_fused_backward_refuses(pkg):
    c, lib = pkg._capi, pkg.load_library()
    ok = dict(grad=64, gdt=c.BF16, v=64, it=c.I64, vo=64, ro=64, ot=c.I64, batch=2, slots=3, dim=8, max_idx=9, nnz=4, pool=c.SUM,
              pad=-1, out=64, odt=c.BF16, rows_out=None, count=None, cap=0, ws=256, ws_bytes=1 << 20)
    for change, status, needle in [
            (dict(batch=-1), c.EINVAL, "batch_size"), (dict(slots=-1), c.EINVAL, "num_slots"), (dict(dim=0), c.EINVAL, "dim"),
            (dict(max_idx=-1), c.EINVAL, "max_idx"), (dict(max_idx=2 ** 31), c.EUNSUPPORTED, "max_idx"), (dict(ot=9), c.EINVAL, "offset type"),
            (dict(pool=2), c.EINVAL, "pooling"), (dict(batch=2 ** 29, slots=3), c.EUNSUPPORTED, "bags"), (dict(pad=10), c.EINVAL, "padding"),
            (dict(vo=None), c.EINVAL, "NULL"), (dict(ro=None), c.EINVAL, "NULL"), (dict(out=None), c.EINVAL, "NULL"),
            (dict(ws=None), c.EWORKSPACE, "needed")]:
        a = {**ok, **change}
        assert lib.cti_ebag_fused_all_slots_backward(*a.values(), None) == status and needle in c.last_error(), change


def test_backward_refuses(pkg):
    c, lib = pkg._capi, pkg.load_library()

    def call(tables=(), **kw):
        descs = (c.Table * max(2, len(tables)))()
        base = [dict(data=4096, rows=10, row_stride=8, dim=8, out_col=0), dict(data=8192, rows=20, row_stride=8, dim=8, out_col=8)]
        for d, t in zip(descs, [{**b, **t} for b, t in zip(base, list(tables) + [{}, {}])]):
            for k, v in t.items():
                setattr(d, k, v)
        a = dict(grad=64, gdt=c.F32, stride=16, v=64, it=c.I64, nnz=4, offs=64, batch=2, fields=2, tables=descs, pool=c.SUM, pad=-1,
                 odt=c.F32, out=None, rows_out=None, count=None, cap=0, ws=256, ws_bytes=1 << 20)
        a.update(kw)
        return lib.cti_ebag_backward(*a.values(), None)

    for kw, status, needle in [
            (dict(fields=0), c.EINVAL, "num_fields"), (dict(fields=65), c.EUNSUPPORTED, "num_fields"), (dict(tables=None), c.EINVAL, "tables"),
            (dict(batch=-1), c.EINVAL, "batch_size"), (dict(pool=3), c.EINVAL, "pooling"), (dict(stride=15), c.EINVAL, "columns"),
            (dict(grad=None), c.EINVAL, "NULL"), (dict(offs=None), c.EINVAL, "NULL"), (dict(ws=None), c.EWORKSPACE, "needed"),
            (dict(pad=10), c.EINVAL, "padding")]:
        tables = kw.pop("tables", ())
        got = call(**kw) if tables is not None else lib.cti_ebag_backward(64, c.F32, 16, 64, c.I64, 4, 64, 2, 2, None, 0, -1, c.F32, None,
                                                                           None, None, 0, 256, 1 << 20, None)
        assert got == status and needle in c.last_error(), kw
    for tables, status, needle in [
            ([dict(rows=0)], c.EINVAL, "rows"), ([dict(dim=0)], c.EINVAL, "dim"), ([dict(row_stride=7)], c.EINVAL, "row_stride"),
            ([dict(data=None)], c.EINVAL, "data"), ([dict(out_col=9)], c.EINVAL, "columns"), ([dict(out_col=-1)], c.EINVAL, "columns"),
            ([{}, dict(data=4096)], c.EINVAL, "share"), ([dict(rows=2 ** 30), dict(rows=2 ** 30)], c.EUNSUPPORTED, "rows")]:
        assert call(tables) == status and needle in c.last_error(), tables
    assert call([{}, dict(dim=4)], rows_out=64, count=64, cap=4, out=64) == c.EUNSUPPORTED and "width" in c.last_error()


def test_dropout_and_norm_refuse(pkg):
    c, lib = pkg._capi, pkg.load_library()
    for p in (-0.1, 1.1, float("nan"), float("inf")):
        assert lib.cti_ebag_dropout(64, None, 64, 2, 8, c.F32, p, 1, 0, None, None) == c.EINVAL and "p must be" in c.last_error()
    for args in ((None, None, 64, 2, 8, c.F32), (64, None, None, 2, 8, c.F32), (64, None, 64, -1, 8, c.F32), (64, None, 64, 2, 0, c.F32),
                 (64, None, 64, 2, 8, 3)):
        assert lib.cti_ebag_dropout(*args, 0.1, 1, 0, None, None) == c.EINVAL
    assert lib.cti_ebag_dropout(64, None, 64, 2 ** 31, 8, c.F32, 0.1, 1, 0, None, None) == c.EUNSUPPORTED
    assert lib.cti_ebag_dropout(64, None, 64, 2, 2 ** 28, c.F32, 0.1, 1, 0, None, None) == c.EUNSUPPORTED
    assert lib.cti_ebag_dropout(None, None, None, 0, 8, c.F32, 0.1, 1, 0, None, None) == c.OK

    ok = dict(x=64, res=None, h=64, y=64, rows=2, cols=8, dt=c.F32, g=64, b=64, pt=c.F32, eps=1e-5, p=0.5, seed=1, off=0, state=None,
              mean=64, rstd=64)
    for change, needle in [(dict(x=None), "NULL"), (dict(y=None), "NULL"), (dict(g=None), "NULL"), (dict(mean=None), "NULL"),
                           (dict(h=None), "h is NULL"), (dict(h=None, p=0.0, res=64), "h is NULL"), (dict(eps=-1.0), "eps"),
                           (dict(eps=float("nan")), "eps"), (dict(pt=5), "parameter dtype"), (dict(p=2.0), "p must be")]:
        assert lib.cti_ebag_dropout_layernorm(*{**ok, **change}.values(), None) == c.EINVAL and needle in c.last_error(), change

    size = lib.cti_ebag_dropout_layernorm_backward_workspace_bytes(300, 8)
    ok = dict(grad=64, h=64, gh=None, mean=64, rstd=64, rows=300, cols=8, dt=c.F32, g=64, pt=c.F32, p=0.5, seed=1, off=0, state=None, dx=64,
              dr=None, dg=64, db=64, ws=256, ws_bytes=size)
    for change, status, needle in [
            (dict(grad=None), c.EINVAL, "NULL"), (dict(dx=None), c.EINVAL, "NULL"), (dict(dg=None), c.EINVAL, "NULL"),
            (dict(ws=None), c.EWORKSPACE, "needed"), (dict(ws_bytes=size - 1), c.EWORKSPACE, "needed"), (dict(ws=260), c.EINVAL, "aligned"),
            (dict(p=-1.0), c.EINVAL, "p must be"), (dict(cols=0), c.EINVAL, "cols"), (dict(rows=2 ** 31), c.EUNSUPPORTED, "rows")]:
        assert lib.cti_ebag_dropout_layernorm_backward(*{**ok, **change}.values(), None) == status and needle in c.last_error(), change
    assert size > 0 and lib.cti_ebag_dropout_layernorm_backward_workspace_bytes(0, 8) == 0


def test_python_refuses_host_tensors(pkg):
    ids, w, x = torch.zeros(3, dtype=torch.int64), torch.zeros(5, 8), torch.zeros(2, 8)
    for call in (lambda: pkg.embedding_lookup(ids, w), lambda: pkg.embedding_lookup_backward(torch.zeros(3, 8), ids, 5),
                 lambda: pkg.dropout(x, 0.1, 1), lambda: pkg.dropout_backward(x, 0.1, 1),
                 lambda: pkg.dropout_add_layer_norm(x, x[0], x[0]),
                 lambda: pkg.dropout_add_layer_norm_backward(x, x, x[:, 0], x[:, 0], x[0]),
                 lambda: pkg.embedding_bag_backward(x, ids, torch.zeros(3, dtype=torch.int64), [w]),
                 lambda: pkg.embedding_bag_train(ids, torch.zeros(3, dtype=torch.int64), [w])):
        with pytest.raises(ValueError, match="GPU tensor"):
            call()


def test_int8_encoder_is_not_trained(pkg):
    enc = pkg.RepEncoder(10, 8, padding_idx=0, slot_num=2, d_model=4)
    enc._int8_linear = (None, None)
    with pytest.raises(ValueError, match="not trained"):
        enc.forward_train({})


def test_oracle_notices_planted_mistakes():
    """The bounds are narrow enough to see a lost contribution, a wrong column of the mask and a norm without its mean."""
    g = torch.Generator().manual_seed(0)
    grad, ids = torch.randn(200, 16, generator=g), torch.randint(0, 20, (200,), generator=g)
    want, absolute, count = ref.table_gradient(grad, ids, 20)
    lost, _, _ = ref.table_gradient(grad[1:], ids[1:], 20)
    with pytest.raises(AssertionError):
        ref.assert_within(lost, want, ref.gradient_bound(want, absolute, count, torch.bfloat16))
    ref.assert_within(want.to(torch.bfloat16), want, ref.gradient_bound(want, absolute, count, torch.bfloat16))
    x = torch.randn(30, 24, generator=g)
    a, b = ref.dropped(x, 0.3, 5, 1), ref.dropped(x, 0.3, 5, 2)
    with pytest.raises(AssertionError):
        ref.assert_within(a, b, ref.rounded(b, torch.bfloat16))
    n = ref.Norm64(x, torch.ones(24), torch.zeros(24), 1e-5, 64)
    with pytest.raises(AssertionError):
        ref.assert_within(x * n.rstd, n.y, ref.rounded(n.y, torch.bfloat16, n.e_y))
    n.backward(torch.randn(30, 24, generator=g))
    with pytest.raises(AssertionError):
        ref.assert_within(n.dgamma * (1 + 1e-3), n.dgamma, ref.rounded(n.dgamma, torch.float32, n.e_dgamma))
    assert np.isfinite(float(n.e_dh.max()))
