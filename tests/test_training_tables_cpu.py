"""The differentiable pooling's way through autograd without a GPU: its two launches replaced by loops."""
import importlib

import pytest
import torch

BATCH, ROWS, DIM = 5, 7, 4


@pytest.fixture
def loops(pkg, monkeypatch):
    """The training module with bags pooled, and their gradients summed, by loops on the CPU."""
    module = importlib.import_module(pkg.__name__ + ".training")

    def pooled(values, offsets, tables, pooling="sum", out_dtype=None):
        fields = len(tables)
        batch = (offsets.numel() - 1) // fields
        return torch.cat([torch.stack([tables[f][values[offsets[f * batch + b]:offsets[f * batch + b + 1]]].sum(0) for b in range(batch)])
                          for f in range(fields)], 1)

    def gradients(index, grad, values, offsets, shapes, alike, dtype, same, *rest, wanted=None, **kw):
        module.asked.append(wanted)
        batch, col, sums = grad.shape[0], 0, {}
        for f, (rows, dim) in enumerate(shapes):
            out = sums.setdefault(same[f] if same is not None else f, torch.zeros(rows, dim, dtype=dtype))
            for b in range(batch):
                for i in values[offsets[f * batch + b]:offsets[f * batch + b + 1]]:
                    out[i] += grad[b, col:col + dim]
            col += dim
        return [sums[same[f] if same is not None else f] if wanted is None or wanted[f] else None for f in range(len(shapes))]

    monkeypatch.setattr(module, "asked", [], raising=False)
    monkeypatch.setattr(module, "embedding_bag_pooled", pooled)
    monkeypatch.setattr(module, "_bag_gradients", gradients)
    return module


def make_fields(fields):
    gen = torch.Generator().manual_seed(fields)
    lens = torch.randint(0, 4, (fields * BATCH,), generator=gen)
    return torch.randint(0, ROWS, (int(lens.sum()),), generator=gen), torch.cat([torch.zeros(1, dtype=torch.int64), lens.cumsum(0)])


def wanted(values, offsets, grad, fields):
    out = torch.zeros(ROWS, DIM)
    for f in fields:
        for b in range(BATCH):
            for i in values[offsets[f * BATCH + b]:offsets[f * BATCH + b + 1]]:
                out[i] += grad[b, f * DIM:(f + 1) * DIM]
    return out


@pytest.mark.parametrize("detached", [(0,), (1,), (0, 2), (1, 2)])
def test_a_detached_alias_adds_nothing(loops, detached):
    values, offsets = make_fields(3)
    w = torch.randn(ROWS, DIM, requires_grad=True)
    out = loops.embedding_bag_train(values, offsets, [w.detach() if f in detached else w for f in range(3)])
    grad = torch.arange(out.numel(), dtype=torch.float32).view_as(out)  # whole numbers: sums are exact in any order
    out.backward(grad)
    assert torch.equal(w.grad, wanted(values, offsets, grad, [f for f in range(3) if f not in detached]))


def test_leaves_over_one_memory_and_shared_tensors(loops):
    values, offsets = make_fields(4)
    a = torch.randn(ROWS, DIM, requires_grad=True)
    b = a.detach().requires_grad_()
    out = loops.embedding_bag_train(values, offsets, [a, b, b, a])
    grad = torch.arange(out.numel(), dtype=torch.float32).view_as(out)
    out.backward(grad)
    assert torch.equal(a.grad, wanted(values, offsets, grad, [0, 3])) and torch.equal(b.grad, wanted(values, offsets, grad, [1, 2]))


def test_tables_may_change_before_the_backward_pass(loops):
    """The gradient reads no table: an optimizer's step in between is no fault."""
    values, offsets = make_fields(2)
    a, b = (torch.randn(ROWS, DIM, requires_grad=True) for _ in range(2))
    out = loops.embedding_bag_train(values, offsets, [a, b])
    with torch.no_grad():
        a.add_(1.0)
        b.zero_()
    grad = torch.arange(out.numel(), dtype=torch.float32).view_as(out)
    out.backward(grad)
    assert torch.equal(a.grad, wanted(values, offsets, grad, [0])) and torch.equal(b.grad, wanted(values, offsets, grad, [1]))


def test_only_tables_that_require_a_gradient_get_one(loops):
    values, offsets = make_fields(4)
    a, b, frozen = torch.randn(ROWS, DIM, requires_grad=True), torch.randn(ROWS, DIM, requires_grad=True), torch.randn(ROWS, DIM)
    out = loops.embedding_bag_train(values, offsets, [frozen, a, frozen, b])
    grad = torch.arange(out.numel(), dtype=torch.float32).view_as(out)
    out.backward(grad)
    assert [tuple(w) for w in loops.asked] == [(False, True, False, True)] and frozen.grad is None
    assert torch.equal(a.grad, wanted(values, offsets, grad, [1])) and torch.equal(b.grad, wanted(values, offsets, grad, [3]))
    out = loops.embedding_bag_train(values, offsets, [a, b, a, b])
    out.backward(grad)
    assert loops.asked[1] is None


def test_gradient_of_some_fields_refuses(pkg):
    """The C ABI; addresses are numbers that nothing reads. Of a field without a gradient only its columns are looked at."""
    c, lib = pkg._capi, pkg.load_library()

    def call(wanted, second=None, **kw):
        descs = (c.Table * 2)()
        rest = dict(data=8192, rows=20, row_stride=8, dim=8, out_col=8)
        for d, t in zip(descs, (dict(data=4096, rows=10, row_stride=8, dim=8, out_col=0), {**rest, **(second or {})})):
            for k, v in t.items():
                setattr(d, k, v)
        a = dict(grad=64, gdt=c.F32, stride=16, v=64, it=c.I64, nnz=4, offs=64, batch=2, fields=2, tables=descs, wanted=wanted, pool=c.SUM,
                 pad=-1, odt=c.F32, out=None, rows_out=None, count=None, cap=0, ws=None, ws_bytes=0)
        a.update(kw)
        status = lib.cti_ebag_backward_fields(*a.values(), None)
        return status, c.last_error()

    for mask in (0, 4, 2 ** 64 - 4):
        status, error = call(mask)
        assert status == c.EINVAL and "no field" in error
    for second in (dict(data=None), dict(rows=0), dict(row_stride=0), dict(data=4096), dict(rows=2 ** 31)):
        assert call(3, second)[0] in (c.EINVAL, c.EUNSUPPORTED), second
        status, error = call(1, second)  # as far as the workspace, which is checked last
        assert status == c.EWORKSPACE and "needed" in error, second
    for second in (dict(dim=0), dict(out_col=9), dict(out_col=-1)):
        assert call(1, second)[0] == c.EINVAL, second
    status, error = call(2, pad=10)  # the first table's rows do not count
    assert status == c.EWORKSPACE, error
    status, error = call(1, pad=10)
    assert status == c.EINVAL and "padding" in error
    # one width is asked of the tables that have a gradient
    compact = dict(rows_out=64, count=64, cap=4, out=64)
    assert call(3, dict(dim=4, row_stride=4), **compact)[0] == c.EUNSUPPORTED
    assert call(1, dict(dim=4, row_stride=4), **compact)[0] == c.EWORKSPACE


def test_rows_of_several_tables_are_told_apart(pkg):
    """Compact rows are numbered one table behind the other."""
    module = importlib.import_module(pkg.__name__ + ".training")
    shapes = [(4, 3), (1, 3), (6, 3), (2, 3)]
    numbers = torch.tensor([0, 3, 5, 9, 10, 11, 12, -1, -1])
    sums = torch.arange(9 * 3, dtype=torch.float32).view(9, 3)
    got = module._sparse_tables((numbers, sums, torch.tensor([7])), shapes)
    want = torch.zeros(13, 3)
    want[numbers[:7]] = sums[:7]
    at = 0
    for g, shape in zip(got, shapes):
        assert g.shape == shape and torch.equal(g.to_dense(), want[at:at + shape[0]])
        at += shape[0]
    assert [g._nnz() for g in got] == [2, 0, 3, 2]
    none = module._sparse_tables((numbers, sums, torch.tensor([0])), shapes)
    assert [g._nnz() for g in none] == [0, 0, 0, 0]


def test_sparse_gradients_need_one_width(pkg):
    ids, offsets = torch.zeros(4, dtype=torch.int64), torch.arange(5)
    wide, narrow = torch.zeros(5, 8, requires_grad=True), torch.zeros(5, 4, requires_grad=True)
    with pytest.raises(pkg.EbagError, match="one width"):
        pkg.embedding_bag_train(ids, offsets, [wide, narrow], sparse_grad=True)
    for tables, sparse in (([wide, narrow.detach()], True), ([wide, narrow], False)):  # only of those that have a gradient
        with pytest.raises(ValueError, match="GPU tensor"):
            pkg.embedding_bag_train(ids, offsets, tables, sparse_grad=sparse)
