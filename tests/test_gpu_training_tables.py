"""Which table a gradient belongs to: fields with the same tensor share one, tensors over the same memory do not, and tables
that need no gradient take none."""
import pytest
import torch

import _training as ref

pytestmark = pytest.mark.gpu

BATCH, ROWS, DIM = 30, 40, 24


def randn(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def make_fields(fields, seed=0, rows=ROWS, max_len=6):
    """(values, global offsets, per field the ids and the samples that they belong to)"""
    gen = torch.Generator().manual_seed(seed)
    lens = torch.randint(0, max_len + 1, (fields, BATCH), generator=gen)
    values = torch.randint(-1, rows + 1, (int(lens.sum()),), generator=gen)
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), lens.reshape(-1).cumsum(0)])
    parts = [(values[offsets[f * BATCH]:offsets[(f + 1) * BATCH]].clamp(0, rows - 1), torch.repeat_interleave(torch.arange(BATCH), lens[f]))
             for f in range(fields)]
    return values, offsets, parts


def assert_gradient(got, parts, grad, fields, dim=DIM, rows=ROWS, padding=None, mean=False):
    """`got` is the sum over these fields' ids."""
    ids = torch.cat([parts[f][0] for f in fields])
    g = torch.cat([grad[:, f * dim:(f + 1) * dim][parts[f][1]] for f in fields])
    weights = None
    if mean:
        weights = torch.cat([1.0 / torch.bincount(parts[f][1], minlength=BATCH)[parts[f][1]].double() for f in fields])
    want, absolute, count = ref.table_gradient(g, ids, rows, padding=padding, weights=weights)
    ref.assert_within(got, want, ref.gradient_bound(want, absolute, count, got.dtype, mean))


@pytest.mark.parametrize("detached", [(0,), (1,), (0, 2), (1, 2)])
def test_a_table_and_its_detached_alias(pkg, dev, detached):
    """The gradient is cut off where the table is detached, in any order of the fields."""
    fields = 3
    values, offsets, parts = make_fields(fields)
    grad = randn(1, BATCH, fields * DIM)
    w = randn(2, ROWS, DIM).to(dev).requires_grad_()
    tables = [w.detach() if f in detached else w for f in range(fields)]
    pkg.embedding_bag_train(values.to(dev), offsets.to(dev), tables).backward(grad.to(dev))
    assert w.grad is not None
    assert_gradient(w.grad, parts, grad, [f for f in range(fields) if f not in detached])


def test_two_leaves_over_one_memory(pkg, dev):
    values, offsets, parts = make_fields(4)
    grad = randn(1, BATCH, 4 * DIM)
    a = randn(2, ROWS, DIM).to(dev).requires_grad_()
    b = a.detach().requires_grad_()
    pkg.embedding_bag_train(values.to(dev), offsets.to(dev), [a, b, b, a]).backward(grad.to(dev))
    assert_gradient(a.grad, parts, grad, [0, 3])
    assert_gradient(b.grad, parts, grad, [1, 2])


def test_views_of_one_table_add_up(pkg, dev):
    """A table and a view of it that autograd knows: both fields' gradients arrive at the leaf."""
    values, offsets, parts = make_fields(3)
    grad = randn(1, BATCH, 3 * DIM)
    w = randn(2, ROWS, DIM).to(dev).requires_grad_()
    pkg.embedding_bag_train(values.to(dev), offsets.to(dev), [w, w.view_as(w), w]).backward(grad.to(dev))
    want, absolute, count = ref.table_gradient(torch.cat([grad[:, f * DIM:(f + 1) * DIM][parts[f][1]] for f in range(3)]),
                                               torch.cat([p[0] for p in parts]), ROWS)
    # two sums, each rounded, and their sum: two roundings more
    ref.assert_within(w.grad, want, ref.gradient_bound(want, absolute, count + 2, torch.float32))


def test_a_shared_table_has_one_gradient(pkg, dev):
    values, offsets, parts = make_fields(4)
    grad = randn(1, BATCH, 4 * DIM)
    a, b = (randn(s, ROWS, DIM).to(dev).requires_grad_() for s in (2, 3))
    pkg.embedding_bag_train(values.to(dev), offsets.to(dev), [a, b, a, b], "mean", padding_idx=1).backward(grad.to(dev))
    assert_gradient(a.grad, parts, grad, [0, 2], padding=1, mean=True)
    assert_gradient(b.grad, parts, grad, [1, 3], padding=1, mean=True)


def test_tables_may_change_before_the_backward_pass(pkg, dev):
    """As with the other differentiable operators: the gradient reads no table."""
    values, offsets, parts = make_fields(2)
    grad = randn(1, BATCH, 2 * DIM)
    tables = [randn(s, ROWS, DIM).to(dev).requires_grad_() for s in (2, 3)]
    out = pkg.embedding_bag_train(values.to(dev), offsets.to(dev), tables)
    with torch.no_grad():
        for t in tables:
            t.add_(1.0)
    out.backward(grad.to(dev))
    for f, t in enumerate(tables):
        assert_gradient(t.grad, parts, grad, [f])


@pytest.mark.parametrize("dims", [(24, 24, 24, 24), (128, 128, 128, 128), (7, 64, 300, 1)])
@pytest.mark.parametrize("frozen", [(0,), (3,), (1, 2), (0, 2, 3)])
@pytest.mark.parametrize("padding", [None, 0, 5])
@pytest.mark.parametrize("max_len", [6, 200])  # ids of one tile, and of several
def test_frozen_tables_take_no_part(pkg, dev, dims, frozen, padding, max_len):
    gen = torch.Generator().manual_seed(max_len)
    rows, fields = (40, 9, 17, 30), len(dims)
    lens = torch.randint(0, max_len + 1, (fields, BATCH), generator=gen)
    values = torch.randint(-1, 41, (int(lens.sum()),), generator=gen)
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), lens.reshape(-1).cumsum(0)])
    grad = randn(1, BATCH, sum(dims))
    tables = [randn(f, rows[f], dims[f]).to(dev).requires_grad_(f not in frozen) for f in range(fields)]
    pkg.embedding_bag_train(values.to(dev), offsets.to(dev), tables, "mean", padding_idx=padding).backward(grad.to(dev))
    for f, t in enumerate(tables):
        if f in frozen:
            assert t.grad is None
            continue
        ids = values[offsets[f * BATCH]:offsets[(f + 1) * BATCH]].clamp(0, rows[f] - 1)
        sample = torch.repeat_interleave(torch.arange(BATCH), lens[f])
        col = sum(dims[:f])
        want, absolute, count = ref.table_gradient(grad[:, col:col + dims[f]][sample], ids, rows[f], padding=padding,
                                                   weights=1.0 / lens[f][sample].double())
        ref.assert_within(t.grad, want, ref.gradient_bound(want, absolute, count, torch.float32, True), f"field {f}")


def test_frozen_tables_take_no_memory(pkg, dev):
    values, offsets, parts = make_fields(2)
    big = torch.zeros(2 ** 20, DIM, device=dev)  # 96 MiB
    w = randn(2, ROWS, DIM).to(dev).requires_grad_()
    grad = randn(1, BATCH, 2 * DIM)
    out = pkg.embedding_bag_train(values.to(dev), offsets.to(dev), [big, w])
    grad_dev = grad.to(dev)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out.backward(grad_dev)
    assert torch.cuda.max_memory_allocated() - before < 2 ** 24
    assert_gradient(w.grad, parts, grad, [1])


def test_tangents_are_refused(pkg, dev):
    """Forward mode: no result without its tangent."""
    w, x, one = randn(1, ROWS, DIM).to(dev), randn(2, 6, DIM).to(dev), torch.ones(DIM, device=dev)
    ids = torch.arange(6, device=dev)
    for call, t in ((lambda t: pkg.embedding_lookup(ids, t), w), (lambda t: pkg.dropout(t, 0.5, 1), x),
                    (lambda t: pkg.dropout(x, 0.5, 1, residual=t), x), (lambda t: pkg.dropout_add_layer_norm(t, one, one), x),
                    (lambda t: pkg.dropout_add_layer_norm(x, t, one), one),
                    (lambda t: pkg.embedding_bag_train(ids, torch.tensor([0, 3, 6], device=dev), [t]), w)):
        with torch.autograd.forward_ad.dual_level():
            with pytest.raises(ValueError, match="tangent"):
                call(torch.autograd.forward_ad.make_dual(t, torch.ones_like(t)))
            call(t)


@pytest.mark.parametrize("shapes", [((1, 24), (24,)), ((24,), (1, 24)), ((24, 1, 1), (2, 12))])
def test_norm_parameters_of_any_dimensions(pkg, dev, shapes):
    """Accepted by the forward pass where they have as many elements as columns; each gradient has its parameter's shape."""
    x, gy = randn(1, 6, 24).to(dev).requires_grad_(), randn(2, 6, 24).to(dev)
    w, b = (randn(3 + i, *s).to(dev).requires_grad_() for i, s in enumerate(shapes))
    flat = [t.detach().reshape(24).requires_grad_() for t in (w, b)]
    y = pkg.dropout_add_layer_norm(x, w, b)[0]
    y.backward(gy)
    dx, x.grad = x.grad, None
    pkg.dropout_add_layer_norm(x, *flat)[0].backward(gy)
    assert torch.equal(dx, x.grad)
    for t, f in zip((w, b), flat):
        assert t.grad.shape == t.shape and torch.equal(t.grad.reshape(24), f.grad)


def test_training_step_follows_the_batchs_tile_order(pkg, dev, monkeypatch):
    """As pooled() does, and with the same result bit for bit."""
    import sys

    slots, dim, batch, rows = 28, 128, 64, 500
    gen = torch.Generator().manual_seed(1)
    lens = torch.randint(0, 12, (slots, batch), generator=gen)
    values = torch.randint(0, rows, (int(lens.sum()),), generator=gen)
    row_offsets = torch.zeros(slots, batch + 1, dtype=torch.int64)
    row_offsets[:, 1:] = lens.cumsum(1)
    val_offsets = (lens.sum(1).cumsum(0) - lens.sum(1)).to(dev)
    order = pkg.make_tile_order(row_offsets.reshape(-1), batch, slots, torch.bfloat16, dim).to(dev)
    enc = pkg.RepEncoder(rows, dim, slot_num=slots, d_model=16).to(dev).bfloat16()
    flat = {"_flat_values": values.to(dev), "_val_offsets": val_offsets, "_flat_row_offsets": row_offsets.reshape(-1).to(dev)}
    module, seen = sys.modules[pkg.__name__ + ".training"], []
    pooled = module.fused_all_slots_embedding
    monkeypatch.setattr(module, "fused_all_slots_embedding", lambda *a, **kw: (seen.append(kw.get("tile_order")), pooled(*a, **kw))[1])
    out = []
    for case in (flat, {**flat, "_tile_order": order}):
        enc.zero_grad()
        y = enc.forward_train(case, dropout=0.2, seed=3, offset=1)
        y.float().square().sum().backward()
        out.append([y.detach(), *(p.grad.clone() for p in enc.parameters())])
    assert seen[0] is None and seen[1] is order
    assert all(torch.equal(a, b) for a, b in zip(*out))


@pytest.mark.parametrize("frozen", [(), (0,), (1, 4)])
@pytest.mark.parametrize("padding,pooling,max_len", [(None, "sum", 6), (0, "mean", 6), (3, "sum", 300), (None, "mean", 0)])
def test_sparse_gradients_of_tables_per_field(pkg, dev, frozen, padding, pooling, max_len):
    """The rows that occur, each once and in order, with the whole gradients' bits where the same call gives these; tables that
    share, frozen ones between; no ids at all."""
    values, offsets, parts = make_fields(5, seed=max_len, rows=ROWS, max_len=max_len)
    grad = randn(1, BATCH, 5 * DIM).to(dev)
    a, b, c, d = (randn(s, ROWS + 7 * s, DIM).to(dev) for s in (0, 1, 2, 3))
    tables = [a, b, c, a, d]  # field 3 shares field 0's
    for f in frozen:
        tables[f] = tables[f].detach()
    leaves = {id(t): t.requires_grad_() for f, t in enumerate(tables) if f not in frozen}
    grads = []
    for sparse in (False, True):
        for t in leaves.values():
            t.grad = None
        out = pkg.embedding_bag_train(values.to(dev), offsets.to(dev), tables, pooling, padding_idx=padding, sparse_grad=sparse)
        out.backward(grad)
        grads.append([t.grad for t in leaves.values()])
    for whole, sparse in zip(*grads):
        assert sparse.is_sparse and sparse.shape == whole.shape and sparse.dtype == whole.dtype
        rows = sparse._indices()[0]  # (torch drops the mark that they are in order)
        assert bool((rows[1:] > rows[:-1]).all()) and torch.equal(sparse.to_dense(), whole)
        assert padding is None or not bool((rows == padding).any())
    assert all(tables[f].grad is None for f in frozen)
    ids = [p[0].unique() for p in parts]
    first = list(leaves.values())[0]
    if first is a:  # fields 0 and 3
        occur = torch.cat([ids[0], ids[3]]).unique()
        occur = occur[occur != padding] if padding is not None else occur
        # ids of the larger tables are not clamped to ROWS there, but a has ROWS rows
        assert torch.equal(grads[1][0]._indices()[0].cpu(), occur)


def test_sparse_gradients_train(pkg, dev):
    """An optimizer of torch's takes them; rows without ids stay."""
    values, offsets, parts = make_fields(2)
    tables = [torch.nn.Parameter(randn(s, 1000, DIM).to(dev)) for s in (2, 3)]
    before = [t.detach().clone() for t in tables]
    opt = torch.optim.SparseAdam(tables, lr=0.1)
    pkg.embedding_bag_train(values.to(dev), offsets.to(dev), tables, sparse_grad=True).square().sum().backward()
    opt.step()
    for f, t in enumerate(tables):
        touched = torch.zeros(1000, dtype=torch.bool)
        ids = values[offsets[f * BATCH]:offsets[(f + 1) * BATCH]].clamp(0, 999)
        touched[ids] = True
        assert torch.equal((t.detach() != before[f]).any(1).cpu(), touched)


@pytest.mark.parametrize("seed", range(30))
def test_any_mix_of_tables(pkg, dev, seed):
    """Fields with tables of their own, shared ones, detached aliases and leaves over one memory, frozen ones; widths alike or not;
    every type; sum and mean; a long bag; whole and sparse."""
    import random

    rng, gen = random.Random(seed), torch.Generator().manual_seed(seed)
    types = [torch.float32, torch.bfloat16, torch.float16]
    fields, batch = rng.choice([1, 2, 5, 13, 64]), rng.choice([1, 7, 33, 200])
    dims = [rng.choice([1, 8, 24, 64, 65, 128, 256])] * fields if rng.random() < 0.5 else [rng.choice([1, 7, 64, 100, 129]) for _ in range(fields)]
    dtype, out_dtype, pooling, padding = rng.choice(types), rng.choice([None, *types]), rng.choice(["sum", "mean"]), rng.choice([None, 0])
    tables = []
    for f in range(fields):
        other = rng.randrange(f) if f and rng.random() < 0.4 else None
        if other is not None and dims[other] == dims[f]:
            tables.append(tables[other] if rng.random() < 0.5 else tables[other].detach().requires_grad_(rng.random() < 0.5))
        else:
            table = torch.randn(rng.choice([1, 5, 100, 3000]), dims[f], generator=gen).to(dtype)
            tables.append(table.to(dev).requires_grad_(rng.random() < 0.7 or f == 0))
    rows = [t.shape[0] for t in tables]
    lens = torch.randint(0, rng.choice([1, 4, 30]) + 1, (fields, batch), generator=gen)
    if rng.random() < 0.4:
        lens[rng.randrange(fields), rng.randrange(batch)] = rng.choice([100, 9000])
    values = torch.cat([torch.randint(-1, rows[f] + 1, (int(lens[f].sum()),), generator=gen) for f in range(fields)])
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), lens.reshape(-1).cumsum(0)])
    trained = {id(t): t for t in tables if t.requires_grad}
    sparse = len({t.shape[1] for t in trained.values()}) == 1 and rng.random() < 0.5
    out = pkg.embedding_bag_train(values.to(dev, rng.choice([torch.int64, torch.int32])), offsets.to(dev), tables, pooling, padding, out_dtype,
                                  sparse_grad=sparse)
    grad = torch.randn(out.shape, generator=gen).to(out.dtype)
    out.backward(grad.to(dev))
    assert all(t.grad is None for t in tables if not t.requires_grad)
    for t in trained.values():
        ids, parts, weights = [], [], []
        for f in range(fields):
            if tables[f] is t:
                sample = torch.repeat_interleave(torch.arange(batch), lens[f])
                ids.append(values[offsets[f * batch]:offsets[(f + 1) * batch]].clamp(0, rows[f] - 1))
                parts.append(grad[:, sum(dims[:f]):sum(dims[:f + 1])].double()[sample])
                weights.append(1.0 / lens[f][sample].double() if pooling == "mean" else torch.ones(sample.numel(), dtype=torch.float64))
        want, absolute, count = ref.table_gradient(torch.cat(parts), torch.cat(ids), t.shape[0], padding=padding, weights=torch.cat(weights))
        assert t.grad.is_sparse == sparse
        ref.assert_within(t.grad.to_dense() if sparse else t.grad, want,
                          ref.gradient_bound(want, absolute, count, t.dtype, pooling == "mean"))
