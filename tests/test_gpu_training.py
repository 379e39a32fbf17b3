"""The training operators on the GPU against plain 64-bit forms (tests/_training.py, whose bounds count fp32 roundings and
one rounding of the result): the scaled lookup and its gradient, the pooled bags' gradients, dropout, the norm with dropout
and residual forward and backward, autograd, captured graphs, streams, and the encoder's training step."""
import numpy as np
import pytest
import torch
from torch import nn

import _training as ref

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def randn(seed, *shape, dtype=torch.float32, size=1.0):
    g = torch.Generator().manual_seed(seed)
    return (size * torch.randn(*shape, generator=g)).to(dtype)


def randint(seed, lo, hi, n, dtype=torch.int64):
    return torch.randint(lo, hi, (n,), generator=torch.Generator().manual_seed(seed)).to(dtype)


# ---------------------------------------------------------------------------------------------
# Lookup
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("n,rows,dim,dtype,out,index", [
    (1, 1, 1, "f32", "f32", torch.int64), (1, 100, 4096, "bf16", "bf16", torch.int64), (3, 7, 8, "f16", "f16", torch.int32),
    (1000, 333, 7, "bf16", "f32", torch.int32), (513, 50, 9, "f32", "bf16", torch.int64), (77, 1000, 333, "f16", "f32", torch.int64),
    (20001, 5000, 64, "bf16", "f16", torch.int64), (300, 40, 1000, "f32", "f16", torch.int32)])
def test_lookup(pkg, dev, n, rows, dim, dtype, out, index):
    w = randn(n, rows, dim, dtype=DT[dtype])
    ids = randint(n + 1, -3, rows + 3, n, index)
    got = pkg.embedding_lookup(ids.to(dev), w.to(dev), 1.7, out_dtype=DT[out])
    scale = float(np.float32(1.7))
    want = w.double()[ids.long().clamp(0, rows - 1)] * scale
    assert got.shape == (n, dim) and got.dtype == DT[out]
    ref.assert_within(got, want, ref.rounded(want, DT[out], ref.U32 * want.abs()))


def test_lookup_shapes_strides_and_extreme_ids(pkg, dev):
    w = randn(1, 9, 24, dtype=torch.bfloat16).to(dev)
    ids = torch.tensor([[-2 ** 63, 2 ** 63 - 1, 0], [8, -1, 4]], device=dev)
    got = pkg.embedding_lookup(ids, w[:, :16])  # row stride 24
    assert got.shape == (2, 3, 16) and torch.equal(got, w[:, :16][ids.clamp(0, 8)])
    odd = w.reshape(-1)[1:1 + 9 * 13].view(9, 13)  # rows at odd addresses
    assert torch.equal(pkg.embedding_lookup(ids, odd), odd[ids.clamp(0, 8)])
    out = torch.empty(2, 3, 16, dtype=torch.float32, device=dev)
    assert pkg.embedding_lookup(ids, w[:, :16], out=out) is out and torch.equal(out, w[:, :16][ids.clamp(0, 8)].float())
    assert pkg.embedding_lookup(ids[:0], w).shape == (0, 3, 24)


# ---------------------------------------------------------------------------------------------
# Gradient of the lookup
# ---------------------------------------------------------------------------------------------
def check_gradient(pkg, dev, grad, ids, rows, scale=1.0, padding=None, out=None, compact=True):
    clamped = ids.long().clamp(0, rows - 1)
    want, absolute, count = ref.table_gradient(grad.reshape(-1, grad.shape[-1]), clamped.reshape(-1), rows, float(np.float32(scale)), padding)
    bound = ref.gradient_bound(want, absolute, count, out or grad.dtype)
    d_grad, d_ids = grad.to(dev), ids.to(dev)
    got = pkg.embedding_lookup_backward(d_grad, d_ids, rows, scale, padding, grad_dtype=out)
    assert got.shape == (rows, grad.shape[-1]) and got.dtype == (out or grad.dtype)
    ref.assert_within(got, want, bound, "whole")
    again = pkg.embedding_lookup_backward(d_grad, d_ids, rows, scale, padding, grad_dtype=out)
    assert torch.equal(got, again)
    if compact:
        numbers, sums, k = pkg.embedding_lookup_backward(d_grad, d_ids, rows, scale, padding, grad_dtype=out, compact=True)
        k, present = int(k), torch.nonzero(count)[:, 0]
        assert k == present.numel() and torch.equal(numbers[:k].cpu(), present) and bool((numbers[k:] == -1).all())
        assert torch.equal(sums[:k], got[numbers[:k]])  # the same sums bit for bit
    return got


@pytest.mark.parametrize("n", [1, 2, 63, 255, 4095, 4096, 4097, 20000])
@pytest.mark.parametrize("rows,dim,dtype,out", [(1, 8, "f32", "f32"), (255, 128, "bf16", "bf16"), (256, 3, "f16", "f32"),
                                                (1003, 333, "bf16", "f32"), (70001, 64, "f32", "bf16")])
def test_lookup_gradient(pkg, dev, n, rows, dim, dtype, out):
    check_gradient(pkg, dev, randn(n, n, dim, dtype=DT[dtype]), randint(n + 1, -2, rows + 2, n), rows, out=DT[out])


@pytest.mark.parametrize("dim", [1, 2, 4, 5, 7, 8, 9, 15, 16, 31, 33, 100, 255, 256, 257, 511, 512, 513, 1000, 2049, 4096])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_lookup_gradient_widths(pkg, dev, dim, dtype):
    n, rows = 700, 90
    check_gradient(pkg, dev, randn(dim, n, dim, dtype=DT[dtype]), randint(dim, 0, rows, n, torch.int32), rows, scale=3.3)


@pytest.mark.parametrize("rows", [2, 3, 127, 128, 2 ** 16 - 1, 2 ** 16, 2 ** 17 + 1, 2 ** 24, 2 ** 31 - 2])
def test_lookup_gradient_row_numbers(pkg, dev, rows):
    """Keys of every number of digits, the last row and the dropped ids' key behind it among them."""
    for n in (300, 9000):
        ids = randint(rows % 1000, 0, rows, n)
        ids[::7], ids[1::7], ids[2::7] = rows - 1, 0, 2 ** 40
        grad = randn(n, n, 8)
        clamped = ids.clamp(0, rows - 1)
        present, place = torch.unique(clamped[clamped != 0], return_inverse=True)
        want, absolute, count = ref.table_gradient(grad[clamped != 0], place, present.numel())
        numbers, sums, k = pkg.embedding_lookup_backward(grad.to(dev), ids.to(dev), rows, padding_idx=0, compact=True)
        k = int(k)
        assert torch.equal(numbers[:k].cpu(), present) and bool((numbers[k:] == -1).all())
        ref.assert_within(sums[:k], want, ref.gradient_bound(want, absolute, count, torch.float32))


@pytest.mark.parametrize("n,dim", [(5000, 128), (40000, 512), (70000, 24), (3000, 1500)])
@pytest.mark.parametrize("shape", ["one", "two", "runs", "sorted"])
def test_lookup_gradient_of_hot_rows(pkg, dev, n, dim, shape):
    """Keys that cross lane groups and workgroups: one row hit by every id, a few, runs of every length up to thousands."""
    rows = 3000
    ids = {"one": torch.full((n,), 7), "two": torch.arange(n) % 2 * 100, "sorted": torch.arange(n) * rows // n,
           "runs": torch.repeat_interleave(torch.arange(rows), torch.arange(rows) ** 2 // 500)[:n]}[shape]
    grad = randn(n, ids.numel(), dim, dtype=torch.bfloat16)
    check_gradient(pkg, dev, grad, ids, rows, out=torch.float32)
    check_gradient(pkg, dev, grad, ids[torch.randperm(ids.numel(), generator=torch.Generator().manual_seed(1))], rows, padding=7)


@pytest.mark.parametrize("n", [2047, 2048, 2049, 8193, 16385, 24576, 32768])
def test_lookup_gradient_of_one_range_of_rows(pkg, dev, n):
    """All ids in neighbouring rows at one end of a large table: one workgroup of the sort holds them, others none or a few."""
    rows = 200_000
    ids = randint(n, rows - 40, rows + 5, n)
    check_gradient(pkg, dev, randn(n, n, 16), ids, rows)
    ids[::1000] = 3
    ids[5::700] = 100_001
    check_gradient(pkg, dev, randn(n + 1, n, 16), ids, rows, padding=rows - 1)


@pytest.mark.parametrize("fields,batch,long", [(9, 800, None), (2, 900, (1000, 3000)), (3, 30, (40, 20_000)), (1, 20_000, (7, 1024)),
                                               (1, 18_000, (17_999, 1025))])
def test_gradient_of_bags_in_small_tiles(pkg, dev, fields, batch, long):
    """Some ten thousand ids in bags: empty and short ones, one over many tiles, one that ends with or just behind a tile."""
    rows, dim, empty = 700, 24, 0.9 if batch >= 18_000 else 0.2
    lens, values, _, val_offsets, row_offsets = make_bags(batch, fields, batch, [rows] * fields, 10, empty=empty, long=long)
    assert 8192 < values.numel() <= 32768
    grad = randn(batch, batch, fields * dim)
    parts = bag_contributions(lens, values, grad, [dim] * fields, "sum")
    want, absolute, count = ref.table_gradient(torch.cat([p[1] for p in parts]), torch.cat([p[0] for p in parts]).clamp(0, rows - 1), rows)
    got = pkg.fused_all_slots_embedding_backward(grad.to(dev), values.to(dev), val_offsets.to(dev), row_offsets.to(dev), batch, dim, rows - 1)
    ref.assert_within(got, want, ref.gradient_bound(want, absolute, count, torch.float32))


def test_lookup_gradient_of_many_ids(pkg, dev):
    """More tiles than a workgroup adds up by itself, more runs than heads are summed in place."""
    n, rows = 1_300_000, 40_000
    check_gradient(pkg, dev, randn(1, n, 2), randint(2, 0, rows, n, torch.int32), rows)
    # few gradient rows behind many ids, wide ones: 100 bags of 13,000
    d = 512
    grad, ids = randn(3, 1, 100 * d, dtype=torch.bfloat16), randint(4, 0, rows, n)
    slots = torch.arange(100) * (n // 100)
    row_offsets = torch.tensor([0, n // 100]).repeat(100)
    numbers, sums, k = pkg.fused_all_slots_embedding_backward(grad.to(dev), ids.to(dev), slots.to(dev), row_offsets.to(dev), 1, d, rows - 1,
                                                              grad_dtype=torch.float32, compact=True)
    hits = torch.zeros(rows, 100, dtype=torch.float64).index_put_((ids, torch.arange(n) // (n // 100)), torch.ones((), dtype=torch.float64),
                                                                 accumulate=True)
    parts = grad.double().view(100, d)
    want, absolute, count = hits @ parts, hits @ parts.abs(), hits.sum(1)
    k = int(k)
    assert torch.equal(numbers[:k].cpu(), torch.nonzero(count)[:, 0])
    ref.assert_within(sums[:k], want[count > 0], ref.gradient_bound(want, absolute, count, torch.float32)[count > 0])


def test_lookup_gradient_edges(pkg, dev):
    # no ids: zeros, or no rows
    empty = torch.empty(0, 16, device=dev)
    none = torch.empty(0, dtype=torch.int64, device=dev)
    assert not pkg.embedding_lookup_backward(empty, none, 5, out=torch.full((5, 16), 3.0, device=dev)).any()
    numbers, sums, k = pkg.embedding_lookup_backward(empty, none, 5, compact=True)
    assert int(k) == 0 and bool((numbers == -1).all())
    # every id the padding row's
    ids = torch.zeros(100, dtype=torch.int64, device=dev)
    assert not pkg.embedding_lookup_backward(torch.ones(100, 16, device=dev), ids, 5, padding_idx=0).any()
    numbers, _, k = pkg.embedding_lookup_backward(torch.ones(100, 16, device=dev), ids, 5, padding_idx=0, compact=True)
    assert int(k) == 0 and bool((numbers == -1).all())
    # buffers longer than needed: rows behind the last are left as they were
    buffers = (torch.full((500,), 9, dtype=torch.int64, device=dev), torch.full((500, 16), 5.0, device=dev), torch.zeros(1, dtype=torch.int64, device=dev))
    numbers, sums, k = pkg.embedding_lookup_backward(torch.ones(100, 16, device=dev), ids + 3, 5, compact=True, out=buffers)
    assert sums is buffers[1] and int(k) == 1 and numbers[0] == 3 and bool((numbers[1:] == -1).all())
    assert bool((sums[0] == 100).all()) and bool((sums[1:] == 5).all())
    # NaN and infinity stay in their rows
    grad = torch.ones(3, 16, device=dev)
    grad[0, 0], grad[1, 1] = float("nan"), float("inf")
    got = pkg.embedding_lookup_backward(grad, torch.tensor([1, 2, 3], device=dev), 5)
    assert bool(got[1, 0].isnan()) and bool(got[2, 1].isinf()) and bool(got[[0, 3, 4]].isfinite().all())
    # 2-D ids and a gradient at an odd address
    flat = randn(5, 1 + 6 * 10, dtype=torch.bfloat16)
    check_gradient(pkg, dev, flat[1:].view(2, 3, 10), randint(6, 0, 4, 6).view(2, 3), 4)
    odd = flat.to(dev)[1:].view(6, 10)
    assert torch.equal(pkg.embedding_lookup_backward(odd, torch.arange(6, device=dev), 6), odd)


# ---------------------------------------------------------------------------------------------
# Gradient of pooled bags
# ---------------------------------------------------------------------------------------------
def make_bags(seed, fields, batch, rows, max_len, empty=0.2, index=torch.int64, long=None):
    """(lengths [F, B], values, global offsets, val_offsets, row_offsets)"""
    lens = randint(seed, 0, max_len + 1, fields * batch)
    lens[torch.rand(fields * batch, generator=torch.Generator().manual_seed(seed)) < empty] = 0
    if long is not None:
        lens[long[0]] = long[1]
    lens = lens.view(fields, batch)
    values = torch.cat([randint(seed + 1 + f, -2, rows[f] + 2, int(lens[f].sum())) for f in range(fields)]).to(index)
    offsets = torch.zeros(fields * batch + 1, dtype=torch.int64)
    offsets[1:] = lens.reshape(-1).cumsum(0)
    row_offsets = torch.zeros(fields, batch + 1, dtype=torch.int64)
    row_offsets[:, 1:] = lens.cumsum(1)
    return lens, values, offsets, offsets[:-1].view(fields, batch)[:, 0].contiguous(), row_offsets.reshape(-1)


def bag_contributions(lens, values, grad, dims, pooling):
    """Per field: (ids, the bag's part of grad for each, weights)."""
    fields, batch = lens.shape
    at, col, out = 0, 0, []
    for f in range(fields):
        n = int(lens[f].sum())
        sample = torch.repeat_interleave(torch.arange(batch), lens[f])
        weights = 1.0 / lens[f][sample].double() if pooling == "mean" else torch.ones(n, dtype=torch.float64)
        out.append((values[at:at + n].long(), grad[:, col:col + dims[f]].double()[sample], weights))
        at, col = at + n, col + dims[f]
    return out


@pytest.mark.parametrize("fields,batch,rows,dim,max_len,dtype,index,otype", [
    (1, 1, 5, 8, 9, "f32", torch.int64, torch.int64), (3, 50, 40, 64, 12, "bf16", torch.int32, torch.int32),
    (28, 300, 5000, 128, 16, "bf16", torch.int64, torch.int64), (28, 33, 100, 20, 5, "f16", torch.int32, torch.int64),
    (70, 90, 2000, 512, 3, "bf16", torch.int64, torch.int32)])
@pytest.mark.parametrize("pooling", ["sum", "mean"])
def test_shared_table_gradient(pkg, dev, fields, batch, rows, dim, max_len, dtype, index, otype, pooling):
    lens, values, _, val_offsets, row_offsets = make_bags(fields, fields, batch, [rows] * fields, max_len, index=index,
                                                          long=(fields * batch // 2, 5000))
    grad = randn(batch, batch, fields * dim, dtype=DT[dtype])
    for padding in (None, 0, rows - 1):
        parts = bag_contributions(lens, values, grad, [dim] * fields, pooling)
        ids = torch.cat([p[0] for p in parts]).clamp(0, rows - 1)
        want, absolute, count = ref.table_gradient(torch.cat([p[1] for p in parts]), ids, rows, padding=padding,
                                                   weights=torch.cat([p[2] for p in parts]))
        args = (grad.to(dev), values.to(dev), val_offsets.to(dev, otype), row_offsets.to(dev, otype), batch, dim, rows - 1)
        got = pkg.fused_all_slots_embedding_backward(*args, pooling=pooling, padding_idx=padding, grad_dtype=torch.float32)
        ref.assert_within(got, want, ref.gradient_bound(want, absolute, count, torch.float32, pooling == "mean"))
        numbers, sums, k = pkg.fused_all_slots_embedding_backward(*args, pooling=pooling, padding_idx=padding, compact=True,
                                                                  grad_dtype=torch.float32)
        assert torch.equal(numbers[:int(k)].cpu(), torch.nonzero(count)[:, 0]) and torch.equal(sums[:int(k)], got[numbers[:int(k)]])


@pytest.mark.parametrize("dims,rows,dtype,out", [
    ((64,), (100,), "f32", "f32"), ((32, 64, 128), (500, 20, 3000), "bf16", "bf16"), ((7, 1, 300, 9), (10, 1, 50, 1000), "f16", "f32"),
    ((512, 513), (40, 30), "f32", "bf16"), ((16,) * 64, (50,) * 64, "bf16", "f32")])
@pytest.mark.parametrize("pooling", ["sum", "mean"])
def test_gradients_of_tables_per_field(pkg, dev, dims, rows, dtype, out, pooling):
    fields, batch = len(dims), 120
    lens, values, offsets, _, _ = make_bags(len(dims), fields, batch, rows, 9, long=(3, 2000))
    grad = randn(1, batch, sum(dims), dtype=DT[dtype])
    tables = [torch.zeros(v, d, dtype=DT[out], device=dev) for v, d in zip(rows, dims)]
    got = pkg.embedding_bag_backward(grad.to(dev), values.to(dev), offsets.to(dev), tables, pooling, padding_idx=0)
    for f, (ids, g, w) in enumerate(bag_contributions(lens, values, grad, dims, pooling)):
        want, absolute, count = ref.table_gradient(g, ids.clamp(0, rows[f] - 1), rows[f], padding=0, weights=w)
        assert got[f].shape == tables[f].shape and got[f].dtype == DT[out]
        ref.assert_within(got[f], want, ref.gradient_bound(want, absolute, count, DT[out], pooling == "mean"), f"field {f}")
    if len(set(dims)) == 1:
        numbers, sums, k = pkg.embedding_bag_backward(grad.to(dev), values.to(dev), offsets.to(dev), tables, pooling, padding_idx=0, compact=True)
        whole, k = torch.cat(got), int(k)
        assert bool((numbers[k:] == -1).all()) and torch.equal(sums[:k], whole[numbers[:k]])
        rest = torch.ones(whole.shape[0], dtype=torch.bool, device=dev)
        rest[numbers[:k]] = False
        assert not whole[rest].any() and bool((numbers[1:k] > numbers[:k - 1]).all())


def test_fields_that_share_a_table(pkg, dev):
    batch, dims, rows = 60, [24, 24, 24, 24], [100, 80, 100, 80]
    lens, values, offsets, _, _ = make_bags(5, 4, batch, rows, 7)
    grad = randn(2, batch, sum(dims))
    a, b = torch.zeros(100, 24, device=dev), torch.zeros(80, 24, device=dev)
    got = pkg.embedding_bag_backward(grad.to(dev), values.to(dev), offsets.to(dev), [a, b, a, b])
    assert got[0] is got[2] and got[1] is got[3]
    parts = bag_contributions(lens, values, grad, dims, "sum")
    for f, r in ((0, 100), (1, 80)):
        want, absolute, count = ref.table_gradient(torch.cat([parts[f][1], parts[f + 2][1]]),
                                                   torch.cat([parts[f][0], parts[f + 2][0]]).clamp(0, r - 1), r)
        ref.assert_within(got[f], want, ref.gradient_bound(want, absolute, count, torch.float32))
    numbers, sums, k = pkg.embedding_bag_backward(grad.to(dev), values.to(dev), offsets.to(dev), [a, b, a, b], compact=True)
    assert torch.equal(sums[:int(k)], torch.cat(got[:2])[numbers[:int(k)]])


def test_bags_that_leave_ids_out(pkg, dev):
    """Ids before the first bag, between slots and behind the last count for none; offsets past the ids are clipped; far more
    empty bags than ids."""
    values = randint(1, 0, 30, 200)
    grad = randn(3, 2, 2 * 16)
    # slot 0: ids 10..50 and 50..60; slot 1: 100..120 and 120..(past the end)
    val_offsets, row_offsets = torch.tensor([10, 100]), torch.tensor([0, 40, 50, 0, 20, 1000])
    got = pkg.fused_all_slots_embedding_backward(grad.to(dev), values.to(dev), val_offsets.to(dev), row_offsets.to(dev), 2, 16, 29)
    g = grad.view(2, 2, 16)
    parts = [(values[10:50], g[0, 0]), (values[50:60], g[1, 0]), (values[100:120], g[0, 1]), (values[120:], g[1, 1])]
    want, absolute, count = ref.table_gradient(torch.cat([p[1].expand(p[0].numel(), 16) for p in parts]), torch.cat([p[0] for p in parts]), 30)
    ref.assert_within(got, want, ref.gradient_bound(want, absolute, count, torch.float32))
    # 60,000 bags, of which every 999th has ids
    batch = 60_000
    lens = torch.zeros(batch, dtype=torch.int64)
    lens[5::999] = 3
    values = randint(4, 0, 30, int(lens.sum()))
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), lens.cumsum(0)])
    grad = randn(5, batch, 8)
    got, = pkg.embedding_bag_backward(grad.to(dev), values.to(dev), offsets.to(dev), [torch.zeros(30, 8, device=dev)])
    want, absolute, count = ref.table_gradient(grad[torch.repeat_interleave(torch.arange(batch), lens)], values, 30)
    ref.assert_within(got, want, ref.gradient_bound(want, absolute, count, torch.float32))
    # no ids, no samples
    t = torch.zeros(30, 8, device=dev)
    none = torch.empty(0, dtype=torch.int64, device=dev)
    assert not pkg.embedding_bag_backward(grad.to(dev), none, torch.zeros(batch + 1, dtype=torch.int64, device=dev), [t])[0].any()
    assert not pkg.embedding_bag_backward(torch.empty(0, 8, device=dev), none, torch.zeros(1, dtype=torch.int64, device=dev), [t])[0].any()


# ---------------------------------------------------------------------------------------------
# Dropout
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 4096), (3, 7), (17, 8), (5, 9), (300, 64), (33, 1021), (70000, 3), (2, 20001)])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_dropout(pkg, dev, rows, cols, dtype):
    x, res = randn(1, rows, cols, dtype=DT[dtype]), randn(2, rows, cols, dtype=DT[dtype])
    for p, seed, offset in ((0.1, 5, 0), (0.5, 2 ** 64 - 1, 2 ** 40 + 3), (0.0, 1, 1), (1.0, 1, 1), (1e-6, 3, 0), (0.999, 2 ** 33, 9)):
        want = ref.dropped(x, p, seed, offset)
        got = pkg.dropout(x.to(dev), p, seed, offset)
        ref.assert_within(got, want, ref.rounded(want, DT[dtype], 2 * ref.U32 * want.abs()))
        assert not got.cpu()[want == 0].any()
        both = want + res.double()
        got = pkg.dropout(x.to(dev), p, seed, offset, residual=res.to(dev))
        ref.assert_within(got, both, ref.rounded(both, DT[dtype], 3 * ref.U32 * (want.abs() + both.abs())))
        assert torch.equal(pkg.dropout_backward(x.to(dev), p, seed, offset), pkg.dropout(x.to(dev), p, seed, offset))


def test_dropout_in_place_shapes_and_states(pkg, dev):
    x = randn(1, 3, 5, 16, dtype=torch.bfloat16).to(dev)
    want = pkg.dropout(x.view(15, 16), 0.3, 11, 7)
    assert torch.equal(pkg.dropout(x, 0.3, 11, 7).view(15, 16), want)
    res = randn(2, 3, 5, 16, dtype=torch.bfloat16).to(dev)
    added = pkg.dropout(x, 0.3, 11, 7, residual=res)
    y = x.clone()
    assert pkg.dropout(y, 0.3, 11, 7, out=y) is y and torch.equal(y.view(15, 16), want)
    r = res.clone()
    assert torch.equal(pkg.dropout(x, 0.3, 11, 7, residual=r, out=r), added)
    # (seed, offset) from the device, the call's own offset added; wraps at 2^64
    state = torch.tensor([11, 5], device=dev)
    assert torch.equal(pkg.dropout(x, 0.3, state, 2).view(15, 16), want)
    assert torch.equal(pkg.dropout(x, 0.3, torch.tensor([11, -1], device=dev), 8).view(15, 16), want)
    # what is dropped is 0 whatever it was
    bad = torch.full((64, 64), float("nan"), device=dev)
    got = pkg.dropout(bad, 0.5, 1)
    keep = ref.keep_mask(64, 64, 0.5, 1, 0).to(dev)
    assert bool(got[keep].isnan().all()) and not got[~keep].any()
    assert not pkg.dropout(bad, 1.0, 1).any()
    assert pkg.dropout(x[:0], 0.3, 1).shape == (0, 5, 16)


# ---------------------------------------------------------------------------------------------
# Norm
# ---------------------------------------------------------------------------------------------
def depth(cols):
    """Additions on an element's way into a row's sum: 8 columns of up to 4 chunks, lanes, wavefronts; wide rows by 1,024 threads."""
    return 32 + 6 + 8 if cols <= 16384 else 8 * (-(-cols // 8192)) + 6 + 16


def check_norm(pkg, dev, rows, cols, dtype, params, p, residual, grad_h, seed=9, offset=4, shift=0.0, eps=1e-5):
    dt, pt = DT[dtype], DT[params]
    x = (randn(1, rows, cols) + shift).to(dt)
    res = randn(2, rows, cols, dtype=dt, size=2.0) if residual else None
    gamma, beta = (1 + randn(3, cols, size=0.1)).to(pt), randn(4, cols, dtype=pt, size=0.1)
    grad, gh = randn(5, rows, cols, dtype=dt), (randn(6, rows, cols, dtype=dt) if grad_h else None)
    d = lambda t: None if t is None else t.to(dev)
    y, h, mean, rstd = pkg.dropout_add_layer_norm(d(x), d(gamma), d(beta), eps, residual=d(res), p=p, seed=seed, offset=offset)
    drop = ref.dropped(x, p, seed, offset)
    want_h = drop + (res.double() if residual else 0)
    ref.assert_within(h, want_h, ref.rounded(want_h, dt, 3 * ref.U32 * (drop.abs() + want_h.abs())), "h")
    n = ref.Norm64(h.cpu(), gamma, beta, float(np.float32(eps)), depth(cols)).backward(grad, gh)
    ref.assert_within(mean[:, None], n.mean, n.e_mean, "mean")
    ref.assert_within(rstd[:, None], n.rstd, n.r_rstd * n.rstd, "rstd")
    ref.assert_within(y, n.y, ref.rounded(n.y, dt, n.e_y), "y")
    back = (d(grad), h, mean, rstd, d(gamma))
    kw = dict(grad_h=d(gh), p=p, seed=seed, offset=offset)
    dx, dgamma, dbeta, dres = pkg.dropout_add_layer_norm_backward(*back, residual=residual, **kw)
    factor = 0.0 if ref.threshold(p) == 65536 else 65536 / (65536 - ref.threshold(p))
    want = ref.dropped(n.dh, p, seed, offset)
    ref.assert_within(dx, want, torch.where(want == 0, 0.0, 1.0) * ref.rounded(want, dt, factor * (n.e_dh + 2 * ref.U32 * n.dh.abs()))
                      if p else ref.rounded(want, dt, n.e_dh), "dx")
    if residual:
        ref.assert_within(dres, n.dh, ref.rounded(n.dh, dt, n.e_dh), "dresidual")
    else:
        assert dres is None
    ref.assert_within(dgamma, n.dgamma, ref.rounded(n.dgamma, pt, n.e_dgamma), "dgamma")
    ref.assert_within(dbeta, n.dbeta, ref.rounded(n.dbeta, pt, n.e_dbeta), "dbeta")
    again = pkg.dropout_add_layer_norm_backward(*back, residual=residual, **kw)
    assert torch.equal(dx, again[0]) and torch.equal(dgamma, again[1]) and torch.equal(dbeta, again[2])


@pytest.mark.parametrize("cols", [1, 2, 7, 8, 9, 63, 64, 65, 127, 128, 200, 256, 333, 512, 513, 1021, 1024, 2047, 2048, 3584, 4096, 5000, 8192,
                                  8193, 14336, 16384, 16385, 20001])
@pytest.mark.parametrize("dtype,params,p,residual,grad_h", [("bf16", "f32", 0.1, True, True), ("f32", "f32", 0.0, False, False),
                                                            ("f16", "f16", 0.5, False, True)])
def test_norm_widths(pkg, dev, cols, dtype, params, p, residual, grad_h):
    check_norm(pkg, dev, 37, cols, dtype, params, p, residual, grad_h)


@pytest.mark.parametrize("rows", [1, 2, 3, 31, 33, 511, 513, 1025, 3001])
@pytest.mark.parametrize("cols,dtype,params", [(40, "bf16", "bf16"), (100, "f32", "bf16"), (600, "f16", "f32"), (1536, "bf16", "f32")])
def test_norm_rows(pkg, dev, rows, cols, dtype, params):
    check_norm(pkg, dev, rows, cols, dtype, params, 0.2, True, False)


@pytest.mark.parametrize("cols", [1, 9, 64, 127, 128, 129, 256, 333, 512, 1021, 2048, 3584, 4096, 5000, 8191, 8192, 8193])
@pytest.mark.parametrize("rows,dtype,params", [(256, "bf16", "bf16"), (257, "bf16", "f32"), (300, "f32", "f16")])
def test_norm_rows_around_the_single_launch(pkg, dev, rows, cols, dtype, params):
    check_norm(pkg, dev, rows, cols, dtype, params, 0.1, True, True)


def test_norm_extremes(pkg, dev):
    check_norm(pkg, dev, 40, 512, "f32", "f32", 0.0, False, False, shift=100.0)  # a mean far from 0
    check_norm(pkg, dev, 5, 256, "bf16", "bf16", 1.0, True, True)                # everything dropped
    check_norm(pkg, dev, 5, 256, "f32", "f32", 1.0, False, False, eps=1e-3)      # rows of zeros
    # no rows: the parameters' gradients are 0
    e = torch.empty(0, 64, device=dev)
    s, w = torch.empty(0, device=dev), torch.ones(64, device=dev)
    assert pkg.dropout_add_layer_norm(e, w, w)[0].shape == (0, 64)
    _, dgamma, dbeta, _ = pkg.dropout_add_layer_norm_backward(e, e, s, s, w)
    assert not dgamma.any() and not dbeta.any()
    # NaN stays in its row, but for the parameters' gradients of every column that it reaches
    x = randn(1, 4, 64).to(dev)
    x[1, 3] = float("nan")
    y = pkg.dropout_add_layer_norm(x, w, w)[0]
    assert bool(y[1].isnan().all()) and bool(y[[0, 2, 3]].isfinite().all())


def test_norm_takes_dropouts_mask(pkg, dev):
    """h is what dropout gives for the same numbers, N-d inputs and a state on the device too."""
    x, res = randn(1, 4, 6, 72, dtype=torch.bfloat16).to(dev), randn(2, 4, 6, 72, dtype=torch.bfloat16).to(dev)
    w = torch.ones(72, device=dev)
    y, h, mean, rstd = pkg.dropout_add_layer_norm(x, w, w, residual=res, p=0.3, seed=5, offset=6)
    assert torch.equal(h, pkg.dropout(x, 0.3, 5, 6, residual=res)) and mean.shape == (4, 6)
    state = torch.tensor([5, 2], device=dev)
    got = pkg.dropout_add_layer_norm(x, w, w, residual=res, p=0.3, seed=state, offset=4)
    assert all(torch.equal(a, b) for a, b in zip(got, (y, h, mean, rstd)))
    a = pkg.dropout_add_layer_norm_backward(y, h, mean, rstd, w, residual=True, p=0.3, seed=5, offset=6)
    b = pkg.dropout_add_layer_norm_backward(y, h, mean, rstd, w, residual=True, p=0.3, seed=state, offset=4)
    assert all(torch.equal(s, t) for s, t in zip(a, b))
    assert torch.equal(a[0] == 0, pkg.dropout(a[3], 0.3, 5, 6) == 0)


# ---------------------------------------------------------------------------------------------
# Autograd, differences, and the operators together
# ---------------------------------------------------------------------------------------------
def test_gradients_against_differences(pkg, dev):
    """Central differences of a 64-bit forward pass against the kernels' gradients. The step's error is below
    h^2 / 6 * |f'''| ~ 1e-6 of the values' size here, that of the kernels (fp32) below 1e-4: 1e-3 holds both."""
    rows, cols, p, seed, offset = 6, 40, 0.3, 3, 1
    x, res, gamma, beta = randn(1, rows, cols).double(), randn(2, rows, cols).double(), 1 + randn(3, cols).double() / 9, randn(4, cols).double()
    gy, gh = randn(5, rows, cols).double(), randn(6, rows, cols).double()
    mask = ref.dropped(torch.ones(rows, cols), p, seed, offset)

    def f(x, res, gamma, beta):
        h = res + mask * x
        dev_ = h - h.mean(1, keepdim=True)
        y = dev_ / torch.sqrt((dev_ ** 2).mean(1, keepdim=True) + 1e-5) * gamma + beta
        return float((y * gy).sum() + (h * gh).sum())

    leaves = [t.float().to(dev).requires_grad_() for t in (x, res, gamma, beta)]
    y, h, _, _ = pkg.dropout_add_layer_norm(leaves[0], leaves[2], leaves[3], 1e-5, residual=leaves[1], p=p, seed=seed, offset=offset)
    ((y * gy.float().to(dev)).sum() + (h * gh.float().to(dev)).sum()).backward()
    args, step = [t.float().double() for t in (x, res, gamma, beta)], 1e-4
    for k, leaf in enumerate(leaves):
        for at in range(0, args[k].numel(), 23):
            moved = [[t.clone() for t in args] for _ in range(2)]
            moved[0][k].view(-1)[at] += step
            moved[1][k].view(-1)[at] -= step
            slope = (f(*moved[0]) - f(*moved[1])) / (2 * step)
            assert abs(float(leaf.grad.view(-1)[at]) - slope) <= 1e-3 * max(1.0, abs(slope)), (k, at)


def test_autograd_of_a_sequence(pkg, dev):
    """Lookup, dropout, norm with a residual, a second use of the table: gradients against torch's in 64 bits."""
    rows, dim, n = 50, 48, 64
    ids, w = randint(1, 0, rows, n).view(4, 16), randn(2, rows, dim)
    gamma, beta, gy, gh = 1 + randn(3, dim) / 9, randn(4, dim), randn(5, 4, 16, dim), randn(6, 4, 16, dim)
    leaves = [t.to(dev).requires_grad_() for t in (w, gamma, beta)]
    e = pkg.embedding_lookup(ids.to(dev), leaves[0], 2.0, padding_idx=3)
    a = pkg.dropout(e, 0.25, 7, 1, residual=e)  # the same input twice
    y, h, _, _ = pkg.dropout_add_layer_norm(a, leaves[1], leaves[2], residual=e, p=0.5, seed=7, offset=2)
    plain, own_h, _, _ = pkg.dropout_add_layer_norm(h, leaves[1], leaves[2])  # neither dropout nor residual: h itself
    assert own_h is h
    ((y + plain) * gy.to(dev) + h * gh.to(dev)).sum().backward()
    w64, g64, b64 = (t.double().requires_grad_() for t in (w, gamma, beta))
    e64 = nn.functional.embedding(ids, w64, padding_idx=3) * 2.0
    m1 = ref.dropped(torch.ones(64, dim), 0.25, 7, 1).view(4, 16, dim)
    m2 = ref.dropped(torch.ones(64, dim), 0.5, 7, 2).view(4, 16, dim)
    h64 = e64 + m2 * (e64 + m1 * e64)
    y64 = nn.functional.layer_norm(h64, (dim,), g64, b64)
    ((2 * y64) * gy.double() + h64 * gh.double()).sum().backward()
    # fp32 throughout: a few hundred roundings of values of size 1 to 100 at the most
    for got, want in zip(leaves, (w64, g64, b64)):
        assert float((got.grad.double().cpu() - want.grad).abs().max()) <= 1e-4 * float(want.grad.abs().max())
    assert not leaves[0].grad[3].any()


def test_autograd_forms(pkg, dev):
    w = randn(1, 30, 16).to(dev).requires_grad_()
    ids = randint(2, 0, 30, 40).to(dev)
    pkg.embedding_lookup(ids, w, sparse_grad=True).sum().backward()  # an expanded gradient
    sparse, w.grad = w.grad, None
    assert sparse.is_sparse and sparse._nnz() == ids.unique().numel()  # no row twice
    pkg.embedding_lookup(ids, w).sum().backward()
    assert torch.equal(sparse.to_dense(), w.grad)
    with pytest.raises(ValueError, match="out does not combine"):
        pkg.embedding_lookup(ids, w, out=torch.empty(40, 16, device=dev))
    with torch.no_grad():
        assert not pkg.embedding_lookup(ids, w).requires_grad
    # only some inputs, only some outputs
    x, r = randn(3, 8, 16).to(dev).requires_grad_(), randn(4, 8, 16).to(dev)
    pkg.dropout(x, 0.5, 1, residual=r).sum().backward()
    assert torch.equal(x.grad, pkg.dropout_backward(torch.ones_like(x), 0.5, 1))
    x.grad = None
    one = torch.ones(16, device=dev)
    _, h, mean, _ = pkg.dropout_add_layer_norm(x, one, one, residual=r, p=0.5, seed=1)
    h.sum().backward()  # y takes no part
    assert torch.equal(x.grad, pkg.dropout_backward(torch.ones_like(x), 0.5, 1)) and not mean.requires_grad
    # bags: shared tables, mean
    tables = [randn(5, 20, 8).to(dev).requires_grad_(), randn(6, 30, 8).to(dev).requires_grad_()]
    values, offsets = randint(7, 0, 20, 60).to(dev), (torch.arange(13) * 5).to(dev)
    pkg.embedding_bag_train(values, offsets, [tables[0], tables[1], tables[0]], "mean", padding_idx=1).square().sum().backward()
    t64 = [t.detach().double().cpu().requires_grad_() for t in tables]
    out = [nn.functional.embedding_bag(values[20 * f:20 * f + 20].cpu(), t64[t], torch.arange(4) * 5, mode="mean")
           for f, t in enumerate((0, 1, 0))]
    torch.cat(out, 1).square().sum().backward()
    for t, want in zip(tables, t64):
        want.grad[1] = 0
        assert float((t.grad.double().cpu() - want.grad).abs().max()) <= 1e-5 * float(want.grad.abs().max())


def test_encoder_training_step(pkg, dev):
    """RepEncoder.forward_train against the reference's modules (segment sums, nn.LayerNorm, nn.Linear) in 64 bits, with the
    dropout's mask given; both batch forms; sparse gradients."""
    slots, dim, rows, batch, d_model = 5, 32, 200, 40, 24
    torch.manual_seed(0)
    enc = pkg.RepEncoder(rows, dim, padding_idx=0, slot_num=slots, d_model=d_model).to(dev)
    lens, values, offsets, val_offsets, row_offsets = make_bags(9, slots, batch, [rows] * slots, 6)
    flat = {"_flat_values": values.to(dev), "_val_offsets": val_offsets.to(dev), "_flat_row_offsets": row_offsets.to(dev)}
    pairs = {f + 1: (values[offsets[f * batch]:offsets[(f + 1) * batch]].to(dev), row_offsets.view(slots, -1)[f].contiguous().to(dev))
             for f in range(slots)}
    gy = randn(10, batch, d_model)
    grads = []
    for case in (flat, pairs):
        enc.zero_grad()
        out = enc.forward_train(case, dropout=0.2, seed=4, offset=8)
        (out * gy.to(dev)).sum().backward()
        grads.append([p.grad.clone() for p in enc.parameters()])
    assert all(torch.equal(a, b) for a, b in zip(*grads))
    ref64 = pkg.RepEncoder(rows, dim, padding_idx=0, slot_num=slots, d_model=d_model).double()
    ref64.load_state_dict({k: v.double().cpu() for k, v in enc.state_dict().items()})
    e = ref64.emb(values.clamp(0, rows - 1))
    bag = torch.repeat_interleave(torch.arange(slots * batch), lens.reshape(-1))
    pooled = torch.zeros(slots * batch, dim, dtype=torch.float64).index_add(0, bag, e).view(slots, batch, dim).transpose(0, 1).reshape(batch, -1)
    mask = ref.dropped(torch.ones(batch, slots * dim), 0.2, 4, 8)
    want = ref64.linear(ref64.input_norm(pooled * mask))
    (want * gy.double()).sum().backward()
    # fp32 sums of at most a few hundred terms on the way
    assert float((out.detach().double().cpu() - want.detach()).abs().max()) <= 1e-4 * float(want.abs().max())
    for (name, p), g in zip(ref64.named_parameters(), grads[0]):
        assert float((g.double().cpu() - p.grad).abs().max()) <= 1e-4 * float(p.grad.abs().max()), name
    assert not grads[0][0][0].any()  # the padding row
    enc.zero_grad()
    (enc.forward_train(flat, dropout=0.2, seed=4, offset=8, sparse_grad=True) * gy.to(dev)).sum().backward()
    assert enc.emb.weight.grad.is_sparse and torch.equal(enc.emb.weight.grad.to_dense(), grads[0][0])
    enc.zero_grad()
    same = enc.forward_train(flat)  # without dropout: forward's result up to the order of the norm's sums
    assert float((same - enc(flat)).abs().max()) <= 1e-4 * float(same.abs().max())


# ---------------------------------------------------------------------------------------------
# Graphs and streams
# ---------------------------------------------------------------------------------------------
def test_captured_training_step(pkg, dev):
    """A step of plain calls (pool, dropout and norm, backward, rows of the table's gradient; a lookup, its whole gradient) in
    a graph: every replay, on new inputs and a new generator state, equals the eager calls bit for bit."""
    slots, dim, rows, batch, n = 6, 64, 3000, 150, 6000
    weight = randn(1, rows, dim, dtype=torch.bfloat16).to(dev)
    gamma, beta = (1 + randn(2, slots * dim) / 9).to(dev), randn(3, slots * dim).to(dev)
    lens, values, _, val_offsets, row_offsets = make_bags(1, slots, batch, [rows] * slots, 20)
    values = torch.cat([values, torch.zeros(20_000 - values.numel(), dtype=torch.int64)])
    inputs = [values.to(dev), val_offsets.to(dev), row_offsets.to(dev), randn(4, batch, slots * dim, dtype=torch.bfloat16).to(dev),
              torch.tensor([5, 0], device=dev), randint(6, 0, rows, n).to(dev), randn(7, n, dim, dtype=torch.bfloat16).to(dev)]

    def step(values, val_offsets, row_offsets, grad, state, ids, grad_rows):
        pooled = torch.empty(batch, slots * dim, dtype=torch.bfloat16, device=dev)
        pkg.fused_all_slots_embedding(values, val_offsets, row_offsets, weight, pooled, batch, dim, rows - 1)
        y, h, mean, rstd = pkg.dropout_add_layer_norm(pooled, gamma, beta, p=0.2, seed=state, offset=1)
        dx, dgamma, dbeta, _ = pkg.dropout_add_layer_norm_backward(grad, h, mean, rstd, gamma, p=0.2, seed=state, offset=1)
        numbers, sums, count = pkg.fused_all_slots_embedding_backward(dx, values, val_offsets, row_offsets, batch, dim, rows - 1, pooling="sum",
                                                                      padding_idx=0, compact=True)
        mean_grad = pkg.fused_all_slots_embedding_backward(dx, values, val_offsets, row_offsets, batch, dim, rows - 1, pooling="mean")
        e = pkg.dropout(pkg.embedding_lookup(ids, weight, 8.0), 0.5, state, 2, residual=grad_rows)
        return [y, h, mean, rstd, dx, dgamma, dbeta, numbers, sums, count, mean_grad, e,
                pkg.embedding_lookup_backward(grad_rows, ids, rows, 8.0)]

    step(*inputs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(*inputs)
    for k in range(4):
        lens, values, _, val_offsets, row_offsets = make_bags(10 + k, slots, batch, [rows] * slots, 20)
        values = torch.cat([values, torch.zeros(20_000 - values.numel(), dtype=torch.int64)])
        fresh = [values, val_offsets, row_offsets, randn(20 + k, batch, slots * dim, dtype=torch.bfloat16), torch.tensor([5 + k, k]),
                 randint(30 + k, 0, rows, n), randn(40 + k, n, dim, dtype=torch.bfloat16)]
        for a, b in zip(inputs, fresh):
            a.copy_(b)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        want = step(*inputs)
        live = int(want[9])
        for i, (a, b) in enumerate(zip(got, want)):
            assert torch.equal(a[:live], b[:live]) if i == 8 else torch.equal(a, b), (k, i)


def test_two_calls_at_once_on_two_streams(pkg, dev):
    n, rows, dim = 30_000, 5000, 128
    ids, grads = [randint(k, 0, rows, n).to(dev) for k in range(2)], [randn(k, n, dim, dtype=torch.bfloat16).to(dev) for k in range(2)]
    want = [pkg.embedding_lookup_backward(g, i, rows) for g, i in zip(grads, ids)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(3):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(pkg.embedding_lookup_backward(grads[k], ids[k], rows))
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(g, want[k]) for g in got[k])


# ---------------------------------------------------------------------------------------------
# Refusals
# ---------------------------------------------------------------------------------------------
def test_refusals(pkg, dev):
    ids, w, g = torch.zeros(4, dtype=torch.int64, device=dev), torch.zeros(9, 16, device=dev), torch.zeros(4, 16, device=dev)
    offs = torch.tensor([0, 2, 4], device=dev)
    bad = [
        (TypeError, lambda: pkg.embedding_lookup(ids.float(), w)), (ValueError, lambda: pkg.embedding_lookup(ids, w.t())),
        (ValueError, lambda: pkg.embedding_lookup(ids, w, out=g[:, :8])), (ValueError, lambda: pkg.embedding_lookup(ids[::2], w)),
        (TypeError, lambda: pkg.embedding_lookup(ids, w.double())), (ValueError, lambda: pkg.embedding_lookup(ids, w[:0])),
        (ValueError, lambda: pkg.embedding_lookup_backward(g, ids[:3], 9)), (ValueError, lambda: pkg.embedding_lookup_backward(g, ids, 0)),
        (ValueError, lambda: pkg.embedding_lookup_backward(g, ids, 9, padding_idx=9)), (ValueError, lambda: pkg.embedding_lookup_backward(g.t(), ids, 9)),
        (ValueError, lambda: pkg.embedding_lookup_backward(g, ids, 9, padding_idx=-1)),
        (ValueError, lambda: pkg.embedding_lookup_backward(g, ids, 9, compact=True, out=w)),
        (ValueError, lambda: pkg.embedding_lookup_backward(g, ids, 9, compact=True, out=(ids[:3], g[:3], ids[:1]))),
        (TypeError, lambda: pkg.embedding_lookup_backward(g, ids, 9, grad_dtype=torch.bfloat16, out=w)),
        (ValueError, lambda: pkg.embedding_bag_backward(g, ids, offs, [w])), (ValueError, lambda: pkg.embedding_bag_backward(g[:2], ids, offs, [])),
        (TypeError, lambda: pkg.embedding_bag_backward(g[:2], ids, offs.int(), [w])),
        (TypeError, lambda: pkg.embedding_bag_backward(g[:2], ids, offs, [(w.to(torch.int8), w[:, 0].contiguous())])),
        (ValueError, lambda: pkg.embedding_bag_backward(g[:2], ids, offs, [w], padding_idx=9)),
        (ValueError, lambda: pkg.embedding_bag_backward(g[:2], ids, offs, [w], pooling="max")),
        (ValueError, lambda: pkg.embedding_bag_backward(g[:1, :].repeat(1, 2), ids, offs, [w, w.clone()], out=[w, w])),
        (ValueError, lambda: pkg.fused_all_slots_embedding_backward(g[:2], ids, offs[:1], offs, 2, 8, 8)),
        (ValueError, lambda: pkg.fused_all_slots_embedding_backward(g[:2], ids, offs[:1], offs[:2], 2, 16, 8)),
        (ValueError, lambda: pkg.dropout(g, 1.5, 1)), (ValueError, lambda: pkg.dropout(g, 0.5, -1)), (ValueError, lambda: pkg.dropout(g, 0.5, 2 ** 64)),
        (ValueError, lambda: pkg.dropout(g, 0.5, 1, -1)), (ValueError, lambda: pkg.dropout(g, 0.5, ids)), (ValueError, lambda: pkg.dropout(g.t(), 0.5, 1)),
        (ValueError, lambda: pkg.dropout(g, 0.5, 1, residual=g[:2])), (TypeError, lambda: pkg.dropout(g.double(), 0.5, 1)),
        (ValueError, lambda: pkg.dropout(g, 0.5, 1, residual=g.bfloat16())), (ValueError, lambda: pkg.dropout(g, float("nan"), 1)),
        (ValueError, lambda: pkg.dropout_add_layer_norm(g, w[0], w[0, :8])), (TypeError, lambda: pkg.dropout_add_layer_norm(g, w[0], w[0].half())),
        (_eb(pkg), lambda: pkg.dropout_add_layer_norm(g, w[0], w[0], eps=-1.0)), (ValueError, lambda: pkg.dropout_add_layer_norm(g, w[0], w[0], residual=g[:2])),
        (ValueError, lambda: pkg.dropout_add_layer_norm_backward(g, g, g[:, 0], g[:, 0].contiguous(), w[0])),
        (ValueError, lambda: pkg.dropout_add_layer_norm_backward(g[:2], g, g[0, :4], g[0, :4], w[0])),
    ]
    for k, (error, call) in enumerate(bad):
        with pytest.raises(error):
            call()
            pytest.fail(f"call {k} was not refused")


def _eb(pkg):
    return pkg.EbagError
