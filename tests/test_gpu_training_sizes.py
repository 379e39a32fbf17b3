"""Training operators at the ends of their ranges: tensors of more than 2^31 elements, ids that all fall into one range of
keys, widths that end inside a vector, in place."""
import numpy as np
import pytest
import torch

import _training as ref

pytestmark = pytest.mark.gpu


def rows_dropped(x, first, p, seed, offset):
    """Dropout in 64 bits of rows `first` on of a longer tensor."""
    blocks, n = (x.shape[1] + 7) // 8, x.shape[0]
    row, block = np.meshgrid(np.arange(first, first + n, dtype=np.uint64), np.arange(blocks, dtype=np.uint64), indexing="ij")
    words = ref.philox(row, block, offset % 2 ** 32, offset >> 32, seed % 2 ** 32, seed >> 32)
    bits = np.stack([half for w in words for half in (w & np.uint64(0xFFFF), w >> np.uint64(16))], axis=2)
    t = ref.threshold(p)
    keep = torch.from_numpy(bits.astype(np.int64).reshape(n, -1)[:, :x.shape[1]] >= t)
    return torch.where(keep, x.double() * (65536 / (65536 - t)), torch.zeros((), dtype=torch.float64))


def test_more_than_two_billion_elements(pkg, dev):
    rows, cols, last = 2 ** 20 + 3, 2048, 5  # 2^31 elements and more
    g = torch.Generator(device=dev).manual_seed(1)
    x = torch.randn(rows, cols, generator=g, device=dev, dtype=torch.bfloat16)
    tail = x[-last:].cpu()
    got = pkg.dropout(x, 0.25, 7, 2 ** 33 + 1)
    want = rows_dropped(tail, rows - last, 0.25, 7, 2 ** 33 + 1)
    ref.assert_within(got[-last:], want, ref.rounded(want, torch.bfloat16, 2 * ref.U32 * want.abs()), "dropout")
    del got
    w = torch.ones(cols, device=dev)
    y, h, mean, rstd = pkg.dropout_add_layer_norm(x, w, w, p=0.25, seed=7, offset=1)
    n = ref.Norm64(h[-last:].cpu(), torch.ones(cols), torch.ones(cols), float(np.float32(1e-5)), 46).backward(tail)
    ref.assert_within(y[-last:], n.y, ref.rounded(n.y, torch.bfloat16, n.e_y), "y")
    want = rows_dropped(tail, rows - last, 0.25, 7, 1)
    ref.assert_within(h[-last:], want, ref.rounded(want, torch.bfloat16, 2 * ref.U32 * want.abs()), "h")
    del y
    dx, _, _, dres = pkg.dropout_add_layer_norm_backward(x, h, mean, rstd, w, residual=True, p=0.25, seed=7, offset=1)
    ref.assert_within(dres[-last:], n.dh, ref.rounded(n.dh, torch.bfloat16, n.e_dh), "dresidual")
    assert bool(((dx[-last:] == 0) | (h[-last:] != 0)).all())  # nothing of x that was dropped
    del dx, dres, h
    # a table of as many elements: its last rows looked up, and their gradient
    ids = torch.tensor([rows - 1, 0, rows - 2, rows - 1], device=dev)
    assert torch.equal(pkg.embedding_lookup(ids, x), x[ids])
    grad = torch.randn(4, cols, generator=g, device=dev, dtype=torch.bfloat16)
    got = pkg.embedding_lookup_backward(grad, ids, rows, out=x)
    want = grad.double().cpu()
    ref.assert_within(got[rows - 2:], torch.stack([want[2], want[0] + want[3]]),
                      ref.rounded(torch.stack([want[2], want[0] + want[3]]), torch.bfloat16, 3 * ref.U32 * (want[0].abs() + want[3].abs())))
    assert torch.equal(got[0], grad[1]) and not got[1:rows - 2].any()


def test_lookup_and_gradient_of_more_than_two_billion_elements(pkg, dev):
    """As many looked-up elements: ids far apart in the output, and rows of grad past 2^31 elements."""
    n, dim, rows = 2 ** 20 + 7, 2048, 100
    w = torch.randn(rows, dim, device=dev, dtype=torch.bfloat16)
    ids = torch.randint(0, rows - 1, (n,), device=dev, dtype=torch.int32)
    ids[-3:] = rows - 1
    out = pkg.embedding_lookup(ids, w)
    assert torch.equal(out[-2000:], w[ids[-2000:].long()])
    numbers, sums, count = pkg.embedding_lookup_backward(out, ids, rows, grad_dtype=torch.float32, compact=True)
    assert int(count) == rows and int(numbers[rows - 1]) == rows - 1
    want = 3 * w[rows - 1].double().cpu()
    ref.assert_within(sums[rows - 1], want, ref.rounded(want, torch.float32, 3 * ref.U32 * want.abs()))


@pytest.mark.parametrize("n", [4097, 8192, 8193, 16384, 16385, 32768, 32769])
@pytest.mark.parametrize("rows", [2, 300, 40_000, 2 ** 23 + 5])
def test_ids_in_one_range_of_keys(pkg, dev, n, rows):
    """The sort's ranges at their ends: all ids in one range, in every position's order, and next to dropped ones."""
    g = torch.Generator().manual_seed(n)
    for low, high in ((0, 1), (rows // 2, min(rows, rows // 2 + 40)), (0, rows)):
        ids = torch.randint(low, max(high, low + 1), (n,), generator=g)
        grad = torch.randn(n, 8, generator=g)
        live = ids != 0
        present, place = torch.unique(ids[live], return_inverse=True)
        want, absolute, count = ref.table_gradient(grad[live], place, present.numel()) if present.numel() else (None, None, None)
        numbers, sums, k = pkg.embedding_lookup_backward(grad.to(dev), ids.to(dev), rows, padding_idx=0, compact=True)
        k = int(k)
        assert k == present.numel() and torch.equal(numbers[:k].cpu(), present) and bool((numbers[k:] == -1).all())
        if k:
            ref.assert_within(sums[:k], want, ref.gradient_bound(want, absolute, count, torch.float32))


@pytest.mark.parametrize("cols", [*range(1, 26), 31, 33, 255, 1001])
def test_dropout_in_place_at_any_width(pkg, dev, cols):
    """The last chunk of a row is read with its neighbour's columns, which another thread may have written already."""
    g = torch.Generator(device=dev).manual_seed(cols)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        x, r = (torch.randn(513, cols, generator=g, device=dev).to(dtype) for _ in range(2))
        want, added = pkg.dropout(x, 0.4, 3, 1), pkg.dropout(x, 0.4, 3, 1, residual=r)
        y = x.clone()
        assert torch.equal(pkg.dropout(y, 0.4, 3, 1, out=y), want)
        y = r.clone()
        assert torch.equal(pkg.dropout(x, 0.4, 3, 1, residual=y, out=y), added)


def test_wide_norms_on_a_stream_of_their_own(pkg, dev):
    """The forms of wide rows (in LDS, and by columns) from two streams at once, several times: the same bits."""
    cases = []
    for cols in (12_000, 16_383, 17_000):
        g = torch.Generator(device=dev).manual_seed(cols)
        x, r = torch.randn(300, cols, generator=g, device=dev), torch.randn(300, cols, generator=g, device=dev)
        cases.append((x, r, torch.ones(cols, device=dev)))

    def step(x, r, w):
        y, h, mean, rstd = pkg.dropout_add_layer_norm(x, w, w, residual=r, p=0.1, seed=1, offset=2)
        return [y, h, *pkg.dropout_add_layer_norm_backward(x, h, mean, rstd, w, grad_h=r, residual=True, p=0.1, seed=1, offset=2)]

    want = [step(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(2):
        for s in streams:
            with torch.cuda.stream(s):
                got.append([step(*c) for c in cases])
    torch.cuda.synchronize()
    for g in got:
        for a, b in zip(g, want):
            assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_lookups_from_a_captured_graph_and_eager_calls_in_turn(pkg, dev):
    """Two graphs of the same calls replayed in turn with eager calls between: none shares a workspace."""
    w = torch.randn(5000, 96, device=dev)
    ids = [torch.randint(0, 5000, (n,), device=dev) for n in (7000, 40_000)]
    grads = [torch.randn(i.numel(), 96, device=dev) for i in ids]
    graphs, outs = [], []
    for i, g in zip(ids, grads):
        pkg.embedding_lookup_backward(g, i, 5000)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(pkg.embedding_lookup_backward(g + pkg.embedding_lookup(i, w, 0.5), i, 5000))
        graphs.append(graph)
    for k in range(3):
        for i, g in zip(ids, grads):
            i.copy_(torch.randint(0, 5000, (i.numel(),), device=dev))
            g.copy_(torch.randn(g.shape, device=dev))
        for graph in graphs:
            graph.replay()
        want = [pkg.embedding_lookup_backward(g + pkg.embedding_lookup(i, w, 0.5), i, 5000) for i, g in zip(ids, grads)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), k
