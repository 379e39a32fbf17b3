"""Training operators at the largest sizes that they take, and at the ends of the norm's single launch."""
import pytest
import torch

import test_gpu_training as training

pytestmark = pytest.mark.gpu


def test_lookup_of_the_widest_rows(pkg, dev):
    """Rows of 2^31 - 1 columns, several launches: every element, the last chunk's too."""
    dim = 2 ** 31 - 1
    weight = torch.empty(2, dim, dtype=torch.float16, device=dev)
    weight.view(torch.int16).random_(0, 2 ** 14)  # no NaN among these
    ids = torch.tensor([1, 0, 1, 7, -3], device=dev)
    out = pkg.embedding_lookup(ids, weight)
    for i, row in enumerate((1, 0, 1, 1, 0)):
        assert torch.equal(out[i].view(torch.int16), weight[row].view(torch.int16)), i


@pytest.mark.parametrize("rows", [1, 15, 16, 17, 32, 33, 127, 128, 129, 200, 255])  # rounds of 16 and 32 rows, and what is left over
@pytest.mark.parametrize("cols", [64, 77, 512, 520, 1021, 1024, 2040, 2047, 2048, 2049, 4093, 8191])  # by 64 columns and by 128
def test_norm_rows_of_the_single_launch(pkg, dev, rows, cols):
    training.check_norm(pkg, dev, rows, cols, "f16" if cols % 2 else "f32", "f32", 0.2, False, False)


def test_norm_of_a_last_row_that_is_not_finite(pkg, dev):
    """What is read in place of rows past the end counts for nothing, NaN among it."""
    rows, cols = 37, 100
    x = torch.randn(rows, cols, generator=torch.Generator().manual_seed(1)).to(dev)
    w = torch.ones(cols, device=dev)
    _, h, mean, rstd = pkg.dropout_add_layer_norm(x, w, w)
    grad = torch.ones_like(x)
    want = pkg.dropout_add_layer_norm_backward(grad, h, mean, rstd, w)
    grad[-1] = float("nan")
    dx, dweight, dbias, _ = pkg.dropout_add_layer_norm_backward(grad, h, mean, rstd, w)
    assert torch.equal(dx[:-1], want[0][:-1]) and bool(dweight.isnan().all()) and bool(dbias.isnan().all())
    grad[-1] = 0.0  # counted more than once, the row would show
    assert torch.equal(pkg.dropout_add_layer_norm_backward(grad, h, mean, rstd, w)[2], torch.full_like(w, rows - 1))
