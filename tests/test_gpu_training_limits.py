"""Training operators at the largest sizes that they take."""
import pytest
import torch

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
