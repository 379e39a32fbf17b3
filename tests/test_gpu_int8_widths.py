"""Rows of every width at which a form of the row quantiser begins or ends, bit for bit the expression that it states."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vectors", [32, 64, 128, 256, 512, 1024, 2048, 4096])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
def test_quantiser_at_the_edges_of_its_forms(pkg, dev, vectors, dt):
    """`vectors` of 16 bytes a row, one element less and one more; at the first element's address and the next one's."""
    per = 16 // torch.empty(0, dtype=dt).element_size()
    for dim in (vectors * per - 1, vectors * per, vectors * per + 1):
        x = torch.randn(23, dim, generator=torch.Generator().manual_seed(dim))
        x[3, dim - 1], x[4, 0], x[5] = 60.0, -60.0, 0.0
        x = x.to(dt)
        want_s = torch.clamp(x.float().abs().amax(1) * np.float32(1 / 127), min=np.float32(1e-8))
        want_q = torch.clamp(torch.round(x.float() / want_s[:, None]), -128, 127).to(torch.int8)
        for shift in (0, 1):
            print(f"quantise dim={dim} {dt} shift={shift}", flush=True)
            view = torch.zeros(23 * dim + shift, dtype=dt, device=dev)[shift:].view(23, dim)
            view.copy_(x)
            q, s = pkg.quantize_embedding_int8(view)
            assert torch.equal(s.cpu(), want_s) and torch.equal(q.cpu(), want_q)


def test_more_rows_than_a_launch_of_four_wavefronts_has(pkg, dev):
    """256 threads a row from 129 vectors on: 2^24 rows are 2^32 threads, which no launch has."""
    rows, dim = 2 ** 24 + 5, 1032
    w = torch.zeros(rows, dim, dtype=torch.bfloat16, device=dev)
    at = torch.tensor([0, 2 ** 24 - 2, 2 ** 24 - 1, 2 ** 24, rows - 1], device=dev)
    some = torch.randn(len(at), dim, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).to(dev)
    w[at] = some
    print("more rows than a launch of four wavefronts has", flush=True)
    for nan_rows in (False, True):
        q, s = pkg.quantize_embedding_int8(w, nan_rows=nan_rows)
        torch.cuda.synchronize()
        want_q, want_s = pkg.quantize_embedding_int8(some)
        assert torch.equal(q[at], want_q) and torch.equal(s[at], want_s)
        assert int((s != np.float32(1e-8)).sum()) == len(at)
        del q
