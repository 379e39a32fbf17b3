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
