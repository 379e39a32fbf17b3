"""The int8 norms in every form that their dispatch can choose, for few rows and for many, at widths of whole vectors and
others, against their definitions in 64 bits (on the device).

test_int8_plans_cpu.py holds the shapes against the dispatch rule.
"""
import numpy as np
import pytest
import torch
from test_gpu_int8_serving import U, _norm, _norm_bounds, _norm_reference

pytestmark = pytest.mark.gpu

# vectors of 16 bytes a row: one element more than as many whole ones, and the whole ones
VECTORS = [1, 7, 32, 40, 64, 100, 128, 200, 256, 300, 511, 512, 700, 1024, 1500, 2047, 2048, 3000, 4096, 4200]
ROWS = [3, 1540]
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def shapes(size):
    """(rows, cols) for elements of `size` bytes."""
    return [(r, n * 16 // size + more) for r in ROWS for n in VECTORS for more in (0, 1, -1) if n * 16 // size + more > 0]


@pytest.mark.parametrize("n", VECTORS)
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("dt", TYPES)
def test_norm_forms(pkg, dev, rows, n, dt):
    for cols in sorted({c for r, c in shapes(torch.empty(0, dtype=dt).element_size())
                        if abs(c - n * 16 // torch.empty(0, dtype=dt).element_size()) <= 1}):
        g = torch.Generator(device=dev).manual_seed(rows + cols)
        x, r = ((torch.randn(rows, cols, generator=g, device=dev) + 0.3).to(dt) for _ in range(2))
        for layer, res, pdt in ((False, r, dt), (True, None, dt), (True, r, torch.float32), (False, None, torch.float16)):
            print(f"norm form rows={rows} cols={cols} {dt} layer={layer} res={res is not None} params={pdt}", flush=True)
            w = (1 + 0.2 * torch.randn(cols, generator=g, device=dev)).to(pdt)
            b = (0.2 * torch.randn(cols, generator=g, device=dev)).to(pdt)
            got = _norm(pkg, layer, x, w, b, 1e-5, residual=res)
            torch.cuda.synchronize()
            h, y = _norm_reference(x, res, w, b, 1e-5, layer)
            if res is not None:
                assert torch.equal(got[2], (x.float() + res.float()).to(dt))
            # the maximum's error / 127, the factor's and the product's rounding; a byte: half a step, y's error, and the
            # rounding of the quotient (128 steps at most)
            err = _norm_bounds(h, y, w, b, 1e-5, layer)
            top, s = y.abs().amax(1), got[1].double()
            assert ((s - torch.clamp(top / 127, min=float(np.float32(1e-8)))).abs() <= err.amax(1) / 127 + (top / 127) * 3 * U).all()
            off = (got[0].double() * s[:, None] - y).abs()
            assert (off <= s[:, None] * (0.5 + 128 * 2 * U) + err).all(), float((off / s[:, None]).max())
