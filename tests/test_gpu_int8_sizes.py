"""Products of more outputs than the fastest form's launch has workgroups for: another form runs them."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,cols,n,gated", [(3, 16, 2 ** 26 + 5, False), (2, 8, 2 ** 26 + 1, True), (2, 40, 2 ** 26 + 16, False)])
@pytest.mark.parametrize("shift", [0, 1])
def test_many_outputs(pkg, dev, rows, cols, n, gated, shift):
    print(f"many outputs {rows}x{cols}->{n} gated={gated} shift={shift}", flush=True)
    g = torch.Generator(device=dev).manual_seed(n)
    wrows = n * (2 if gated else 1)

    def int8(*shape):
        count = shape[0] * shape[1]
        t = torch.empty(count + shift, dtype=torch.int8, device=dev)[shift:].view(shape)
        t.random_(-127, 128, generator=g)
        return t

    q, w = int8(rows, cols), int8(wrows, cols)
    s = torch.rand(rows, generator=g, device=dev) / 100
    ws = torch.rand(wrows, generator=g, device=dev) / 100
    f = pkg.gated_linear_int8 if gated else pkg.linear_int8
    kw = dict(activation="relu") if gated else {}
    for split in (True, False):
        y = f(q, s, w, ws, split_k=split, **kw)
        torch.cuda.synchronize()
        # pieces of the outputs: exact sums in float64, then one rounding an operation
        for lo in (0, 2 ** 22 - 1000, n // 2, n - 70001):
            at = slice(lo, lo + 70001)

            def value(first):
                t = q.double() @ w[first + at.start:first + at.stop].double().t().contiguous()
                return (t.float() * s[:, None]) * ws[None, first + at.start:first + at.stop]

            want = torch.clamp(value(0), min=0.0) * value(n) if gated else value(0)
            assert torch.equal(y[:, at], want.to(torch.bfloat16)), (split, lo)
        del y
