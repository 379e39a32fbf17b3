"""Operands at odd addresses through the Python entry points: they are given the workspace that the library copies them
into, as operands of odd widths are."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,cols,n,gated", [(1024, 2048, 1024, False), (300, 1024, 640, False), (513, 512, 700, True),
                                               (40, 8192, 100, False), (3, 256, 64, True)])
@pytest.mark.parametrize("at", [(1, 0), (0, 4), (9, 9)])
def test_odd_addresses_have_the_workspace_that_they_use(pkg, dev, monkeypatch, rows, cols, n, gated, at):
    g = torch.Generator(device=dev).manual_seed(rows)
    wrows = 2 * n if gated else n

    def int8(shift, *shape):
        t = torch.empty(shape[0] * shape[1] + shift, dtype=torch.int8, device=dev)[shift:].view(shape)
        return t.random_(-127, 128, generator=g)

    q, w = int8(at[0], rows, cols), int8(at[1], wrows, cols)
    s, ws = (torch.rand(k, generator=g, device=dev) / 100 for k in (rows, wrows))
    f = pkg.gated_linear_int8 if gated else pkg.linear_int8
    want = f(q.clone(), s, w.clone(), ws)
    given = []
    launch = pkg.ops._launch
    monkeypatch.setattr(pkg.ops, "_launch", lambda index, fn, *args: (given.append(args[-1]), launch(index, fn, *args))[1])
    print(f"odd addresses {rows}x{cols}->{n} gated={gated} {at}", flush=True)
    got = f(q, s, w, ws)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    c = pkg._capi
    gate = c.GATE_SILU if gated else c.GATE_NONE
    assert given == [c.lib().cti_ebag_linear_int8_workspace_bytes_unaligned(rows, cols, n, gate)]
