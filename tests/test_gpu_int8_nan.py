"""Rows that are not finite on their way through the int8 operators: a row of activations with NaN or infinity in it
is NaN behind every one of them, and no other row is.

``quantize_embedding_int8(x, nan_rows=True)`` marks such a row (scale NaN, q 0) as the norms do; without it the
quantiser leaves NaN out, which is for tables.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _gen(seed):
    return torch.Generator().manual_seed(seed)


# (widths of every form: chunks of 16 bytes down to one element, rows in a workgroup's registers, the loop)
@pytest.mark.parametrize("dim", [1, 5, 50, 64, 128, 129, 256, 300, 500, 1000, 1021, 2056, 5632, 16391, 40001])
@pytest.mark.parametrize("dt", TYPES)
def test_the_quantiser_marks_rows_that_are_not_finite(pkg, dev, dim, dt):
    g = _gen(dim)
    rows = 70
    x = torch.randn(rows, dim, generator=g).to(dt)
    at = torch.randint(0, dim, (rows,), generator=g)
    nan, inf = float("nan"), float("inf")
    bad = torch.zeros(rows, dtype=torch.bool)
    for r in range(0, 60, 3):  # NaN, infinities, one place a row
        x[r, at[r]] = (nan, inf, -inf, -nan)[r // 3 % 4]
        bad[r] = True
    x[60] = nan
    x[61], x[61, at[61]] = inf, nan
    x[62], x[62, 0] = nan, 1.0
    bad[60:63] = True
    bad[62] = dim > 1
    x[63] = torch.finfo(dt).max  # finite all the same
    x[64] = 0.0
    x[65] = torch.finfo(dt).smallest_normal
    for shift, pad in ((0, 0), (1, 0), (0, 5)):
        print(f"nan rows dim={dim} {dt} shift={shift} pad={pad}", flush=True)
        base = torch.zeros(rows * (dim + pad) + shift, dtype=dt, device=dev)
        view = base[shift:].view(rows, dim + pad)[:, :dim]
        view.copy_(x)
        q, s = (t.cpu() for t in pkg.quantize_embedding_int8(view, nan_rows=True))
        assert torch.equal(torch.isnan(s), bad)
        assert not q[bad].any()
        # the other rows: the expression as it stands, bit for bit
        v = x[~bad].float()
        want_s = torch.clamp(v.abs().amax(1) * np.float32(1 / 127), min=np.float32(1e-8))
        want_q = torch.clamp(torch.round(v / want_s[:, None]), -128, 127).to(torch.int8)
        assert torch.equal(s[~bad], want_s) and torch.equal(q[~bad], want_q)


@pytest.mark.parametrize("dim", [64, 300, 2056, 40001])
def test_what_rows_without_nan_give_does_not_depend_on_it(pkg, dev, dim):
    x = torch.randn(40, dim, generator=_gen(dim)).to(torch.bfloat16).to(dev)
    a, b = pkg.quantize_embedding_int8(x), pkg.quantize_embedding_int8(x, nan_rows=True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("rows,width,hidden", [(9, 64, 40), (40, 512, 1376), (300, 1021, 333)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_a_feed_forward_block_keeps_nan_rows(pkg, dev, rows, width, hidden, dt):
    """The block as it is documented: norm with the residual, gated product, rows quantised, product back."""
    g = _gen(rows)
    x, r = (torch.randn(rows, width, generator=g).to(dt) for _ in range(2))
    bad = torch.zeros(rows, dtype=torch.bool)
    x[1, 3], x[2, 0], r[4, width - 1] = float("nan"), float("inf"), -float("inf")
    x[6] = 3e38 / 2  # finite, but its squares leave fp32's range: no norm
    r[6] = 0.0
    bad[[1, 2, 4, 6]] = True
    norm = torch.ones(width, dtype=dt, device=dev)
    up = pkg.quantize_embedding_int8(torch.randn(2 * hidden, width, generator=g).to(dev) / width ** 0.5)
    down = pkg.quantize_embedding_int8(torch.randn(width, hidden, generator=g).to(dev) / hidden ** 0.5)

    def block(x, r, up):
        q, s, h = pkg.rms_norm_int8(x.to(dev), norm, 1e-5, residual=r.to(dev))
        a = pkg.gated_linear_int8(q, s, *up, out_dtype=dt)
        return pkg.linear_int8(*pkg.quantize_embedding_int8(a, nan_rows=True), *down, out_dtype=dt)

    print(f"block rows={rows} {width}/{hidden} {dt}", flush=True)
    y = block(x, r, up).cpu()
    assert torch.equal(torch.isnan(y).all(1), bad) and torch.equal(torch.isnan(y).any(1), bad)
    # the other rows are what they are without those beside them
    x[bad], r[bad] = 0.0, 0.0
    assert torch.equal(block(x, r, up).cpu()[~bad], y[~bad])
    # one gate's scale NaN: one column of the activations in every row, so every row of the product back
    scale = up[1].clone()
    scale[hidden // 2] = float("nan")
    assert torch.isnan(block(x, r, (up[0], scale))).all()


def test_a_channel_of_the_encoders_linear_that_is_not_finite(pkg, dev):
    """As with the float Linear: the channel's outputs are NaN, the others what they were."""
    torch.manual_seed(0)
    enc = pkg.RepEncoder(500, 64, 0, 4, 96).to(dev)
    rng = np.random.default_rng(0)
    lens = rng.integers(0, 6, size=(4, 50))
    batch = {"_flat_values": torch.from_numpy(rng.integers(0, 500, size=int(lens.sum()))).to(dev),
             "_val_offsets": torch.from_numpy(np.concatenate([[0], np.cumsum(lens.sum(axis=1))[:-1]])).to(dev),
             "_flat_row_offsets": torch.from_numpy(np.concatenate([np.concatenate([[0], np.cumsum(l)]) for l in lens])).to(dev)}
    with torch.no_grad():
        want = enc.quantize_linear_int8_()(batch)
        enc.linear.weight[7, 5] = float("nan")
        got = enc.quantize_linear_int8_()(batch)
    bad = torch.zeros(96, dtype=torch.bool, device=dev)
    bad[7] = True
    assert torch.isnan(got[:, bad]).all() and torch.equal(got[:, ~bad], want[:, ~bad])
