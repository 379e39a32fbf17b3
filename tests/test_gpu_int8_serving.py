"""The int8 serving operators on the GPU, against their definitions in 64 bits (numpy and torch on the CPU, or
torch in float64 on the device for the large shapes).

Bar:
- norms: the residual's sum is the fp32 sum rounded once, bit for bit; every scale is the largest normalised
  value / 127 and every q the nearest step to its value, within what fp32 arithmetic can move them (derived in
  _norm_bounds); rows that are not finite have the scale NaN and q = 0 and disturb no other row;
- linear_int8: bit for bit (float32(integer sum) * scale * weight_scale + bias, each operation rounded once);
- gated_linear_int8: the activation within 8 fp32 roundings (derived at the test), the rest as above;
- dequantize_embedding_int8: bit for bit;
- all of them: odd sizes and addresses, streams, graphs replayed on new inputs, offsets past 32 bits.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # half a step of fp32
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: U}
SMALLEST = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24, torch.float32: 2.0 ** -149}


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _at_offset(t, dev, shift):
    """`t` on the device, contiguous, `shift` elements into its allocation."""
    if not shift:
        return t.to(dev)
    buf = torch.empty(t.numel() + shift, dtype=t.dtype, device=dev)
    out = buf[shift:].view(t.shape)
    out.copy_(t)
    return out


# ------------------------------------------------------------------------------------------------
# Norms
# ------------------------------------------------------------------------------------------------
def _norm_reference(x, res, w, b, eps, layer):
    """(h, y) in float64; h unrounded."""
    h = x.double()
    if res is not None:
        h = h + res.double()
    d = h - h.mean(1, keepdim=True) if layer else h
    y = d / torch.sqrt(d.pow(2).mean(1, keepdim=True) + eps) * w.double()
    return h, (y + b.double() if layer else y)


def _norm_bounds(h, y, w, b, eps, layer):
    """How far fp32 arithmetic can move each y. h is one rounding of the sum. A mean or a sum of squares over n
    terms adds at most T = 80 terms in a row per thread (16 384 columns over 256 threads and up to 8 vectors; the
    loop kernel n / 256) and 12 levels of tree: relative error (T + 14) u of the mean of the |terms|. Half of it
    reaches rstd; rstd, the subtraction and the three operations after it add at most 6 roundings."""
    n = h.shape[1]
    t = max(80, n / 256) + 14
    d = h - h.mean(1, keepdim=True) if layer else h
    rstd = 1 / torch.sqrt(d.pow(2).mean(1, keepdim=True) + eps)
    wa = w.double().abs()
    core = (d * rstd).abs() * wa
    err = core * (t + 8) * U + h.abs() * rstd * wa * 2 * U
    if layer:
        shift = h.abs().mean(1, keepdim=True) * (t + 2) * U  # of the mean
        err = err + shift * rstd * wa * 2 + (b.double().abs() + y.abs()) * U * 2
        # the deviations' error also reaches the variance: relative 2 shift / sigma of it, half of that rstd's
        err = err + core * shift * rstd * 2
    return err


def _check_norm(got, x, res, w, b, eps, layer):
    q, s = got[0].cpu(), got[1].cpu()
    h, y = _norm_reference(x, res, w, b, eps, layer)
    if res is not None:
        want = (x.float() + res.float()).to(x.dtype)
        assert torch.equal(got[2].cpu().view(torch.uint8), want.view(torch.uint8))
    err = _norm_bounds(h, y, w, b, eps, layer)
    top = y.abs().amax(1)
    s64 = s.double()
    # the maximum's error / 127, the factor's and the product's rounding
    ds = err.amax(1) / 127 + (top / 127) * 3 * U
    want_s = torch.clamp(top / 127, min=float(np.float32(1e-8)))
    assert ((s64 - want_s).abs() <= ds).all()
    # nearest step: half a step, y's error, and the division's rounding (128 steps * u)
    off = (q.double() * s64[:, None] - y).abs()
    assert (off <= s64[:, None] * (0.5 + 128 * 2 * U) + err).all(), float((off / s64[:, None]).max())


def _norm(pkg, layer, x, w, b, eps, **kw):
    if layer:
        return pkg.layer_norm_int8(x, w, b, eps, **kw)
    return pkg.rms_norm_int8(x, w, eps, **kw)


NORM_SHAPES = [(1, 1), (3, 7), (2, 8), (5, 9), (4, 64), (7, 129), (1, 512), (33, 1021), (2, 2048), (3, 8200), (2, 16384),
               (2, 32768), (1, 40001), (1, 70001),
               # from 1,024 rows on a row has fewer wavefronts
               (1030, 4), (1025, 511), (1024, 1000), (1027, 2047), (1024, 4096), (1025, 4104), (1024, 10001), (1024, 20000)]


@pytest.mark.parametrize("rows,cols", NORM_SHAPES)
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
def test_norms(pkg, dev, rows, cols, dt):
    g = _gen(rows * 7 + cols)
    size = torch.exp(torch.randn(rows, 1, generator=g))
    x = ((torch.randn(rows, cols, generator=g) + 0.3) * size).to(dt)
    r = (torch.randn(rows, cols, generator=g) * 0.7).to(dt)
    for layer in (False, True):
        for res, pdt in ((None, torch.float32), (r, dt), (r, torch.float16)):
            print(f"norm rows={rows} cols={cols} {dt} layer={layer} res={res is not None} params={pdt}", flush=True)
            w = (1 + 0.2 * torch.randn(cols, generator=g)).to(pdt)
            b = (0.2 * torch.randn(cols, generator=g)).to(pdt)
            got = _norm(pkg, layer, x.to(dev), w.to(dev), b.to(dev), 1e-5,
                        residual=res.to(dev) if res is not None else None)
            torch.cuda.synchronize()
            _check_norm(got, x, res, w, b, 1e-5, layer)


@pytest.mark.parametrize("cols", [1024, 1021, 24])
@pytest.mark.parametrize("shift", [1, 3])
@pytest.mark.parametrize("rows", [5, 1100])
def test_norms_at_odd_addresses(pkg, dev, rows, cols, shift):
    g = _gen(cols + shift)
    for dt in (torch.bfloat16, torch.float32):
        x, r = ((torch.randn(rows, cols, generator=g)).to(dt) for _ in range(2))
        w, b = torch.randn(cols, generator=g).to(dt), torch.randn(cols, generator=g).to(dt)
        print(f"norm rows={rows} cols={cols} shift={shift} {dt}", flush=True)
        q = _at_offset(torch.zeros(rows, cols, dtype=torch.int8), dev, shift)
        out = _at_offset(torch.zeros(rows, cols, dtype=dt), dev, shift)
        got = _norm(pkg, True, _at_offset(x, dev, shift), _at_offset(w, dev, shift), _at_offset(b, dev, shift), 1e-5,
                    residual=_at_offset(r, dev, shift), q=q, residual_out=out)
        torch.cuda.synchronize()
        assert got[0] is q and got[2] is out
        _check_norm(got, x, r, w, b, 1e-5, True)


@pytest.mark.parametrize("rows,cols", [(9, 1000), (1500, 1000), (1100, 1021), (2, 70001), (4, 3)])
def test_residual_in_place(pkg, dev, rows, cols):
    g = _gen(5)
    x, r = (torch.randn(rows, cols, generator=g).to(torch.bfloat16).to(dev) for _ in range(2))
    w = torch.ones(cols, device=dev)
    want = pkg.rms_norm_int8(x, w, residual=r)
    for which in ("residual", "x"):
        a, b = x.clone(), r.clone()
        got = pkg.rms_norm_int8(a, w, residual=b, residual_out=b if which == "residual" else a)
        torch.cuda.synchronize()
        assert all(torch.equal(u, v) for u, v in zip(got, want)), which
        assert torch.equal(b, want[2]) if which == "residual" else torch.equal(b, r)


@pytest.mark.parametrize("layer", [False, True])
@pytest.mark.parametrize("rows,cols", [(40, 520), (1200, 520), (40, 70001)])
def test_rows_that_are_not_finite_or_have_no_scale(pkg, dev, layer, rows, cols):
    g = _gen(11)
    for dt in (torch.bfloat16, torch.float32, torch.float16):
        x = torch.randn(rows, cols, generator=g).to(dt)
        top = torch.finfo(dt).max
        x[3, 17] = float("nan")
        x[5, 0] = float("inf")
        x[7, cols - 1] = -float("inf")
        x[9] = 0.0                       # nothing in the row
        x[11] = torch.finfo(dt).tiny     # squares below fp32's range: the variance is 0
        x[13] = 2.5                      # LayerNorm's variance is 0
        x[15] = 0.0
        x[15, 8] = 3.0                   # one value
        big = [20] if dt == torch.float16 else [19, 20]
        for i in big:
            x[i] = x[i].sign() * top     # lowest and largest values of the type
        w = torch.ones(cols)
        b = torch.zeros(cols)
        print(f"special rows={rows} cols={cols} {dt} layer={layer}", flush=True)
        got = _norm(pkg, layer, x.to(dev), w.to(dev), b.to(dev), 1e-5)
        torch.cuda.synchronize()
        q, s = got[0].cpu(), got[1].cpu()
        # fp16's largest squares fit into fp32, those of the others do not: the row has no norm in fp32
        bad = torch.zeros(rows, dtype=torch.bool)
        bad[[3, 5, 7]] = True
        if dt != torch.float16:
            bad[big] = True
        assert torch.equal(torch.isnan(s), bad)
        assert (q[bad] == 0).all()
        assert s[9] == np.float32(1e-8) and (q[9] == 0).all()
        keep = ~bad
        keep[11] = False  # its y (about 2^-110 / sqrt(eps) or less) are below the smallest scale's half step
        assert (q[11] == 0).all() and s[11] == np.float32(1e-8) or dt == torch.float16
        _check_norm((got[0][keep.to(dev)], got[1][keep.to(dev)]), x[keep], None, w, b, 1e-5, layer)
        # what such a row's products are: NaN, its own only
        wt = torch.randint(-127, 128, (48, cols), generator=g, dtype=torch.int8).to(dev)
        y = pkg.linear_int8(got[0], got[1], wt, torch.ones(48, device=dev)).float().cpu()
        assert torch.equal(torch.isnan(y).all(1), bad) and torch.equal(torch.isnan(y).any(1), bad)


def test_weights_that_are_not_finite_make_their_rows_nan(pkg, dev):
    x = torch.ones(3, 64, device=dev)
    w = torch.ones(64, device=dev)
    w[5] = float("inf")
    q, s = pkg.rms_norm_int8(x, w)
    assert torch.isnan(s).all() and (q == 0).all()


@pytest.mark.parametrize("rows,cols", [(6, 4096), (2000, 1024), (1100, 1021)])
def test_norm_rows_stand_for_themselves(pkg, dev, rows, cols):
    """A row's result does not depend on the rows beside it, and two runs agree bit for bit."""
    g = _gen(3)
    x = torch.randn(rows, cols, generator=g).to(torch.bfloat16).to(dev)
    w = torch.ones(cols, device=dev, dtype=torch.bfloat16)
    a, b = pkg.rms_norm_int8(x, w), pkg.rms_norm_int8(x, w)
    c = pkg.rms_norm_int8(torch.flip(x, (0,)), w)
    assert all(torch.equal(u, v) for u, v in zip(a, b))
    assert torch.equal(torch.flip(c[0], (0,)), a[0]) and torch.equal(torch.flip(c[1], (0,)), a[1])


def test_no_rows(pkg, dev):
    x = torch.empty(0, 64, device=dev)
    w = torch.ones(64, device=dev)
    q, s, h = pkg.rms_norm_int8(x, w, residual=x)
    assert q.shape == (0, 64) and s.shape == (0,) and h.shape == (0, 64)
    wt = torch.zeros(6, 64, dtype=torch.int8, device=dev)
    ws = torch.ones(6, device=dev)
    assert pkg.linear_int8(q, s, wt, ws).shape == (0, 6)
    assert pkg.gated_linear_int8(q, s, wt, ws).shape == (0, 3)
    assert pkg.dequantize_embedding_int8(q, s).shape == (0, 64)


# ------------------------------------------------------------------------------------------------
# Products
# ------------------------------------------------------------------------------------------------
def _operands(rows, cols, n, seed, full=False):
    g = _gen(seed)
    lo = -128 if full else -127
    q = torch.randint(lo, 128, (rows, cols), generator=g, dtype=torch.int8)
    w = torch.randint(lo, 128, (n, cols), generator=g, dtype=torch.int8)
    s = torch.exp(torch.randn(rows, generator=g)) / 100
    ws = torch.exp(torch.randn(n, generator=g)) / 100
    bias = torch.randn(n, generator=g)
    return q, s, w, ws, bias


def _value(q, s, w, ws, bias):
    """v of the definition: exact sums (float64 holds them), then fp32 operations, each rounded once."""
    t = (q.double() @ w.double().t()).numpy().astype(np.float32)
    v = (t * s.numpy()[:, None]).astype(np.float32) * ws.numpy()[None, :]
    v = v.astype(np.float32)
    return v if bias is None else (v + bias.float().numpy()).astype(np.float32)


SHAPES = [  # rows, cols, outputs
    (1, 1, 1), (1, 16, 16), (1, 127, 5), (2, 128, 33), (7, 1021, 100), (16, 4096, 48), (17, 200, 64), (31, 130, 17),
    (32, 3584, 64), (33, 15, 3), (40, 128, 128), (64, 257, 130), (65, 1024, 1000), (77, 8192, 100), (128, 14336, 64),
    (129, 640, 257), (200, 48, 511), (255, 1040, 256), (300, 3584, 512), (513, 1021, 777), (1000, 96, 1500),
    (2049, 256, 512), (4100, 528, 130), (1024, 2048, 1536)]


@pytest.mark.parametrize("rows,cols,n", SHAPES)
def test_linear_is_exact(pkg, dev, rows, cols, n):
    q, s, w, ws, bias = _operands(rows, cols, n, rows + cols + n)
    for b, odt in ((None, torch.float32), (bias, torch.float32), (bias.to(torch.bfloat16), torch.bfloat16),
                   (bias.to(torch.float16), torch.float16)):
        print(f"linear rows={rows} cols={cols} n={n} bias={b is not None} {odt}", flush=True)
        want = torch.from_numpy(_value(q, s, w, ws, b)).to(odt)
        for split in (True, False):
            got = pkg.linear_int8(q.to(dev), s.to(dev), w.to(dev), ws.to(dev), b.to(dev) if b is not None else None,
                                  out_dtype=odt, split_k=split)
            torch.cuda.synchronize()
            assert torch.equal(got.cpu(), want), (split, int((got.cpu() != want).sum()))


# Products too large for the CPU: every form of the large plans (256 x 256 tiles with and without a rest of K, a rest of
# columns in another form, operands copied to whole steps), against float64 on the device.
LARGE = [(8192, 256, 2048, False), (4100, 640, 4100, False), (4100, 272, 4100, False), (4096, 1000, 4200, False),
         (8000, 130, 4099, False), (2500, 1040, 2049, False), (4100, 640, 2050, True), (4096, 1008, 2176, True),
         (3001, 333, 1500, True), (8192, 512, 1024, True), (2048, 2048, 2048, False),
         # about as many tiles as CUs, or K split over as many: the rings of one tile to a CU
         (4096, 3584, 512, False), (2000, 1040, 1003, False), (1000, 8192, 1000, False), (600, 16016, 700, False),
         (512, 4096, 2048, True), (700, 9216, 500, True), (520, 3600, 4100, False), (900, 12304, 900, False),
         (500, 1040, 2100, True), (2048, 2048, 1024, True), (300, 15360, 2500, False)]


@pytest.mark.parametrize("rows,cols,n,gated", LARGE)
def test_large_products(pkg, dev, rows, cols, n, gated):
    print(f"large rows={rows} cols={cols} n={n} gated={gated}", flush=True)
    wrows = 2 * n if gated else n
    q, s, w, ws, bias = (t.to(dev) for t in _operands(rows, cols, wrows, rows + n))
    t = q.double() @ w.double().t().contiguous()
    v = (t.float() * s[:, None]) * ws[None, :] + bias[None, :]  # as _value: one rounding an operation
    for odt in (torch.bfloat16, torch.float32):
        if gated:
            got = pkg.gated_linear_int8(q, s, w, ws, bias, activation="relu", out_dtype=odt)
            want = torch.clamp(v[:, :n], min=0.0) * v[:, n:]
        else:
            got = pkg.linear_int8(q, s, w, ws, bias, out_dtype=odt)
            want = v
        torch.cuda.synchronize()
        assert torch.equal(got, want.to(odt)), int((got != want.to(odt)).sum())


@pytest.mark.parametrize("rows,cols,n", [(1, 131071, 20), (40, 131071, 24), (300, 131071, 40)])
def test_the_largest_sums_do_not_overflow(pkg, dev, rows, cols, n):
    print(f"largest sums rows={rows}", flush=True)
    q = torch.full((rows, cols), -128, dtype=torch.int8, device=dev)
    w = torch.full((n, cols), -128, dtype=torch.int8, device=dev)
    w[1::2] = 127
    one = (lambda k: torch.ones(k, device=dev))
    got = pkg.linear_int8(q, one(rows), w, one(n), out_dtype=torch.float32).cpu()
    assert (got[:, ::2] == float(np.float32(cols * 16384))).all()
    assert (got[:, 1::2] == float(np.float32(-cols * 127 * 128))).all()


@pytest.mark.parametrize("rows,cols,n", [(3, 64, 32), (20, 1024, 48), (70, 512, 200), (300, 1024, 300)])
@pytest.mark.parametrize("shift", [1, 4, 7])
def test_products_at_odd_addresses(pkg, dev, rows, cols, n, shift):
    q, s, w, ws, bias = _operands(rows, cols, n, 9, full=True)
    want = torch.from_numpy(_value(q, s, w, ws, bias)).to(torch.bfloat16)
    print(f"linear shift={shift} rows={rows} cols={cols} n={n}", flush=True)
    out = _at_offset(torch.zeros(rows, n, dtype=torch.bfloat16), dev, shift)
    for a, b in ((shift, 0), (0, shift), (shift, shift)):
        pkg.linear_int8(_at_offset(q, dev, a), _at_offset(s, dev, a), _at_offset(w, dev, b), _at_offset(ws, dev, b),
                        _at_offset(bias, dev, b), out=out)
        torch.cuda.synchronize()
        assert torch.equal(out.cpu(), want), (a, b)


@pytest.mark.parametrize("rows,n", [(5, 40), (24, 17), (100, 130), (300, 640)])
def test_nothing_is_written_past_the_output(pkg, dev, rows, n):
    """Rows before and behind the output stay as they were, whatever the tiles cover."""
    q, s, w, ws, bias = (t.to(dev) for t in _operands(rows, 1024, n, 21))
    for dt in (torch.bfloat16, torch.float32):
        for gated in (False, True):
            cols_out = n // 2 if gated else n
            weight, wsc = (w[:2 * cols_out].contiguous(), ws[:2 * cols_out].contiguous()) if gated else (w, ws)
            buf = torch.full((rows + 600, cols_out), 7.0, dtype=dt, device=dev)
            out = buf[300:300 + rows]
            f = pkg.gated_linear_int8 if gated else pkg.linear_int8
            f(q, s, weight, wsc, out=out)
            torch.cuda.synchronize()
            assert (buf[:300] == 7).all() and (buf[300 + rows:] == 7).all()
            assert torch.equal(out, f(q, s, weight, wsc, out_dtype=dt))


def _activation(v, name):
    """float64 of the activation of a float32 array."""
    g = torch.from_numpy(v).double()
    if name == "silu":
        return g * torch.sigmoid(g)
    if name == "gelu":
        return 0.5 * g * torch.special.erfc(-g / math.sqrt(2))
    return torch.clamp(g, min=0.0)


@pytest.mark.parametrize("rows,cols,n", [(1, 1, 1), (1, 4096, 40), (3, 127, 33), (16, 1024, 100), (17, 640, 17),
                                         (32, 256, 5), (33, 100, 70), (64, 2048, 200), (77, 1021, 64), (130, 512, 129),
                                         (513, 384, 300), (1030, 1040, 257)])
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
def test_gated(pkg, dev, rows, cols, n, act):
    """v is exact (as linear_int8's). fp32 roundings of act(v) * u: silu exp (2 half steps, and the rounding of
    1 + exp), division, product; gelu the argument (its rounding moves erfc by up to 2 x^2 + 1 times that) and erfc (2
    ulp), two products; at most 8 half steps, gelu (4 x^2 + 8); below fp32's normal range a few times its
    smallest value times the other factor. Then the output's rounding."""
    q, s, w, ws, bias = _operands(rows, cols, 2 * n, rows + cols)
    s = s / cols ** 0.5
    for b, odt in ((None, torch.float32), (bias.to(torch.bfloat16), torch.bfloat16), (bias, torch.float16)):
        print(f"gated rows={rows} cols={cols} n={n} {act} {odt}", flush=True)
        v = _value(q, s, w, ws, b)
        a = _activation(np.ascontiguousarray(v[:, :n]), act)
        u = torch.from_numpy(np.ascontiguousarray(v[:, n:])).double()
        ref = a * u
        x2 = torch.from_numpy(v[:, :n].astype(np.float64) ** 2 / 2) if act == "gelu" else torch.zeros_like(ref)
        tol = ref.abs() * ((4 * x2 + 8) * U + HALF_STEP[odt] * 1.001) + 4 * 2.0 ** -126 * u.abs() + SMALLEST[odt]
        got = pkg.gated_linear_int8(q.to(dev), s.to(dev), w.to(dev), ws.to(dev), b.to(dev) if b is not None else None,
                                    activation=act, out_dtype=odt)
        torch.cuda.synchronize()
        got = got.cpu().double()
        inside = ref.abs() < torch.finfo(odt).max * 0.99
        assert ((got - ref).abs() <= tol)[inside].all(), float(((got - ref).abs() / tol)[inside].max())
        assert torch.isfinite(got[inside]).all()


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
def test_gates_far_out(pkg, dev, act):
    """Gates from -2000 to 2000: no overflow on the way, limits 0 and the gate itself."""
    gate = torch.tensor([-2000.0, -200.0, -88.8, -30.0, -1.0, 0.0, 1.0, 30.0, 200.0, 2000.0])
    q = torch.ones(1, 16, dtype=torch.int8)
    w = torch.zeros(20, 16, dtype=torch.int8)
    bias = torch.cat([gate, torch.ones(10)])
    got = pkg.gated_linear_int8(q.to(dev), torch.ones(1, device=dev), w.to(dev), torch.ones(20, device=dev),
                                bias.to(dev), activation=act, out_dtype=torch.float32).cpu()[0].double()
    ref = _activation(gate.numpy(), act)
    x2 = gate.double() ** 2 / 2
    assert torch.isfinite(got).all()
    tol = ref.abs() * ((4 * torch.clamp(x2, max=200.0) if act == "gelu" else 0) + 8) * U + 4 * 2.0 ** -126
    assert ((got - ref).abs() <= tol).all()


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
def test_nan_scales_reach_their_products_only(pkg, dev, act):
    q, s, w, ws, _ = _operands(50, 128, 64, 4)
    s[3] = float("nan")
    ws[5] = float("nan")       # gate of column 5
    ws[32 + 9] = float("nan")  # value of column 9
    got = pkg.gated_linear_int8(q.to(dev), s.to(dev), w.to(dev), ws.to(dev), activation=act).cpu()
    want = torch.zeros(50, 32, dtype=torch.bool)
    want[3] = True
    want[:, 5] = want[:, 9] = True
    assert torch.equal(torch.isnan(got), want)


def test_workspaces_of_any_size(pkg, dev):
    """Through the C ABI: no workspace, less than the query, the query: the same result bit for bit, and nothing
    written past the workspace."""
    c = pkg._capi
    lib = c.lib()
    for rows, cols, n, gate in ((128, 14336, 512, 0), (77, 8192, 1000, 0), (64, 4096, 256, c.GATE_SILU)):
        wrows = n * (2 if gate else 1)
        q, s, w, ws, _ = (t.to(dev) for t in _operands(rows, cols, wrows, 1))
        need = lib.cti_ebag_linear_int8_workspace_bytes(rows, cols, n, gate)
        outs = []
        for nbytes in sorted({0, 16, need // 3 // 16 * 16, need}):
            print(f"workspace {rows}x{cols}x{n} {nbytes} of {need}", flush=True)
            buf = torch.full((nbytes + 4096,), 171, dtype=torch.uint8, device=dev)
            out = torch.empty(rows, n, dtype=torch.float32, device=dev)
            c.check(lib.cti_ebag_linear_int8(q.data_ptr(), s.data_ptr(), rows, cols, w.data_ptr(), ws.data_ptr(), n, None,
                                             c.F32, gate, out.data_ptr(), c.F32, buf.data_ptr(), nbytes,
                                             torch.cuda.current_stream(dev).cuda_stream))
            torch.cuda.synchronize()
            assert (buf[nbytes:] == 171).all()
            outs.append(out)
        assert all(torch.equal(o, outs[0]) for o in outs)


# ------------------------------------------------------------------------------------------------
# Read-back
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 5), (2, 16), (100, 17), (33, 1021), (7, 4096), (50000, 3), (1000, 128)])
def test_dequantize(pkg, dev, rows, cols):
    g = _gen(rows + cols)
    q = torch.randint(-128, 128, (rows, cols), generator=g, dtype=torch.int8)
    s = torch.exp(torch.randn(rows, generator=g))
    s[rows // 2] = float("nan")
    for dt in (torch.bfloat16, torch.float16, torch.float32):
        want = (q.float() * s[:, None]).to(dt)
        for shift in (0, 1, 5):
            print(f"dequantize rows={rows} cols={cols} {dt} shift={shift}", flush=True)
            out = _at_offset(torch.zeros(rows, cols, dtype=dt), dev, shift)
            pkg.dequantize_embedding_int8(_at_offset(q, dev, shift), _at_offset(s, dev, shift), out=out)
            torch.cuda.synchronize()
            assert torch.equal(out.cpu().nan_to_num(9.0), want.nan_to_num(9.0))
            assert torch.equal(out.cpu().isnan(), want.isnan())


def test_quantize_and_back(pkg, dev):
    x = torch.randn(100, 300, generator=_gen(1)).to(dev)
    q, s = pkg.quantize_embedding_int8(x)
    back = pkg.dequantize_embedding_int8(q, s, torch.float32)
    assert ((back - x).abs() <= s[:, None] * 0.5001).all()


# ------------------------------------------------------------------------------------------------
# Offsets past 32 bits
# ------------------------------------------------------------------------------------------------
def test_norm_and_read_back_past_32_bits(pkg, dev):
    cols = 8192
    rows = 2 ** 32 // cols + 5  # elements past 2^32
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device=dev)
    tail = torch.randn(7, cols, generator=_gen(2)).to(torch.bfloat16)
    x[-7:] = tail.to(dev)
    w = torch.ones(cols)
    print("norm past 32 bits", flush=True)
    q, s, h = pkg.rms_norm_int8(x, w.to(dev), residual=x, residual_out=x)
    torch.cuda.synchronize()
    assert h is x
    _check_norm((q[-7:], s[-7:], x[-7:]), tail, tail, w, None, 1e-5, False)
    assert (s[:-7] == np.float32(1e-8)).all()
    print("read-back past 32 bits", flush=True)
    v = pkg.dequantize_embedding_int8(q, s, out=x)
    torch.cuda.synchronize()
    assert torch.equal(v[-7:].cpu(), (q[-7:].cpu().float() * s[-7:].cpu()[:, None]).to(torch.bfloat16))
    assert not v[:-7].any()


@pytest.mark.parametrize("rows,cols,n", [(70000, 65536, 40), (150000, 32, 16400)])
def test_products_past_32_bits(pkg, dev, rows, cols, n):
    """Inputs, or outputs, of more than 2^32 elements and 2^31 bytes."""
    q = torch.zeros(rows, cols, dtype=torch.int8, device=dev)
    tq, s, w, ws, _ = _operands(5, cols, n, 6)
    q[-5:] = tq.to(dev)
    scale = torch.ones(rows, device=dev)
    scale[-5:] = s.to(dev)
    print(f"product past 32 bits {rows}x{cols}x{n}", flush=True)
    y = pkg.linear_int8(q, scale, w.to(dev), ws.to(dev))
    torch.cuda.synchronize()
    assert torch.equal(y[-5:].cpu(), torch.from_numpy(_value(tq, s, w, ws, None)).to(torch.bfloat16))
    assert not y[:-5].any()


# ------------------------------------------------------------------------------------------------
# Together: a feed-forward block, the encoder; streams and graphs
# ------------------------------------------------------------------------------------------------
class _Block:
    """norm + residual -> gated -> rows quantised -> product back, on `dev`."""

    def __init__(self, pkg, dev, width, hidden, dt, seed=0):
        g = _gen(seed)
        self.pkg = pkg
        self.norm = (1 + 0.1 * torch.randn(width, generator=g)).to(dt).to(dev)
        up = torch.randn(2 * hidden, width, generator=g).to(dev) / width ** 0.5
        down = torch.randn(width, hidden, generator=g).to(dev) / hidden ** 0.5
        self.up, self.down = pkg.quantize_embedding_int8(up), pkg.quantize_embedding_int8(down)

    def __call__(self, x, res):
        q, s, h = self.pkg.rms_norm_int8(x, self.norm, 1e-5, residual=res)
        a = self.pkg.gated_linear_int8(q, s, *self.up, out_dtype=x.dtype)
        return self.pkg.linear_int8(*self.pkg.quantize_embedding_int8(a), *self.down, out_dtype=x.dtype), h

    def float64(self, x, res):
        """The block without any quantisation of rows (the weights are the int8 ones)."""
        h = x.double() + res.double()
        y = h / torch.sqrt(h.pow(2).mean(1, keepdim=True) + 1e-5) * self.norm.double()
        g, u = (y @ (self.up[0].double() * self.up[1].double()[:, None]).t().contiguous()).chunk(2, 1)
        return (g * torch.sigmoid(g) * u) @ (self.down[0].double() * self.down[1].double()[:, None]).t().contiguous()


@pytest.mark.parametrize("rows", [1, 9, 40, 300, 1100])
@pytest.mark.parametrize("width,hidden", [(512, 1376), (1021, 333)])
def test_feed_forward_block(pkg, dev, rows, width, hidden):
    """Rows quantised to 8 bits carry errors uniform over a step: s / sqrt(12) an element. The products add them
    with independent signs, so the block's output is off by a few percent of its root mean square; a wrong
    row, column, scale or half is off by as much as the output itself."""
    block = _Block(pkg, dev, width, hidden, torch.bfloat16)
    g = _gen(rows)
    x, r = (torch.randn(rows, width, generator=g).to(torch.bfloat16).to(dev) for _ in range(2))
    print(f"block rows={rows} {width}/{hidden}", flush=True)
    y, h = block(x, r)
    torch.cuda.synchronize()
    ref = block.float64(x, r)
    # per row: step of the norm's rows max/127 <= 6 sigma / 127, error sigma_e = step / sqrt(12) = 1.4% of sigma; the
    # gate passes at most its slope (1.1) of it on each factor, and the second quantisation has heavier tails (max
    # up to about 20 rms): 20 / 127 / sqrt(12) = 4.5%; together below 8% of the row's root mean square
    err = (y.double() - ref).pow(2).mean(1).sqrt() / ref.pow(2).mean(1).sqrt()
    assert err.max() < 0.08, float(err.max())
    assert torch.equal(h, (x.float() + r.float()).to(torch.bfloat16))


def _batch(rng, S, B, V, dev):
    lens = rng.integers(0, 6, size=(S, B))
    ids = rng.integers(0, V, size=int(lens.sum()))
    ro = np.concatenate([np.concatenate([[0], np.cumsum(l)]) for l in lens]).astype(np.int64)
    vo = np.concatenate([[0], np.cumsum(lens.sum(axis=1))[:-1]]).astype(np.int64)
    return {"_flat_values": torch.from_numpy(ids).to(dev), "_val_offsets": torch.from_numpy(vo).to(dev),
            "_flat_row_offsets": torch.from_numpy(ro).to(dev)}


@pytest.mark.parametrize("B", [1, 50, 700])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("int8_table", [False, True])
def test_encoder_with_an_int8_linear(pkg, dev, B, dt, int8_table):
    torch.manual_seed(0)
    enc = pkg.RepEncoder(500, 64, 0, 28, 96).to(dev).to(dt)
    batch = _batch(np.random.default_rng(B), 28, B, 500, dev)
    if int8_table:
        enc.quantize_int8_()
    print(f"encoder int8 linear B={B} {dt} int8_table={int8_table}", flush=True)
    with torch.no_grad():
        before = enc(batch)
        pooled = enc.pooled(batch)
        assert enc.quantize_linear_int8_() is enc
        got = enc(batch)
        assert got.dtype == dt and got.shape == (B, 96)
        q, s = pkg.layer_norm_int8(pooled, enc.input_norm.weight, enc.input_norm.bias, enc.input_norm.eps)
        wq, wsc = pkg.quantize_embedding_int8(enc.linear.weight.detach())
        bias = enc.linear.bias.detach()
        want = torch.from_numpy(_value(q.cpu(), s.cpu(), wq.cpu(), wsc.cpu(), bias.cpu())).to(dt)
        assert torch.equal(got.cpu(), want)
        with pytest.raises(ValueError, match="int8 Linear"):
            enc(batch, fused_linear=True)
        enc.dequantize_linear_()
        assert torch.equal(enc(batch), before)


def test_calls_follow_their_streams(pkg, dev):
    """Two blocks on two streams at once, each behind work of its own stream, give what they give alone."""
    block = _Block(pkg, dev, 512, 1376, torch.bfloat16)
    ins = [tuple(torch.randn(200 + 37 * i, 512, generator=_gen(i)).to(torch.bfloat16).to(dev) for _ in range(2))
           for i in range(2)]
    want = [block(*p) for p in ins]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for rep in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                x = ins[i][0].clone()
                torch.cuda._sleep(200_000)
                got[i].append(block(x, ins[i][1]))
    torch.cuda.synchronize()
    for i in range(2):
        for y, h in got[i]:
            assert torch.equal(y, want[i][0]) and torch.equal(h, want[i][1])


@pytest.mark.parametrize("rows", [1, 20, 77, 300])
def test_graph_replays(pkg, dev, rows):
    """A captured block and another captured one of the same shape (workspaces of their own) replayed on new
    inputs, with eager calls between the replays."""
    block = _Block(pkg, dev, 1024, 512, torch.bfloat16)
    bufs = [tuple(torch.zeros(rows, 1024, dtype=torch.bfloat16, device=dev) for _ in range(2)) for _ in range(2)]
    block(*bufs[0])
    torch.cuda.synchronize()
    graphs, outs = [], []
    for b in bufs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(block(*b))
        graphs.append(g)
    for rep in range(4):
        new = [tuple(torch.randn(rows, 1024, generator=_gen(10 * rep + i)).to(torch.bfloat16).to(dev) for _ in range(2))
               for i in range(2)]
        for b, v in zip(bufs, new):
            for d, t in zip(b, v):
                d.copy_(t)
        for g in graphs:
            g.replay()
        want = [block(*v) for v in new]
        torch.cuda.synchronize()
        for o, t in zip(outs, want):
            assert torch.equal(o[0], t[0]) and torch.equal(o[1], t[1]), rep


def test_python_refusals(pkg, dev):
    q, s, w, ws, bias = (t.to(dev) for t in _operands(4, 64, 32, 0))
    x = torch.ones(4, 64, device=dev)
    g = torch.ones(64, device=dev)
    bad = [
        (lambda: pkg.linear_int8(q.float(), s, w, ws), TypeError, "int8"),
        (lambda: pkg.linear_int8(q, s.double(), w, ws), TypeError, "float32"),
        (lambda: pkg.linear_int8(q, s[:3], w, ws), ValueError, "shape"),
        (lambda: pkg.linear_int8(q, s, w[:, :60].contiguous(), ws), ValueError, "columns"),
        (lambda: pkg.linear_int8(q, s, w[:, :60], ws), ValueError, "contiguous"),
        (lambda: pkg.linear_int8(q.t(), ws[:1].expand(64), w, ws), ValueError, "contiguous"),
        (lambda: pkg.linear_int8(q, s, w, ws, bias[:5]), ValueError, "bias"),
        (lambda: pkg.linear_int8(q, s, w, ws, bias.double()), TypeError, "element type"),
        (lambda: pkg.linear_int8(q, s, w, ws, out=torch.empty(4, 31, device=dev)), ValueError, "shape"),
        (lambda: pkg.linear_int8(q, s, w, ws, out_dtype=torch.float64), TypeError, "element type"),
        (lambda: pkg.linear_int8(q, s, w[:0], ws[:0]), ValueError, "no rows"),
        (lambda: pkg.gated_linear_int8(q, s, w[:31], ws[:31]), ValueError, "even"),
        (lambda: pkg.rms_norm_int8(x[0], g), ValueError, "2-D"),
        (lambda: pkg.rms_norm_int8(x, g[:5]), ValueError, "elements"),
        (lambda: pkg.rms_norm_int8(x.t(), g), ValueError, "contiguous"),
        (lambda: pkg.rms_norm_int8(x.double(), g), TypeError, "element type"),
        (lambda: pkg.rms_norm_int8(x, g, residual=x.half()), ValueError, "residual"),
        (lambda: pkg.rms_norm_int8(x, g, residual_out=x), ValueError, "needs a residual"),
        (lambda: pkg.rms_norm_int8(x, g, q=x), TypeError, "q must be"),
        (lambda: pkg.layer_norm_int8(x, g, g.half()), TypeError, "dtypes differ"),
        (lambda: pkg.dequantize_embedding_int8(x, s), TypeError, "int8"),
    ]
    for call, kind, needle in bad:
        with pytest.raises(kind, match=needle):
            call()
    flat = torch.zeros(4 * 64 + 1, device=dev)
    with pytest.raises(pkg.EbagError, match="overlaps"):
        pkg.rms_norm_int8(flat[:-1].view(4, 64), g, residual=x, residual_out=flat[1:].view(4, 64))


@pytest.mark.parametrize("dim", [513, 1000, 1021, 2048, 4097, 5632, 14336, 16391, 32768, 40000])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
def test_wide_rows_are_quantised_as_narrow_ones(pkg, dev, dim, dt):
    """Bit for bit the expression that quantize_embedding_int8 states, rows with a stride and odd addresses too."""
    g = _gen(dim)
    x = torch.randn(37, dim, generator=g) * torch.exp(torch.randn(37, 1, generator=g))
    x[5] = 0
    x[7, dim - 1] = 50.0
    x = x.to(dt)
    for shift, pad in ((0, 0), (1, 0), (0, 5), (3, 8)):
        print(f"wide rows dim={dim} {dt} shift={shift} pad={pad}", flush=True)
        base = torch.zeros(37 * (dim + pad) + shift, dtype=dt, device=dev)
        view = base[shift:].view(37, dim + pad)[:, :dim]
        view.copy_(x)
        q, s = pkg.quantize_embedding_int8(view)
        want_s = torch.clamp(x.float().abs().amax(1) * np.float32(1 / 127), min=np.float32(1e-8))
        want_q = torch.clamp(torch.round(x.float() / want_s[:, None]), -128, 127).to(torch.int8)
        assert torch.equal(s.cpu(), want_s) and torch.equal(q.cpu(), want_q)


def test_more_wide_rows_than_a_launch_has(pkg, dev):
    """A workgroup of 256 threads a row: 2^24 rows and more are 2^32 threads, which no launch has."""
    rows, dim = 2 ** 24 + 5, 513
    w = torch.zeros(rows, dim, dtype=torch.bfloat16, device=dev)
    g = _gen(4)
    at = torch.tensor([0, 2 ** 24 - 2, 2 ** 24 - 1, 2 ** 24, rows - 1])
    some = torch.randn(len(at), dim, generator=g).to(torch.bfloat16)
    w[at.to(dev)] = some.to(dev)
    print("more wide rows than a launch has", flush=True)
    q, s = pkg.quantize_embedding_int8(w)
    torch.cuda.synchronize()
    del w
    want_q, want_s = pkg.quantize_embedding_int8(some.to(dev))
    assert torch.equal(q[at.to(dev)], want_q) and torch.equal(s[at.to(dev)], want_s)
    assert int((s != np.float32(1e-8)).sum()) == len(at)


@pytest.mark.parametrize("cols", [3, 40])
def test_more_norm_rows_than_a_launch_has(pkg, dev, cols):
    """Up to 1,024 threads a row, fewer than 2^32 in a launch: the rows of several launches."""
    rows = 2 ** 24 + 5
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device=dev)
    edge = (2 ** 32 - 1) // 1024  # the first launch's rows, if it has as many as 1,024 threads for each allow
    at = torch.tensor([0, edge - 1, edge, 2 * edge - 1, 2 * edge, 4 * edge, 2 ** 24 - 1, 2 ** 24, rows - 1])
    some = torch.randn(len(at), cols, generator=_gen(5)).to(torch.bfloat16)
    x[at.to(dev)] = some.to(dev)
    w = torch.ones(cols)
    print(f"more norm rows than a launch has, {cols} wide", flush=True)
    q, s, h = pkg.rms_norm_int8(x, w.to(dev), residual=x, residual_out=x)
    torch.cuda.synchronize()
    _check_norm((q[at.to(dev)], s[at.to(dev)], h[at.to(dev)]), some, some, w, None, 1e-5, False)
    assert int((s != np.float32(1e-8)).sum()) == len(at) and int(h.any(1).sum()) == len(at)


@pytest.mark.parametrize("cols", [20, 32])
def test_more_product_rows_than_a_launch_takes(pkg, dev, cols):
    """2^20 rows a launch: the rows of three, the last of a few."""
    rows, n = 2 ** 21 + 37, 24
    q, s, w, ws, bias = _operands(rows, cols, n, 7)
    args = [t.to(dev) for t in (q, s, w, ws)]
    print(f"more product rows than a launch takes, {cols} wide", flush=True)
    y = pkg.linear_int8(*args, bias=bias.to(dev))
    torch.cuda.synchronize()
    at = torch.cat([torch.arange(70), *(torch.arange(e - 70, e + 37) for e in (2 ** 20, 2 ** 21))])
    assert torch.equal(y[at.to(dev)].cpu(), torch.from_numpy(_value(q[at], s[at], w, ws, bias)).to(torch.bfloat16))
    # every other row against the same product of the rows around it
    for lo in range(0, rows, 300000):
        part = pkg.linear_int8(args[0][lo:lo + 300000], args[1][lo:lo + 300000], *args[2:], bias=bias.to(dev))
        assert torch.equal(y[lo:lo + 300000], part)
    z = pkg.gated_linear_int8(*args, bias=bias.to(dev))
    assert torch.equal(z[2 ** 20 - 9:2 ** 20 + 9], pkg.gated_linear_int8(args[0][2 ** 20 - 9:2 ** 20 + 9], args[1][2 ** 20 - 9:2 ** 20 + 9],
                                                                         *args[2:], bias=bias.to(dev)))
