"""The bytes that the int8 norms write are the quotients', rint(y / scale) with IEEE division as
``quantize_embedding_int8`` rounds, next to the middle of two steps too, in every form of the kernel.

Rows of +1 and -1 have a mean square of 1 (and as many of each a mean of 0) exactly, and with eps = 0 the norm leaves
weight * x: the values to be quantised are the weights, whatever order the sums are taken in.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _weights(cols, seed):
    """fp32 values of which the first is the largest and the others lie within three of their last places of the middle
    of two steps; and their scale and bytes."""
    rng = np.random.default_rng(seed)
    top = np.float32(rng.uniform(0.5, 2.0))
    s = max(np.float32(top * np.float32(1 / 127)), np.float32(1e-8))
    step = rng.integers(0, 127, cols)
    w = ((step + 0.5) * np.float64(s)).astype(np.float32)
    w = (w.view(np.int32) + rng.integers(-3, 4, cols).astype(np.int32)).view(np.float32)
    w = np.minimum(w, top) * rng.choice(np.array([-1, 1], np.float32), cols)
    w[0] = top
    return w, s, np.clip(np.rint(w / s), -128, 127).astype(np.int8)


def test_the_weights_tell_a_quotient_from_a_product_with_the_reciprocal():
    """About one in ten of these values, whether the product is rounded before it is taken to a byte or not."""
    w, s, q = _weights(16384, 1)
    inv = np.float64(np.float32(1) / s)
    assert (np.rint(w.astype(np.float64) * inv).astype(np.int8) != q).sum() > 100
    assert (np.rint((w * np.float32(inv)).astype(np.float32)).astype(np.int8) != q).sum() > 100


@pytest.mark.parametrize("cols", [2, 6, 24, 64, 130, 256, 500, 1000, 1022, 2000, 4000, 4104, 8000, 10002, 16000, 32000, 40002])
@pytest.mark.parametrize("rows", [3, 1600])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_norms_round_quotients(pkg, dev, rows, cols, dt):
    w, s, q = _weights(cols, cols + rows)
    sign = np.ones((rows, cols), np.int8)
    order = np.random.default_rng(cols).permutation(cols)
    sign[:, order[: cols // 2]] = -1
    sign[1::2] *= -1
    x = torch.from_numpy(sign).to(dt).to(dev)
    weight = torch.from_numpy(w).to(dev)
    want_q = torch.from_numpy(sign * q[None, :])  # (-128 does not occur: the largest is 127 steps)
    for layer in (False, True):
        print(f"rounding rows={rows} cols={cols} {dt} layer={layer}", flush=True)
        got, scale = (pkg.layer_norm_int8(x, weight, torch.zeros_like(weight), 0.0) if layer
                      else pkg.rms_norm_int8(x, weight, 0.0))
        assert (scale.cpu().numpy() == s).all()
        off = got.cpu() != want_q
        assert not off.any(), (layer, int(off.sum()))


def test_read_back_is_rounded_to_fp32_and_then_to_fp16(pkg, dev):
    """Scales of which q * scale in fp32 is the middle of two fp16 numbers while the product itself is not: the last
    elements of an array, which are taken one by one, as well as whole vectors."""
    rng = np.random.default_rng(0)
    q = rng.integers(1, 128, 4_000_000).astype(np.int8)
    s = rng.uniform(0.001, 1, q.size).astype(np.float32)
    exact = q.astype(np.float64) * s  # 8 and 24 bits: exact
    twice = (q * s).astype(np.float32).astype(np.float16)
    at = np.flatnonzero(twice != exact.astype(np.float16))[:200]
    assert len(at) > 50
    q, s, twice = (torch.from_numpy(a[at]).to(dev) for a in (q, s, twice))
    for n in (1, 3, 8, 11, 16, len(at)):
        print(f"read back {n}", flush=True)
        for lo in range(0, len(at) - n + 1, n):
            got = pkg.dequantize_embedding_int8(q[lo:lo + n].view(n, 1), s[lo:lo + n], torch.float16)
            assert torch.equal(got[:, 0], twice[lo:lo + n]), (n, lo)
    # rows of 5 such elements of one scale each
    wide = q[:, None].expand(-1, 5).contiguous()
    assert torch.equal(pkg.dequantize_embedding_int8(wide, s, torch.float16), twice[:, None].expand(-1, 5))
