"""Sizes of the int8 Linear past its limits, without a GPU: the tensors' checks and the launch are replaced, so the
sizes alone are at work."""
import types

import pytest
import torch


@pytest.fixture
def linear(pkg, monkeypatch):
    """linear(rows, cols, weight rows, gate): what _linear_int8 hands to the library for operands of these sizes."""
    ops = pkg.ops
    launched = []

    def check(name, q, scale_name, scale, index=None):
        return (*q.sizes, 0)

    monkeypatch.setattr(ops, "_check_int8_rows", check)
    monkeypatch.setattr(ops, "_launch", lambda index, fn, *args: launched.append(args))

    def operand(*sizes):
        return types.SimpleNamespace(sizes=sizes, device=torch.device("cpu"), data_ptr=lambda: 4096)

    def call(rows, cols, w_rows, gate=0, split_k=True):
        launched.clear()
        # (an output of no rows: no memory behind the sizes)
        out = torch.empty(0, dtype=torch.bfloat16)
        monkeypatch.setattr(ops, "_float_output", lambda *a: (out, pkg._capi.BF16))
        ops._linear_int8(operand(rows, cols), operand(rows), operand(w_rows, cols), operand(w_rows), None, gate, None,
                         torch.bfloat16, split_k)
        return launched[0]

    return call


@pytest.mark.parametrize("split_k", [False, True])
@pytest.mark.parametrize("rows,cols,w_rows,gate,needle", [
    (1, 131072, 32, 0, "cols"), (0, 2 ** 32 + 64, 32, 0, "cols"), (1, 2 ** 32 + 64, 32, 1, "cols"),
    (1, 2 ** 32, 32, 0, "cols"), (1, 64, 2 ** 32 + 5, 0, "out_features"), (0, 64, 2 ** 33 + 10, 1, "out_features"),
    (1, 64, 2 ** 30 + 1, 0, "out_features"), (1, 64, 2 ** 31 + 2, 2, "out_features"),
])
def test_sizes_that_32_bits_do_not_hold_are_refused(pkg, linear, rows, cols, w_rows, gate, needle, split_k):
    """The library takes columns and outputs as 32-bit numbers, and 2^32 + 64 columns would pass for 64."""
    with pytest.raises(pkg.EbagError, match=needle) as e:
        linear(rows, cols, w_rows, gate, split_k)
    assert e.value.status == pkg._capi.EUNSUPPORTED


def test_sizes_up_to_the_limits_reach_the_library_as_they_are(linear):
    for rows, cols, w_rows, gate, n in ((3, 131071, 7, 0, 7), (2 ** 33, 64, 32, 1, 16), (1, 1, 2 ** 30, 0, 2 ** 30)):
        args = linear(rows, cols, w_rows, gate, split_k=False)
        assert args[2] == rows and args[3] == cols and args[6] == n
