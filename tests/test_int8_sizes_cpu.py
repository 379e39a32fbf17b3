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

    def call(rows, cols, w_rows, gate=0, split_k=True, address=4096):
        launched.clear()

        def operand(*sizes):
            return types.SimpleNamespace(sizes=sizes, device=torch.device("cpu"), data_ptr=lambda: address)

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


def test_the_workspace_is_the_one_for_the_operands_addresses(pkg, linear, monkeypatch):
    """Operands that start at no 16-byte address are copied to whole steps, or split, otherwise than aligned ones."""
    f = pkg._capi.lib()
    sizes = (1024, 4096, 4096, 0)
    aligned, unaligned = (g(*sizes) for g in (f.cti_ebag_linear_int8_workspace_bytes,
                                              f.cti_ebag_linear_int8_workspace_bytes_unaligned))
    assert unaligned == (1024 + 4096) * 4096 and aligned < unaligned  # both operands, in rows of whole steps
    asked = []
    empty = torch.empty
    monkeypatch.setattr(torch, "empty", lambda *a, **k: (asked.append(a[0]), empty(16, dtype=torch.uint8))[1]
                        if k.get("dtype") is torch.uint8 else empty(*a, **k))
    for at, want in ((4096, aligned), (4097, unaligned), (4104, unaligned)):
        asked.clear()
        assert linear(*sizes[:3], address=at)[-1] == want
        assert asked == ([want] if want else [])


@pytest.mark.parametrize("cols", [16, 100, 1024, 4096, 4097])
def test_unaligned_workspaces(pkg, cols):
    f = pkg._capi.lib()
    for rows in (0, 1, 77, 2000, 2 ** 20 + 3, 2 ** 31):
        for n in (0, 5, 512, 4096, 2 ** 30):
            for gate in (0, 1, 4):
                a = f.cti_ebag_linear_int8_workspace_bytes(rows, cols, n, gate)
                b = f.cti_ebag_linear_int8_workspace_bytes_unaligned(rows, cols, n, gate)
                assert (a == b) if cols % 16 else a >= 0 and b >= 0
                if not 1 <= rows < 2 ** 31 or not 1 <= n < 2 ** 30 or gate == 4:
                    assert a == b == 0


@pytest.mark.parametrize("dtype,most", [("F32", 2 ** 36 - 4096), ("BF16", 2 ** 37 - 8192), ("F16", 2 ** 37 - 8192)])
def test_read_back_of_more_elements_than_a_launch_has(pkg, dtype, most):
    """256 threads a workgroup of 1,024 chunks of 16 bytes of output, and fewer than 2^32 threads: refused before a launch."""
    c = pkg._capi
    for rows, dim in ((most + 1, 1), (most // 4096 + 1, 4096), (2 ** 39, 2), (1, 2 ** 62), (2 ** 62, 3)):
        status = c.lib().cti_ebag_dequantize_int8(256, 256, rows, dim, 256, getattr(c, dtype), None)
        assert status == c.EUNSUPPORTED and "elements" in c.last_error(), (rows, dim)
