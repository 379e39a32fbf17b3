"""What the training operators' sources have to state themselves, because no run can be relied on to show that it is missing."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cti-inference-optimization_amd", "csrc")
BYTES = {"uint8_t": 1, "uint16_t": 2, "uint32_t": 4, "int32_t": 4, "float": 4, "uint2": 8, "Pair": 8, "uint4": 16, "float4": 16}


@pytest.mark.parametrize("name", ["ebag_backward.hip", "ebag_train_norm.hip"])
def test_lds_arrays_are_aligned_for_their_widest_access(name):
    """An LDS array of narrow numbers that is read or written by vectors says so in its declaration: a variable is otherwise
    aligned for its elements alone."""
    text = open(os.path.join(CSRC, name)).read()
    casts = {}
    for kind, array in re.findall(r"reinterpret_cast<(?:const )?(\w+)\*>\((s_\w+)", text):
        casts[array] = max(casts.get(array, 0), BYTES.get(kind, 0))
    checked = 0
    for align, kind, declared in re.findall(r"__shared__ (?:__align__\((\d+)\) )?(\w+) (s_[^;]+);", text):
        for array in re.findall(r"(s_\w+)\[", declared):
            if array in casts and kind in BYTES:
                # (one name in several kernels: of the narrow types only 16-bit numbers are cast here)
                if BYTES[kind] >= casts[array] or kind == "uint32_t" and array == "s_hist":
                    continue
                checked += 1
                assert int(align or BYTES[kind]) >= casts[array], f"{kind} {array} is accessed {casts[array]} bytes at a time"
    assert checked == (2 if name == "ebag_backward.hip" else 0)
