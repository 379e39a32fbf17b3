"""The int8 Linear in every form that its dispatch can choose: each of them plain and gated, whole and with K split, as
the whole product and as the columns left over behind rounds of large tiles, with and without a rest of K, and the rows
form in each of its step classes. Bit for bit: sums in float64 are exact, then one rounding an operation.

test_int8_plans_cpu.py holds the list against the dispatch rules.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

# rows, columns, outputs, 16-byte addresses, workspace
PLAIN = [
    (7926, 2, 4087, 0, 1), (2533, 64, 12775, 1, 1),
    (1, 1, 1, 0, 0), (1, 514, 1, 0, 1), (1, 1027, 1, 0, 1), (1, 2057, 1, 0, 1), (1, 4222, 1, 0, 1),
    (1, 4574, 1, 0, 1), (2, 2112, 199, 1, 1), (66, 2, 13845, 0, 1), (6, 2176, 199, 1, 1), (5, 3200, 332, 1, 1),
    (2, 912, 3218, 1, 1), (329, 3168, 6, 1, 1), (75, 10768, 12, 1, 1), (13057, 1, 1025, 0, 1), (52, 10880, 24, 1, 1),
    (13060, 1, 1059, 0, 1), (13142, 1, 1157, 0, 1), (13069, 1, 1234, 0, 1), (13387, 1, 1219, 0, 1),
    (10, 11648, 142, 1, 1), (11, 12096, 139, 1, 1), (907, 2, 11744, 0, 1), (67, 5286, 70, 0, 1),
    (3044, 1024, 9, 1, 1), (117, 4862, 68, 0, 1), (34, 12752, 97, 1, 1), (37, 15104, 81, 1, 1),
    (82, 14784, 39, 1, 1), (131, 9088, 50, 1, 1), (98, 4634, 148, 0, 1), (150, 5767, 124, 0, 1),
    (962, 16, 11464, 1, 1), (1250, 656, 259, 1, 1), (13060, 16, 1057, 1, 0), (318, 646, 1085, 0, 1),
    (183, 7488, 172, 1, 1), (13106, 16, 1153, 1, 0), (13075, 16, 1226, 1, 0), (13058, 16, 1239, 1, 0),
    (1026, 513, 13066, 0, 1), (1026, 1040, 13059, 1, 1), (1025, 2057, 13058, 0, 1), (13803, 16192, 132, 1, 1),
    (11018, 3229, 1281, 0, 1), (13065, 3488, 1025, 1, 1), (15649, 3232, 1025, 1, 1), (391, 11930, 11138, 0, 1),
    (15514, 3294, 1025, 0, 1), (1026, 4111, 13057, 0, 1), (9299, 4448, 1537, 1, 1), (9274, 4480, 1537, 1, 1),
    (1808, 5100, 8262, 0, 1), (1378, 5168, 10847, 1, 1), (1862, 5888, 8211, 1, 1), (1291, 6704, 10770, 1, 1),
    (1814, 8320, 8207, 1, 1), (1677, 8192, 9217, 1, 1), (13222, 14828, 1156, 0, 1), (11189, 15632, 1413, 1, 1),
]
GATED = [
    (1, 1, 1, 0, 0), (1, 522, 1, 0, 1), (1, 1040, 1, 1, 1), (1, 2080, 1, 1, 1), (1, 2371, 1, 0, 1),
    (1, 3312, 1, 1, 1), (1, 3328, 1, 1, 1), (1, 4108, 1, 0, 1), (2, 2112, 98, 1, 1), (11957, 1, 35, 0, 0),
    (5, 2176, 104, 1, 1), (164, 5741, 2, 0, 1), (1, 768, 2973, 1, 1), (263, 8768, 2, 1, 1), (3, 1008, 1567, 1, 0),
    (3, 1024, 1559, 1, 1), (67, 11136, 7, 1, 1), (513, 1, 10881, 0, 1), (13111, 1, 529, 0, 1), (40, 10976, 17, 1, 1),
    (13067, 1, 581, 0, 1), (130, 11872, 6, 1, 1), (65, 16, 8989, 1, 0), (136, 12032, 6, 1, 1), (49, 8832, 30, 1, 1),
    (46, 7680, 47, 0, 1), (143, 6288, 33, 1, 1), (48, 9088, 69, 1, 1), (4107, 2, 3744, 0, 1), (196, 3046, 67, 0, 1),
    (377, 3918, 33, 0, 1), (3, 9216, 2120, 0, 1), (898, 16, 8468, 1, 0), (11355, 16, 705, 1, 0),
    (4003, 16, 3520, 1, 0), (13438, 129, 639, 0, 1), (9875, 129, 870, 0, 1), (13610, 144, 633, 1, 0),
    (14883, 144, 1089, 1, 1), (513, 513, 10883, 0, 1), (514, 1028, 10881, 0, 1), (15553, 907, 792, 0, 1),
    (517, 2052, 10889, 0, 1), (136, 9344, 11227, 1, 1), (132, 8608, 13599, 1, 1), (15591, 1088, 1307, 1, 1),
    (13192, 3468, 513, 0, 1), (14560, 3472, 513, 1, 1), (14940, 3475, 513, 0, 1), (11927, 3552, 641, 1, 1),
    (7276, 3878, 1026, 0, 1), (8043, 3776, 1025, 1, 1), (513, 5922, 10976, 0, 1), (516, 6208, 10895, 1, 1),
    (3101, 4976, 2447, 1, 1), (564, 6529, 10882, 0, 1), (1086, 5693, 6530, 0, 1), (586, 6355, 10928, 0, 1),
    (834, 6227, 8222, 0, 1), (13478, 14832, 578, 1, 1), (13302, 12164, 726, 0, 1),
]
CASES = [(*c, 0) for c in PLAIN] + [(*c, 1) for c in GATED]


@pytest.mark.parametrize("rows,cols,n,aligned,workspace,gated", CASES)
def test_every_form(pkg, dev, rows, cols, n, aligned, workspace, gated):
    print(f"form {rows}x{cols}->{n} aligned={aligned} workspace={workspace} gated={gated}", flush=True)
    g = torch.Generator(device=dev).manual_seed(rows + n)
    wrows = 2 * n if gated else n

    def int8(count, width):
        t = torch.empty(count * width + 1, dtype=torch.int8, device=dev)[0 if aligned else 1:][:count * width].view(count, width)
        return t.random_(-128, 128, generator=g)

    q, w = int8(rows, cols), int8(wrows, cols)
    s, ws = (torch.rand(k, generator=g, device=dev) / 100 for k in (rows, wrows))
    bias = torch.randn(wrows, generator=g, device=dev)
    v = q.double() @ w.double().t().contiguous()
    v = (v.float() * s[:, None]) * ws[None, :] + bias[None, :]
    if gated:
        v = torch.clamp(v[:, :n], min=0.0) * v[:, n:]
    for odt in (torch.bfloat16, torch.float16, torch.float32):
        if gated:
            got = pkg.gated_linear_int8(q, s, w, ws, bias, activation="relu", out_dtype=odt, split_k=bool(workspace))
        else:
            got = pkg.linear_int8(q, s, w, ws, bias, out_dtype=odt, split_k=bool(workspace))
        torch.cuda.synchronize()
        want = v.to(odt)
        assert torch.equal(got, want), (odt, int((got != want).sum()))
