"""The training operators of this package as cases that can be timed and compared: the embedding lookup
with a scale and its gradient by sorted ids, the gradient of the pooled bags, dropout from a
counter-based generator, the layer norm with dropout and the residual's addition in it, forward and
backward, and the encoder's front end as a training step runs it.

listed() gives the cases, draw() more of the same ranges, prepare() what the program holds before the
call, run() one call, work() the bytes and operations it cannot do without, exact() the results in 64
bits. Where `own` is false run() computes the plain form with elementary torch operations in 32 bits.
"""
from __future__ import annotations

import functools
import importlib.util
import math
import os
import sys

import numpy as np
import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_PACKAGE = "cti_inference_optimization_amd"
_EPS = 1e-5


def _package():
    """The package of the tree in the working folder (its folder's name is no Python identifier)."""
    if _PACKAGE in sys.modules:
        return sys.modules[_PACKAGE]
    folder = os.path.join(os.getcwd(), "cti-inference-optimization_amd")
    spec = importlib.util.spec_from_file_location(_PACKAGE, os.path.join(folder, "__init__.py"),
                                                  submodule_search_locations=[folder])
    module = importlib.util.module_from_spec(spec)
    sys.modules[_PACKAGE] = module
    spec.loader.exec_module(module)
    return module


# ------------------------------------------------------------------------------------------------
# The cases
# ------------------------------------------------------------------------------------------------
def _lookup(name, **kw):
    """Rows of a table, scaled (a model's input embedding)."""
    case = dict(name=name, kind="lookup", ids=1024, rows=32000, dim=4096, dtype="bf16", index="int64")
    case.update(kw)
    return case


def _lookup_grad(name, **kw):
    """The dense gradient of the table behind such a lookup: Zipf ids, as tokens have them."""
    case = dict(name=name, kind="lookup_grad", ids=16384, rows=32000, dim=2048, dtype="bf16", out="bf16",
                index="int64", zipf=1.1, padding=False)
    case.update(kw)
    return case


def _bag_grad(name, **kw):
    """The gradient of the tables behind pooled bags: one table that all slots share, in the reference's
    layout, as the rows that were looked up (`compact`); or a table for each field, whole."""
    case = dict(name=name, kind="bag_grad", batch=4096, fields=28, rows=2_000_000, dim=128, mean_len=8.0, cap=256,
                pooling="sum", shared=True, compact=True, dtype="bf16", out="bf16", index="int64", zipf=1.1, padding=False)
    case.update(kw)
    return case


def _dropout(name, **kw):
    """Dropout forward and backward (the mask made twice, stored never), with the residual's addition or without."""
    case = dict(name=name, kind="dropout", rows=1024, cols=4096, p=0.1, residual=True, dtype="bf16")
    case.update(kw)
    return case


def _norm(name, **kw):
    """Dropout, the residual's addition and the layer norm, forward and backward, with the gradients of
    the norm's parameters and a gradient arriving at the residual stream."""
    case = dict(name=name, kind="norm", rows=1024, cols=4096, p=0.1, residual=True, dtype="bf16", params="bf16")
    case.update(kw)
    return case


def _front(name, **kw):
    """The encoder's front end in a training step: bags pooled, dropout, layer norm; back to the rows of
    the table that were looked up."""
    case = dict(name=name, kind="front", batch=4096, fields=28, rows=2_000_000, dim=128, mean_len=8.0, cap=256, p=0.1,
                dtype="bf16", params="fp32", index="int64", zipf=1.1)
    case.update(kw)
    return case


def listed():
    return [
        # One id: launch latency is all there is.
        _lookup("lookup-one", ids=1),
        # The tokens of a batch of prompts, a wide table: a gather at the memory's rate.
        _lookup("lookup-prompt", ids=16384, rows=128000),
        # A language model's embedding after a step of 16,384 tokens: the whole table's gradient.
        _lookup_grad("lookup-grad-tokens"),
        # Odd sizes in every direction, a padding row, few rows that are hit often, 32-bit ids.
        _lookup_grad("lookup-grad-odd", ids=5001, rows=1003, dim=333, dtype="fp16", out="fp32", index="int32",
                     padding=True),
        # The package's headline batch and table, backwards.
        _bag_grad("bag-grad-4096"),
        # The package's small configuration: fp32 tables of 10,000 x 64, one for each field, short bags.
        _bag_grad("bag-grad-fields", batch=256, rows=10_000, dim=64, mean_len=3.0, cap=32, shared=False, compact=False,
                  dtype="fp32", out="fp32", zipf=0.0),
        # A few rows of a small batch: latency.
        _dropout("dropout-few", rows=16, cols=1024),
        # A training batch: one pass over memory each way.
        _dropout("dropout-batch", rows=16384),
        # The encoder's rows of a small batch.
        _norm("norm-few", rows=128, cols=28 * 128, p=0.0, residual=False, params="fp32"),
        # An odd number of rows of an odd width, half precision.
        _norm("norm-odd", rows=3001, cols=1021, dtype="fp16", params="fp32"),
        # A block's norm over a training batch: the largest pass over memory here.
        _norm("norm-batch", rows=16384),
        # Everything together at the headline batch.
        _front("front-4096"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed cases' ranges: sizes spread over them, odd ones among them."""
    kind = rng.choice(["lookup", "lookup_grad", "lookup_grad", "bag_grad", "bag_grad", "dropout", "norm", "norm", "front"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    step = rng.choice([1, 2, 8, 16, 64])  # what a width is a multiple of

    def width(lo, hi):
        return max(step, _log(rng, lo, hi) // step * step)

    index = rng.choice(["int64", "int32"])
    if kind == "lookup":
        dim = width(16, 8192)
        rows = min(_log(rng, 1000, 2_000_000), 2 ** 29 // dim)
        return _lookup("", ids=min(_log(rng, 1, 65536), 2 ** 26 // dim), rows=rows, dim=dim, dtype=dtype, index=index)
    if kind == "lookup_grad":
        dim = width(16, 8192)
        return _lookup_grad("", ids=min(_log(rng, 1, 65536), 2 ** 25 // dim), rows=min(_log(rng, 100, 200_000), 2 ** 26 // dim),
                            dim=dim, dtype=dtype, out=rng.choice([dtype, "fp32"]), index=index,
                            zipf=rng.choice([0.0, 0.8, 1.1]), padding=rng.random() < 0.5)
    if kind == "bag_grad":
        shared = rng.random() < 0.6
        fields = rng.choice([1, 3, 13, 28])
        dim = min(width(16, 512), 512)
        mean_len = rng.choice([1.0, 3.0, 8.0, 16.0])
        batch = max(1, min(_log(rng, 1, 8192), int(2 ** 26 / (fields * dim * mean_len))))
        rows = _log(rng, 100, 2_000_000) if shared else min(_log(rng, 100, 50_000), 2 ** 26 // (dim * fields))
        return _bag_grad("", batch=batch, fields=fields, rows=rows, dim=dim, mean_len=mean_len, shared=shared, compact=shared,
                         pooling=rng.choice(["sum", "mean"]), dtype=dtype, out=rng.choice([dtype, "fp32"]), index=index,
                         zipf=rng.choice([0.0, 0.8, 1.1]), padding=rng.random() < 0.3)
    if kind == "front":
        dim = rng.choice([16, 32, 64, 128, 256])
        return _front("", batch=_log(rng, 16, 4096), fields=rng.choice([7, 28]), rows=_log(rng, 1000, 1_000_000), dim=dim,
                      mean_len=rng.choice([1.0, 4.0, 8.0]) * min(1.0, 128 / dim), p=rng.choice([0.0, 0.1, 0.5]),
                      dtype=rng.choice(["bf16", "fp32"]), index=index)
    cols = width(64, 16384)
    rows = max(1, min(_log(rng, 1, 32768), 2 ** 26 // cols // (2 if dtype == "fp32" else 1)))
    p = rng.choice([0.05, 0.1, 0.2, 0.5])
    if kind == "dropout":
        return _dropout("", rows=rows, cols=cols, p=p, residual=rng.random() < 0.5, dtype=dtype)
    return _norm("", rows=rows, cols=cols, p=rng.choice([0.0, p]), residual=rng.random() < 0.7, dtype=dtype,
                 params=rng.choice([dtype, "fp32"]))


# ------------------------------------------------------------------------------------------------
# Inputs
# ------------------------------------------------------------------------------------------------
def _zipf(gen, n, rows, s):
    """n ids of `rows`: uniform (s = 0), or bounded Zipf with the frequent ones scattered over the table."""
    if s == 0.0:
        return torch.randint(0, rows, (n,), generator=gen, device="cuda")
    weight = torch.arange(1, rows + 1, device="cuda", dtype=torch.float64).pow_(-s).cumsum_(0)
    u = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64) * weight[-1]
    rank = torch.searchsorted(weight, u).clamp_(max=rows - 1)
    a = next(k for k in (2654435761, 40503, 7919, 1) if math.gcd(k, rows) == 1)
    return (rank * a + 12345) % rows


def _bags(gen, case):
    """Lengths [fields, batch], geometric with the case's mean and an end, a few ids outside the table."""
    shape = (case["fields"], case["batch"])
    u = torch.rand(shape, generator=gen, device="cuda", dtype=torch.float64)
    lens = torch.floor(torch.log1p(-u) / math.log(1 - 1 / (case["mean_len"] + 1))).clamp_(0, case["cap"]).long()
    n = int(lens.sum())
    values = _zipf(gen, n, case["rows"], case["zipf"])
    if n:
        values[torch.rand(n, generator=gen, device="cuda") < 1e-3] = case["rows"] + 5  # clamped to the last row
    return lens, values


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    st = dict(case)
    kind = case["kind"]

    def randn(*shape, dtype=dt, size=1.0):
        return (size * torch.randn(*shape, generator=gen, device="cuda")).to(dtype)

    def seeds():
        # the generator's seed and the step's number: plain numbers that the training loop holds
        pair = torch.randint(0, 2 ** 62, (2,), generator=gen, device="cuda").tolist()
        st["seed"], st["offset"] = pair[0], pair[1] % 100_000

    if kind in ("lookup", "lookup_grad"):
        n, rows, dim = case["ids"], case["rows"], case["dim"]
        st["values"] = _zipf(gen, n, rows, case.get("zipf", 1.1)).to(getattr(torch, case["index"]))
        st["scale"] = math.sqrt(dim)
        if kind == "lookup":
            st["weight"] = randn(rows, dim, size=dim ** -0.5)
        else:
            st["grad"] = randn(n, dim)
    if kind in ("bag_grad", "front"):
        lens, values = _bags(gen, case)
        b, f, dim, n = case["batch"], case["fields"], case["dim"], values.numel()
        st["lens"], st["values"] = lens, values.to(getattr(torch, case["index"]))
        row_offsets = torch.zeros(f, b + 1, dtype=torch.int64, device="cuda")
        row_offsets[:, 1:] = lens.cumsum(1)
        st["row_offsets"] = row_offsets.reshape(-1)
        ends = lens.sum(1).cumsum(0)
        st["val_offsets"] = ends - lens.sum(1)
        st["offsets"] = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), lens.reshape(-1).cumsum(0)])
        if kind == "front":
            st["weight"] = randn(case["rows"], dim, size=0.01)
        elif not case["shared"]:
            st["tables"] = [torch.zeros(case["rows"], dim, dtype=_DTYPES[case["out"]], device="cuda") for _ in range(f)]
        if kind == "front" or case["compact"]:
            # buffers that a training loop keeps: as long as eight standard deviations above the mean of its batches
            bags, mean = b * f, case["mean_len"]
            most = min(int(bags * mean + 8 * math.sqrt(bags * mean * (mean + 1))) + 16, case["rows"])
            assert n <= most or most == case["rows"], "a batch past its buffers"
            st["grad_rows"] = (torch.full((most,), -1, dtype=torch.int64, device="cuda"),
                               torch.zeros(most, dim, dtype=_DTYPES[case.get("out", case["dtype"])], device="cuda"),
                               torch.zeros(1, dtype=torch.int64, device="cuda"))
        if kind == "bag_grad":
            st["grad"] = randn(b, f * dim)
        else:
            case = dict(case, rows=b, cols=f * dim, residual=False)
    if kind in ("dropout", "norm", "front"):
        rows, cols = case["rows"], case["cols"]
        seeds()
        if kind != "front":
            st["x"] = randn(rows, cols)
        st["residual_in"] = randn(rows, cols, size=2.0) if case["residual"] else None
        st["grad"] = randn(rows, cols)
        if kind != "dropout":
            pt = _DTYPES[case["params"]]
            st["gamma"] = randn(cols, dtype=torch.float32, size=0.1).add_(1.0).to(pt)
            st["beta"] = randn(cols, dtype=pt, size=0.1)
            st["grad_h"] = randn(rows, cols) if case["residual"] else None
    return st


# ------------------------------------------------------------------------------------------------
# The plain forms
# ------------------------------------------------------------------------------------------------
def _keep(st, rows, cols):
    """(what is kept [rows, cols], the factor of what is kept). Philox4x32-10 (Salmon et al., 2011) of the
    counter (row, column // 8, offset low, offset high) and the key (seed low, seed high) gives four words:
    16 bits for each of 8 columns, low half first. Dropped where they are below round(65536 p)."""
    mask32 = 0xFFFFFFFF
    t = math.floor(65536 * st["p"] + 0.5)
    blocks = (cols + 7) // 8
    c = [torch.arange(rows, device="cuda").repeat_interleave(blocks), torch.arange(blocks, device="cuda").repeat(rows),
         torch.full((rows * blocks,), st["offset"] & mask32, device="cuda"),
         torch.full((rows * blocks,), st["offset"] >> 32, device="cuda")]
    k0, k1 = st["seed"] & mask32, st["seed"] >> 32
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57  # 64 bits, of which the sign is one
        c = [((b >> 32) & mask32) ^ c[1] ^ k0, b & mask32, ((a >> 32) & mask32) ^ c[3] ^ k1, a & mask32]
        k0, k1 = (k0 + 0x9E3779B9) & mask32, (k1 + 0xBB67AE85) & mask32
    words = torch.stack(c, dim=1)
    halves = torch.stack([words & 0xFFFF, words >> 16], dim=2).reshape(rows, blocks * 8)[:, :cols]
    return halves >= t, (65536.0 / (65536 - t) if t < 65536 else 0.0)


def _plain_dropout(st, x):
    if st["p"] == 0.0:
        return x
    keep, factor = _keep(st, *x.shape)
    return torch.where(keep, x * factor, torch.zeros_like(x))


def _plain_sums(rows, ids, contributions, padding):
    """Sums of the contributions of each id: [rows, dim]."""
    if padding:
        contributions = torch.where((ids == 0)[:, None], torch.zeros_like(contributions), contributions)
    return torch.zeros(rows, contributions.shape[1], device="cuda").index_add_(0, ids, contributions)


def _plain_compact(st, ids, contributions, rows, grads, padding):
    """The same for the ids that occur, in their order: padded with -1 and 0 to the buffers' length."""
    if padding:
        contributions, ids = contributions[ids != 0], ids[ids != 0]
    present, place = torch.unique(ids, return_inverse=True)
    sums = torch.zeros(grads.shape, device="cuda").index_add_(0, place, contributions)
    out = torch.full_like(rows, -1)
    out[:present.numel()] = present
    return out, sums.to(grads.dtype), torch.full((1,), present.numel(), dtype=torch.int64, device="cuda")


def _field_and_sample(st):
    """The field and the sample of each id."""
    bag = torch.repeat_interleave(torch.arange(st["lens"].numel(), device="cuda"), st["lens"].reshape(-1))
    return bag // st["batch"], bag % st["batch"]


def _plain_bag_grad(st, grad):
    """As a list: the compact rows' numbers, sums and count, or each table's gradient."""
    f, b = _field_and_sample(st)
    ids = st["values"].long().clamp(0, st["rows"] - 1)
    g = grad.float().view(st["batch"], st["fields"], st["dim"])[b, f]
    if st.get("pooling") == "mean":
        g = g / st["lens"][f, b][:, None].float()
    if "grad_rows" in st:
        return list(_plain_compact(st, ids, g, *st["grad_rows"][:2], st.get("padding", False)))
    if st["padding"]:
        g = torch.where((ids == 0)[:, None], torch.zeros_like(g), g)
    sums = _plain_sums(st["rows"] * st["fields"], f * st["rows"] + ids, g, False)
    return list(sums.to(_DTYPES[st["out"]]).view(st["fields"], st["rows"], st["dim"]).unbind(0))


def _plain_norm(st, x, dt):
    """Forward and backward; what is stored between them is stored in the case's type."""
    h = _plain_dropout(st, x.float())
    if st.get("residual_in") is not None:
        h = h + st["residual_in"].float()
    h = h.to(dt)
    v = h.float()
    mean = v.mean(dim=1, keepdim=True)
    rstd = torch.rsqrt(((v - mean) ** 2).mean(dim=1, keepdim=True) + _EPS)
    hat, gamma, g = (v - mean) * rstd, st["gamma"].float(), st["grad"].float()
    y = hat * gamma + st["beta"].float()
    gg = g * gamma
    dh = rstd * (gg - gg.mean(dim=1, keepdim=True) - hat * (gg * hat).mean(dim=1, keepdim=True))
    if st.get("grad_h") is not None:
        dh = dh + st["grad_h"].float()
    dx = _plain_dropout(st, dh)
    pt = st["gamma"].dtype
    out = [y.to(dt), h, mean[:, 0], rstd[:, 0], dx.to(dt), (g * hat).sum(0).to(pt), g.sum(0).to(pt)]
    return out + [dh.to(dt)] if st.get("residual_in") is not None else out


def run(st):
    kind, dt = st["kind"], _DTYPES[st["dtype"]]
    if own:
        return _run_own(st, kind)
    if kind == "lookup":
        return (st["weight"][st["values"].long()].float() * st["scale"]).to(dt)
    if kind == "lookup_grad":
        ids = st["values"].long()
        return (_plain_sums(st["rows"], ids, st["grad"].float(), st["padding"]) * st["scale"]).to(_DTYPES[st["out"]])
    if kind == "bag_grad":
        return _plain_bag_grad(st, st["grad"])
    if kind == "dropout":
        y = _plain_dropout(st, st["x"].float())
        if st["residual_in"] is not None:
            y = y + st["residual_in"].float()
        return [y.to(dt), _plain_dropout(st, st["grad"].float()).to(dt)]
    if kind == "norm":
        return _plain_norm(st, st["x"], dt)
    f, b = _field_and_sample(st)
    rows = st["weight"][st["values"].long().clamp(0, st["rows"] - 1)].float()
    pooled = torch.zeros(st["batch"] * st["fields"], st["dim"], device="cuda").index_add_(0, b * st["fields"] + f, rows)
    out = _plain_norm(st, pooled.view(st["batch"], -1).to(dt), dt)
    return [*out, *_plain_bag_grad(st, out[4])]


def _run_own(st, kind):
    """The calls that a user makes of the package."""
    pkg = _package()
    if kind == "lookup":
        return pkg.embedding_lookup(st["values"], st["weight"], st["scale"])
    if kind == "lookup_grad":
        return pkg.embedding_lookup_backward(st["grad"], st["values"], st["rows"], st["scale"],
                                             padding_idx=0 if st["padding"] else None, grad_dtype=_DTYPES[st["out"]])
    if kind == "bag_grad":
        padding = 0 if st["padding"] else None
        if st["shared"]:
            return list(pkg.fused_all_slots_embedding_backward(
                st["grad"], st["values"], st["val_offsets"], st["row_offsets"], st["batch"], st["dim"], st["rows"] - 1,
                pooling=st["pooling"], padding_idx=padding, compact=True, out=st["grad_rows"]))
        return pkg.embedding_bag_backward(st["grad"], st["values"], st["offsets"], st["tables"], pooling=st["pooling"],
                                          padding_idx=padding)
    if kind == "dropout":
        return [pkg.dropout(st["x"], st["p"], st["seed"], st["offset"], residual=st["residual_in"]),
                pkg.dropout_backward(st["grad"], st["p"], st["seed"], st["offset"])]
    x = st.get("x")
    if kind == "front":
        x = torch.empty(st["batch"], st["fields"] * st["dim"], dtype=st["weight"].dtype, device="cuda")
        pkg.fused_all_slots_embedding(st["values"], st["val_offsets"], st["row_offsets"], st["weight"], x, st["batch"],
                                      st["dim"], st["rows"] - 1)
    y, h, mean, rstd = pkg.dropout_add_layer_norm(x, st["gamma"], st["beta"], _EPS, residual=st["residual_in"], p=st["p"],
                                                  seed=st["seed"], offset=st["offset"])
    dx, dgamma, dbeta, dh = pkg.dropout_add_layer_norm_backward(
        st["grad"], h, mean, rstd, st["gamma"], grad_h=st["grad_h"], residual=st["residual_in"] is not None, p=st["p"],
        seed=st["seed"], offset=st["offset"])
    out = [y, h, mean, rstd, dx, dgamma, dbeta]
    if kind == "norm":
        return out if dh is None else out + [dh]
    return [*out, *pkg.fused_all_slots_embedding_backward(
        dx, st["values"], st["val_offsets"], st["row_offsets"], st["batch"], st["dim"], st["rows"] - 1, compact=True,
        out=st["grad_rows"])]


# ------------------------------------------------------------------------------------------------
# The work and the results in 64 bits
# ------------------------------------------------------------------------------------------------
@functools.lru_cache(maxsize=256)
def _distinct(n, rows, s):
    """How many of the rows n ids hit on average."""
    if s == 0.0:
        return rows * -math.expm1(n * math.log1p(-1 / rows)) if rows > 1 else 1.0
    p = np.arange(1, rows + 1, dtype=np.float64) ** -s
    p /= p.sum()
    return float(-np.expm1(n * np.log1p(-np.minimum(p, 1 - 1e-12))).sum())


def work(case):
    kind, b = case["kind"], _BYTES[case["dtype"]]
    ids = {"int64": 8, "int32": 4}.get(case.get("index"), 0)
    if kind == "lookup":
        n, d = case["ids"], case["dim"]
        return {"bytes": _distinct(n, case["rows"], 1.1) * d * b + n * (ids + d * b), "flops": n * d}
    if kind == "lookup_grad":
        n, d = case["ids"], case["dim"]
        return {"bytes": n * (ids + d * b) + case["rows"] * d * _BYTES[case["out"]], "flops": n * d}
    if kind in ("bag_grad", "front"):
        bags, d = case["batch"] * case["fields"], case["dim"]
        n = int(bags * case["mean_len"])
        distinct = _distinct(n, case["rows"], case["zipf"])
        written = case["rows"] * case["fields"] if kind == "bag_grad" and not case["compact"] else distinct
        back = {"bytes": bags * (d * b + 8) + n * ids + written * (d * _BYTES[case.get("out", case["dtype"])] + 8),
                "flops": n * d}
        if kind == "bag_grad":
            return back
        # table rows in; y and grad once, and the pooled block, h and dx, which one call writes and the next one reads
        block = bags * d
        return {"bytes": back["bytes"] + (distinct * d + (7 if case["p"] else 6) * block) * b + n * ids,
                "flops": back["flops"] + n * d + 30 * block}
    m, c = case["rows"], case["cols"]
    if kind == "dropout":
        return {"bytes": (5 if case["residual"] else 4) * m * c * b, "flops": 20 * m * c}
    # x in, y out; grad and h in, dx out; h out where it is not x itself; residual and grad_h in, its own gradient out
    arrays = 5 + (1 if case["residual"] or case["p"] else 0) + (2 if case["residual"] else 0)
    arrays += 1 if case["residual"] and case["p"] else 0
    return {"bytes": arrays * m * c * b + 16 * m + 4 * c * _BYTES[case["params"]], "flops": 30 * m * c}


def exact(case, seed):
    st = prepare(case, seed)
    kind, d, dt = case["kind"], torch.float64, _DTYPES[case["dtype"]]

    def dropped(v):
        if case["p"] == 0.0:
            return v
        rows, cols = v.shape
        blocks, u = -(-cols // 8), np.uint64
        low = u(0xFFFFFFFF)
        row, block = np.meshgrid(np.arange(rows, dtype=u), np.arange(blocks, dtype=u), indexing="ij")
        x0, x1 = row, block
        x2, x3 = np.full_like(row, st["offset"] % 2 ** 32), np.full_like(row, st["offset"] // 2 ** 32)
        for r in range(10):
            key0 = u((st["seed"] % 2 ** 32 + r * 0x9E3779B9) % 2 ** 32)
            key1 = u((st["seed"] // 2 ** 32 + r * 0xBB67AE85) % 2 ** 32)
            left, right = x0 * u(0xD2511F53), x2 * u(0xCD9E8D57)
            x0, x1, x2, x3 = (right >> u(32)) ^ x1 ^ key0, right & low, (left >> u(32)) ^ x3 ^ key1, left & low
        bits = np.empty((rows, blocks, 8), dtype=np.int32)
        for j, w in enumerate((x0, x1, x2, x3)):
            bits[:, :, 2 * j], bits[:, :, 2 * j + 1] = w % u(65536), w // u(65536)
        t = round(case["p"] * 65536)
        gone = torch.from_numpy(bits.reshape(rows, -1)[:, :cols] < t).to(v.device)
        return (v / (1 - t / 65536)).masked_fill(gone, 0.0)

    def sums(ids, rows_of):
        """(ids that occur, their sums) by differences of running sums over the sorted list."""
        order = torch.argsort(ids, stable=True)
        running = torch.cumsum(rows_of(order), dim=0)
        present, counts = torch.unique_consecutive(ids[order], return_counts=True)
        last = counts.cumsum(0) - 1
        total = running[last]
        total[1:] -= running[last[:-1]]
        return present, total

    def bag_grad(grad):
        flat = st["lens"].flatten()
        starts = torch.nn.functional.pad(flat.cumsum(0), (1, 0))
        position = torch.arange(st["values"].numel(), device="cuda")
        bag = torch.searchsorted(starts[1:].contiguous(), position, right=True)
        field, sample = bag.div(case["batch"], rounding_mode="floor"), bag.remainder(case["batch"])
        ids = torch.minimum(st["values"].to(torch.int64), torch.tensor(case["rows"] - 1, device="cuda"))
        blocks = grad.to(d).reshape(case["batch"] * case["fields"], case["dim"])
        weight = 1.0 / flat.to(d)[bag] if case.get("pooling") == "mean" else torch.ones(bag.numel(), dtype=d, device="cuda")
        live = torch.nonzero(ids != 0)[:, 0] if case.get("padding") else position

        def rows_of(order):
            at = live[order]
            return blocks[sample[at] * case["fields"] + field[at]] * weight[at, None]

        compact = "grad_rows" in st
        key = ids[live] if compact else ids[live] + field[live] * case["rows"]
        if key.numel():
            present, total = sums(key, rows_of)
        else:
            present, total = key, torch.zeros(0, case["dim"], dtype=d, device="cuda")
        if compact:
            rows, grads = torch.full_like(st["grad_rows"][0], -1), torch.zeros(st["grad_rows"][1].shape, dtype=d, device="cuda")
            rows[:len(present)], grads[:len(present)] = present, total
            return [rows, grads, torch.tensor([len(present)], device="cuda")]
        whole = torch.zeros(case["rows"] * case["fields"], case["dim"], dtype=d, device="cuda")
        whole[present] = total
        return list(whole.split(case["rows"]))

    def norm(x):
        h = dropped(x.to(d))
        if st.get("residual_in") is not None:
            h = h + st["residual_in"].to(d)
        h_out = h
        h = h.to(dt).to(d)  # the norm and its gradient are of what is stored
        n = h.shape[1]
        mean = h.sum(1) / n
        var = (h * h).sum(1) / n - mean * mean
        inv = 1 / torch.sqrt(var + _EPS)
        z = (h - mean.unsqueeze(1)) * inv.unsqueeze(1)
        g = st["grad"].to(d)
        a = g * st["gamma"].to(d).unsqueeze(0)
        dh = (n * a - a.sum(1, keepdim=True) - z * (a * z).sum(1, keepdim=True)) * (inv / n).unsqueeze(1)
        if st.get("grad_h") is not None:
            dh = dh + st["grad_h"].to(d)
        y = torch.addcmul(st["beta"].to(d).unsqueeze(0), z, st["gamma"].to(d).unsqueeze(0))
        out = [y, h_out, mean, inv, dropped(dh), torch.sum(g * z, 0), torch.sum(g, 0)]
        return [*out, dh] if st.get("residual_in") is not None else out

    if kind == "lookup":
        return torch.nn.functional.embedding(st["values"].long(), st["weight"]).to(d) * math.sqrt(case["dim"])
    if kind == "lookup_grad":
        ids = st["values"].long()
        live = torch.nonzero(ids != 0)[:, 0] if case["padding"] else torch.arange(ids.numel(), device="cuda")
        out = torch.zeros(case["rows"], case["dim"], dtype=d, device="cuda")
        if live.numel():
            present, total = sums(ids[live], lambda order: st["grad"][live[order]].to(d))
            out[present] = total * st["scale"]
        return out
    if kind == "bag_grad":
        return bag_grad(st["grad"])
    if kind == "dropout":
        y = dropped(st["x"].to(d))
        return [y if st["residual_in"] is None else y + st["residual_in"].to(d), dropped(st["grad"].to(d))]
    if kind == "norm":
        return norm(st["x"])
    # the pooled block is rows of the case's type, as is the gradient that goes back through it
    ids = st["values"].long().clamp(max=case["rows"] - 1)
    ends = st["lens"].flatten().cumsum(0)
    running = torch.nn.functional.pad(torch.cumsum(st["weight"][ids].to(d), dim=0), (0, 0, 1, 0))
    pooled = running[ends] - running[ends - st["lens"].flatten()]
    pooled = pooled.view(case["fields"], case["batch"], case["dim"]).transpose(0, 1).reshape(case["batch"], -1)
    out = norm(pooled.float().to(dt))
    return [*out, *bag_grad(out[4].to(dt))]
