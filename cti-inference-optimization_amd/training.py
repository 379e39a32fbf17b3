"""Operators of a training step in front of and behind the encoder: the embedding lookup with a scale, the
gradients of tables behind lookups and pooled bags, dropout, and the layer norm with dropout and the
residual's addition in it.

The reference's kernels are forward-only; what its modules would train is what torch's do
(``nn.Embedding`` with ``padding_idx`` and ``nn.LayerNorm``, online_best/infer.py:948-950), and the
gradients here are theirs. Each operator comes as plain calls, forward and backward, that a training
loop or a captured graph makes itself (``embedding_lookup_backward``, ``embedding_bag_backward``,
``fused_all_slots_embedding_backward``, ``dropout_backward``, ``dropout_add_layer_norm_backward``), and
``embedding_lookup``, ``dropout``, ``dropout_add_layer_norm``, ``embedding_bag_train`` and
``fused_embedding_train`` take part in autograd by themselves where an input requires a gradient, in reverse
mode and once; inputs with a tangent (forward mode) are refused.

Gradients of tables come whole, or as the rows that occur (``compact``): ``rows`` (their numbers, ascending,
then -1), their sums and how many they are, all on the device, so that nothing waits for the count. The ids
are sorted for it and no sum is taken by atomics: results are the same bits in every run.

Dropout's mask is a function of seed, offset, row and column that both directions compute: nothing is stored.
A training loop gives each layer and step an offset of its own. ``seed`` may be an int64 tensor of two
numbers on the device, (seed, offset), to which the call's own offset is added: for captured graphs, which
replay the numbers that a call was given but read what lies in the tensor.

Arguments are validated on the host (no device synchronisation): ``ValueError`` / ``TypeError`` for
malformed calls, ``EbagError`` when the C ABI reports a failure. Everything runs on torch's current stream;
workspaces come from torch's allocator for the call.
"""
from __future__ import annotations

import ctypes
import functools
import itertools
import struct
from typing import Optional, Sequence

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _capi
from .ops import (_check_flat_layout, _check_output, _launch, _require_on, _same_offset_type, _table_descs,
                  embedding_bag_pooled, fused_all_slots_embedding)

_INDEX_TYPES = (torch.int64, torch.int32)
_FLOATS = (torch.float32, torch.bfloat16, torch.float16)


_grad_enabled = torch.is_grad_enabled


def _any_requires_grad(*tensors) -> bool:
    for t in tensors:
        if t is not None and t.requires_grad:
            return True
    return False


def _refuse_tangents(*tensors) -> None:
    """There is no forward mode, and a dual tensor has no requires_grad by which it would take autograd's way and be refused there."""
    if getattr(forward_ad, "_current_level", 0) >= 0:  # -1 outside of dual levels: unpack_dual takes as long as a small kernel
        for t in tensors:
            if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
                raise ValueError("an input has a tangent: this operator is differentiated in reverse mode only")


def _check_index(name: str, t: torch.Tensor, index: Optional[int] = None) -> int:
    index = _require_on(name, t, index)
    if t.dtype not in _INDEX_TYPES:
        raise TypeError(f"{name} must be int64 or int32 (got {t.dtype})")
    return index


def _check_padding(padding_idx: Optional[int], rows: int) -> int:
    if padding_idx is None:
        return -1
    if not 0 <= padding_idx < rows:
        raise ValueError(f"padding_idx {padding_idx} outside [0, {rows - 1}]")
    return int(padding_idx)


def _check_dim(dim: int) -> None:
    if dim >= 2 ** 31:  # ctypes drops the bits above
        raise _capi.EbagError(_capi.EUNSUPPORTED, f"dim {dim} >= 2^31")


_MOST_IDS, _MOST_ROWS, _MOST_COLUMNS, _MOST_FIELDS = 2 ** 30, 2 ** 31 - 2, 2 ** 22, 64  # of a gradient, as the library has them


def _check_gradient(ids: int, bags: int, rows: int, dim: int) -> None:
    """Refuse in the forward pass what its backward pass would."""
    if ids > _MOST_IDS or bags > _MOST_IDS or rows > _MOST_ROWS or dim > _MOST_COLUMNS:
        raise _capi.EbagError(_capi.EUNSUPPORTED, f"no gradient for {ids} ids in {bags} bags of {rows} rows of {dim} columns: at most 2^30 "
                                                  "ids and bags, 2^31 - 2 rows of tables, 2^22 columns")


# ------------------------------------------------------------------------------------------------
# Lookup
# ------------------------------------------------------------------------------------------------
# A call's way through Python takes as long as a small kernel: what these operators check on every call is one expression, explained
# only when it fails (as in ops.py).
def _lookup(ids, weight, scale, out, out_dtype):
    if not (isinstance(weight, torch.Tensor) and isinstance(ids, torch.Tensor) and weight.is_cuda and ids.is_cuda
            and weight.dim() == 2 and (weight.is_contiguous() or _row_major(weight)) and ids.is_contiguous()
            and (ids.dtype is torch.int64 or ids.dtype is torch.int32) and ids.get_device() == weight.get_device()):
        if not isinstance(weight, torch.Tensor) or not weight.is_cuda:
            _require_on("weight", weight)
        _check_index("ids", ids, weight.get_device())
        raise ValueError("weight must be a row-major 2-D tensor with unit column stride")
    index = weight.get_device()
    rows, dim = weight.shape
    if rows < 1 or not 1 <= dim < 2 ** 31:
        if rows >= 1 and dim >= 1:
            _check_dim(dim)
        raise ValueError(f"weight has shape {tuple(weight.shape)}: no rows or no columns")
    dtype = weight.dtype
    code = out_code = _capi.dtype_code(dtype)
    if out is None:
        if out_dtype is not None:
            dtype, out_code = out_dtype, _capi.dtype_code(out_dtype)
        out = torch.empty(*ids.shape, dim, dtype=dtype, device=weight.device)
    else:
        _check_output("out", out, (*ids.shape, dim), out_dtype or out.dtype, index)
        out_code = _capi.dtype_code(out.dtype)
    _launch(index, _capi.lib().cti_ebag_lookup, ids.data_ptr(), _capi.I64 if ids.dtype is torch.int64 else _capi.I32, ids.numel(),
            weight.data_ptr(), code, rows, weight.stride(0), dim, scale, out.data_ptr(), out_code)
    return out


def _row_major(t: torch.Tensor) -> bool:
    return t.stride(1) == 1 and t.stride(0) >= t.shape[1]


class _Lookup(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, ids, scale, padding_idx, out_dtype, sparse_grad):
        ctx.save_for_backward(ids)
        ctx.info = (weight.shape[0], weight.shape[1], weight.dtype, scale, padding_idx, sparse_grad)
        return _lookup(ids, weight, scale, None, out_dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        ids, = ctx.saved_tensors
        rows, dim, dtype, scale, padding_idx, sparse_grad = ctx.info
        got = embedding_lookup_backward(grad.contiguous(), ids, rows, scale, padding_idx, grad_dtype=dtype, compact=sparse_grad)
        return (_sparse(got, rows, dim) if sparse_grad else got), None, None, None, None, None


def _sparse(got, rows: int, dim: int) -> torch.Tensor:
    """Compact rows as a sparse tensor of torch; waits for their count."""
    numbers, sums, count = got
    n = int(count.item())
    return torch.sparse_coo_tensor(numbers[:n].unsqueeze(0), sums[:n], (rows, dim), is_coalesced=True, check_invariants=False)


def embedding_lookup(
    ids: torch.Tensor,
    weight: torch.Tensor,
    scale: float = 1.0,
    padding_idx: Optional[int] = None,
    out: Optional[torch.Tensor] = None,
    out_dtype: Optional[torch.dtype] = None,
    sparse_grad: bool = False,
) -> torch.Tensor:
    """Rows of a table, scaled: ``out[..., :] = scale * weight[clamp(ids[...], 0, rows - 1)]`` in fp32, rounded
    once to ``out_dtype`` (the table's type by default; or ``out``'s).

    ``ids`` int64 or int32 of any shape, contiguous; ``weight`` ``[rows, dim]`` fp32 / bf16 / fp16 with unit
    column stride. Ids outside the table are clamped, as everywhere in this package. Returns ``out`` of shape
    ``ids.shape + (dim,)``; ``out`` overlaps no input.

    Differentiable in ``weight`` (``out`` must then be None, and the limits are the gradient's: 2^30 ids, 2^31 - 2 rows, 2^22
    columns): the gradient is ``embedding_lookup_backward``'s,
    0 for row ``padding_idx``, which the lookup itself reads like any row. With ``sparse_grad`` it is a
    sparse tensor of the rows that occur, each once, whose making waits for their count (not within a captured graph).
    """
    scale = float(scale)
    _refuse_tangents(weight)
    if _grad_enabled() and isinstance(weight, torch.Tensor) and weight.requires_grad:
        if out is not None:
            raise ValueError("out does not combine with a gradient: detach the weight or leave out None")
        if weight.dim() == 2 and isinstance(ids, torch.Tensor):
            _check_padding(padding_idx, weight.shape[0])
            _check_gradient(ids.numel(), 0, *weight.shape)
            return _Lookup.apply(weight, ids, scale, padding_idx, out_dtype, sparse_grad)
    elif padding_idx is not None and isinstance(weight, torch.Tensor) and weight.dim() == 2:
        _check_padding(padding_idx, weight.shape[0])
    return _lookup(ids, weight, scale, out, out_dtype)


# ------------------------------------------------------------------------------------------------
# Gradients of tables
# ------------------------------------------------------------------------------------------------
@functools.lru_cache(maxsize=4096)
def _backward_workspace(nnz: int, bags: int, rows: int, dim: int, pooling: int) -> int:
    return _capi.lib().cti_ebag_backward_workspace_bytes(nnz, bags, rows, dim, pooling)


def _workspace(nnz, bags, rows, dim, pooling, device):
    """(the workspace, its address, its bytes); kept alive until the launches are enqueued."""
    size = _backward_workspace(nnz, bags, rows, dim, pooling)
    if size <= 0:
        return None, None, 0
    ws = torch.empty(size, dtype=torch.uint8, device=device)
    return ws, ws.data_ptr(), size


def _compact_output(out, nnz: int, rows: int, dim: int, dtype, device, index: int):
    """Buffers of the compact form, checked or new: (numbers, sums, count), and their capacity."""
    need = max(1, min(nnz, rows))
    if out is None:
        return (torch.empty(need, dtype=torch.int64, device=device), torch.empty(need, dim, dtype=dtype, device=device),
                torch.empty(1, dtype=torch.int64, device=device)), need
    if not isinstance(out, (tuple, list)) or len(out) != 3:
        raise ValueError("out of the compact form is (rows, grads, count)")
    numbers, sums, count = out
    _require_on("out[0] (rows)", numbers, index)
    if numbers.dim() != 1 or numbers.dtype != torch.int64 or numbers.numel() < need:
        raise ValueError(f"out[0] (rows) must be 1-D int64 with at least {need} entries")
    _check_output("out[1] (grads)", sums, (numbers.numel(), dim), dtype or sums.dtype, index)
    _check_output("out[2] (count)", count, (1,), torch.int64, index)
    return (numbers, sums, count), numbers.numel()


def embedding_lookup_backward(
    grad: torch.Tensor,
    ids: torch.Tensor,
    num_rows: int,
    scale: float = 1.0,
    padding_idx: Optional[int] = None,
    grad_dtype: Optional[torch.dtype] = None,
    compact: bool = False,
    out=None,
):
    """The gradient of ``embedding_lookup``'s table of ``num_rows`` rows: row v is ``scale`` times the sum of
    ``grad``'s rows whose id, clamped, is v; row ``padding_idx`` is 0.

    ``grad`` ``ids.shape + (dim,)`` fp32 / bf16 / fp16, contiguous. Sums in fp32, in an order that sizes and ids
    fix (the same call gives the same bits in every run), rounded once to ``grad_dtype`` (``grad``'s type by default; or ``out``'s). Returns ``[num_rows, dim]``
    (``out``), or with ``compact`` ``(rows, grads, count)``: the numbers of the rows that occur, ascending, then -1;
    their sums, where what lies behind the last row is left as it was; and how many they are, int64 ``[1]``. There
    ``out`` is a tuple of three such buffers of any capacity of at least ``min(ids, num_rows)`` (and 1) rows.
    Nothing waits for the device. ``out`` overlaps no input.
    """
    index = _require_on("grad", grad)
    _check_index("ids", ids, index)
    if grad.dim() != ids.dim() + 1 or grad.shape[:-1] != ids.shape or grad.shape[-1] < 1:
        raise ValueError(f"grad has shape {tuple(grad.shape)}, expected {tuple(ids.shape)} and columns")
    dim, n, num_rows = grad.shape[-1], ids.numel(), int(num_rows)
    _check_dim(dim)
    if num_rows < 1:
        raise ValueError(f"num_rows must be >= 1, got {num_rows}")
    padding = _check_padding(padding_idx, num_rows)
    code = _capi.dtype_code(grad.dtype)
    numbers = count = None
    capacity = 0
    if compact:
        got, capacity = _compact_output(out, n, num_rows, dim, grad_dtype or (grad.dtype if out is None else None), grad.device, index)
        numbers, out, count = got
    elif out is None:
        out = torch.empty(num_rows, dim, dtype=grad_dtype or grad.dtype, device=grad.device)
    else:
        _check_output("out", out, (num_rows, dim), grad_dtype or out.dtype, index)
    ws, ws_ptr, ws_bytes = _workspace(n, n, num_rows, dim, _capi.SUM, grad.device)
    _launch(index, _capi.lib().cti_ebag_lookup_backward, grad.data_ptr(), code, ids.data_ptr(), _capi.index_code(ids.dtype), n,
            num_rows, dim, float(scale), padding, out.data_ptr(), _capi.dtype_code(out.dtype),
            numbers.data_ptr() if compact else None, count.data_ptr() if compact else None, capacity, ws_ptr, ws_bytes)
    return (numbers, out, count) if compact else out


def fused_all_slots_embedding_backward(
    grad: torch.Tensor,
    flat_values: torch.Tensor,
    val_offsets: torch.Tensor,
    flat_row_offsets: torch.Tensor,
    batch_size: int,
    emb_dim: int,
    max_idx: int,
    pooling: str = "sum",
    padding_idx: Optional[int] = None,
    grad_dtype: Optional[torch.dtype] = None,
    compact: bool = False,
    out=None,
):
    """The gradient of ``fused_all_slots_embedding``'s table (``max_idx + 1`` rows), given ``grad`` ``[B,
    S*emb_dim]``, the gradient of its output: row v is the sum over ids that are v, clamped, of their bag's part of
    ``grad`` (under ``pooling="mean"`` divided by the bag's length); row ``padding_idx`` is 0.

    The batch's arguments as ``fused_all_slots_embedding`` takes them; the bags lie in ``flat_values`` in the order of
    slots and samples, as ``collate_flat_layout``, ``pack_slots`` and ``merge_batches`` lay them out (a batch whose
    offsets descend gives unspecified sums). The rest as in ``embedding_lookup_backward``.
    """
    index = _require_on("grad", grad)
    icode, ocode = _check_flat_layout(flat_values, val_offsets, flat_row_offsets, grad, grad.device)
    val_offsets = _same_offset_type(val_offsets, flat_row_offsets, flat_values.numel())
    batch_size, emb_dim, max_idx = int(batch_size), int(emb_dim), int(max_idx)
    slots, n = val_offsets.numel(), flat_values.numel()
    if batch_size < 0 or emb_dim < 1 or max_idx < 0:
        raise ValueError(f"batch_size {batch_size}, emb_dim {emb_dim}, max_idx {max_idx}: expected >= 0, >= 1, >= 0")
    _check_dim(emb_dim)
    if flat_row_offsets.numel() != slots * (batch_size + 1):
        raise ValueError(f"flat_row_offsets has {flat_row_offsets.numel()} entries, expected {slots} * ({batch_size} + 1)")
    if tuple(grad.shape) != (batch_size, slots * emb_dim):
        raise ValueError(f"grad has shape {tuple(grad.shape)}, expected ({batch_size}, {slots * emb_dim})")
    padding = _check_padding(padding_idx, max_idx + 1)
    code, pool = _capi.dtype_code(grad.dtype), _capi.pooling_code(pooling)
    numbers = count = None
    capacity = 0
    if compact:
        got, capacity = _compact_output(out, n, max_idx + 1, emb_dim, grad_dtype or (grad.dtype if out is None else None), grad.device,
                                        index)
        numbers, out, count = got
    elif out is None:
        out = torch.empty(max_idx + 1, emb_dim, dtype=grad_dtype or grad.dtype, device=grad.device)
    else:
        _check_output("out", out, (max_idx + 1, emb_dim), grad_dtype or out.dtype, index)
    ws, ws_ptr, ws_bytes = _workspace(n, batch_size * slots, max_idx + 1, emb_dim, pool, grad.device)
    _launch(index, _capi.lib().cti_ebag_fused_all_slots_backward, grad.data_ptr(), code, flat_values.data_ptr(), icode,
            val_offsets.data_ptr(), flat_row_offsets.data_ptr(), ocode, batch_size, slots, emb_dim, max_idx, n, pool, padding,
            out.data_ptr(), _capi.dtype_code(out.dtype), numbers.data_ptr() if compact else None,
            count.data_ptr() if compact else None, capacity, ws_ptr, ws_bytes)
    return (numbers, out, count) if compact else out


def embedding_bag_backward(
    grad: torch.Tensor,
    values: torch.Tensor,
    offsets: torch.Tensor,
    tables: Sequence[torch.Tensor],
    pooling: str = "sum",
    padding_idx: Optional[int] = None,
    grad_dtype: Optional[torch.dtype] = None,
    compact: bool = False,
    out=None,
):
    """The gradients of ``embedding_bag_pooled``'s tables, given ``grad`` ``[B, sum(D_f)]``, the gradient of its
    output. ``values``, ``offsets`` and ``tables`` as that call takes them (offsets ascend; tables are float tensors,
    of which only shape, type and identity are read; at most 64).

    Returns a list with the gradient ``[V_f, D_f]`` of each field's table, of ``grad_dtype`` (the tables' type by
    default); fields that share a table (the same memory, shape and strides) share its gradient (the same tensor). ``out``: such a
    list.
    With ``compact`` (tables of one width) ``(rows, grads, count)`` as in ``embedding_lookup_backward``, where row r
    of a table has the number (rows of the tables before it, shared ones counted once) + r. ``padding_idx`` is every
    table's.
    """
    index = _require_on("grad", grad)
    shapes, pointers, alike = _plain_tables(tables, index)
    if shapes is None:
        code, table_dev = _table_descs(tables)[2:0:-1]  # explains what is wrong with them
        if code == _capi.I8:
            raise TypeError("int8 tables have no gradient")
        raise ValueError(f"tables are on {table_dev}, grad on {grad.device}" if table_dev != grad.device else "a table has no columns")
    same = None  # the first field with the table
    if len(set(pointers)) != len(pointers):
        first = {}  # a table is its address, shape and strides
        same = [first.setdefault((pointers[f], shapes[f], t.stride()), f) for f, t in enumerate(tables)]
    return _bag_gradients(index, grad, values, offsets, shapes, alike, tables[0].dtype, same, pooling, padding_idx, grad_dtype, compact, out)


def _bag_gradients(index, grad, values, offsets, shapes, alike, dtype, same, pooling, padding_idx, grad_dtype=None, compact=False,
                   out=None, wanted=None):
    """``embedding_bag_backward`` of tables of these shapes (``alike``: all the same) and this type; ``same[f]``: the first field with
    field f's table (None: no field shares one); ``wanted[f]``: whether its table has a gradient (None: every field's; the whole
    form gives None for the others, the compact one does not count their rows)."""
    dev = grad.device
    fields = len(shapes)
    width = fields * shapes[0][1] if alike else sum(shape[1] for shape in shapes)
    _check_index("values", values, index)
    _require_on("offsets", offsets, index)
    if offsets.dtype != torch.int64:
        raise TypeError(f"offsets must be int64 (got {offsets.dtype})")
    if offsets.numel() < 1 or (offsets.numel() - 1) % fields:
        raise ValueError(f"offsets has {offsets.numel()} entries; expected F*B+1 with F={fields}")
    batch = (offsets.numel() - 1) // fields
    if grad.shape != (batch, width):
        raise ValueError(f"grad has shape {tuple(grad.shape)}, expected ({batch}, {width})")
    if width >= 2 ** 31:
        raise _capi.EbagError(_capi.EUNSUPPORTED, f"{width} columns >= 2^31")
    pool = _capi.pooling_code(pooling)
    with_grad = shapes if wanted is None else [shape for f, shape in enumerate(shapes) if wanted[f]]
    if same is None:
        same, rows = range(fields), len(with_grad) * shapes[0][0] if alike else sum(shape[0] for shape in with_grad)
    else:
        rows = sum(shapes[f][0] for f in set(same) if wanted is None or wanted[f])
    padding = _check_padding(padding_idx, shapes[0][0] if alike else min(shape[0] for shape in with_grad))
    dim = shapes[0][1] if alike else max(shape[1] for shape in with_grad)
    odt = grad_dtype or dtype
    n = values.numel()
    numbers = sums = count = grads = None
    capacity = 0
    if compact:
        got, capacity = _compact_output(out, n, rows, dim, odt, dev, index)
        numbers, sums, count = got
        pointers = [f + 1 for f in same]  # only tells the tables apart
    elif out is None:
        if alike and rows == fields * shapes[0][0]:  # tables alike and none shared: one allocation
            whole = torch.empty((rows, dim), dtype=odt, device=dev)
            grads = list(torch.unsafe_chunk(whole, fields))
            size = shapes[0][0] * dim * whole.element_size()
            pointers = range(whole.data_ptr(), whole.data_ptr() + fields * size, size)
        else:
            made = {f: torch.empty(shapes[f], dtype=odt, device=dev) if wanted is None or wanted[f] else None for f in set(same)}
            grads = [made[f] for f in same]
            pointers = [0 if g is None else g.data_ptr() for g in grads]
    else:
        grads = list(out)
        if len(grads) != fields:
            raise ValueError(f"out has {len(grads)} tensors for {fields} tables")
        for f, g in enumerate(grads):
            _check_output(f"out[{f}]", g, shapes[f], odt, index)
        pointers = [g.data_ptr() for g in grads]
        if any(pointers[f] != pointers[same[f]] for f in range(fields)) or len(set(pointers)) != len(set(same)):
            raise ValueError("out: fields of one table expect one tensor, and different tables different ones")
    # cti_ebag_table of every field: data, rows, row_stride, dim, out_col, row_scale
    descs = [0] * (6 * fields)
    descs[0::6] = pointers
    if alike:
        descs[1::6], descs[2::6], descs[3::6] = [shapes[0][0]] * fields, [dim] * fields, [dim] * fields
        descs[4::6] = range(0, width, dim)
    else:
        descs[1::6], dims = [shape[0] for shape in shapes], [shape[1] for shape in shapes]
        descs[2::6], descs[3::6] = dims, dims
        descs[4::6] = itertools.accumulate(dims[:-1], initial=0)
    packed = struct.pack("QqqiiQ" * fields, *descs)
    ws, ws_ptr, ws_bytes = _workspace(n, batch * fields, rows, dim, pool, dev)
    mask = 2 ** 64 - 1 if wanted is None else sum(1 << f for f in range(fields) if wanted[f])
    _launch(index, _capi.lib().cti_ebag_backward_fields, grad.data_ptr(), _capi.dtype_code(grad.dtype), width, values.data_ptr(),
            _capi.index_code(values.dtype), n, offsets.data_ptr(), batch, fields,
            ctypes.cast(ctypes.c_char_p(packed), ctypes.POINTER(_capi.Table)), mask, pool, padding,
            _capi.dtype_code(sums.dtype if compact else odt), sums.data_ptr() if compact else None,
            numbers.data_ptr() if compact else None, count.data_ptr() if compact else None, capacity, ws_ptr, ws_bytes)
    return (numbers, sums, count) if compact else grads


def _plain_tables(tables, index: int):
    """(shapes, addresses, whether the shapes are all the same) of float tables of one type on device `index`, row-major,
    with rows and columns; (None, None, False) if that is not what they are."""
    bad = None, None, False
    if not tables:
        return bad
    dtype = getattr(tables[0], "dtype", None)
    if dtype not in _FLOATS:
        return bad
    shapes, pointers = [], []
    for t in tables:
        if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype is dtype and t.get_device() == index
                and (t.is_contiguous() or t.dim() == 2 and _row_major(t))):
            return bad
        shapes.append(t.shape)
        pointers.append(t.data_ptr())
    alike = shapes.count(shapes[0]) == len(shapes)
    for shape in shapes[:1] if alike else shapes:
        if len(shape) != 2 or shape[0] < 1 or shape[1] < 1:
            return bad
    return shapes, pointers, alike


class _PooledTables(torch.autograd.Function):
    @staticmethod
    def forward(ctx, values, offsets, pooling, padding_idx, out_dtype, sparse_grad, known, *tables):
        out = embedding_bag_pooled(values, offsets, tables, pooling, out_dtype)
        ctx.save_for_backward(values, offsets)  # of the tables, only what the gradient needs to know: they may change until then
        ctx.info = (pooling, padding_idx, sparse_grad, *known, tables[0].dtype)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        values, offsets = ctx.saved_tensors
        pooling, padding_idx, sparse_grad, shapes, alike, same, dtype = ctx.info
        wanted = ctx.needs_input_grad[7:]
        grads = _bag_gradients(grad.get_device(), grad.contiguous(), values, offsets, shapes, alike, dtype, same, pooling, padding_idx,
                               compact=sparse_grad, wanted=None if all(wanted) else wanted)
        if sparse_grad:
            first = [f for f in range(len(shapes)) if wanted[f] and (same is None or same[f] == f)]
            made = dict(zip(first, _sparse_tables(grads, [shapes[f] for f in first])))
            grads = [made.get(f) for f in range(len(shapes))]
        elif same is not None:  # autograd adds up the fields' gradients of one table: its sum is in the first
            grads = [g if same[f] == f else None for f, g in enumerate(grads)]
        return (None, None, None, None, None, None, None, *grads)


def _sparse_tables(got, shapes):
    """Compact rows of tables of these shapes, numbered one table behind the other, as a sparse tensor of torch each; waits for
    their count."""
    numbers, sums, count = got
    numbers = numbers[:int(count.item())]
    starts = [0, *itertools.accumulate(shape[0] for shape in shapes)]
    ends = torch.searchsorted(numbers, torch.tensor(starts, device=numbers.device)).tolist()
    return [torch.sparse_coo_tensor((numbers[a:b] - start).unsqueeze(0), sums[a:b], shape, is_coalesced=True, check_invariants=False)
            for a, b, start, shape in zip(ends, ends[1:], starts, shapes)]


def embedding_bag_train(
    values: torch.Tensor,
    offsets: torch.Tensor,
    tables: Sequence[torch.Tensor],
    pooling: str = "sum",
    padding_idx: Optional[int] = None,
    out_dtype: Optional[torch.dtype] = None,
    sparse_grad: bool = False,
) -> torch.Tensor:
    """``embedding_bag_pooled`` of float tables, differentiable in them (``embedding_bag_backward``). Fields share a table where they
    are given the same tensor. Tensors that only share memory, a table and what ``detach()`` makes of it among them, are tables of
    their own, as autograd sees them. Tables that require no gradient take no memory and no sums in the backward pass. Where one
    requires it there are at most 64 fields, 2^30 ids and bags, 2^31 - 2 rows of such tables and 2^22 columns of each, and the
    offsets ascend (else the gradients are unspecified). With ``sparse_grad`` (such tables then have one width) gradients are sparse
    tensors of the rows that occur, as ``embedding_lookup``'s, and their making waits for their count.

    Row ``padding_idx`` of every table gets the gradient 0, and that is all: unlike ``nn.EmbeddingBag``'s, the forward pass reads the
    row like any other, and its ids count in a mean's length.
    """
    shapes = []  # looked up once: for 28 tables each pass over them takes as long as a launch
    for f, t in enumerate(tables):
        if not isinstance(t, torch.Tensor):
            raise TypeError("tables must be tensors: int8 pairs have no gradient")
        shape = t.shape
        if len(shape) != 2:
            raise ValueError(f"tables[{f}] must be 2-D, got shape {tuple(shape)}")
        shapes.append(shape)
    if padding_idx is not None and shapes:
        _check_padding(padding_idx, min(shape[0] for shape in shapes))
    _refuse_tangents(*tables)
    fields = len(shapes)
    alike = fields > 0 and shapes.count(shapes[0]) == fields
    same = None  # the first field with the table
    if len(set(map(id, tables))) != fields:
        first = {}
        same = [first.setdefault(id(t), f) for f, t in enumerate(tables)]
    needs = [t.requires_grad for t in tables]
    if True in needs and _grad_enabled():
        if fields > _MOST_FIELDS:
            raise _capi.EbagError(_capi.EUNSUPPORTED, f"no gradient for {fields} fields: at most {_MOST_FIELDS} in a call")
        trained = [shape for f, shape in enumerate(shapes) if needs[f] and (same is None or same[f] == f)]
        dim = trained[0][1] if alike else max(shape[1] for shape in trained)
        if sparse_grad and not alike and min(shape[1] for shape in trained) != dim:
            raise _capi.EbagError(_capi.EUNSUPPORTED, "sparse gradients need tables of one width")
        if isinstance(values, torch.Tensor) and isinstance(offsets, torch.Tensor):
            rows = len(trained) * trained[0][0] if alike else sum(shape[0] for shape in trained)
            _check_gradient(values.numel(), offsets.numel() - 1, rows, dim)
    return _PooledTables.apply(values, offsets, pooling, padding_idx, out_dtype, sparse_grad, (shapes, alike, same), *tables)


class _PooledShared(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, flat_values, val_offsets, flat_row_offsets, batch_size, padding_idx, sparse_grad, tile_order):
        ctx.save_for_backward(flat_values, val_offsets, flat_row_offsets)
        rows, dim = weight.shape
        ctx.info = (rows, dim, batch_size, padding_idx, sparse_grad)
        out = torch.empty(batch_size, val_offsets.numel() * dim, dtype=weight.dtype, device=weight.device)
        return fused_all_slots_embedding(flat_values, val_offsets, flat_row_offsets, weight, out, batch_size, dim, rows - 1,
                                         tile_order=tile_order)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        rows, dim, batch_size, padding_idx, sparse_grad = ctx.info
        got = fused_all_slots_embedding_backward(grad.contiguous(), *ctx.saved_tensors, batch_size, dim, rows - 1,
                                                 padding_idx=padding_idx, compact=sparse_grad)
        return (_sparse(got, rows, dim) if sparse_grad else got), None, None, None, None, None, None, None


def fused_embedding_train(
    flat_values: torch.Tensor,
    val_offsets: torch.Tensor,
    flat_row_offsets: torch.Tensor,
    weight: torch.Tensor,
    padding_idx: Optional[int] = None,
    sparse_grad: bool = False,
    tile_order: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """The fused step of a flat-layout batch, ``[B, S*D]`` as ``fused_all_slots_embedding`` pools it, differentiable in
    the table (``fused_all_slots_embedding_backward``; ``padding_idx``, ``sparse_grad`` and the limits, of bags too, as in
    ``embedding_lookup``). ``tile_order``: the batch's dispatch order for the forward pass, as ``fused_all_slots_embedding`` takes
    it.

    The bags have to lie in ``flat_values`` in the order of slots and samples, none over another, as ``collate_flat_layout``,
    ``pack_slots`` and ``merge_batches`` lay them out. The forward pass pools any other batch too (slots in another order, bags
    that share ids), but its gradient is unspecified, without an error."""
    for name, t in (("flat_values", flat_values), ("val_offsets", val_offsets), ("flat_row_offsets", flat_row_offsets), ("weight", weight)):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    if weight.dim() != 2:
        raise ValueError(f"weight must be 2-D [V, D], got shape {tuple(weight.shape)}")
    slots = val_offsets.numel()
    if slots < 1 or flat_row_offsets.numel() < slots or flat_row_offsets.numel() % slots:
        raise ValueError(f"flat_row_offsets has {flat_row_offsets.numel()} entries for {slots} slots")
    _check_padding(padding_idx, weight.shape[0])
    _refuse_tangents(weight)
    batch_size = flat_row_offsets.numel() // slots - 1
    if _grad_enabled() and weight.requires_grad:
        _check_gradient(flat_values.numel(), slots * batch_size, *weight.shape)
    return _PooledShared.apply(weight, flat_values, val_offsets, flat_row_offsets, batch_size, padding_idx, sparse_grad, tile_order)


# ------------------------------------------------------------------------------------------------
# Dropout
# ------------------------------------------------------------------------------------------------
def _check_seed(p, seed, offset, index: int):
    """(p, seed, offset, the state's address) as the library takes them."""
    p, offset = float(p), int(offset)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"p must be in [0, 1], got {p}")
    if not 0 <= offset < 2 ** 64:
        raise ValueError(f"offset must be in [0, 2^64), got {offset}")
    if isinstance(seed, torch.Tensor):
        _require_on("seed", seed, index)
        if seed.dtype != torch.int64 or seed.numel() != 2:
            raise ValueError(f"seed must be an int or an int64 tensor of 2 (seed, offset), got {tuple(seed.shape)} {seed.dtype}")
        return p, 0, offset, seed.data_ptr()
    seed = int(seed)
    if not 0 <= seed < 2 ** 64:
        raise ValueError(f"seed must be in [0, 2^64), got {seed}")
    return p, seed, offset, None


def _rows_of(name: str, x) -> tuple:
    """(device index, type code, rows, columns) of a contiguous tensor of rows."""
    if isinstance(x, torch.Tensor) and x.is_cuda and x.is_contiguous():
        shape = x.shape
        if len(shape) == 2 and shape[1] >= 1:
            return x.get_device(), _capi.dtype_code(x.dtype), shape[0], shape[1]
    index = _require_on(name, x)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"{name} must have columns, got shape {tuple(x.shape)}")
    return index, _capi.dtype_code(x.dtype), x.numel() // x.shape[-1], x.shape[-1]


def _check_like(name: str, t, x, index: int) -> int:
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.get_device() == index and t.is_contiguous() and t.dtype is x.dtype
            and t.shape == x.shape):
        _require_on(name, t, index)
        raise ValueError(f"{name} must be {tuple(x.shape)} {x.dtype}, got {tuple(t.shape)} {t.dtype}")
    return t.data_ptr()


def _dropout(x, p, seed, offset, residual, out):
    index, code, rows, cols = _rows_of("x", x)
    p, seed, offset, state = _check_seed(p, seed, offset, index)
    res = None if residual is None else _check_like("residual", residual, x, index)
    if out is None:
        out = torch.empty_like(x)
    else:
        _check_like("out", out, x, index)
    _launch(index, _capi.lib().cti_ebag_dropout, x.data_ptr(), res, out.data_ptr(), rows, cols, code, p, seed, offset, state)
    return out


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, offset):
        ctx.state = None if isinstance(seed, torch.Tensor) else (p, seed, offset)
        if ctx.state is None:
            ctx.save_for_backward(seed)
            ctx.rest = (p, offset)
        return _dropout(x, p, seed, offset, residual, None)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        p, seed, offset = ctx.state or (ctx.rest[0], ctx.saved_tensors[0], ctx.rest[1])
        dx = _dropout(grad.contiguous(), p, seed, offset, None, None) if ctx.needs_input_grad[0] else None
        return dx, (grad if ctx.needs_input_grad[1] else None), None, None, None


def dropout(
    x: torch.Tensor,
    p: float,
    seed,
    offset: int = 0,
    residual: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """``residual + (kept ? x / (1 - p) : 0)`` in fp32, rounded once to x's type; without a residual the dropout alone.

    ``x`` (fp32 / bf16 / fp16, contiguous, any shape; its last dimension are the columns, the others the rows) is kept
    where 16 bits of Philox4x32-10 with key ``seed`` and counter (row, column / 8, ``offset``) reach
    ``t = round(65536 p)``; p counts as t / 65536, for the factor too. Dropped elements give 0 whatever x is (NaN too).
    ``seed`` is a number below 2^64, or an int64 tensor (seed, offset) on the device. ``out`` may be x or residual.
    Differentiable in ``x`` and ``residual`` (``out`` must then be None); the mask is made again for it, not stored.
    """
    _refuse_tangents(x, residual)
    if _grad_enabled() and _any_requires_grad(x, residual):
        if out is not None:
            raise ValueError("out does not combine with a gradient: detach the inputs or leave out None")
        return _Dropout.apply(x, residual, p, seed, offset)
    return _dropout(x, p, seed, offset, residual, out)


def dropout_backward(grad: torch.Tensor, p: float, seed, offset: int = 0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The gradient of ``dropout``'s ``x`` (that of its residual is ``grad`` itself); ``out`` may be ``grad``."""
    return _dropout(grad, p, seed, offset, None, out)


# ------------------------------------------------------------------------------------------------
# Layer norm
# ------------------------------------------------------------------------------------------------
def _check_param(name: str, t, cols: int, index: int) -> int:
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.get_device() == index and t.is_contiguous() and t.numel() == cols):
        _require_on(name, t, index)
        raise ValueError(f"{name} has {t.numel()} elements, expected {cols}")
    return t.data_ptr()


def _check_stats(name: str, t, rows: int, index: int) -> int:
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.get_device() == index and t.is_contiguous() and t.dtype is torch.float32
            and t.numel() == rows):
        _require_on(name, t, index)
        raise ValueError(f"{name} must be a contiguous float32 tensor of {rows} elements")
    return t.data_ptr()


def _threshold(p: float) -> int:
    return int(p * 65536.0 + 0.5)


def _norm(x, weight, bias, eps, residual, p, seed, offset):
    index, code, rows, cols = _rows_of("x", x)
    gamma, beta = _check_param("weight", weight, cols, index), _check_param("bias", bias, cols, index)
    if weight.dtype is not bias.dtype:
        raise TypeError(f"weight and bias dtypes differ ({weight.dtype} vs {bias.dtype})")
    param = _capi.dtype_code(weight.dtype)
    p, seed, offset, state = _check_seed(p, seed, offset, index)
    res = None if residual is None else _check_like("residual", residual, x, index)
    y = torch.empty_like(x)
    h = torch.empty_like(x) if residual is not None or _threshold(p) else None
    mean = torch.empty(*x.shape[:-1], dtype=torch.float32, device=x.device) if x.dim() > 1 else torch.empty((), dtype=torch.float32, device=x.device)
    rstd = torch.empty_like(mean)
    _launch(index, _capi.lib().cti_ebag_dropout_layernorm, x.data_ptr(), res, None if h is None else h.data_ptr(), y.data_ptr(), rows,
            cols, code, gamma, beta, param, eps, p, seed, offset, state, mean.data_ptr(), rstd.data_ptr())
    return y, h, mean, rstd


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps, p, seed, offset):
        y, h, mean, rstd = _norm(x, weight, bias, eps, residual, p, seed, offset)
        on_device = isinstance(seed, torch.Tensor)
        ctx.save_for_backward(x if h is None else h, mean, rstd, weight, *((seed,) if on_device else ()))
        ctx.info = (p, None if on_device else seed, offset, residual is not None, h is not None)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(mean, rstd)
        ctx.bias_shape = None if bias.shape == weight.shape else bias.shape  # as many elements, not always the same dimensions
        return (y, mean, rstd) if h is None else (y, mean, rstd, h)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad, _mean, _rstd, grad_h=None):
        h, mean, rstd, weight, *rest = ctx.saved_tensors
        p, seed, offset, residual, _ = ctx.info
        grad = torch.zeros_like(h) if grad is None else grad.contiguous()
        dx, dweight, dbias, dres = dropout_add_layer_norm_backward(
            grad, h, mean, rstd, weight, None if grad_h is None else grad_h.contiguous(), residual, p, rest[0] if rest else seed, offset)
        return dx, dres, dweight, dbias if ctx.bias_shape is None else dbias.view(ctx.bias_shape), None, None, None, None


def dropout_add_layer_norm(
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: torch.Tensor,
    eps: float = 1e-5,
    residual: Optional[torch.Tensor] = None,
    p: float = 0.0,
    seed=0,
    offset: int = 0,
):
    """``h = residual + dropout(x, p, seed, offset)`` (rounded to x's type) and its LayerNorm in one pass over memory.

    ``x`` (and ``residual``) ``[..., cols]`` fp32 / bf16 / fp16, contiguous, ``weight`` and ``bias`` ``[cols]`` of one of
    these types. Returns ``(y, h, mean, rstd)``: ``y = (h - mean) * rstd * weight + bias`` of h as it is stored, rounded
    once; ``mean`` and ``rstd`` fp32, one a row. Without dropout and residual h is x itself. ``p``, ``seed`` and
    ``offset`` as in ``dropout``. Differentiable in x, residual, weight and bias, through y and h.
    """
    eps = float(eps)
    _refuse_tangents(x, residual, weight, bias)
    if _grad_enabled() and _any_requires_grad(x, residual, weight, bias):
        y, mean, rstd, *h = _Norm.apply(x, residual, weight, bias, eps, p, seed, offset)
        return y, (h[0] if h else x), mean, rstd
    y, h, mean, rstd = _norm(x, weight, bias, eps, residual, p, seed, offset)
    return y, (x if h is None else h), mean, rstd


@functools.lru_cache(maxsize=4096)
def _norm_workspace(rows: int, cols: int) -> int:
    return _capi.lib().cti_ebag_dropout_layernorm_backward_workspace_bytes(rows, cols)


def dropout_add_layer_norm_backward(
    grad: torch.Tensor,
    h: torch.Tensor,
    mean: torch.Tensor,
    rstd: torch.Tensor,
    weight: torch.Tensor,
    grad_h: Optional[torch.Tensor] = None,
    residual: bool = False,
    p: float = 0.0,
    seed=0,
    offset: int = 0,
):
    """The gradients of ``dropout_add_layer_norm``: ``grad`` is that of y, ``grad_h`` what arrives at h itself (the
    residual stream's, or None), ``h``, ``mean`` and ``rstd`` are what it returned. Returns ``(dx, dweight, dbias,
    dresidual)``; ``dresidual`` is None unless ``residual`` is set, and dx itself without dropout. dweight and dbias
    are summed in fp32 over the rows, in a fixed order, and rounded once to the weight's type.
    """
    index, code, rows, cols = _rows_of("h", h)
    g = _check_like("grad", grad, h, index)
    gh = None if grad_h is None else _check_like("grad_h", grad_h, h, index)
    stats = _check_stats("mean", mean, rows, index), _check_stats("rstd", rstd, rows, index)
    gamma = _check_param("weight", weight, cols, index)
    p, seed, offset, state = _check_seed(p, seed, offset, index)
    param = _capi.dtype_code(weight.dtype)
    dx = torch.empty_like(h)
    dres = None
    if residual:
        dres = torch.empty_like(h) if _threshold(p) else dx
    dweight, dbias = torch.empty_like(weight), torch.empty_like(weight)
    size = _norm_workspace(rows, cols)
    ws = torch.empty(size, dtype=torch.uint8, device=h.device) if size > 0 else None
    _launch(index, _capi.lib().cti_ebag_dropout_layernorm_backward, g, h.data_ptr(), gh, *stats,
            rows, cols, code, gamma, param, p, seed, offset, state, dx.data_ptr(),
            dres.data_ptr() if dres is not None and dres is not dx else None, dweight.data_ptr(), dbias.data_ptr(),
            None if ws is None else ws.data_ptr(), size)
    return dx, dweight, dbias, dres
