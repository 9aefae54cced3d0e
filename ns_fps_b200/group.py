"""Grouping after sampling on CUDA tensors: the PointNet++ operators that
follow farthest point sampling.

* ``ball_query(points, centers, radius, nsample)``: for each centre, the
  first ``nsample`` point indices (ascending) within ``radius``; the unfilled
  slots repeat the first hit (index 0 when there is none), and ``hits`` holds
  how many were found (at most ``nsample``).
* ``gather_points(points, idx)``: the coordinates of the indexed points.
* ``group_points(points, centers, idx)``: those of ``idx`` (M, nsample)
  minus their centre, shape (M, nsample, 3).
* ``gather_rows(table, idx, scale)``: the feature rows that indices name,
  with their gradient.

The first three take coordinates.  Each takes one cloud (N, 3) or a batch (B, N, 3) with matching (B, M, ...)
centres / indices, runs on PyTorch's current stream through the C ABI
(``nsfps_ball_query_device`` and friends) and returns CUDA tensors.  The
distance test is the sampler's: d2 = (dx*dx + dy*dy) + dz*dz, fp32 rounded
per operation without multiply-add contraction, hit iff d2 < radius * radius.
"""
from __future__ import annotations

import ctypes

from . import capi

__all__ = ["ball_query", "gather_points", "group_points", "gather_rows"]


def _cloud_batch(t, name):
    import torch
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor")
    if t.dtype != torch.float32:
        raise TypeError(f"{name} must be float32")
    single = t.dim() == 2
    if single:
        t = t.unsqueeze(0)
    if t.dim() != 3 or t.shape[2] != 3:
        raise ValueError(f"{name}: expected shape (N, 3) or (B, N, 3)")
    return t.contiguous(), single


def _offsets(B, n):
    return [i * n for i in range(B + 1)]


def ball_query(points, centers, radius: float, nsample: int):
    """Returns (idx int64 (M, nsample) or (B, M, nsample), hits int32 (M,) or
    (B, M))."""
    import torch
    pts, single = _cloud_batch(points, "points")
    ctr, single_c = _cloud_batch(centers, "centers")
    if single != single_c or pts.shape[0] != ctr.shape[0]:
        raise ValueError("points and centers must have the same batch layout")
    if pts.device != ctr.device:
        raise ValueError("points and centers must be on the same device")
    B, N, M = int(pts.shape[0]), int(pts.shape[1]), int(ctr.shape[1])
    S = int(nsample)
    idx = torch.empty((B, M, S), dtype=torch.int64, device=pts.device)
    hits = torch.empty((B, M), dtype=torch.int32, device=pts.device)
    with torch.cuda.device(pts.device):
        stream = torch.cuda.current_stream(pts.device)
        capi.ball_query_device(pts.data_ptr(), _offsets(B, N), ctr.data_ptr(), _offsets(B, M),
                               float(radius), S, idx.data_ptr(), hits.data_ptr(),
                               stream.cuda_stream)
    return (idx[0], hits[0]) if single else (idx, hits)


def gather_points(points, idx):
    """Coordinates of the points ``idx`` ((M,) or (B, M) int64) selects:
    (M, 3) or (B, M, 3)."""
    import torch
    pts, single = _cloud_batch(points, "points")
    if idx.dtype != torch.int64 or not idx.is_cuda:
        raise TypeError("idx must be an int64 CUDA tensor")
    ix = idx.unsqueeze(0) if single else idx
    if ix.dim() != 2 or ix.shape[0] != pts.shape[0]:
        raise ValueError("idx must have shape (M,) for (N, 3) points or (B, M) for (B, N, 3)")
    ix = ix.contiguous()
    B, N, M = int(pts.shape[0]), int(pts.shape[1]), int(ix.shape[1])
    out = torch.empty((B, M, 3), dtype=torch.float32, device=pts.device)
    with torch.cuda.device(pts.device):
        stream = torch.cuda.current_stream(pts.device)
        capi.gather_points_device(pts.data_ptr(), _offsets(B, N), ix.data_ptr(), _offsets(B, M),
                                  out.data_ptr(), stream.cuda_stream)
    return out[0] if single else out


def group_points(points, centers, idx):
    """``points[idx] - centers`` per group: (M, nsample, 3) or
    (B, M, nsample, 3), idx as returned by ``ball_query``."""
    import torch
    pts, single = _cloud_batch(points, "points")
    ctr, single_c = _cloud_batch(centers, "centers")
    if single != single_c or pts.shape[0] != ctr.shape[0]:
        raise ValueError("points and centers must have the same batch layout")
    if idx.dtype != torch.int64 or not idx.is_cuda:
        raise TypeError("idx must be an int64 CUDA tensor")
    ix = idx.unsqueeze(0) if single else idx
    if ix.dim() != 3 or ix.shape[0] != pts.shape[0] or ix.shape[1] != ctr.shape[1]:
        raise ValueError("idx must have shape (M, nsample) or (B, M, nsample)")
    ix = ix.contiguous()
    B, N, M, S = int(pts.shape[0]), int(pts.shape[1]), int(ctr.shape[1]), int(ix.shape[2])
    out = torch.empty((B, M, S, 3), dtype=torch.float32, device=pts.device)
    with torch.cuda.device(pts.device):
        stream = torch.cuda.current_stream(pts.device)
        capi.group_points_device(pts.data_ptr(), _offsets(B, N), ctr.data_ptr(), _offsets(B, M),
                                 S, ix.data_ptr(), out.data_ptr(), stream.cuda_stream)
    return out[0] if single else out


_FLOATS = (capi.F32, capi.F16, capi.BF16)
_codes = {}


def _dtype_code(t, name, allowed):
    """The C code of t's type."""
    if not _codes:
        import torch
        _codes.update({torch.float32: capi.F32, torch.float16: capi.F16,
                       torch.bfloat16: capi.BF16})
    code = _codes.get(t.dtype)
    if code not in allowed:
        names = {capi.F32: "float32", capi.F16: "float16", capi.BF16: "bfloat16"}
        raise TypeError(f"{name} must be " + " or ".join(names[a] for a in allowed))
    return code


def _enter(index):
    """Makes device `index` current; what it was, or None.  (Small calls cost
    their launches and little else, so the common case is one comparison.)"""
    import torch
    before = torch._C._cuda_getDevice()
    if before == index:
        return None
    torch.cuda.set_device(index)
    return before


def _leave(before):
    if before is not None:
        import torch
        torch.cuda.set_device(before)


def _no_tangents(*tensors):
    """Refuses forward-mode differentiation: a kernel's result has no tangent,
    which would read as a derivative of zero.  (A dual tensor need not require
    a gradient, so the autograd node would not see it.)"""
    import torch
    forward_ad = torch.autograd.forward_ad
    if forward_ad._current_level >= 0 and any(
            forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError("no forward-mode derivative: only gradients (backward)")


def _number(scale):
    """A scale as the plain number that it is now.  (A tensor would be another
    number at the next call, and still the same key of a plan.)"""
    if type(scale) is float:
        return scale
    import torch
    if isinstance(scale, torch.Tensor):
        _no_tangents(scale)
        if scale.requires_grad and torch.is_grad_enabled():
            raise TypeError("scale takes no gradient: multiply by it outside, or pass a number")
    return float(scale)


class _Plans(dict):
    """What a call's shapes, strides and types settle once: its checks, its
    descriptor, its scratch.  Bounded; a plan holds no tensor."""

    def keep(self, key, plan):
        if len(self) >= 512:
            self.clear()
        self[key] = plan
        return plan


_rows_plans, _rows_grad_plans = _Plans(), _Plans()


def _rows_plan(table, idx, scale):
    """Checks a lookup: (descriptor, its address, shape of the result, whether
    the table has to be copied)."""
    import torch
    if not isinstance(table, torch.Tensor) or not table.is_cuda:
        raise TypeError("table must be a CUDA tensor")
    if not isinstance(idx, torch.Tensor) or not idx.is_cuda or idx.dtype != torch.int64:
        raise TypeError("idx must be an int64 CUDA tensor")
    code = _dtype_code(table, "table", _FLOATS)
    if table.dim() not in (2, 3):
        raise ValueError("table: expected shape (N, C) or (B, N, C)")
    if table.dim() == 3 and (idx.dim() < 1 or idx.shape[0] != table.shape[0]):
        raise ValueError("idx must have shape (B, ...) for a (B, N, C) table")
    if table.device != idx.device:
        raise ValueError("table and idx must be on the same device")
    shape = table.shape
    B, N, C = (1, *shape) if len(shape) == 2 else shape
    copy = (C > 1 and table.stride(-1) != 1) or C == 0
    strides = (N * C, C, 1) if copy else (0, *table.stride())[-3:]
    desc = capi.RowsDesc(B, N, C, idx.numel() // B if B else 0,
                         strides[0] if len(shape) == 3 else 0, strides[1], scale, code)
    return desc, ctypes.addressof(desc), (*idx.shape, C), copy


def _gather_rows_forward(table, idx, scale, plan):
    import torch
    if plan[3]:
        table = table.contiguous()
    idx = idx.contiguous()
    out = table.new_empty(plan[2])
    device = table.get_device()
    before = _enter(device)
    try:
        capi.call("nsfps_gather_rows_device", plan[1], table.data_ptr(), idx.data_ptr(),
                  out.data_ptr(), torch._C._cuda_getCurrentRawStream(device))
    finally:
        _leave(before)
    return out


def _gather_rows_backward(dout, idx, shape, scale):
    import torch
    dout, idx = dout.contiguous(), idx.contiguous()
    grad = dout.new_empty(shape)
    key = (shape, idx.shape, scale, dout.dtype)
    plan = _rows_grad_plans.get(key)
    if plan is None:
        B, N, C = (1, *shape) if len(shape) == 2 else shape
        desc = capi.RowsDesc(B, N, C, idx.numel() // B if B else 0, 0, 0, scale,
                             _dtype_code(dout, "grad", _FLOATS))
        plan = _rows_grad_plans.keep(key, (desc, ctypes.addressof(desc),
                                           capi.gather_rows_grad_workspace(desc)))
    device = dout.get_device()
    before = _enter(device)
    try:
        work = dout.new_empty(plan[2], dtype=torch.uint8)
        capi.call("nsfps_gather_rows_grad_device", plan[1], dout.data_ptr(), idx.data_ptr(),
                  grad.data_ptr(), work.data_ptr(), plan[2],
                  torch._C._cuda_getCurrentRawStream(device))
    finally:
        _leave(before)
    return grad


_gather_rows_function = None


def _gather_rows_autograd():
    """The autograd node, made at its first use (the module itself does not
    need PyTorch)."""
    global _gather_rows_function
    if _gather_rows_function is None:
        import torch
        from torch.autograd.function import once_differentiable

        class GatherRows(torch.autograd.Function):
            @staticmethod
            def forward(ctx, table, idx, scale, plan):
                ctx.save_for_backward(idx)
                ctx.shape, ctx.scale = table.shape, scale
                return _gather_rows_forward(table, idx, scale, plan)

            @staticmethod
            @once_differentiable
            def backward(ctx, dout):
                _no_tangents(dout)
                idx, = ctx.saved_tensors
                return _gather_rows_backward(dout, idx, ctx.shape, ctx.scale), None, None, None

        _gather_rows_function = GatherRows
    return _gather_rows_function


def gather_rows(table, idx, scale: float = 1.0):
    """``scale * table[idx]``: the feature rows that ``idx`` names, with a
    gradient for ``table``.

    table  (N, C), or (B, N, C) for B clouds: float32, float16 or bfloat16
    idx    int64: any shape for (N, C); (B, ...) for (B, N, C)
    scale  a number (what a tensor holds is read, which waits for a CUDA tensor,
           and has no gradient)

    Returns idx.shape + (C,) in the table's type (the product in float32,
    rounded once).  A negative index stands for no row: zeros, and no gradient.
    An index of N or more is never read: its row is NaN, and its gradient goes
    nowhere.  The gradient adds a row's entries in float32 in index order, so
    it is the same every time.  Forward-mode derivatives are refused.  Runs on
    PyTorch's current stream without waiting for it.
    """
    import torch
    scale = _number(scale)
    try:
        key = (table.shape, table.stride(), table.dtype, table.device, idx.shape, idx.dtype,
               idx.device, scale)
        plan = _rows_plans.get(key)
    except AttributeError:  # not tensors
        key = plan = None
    if plan is None:
        plan = _rows_plans.keep(key, _rows_plan(table, idx, scale))
    _no_tangents(table)
    if table.requires_grad and torch.is_grad_enabled():
        return _gather_rows_autograd().apply(table, idx, scale, plan)
    return _gather_rows_forward(table, idx, scale, plan)
