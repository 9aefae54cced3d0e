"""Attention of sampled centres over nearby blocks of their cloud.

* ``select_blocks(points, centers, block, top)``: for each centre, the ``top``
  blocks of ``block`` consecutive points whose bounding boxes are nearest.
* ``block_attention(q, k, v, blocks, block)``: every query attends to the keys
  of the blocks listed for it, with gradients for q, k and v.

Both take one cloud or a batch of padded clouds (``lengths``), run on
PyTorch's current stream through the C ABI (``nsfps_select_blocks_device``,
``nsfps_block_attention_device``, ``nsfps_block_attention_grad_device``)
without waiting for it, and return CUDA tensors.  Blocks are runs of
consecutive points: order a cloud along a space-filling curve (or keep a
scan's own order) so that a block is a small region.

With the sampler and the grouping operators:

    s = torch_fps.fps(pts, 4096)                              # samples
    q = to_q(group.gather_rows(feats, s)).view(-1, H, D)      # their features
    blocks, d2 = attention.select_blocks(pts, pts[s], 64, 16)
    out = attention.block_attention(q, k, v, blocks, 64)      # k, v: (N, H, D)
"""
from __future__ import annotations

import ctypes
import math

from . import capi
from .group import _cloud_batch, _dtype_code, _enter, _leave, _no_tangents, _number, _Plans

__all__ = ["select_blocks", "block_attention"]

_BLOCKS = (16, 32, 64, 128)
_MAX_TOP = 64


def _check_block(block, top):
    if block not in _BLOCKS:
        raise ValueError("block must be 16, 32, 64 or 128")
    if not 1 <= top <= _MAX_TOP:
        raise ValueError(f"top must be in 1..{_MAX_TOP}")


def _check_lengths(lengths, B, device):
    import torch
    if lengths is None:
        return
    if not isinstance(lengths, torch.Tensor) or not lengths.is_cuda or lengths.dtype != torch.int32:
        raise TypeError("lengths must be an int32 CUDA tensor")
    if lengths.numel() != B or lengths.dim() > 1:
        raise ValueError("lengths must hold one length per cloud")
    if lengths.device != device:
        raise ValueError("lengths must be on the clouds' device")


def _look(t):
    """What a call's checks read of a tensor (None: None)."""
    return None if t is None else (t.shape, t.stride(), t.dtype, t.device)


_select_plans, _attention_plans = _Plans(), _Plans()


def _select_plan(points, centers, block, top, lengths):
    pts, single = _cloud_batch(points, "points")
    ctr, single_c = _cloud_batch(centers, "centers")
    if single != single_c or pts.shape[0] != ctr.shape[0]:
        raise ValueError("points and centers must have the same batch layout")
    if pts.device != ctr.device:
        raise ValueError("points and centers must be on the same device")
    _check_block(block, top)
    B, N, M = int(pts.shape[0]), int(pts.shape[1]), int(ctr.shape[1])
    _check_lengths(lengths, B, pts.device)
    desc = capi.SelectDesc(B, N, M, block, top)
    return (desc, ctypes.addressof(desc), capi.select_blocks_workspace(desc),
            (M, top) if single else (B, M, top))


def select_blocks(points, centers, block: int, top: int, lengths=None):
    """The ``top`` blocks nearest to each centre.

    points   float32 (N, 3), or (B, N, 3) for B clouds
    centers  float32 (M, 3) or (B, M, 3)
    block    points per block: 16, 32, 64 or 128
    top      1 to 64
    lengths  None, or int32 (B,): the points of each padded cloud

    Returns (blocks int64 (M, top) or (B, M, top), d2 float32 of that shape):
    block indices by ascending squared distance from the centre to the block's
    bounding box, the lower index first among equals, -1 (d2 = inf) behind the
    last block.  d2 is the sampler's arithmetic, (dx*dx + dy*dy) + dz*dz in
    float32 without contraction, so the choice is exact.  To cut the list at a
    radius: ``blocks.masked_fill(d2 > radius * radius, -1)``.  Points and centres
    are data here, as for ``ball_query``: d2 carries no derivative.
    """
    import torch
    block, top = int(block), int(top)
    try:
        key = (_look(points), _look(centers), _look(lengths), block, top)
        plan = _select_plans.get(key)
    except AttributeError:  # not tensors
        key = plan = None
    if plan is None:
        plan = _select_plans.keep(key, _select_plan(points, centers, block, top, lengths))
    points, centers = points.contiguous(), centers.contiguous()
    lengths = None if lengths is None else lengths.contiguous()
    blocks = points.new_empty(plan[3], dtype=torch.int64)
    d2 = points.new_empty(plan[3])
    device = points.get_device()
    before = _enter(device)
    try:
        work = points.new_empty(plan[2], dtype=torch.uint8)
        capi.call("nsfps_select_blocks_device", plan[1], points.data_ptr(),
                  0 if lengths is None else lengths.data_ptr(), centers.data_ptr(),
                  blocks.data_ptr(), d2.data_ptr(), work.data_ptr(), plan[2],
                  torch._C._cuda_getCurrentRawStream(device))
    finally:
        _leave(before)
    return blocks, d2


def _strides(t):
    """Strides of batch, row and head; an axis of one entry is never stepped."""
    return [s if n > 1 else 0 for s, n in zip(t.stride()[:3], t.shape[:3])]


def _needs_copy(t):
    return t.stride(-1) != 1 or any(s % 8 for s in _strides(t))


def _rows16(t, copy):
    """t with contiguous heads and 16-byte aligned rows: t itself when it is."""
    if copy:
        t = t.contiguous()
    return t.clone(memory_format=_contiguous()) if t.data_ptr() % 16 else t


def _contiguous():
    import torch
    return torch.contiguous_format


def _attention_plan(q, k, v, blocks, block, lengths, scale):
    """Checks a call: (q, k, v to be copied, the arguments of _desc)."""
    import torch
    single = isinstance(q, torch.Tensor) and q.dim() == 3
    for name, t in (("q", q), ("k", k), ("v", v)):
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise TypeError(f"{name} must be a CUDA tensor")
        code = _dtype_code(t, name, (capi.F16, capi.BF16))
        if t.dim() != (3 if single else 4):
            raise ValueError("q: expected shape (M, H, D) or (B, M, H, D), k and v alike")
        if t.dtype != q.dtype:
            raise TypeError("q, k and v must have the same type")
        if t.device != q.device:
            raise ValueError("q, k and v must be on the same device")
    if not isinstance(blocks, torch.Tensor) or not blocks.is_cuda or blocks.dtype != torch.int64:
        raise TypeError("blocks must be an int64 CUDA tensor")
    if blocks.device != q.device:
        raise ValueError("blocks must be on q's device")
    if single:
        q, k, v, blocks = q.unsqueeze(0), k.unsqueeze(0), v.unsqueeze(0), blocks.unsqueeze(0)
    if k.shape != v.shape:
        raise ValueError("k and v must have the same shape")
    B, M, H, D = q.shape
    if k.shape[0] != B or k.shape[3] != D:
        raise ValueError("q and k must have the same batch and head size")
    G = k.shape[2]
    if not 1 <= H <= 256 or G < 1 or H % G:
        raise ValueError("q's heads must be a multiple of k's, at most 256")
    if D % 8 or not 8 <= D <= 128:
        raise ValueError("the head size must be a multiple of 8 in 8..128")
    if blocks.dim() != 3 or blocks.shape[:2] != (B, M):
        raise ValueError("blocks must have shape (M, top) or (B, M, top)")
    _check_block(block, blocks.shape[2])
    _check_lengths(lengths, B, q.device)
    copies = tuple(_needs_copy(t) for t in (q, k, v))
    # (a copy of a view whose rows begin off a 16-byte boundary is dense, too:
    # such a view is copied in the call, and its strides are these)
    dense = [(n * h * D, h * D, D) for n, h in ((M, H), (k.shape[1], G), (k.shape[1], G))]
    strides = tuple(_strides(t) for t in (q, k, v))
    head = (B, M, k.shape[1], H, G, D, block, blocks.shape[2], code)
    return copies, (head, strides, dense, 1.0 / math.sqrt(D) if scale is None else scale)


def _desc(plan, moved, backward):
    """The descriptor of a call whose q, k, v lie densely where moved says so:
    (descriptor, its address, its scratch bytes)."""
    key = (moved, backward)
    got = plan[2].get(key)
    if got is None:
        head, strides, dense, scale = plan[1]
        three = ctypes.c_int64 * 3
        lie = [three(*(d if m else s)) for m, s, d in zip(moved, strides, dense)]
        desc = capi.AttentionDesc(*head, *lie, scale, 0)
        got = plan[2][key] = (desc, ctypes.addressof(desc),
                              capi.block_attention_workspace(desc, backward))
    return got


def _forward(q, k, v, blocks, lengths, plan, train):
    """out, and what the gradient needs besides: what the rounding of out left,
    and behind it the logs of the softmax sums, as bytes."""
    import torch
    copies = plan[0]
    qp, kp, vp = q.data_ptr(), k.data_ptr(), v.data_ptr()
    if (qp | kp | vp) & 15 or copies != (False, False, False):
        copies = tuple(c or t.data_ptr() % 16 != 0 for c, t in zip(copies, (q, k, v)))
        q, k, v = (_rows16(t, c) for t, c in zip((q, k, v), copies))
        qp, kp, vp = q.data_ptr(), k.data_ptr(), v.data_ptr()
    blocks = blocks.contiguous()
    lengths = None if lengths is None else lengths.contiguous()
    out = q.new_empty(q.shape)
    keep, rest, lse = None, 0, 0
    if train:
        keep = q.new_empty(2 * q.numel() + 4 * (q.numel() // q.shape[-1]), dtype=torch.uint8)
        rest = keep.data_ptr()
        lse = rest + 2 * q.numel()
    desc, address, need = _desc(plan, copies, False)
    device = q.get_device()
    before = _enter(device)
    try:
        work = q.new_empty(need, dtype=torch.uint8)
        capi.call("nsfps_block_attention_device", address, qp, kp, vp, blocks.data_ptr(),
                  0 if lengths is None else lengths.data_ptr(), out.data_ptr(),
                  lse, rest, work.data_ptr(), need,
                  torch._C._cuda_getCurrentRawStream(device))
    finally:
        _leave(before)
    return out, keep


def _backward(q, k, v, blocks, lengths, plan, out, keep, dout):
    import torch
    copies = tuple(c or t.data_ptr() % 16 != 0 for c, t in zip(plan[0], (q, k, v)))
    dq, dk, dv = q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)
    q, k, v = (_rows16(t, c) for t, c in zip((q, k, v), copies))
    dout, blocks = _rows16(dout, True), blocks.contiguous()
    lengths = None if lengths is None else lengths.contiguous()
    rest = keep.data_ptr()
    desc, address, need = _desc(plan, copies, True)
    device = q.get_device()
    before = _enter(device)
    try:
        work = q.new_empty(need, dtype=torch.uint8)
        capi.call("nsfps_block_attention_grad_device", address, q.data_ptr(), k.data_ptr(),
                  v.data_ptr(), blocks.data_ptr(), 0 if lengths is None else lengths.data_ptr(),
                  out.data_ptr(), rest + 2 * q.numel(), rest, dout.data_ptr(),
                  dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), work.data_ptr(), need,
                  torch._C._cuda_getCurrentRawStream(device))
    finally:
        _leave(before)
    return dq, dk, dv


_function = None


def _autograd():
    """The autograd node, made at its first use (the module itself does not
    need PyTorch)."""
    global _function
    if _function is None:
        import torch
        from torch.autograd.function import once_differentiable

        class BlockAttention(torch.autograd.Function):
            @staticmethod
            def forward(ctx, q, k, v, blocks, lengths, plan):
                out, keep = _forward(q, k, v, blocks, lengths, plan, True)
                ctx.save_for_backward(q, k, v, blocks, lengths, out, keep)
                ctx.plan = plan
                return out

            @staticmethod
            @once_differentiable
            def backward(ctx, dout):
                _no_tangents(dout)
                q, k, v, blocks, lengths, out, keep = ctx.saved_tensors
                grads = _backward(q, k, v, blocks, lengths, ctx.plan, out, keep, dout)
                return (*grads, None, None, None)

        _function = BlockAttention
    return _function


def block_attention(q, k, v, blocks, block: int, lengths=None, scale: float | None = None):
    """softmax(scale * q k^T) v over the keys of the blocks listed per query.

    q        (M, H, D), or (B, M, H, D) for B clouds: float16 or bfloat16
    k, v     (N, G, D) or (B, N, G, D) of q's type; H a multiple of G, query
             head h reads key head h // (H / G)
    blocks   int64 (M, top) or (B, M, top), as ``select_blocks`` gives them: a
             set of blocks of ``block`` consecutive keys; entries that are
             negative, repeated, or name no block count for nothing
    lengths  None, or int32 (B,): the keys of each padded cloud; what lies
             behind them, or in blocks that no query lists, is never part of a
             result.  Values that are listed have to be finite, and so have
             their scores in float32.
    scale    a number, by default 1 / sqrt(D) (what a tensor holds is read, which
             waits for a CUDA tensor, and has no gradient)

    D is a multiple of 8 up to 128, H at most 256.  Returns a tensor like q,
    dense; a query without any key gets zeros.  Scores and sums are float32;
    the softmax weights are rounded to q's type for the product with v.
    Gradients reach q, k and v (zeros for keys that no query lists), summed in
    a fixed order; forward-mode derivatives are refused.  Inputs whose rows are
    not 16-byte aligned are copied first.
    """
    import torch
    block, scale = int(block), None if scale is None else _number(scale)
    try:
        key = (_look(q), _look(k), _look(v), _look(blocks), _look(lengths), block, scale)
        plan = _attention_plans.get(key)
    except AttributeError:  # not tensors
        key = plan = None
    if plan is None:
        copies, shape = _attention_plan(q, k, v, blocks, block, lengths, scale)
        plan = _attention_plans.keep(key, (copies, shape, {}))
    _no_tangents(q, k, v)
    if (q.requires_grad or k.requires_grad or v.requires_grad) and torch.is_grad_enabled():
        return _autograd().apply(q, k, v, blocks, lengths, plan)
    return _forward(q, k, v, blocks, lengths, plan, False)[0]
