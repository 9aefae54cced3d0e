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
import functools
import math

from . import capi
from .group import _cloud_batch, _dtype_code, _on

__all__ = ["select_blocks", "block_attention"]

_BLOCKS = (16, 32, 64, 128)
_MAX_TOP = 64


def _check_block(block, top):
    if block not in _BLOCKS:
        raise ValueError("block must be 16, 32, 64 or 128")
    if not 1 <= top <= _MAX_TOP:
        raise ValueError(f"top must be in 1..{_MAX_TOP}")


def _check_lengths(lengths, B, device):
    """Address of the clouds' lengths (0 for None)."""
    import torch
    if lengths is None:
        return 0, None
    if not isinstance(lengths, torch.Tensor) or not lengths.is_cuda or lengths.dtype != torch.int32:
        raise TypeError("lengths must be an int32 CUDA tensor")
    if lengths.numel() != B or lengths.dim() > 1:
        raise ValueError("lengths must hold one length per cloud")
    if lengths.device != device:
        raise ValueError("lengths must be on the clouds' device")
    lengths = lengths.contiguous()
    return lengths.data_ptr(), lengths


@functools.lru_cache(maxsize=256)
def _select_desc(B, N, M, block, top):
    desc = capi.SelectDesc(B, N, M, block, top)
    return desc, capi.select_blocks_workspace(desc)


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
    radius: ``blocks.masked_fill(d2 > radius * radius, -1)``.
    """
    import torch
    pts, single = _cloud_batch(points, "points")
    ctr, single_c = _cloud_batch(centers, "centers")
    if single != single_c or pts.shape[0] != ctr.shape[0]:
        raise ValueError("points and centers must have the same batch layout")
    if pts.device != ctr.device:
        raise ValueError("points and centers must be on the same device")
    block, top = int(block), int(top)
    _check_block(block, top)
    B, N, M = int(pts.shape[0]), int(pts.shape[1]), int(ctr.shape[1])
    len_ptr, _len = _check_lengths(lengths, B, pts.device)
    blocks = pts.new_empty((B, M, top), dtype=torch.int64)
    d2 = pts.new_empty((B, M, top))
    desc, need = _select_desc(B, N, M, block, top)
    with _on(pts) as stream:
        work = pts.new_empty(need, dtype=torch.uint8)
        capi.select_blocks_device(desc, pts.data_ptr(), len_ptr, ctr.data_ptr(),
                                  blocks.data_ptr(), d2.data_ptr(), work.data_ptr(), need, stream)
    return (blocks[0], d2[0]) if single else (blocks, d2)


def _rows16(t):
    """t with contiguous heads, 16-byte aligned rows: t itself when it is."""
    if t.stride(-1) != 1 or t.data_ptr() % 16 or any(s % 8 for s in _strides(t)):
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone()
    return t


def _strides(t):
    """Strides of batch, row and head; an axis of one entry is never stepped."""
    return tuple([s if n > 1 else 0 for s, n in zip(t.stride()[:3], t.shape[:3])])


@functools.lru_cache(maxsize=256)
def _make_desc(q_shape, k_shape, top, q_strides, k_strides, v_strides, code, block, scale,
               backward):
    B, M, H, D = q_shape
    three = ctypes.c_int64 * 3
    desc = capi.AttentionDesc(B, M, k_shape[1], H, k_shape[2], D, block, top, code,
                              three(*q_strides), three(*k_strides), three(*v_strides), scale, 0)
    return desc, capi.block_attention_workspace(desc, backward)


def _desc(q, k, v, blocks, block, scale, backward):
    """The call's descriptor and its scratch bytes."""
    return _make_desc(q.shape, k.shape, blocks.shape[2], _strides(q), _strides(k), _strides(v),
                      _dtype_code(q, "q", (capi.F16, capi.BF16)), block, scale, backward)


def _forward(q, k, v, blocks, block, lengths, scale, want_lse):
    import torch
    q, k, v, blocks = _rows16(q), _rows16(k), _rows16(v), blocks.contiguous()
    len_ptr, _len = _check_lengths(lengths, q.shape[0], q.device)
    out = q.new_empty(q.shape)
    lse = q.new_empty(q.shape[:3], dtype=torch.float32) if want_lse else None
    desc, need = _desc(q, k, v, blocks, block, scale, False)
    with _on(q) as stream:
        work = q.new_empty(need, dtype=torch.uint8)
        capi.block_attention_device(desc, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                                    blocks.data_ptr(), len_ptr, out.data_ptr(),
                                    lse.data_ptr() if want_lse else 0, work.data_ptr(), need,
                                    stream)
    return out, lse


def _backward(q, k, v, blocks, block, lengths, scale, out, lse, dout):
    import torch
    q, k, v, dout, blocks = _rows16(q), _rows16(k), _rows16(v), dout.contiguous(), blocks.contiguous()
    dout = _rows16(dout)
    len_ptr, _len = _check_lengths(lengths, q.shape[0], q.device)
    dq, dk, dv = q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)
    desc, need = _desc(q, k, v, blocks, block, scale, True)
    with _on(q) as stream:
        work = q.new_empty(need, dtype=torch.uint8)
        capi.block_attention_grad_device(
            desc, q.data_ptr(), k.data_ptr(), v.data_ptr(), blocks.data_ptr(), len_ptr,
            out.data_ptr(), lse.data_ptr(), dout.data_ptr(), dq.data_ptr(), dk.data_ptr(),
            dv.data_ptr(), work.data_ptr(), need, stream)
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
            def forward(ctx, q, k, v, blocks, block, lengths, scale):
                out, lse = _forward(q, k, v, blocks, block, lengths, scale, True)
                ctx.save_for_backward(q, k, v, blocks, lengths, out, lse)
                ctx.block, ctx.scale = block, scale
                return out

            @staticmethod
            @once_differentiable
            def backward(ctx, dout):
                q, k, v, blocks, lengths, out, lse = ctx.saved_tensors
                grads = _backward(q, k, v, blocks, ctx.block, lengths, ctx.scale, out, lse, dout)
                return (*grads, None, None, None, None)

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
             behind them is never read into a result
    scale    default 1 / sqrt(D)

    D is a multiple of 8 up to 128, H at most 256.  Returns a tensor like q,
    dense; a query without any key gets zeros.  Scores and sums are float32;
    the softmax weights are rounded to q's type for the product with v.
    Gradients reach q, k and v (zeros for keys that no query lists), summed in
    a fixed order.  Inputs whose rows are not 16-byte aligned are copied first.
    """
    import torch
    single = isinstance(q, torch.Tensor) and q.dim() == 3
    for name, t in (("q", q), ("k", k), ("v", v)):
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise TypeError(f"{name} must be a CUDA tensor")
        _dtype_code(t, name, (capi.F16, capi.BF16))
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
    block = int(block)
    _check_block(block, blocks.shape[2])
    _check_lengths(lengths, B, q.device)
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        out = _autograd().apply(q, k, v, blocks, block, lengths, scale)
    else:
        out = _forward(q, k, v, blocks, block, lengths, scale, False)[0]
    return out[0] if single else out
