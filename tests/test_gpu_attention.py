"""Attention over listed blocks and its gradients against 64-bit formulas,
with tolerances that count the roundings of the definition."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

U32 = 2.0 ** -24


def _normal(shape, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def _lists(B, M, nb, top, seed):
    """Distinct blocks per query in no order, -1 behind the last block."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    order = torch.rand(B, M, nb, device="cuda", generator=g).argsort(2)[..., :top]
    return torch.nn.functional.pad(order, (0, top - order.shape[2]), value=-1)


def _seen(blocks, block, N, lengths, B):
    """(B, M, N): whether a query reads a key."""
    nb = (N + block - 1) // block
    member = torch.zeros(*blocks.shape[:2], nb + 1, dtype=torch.bool, device="cuda")
    member.scatter_(2, torch.where((blocks < 0) | (blocks >= nb), nb, blocks), True)
    seen = member[..., :nb].repeat_interleave(block, dim=2)[..., :N]
    if lengths is not None:
        seen = seen & (torch.arange(N, device="cuda") < lengths[:, None])[:, None, :]
    return seen


class Exact:
    """out, dq, dk, dv in 64 bits, and how far the operator may be off.

    The operator works in fp32 and rounds, besides its outputs, the weights p
    (for p v and p^T dout) and ds (for ds k and ds^T q) to the type, half a
    step u each (at least half a step of the smallest numbers); its delta comes
    from the rounded out.  An fp32 score is off by at most (D + 4) U32 of the
    sum of its terms' magnitudes, which p takes on as a relative error."""

    def __init__(self, q, k, v, blocks, block, lengths=None, scale=None, dout=None):
        dtype, (B, M, H, D), (N, G) = q.dtype, q.shape, k.shape[1:3]
        scale = 1 / math.sqrt(D) if scale is None else scale
        u = torch.finfo(dtype).eps / 2
        tiny = torch.finfo(dtype).smallest_normal * u
        seen = _seen(blocks, block, N, lengths, B)[:, None]             # B 1 M N
        valid = torch.ones(B, N, dtype=torch.bool, device="cuda")
        if lengths is not None:
            valid = torch.arange(N, device="cuda") < lengths[:, None]
        clean = [torch.where(valid[..., None, None], t.double(), 0.0) for t in (k, v)]
        kh, vh = (t.repeat_interleave(H // G, dim=2).transpose(1, 2) for t in clean)
        qh = q.double().transpose(1, 2)
        s = (qh @ kh.transpose(2, 3) * scale).masked_fill(~seen, -math.inf)
        p = torch.softmax(s, dim=-1).nan_to_num(0.0)
        off_s = (qh.abs() @ kh.abs().transpose(2, 3)) * abs(scale) * (D + 4) * U32
        off_s = torch.where(seen, off_s, 0.0).amax(-1, keepdim=True)
        rel = 2 * off_s + (64 + seen.sum(-1, keepdim=True)) * U32        # of p, in fp32
        out = p @ vh
        mag = (p * (u + rel) + tiny) @ vh.abs() * 1.01
        self.out, self.out_off = out.transpose(1, 2), (mag + u * out.abs() + tiny).transpose(1, 2)
        if dout is None:
            return
        do = dout.double().transpose(1, 2)
        dp = do @ vh.transpose(2, 3)
        delta = (p * dp).sum(-1, keepdim=True)
        ds = p * (dp - delta) * scale
        off_delta = (do.abs() * (mag + u * out.abs() + tiny)).sum(-1, keepdim=True)
        off_dp = (do.abs() @ vh.abs().transpose(2, 3)) * (D + 4) * U32
        # ds is rounded before the scale multiplies the sums of its products: below
        # the smallest normal number its half step is tiny, times |scale| in the result
        off_ds = (abs(scale) * p * (off_delta + off_dp + (dp.abs() + delta.abs()) * rel) * 1.01 +
                  u * ds.abs() * 1.01 + tiny * abs(scale))
        off_ds = torch.where(seen, off_ds, 0.0)
        n = (64 + M * H // G + N) * U32                                  # fp32 sums

        def heads(t):  # B H N D -> B N G D, query heads of a key head summed
            return t.reshape(B, G, H // G, N, D).sum(2).transpose(1, 2)

        dq = ds @ kh
        self.dq = dq.transpose(1, 2)
        self.dq_off = (off_ds @ kh.abs() + u * dq.abs() + n * (ds.abs() @ kh.abs()) +
                       tiny).transpose(1, 2)
        off_p = torch.where(seen, p * (u + rel) * 1.01 + tiny, 0.0)
        self.dk = heads(ds.transpose(2, 3) @ qh)
        self.dk_off = (heads(off_ds.transpose(2, 3) @ qh.abs() +
                             n * (ds.abs().transpose(2, 3) @ qh.abs())) + u * self.dk.abs() + tiny)
        self.dv = heads(p.transpose(2, 3) @ do)
        self.dv_off = (heads(off_p.transpose(2, 3) @ do.abs() +
                             n * (p.transpose(2, 3) @ do.abs())) + u * self.dv.abs() + tiny)


def _check(q, k, v, blocks, block, lengths=None, scale=None, train=True):
    from ns_fps_b200 import attention
    dout = _normal(q.shape, q.dtype, 99) if train else None
    ref = Exact(q, k, v, blocks, block, lengths, scale, dout)
    out = attention.block_attention(q, k, v, blocks, block, lengths=lengths, scale=scale)
    assert out.shape == q.shape and out.dtype == q.dtype
    assert bool(((out.double() - ref.out).abs() <= ref.out_off).all())
    if not train:
        return out
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    again = attention.block_attention(*leaves, blocks, block, lengths=lengths, scale=scale)
    assert torch.equal(again.detach(), out)
    grads = torch.autograd.grad(again, leaves, dout)
    for name, g, t in zip(("dq", "dk", "dv"), grads, (q, k, v)):
        assert g.shape == t.shape and g.dtype == t.dtype
        off = (g.double() - getattr(ref, name)).abs()
        assert bool((off <= getattr(ref, name + "_off")).all()), name
    return out


CASES = [  # B, M, N, H, G, D, block, top
    (1, 1, 1, 1, 1, 8, 16, 1),
    (1, 1, 1000, 8, 8, 64, 64, 16),
    (1, 3, 40, 2, 1, 16, 16, 64),
    (2, 37, 333, 4, 2, 40, 16, 5),
    (1, 130, 513, 6, 2, 72, 32, 9),
    (3, 65, 200, 3, 1, 128, 128, 2),
    (1, 20, 4500, 16, 1, 64, 64, 64),
    (1, 300, 2100, 2, 2, 64, 32, 16),
    (1, 500, 96, 4, 4, 32, 16, 6),
    (2, 257, 1030, 8, 2, 128, 64, 8),
    (1, 64, 700, 48, 2, 24, 128, 5),
    (1, 1000, 3000, 1, 1, 112, 32, 24),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", CASES)
def test_matches_the_formulas(case, dtype):
    B, M, N, H, G, D, block, top = case
    q, k, v = _normal((B, M, H, D), dtype, 1), _normal((B, N, G, D), dtype, 2), \
        _normal((B, N, G, D), dtype, 3)
    _check(q, k, v, _lists(B, M, (N + block - 1) // block, top, 4), block)


@pytest.mark.parametrize("block", [16, 32, 64, 128])
def test_padded_clouds_and_lists_that_name_nothing(block):
    """Lengths of 0, 1, inside a block and behind the end; entries that repeat,
    are negative or too large; queries without a key; NaN and infinities in
    what is padding."""
    B, M, N, H, G, D, top = 5, 90, 390, 4, 2, 64, 6
    dtype = torch.bfloat16
    q, k, v = _normal((B, M, H, D), dtype, 1), _normal((B, N, G, D), dtype, 2), \
        _normal((B, N, G, D), dtype, 3)
    lengths = torch.tensor([N, 0, 1, 200, 139], dtype=torch.int32, device="cuda")
    pad = torch.arange(N, device="cuda")[None, :] >= lengths[:, None]
    k[pad], v[pad] = math.nan, math.inf
    nb = (N + block - 1) // block
    blocks = _lists(B, M, nb, top, 4)
    blocks[:, ::7, 3] = blocks[:, ::7, 0]
    blocks[:, 1::7, :2] = -5
    blocks[:, 2::7, 1] = nb
    blocks[:, 3::7, 2] = 2 ** 40
    blocks[:, 4::7] = -1
    blocks[:, 5::7] = 0
    out = _check(q, k, v, blocks, block, lengths)
    assert not out[1].any() and not out[:, 4::7].any()


@pytest.mark.parametrize("M", [40, 6000])  # the direct path and the tiles
@pytest.mark.parametrize("block", [16, 64])
def test_blocks_that_nobody_lists_are_never_part_of_a_result(M, block):
    """NaN and infinities beside listed blocks, and in rows of q and dout whose
    query lists nothing; q, k and v gradients zero there and right elsewhere."""
    from ns_fps_b200 import attention
    B, N, H, G, D = 1, 1000, 4, 2, 64
    q, k, v = _normal((B, M, H, D), torch.bfloat16, 1), _normal((B, N, G, D), torch.bfloat16, 2), \
        _normal((B, N, G, D), torch.bfloat16, 3)
    nb = (N + block - 1) // block
    blocks = _lists(B, M, nb, 5, 4)
    blocks[blocks % 2 == 1] = -1  # odd blocks: not listed
    blocks[:, ::9] = -1
    dout = _normal(q.shape, torch.bfloat16, 5)
    ref = Exact(q, k, v, blocks, block, None, None, dout)
    odd = (torch.arange(N, device="cuda") // block) % 2 == 1
    k[:, odd], v[:, odd] = math.nan, math.inf
    q[:, ::9], dout[:, ::9] = math.nan, math.inf
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = attention.block_attention(*leaves, blocks, block)
    got = (out.detach(), *torch.autograd.grad(out, leaves, dout))
    for g, name in zip(got, ("out", "dq", "dk", "dv")):
        off = (g.double() - getattr(ref, name)).abs()
        assert bool((off <= getattr(ref, name + "_off")).all()), name
    assert not got[2][:, odd].any() and not got[3][:, odd].any() and not got[0][:, ::9].any()


def test_long_lists():
    """More pairs than a pass of short tiles sorts, in two clouds."""
    q, k, v = _normal((2, 20_000, 1, 16), torch.bfloat16, 1), \
        _normal((2, 500, 1, 16), torch.bfloat16, 2), _normal((2, 500, 1, 16), torch.bfloat16, 3)
    _check(q, k, v, _lists(2, 20_000, 32, 14, 4), 16)


def test_calls_taken_in_turns_equal_calls_apart():
    """A call whose partial results pass the limit takes its heads, then its
    clouds, in turns; each cloud and head by itself gives the same bits."""
    from ns_fps_b200 import attention
    B, M, N, H, D, top, block = 5, 40_000, 2000, 2, 128, 16, 16
    q, k, v, dout = (_normal((B, n, H, D), torch.bfloat16, i)
                     for i, n in enumerate((M, N, N, M)))
    blocks = _lists(B, M, (N + block - 1) // block, top, 9)

    def step(*x):
        leaves = [t.detach().requires_grad_() for t in x[:3]]
        out = attention.block_attention(*leaves, x[3], block)
        return (out.detach(), *torch.autograd.grad(out, leaves, x[4]))

    all_at_once = step(q, k, v, blocks, dout)
    for b in (0, B - 1):
        for h in range(H):
            part = step(*(t[b:b + 1, :, h:h + 1] for t in (q, k, v)), blocks[b:b + 1],
                        dout[b:b + 1, :, h:h + 1])
            for x, y in zip(all_at_once, part):
                assert torch.equal(x[b:b + 1, :, h:h + 1], y)


def test_every_query_lists_the_same_block():
    q, k, v = _normal((1, 5000, 2, 64), torch.bfloat16, 1), \
        _normal((1, 100, 1, 64), torch.bfloat16, 2), _normal((1, 100, 1, 64), torch.bfloat16, 3)
    blocks = torch.full((1, 5000, 3), 1, dtype=torch.int64, device="cuda")
    _check(q, k, v, blocks, 16)


@pytest.mark.parametrize("scale", [0.0, 4.0, -0.3])
def test_scales(scale):
    """Uniform weights, weights of nearly one key, and a negative scale."""
    q, k, v = _normal((1, 60, 2, 48), torch.float16, 1), _normal((1, 500, 2, 48), torch.float16, 2), \
        _normal((1, 500, 2, 48), torch.float16, 3)
    _check(q, k, v, _lists(1, 60, 32, 7, 4), 16, scale=scale)


def test_single_cloud_views_and_unaligned_inputs():
    from ns_fps_b200 import attention
    packed = _normal((2, 300, 3, 4, 64), torch.bfloat16, 1)
    q, k, v = packed[:, :70, 0], packed[:, :, 1], packed[:, :, 2]
    blocks = _lists(2, 70, 10, 4, 2)
    out = _check(q, k, v, blocks, 32)
    one = attention.block_attention(q[1], k[1], v[1], blocks[1], 32)
    # (a batch of one, not the batch of two: how a row's keys are split over
    # partial sums depends on the number of queries of a call)
    same = attention.block_attention(q[1:], k[1:], v[1:], blocks[1:], 32)
    assert torch.equal(one, same[0])
    wide = _normal((2, 300, 4, 67), torch.bfloat16, 5)
    _check(wide[:, :70, :, 3:], wide[..., 1:65], wide[..., 2:66], blocks, 32)
    _check(k.transpose(1, 2).contiguous().transpose(1, 2)[:, :70], k, v, blocks, 32)
    _check(k[:1, :70].expand(2, 70, 4, 64), k[:1].expand(2, 300, 4, 64), v, blocks, 32)


def test_empty_sizes():
    from ns_fps_b200 import attention
    for B, M, N in [(0, 3, 4), (2, 0, 40), (2, 3, 0)]:
        leaves = [torch.zeros(B, n, 2, 16, device="cuda", dtype=torch.float16, requires_grad=True)
                  for n in (M, N, N)]
        blocks = torch.zeros(B, M, 2, dtype=torch.int64, device="cuda")
        out = attention.block_attention(*leaves, blocks, 16)
        assert out.shape == (B, M, 2, 16) and not out.any()
        for g, t in zip(torch.autograd.grad(out, leaves, torch.ones_like(out)), leaves):
            assert g.shape == t.shape and not g.any()


def test_gradient_matches_differences():
    """Differences of the 64-bit formula along a direction against the
    operator's gradient."""
    from ns_fps_b200 import attention
    x = [_normal(s, torch.float16, i) for i, s in enumerate([(1, 30, 2, 32), (1, 90, 1, 32),
                                                            (1, 90, 1, 32)])]
    d = [_normal(t.shape, torch.float64, 10 + i) for i, t in enumerate(x)]
    blocks, w = _lists(1, 30, 6, 3, 7), _normal(x[0].shape, torch.float16, 8)
    leaves = [t.detach().requires_grad_() for t in x]
    grads = torch.autograd.grad(attention.block_attention(*leaves, blocks, 16), leaves, w)
    got = sum(float((g.double() * y).sum()) for g, y in zip(grads, d))
    h = 1e-4

    def value(s):
        q, k, v = (t.double() + s * h * y for t, y in zip(x, d))
        kh, vh = (t.expand(1, 90, 2, 32).transpose(1, 2) for t in (k, v))
        a = q.transpose(1, 2) @ kh.transpose(2, 3) / math.sqrt(32)
        a = a.masked_fill(~_seen(blocks, 16, 90, None, 1)[:, None], -math.inf)
        return float(((torch.softmax(a, -1) @ vh).transpose(1, 2) * w.double()).sum())

    ref = Exact(*x, blocks, 16, None, None, w)
    bound = sum(float((getattr(ref, n + "_off") * y.abs()).sum())
                for n, y in zip(("dq", "dk", "dv"), d))
    # the difference itself is off by a third derivative times h^2 / 6
    assert abs((value(1) - value(-1)) / (2 * h) - got) <= bound + 1e-3


def test_same_bits_again_on_another_stream_and_in_graphs():
    from ns_fps_b200 import attention
    q, k, v = _normal((2, 400, 4, 64), torch.bfloat16, 1), _normal((2, 1500, 2, 64), torch.bfloat16, 2), \
        _normal((2, 1500, 2, 64), torch.bfloat16, 3)
    blocks, dout = _lists(2, 400, 47, 9, 4), _normal(q.shape, torch.bfloat16, 5)

    def step():
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = attention.block_attention(*leaves, blocks, 32)
        return (out.detach(), *torch.autograd.grad(out, leaves, dout))

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kept = step()
        graphs.append((graph, kept))
    for graph, _ in graphs:
        graph.replay()
    torch.cuda.synchronize()
    for got in (step(), other, graphs[0][1], graphs[1][1]):
        for a, b in zip(first, got):
            assert torch.equal(a, b)


def test_sampler_to_attention_together():
    """The run a point network makes: samples, their features, nearby blocks,
    attention, and the gradient back into the features."""
    import numpy as np

    from ns_fps_b200 import attention, group, synthetic, torch_fps
    cloud = synthetic.cluster_cloud(5000, seed=5)
    cloud = cloud[np.lexsort(cloud.T)]
    pts = torch.from_numpy(np.ascontiguousarray(cloud)).cuda()
    H, D, block = 2, 32, 32
    feats = _normal((5000, H * D), torch.bfloat16, 1).requires_grad_()
    s = torch_fps.fps(pts, 256)
    q = group.gather_rows(feats, s).view(-1, H, D)
    blocks, d2 = attention.select_blocks(pts, group.gather_points(pts, s), block, 6)
    assert bool((d2[:, 0] == 0).all())  # a sample lies in a box
    kv = feats.view(-1, H, D)
    out = attention.block_attention(q, kv, kv, blocks, block)
    dout = _normal(out.shape, torch.bfloat16, 2)
    grad, = torch.autograd.grad(out, feats, dout)
    x = feats.detach().view(1, -1, H, D)
    ref = Exact(x[:, s], x, x, blocks[None], block, None, None, dout[None])
    assert bool(((out[None].double() - ref.out).abs() <= ref.out_off).all())
    total, off = ref.dk + ref.dv, ref.dk_off + ref.dv_off
    total[:, s] += ref.dq
    off[:, s] += ref.dq_off
    # PyTorch adds the three gradients in bf16: two more roundings
    size = ref.dk.abs() + ref.dv.abs() + off
    size[:, s] += ref.dq.abs()
    err = (grad.view(1, -1, H, D).double() - total).abs()
    assert bool((err <= off + 2 * 2.0 ** -8 * size * 1.01).all())


def test_refusals():
    from ns_fps_b200 import attention
    q, k = _normal((1, 5, 4, 64), torch.bfloat16, 1), _normal((1, 50, 2, 64), torch.bfloat16, 2)
    blocks = _lists(1, 5, 4, 2, 3)
    one = torch.zeros(1, dtype=torch.int32, device="cuda")
    for args, error in [
            ((q.float(), k.float(), k.float(), blocks, 16), TypeError),
            ((q, k.half(), k.half(), blocks, 16), TypeError),
            ((q, k, k[:, :40], blocks, 16), ValueError),
            ((q, k, k, blocks.int(), 16), TypeError),
            ((q, k, k, blocks, 20), ValueError),
            ((q, k, k, blocks[:, :3], 16), ValueError),
            ((q, k, k, blocks[..., :0], 16), ValueError),
            ((q, k, k, blocks.repeat(1, 1, 40), 16), ValueError),
            ((q[:, :, :3], k, k, blocks, 16), ValueError),
            ((q[..., :60], k[..., :60], k[..., :60], blocks, 16), ValueError),
            ((q[0], k, k, blocks, 16), ValueError),
            ((q, k, k, blocks, 16, one.repeat(2)), ValueError),
            ((q, k, k, blocks, 16, one.long()), TypeError),
            ((q, k, k, blocks, 16, None, math.inf), RuntimeError)]:
        with pytest.raises(error):
            attention.block_attention(*args)


def _one_block(B, M, N, H, G, D, dtype, seed):
    """A call in which every query reads all N keys, of one block of 16."""
    q, dout = _normal((B, M, H, D), dtype, seed), _normal((B, M, H, D), dtype, seed + 1)
    k, v = _normal((B, N, G, D), dtype, seed + 2), _normal((B, N, G, D), dtype, seed + 3)
    return q, k, v, torch.zeros(B, M, 1, dtype=torch.int64, device="cuda"), dout


def _grads(q, k, v, blocks, dout, block=16, lengths=None):
    from ns_fps_b200 import attention
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = attention.block_attention(*leaves, blocks, block, lengths=lengths)
    return torch.autograd.grad(out, leaves, dout)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,queries", [(64, 1), (64, 300), (128, 70), (24, 9)])
def test_one_key_moves_no_score(D, queries, dtype):
    """A query with one key gives it weight one wherever it lies: dq and dk
    are zero, dv is dout.  Queries beside it that read more keys keep theirs."""
    B, N, H, G = 2, 33, 4, 2
    q, k, v = (_normal(s, dtype, i) for i, s in
               enumerate([(B, queries, H, D), (B, N, G, D), (B, N, G, D)]))
    dout = _normal(q.shape, dtype, 7)
    blocks = torch.full((B, queries, 2), 2, dtype=torch.int64, device="cuda")
    dq, dk, dv = _grads(q, k, v, blocks, dout)
    assert not bool(dq.any()) and not bool(dk.any())
    # p is 1 up to the errors of an fp32 score, far less than the 2^-12 that
    # would round it to anything but 1; the sum's 600 terms are added in fp32
    sums = dout.double().reshape(B, queries, G, H // G, D).sum((1, 3))
    mag = dout.double().abs().reshape(B, queries, G, H // G, D).sum((1, 3))
    u = torch.finfo(dtype).eps / 2
    assert bool(((dv[:, 32].double() - sums).abs() <= u * sums.abs() + 1e-4 * mag + 2e-7).all())
    assert not bool(dv[:, :32].any())
    blocks[:, ::2, 1] = 0  # every other query reads 16 keys more
    dq = _grads(q, k, v, blocks, dout)[0]
    assert bool(dq[:, ::2].any()) and not bool(dq[:, 1::2].any())
    lengths = torch.tensor([1, 17], dtype=torch.int32, device="cuda")
    dq, dk, _ = _grads(q, k, v, torch.ones_like(blocks) * lengths[:, None, None] // 17, dout,
                       lengths=lengths)
    assert not bool(dq.any()) and not bool(dk.any())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N", [2, 3, 5, 11])
def test_gradients_of_few_keys(N, dtype):
    """dp - delta cancels where few keys share the weight.  dq and dk are off
    by the roundings of ds and of themselves alone.  A rounding error is uniform
    within half a step, at most u of the value, so over many independent values
    its 2-norm is at most u / sqrt(3) of theirs, and that of the two roundings
    together at most sqrt(2 / 3) u."""
    B, M, H, G, D = 2, 400, 4, 2, 64
    q, k, v, blocks, dout = _one_block(B, M, N, H, G, D, dtype, 3)
    ref = Exact(q, k, v, blocks, 16, dout=dout)
    dq, dk, _ = _grads(q, k, v, blocks, dout)
    u = torch.finfo(dtype).eps / 2
    for name, got, want in (("dq", dq, ref.dq), ("dk", dk, ref.dk)):
        off = float((got.double() - want).norm() / want.norm())
        assert off <= math.sqrt(2 / 3) * u, (name, off / u)


@pytest.mark.parametrize("N", [2, 7])
def test_gradients_of_few_keys_of_many_queries(N):
    """The same where the queries are enough to be gathered into tiles (above
    65,535, whatever they read)."""
    B, M, H, G, D, dtype = 2, 33_000, 1, 1, 64, torch.bfloat16
    q, k, v, blocks, dout = _one_block(B, M, N, H, G, D, dtype, 5)
    ref = Exact(q, k, v, blocks, 16, dout=dout)
    dq, dk, _ = _grads(q, k, v, blocks, dout)
    u = torch.finfo(dtype).eps / 2
    off = float((dq.double() - ref.dq).norm() / ref.dq.norm())
    assert off <= math.sqrt(2 / 3) * u, off / u
    # dk adds M terms in fp32 besides
    off = float((dk.double() - ref.dk).norm() / ref.dk.norm())
    assert off <= math.sqrt(2 / 3) * u + M * U32, off / u


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M", [16_384, 14_000])
def test_a_last_turn_of_fewer_clouds(M, dtype):
    """Three clouds whose partial results make turns of two and one: the
    forward's (M = 16,384) or the gradient's (14,000).  The last turn sorts half
    the pairs of a full one (786,432 or 672,000) in its scratch.  Each cloud by
    itself gives the same bits."""
    from ns_fps_b200 import attention
    B, N, H, G, D, top, block = 3, 600, 4, 2, 128, 24, 16
    q, dout = _normal((B, M, H, D), dtype, 1), _normal((B, M, H, D), dtype, 2)
    k, v = _normal((B, N, G, D), dtype, 3), _normal((B, N, G, D), dtype, 4)
    dout[1] *= 2.0 ** -12  # (in half precision each cloud has its own factor)
    blocks = _lists(B, M, (N + block - 1) // block, top, 5)

    def step(*x):
        leaves = [t.detach().requires_grad_() for t in x[:3]]
        out = attention.block_attention(*leaves, x[3], block)
        return (out.detach(), *torch.autograd.grad(out, leaves, x[4]))

    together = step(q, k, v, blocks, dout)
    for b in range(B):
        apart = step(*(t[b:b + 1] for t in (q, k, v, blocks, dout)))
        for x, y in zip(together, apart):
            assert torch.equal(x[b:b + 1], y)


@pytest.mark.parametrize("device", ["cpu", "cuda"])
def test_a_scale_that_changes_in_place(device):
    """A scale held in a tensor is read at every call, and not kept."""
    import gc
    import weakref

    from ns_fps_b200 import attention
    q, k, v = (_normal((1, n, 2, 32), torch.float16, i) for i, n in enumerate((9, 100, 100)))
    blocks, dout = _lists(1, 9, 7, 3, 4), _normal(q.shape, torch.float16, 5)

    def step(scale):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = attention.block_attention(*leaves, blocks, 16, scale=scale)
        return (out.detach(), *torch.autograd.grad(out, leaves, dout))

    scale = torch.tensor(0.25, device=device)
    for value in (0.25, 2.0, 0.0):
        scale.fill_(value)
        for x, y in zip(step(scale), step(value)):
            assert torch.equal(x, y)
    kept = weakref.ref(scale)
    del scale
    gc.collect()
    assert kept() is None


def test_forward_mode_derivatives_are_refused():
    """They are not computed, and no result without a tangent stands for one."""
    from torch.autograd import forward_ad

    from ns_fps_b200 import attention
    x = [_normal((n, 2, 32), torch.float16, i) for i, n in enumerate((9, 100, 100))]
    blocks, dout = _lists(1, 9, 7, 3, 4)[0], _normal(x[0].shape, torch.float16, 5)
    plain = attention.block_attention(*x, blocks, 16)
    with forward_ad.dual_level():
        for i in range(3):
            for leaf in (False, True):
                args = [t.detach().requires_grad_(leaf) for t in x]
                args[i] = forward_ad.make_dual(args[i], torch.ones_like(x[i]))
                with pytest.raises(RuntimeError, match="forward"):
                    attention.block_attention(*args, blocks, 16)
        scale = forward_ad.make_dual(torch.tensor(0.5), torch.tensor(1.0))
        with pytest.raises(RuntimeError, match="forward"):
            attention.block_attention(*x, blocks, 16, scale=scale)
        leaves = [t.detach().requires_grad_() for t in x]
        out = attention.block_attention(*leaves, blocks, 16)
        with pytest.raises(RuntimeError, match="forward"):
            torch.autograd.grad(out, leaves, forward_ad.make_dual(dout, torch.ones_like(dout)))
        assert torch.equal(attention.block_attention(*x, blocks, 16), plain)  # no tangent: as ever
    assert torch.equal(attention.block_attention(*x, blocks, 16), plain)


@pytest.mark.parametrize("size,v_size,M,N,D", [
    (1e-4, 1.0, 200, 2048, 64), (1e-3, 1.0, 200, 2048, 64), (1.0, 1.0, 200, 2048, 64),
    (1e-3, 1.0, 100, 512, 128), (1e-2, 1.0, 70, 2000, 24), (8000.0, 1.0, 8, 3, 64),
    (8000.0, 1.0, 8, 3, 128), (1e-3, 500.0, 200, 2048, 64), (10.0, 0.002, 200, 2048, 64)])
def test_half_precision_gradients_of_any_size(size, v_size, M, N, D):
    """float16 gradients where the incoming one is small, as it is without a
    scaled loss, and large, as with one: dq, dk and dv are off by the roundings
    of ds or p and of themselves alone.  A rounding error is uniform within half
    a step, at most u of the value or 2^-25 below the smallest normal number, so
    its square is at most a third of that on average; the two roundings are
    independent.  ds and p keep clear of the smallest numbers, whatever the size
    of dout; the results may lie among them.  (64 roundings of fp32 besides.)"""
    B, H, G, block = 1, 2, 1, 128
    q, k, v = (_normal(s, torch.float16, i) for i, s in
               enumerate([(B, M, H, D), (B, N, G, D), (B, N, G, D)]))
    v = (v.float() * v_size).half()
    dout = (_normal(q.shape, torch.float32, 9) * size).half()
    blocks = _lists(B, M, (N + block - 1) // block, 16, 4)
    ref = Exact(q, k, v, blocks, block, None, None, dout)
    got = _grads(q, k, v, blocks, dout, block)
    u = 2.0 ** -11
    for name, g in zip(("dq", "dk", "dv"), got):
        want = getattr(ref, name)
        assert bool(torch.isfinite(g).all()), name
        off = float((g.double() - want).norm())
        own = math.sqrt(2 / 3) * u * float(want.norm())
        low = 2.0 ** -25 * math.sqrt(want.numel() / 3)
        assert off <= math.hypot(own, low) + 64 * U32 * float(want.norm()), (name, off, own, low)


def test_half_precision_gradients_of_unlike_rows():
    """A query whose incoming gradient is a thousandth of its neighbours', in the
    same tiles, keeps its dq to the roundings; an infinite one spoils its own."""
    B, M, N, H, G, D, block = 1, 64, 1024, 2, 1, 64, 128
    q, k, v = (_normal(s, torch.float16, i) for i, s in
               enumerate([(B, M, H, D), (B, N, G, D), (B, N, G, D)]))
    dout = _normal(q.shape, torch.float32, 9)
    dout[:, ::2] *= 1e-3
    dout = dout.half()
    blocks = _lists(B, M, 8, 8, 4)
    ref = Exact(q, k, v, blocks, block, None, None, dout)
    u = 2.0 ** -11

    def small(dq, rows):
        want = ref.dq[:, rows]
        off = float((dq[:, rows].double() - want).norm())
        low = 2.0 ** -25 * math.sqrt(want.numel() / 3)
        bound = math.hypot(math.sqrt(2 / 3) * u * float(want.norm()), low)
        assert off <= bound + 64 * U32 * float(want.norm()), (off, bound)

    small(_grads(q, k, v, blocks, dout, block)[0], slice(0, None, 2))
    dout[0, 1, 0, 5] = math.inf
    dq = _grads(q, k, v, blocks, dout, block)[0]
    assert not bool(torch.isfinite(dq[0, 1, 0]).all())
    small(dq, slice(2, None, 2))


def test_one_cloud_beyond_the_limit_of_a_turn():
    """One cloud and key head whose partial results pass 1 GiB stay together;
    parts of the queries give the same within the roundings, and their dk and
    dv add up."""
    from ns_fps_b200 import attention, capi
    import ctypes
    M, N, H, D, top, block, dtype = 66_000, 400, 2, 128, 16, 16, torch.bfloat16
    three = ctypes.c_int64 * 3
    desc = capi.AttentionDesc(1, M, N, H, 1, D, block, top, capi.BF16, three(0, H * D, D),
                              three(0, D, 0), three(0, D, 0), 0.1, 0)
    assert 1 << 30 < M * top * H * 4 * (D + 1) <= capi.block_attention_workspace(desc, False)
    q, dout = _normal((1, M, H, D), dtype, 1), _normal((1, M, H, D), dtype, 2)
    k, v = _normal((1, N, 1, D), dtype, 3), _normal((1, N, 1, D), dtype, 4)
    blocks = _lists(1, M, N // block, top, 5)

    def step(part):
        leaves = [t.detach().requires_grad_() for t in (q[:, part], k, v)]
        out = attention.block_attention(*leaves, blocks[:, part], block)
        return (out.detach(), *torch.autograd.grad(out, leaves, dout[:, part]))

    out, dq, dk, dv = step(slice(None))
    sums = [torch.zeros_like(t, dtype=torch.float64) for t in (dk, dv)]
    offs = [torch.zeros_like(t) for t in sums]
    for at in range(0, M, 11_000):
        part = slice(at, at + 11_000)
        ref = Exact(q[:, part], k, v, blocks[:, part], block, None, None, dout[:, part])
        assert bool(((out[:, part].double() - ref.out).abs() <= ref.out_off).all())
        assert bool(((dq[:, part].double() - ref.dq).abs() <= ref.dq_off).all())
        for i, name in enumerate(("dk", "dv")):
            sums[i] += getattr(ref, name)
            offs[i] += getattr(ref, name + "_off")
        del ref
    # (the parts' bounds count a rounding of the result each, and fp32 sums over
    # the part's rows: six times as many here)
    for got, want, off in zip((dk, dv), sums, offs):
        u = torch.finfo(dtype).eps / 2
        assert bool(((got.double() - want).abs() <= 6 * off + u * want.abs()).all())


def test_half_precision_same_bits_again_on_another_stream_and_in_graphs():
    """The factor of ds comes from maxima that CTAs raise in any order, in the
    call's own scratch: two captured calls and an eager one side by side."""
    from ns_fps_b200 import attention
    q, k, v = _normal((2, 700, 4, 64), torch.float16, 1), _normal((2, 1500, 2, 64), torch.float16, 2), \
        _normal((2, 1500, 2, 64), torch.float16, 3)
    blocks, dout = _lists(2, 700, 47, 9, 4), _normal(q.shape, torch.float16, 5)

    def step(size):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = attention.block_attention(*leaves, blocks, 32)
        return (out.detach(), *torch.autograd.grad(out, leaves, dout * size))

    sizes = (1.0, 1e-3)
    first = [step(s) for s in sizes]
    graphs = []
    for s in sizes:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kept = step(s)
        graphs.append((graph, kept))
    side = [torch.cuda.Stream() for _ in sizes]
    for _ in range(3):
        for s, (graph, _) in zip(side, graphs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                graph.replay()
        eager = [step(s) for s in sizes]
        torch.cuda.synchronize()
        for i in range(2):
            for a, b, c in zip(first[i], graphs[i][1], eager[i]):
                assert torch.equal(a, b) and torch.equal(a, c)
