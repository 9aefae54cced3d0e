"""The nearest blocks of a cloud against a restatement in the same fp32
arithmetic, index for index, and its distances in 64 bits."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def _cloud(B, N, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    p = torch.randn(B, N, 3, device="cuda", generator=g)
    # runs of near points: sorted along x within the cloud
    return torch.gather(p, 1, p[..., :1].argsort(1).expand(B, N, 3)).contiguous()


def _reference(points, centers, block, top, lengths=None):
    """One cloud at a time; (d2, index) order by a stable sort."""
    outs = []
    for b in range(points.shape[0]):
        n = points.shape[1] if lengths is None else min(max(int(lengths[b]), 0), points.shape[1])
        M = centers.shape[1]
        blocks = torch.full((M, top), -1, dtype=torch.int64, device="cuda")
        d2 = torch.full((M, top), math.inf, device="cuda")
        if n:
            parts = points[b, :n].split(block)
            lo = torch.stack([p.nan_to_num(math.inf, math.inf, -math.inf).amin(0) for p in parts])
            hi = torch.stack([p.nan_to_num(-math.inf, math.inf, -math.inf).amax(0) for p in parts])
            d = []
            for a in range(3):
                c = centers[b, :, a, None]
                gap = torch.fmax(torch.fmax(lo[:, a] - c, c - hi[:, a]), torch.zeros_like(c))
                d.append(gap * gap)
            far = (d[0] + d[1]) + d[2]
            s = torch.sort(far, dim=1, stable=True)
            k = min(top, len(parts))
            blocks[:, :k], d2[:, :k] = s.indices[:, :k], s.values[:, :k]
        outs.append((blocks, d2))
    return torch.stack([o[0] for o in outs]), torch.stack([o[1] for o in outs])


def _check(points, centers, block, top, lengths=None):
    from ns_fps_b200 import attention
    got = attention.select_blocks(points, centers, block, top, lengths=lengths)
    ref = _reference(points, centers, block, top, lengths)
    assert torch.equal(got[0], ref[0])
    assert torch.equal(got[1], ref[1])


@pytest.mark.parametrize("B,N,M,block,top", [
    (1, 1, 1, 16, 1), (1, 17, 3, 16, 64), (2, 1000, 50, 16, 7), (1, 5000, 1, 32, 16),
    (1, 5000, 2500, 32, 33), (3, 2049, 1000, 64, 16), (1, 130_000, 5, 16, 64),
    (1, 40_000, 4000, 128, 32), (1, 65_537, 9, 64, 1)])
def test_matches_the_restatement(B, N, M, block, top):
    pts, ctr = _cloud(B, N, 1), _cloud(B, M, 2)
    _check(pts, ctr, block, top)
    _check(pts, pts[:, : min(M, N)].contiguous(), block, top)  # inside boxes: many ties at 0


def test_padded_clouds():
    from ns_fps_b200 import attention
    pts, ctr = _cloud(6, 600, 3), _cloud(6, 700, 4)
    lengths = torch.tensor([600, 0, 1, 17, 900, -4], dtype=torch.int32, device="cuda")
    keep = torch.arange(600, device="cuda")[None, :, None] < lengths[:, None, None].clamp(max=600)
    pts = torch.where(keep, pts, math.nan)  # padding is never read into a box
    _check(pts, ctr, 16, 20, lengths)
    one = attention.select_blocks(pts[3], ctr[3], 16, 20, lengths=lengths[3])
    both = attention.select_blocks(pts, ctr, 16, 20, lengths=lengths)
    assert torch.equal(one[0], both[0][3]) and torch.equal(one[1], both[1][3])


def test_ties_take_the_lower_index():
    pts = torch.zeros(1, 5000, 3, device="cuda")
    ctr = _cloud(1, 40, 5)
    _check(pts, ctr, 16, 40)
    _check(pts.repeat(1, 1, 1), ctr.repeat(1, 100, 1), 16, 40)
    # distances that fall with the index: every block displaces the list
    line = torch.zeros(1, 20_000, 3, device="cuda")
    line[0, :, 0] = torch.arange(20_000, 0, -1, device="cuda")
    _check(line, torch.zeros(1, 30, 3, device="cuda"), 16, 64)
    _check(line, torch.zeros(1, 3000, 3, device="cuda"), 16, 20)


def test_values_at_the_edges():
    """Overflowing distances, infinities, NaN coordinates and centres."""
    pts = _cloud(1, 800, 6)
    pts[0, 100:140] *= 1e30
    pts[0, 200, 1] = math.inf
    pts[0, 300, 2] = -math.inf
    pts[0, 400:450, 0] = math.nan
    ctr = _cloud(1, 60, 7)
    ctr[0, 0, 0] = math.nan
    ctr[0, 1] = math.inf
    ctr[0, 2] = -math.inf
    ctr[0, 3] = 3e38
    _check(pts, ctr, 16, 64)
    _check(pts, ctr.repeat(1, 50, 1), 16, 30)


def test_distances_in_64_bits():
    from ns_fps_b200 import attention
    pts, ctr = _cloud(1, 3000, 8), _cloud(1, 100, 9)
    blocks, d2 = attention.select_blocks(pts, ctr, 32, 10)
    parts = pts[0].double().split(32)
    lo, hi = (torch.stack([getattr(p, f)(0) for p in parts]) for f in ("amin", "amax"))
    c = ctr[0].double()[:, None]
    gap = torch.clamp(torch.maximum(lo - c, c - hi), min=0)
    ref = torch.gather((gap ** 2).sum(-1), 1, blocks[0])
    # a difference, a square and two sums, half a step each: 2 * 1 + 1 + 2
    assert bool(((d2[0].double() - ref).abs() <= ref * 5.01 * 2.0 ** -24).all())


def test_empty_sizes_streams_graphs_and_refusals():
    from ns_fps_b200 import attention
    z = torch.zeros(2, 0, 3, device="cuda")
    blocks, d2 = attention.select_blocks(z, _cloud(2, 3, 1), 16, 2)
    assert bool((blocks == -1).all()) and bool(torch.isinf(d2).all())
    assert attention.select_blocks(_cloud(2, 9, 1), z, 16, 2)[0].shape == (2, 0, 2)
    pts, ctr = _cloud(2, 5000, 1), _cloud(2, 3000, 2)
    ref = _reference(pts, ctr, 32, 8)
    graph = torch.cuda.CUDAGraph()
    attention.select_blocks(pts, ctr, 32, 8)
    with torch.cuda.graph(graph):
        kept = attention.select_blocks(pts, ctr, 32, 8)
    graph.replay()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = attention.select_blocks(pts, ctr, 32, 8)
    torch.cuda.synchronize()
    for got in (kept, other):
        assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    for args, error in [((pts, ctr, 24, 8), ValueError), ((pts, ctr, 32, 0), ValueError),
                        ((pts, ctr, 32, 65), ValueError), ((pts.double(), ctr, 32, 8), TypeError),
                        ((pts, ctr[:1], 32, 8), ValueError), ((pts[0], ctr, 32, 8), ValueError),
                        ((pts, ctr, 32, 8, torch.zeros(3, dtype=torch.int32, device="cuda")),
                         ValueError),
                        ((pts, ctr, 32, 8, torch.zeros(2, device="cuda")), TypeError)]:
        with pytest.raises(error):
            attention.select_blocks(*args)
