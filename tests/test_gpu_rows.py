"""Row lookup by index and its gradient against 64-bit restatements."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def _table(B, N, C, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    shape = (N, C) if B is None else (B, N, C)
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def _idx(shape, N, seed=1, lo=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(lo, max(N, 1), shape, device="cuda", generator=g)


def _forward(table, idx, scale):
    """64 bits; negative -> 0, too large -> NaN."""
    N, C = table.shape[-2:]
    t = table.double()
    safe = idx.clamp(0, N - 1)
    if table.dim() == 2:
        out = t[safe]
    else:
        flat = safe.reshape(safe.shape[0], -1)
        out = torch.stack([t[b][flat[b]] for b in range(t.shape[0])]).reshape(*idx.shape, C)
    out = out * scale
    out = torch.where((idx < 0)[..., None], 0.0, out)
    return torch.where((idx >= N)[..., None], math.nan, out)


def _backward(dout, idx, shape, scale):
    """64 bits, and the sum of magnitudes."""
    N, C = shape[-2:]
    B = 1 if len(shape) == 2 else shape[0]
    out = torch.zeros(B, N, C, dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(out)
    num = torch.zeros(B, N, 1, dtype=torch.float64, device="cuda")
    for b in range(B):
        i = idx.reshape(-1) if len(shape) == 2 else idx[b].reshape(-1)
        d = (dout.reshape(-1, C) if len(shape) == 2 else dout[b].reshape(-1, C)).double()
        ok = (i >= 0) & (i < N)
        out[b].index_add_(0, i[ok], d[ok])
        mag[b].index_add_(0, i[ok], d[ok].abs())
        num[b].index_add_(0, i[ok], torch.ones(int(ok.sum()), 1, dtype=torch.float64, device="cuda"))
    s = abs(scale)
    return (out * scale).reshape(shape), (mag * s).reshape(shape), num.expand(B, N, C).reshape(shape)


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _tiny(dtype):
    """Half a step below the smallest normal number."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


CASES = [  # B, N, C, idx shape, scale
    (None, 1, 1, (1,), 1.0),
    (None, 7, 3, (5, 4), 2.5),
    (None, 10_000, 64, (1000,), 1.0),
    (None, 501, 200, (33, 7, 3), math.sqrt(200.0)),
    (None, 3, 17, (2000,), 0.5),
    (1, 1, 8, (1, 1), -1.0),
    (3, 130, 96, (3, 77, 5), 1.0),
    (2, 1000, 10, (2, 1), 1.0),
    (4, 65, 260, (4, 300), 0.3),
    (2, 5, 1030, (2, 41), 1.0),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("case", CASES)
def test_lookup_and_gradient(case, dtype):
    from ns_fps_b200 import group
    B, N, C, shape, scale = case
    table = _table(B, N, C, dtype).requires_grad_()
    idx = _idx(shape, N, lo=-1)
    out = group.gather_rows(table, idx, scale)
    assert out.shape == (*shape, C) and out.dtype == dtype
    ref = _forward(table.detach(), idx, scale)
    # scale rounded to fp32, the product rounded to fp32 and then to the type
    tol = ref.abs() * (_half_step(dtype) + 3 * 2.0 ** -24) + _tiny(dtype)
    assert bool(((out.detach().double() - ref).abs() <= tol).all())
    if scale == 1.0:
        assert bool((out.detach().double() == ref).all())
    dout = _table(None, math.prod(shape), C, dtype, 5).reshape(*shape, C)
    grad, = torch.autograd.grad(out, table, dout)
    ref, mag, num = _backward(dout, idx, table.shape, scale)
    # a sum of n terms in fp32 is off by at most n half steps of the sum of magnitudes
    tol = ref.abs() * _half_step(dtype) + mag * (num + 3) * 2.0 ** -24 * 1.01 + _tiny(dtype)
    assert bool(((grad.double() - ref).abs() <= tol).all())
    assert bool((grad[num == 0] == 0).all())


@pytest.mark.parametrize("count", [255, 256, 257, 512, 513, 5000, 100_003])
def test_gradient_of_a_row_that_many_entries_name(count):
    """Whole numbers whose sums fp32 holds exactly: one hot row, two that meet
    in a tile, short ones between."""
    from ns_fps_b200 import group
    N, C = 9, 24
    idx = torch.full((count,), 4, dtype=torch.int64, device="cuda")
    idx[: count // 2] = 2
    idx[::97] = 3
    idx[5] = 0
    idx[-1] = 8
    table = torch.zeros(N, C, device="cuda", requires_grad=True)
    dout = _idx((count, C), 16, seed=3).float()
    grad, = torch.autograd.grad(group.gather_rows(table, idx), table, dout)
    ref, _, _ = _backward(dout, idx, (N, C), 1.0)
    assert torch.equal(grad.double(), ref)


@pytest.mark.parametrize("count,N", [(70_001, 9), (90_000, 70_001), (600_011, 70_001),
                                     (530_000, 200)])
def test_gradient_of_long_lists(count, N):
    """Lists of many tiles and of two and three digits; whole numbers, exact."""
    from ns_fps_b200 import group
    table = torch.zeros(N, 3, device="cuda", requires_grad=True)
    idx = _idx((count,), N, lo=-N // 50 - 1)
    dout = _idx((count, 3), 4, seed=3).float()
    grad, = torch.autograd.grad(group.gather_rows(table, idx), table, dout)
    assert torch.equal(grad.double(), _backward(dout, idx, (N, 3), 1.0)[0])


def test_indices_that_name_no_row():
    from ns_fps_b200 import group
    table = _table(2, 6, 5, torch.float32).requires_grad_()
    idx = torch.tensor([[-1, 5, 6, -2 ** 63], [2 ** 62, 0, -5, 5]], device="cuda")
    out = group.gather_rows(table, idx)
    ref = _forward(table.detach(), idx, 1.0)
    assert torch.equal(out.detach().double().nan_to_num(7e7), ref.nan_to_num(7e7))
    grad, = torch.autograd.grad(out, table, torch.ones_like(out))
    assert torch.equal(grad.double(), _backward(torch.ones_like(out), idx, table.shape, 1.0)[0])


def test_empty_sizes():
    from ns_fps_b200 import group
    for shape, ishape in [((0, 4), (0,)), ((5, 4), (0,)), ((5, 0), (3,)), ((0, 3, 4), (0, 2)),
                          ((2, 3, 4), (2, 0)), ((2, 0, 4), (2, 3))]:
        table = torch.zeros(shape, device="cuda", requires_grad=True)
        idx = torch.full(ishape, -1, dtype=torch.int64, device="cuda")
        out = group.gather_rows(table, idx)
        assert out.shape == (*ishape, shape[-1])
        grad, = torch.autograd.grad(out, table, torch.ones_like(out))
        assert grad.shape == table.shape and not grad.any()


def test_views_and_shared_tables():
    """Rows with a stride, an offset that breaks alignment, an expanded batch
    and an expanded incoming gradient."""
    from ns_fps_b200 import group
    big = _table(2, 50, 40, torch.bfloat16)
    idx = _idx((2, 33), 50)
    for view in (big[..., 3:20], big[..., ::2], big[:, ::2], big.transpose(0, 1)[:2],
                 big[0].expand(2, 50, 40)):
        i = idx.clamp(max=view.shape[1] - 1)
        assert torch.equal(group.gather_rows(view, i).double(), _forward(view, i, 1.0))
    shared = big[0].clone().requires_grad_()
    out = group.gather_rows(shared.expand(2, 50, 40), idx)
    grad, = torch.autograd.grad(out.float().sum(), shared)
    ref = torch.zeros(50, 40, dtype=torch.float64, device="cuda")
    ref += torch.bincount(idx.reshape(-1), minlength=50)[:, None]
    # small whole numbers: exact in bf16
    assert torch.equal(grad.double(), ref)


def test_gradient_matches_differences():
    from ns_fps_b200 import group
    table, idx = _table(2, 12, 6, torch.float32), _idx((2, 40), 12, lo=-1)
    w, step = _table(2, 40, 6, torch.float32, 3), _table(2, 12, 6, torch.float32, 4)
    leaf = table.clone().requires_grad_()
    grad, = torch.autograd.grad((group.gather_rows(leaf, idx, 1.5) * w).sum(), leaf)
    # the lookup is linear: a difference of any size is exact up to rounding
    ends = [(group.gather_rows(table + s * step, idx, 1.5).double() * w.double()).sum()
            for s in (1.0, -1.0)]
    got = (grad.double() * step.double()).sum()
    terms = (_forward(table.abs() + step.abs(), idx, 1.5) * w.double().abs()).sum()
    assert abs(float((ends[0] - ends[1]) / 2 - got)) <= float(terms) * 64 * 2.0 ** -24


def test_same_bits_again_on_another_stream_and_in_a_graph():
    from ns_fps_b200 import group
    table, idx = _table(3, 700, 72, torch.bfloat16).requires_grad_(), _idx((3, 9000), 700)
    dout = _table(3, 9000, 72, torch.bfloat16, 8)

    def both(leaf):
        out = group.gather_rows(leaf, idx, 0.75)
        return out.detach(), torch.autograd.grad(out, leaf, dout)[0]

    first = both(table)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = both(table.detach().requires_grad_())
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kept = both(table.detach().requires_grad_())
        graphs.append((graph, kept))
    for graph, _ in graphs:
        graph.replay()
    torch.cuda.synchronize()
    for got in (other, graphs[0][1], graphs[1][1]):
        assert torch.equal(first[0], got[0]) and torch.equal(first[1], got[1])


def test_refusals():
    from ns_fps_b200 import group
    table, idx = _table(None, 5, 4, torch.float32), _idx((3,), 5)
    for bad, error in [((table.double(), idx), TypeError), ((table, idx.int()), TypeError),
                       ((table[0], idx), ValueError), ((table[None], idx), ValueError),
                       ((table, idx.cpu()), TypeError), ((table, idx, math.nan), RuntimeError)]:
        with pytest.raises(error):
            group.gather_rows(*bad)


def test_forward_mode_derivatives_are_refused():
    """They are not computed, and no result without a tangent stands for one."""
    from torch.autograd import forward_ad

    from ns_fps_b200 import group
    table = torch.ones(5, 4, device="cuda")
    idx = torch.tensor([1, 3], device="cuda")
    with forward_ad.dual_level():
        for leaf in (False, True):
            dual = forward_ad.make_dual(table.detach().requires_grad_(leaf), table)
            with pytest.raises(RuntimeError, match="forward"):
                group.gather_rows(dual, idx)
        scale = forward_ad.make_dual(torch.tensor(0.5), torch.tensor(1.0))
        with pytest.raises(RuntimeError, match="forward"):
            group.gather_rows(table, idx, scale)
        leaf = table.detach().requires_grad_()
        out = group.gather_rows(leaf, idx)
        dout = forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out))
        with pytest.raises(RuntimeError, match="forward"):
            torch.autograd.grad(out, leaf, dout)
        assert torch.equal(group.gather_rows(table, idx), table[idx])
