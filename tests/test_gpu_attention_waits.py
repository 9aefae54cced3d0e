"""Waits of the attention kernels that run out, driven without faulting the GPU.

One CTA issues a product and does not announce it (a commit that nothing else
makes), so every wait for it in that CTA gives up after 0.2 s.  The calls do not
wait for their kernels and return as ever; what could be wrong must then be
NaN, nothing may hang, and the next call must give the bits it always gave."""
import pytest

from tests import capi

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

WAIT_NS = 200_000_000


@pytest.fixture(autouse=True)
def _reset_hooks():
    capi.set_test_hooks(reset=True)
    yield
    capi.set_test_hooks(reset=True)


def _call(D, dtype, M=1500, N=5000):
    """One cloud in both directions, on tiles: (inputs, forward, gradient)."""
    from ns_fps_b200 import attention
    g = torch.Generator(device="cuda").manual_seed(5)
    q, k, v, dout = (torch.randn(1, n, 2, D, device="cuda", generator=g).to(dtype)
                     for n in (M, N, N, M))
    blocks = torch.rand(1, M, N // 16, device="cuda", generator=g).argsort(2)[..., :64]
    blocks[:, ::50] = -1  # some queries without a key

    def forward():
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        return attention.block_attention(*leaves, blocks, 16), leaves

    def gradient(out, leaves):
        return torch.autograd.grad(out, leaves, dout, retain_graph=True)

    return forward, gradient


def _same(xs, ys):
    return all(torch.equal(x, y) for x, y in zip(xs, ys))


@pytest.mark.parametrize("D,dtype", [(64, torch.bfloat16), (128, torch.float16)])
def test_forward(D, dtype):
    forward, gradient = _call(D, dtype)
    out, leaves = forward()
    grads = gradient(out, leaves)
    assert bool(torch.isfinite(out).all())
    capi.set_test_hooks(wait_limit_ns=WAIT_NS, withhold_cta=3, withhold_step=0)
    got, _ = forward()
    torch.cuda.synchronize()
    capi.set_test_hooks(reset=True)
    assert bool(torch.isnan(got).all())
    again, leaves = forward()
    assert _same([again, *gradient(again, leaves)], [out, *grads])


@pytest.mark.parametrize("step", [0, 1])
@pytest.mark.parametrize("M", [400, 1500])  # spans of keys of one CTA each; shared ones
@pytest.mark.parametrize("D,dtype", [(64, torch.bfloat16), (64, torch.float16),
                                     (128, torch.bfloat16)])
def test_gradient(D, dtype, M, step):
    forward, gradient = _call(D, dtype, M)
    out, leaves = forward()
    grads = gradient(out, leaves)
    assert all(bool(torch.isfinite(t).all()) for t in grads)
    capi.set_test_hooks(wait_limit_ns=WAIT_NS, withhold_cta=2, withhold_step=step)
    dq, dk, dv = gradient(out, leaves)
    torch.cuda.synchronize()
    capi.set_test_hooks(reset=True)
    assert bool(torch.isnan(dq).all())
    for got, right in ((dk, grads[1]), (dv, grads[2])):
        gone = torch.isnan(got)
        assert bool(gone.any()) and torch.equal(got[~gone], right[~gone])
        assert M > 400 or not bool(gone.all())
    assert _same(gradient(out, leaves), grads)


def test_a_cta_that_the_grid_does_not_have_changes_nothing():
    forward, gradient = _call(64, torch.bfloat16)
    out, leaves = forward()
    grads = gradient(out, leaves)
    capi.set_test_hooks(wait_limit_ns=WAIT_NS, withhold_cta=1_000_000)
    again, leaves = forward()
    assert _same([again, *gradient(again, leaves)], [out, *grads])
