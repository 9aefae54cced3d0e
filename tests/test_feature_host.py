"""Feature operators, host side (no GPU): the C ABI refuses bad arguments
before touching a device, workspaces grow with the work, and the Python entry
points refuse what is not a CUDA tensor."""
import ctypes

import pytest

from tests import capi


def _rows(**kw):
    d = dict(batch=1, rows=4, width=8, count=2, batch_stride=0, row_stride=8, scale=1.0, dtype=0)
    d.update(kw)
    return capi.RowsDesc(**d)


def _select(**kw):
    d = dict(batch=1, points=100, centers=3, block=16, top=4)
    d.update(kw)
    return capi.SelectDesc(**d)


def _attention(**kw):
    d = dict(batch=1, queries=4, keys=64, heads=4, kv_heads=2, head_dim=64, block=16, top=2,
             dtype=2, scale=0.125, reserved=0)
    d.update(kw)
    s = d.pop("stride", 8)
    three = ctypes.c_int64 * 3
    return capi.AttentionDesc(**d, q_stride=three(s, s, s), k_stride=three(s, s, s),
                              v_stride=three(s, s, s))


P = 1 << 20  # a non-null, aligned address that no refused call touches


@pytest.mark.parametrize("bad", [dict(dtype=3), dict(dtype=-1), dict(scale=float("nan")),
                                 dict(scale=float("inf"))])
def test_rows_refuses_arguments(bad):
    with pytest.raises(RuntimeError, match=f"rc={capi.ERR_ARG}"):
        capi.gather_rows_device(_rows(**bad), P, P, P)
    with pytest.raises(RuntimeError, match=f"rc={capi.ERR_ARG}"):
        capi.gather_rows_grad_workspace(_rows(**bad))


@pytest.mark.parametrize("bad", [dict(rows=1 << 31), dict(batch=1 << 16, rows=1 << 16),
                                 dict(batch=1 << 16, count=1 << 16), dict(width=1 << 24),
                                 dict(batch=1 << 63, rows=2)])
def test_rows_refuses_sizes(bad):
    with pytest.raises(RuntimeError, match=f"rc={capi.ERR_UNSUPPORTED}"):
        capi.gather_rows_device(_rows(**bad), P, P, P)


def test_rows_refuses_pointers():
    d = _rows()
    for args in [(0, P, P), (P, 0, P), (P, P, 0), (P + 2, P, P), (P, P + 4, P), (P, P, P + 1)]:
        with pytest.raises(RuntimeError, match=f"rc={capi.ERR_ARG}"):
            capi.gather_rows_device(d, *args)
    need = capi.gather_rows_grad_workspace(d)
    for args in [(0, P, P, P, need), (P, 0, P, P, need), (P, P, 0, P, need), (P, P, P, 0, need),
                 (P, P, P, P + 16, need), (P, P, P, P, need - 1)]:
        with pytest.raises(RuntimeError, match=f"rc={capi.ERR_ARG}"):
            capi.gather_rows_grad_device(d, *args)
    with pytest.raises(RuntimeError, match="strides"):
        capi.gather_rows_device(_rows(row_stride=-8), P, P, P)
    assert capi.lib().nsfps_gather_rows_device(None, None, None, None, None) == capi.ERR_ARG


def test_rows_with_nothing_to_do_touch_no_device():
    capi.gather_rows_device(_rows(count=0), 0, 0, 0)
    capi.gather_rows_device(_rows(batch=0), 0, 0, 0)
    capi.gather_rows_device(_rows(width=0), 0, 0, 0)
    capi.gather_rows_grad_device(_rows(rows=0), 0, 0, 0, 0, 0)


@pytest.mark.parametrize("bad", [dict(block=0), dict(block=48), dict(block=256), dict(top=0),
                                 dict(top=65)])
def test_select_refuses_arguments(bad):
    with pytest.raises(RuntimeError, match=f"rc={capi.ERR_ARG}"):
        capi.select_blocks_workspace(_select(**bad))
    with pytest.raises(RuntimeError, match=f"rc={capi.ERR_ARG}"):
        capi.select_blocks_device(_select(**bad), P, 0, P, P, P, P, 1 << 40)


def test_select_refuses_sizes_and_pointers():
    for bad in [dict(points=1 << 31), dict(batch=1 << 20, centers=1 << 11)]:
        with pytest.raises(RuntimeError, match=f"rc={capi.ERR_UNSUPPORTED}"):
            capi.select_blocks_workspace(_select(**bad))
    d = _select()
    need = capi.select_blocks_workspace(d)
    assert need >= 7 * 6 * 4
    for args in [(0, 0, P, P, P, P, need), (P, 0, 0, P, P, P, need), (P, 0, P, 0, P, P, need),
                 (P, 0, P, P, P, 0, need), (P, 0, P, P, P, P, need - 1),
                 (P, 0, P, P, P, P + 8, need), (P, 2, P, P, P, P, need),
                 (P, 0, P, P + 4, P, P, need)]:
        with pytest.raises(RuntimeError, match=f"rc={capi.ERR_ARG}"):
            capi.select_blocks_device(d, *args)
    capi.select_blocks_device(_select(centers=0), 0, 0, 0, 0, 0, 0, 0)
    capi.select_blocks_device(_select(batch=0), 0, 0, 0, 0, 0, 0, 0)


@pytest.mark.parametrize("bad", [dict(dtype=0), dict(dtype=7), dict(head_dim=0),
                                 dict(head_dim=12), dict(head_dim=136), dict(kv_heads=0),
                                 dict(heads=0), dict(kv_heads=3), dict(heads=512, kv_heads=1),
                                 dict(block=8), dict(top=0), dict(top=65),
                                 dict(scale=float("nan")), dict(stride=4), dict(stride=-8),
                                 dict(reserved=1)])
def test_attention_refuses_arguments(bad):
    with pytest.raises(RuntimeError, match=f"rc={capi.ERR_ARG}"):
        capi.block_attention_workspace(_attention(**bad), False)
    with pytest.raises(RuntimeError, match=f"rc={capi.ERR_ARG}"):
        capi.block_attention_device(_attention(**bad), P, P, P, P, 0, P, P, P, 1 << 40)
    with pytest.raises(RuntimeError, match=f"rc={capi.ERR_ARG}"):
        capi.block_attention_grad_device(_attention(**bad), P, P, P, P, 0, P, P, P, P, P, P, P,
                                         1 << 40)


def test_attention_refuses_sizes_and_pointers():
    for bad in [dict(keys=1 << 30), dict(batch=1 << 10, keys=1 << 20),
                dict(queries=1 << 26, top=16), dict(batch=1 << 40)]:
        with pytest.raises(RuntimeError, match=f"rc={capi.ERR_UNSUPPORTED}"):
            capi.block_attention_workspace(_attention(**bad), False)
    d = _attention()
    need = capi.block_attention_workspace(d, False)
    ok = [P, P, P, P, 0, P, 0, P]  # q, k, v, blocks, lengths, out, lse, work
    for i, value in [(0, 0), (1, 0), (2, 0), (3, 0), (5, 0), (7, 0), (0, P + 8), (1, P + 2),
                     (2, P + 4), (3, P + 4), (4, 2), (5, P + 8), (6, 2), (7, P + 64)]:
        args = list(ok)
        args[i] = value
        with pytest.raises(RuntimeError, match=f"rc={capi.ERR_ARG}"):
            capi.block_attention_device(d, *args, need)
    with pytest.raises(RuntimeError, match=f"rc={capi.ERR_ARG}"):
        capi.block_attention_device(d, *ok, need - 1)
    need = capi.block_attention_workspace(d, True)
    ok = [P, P, P, P, 0, P, P, P, P, P, P, P]  # ..., out, lse, dout, dq, dk, dv, work
    for i in (0, 1, 2, 3, 5, 6, 7, 8, 9, 10, 11):
        args = list(ok)
        args[i] = 0
        with pytest.raises(RuntimeError, match=f"rc={capi.ERR_ARG}"):
            capi.block_attention_grad_device(d, *args, need)
    with pytest.raises(RuntimeError, match=f"rc={capi.ERR_ARG}"):
        capi.block_attention_grad_device(d, *ok, need - 1)
    capi.block_attention_device(_attention(queries=0), 0, 0, 0, 0, 0, 0, 0, 0, 0)
    capi.block_attention_grad_device(_attention(batch=0), *([0] * 12), 0)


def test_workspaces_grow_with_the_work():
    assert (capi.gather_rows_grad_workspace(_rows(count=100_000)) >
            capi.gather_rows_grad_workspace(_rows(count=100)))
    assert (capi.select_blocks_workspace(_select(points=100_000)) >
            capi.select_blocks_workspace(_select()))
    assert (capi.block_attention_workspace(_attention(queries=100_000), True) >
            capi.block_attention_workspace(_attention(), True))


def test_python_entries_refuse_host_tensors():
    torch = pytest.importorskip("torch")
    from ns_fps_b200 import attention, group
    with pytest.raises(TypeError, match="CUDA"):
        group.gather_rows(torch.zeros(3, 4), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(TypeError, match="CUDA"):
        attention.select_blocks(torch.zeros(9, 3), torch.zeros(2, 3), 16, 2)
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(TypeError, match="CUDA"):
        attention.block_attention(x, x, x, torch.zeros(4, 1, dtype=torch.int64), 16)


def test_attention_refuses_a_rest_off_its_alignment():
    d = _attention()
    with pytest.raises(RuntimeError, match=f"rc={capi.ERR_ARG}.*rest"):
        capi.block_attention_device(d, P, P, P, P, 0, P, P, P, 1 << 40, rest=P + 8)
    with pytest.raises(RuntimeError, match=f"rc={capi.ERR_ARG}.*rest"):
        capi.block_attention_grad_device(d, P, P, P, P, 0, P, P, P, P, P, P, P, 1 << 40,
                                         rest=P + 2)


def test_python_entries_refuse_a_scale_that_wants_a_gradient():
    torch = pytest.importorskip("torch")
    from ns_fps_b200 import attention, group
    scale = torch.tensor(0.5, requires_grad=True)
    x, idx = torch.zeros(4, 2, 64, dtype=torch.bfloat16), torch.zeros(4, 1, dtype=torch.int64)
    with pytest.raises(TypeError, match="scale.*gradient"):
        attention.block_attention(x, x, x, idx, 16, scale=scale)
    with pytest.raises(TypeError, match="scale.*gradient"):
        group.gather_rows(x[:, 0], idx, scale)
    with torch.no_grad(), pytest.raises(TypeError, match="CUDA"):  # a number then
        attention.block_attention(x, x, x, idx, 16, scale=scale)


@pytest.mark.parametrize("scale", [3e38, -3e38])
def test_attention_refuses_a_scale_beyond_base_two(scale):
    """Scores are taken in base 2: scale * log2(e) has to be finite, too."""
    for backward in (False, True):
        with pytest.raises(RuntimeError, match=f"rc={capi.ERR_ARG}.*scale"):
            capi.block_attention_workspace(_attention(scale=scale), backward)
        capi.block_attention_workspace(_attention(scale=scale / 2), backward)
