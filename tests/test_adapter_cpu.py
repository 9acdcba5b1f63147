"""The learned adapter's and the clipping's argument checks: every refusal comes before any device
work, so they run without a GPU (addresses are made up and never followed)."""
import math

import pytest

import xvec_b200 as xb

A = 1 << 20  # a made-up address; regions below are 1 MiB apart


def at(i):
    return A * (i + 1)


def refuse(call, text):
    with pytest.raises(xb.XvecGPUError) as e:
        call()
    assert e.value.status == xb.INVALID_ARGUMENT and text in str(e.value), str(e.value)


def linear(**kw):
    a = dict(device=0, storage=1, n=4, in_dim=16, out_dim=8, x_ptr=at(0), weight_ptr=at(1), y_ptr=at(2))
    a.update(kw)
    return lambda: xb.linear_device(**a)


def gated(**kw):
    a = dict(device=0, storage=1, n=4, in_dim=16, out_dim=8, x_ptr=at(0), gate_weight_ptr=at(1),
             up_weight_ptr=at(2), h_ptr=at(3))
    a.update(kw)
    return lambda: xb.gated_device(**a)


def linear_backward(**kw):
    a = dict(device=0, storage=1, n=4, in_dim=16, out_dim=8, dy_ptr=at(0), x_ptr=at(1),
             weight_ptr=at(2), dx_ptr=at(3), dw_ptr=at(4), db_ptr=at(5))
    a.update(kw)
    return lambda: xb.linear_backward_device(**a)


def gated_backward(**kw):
    a = dict(device=0, storage=1, n=4, in_dim=16, out_dim=8, dh_ptr=at(0), x_ptr=at(1),
             gate_weight_ptr=at(2), up_weight_ptr=at(3), gate_ptr=at(4), up_ptr=at(5), dx_ptr=at(6),
             dgate_weight_ptr=at(7), dup_weight_ptr=at(8), dgate_bias_ptr=at(9), dup_bias_ptr=at(10))
    a.update(kw)
    return lambda: xb.gated_backward_device(**a)


@pytest.mark.parametrize("call", [linear, gated, linear_backward, gated_backward])
def test_shapes_and_types(call):
    for storage in (0, 4, -1):
        refuse(call(storage=storage), "storage")
    for activation in (-1, 4):
        refuse(call(activation=activation), "activation")
    for dim in (0, -3, (1 << 20) + 1):
        refuse(call(in_dim=dim), "dimensions")
        refuse(call(out_dim=dim), "dimensions")
    for n in (-1, 2 ** 31 - 1, 2 ** 40):
        refuse(call(n=n), "row count")
    refuse(call(ldx=15), "leading dimension")
    refuse(call(ldw=3), "leading dimension")
    refuse(call(ldx=-16), "leading dimension")
    refuse(call(ldx=(1 << 27) + 1), "too large")


def test_missing_operands():
    for name in ("x_ptr", "weight_ptr", "y_ptr"):
        refuse(linear(**{name: 0}), "required")
    for name in ("x_ptr", "gate_weight_ptr", "up_weight_ptr", "h_ptr"):
        refuse(gated(**{name: 0}), "required")
    refuse(gated(gate_ptr=at(5)), "together")
    refuse(gated(up_ptr=at(5)), "together")
    refuse(linear_backward(dy_ptr=0), "required")
    refuse(linear_backward(weight_ptr=0), "needs weight")
    refuse(linear_backward(x_ptr=0), "needs x")
    refuse(linear_backward(activation=xb.ACT_GELU), "needs preact")
    for name in ("dh_ptr", "gate_ptr", "up_ptr"):
        refuse(gated_backward(**{name: 0}), "required")
    refuse(gated_backward(up_weight_ptr=0), "both weights")
    refuse(gated_backward(x_ptr=0), "need x")


def test_alignment():
    refuse(linear(x_ptr=at(0) + 2), "aligned")
    refuse(linear(storage=2, bias_ptr=at(5) + 1), "aligned")
    refuse(linear_backward(db_ptr=at(5) + 1), "aligned")
    refuse(gated(h_ptr=at(3) + 3), "aligned")
    refuse(gated_backward(dup_weight_ptr=at(8) + 2), "aligned")


def test_overlaps():
    refuse(linear(y_ptr=at(0)), "y overlaps x")
    refuse(linear(y_ptr=at(1) + 4 * 16), "y overlaps weight")
    refuse(linear(bias_ptr=at(2) + 4 * 31), "y overlaps bias")
    refuse(linear(preact_ptr=at(2)), "y overlaps preact")
    # y may be the residual itself, with the same rows only.
    refuse(linear(residual_ptr=at(2), ldr=16), "y overlaps residual")
    refuse(linear(residual_ptr=at(2) + 4), "y overlaps residual")
    refuse(linear(residual_ptr=at(5), preact_ptr=at(5)), "preact overlaps residual")
    # Columns of one wider matrix: disjoint ones pass (and then find no device here or work),
    # overlapping ones do not.
    wide = dict(ldx=32, ldy=32, x_ptr=at(0))
    refuse(linear(y_ptr=at(0) + 4 * 15, **wide), "y overlaps x")
    refuse(linear(y_ptr=at(0) + 4 * 25, **wide), "y overlaps x")  # wraps into the next row
    refuse(gated(h_ptr=at(2)), "h overlaps up_weight")
    refuse(gated(gate_ptr=at(6), up_ptr=at(6) + 4 * 8), "gate overlaps up")
    refuse(linear_backward(dx_ptr=at(1)), "dx overlaps x")
    refuse(linear_backward(dw_ptr=at(2)), "dweight overlaps weight")
    refuse(linear_backward(db_ptr=at(4)), "dweight overlaps dbias")
    refuse(gated_backward(dup_weight_ptr=at(7)), "dgate_weight overlaps dup_weight")
    refuse(gated_backward(dx_ptr=at(0)), "dx overlaps dh")


def test_interleaved_columns_pass_the_checks():
    """x and y as disjoint columns of one matrix, and an output that is its residual, are no
    overlaps: without a device the call then says so."""
    if xb.device_count() > 0:
        pytest.skip("a device is visible: the made-up addresses would be followed")
    for call in (linear(y_ptr=at(0) + 4 * 16, ldx=32, ldy=32), linear(residual_ptr=at(2)),
                 linear(), gated(), linear_backward(), gated_backward(),
                 linear_backward(n=0, dy_ptr=0, x_ptr=0)):
        with pytest.raises(xb.XvecGPUError) as e:
            call()
        assert e.value.status == xb.UNSUPPORTED


def test_nothing_to_do_needs_no_device():
    linear(n=0, x_ptr=0, y_ptr=0)()
    gated(n=0, x_ptr=0, h_ptr=0)()


def test_nil_arguments():
    lib = xb.library()
    for name in ("linear", "linear_backward", "gated", "gated_backward"):
        assert getattr(lib, f"xvec_gpu_{name}_device")(None) == xb.INVALID_ARGUMENT
    args = xb.LinearArgs(0, 1, 0, 16, 8, 7, 4, at(0), at(1), 0, 0, at(2))
    import ctypes
    assert lib.xvec_gpu_linear_device(ctypes.byref(args)) == xb.INVALID_ARGUMENT
    assert "reserved" in xb.last_error()


def clip(tensors, max_norm=1.0, norm_ptr=at(50)):
    return lambda: xb.clip_gradients_device(0, tensors, max_norm, norm_ptr)


def test_clip_refusals():
    ok = (1, at(0), at(0), 100)
    refuse(clip([ok], max_norm=-1.0), "max_norm")
    refuse(clip([ok], max_norm=math.nan), "max_norm")
    refuse(clip([ok], norm_ptr=0), "norm")
    refuse(clip([ok], norm_ptr=at(50) + 2), "norm")
    refuse(clip([(0, at(0), at(0), 1)]), "storage")
    refuse(clip([(4, at(0), at(0), 1)]), "storage")
    refuse(clip([(1, at(0), at(0), -1)]), "count")
    refuse(clip([(1, at(0), at(0), (1 << 40) + 1)]), "count")
    refuse(clip([(1, 0, at(0), 1)]), "nil")
    refuse(clip([(1, at(0), 0, 1)]), "nil")
    refuse(clip([(1, at(0) + 2, at(1), 1)]), "aligned")
    refuse(clip([(2, at(0), at(1) + 1, 1)]), "aligned")


def test_clip_overlaps():
    refuse(clip([(1, at(0), at(0), 100), (1, at(0), at(0), 100)]), "overlaps")  # the same twice
    refuse(clip([(1, at(0), at(1), 100), (1, at(1) + 396, at(2), 4)]), "overlaps")
    refuse(clip([(1, at(0), at(0) + 4, 100)]), "overlaps")
    refuse(clip([(1, at(0), at(0), 100), (1, at(3), at(0) + 396, 1)]), "overlaps")
    refuse(clip([(1, at(0), at(0), 100)], norm_ptr=at(0) + 396), "overlaps")
    refuse(clip([(1, at(0), at(1), 100)], norm_ptr=at(1)), "overlaps")
    if xb.device_count() == 0:
        for tensors in ([], [(1, at(0), at(0), 100), (1, at(0) + 400, at(0) + 400, 100)],
                        [(1, at(0), at(1), 100), (1, at(0), at(2), 100)], [(1, 0, 0, 0)]):
            with pytest.raises(xb.XvecGPUError) as e:
                clip(tensors)()
            assert e.value.status == xb.UNSUPPORTED
