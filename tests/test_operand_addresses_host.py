"""Operands that do not start on an element are refused before anything is launched: norm, distillation, gated product."""
import pytest

import test_gated_host as gated
import test_norm_distill_host as host
from superfloat.python_b200 import _lib
from test_norm_distill_host import A, lib  # noqa: F401

F32, BF16, F16, I8 = 0, 2, 3, 4


@pytest.mark.parametrize("bad", [
    dict(x=A + 1), dict(y=2 * A + 1), dict(stats=3 * A + 4), dict(dtype=F32, x=A + 2), dict(w=A + 2, w_dtype=F32), dict(w=A + 1, w_dtype=F16),
    dict(b=A + 1, b_dtype=BF16), dict(b=A + 2, b_dtype=F32)])
def test_norm(lib, bad):  # noqa: F811
    for fn in (lib.sfb_norm_forward, lib.sfb_norm_backward):
        assert host.call(fn, _lib.NORM_CALL, host.NORM, bad) == _lib.SFB_EINVAL and lib.sfb_last_error()
    for more in (dict(dx=A + 1), dict(dw=A + 2, w_dtype=F32), dict(db=A + 1, b_dtype=F16)):
        assert host.call(lib.sfb_norm_backward, _lib.NORM_CALL, host.NORM, more) == _lib.SFB_EINVAL


@pytest.mark.parametrize("bad", [
    dict(teacher=2 * A + 2), dict(teacher=2 * A + 1, t_dtype=BF16), dict(index=3 * A + 4), dict(index=3 * A + 2, i_long=0),
    dict(weight=A + 2, w_dtype=F32), dict(weight=A + 1, w_dtype=F16), dict(loss=4 * A + 2), dict(rows=5 * A + 2), dict(parts=6 * A + 1),
    dict(stats=7 * A + 2), dict(weights=11 * A + 2)])
def test_distillation_forward(lib, bad):  # noqa: F811
    assert host.call(lib.sfb_distill_forward, _lib.DISTILL_CALL, host.DISTILL, bad) == _lib.SFB_EINVAL and lib.sfb_last_error()


def test_distillation_backward(lib):  # noqa: F811
    for bad in (dict(upstream=9 * A + 2), dict(stats=7 * A + 1)):
        assert host.call(lib.sfb_distill_backward, _lib.DISTILL_CALL, host.DISTILL, bad) == _lib.SFB_EINVAL


@pytest.mark.parametrize("bad", [
    dict(y=6 * A + 1), dict(gate=2 * A + 2), dict(up=3 * A + 1, w_dtype=BF16), dict(gate_bias=A + 2), dict(up_bias=A + 1, up_bias_dtype=F16),
    dict(scale=5 * A + 2), dict(z=7 * A + 2), dict(w_dtype=I8, gate_scale=A + 2, up_scale=A), dict(w_dtype=I8, gate_scale=A, up_scale=A + 1),
    dict(per_channel=0, work=8 * A + 2), dict(x=A + 1, xpad=A, ldp=64)])
def test_gated_forward(lib, bad):  # noqa: F811
    assert gated.call(lib.sfb_gated_forward, **bad) == _lib.SFB_EINVAL and lib.sfb_last_error()


@pytest.mark.parametrize("bad", [
    dict(dx=12 * A + 1), dict(dgate=A + 2), dict(dup=A + 1, w_dtype=F16), dict(dgate_bias=A + 2), dict(dup_bias=A + 1, up_bias_dtype=BF16),
    dict(dtype=F16, top=9 * A + 2), dict(dgate_bias=A, work=8 * A + 2)])
def test_gated_backward(lib, bad):  # noqa: F811
    assert gated.call(lib.sfb_gated_backward, **bad) == _lib.SFB_EINVAL and lib.sfb_last_error()
