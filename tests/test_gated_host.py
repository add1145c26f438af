"""The gated product's checks on the host, without a GPU: refusals before anything is launched."""
from array import array

import pytest
import torch

import superfloat.python_b200.torch as sft
from superfloat.python_b200 import _lib, build
from superfloat.python_b200._errors import SFShapeError, SFTypeError


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


A = 1 << 20                                    # addresses that no launch ever sees
GOOD = dict(dtype=2, bits=8, act=4, M=100, N=60, K=64, x=A, ldx=64, gate=2 * A, up=3 * A, ldg=64, ldu=64, w_dtype=0,
            per_channel=1, codes=4 * A, ldc=64, scale=5 * A, y=6 * A, ldy=64, z=7 * A, ldz=128, work=8 * A, top=9 * A, dz=10 * A,
            dzs=11 * A, ldd=128, dx=12 * A)


def call(fn, **kw):
    c = {**GOOD, **kw}
    words = array("q", [int(c.get(f, 0)) for f in _lib.GATED_CALL])
    return fn(words.buffer_info()[0], None)


@pytest.mark.parametrize("bad", [
    dict(dtype=0), dict(bits=3), dict(bits=9), dict(act=5), dict(act=-1), dict(M=-1), dict(N=0), dict(K=0), dict(codes=0),
    dict(codes=4 * A + 2), dict(ldc=60), dict(ldc=68), dict(scale=0), dict(w_dtype=7), dict(gate=0), dict(up=0), dict(x=0), dict(y=0),
    dict(ldx=63), dict(ldg=63), dict(ldu=63), dict(ldy=59), dict(ldz=127), dict(gate_bias=A, gate_bias_dtype=9),
    dict(up_bias=A, up_bias_dtype=4), dict(per_channel=0, work=0), dict(x=A + 2), dict(ldx=65), dict(x=A + 2, xpad=A, ldp=63),
    dict(x=A + 2, xpad=A + 2, ldp=64), dict(w_dtype=4), dict(w_dtype=4, gate_scale=A), dict(w_dtype=4, codes=0, M=49),
    dict(w_dtype=4, codes=0, M=8)])
def test_forward_refusals(lib, bad):
    assert call(lib.sfb_gated_forward, **bad) == _lib.SFB_EINVAL and lib.sfb_last_error()


@pytest.mark.parametrize("bad", [
    dict(dtype=0), dict(M=0), dict(codes=0), dict(scale=0), dict(y=0), dict(x=0), dict(z=0), dict(z=7 * A + 4), dict(ldz=127),
    dict(ldz=130), dict(ldd=120), dict(ldd=132), dict(x=A + 2), dict(ldx=65), dict(dgate_bias=A, work=0),
    dict(dup_bias=A, up_bias_dtype=7), dict(dgate=A, w_dtype=4), dict(dup=A, dz=0), dict(dzs=0), dict(dzs=11 * A + 2),
    dict(dtype=3, top=0)])
def test_backward_refusals(lib, bad):
    assert call(lib.sfb_gated_backward, **bad) == _lib.SFB_EINVAL and lib.sfb_last_error()


def test_sizes_beyond_the_tiles(lib):
    for kw in (dict(M=1 << 31), dict(N=1 << 30, ldy=1 << 30, ldz=1 << 31, ldd=1 << 31), dict(K=1 << 31, ldx=1 << 31, ldg=1 << 31, ldu=1 << 31, ldc=1 << 31)):
        assert call(lib.sfb_gated_forward, **kw) == call(lib.sfb_gated_backward, **kw) == _lib.SFB_ERANGE
    assert lib.sfb_gated_forward(None, None) == lib.sfb_gated_backward(None, None) == _lib.SFB_EINVAL
    assert lib.sfb_gated_sums(65, 17) == 8 * 2 * 32


def test_python_refusals():
    x, w = torch.zeros(3, 8, dtype=torch.bfloat16), torch.zeros(4, 8)
    p, q = (sft.SFPackedWeight(torch.zeros(4, 8, dtype=torch.int8), torch.ones(4), bits) for bits in (8, 6))
    with pytest.raises(SFShapeError, match="CUDA"):
        sft.tensor_gated(x, w, w)
    with pytest.raises(SFShapeError, match="CUDA"):
        sft.tensor_gated(x, p, p)
    with pytest.raises(SFShapeError, match="shapes"):
        sft.tensor_gated(x, w, w[:3])
    for args in ((p, w), (p, q)):
        with pytest.raises(SFTypeError):
            sft.tensor_gated(x, *args)
