"""The tensor-core linear's checks on the host, without a GPU: refusals before
anything is launched, configuration and conversion, and the call struct."""
import re

import os
import pytest
import torch
import torch.nn as nn

import superfloat.python_b200.torch as sft
from array import array
from conftest import REPO
from superfloat.python_b200 import _lib, build
from superfloat.python_b200._errors import SFShapeError, SFTypeError, SFUnsupportedError


def test_the_call_struct_is_the_headers():
    """Python fills sfb_tensor_call as an array of 8-byte words: the header's fields in the header's order."""
    text = open(os.path.join(REPO, "include", "sfb200.h")).read()
    body = re.sub(r"/\*.*?\*/", "", re.search(r"typedef struct sfb_tensor_call \{(.*?)\}", text, re.S)[1], flags=re.S)
    names = []
    for decl in filter(None, (d.strip() for d in body.split(";"))):
        assert decl.startswith("int64_t ") or "*" in decl, decl
        names += [re.sub(r"[\s*]", "", d.split()[-1]) for d in decl.split(",")]
    assert tuple(names) == _lib.TENSOR_CALL


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


A = 1 << 20                                    # addresses that no launch ever sees
GOOD = dict(dtype=2, bits=8, act=0, M=100, N=64, K=64, x=A, ldx=64, w=2 * A, ldw=64, w_dtype=0, per_channel=1,
            codes=3 * A, ldc=64, scale=4 * A, y=5 * A, ldy=64, z=6 * A, ldz=64, ldd=64, dz=7 * A, dzs=8 * A, dx=9 * A,
            work=10 * A, top=11 * A)


def call(fn, **kw):
    c = {**GOOD, **kw}
    words = array("q", [int(c.get(f, 0)) for f in _lib.TENSOR_CALL])
    return fn(words.buffer_info()[0], None)


@pytest.mark.parametrize("bad", [
    dict(dtype=0), dict(bits=3), dict(bits=9), dict(act=5), dict(act=-1), dict(M=-1), dict(N=0), dict(K=0),
    dict(codes=0), dict(codes=3 * A + 2), dict(ldc=60), dict(ldc=68), dict(scale=0), dict(w_dtype=7), dict(w=0),
    dict(x=0), dict(y=0), dict(ldx=63), dict(ldw=63), dict(ldy=63), dict(ldz=63), dict(bias=A, bias_dtype=9),
    dict(residual=A, ldr=63), dict(per_channel=0, work=0), dict(x=A + 2), dict(ldx=65), dict(x=A + 2, xpad=A, ldp=63),
    dict(x=A + 2, xpad=A + 2, ldp=64), dict(w_dtype=4, codes=0, M=49), dict(w_dtype=4, codes=0, M=8)])
def test_forward_refusals(lib, bad):
    assert call(lib.sfb_tensor_forward, **bad) == _lib.SFB_EINVAL and lib.sfb_last_error()


@pytest.mark.parametrize("bad", [
    dict(dtype=0), dict(M=0), dict(codes=0), dict(scale=0), dict(y=0), dict(x=0), dict(act=2, z=0), dict(ldd=60),
    dict(ldd=68), dict(x=A + 2), dict(ldx=65), dict(db=A, db_dtype=0, work=0), dict(db=A, db_dtype=7),
    dict(dw=A, w_dtype=4), dict(dzs=0), dict(dzs=8 * A + 2), dict(act=2, dw=A, dz=0), dict(dtype=3, top=0)])
def test_backward_refusals(lib, bad):
    assert call(lib.sfb_tensor_backward, **bad) == _lib.SFB_EINVAL and lib.sfb_last_error()


def test_sizes_beyond_the_tiles(lib):
    for kw in (dict(M=1 << 31), dict(N=1 << 31), dict(K=1 << 31, ldx=1 << 31, ldw=1 << 31, ldc=1 << 31),
               dict(M=(1 << 31) - 1024, N=1 << 20)):
        assert call(lib.sfb_tensor_forward, **kw) == _lib.SFB_ERANGE
    assert lib.sfb_tensor_forward(None, None) == _lib.SFB_EINVAL
    assert lib.sfb_tensor_backward(None, None) == _lib.SFB_EINVAL
    assert lib.sfb_tensor_failures(None) == _lib.SFB_EINVAL
    assert lib.sfb_code_quantize(None, 0, 4, 4, 4, 9, 1, None, 4, None, None, None) == _lib.SFB_EINVAL
    assert lib.sfb_code_quantize(None, 1, 4, 4, 4, 8, 1, None, 4, None, None, None) == _lib.SFB_EINVAL
    assert lib.sfb_code_quantize(None, 0, 4, 4, 3, 8, 1, None, 4, None, None, None) == _lib.SFB_EINVAL
    assert lib.sfb_code_quantize(None, 0, 4, 4, 4, 8, 1, None, 4, None, None, None) == _lib.SFB_EINVAL
    assert lib.sfb_code_quantize(None, 0, 0, 4, 4, 8, 1, None, 4, None, None, None) == _lib.SFB_OK


def test_python_refusals():
    x, w = torch.zeros(3, 8, dtype=torch.bfloat16), torch.zeros(4, 8)
    with pytest.raises(SFShapeError, match="CUDA"):
        sft.tensor_linear(x, w)
    with pytest.raises(SFShapeError, match="CUDA"):
        sft.pack_weight(w)
    for bits in (9, 16):
        with pytest.raises(SFUnsupportedError):
            sft.tensor_linear(x, w, dtype=f"sf{bits}")
    with pytest.raises(SFTypeError):
        sft.SFPackedWeight(w, torch.zeros(4))
    p = sft.SFPackedWeight(torch.zeros(4, 8, dtype=torch.int8), torch.ones(4), 8)
    with pytest.raises(SFShapeError, match="CUDA"):
        sft.tensor_linear(x, p)
    with pytest.raises(SFTypeError, match="float32"):
        sft.tensor_linear(x.float(), p)


def test_configuration():
    assert "accumulate=tensor" in sft.SFConfig(8, "per_channel", accumulate="tensor").describe()
    for bits in (9, 16):
        with pytest.raises(SFUnsupportedError, match="sf4..sf8"):
            sft.SFConfig(bits, accumulate="tensor")
    with pytest.raises(ValueError, match="shift"):
        sft.SFConfig(8, accumulate="tensor", shift=1)
    with pytest.raises(ValueError, match="accumulate"):
        sft.SFConfig(8, accumulate="tensors")
    with pytest.raises(SFUnsupportedError, match="linear layers"):
        sft.matmul(torch.zeros(2, 2), torch.zeros(2, 2), dtype="sf8", accumulate="tensor")


def test_conversion():
    net = nn.Sequential(nn.Embedding(32, 16), nn.Linear(16, 24), nn.GELU(), nn.Linear(24, 32))
    m = sft.convert(net, dtype="sf6", accumulate="tensor", scale="per_channel", widths={"3": "sf8"})
    assert [type(c).__name__ for c in m] == ["Embedding", "SFLinear", "GELU", "SFLinear"]
    assert m[1].sf.accumulate == "tensor" and m[1].sf.bits == 6 and m[3].sf.bits == 8
    assert not sft.conversion_report(m).kept_sf16          # the head (a vocabulary of 32) is converted too
    with pytest.raises(ValueError, match="keep_sf16"):
        sft.convert(net, dtype="sf8", accumulate="tensor", keep_sf16=["1"])
    with pytest.raises(SFUnsupportedError):
        sft.convert(net, dtype="sf16", accumulate="tensor")
    chain = sft.convert(net, dtype="sf8")
    assert sft.pack(chain)[1].__class__.__name__ == "SFLinear"     # other modes are left alone
