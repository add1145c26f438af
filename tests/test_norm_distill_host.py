"""Layer norm's and the distillation loss's checks on the host, without a GPU: refusals before anything is launched, and
the call structs."""
import math
import os
import re
from array import array

import pytest
import torch

import superfloat.python_b200.torch as sft
from conftest import REPO
from superfloat.python_b200 import _lib, build
from superfloat.python_b200._errors import SFShapeError
from superfloat.python_b200.torch._distill import _like, _strides_of, _two_strides


@pytest.mark.parametrize("name,fields", [("norm", _lib.NORM_CALL), ("distill", _lib.DISTILL_CALL), ("gated", _lib.GATED_CALL)])
def test_the_call_structs_are_the_headers(name, fields):
    """Python fills the structs as arrays of 8-byte words: the header's fields in the header's order, none shorter."""
    text = open(os.path.join(REPO, "include", "sfb200.h")).read()
    body = re.sub(r"/\*.*?\*/", "", re.search(r"typedef struct sfb_%s_call \{(.*?)\}" % name, text, re.S)[1], flags=re.S)
    names = []
    for decl in filter(None, (d.strip() for d in body.split(";"))):
        assert decl.startswith(("int64_t ", "double ")) or "*" in decl, decl
        names += [re.sub(r"[\s*]", "", d.split()[-1]) for d in decl.split(",")]
    assert tuple(names) == fields


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


A = 1 << 20                                    # addresses that no launch ever sees
NORM = dict(dtype=2, M=10, D=64, x=A, ldx=64, y=2 * A, ldy=64, eps=_lib.bits_of(1e-5), stats=3 * A, dx=4 * A, lddx=64, work=5 * A)
DISTILL = dict(dtype=2, M=10, V=64, logits=A, inner=10, si=64, K=4, teacher=2 * A, ldt=4, index=3 * A, i_long=1, ldi=4,
               w_dtype=-2, reduction=2, temperature=_lib.bits_of(1.0), loss=4 * A, rows=5 * A, parts=6 * A, stats=7 * A, block=10 * A, weights=11 * A,
               grad=8 * A, gi=64, upstream=9 * A)


def call(fn, fields, good, kw):
    c = {**good, **kw}
    words = array("q", [int(c.get(f, 0)) for f in fields])
    return fn(words.buffer_info()[0], None)


@pytest.mark.parametrize("bad", [
    dict(dtype=4), dict(dtype=7), dict(M=-1), dict(D=0), dict(x=0), dict(y=0), dict(ldx=63), dict(ldy=63), dict(w=A, w_dtype=9),
    dict(b=A, b_dtype=4), dict(eps=_lib.bits_of(-1.0)), dict(eps=_lib.bits_of(math.nan))])
def test_norm_forward_refusals(lib, bad):
    assert call(lib.sfb_norm_forward, _lib.NORM_CALL, NORM, bad) == _lib.SFB_EINVAL and lib.sfb_last_error()


@pytest.mark.parametrize("bad", [
    dict(dtype=4), dict(M=0), dict(D=0), dict(x=0), dict(y=0), dict(stats=0), dict(stats=A + 4), dict(lddx=63), dict(dw=A, work=0),
    dict(db=A, work=5 * A + 8), dict(dw=A, w_dtype=9), dict(db=A, b_dtype=4)])
def test_norm_backward_refusals(lib, bad):
    assert call(lib.sfb_norm_backward, _lib.NORM_CALL, NORM, bad) == _lib.SFB_EINVAL and lib.sfb_last_error()


@pytest.mark.parametrize("bad", [
    dict(dtype=4), dict(t_dtype=4), dict(w_dtype=4), dict(M=-1), dict(V=0), dict(K=-1), dict(inner=0), dict(ldt=3), dict(ldi=3),
    dict(temperature=0), dict(temperature=_lib.bits_of(math.nan)), dict(temperature=_lib.bits_of(1e7)), dict(reduction=3),
    dict(reduction=-1), dict(logits=0), dict(so=-1), dict(gi=-8), dict(logits=A + 1), dict(grad=8 * A + 1)])
def test_distill_refusals(lib, bad):
    for fn in (lib.sfb_distill_forward, lib.sfb_distill_backward):
        assert call(fn, _lib.DISTILL_CALL, DISTILL, bad) == _lib.SFB_EINVAL and lib.sfb_last_error()


def test_more_refusals(lib):
    forward, backward, fields = lib.sfb_distill_forward, lib.sfb_distill_backward, _lib.DISTILL_CALL
    for bad in (dict(loss=0), dict(rows=0), dict(parts=0), dict(weights=0), dict(block=0), dict(teacher=0), dict(index=0), dict(w_dtype=0)):
        assert call(forward, fields, DISTILL, bad) == _lib.SFB_EINVAL
    for bad in (dict(grad=0), dict(stats=0), dict(block=0), dict(block=A + 4), dict(upstream=0)):
        assert call(backward, fields, DISTILL, bad) == _lib.SFB_EINVAL
    for bad in (dict(K=1025, ldt=1025, ldi=1025), dict(V=1 << 31)):
        assert call(forward, fields, DISTILL, bad) == call(backward, fields, DISTILL, bad) == _lib.SFB_ERANGE
    assert call(lib.sfb_norm_forward, _lib.NORM_CALL, NORM, dict(D=65537, ldx=65537, ldy=65537)) == _lib.SFB_ERANGE
    for fn in (forward, backward, lib.sfb_norm_forward, lib.sfb_norm_backward):
        assert fn(None, None) == _lib.SFB_EINVAL
    # nothing to do
    assert call(lib.sfb_norm_forward, _lib.NORM_CALL, NORM, dict(M=0, x=0, y=0)) == _lib.SFB_OK
    assert call(backward, fields, DISTILL, dict(M=0)) == _lib.SFB_OK
    assert lib.sfb_distill_failures(None) == lib.sfb_norm_failures(None) == _lib.SFB_EINVAL
    assert lib.sfb_distill_parts(0) == 0 and lib.sfb_distill_parts(9) == 2
    assert lib.sfb_norm_work(0, 0) == 0 and lib.sfb_norm_work(5, 65537) == 0


def test_python_refusals():
    x = torch.zeros(3, 8)
    with pytest.raises(SFShapeError, match="CUDA"):
        sft.layer_norm(x)
    with pytest.raises(SFShapeError, match="CUDA"):
        sft.distill_loss(x, x[:, :2], torch.zeros(3, 2, dtype=torch.int64))


def test_rows_as_two_runs():
    """(rows of the inner run, outer stride, inner stride) reach the rows in their order, without a copy where two runs are enough."""
    x = torch.arange(4 * 10 * 17 * 3).view(4, 10, 3, 17)
    views = [x, x[:, :-1], x[..., :5], x[0, 0], x[0, 0, 0], x.transpose(0, 1), x[:, :, 1], x[:, ::2, 0], x[:0], x[:1, :1].expand(3, 5, 3, 17),
             x.transpose(1, 3), x[..., :1], x[:, :-1, :, 2:9], x[1:, :, :-1]]
    copies = 0
    for v in views:
        t, inner, so, si = _two_strides(v)
        copies += t.data_ptr() != v.data_ptr()
        rows = t.reshape(-1, v.shape[-1])
        base = torch.as_strided(t, (x.numel(),), (1,), 0) if t.data_ptr() == v.data_ptr() else t.reshape(-1)
        at = t.storage_offset() if t.data_ptr() == v.data_ptr() else 0
        for r in range(rows.shape[0]):
            start = at + r // inner * so + r % inner * si
            assert int(base[start]) == int(rows[r, 0])
        g = _like(t)
        assert g.shape == t.shape
        go, gi = _strides_of(g, t)
        places = [r // inner * go + r % inner * gi for r in range(rows.shape[0])]
        want = [g.stride() and sum(int(i) * s for i, s in zip(torch.unravel_index(torch.tensor(r), t.shape[:-1]), g.stride()))
                for r in range(rows.shape[0])]
        assert places == want and len(set(places)) == len(places)
    assert copies == 2                             # transposed columns, and three runs of rows
