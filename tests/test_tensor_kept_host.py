"""What the tensor-core linear's backward pass reads of what the forward pass
kept, where saved-tensor hooks (activation offloading) hand it back in another
layout.  Without a GPU: the library's calls are recorded instead of made, and
each address that one names is compared with the memory of the tensors.
"""
import ctypes

import pytest
import torch

from superfloat.python_b200 import _lib
from superfloat.python_b200._errors import SFShapeError, SFTypeError
from superfloat.python_b200.torch import _tensor


@pytest.fixture
def calls(monkeypatch):
    made = {}
    monkeypatch.setattr(_lib, "tensor_forward", lambda index, call: made.update(forward=dict(zip(_lib.TENSOR_CALL, call))))
    monkeypatch.setattr(_lib, "tensor_backward",
                        lambda index, call: made.update(backward=dict(zip(_lib.TENSOR_CALL, call))))
    monkeypatch.setattr(_lib, "tensor_sums", lambda M, N: 4 * -(-M // 64) * N)
    return made


class Relaid(torch.autograd.graph.saved_tensors_hooks):
    """Keeps each tensor as `how` lays it out; `back` is what was handed back."""

    def __init__(self, how):
        self.back = []

        def unpack(t):
            self.back.append(t)
            return t
        super().__init__(how, unpack)


def compact(t):
    return torch.empty(t.shape, dtype=t.dtype).copy_(t)


def odd(t):
    """The same values at an odd element of a wider buffer."""
    wide = torch.empty(*t.shape[:-1], t.shape[-1] + 3, dtype=t.dtype)[..., 1:1 + t.shape[-1]]
    return wide.copy_(t)


def turned(t):
    return compact(t.t()).t() if t.dim() == 2 else compact(t)


def inside(first, elements, size, tensors):
    """Whether so many elements of `size` bytes from address `first` on are within one of the tensors' memory."""
    for t in tensors:
        if t is not None:
            s = t.untyped_storage()
            if s.data_ptr() <= first and first + elements * size <= s.data_ptr() + s.nbytes():
                return True
    return False


def values(first, ld, M, K, like):
    """What lies at an address, as M rows of K, ld apart."""
    out = torch.empty(M, K, dtype=like)
    for m in range(M):
        ctypes.memmove(out.data_ptr() + m * K * 2, first + m * ld * 2, K * 2)
    return out


@pytest.mark.parametrize("how", [compact, odd, turned])
@pytest.mark.parametrize("M,K,wide", [(40, 64, 192), (40, 64, 64), (33, 40, 48), (40, 13, 16), (40, 13, 13), (1, 24, 96),
                                      (1, 13, 40), (5, 1, 8)])
def test_x_in_another_layout(calls, how, M, K, wide):
    """x is a slice of a wider buffer (a fused projection's, say) whose rows start on 16 bytes where `wide` allows."""
    g = torch.Generator().manual_seed(M + K)
    x = torch.randn(M, wide, generator=g).bfloat16()[:, :K]
    w, b = torch.randn(24, K, generator=g).requires_grad_(), torch.randn(24, generator=g).requires_grad_()
    hooks = Relaid(how)
    with hooks:
        y = _tensor._TensorLinear.apply(x, w, None, b, None, 8, "per_channel", _lib.ACTIVATIONS["gelu"])
    made, seen = [], {}
    rows, dense, clone, record = _tensor._rows_on16, torch.Tensor.contiguous, torch.Tensor.clone, _lib.tensor_backward

    def noted(fn, pick):                                # the copies that the pass makes itself
        def call(*args):
            out = fn(*args)
            made.append(pick(out))
            return out
        return call

    def look(index, call):                              # while the copies live
        record(index, call)
        c, known = calls["backward"], hooks.back + made
        assert c["x"] % 16 == 0 and c["ldx"] % 8 == 0 and c["ldx"] >= K and c["codes"] % 16 == 0 and c["ldz"] == 24
        assert inside(c["x"], (M - 1) * c["ldx"] + K, 2, known)
        assert inside(c["z"], M * 24, 2, known) and inside(c["codes"], 24 * c["ldc"], 2, known)
        assert inside(c["scale"], 24, 4, known)
        seen["x"] = values(c["x"], c["ldx"], M, K, x.dtype)

    with pytest.MonkeyPatch.context() as mp:
        mp.setattr(_lib, "tensor_backward", look)
        mp.setattr(_tensor, "_rows_on16", noted(rows, lambda out: out[0]))
        mp.setattr(torch.Tensor, "contiguous", noted(dense, lambda out: out))
        mp.setattr(torch.Tensor, "clone", noted(clone, lambda out: out))
        y.backward(torch.ones_like(y))
    if wide % 8 == 0:                                   # (else the forward pass's own copy, which is not made here)
        assert torch.equal(seen["x"], x)


def test_other_tensors_than_were_kept_are_refused(calls):
    x, w = torch.randn(40, 64).bfloat16(), torch.randn(24, 64).requires_grad_()
    for change, error in ((lambda t: t.float() if t.dtype == torch.bfloat16 else t, SFTypeError),
                          (lambda t: t[:20] if t.dtype == torch.bfloat16 else t, SFShapeError),
                          (lambda t: t[:100] if t.dtype == torch.uint8 else t, SFShapeError),
                          (lambda t: t.to("meta"), SFShapeError)):
        with torch.autograd.graph.saved_tensors_hooks(change, lambda t: t):
            y = _tensor._TensorLinear.apply(x, w, None, None, None, 8, "per_channel", _lib.ACTIVATIONS["gelu"])
        calls.clear()
        with pytest.raises(error, match="kept"):
            y.backward(torch.ones_like(y))
        assert "backward" not in calls


def test_a_padded_x_is_kept_once(calls):
    """The copy of x with its rows on 16 bytes lies beside the codes: the hooks see it once."""
    sizes = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: sizes.append(t.numel() * t.element_size()) or t, lambda t: t):
        _tensor._TensorLinear.apply(torch.randn(40, 13).bfloat16(), torch.randn(24, 13).requires_grad_(), None, None, None,
                                    8, "per_channel", 0)
    assert len(sizes) == 1
