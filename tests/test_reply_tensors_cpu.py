"""What the torch module of the reply calls refuses to read: tensors of the host (device -1) up to the library's own refusal of a context that is none."""
import pytest

from imagecaptioner_amd import TagPipeError
from imagecaptioner_amd.replies import _native

torch = pytest.importorskip("torch")
ROWS, VOCAB = 2, 40


def arguments():
    """Plain tensors of every kind that a call takes."""
    f, i = lambda *s: torch.ones(*s), lambda *s: torch.ones(*s, dtype=torch.int32)
    return dict(logits=f(ROWS, VOCAB), temperature=f(ROWS), uniform=f(ROWS), history=i(ROWS, 5), history_len=i(ROWS), prompt_len=i(ROWS), repetition=f(ROWS), frequency=f(ROWS),
                presence=f(ROWS), bias=f(3, VOCAB), bias_row=i(ROWS), mask=i(3, 2), mask_row=i(ROWS))


def choose(**kw):
    return _native().choose(None, -1, 0, kw.pop("logits"), kw.pop("temperature"), kw.pop("uniform"), kw)


def shape_into(out):
    return _native().shape(None, -1, 0, torch.ones(ROWS, VOCAB), out, {})


def test_plain_tensors_reach_the_library():
    with pytest.raises(TagPipeError, match="null argument"):
        choose(**arguments())


def test_tangents_are_refused():
    """A forward-mode derivative is refused like a backward one, and taken where derivatives are off."""
    from torch.autograd import forward_ad
    floats = [k for k, v in arguments().items() if v.is_floating_point()]
    with forward_ad.dual_level():
        def dual(x):
            return forward_ad.make_dual(x, torch.ones_like(x))
        for k in floats:
            args = arguments()
            args[k] = dual(args[k])
            with pytest.raises(ValueError, match=k + " requires a gradient"):
                choose(**args)
            with forward_ad._set_fwd_grad_enabled(False), pytest.raises(TagPipeError, match="null argument"):
                choose(**args)
            args[k] = forward_ad.unpack_dual(args[k]).primal
            with pytest.raises(TagPipeError, match="null argument"):
                choose(**args)
        with pytest.raises(ValueError, match="out requires a gradient"):
            shape_into(dual(torch.ones(ROWS, VOCAB)))


def test_values_that_do_not_stand_in_memory_are_refused():
    """The imaginary part of a conjugate is a view with the opposite sign in memory; torch's efficient zeros have no memory at all."""
    for k, v in arguments().items():
        lazy = [torch._efficientzerotensor(v.shape, dtype=v.dtype)]
        if v.is_floating_point():
            lazy.append(torch._neg_view(v))
        for t in lazy:
            args = arguments()
            args[k] = t
            with pytest.raises(ValueError, match=k + " does not stand in memory"):
                choose(**args)
            args[k] = t.resolve_neg().clone() if t.is_neg() else torch.zeros(t.shape, dtype=t.dtype)
            with pytest.raises(TagPipeError, match="null argument"):
                choose(**args)
    with pytest.raises(ValueError, match="out does not stand in memory"):
        shape_into(torch._neg_view(torch.ones(ROWS, VOCAB)))
