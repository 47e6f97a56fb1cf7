"""CPU: what the 16-bit operators' Python forms refuse because it would be lost without a word."""
import pytest

torch = pytest.importorskip("torch")


def _calls():
    from edge_maskgit_b200 import runtime as rt
    f16 = torch.float16
    return {
        "linear": (rt.linear, [torch.zeros(2, 64, dtype=f16), torch.zeros(8, 64, dtype=f16)]),
        "attention": (rt.attention, [torch.zeros(1, 2, 2, 64, dtype=f16) for _ in range(3)]),
        "logits_adjust": (rt.logits_adjust, [torch.zeros(2, 40)]),
    }


@pytest.mark.parametrize("name", ["linear", "attention", "logits_adjust"])
def test_forward_mode_tangents_are_refused(name):
    import torch.autograd.forward_ad as fwd
    from edge_maskgit_b200.runtime import MgcError
    fn, args = _calls()[name]
    for i in range(len(args)):
        with fwd.dual_level():
            with_tangent = list(args)
            with_tangent[i] = fwd.make_dual(args[i], torch.ones_like(args[i]))
            with pytest.raises(MgcError, match="tangent"):
                fn(*with_tangent)
            with pytest.raises(MgcError, match="CUDA"):   # a level alone is no reason
                fn(*args)


def test_optional_arguments_with_tangents_are_refused():
    import torch.autograd.forward_ad as fwd
    from edge_maskgit_b200.runtime import MgcError
    with fwd.dual_level():
        for name, key, shape in (("linear", "bias", (8,)), ("attention", "slopes", (2,)), ("attention", "dist_bias", (2, 3)),
                                 ("logits_adjust", "bias", (40,))):
            fn, args = _calls()[name]
            with pytest.raises(MgcError, match=key + " carries"):
                fn(*args, **{key: fwd.make_dual(torch.zeros(shape), torch.ones(shape))})


@pytest.mark.parametrize("name", ["linear", "attention", "logits_adjust"])
def test_traces_are_refused(name):
    from edge_maskgit_b200.runtime import MgcError
    fn, args = _calls()[name]
    with pytest.raises(MgcError, match="trace"):
        torch.jit.trace(fn, tuple(args))
