"""Calls of the autograd functions between the towers (declip_amd/fusion.py) that go wrong without a word if nobody looks: on the host emulation."""
import pytest
import torch

from hipemu_util import emulated_gpu


def rnd(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("which", ["post", "pre"])
def test_a_bias_without_its_weight_is_refused(which):
    """as ops.join_norm_fwd refuses it; dropped, the call would answer without the norm and its bias would get no gradient"""
    from declip_amd import fusion
    from declip_amd.lib import DeclipHipError
    with emulated_gpu():
        x, b = rnd(4, 64), rnd(64, seed=1).requires_grad_(True)
        with pytest.raises(DeclipHipError, match="weight"):
            fusion.join_norm(x, x, **{which: (None, b)})
        assert fusion.join_norm(x, x, **{which: (None, None)})[1] is None
