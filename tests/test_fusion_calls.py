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


def test_the_backward_takes_the_numbers_the_forward_took():
    """alpha, theta and the like may come as tensors or lists that a schedule writes to before the backward runs"""
    from declip_amd import fusion
    with emulated_gpu():
        x, y = rnd(4, 64).requires_grad_(True), rnd(4, 64, seed=1).requires_grad_(True)
        alpha = torch.tensor(2.0)
        out, _ = fusion.join_norm(x, y, alpha=alpha)
        alpha.fill_(5.0)
        dx, dy = torch.autograd.grad(out, [x, y], torch.ones_like(out))
        assert torch.equal(dx, torch.full_like(x, 2.0)) and torch.equal(dy, torch.ones_like(y))
        pos, theta, sections = torch.arange(4, dtype=torch.int32)[:, None].contiguous(), [100.0], [16]
        out = fusion.rope_axes(x, pos, 2, sections, theta)
        theta[0], sections[0] = 1e6, 8
        back, = torch.autograd.grad(out, [x], out.detach())
        assert float((back - x).abs().max()) < 1e-5          # rotated there and back
        scale, most = torch.tensor(0.5), torch.tensor(4)
        a, = torch.autograd.grad(fusion.cross_attention(x, y, y, 2, batch=1, scale=0.5).sum(), [x])
        out = fusion.cross_attention(x, y, y, 2, batch=1, scale=scale, max_q=most)
        scale.fill_(0.1)
        b, = torch.autograd.grad(out.sum(), [x])
        assert torch.equal(a, b)


def test_a_trainable_number_is_refused():
    """a learned scale, alpha or base: these operators have no gradient for it, and would leave it where it is without a word"""
    from declip_amd import fusion
    from declip_amd.lib import DeclipHipError
    with emulated_gpu():
        x, pos, t = rnd(4, 64), torch.arange(4, dtype=torch.int32)[:, None].contiguous(), torch.tensor(2.0, requires_grad=True)
        for call, name in ((lambda v: fusion.cross_attention(x, x, x, 2, batch=1, scale=v), "scale"), (lambda v: fusion.join_norm(x, x, alpha=v), "alpha"),
                           (lambda v: fusion.join_norm(x, x, eps=v), "eps"), (lambda v: fusion.rope_axes(x, pos, 2, (4,), theta=v), "theta"),
                           (lambda v: fusion.rope_axes(x, pos, 2, (4,), theta=[v]), "theta")):
            with pytest.raises(DeclipHipError, match=name):
                call(t)
            call(t.detach())
            with torch.no_grad():
                call(t)
