"""Autograd functions of the operators between the towers: cross attention to an encoder's states of another length, rotary positions with
several axes, and the norms around a block fused with its gate and residual scale (declip_amd.ops: xattn_*, rope_axes, join_norm_*).

They are what a caption decoder or fusion tower over the image tower's tokens is built from -- the branch that the reference declares
(return_caption, model/declip.py:166-167) and refuses:

    q = fusion.rope_axes(q, pos_q, heads, sections)
    a = fusion.cross_attention(q, k, v, heads, cu_q=cu, batch=b)
    x, h = fusion.join_norm(x, project(a), post=(w1, b1), gate=g, scale=s, pre=(w2, b2))

Gradients of parameters come back as ordinary autograd gradients (fp32).  As with every autograd graph: do not capture a backward pass into a
hipGraph while an eager graph over the same leaves is alive (its AccumulateGrad nodes carry the eager stream into the capture)."""
import torch
from torch.autograd.function import once_differentiable

from . import ops
from .lib import DeclipHipError

TABLES = ("cu_q", "cu_kv", "kv_len", "key_mask")


def _number(name, v):
    """a plain number, also of a tensor of one element: read once, in the forward, so that the backward goes by the same; one that asks for a gradient would get none"""
    if torch.is_tensor(v):
        if v.requires_grad and torch.is_grad_enabled():
            raise DeclipHipError("bad argument: %s carries no gradient (detach it, or multiply outside)" % name)
        return v.detach().item()
    return v


def _rows16(t):
    """contiguous columns, 16-byte aligned rows less than 2^22 elements apart: what the kernels read; anything else is copied"""
    unit = 16 // t.element_size()
    ok = t.dim() == 2 and (t.shape[1] == 1 or t.stride(1) == 1) and t.data_ptr() % 16 == 0
    if ok and t.shape[0] > 1:
        ok = t.shape[1] <= t.stride(0) < 1 << 22 and t.stride(0) % unit == 0
    return t if ok else t.clone(memory_format=torch.contiguous_format)


class CrossAttnFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, heads, geometry):
        q, k, v = _rows16(q), _rows16(k), _rows16(v)
        out, lse = ops.xattn_fwd(q, k, v, heads, **geometry)
        ctx.heads = heads
        ctx.plain = {n: t for n, t in geometry.items() if not torch.is_tensor(t)}
        ctx.tables = [n for n, t in geometry.items() if torch.is_tensor(t)]
        ctx.save_for_backward(q, k, v, out, lse, *(geometry[n] for n in ctx.tables))
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, _dlse):
        q, k, v, out, lse, *tables = ctx.saved_tensors
        dq, dk, dv = ops.xattn_bwd(q, k, v, out, _rows16(dout), lse, ctx.heads, **ctx.plain, **dict(zip(ctx.tables, tables)))
        return dq, dk, dv, None, None


def cross_attention(q, k, v, heads, *, need_lse=False, **geometry):
    """ops.xattn_fwd with its gradient: out [rows_q, heads*hd] (need_lse: (out, lse); lse and scale carry no gradient)."""
    geometry = {n: t if n in TABLES else _number(n, t) for n, t in geometry.items()}
    out, lse = CrossAttnFn.apply(q, k, v, heads, geometry)
    return (out, lse) if need_lse else out


class RopeAxesFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, pos, heads, sections, how):
        ctx.args = (heads, sections, how)
        ctx.save_for_backward(pos)
        x = x if x.dim() == 2 and (x.shape[1] == 1 or x.stride(1) == 1) and (x.shape[0] <= 1 or x.stride(0) >= x.shape[1]) else x.contiguous()
        return ops.rope_axes(x, pos, heads, sections, **how)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        heads, sections, how = ctx.args
        return ops.rope_axes(dy.contiguous(), ctx.saved_tensors[0], heads, sections, inverse=True, **how), None, None, None, None


def rope_axes(x, pos, heads, sections, theta=10000.0, *, joint=False, interleaved=False):
    """ops.rope_axes with its gradient (the rotation back); pos and theta carry none."""
    theta = tuple(_number("theta", t) for t in theta) if isinstance(theta, (tuple, list)) else _number("theta", theta)
    return RopeAxesFn.apply(x, pos, heads, tuple(sections), dict(theta=theta, joint=joint, interleaved=interleaved))


class JoinNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, post_w, post_b, gate, scale, pre_w, pre_b, how):
        c = lambda t: None if t is None else t.contiguous()  # noqa: E731
        x, y, *params = (c(t) for t in (x, y, post_w, post_b, gate, scale, pre_w, pre_b))
        x_out, n, stats = ops.join_norm_fwd(x, y, **JoinNormFn._named(params), **how)
        ctx.how = how
        ctx.save_for_backward(x, y, stats, *params)
        ctx.set_materialize_grads(False)
        return x_out, n

    @staticmethod
    def _named(params):
        post_w, post_b, gate, scale, pre_w, pre_b = params
        pair = lambda w, b: None if w is None and b is None else (w, b)  # noqa: E731 -- (a bias alone goes on, and is refused)
        return dict(post=pair(post_w, post_b), gate=gate, scale=scale, pre=pair(pre_w, pre_b))

    @staticmethod
    @once_differentiable
    def backward(ctx, dx_out, dn):
        x, y, stats, *params = ctx.saved_tensors
        if dx_out is None and dn is None:
            return (None,) * 9
        c = lambda t: None if t is None else t.contiguous()  # noqa: E731
        dx, dy, grads = ops.join_norm_bwd(x, y, c(dx_out), c(dn), stats, **JoinNormFn._named(params), **ctx.how)
        return (dx, dy, *grads, None)


def join_norm(x, y, *, post=None, gate=None, scale=None, pre=None, alpha=1.0, eps=1e-5, rms=False, gate_tanh=False):
    """ops.join_norm_fwd with its gradient: (x_out, n), n = None without `pre`; alpha and eps carry none."""
    alpha, eps = _number("alpha", alpha), _number("eps", eps)
    post, pre = post or (None, None), pre or (None, None)
    return JoinNormFn.apply(x, y, *post, gate, scale, *pre, dict(alpha=alpha, eps=eps, rms=rms, gate_tanh=gate_tanh))
