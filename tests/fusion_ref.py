"""References of the operators between the towers in 64 bits, with the error that their kernels may have at every element.

A rounding to bf16 is off by at most UB = 2^-8 of the value, one to fp32 by UF = 2^-24.  The bounds below add up the roundings that a kernel
makes: its sums of n products in fp32 (n UF of the sum of magnitudes, any order), the hardware's exp2 / log2 / sin / rsqrt (within 4 UF of
the result), P and dS rounded to the operand type, and the result's own rounding."""
import math

import torch

UB, UF = 2.0 ** -8, 2.0 ** -24
F64 = torch.float64


def unit(dtype):
    return UB if dtype == torch.bfloat16 else UF


def lengths(cu, rows, batch):
    if cu is None:
        n = rows // batch
        return [(i * n, n) for i in range(batch)]
    return [(int(cu[i]), int(cu[i + 1]) - int(cu[i])) for i in range(batch)]


def xattn(q, k, v, heads, dout=None, kv_heads=None, batch=None, cu_q=None, cu_kv=None, kv_len=None, key_mask=None, scale=None):
    """{name: (value, bound)} of out, lse (, dq, dk, dv)"""
    u = unit(q.dtype)
    up = u if q.dtype == torch.bfloat16 else 0.0
    kv_heads = kv_heads or heads
    hd, rep = q.shape[1] // heads, heads // kv_heads
    scale = hd ** -0.5 if scale is None else scale
    batch = batch or (cu_q if cu_q is not None else cu_kv).numel() - 1
    z = lambda *s: torch.zeros(*s, dtype=F64)  # noqa: E731
    out, eo = z(q.shape[0], heads, hd), z(q.shape[0], heads, hd)
    lse, el = torch.full((heads, q.shape[0]), -math.inf, dtype=F64), z(heads, q.shape[0])
    dq, edq = z(q.shape[0], heads, hd), z(q.shape[0], heads, hd)
    dk, edk, dv, edv = (z(k.shape[0], kv_heads, hd) for _ in range(4))
    for i, ((q0, nq), (k0, nk)) in enumerate(zip(lengths(cu_q, q.shape[0], batch), lengths(cu_kv, k.shape[0], batch))):
        if kv_len is not None:
            nk = min(nk, max(int(kv_len[i]), 0))
        keys = torch.arange(k0, k0 + nk)
        if key_mask is not None:
            keys = keys[key_mask.reshape(-1)[keys].bool()]
        n = keys.numel()
        if n == 0 or nq == 0:
            continue
        rows = slice(q0, q0 + nq)
        for h in range(heads):
            g = h // rep
            Q, K, V = q[rows, h * hd:(h + 1) * hd].to(F64), k[keys, g * hd:(g + 1) * hd].to(F64), v[keys, g * hd:(g + 1) * hd].to(F64)
            s = scale * (Q @ K.T)
            L = torch.logsumexp(s, 1)
            P = torch.exp(s - L[:, None])
            # a score in units of log2: sum of hd products, the products with scale and log2(e), the subtraction of the running maximum
            es = scale * (Q.abs() @ K.abs().T) * (hd + 4) * UF + 4 * UF * s.abs().amax(1, keepdim=True)
            es = es.amax(1, keepdim=True)
            rel = 2 * es + (n + 16) * UF                                   # of p: numerator, and the sum that divides it
            o = P @ V
            pv = P @ V.abs()
            out[rows, h], eo[rows, h] = o, (rel + up + n * UF) * pv + u * o.abs()
            lse[h, rows], el[h, rows] = L, (2 * es[:, 0] + (n + 16) * UF) + 4 * UF * L.abs()
            if dout is None:
                continue
            do = dout[rows, h * hd:(h + 1) * hd].to(F64)
            dp = do @ V.T
            D = (do * o).sum(1, keepdim=True)
            edp = (hd + 2) * UF * (do.abs() @ V.abs().T)
            eD = (do.abs() * (eo[rows, h] + (hd + n + 4) * UF * pv)).sum(1, keepdim=True)
            # lse's error moves every p of the row as well
            rp = rel + 2 * el[h, rows][:, None] + 8 * UF * (1 + L.abs()[:, None])
            ds = P * (dp - D)
            eds = P * (edp + eD) + (rp + up + 4 * UF) * ds.abs()
            dq[rows, h] = scale * (ds @ K)
            edq[rows, h] = scale * (eds @ K.abs() + n * UF * (ds.abs() @ K.abs())) + u * dq[rows, h].abs()
            dk[keys, g] += scale * (ds.T @ Q)
            edk[keys, g] += scale * (eds.T @ Q.abs() + nq * rep * UF * (ds.abs().T @ Q.abs()))
            dv[keys, g] += P.T @ do
            edv[keys, g] += ((rp + up).expand_as(P) * P).T @ do.abs() + nq * rep * UF * (P.T @ do.abs())
    flat = lambda t: t.reshape(t.shape[0], -1)  # noqa: E731
    res = {"out": (flat(out), flat(eo)), "lse": (lse, el)}
    if dout is not None:
        res.update(dq=(flat(dq), flat(edq)), dk=(flat(dk), flat(edk) + u * flat(dk).abs()), dv=(flat(dv), flat(edv) + u * flat(dv).abs()))
    return res


def rope(x, pos, heads, sections, theta=10000.0, joint=False, interleaved=False, inverse=False):
    """(value, bound)"""
    hd, P = x.shape[1] // heads, sum(sections)
    th = theta if isinstance(theta, (tuple, list)) else [theta] * len(sections)
    ang = torch.empty(pos.shape[0], P, dtype=F64)
    i = 0
    for a, n in enumerate(sections):
        for j in range(n):
            ang[:, i] = pos[:, a].to(F64) * th[a] ** -(i / P if joint else j / n)
            i += 1
    ang = ang.repeat(x.shape[0] // pos.shape[0], 1)[:, None, :] * (-1 if inverse else 1)
    h = x.to(F64).reshape(x.shape[0], heads, hd)
    ia = torch.arange(P) * 2 if interleaved else torch.arange(P)
    ib = ia + 1 if interleaved else ia + P
    a, b = h[..., ia], h[..., ib]
    y, mag = h.clone(), torch.zeros_like(h)
    y[..., ia], y[..., ib] = a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos()
    mag[..., ia] = mag[..., ib] = a.abs() + b.abs()
    # sin and cos of a fraction of a turn in fp32 (the fraction's rounding: half a turn times UF, times 2 pi; the functions: 2 UF), two products and a
    # sum; the 64-bit angle itself: |turns| 2^-52
    bound = (12 * UF + ang.abs().amax() * 2.0 ** -50) * mag + unit(x.dtype) * y.abs()
    return y.reshape(x.shape), bound.reshape(x.shape)


def _norm(z, w, b, rms, eps):
    mu = torch.zeros(z.shape[0], 1, dtype=F64) if rms else z.mean(1, keepdim=True)
    c = z - mu
    return c / torch.sqrt((c * c).mean(1, keepdim=True) + eps) * w + (0 if b is None else b)


def join(x, y, post, gate, scale, pre, alpha=1.0, eps=1e-5, rms=False, gate_tanh=False, dx_out=None, dn=None):
    """values in 64 bits (dict), gradients by torch's autograd"""
    leaf = lambda t: None if t is None else t.detach().to(F64).requires_grad_(True)  # noqa: E731
    X, Y, G, S = leaf(x), leaf(y), leaf(gate), leaf(scale)
    po = None if post is None else [leaf(t) for t in post]
    pr = None if pre is None else [leaf(t) for t in pre]
    t = Y if po is None else _norm(Y, po[0], po[1], rms, eps)
    if G is not None:
        g = (torch.tanh(G) if gate_tanh else G).reshape(-1) if G.dim() < 2 else (torch.tanh(G) if gate_tanh else G)
        g = g.repeat_interleave(x.shape[0] // g.shape[0], 0)
        t = t * (g if g.dim() == 2 else g[:, None])
    if S is not None:
        t = t * S
    xo = alpha * X + t
    n = None if pr is None else _norm(xo, pr[0], pr[1], rms, eps)
    res = {"x_out": xo.detach()}
    if n is not None:
        res["n"] = n.detach()
    if dx_out is not None or dn is not None:
        total = 0.0
        if dx_out is not None:
            total = total + (xo * dx_out.to(F64)).sum()
        if dn is not None:
            total = total + (n * dn.to(F64)).sum()
        names = ["dx", "dy", "post_w", "post_b", "gate", "scale", "pre_w", "pre_b"]
        leaves = [X, Y, *(po or (None, None)), G, S, *(pr or (None, None))]
        have = [(a, b) for a, b in zip(names, leaves) if b is not None]
        for (a, b), gr in zip(have, torch.autograd.grad(total, [b for _, b in have], allow_unused=True)):
            res[a] = torch.zeros_like(b) if gr is None else gr
    return res


def join_bounds(ref, x, y, post, gate, scale, pre, alpha=1.0, eps=1e-5, rms=False, gate_tanh=False, dx_out=None, dn=None):
    """{name: bound} for join()'s values.  A norm's statistics are sums of d terms, at most 40 of them one after the other (32 per lane, then trees): a norm or
    its gradient is off by at most 100 UF of the magnitudes it adds; four of them follow one another at most, plus a dozen products: 500 UF.  A column
    sum adds one rounding per row."""
    W = lambda t: None if t is None else t.to(F64)  # noqa: E731
    c, u, rows = 500 * UF, unit(x.dtype), x.shape[0]
    X, Y = W(x), W(y)

    def stats(z):
        mu = torch.zeros(rows, 1, dtype=F64) if rms else z.mean(1, keepdim=True)
        r = 1 / torch.sqrt(((z - mu) ** 2).mean(1, keepdim=True) + eps)
        return (z - mu) * r, r, z.abs().mean(1, keepdim=True) * r

    one = torch.ones(1, x.shape[1], dtype=F64)
    g = one
    if gate is not None:
        g = (torch.tanh(W(gate)) if gate_tanh else W(gate))
        g = g.reshape(-1, 1) if g.dim() < 2 else g
        g = g.repeat_interleave(rows // g.shape[0], 0)
    sc = one if scale is None else W(scale)[None]
    yh, rs, ky = stats(Y) if post is not None else (Y, torch.ones(rows, 1, dtype=F64), torch.zeros(rows, 1, dtype=F64))
    w1 = one if post is None else W(post[0])[None].abs()
    b1 = 0 * one if post is None or post[1] is None else W(post[1])[None].abs()
    p = (yh.abs() + ky) * w1 + b1
    t = p * (sc * g).abs()
    mx = alpha * X.abs() + t
    out = {"x_out": c * mx + u * ref["x_out"].abs()}
    if pre is not None:
        xh, r2, kx = stats(ref["x_out"])
        w2 = W(pre[0])[None].abs()
        mh = mx * r2 + kx                                  # magnitude behind xhat, cancellation in x_out and in its mean included
        mh = mh + xh.abs() * (mh * xh.abs()).mean(1, keepdim=True)
        out["n"] = c * (mh * w2 + (0 if pre[1] is None else W(pre[1]).abs())) + u * ref["n"].abs()
    if dx_out is None and dn is None:
        return out
    mG = 0 * X if dx_out is None else W(dx_out).abs()
    if dn is not None:
        wn = W(dn).abs() * w2
        mm = mh + xh.abs()
        mG = mG + r2 * (wn + wn.mean(1, keepdim=True) + mm * (wn * mm).mean(1, keepdim=True)) * (1 + mm)
        out["pre_w"] = (c + rows * UF) * (W(dn).abs() * mm).sum(0)
        out["pre_b"] = (c + rows * UF) * W(dn).abs().sum(0)
    elif pre is not None:
        out["pre_w"] = out["pre_b"] = torch.zeros(x.shape[1], dtype=F64)
    out["dx"] = c * alpha * mG + u * ref["dx"].abs()
    q = mG * sc.abs()
    dp = q * g.abs()
    if post is None:
        out["dy"] = c * dp + u * ref["dy"].abs()
    else:
        my, wn = yh.abs() + ky, dp * w1
        out["dy"] = c * rs * (wn + wn.mean(1, keepdim=True) + my * (wn * my).mean(1, keepdim=True)) * (1 + my) + u * ref["dy"].abs()
        out["post_w"] = (c + rows * UF) * (dp * my).sum(0)
        out["post_b"] = (c + rows * UF) * dp.sum(0)
    if scale is not None:
        out["scale"] = (c + rows * UF) * (mG * g.abs() * p).sum(0)
    if gate is not None:
        e = q * p
        e = e.sum(1) if gate.dim() < 2 else e
        n = gate.shape[0] if gate.dim() else 1
        e = e.reshape(n, rows // n, *e.shape[1:]).sum(1)
        out["gate"] = ((c + (rows + x.shape[1]) * UF) * e).reshape(gate.shape)
    return out
