"""dq and dk of cross attention in 64 bits, with the norm that the error of each may have."""
import math

import torch

from fusion_ref import F64, UF, lengths, unit


def gradients(q, k, v, heads, dout, kv_heads=None, batch=None, cu_q=None, cu_kv=None, kv_len=None, key_mask=None, scale=None):
    """{name: (value, norm its error may have)} of dq, dk.
    Relative roundings spread over at most [-u, u] have a mean square of u^2 / 3 at most, independent ones add up in squares, and the norm of a few hundred
    of them stays within 15 % of that: dS is rounded to the operand type element by element, the result once more.  fp32's roundings are counted the
    same way (a sum of n products: sqrt(n / 3) UF of the magnitudes), twice what they come to; what moves a whole row (D = sum p dp from
    unrounded p and dp, lse) is added up before it is squared."""
    kv_heads = kv_heads or heads
    hd, rep = q.shape[1] // heads, heads // kv_heads
    scale = hd ** -0.5 if scale is None else scale
    batch = batch or (cu_q if cu_q is not None else cu_kv).numel() - 1
    val = {"dq": torch.zeros(q.shape[0], heads, hd, dtype=F64), "dk": torch.zeros(k.shape[0], kv_heads, hd, dtype=F64)}
    operand, fine = {"dq": 0.0, "dk": 0.0}, {"dq": 0.0, "dk": 0.0}
    for i, ((q0, nq), (k0, nk)) in enumerate(zip(lengths(cu_q, q.shape[0], batch), lengths(cu_kv, k.shape[0], batch))):
        keys = torch.arange(k0, k0 + (nk if kv_len is None else min(nk, int(kv_len[i]))))
        if key_mask is not None:
            keys = keys[key_mask.reshape(-1)[keys].bool()]
        n, rows = keys.numel(), slice(q0, q0 + nq)
        if n == 0 or nq == 0:
            continue
        for h in range(heads):
            g = h // rep
            Q, K, V = q[rows, h * hd:(h + 1) * hd].to(F64), k[keys, g * hd:(g + 1) * hd].to(F64), v[keys, g * hd:(g + 1) * hd].to(F64)
            do = dout[rows, h * hd:(h + 1) * hd].to(F64)
            s = scale * (Q @ K.T)
            L = torch.logsumexp(s, 1, keepdim=True)
            P, dp = torch.exp(s - L), do @ V.T
            ds = P * (dp - (P * dp).sum(1, keepdim=True))
            val["dq"][rows, h] = scale * (ds @ K)
            val["dk"][keys, g] += scale * (ds.T @ Q)
            operand["dq"] += scale ** 2 * float((ds ** 2 @ (K * K)).sum())
            operand["dk"] += scale ** 2 * float((ds.T ** 2 @ (Q * Q)).sum())
            # fp32: a score and its exponential, a row's lse, dp; what they make of an element of dS, and of the row's D
            one = scale * (Q.abs() @ K.abs().T) * math.sqrt((hd + 4) / 3) * UF + 4 * UF * s.abs()
            row = (P * one).sum(1, keepdim=True) + (math.sqrt(n) + 16) * UF + 8 * UF * (1 + L.abs())
            edp = (do.abs() @ V.abs().T) * math.sqrt((hd + 2) / 3) * UF
            e1 = P * edp + (one + row + 4 * UF) * ds.abs()
            e2 = (P * (edp + (one + row + math.sqrt(n / 3) * UF) * dp.abs())).sum(1, keepdim=True)
            fine["dq"] += scale ** 2 * float((e1 ** 2 @ (K * K) + (e2 * (P @ K)) ** 2 + n * UF ** 2 * (ds ** 2 @ (K * K))).sum())
            fine["dk"] += scale ** 2 * float(((e1 + P * e2).T ** 2 @ (Q * Q) + nq * rep * UF ** 2 * (ds.T ** 2 @ (Q * Q))).sum())
    u = unit(q.dtype)
    return {name: (t.reshape(t.shape[0], -1), 1.15 * u / math.sqrt(3) * math.sqrt((operand[name] if q.dtype == torch.bfloat16 else 0.0) + float((t * t).sum()))
                   + 2 * math.sqrt(fine[name])) for name, t in val.items()}
