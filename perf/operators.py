"""Workloads of the cross-tower operators: cross attention to an encoder's states of another length, rotary positions with
several axes, and the norms around a block fused with its gate and residual scale.

`run` computes a pass either from elementary torch operations in 32 bits (`own = False`) or through declip_amd.ops."""
import math

import torch

own = False

BF16, FP32 = torch.bfloat16, torch.float32


# ------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # a caption decoder's training step: packed captions of 5..77 tokens on the 197 states of a ViT-B/16 image tower
        dict(name="xattn_captions_train", op="xattn", train=True, dtype="bf16", b=256, heads=8, kv_heads=8, hd=64, lq=77, lq_lo=5, s=197, s_lo=197,
             packed=True, mask=0.0),
        # the longest training: text on 16 video frames of 196 patches, shared kv heads, dropped patches
        dict(name="xattn_video_train", op="xattn", train=True, dtype="bf16", b=4, heads=16, kv_heads=4, hd=128, lq=1024, lq_lo=1024, s=3136, s_lo=1568,
             packed=False, mask=0.1),
        # scoring a long text against a long encoder sequence, forward only
        dict(name="xattn_prompt", op="xattn", train=False, dtype="bf16", b=2, heads=12, kv_heads=12, hd=64, lq=2047, lq_lo=2047, s=6272, s_lo=6001,
             packed=False, mask=0.0),
        # serving: one new token per sequence, long encoder states of different lengths
        dict(name="xattn_decode", op="xattn", train=False, dtype="bf16", b=64, heads=16, kv_heads=4, hd=64, lq=1, lq_lo=1, s=3136, s_lo=196,
             packed=False, mask=0.0),
        # serving at its smallest: latency (50 states of a ViT-B/32 image tower)
        dict(name="xattn_decode_small", op="xattn", train=False, dtype="bf16", b=4, heads=8, kv_heads=8, hd=64, lq=1, lq_lo=1, s=50, s_lo=50,
             packed=False, mask=0.0),
        # the validation precision, a head size that is no power of two, sequences without a key
        dict(name="xattn_fp32_train", op="xattn", train=True, dtype="fp32", b=16, heads=12, kv_heads=12, hd=80, lq=77, lq_lo=1, s=257, s_lo=0,
             packed=True, mask=0.2),
        # q and k columns of a fused projection, video positions (time, height, width), rotation and its gradient
        dict(name="rope_video_train", op="rope", train=True, dtype="bf16", rows=25088, pos_rows=1568, heads=24, extra=12, hd=64, sections="8,12,12",
             joint=False, interleaved=False, far=32, frac=False),
        # serving: one token per sequence at far positions, one ladder shared by the axes
        dict(name="rope_tokens", op="rope", train=False, dtype="bf16", rows=32, pos_rows=32, heads=20, extra=4, hd=128, sections="16,24,24",
             joint=True, interleaved=False, far=1000000, frac=False),
        # an image grid resampled to fractional positions, part of each head rotated, neighbouring pairs, validation precision
        dict(name="rope_image_fp32", op="rope", train=True, dtype="fp32", rows=4096 + 15, pos_rows=4096 + 15, heads=12, extra=0, hd=80, sections="16,16",
             joint=False, interleaved=True, far=64, frac=True),
        # a ViT-B block boundary at the batch of the headline benchmark: LayerScale and a per-image gate
        dict(name="join_train", op="join", train=True, dtype="bf16", rows=25600, d=768, groups=512, gate="channel", tanh=False, scale=True, post=True, pre=True,
             rms=False, alpha=1.0),
        # a wide RMS-normed block with one tanh gate, an odd number of rows
        dict(name="join_wide_train", op="join", train=True, dtype="bf16", rows=8191, d=4096, groups=1, gate="row", tanh=True, scale=False, post=True, pre=True,
             rms=True, alpha=1.0),
        # serving: a few tokens
        dict(name="join_tokens", op="join", train=False, dtype="bf16", rows=64, d=1024, groups=64, gate="row", tanh=False, scale=True, post=True, pre=True,
             rms=False, alpha=1.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["xattn", "xattn", "rope", "join"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if op == "xattn":
        kv_heads = rng.choice([1, 2, 3, 4, 8])
        heads = kv_heads * rng.choice([1, 1, 2, 4])
        hd = rng.choice([32, 64, 64, 80, 96, 128])
        form = rng.choice(["train", "train", "prompt", "decode"])
        lq = rng.randint(1, 2) if form == "decode" else _log(rng, 2, 2048)
        s = _log(rng, 1, 6272)
        most = min(64 if form != "decode" else 256, 400_000_000 // (heads * hd * lq * s) * 16, 100_000_000 // (heads * lq * s), 100_000_000 // (kv_heads * hd * s),
                   100_000_000 // (heads * hd * lq))
        return dict(op="xattn", train=form == "train", dtype=dtype, b=_log(rng, 1, max(1, most)), heads=heads, kv_heads=kv_heads, hd=hd, lq=lq,
                    lq_lo=rng.randint(1, lq), s=s, s_lo=rng.randint(0, s), packed=rng.random() < 0.5, mask=rng.choice([0.0, 0.0, 0.1, 0.5]))
    if op == "rope":
        hd = rng.choice([32, 64, 80, 96, 128])
        axes = rng.randint(1, 3)
        room = rng.choice([hd // 2, hd // 2, hd // 4])
        cut = sorted(rng.sample(range(1, room), axes - 1))
        sections = ",".join(str(b - a) for a, b in zip([0] + cut, cut + [room]))
        heads = rng.randint(1, 24)
        rows = _log(rng, 1, min(32768, 40_000_000 // (heads * hd)))
        rep = rng.choice([1, 1, 2, 4])
        return dict(op="rope", train=rng.random() < 0.7, dtype=dtype, rows=rows * rep if rows < 8192 else rows, pos_rows=rows, heads=heads, extra=rng.choice([0, 1, 12]),
                    hd=hd, sections=sections, joint=rng.random() < 0.5, interleaved=rng.random() < 0.5, far=_log(rng, 8, 1000000), frac=rng.random() < 0.3)
    d = rng.choice([_log(rng, 16, 8192), 8 * _log(rng, 4, 1024)])
    groups = _log(rng, 1, 512)
    per = _log(rng, 1, max(1, min(32768, 33_000_000 // d) // groups))
    return dict(op="join", train=rng.random() < 0.7, dtype=dtype, rows=groups * per, d=d, groups=groups, gate=rng.choice(["none", "row", "channel", "token"]),
                tanh=rng.random() < 0.4, scale=rng.random() < 0.6, post=rng.random() < 0.7, pre=rng.random() < 0.8, rms=rng.random() < 0.4,
                alpha=rng.choice([1.0, 1.0, 2.5]))


def _lengths(n, lo, hi, step):
    """n lengths over [lo, hi], the longest first"""
    return [hi - (i * step) % (hi - lo + 1) for i in range(n)]


def _geometry(c):
    ql, sl = _lengths(c["b"], c["lq_lo"], c["lq"], 29), _lengths(c["b"], c["s_lo"], c["s"], 37)
    if not c["packed"]:
        ql = [c["lq"]] * c["b"]
    return ql, sl


def _elem(c):
    return 4 if c["dtype"] == "fp32" else 2


def work(case):
    c, e = case, _elem(case)
    if c["op"] == "xattn":
        ql, sl = _geometry(c)
        rq, rk = sum(ql), sum(sl)
        pairs = sum(a * b for a, b in zip(ql, sl))
        q, kv, lse = rq * c["heads"] * c["hd"] * e, rk * c["kv_heads"] * c["hd"] * e, rq * c["heads"] * 4
        fwd = 2 * q + 2 * kv + lse
        # the backward pass meets the forward's inputs again as the same data: read once for the training step
        return {"bytes": fwd + (2 * q + 2 * kv if c["train"] else 0), "flops": (14 if c["train"] else 4) * pairs * c["heads"] * c["hd"]}
    if c["op"] == "rope":
        n = c["rows"] * c["heads"] * c["hd"]
        ways = 2 if c["train"] else 1
        return {"bytes": ways * 2 * n * e + c["pos_rows"] * len(c["sections"].split(",")) * 4, "flops": ways * 3 * n}
    n = c["rows"] * c["d"]
    tensors = 2 + 1 + int(c["pre"])
    if c["train"]:
        tensors += 1 + int(c["pre"]) + 2
    small = {"none": 0, "row": c["groups"], "token": c["rows"], "channel": c["groups"] * c["d"]}[c["gate"]] * 4
    return {"bytes": tensors * n * e + small * (2 if c["train"] else 1), "flops": n * (40 if c["train"] else 15)}


# ------------------------------------------------------------------------------------------------- what a program has in hand
def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(int(seed) % (1 << 60) + 1)
    dt = FP32 if c["dtype"] == "fp32" else BF16

    def rnd(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)

    s = dict(c)
    if c["op"] == "xattn":
        ql, sl = _geometry(c)
        b, dq, dk = c["b"], c["heads"] * c["hd"], c["kv_heads"] * c["hd"]
        if c["packed"]:                    # the packed row counts are whole tiles: rows behind the last sequence belong to nobody
            rows_q, rows_kv = (sum(ql) + 63) // 64 * 64, (sum(sl) + 63) // 64 * 64
            s["cu_q"] = torch.tensor([0] + ql, device="cuda").cumsum(0).to(torch.int32)
            s["cu_kv"] = torch.tensor([0] + sl, device="cuda").cumsum(0).to(torch.int32)
            s["kv_len"] = None
        else:
            rows_q, rows_kv = b * c["lq"], b * c["s"]
            s["cu_q"] = s["cu_kv"] = None
            s["kv_len"] = None if min(sl) == c["s"] else torch.tensor(sl, device="cuda", dtype=torch.int32)
        rows_kv = max(rows_kv, 1)
        s["q"] = rnd(rows_q, dq)
        kv = rnd(rows_kv, 2 * dk)          # one projection makes both
        s["k"], s["v"] = kv[:, :dk], kv[:, dk:]
        s["key_mask"] = (torch.rand(rows_kv, device="cuda", generator=g) >= c["mask"]) if c["mask"] else None
        s["scale"] = c["hd"] ** -0.5
        if c["train"]:
            s["dout"] = rnd(rows_q, dq)
    elif c["op"] == "rope":
        s["sections"] = [int(n) for n in c["sections"].split(",")]
        width, axes = c["heads"] * c["hd"], len(s["sections"])
        buf = rnd(c["rows"], width + c["extra"] * c["hd"])
        s["x"] = buf[:, :width]
        if c["frac"]:
            s["pos"] = torch.rand(c["pos_rows"], axes, device="cuda", generator=g) * c["far"]
        else:
            s["pos"] = torch.randint(0, c["far"], (c["pos_rows"], axes), device="cuda", generator=g, dtype=torch.int32)
        if c["train"]:
            s["dy"] = rnd(c["rows"], width)
    else:
        rows, d = c["rows"], c["d"]
        s["x"], s["y"] = rnd(rows, d, scale=2.0), rnd(rows, d)
        vec = lambda mid: mid + 0.2 * torch.randn(d, device="cuda", generator=g)  # noqa: E731
        bias = lambda: None if c["rms"] else vec(0.0)  # noqa: E731
        s["post"] = (vec(1.0), bias()) if c["post"] else None
        s["pre"] = (vec(1.0), bias()) if c["pre"] else None
        s["scale"] = vec(0.5) if c["scale"] else None
        shape = {"none": None, "row": (c["groups"],), "token": (rows,), "channel": (c["groups"], d)}[c["gate"]]
        s["gate"] = None if shape is None else torch.randn(*shape, device="cuda", generator=g)
        if c["train"]:
            s["dx_out"] = rnd(rows, d)
            s["dn"] = rnd(rows, d) if c["pre"] else None
    return s


# ------------------------------------------------------------------------------------------------- plain forms
def _padded(s, ql_max, sl_max):
    """index [b, Lmax] and validity of every query / key slot"""
    dev, b = s["q"].device, s["b"]
    rq, rk = s["q"].shape[0], s["k"].shape[0]
    aq, ak = torch.arange(ql_max, device=dev), torch.arange(sl_max, device=dev)
    if s["packed"]:
        q0, qn = s["cu_q"][:-1].long(), (s["cu_q"][1:] - s["cu_q"][:-1]).long()
        k0, kn = s["cu_kv"][:-1].long(), (s["cu_kv"][1:] - s["cu_kv"][:-1]).long()
    else:
        q0, k0 = torch.arange(b, device=dev) * s["lq"], torch.arange(b, device=dev) * s["s"]
        qn = torch.full((b,), s["lq"], device=dev)
        kn = torch.full((b,), s["s"], device=dev) if s["kv_len"] is None else s["kv_len"].long()
    qi, qok = (q0[:, None] + aq).clamp(max=rq - 1), aq < qn[:, None]
    ki, kok = (k0[:, None] + ak).clamp(max=rk - 1), ak < kn[:, None]
    if s["key_mask"] is not None:
        kok = kok & s["key_mask"][ki]
    return qi, qok, ki, kok


def _xattn_plain(s):
    H, G, hd, b = s["heads"], s["kv_heads"], s["hd"], s["b"]
    qi, qok, ki, kok = _padded(s, s["lq"], max(s["s"], 1))
    Lq, S = qi.shape[1], ki.shape[1]
    rep = H // G
    zq, zk = qok[:, :, None], kok[:, :, None]
    q = torch.where(zq, s["q"].float()[qi], 0.0).view(b, Lq, G, rep, hd).permute(0, 2, 3, 1, 4).reshape(b, G, rep * Lq, hd)
    k = torch.where(zk, s["k"].float()[ki], 0.0).view(b, S, G, hd).permute(0, 2, 1, 3).contiguous()
    v = torch.where(zk, s["v"].float()[ki], 0.0).view(b, S, G, hd).permute(0, 2, 1, 3).contiguous()
    sc = torch.matmul(q, k.transpose(2, 3)) * s["scale"]
    sc = sc.masked_fill(~kok[:, None, None, :], -math.inf)
    m = sc.amax(3, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p = torch.exp(sc - m)
    l = p.sum(3, keepdim=True)
    lse_p = (m + torch.log(l)).view(b, H, Lq)
    p = p / torch.where(l == 0, 1.0, l)
    o = torch.matmul(p, v)

    def rows_of(t):                       # [b, G, rep * Lq, hd] -> the query rows, zero where nobody owns the row
        full = torch.zeros_like(s["q"])
        full[qi[qok]] = t.view(b, G, rep, Lq, hd).permute(0, 3, 1, 2, 4).reshape(b, Lq, H * hd)[qok].to(full.dtype)
        return full

    out = rows_of(o)
    lse = torch.full((H, s["q"].shape[0]), -math.inf, device=out.device)
    lse[:, qi[qok]] = lse_p.permute(1, 0, 2)[:, qok]
    if not s["train"]:
        return out, lse
    do = torch.where(zq, s["dout"].float()[qi], 0.0).view(b, Lq, G, rep, hd).permute(0, 2, 3, 1, 4).reshape(b, G, rep * Lq, hd)
    delta = (do * o).sum(3, keepdim=True)
    dv = torch.matmul(p.transpose(2, 3), do)
    ds = p * (torch.matmul(do, v.transpose(2, 3)) - delta) * s["scale"]
    dq = rows_of(torch.matmul(ds, k))
    dk = torch.matmul(ds.transpose(2, 3), q)
    real = kok

    def kv_rows(t):
        full = torch.zeros(s["k"].shape, device=out.device, dtype=s["k"].dtype)
        full[ki[real]] = t.permute(0, 2, 1, 3).reshape(b, S, G * hd)[real].to(full.dtype)
        return full

    return out, lse, dq, kv_rows(dk), kv_rows(dv)


def _frequencies(c, dev):
    """(frequency in 64 bits, axis) of every pair"""
    n = torch.tensor(c["sections"], device=dev)
    axis = torch.repeat_interleave(torch.arange(len(c["sections"]), device=dev), n)
    P = int(sum(c["sections"]))
    p = torch.arange(P, device=dev, dtype=torch.float64)
    if c["joint"]:
        return 10000.0 ** (-p / P), axis
    first = (torch.cumsum(n, 0) - n)[axis].double()
    return 10000.0 ** (-(p - first) / n[axis].double()), axis


def _rotate(c, x, ang, sign, wide):
    P, heads, hd = ang.shape[1], c["heads"], c["hd"]
    rep = x.shape[0] // ang.shape[0]
    cos, sin = ang.cos().to(wide).repeat(rep, 1)[:, None], (sign * ang.sin()).to(wide).repeat(rep, 1)[:, None]
    h = x.to(wide).reshape(x.shape[0], heads, hd)
    if c["interleaved"]:
        a, b = h[..., 0:2 * P:2], h[..., 1:2 * P:2]
        r = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(2)
    else:
        a, b = h[..., :P], h[..., P:2 * P]
        r = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((r, h[..., 2 * P:]), -1).reshape(x.shape[0], heads * hd)


def _rope_plain(s):
    f, axis = _frequencies(s, s["x"].device)
    ang = s["pos"].double()[:, axis] * f
    y = _rotate(s, s["x"], ang, 1.0, FP32).to(s["x"].dtype)
    if not s["train"]:
        return (y,)
    return y, _rotate(s, s["dy"], ang, -1.0, FP32).to(s["x"].dtype)


def _norm(x, rms, eps=1e-5):
    mu = 0.0 if rms else x.mean(1, keepdim=True)
    c = x - mu
    r = torch.rsqrt((c * c).mean(1, keepdim=True) + eps)
    return c * r, r


def _norm_grad(g, xhat, r, rms):
    t = g - xhat * (g * xhat).mean(1, keepdim=True)
    return r * (t if rms else t - g.mean(1, keepdim=True))


def _join_formula(s, wide):
    rms, rows, d = s["rms"], s["rows"], s["d"]
    W = lambda t: None if t is None else t.to(wide)  # noqa: E731
    x, y, gate, scale = W(s["x"]), W(s["y"]), W(s["gate"]), W(s["scale"])
    hat, p, r_post = None, y, None
    if s["post"] is not None:
        w1, b1 = W(s["post"][0]), W(s["post"][1])
        hat, r_post = _norm(y, rms)
        p = hat * w1 if b1 is None else hat * w1 + b1
    g = act = None
    if gate is not None:
        act = torch.tanh(gate) if s["tanh"] else gate
        g = act.repeat_interleave(rows // act.shape[0], 0)
        g = g[:, None] if g.dim() == 1 else g
    t = p if g is None else p * g
    t = t if scale is None else t * scale
    x_out = s["alpha"] * x + t
    n = xhat = r_pre = w2 = None
    if s["pre"] is not None:
        w2, b2 = W(s["pre"][0]), W(s["pre"][1])
        xhat, r_pre = _norm(x_out, rms)
        n = xhat * w2 if b2 is None else xhat * w2 + b2
    dt = wide if wide == torch.float64 else s["x"].dtype
    out = [x_out.to(dt)] + ([] if n is None else [n.to(dt)])
    if not s["train"]:
        return tuple(out)
    G = W(s["dx_out"])
    if n is not None:
        dn = W(s["dn"])
        G = G + _norm_grad(dn * w2, xhat, r_pre, rms)
    q = G if scale is None else G * scale
    dp = q if g is None else q * g
    dy = dp if hat is None else _norm_grad(dp * w1, hat, r_post, rms)
    out += [(s["alpha"] * G).to(dt), dy.to(dt)]
    if hat is not None:
        out.append((dp * hat).sum(0))
        if not rms:
            out.append(dp.sum(0))
    if gate is not None:
        e = q * p
        e = (e.sum(1) if act.dim() == 1 else e).reshape(act.shape[0], rows // act.shape[0], *act.shape[1:]).sum(1)
        out.append(e * (1 - act * act) if s["tanh"] else e)
    if scale is not None:
        out.append((G * p if g is None else G * g * p).sum(0))
    if n is not None:
        out.append((dn * xhat).sum(0))
        if not rms:
            out.append(dn.sum(0))
    return tuple(out)


# ------------------------------------------------------------------------------------------------- a pass
def _run_own(s):
    from declip_amd import ops
    if s["op"] == "xattn":
        shape = dict(kv_heads=s["kv_heads"], batch=s["b"], cu_q=s["cu_q"], cu_kv=s["cu_kv"], kv_len=s["kv_len"], key_mask=s["key_mask"], scale=s["scale"],
                     max_q=s["lq"], max_kv=s["s"])
        out, lse = ops.xattn_fwd(s["q"], s["k"], s["v"], s["heads"], **shape)
        if not s["train"]:
            return out, lse
        return (out, lse, *ops.xattn_bwd(s["q"], s["k"], s["v"], out, s["dout"], lse, s["heads"], **shape))
    if s["op"] == "rope":
        how = dict(joint=s["joint"], interleaved=s["interleaved"])
        y = ops.rope_axes(s["x"], s["pos"], s["heads"], s["sections"], **how)
        if not s["train"]:
            return (y,)
        return y, ops.rope_axes(s["dy"], s["pos"], s["heads"], s["sections"], inverse=True, **how)
    how = dict(post=s["post"], gate=s["gate"], scale=s["scale"], pre=s["pre"], alpha=s["alpha"], rms=s["rms"], gate_tanh=s["tanh"])
    x_out, n, stats = ops.join_norm_fwd(s["x"], s["y"], **how)
    out = [x_out] + ([] if n is None else [n])
    if not s["train"]:
        return tuple(out)
    dx, dy, grads = ops.join_norm_bwd(s["x"], s["y"], s["dx_out"], s["dn"], stats, **how)
    out += [dx, dy] + [t for t in grads if t is not None]
    return tuple(out)


def run(state):
    if own:
        return _run_own(state)
    if state["op"] == "xattn":
        return _xattn_plain(state)
    if state["op"] == "rope":
        return _rope_plain(state)
    return _join_formula(state, FP32)


# ------------------------------------------------------------------------------------------------- the definition in 64 bits
def _xattn_exact(s):
    H, G, hd = s["heads"], s["kv_heads"], s["hd"]
    F64 = torch.float64
    dev, rq, rk = s["q"].device, s["q"].shape[0], s["k"].shape[0]
    ql, sl = _geometry(s)
    out, lse = torch.zeros(rq, H, hd, device=dev, dtype=F64), torch.full((H, rq), -math.inf, device=dev, dtype=F64)
    dq, dk, dv = torch.zeros_like(out), torch.zeros(rk, G, hd, device=dev, dtype=F64), torch.zeros(rk, G, hd, device=dev, dtype=F64)
    q0 = k0 = 0
    for i in range(s["b"]):
        if not s["packed"]:
            q0, k0 = i * s["lq"], i * s["s"]
        a, e = slice(q0, q0 + ql[i]), slice(k0, k0 + sl[i])
        q0, k0 = q0 + ql[i], k0 + sl[i]
        live = torch.arange(e.start, e.stop, device=dev)
        if s["key_mask"] is not None:
            live = live[s["key_mask"][e]]
        if live.numel() == 0:
            continue
        for h in range(H):
            c, kc = slice(h * hd, (h + 1) * hd), slice(h // (H // G) * hd, (h // (H // G) + 1) * hd)
            q, k, v = s["q"][a, c].to(F64), s["k"][live][:, kc].to(F64), s["v"][live][:, kc].to(F64)
            z = q @ k.T * s["scale"]
            lse[h, a] = torch.logsumexp(z, 1)
            p = torch.softmax(z, 1)
            o = p @ v
            out[a, h] = o
            if s["train"]:
                do = s["dout"][a, c].to(F64)
                ds = p * (do @ v.T - (do * o).sum(1, keepdim=True)) * s["scale"]
                dq[a, h] = ds @ k
                dk[live, h // (H // G)] += ds.T @ q
                dv[live, h // (H // G)] += p.T @ do
    out = out.view(rq, H * hd)
    if not s["train"]:
        return out, lse
    return out, lse, dq.view(rq, H * hd), dk.view(rk, G * hd), dv.view(rk, G * hd)


def _rope_exact(s):
    """every pair as a complex number, turned by the angle of its position"""
    F64, P, heads, hd = torch.float64, sum(s["sections"]), s["heads"], s["hd"]
    pos, cols, i = s["pos"].to(F64), [], 0
    for a, n in enumerate(s["sections"]):
        for j in range(n):
            cols.append(pos[:, a] * 10000.0 ** (-(i / P if s["joint"] else j / n)))
            i += 1
    turn = torch.polar(torch.ones((), dtype=F64, device=pos.device), torch.stack(cols, 1))
    turn = turn[torch.arange(s["rows"], device=pos.device) % pos.shape[0]][:, None]

    def turned(x, by):
        h = x.to(F64).reshape(s["rows"], heads, hd).clone()
        one, two = (slice(0, 2 * P, 2), slice(1, 2 * P, 2)) if s["interleaved"] else (slice(0, P), slice(P, 2 * P))
        z = torch.complex(h[..., one].contiguous(), h[..., two].contiguous()) * by
        h[..., one], h[..., two] = z.real, z.imag
        return h.view(s["rows"], heads * hd)

    y = turned(s["x"], turn)
    return (y, turned(s["dy"], turn.conj())) if s["train"] else (y,)


def _join_exact(s):
    """torch's own derivative of the forward's definition in 64 bits"""
    F64 = torch.float64
    leaf = lambda t: None if t is None else t.detach().to(F64).requires_grad_(True)  # noqa: E731
    x, y, gate, scale = leaf(s["x"]), leaf(s["y"]), leaf(s["gate"]), leaf(s["scale"])
    post = None if s["post"] is None else [leaf(t) for t in s["post"]]
    pre = None if s["pre"] is None else [leaf(t) for t in s["pre"]]

    def norm(v, w, b):
        var = (v * v).mean(1, keepdim=True) if s["rms"] else v.var(1, unbiased=False, keepdim=True)
        v = v if s["rms"] else v - v.mean(1, keepdim=True)
        v = v / torch.sqrt(var + 1e-5) * w
        return v if b is None else v + b

    t = y if post is None else norm(y, *post)
    if gate is not None:
        g = torch.tanh(gate) if s["tanh"] else gate
        where = torch.arange(s["rows"], device=x.device) // (s["rows"] // g.shape[0])
        t = t * (g[where] if g.dim() == 2 else g[where].unsqueeze(1))
    if scale is not None:
        t = t * scale
    x_out = s["alpha"] * x + t
    n = None if pre is None else norm(x_out, *pre)
    outs = [x_out] + ([] if n is None else [n])
    if not s["train"]:
        return tuple(o.detach() for o in outs)
    total = (x_out * s["dx_out"].to(F64)).sum()
    if n is not None:
        total = total + (n * s["dn"].to(F64)).sum()
    leaves = [x, y] + [t for t in (post or []) if t is not None] + [t for t in (gate, scale) if t is not None] + [t for t in (pre or []) if t is not None]
    return tuple(o.detach() for o in outs) + torch.autograd.grad(total, leaves)


def exact(case, seed):
    s = prepare(case, seed)
    return {"xattn": _xattn_exact, "rope": _rope_exact, "join": _join_exact}[s["op"]](s)
