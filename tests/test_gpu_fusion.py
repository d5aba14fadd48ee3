"""The operators between the towers (cross attention, multi-axis rotary positions, block-boundary norms) against their definitions in 64
bits (tests/fusion_ref.py: value and bound of every element)."""
import math

import pytest
import torch

import fusion_ref as R

pytestmark = pytest.mark.gpu

cuda = torch.device("cuda")
BF16, F32 = torch.bfloat16, torch.float32
NAN, INF = float("nan"), float("inf")


def _ops():
    from declip_amd import ops
    return ops


def rnd(*shape, seed=0, dtype=F32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def check(got, value, bound, name):
    got = got.detach().cpu().double().reshape(value.shape)
    fin = torch.isfinite(value)
    assert torch.equal(torch.isfinite(got), fin) and torch.equal(got[~fin], value[~fin]), name + ": infinities or NaN"
    off = (got - value).abs()[fin] - bound.expand_as(value)[fin] - 1e-30
    worst = ((got - value).abs()[fin] / (bound.expand_as(value)[fin] + 1e-30)).max() if off.numel() else 0
    assert not off.numel() or float(off.max()) <= 0, "%s: %.3g times its bound" % (name, float(worst))


def dev(t):
    return t.to(cuda) if torch.is_tensor(t) else t


# ----------------------------------------------------------------------------- cross attention
def geometry(b, lq, s, packed, seed=0, lo_q=1, lo_s=0, extra=0):
    """(rows_q, rows_kv, arguments) of b sequences with lq / s rows at most"""
    g = torch.Generator().manual_seed(seed)
    if not packed:
        kv_len = torch.randint(lo_s, s + 1, (b,), generator=g).int()
        kv_len[0] = s
        return b * lq, b * s, dict(batch=b, kv_len=kv_len)
    ql, sl = torch.randint(lo_q, lq + 1, (b,), generator=g), torch.randint(lo_s, s + 1, (b,), generator=g)
    ql[0], sl[0] = lq, s
    cu_q, cu_kv = (torch.cat([torch.tensor([extra]), extra + n.cumsum(0)]).int() for n in (ql, sl))
    return int(cu_q[-1]) + extra, int(cu_kv[-1]) + extra, dict(cu_q=cu_q, cu_kv=cu_kv)


def xattn_case(dtype, heads, kv_heads, hd, rows_q, rows_kv, kw, seed=1, mask=0.0, scale=None, grads=True, poison=True):
    """runs forward and backward, checks every element; k, v, out rows that nobody reads hold NaN"""
    ops = _ops()
    q, dout = rnd(rows_q, heads * hd, seed=seed, dtype=dtype), rnd(rows_q, heads * hd, seed=seed + 1, dtype=dtype)
    kv = rnd(rows_kv, 2 * kv_heads * hd, seed=seed + 2, dtype=dtype)
    w = kv_heads * hd
    kw = dict(kw, kv_heads=kv_heads, scale=scale)
    if mask:
        kw["key_mask"] = torch.rand(rows_kv, generator=torch.Generator().manual_seed(seed + 3)) >= mask
    ref = R.xattn(q, kv[:, :w], kv[:, w:], heads, dout, **kw)
    if poison:
        batch = kw.get("batch") or (kw["cu_q"] if "cu_q" in kw else kw["cu_kv"]).numel() - 1
        used = torch.zeros(rows_kv, dtype=torch.bool)
        for i, (k0, n) in enumerate(R.lengths(kw.get("cu_kv"), rows_kv, batch)):
            used[k0:k0 + (n if kw.get("kv_len") is None else min(n, int(kw["kv_len"][i])))] = True
        if mask:
            used &= kw["key_mask"]
        kv[~used] = torch.tensor([NAN, INF, -INF, torch.finfo(dtype).min]).to(dtype).repeat(kv.shape[1] // 4)
    kd = kv.to(cuda)
    args = {n: dev(t) for n, t in kw.items()}
    out, lse = ops.xattn_fwd(q.to(cuda), kd[:, :w], kd[:, w:], heads, **args)
    check(out, *ref["out"], "out")
    check(lse, *ref["lse"], "lse")
    if grads:
        got = ops.xattn_bwd(q.to(cuda), kd[:, :w], kd[:, w:], out, dout.to(cuda), lse, heads, **args)
        for name, t in zip(("dq", "dk", "dv"), got):
            check(t, *ref[name], name)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads,kv_heads,hd,b,lq,s,packed,mask", [
    (2, 2, 64, 3, 77, 197, True, 0.0), (4, 2, 64, 2, 50, 70, False, 0.3), (4, 1, 32, 3, 33, 65, True, 0.5), (2, 2, 80, 2, 20, 129, True, 0.0),
    (3, 3, 96, 2, 5, 64, False, 0.0), (2, 1, 128, 2, 130, 63, True, 0.2), (1, 1, 8, 1, 1, 1, False, 0.0), (8, 2, 40, 2, 1, 300, False, 0.1),
    (2, 2, 64, 1, 129, 1, False, 0.0), (2, 2, 24, 4, 2, 3, True, 0.5), (6, 3, 64, 5, 31, 33, True, 0.0)])
def test_xattn(dtype, heads, kv_heads, hd, b, lq, s, packed, mask):
    xattn_case(dtype, heads, kv_heads, hd, *geometry(b, lq, s, packed, seed=lq), mask=mask)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_xattn_rows_without_owner_are_zero_and_tables_may_start_late(dtype):
    xattn_case(dtype, 2, 2, 64, *geometry(3, 40, 50, True, seed=4, extra=7))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("what", ["no_keys", "all_masked", "no_queries"])
def test_xattn_empty(dtype, what):
    ops = _ops()
    q, kv = rnd(6, 64, seed=1, dtype=dtype).to(cuda), torch.full((8, 64), NAN, dtype=dtype, device=cuda)
    kw = dict(batch=2)
    if what == "no_keys":
        kv = kv[:0]
    elif what == "all_masked":
        kw["key_mask"] = torch.zeros(8, dtype=torch.uint8, device=cuda)
    else:
        q, kv = q[:0], torch.ones_like(kv)
    out, lse = ops.xattn_fwd(q, kv, kv, 1, **kw)
    dq, dk, dv = ops.xattn_bwd(q, kv, kv, out, torch.full_like(out, NAN), lse, 1, **kw)
    assert bool((out == 0).all()) and bool((lse == -INF).all())
    for t in (dq, dk, dv):
        assert bool((t == 0).all())
    assert dk.shape == kv.shape and dq.shape == q.shape


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads,kv_heads,hd,b,lq,s", [(8, 8, 64, 4, 1, 50), (16, 4, 64, 3, 1, 3000), (4, 4, 128, 1, 2, 5001), (6, 2, 80, 2, 1, 1025), (4, 1, 32, 1, 7, 700)])
def test_xattn_single_tokens_over_long_keys(dtype, heads, kv_heads, hd, b, lq, s):
    """few rows: the key axis is split over blocks and joined"""
    xattn_case(dtype, heads, kv_heads, hd, *geometry(b, lq, s, False, seed=s), mask=0.1, grads=False)
    xattn_case(dtype, heads, kv_heads, hd, *geometry(b, lq, s, True, seed=s), grads=False)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads,kv_heads,hd,b,lq,s,packed,mask", [
    (2, 2, 64, 1, 600, 50, False, 0.2), (2, 1, 64, 2, 700, 40, True, 0.0), (2, 2, 128, 3, 77, 100, True, 0.0), (2, 1, 128, 2, 200, 300, True, 0.1), (3, 3, 96, 2, 150, 260, False, 0.0),
    (1, 1, 128, 1, 300, 1500, False, 0.3), (2, 2, 64, 1, 150, 2100, True, 0.0), (4, 1, 64, 1, 70, 3100, False, 0.1), (2, 2, 32, 2, 900, 300, True, 0.0), (2, 2, 72, 1, 129, 700, False, 0.0)])
def test_xattn_block_shapes_and_split_axes(dtype, heads, kv_heads, hd, b, lq, s, packed, mask):
    """1 to 8 waves per block, the other axis whole and in ranges, for each of the three kernels"""
    xattn_case(dtype, heads, kv_heads, hd, *geometry(b, lq, s, packed, seed=lq + s), mask=mask)


def test_xattn_rows_far_apart():
    """element offsets beyond 2^31: the rows of a long cache, 2^21 elements apart"""
    ops = _ops()
    rows_q, rows_kv, ld, w = 1040, 1100, 1 << 21, 128
    q, k, v, dout = (rnd(n, w, seed=i, dtype=BF16) for i, n in enumerate((rows_q, rows_kv, rows_kv, rows_q)))
    ref = R.xattn(q, k, v, 2, dout, batch=1)
    cache = torch.empty(rows_kv, ld, dtype=BF16, device=cuda)
    cache[:, 256:256 + w], cache[:, ld - w:] = k.to(cuda), v.to(cuda)
    far = torch.empty(rows_q, ld, dtype=BF16, device=cuda)
    far[:, 8:8 + w], far[:, 512:512 + w] = q.to(cuda), dout.to(cuda)
    qd, dd, kd, vd = far[:, 8:8 + w], far[:, 512:512 + w], cache[:, 256:256 + w], cache[:, ld - w:]
    out, lse = ops.xattn_fwd(qd, kd, vd, 2, batch=1)
    check(out, *ref["out"], "out")
    for name, t in zip(("dq", "dk", "dv"), ops.xattn_bwd(qd, kd, vd, out, dd, lse, 2, batch=1)):
        check(t, *ref[name], name)
    pos = torch.arange(rows_q, dtype=torch.int32)[:, None].contiguous()
    y = ops.rope_axes(qd, pos.to(cuda), 2, (32,))
    check(y, *R.rope(q, pos, 2, (32,)), "rope")


def test_xattn_split_ranges_without_a_key():
    """whole ranges of the split key axis are masked, one sequence has nothing but masked keys"""
    ops = _ops()
    q, k, v = rnd(2, 64, seed=1, dtype=BF16), rnd(2 * 4000, 64, seed=2, dtype=BF16), rnd(2 * 4000, 64, seed=3, dtype=BF16)
    mask = torch.zeros(2, 4000, dtype=torch.bool)
    mask[0, 3990] = True
    ref = R.xattn(q, k, v, 1, batch=2, key_mask=mask)
    out, lse = ops.xattn_fwd(q.to(cuda), k.to(cuda), v.to(cuda), 1, batch=2, key_mask=mask.to(cuda))
    check(out, *ref["out"], "out")
    check(lse, *ref["lse"], "lse")
    assert bool((out[1] == 0).all()) and float(lse[0, 1]) == -INF


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_xattn_large_scores(dtype):
    """peaked and far-off scores: the running maximum moves from tile to tile"""
    ops = _ops()
    q, v = rnd(40, 64, seed=1, dtype=dtype, scale=6.0), rnd(300, 64, seed=3, dtype=dtype)
    k = (rnd(300, 64, seed=2, scale=6.0) * torch.linspace(0.1, 1.0, 300)[:, None]).to(dtype)
    dout = rnd(40, 64, seed=4, dtype=dtype)
    ref = R.xattn(q, k, v, 1, dout, batch=1)
    qd, kd, vd = q.to(cuda), k.to(cuda), v.to(cuda)
    out, lse = ops.xattn_fwd(qd, kd, vd, 1, batch=1)
    check(out, *ref["out"], "out")
    check(lse, *ref["lse"], "lse")
    for name, t in zip(("dq", "dk", "dv"), ops.xattn_bwd(qd, kd, vd, out, dout.to(cuda), lse, 1, batch=1)):
        check(t, *ref[name], name)


def test_xattn_lengths_beyond_the_hint_and_strided_rows():
    """max_q / max_kv only lay out the grid; q, dout and the key rows have strides of their own"""
    ops = _ops()
    rows_q, rows_kv, kw = geometry(2, 300, 290, True, seed=5)
    wide_q, wide_d = rnd(rows_q, 3 * 128, seed=1, dtype=BF16), rnd(rows_q, 2 * 128, seed=2, dtype=BF16)
    wide_k = rnd(rows_kv, 4 * 128, seed=3, dtype=BF16)
    q, dout, k, v = wide_q[:, 128:256], wide_d[:, :128], wide_k[:, 256:384], wide_k[:, :128]
    ref = R.xattn(q, k, v, 2, dout, scale=0.05, **kw)
    dq_, dd_, dk_ = wide_q.to(cuda), wide_d.to(cuda), wide_k.to(cuda)
    q, dout, k, v = dq_[:, 128:256], dd_[:, :128], dk_[:, 256:384], dk_[:, :128]
    args = dict({n: dev(t) for n, t in kw.items()}, max_q=3, max_kv=5, scale=0.05)
    out, lse = ops.xattn_fwd(q, k, v, 2, **args)
    check(out, *ref["out"], "out")
    for name, t in zip(("dq", "dk", "dv"), ops.xattn_bwd(q, k, v, out, dout, lse, 2, **args)):
        check(t, *ref[name], name)


def test_xattn_tables_out_of_range_stay_inside():
    """entries beyond the row counts are clamped, descending ones own nothing: wrong tables give wrong rows, never a foreign access"""
    ops = _ops()
    q, kv = rnd(64, 64, seed=1, dtype=BF16).to(cuda), rnd(96, 64, seed=2, dtype=BF16).to(cuda)
    cu = torch.tensor([0, 64], dtype=torch.int32, device=cuda)
    far = torch.tensor([-5, 2_000_000_000], dtype=torch.int32, device=cuda)
    out, lse = ops.xattn_fwd(q, kv, kv, 1, cu_q=far, cu_kv=far, kv_len=torch.tensor([-3], dtype=torch.int32, device=cuda))
    assert bool((out == 0).all())
    out, lse = ops.xattn_fwd(q, kv, kv, 1, cu_q=far, cu_kv=far, kv_len=torch.tensor([1 << 30], dtype=torch.int32, device=cuda))
    want, lse2 = ops.xattn_fwd(q, kv, kv, 1, cu_q=cu, cu_kv=torch.tensor([0, 96], dtype=torch.int32, device=cuda))
    assert torch.equal(out, want) and torch.equal(lse, lse2)
    ops.xattn_bwd(q, kv, kv, out, out, lse, 1, cu_q=far, cu_kv=torch.tensor([90, 3], dtype=torch.int32, device=cuda))
    torch.cuda.synchronize()


def test_xattn_same_bits_on_every_run():
    ops = _ops()
    rows_q, rows_kv, kw = geometry(4, 200, 500, True, seed=6)
    q, k, v, d = (rnd(n, 4 * 64, seed=i, dtype=BF16).to(cuda) for i, n in enumerate((rows_q, rows_kv, rows_kv, rows_q)))
    args = {n: dev(t) for n, t in kw.items()}
    out, lse = ops.xattn_fwd(q, k, v, 4, **args)
    first = (out, lse, *ops.xattn_bwd(q, k, v, out, d, lse, 4, **args))
    for _ in range(3):
        o, l = ops.xattn_fwd(q, k, v, 4, **args)
        for a, b in zip(first, (o, l, *ops.xattn_bwd(q, k, v, o, d, l, 4, **args))):
            assert torch.equal(a, b)


# ----------------------------------------------------------------------------- rotary positions
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,pos_rows,heads,hd,sections,joint,interleaved,frac,far", [
    (1568, 1568, 12, 64, (8, 12, 12), False, False, False, 32), (37, 37, 3, 64, (8, 12, 12), True, False, False, 1_000_000), (12, 4, 2, 80, (16, 16), False, True, True, 64),
    (1, 1, 1, 128, (64,), False, False, False, 5), (9, 9, 5, 32, (3, 5), False, True, False, 100), (10, 5, 2, 40, (3, 4), True, False, True, 50),
    (3000, 1000, 2, 96, (12, 12, 12), True, True, False, 2_000_000_000), (7, 7, 1, 6, (1, 1, 1), False, False, False, 9), (5, 5, 2, 256, (64, 64), False, False, False, 999)])
def test_rope_axes(dtype, rows, pos_rows, heads, hd, sections, joint, interleaved, frac, far):
    ops = _ops()
    x = rnd(rows, heads * hd, seed=rows, dtype=dtype)
    g = torch.Generator().manual_seed(1)
    n = len(sections)
    pos = torch.rand(pos_rows, n, generator=g) * far if frac else torch.randint(-far if far < 1000 else 0, far, (pos_rows, n), generator=g, dtype=torch.int32)
    for inverse in (False, True):
        kw = dict(joint=joint, interleaved=interleaved, inverse=inverse)
        y = ops.rope_axes(x.to(cuda), pos.to(cuda), heads, sections, **kw)
        check(y, *R.rope(x, pos, heads, sections, **kw), "rope")


def test_rope_axes_strided_in_place_and_bases():
    """the q and k columns of a fused projection, rotated in place, v untouched; a base per axis; odd strides"""
    ops = _ops()
    qkv = rnd(50, 3 * 128, seed=1, dtype=BF16)
    pos = torch.randint(0, 20, (50, 2), dtype=torch.int32)
    ref = R.rope(qkv[:, :256].contiguous(), pos, 4, (16, 16), theta=[100.0, 10000.0])
    buf = qkv.to(cuda)
    got = ops.rope_axes(buf[:, :256], pos.to(cuda), 4, (16, 16), theta=(100.0, 10000.0), out=buf[:, :256])
    assert got.data_ptr() == buf.data_ptr()
    check(buf[:, :256], *ref, "in place")
    assert torch.equal(buf[:, 256:].cpu(), qkv[:, 256:])
    odd = rnd(9, 67, seed=2)
    got = ops.rope_axes(odd.to(cuda)[:, 3:67], pos[:9].to(cuda), 1, (16, 16))
    check(got, *R.rope(odd[:, 3:67].contiguous(), pos[:9], 1, (16, 16)), "odd stride")


# ----------------------------------------------------------------------------- block boundary
JOINS = [  # rows, d, groups, gate, tanh, scale, post, bias, pre, rms, alpha
    (50, 768, 5, "channel", False, True, True, True, True, False, 1.0), (33, 512, 33, "row", True, False, True, True, True, True, 2.0),
    (1, 1024, 1, "row", False, True, True, False, True, False, 1.0), (20, 2048, 1, "none", False, True, True, True, False, False, 1.0),
    (9, 4096, 3, "row", True, True, False, True, True, False, 0.5), (6, 8192, 2, "channel", True, False, True, True, True, True, 1.0),
    (14, 33, 7, "row", False, True, True, True, True, False, 1.0), (5, 257, 1, "channel", False, False, True, False, True, False, 1.0),
    (4, 3001, 4, "row", False, False, False, True, True, True, 1.0), (2000, 264, 4, "row", False, True, True, True, True, False, 1.0),
    (1500, 96, 1500, "channel", False, True, False, True, False, False, 1.0), (3, 8191, 1, "none", False, True, True, True, True, False, 1.0), (6, 1, 2, "row", False, True, False, True, False, False, 1.0)]


def join_inputs(dtype, rows, d, groups, gate, scale, post, bias, pre, rms, seed=3):
    vec = lambda i, mid: mid + 0.2 * rnd(d, seed=seed + i)  # noqa: E731
    b = lambda i: vec(i, 0.0) if bias and not rms else None  # noqa: E731
    return dict(x=rnd(rows, d, seed=seed, dtype=dtype, scale=2.0), y=rnd(rows, d, seed=seed + 1, dtype=dtype)), dict(
        post=(vec(2, 1.0), b(3)) if post else None, pre=(vec(4, 1.0), b(5)) if pre else None, scale=vec(6, 0.5) if scale else None,
        gate={"none": None, "row": rnd(groups, seed=seed + 7), "channel": rnd(groups, d, seed=seed + 8)}[gate])


def on_gpu(kw):
    return {n: tuple(dev(t) for t in v) if isinstance(v, tuple) else dev(v) for n, v in kw.items()}


def join_check(dtype, xy, kw, how, dx_out, dn):
    ops = _ops()
    x, y = xy["x"], xy["y"]
    ref = R.join(x, y, **kw, **how, dx_out=dx_out, dn=dn)
    tol = R.join_bounds(ref, x, y, **kw, **how, dx_out=dx_out, dn=dn)
    x_out, n, stats = ops.join_norm_fwd(x.to(cuda), y.to(cuda), **on_gpu(kw), **how)
    check(x_out, ref["x_out"], tol["x_out"], "x_out")
    assert (n is None) == (kw["pre"] is None)
    if n is not None:
        check(n, ref["n"], tol["n"], "n")
    dx, dy, grads = ops.join_norm_bwd(x.to(cuda), y.to(cuda), None if dx_out is None else dx_out.to(cuda), None if dn is None else dn.to(cuda), stats, **on_gpu(kw), **how)
    for name, t in dict(dx=dx, dy=dy, **grads._asdict()).items():
        assert (t is None) == (name not in ref), name
        if t is not None:
            assert t.shape == ref[name].shape
            check(t, ref[name], tol[name], name)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("case", JOINS, ids=["%dx%d-%s" % (c[0], c[1], c[3]) for c in JOINS])
def test_join_norm(dtype, case):
    rows, d, groups, gate, tanh, scale, post, bias, pre, rms, alpha = case
    xy, kw = join_inputs(dtype, rows, d, groups, gate, scale, post, bias, pre, rms)
    how = dict(alpha=alpha, rms=rms, gate_tanh=tanh)
    dx_out, dn = rnd(rows, d, seed=20, dtype=dtype), rnd(rows, d, seed=21, dtype=dtype) if pre else None
    join_check(dtype, xy, kw, how, dx_out, dn)


@pytest.mark.parametrize("which", ["dn", "dx_out"])
def test_join_norm_one_gradient_only(which):
    xy, kw = join_inputs(BF16, 40, 768, 4, "row", True, True, True, True, False)
    g = rnd(40, 768, seed=20, dtype=BF16)
    join_check(BF16, xy, kw, {}, g if which == "dx_out" else None, g if which == "dn" else None)


def test_join_norm_unaligned_rows_and_same_bits():
    """addresses that rule 16-byte accesses out go element by element; a run repeats its bits"""
    ops = _ops()
    xy, kw = join_inputs(BF16, 300, 768, 6, "channel", True, True, True, True, False)
    a = ops.join_norm_fwd(xy["x"].to(cuda), xy["y"].to(cuda), **on_gpu(kw))
    shifted = torch.empty(300 * 768 + 1, dtype=BF16, device=cuda)[1:].view(300, 768)
    shifted.copy_(xy["x"])
    b = ops.join_norm_fwd(shifted, xy["y"].to(cuda), **on_gpu(kw))
    ref = R.join(xy["x"], xy["y"], **kw)
    tol = R.join_bounds(ref, xy["x"], xy["y"], **kw)
    check(b[0], ref["x_out"], tol["x_out"], "x_out")
    check(b[1], ref["n"], tol["n"], "n")
    g = rnd(300, 768, seed=9, dtype=BF16).to(cuda)
    runs = [ops.join_norm_bwd(xy["x"].to(cuda), xy["y"].to(cuda), g, g, a[2], **on_gpu(kw)) for _ in range(3)]
    for r in runs[1:]:
        for s, t in zip(runs[0][:2] + tuple(runs[0][2]), r[:2] + tuple(r[2])):
            assert torch.equal(s, t)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rms", [False, True])
def test_join_norm_rows_far_from_zero(dtype, rms):
    """rows whose mean is a thousand times their deviation, and rows of one value (their deviation is eps's)"""
    xy, kw = join_inputs(dtype, 40, 520, 4, "row", True, True, True, True, rms)
    far = torch.linspace(-2000, 2000, 40)[:, None]
    xy = {n: (t.float() + far).to(dtype) for n, t in xy.items()}
    xy["y"][7] = 3.0
    xy["x"][9], xy["y"][9] = 0.0, -0.0
    join_check(dtype, xy, kw, dict(rms=rms), rnd(40, 520, seed=20, dtype=dtype), rnd(40, 520, seed=21, dtype=dtype))


def test_join_norm_more_elements_than_31_bits():
    ops = _ops()
    rows, d = (1 << 18) + 3, 8192
    xy, kw = join_inputs(BF16, 4, d, 1, "row", True, True, True, True, False)
    some = torch.tensor([0, 1, rows - 2, rows - 1], device=cuda)
    full = {n: torch.zeros(rows, d, dtype=BF16, device=cuda).index_copy_(0, some, t.to(cuda)) for n, t in xy.items()}
    g = rnd(4, d, seed=20, dtype=BF16)
    gd = torch.zeros(rows, d, dtype=BF16, device=cuda).index_copy_(0, some, g.to(cuda))
    ref = R.join(**xy, **kw, dx_out=g, dn=g)
    tol = R.join_bounds(ref, **xy, **kw, dx_out=g, dn=g)
    x_out, n, stats = ops.join_norm_fwd(**full, **on_gpu(kw))
    dx, dy, grads = ops.join_norm_bwd(full["x"], full["y"], gd, gd, stats, **on_gpu(kw))
    for name, t in dict(x_out=x_out, n=n, dx=dx, dy=dy).items():
        check(t[some], ref[name], tol[name], name)
    for name in ("post_w", "pre_w", "gate", "scale"):        # (rows without a gradient add zeros)
        check(getattr(grads, name), ref[name], tol[name], name)


def test_join_norm_no_rows():
    ops = _ops()
    xy, kw = join_inputs(F32, 0, 64, 1, "none", True, True, True, True, False)
    x_out, n, stats = ops.join_norm_fwd(xy["x"].to(cuda), xy["y"].to(cuda), **on_gpu(kw))
    dx, dy, grads = ops.join_norm_bwd(x_out, x_out, x_out, n, stats, **on_gpu(kw))
    assert dx.shape == (0, 64) and bool((grads.scale == 0).all()) and grads.gate is None


# ----------------------------------------------------------------------------- together, as they are used
class Block:
    """x, h -> the next x, h: queries of h attend to the encoder's states, the result joins the stream (q, k, v, out projections in torch)"""

    def __init__(self, d, heads, hd, dtype, seed=0):
        self.heads, self.hd, self.dtype = heads, hd, dtype
        self.w = {n: rnd(*s, seed=seed + i, scale=s[1] ** -0.5) for i, (n, s) in enumerate((("q", (heads * hd, d)), ("kv", (2 * heads * hd, d)), ("o", (d, heads * hd))))}
        self.p = dict(w1=1 + 0.1 * rnd(d, seed=seed + 5), b1=0.1 * rnd(d, seed=seed + 6), gate=rnd(1, seed=seed + 7), scale=0.5 + 0.1 * rnd(d, seed=seed + 8),
                      w2=1 + 0.1 * rnd(d, seed=seed + 9), b2=0.1 * rnd(d, seed=seed + 10))

    def leaves(self, to):
        return {n: to(t).requires_grad_(True) for n, t in {**self.w, **self.p}.items()}


def run_block(blk, L, x, h, enc, pos_q, pos_k, kw, fused, trace):
    heads, hd, w = blk.heads, blk.hd, blk.heads * blk.hd
    sections = (hd // 4, hd // 4)
    if fused:
        from declip_amd import fusion
        c = lambda t: t.to(x.dtype)  # noqa: E731
        q = fusion.rope_axes(h @ c(L["q"]).t(), pos_q, heads, sections)
        kv = enc @ c(L["kv"]).t()
        k = fusion.rope_axes(kv[:, :w], pos_k, heads, sections)
        a = fusion.cross_attention(q, k, kv[:, w:], heads, **kw)
        return fusion.join_norm(x, a @ c(L["o"]).t(), post=(L["w1"], L["b1"]), gate=L["gate"], gate_tanh=True, scale=L["scale"], pre=(L["w2"], L["b2"]))
    turn = lambda t, pos: torch.cat([torch.cat(_turned(t[:, i * hd:(i + 1) * hd], pos, sections), 1) for i in range(heads)], 1)  # noqa: E731
    q, kv = turn(h @ L["q"].t(), pos_q), enc @ L["kv"].t()
    k, v = turn(kv[:, :w], pos_k), kv[:, w:]
    a = torch.zeros_like(q)
    n = kw["cu_q"].numel() - 1
    for (q0, nq), (k0, nk) in zip(R.lengths(kw["cu_q"], q.shape[0], n), R.lengths(kw["cu_kv"], k.shape[0], n)):
        for i in range(heads):
            s = slice(i * hd, (i + 1) * hd)
            if nk:
                a[q0:q0 + nq, s] = torch.softmax(q[q0:q0 + nq, s] @ k[k0:k0 + nk, s].t() * hd ** -0.5, 1) @ v[k0:k0 + nk, s]
    y = R._norm(a @ L["o"].t(), L["w1"], L["b1"], False, 1e-5)
    trace.append(y)
    xo = x + L["scale"] * torch.tanh(L["gate"]) * y
    return xo, R._norm(xo, L["w2"], L["b2"], False, 1e-5)


def _turned(t, pos, sections):
    P = sum(sections)
    ang = torch.cat([pos[:, a:a + 1].double() * 10000.0 ** (-torch.arange(n, dtype=torch.float64) / n) for a, n in enumerate(sections)], 1)
    a, b = t[:, :P], t[:, P:2 * P]
    return a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gated_cross_attention_blocks_and_their_gradients(dtype):
    """two blocks one after the other through the autograd functions, all gradients against torch's in 64 bits"""
    d, heads, hd = 64, 2, 32
    rows_q, rows_kv, kw = geometry(3, 20, 30, True, seed=8, lo_s=1)
    blocks = [Block(d, heads, hd, dtype, seed=40 * i) for i in (1, 2)]
    x0, enc0 = rnd(rows_q, d, seed=1), rnd(rows_kv, d, seed=2)
    pos_q, pos_k = torch.stack([torch.arange(rows_q), torch.zeros(rows_q)], 1).int(), torch.stack([torch.arange(rows_kv) // 6, torch.arange(rows_kv) % 6], 1).int()
    gx, gh = rnd(rows_q, d, seed=3), rnd(rows_q, d, seed=4)
    results = []
    for fused in (False, True):
        to = (lambda t: t.to(cuda)) if fused else (lambda t: t.double())
        act = (lambda t: t.to(cuda, dtype)) if fused else (lambda t: t.to(dtype).double())
        L = [b.leaves(to) for b in blocks]
        x, enc = act(x0).requires_grad_(True), act(enc0).requires_grad_(True)
        g = {n: dev(t) for n, t in kw.items()} if fused else kw
        pq, pk = (pos_q.to(cuda), pos_k.to(cuda)) if fused else (pos_q, pos_k)
        s, h, trace = x, x, []
        for b, leaf in zip(blocks, L):
            s, h = run_block(b, leaf, s, h, enc, pq, pk, g, fused, trace)
        leaves = [x, enc] + [t for leaf in L for t in leaf.values()]
        names = ["s", "h", "x", "enc"] + [n for leaf in L for n in leaf]
        grads = torch.autograd.grad([s, h], leaves + trace, [act(gx), act(gh)])
        results.append([t.detach().cpu().double() for t in (s, h, *grads[:len(leaves)])])
        if not fused:
            # a gate's gradient is ONE sum, of a = G scale (1 - tanh^2) times b = p over all elements, and may cancel: with a and b each off by tol of their
            # norms it is off by 2 tol |a| |b| (Cauchy-Schwarz), whatever its own size.  dL/dp = G scale tanh gives |a|.
            th = [math.tanh(float(b.p["gate"])) for b in blocks]
            sums = [2 * float(gy.norm()) * (1 - c * c) / abs(c) * float(y.detach().norm()) for gy, y, c in zip(grads[len(leaves):], trace, th)]
    # fp32: about 30 chained products and sums of at most 64 terms, each off by at most 64 UF: 2000 UF of the result's norm; bf16: about 30 roundings
    # of UB each along the longest path, of which the norm of many independent ones keeps the square root: 2 sqrt(30) UB
    tol = 2000 * R.UF if dtype == F32 else 2 * math.sqrt(30) * R.UB
    for n, a, b in zip(names, *results):
        assert float((a - b).norm()) <= tol * (sums.pop(0) if n == "gate" else float(a.norm())), n


def test_gradients_that_arrive_expanded_or_far_apart():
    """the gradient of a sum is one element seen everywhere; rows may come with any stride"""
    from declip_amd import fusion
    q, k, v = (rnd(n, 64, seed=i).to(cuda) for i, n in enumerate((6, 10, 10)))
    pos = torch.arange(6, dtype=torch.int32, device=cuda)[:, None].contiguous()
    w = torch.ones(64, device=cuda)

    def grads(out_of, *leaves):
        leaves = [t.clone().requires_grad_(True) for t in leaves]
        outs = out_of(*leaves)
        ones = torch.autograd.grad([o.sum() for o in outs], leaves)
        return ones, torch.autograd.grad(out_of(*leaves), leaves, [torch.ones_like(o) for o in outs])

    for a, b in (grads(lambda *t: (fusion.cross_attention(*t, 2, batch=2),), q, k, v), grads(lambda t: (fusion.rope_axes(t, pos, 2, (16,)),), q),
                 grads(lambda x, y: fusion.join_norm(x, y, post=(w, None), pre=(w, None)), q, q * 2)):
        for s, t in zip(a, b):
            assert torch.equal(s, t)
    apart = torch.zeros(10 * (1 << 22) + 64, device=cuda).as_strided((10, 64), (1 << 22, 1))
    apart.copy_(k)
    assert torch.equal(fusion.cross_attention(q, apart, v, 2, batch=2), fusion.cross_attention(q, k, v, 2, batch=2))


def test_numbers_given_as_tensors_are_read_on_every_call():
    ops = _ops()
    q, k = rnd(6, 64, seed=1).to(cuda), rnd(10, 64, seed=2).to(cuda)
    scale, most = torch.tensor(0.5, device=cuda), torch.tensor(3, device=cuda)
    first = ops.xattn_fwd(q, k, k, 2, batch=2, scale=scale, max_q=most)[0]
    scale.fill_(0.125)
    second = ops.xattn_fwd(q, k, k, 2, batch=2, scale=scale, max_q=most)[0]
    assert torch.equal(first, ops.xattn_fwd(q, k, k, 2, batch=2, scale=0.5)[0]) and torch.equal(second, ops.xattn_fwd(q, k, k, 2, batch=2, scale=0.125)[0])
    alpha = torch.tensor(2.0)
    first = ops.join_norm_fwd(q, q, alpha=alpha)[0]
    alpha.fill_(3.0)
    assert torch.equal(first, 3 * q) and torch.equal(ops.join_norm_fwd(q, q, alpha=alpha)[0], 4 * q)


def test_finite_differences():
    """the gradients against differences of the forwards themselves, in fp32 with steps along random directions"""
    from declip_amd import fusion
    rows_q, rows_kv, kw = geometry(2, 9, 12, True, seed=9, lo_s=1)
    kw = {n: dev(t) for n, t in kw.items()}
    pos = torch.randint(0, 9, (rows_q, 2), dtype=torch.int32).to(cuda)
    q, k, v = (rnd(n, 64, seed=i).to(cuda) for i, n in enumerate((rows_q, rows_kv, rows_kv)))
    x, gate, scale = rnd(rows_q, 64, seed=5).to(cuda), rnd(1, seed=6).to(cuda), rnd(64, seed=7).to(cuda)
    w1, w2 = 1 + 0.1 * rnd(64, seed=8).to(cuda), 1 + 0.1 * rnd(64, seed=9).to(cuda)
    c1, c2 = rnd(rows_q, 64, seed=10).double(), rnd(rows_q, 64, seed=11).double()

    def f(q, k, v, x, gate, scale, w1, w2):
        a = fusion.cross_attention(fusion.rope_axes(q, pos, 2, (8, 8)), k, v, 2, **kw)
        return fusion.join_norm(x, a, post=(w1, None), gate=gate, gate_tanh=True, scale=scale, pre=(w2, None), rms=True)

    leaves = [t.clone().requires_grad_(True) for t in (q, k, v, x, gate, scale, w1, w2)]
    grads = torch.autograd.grad(f(*leaves), leaves, [c1.float().to(cuda), c2.float().to(cuda)])
    total = lambda args: sum(float((o.detach().cpu().double() * c).sum()) for o, c in zip(f(*args), (c1, c2)))  # noqa: E731
    for i, t in enumerate(leaves):
        step = rnd(*t.shape, seed=50 + i).to(cuda)
        e = 2.0 ** -7 / max(1.0, float(step.abs().max()))
        up, down = ([s.detach() + (sign * e * step if j == i else 0) for j, s in enumerate(leaves)] for sign in (1, -1))
        diff = (total(up) - total(down)) / (2 * e)
        want = float((grads[i].detach().cpu().double() * step.cpu().double()).sum())
        # third derivatives: e^2 = 6e-5 of quantities as large as the gradient's norm times the step's; the forward's own roundings: 30 UF of the summed
        # magnitudes (about 2 * rows * 64) over e
        size = float(grads[i].double().norm()) * float(step.double().norm())
        assert abs(diff - want) <= 20 * e * e * size + 30 * R.UF * 2 * rows_q * 64 / e / 8, i


# ----------------------------------------------------------------------------- streams and graphs
def test_side_stream_and_captured_replays():
    """a captured forward and backward of all three, replayed on new contents of its inputs between eager calls on another stream; two graphs at a time"""
    ops = _ops()
    rows_q, rows_kv, kw = geometry(3, 1, 900, True, seed=10, lo_s=5)
    kw = {n: dev(t) for n, t in kw.items()}
    params = on_gpu(join_inputs(BF16, rows_q, 256, rows_q, "row", True, True, True, True, False)[1])
    pos = torch.arange(rows_q, dtype=torch.int32, device=cuda)[:, None].contiguous()

    def step(q, k, v):
        r = ops.rope_axes(q, pos, 4, (32,))
        a, lse = ops.xattn_fwd(r, k, v, 4, **kw)
        x, n, stats = ops.join_norm_fwd(q, a, **params)
        dx, da, grads = ops.join_norm_bwd(q, a, x, n, stats, **params)
        dr, dk, dv = ops.xattn_bwd(r, k, v, a, da, lse, 4, **kw)
        return (a, lse, x, n, dx, dk, dv, ops.rope_axes(dr, pos, 4, (32,), inverse=True), *grads)

    def inputs(seed):
        return [rnd(n, 256, seed=seed + i, dtype=BF16).to(cuda) for i, n in enumerate((rows_q, rows_kv, rows_kv))]

    side = torch.cuda.Stream()
    graphs = []
    for i in range(2):
        held = inputs(100 * i)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(*held)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = step(*held)
        graphs.append((g, held, outs))
    for round_ in range(3):
        fresh = [inputs(1000 + 10 * round_ + i) for i in range(2)]
        for (g, held, _), new in zip(graphs, fresh):
            for h, t in zip(held, new):
                h.copy_(t)
            g.replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = [step(*new) for new in fresh]
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        for (_, _, outs), ref in zip(graphs, want):
            for a, b in zip(outs, ref):
                assert (a is None and b is None) or torch.equal(a, b)
