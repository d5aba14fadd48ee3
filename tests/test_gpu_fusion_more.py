"""More of the operators between the towers: every block shape of the boundary norms, head ratios that are no powers of two with their gradients, single results
and gradients that are not asked for."""
import pytest
import torch

import fusion_ref as R
from test_gpu_fusion import geometry, join_check, join_inputs, on_gpu, rnd, xattn_case

pytestmark = pytest.mark.gpu

cuda = torch.device("cuda")
BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("d", [260, 508, 772, 1020, 1100, 1532, 1540, 2044, 2052, 4092, 4100, 8188])
@pytest.mark.parametrize("gate,rms", [("channel", False), ("row", True)])
def test_join_norm_widths_that_no_vector_of_eight_divides(dtype, d, gate, rms):
    rows = 10
    xy, kw = join_inputs(dtype, rows, d, 2, gate, True, True, True, True, rms)
    join_check(dtype, xy, kw, dict(rms=rms, gate_tanh=gate == "row"), rnd(rows, d, seed=20, dtype=dtype), rnd(rows, d, seed=21, dtype=dtype))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,d", [(4000, 64), (600, 1024)])
def test_join_norm_a_gate_vector_per_token(dtype, rows, d):
    xy, kw = join_inputs(dtype, rows, d, rows, "channel", True, True, True, True, False)
    join_check(dtype, xy, kw, dict(gate_tanh=True), rnd(rows, d, seed=20, dtype=dtype), rnd(rows, d, seed=21, dtype=dtype))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads,kv_heads,hd,b,lq,s,packed,mask", [
    (6, 2, 64, 3, 21, 50, True, 0.0), (5, 1, 32, 2, 40, 70, False, 0.2), (7, 1, 64, 2, 9, 40, True, 0.0), (14, 2, 128, 1, 30, 35, False, 0.0), (3, 1, 96, 2, 60, 140, True, 0.1),
    (12, 1, 64, 1, 1, 300, False, 0.0), (11, 1, 64, 1, 200, 400, False, 0.0)])
def test_xattn_head_ratios(dtype, heads, kv_heads, hd, b, lq, s, packed, mask):
    xattn_case(dtype, heads, kv_heads, hd, *geometry(b, lq, s, packed, seed=lq), mask=mask)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_lse_beside_the_result_and_gradients_of_some_inputs_only(dtype):
    from declip_amd import fusion
    q, k, v = (rnd(n, 64, seed=i, dtype=dtype).to(cuda) for i, n in enumerate((6, 10, 10)))
    ref = R.xattn(q.cpu(), k.cpu(), v.cpu(), 2, batch=2)
    out, lse = fusion.cross_attention(q, k, v, 2, batch=2, need_lse=True)
    assert bool(((lse.cpu().double() - ref["lse"][0]).abs() <= ref["lse"][1]).all())
    assert torch.equal(out, fusion.cross_attention(q, k, v, 2, batch=2))
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    out, lse = fusion.cross_attention(*leaves, 2, batch=2, need_lse=True)
    assert out.requires_grad and not lse.requires_grad
    full = torch.autograd.grad(out.sum(), leaves)
    for wanted in ((0,), (1,), (2,), (1, 2), (0, 2)):
        mixed = [t.clone().requires_grad_(True) if i in wanted else t for i, t in enumerate((q, k, v))]
        got = torch.autograd.grad(fusion.cross_attention(*mixed, 2, batch=2).sum(), [mixed[i] for i in wanted])
        for i, g in zip(wanted, got):
            assert torch.equal(g, full[i])
    x, y, w, gate = q, q * 2, 1 + 0.1 * rnd(64, seed=7).to(cuda), rnd(3, seed=8).to(cuda)
    names = ["x", "y", "w", "gate"]
    call = lambda t: fusion.join_norm(t["x"], t["y"], post=(t["w"], None), gate=t["gate"], pre=(w, None))  # noqa: E731
    leaves = {n: t.clone().requires_grad_(True) for n, t in zip(names, (x, y, w, gate))}
    full = dict(zip(names, torch.autograd.grad([o.float().sum() for o in call(leaves)], list(leaves.values()))))
    for wanted in (("x",), ("y",), ("w",), ("gate", "x")):
        mixed = {n: t.clone().requires_grad_(True) if n in wanted else t for n, t in zip(names, (x, y, w, gate))}
        for n, g in zip(wanted, torch.autograd.grad([o.float().sum() for o in call(mixed)], [mixed[n] for n in wanted])):
            assert torch.equal(g, full[n])


def test_join_norm_repeats_its_bits_with_a_gate_vector_per_token():
    from declip_amd import ops
    xy, kw = join_inputs(BF16, 2000, 264, 2000, "channel", True, True, True, True, False)
    x, y, g, kw = xy["x"].to(cuda), xy["y"].to(cuda), rnd(2000, 264, seed=9, dtype=BF16).to(cuda), on_gpu(kw)
    stats = ops.join_norm_fwd(x, y, **kw)[2]
    first = ops.join_norm_bwd(x, y, g, g, stats, **kw)
    again = ops.join_norm_bwd(x, y, g, g, stats, **kw)
    for a, b in zip(first[:2] + tuple(first[2]), again[:2] + tuple(again[2])):
        assert torch.equal(a, b)
