"""The cross-attention backward where the gradients of the scores cancel: a softmax with most of its weight on one key, a mask that leaves two keys.
dS = p (dp - D) is then small beside dp and D, and an error of D shows in full."""
import pytest
import torch

from test_gpu_fusion import dev, geometry, rnd
from xattn_norms import gradients

pytestmark = pytest.mark.gpu

cuda = torch.device("cuda")
BF16, F32 = torch.bfloat16, torch.float32


def run(dtype, heads, kv_heads, hd, rows_q, rows_kv, kw, sharp, mask=None):
    from declip_amd import ops
    q, k, v = rnd(rows_q, heads * hd, seed=1, dtype=dtype, scale=sharp), rnd(rows_kv, kv_heads * hd, seed=2, dtype=dtype, scale=sharp), rnd(rows_kv, kv_heads * hd, seed=3, dtype=dtype)
    dout = rnd(rows_q, heads * hd, seed=4, dtype=dtype)
    kw = dict(kw, kv_heads=kv_heads)
    if mask is not None:
        kw["key_mask"] = mask
    ref = gradients(q, k, v, heads, dout, **kw)
    args = {n: dev(t) for n, t in kw.items()}
    qd, kd, vd = q.to(cuda), k.to(cuda), v.to(cuda)
    out, lse = ops.xattn_fwd(qd, kd, vd, heads, **args)
    dq, dk, dv = ops.xattn_bwd(qd, kd, vd, out, dout.to(cuda), lse, heads, **args)
    for name, t in (("dq", dq), ("dk", dk)):
        value, allowed = ref[name]
        off, size = float((t.cpu().double() - value).norm()), float(value.norm())
        assert off <= allowed, "%s: off by %.3g of its norm, %.3g allowed" % (name, off / size, allowed / size)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads,kv_heads,hd,rows_q,rows_kv,sharp", [
    (2, 2, 64, 40, 32, 3.0), (2, 2, 64, 40, 33, 3.0), (2, 2, 64, 40, 197, 3.0), (6, 2, 64, 40, 197, 2.0), (1, 1, 128, 150, 100, 2.0), (2, 2, 128, 20, 197, 2.0), (2, 1, 96, 150, 300, 2.0),
    (2, 2, 32, 77, 150, 4.0), (1, 1, 64, 20, 900, 3.0), (2, 1, 80, 9, 1100, 2.0), (1, 1, 128, 300, 700, 2.0)])
def test_a_softmax_on_one_key(dtype, heads, kv_heads, hd, rows_q, rows_kv, sharp):
    run(dtype, heads, kv_heads, hd, rows_q, rows_kv, dict(batch=1), sharp)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hd,rows_q,rows_kv", [(64, 100, 197), (128, 100, 197), (64, 20, 1200), (80, 150, 64)])
def test_two_keys_left_by_the_mask(dtype, hd, rows_q, rows_kv):
    mask = torch.zeros(rows_kv, dtype=torch.bool)
    mask[3] = mask[rows_kv - 2] = True
    run(dtype, 2, 2, hd, rows_q, rows_kv, dict(batch=1), 1.0, mask)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_packed_sequences_of_one_and_several_tiles(dtype):
    rows_q, rows_kv, kw = geometry(6, 60, 150, True, seed=2, lo_s=0, extra=3)
    run(dtype, 3, 1, 64, rows_q, rows_kv, kw, 3.0)


def test_the_key_axis_in_ranges_of_packed_sequences():
    rows_q, rows_kv, kw = geometry(3, 5, 1500, True, seed=3, lo_s=0)
    run(BF16, 2, 2, 64, rows_q, rows_kv, kw, 3.0)
