"""The operators between the towers without a GPU: their GPU tests on the host emulation of the kernels, and every refusal."""
import ctypes

import pytest
import torch

from hipemu_util import emulated_gpu

F32, BF16 = torch.float32, torch.bfloat16
CASES = ([("test_xattn", (dt,) + c) for dt in (BF16, F32) for c in [
    (2, 2, 64, 3, 40, 70, True, 0.0), (4, 2, 64, 2, 20, 70, False, 0.3), (4, 1, 32, 3, 33, 65, True, 0.5), (2, 2, 80, 2, 20, 33, True, 0.0), (2, 1, 128, 1, 33, 63, True, 0.2),
    (1, 1, 8, 1, 1, 1, False, 0.0), (2, 2, 24, 4, 2, 3, True, 0.5)]]
         + [("test_xattn_rows_without_owner_are_zero_and_tables_may_start_late", (BF16,)), ("test_xattn_large_scores", (BF16,)), ("test_xattn_large_scores", (F32,)),
            ("test_xattn_split_ranges_without_a_key", ()), ("test_xattn_tables_out_of_range_stay_inside", ())]
         + [("test_xattn_empty", (BF16, w)) for w in ("no_keys", "all_masked", "no_queries")]
         + [("test_xattn_single_tokens_over_long_keys", (dt, 6, 2, 80, 2, 1, 700)) for dt in (BF16, F32)]
         + [("test_rope_axes", (dt,) + c) for dt in (BF16, F32) for c in [
             (37, 37, 3, 64, (8, 12, 12), True, False, False, 1_000_000), (12, 4, 2, 80, (16, 16), False, True, True, 64), (9, 9, 5, 32, (3, 5), False, True, False, 100),
             (10, 5, 2, 40, (3, 4), True, False, True, 50), (7, 7, 1, 6, (1, 1, 1), False, False, False, 9), (5, 5, 2, 256, (64, 64), False, False, False, 999)]]
         + [("test_rope_axes_strided_in_place_and_bases", ())]
         + [("test_join_norm", (dt, c)) for dt in (BF16, F32) for c in [
             (50, 768, 5, "channel", False, True, True, True, True, False, 1.0), (33, 512, 33, "row", True, False, True, True, True, True, 2.0),
             (9, 2056, 3, "row", True, True, False, True, True, False, 0.5), (6, 5000, 2, "channel", True, False, True, True, True, True, 1.0),
             (14, 33, 7, "row", False, True, True, True, True, False, 1.0), (5, 257, 1, "channel", False, False, True, False, True, False, 1.0),
             (4, 3001, 4, "row", False, False, False, True, True, True, 1.0), (6, 1, 2, "row", False, True, False, True, False, False, 1.0)]]
         + [("test_xattn_block_shapes_and_split_axes", (BF16,) + c) for c in [
             (2, 2, 64, 1, 300, 20, False, 0.2), (1, 1, 128, 1, 33, 40, True, 0.0), (1, 1, 128, 1, 130, 140, True, 0.1), (1, 1, 64, 1, 130, 2050, True, 0.0), (1, 1, 96, 1, 130, 300, False, 0.0)]]
         + [("test_join_norm_rows_far_from_zero", (dt, rms)) for dt in (BF16, F32) for rms in (False, True)]
         + [("test_gradients_that_arrive_expanded_or_far_apart", ()), ("test_numbers_given_as_tensors_are_read_on_every_call", ())]
         + [("test_join_norm_one_gradient_only", (w,)) for w in ("dn", "dx_out")] + [("test_join_norm_no_rows", ())]
         + [("test_gated_cross_attention_blocks_and_their_gradients", (dt,)) for dt in (F32, BF16)] + [("test_finite_differences", ())])


@pytest.mark.parametrize("name,args", CASES, ids=["%s-%d" % (c[0], i) for i, c in enumerate(CASES)])
def test_gpu_test_on_host_emulation(monkeypatch, name, args):
    import test_gpu_fusion as T
    monkeypatch.setattr(T, "cuda", torch.device("cpu"))
    with emulated_gpu():
        getattr(T, name)(*args)


def _refused(call, *words):
    from declip_amd.lib import DeclipHipError
    with pytest.raises(DeclipHipError) as e:
        call()
    for w in words:
        assert w in str(e.value), str(e.value)


def test_xattn_refusals():
    with emulated_gpu() as ops:
        z = lambda *s, dtype=BF16: torch.zeros(*s, dtype=dtype)  # noqa: E731
        q, k = z(4, 128), z(6, 128)
        i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
        f = ops.xattn_fwd
        _refused(lambda: f(q, k, k, 2), "batch")
        _refused(lambda: f(q, k, k, 3, batch=1), "heads")
        _refused(lambda: f(q, k, k, 2, kv_heads=3, batch=1), "kv_heads")
        _refused(lambda: f(q, k, k, 2, kv_heads=1, batch=1), "k: [rows, 64]")
        _refused(lambda: f(q, k.float(), k, 2, batch=1), "dtype")
        _refused(lambda: f(q.half(), k.half(), k.half(), 2, batch=1), "dtype")
        _refused(lambda: f(q, k, z(5, 128), 2, batch=1), "shape")
        _refused(lambda: f(q, k, k, 2, batch=3), "do not divide")
        _refused(lambda: f(q, k, k, 2, batch=4), "key rows do not divide")
        _refused(lambda: f(q, k, k, 2, batch=1, scale=0.0), "scale")
        _refused(lambda: f(q, k, k, 2, batch=1, scale=-1.0), "scale")
        _refused(lambda: f(q, k, k, 2, batch=1, scale=float("nan")), "scale")
        _refused(lambda: f(q, k, k, 2, cu_q=i32(0, 4), cu_kv=i32(0, 3, 6)), "batch + 1")
        _refused(lambda: f(q, k, k, 2, batch=2, cu_q=i32(0, 4)), "batch + 1")
        _refused(lambda: f(q, k, k, 2, cu_q=torch.tensor([0, 4])), "int32")
        _refused(lambda: f(q, k, k, 2, batch=2, kv_len=i32(1)), "kv_len")
        _refused(lambda: f(q, k, k, 2, batch=2, key_mask=torch.ones(5, dtype=torch.bool)), "key_mask")
        _refused(lambda: f(q, k, k, 2, batch=2, key_mask=torch.ones(6)), "key_mask")
        _refused(lambda: f(z(4, 132), z(6, 132), z(6, 132), 1, batch=1), "head size 132")
        _refused(lambda: f(z(4, 20), z(6, 20), z(6, 20), 1, batch=1), "head size 20")
        _refused(lambda: f(q.t(), k, k, 1, batch=1), "contiguous columns")
        _refused(lambda: f(z(4, 131)[:, 3:], k, k, 2, batch=1), "16-byte")
        _refused(lambda: f(q, z(1, 128).expand(6, 128), k, 2, batch=1), "16-byte")
        far = z((1 << 22) + 128).as_strided((2, 128), (1 << 22, 1))
        _refused(lambda: f(q, far, far, 2, batch=1), "2^22")
        many = z(1).expand(1 << 30, 8)
        _refused(lambda: f(many, z(6, 8), z(6, 8), 1, batch=1), "2^30")
        out, lse = f(q, k, k, 2, batch=1)
        b = ops.xattn_bwd
        _refused(lambda: b(q, k, k, out, out[:3], lse, 2, batch=1), "dout")
        _refused(lambda: b(q, k, k, out, out.float(), lse, 2, batch=1), "dout")
        _refused(lambda: b(q, k, k, out, out, lse[:1], 2, batch=1), "lse")
        _refused(lambda: b(q, k, k, out, out, lse.double(), 2, batch=1), "lse")


def test_rope_refusals():
    with emulated_gpu() as ops:
        x, pos = torch.zeros(6, 128, dtype=BF16), torch.zeros(6, 2, dtype=torch.int32)
        f = ops.rope_axes
        _refused(lambda: f(x, pos, 3, (4, 4)), "heads")
        _refused(lambda: f(x, pos, 2, (4, 4, 4)), "pos")
        _refused(lambda: f(x, pos.long(), 2, (4, 4)), "int32")
        _refused(lambda: f(x, pos[:4], 2, (4, 4)), "6 rows, 4 positions")
        _refused(lambda: f(x, pos[:0], 2, (4, 4)), "positions")
        _refused(lambda: f(x, pos, 2, (20, 20)), "40 pairs")
        _refused(lambda: f(x, pos, 2, (0, 4)), "section 0")
        _refused(lambda: f(x, pos, 2, (-1, 4)), "section -1")
        _refused(lambda: f(x, pos, 2, (4, 4), theta=0.0), "theta")
        _refused(lambda: f(x, pos, 2, (4, 4), theta=(10.0, 20.0, 30.0)), "theta")
        _refused(lambda: f(x, pos, 2, (4, 4), theta=(10.0, 20.0), joint=True), "joint")
        _refused(lambda: f(x.half(), pos, 2, (4, 4)), "dtype")
        _refused(lambda: f(x.t(), pos, 2, (4, 4)), "contiguous columns")
        _refused(lambda: f(x, pos, 2, (4, 4), out=x[:5]), "out")
        _refused(lambda: f(x[:1, :1].expand(1 << 30, 8), pos, 1, (4,)), "2^30")
        wide = torch.zeros(7, 128, dtype=BF16)
        _refused(lambda: f(wide[:6], pos, 2, (4, 4), out=wide[1:]), "out")


def test_join_norm_refusals():
    with emulated_gpu() as ops:
        x, w = torch.zeros(6, 64, dtype=BF16), torch.ones(64)
        f = ops.join_norm_fwd
        _refused(lambda: f(x, x[:5]), "x and y")
        _refused(lambda: f(x, x.float()), "x and y")
        _refused(lambda: f(x[:, ::2], x[:, ::2]), "contiguous")
        _refused(lambda: f(x, x, post=(w[:3], None)), "post_w")
        _refused(lambda: f(x, x, post=(w.to(BF16), None)), "post_w")
        _refused(lambda: f(x, x, post=(w, w), rms=True), "bias")
        _refused(lambda: f(x, x, pre=(None, w)), "bias")
        _refused(lambda: f(x, x, scale=w[:1]), "scale")
        _refused(lambda: f(x, x, gate=torch.ones(4)), "groups")
        _refused(lambda: f(x, x, gate=torch.ones(2, 3)), "gate")
        _refused(lambda: f(x, x, gate=torch.ones(0)), "groups")
        _refused(lambda: f(x, x, eps=-1.0), "eps")
        many = x[:1, :1].expand(1 << 30, 8)
        _refused(lambda: f(many, many), "2^30")
        _refused(lambda: f(torch.zeros(2, 8200), torch.zeros(2, 8200)), "8192")
        _refused(lambda: f(torch.zeros(2, 0), torch.zeros(2, 0)), "width 0")
        _, n, st = f(x, x, pre=(w, None))
        b = ops.join_norm_bwd
        _refused(lambda: b(x, x, None, None, st, pre=(w, None)), "no gradient")
        _refused(lambda: b(x, x, x, x, st), "dn without")
        _refused(lambda: b(x, x, x[:3], None, st), "dx_out")
        _refused(lambda: b(x, x, x, None, st[:2]), "stats")


def test_c_entries_check_before_they_launch():
    """the real library: bad structs and small workspaces come back as codes with a message"""
    from declip_amd import lib as L
    lib = L.load()
    assert lib.dh_xattn_fwd(None, None) == -1 and lib.dh_xattn_bwd(None, None) == -1 and lib.dh_xattn_ws_bytes(None, 0) == -1
    assert lib.dh_join_norm_fwd(None, None) == -1 and lib.dh_join_norm_bwd(None, None) == -1 and lib.dh_join_norm_bwd_ws_bytes(None) == -1
    a = L.XattnArgs()
    assert lib.dh_xattn_fwd(ctypes.byref(a), None) == -1 and lib.dh_xattn_ws_bytes(ctypes.byref(a), 1) == -1
    a.dtype, a.batch, a.heads, a.kv_heads, a.hd, a.rows_q, a.rows_kv, a.scale = 1, 1, 4, 4, 64, 1, 100000, 1.0
    one = ctypes.c_void_p(16)
    a.q = a.k = a.v = a.out = a.lse = a.dout = a.dq = a.dk = a.dv = one
    a.ldq = a.ldk = a.ldv = a.ldo = a.lddo = a.lddq = a.lddk = a.lddv = 256
    assert lib.dh_xattn_ws_bytes(ctypes.byref(a), 0) > 0
    assert lib.dh_xattn_fwd(ctypes.byref(a), None) == -1 and b"workspace" in lib.dh_last_error()
    assert lib.dh_xattn_bwd(ctypes.byref(a), None) == -1 and b"workspace" in lib.dh_last_error()
    a.dk = None
    assert lib.dh_xattn_bwd(ctypes.byref(a), None) == -1 and b"dk is NULL" in lib.dh_last_error()
    a.dk, a.rows_q = one, 1 << 30
    assert lib.dh_xattn_fwd(ctypes.byref(a), None) == -1 and b"too many rows" in lib.dh_last_error()
    j = L.JoinNormArgs()
    j.dtype, j.rows, j.d, j.x, j.y, j.stats, j.dx, j.dy, j.dx_out = 1, 8, 64, one, one, one, one, one, one
    assert lib.dh_join_norm_fwd(ctypes.byref(j), None) == -1 and b"null output" in lib.dh_last_error()
    assert lib.dh_join_norm_bwd(ctypes.byref(j), None) == -1 and b"workspace" in lib.dh_last_error()
    sec, th = (ctypes.c_int * 1)(4), (ctypes.c_double * 1)(1e4)
    plan = L.RopePlan()
    p = ctypes.byref(plan)
    assert lib.dh_rope_axes(p, 1, one, 64, one, 64, 2, 1, one, 0, 1, 0, None) == -1 and b"not initialised" in lib.dh_last_error()
    assert lib.dh_rope_plan_init(None, 64, sec, th, 1, 0, 0) == -1 and lib.dh_rope_plan_init(p, 4, sec, th, 1, 0, 0) == -1 and b"4 pairs in a head of 4" in lib.dh_last_error()
    assert lib.dh_rope_plan_init(p, 64, sec, th, 1, 0, 0) == 0
    assert lib.dh_rope_axes(p, 7, one, 64, one, 64, 2, 1, one, 0, 1, 0, None) == -1 and b"dtype" in lib.dh_last_error()
    assert lib.dh_rope_axes(p, 1, one, 32, one, 64, 2, 1, one, 0, 1, 0, None) == -1 and b"strides" in lib.dh_last_error()
    assert lib.dh_rope_axes(p, 1, None, 64, one, 64, 2, 1, one, 0, 1, 0, None) == -1


def test_cpu_tensors_and_mixed_devices_are_refused():
    from declip_amd import ops
    x = torch.zeros(4, 64)
    _refused(lambda: ops.xattn_fwd(x, x, x, 1, batch=1), "HIP device")
    _refused(lambda: ops.rope_axes(x, torch.zeros(4, 1, dtype=torch.int32), 1, (4,)), "HIP device")
    _refused(lambda: ops.join_norm_fwd(x, x), "HIP device")
    _refused(lambda: ops.xattn_fwd(x, x.to("meta"), x, 1, batch=1), "different devices")


def test_a_call_goes_to_its_tensors_device(monkeypatch):
    """tensors of another device than the current one: the device is switched for the call"""
    from declip_amd import ops
    seen = []

    class Guard:
        def __init__(self, dev):
            seen.append(dev)

        def __enter__(self):
            monkeypatch.setattr(torch.cuda, "current_device", lambda: seen[-1])

        def __exit__(self, *a):
            pass

    for call in (lambda x: ops.xattn_fwd(x, x, x, 1, batch=1), lambda x: ops.rope_axes(x, x, 1, (4,)), lambda x: ops.join_norm_fwd(x, x)):
        monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
        monkeypatch.setattr(torch.cuda, "device", Guard)
        monkeypatch.setattr(ops, "_device_of", lambda *a: 3)
        monkeypatch.setattr(ops, "_plan", lambda *a: (_ for _ in ()).throw(RuntimeError("planned on %d" % torch.cuda.current_device())))
        with pytest.raises(RuntimeError, match="planned on 3"):
            call(torch.zeros(2, 8))
    assert seen == [3, 3, 3]
