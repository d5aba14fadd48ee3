"""tests/test_gpu_fusion_more.py on the host emulation of the kernels."""
import pytest
import torch

from hipemu_util import emulated_gpu

F32, BF16 = torch.float32, torch.bfloat16
CASES = ([("test_join_norm_widths_that_no_vector_of_eight_divides", (dt, d) + g) for dt, g in ((BF16, ("channel", False)), (F32, ("row", True)))
          for d in (260, 508, 772, 1020, 1100, 1532, 1540, 2044, 2052, 4092, 4100, 8188)]
         + [("test_join_norm_a_gate_vector_per_token", (BF16, 40, 64))]
         + [("test_xattn_head_ratios", (dt,) + c) for dt in (BF16, F32) for c in [
             (6, 2, 64, 3, 21, 50, True, 0.0), (5, 1, 32, 2, 20, 40, False, 0.2), (7, 1, 64, 2, 9, 40, True, 0.0), (14, 2, 128, 1, 10, 35, False, 0.0), (3, 1, 96, 2, 30, 70, True, 0.1)]]
         + [("test_lse_beside_the_result_and_gradients_of_some_inputs_only", (dt,)) for dt in (BF16, F32)])


@pytest.mark.parametrize("name,args", CASES, ids=["%s-%d" % (c[0], i) for i, c in enumerate(CASES)])
def test_gpu_test_on_host_emulation(monkeypatch, name, args):
    import test_gpu_fusion as F
    import test_gpu_fusion_more as T
    monkeypatch.setattr(T, "cuda", torch.device("cpu"))
    monkeypatch.setattr(F, "cuda", torch.device("cpu"))
    with emulated_gpu():
        getattr(T, name)(*args)
