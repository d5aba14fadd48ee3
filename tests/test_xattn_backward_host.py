"""tests/test_gpu_xattn_backward.py on the host emulation of the kernels."""
import pytest
import torch

from hipemu_util import emulated_gpu

F32, BF16 = torch.float32, torch.bfloat16
CASES = ([("test_a_softmax_on_one_key", (dt,) + c) for dt in (BF16, F32) for c in [
    (2, 2, 64, 40, 32, 3.0), (2, 2, 64, 40, 33, 3.0), (2, 2, 64, 40, 197, 3.0), (6, 2, 64, 13, 100, 2.0), (1, 1, 128, 150, 100, 2.0), (2, 1, 96, 20, 100, 2.0), (1, 1, 64, 20, 900, 3.0)]]
         + [("test_two_keys_left_by_the_mask", (BF16,) + c) for c in [(64, 100, 197), (64, 20, 700), (80, 150, 64)]]
         + [("test_packed_sequences_of_one_and_several_tiles", (BF16,)), ("test_the_key_axis_in_ranges_of_packed_sequences", ())])


@pytest.mark.parametrize("name,args", CASES, ids=["%s-%d" % (c[0], i) for i, c in enumerate(CASES)])
def test_gpu_test_on_host_emulation(monkeypatch, name, args):
    import test_gpu_fusion as F
    import test_gpu_xattn_backward as T
    monkeypatch.setattr(T, "cuda", torch.device("cpu"))
    monkeypatch.setattr(F, "cuda", torch.device("cpu"))
    with emulated_gpu():
        getattr(T, name)(*args)
