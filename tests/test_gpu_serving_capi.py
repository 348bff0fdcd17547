"""The serving operators' C entry points on device tensors, called as a host without Python would."""
import ctypes

import pytest
import torch

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")]


@pytest.mark.parametrize("biases", [0, 5, 1000, -3])
def test_biases_without_a_list_are_left_out(biases):
    """NULL members are left out: a count beside a NULL list adds nothing and reads nothing."""
    from aria_b200 import _lib
    x = torch.randn(3, 2001, device="cuda")
    out = torch.zeros_like(x)
    r = _lib.LogitRulesStruct(biases=biases, bias_row=biases)
    status = _lib.lib().aria_logits_adjust(ctypes.addressof(r), x.data_ptr(), _lib.F32, 2001, 3, 2001, out.data_ptr(),
                                           _lib.F32, 2001, None, None, 0, torch.cuda.current_stream().cuda_stream)
    assert status == _lib.OK
    assert torch.equal(out, x)
