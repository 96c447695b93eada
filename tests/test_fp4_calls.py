"""The front end of the 4-bit cache's operators (a module of the host's compiler) on the host: what does not fit is answered with None."""

import torch


def test_a_flag_without_a_truth_value_does_not_fit():
    from torchllms_b200.kernels.build import load_extension
    calls = load_extension("fp4_calls")
    x = torch.zeros((2, 8 * 64))
    args = [x, x, x, 4, 2, 64, torch.zeros(2), None, None, None, 16, -1, None, 0.0, 0.0]       # (two numbers are neither true nor false)
    assert calls.write(*args) is None
    args[6] = True
    assert calls.write(*args) is None                                                           # (nothing lies on a GPU)
