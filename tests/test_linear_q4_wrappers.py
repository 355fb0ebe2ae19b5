"""What the Python entry point of the 4-bit projection refuses before the library is called. No GPU: stand-ins of tensors on a GPU, and of the library."""
import pytest
import torch

from fngine_b200 import lib as L
from fngine_b200 import linear


class OnGpu:
    """A CPU tensor that says it is on a GPU."""

    is_cuda = True

    def __init__(self, x, device=0):
        self.x, self.device_number = x, device

    def __getattr__(self, name):
        return getattr(self.x, name)

    def get_device(self):
        return self.device_number


def codes(n=6, k=256, device=0):
    return OnGpu(torch.zeros(n, k // 2, dtype=torch.uint8), device)


def per_group(dtype, n=6, groups=4, device=0):
    return OnGpu(torch.zeros(n, groups, dtype=dtype), device)


def test_a_weight_lies_on_one_device():
    for device in (0, 1):
        w = linear.Q4GroupWeight(codes(device=device), per_group(torch.float32, device=device), per_group(torch.uint8, device=device))
        assert (w.n, w.k, w.group) == (6, 256, 64)
    linear.Q4GroupWeight(codes(), per_group(torch.bfloat16))
    for scales, zeros in ((1, None), (0, 1), (1, 1), (1, 0)):
        with pytest.raises(AssertionError):
            linear.Q4GroupWeight(codes(), per_group(torch.float16, device=scales), None if zeros is None else per_group(torch.uint8, device=zeros))
