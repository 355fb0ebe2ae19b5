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


def test_epilogue_inputs_of_fewer_tokens_or_another_device(monkeypatch):
    """inj is [tokens][4]; gate_logit reaches the last token's logit: [tokens][513] from column 512 on, one logit per token, one for all."""
    made = []
    monkeypatch.setattr(L, "load", lambda: type("Library", (), {"fb_linear_q4_decode": lambda self, *a: made.append(a) or 0})())
    monkeypatch.setattr(L, "stream", lambda: None)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    w = linear.Q4GroupWeight(codes(), per_group(torch.float32))
    gpu = lambda *shape, dtype=torch.float32, device=0: OnGpu(torch.zeros(*shape, dtype=dtype), device)
    x, T = gpu(5, 256, dtype=torch.bfloat16), 5
    write = lambda inj: linear.gr_write(gpu(T, 4, 6), inj)
    scale = lambda gate, stride: linear.shared_scale(gpu(T, 6), gate, stride)
    logits = torch.zeros(T, 513)
    good = [write(gpu(T, 4)), scale(OnGpu(logits[:, 512:]), 513), scale(OnGpu(logits.view(-1)[512:]), 513), scale(gpu(T), 1), scale(gpu(1), 0), scale(OnGpu(logits), 513)]
    for epilogue in good:
        linear.linear_q4_decode(x, w, epilogue)
    assert len(made) == len(good)
    for epilogue in [write(gpu(T - 1, 4)), write(gpu(T + 1, 4)), write(gpu(T, 4, device=1)), scale(OnGpu(logits[:T - 1, 512:]), 513),
                     scale(OnGpu(logits.view(-1)[513:]), 513), scale(gpu(T - 1), 1), scale(gpu(T), 2), scale(gpu(0), 0), scale(gpu(T), -1), scale(gpu(T, device=1), 1)]:
        with pytest.raises(AssertionError):
            linear.linear_q4_decode(x, w, epilogue)
    assert len(made) == len(good)


def test_epilogue_inputs_that_are_not_aligned(fb_built):
    from test_linear_q4_arguments import call
    lib = L.load()
    for bad in (dict(kind=L.EPI_GR_WRITE, inj=0x600002), dict(kind=L.EPI_GR_WRITE, inj=0x600001), dict(kind=L.EPI_SHARED_SCALE, gate=0x600002)):
        st, msg = call(lib, **bad)
        assert st == 1 and b"inj or gate_logit is not aligned" in msg
