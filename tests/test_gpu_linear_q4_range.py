"""Small and infinite activations of the 4-bit projection. Its sums are fp32 numbers in a scale of 2^-69 (2^-133 for a token that has an
activation of 2^63 or more), so their smallest step, 2^-149 there, is 2^-80 (2^-16) in the activations' own scale."""
import pytest

from test_gpu_linear_q4 import make, run, weight64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("T", [1, 5, 9, 16])
def test_sums_are_exact_down_to_their_smallest_step(T, zeros):
    """Whole numbers of at most 8 times 2^e and scales 2^-6 .. 1: every product and sum is a whole multiple of 2^(e - 6) below 2^24 of them, exact
    while that is 2^-80 or more."""
    import torch
    codes, scales, z, x = make(torch, 70, 1024, 32, torch.float32, zeros, T, True, 8)
    w = weight64(torch, codes, scales, z, 32)
    for e in (-74, -70, -63, -58, -57, -56, -30):
        small = x * 2.0 ** e
        assert torch.equal(run(torch, "store_f32", codes, scales, z, small).double(), small.double() @ w.T), e
    mixed = x * torch.exp2(torch.randint(-74, 0, (T, 1), device="cuda", generator=torch.Generator(device="cuda").manual_seed(T)).float()).bfloat16()
    mixed[0] = x[0] * 2.0 ** 64  # a token of large activations beside them
    assert torch.equal(run(torch, "store_f32", codes, scales, z, mixed).double(), mixed.double() @ w.T)


@pytest.mark.parametrize("group,zeros", [(32, True), (128, False), (64, True)])
def test_below_the_smallest_step(group, zeros):
    """Any activations of 2^-86 .. 2^-60. Per group: the products' additions cut 2^-80 each, group / 16 of them; a rounded activation is off by 2^-81,
    group of them times a zero point of 15; their difference by 2^-81. That times the scale, and 2^-80 for each of the k / group + 20 additions of
    scaled sums; beside that fp32's (k / 16 + k / group + 20) 2^-22 sum |w x|, where w x counts as |c x| + |z x|."""
    import torch
    n, k, T = 90, 1024, 7
    codes, scales, z, x = make(torch, n, k, group, torch.float32, zeros, T, False, 3)
    scales = scales * 50
    w = weight64(torch, codes, scales, z, group)
    for e in (-60, -70, -76, -80, -86):
        small = x * 2.0 ** e
        size = small.double().abs() @ (30 * scales.double().repeat_interleave(group, 1)).T
        step = (scales.double().sum(1) * (group / 16 + 7.5 * group + 1) + k // group + 20) * 2.0 ** -80
        got = run(torch, "store_f32", codes, scales, z, small).double()
        assert bool(((got - small.double() @ w.T).abs() <= (k // 16 + k // group + 20) * 2.0 ** -22 * size + step).all()), e


@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")])
@pytest.mark.parametrize("T", [1, 11])
def test_an_activation_that_is_not_finite_makes_its_token_not_a_number(T, value):
    """Whatever the weight that it meets: below, at and above the zero point, with and without zero points, and in no other token."""
    import torch
    n, k = 48, 256
    for group in (32, 64, 128):
        codes = (torch.arange(n, device="cuda", dtype=torch.uint8) % 16 * 17)[:, None].expand(n, k // 2).contiguous()
        scales = torch.ones(n, k // group, device="cuda")
        x = torch.randn(T, k, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).bfloat16()
        for z in (None, torch.zeros(n, k // group, dtype=torch.uint8, device="cuda"), torch.full((n, k // group), 15, dtype=torch.uint8, device="cuda")):
            want = run(torch, "store_f32", codes, scales, z, x)
            bad = x.clone()
            bad[T // 2, 200] = value
            got = run(torch, "store_f32", codes, scales, z, bad)
            others = [t for t in range(T) if t != T // 2]
            assert bool(torch.isnan(got[T // 2]).all()) and torch.equal(got[others], want[others])
