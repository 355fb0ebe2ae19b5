"""The 4-bit projection at decode width against its formula in 64 bits.

Two kinds of inputs. Whole activations of at most 8 and scales that are powers of two: every sum is a whole number times
2^-6 below 2^24 steps, so fp32 outputs are the formula's to the last bit, whatever the order. Normal activations and
any scales: each output adds its k products, k / group scaled sums and the partial sums of up to sixteen warps in fp32; every addition is off by
at most 2^-22 of A = sum |w x| (the tensor core cuts where fp32 rounds), in chains of k / 16 + k / group + 20 additions, and the
scale multiplication by 2^-24: |error| <= (k / 16 + k / group + 20) 2^-22 A, and half a bf16 step (2^-8 of the value) where
the output is bf16."""
import pytest

pytestmark = pytest.mark.gpu


def _torch():
    import torch
    assert torch.cuda.is_available()
    return torch


def make(torch, n, k, group, sdtype, zeros, T, whole, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(0, 256, (n, k // 2), generator=gen, device="cuda", dtype=torch.uint8)
    z = torch.randint(0, 16, (n, k // group), generator=gen, device="cuda", dtype=torch.uint8) if zeros else None
    if whole:
        scales = torch.exp2(torch.randint(-6, 1, (n, k // group), generator=gen, device="cuda").float()).to(sdtype)
        x = torch.randint(-8, 9, (T, k), generator=gen, device="cuda").to(torch.bfloat16)
    else:
        scales = (torch.rand(n, k // group, generator=gen, device="cuda") * 0.02 + 0.001).to(sdtype)
        x = (torch.randn(T, k, generator=gen, device="cuda") * 1.7).to(torch.bfloat16)
    return codes, scales, z, x


def weight64(torch, codes, scales, zeros, group):
    c = torch.stack((codes % 16, codes // 16), dim=2).reshape(codes.shape[0], -1).double()
    z = torch.full(scales.shape, 8.0, device="cuda", dtype=torch.float64) if zeros is None else (zeros % 16).double()
    return (c - z.repeat_interleave(group, 1)) * scales.double().repeat_interleave(group, 1)


def run(torch, kind, codes, scales, zeros, x, extra=None):
    from fngine_b200 import linear
    T, n = x.shape[0], codes.shape[0]
    w = linear.Q4GroupWeight(codes, scales, zeros)
    if kind == "store_bf16":
        out = torch.full((T, n), float("nan"), dtype=torch.bfloat16, device="cuda")
        linear.linear_q4_decode(x, w, linear.store_bf16(out))
    elif kind == "store_f32":
        out = torch.full((T, n), float("nan"), device="cuda")
        linear.linear_q4_decode(x, w, linear.store_f32(out))
    elif kind == "swiglu":
        out = torch.full((T, n // 2), float("nan"), dtype=torch.bfloat16, device="cuda")
        linear.linear_q4_decode(x, w, linear.swiglu(out))
    elif kind == "shared_scale":
        out = torch.full((T, n), float("nan"), device="cuda")
        linear.linear_q4_decode(x, w, linear.shared_scale(out, extra[:, 512:], 513))
    else:
        out = extra[1].clone()
        linear.linear_q4_decode(x, w, linear.gr_write(out, extra[0]))
    torch.cuda.synchronize()
    return out


# n, k, group, scales, zeros, tokens: one row, odd rows, ragged row tiles, one K step, every number of warps per row tile,
# activations that do not fit shared memory at once (10240 and up), more row tiles than warps
SHAPES = [(1, 128, 32, "bfloat16", False, 1), (7, 256, 64, "float16", True, 2), (33, 384, 128, "float32", True, 3),
          (161, 640, 32, "float32", False, 5), (1003, 2560, 64, "bfloat16", True, 8), (2560, 640, 32, "float16", True, 9),
          (513, 10240, 128, "bfloat16", True, 16), (2050, 4096, 32, "float32", True, 16), (16384, 1280, 128, "float16", False, 4),
          (40001, 256, 64, "float32", False, 13), (96, 20480, 64, "float16", True, 11), (5000, 1152, 64, "bfloat16", True, 7),
          (24001, 1536, 128, "bfloat16", False, 16)]


@pytest.mark.parametrize("n,k,group,sdtype,zeros,T", SHAPES)
def test_whole_numbers_are_exact(n, k, group, sdtype, zeros, T):
    torch = _torch()
    codes, scales, z, x = make(torch, n, k, group, getattr(torch, sdtype), zeros, T, True, n + k)
    got = run(torch, "store_f32", codes, scales, z, x)
    assert torch.equal(got.double(), x.double() @ weight64(torch, codes, scales, z, group).T)
    assert torch.equal(run(torch, "store_f32", codes, scales, z, x), got)


@pytest.mark.parametrize("kind", ["store_bf16", "store_f32", "swiglu", "shared_scale", "gr_write"])
@pytest.mark.parametrize("n,k,group,sdtype,zeros,T", [(1280, 2560, 128, "bfloat16", True, 1), (330, 640, 32, "float16", False, 16),
                                                      (2560, 6144, 64, "float32", True, 6), (34, 12800, 128, "float16", True, 12)])
def test_epilogues(kind, n, k, group, sdtype, zeros, T):
    torch = _torch()
    codes, scales, z, x = make(torch, n, k, group, getattr(torch, sdtype), zeros, T, False, n + T)
    w = weight64(torch, codes, scales, z, group)
    acc, A = x.double() @ w.T, x.double().abs() @ w.abs().T
    e = (k // 16 + k // group + 20) * 2.0 ** -22 * A
    extra = None
    if kind == "swiglu":
        g, u, eg, eu = acc[:, :n // 2], acc[:, n // 2:], e[:, :n // 2], e[:, n // 2:]
        ref = g * torch.sigmoid(g) * u
        # silu has slope below 1.1; exp, division and product add 2^-20 of the value
        tol = 1.1 * eg * (u.abs() + eu) + g.abs() * eu + 2.0 ** -20 * ref.abs()
    elif kind == "shared_scale":
        extra = torch.randn(T, 513, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
        s = torch.sigmoid(extra[:, 512].double())[:, None]
        ref, tol = acc * s, e * s + 2.0 ** -21 * (acc * s).abs()
    elif kind == "gr_write":
        gen = torch.Generator(device="cuda").manual_seed(2)
        extra = (torch.randn(T, 4, device="cuda", generator=gen), torch.randn(T, 4, n, device="cuda", generator=gen))
        add = extra[0].double()[:, :, None] * acc[:, None, :]
        ref = extra[1].double() + add
        tol = extra[0].double().abs()[:, :, None] * e[:, None, :] + 2.0 ** -23 * (add.abs() + ref.abs())
    else:
        ref, tol = acc, e
    got = run(torch, kind, codes, scales, z, x, extra)
    if kind in ("store_bf16", "swiglu"):
        tol = tol + 2.0 ** -8 * (ref.abs() + tol)
    assert bool(((got.double() - ref).abs() <= tol).all())
    if kind != "gr_write":
        assert torch.equal(run(torch, kind, codes, scales, z, x, extra), got)


@pytest.mark.parametrize("zeros", [False, True])
def test_activations_of_any_size(zeros):
    """Activations from 2^-56 to the largest bf16 numbers, tokens of both kinds in one call: the kernel scales them by powers of two."""
    torch = _torch()
    codes, scales, z, x = make(torch, 70, 1024, 32, torch.float32, zeros, 5, True, 8)
    scales = scales * 2.0 ** -14
    x = x * torch.tensor([2.0 ** -50, 1.0, 2.0 ** 62, 2.0 ** 100, 2.0 ** 124], device="cuda")[:, None].to(torch.bfloat16)
    want = x.double() @ weight64(torch, codes, scales, z, 32).T
    assert torch.equal(run(torch, "store_f32", codes, scales, z, x).double(), want)
    assert torch.equal(run(torch, "store_f32", codes, scales, z, x[:3].contiguous()).double(), want[:3])
    assert torch.equal(run(torch, "store_f32", codes, scales, z, x[3:].contiguous()).double(), want[3:])


def test_zero_points_count_their_low_four_bits():
    torch = _torch()
    codes, scales, z, x = make(torch, 50, 256, 32, torch.float32, True, 3, True, 5)
    assert torch.equal(run(torch, "store_f32", codes, scales, z + 0xB0, x), run(torch, "store_f32", codes, scales, z, x))


def test_a_captured_call_replays_and_another_stream_is_ordered():
    torch = _torch()
    from fngine_b200 import linear
    codes, scales, z, x = make(torch, 700, 1280, 64, torch.bfloat16, True, 4, True, 9)
    w = linear.Q4GroupWeight(codes, scales, z)
    out = torch.zeros(4, 700, device="cuda")
    want = run(torch, "store_f32", codes, scales, z, x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        linear.linear_q4_decode(x, w, linear.store_f32(out))
        out.zero_()
        with torch.cuda.graph(graph, stream=s):
            for _ in range(3):  # each behind the one before, which may still run when it starts
                linear.linear_q4_decode(x, w, linear.store_f32(out))
                x.add_(1)
        graph.replay()
    torch.cuda.synchronize()
    got = run(torch, "store_f32", codes, scales, z, x - 1)
    assert torch.equal(out, got) and not torch.equal(out, want)


def test_values_that_are_not_finite_stay_with_their_token():
    torch = _torch()
    codes, scales, z, x = make(torch, 130, 512, 64, torch.bfloat16, True, 7, True, 3)
    want = run(torch, "store_f32", codes, scales, z, x)
    x[2, 100], x[5, 300] = float("inf"), float("nan")
    got = run(torch, "store_f32", codes, scales, z, x)
    keep = [0, 1, 3, 4, 6]
    assert torch.equal(got[keep], want[keep]) and not bool(torch.isfinite(got[2]).any()) and bool(torch.isnan(got[5]).all())


def test_offsets_beyond_32_bits():
    """Outputs some 4.5 GB behind the first one (sampled rows), and an output of the wrong size."""
    torch = _torch()
    from fngine_b200 import linear
    n, k, T = 70000003, 128, 16
    codes = torch.empty(n, k // 2, dtype=torch.uint8, device="cuda")
    codes.view(-1)[: n * 64 // 8 * 8].view(torch.int64).random_(generator=torch.Generator(device="cuda").manual_seed(3))
    scales = torch.exp2((torch.arange(n, device="cuda") % 7 - 6).float())[:, None].bfloat16()
    x = torch.randint(-8, 9, (T, k), generator=torch.Generator(device="cuda").manual_seed(4), device="cuda").to(torch.bfloat16)
    w, out = linear.Q4GroupWeight(codes, scales), torch.empty(T, n, device="cuda")
    linear.linear_q4_decode(x, w, linear.store_f32(out))
    torch.cuda.synchronize()
    rows = torch.cat((torch.arange(0, n, 99991, device="cuda"), torch.arange(n - 300, n, device="cuda")))
    want = x.double() @ weight64(torch, codes[rows], scales[rows], None, 128).T
    assert torch.equal(out[:, rows].double(), want)
    for wrong in (linear.store_f32(out[:15]), linear.store_bf16(torch.empty(T, n - 1, dtype=torch.bfloat16, device="cuda"))):
        with pytest.raises(AssertionError):
            linear.linear_q4_decode(x, w, wrong)
