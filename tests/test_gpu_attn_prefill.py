"""Causal attention over packed prompts against its formula in 64 bits.

The tolerance: weights are rounded once to the type of v (half a step h of each: bf16 2^-8, fp16 2^-11), so an output is off by at most h
sum_j w_j |v_j| = h B; scores are fp32 sums of D products (D 2^-23 sum |scale q k|, which moves a weight by that relative part, and the
exponential another 2^-18, of which a polynomial's 2.7e-6 < 2^-18.4 is the most, its roundings and the scaled score's 2^-21): 2 (D
2^-23 S + 2^-18) B with S the row's largest sum |scale q k|; sums over the keys 2^-18 B; and half a step of the output. Weights below fp16's normal range are off by 2^-25 of the largest at most (the largest in use is at
least 2^-8 of the one that the exponents refer to, which loses eight bits there: 2^-17): 2^-17 sum |v| w_max over the keys."""
import pytest

pytestmark = pytest.mark.gpu
HALF = {"bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}


def _torch():
    import torch
    assert torch.cuda.is_available()
    return torch


def inputs(torch, tokens, heads, kv, dim, dtype, seed, gain=1.5):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = getattr(torch, dtype)
    return [(torch.randn(tokens, h, dim, generator=gen, device="cuda") * f).to(dt) for h, f in ((heads, gain), (kv, 1.0), (kv, 1.0))]


def check(torch, out, q, k, v, a, b, scale=None):
    """Compares out[a:b] with the formula for the sequence a..b."""
    H, D, kv = q.shape[1], q.shape[2], k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    h = HALF[str(q.dtype).split(".")[1]]
    n = b - a
    later = torch.ones(n, n, dtype=torch.bool, device="cuda").triu_(1)
    for g in range(H):
        qq, kk, vv = q[a:b, g].double(), k[a:b, g * kv // H].double(), v[a:b, g * kv // H].double()
        w = torch.softmax((qq @ kk.T * scale).masked_fill_(later, -float("inf")), 1)
        want, B = w @ vv, w @ vv.abs()
        S = ((qq.abs() @ kk.abs().T) * scale).masked_fill_(later, 0).amax(1, keepdim=True)
        tol = (h + 2 * (D * 2.0 ** -23 * S + 2.0 ** -18) + 2.0 ** -18) * B
        least = 0.0
        if q.dtype == torch.float16:
            tol = tol + 2.0 ** -17 * w.amax(1, keepdim=True) * vv.abs().cumsum(0)
            least = 2.0 ** -25
        tol = tol + h * (want.abs() + tol) + least
        off = (out[a:b, g].double() - want).abs()
        if not bool((off <= tol).all()):
            at = int((off - tol).nan_to_num(1e30).argmax())
            raise AssertionError("sequence %d..%d head %d: %d of %d values off, at row %d: %r against %r, tolerance %r" % (
                a, b, g, int((~(off <= tol)).sum()), off.numel(), at // D, float(out[a:b, g].reshape(-1)[at]), float(want.reshape(-1)[at]), float(tol.reshape(-1)[at])))


# lengths, heads, kv heads, dim, type
CASES = [([1], 1, 1, 64, "bfloat16"), ([1], 2, 1, 128, "float16"), ([128], 2, 2, 128, "bfloat16"), ([129, 127], 3, 1, 128, "bfloat16"),
         ([0, 5, 0, 0, 256, 257, 0], 4, 2, 64, "float16"), ([255, 1, 384, 2, 511], 6, 2, 128, "float16"), ([640], 5, 5, 64, "bfloat16"),
         ([3] * 90, 2, 1, 64, "bfloat16"), ([2048, 1000], 8, 2, 128, "bfloat16"), ([1537], 14, 2, 64, "float16"), ([4100], 3, 1, 128, "float16"),
         ([17, 300, 33, 700, 100, 1, 64], 12, 4, 128, "bfloat16")]


@pytest.mark.parametrize("lengths,heads,kv,dim,dtype", CASES)
def test_against_the_formula(lengths, heads, kv, dim, dtype):
    torch = _torch()
    from fngine_b200 import attention as A
    tokens = sum(lengths)
    q, k, v = inputs(torch, tokens, heads, kv, dim, dtype, tokens + heads)
    ends = [0]
    for n in lengths:
        ends.append(ends[-1] + n)
    cu = torch.tensor(ends, device="cuda", dtype=torch.int32)
    out, status = torch.full_like(q, float("nan")), torch.zeros(1, dtype=torch.int32, device="cuda")
    A.attn_prefill(q, k, v, cu, out, status=status)
    torch.cuda.synchronize()
    assert int(status) == 0
    for a, b in zip(ends, ends[1:]):
        if b > a:
            check(torch, out, q, k, v, a, b)
    again = torch.full_like(q, float("nan"))
    A.attn_prefill(q, k, v, cu, again)
    assert torch.equal(out, again)


def test_a_sequence_does_not_depend_on_its_neighbours():
    """NaN and infinities in the tokens in front of, between and behind the sequences; those tokens' outputs stay as they were."""
    torch = _torch()
    from fngine_b200 import attention as A
    for dim, dtype in ((64, "float16"), (128, "bfloat16")):
        q, k, v = inputs(torch, 900, 4, 2, dim, dtype, 7)
        cu = torch.tensor([40, 240, 240, 541], device="cuda", dtype=torch.int32)
        clean = torch.full_like(q, 3.0)
        A.attn_prefill(q, k, v, cu, clean)
        for x, bad in ((q, float("inf")), (k, float("nan")), (v, float("nan"))):
            x[:40] = bad
            x[541:] = bad
        v[600:] = float("inf")
        out = torch.full_like(q, 3.0)
        A.attn_prefill(q, k, v, cu, out)
        torch.cuda.synchronize()
        assert torch.equal(out, clean) and bool((out[:40] == 3).all()) and bool((out[541:] == 3).all())
        check(torch, out, q, k, v, 40, 240)
        check(torch, out, q, k, v, 240, 541)
        k[240:541], v[240:541] = float("nan"), float("inf")  # one sequence's values do not reach the other
        A.attn_prefill(q, k, v, cu, out)
        torch.cuda.synchronize()
        assert torch.equal(out[40:240], clean[40:240]) and bool(torch.isnan(out[240:541]).all())


def test_parts_of_one_projection():
    """q, k and v as parts of wider rows, the output into wider rows, another scale."""
    torch = _torch()
    from fngine_b200 import attention as A
    T, H, K, D = 700, 6, 2, 128
    wide = torch.randn(T, (H + 2 * K) * D + 64, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5)).bfloat16()
    q, k, v = (wide[:, a * D + 32:b * D + 32].unflatten(1, (b - a, D)) for a, b in ((0, H), (H, H + K), (H + K, H + 2 * K)))
    rows = torch.zeros(T, H * D + 128, device="cuda", dtype=torch.bfloat16)
    out = rows[:, 64:64 + H * D].unflatten(1, (H, D))
    A.attn_prefill(q, k, v, torch.tensor([0, 300, 700], device="cuda", dtype=torch.int32), out, scale=0.05)
    torch.cuda.synchronize()
    check(torch, out, q, k, v, 0, 300, 0.05)
    check(torch, out, q, k, v, 300, 700, 0.05)
    assert not bool(rows[:, :64].any()) and not bool(rows[:, 64 + H * D:].any())


@pytest.mark.parametrize("dim,dtype", [(64, "bfloat16"), (128, "float16"), (128, "bfloat16")])
def test_maxima_that_rise_late(dim, dtype):
    """Scores that grow along the keys by far more than the slack in which the outputs are left alone, and a last key that takes all."""
    torch = _torch()
    from fngine_b200 import attention as A
    q, k, v = inputs(torch, 1000, 2, 1, dim, dtype, 9, 1.0)
    lift = torch.linspace(0.0, 60.0, 1000, device="cuda")[:, None]
    k[:, 0] = (k[:, 0].float() * 0.3).to(k.dtype)
    k[:, 0, 0] = lift[:, 0].to(k.dtype)
    q[:, :, 0] = 8.0
    cu = torch.tensor([0, 1000], device="cuda", dtype=torch.int32)
    out = torch.empty_like(q)
    A.attn_prefill(q, k, v, cu, out)
    torch.cuda.synchronize()
    check(torch, out, q, k, v, 0, 1000)
    k[:, 0, 0] = lift.flip(0)[:, 0].to(k.dtype)  # and ones that fall
    A.attn_prefill(q, k, v, cu, out)
    torch.cuda.synchronize()
    check(torch, out, q, k, v, 0, 1000)
    k[500, 0] = 100.0
    q[500:] = 4.0
    A.attn_prefill(q, k, v, cu, out)
    torch.cuda.synchronize()
    check(torch, out, q, k, v, 0, 1000)


def test_captured_calls_follow_the_lengths():
    torch = _torch()
    from fngine_b200 import attention as A
    q, k, v = inputs(torch, 800, 4, 2, 64, "bfloat16", 2)
    cu = torch.tensor([0, 400, 800], device="cuda", dtype=torch.int32)
    out = torch.empty_like(q)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        A.attn_prefill(q, k, v, cu, out)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            A.attn_prefill(q, k, v, cu, out)
            A.attn_prefill(q, k, v, cu, out)
        for ends in ([0, 400, 800], [0, 0, 800], [10, 700, 701]):
            cu.copy_(torch.tensor(ends, dtype=torch.int32))
            graph.replay()
            s.synchronize()
            for a, b in zip(ends, ends[1:]):
                if b > a:
                    check(torch, out, q, k, v, a, b)


def test_lengths_that_make_no_sense_stay_within_the_tensors():
    """Device values outside of 0 .. tokens are taken as the nearer end, a falling end as an empty sequence."""
    torch = _torch()
    from fngine_b200 import attention as A
    q, k, v = inputs(torch, 300, 2, 1, 64, "float16", 2)
    out = torch.full_like(q, 5.0)
    A.attn_prefill(q, k, v, torch.tensor([120, 100, 4000], device="cuda", dtype=torch.int32), out)
    torch.cuda.synchronize()
    check(torch, out, q, k, v, 100, 300)
    assert bool((out[:100] == 5).all())
    A.attn_prefill(q, k, v, torch.tensor([-7, 50, -3], device="cuda", dtype=torch.int32), out)
    torch.cuda.synchronize()
    check(torch, out, q, k, v, 0, 50)
    assert bool((out[50:100] == 5).all())


@pytest.mark.parametrize("dim", [64, 128])
def test_a_key_that_is_not_a_number_reaches_the_rows_that_see_it(dim):
    """One key that is not a number, at every place of a group of 32: NaN in the rows from it on, and in no other."""
    torch = _torch()
    from fngine_b200 import attention as A
    g = torch.Generator(device="cuda").manual_seed(5)
    q, k, v = (torch.randn(300, 2, dim, generator=g, device="cuda").bfloat16() for _ in range(3))
    cu = torch.tensor([0, 300], dtype=torch.int32, device="cuda")
    for at in list(range(32)) + [33, 101, 127, 128, 140, 172, 255, 256, 299]:
        bad, out = k.clone(), torch.zeros_like(q)
        bad[at, 1, dim // 2] = float("nan")
        A.attn_prefill(q, bad, v, cu, out)
        torch.cuda.synchronize()
        nan = torch.isnan(out)
        assert not bool(nan[:, 0].any()) and not bool(nan[:at, 1].any()) and bool(nan[at:, 1].all()), at


def test_offsets_beyond_32_bits():
    """Tokens that lie some 10 GB behind the first one."""
    torch = _torch()
    from fngine_b200 import attention as A
    tokens, H, K, D = 200000, 2, 1, 128
    wide = torch.empty(tokens, 24576, dtype=torch.bfloat16, device="cuda")
    first = tokens - 700
    wide[first:] = torch.randn(700, 24576, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda").bfloat16()
    q, k, v, out = wide[:, 128:128 + H * D].unflatten(1, (H, D)), wide[:, 1024:1024 + D].unflatten(1, (K, D)), wide[:, 24448:].unflatten(1, (K, D)), None
    out = wide[:, 4096:4096 + H * D].unflatten(1, (H, D))
    cu = torch.tensor([first, tokens - 200, tokens], dtype=torch.int32, device="cuda")
    A.attn_prefill(q, k, v, cu, out)
    torch.cuda.synchronize()
    last = lambda x: x[first:]
    check(torch, last(out), last(q), last(k), last(v), 0, 500)
    check(torch, last(out), last(q), last(k), last(v), 500, 700)
