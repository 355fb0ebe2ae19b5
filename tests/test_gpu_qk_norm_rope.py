"""Norms and rotation of queries and keys against the formula in 64 bits.

The tolerance counts what fp32 does: the mean of squares, its root (2 ulp), two products by it (together below 2^-21
relative), and the sine and cosine of an angle reduced in 64 bits (below 2^-21): (|a| + |b|) 2^-19 for a pair (a, b), then half a
step of the output's type (bf16 2^-8, fp16 2^-11 of the value; below fp16's smallest normal number 2^-14 its steps are all
2^-24, half of one 2^-25, whatever the value)."""
import pytest

pytestmark = pytest.mark.gpu
HALF_STEP = {"bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}


def _torch():
    import torch
    assert torch.cuda.is_available()
    return torch


def reference(torch, x, weight, eps, inv_freq, positions, sections, adjacent):
    """(y, |a| + |b| of every value's pair) of x [tokens][heads][dim]."""
    x = x.double()
    if weight is not None:
        x = x / (x.pow(2).mean(2, keepdim=True) + eps).sqrt() * weight.double()
    if inv_freq is None:
        return x, x.abs()
    rot = 2 * inv_freq.numel()
    pos = torch.cat([positions[a].double()[:, None].expand(-1, n) for a, n in enumerate(sections)], 1)
    angle = (pos * inv_freq.double())[:, None, :]
    c, s = angle.cos(), angle.sin()
    y, size = x.clone(), x.abs()
    lo, hi = (slice(0, rot, 2), slice(1, rot, 2)) if adjacent else (slice(0, rot // 2), slice(rot // 2, rot))
    a, b = x[:, :, lo], x[:, :, hi]
    y[:, :, lo], y[:, :, hi] = a * c - b * s, b * c + a * s
    size[:, :, lo] = size[:, :, hi] = a.abs() + b.abs()
    return y, size


def check(torch, got, want, size):
    tol = size * 2.0 ** -19
    least = 2.0 ** -14 if got.dtype == torch.float16 else 0.0  # (fp16: subnormal results)
    tol = tol + HALF_STEP[str(got.dtype).split(".")[1]] * (want.abs() + tol).clamp(min=least)
    off = (got.double() - want).abs()
    if not bool((off <= tol).all()):
        at = int((off / tol).argmax())
        raise AssertionError("%d values off, worst %r against %r, tolerance %r" % (int((off > tol).sum()), float(got.reshape(-1)[at]), float(want.reshape(-1)[at]), float(tol.reshape(-1)[at])))


# tokens, heads, kv heads, dim, rotated, sections, adjacent, type, weights' type, slots, far
CASES = [(1, 1, 1, 64, 64, None, False, "bfloat16", "bfloat16", False, 10), (3, 48, 8, 128, 128, None, False, "bfloat16", "float32", True, 2000000000),
         (5, 7, 1, 128, 32, None, True, "float16", "float16", True, 1000000), (130, 16, 2, 256, 64, None, False, "bfloat16", "bfloat16", False, 40000),
         (67, 14, 2, 64, 48, (4, 10, 10), False, "float16", "float32", False, 9000), (33, 32, 8, 128, 128, (16, 24, 24), True, "bfloat16", "bfloat16", True, 500),
         (9, 100, 40, 256, 256, (1, 0, 120, 7), False, "float16", "bfloat16", True, 100000), (4100, 6, 2, 128, 112, (30, 26), False, "bfloat16", "float32", False, 8192),
         (2, 513, 511, 64, 16, None, False, "bfloat16", "float16", False, 77)]


@pytest.mark.parametrize("tokens,heads,kv,dim,rot,sections,adjacent,dtype,wtype,slots,far", CASES)
def test_against_the_formula(tokens, heads, kv, dim, rot, sections, adjacent, dtype, wtype, slots, far):
    torch = _torch()
    from fngine_b200 import attention as A
    gen = torch.Generator(device="cuda").manual_seed(tokens + heads)
    dt = getattr(torch, dtype)
    # parts of one projection's output, with something between the tokens
    wide = (torch.randn(tokens, (heads + 2 * kv) * dim + 24, generator=gen, device="cuda") * 3).to(dt)
    q, k, v = (wide[:, a * dim:b * dim].unflatten(1, (b - a, dim)) for a, b in ((0, heads), (heads, heads + kv), (heads + kv, heads + 2 * kv)))
    qw, kw = ((torch.rand(dim, generator=gen, device="cuda") + 0.5).to(getattr(torch, wtype)) for _ in "qk")
    inv = (1e6 ** (-torch.arange(rot // 2, device="cuda", dtype=torch.float64) / (rot // 2))).float()
    sections = sections or (rot // 2,)
    pos = torch.randint(0, far + 1, (len(sections), tokens), generator=gen, device="cuda", dtype=torch.int32)
    pos[0, 0] = far
    rows, at, where = tokens, torch.arange(tokens, device="cuda"), None
    if slots:
        rows = tokens + 11
        at = torch.randperm(rows, generator=gen, device="cuda")[:tokens]
        where = at.clone()
    q_out = torch.full((tokens, heads, dim), 7.0, device="cuda", dtype=dt)
    k_out, v_out = torch.full((rows, kv, dim), 7.0, device="cuda", dtype=dt), torch.full((rows, kv, dim), 7.0, device="cuda", dtype=dt)
    A.qk_norm_rope(q, k, v, qw, kw, 1e-6, A.Rope(inv, sections, adjacent), pos, q_out, k_out, v_out, slots=where)
    torch.cuda.synchronize()
    check(torch, q_out, *reference(torch, q, qw, 1e-6, inv, pos, sections, adjacent))
    check(torch, k_out[at], *reference(torch, k, kw, 1e-6, inv, pos, sections, adjacent))
    assert torch.equal(v_out[at], v)
    rest = torch.ones(rows, dtype=torch.bool, device="cuda")
    rest[at] = False
    assert bool((k_out[rest] == 7).all()) and bool((v_out[rest] == 7).all())


def test_parts_that_are_left_out():
    """No rotation, no norm of q, of k, of either; keys without values; in place; slots that store nothing; no tokens."""
    torch = _torch()
    from fngine_b200 import attention as A
    gen = torch.Generator(device="cuda").manual_seed(3)
    T, H, K, D = 21, 6, 2, 128
    q, k, v = (torch.randn(T, h, D, generator=gen, device="cuda").to(torch.bfloat16) for h in (H, K, K))
    w = torch.rand(D, generator=gen, device="cuda") + 0.5
    inv = torch.rand(64, generator=gen, device="cuda")
    pos = torch.arange(T, device="cuda", dtype=torch.int32) - 5  # before the start, too
    rope = A.Rope(inv)
    for qw, kw, turn in ((w, None, rope), (None, w, rope), (None, None, rope), (w, w, None), (None, None, None)):
        qo, ko, vo = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
        A.qk_norm_rope(q, k, v, qw, kw, 1e-5, turn, pos, qo, ko, vo)
        f, p = (inv, pos[None]) if turn else (None, None)
        check(torch, qo, *reference(torch, q, qw, 1e-5, f, p, (64,), False))
        check(torch, ko, *reference(torch, k, kw, 1e-5, f, p, (64,), False))
        assert torch.equal(vo, v)
        ko2 = torch.zeros_like(k)
        A.qk_norm_rope(q, k, None, qw, kw, 1e-5, turn, pos, qo, ko2, None)
        assert torch.equal(ko2, ko)
        q2, k2, v2 = q.clone(), k.clone(), v.clone()
        A.qk_norm_rope(q2, k2, v2, qw, kw, 1e-5, turn, pos, q2, k2, v2)
        assert torch.equal(q2, qo) and torch.equal(k2, ko) and torch.equal(v2, v)
    slots = torch.arange(T, device="cuda")
    slots[4], slots[5], slots[6] = -1, T, 2 ** 40
    ko, vo = torch.zeros_like(k), torch.zeros_like(v)
    A.qk_norm_rope(q, k, v, None, None, 0.0, None, pos, torch.empty_like(q), ko, vo, slots=slots)
    keep = torch.ones(T, dtype=torch.bool, device="cuda")
    keep[4:7] = False
    assert torch.equal(ko[keep], k[keep]) and torch.equal(vo[keep], v[keep]) and not bool(ko[4:7].any()) and not bool(vo[4:7].any())
    A.qk_norm_rope(q[:0], k[:0], v[:0], w, w, 1e-5, rope, pos[:0], qo[:0], ko[:0], vo[:0])
    torch.cuda.synchronize()


def test_rows_of_zeros_and_values_that_are_not_finite():
    torch = _torch()
    from fngine_b200 import attention as A
    q = torch.randn(4, 3, 64, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).half()
    q[1, 1] = 0
    q[2, 0, 5] = float("inf")
    w = torch.ones(64, device="cuda")
    out, ko = torch.empty_like(q), torch.empty_like(q)
    A.qk_norm_rope(q, q, None, w, w, 1e-6, None, None, out, ko, None)
    want = reference(torch, q, w, 1e-6, None, None, None, False)[0]
    assert not bool(out[1, 1].any()) and bool(torch.isnan(out[2, 0, 5]))
    rows = [(t, h) for t in range(4) for h in range(3) if (t, h) != (2, 0)]
    for t, h in rows:
        check(torch, out[t, h], want[t, h], want[t, h].abs())


def test_captured_and_chained():
    """Replayed from a graph, each call behind a kernel that writes its input."""
    torch = _torch()
    from fngine_b200 import attention as A
    q = torch.randn(5, 4, 128, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).bfloat16()
    k, v = q[:, :2].contiguous(), q[:, 2:].contiguous()
    w = torch.ones(128, device="cuda")
    rope, pos = A.Rope(torch.rand(32, device="cuda")), torch.arange(5, device="cuda", dtype=torch.int32)
    mid, out, ko, vo = (torch.zeros_like(t) for t in (q, q, k, v))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run = lambda: (A.qk_norm_rope(q, k, v, w, w, 1e-6, rope, pos, mid, ko, vo), A.qk_norm_rope(mid, k, v, None, None, 0.0, rope, pos, out, ko, vo))
        run()
        s.synchronize()
        want = out.clone()
        mid.zero_(), out.zero_()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            run()
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_one_row_of_positions_for_all_axes():
    """A position row that is expanded to the axes (no memory of its own) is the same as three equal rows, and as one axis."""
    torch = _torch()
    from fngine_b200 import attention as A
    gen = torch.Generator(device="cuda").manual_seed(9)
    q, k = torch.randn(50, 4, 64, generator=gen, device="cuda").bfloat16(), torch.randn(50, 2, 64, generator=gen, device="cuda").bfloat16()
    pos = torch.randint(0, 5000, (1, 50), generator=gen, device="cuda", dtype=torch.int32)
    inv = (1e4 ** (-torch.arange(32, device="cuda") / 32)).float()
    outs = []
    for sections, p in (((10, 12, 10), pos.expand(3, 50)), ((10, 12, 10), pos.repeat(3, 1)), (None, pos)):
        qo, ko = torch.empty_like(q), torch.empty_like(k)
        A.qk_norm_rope(q, k, None, None, None, 0.0, A.Rope(inv, sections), p, qo, ko, None)
        outs.append((qo, ko))
    torch.cuda.synchronize()
    for a, b in outs[1:]:
        assert torch.equal(a, outs[0][0]) and torch.equal(b, outs[0][1])


def test_offsets_beyond_32_bits():
    """Tokens some 10 GB behind the first one, into slots as far behind the first one."""
    torch = _torch()
    from fngine_b200 import attention as A
    tokens, H, K, D = 200000, 2, 1, 128
    wide = torch.zeros(tokens, 24576, dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(2)
    wide[-300:] = torch.randn(300, 24576, generator=gen, device="cuda").bfloat16()
    q, k, v = wide[:, 128:384].unflatten(1, (H, D)), wide[:, 1024:1152].unflatten(1, (K, D)), wide[:, 24448:].unflatten(1, (K, D))
    ko, vo = (wide[:, c:c + D].unflatten(1, (K, D)) for c in (8192, 16384))
    slots = torch.full((tokens,), -1, device="cuda")
    slots[-300:] = torch.arange(tokens - 1, tokens - 301, -1, device="cuda")
    pos = torch.arange(tokens, device="cuda", dtype=torch.int32)
    inv = (1e4 ** (-torch.arange(64, device="cuda") / 64)).float()
    want = [reference(torch, x[-300:], None, 0.0, inv, pos[None, -300:], (64,), False) for x in (q, k)]
    A.qk_norm_rope(q, k, v, None, None, 0.0, A.Rope(inv), pos, q, ko, vo, slots=slots)
    torch.cuda.synchronize()
    check(torch, q[-300:], *want[0])
    check(torch, ko[-300:].flip(0), *want[1])
    assert torch.equal(vo[-300:].flip(0), v[-300:]) and not bool(ko[:-300].any())
