"""One key far above many others, whose weights are small one by one and not in sum: they must not fall below the smallest number of the weights'
type. fp16 has steps of 2^-24 there, half of one is the most that a weight may be off; the kernels keep fp16 weights at 2^7 times the formula's
(2^(7 + 8) at most), so that is 2^-32 of the largest weight: 2^-32 sum |v| in all, beside half a step 2^-11 (bf16: 2^-8) of every
weight, 2 (D 2^-23 S + 2^-18) + 2^-18 from scores, exponentials and sums, and half a step of the output."""
import math

import pytest

pytestmark = pytest.mark.gpu
HALF = {"bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}


def bound(want, dtype, S, dim, weights):
    """v is 0 at the key above and 1 at the others, so an output is the others' weight."""
    h = HALF[dtype]
    tol = (h + 2 * (dim * 2.0 ** -23 * S + 2.0 ** -18) + 2.0 ** -18) * want + (2.0 ** -32 * weights if dtype == "float16" else 0.0)
    return tol + h * (want + tol) + (2.0 ** -25 if dtype == "float16" else 0.0)


def above(torch, dim, octaves, dt):
    """A value that every element of the key above has; its scores are `octaves` powers of two over the others' zeros, up to rounding."""
    return (torch.tensor(octaves * math.log(2) * dim ** -0.5)).to(dt)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("octaves", [14.0, 20.0, 25.5, 28.0])
def test_drafted_tokens(octaves, dim, dtype):
    import torch
    from fngine_b200 import attention as A
    page, drafted, heads, kv = 64, 3, 8, 2
    dt = getattr(torch, dtype)
    for n in (60000, 700):
        pages = -(-(n + drafted) // page)
        for place in (0, n // 2, n - 1):
            kc, vc = torch.zeros(pages, page, kv, dim, device="cuda", dtype=dt), torch.ones(pages, page, kv, dim, device="cuda", dtype=dt)
            a = above(torch, dim, octaves, dt)
            kc[place // page, place % page], vc[place // page, place % page] = a.item(), 0
            q = torch.ones(1, drafted, heads, dim, device="cuda", dtype=dt)
            out, ws = torch.full_like(q, float("nan")), A.attn_tree_workspace(1, drafted, heads, kv, dim)
            A.attn_tree_decode(q, A.KvCache(kc, vc), torch.arange(pages, device="cuda", dtype=torch.int32)[None], torch.tensor([n], device="cuda", dtype=torch.int32), out, ws)
            torch.cuda.synchronize()
            score = float(a) * dim * dim ** -0.5
            for i in range(drafted):
                others = (n + i) * math.exp(-score)
                want = others / (1 + others)
                assert bool(((out[0, i].double() - want).abs() <= bound(want, dtype, score, dim, n + i)).all()), (n, place, i, float(out[0, i].double().mean()), want)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("octaves", [14.0, 20.0, 25.5, 28.0])
def test_prompts(octaves, dim, dtype):
    import torch
    from fngine_b200 import attention as A
    dt, n = getattr(torch, dtype), 20000
    for place in (0, 300):
        k, v = torch.zeros(n, 1, dim, device="cuda", dtype=dt), torch.ones(n, 1, dim, device="cuda", dtype=dt)
        a = above(torch, dim, octaves, dt)
        k[place], v[place] = a.item(), 0
        q = torch.ones(n, 1, dim, device="cuda", dtype=dt)
        out = torch.full_like(q, float("nan"))
        A.attn_prefill(q, k, v, torch.tensor([0, n], device="cuda", dtype=torch.int32), out)
        torch.cuda.synchronize()
        score = float(a) * dim * dim ** -0.5
        row = torch.arange(n, device="cuda", dtype=torch.float64)
        others = row * math.exp(-score)
        want = torch.where(row < place, torch.ones_like(others), others / (1 + others))
        # (a row's largest weight is the key's above: the exponents refer to it, or to a score that is at most eight powers of two below)
        assert bool(((out[:, 0].double() - want[:, None]).abs() <= bound(want, dtype, score, dim, row)[:, None]).all())
