"""Scores of thousands: where one key is more than 40 above all others (natural units), the row is that key's value. A score is an fp32 sum of D
products, off by at most e = D 2^-23 sum |scale q k|, so the distance of two is off by 2 e at most, and n other keys weigh no more than n exp(-(40 - 2 e))
beside the one: the output is off by that part of the largest value (as much again in the sum of weights: twice it). The one weight is 2^0 .. 2^8 of the maximum
in use and rounded to the type of v, half a step h of it, while the sum is not; then the output is rounded: (1 + h)^2 - 1 = 2 h + h^2 of the value,
and 2^-18 from the exponential, the sum and the quotient."""
import math

import pytest

from test_gpu_attn_prefill import inputs
from test_gpu_attn_tree import HALF, setup, tree_mask

pytestmark = pytest.mark.gpu


def check_rows(torch, out, q, k, v, sees, scale):
    """out, q [rows][dim], k, v [keys][dim], sees [rows][keys]. Returns how many rows one key takes."""
    s = (q.double() @ k.double().T * scale).masked_fill(~sees, -float("inf"))
    e = q.shape[1] * 2.0 ** -23 * float(((q.double().abs() @ k.double().abs().T) * scale).amax())
    two = s.topk(2, dim=1)
    rows = two.values[:, 0] - two.values[:, 1] > 40
    want, h = v.double()[two.indices[:, 0]], HALF[str(q.dtype).split(".")[1]]
    tol = (2 * h + h * h + 2.0 ** -18) * want.abs() + (2.0 ** -25 if q.dtype == torch.float16 else 0) + 2 * k.shape[0] * math.exp(2 * e - 40) * float(v.double().abs().max())
    assert bool((((out.double() - want).abs() <= tol) | ~rows[:, None]).all())
    return int(rows.sum())


@pytest.mark.parametrize("dim,drafted,heads,kv,dtype,factor", [(64, 3, 4, 2, "bfloat16", 3000.0), (128, 16, 12, 2, "bfloat16", 3000.0), (64, 40, 2, 2, "float16", 2000.0),
                                                               (128, 5, 6, 2, "float16", 1000.0)])
def test_drafted_tokens(dim, drafted, heads, kv, dtype, factor):
    import torch
    from fngine_b200 import attention as A
    contexts = [500, 90]
    q, kc, vc, table, ctx = setup(torch, 2, drafted, heads, kv, dim, 16, contexts, dtype, 11)
    q, mask = q * factor, tree_mask(torch, 2, drafted, 4)
    ws, out = A.attn_tree_workspace(2, drafted, heads, kv, dim), torch.full_like(q, float("nan"))
    A.attn_tree_decode(q, A.KvCache(kc, vc), table, ctx, out, ws, mask=mask)
    torch.cuda.synchronize()
    found = 0
    for s, c in enumerate(contexts):
        used = table[s, :-(-(c + drafted) // 16)].long()
        k, v = (x[used].reshape(-1, kv, dim)[:c + drafted] for x in (kc, vc))
        sees = torch.ones(drafted, c + drafted, dtype=torch.bool, device="cuda")
        for d in range(drafted):
            sees[:, c + d] = ((mask[s] >> d) & 1).bool()
        for h in range(heads):
            found += check_rows(torch, out[s, :, h], q[s, :, h], k[:, h * kv // heads], v[:, h * kv // heads], sees, dim ** -0.5)
    assert found > drafted * heads  # more than half of the rows


@pytest.mark.parametrize("dim,dtype,factor", [(64, "bfloat16", 3000.0), (128, "bfloat16", 3000.0), (64, "float16", 2000.0), (128, "float16", 1000.0)])
def test_prompts(dim, dtype, factor):
    import torch
    from fngine_b200 import attention as A
    n = 700
    q, k, v = inputs(torch, n, 4, 2, dim, dtype, 3, factor)
    out = torch.full_like(q, float("nan"))
    A.attn_prefill(q, k, v, torch.tensor([0, n], device="cuda", dtype=torch.int32), out)
    torch.cuda.synchronize()
    sees = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
    found = sum(check_rows(torch, out[1:, h], q[1:, h], k[:, h // 2], v[:, h // 2], sees[1:], dim ** -0.5) for h in range(4))
    assert found > 2 * n
