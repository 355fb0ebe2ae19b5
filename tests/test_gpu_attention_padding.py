"""Prompts in a batch that is padded to a fixed width: tokens in front of the first and behind the last sequence have no attention. Their rows of
attn_prefill's output are zeros where the caller asks for that, and the branch adds nothing to their residual streams."""
import pytest

from test_gpu_attention_branch import DIM, HEADS, HIDDEN, KV, make_branch
from test_gpu_attn_prefill import check, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kv,dim,dtype", [(4, 2, 64, "float16"), (6, 2, 128, "bfloat16"), (1, 1, 128, "float16")])
@pytest.mark.parametrize("ends", [[0, 900], [40, 240, 240, 541], [0, 256, 512], [300, 300], [0], [900, 900], [0, 0, 899], [899, 900], [1, 5, 900], [0, 1]])
def test_rows_outside_of_all_sequences_are_zeros(ends, heads, kv, dim, dtype):
    """Every other row as without the padding, bit for bit; nothing beside the rows' heads is written."""
    import torch
    from fngine_b200 import attention as A
    q, k, v = inputs(torch, 900, heads, kv, dim, dtype, 7)
    cu = torch.tensor(ends, device="cuda", dtype=torch.int32)
    first, last = ends[0], ends[-1]
    for x in (q, k, v):
        x[:first] = float("nan")
        x[last:] = float("nan")
    plain = torch.zeros_like(q)
    A.attn_prefill(q, k, v, cu, plain)
    wide = torch.full((900, heads * dim + 64), 3.0, device="cuda", dtype=q.dtype)
    out, status = wide[:, 32:32 + heads * dim].unflatten(1, (heads, dim)), torch.zeros(1, dtype=torch.int32, device="cuda")
    out.fill_(float("nan"))
    A.attn_prefill(q, k, v, cu, out, status=status, padded=True)
    torch.cuda.synchronize()
    assert int(status) == 0 and torch.equal(out, plain)
    assert not bool(out[:first].any()) and not bool(out[last:].any())
    assert bool((wide[:, :32] == 3).all()) and bool((wide[:, 32 + heads * dim:] == 3).all())
    for a, b in zip(ends, ends[1:]):
        if b > a:
            check(torch, out, q, k, v, a, b)


def test_ends_that_fall_or_lie_outside():
    """Ends outside of 0 .. tokens are taken as the nearer end: what no sequence covers is zeros."""
    import torch
    from fngine_b200 import attention as A
    q, k, v = inputs(torch, 300, 2, 1, 64, "float16", 2)
    for ends, a, b in (([120, 100, 4000], 100, 300), ([-7, 50, -3], 0, 50), ([400, 500], 300, 300), ([2 ** 31 - 1, -2 ** 31], 300, 300)):
        out = torch.full_like(q, float("nan"))
        A.attn_prefill(q, k, v, torch.tensor(ends, device="cuda", dtype=torch.int32), out, padded=True)
        torch.cuda.synchronize()
        if b > a:
            check(torch, out, q, k, v, a, b)
        assert not bool(out[:a].any()) and not bool(out[b:].any())


@pytest.mark.parametrize("kind,tokens", [("fp8", 512), ("fp8", 100), ("q4", 16)])
def test_a_padded_batch_adds_nothing_to_its_padding(kind, tokens):
    """The branch over sequences that leave tokens out, after a call that filled its buffers and with buffers that hold NaN; eager and replayed
    as the ends move. The sequences' rows are those of a call without the padding."""
    import torch
    from fngine_b200 import attention as A
    branch = make_branch(torch, kind, tokens)
    gen = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(tokens, HIDDEN, generator=gen, device="cuda").bfloat16()
    inj, before = torch.randn(tokens, 4, generator=gen, device="cuda"), torch.randn(tokens, 4, HIDDEN, generator=gen, device="cuda")
    pos, X = torch.arange(tokens, device="cuda", dtype=torch.int32) % 97, before.clone()
    t = lambda f: int(f * tokens)
    cases = [[0, t(0.4), tokens], [0, t(0.3), t(0.6)], [t(0.2), t(0.5), tokens], [t(0.1), t(0.1), t(0.2)], [0, 0, 0], [tokens, tokens, tokens], [1, 2, tokens - 1]]
    cu = torch.tensor(cases[0], device="cuda", dtype=torch.int32)
    step = lambda: A.forward_attention_prefill(branch, x, cu, pos, X, inj)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        step()
        with torch.cuda.graph(graph, stream=s):
            step()
    torch.cuda.synchronize()
    for ends in cases:
        cu.copy_(torch.tensor(ends, dtype=torch.int32))
        results = []
        for run in (step, graph.replay):
            branch.o.fill_(float("nan"))
            X.copy_(before)
            run()
            torch.cuda.synchronize()
            results.append(X.clone())
        a, b = ends[0], ends[-1]
        assert torch.equal(results[0], results[1])
        assert torch.equal(results[0][:a], before[:a]) and torch.equal(results[0][b:], before[b:])
        assert bool(torch.isfinite(results[0]).all()) and (a == b or bool((results[0][a:b] != before[a:b]).any(2).all()))
        assert not bool(branch.o[:a].any()) and not bool(branch.o[b:tokens].any())
    assert branch.status() == 0
