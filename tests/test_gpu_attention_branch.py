"""The operators of the attention branch together, as a model runs them: prompts through projection, norms and rotation, attention and the
residual write, their keys and values into a paged cache, then drafted tokens on top of them. Each stage is held against its formula
on the stage before it, so the tolerances are the operators' own; a prompt in two parts (the second as drafted tokens) is held
against the prompt as a whole."""
import pytest

from test_gpu_attn_prefill import check as check_prompt
from test_gpu_attn_tree import compare, reference, tree_mask
from test_gpu_qk_norm_rope import check as check_rope, reference as rope_reference

pytestmark = pytest.mark.gpu
HIDDEN, HEADS, KV, DIM = 1280, 12, 4, 64


def _torch():
    import torch
    assert torch.cuda.is_available()
    return torch


def make_branch(torch, kind, max_tokens):
    from fngine_b200 import attention as A, linear
    gen = torch.Generator(device="cuda").manual_seed(17)

    def weight(n, k):
        if kind == "q4":
            codes = torch.randint(0, 256, (n, k // 2), generator=gen, device="cuda", dtype=torch.uint8)
            return linear.Q4GroupWeight(codes, (torch.rand(n, k // 64, generator=gen, device="cuda") * 0.01 + 0.002).bfloat16())
        codes = (torch.randn(n, k, generator=gen, device="cuda") * 20).to(torch.float8_e4m3fn).view(torch.uint8)
        return linear.Fp8RowWeight(codes, torch.rand(n, generator=gen, device="cuda") * 0.002 + 0.0005)

    qw, kw = (torch.rand(DIM, generator=gen, device="cuda") + 0.5 for _ in "qk")
    inv = (1e5 ** (-torch.arange(DIM // 2, device="cuda", dtype=torch.float64) / (DIM // 2))).float()
    return A.AttentionBranch(weight((HEADS + 2 * KV) * DIM, HIDDEN), weight(HIDDEN, HEADS * DIM), qw, kw, 1e-6, A.Rope(inv), HEADS, KV, DIM, max_tokens)


def dense(torch, w):
    """A weight in 64 bits."""
    if hasattr(w, "group"):
        c = torch.stack((w.codes % 16, w.codes // 16), 2).reshape(w.n, w.k).double() - 8
        return c * w.scales.double().repeat_interleave(w.group, 1)
    return w.codes.view(torch.float8_e4m3fn).double() * w.scales.double()[:, None]


def check_product(torch, got, x, w, factor=None):
    """A projection in fp32 or bf16 against 64 bits: additions in chains of k / 16 + 60, each within 2^-22 of sum |w x| (the FP8 route drops
    activations below 2^-17 of their row's largest: 2^-17 max|x| sum |w|), half a step of bf16 on top."""
    d = dense(torch, w)
    want, size = x.double() @ d.T, x.double().abs() @ d.abs().T
    tol = (w.k // 16 + 60) * 2.0 ** -22 * size + 2.0 ** -17 * x.double().abs().amax(1, keepdim=True) * d.abs().sum(1)
    if factor is not None:  # the four residual streams
        want, tol = factor.double()[:, :, None] * want[:, None], factor.double().abs()[:, :, None] * tol[:, None]
        tol = tol + 2.0 ** -22 * want.abs()  # (product and sum)
    elif got.dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * (want.abs() + tol)
    assert bool(((got.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("kind,lengths,drafted", [("fp8", [70, 1, 333], 5), ("fp8", [17, 40], 1), ("q4", [3, 2, 9], 4)])
def test_prompts_then_drafted_tokens(kind, lengths, drafted):
    torch = _torch()
    from fngine_b200 import attention as A
    seqs, tokens, page = len(lengths), sum(lengths), 16
    branch = make_branch(torch, kind, 512)
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(tokens, HIDDEN, generator=gen, device="cuda").bfloat16()
    inj = torch.randn(tokens, 4, generator=gen, device="cuda")
    X = torch.zeros(tokens, 4, HIDDEN, device="cuda")
    pages = [-(-(n + drafted) // page) for n in lengths]
    table = torch.full((seqs, max(pages)), -1, dtype=torch.int32, device="cuda")
    order, at = torch.randperm(sum(pages), generator=gen, device="cuda").int(), 0
    for s, p in enumerate(pages):
        table[s, :p] = order[at:at + p]
        at += p
    kc, vc = (torch.zeros(sum(pages) + 1, page, KV, DIM, device="cuda", dtype=torch.bfloat16) for _ in "kv")
    cache = A.KvCache(kc, vc)
    slot = lambda s, p: int(table[s, p // page]) * page + p % page
    where = torch.tensor([slot(s, p) for s, n in enumerate(lengths) for p in range(n)], device="cuda")
    pos = torch.tensor([p for n in lengths for p in range(n)], device="cuda", dtype=torch.int32)
    ends = [0]
    for n in lengths:
        ends.append(ends[-1] + n)
    cu = torch.tensor(ends, device="cuda", dtype=torch.int32)
    if tokens <= 16 or kind == "fp8":
        A.forward_attention_prefill(branch, x, cu, pos, X, inj, cache, where)
    torch.cuda.synchronize()
    q, k, v = branch.parts(tokens)
    raw = torch.empty_like(branch.rows[:tokens])
    from fngine_b200 import linear
    branch.project(x, 0, linear.store_bf16(raw))
    check_product(torch, raw, x, branch.qkv)
    rq, rk, rv = (r.unflatten(1, (-1, DIM)) for r in raw.split([HEADS * DIM, KV * DIM, KV * DIM], 1))
    check_rope(torch, q, *rope_reference(torch, rq, branch.q_weight, 1e-6, branch.rope.inv_freq, pos[None], (DIM // 2,), False))
    check_rope(torch, k, *rope_reference(torch, rk, branch.k_weight, 1e-6, branch.rope.inv_freq, pos[None], (DIM // 2,), False))
    assert torch.equal(v, rv) and torch.equal(cache.k_rows[where], k) and torch.equal(cache.v_rows[where], v)
    for a, b in zip(ends, ends[1:]):
        check_prompt(torch, branch.o[:tokens], q, k, v, a, b)
    check_product(torch, X, branch.o[:tokens].flatten(1), branch.out, inj)

    # drafted tokens on top
    T = seqs * drafted
    y, inj2 = torch.randn(T, HIDDEN, generator=gen, device="cuda").bfloat16(), torch.randn(T, 4, generator=gen, device="cuda")
    X2 = torch.zeros(T, 4, HIDDEN, device="cuda")
    ctx = torch.tensor(lengths, device="cuda", dtype=torch.int32)
    where2 = torch.tensor([slot(s, n + d) for s, n in enumerate(lengths) for d in range(drafted)], device="cuda")
    pos2 = torch.tensor([n + d for n in lengths for d in range(drafted)], device="cuda", dtype=torch.int32)
    mask = tree_mask(torch, seqs, drafted, 2)
    ws = A.attn_tree_workspace(seqs, drafted, HEADS, KV, DIM)
    A.forward_attention_decode(branch, y, drafted, cache, table, ctx, where2, pos2, ws, X2, inj2, mask=mask)
    torch.cuda.synchronize()
    q2 = branch.parts(T)[0].unflatten(0, (seqs, drafted))
    compare(branch.o[:T].unflatten(0, (seqs, drafted)), *reference(torch, q2, kc, vc, table, lengths, mask))
    check_product(torch, X2, branch.o[:T].flatten(1), branch.out, inj2)
    assert A.attn_tree_status(ws) == 0


def test_the_end_of_a_prompt_as_drafted_tokens():
    """The last tokens of a prompt as a chain of drafted ones, without a mask: the formula is the prompt's, on the keys and values in
    the cache. Both parts put there what the whole prompt does, up to a bf16 step (a projection's sums depend on the number of tokens)."""
    torch = _torch()
    from fngine_b200 import attention as A
    branch = make_branch(torch, "fp8", 512)
    gen = torch.Generator(device="cuda").manual_seed(8)
    n, last, page = 200, 20, 32
    x = torch.randn(n, HIDDEN, generator=gen, device="cuda").bfloat16()
    inj = torch.ones(n, 4, device="cuda")
    table = torch.arange(7, device="cuda", dtype=torch.int32).flip(0)[None].contiguous()
    where = torch.tensor([int(table[0, p // page]) * page + p % page for p in range(n)], device="cuda")
    pos = torch.arange(n, device="cuda", dtype=torch.int32)
    X = torch.zeros(n, 4, HIDDEN, device="cuda")
    caches = []
    for _ in range(2):
        kc, vc = (torch.zeros(7, page, KV, DIM, device="cuda", dtype=torch.bfloat16) for _ in "kv")
        caches.append(A.KvCache(kc, vc))
    A.forward_attention_prefill(branch, x, torch.tensor([0, n], device="cuda", dtype=torch.int32), pos, X, inj, caches[0], where)
    A.forward_attention_prefill(branch, x[:n - last], torch.tensor([0, n - last], device="cuda", dtype=torch.int32), pos[:n - last], X[:n - last].clone(),
                                inj[:n - last], caches[1], where[:n - last])
    ws = A.attn_tree_workspace(1, last, HEADS, KV, DIM)
    A.forward_attention_decode(branch, x[n - last:], last, caches[1], table, torch.tensor([n - last], device="cuda", dtype=torch.int32), where[n - last:],
                               pos[n - last:], ws, X[n - last:].clone(), inj[n - last:])
    torch.cuda.synchronize()
    a, b = caches[0].v_rows[where].double(), caches[1].v_rows[where].double()
    size = (x.double().abs() @ dense(torch, branch.qkv)[-KV * DIM:].abs().T).unflatten(1, (KV, DIM))
    assert bool(((a - b).abs() <= 2.0 ** -7 * torch.maximum(a.abs(), b.abs()) + 2.0 ** -12 * size).all())
    q = branch.parts(last)[0][None]
    compare(branch.o[None, :last], *reference(torch, q, caches[1].k, caches[1].v, table, [n - last], None))


def test_arguments():
    torch = _torch()
    from fngine_b200 import attention as A
    branch = make_branch(torch, "q4", 16)
    with pytest.raises(ValueError):
        A.AttentionBranch(branch.qkv, branch.out, None, None, 0.0, None, HEADS, KV + 1, DIM, 4)
    x, X = torch.zeros(4, HIDDEN, device="cuda", dtype=torch.bfloat16), torch.zeros(4, 4, HIDDEN, device="cuda")
    with pytest.raises(ValueError):
        A.forward_attention_decode(branch, x, 3, None, None, torch.zeros(2, device="cuda", dtype=torch.int32), None, None, None, X, torch.ones(4, 4, device="cuda"))
    q = torch.zeros(4, HEADS, DIM, dtype=torch.bfloat16)  # not on the GPU
    with pytest.raises(ValueError):
        A.attn_prefill(q, q, q, torch.tensor([0, 4], dtype=torch.int32), q)


def test_a_branch_refuses_what_does_not_fit():
    """More tokens than its buffers hold, streams or inj of other shapes; no tokens at all are not an error."""
    torch = _torch()
    from fngine_b200 import attention as A
    branch = make_branch(torch, "fp8", 32)
    make = lambda t: (torch.zeros(t, HIDDEN, device="cuda", dtype=torch.bfloat16), torch.zeros(t, 4, HIDDEN, device="cuda"), torch.ones(t, 4, device="cuda"))
    cu, pos = torch.tensor([0, 0], device="cuda", dtype=torch.int32), torch.zeros(33, device="cuda", dtype=torch.int32)
    for x, X, inj in (make(33), (make(4)[0], make(3)[1], make(4)[2]), (make(4)[0], make(4)[1], make(5)[2]), (make(4)[0][:, :640].contiguous(), *make(4)[1:]),
                      (make(4)[0], make(4)[1].cpu(), make(4)[2])):
        with pytest.raises(ValueError):
            A.forward_attention_prefill(branch, x, cu, pos[:x.shape[0]], X, inj)
        with pytest.raises(ValueError):
            A.forward_attention_decode(branch, x, 1, None, None, torch.zeros(x.shape[0], device="cuda", dtype=torch.int32), None, pos[:x.shape[0]], None, X, inj)
    x, X, inj = make(0)
    A.forward_attention_prefill(branch, x, cu, pos[:0], X, inj)
    A.forward_attention_decode(branch, x, 1, None, None, torch.zeros(0, device="cuda", dtype=torch.int32), None, pos[:0], None, X, inj)


def test_a_captured_decode_step_follows_its_inputs():
    """A step captured once and replayed as the sequences grow, on another stream than it was captured on, against steps without a graph."""
    torch = _torch()
    from fngine_b200 import attention as A
    seqs, page = 3, 16
    branch = make_branch(torch, "q4", 16)
    gen = torch.Generator(device="cuda").manual_seed(23)
    kc, vc = (torch.randn(40, page, KV, DIM, generator=gen, device="cuda").bfloat16() for _ in "kv")
    table = torch.randperm(39, generator=gen, device="cuda").int().view(3, 13)
    cache, ws = A.KvCache(kc, vc), A.attn_tree_workspace(seqs, 1, HEADS, KV, DIM)
    x, inj = torch.randn(seqs, HIDDEN, generator=gen, device="cuda").bfloat16(), torch.randn(seqs, 4, generator=gen, device="cuda")
    X, ctx, slots = torch.zeros(seqs, 4, HIDDEN, device="cuda"), torch.zeros(seqs, dtype=torch.int32, device="cuda"), torch.zeros(seqs, dtype=torch.int64, device="cuda")
    step = lambda: A.forward_attention_decode(branch, x, 1, cache, table, ctx, slots, ctx, ws, X, inj)

    def at(contexts):
        ctx.copy_(torch.tensor(contexts, dtype=torch.int32))
        slots.copy_(torch.tensor([int(table[s, c // page]) * page + c % page for s, c in enumerate(contexts)]))
        X.zero_()

    at([0, 5, 100])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        step()
        with torch.cuda.graph(graph, stream=s):
            step()
    torch.cuda.synchronize()
    for contexts in ([0, 5, 100], [1, 6, 101], [200, 31, 32]):
        at(contexts)
        graph.replay()
        got = X.clone()
        at(contexts)
        step()
        assert torch.equal(got, X) and bool(got.any())
    torch.cuda.synchronize()
    assert A.attn_tree_status(ws) == 0
