"""Calls that overlap on two streams, with a branch and a workspace each: results are those of the same calls one after another, bit for bit."""
import pytest

from test_gpu_attention_branch import DIM, HEADS, HIDDEN, KV, make_branch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,lengths", [("fp8", [300, 17, 500]), ("q4", [5, 2, 9])])
def test_two_branches_at_once(kind, lengths):
    """Prompts and then decode steps of two users' batches: each on its own stream, many times over, against one stream."""
    import torch
    from fngine_b200 import attention as A
    tokens, seqs, page, steps = sum(lengths), len(lengths), 16, 6
    columns = -(-(max(lengths) + steps) // page)

    def user(seed):
        """A function that runs everything and returns the residual streams after it."""
        branch = make_branch(torch, kind, max(tokens, 16))
        gen = torch.Generator(device="cuda").manual_seed(seed)
        x, y = (torch.randn(n, HIDDEN, generator=gen, device="cuda").bfloat16() for n in (tokens, seqs))
        inj = torch.randn(tokens, 4, generator=gen, device="cuda")
        X, Y = torch.zeros(tokens, 4, HIDDEN, device="cuda"), torch.zeros(seqs, 4, HIDDEN, device="cuda")
        cache = A.KvCache(*(torch.zeros(seqs * columns, page, KV, DIM, device="cuda", dtype=torch.bfloat16) for _ in "kv"))
        table = torch.randperm(seqs * columns, generator=gen, device="cuda").int().view(seqs, columns)
        ends = [sum(lengths[:i]) for i in range(seqs + 1)]
        cu = torch.tensor(ends, device="cuda", dtype=torch.int32)
        host = table.cpu()
        slot = lambda s, p: int(host[s, p // page]) * page + p % page
        where = torch.tensor([slot(s, p) for s, n in enumerate(lengths) for p in range(n)], device="cuda")
        pos = torch.tensor([p for n in lengths for p in range(n)], device="cuda", dtype=torch.int32)
        later = [(torch.tensor([n + i for n in lengths], device="cuda", dtype=torch.int32), torch.tensor([slot(s, n + i) for s, n in enumerate(lengths)], device="cuda"))
                 for i in range(steps)]
        ws = A.attn_tree_workspace(seqs, 1, HEADS, KV, DIM)

        def run():
            X.zero_(), Y.zero_()
            A.forward_attention_prefill(branch, x, cu, pos, X, inj, cache, where)
            for ctx, to in later:
                A.forward_attention_decode(branch, y, 1, cache, table, ctx, to, ctx, ws, Y, inj[:seqs])
            return X.clone(), Y.clone()

        return run, lambda: branch.status() | A.attn_tree_status(ws)

    users = [user(1), user(2)]
    want = [run() for run, _ in users]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(8):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(users[i][0]())
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for pair in got[i] for a, b in zip(pair, want[i])) and users[i][1]() == 0
    assert not torch.equal(want[0][0], want[1][0]) and bool(want[0][1].any())
