"""Attention of drafted tokens through a block table that is a range of a wider one's columns: the columns beside it belong to others."""
import pytest

from test_gpu_attn_tree import compare, reference, setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("first,columns", [(0, 3), (90, 10), (37, 4), (99, 1)])
@pytest.mark.parametrize("page,dim,dtype", [(16, 128, "bfloat16"), (5, 64, "float16")])
def test_contexts_end_at_the_columns_of_the_view(first, columns, page, dim, dtype):
    """Contexts inside, at and behind the view's last column, with pages of others that hold large keys and values in the hidden columns: bit
    for bit what the same columns give as a table of their own."""
    import torch
    from fngine_b200 import attention as A
    seqs, drafted, room = 3, 4, columns * page
    q, kc, vc, _, _ = setup(torch, seqs, drafted, 6, 2, dim, page, [room] * seqs, dtype, 31 + first)
    spare = 7
    others = torch.full((spare, page, 2, dim), 40.0, device="cuda", dtype=kc.dtype)
    kc, vc = torch.cat((kc, others)), torch.cat((vc, others))
    own = kc.shape[0] - spare
    wide = own + torch.randint(0, spare, (seqs, 100), device="cuda", dtype=torch.int32, generator=torch.Generator(device="cuda").manual_seed(2))
    wide[:, first:first + columns] = torch.randperm(own, device="cuda", dtype=torch.int32, generator=torch.Generator(device="cuda").manual_seed(3))[:seqs * columns].view(seqs, columns)
    view, ws = wide[:, first:first + columns], A.attn_tree_workspace(seqs, drafted, 6, 2, dim)
    cache = A.KvCache(kc, vc)
    for contexts in ([0, room - drafted, room - 1], [room - 2, room, room + 1], [room + 1000, 2 ** 31 - 1, 1], [room - drafted + 1, room, room]):
        ctx = torch.tensor([min(c, 2 ** 31 - 1) for c in contexts], device="cuda", dtype=torch.int32)
        out, plain = torch.full_like(q, float("nan")), torch.full_like(q, float("nan"))
        A.attn_tree_decode(q, cache, view, ctx, out, ws)
        A.attn_tree_decode(q, cache, view.contiguous(), ctx, plain, ws)
        torch.cuda.synchronize()
        assert torch.equal(out, plain)
        compare(out, *reference(torch, q, kc, vc, view, contexts, None))
        one = torch.full_like(q, float("nan"))
        for s in range(seqs):  # a sequence by itself sees the same
            A.attn_tree_decode(q[s:s + 1], cache, view[s:s + 1], ctx[s:s + 1], one[s:s + 1], ws)
        torch.cuda.synchronize()
        compare(one, *reference(torch, q, kc, vc, view, contexts, None))
    assert A.attn_tree_status(ws) == 0
