"""Attention of drafted tokens over a paged cache against its formula in 64 bits.

The tolerance: weights are rounded once to the type of v (half a step h of each: bf16 2^-8, fp16 2^-11), so an output is off by at most h
sum_j w_j |v_j| = h B; scores are fp32 sums of D products (D 2^-23 sum |scale q k|, which moves a weight by that relative part, and the
exponential another 2^-21): 2 (D 2^-23 S + 2^-21) B with S the row's largest sum |scale q k|; sums over the keys 2^-18 B; and
half a step of the output. Weights below fp16's normal range are off by 2^-25 of the largest at most: 2^-25 sum |v| over the keys."""
import pytest

pytestmark = pytest.mark.gpu
HALF = {"bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}


def _torch():
    import torch
    assert torch.cuda.is_available()
    return torch


def setup(torch, seqs, drafted, heads, kv, dim, page, contexts, dtype, seed, spare=3):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = getattr(torch, dtype)
    pages = [-(-(max(0, c) + drafted) // page) for c in contexts]
    total, most = sum(pages) + spare, max(pages) + 2
    order = torch.randperm(total, generator=gen, device="cuda", dtype=torch.int32)
    table = torch.full((seqs, most), -7, device="cuda", dtype=torch.int32)  # columns behind a sequence's pages are not looked at
    at = 0
    for s, p in enumerate(pages):
        table[s, :p] = order[at:at + p]
        at += p
    kc, vc = (torch.randn(total, page, kv, dim, generator=gen, device="cuda").to(dt) for _ in "kv")
    q = (torch.randn(seqs, drafted, heads, dim, generator=gen, device="cuda") * 1.5).to(dt)
    ctx = torch.tensor(contexts, device="cuda", dtype=torch.int32)
    return q, kc, vc, table, ctx


def tree_mask(torch, seqs, drafted, seed):
    import random
    rng = random.Random(seed)
    rows = []
    for _ in range(seqs):
        m = []
        for i in range(drafted):
            p = rng.randrange(-1, i) if i else -1
            m.append((m[p] if p >= 0 else 0) | 1 << i)
        rows.append([x - (1 << 64) if x >= 1 << 63 else x for x in m])
    return torch.tensor(rows, dtype=torch.int64, device="cuda")


def reference(torch, q, kc, vc, table, contexts, mask, scale=None):
    """(out, tolerance) in 64 bits."""
    seqs, T, H, D = q.shape
    page, kv = kc.shape[1], kc.shape[2]
    scale = D ** -0.5 if scale is None else scale
    h = HALF[str(q.dtype).split(".")[1]]
    room = table.shape[1] * page
    out, tol = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for s in range(seqs):
        c = min(max(0, int(contexts[s])), room)
        n = min(c + T, room)
        if n == 0:
            continue
        idx = table[s, :-(-n // page)].long()
        bad = (idx < 0) | (idx >= kc.shape[0])
        k, v = (x[idx.clamp(0, kc.shape[0] - 1)].double().masked_fill(bad[:, None, None, None], 0).reshape(-1, kv, D)[:n] for x in (kc, vc))
        sees = torch.ones(T, n, dtype=torch.bool, device="cuda")
        for d in range(n - c):
            sees[:, c + d] = ((mask[s] >> d) & 1).bool() if mask is not None else torch.arange(T, device="cuda") >= d
        used = sees.any(0)
        k, v = k * used[:, None, None], torch.where(used[:, None, None], v, torch.zeros_like(v))
        k = torch.where(used[:, None, None], k, torch.zeros_like(k))
        for g in range(H):
            kk, vv, qq = k[:, g * kv // H], v[:, g * kv // H], q[s, :, g].double()
            sc = (qq @ kk.T * scale).masked_fill(~sees, -float("inf"))
            w = torch.where(sees.any(1, keepdim=True), torch.softmax(sc, 1), torch.zeros_like(sc)).nan_to_num(0.0) if not sees.any(1).all() else torch.softmax(sc, 1)
            out[s, :, g] = w @ vv
            B = w @ vv.abs()
            S = ((qq.abs() @ kk.abs().T) * scale).masked_fill(~sees, 0).amax(1, keepdim=True)
            small = 2.0 ** -25 * w.amax(1, keepdim=True) * (sees.double() @ vv.abs()) if q.dtype == torch.float16 else 0
            tol[s, :, g] = (h + 2 * (D * 2.0 ** -23 * S + 2.0 ** -21) + 2.0 ** -18) * B + small
    return out, tol + h * (out.abs() + tol) + (2.0 ** -25 if q.dtype == torch.float16 else 0)


def compare(got, want, tol):
    off = (got.double() - want).abs()
    if not bool((off <= tol).all()):
        at = int((off - tol).nan_to_num(1e30).argmax())
        raise AssertionError("%d of %d values off; %r against %r, tolerance %r" % (int((~(off <= tol)).sum()), off.numel(), float(got.reshape(-1)[at]),
                                                                                 float(want.reshape(-1)[at]), float(tol.reshape(-1)[at])))


# sequences, drafted, heads, kv heads, dim, page, contexts, type, masked
CASES = [
    (1, 1, 1, 1, 64, 16, [0], "bfloat16", False),                     # one key in all
    (1, 1, 8, 2, 128, 16, [1003], "bfloat16", False),                 # plain decoding
    (3, 1, 6, 1, 128, 1, [0, 5, 300], "float16", False),              # pages of one
    (4, 5, 6, 2, 128, 48, [127, 128, 129, 1], "bfloat16", True),      # pages of no power of two, tiles that end at the context
    (5, 16, 12, 2, 128, 64, [700, 0, 64, 2047, 31], "float16", True),  # 96 rows
    (2, 64, 16, 2, 64, 256, [500, 77], "bfloat16", True),             # 512 rows: four row tiles, all mask bits
    (2, 31, 7, 7, 64, 32, [63, 640], "float16", True),
    (1, 3, 5, 1, 128, 64, [40000], "bfloat16", True),                 # one segment cut into over a hundred pieces
    (300, 2, 4, 2, 64, 16, [(37 * j) % 211 for j in range(300)], "bfloat16", True),  # more sequences than threads
    (9, 4, 32, 8, 128, 128, [0, 1, 2, 3, 1000, 1, 0, 5000, 9], "float16", True),
    (1, 64, 3, 1, 128, 16, [0], "float16", False),
    (3, 16, 48, 8, 128, 64, [4096, 2500, 3001], "bfloat16", True),    # many key blocks per multiprocessor
    (2, 2, 8, 8, 64, 16, [12000, 9000], "float16", True),
    (2, 9, 100, 1, 64, 16, [300, 41], "bfloat16", True),              # a hundred heads of one key head: a token per row tile
    (3, 11, 45, 5, 128, 32, [260, 0, 513], "float16", True),          # 99 rows
    (2, 10, 8, 2, 64, 16, [3000, 129], "bfloat16", True),             # 40 rows, twice in the lanes
    (5, 16, 16, 4, 128, 64, [0, 1, 1700, 64, 4000], "float16", True),  # 64 rows
    (2, 3, 11, 1, 128, 16, [900, 2500], "bfloat16", False),           # 33 rows
    (3, 8, 8, 2, 64, 64, [2222, 31, 555], "float16", True),           # 32 rows, four times
    (7, 8, 8, 8, 128, 16, [15, 16, 17, 143, 144, 145, 120], "bfloat16", False),
]


@pytest.mark.parametrize("seqs,drafted,heads,kv,dim,page,contexts,dtype,masked", CASES)
def test_against_the_formula(seqs, drafted, heads, kv, dim, page, contexts, dtype, masked):
    torch = _torch()
    from fngine_b200 import attention as A
    q, kc, vc, table, ctx = setup(torch, seqs, drafted, heads, kv, dim, page, contexts, dtype, seqs + drafted)
    mask = tree_mask(torch, seqs, drafted, 5) if masked else None
    cache, ws = A.KvCache(kc, vc), A.attn_tree_workspace(seqs, drafted, heads, kv, dim)
    out = torch.full_like(q, float("nan"))
    A.attn_tree_decode(q, cache, table, ctx, out, ws, mask=mask)
    torch.cuda.synchronize()
    compare(out, *reference(torch, q, kc, vc, table, contexts, mask))
    again = torch.full_like(q, float("nan"))
    A.attn_tree_decode(q, cache, table, ctx, again, ws, mask=mask)
    assert torch.equal(again, out)  # and the counters were left clear
    assert not bool(ws[:256].any())  # no wait ran out


def test_what_nobody_sees_is_not_looked_at():
    """NaN and infinities in the cache behind a sequence, in drafted tokens that no token sees, and in pages of others; a row that sees
    nothing gives zeros; pages outside of the cache read as zeros; contexts outside of the table."""
    torch = _torch()
    from fngine_b200 import attention as A
    contexts = [0, 130, 70, 10, 5]
    q, kc, vc, table, ctx = setup(torch, 5, 4, 4, 2, 64, 32, contexts, "bfloat16", 3)
    mask = torch.tensor([[0, 0, 4, 0], [1, 2, 3, 0], [1, 1, 1, 1], [1, 3, 0, 0], [0, 0, 0, 0]], device="cuda")
    used = torch.zeros(kc.shape[0] * 32, dtype=torch.bool, device="cuda")
    for s, c in enumerate(contexts):
        union = int(mask[s].sum()) and [d for d in range(4) if any((int(m) >> d) & 1 for m in mask[s])] or []
        for p in list(range(c)) + [c + d for d in union]:
            used[int(table[s, p // 32]) * 32 + p % 32] = True
    for x in (kc, vc):
        flat = x.view(-1, 2, 64)
        flat[~used] = float("nan")
        flat[(~used).nonzero()[::2, 0]] = float("inf")
    table[3, 0] = 10 ** 6  # sequence 3 reads zeros
    cache, ws = A.KvCache(kc, vc), A.attn_tree_workspace(5, 4, 4, 2, 64)
    out = torch.full_like(q, float("nan"))
    A.attn_tree_decode(q, cache, table, ctx, out, ws, mask=mask)
    torch.cuda.synchronize()
    want, tol = reference(torch, q, kc, vc, table, contexts, mask)
    compare(out, want, tol)
    assert not bool(out[0, [0, 1, 3]].any()) and bool(out[0, 2].any()) and not bool(out[3].any())
    q, kc, vc, table, ctx = setup(torch, 3, 2, 2, 1, 64, 16, [40, 40, 40], "float16", 4)
    table = table[:, :2].contiguous()  # room for 32 keys
    for bad in (-5, 1000, 32, 31, 2 ** 31 - 1):
        ctx = torch.tensor([bad, 3, bad], device="cuda", dtype=torch.int32)
        out = torch.full_like(q, float("nan"))
        A.attn_tree_decode(q, A.KvCache(kc, vc), table, ctx, out, ws, scale=0.3)
        torch.cuda.synchronize()
        compare(out, *reference(torch, q, kc, vc, table, [bad, 3, bad], None, 0.3))


def test_strided_tokens_and_a_wide_table():
    torch = _torch()
    from fngine_b200 import attention as A
    q, kc, vc, table, ctx = setup(torch, 3, 5, 6, 2, 128, 16, [100, 20, 333], "bfloat16", 8)
    wide = torch.zeros(15, 1000, dtype=q.dtype, device="cuda")
    wide[:, 64:64 + 768] = q.view(15, 768)
    qs = wide[:, 64:64 + 768].unflatten(1, (6, 128)).unflatten(0, (3, 5))
    to = torch.zeros(15, 2048, dtype=q.dtype, device="cuda")
    out = to[:, 512:512 + 768].unflatten(1, (6, 128)).unflatten(0, (3, 5))
    big = torch.zeros(3, 100, dtype=torch.int32, device="cuda")
    big[:, :table.shape[1]] = table
    ws = A.attn_tree_workspace(3, 5, 6, 2, 128)
    A.attn_tree_decode(qs, A.KvCache(kc, vc), big[:, :table.shape[1]], ctx, out, ws)
    torch.cuda.synchronize()
    compare(out, *reference(torch, q, kc, vc, table, [100, 20, 333], None))
    assert not bool(to[:, :512].any()) and not bool(to[:, 512 + 768:].any())


def test_extreme_scores():
    """Scores of thousands (one key takes all), equal scores, scores of the type's largest values."""
    torch = _torch()
    from fngine_b200 import attention as A
    q, kc, vc, table, ctx = setup(torch, 2, 3, 4, 2, 64, 16, [500, 90], "bfloat16", 11)
    ws = A.attn_tree_workspace(2, 3, 4, 2, 64)
    for f in (0.0, 60.0, 3000.0):
        out = torch.full_like(q, float("nan"))
        A.attn_tree_decode(q * f, A.KvCache(kc, vc), table, ctx, out, ws)
        torch.cuda.synchronize()
        want, tol = reference(torch, q * f, kc, vc, table, [500, 90], None)
        if f < 3000:
            compare(out, want, tol)
        else:
            assert bool(torch.isfinite(out).all())


def test_captured_calls_follow_the_contexts():
    torch = _torch()
    from fngine_b200 import attention as A
    q, kc, vc, table, ctx = setup(torch, 3, 2, 8, 2, 128, 16, [900, 900, 900], "float16", 21)
    cache, ws = A.KvCache(kc, vc), A.attn_tree_workspace(3, 2, 8, 2, 128)
    out = torch.empty_like(q)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        A.attn_tree_decode(q, cache, table, ctx, out, ws)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            A.attn_tree_decode(q, cache, table, ctx, out, ws)
            A.attn_tree_decode(q, cache, table, ctx, out, ws)
        for contexts in ([900, 900, 900], [0, 1, 899], [5, 700, 128]):
            ctx.copy_(torch.tensor(contexts, dtype=torch.int32))
            graph.replay()
            s.synchronize()
            compare(out, *reference(torch, q, kc, vc, table, contexts, None))


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("drafted", [64, 24, 16])
def test_rows_that_see_nothing_and_rows_that_see_one_key(drafted, dim, dtype):
    """Exact zeros and exact copies: a weight of a hidden key that is not zero, however small, would show in both."""
    torch = _torch()
    from fngine_b200 import attention as A
    q, kc, vc, table, ctx = setup(torch, 2, drafted, 4, 2, dim, 16, [0, 0], dtype, 12)
    mask = torch.tensor([[0 if i % 3 else 1 << i if i < 63 else -(1 << 63) for i in range(drafted)]] * 2, device="cuda")
    ws, out = A.attn_tree_workspace(2, drafted, 4, 2, dim), torch.full_like(q, float("nan"))
    A.attn_tree_decode(q, A.KvCache(kc, vc), table, ctx, out, ws, mask=mask)
    torch.cuda.synchronize()
    for s in range(2):
        for i in range(drafted):
            v = vc[int(table[s, i // 16]), i % 16].repeat_interleave(2, 0)
            assert torch.equal(out[s, i], v if i % 3 == 0 else torch.zeros_like(v))
    vc[int(table[1, 0]), 6] = float("nan")  # a key that one row sees: NaN in that row
    A.attn_tree_decode(q, A.KvCache(kc, vc), table, ctx, out, ws, mask=mask)
    torch.cuda.synchronize()
    assert bool(torch.isnan(out[1, 6]).all()) and not bool(torch.isnan(out[0]).any())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("drafted", [3, 20, 50])
def test_not_a_number_reaches_the_rows_that_see_it(drafted, dim):
    """A key of the context that is not a number: every row of its sequence and key head, and no other."""
    torch = _torch()
    from fngine_b200 import attention as A
    for at in range(0, 300, 37):
        q, kc, vc, table, ctx = setup(torch, 2, drafted, 4, 2, dim, 16, [300, 200], "bfloat16", 13)
        kc[int(table[0, at // 16]), at % 16, 1] = float("nan")
        ws, out = A.attn_tree_workspace(2, drafted, 4, 2, dim), torch.zeros_like(q)
        A.attn_tree_decode(q, A.KvCache(kc, vc), table, ctx, out, ws)
        torch.cuda.synchronize()
        assert bool(torch.isnan(out[0, :, 2:]).all()) and not bool(torch.isnan(out[0, :, :2]).any()) and not bool(torch.isnan(out[1]).any())


def test_calls_of_different_shapes_share_a_workspace():
    """More sequences, fewer, another head_dim, another number of row tiles, one after another and back."""
    torch = _torch()
    from fngine_b200 import attention as A
    shapes = [(2, 3, 8, 2, 128, [9000, 12000]), (300, 2, 4, 2, 64, [(53 * j) % 700 for j in range(300)]), (3, 16, 48, 2, 128, [4000, 2000, 77]),
              (1, 1, 4, 4, 64, [30000])]
    size = max((A.attn_tree_workspace(*s[:5]) for s in shapes), key=lambda w: w.numel())
    ws = torch.zeros(size.numel() + 256, dtype=torch.uint8, device="cuda")
    ws = ws[-ws.data_ptr() % 256:][:size.numel()]
    first = []
    for turn in range(2):
        for i, (seqs, drafted, heads, kv, dim, contexts) in enumerate(shapes if not turn else shapes[::-1]):
            q, kc, vc, table, ctx = setup(torch, seqs, drafted, heads, kv, dim, 16, contexts, "bfloat16", dim + seqs)
            out = torch.full_like(q, float("nan"))
            A.attn_tree_decode(q, A.KvCache(kc, vc), table, ctx, out, ws)
            torch.cuda.synchronize()
            if turn:
                assert torch.equal(out, first[-1 - i])
            else:
                compare(out, *reference(torch, q, kc, vc, table, contexts, None))
                first.append(out)
    assert A.attn_tree_status(ws) == 0


@pytest.mark.parametrize("page", [16, 5])
def test_offsets_beyond_32_bits(page):
    """A cache of some 10 GB each of keys and values, with pages from both of its ends; pages of no power of two go the other way."""
    torch = _torch()
    from fngine_b200 import attention as A
    kv, dim, contexts = 8, 128, [700, 333]
    n = 5 * 2 ** 30 // (page * kv * dim)
    kc, vc = (torch.empty(n, page, kv, dim, dtype=torch.bfloat16, device="cuda") for _ in "kv")
    gen = torch.Generator(device="cuda").manual_seed(6)
    need = [-(-(c + 4) // page) for c in contexts]
    table = torch.zeros(2, max(need), dtype=torch.int32, device="cuda")
    table[0] = n - 1 - torch.arange(max(need), device="cuda", dtype=torch.int32)
    table[1] = torch.arange(max(need), device="cuda", dtype=torch.int32) * 2 + n // 2
    for x in (kc, vc):
        for s in range(2):
            x[table[s].long()] = torch.randn(max(need), page, kv, dim, generator=gen, device="cuda").bfloat16()
    q = torch.randn(2, 4, 16, dim, generator=gen, device="cuda").bfloat16()
    ws, out = A.attn_tree_workspace(2, 4, 16, kv, dim), torch.full_like(q, float("nan"))
    A.attn_tree_decode(q, A.KvCache(kc, vc), table, torch.tensor(contexts, dtype=torch.int32, device="cuda"), out, ws)
    torch.cuda.synchronize()
    compare(out, *reference(torch, q, kc, vc, table, contexts, None))
