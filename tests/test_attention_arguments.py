"""The entry points of the attention branch refuse what they do not take before anything is launched. No GPU: addresses are made up."""
import ctypes as C

import pytest

from fngine_b200 import lib as L

P = 0x100000


def test_qk_norm_rope_refusals(fb_built):
    lib = L.load()

    def call(tokens=5, given={}, norm={}, rope={}, out={}, no=()):
        q = dict(q=P, k=2 * P, v=3 * P, q_stride=1024, k_stride=256, v_stride=256, dtype=L.DT_BF16, heads=8, kv_heads=2, head_dim=128, **{})
        q.update(given)
        n = dict(q_weight=4 * P, k_weight=5 * P, weight_dtype=L.DT_F32, eps=1e-6)
        n.update(norm)
        r = dict(inv_freq=6 * P, positions=7 * P, axis_stride=5, rot_dim=64, axes=1, sections=(C.c_int32 * 4)(*rope.pop("sections", (0,) * 4)), adjacent=0)
        r.update(rope)
        o = dict(q=8 * P, k=9 * P, v=10 * P, q_stride=1024, k_stride=256, v_stride=256, slots=None, n_slots=0)
        o.update(out)
        a = [L.Qkv(**q), L.QkNorm(**n), L.RopeArgs(**r), L.QkvOut(**o)]
        a = [None if i in no else C.byref(x) for i, x in enumerate(a)]
        return lib.fb_qk_norm_rope(a[0], tokens, a[1], a[2], a[3], None), lib.fb_last_error_string()

    for bad, word in [(dict(no=(0,)), b"null"), (dict(no=(3,)), b"null"), (dict(tokens=-1), b"negative"), (dict(given=dict(head_dim=96)), b"head_dim"),
                      (dict(given=dict(dtype=L.DT_F32)), b"bf16 or fp16"), (dict(given=dict(heads=0)), b"without heads"), (dict(given=dict(heads=-1)), b"heads"),
                      (dict(given=dict(kv_heads=1025)), b"heads"), (dict(given=dict(q=P + 8)), b"16 bytes"), (dict(given=dict(q_stride=1028)), b"16 bytes"),
                      (dict(given=dict(q_stride=512)), b"stride"), (dict(out=dict(k_stride=128)), b"stride"), (dict(out=dict(v=10 * P + 2)), b"16 bytes"),
                      (dict(out=dict(q=None)), b"together"), (dict(given=dict(v=None)), b"together"),
                      (dict(given=dict(q=None, k=None, v=None), out=dict(q=None, k=None, v=None)), b"nothing"),
                      (dict(norm=dict(weight_dtype=9)), b"weights"), (dict(norm=dict(eps=-1.0)), b"eps"), (dict(norm=dict(eps=float("nan"))), b"eps"),
                      (dict(norm=dict(q_weight=4 * P + 2)), b"aligned"), (dict(rope=dict(rot_dim=0)), b"rot_dim"), (dict(rope=dict(rot_dim=24)), b"rot_dim"),
                      (dict(rope=dict(rot_dim=144)), b"rot_dim"), (dict(rope=dict(axes=0)), b"axes"), (dict(rope=dict(axes=5)), b"axes"),
                      (dict(rope=dict(inv_freq=None)), b"without"), (dict(rope=dict(positions=None)), b"without"), (dict(rope=dict(positions=7 * P + 1)), b"aligned"),
                      (dict(rope=dict(axes=2, sections=(16, 15, 0, 0))), b"add up"), (dict(rope=dict(axes=2, sections=(33, -1, 0, 0))), b"section"),
                      (dict(rope=dict(axes=2, sections=(16, 16, 0, 0), axis_stride=4)), b"axis_stride"),
                      (dict(out=dict(slots=11 * P)), b"n_slots"), (dict(out=dict(slots=11 * P + 4, n_slots=9)), b"aligned")]:
        st, msg = call(**bad)
        assert st == 1 and word in msg, (bad, st, msg)
    assert call(tokens=0)[0] == 0  # nothing to do is not an error


def test_python_mirror_refuses_what_does_not_fit():
    import torch
    from fngine_b200 import attention as A
    q, k = torch.zeros(3, 4, 64, dtype=torch.bfloat16), torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    bad = [dict(q=q.float()), dict(k=k.half()), dict(k=k[:2]), dict(q_out=q[:, :3]), dict(k_out=k[:2]), dict(q=q.transpose(0, 1).contiguous().transpose(0, 1)),
           dict(v=k), dict(q_weight=torch.ones(63)), dict(q_weight=torch.ones(64), k_weight=torch.ones(64).half()), dict(slots=torch.zeros(3, dtype=torch.int32))]
    for change in bad:
        a = dict(q=q, k=k, v=None, q_weight=None, k_weight=None, eps=0.0, rope=None, positions=None, q_out=q, k_out=k, v_out=None)
        a.update(change)
        with pytest.raises((ValueError, AttributeError)):
            A.qk_norm_rope(**a)


def test_attn_tree_refusals(fb_built):
    lib = L.load()
    size = lib.fb_attn_tree_workspace_bytes
    need = size(2, 3, 8, 2, 128)
    assert need == 512 + 512 * 128 * 130 * 4 and size(2, 64, 8, 1, 64) == 512 + 512 * 128 * 130 * 4  # partial results at one size for all shapes
    assert size(100, 64, 16, 2, 64) == 256 + 100 * 2 * 4 * 4 + 128 + 512 * 128 * 130 * 4  # four row tiles of sixteen tokens
    for bad in [(-1, 3, 8, 2, 128), (2, 0, 8, 2, 128), (2, 65, 8, 2, 128), (2, 3, 9, 2, 128), (2, 3, 8, 0, 128), (2, 3, 2, 8, 128), (2, 3, 8, 2, 96), (2, 1, 129, 1, 64)]:
        assert size(*bad) == 0

    def call(q=P, q_stride=1024, heads=8, n_seqs=2, drafted=3, cache={}, no_cache=False, table=2 * P, table_stride=4, contexts=3 * P, mask=4 * P,
             scale=0.1, out=5 * P, out_stride=1024, workspace=6 * P, bytes=need):
        c = dict(k=7 * P, v=8 * P, n_pages=9, page_size=16, dtype=L.DT_F16, kv_heads=2, head_dim=128)
        c.update(cache)
        c = L.KvCacheArgs(**c)
        st = lib.fb_attn_tree_decode(q, q_stride, heads, n_seqs, drafted, None if no_cache else C.byref(c), table, table_stride, contexts, mask, scale,
                                     out, out_stride, workspace, bytes, None)
        return st, lib.fb_last_error_string()

    for bad, word in [(dict(no_cache=True), b"null"), (dict(q=None), b"null"), (dict(out=None), b"null"), (dict(table=None), b"null"),
                      (dict(contexts=None), b"null"), (dict(cache=dict(k=None)), b"null"), (dict(cache=dict(v=None)), b"null"),
                      (dict(cache=dict(dtype=L.DT_F32)), b"bf16 or fp16"), (dict(drafted=0), b"1..64"), (dict(drafted=65), b"1..64"),
                      (dict(heads=7), b"shape"), (dict(n_seqs=-1), b"shape"), (dict(cache=dict(kv_heads=0)), b"shape"), (dict(cache=dict(head_dim=80)), b"shape"),
                      (dict(cache=dict(page_size=0)), b"pages"), (dict(cache=dict(n_pages=0)), b"pages"), (dict(table_stride=0), b"columns"),
                      (dict(table_stride=2 ** 27), b"2^30"), (dict(cache=dict(n_pages=2 ** 27)), b"2^31"), (dict(q_stride=2 ** 39), b"too large"), (dict(q_stride=1016), b"stride"), (dict(out_stride=512), b"stride"), (dict(q_stride=1028), b"16 bytes"),
                      (dict(q=P + 8), b"16 bytes"), (dict(cache=dict(v=8 * P + 2)), b"16 bytes"), (dict(table=2 * P + 2), b"aligned"),
                      (dict(mask=4 * P + 4), b"aligned"), (dict(scale=0.0), b"scale"), (dict(scale=-1.0), b"scale"), (dict(scale=float("nan")), b"scale"),
                      (dict(scale=float("inf")), b"scale"), (dict(workspace=None), b"workspace"), (dict(workspace=6 * P + 128), b"workspace"), (dict(bytes=need - 1), b"workspace")]:
        st, msg = call(**bad)
        assert st == 1 and word in msg, (bad, st, msg)
    assert call(n_seqs=0)[0] == 0


def test_how_tree_tiles_are_cut():
    """The kernel's arithmetic: block b takes tiles [b total / blocks, (b + 1) total / blocks) of all segments' tiles. The blocks that a
    segment says it has pieces in are those that hold some of its tiles, and a block's partial pieces go to different slots."""
    import random
    rng = random.Random(3)
    for _ in range(300):
        tiles = [rng.choice([1, 1, 2, 3, 17, 200]) for _ in range(rng.randint(1, 60))]
        total = sum(tiles)
        blocks = min(total, rng.choice([1, 2, 7, 148]))
        owner = {}
        for b in range(blocks):
            lo, hi = b * total // blocks, (b + 1) * total // blocks
            assert hi > lo
            for t in range(lo, hi):
                owner[t] = b
        assert sorted(owner) == list(range(total))
        slots, begin = {}, 0
        for s, n in enumerate(tiles):
            first, last = ((begin + 1) * blocks - 1) // total, ((begin + n) * blocks - 1) // total
            assert {owner[t] for t in range(begin, begin + n)} == set(range(first, last + 1))
            if first != last:
                for b in range(first, last + 1):
                    slot = 2 * b + (1 if max(begin, b * total // blocks) == begin else 0)
                    assert slots.setdefault(slot, s) == s and slot == (2 * first + 1 if b == first else 2 * b)
            begin += n


def test_attn_prefill_refusals(fb_built):
    lib = L.load()

    def call(given={}, none=False, tokens=70, cu=4 * P, n_seqs=2, scale=0.1, out=5 * P, out_stride=1024, status=None):
        q = dict(q=P, k=2 * P, v=3 * P, q_stride=1024, k_stride=256, v_stride=256, dtype=L.DT_BF16, heads=8, kv_heads=2, head_dim=128)
        q.update(given)
        return lib.fb_attn_prefill(None if none else C.byref(L.Qkv(**q)), tokens, cu, n_seqs, scale, out, out_stride, status, None), lib.fb_last_error_string()

    for bad, word in [(dict(none=True), b"null"), (dict(given=dict(q=None)), b"null"), (dict(given=dict(k=None)), b"null"), (dict(given=dict(v=None)), b"null"),
                      (dict(out=None), b"null"), (dict(cu=None), b"null"), (dict(given=dict(dtype=L.DT_F32)), b"bf16 or fp16"),
                      (dict(given=dict(head_dim=256)), b"head_dim"), (dict(given=dict(heads=7)), b"multiple"), (dict(given=dict(kv_heads=0)), b"multiple"),
                      (dict(given=dict(heads=0)), b"multiple"), (dict(given=dict(heads=1026)), b"multiple"), (dict(tokens=-1), b"negative"), (dict(n_seqs=-1), b"negative"),
                      (dict(given=dict(q_stride=512)), b"stride"), (dict(given=dict(v_stride=248)), b"stride"), (dict(out_stride=1000), b"stride"),
                      (dict(given=dict(k_stride=260)), b"16 bytes"), (dict(given=dict(q=P + 8)), b"16 bytes"), (dict(out=5 * P + 4), b"16 bytes"),
                      (dict(given=dict(k_stride=2 ** 39)), b"too large"), (dict(cu=4 * P + 2), b"aligned"), (dict(status=P + 1), b"aligned"),
                      (dict(scale=0.0), b"scale"), (dict(scale=-0.1), b"scale"), (dict(scale=float("nan")), b"scale"), (dict(scale=float("inf")), b"scale"),
                      (dict(tokens=2 ** 31 - 1), b"65535"), (dict(tokens=70000, n_seqs=70000), b"65535")]:
        st, msg = call(**bad)
        assert st == 1 and word in msg, (bad, st, msg)
    assert call(tokens=0)[0] == 0 and call(n_seqs=0)[0] == 0
