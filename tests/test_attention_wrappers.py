"""What the Python entry points of the attention branch hand to the library, and what they refuse before it is called. No GPU: the tensors are
the CPU's, whose device number stands for the current device's, and the library is a stand-in that notes its arguments."""
import ctypes as C
import types

import pytest
import torch

from fngine_b200 import attention as A
from fngine_b200 import lib as L

BF16 = torch.bfloat16


class Calls:
    """A library whose functions note their name and arguments and succeed."""

    def __init__(self):
        self.made = []

    def __getattr__(self, name):
        def call(*args):
            self.made.append((name, args))
            return 0
        return call


@pytest.fixture
def calls(monkeypatch):
    made = Calls()
    monkeypatch.setattr(L, "load", lambda: made)
    monkeypatch.setattr(L, "stream", lambda: None)
    monkeypatch.setattr(A, "_device", lambda: -1)
    return made


def cache_of(pages=9, page=16, kv=2, dim=64, dtype=BF16):
    """A KvCache of CPU tensors (its constructor wants the GPU's)."""
    c = types.SimpleNamespace(k=torch.zeros(pages, page, kv, dim, dtype=dtype), v=torch.zeros(pages, page, kv, dim, dtype=dtype), n_pages=pages,
                              page_size=page, kv_heads=kv, head_dim=dim, dtype=dtype)
    c.c = L.KvCacheArgs(c.k.data_ptr(), c.v.data_ptr(), pages, page, A._DTYPES[dtype], kv, dim)
    c.ref = C.byref(c.c)
    c.k_rows, c.v_rows = c.k.view(-1, kv, dim), c.v.view(-1, kv, dim)
    return c


def tree(table, seqs=3, drafted=2, **change):
    a = dict(q=torch.zeros(seqs, drafted, 4, 64, dtype=BF16), cache=cache_of(), block_table=table, contexts=torch.zeros(seqs, dtype=torch.int32),
             out=torch.zeros(seqs, drafted, 4, 64, dtype=BF16), workspace=torch.zeros(1024, dtype=torch.uint8))
    a.update(change)
    return A.attn_tree_decode(**a)


def test_a_table_of_some_columns_has_a_stride_and_a_width(calls):
    """Columns of a wider table: the width is the view's, whatever lies beside it, for one sequence as for several."""
    wide = torch.zeros(3, 100, dtype=torch.int32)
    for table, seqs, stride, columns in [(wide, 3, 100, 100), (wide[:, :10], 3, 100, 10), (wide[:, 90:], 3, 100, 10), (wide[:, 5:6], 3, 100, 1),
                                         (wide[1:2, 90:], 1, 10, 10), (wide[:, :10].contiguous(), 3, 10, 10), (wide[:1].expand(3, 100)[:, :100].contiguous(), 3, 100, 100),
                                         (torch.zeros(1, 3, dtype=torch.int32).T, 3, 1, 1)]:
        tree(table, seqs)
        name, args = calls.made.pop()
        assert name == "fb_attn_tree_decode_view" and args[6:9] == (table.data_ptr(), stride, columns)
    for table in (wide.T[:3], wide[:2], wide[:, ::2], wide[:1, :10].expand(3, 10), wide.long()):
        with pytest.raises(ValueError):
            tree(table)
    assert not calls.made


def test_tree_table_refusals(fb_built):
    """The library's own checks of a table's stride and width; addresses are made up."""
    P = 0x100000
    lib = L.load()
    size = lib.fb_attn_tree_workspace_bytes(2, 3, 8, 2, 128)
    c = L.KvCacheArgs(7 * P, 8 * P, 9, 16, L.DT_F16, 2, 128)

    def call(stride, columns, n_seqs=2):
        st = lib.fb_attn_tree_decode_view(P, 1024, 8, n_seqs, 3, C.byref(c), 2 * P, stride, columns, 3 * P, None, 0.1, 5 * P, 1024, 6 * P, size, None)
        return st, lib.fb_last_error_string()

    for stride, columns, word in [(4, 0, b"columns"), (4, -1, b"columns"), (4, 5, b"overlap"), (0, 4, b"overlap"), (-4, 4, b"overlap"), (2 ** 31, 4, b"far apart"),
                                  (2 ** 27, 2 ** 27, b"2^30")]:
        st, msg = call(stride, columns)
        assert st == 1 and word in msg, (stride, columns, st, msg)
    assert call(4, 4, 0)[0] == 0


def branch_of(monkeypatch, tokens=8, heads=4, kv=2, dim=64, hidden=256):
    """An AttentionBranch over stand-ins of its projections, which note what they are called with."""
    made = []
    monkeypatch.setattr(A.linear, "linear_fp8", lambda x, w, epilogue, work: made.append(w.name))
    weight = lambda name, n, k: types.SimpleNamespace(name=name, n=n, k=k, codes=torch.zeros(1, dtype=torch.uint8))
    b = A.AttentionBranch(weight("qkv", (heads + 2 * kv) * dim, hidden), weight("out", hidden, heads * dim), None, None, 1e-6, None, heads, kv, dim, tokens)
    b.made, b.hidden = made, hidden
    return b


def prompt(b, tokens=4, ends=(0, 2, 4), **more):
    return A.forward_attention_prefill(b, torch.zeros(tokens, b.hidden, dtype=BF16), torch.tensor(ends, dtype=torch.int32), None,
                                       torch.zeros(tokens, 4, b.hidden), torch.zeros(tokens, 4), **more)


def test_the_branch_asks_for_zeros_where_there_is_no_sequence(calls, monkeypatch):
    b = branch_of(monkeypatch)
    prompt(b)
    assert [name for name, _ in calls.made] == ["fb_qk_norm_rope", "fb_attn_prefill_padded"] and b.made == ["qkv", "out"]
    A.attn_prefill(b.o, b.o[:, :2], b.o[:, :2].clone(), torch.tensor([0, 8], dtype=torch.int32), b.o.clone())
    assert calls.made[-1][0] == "fb_attn_prefill"


def test_the_branch_reports_a_wait_that_ran_out(calls, monkeypatch):
    """The prompts' attention gets the branch's own status word, a zero until then, and status() reads it."""
    b = branch_of(monkeypatch)
    assert b.status() == 0
    prompt(b)
    args = dict(calls.made)["fb_attn_prefill_padded"]
    C.c_int32.from_address(args[7]).value = 1  # as the kernel does
    assert b.status() == 1
    assert branch_of(monkeypatch).status() == 0  # a word of its own each


class Elsewhere:
    """A tensor as it is, but on a GPU: another device than the current one (of device=-1: the current one)."""

    is_cuda = True

    def __init__(self, x, device=1):
        self.x, self.device_number = x, device

    def __getattr__(self, name):
        return getattr(self.x, name)

    def get_device(self):
        return self.device_number


def test_kv_store_wants_its_cache_on_the_current_device(calls):
    k, slots = torch.zeros(3, 2, 64, dtype=BF16), torch.zeros(3, dtype=torch.int64)
    cache = cache_of()
    A.kv_store(k, k.clone(), cache, slots)
    assert [name for name, _ in calls.made] == ["fb_qk_norm_rope"]
    cache.k, cache.v = Elsewhere(cache.k), Elsewhere(cache.v)
    with pytest.raises(ValueError, match="cache"):
        A.kv_store(k, k.clone(), cache, slots)
    assert len(calls.made) == 1


def test_the_rotation_wants_its_frequencies_on_the_current_device(calls):
    q, k, pos = torch.zeros(3, 4, 64, dtype=BF16), torch.zeros(3, 2, 64, dtype=BF16), torch.zeros(3, dtype=torch.int32)
    here, there = (A.Rope(Elsewhere(torch.ones(32), d)) for d in (-1, 1))
    A.qk_norm_rope(q, k, None, None, None, 0.0, here, pos, q, k, None)
    assert len(calls.made) == 1
    with pytest.raises(ValueError, match="frequencies"):
        A.qk_norm_rope(q, k, None, None, None, 0.0, there, pos, q, k, None)
    assert len(calls.made) == 1


def rotate(**change):
    q, k = torch.zeros(3, 4, 64, dtype=BF16), torch.zeros(3, 2, 64, dtype=BF16)
    a = dict(q=q, k=k, v=None, q_weight=None, k_weight=None, eps=0.0, rope=None, positions=None, q_out=q, k_out=k, v_out=None)
    a.update(change)
    return A.qk_norm_rope(**a)


def test_each_refusal_of_the_norms_and_rotation_is_its_own(calls):
    """The arguments without a fault reach the library; each fault by itself has its own message."""
    q, k, one = torch.zeros(3, 4, 64, dtype=BF16), torch.zeros(3, 2, 64, dtype=BF16), torch.ones(64)
    rope = A.Rope(Elsewhere(torch.ones(32), -1))
    axes = A.Rope(Elsewhere(torch.ones(32), -1), sections=(8, 24))
    pos = torch.zeros(3, dtype=torch.int32)
    good = [dict(), dict(q_weight=one), dict(k_weight=one.half()), dict(v=k, v_out=k), dict(slots=torch.zeros(3, dtype=torch.int64)), dict(rope=rope, positions=pos),
            dict(rope=rope, positions=pos[None]), dict(rope=axes, positions=pos[None].expand(2, 3)), dict(k_out=torch.zeros(9, 2, 64, dtype=BF16), slots=torch.zeros(3, dtype=torch.int64))]
    for change in good:
        rotate(**change)
    assert [name for name, _ in calls.made] == ["fb_qk_norm_rope"] * len(good)
    for change, word in [(dict(q=q.float()), "bf16 or fp16"), (dict(k=k.half()), "^k: "), (dict(k=k[:2]), "^k: "), (dict(q_out=q[:, :3]), "^q_out: "),
                         (dict(k_out=k[:2]), "another number"), (dict(q=q.transpose(0, 1).contiguous().transpose(0, 1)), "side by side"), (dict(v=k), "together"),
                         (dict(v_out=k), "together"), (dict(v=k.half(), v_out=k), "^v: "), (dict(v=k, v_out=q), "^v_out: "), (dict(q_weight=torch.ones(63)), "^q_weight: "),
                         (dict(q_weight=one, k_weight=one.half()), "^k_weight: "), (dict(k_weight=torch.ones(128)[::2]), "^k_weight: "),
                         (dict(q_weight=one.double()), "weights are"), (dict(slots=torch.zeros(3, dtype=torch.int32)), "^slots: "), (dict(slots=torch.zeros(2, dtype=torch.int64)), "^slots: "),
                         (dict(rope=rope, positions=pos[:2]), "^positions: "), (dict(rope=rope, positions=pos.long()), "^positions: "), (dict(rope=axes, positions=pos), "^positions: "),
                         (dict(rope=rope, positions=torch.zeros(6, dtype=torch.int32)[::2]), "^positions: "),
                         (dict(rope=rope, positions=Elsewhere(pos)), "positions: not on"), (dict(q=Elsewhere(q)), "^q: not on"), (dict(k_out=Elsewhere(k)), "^k_out: not on"),
                         (dict(q_weight=Elsewhere(one)), "^q_weight: not on"), (dict(slots=Elsewhere(torch.zeros(3, dtype=torch.int64))), "^slots: not on")]:
        with pytest.raises(ValueError, match=word):
            rotate(**change)
    assert len(calls.made) == len(good)


def test_masks_are_64_bit_words(calls):
    """Words of another size are not taken two or eight at a time."""
    table = torch.zeros(3, 4, dtype=torch.int32)
    for mask in (None, torch.ones(3, 2, dtype=torch.int64), torch.ones(3, 2, dtype=torch.uint64)):
        tree(table, mask=mask)
    assert len(calls.made) == 3 and [c[1][10] is None for c in calls.made] == [True, False, False]
    for mask in (torch.ones(3, 4, dtype=torch.int32), torch.ones(3, 16, dtype=torch.bool), torch.ones(3, 2, dtype=torch.float64), torch.ones(3, 3, dtype=torch.int64),
                 torch.ones(3, 4, dtype=torch.int64)[:, ::2]):
        with pytest.raises(ValueError, match="^mask"):
            tree(table, mask=mask)
    assert len(calls.made) == 3


def test_each_refusal_of_the_tree_is_its_own(calls):
    table, q = torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3, 2, 4, 64, dtype=BF16)
    tree(table)
    for change, word in [(dict(q=q.half()), "cache's type"), (dict(out=q.half()), "cache's type"), (dict(out=q[:, :1]), "cache's type"), (dict(cache=cache_of(dim=128)), "cache's type"),
                         (dict(q=q.transpose(1, 2).contiguous().transpose(1, 2)), "one stride"), (dict(out=torch.zeros(3, 4, 4, 64, dtype=BF16)[:, ::3]), "one stride"),
                         (dict(block_table=table.long()), "block_table"), (dict(block_table=table[:2]), "block_table"), (dict(contexts=torch.zeros(2, dtype=torch.int32)), "^contexts"),
                         (dict(contexts=torch.zeros(3, dtype=torch.int64)), "^contexts"), (dict(q=Elsewhere(q)), "current device"),
                         (dict(workspace=Elsewhere(torch.zeros(8, dtype=torch.uint8))), "current device")]:
        with pytest.raises(ValueError, match=word):
            a = dict(table=table)
            if "block_table" in change:
                a = dict(table=change.pop("block_table"))
            tree(**a, **change)
    assert len(calls.made) == 1


def test_a_branch_refuses_projections_that_its_calls_could_not_use(monkeypatch):
    """Another head_dim than attention takes, projections on two devices: before any buffer is made."""
    assert branch_of(monkeypatch, dim=128).head_dim == 128
    for dim in (32, 96, 256):
        with pytest.raises(ValueError, match="head_dim"):
            branch_of(monkeypatch, dim=dim)
    here, there = (types.SimpleNamespace(n=512, k=256, codes=Elsewhere(torch.zeros(1, dtype=torch.uint8), d)) for d in (0, 1))
    with pytest.raises(ValueError, match="one device"):
        A.AttentionBranch(here, there, None, None, 1e-6, None, 4, 2, 64, 8)
