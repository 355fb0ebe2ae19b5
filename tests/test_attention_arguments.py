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
