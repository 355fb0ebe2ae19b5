"""The attention branch of a layer: norms and rotation of queries and keys, attention over packed prompts, attention of drafted
tokens over a paged cache. Every call goes through the C ABI; torch only owns the device buffers."""
import ctypes

import torch

from . import lib as L

_DTYPES = {torch.bfloat16: L.DT_BF16, torch.float16: L.DT_F16}
_WEIGHT_DTYPES = {torch.float32: L.DT_F32, torch.bfloat16: L.DT_BF16, torch.float16: L.DT_F16}


def _heads(x, what):
    """(address, stride between tokens) of a [tokens][heads][head_dim] tensor whose heads lie side by side."""
    s = x.stride()
    if len(s) != 3 or s[2] != 1 or (s[1] != x.shape[2] and x.shape[1] > 1):
        raise ValueError("%s: [tokens][heads][head_dim] with the heads of a token side by side" % what)
    # (a tensor of one token may state any stride)
    return x.data_ptr(), s[0] if x.shape[0] > 1 else x.shape[1] * x.shape[2]


def _here(what, *tensors):
    """Raises unless every tensor (None is passed over) lies on the current device, whose stream the call goes to."""
    dev = torch._C._cuda_getDevice()
    for x in tensors:
        if x is not None and x.get_device() != dev:
            raise ValueError("%s: tensors on the current device" % what)


class Rope:
    """The rotation of a model: inv_freq fp32 [rot_dim / 2]; `sections` says how many frequencies each position axis turns, in their
    order (None: one axis); `adjacent`: frequency j turns (2j, 2j + 1) instead of (j, j + rot_dim / 2)."""

    def __init__(self, inv_freq, sections=None, adjacent=False):
        assert inv_freq.is_cuda and inv_freq.dtype == torch.float32 and inv_freq.is_contiguous() and inv_freq.dim() == 1
        sections = [inv_freq.numel()] if sections is None else [int(s) for s in sections]
        assert 1 <= len(sections) <= 4 and sum(sections) == inv_freq.numel() and min(sections) >= 0
        self.inv_freq, self.axes = inv_freq, len(sections)
        self._frozen = (inv_freq.data_ptr(), 2 * inv_freq.numel(), self.axes, (ctypes.c_int32 * 4)(*sections), int(bool(adjacent)))

    def c(self, positions, tokens):
        """fb_rope for int32 positions [axes][tokens] (or [tokens], for one axis)."""
        if positions.dim() == 1:
            positions = positions.unsqueeze(0)
        if positions.dtype != torch.int32 or positions.shape != (self.axes, tokens) or (tokens > 1 and positions.stride(1) != 1):
            raise ValueError("positions: int32 [%d axes][%d tokens], contiguous along the tokens" % (self.axes, tokens))
        f = self._frozen
        return L.RopeArgs(f[0], positions.data_ptr(), positions.stride(0) if self.axes > 1 else tokens, f[1], f[2], f[3], f[4], 0)


def qk_norm_rope(q, k, v, q_weight, k_weight, eps, rope, positions, q_out, k_out, v_out, slots=None):
    """fb_qk_norm_rope: norms of q and k per head (a weight None: no norm), rotation (rope None: none), v copied. q, k, v and the
    outputs are [tokens][heads][head_dim] views, v and v_out may be None. With `slots` (int64 [tokens]) k_out and v_out are rows of a
    cache, [rows][kv_heads][head_dim]: KvCache.k_rows and .v_rows of a paged one; a slot outside of them stores nothing."""
    tokens, heads, dim = q.shape
    kv_heads = k.shape[1]
    if q.dtype not in _DTYPES or not (q.dtype == k.dtype == q_out.dtype == k_out.dtype):
        raise ValueError("qk_norm_rope: bf16 or fp16, the same for all tensors")
    rows = k_out.shape[0]
    if k.shape != (tokens, kv_heads, dim) or q_out.shape != q.shape or k_out.shape[1:] != k.shape[1:] or (slots is None and rows != tokens):
        raise ValueError("qk_norm_rope: shapes do not fit")
    q_at, k_at, qo_at, ko_at = _heads(q, "q"), _heads(k, "k"), _heads(q_out, "q_out"), _heads(k_out, "k_out")
    v_at = vo_at = (None, 0)
    if v is not None:
        if v.shape != k.shape or v_out.shape != k_out.shape or v.dtype != q.dtype or v_out.dtype != q.dtype:
            raise ValueError("qk_norm_rope: v does not fit k")
        v_at, vo_at = _heads(v, "v"), _heads(v_out, "v_out")
    norm = None
    if q_weight is not None or k_weight is not None:
        one = q_weight if q_weight is not None else k_weight
        for w in (q_weight, k_weight):
            if w is not None and (w.dtype != one.dtype or w.shape != (dim,) or not w.is_contiguous()):
                raise ValueError("qk_norm_rope: weights [head_dim] of one type")
        norm = L.QkNorm(None if q_weight is None else q_weight.data_ptr(), None if k_weight is None else k_weight.data_ptr(),
                        _WEIGHT_DTYPES[one.dtype], eps)
    if slots is not None and (slots.dtype != torch.int64 or slots.shape != (tokens,) or not slots.is_contiguous()):
        raise ValueError("qk_norm_rope: slots int64 [tokens]")
    _here("qk_norm_rope", q, k, v, q_weight, k_weight, positions if rope else None, q_out, k_out, v_out, slots)
    given = L.Qkv(q_at[0], k_at[0], v_at[0], q_at[1], k_at[1], v_at[1], _DTYPES[q.dtype], heads, kv_heads, dim)
    out = L.QkvOut(qo_at[0], ko_at[0], vo_at[0], qo_at[1], ko_at[1], vo_at[1], None if slots is None else slots.data_ptr(), rows)
    st = L.load().fb_qk_norm_rope(given, tokens, norm, None if rope is None else rope.c(positions, tokens), out, L.stream())
    if st:
        L.check(st, "qk_norm_rope")


def attn_prefill(q, k, v, cu_seqlens, out, scale=None, status=None):
    """fb_attn_prefill: q and out [tokens][heads][head_dim], k and v [tokens][kv_heads][head_dim], cu_seqlens int32 [n_seqs + 1]; scale
    1 / sqrt(head_dim) unless given. status: a word (int32 [1]) that a wait which ran out sets."""
    tokens, heads, dim = q.shape
    kv_heads = k.shape[1]
    if q.dtype not in _DTYPES or not (q.dtype == k.dtype == v.dtype == out.dtype):
        raise ValueError("attn_prefill: bf16 or fp16, the same for all tensors")
    if k.shape != (tokens, kv_heads, dim) or v.shape != k.shape or out.shape != q.shape:
        raise ValueError("attn_prefill: shapes do not fit")
    if cu_seqlens.dtype != torch.int32 or cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 1 or not cu_seqlens.is_contiguous():
        raise ValueError("attn_prefill: cu_seqlens int32 [n_seqs + 1]")
    q_at, k_at, v_at, o_at = _heads(q, "q"), _heads(k, "k"), _heads(v, "v"), _heads(out, "out")
    _here("attn_prefill", q, k, v, cu_seqlens, out, status)
    given = L.Qkv(q_at[0], k_at[0], v_at[0], q_at[1], k_at[1], v_at[1], _DTYPES[q.dtype], heads, kv_heads, dim)
    st = L.load().fb_attn_prefill(given, tokens, cu_seqlens.data_ptr(), cu_seqlens.shape[0] - 1, dim ** -0.5 if scale is None else scale,
                                  o_at[0], o_at[1], None if status is None else status.data_ptr(), L.stream())
    if st:
        L.check(st, "attn_prefill")


class KvCache:
    """fb_kv_cache: k and v [n_pages][page_size][kv_heads][head_dim], bf16 or fp16. k_rows and v_rows are its slots one after
    another (page * page_size + offset), the rows that qk_norm_rope writes to."""

    def __init__(self, k, v):
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.dtype not in _DTYPES or not (k.is_contiguous() and v.is_contiguous()):
            raise ValueError("KvCache: k and v [n_pages][page_size][kv_heads][head_dim] of one type, contiguous")
        _here("KvCache", k, v)
        self.k, self.v = k, v
        self.n_pages, self.page_size, self.kv_heads, self.head_dim = k.shape
        self.dtype = k.dtype
        self.k_rows, self.v_rows = (x.view(-1, self.kv_heads, self.head_dim) for x in (k, v))
        self.c = L.KvCacheArgs(k.data_ptr(), v.data_ptr(), self.n_pages, self.page_size, _DTYPES[k.dtype], self.kv_heads, self.head_dim)
        self.ref = ctypes.byref(self.c)


def attn_tree_workspace(n_seqs, drafted, heads, kv_heads, head_dim, device="cuda"):
    """Zero-filled workspace of attn_tree_decode for up to n_seqs sequences of these shapes; every call leaves it ready for the next."""
    n = L.load().fb_attn_tree_workspace_bytes(n_seqs, drafted, heads, kv_heads, head_dim)
    if not n:
        raise ValueError("attn_tree_workspace: unsupported shape")
    buf = torch.zeros(n + 256, dtype=torch.uint8, device=device)
    off = (-buf.data_ptr()) % 256
    return buf[off:off + n]


def attn_tree_decode(q, cache, block_table, contexts, out, workspace, mask=None, scale=None):
    """fb_attn_tree_decode: q and out [n_seqs][drafted][heads][head_dim], block_table int32 [n_seqs][columns], contexts int32 [n_seqs],
    mask int64 or uint64 [n_seqs][drafted] (bit d of token i: it sees drafted token d; None: d <= i), scale 1 / sqrt(head_dim) unless given."""
    n_seqs, drafted, heads, dim = q.shape
    if q.dtype != cache.dtype or out.dtype != q.dtype or out.shape != q.shape or dim != cache.head_dim:
        raise ValueError("attn_tree_decode: q and out [n_seqs][drafted][heads][head_dim] of the cache's type")
    strides = []
    for x in (q, out):
        s = x.stride()
        token = s[1] if drafted > 1 else s[0] if n_seqs > 1 else heads * dim
        if s[3] != 1 or (heads > 1 and s[2] != dim) or (n_seqs > 1 and s[0] != drafted * token):
            raise ValueError("attn_tree_decode: the tokens of q and out lie at one stride, the heads of a token side by side")
        strides.append(token)
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.shape[0] != n_seqs or block_table.stride(1) != 1:
        raise ValueError("attn_tree_decode: block_table int32 [n_seqs][columns]")
    if contexts.dtype != torch.int32 or contexts.shape != (n_seqs,) or not contexts.is_contiguous():
        raise ValueError("attn_tree_decode: contexts int32 [n_seqs]")
    if mask is not None and (mask.dtype not in (torch.int64, torch.uint64) or mask.shape != (n_seqs, drafted) or not mask.is_contiguous()):
        raise ValueError("attn_tree_decode: mask int64 [n_seqs][drafted]")
    columns = block_table.stride(0) if n_seqs > 1 else block_table.shape[1]
    if columns < block_table.shape[1]:
        raise ValueError("attn_tree_decode: rows of block_table overlap")
    _here("attn_tree_decode", q, out, block_table, contexts, mask, workspace)
    st = L.load().fb_attn_tree_decode(q.data_ptr(), strides[0], heads, n_seqs, drafted, cache.ref, block_table.data_ptr(), columns,
                                      contexts.data_ptr(), None if mask is None else mask.data_ptr(), dim ** -0.5 if scale is None else scale,
                                      out.data_ptr(), strides[1], workspace.data_ptr(), workspace.numel(), L.stream())
    if st:
        L.check(st, "attn_tree_decode")
