"""The attention branch of a layer: norms and rotation of queries and keys, attention over packed prompts, attention of drafted
tokens over a paged cache. Every call goes through the C ABI; torch only owns the device buffers."""
import ctypes

import torch

from . import lib as L
from . import linear

_DTYPES = {torch.bfloat16: L.DT_BF16, torch.float16: L.DT_F16}
_WEIGHT_DTYPES = {torch.float32: L.DT_F32, torch.bfloat16: L.DT_BF16, torch.float16: L.DT_F16}


def _device():
    """Index of the current device; a number that no tensor's device has while there is none in use."""
    return torch._C._cuda_getDevice() if torch.cuda.is_initialized() else -2


def _heads(x, tokens, heads, dim, dtype, dev, what):
    """(address, stride between tokens) of a [tokens][heads][head_dim] tensor whose heads lie side by side, on the current device
    (whose stream the call goes to)."""
    s = x.stride()
    if x.shape != (tokens, heads, dim) or x.dtype is not dtype:
        raise ValueError("%s: [%d tokens][%d heads][%d] of %s" % (what, tokens, heads, dim, dtype))
    if s[1] != dim and heads > 1 or s[2] != 1:
        raise ValueError("%s: [tokens][heads][head_dim] with the heads of a token side by side" % what)
    if x.get_device() != dev:
        raise ValueError("%s: not on the current device" % what)
    return x.data_ptr(), s[0] if tokens > 1 else heads * dim  # (a tensor of one token may state any stride)


def _plain(x, shape, dtype, dev, what):
    """Address of a contiguous tensor of this shape and type on the current device."""
    if x.shape != shape or x.dtype is not dtype or not x.is_contiguous():
        raise ValueError("%s: %s %s, contiguous" % (what, dtype, list(shape)))
    if x.get_device() != dev:
        raise ValueError("%s: not on the current device" % what)
    return x.data_ptr()


class Rope:
    """The rotation of a model: inv_freq fp32 [rot_dim / 2]; `sections` says how many frequencies each position axis turns, in their
    order (None: one axis); `adjacent`: frequency j turns (2j, 2j + 1) instead of (j, j + rot_dim / 2)."""

    def __init__(self, inv_freq, sections=None, adjacent=False):
        assert inv_freq.is_cuda and inv_freq.dtype == torch.float32 and inv_freq.is_contiguous() and inv_freq.dim() == 1
        sections = [inv_freq.numel()] if sections is None else [int(s) for s in sections]
        assert 1 <= len(sections) <= 4 and sum(sections) == inv_freq.numel() and min(sections) >= 0
        self.inv_freq, self.axes = inv_freq, len(sections)
        self._frozen = bytes(L.RopeArgs(inv_freq.data_ptr(), None, 0, 2 * inv_freq.numel(), self.axes, (ctypes.c_int32 * 4)(*sections),
                                        int(bool(adjacent)), 0))

    def c(self, positions, tokens, dev):
        """fb_rope for int32 positions [axes][tokens] (or [tokens], for one axis)."""
        shape, s = positions.shape, positions.stride()
        if shape != (self.axes, tokens) and (self.axes > 1 or shape != (tokens,)) or positions.dtype is not torch.int32 or (tokens > 1 and s[-1] != 1):
            raise ValueError("positions: int32 [%d axes][%d tokens], contiguous along the tokens" % (self.axes, tokens))
        if positions.get_device() != dev:
            raise ValueError("positions: not on the current device")
        if self.inv_freq.get_device() != dev:
            raise ValueError("rope: its frequencies are not on the current device")
        r = L.RopeArgs.from_buffer_copy(self._frozen)
        r.positions = positions.data_ptr()
        if self.axes > 1:
            r.axis_stride = s[0]
        return r


def qk_norm_rope(q, k, v, q_weight, k_weight, eps, rope, positions, q_out, k_out, v_out, slots=None):
    """fb_qk_norm_rope: norms of q and k per head (a weight None: no norm), rotation (rope None: none), v copied. q, k, v and the
    outputs are [tokens][heads][head_dim] views, v and v_out may be None. With `slots` (int64 [tokens]) k_out and v_out are rows of a
    cache, [rows][kv_heads][head_dim]: KvCache.k_rows and .v_rows of a paged one; a slot outside of them stores nothing."""
    tokens, heads, dim = q.shape
    kv_heads, rows, dtype = k.shape[1], k_out.shape[0], q.dtype
    if dtype not in _DTYPES:
        raise ValueError("qk_norm_rope: bf16 or fp16")
    if slots is None and rows != tokens:
        raise ValueError("qk_norm_rope: k_out has another number of tokens than k")
    if (v is None) != (v_out is None):
        raise ValueError("qk_norm_rope: v and v_out are given together, or neither")
    dev = _device()
    q_at, q_stride = _heads(q, tokens, heads, dim, dtype, dev, "q")
    k_at, k_stride = _heads(k, tokens, kv_heads, dim, dtype, dev, "k")
    qo_at, qo_stride = _heads(q_out, tokens, heads, dim, dtype, dev, "q_out")
    ko_at, ko_stride = _heads(k_out, rows, kv_heads, dim, dtype, dev, "k_out")
    v_at = vo_at = None
    v_stride = vo_stride = 0
    if v is not None:
        v_at, v_stride = _heads(v, tokens, kv_heads, dim, dtype, dev, "v")
        vo_at, vo_stride = _heads(v_out, rows, kv_heads, dim, dtype, dev, "v_out")
    norm = None
    if q_weight is not None or k_weight is not None:
        w_dtype = (k_weight if q_weight is None else q_weight).dtype
        if w_dtype not in _WEIGHT_DTYPES:
            raise ValueError("qk_norm_rope: weights are fp32, bf16 or fp16")
        norm = L.QkNorm(None if q_weight is None else _plain(q_weight, (dim,), w_dtype, dev, "q_weight"),
                        None if k_weight is None else _plain(k_weight, (dim,), w_dtype, dev, "k_weight"), _WEIGHT_DTYPES[w_dtype], eps)
    s_at = None if slots is None else _plain(slots, (tokens,), torch.int64, dev, "slots")
    st = L.load().fb_qk_norm_rope(L.Qkv(q_at, k_at, v_at, q_stride, k_stride, v_stride, _DTYPES[dtype], heads, kv_heads, dim), tokens, norm,
                                  None if rope is None else rope.c(positions, tokens, dev),
                                  L.QkvOut(qo_at, ko_at, vo_at, qo_stride, ko_stride, vo_stride, s_at, rows), L.stream())
    if st:
        L.check(st, "qk_norm_rope")


def attn_prefill(q, k, v, cu_seqlens, out, scale=None, status=None, padded=False):
    """fb_attn_prefill: q and out [tokens][heads][head_dim], k and v [tokens][kv_heads][head_dim], cu_seqlens int32 [n_seqs + 1]; scale
    1 / sqrt(head_dim) unless given. status: a word (int32 [1]) that a wait which ran out sets. Tokens outside of all sequences are left as
    they were in out; padded (fb_attn_prefill_padded): they get zeros."""
    tokens, heads, dim = q.shape
    kv_heads, dtype = k.shape[1], q.dtype
    if dtype not in _DTYPES:
        raise ValueError("attn_prefill: bf16 or fp16")
    if cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 1:
        raise ValueError("attn_prefill: cu_seqlens int32 [n_seqs + 1]")
    dev = _device()
    q_at, q_stride = _heads(q, tokens, heads, dim, dtype, dev, "q")
    k_at, k_stride = _heads(k, tokens, kv_heads, dim, dtype, dev, "k")
    v_at, v_stride = _heads(v, tokens, kv_heads, dim, dtype, dev, "v")
    o_at, o_stride = _heads(out, tokens, heads, dim, dtype, dev, "out")
    n_seqs = cu_seqlens.shape[0] - 1
    call = L.load().fb_attn_prefill_padded if padded else L.load().fb_attn_prefill
    st = call(L.Qkv(q_at, k_at, v_at, q_stride, k_stride, v_stride, _DTYPES[dtype], heads, kv_heads, dim), tokens,
              _plain(cu_seqlens, (n_seqs + 1,), torch.int32, dev, "cu_seqlens"), n_seqs, dim ** -0.5 if scale is None else scale, o_at, o_stride,
              None if status is None else _plain(status, (1,), torch.int32, dev, "status"), L.stream())
    if st:
        L.check(st, "attn_prefill")


class KvCache:
    """fb_kv_cache: k and v [n_pages][page_size][kv_heads][head_dim], bf16 or fp16. k_rows and v_rows are its slots one after
    another (page * page_size + offset), the rows that qk_norm_rope writes to."""

    def __init__(self, k, v):
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.dtype not in _DTYPES or not (k.is_contiguous() and v.is_contiguous()):
            raise ValueError("KvCache: k and v [n_pages][page_size][kv_heads][head_dim] of one type, contiguous")
        if k.get_device() < 0 or k.get_device() != v.get_device():
            raise ValueError("KvCache: k and v on one device")
        self.k, self.v = k, v
        self.n_pages, self.page_size, self.kv_heads, self.head_dim = k.shape
        self.dtype = k.dtype
        self.k_rows, self.v_rows = (x.view(-1, self.kv_heads, self.head_dim) for x in (k, v))
        self.c = L.KvCacheArgs(k.data_ptr(), v.data_ptr(), self.n_pages, self.page_size, _DTYPES[k.dtype], self.kv_heads, self.head_dim)
        self.ref = ctypes.byref(self.c)


def attn_tree_workspace(n_seqs, drafted, heads, kv_heads, head_dim, device="cuda"):
    """Zero-filled workspace of attn_tree_decode for up to n_seqs sequences of these shapes, and for all others that need no more bytes;
    every call leaves it ready for the next."""
    n = L.load().fb_attn_tree_workspace_bytes(n_seqs, drafted, heads, kv_heads, head_dim)
    if not n:
        raise ValueError("attn_tree_workspace: unsupported shape")
    buf = torch.zeros(n + 256, dtype=torch.uint8, device=device)
    off = (-buf.data_ptr()) % 256
    return buf[off:off + n]


def attn_tree_status(workspace):
    """FB_STATUS_* of the calls that used this workspace (waits for them)."""
    return int(workspace[:4].view(torch.int32).item())


def attn_tree_decode(q, cache, block_table, contexts, out, workspace, mask=None, scale=None):
    """fb_attn_tree_decode_view: q and out [n_seqs][drafted][heads][head_dim], block_table int32 [n_seqs][columns] (some columns of a wider
    table too: the others are not read), contexts int32 [n_seqs],
    mask int64 or uint64 [n_seqs][drafted] (bit d of token i: it sees drafted token d; None: d <= i), scale 1 / sqrt(head_dim) unless given."""
    n_seqs, drafted, heads, dim = q.shape
    if q.dtype is not cache.dtype or out.dtype is not q.dtype or out.shape != q.shape or dim != cache.head_dim:
        raise ValueError("attn_tree_decode: q and out [n_seqs][drafted][heads][head_dim] of the cache's type")
    dev = _device()
    strides = []
    for x in (q, out):
        s = x.stride()
        token = s[1] if drafted > 1 else s[0] if n_seqs > 1 else heads * dim
        if s[3] != 1 or (heads > 1 and s[2] != dim) or (n_seqs > 1 and s[0] != drafted * token):
            raise ValueError("attn_tree_decode: the tokens of q and out lie at one stride, the heads of a token side by side")
        strides.append(token)
    if block_table.dtype is not torch.int32 or block_table.dim() != 2 or block_table.shape[0] != n_seqs or (block_table.shape[1] > 1 and block_table.stride(1) != 1):
        raise ValueError("attn_tree_decode: block_table int32 [n_seqs][columns]")
    columns = block_table.shape[1]
    table_stride = block_table.stride(0) if n_seqs > 1 else columns
    if table_stride < columns:
        raise ValueError("attn_tree_decode: rows of block_table overlap")
    if not (q.get_device() == out.get_device() == block_table.get_device() == workspace.get_device() == cache.k.get_device() == dev):
        raise ValueError("attn_tree_decode: not on the current device")
    if mask is not None and mask.dtype is torch.uint64:
        mask = mask.view(torch.int64)
    st = L.load().fb_attn_tree_decode_view(q.data_ptr(), strides[0], heads, n_seqs, drafted, cache.ref, block_table.data_ptr(), table_stride, columns,
                                           _plain(contexts, (n_seqs,), torch.int32, dev, "contexts"),
                                           None if mask is None else _plain(mask, (n_seqs, drafted), torch.int64, dev, "mask"),
                                           dim ** -0.5 if scale is None else scale, out.data_ptr(), strides[1], workspace.data_ptr(),
                                           workspace.numel(), L.stream())
    if st:
        L.check(st, "attn_tree_decode")


def kv_store(k, v, cache, slots):
    """Copies keys and values of packed tokens ([tokens][kv_heads][head_dim]) to slots of a paged cache (int64 [tokens]; one outside of
    the cache stores nothing): fb_qk_norm_rope without queries, norms and rotation."""
    tokens, dev = k.shape[0], _device()
    k_at, k_stride = _heads(k, tokens, cache.kv_heads, cache.head_dim, cache.dtype, dev, "k")
    v_at, v_stride = _heads(v, tokens, cache.kv_heads, cache.head_dim, cache.dtype, dev, "v")
    if cache.k.get_device() != dev:
        raise ValueError("kv_store: the cache is not on the current device")
    slot = cache.kv_heads * cache.head_dim
    st = L.load().fb_qk_norm_rope(L.Qkv(None, k_at, v_at, 0, k_stride, v_stride, _DTYPES[cache.dtype], 0, cache.kv_heads, cache.head_dim), tokens,
                                  None, None, L.QkvOut(None, cache.c.k, cache.c.v, 0, slot, slot, _plain(slots, (tokens,), torch.int64, dev, "slots"),
                                                       cache.n_pages * cache.page_size), L.stream())
    if st:
        L.check(st, "kv_store")


class AttentionBranch:
    """The attention branch of one layer: qkv = a weight of (heads + 2 kv_heads) head_dim rows, out = one of hidden rows, both
    linear.Fp8RowWeight (any number of tokens) or linear.Q4GroupWeight (up to 16), the norms' weights, the rotation. Owns the workspaces
    and the intermediate buffers (bf16) of up to max_tokens tokens; calls that overlap need a branch each."""

    def __init__(self, qkv, out, q_weight, k_weight, eps, rope, heads, kv_heads, head_dim, max_tokens):
        if qkv.n != (heads + 2 * kv_heads) * head_dim or out.k != heads * head_dim:
            raise ValueError("AttentionBranch: the projections do not fit the heads")
        if head_dim not in (64, 128):
            raise ValueError("AttentionBranch: head_dim 64 or 128")
        if qkv.codes.get_device() != out.codes.get_device():
            raise ValueError("AttentionBranch: the projections are not on one device")
        self.qkv, self.out, self.q_weight, self.k_weight, self.eps, self.rope = qkv, out, q_weight, k_weight, eps, rope
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        device = qkv.codes.device
        self.rows = torch.empty(max_tokens, qkv.n, dtype=torch.bfloat16, device=device)
        self.o = torch.empty(max_tokens, heads, head_dim, dtype=torch.bfloat16, device=device)
        self.status_word = torch.zeros(1, dtype=torch.int32, device=device)
        self._work = [linear.linear_fp8_workspace(w, max_tokens, device) if isinstance(w, linear.Fp8RowWeight) else None for w in (qkv, out)]

    def status(self):
        """FB_STATUS_* of the prompts' attention so far (waits for it): not zero once a bounded wait has run out, and the residual streams of that call
        are not to be used. That of the drafted tokens' is in their workspace (attn_tree_status)."""
        return int(self.status_word.item())

    def parts(self, tokens):
        """q, k and v of the projection's output, [tokens][heads or kv_heads][head_dim]."""
        q, k, v = self.rows[:tokens].split([self.heads * self.head_dim, self.kv_heads * self.head_dim, self.kv_heads * self.head_dim], dim=1)
        return tuple(x.unflatten(1, (-1, self.head_dim)) for x in (q, k, v))

    def check(self, x, X, inj):
        """Number of tokens of x [tokens][hidden], once everything that the calls behind go by fits it."""
        tokens, hidden = x.shape
        if tokens > self.o.shape[0]:
            raise ValueError("AttentionBranch: %d tokens, made for up to %d" % (tokens, self.o.shape[0]))
        if hidden != self.qkv.k or X.shape != (tokens, 4, self.out.n) or inj.shape != (tokens, 4):
            raise ValueError("AttentionBranch: x [tokens][%d], X [tokens][4][%d], inj [tokens][4]" % (self.qkv.k, self.out.n))
        dev = _device()
        if not (x.get_device() == X.get_device() == inj.get_device() == self.o.get_device() == dev):
            raise ValueError("AttentionBranch: not on the current device")
        return tokens

    def project(self, x, which, epilogue):
        w = self.out if which else self.qkv
        if isinstance(w, linear.Q4GroupWeight):
            linear.linear_q4_decode(x, w, epilogue)
        else:
            linear.linear_fp8(x, w, epilogue, self._work[which])


def forward_attention_prefill(branch, x, cu_seqlens, positions, X, inj, cache=None, slots=None):
    """The attention branch over packed prompts: projection, norms and rotation, causal attention, projection with the residual write X
    += inj * y (X fp32 [T][4][hidden], inj [T][4]). x bf16 [T][hidden]. Tokens outside of all sequences (padding) add nothing to X. With
    `cache` the keys and values are put to `slots` for forward_attention_decode."""
    tokens = branch.check(x, X, inj)
    if not tokens:
        return
    branch.project(x, 0, linear.store_bf16(branch.rows[:tokens]))
    q, k, v = branch.parts(tokens)
    qk_norm_rope(q, k, None, branch.q_weight, branch.k_weight, branch.eps, branch.rope, positions, q, k, None)
    if cache is not None:
        kv_store(k, v, cache, slots)
    o = branch.o[:tokens]
    attn_prefill(q, k, v, cu_seqlens, o, status=branch.status_word, padded=True)
    branch.project(o.flatten(1), 1, linear.gr_write(X, inj))


def forward_attention_decode(branch, x, drafted, cache, block_table, contexts, slots, positions, workspace, X, inj, mask=None):
    """The attention branch of a decode step: x bf16 [n_seqs * drafted][hidden], the tokens of a sequence one after another; their
    keys and values go to `slots` of the cache, which are positions contexts[s] .. contexts[s] + drafted - 1 of sequence s. `workspace` of
    attn_tree_workspace; `mask` as in attn_tree_decode (one token per sequence: plain decoding)."""
    tokens = branch.check(x, X, inj)
    n_seqs = contexts.shape[0]
    if tokens != n_seqs * drafted:
        raise ValueError("forward_attention_decode: x holds another number of tokens than contexts say")
    if not tokens:
        return
    branch.project(x, 0, linear.store_bf16(branch.rows[:tokens]))
    q, k, v = branch.parts(tokens)
    qk_norm_rope(q, k, v, branch.q_weight, branch.k_weight, branch.eps, branch.rope, positions, q, cache.k_rows, cache.v_rows, slots=slots)
    o = branch.o[:tokens]
    attn_tree_decode(q.unflatten(0, (n_seqs, drafted)), cache, block_table, contexts, o.unflatten(0, (n_seqs, drafted)), workspace, mask=mask)
    branch.project(o.flatten(1), 1, linear.gr_write(X, inj))
