"""The operators of a layer's attention branch, as a program that serves a model calls them.

Four kinds of work:

  q4       a projection with 4-bit weights and group scales at decode width (up to 16 tokens), with the epilogues of the
           FP8-row projection
  rope     norms of queries and keys per head and their rotation in one pass, positions of one to four axes; keys and values
           go to packed rows or to slots of a cache
  prompt   causal attention over packed prompts of different lengths, grouped heads
  tree     attention of drafted tokens over a paged cache, each token seeing its ancestors; one token per sequence is plain
           decoding

The plain forms are elementary torch operations in 32 bits (rotation angles in 64), rounded once at the end.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
LARGEST_PROMPT = 8192


def listed():
    return [
        # the shared expert's down projection for one user's token: latency, the smallest group
        dict(name="q4_shared_down_t1", kind="q4", n=2560, k=640, tokens=1, group=32, scales="f16", zeros=False, epilogue="shared_scale"),
        # the wide projection in front of a layer's mixer, five tokens of a drafted step, weights with zero points
        dict(name="q4_qkvz_t5", kind="q4", n=16384, k=2560, tokens=5, group=64, scales="bf16", zeros=True, epilogue="store_bf16"),
        # the vocabulary matrix for a full decode batch: the largest matrix of a model
        dict(name="q4_lm_head_t16", kind="q4", n=248320, k=2560, tokens=16, group=128, scales="bf16", zeros=False, epilogue="store_f32"),
        # three tokens of a decode step far into a long context, keys and values to the cache
        dict(name="rope_decode_t3", kind="rope", tokens=3, heads=48, kv_heads=8, dim=128, rot=128, axes=1, far=900000, adjacent=False, slots=True, dtype="bf16"),
        # a prompt chunk of odd length, half of a head rotated, into the cache
        dict(name="rope_prompt_4093", kind="rope", tokens=4093, heads=48, kv_heads=8, dim=128, rot=64, axes=1, far=30000, adjacent=False, slots=True, dtype="bf16"),
        # a prompt of text, images and video: time, height and width, fp16, packed rows
        dict(name="rope_axes_8192", kind="rope", tokens=8192, heads=32, kv_heads=8, dim=128, rot=128, axes=3, far=8192, adjacent=False, slots=False, dtype="f16"),
        # a few short prompts that came in together, one of a single token and one empty
        dict(name="prompt_short", kind="prompt", tokens=437, seqs=6, spread="short", heads=14, kv_heads=2, dim=64, dtype="f16"),
        # four users' prompts of different lengths in one batch
        dict(name="prompt_packed_4000", kind="prompt", tokens=4000, seqs=4, spread="ragged", heads=48, kv_heads=8, dim=128, dtype="bf16"),
        # one long prompt
        dict(name="prompt_one_8192", kind="prompt", tokens=8192, seqs=1, spread="one", heads=48, kv_heads=8, dim=128, dtype="bf16"),
        # plain decoding of one user: one token, a short context
        dict(name="tree_one_t1", kind="tree", seqs=1, drafted=1, context=1003, heads=48, kv_heads=8, dim=128, page=16, dtype="bf16"),
        # eight users with sixteen drafted tokens each
        dict(name="tree_drafts_t16", kind="tree", seqs=8, drafted=16, context=4096, heads=48, kv_heads=8, dim=128, page=64, dtype="bf16"),
        # many users with long contexts, four drafted tokens each: the cache is what is read
        dict(name="tree_long_t4", kind="tree", seqs=32, drafted=4, context=16384, heads=32, kv_heads=8, dim=128, page=64, dtype="f16"),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["q4", "rope", "prompt", "tree"])
    if kind == "q4":
        n, k = _log(rng, 64, 60000), 128 * _log(rng, 1, 80)
        epilogue = rng.choice(["store_bf16", "store_f32", "swiglu", "shared_scale"])
        return dict(kind=kind, n=n + n % 2 if epilogue == "swiglu" else n, k=k, tokens=rng.randint(1, 16), group=rng.choice([32, 64, 128]),
                    scales=rng.choice(["f32", "bf16", "f16"]), zeros=rng.random() < 0.5, epilogue=epilogue)
    dtype = rng.choice(["bf16", "bf16", "f16"])
    dim = rng.choice([64, 128, 128])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 6, 7, 8]) if kv_heads < 8 else kv_heads * rng.choice([1, 2, 3, 4, 6])
    if kind == "rope":
        return dict(kind=kind, tokens=_log(rng, 1, 8192), heads=heads, kv_heads=kv_heads, dim=dim, rot=rng.choice([32, dim // 2, dim, dim]),
                    axes=rng.choice([1, 1, 2, 3, 4]), far=_log(rng, 100, 1000000), adjacent=rng.random() < 0.3, slots=rng.random() < 0.6, dtype=dtype)
    if kind == "prompt":
        tokens = _log(rng, 1, LARGEST_PROMPT)
        return dict(kind=kind, tokens=tokens, seqs=rng.randint(1, min(9, tokens)), spread=rng.choice(["short", "ragged", "ragged"]), heads=heads,
                    kv_heads=kv_heads, dim=dim, dtype=dtype)
    context = _log(rng, 1, 32768)
    return dict(kind=kind, seqs=_log(rng, 1, max(1, min(64, 500000 // context))), drafted=rng.choice([1, 1, 2, 3, 5, 8, 16, 31, 64]), context=context, heads=heads,
                kv_heads=kv_heads, dim=dim, page=rng.choice([1, 16, 48, 64, 256]), dtype=dtype)


def _lengths(case):
    """The prompts' lengths, from the case alone: they add up to its tokens."""
    tokens, seqs = case["tokens"], case["seqs"]
    if seqs == 1:
        return [tokens]
    if case["spread"] == "short":  # one of one token and one empty, the rest in falling shares
        share = [0.0, 0.0] + [1.0 / (j + 1) for j in range(seqs - 2)]
        lens = [1 if j == 0 else 0 for j in range(seqs)]
    else:
        share = [1.0 + 0.37 * ((5 * j + 2) % 7) for j in range(seqs)]
        lens = [0] * seqs
    left, total = tokens - sum(lens), sum(share) or 1.0
    lens = [a + int(left * b / total) for a, b in zip(lens, share)]
    lens[-1] += tokens - sum(lens)
    return lens


def _contexts(case):
    """The sequences' lengths in the cache, from the case alone: ragged, the longest at the stated context."""
    return [max(0, case["context"] - (case["context"] * ((3 * j) % 8)) // 16 - j % 5) for j in range(case["seqs"])]


def work(case):
    kind, item = case["kind"], 2
    if kind == "q4":
        n, k, t = case["n"], case["k"], case["tokens"]
        out = {"store_bf16": n * 2, "store_f32": n * 4, "swiglu": n // 2 * 2, "shared_scale": n * 4}[case["epilogue"]]
        per_group = (4 if case["scales"] == "f32" else 2) + (1 if case["zeros"] else 0)
        return {"bytes": n * k // 2 + n * (k // case["group"]) * per_group + t * (2 * k + out), "flops": 2 * t * n * k}
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    if kind == "rope":
        rows = case["tokens"] * (heads + 2 * kv)
        return {"bytes": 2 * rows * dim * item + 4 * case["tokens"] * case["axes"], "flops": 10 * rows * dim}
    if kind == "prompt":
        lens = _lengths(case)
        return {"bytes": case["tokens"] * (2 * heads + 2 * kv) * dim * item, "flops": 2 * dim * heads * sum(m * (m + 1) for m in lens)}
    keys, rows = sum(c + case["drafted"] for c in _contexts(case)), case["seqs"] * case["drafted"]
    return {"bytes": keys * kv * 2 * dim * item + 2 * rows * heads * dim * item, "flops": 4 * dim * heads * keys * case["drafted"]}


# ---------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)

    def uniform(*shape):
        return torch.rand(*shape, generator=gen, device="cuda")

    return {"q4": _prepare_q4, "rope": _prepare_rope, "prompt": _prepare_prompt, "tree": _prepare_tree}[case["kind"]](case, gen, normal, uniform)


def _prepare_q4(case, gen, normal, uniform):
    n, k, t, group = case["n"], case["k"], case["tokens"], case["group"]
    st = dict(case=case)
    st["codes"] = torch.randint(0, 256, (n, k // 2), generator=gen, device="cuda", dtype=torch.uint8)
    # a weight matrix of unit gain: codes spread over 16 steps of the scale
    st["scales"] = ((0.5 + uniform(n, k // group)) * (0.2 / math.sqrt(k))).to(DTYPES[case["scales"]])
    st["zeros"] = torch.randint(4, 12, (n, k // group), generator=gen, device="cuda", dtype=torch.uint8) if case["zeros"] else None
    st["x"] = normal(t, k, dtype=torch.bfloat16)
    if case["epilogue"] == "shared_scale":
        st["gate"] = normal(t, 513)
    width = n // 2 if case["epilogue"] == "swiglu" else n
    st["out"] = torch.zeros(t, width, device="cuda", dtype=torch.bfloat16 if case["epilogue"] in ("store_bf16", "swiglu") else torch.float32)
    return st


def _sections(case):
    """How many frequencies each axis turns: time the fewest, the others even."""
    half, axes = case["rot"] // 2, case["axes"]
    if axes == 1:
        return [half]
    each = half * 3 // (3 * axes - 1) if axes > 1 else half
    return [half - each * (axes - 1)] + [each] * (axes - 1)


def _prepare_rope(case, gen, normal, uniform):
    t, heads, kv, dim, dtype = case["tokens"], case["heads"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
    st = dict(case=case)
    # the projection's output: q, k and v of a token side by side, heads of different sizes
    qkv = normal(t, heads + 2 * kv, dim) * (0.3 + 2 * uniform(1, heads + 2 * kv, 1))
    st["qkv"] = qkv.to(dtype).view(t, (heads + 2 * kv) * dim)
    st["q_weight"] = (0.5 + uniform(dim)).to(dtype)
    st["k_weight"] = (0.5 + uniform(dim)).to(dtype)
    st["inv_freq"] = torch.pow(torch.tensor(1.0e6, device="cuda", dtype=torch.float64), torch.arange(case["rot"] // 2, device="cuda", dtype=torch.float64) * (-2.0 / case["rot"])).float()
    first = max(0, case["far"] - t)
    if case["axes"] == 1:
        st["positions"] = (first + torch.arange(t, device="cuda", dtype=torch.int32)).view(1, t)
    else:
        st["positions"] = torch.randint(0, case["far"] + 1, (case["axes"], t), generator=gen, device="cuda", dtype=torch.int32)
    st["sections"] = _sections(case)
    rows = t
    if case["slots"]:  # pages of a cache handed out in no order, some of it in use by others
        rows = t + 37
        st["slots"] = torch.randperm(rows, generator=gen, device="cuda")[:t].contiguous()
    else:
        st["slots"] = None
    st["q_out"] = torch.zeros(t, heads, dim, device="cuda", dtype=dtype)
    st["k_out"] = torch.zeros(rows, kv, dim, device="cuda", dtype=dtype)
    st["v_out"] = torch.zeros(rows, kv, dim, device="cuda", dtype=dtype)
    return st


def _prepare_prompt(case, gen, normal, uniform):
    t, heads, kv, dim, dtype = case["tokens"], case["heads"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
    st = dict(case=case, lens=_lengths(case))
    st["q"], st["k"], st["v"] = normal(t, heads, dim, dtype=dtype), normal(t, kv, dim, dtype=dtype), normal(t, kv, dim, dtype=dtype)
    ends = [0]
    for m in st["lens"]:
        ends.append(ends[-1] + m)
    st["starts"] = ends
    st["cu_seqlens"] = torch.tensor(ends, device="cuda", dtype=torch.int32)
    st["out"] = torch.zeros(t, heads, dim, device="cuda", dtype=dtype)
    return st


def _prepare_tree(case, gen, normal, uniform):
    seqs, t, heads, kv, dim, page, dtype = (case[x] for x in ("seqs", "drafted", "heads", "kv_heads", "dim", "page", "dtype"))
    dtype = DTYPES[dtype]
    contexts = _contexts(case)
    pages = [-(-(c + t) // page) for c in contexts]
    st = dict(case=case)
    total, most = sum(pages), max(pages)
    order = torch.randperm(total, generator=gen, device="cuda", dtype=torch.int32)
    table = torch.zeros(seqs, most, device="cuda", dtype=torch.int32)
    at = 0
    for s, p in enumerate(pages):
        table[s, :p] = order[at:at + p]
        at += p
    st["table"] = table
    st["contexts"] = torch.tensor(contexts, device="cuda", dtype=torch.int32)
    st["k_cache"], st["v_cache"] = normal(total, page, kv, dim, dtype=dtype), normal(total, page, kv, dim, dtype=dtype)
    st["q"] = normal(seqs, t, heads, dim, dtype=dtype)
    # drafted token i hangs below an earlier one, or below the context, and sees its ancestors and itself
    parent = (uniform(seqs, t) * torch.arange(1, t + 1, device="cuda")).long() - 1
    mask = torch.zeros(seqs, t + 1, device="cuda", dtype=torch.int64)  # the last column: no parent
    for i in range(t):
        mask[:, i] = mask.gather(1, parent[:, i:i + 1] % (t + 1))[:, 0] | (1 << i if i < 63 else -(1 << 63))
    st["mask"] = mask[:, :t].contiguous()
    st["out"] = torch.zeros(seqs, t, heads, dim, device="cuda", dtype=dtype)
    return st


# ---------------------------------------------------------------------------------------------- one pass
def run(st):
    return {"q4": _run_q4, "rope": _run_rope, "prompt": _run_prompt, "tree": _run_tree}[st["case"]["kind"]](st)


def _run_q4(st):
    case = st["case"]
    if own:
        from fngine_b200 import linear
        if "weight" not in st:
            st["weight"] = linear.Q4GroupWeight(st["codes"], st["scales"], st["zeros"])
        kind = case["epilogue"]
        if kind == "store_bf16":
            epilogue = linear.store_bf16(st["out"])
        elif kind == "store_f32":
            epilogue = linear.store_f32(st["out"])
        elif kind == "swiglu":
            epilogue = linear.swiglu(st["out"])
        else:
            epilogue = linear.shared_scale(st["out"], st["gate"][:, 512:], 513)
        linear.linear_q4_decode(st["x"], st["weight"], epilogue)
        return st["out"]
    n, k, group = case["n"], case["k"], case["group"]
    codes = torch.stack((st["codes"] & 15, st["codes"] >> 4), dim=2).view(n, k // group, group).float()
    zeros = 8.0 if st["zeros"] is None else st["zeros"].float()[:, :, None]
    weight = ((codes - zeros) * st["scales"].float()[:, :, None]).view(n, k)
    acc = st["x"].float() @ weight.T
    if case["epilogue"] == "store_bf16":
        return acc.to(torch.bfloat16)
    if case["epilogue"] == "swiglu":
        gate, up = acc[:, :n // 2], acc[:, n // 2:]
        return (gate / (1 + torch.exp(-gate)) * up).to(torch.bfloat16)
    if case["epilogue"] == "shared_scale":
        return acc / (1 + torch.exp(-st["gate"][:, 512:]))
    return acc


def _run_rope(st):
    case = st["case"]
    t, heads, kv, dim, rot = case["tokens"], case["heads"], case["kv_heads"], case["dim"], case["rot"]
    q, k, v = (x.view(t, -1, dim) for x in st["qkv"].split([heads * dim, kv * dim, kv * dim], dim=1))
    if own:
        from fngine_b200 import attention
        if "rope" not in st:
            st["rope"] = attention.Rope(st["inv_freq"], sections=st["sections"], adjacent=case["adjacent"])
        attention.qk_norm_rope(q, k, v, st["q_weight"], st["k_weight"], 1e-6, st["rope"], st["positions"], st["q_out"], st["k_out"], st["v_out"], slots=st["slots"])
        return [st["q_out"], st["k_out"], st["v_out"]]
    axis = torch.repeat_interleave(torch.arange(case["axes"], device="cuda"), torch.tensor(st["sections"], device="cuda"), output_size=rot // 2)
    angle = st["positions"].double()[axis].T * st["inv_freq"].double()  # [t][rot / 2]
    cos, sin = torch.cos(angle).float()[:, None, :], torch.sin(angle).float()[:, None, :]

    def turn(x, weight):
        x = x.float()
        x = x * torch.rsqrt((x * x).mean(dim=2, keepdim=True) + 1e-6) * weight.float()
        a, b = (x[:, :, 0:rot:2], x[:, :, 1:rot:2]) if case["adjacent"] else (x[:, :, :rot // 2], x[:, :, rot // 2:rot])
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=3 if case["adjacent"] else 2).reshape(x.shape[0], x.shape[1], rot)
        return torch.cat((y, x[:, :, rot:]), dim=2).to(DTYPES[case["dtype"]])

    k_out, v_out = st["k_out"], st["v_out"]
    if st["slots"] is None:
        return [turn(q, st["q_weight"]), turn(k, st["k_weight"]), v.clone()]
    k_out[st["slots"]] = turn(k, st["k_weight"])
    v_out[st["slots"]] = v
    return [turn(q, st["q_weight"]), k_out, v_out]


def _run_prompt(st):
    case = st["case"]
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    if own:
        from fngine_b200 import attention
        attention.attn_prefill(st["q"], st["k"], st["v"], st["cu_seqlens"], st["out"])
        return st["out"]
    q, k, v, out = st["q"], st["k"], st["v"], st["out"]
    for a, b in zip(st["starts"], st["starts"][1:]):  # each prompt by itself: their scores have different shapes
        m = b - a
        if m == 0:
            continue
        qs = q[a:b].float().view(m, kv, heads // kv, dim).permute(1, 2, 0, 3)
        ks, vs = k[a:b].float().permute(1, 2, 0)[:, None], v[a:b].float().permute(1, 0, 2)[:, None]
        s = (qs @ ks).mul_(1 / math.sqrt(dim))
        s.masked_fill_(torch.ones(m, m, device="cuda", dtype=torch.bool).triu_(1), -math.inf)
        s = s.sub_(s.amax(dim=3, keepdim=True)).exp_()
        o = (s @ vs) / s.sum(dim=3, keepdim=True)
        out[a:b] = o.permute(2, 0, 1, 3).reshape(m, heads, dim).to(out.dtype)
    return out


def _run_tree(st):
    case = st["case"]
    seqs, t, heads, kv, dim, page = (case[x] for x in ("seqs", "drafted", "heads", "kv_heads", "dim", "page"))
    if own:
        from fngine_b200 import attention
        if "cache" not in st:
            st["cache"] = attention.KvCache(st["k_cache"], st["v_cache"])
            st["workspace"] = attention.attn_tree_workspace(seqs, t, heads, kv, dim)
        attention.attn_tree_decode(st["q"], st["cache"], st["table"], st["contexts"], st["out"], st["workspace"], mask=st["mask"])
        return st["out"]
    length = st["table"].shape[1] * page
    at = torch.arange(length, device="cuda")
    slot = st["table"].long()[:, at // page] * page + at % page
    k = st["k_cache"].view(-1, kv, dim)[slot].permute(0, 2, 3, 1).float()  # [seqs][kv][dim][length]
    v = st["v_cache"].view(-1, kv, dim)[slot].permute(0, 2, 1, 3).float()
    q = st["q"].float().view(seqs, t, kv, heads // kv, dim).permute(0, 2, 1, 3, 4).reshape(seqs, kv, t * (heads // kv), dim)
    s = (q @ k).mul_(1 / math.sqrt(dim)).view(seqs, kv, t, heads // kv, length)
    ctx = st["contexts"].long()[:, None]
    drafted = at[None, :] - ctx  # [seqs][length]
    seen = (st["mask"][:, :, None] >> drafted.clamp(0, 63)[:, None, :]) & 1  # [seqs][t][length]
    seen = (drafted < 0)[:, None, :] | ((seen == 1) & (drafted < t)[:, None, :])
    s.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    s = s.sub_(s.amax(dim=4, keepdim=True).clamp_(min=-1e30)).exp_()
    o = (s.view(seqs, kv, t * (heads // kv), length) @ v) / s.sum(dim=4).view(seqs, kv, t * (heads // kv), 1)
    return o.view(seqs, kv, t, heads // kv, dim).permute(0, 2, 1, 3, 4).reshape(seqs, t, heads, dim).to(st["out"].dtype)


# ---------------------------------------------------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    return {"q4": _exact_q4, "rope": _exact_rope, "prompt": _exact_prompt, "tree": _exact_tree}[case["kind"]](case, st)


def _exact_q4(case, st):
    n, k, group = case["n"], case["k"], case["group"]
    x = st["x"].double()
    acc = torch.zeros(case["tokens"], n, device="cuda", dtype=torch.float64)
    for r in range(0, n, 8192):  # rows at a time: a matrix in 64 bits is sixteen times its codes
        byte = st["codes"][r:r + 8192].double()
        high = torch.floor(byte / 16)
        w = torch.empty(byte.shape[0], k, device="cuda", dtype=torch.float64)
        w[:, 0::2], w[:, 1::2] = byte - 16 * high, high
        zero = torch.full_like(st["scales"][r:r + 8192], 8).double() if st["zeros"] is None else st["zeros"][r:r + 8192].double()
        w -= zero.repeat_interleave(group, dim=1)
        w *= st["scales"][r:r + 8192].double().repeat_interleave(group, dim=1)
        acc[:, r:r + 8192] = x @ w.T
    if case["epilogue"] == "swiglu":
        return torch.nn.functional.silu(acc[:, :n // 2]) * acc[:, n // 2:]
    if case["epilogue"] == "shared_scale":
        return torch.sigmoid(st["gate"][:, 512].double())[:, None] * acc
    return acc


def _exact_rope(case, st):
    t, heads, kv, dim, rot = case["tokens"], case["heads"], case["kv_heads"], case["dim"], case["rot"]
    x = st["qkv"].double().view(t, heads + 2 * kv, dim)
    position = torch.cat([st["positions"][a].double()[:, None].expand(t, m) for a, m in enumerate(st["sections"])], dim=1)
    turn = torch.polar(torch.ones_like(position), position * st["inv_freq"].double())[:, None, :]

    def norm_and_turn(y, weight):
        y = y / torch.sqrt((y ** 2).mean(dim=2, keepdim=True) + 1e-6) * weight.double()
        if case["adjacent"]:
            z = torch.view_as_complex(y[:, :, :rot].reshape(t, -1, rot // 2, 2).contiguous()) * turn
            y[:, :, :rot] = torch.view_as_real(z).reshape(t, -1, rot)
        else:
            z = torch.complex(y[:, :, :rot // 2].contiguous(), y[:, :, rot // 2:rot].contiguous()) * turn
            y[:, :, :rot] = torch.cat((z.real, z.imag), dim=2)
        return y

    q = norm_and_turn(x[:, :heads].clone(), st["q_weight"])
    k = torch.zeros(st["k_out"].shape, device="cuda", dtype=torch.float64)
    v = torch.zeros_like(k)
    rows = torch.arange(t, device="cuda") if st["slots"] is None else st["slots"]
    k[rows], v[rows] = norm_and_turn(x[:, heads:heads + kv].clone(), st["k_weight"]), x[:, heads + kv:]
    return [q, k, v]


def _exact_prompt(case, st):
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    out = torch.zeros(case["tokens"], heads, dim, device="cuda", dtype=torch.float64)
    for a, b in zip(st["starts"], st["starts"][1:]):
        if a == b:
            continue
        future = torch.arange(b - a, device="cuda")[None, :] > torch.arange(b - a, device="cuda")[:, None]
        for h in range(heads):
            s = st["q"][a:b, h].double() @ st["k"][a:b, h * kv // heads].double().T / math.sqrt(dim)
            out[a:b, h] = torch.softmax(s.masked_fill_(future, -math.inf), dim=1) @ st["v"][a:b, h * kv // heads].double()
    return out


def _exact_tree(case, st):
    seqs, t, heads, kv, dim, page = (case[x] for x in ("seqs", "drafted", "heads", "kv_heads", "dim", "page"))
    out = torch.zeros(seqs, t, heads, dim, device="cuda", dtype=torch.float64)
    for s, c in enumerate(_contexts(case)):
        used = st["table"][s, :-(-(c + t) // page)].long()
        k = st["k_cache"][used].reshape(-1, kv, dim)[:c + t].double()
        v = st["v_cache"][used].reshape(-1, kv, dim)[:c + t].double()
        sees = torch.ones(t, c + t, device="cuda", dtype=torch.bool)
        for d in range(t):
            sees[:, c + d] = (st["mask"][s] >> d) & 1 == 1
        for h in range(kv):
            q = st["q"][s, :, h * (heads // kv):(h + 1) * (heads // kv)].double()  # [t][group][dim]
            score = torch.einsum("tgd,ld->tgl", q, k[:, h]) / math.sqrt(dim)
            weight = torch.softmax(score.masked_fill(~sees[:, None, :], -math.inf), dim=2)
            out[s, :, h * (heads // kv):(h + 1) * (heads // kv)] = torch.einsum("tgl,ld->tgd", weight, v[:, h])
    return out
