"""The workloads that the positional, windowed and cached-attention operators are measured on.

Four operators: rotary positions with several axes (``rotary_nd``), causal sliding-window attention with sink tokens,
forward and backward (``window_attn_fwd`` / ``window_attn_bwd``), attention of new tokens or of a tree of drafted
tokens over a paged cache (``cached_attn_fwd``), and the writes of that cache (``cache_append`` / ``cache_keep``).
``run`` computes a case with elementary torch operations in 32 bits, or, with ``own`` set, through the framework.
"""
import math
import os
import sys

import torch

own = False

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one decoding step of a batch: every sequence rotates the query and key of its newest token
        {"name": "rotary_token", "op": "rotary", "B": 64, "S": 1, "Hq": 32, "Hkv": 8, "D": 128, "dtype": "bf16",
         "axes": "16,24,24", "interleaved": False, "layout": "bhsd", "grid": "", "train": False},
        # a training step's rotations of a video of 16 x 60 x 80 latent tokens: q, k and the gradients coming back
        {"name": "rotary_video_train", "op": "rotary", "B": 1, "S": 76800, "Hq": 24, "Hkv": 24, "D": 128,
         "dtype": "bf16", "axes": "22,21,21", "interleaved": True, "layout": "bhsd", "grid": "16,60,80", "train": True},
        # images with grouped heads, part of each head rotated, tokens before heads, an odd number of tokens
        {"name": "rotary_image_odd", "op": "rotary", "B": 3, "S": 4097, "Hq": 16, "Hkv": 4, "D": 96, "dtype": "fp16",
         "axes": "16,16", "interleaved": False, "layout": "bshd", "grid": "", "train": False},
        # prefill of a long prompt with grouped heads
        {"name": "window_prefill", "op": "window", "B": 1, "Hq": 32, "Hkv": 8, "Sq": 32768, "Sk": 32768, "D": 128,
         "dtype": "bf16", "window": 2048, "sinks": 4, "ragged": False, "train": False},
        # the last chunk of a chunked prefill of a padded batch
        {"name": "window_prefill_chunk", "op": "window", "B": 4, "Hq": 16, "Hkv": 4, "Sq": 1000, "Sk": 9000, "D": 64,
         "dtype": "fp16", "window": 1500, "sinks": 16, "ragged": True, "train": False},
        # a training step's attention, one head of keys for each head of queries
        {"name": "window_train", "op": "window", "B": 1, "Hq": 16, "Hkv": 16, "Sq": 16384, "Sk": 16384, "D": 128,
         "dtype": "bf16", "window": 1024, "sinks": 4, "ragged": False, "train": True},
        # a training step on a padded batch with odd sizes, grouped heads (gradients of shared heads) and many sinks
        {"name": "window_train_ragged", "op": "window", "B": 2, "Hq": 12, "Hkv": 4, "Sq": 4999, "Sk": 4999, "D": 96,
         "dtype": "fp16", "window": 700, "sinks": 64, "ragged": True, "train": True},
        # one token of one user: latency
        {"name": "cached_token_one", "op": "cached", "B": 1, "Hq": 32, "Hkv": 8, "T": 1, "ctx": 3000, "page": 16,
         "D": 128, "dtype": "bf16", "window": 1024, "sinks": 4, "tree": False},
        # one token of each of many users with long contexts
        {"name": "cached_token_batch", "op": "cached", "B": 64, "Hq": 32, "Hkv": 8, "T": 1, "ctx": 32768, "page": 64,
         "D": 128, "dtype": "bf16", "window": 4096, "sinks": 4, "tree": False},
        # verification of a tree of drafted tokens, all of the context visible
        {"name": "cached_tree", "op": "cached", "B": 8, "Hq": 32, "Hkv": 8, "T": 48, "ctx": 16384, "page": 128,
         "D": 128, "dtype": "bf16", "window": 0, "sinks": 0, "tree": True},
        # drafts are written, then the accepted path of each sequence is moved to the front
        {"name": "cache_accept", "op": "cache", "B": 64, "Hkv": 8, "T": 32, "ctx": 1024, "page": 16, "D": 128,
         "dtype": "bf16", "keep": 8},
        # a prefill chunk of a batch is written into its pages
        {"name": "cache_prefill", "op": "cache", "B": 8, "Hkv": 8, "T": 2048, "ctx": 4096, "page": 64, "D": 128,
         "dtype": "bf16", "keep": 0},
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["rotary", "window", "window", "cached", "cached", "cache"])
    dtype = rng.choice(["bf16", "fp16"])
    hkv = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 1, 2, 3, 4, 8])
    if op == "rotary":
        D = rng.choice([64, 96, 128])
        most = D // 2
        first = rng.randint(4, most // 2)
        axes = rng.choice([(most,), (first, most - first), (most - 2 * (most // 3), most // 3, most // 3),
                           (most // 4, most // 4)])
        return {"op": op, "B": rng.randint(1, 4), "S": spread(1, 16384), "Hq": hkv * group, "Hkv": hkv, "D": D,
                "dtype": rng.choice(["bf16", "fp16", "fp32"]), "axes": ",".join(map(str, axes)),
                "interleaved": rng.random() < 0.5, "layout": rng.choice(["bhsd", "bshd"]), "grid": "",
                "train": rng.random() < 0.5}
    if op == "window":
        sq = spread(1, 8192)
        sk = sq if rng.random() < 0.6 else sq + spread(1, 8192)
        return {"op": op, "B": rng.randint(1, 2), "Hq": hkv * group, "Hkv": hkv, "Sq": sq, "Sk": sk,
                "D": rng.choice([64, 96, 128]), "dtype": dtype, "window": spread(1, 2048), "sinks": rng.choice([0, 1, 4, 30, 128]),
                "ragged": rng.random() < 0.5, "train": rng.random() < 0.5}
    page = rng.choice([16, 32, 64, 128, 256])
    if op == "cached":
        tree = rng.random() < 0.4
        return {"op": op, "B": spread(1, 32), "Hq": hkv * group, "Hkv": hkv, "T": rng.randint(1, 64) if tree else spread(1, 64),
                "ctx": spread(65, 16384), "page": page, "D": rng.choice([64, 96, 128]), "dtype": dtype,
                "window": rng.choice([0, spread(1, 4096)]), "sinks": rng.choice([0, 1, 4, 100]), "tree": tree}
    T = spread(1, 1024)
    return {"op": op, "B": rng.randint(1, 32), "Hkv": hkv, "T": T, "ctx": T + spread(1, 2048), "page": page,
            "D": rng.choice([64, 96, 128]), "dtype": dtype, "keep": rng.randint(0, min(T, 16))}


# ------------------------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------------------------
def _axes(case):
    return [int(x) for x in case["axes"].split(",")]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DT[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32 if dt == torch.float32 else dt)

    def whole(lo, hi, *shape):  # lo <= value < hi
        return torch.randint(lo, hi, shape, generator=gen, device="cuda", dtype=torch.int32)

    st = {"case": case}
    D = case["D"]
    if case["op"] == "rotary":
        B, S = case["B"], case["S"]
        axes = _axes(case)
        shape = (lambda h: (B, h, S, D)) if case["layout"] == "bhsd" else (lambda h: (B, S, h, D))
        if case["grid"]:
            # every token's place in the video, the video starting at a random frame
            t, y, x = [int(n) for n in case["grid"].split(",")]
            at = torch.stack(torch.meshgrid(*(torch.arange(n, device="cuda", dtype=torch.int32) for n in (t, y, x)),
                                            indexing="ij"), -1).reshape(1, S, 3)
            at = at + torch.tensor([1, 0, 0], device="cuda", dtype=torch.int32) * whole(0, 1000, 1, 1, 1)
            st["positions"] = at.expand(B, S, 3).contiguous()
        else:
            st["positions"] = whole(0, 32768, B, S, len(axes))
        # one falling ladder of frequencies for each axis
        st["inv_freq"] = torch.cat([10000.0 ** (-torch.arange(n, device="cuda", dtype=torch.float64) / n) for n in axes]).float()
        st["q"], st["k"] = normal(*shape(case["Hq"])), normal(*shape(case["Hkv"]))
        if case["train"]:
            st["gq"], st["gk"] = normal(*shape(case["Hq"])), normal(*shape(case["Hkv"]))
        return st
    if case["op"] == "window":
        B, Sq, Sk = case["B"], case["Sq"], case["Sk"]
        st["q"] = normal(B, case["Hq"], Sq, D)
        st["k"], st["v"] = normal(B, case["Hkv"], Sk, D), normal(B, case["Hkv"], Sk, D)
        if case["train"]:
            st["dout"] = normal(B, case["Hq"], Sq, D)
        if case["ragged"]:
            lens = whole(Sk - Sq // 2, Sk + 1, B)  # padding reaches into the last half of the new tokens
            lens[0] = Sk
            st["lens"] = lens
        return st
    # paged caches: every sequence owns pages anywhere in the pool, in any order; what it does not own is -1
    B, page, ctx, T = case["B"], case["page"], case["ctx"], case["T"]
    most = -(-ctx // page)
    lens = whole(max(T, ctx // 2), ctx + 1, B)
    lens[0] = ctx
    pool = torch.randperm(B * most, generator=gen, device="cuda").to(torch.int32).view(B, most)
    live = torch.arange(most, device="cuda") * page < lens[:, None]
    st["page_table"] = torch.where(live, pool, -1).to(torch.int32).contiguous()
    st["lens"] = lens
    st["k_cache"] = normal(B * most, case["Hkv"], page, D)
    st["v_cache"] = normal(B * most, case["Hkv"], page, D)
    if case["op"] == "cached":
        st["q"] = normal(B, case["Hq"], T, D)
        if case["tree"]:
            # a draft continues any earlier draft, or the last accepted token (-1)
            r = torch.rand(B, T, generator=gen, device="cuda")
            st["parents"] = (r * torch.arange(1, T + 1, device="cuda")).floor().to(torch.int32) - 1
        return st
    st["k"], st["v"] = normal(B, case["Hkv"], T, D), normal(B, case["Hkv"], T, D)
    keep = case["keep"]
    if keep:
        order = torch.rand(B, T, generator=gen, device="cuda").argsort(-1)[:, :keep].sort(-1).values
        st["path"] = order.to(torch.int32).contiguous()
        st["path_lens"] = whole(0, keep + 1, B)
    return st


# ------------------------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------------------------
if os.path.isdir("block-sparse-attention_b200"):
    sys.path.insert(0, os.path.abspath("block-sparse-attention_b200"))


def run(st):
    case = st["case"]
    if own:
        return _own(st, case)
    return {"rotary": _plain_rotary, "window": _plain_window, "cached": _plain_cached, "cache": _plain_cache}[case["op"]](st, case)


def _own(st, case):
    import block_sparse_attention as bsa
    if case["op"] == "rotary":
        how = dict(interleaved=case["interleaved"], layout=case["layout"])
        res = bsa.rotary_nd(st["q"], st["k"], st["positions"], st["inv_freq"], _axes(case), **how)
        if case["train"]:
            res += bsa.rotary_nd(st["gq"], st["gk"], st["positions"], st["inv_freq"], _axes(case), inverse=True, **how)
        return res
    if case["op"] == "window":
        how = dict(kv_lens=st.get("lens"))
        args = (case["window"], case["sinks"])
        if not case["train"]:
            return (bsa.window_attn_fwd(st["q"], st["k"], st["v"], *args, **how)[0],)
        out, lse = bsa.window_attn_fwd(st["q"], st["k"], st["v"], *args, return_lse=True, **how)
        return (out, lse) + tuple(bsa.window_attn_bwd(st["dout"], st["q"], st["k"], st["v"], out, lse, *args, **how))
    if case["op"] == "cached":
        mask = bsa.tree_mask_from_parents(st["parents"]) if case["tree"] else None
        out, _ = bsa.cached_attn_fwd(st["q"], st["k_cache"], st["v_cache"], st["page_table"], st["lens"], tree_mask=mask,
                                     window=case["window"] or None, sink_tokens=case["sinks"])
        return (out,)
    bsa.cache_append(st["k"], st["v"], st["k_cache"], st["v_cache"], st["page_table"], st["lens"])
    if not case["keep"]:
        return st["k_cache"], st["v_cache"]
    lens = bsa.cache_keep(st["k_cache"], st["v_cache"], st["page_table"], st["lens"], st["path"], st["path_lens"], case["T"])
    return st["k_cache"], st["v_cache"], lens


def _plain_rotary(st, case):
    axes = _axes(case)
    half = sum(axes)
    # angles of far positions lose their fraction in 32 bits
    which = torch.repeat_interleave(torch.arange(len(axes), device="cuda"), torch.tensor(axes, device="cuda"))
    angle = st["positions"][..., which].double() * st["inv_freq"].double()
    cos, sin = angle.cos().float(), angle.sin().float()
    at = 1 if case["layout"] == "bhsd" else 2
    cos, sin = cos.unsqueeze(at), sin.unsqueeze(at)

    def turn(x, sign):
        f = x.float()
        if case["interleaved"]:
            a, b = f[..., 0:2 * half:2], f[..., 1:2 * half:2]
            turned = torch.stack((a * cos - b * (sin * sign), a * (sin * sign) + b * cos), -1).flatten(-2)
        else:
            a, b = f[..., :half], f[..., half:2 * half]
            turned = torch.cat((a * cos - b * (sin * sign), a * (sin * sign) + b * cos), -1)
        return torch.cat((turned, f[..., 2 * half:]), -1).to(x.dtype)

    res = turn(st["q"], 1.0), turn(st["k"], 1.0)
    return res + (turn(st["gq"], -1.0), turn(st["gk"], -1.0)) if case["train"] else res


def _window_forward(q, k, v, W, sinks, lens, scale):
    """Local attention by blocks of 128 queries: each block meets its W + 127 keys and, apart from them, the sinks."""
    B, Hq, Sq, D = q.shape
    Hkv, Sk = k.shape[1], k.shape[2]
    G, C, off = Hq // Hkv, 128, Sk - Sq
    W = min(W, Sk)
    n = -(-Sq // C)
    E, front = W + C - 1, max(0, W - 1 - off)
    first = off - (W - 1) + front
    pad = torch.nn.functional.pad
    qb = pad(q, (0, 0, 0, n * C - Sq)).view(B, Hkv, G, n, C, D).transpose(2, 3).reshape(B, Hkv, n, G * C, D)
    kw = pad(k, (0, 0, front, n * C - Sq))[:, :, first:].unfold(2, E, C)  # [B, Hkv, n, D, E]
    vw = pad(v, (0, 0, front, n * C - Sq))[:, :, first:].unfold(2, E, C)
    at_q = off + torch.arange(n * C, device="cuda").view(1, 1, n, 1, C, 1)
    at_k = (off - (W - 1) + C * torch.arange(n, device="cuda")).view(1, 1, n, 1, 1, 1) + torch.arange(E, device="cuda")
    live = at_q < lens.view(B, 1, 1, 1, 1, 1)
    near = (at_k >= 0) & (at_k <= at_q) & (at_k > at_q - W) & live
    far = (torch.arange(sinks, device="cuda") <= at_q - W) & live  # a sink inside the window counts there
    s = torch.where(near, (qb @ kw).view(B, Hkv, n, G, C, E) * scale, -math.inf)
    t = (qb @ k[:, :, None, :sinks].transpose(-1, -2)).view(B, Hkv, n, G, C, min(sinks, Sk)) * scale
    s = torch.cat((s, torch.where(far[..., :min(sinks, Sk)], t, -math.inf)), -1)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = (p / torch.where(total == 0, 1.0, total)).view(B, Hkv, n, G * C, -1)
    o = p[..., :E] @ vw.transpose(-1, -2) + p[..., E:] @ v[:, :, None, :sinks]
    lse = (top + torch.log(total)).view(B, Hkv, n, G, C)

    def back(x):
        return x.reshape(B, Hkv, n, G, C, -1).transpose(2, 3).reshape(B, Hq, n * C, -1)[:, :, :Sq]

    return back(o), back(lse)[..., 0]


def _plain_window(st, case):
    q, k, v = (st[n].float() for n in "qkv")
    lens = st["lens"] if case["ragged"] else torch.full((case["B"],), case["Sk"], device="cuda")
    scale, dt = case["D"] ** -0.5, DT[case["dtype"]]
    if not case["train"]:
        return (_window_forward(q, k, v, case["window"], case["sinks"], lens, scale)[0].to(dt),)
    for_grad = [t.requires_grad_() for t in (q, k, v)]
    out, lse = _window_forward(q, k, v, case["window"], case["sinks"], lens, scale)
    dq, dk, dv = torch.autograd.grad(out, for_grad, st["dout"].float())
    return out.detach().to(dt), lse.detach(), dq.to(dt), dk.to(dt), dv.to(dt)


def _ancestors(parents):
    """[B, T, T]: which drafts a draft sees, itself among them."""
    B, T = parents.shape
    a = (parents[:, :, None] == torch.arange(T, device="cuda")).float() + torch.eye(T, device="cuda")
    a = ((a @ a) > 0).float()
    a = ((a @ a) > 0).float()
    a = ((a @ a) > 0).float()
    a = ((a @ a) > 0).float()
    a = ((a @ a) > 0).float()
    return (a @ a) > 0  # paths of up to 64 drafts


def _plain_cached(st, case):
    q, table, lens = st["q"].float(), st["page_table"].long(), st["lens"].long()
    B, Hq, T, D = q.shape
    Hkv, page, W, sinks = case["Hkv"], case["page"], case["window"], case["sinks"]
    base = lens - T
    # the tokens that some row can see: the sinks, and the window of the first new token up to the newest one
    span = min(case["ctx"], W + T - 1) if W else case["ctx"]
    near = (lens[:, None] - span + torch.arange(span, device="cuda"))  # [B, span], negative: no such token
    first = torch.arange(min(sinks, case["ctx"]) if W else 0, device="cuda").expand(B, -1)
    at = torch.cat((near, first), 1)
    there = torch.cat((near >= 0, first < near[:, :1]), 1)  # a sink that the span holds counts there
    at = at.clamp_min(0)
    pages = table.gather(1, at // page).clamp_min(0)
    k = st["k_cache"][pages, :, at % page].transpose(1, 2).float()  # [B, Hkv, n, D]
    v = st["v_cache"][pages, :, at % page].transpose(1, 2).float()
    at_k, drafts = at[:, None], torch.arange(T, device="cuda")
    if case["tree"]:
        sees = _ancestors(st["parents"])
        depth = sees.sum(-1) - 1
        at_q = base[:, None, None] + depth[:, :, None]
        draft = (at_k - base[:, None, None]).clamp(0, T - 1).expand(B, T, -1)
        rank = torch.where(at_k < base[:, None, None], at_k, base[:, None, None] + depth[:, None].expand(B, T, T).gather(2, draft))
        visible = (at_k < base[:, None, None]) | sees.gather(2, draft)
    else:
        at_q = (base[:, None] + drafts)[:, :, None]
        rank = at_k.expand(B, T, -1)
        visible = rank <= at_q
    if W:
        visible = visible & ((rank > at_q - W) | (rank < sinks))
    visible = (visible & there[:, None])[:, None, None]
    s = (q.view(B, Hkv, -1, D) @ k.transpose(-1, -2)).view(B, Hkv, Hq // Hkv, T, -1) * D ** -0.5
    s = torch.where(visible, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    return ((p.view(B, Hkv, -1, p.shape[-1]) @ v).view(B, Hq, T, D).to(st["q"].dtype),)


def _plain_cache(st, case):
    table, lens, page, T = st["page_table"].long(), st["lens"].long(), case["page"], case["T"]
    base = lens - T
    at = base[:, None] + torch.arange(T, device="cuda")
    pages = table.gather(1, at // page)
    st["k_cache"][pages, :, at % page] = st["k"].transpose(1, 2)
    st["v_cache"][pages, :, at % page] = st["v"].transpose(1, 2)
    if not case["keep"]:
        return st["k_cache"], st["v_cache"]
    steps = torch.arange(case["keep"], device="cuda")
    # entries past the accepted length move a token onto itself
    src = torch.where(steps < st["path_lens"][:, None], st["path"].long(), steps) + base[:, None]
    dst = steps + base[:, None]
    keep = (steps < st["path_lens"][:, None]) | (src == dst)
    sp, dp = table.gather(1, src // page), table.gather(1, dst // page)
    hold = keep[:, :, None, None]
    for_k = torch.where(hold, st["k_cache"][sp, :, src % page], st["k_cache"][dp, :, dst % page])
    for_v = torch.where(hold, st["v_cache"][sp, :, src % page], st["v_cache"][dp, :, dst % page])
    st["k_cache"][dp, :, dst % page] = for_k
    st["v_cache"][dp, :, dst % page] = for_v
    return st["k_cache"], st["v_cache"], (base + st["path_lens"]).to(torch.int32)


# ------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------------------------------
def _pairs(Sq, Sk, W, sinks):
    """Visible (query, key) pairs of one head of a sequence without padding."""
    lo, hi = Sk - Sq, Sk  # positions of the queries
    full = lambda n, w: n * (n + 1) // 2 if n <= w else w * (w + 1) // 2 + (n - w) * w  # noqa: E731
    near = full(hi, W) - full(max(lo, 0), W)
    # at position p, the sinks that the window has left behind
    gone = lambda n: full(max(n - W, 0), sinks)  # noqa: E731
    return near + gone(hi) - gone(max(lo, 0))


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    D = case["D"]
    if case["op"] == "rotary":
        n = case["B"] * case["S"] * (case["Hq"] + case["Hkv"]) * (2 if case["train"] else 1)
        pairs = sum(_axes(case))
        return {"bytes": 2 * n * D * size + case["B"] * case["S"] * 4 * len(_axes(case)), "flops": 6 * n * pairs}
    if case["op"] == "window":
        B, Sq, Sk = case["B"], case["Sq"], case["Sk"]
        qs, ks = B * case["Hq"] * Sq * D * size, B * case["Hkv"] * min(Sk, Sq + case["window"] + case["sinks"]) * D * size
        pairs = B * case["Hq"] * _pairs(Sq, Sk, case["window"], case["sinks"])
        if case["ragged"]:
            pairs = pairs * (1 + 3 * B) // (4 * B)  # three quarters of the rows of all sequences but the first, on average
        if not case["train"]:
            return {"bytes": 2 * qs + 2 * ks, "flops": 4 * D * pairs}
        return {"bytes": 4 * qs + 4 * ks + B * case["Hq"] * Sq * 4, "flops": 14 * D * pairs}
    B, T = case["B"], case["T"]
    if case["op"] == "cached":
        mean = case["ctx"] * 3 // 4 if B > 1 else case["ctx"]
        seen = min(mean, case["window"] + case["sinks"] + T - 1) if case["window"] else mean
        return {"bytes": 2 * B * case["Hkv"] * seen * D * size + 2 * B * case["Hq"] * T * D * size,
                "flops": 4 * B * case["Hq"] * T * seen * D}
    moved = B * case["Hkv"] * D * size * 2
    return {"bytes": 2 * moved * T + moved * case["keep"], "flops": 0}


# ------------------------------------------------------------------------------------------------------------------
# the definition, in 64 bits
# ------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "rotary":
        res = [_exact_turn(st[n], st, case, n.startswith("g")) for n in (("q", "k", "gq", "gk") if case["train"] else ("q", "k"))]
        return tuple(res)
    if case["op"] == "window":
        return _exact_window(st, case)
    if case["op"] == "cached":
        return (_exact_cached(st, case),)
    return _exact_cache(st, case)


def _exact_turn(x, st, case, inverse):
    """Pairs as complex numbers times exp(i angle)."""
    x = x.double() if case["layout"] == "bhsd" else x.double().transpose(1, 2)
    res, pair = x.clone(), 0
    n = sum(_axes(case))
    for axis, count in enumerate(_axes(case)):
        for _ in range(count):
            a, b = (2 * pair, 2 * pair + 1) if case["interleaved"] else (pair, n + pair)
            angle = st["positions"][:, None, :, axis].double() * st["inv_freq"][pair].double()
            z = torch.complex(x[..., a], x[..., b]) * torch.polar(torch.ones_like(angle), -angle if inverse else angle)
            res[..., a], res[..., b] = z.real, z.imag
            pair += 1
    return res if case["layout"] == "bhsd" else res.transpose(1, 2)


def _exact_window(st, case):
    """Row blocks against the whole range of keys that any of them can see, one group of heads at a time."""
    B, Hq, Sq, D = st["q"].shape
    Hkv, Sk, W, sinks = case["Hkv"], case["Sk"], case["window"], case["sinks"]
    G, off, scale = Hq // Hkv, Sk - Sq, D ** -0.5
    out = torch.zeros(B, Hq, Sq, D, dtype=torch.float64, device="cuda")
    lse = torch.full((B, Hq, Sq), -math.inf, dtype=torch.float64, device="cuda")
    dq, dk, dv = torch.zeros_like(out), torch.zeros(B, Hkv, Sk, D, dtype=torch.float64, device="cuda"), None
    dv = torch.zeros_like(dk)
    for b in range(B):
        n = int(st["lens"][b]) if case["ragged"] else Sk
        for h in range(Hkv):
            k, v = st["k"][b, h].double(), st["v"][b, h].double()
            for lo in range(0, Sq, 1024):
                hi = min(lo + 1024, Sq)
                if off + lo >= n:
                    continue
                i = torch.arange(lo, hi, device="cuda")[:, None] + off
                start = max(0, off + lo - W + 1)
                j = torch.cat((torch.arange(min(sinks, start), device="cuda"), torch.arange(start, off + hi, device="cuda")))
                seen = (j <= i) & ((j > i - W) | (j < sinks)) & (i < n)
                rows = slice(h * G, (h + 1) * G)
                qs = st["q"][b, rows, lo:hi].double()
                s = (qs @ k[j].T * scale).masked_fill(~seen, -math.inf)
                z = torch.logsumexp(s, -1)
                p = torch.exp(s - torch.where(z == -math.inf, 0.0, z)[..., None])
                lse[b, rows, lo:hi], out[b, rows, lo:hi] = z, p @ v[j]
                if case["train"]:
                    g = st["dout"][b, rows, lo:hi].double()
                    ds = p * (g @ v[j].T - (g * out[b, rows, lo:hi]).sum(-1, keepdim=True)) * scale
                    dq[b, rows, lo:hi] = ds @ k[j]
                    dk[b, h].index_add_(0, j, (ds.transpose(1, 2) @ qs).sum(0))
                    dv[b, h].index_add_(0, j, (p.transpose(1, 2) @ g).sum(0))
    return (out, lse, dq, dk, dv) if case["train"] else (out,)


def _exact_cached(st, case):
    B, Hq, T, D = st["q"].shape
    Hkv, page, W, sinks = case["Hkv"], case["page"], case["window"] or 1 << 40, case["sinks"]
    out = torch.zeros(B, Hq, T, D, dtype=torch.float64, device="cuda")
    parents = st["parents"].tolist() if case["tree"] else None
    for b in range(B):
        n = int(st["lens"][b])
        base = n - T
        j = torch.arange(n, device="cuda")
        seen = torch.zeros(T, n, dtype=torch.bool)
        place = torch.arange(n)  # of each token: where its text has it
        at = [base + t for t in range(T)]
        chains = [[t] for t in range(T)]
        if parents:
            for t in range(T):
                up = parents[b][t]
                chains[t] = [t] + (chains[up] if up >= 0 else [])
                at[t] = base + len(chains[t]) - 1
                place[base + t] = at[t]
        else:
            chains = [list(range(t + 1)) for t in range(T)]
        for t in range(T):
            mine = torch.zeros(n, dtype=torch.bool)
            mine[:base] = True
            mine[[base + u for u in chains[t]]] = True
            seen[t] = mine & ((place > at[t] - W) | (place < sinks))
        seen = seen.cuda()
        some = seen.any(0)
        j, seen = j[some], seen[:, some]
        pages = st["page_table"][b].long()[j // page]
        k, v = (st[c][pages, :, j % page].transpose(0, 1).double() for c in ("k_cache", "v_cache"))
        for h in range(Hkv):
            rows = slice(h * Hq // Hkv, (h + 1) * Hq // Hkv)
            s = (st["q"][b, rows].double() @ k[h].T * D ** -0.5).masked_fill(~seen, -math.inf)
            out[b, rows] = torch.softmax(s, -1) @ v[h]
    return out


def _exact_cache(st, case):
    k, v = st["k_cache"].double(), st["v_cache"].double()
    page, T = case["page"], case["T"]
    table, lens = st["page_table"].tolist(), st["lens"].tolist()
    path, count = (st["path"].tolist(), st["path_lens"].tolist()) if case["keep"] else ([], [0] * case["B"])
    for b in range(case["B"]):
        base = lens[b] - T
        for t in range(T):
            # the draft that ends at this place: the accepted one, where there is one
            u = path[b][t] if t < count[b] else t
            p, r = table[b][(base + t) // page], (base + t) % page
            k[p, :, r], v[p, :, r] = st["k"][b, :, u].double(), st["v"][b, :, u].double()
    if not case["keep"]:
        return k, v
    return k, v, torch.tensor([n - T + c for n, c in zip(lens, count)], dtype=torch.int32, device="cuda")
