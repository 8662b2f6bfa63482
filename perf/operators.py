"""The serving and position operators that stand beside ring attention, as cases to measure.

Five operators: rotary positions (forward and backward), writing new tokens
into a paged key/value cache, copying pages of it, keeping the accepted path of
a drafted tree, and the attention of drafted trees, single tokens and chunks
over the cache.  ``run`` computes them in elementary torch operations, or with
this package's kernels where ``own`` is true.

Shapes follow the package: tokens are ``[tokens, heads, dim]`` packed over the
requests (``cu_q`` holds their borders), pages are
``[pages, kv heads, page size, dim]`` with an optional leading layer dimension.
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


# --------------------------------------------------------------------------- cases
def listed():
    return [
        # positions of one decoding step far into a long context: 32 requests, part of the head rotated
        dict(name="rotary_step_far", op="rotary", dtype="fp16", tokens=32, heads=32, heads_kv=8, dim=128,
             rotary=64, interleaved=True, far=1 << 20, base=500000.0, scale=1.0, grad=False),
        # training step of a 16384-token shard, q and k as slices of one projection, forward and backward
        dict(name="rotary_train_16k", op="rotary", dtype="bf16", tokens=16384, heads=32, heads_kv=8, dim=128,
             rotary=128, interleaved=False, far=1 << 17, base=1000000.0, scale=1.0, grad=True),
        # one new token of each of 64 requests written into the cache, its query rotated with it
        dict(name="append_step_64", op="append", dtype="bf16", batch=64, q_lo=1, q_hi=1, ctx_lo=100, ctx_hi=6000,
             heads=32, heads_kv=8, dim=128, page=16, rotary=128, interleaved=False, base=500000.0),
        # ragged prompts, 5 of them, written into the cache
        dict(name="append_prompts", op="append", dtype="fp16", batch=5, q_lo=777, q_hi=6001, ctx_lo=0, ctx_hi=1000,
             heads=32, heads_kv=8, dim=128, page=64, rotary=64, interleaved=True, base=10000.0),
        # a forked request's last, partly filled page copied in every layer, for 8 samples
        dict(name="copy_fork_8", op="copy", dtype="bf16", layers=32, pages=64, pairs=8, heads_kv=8, dim=128, page=16),
        # pages moved to the front of a pool so that its tail can be given back
        dict(name="copy_defrag", op="copy", dtype="fp16", layers=8, pages=2048, pairs=700, heads_kv=8, dim=128, page=16),
        # the accepted path of 4 requests' drafted trees, 32 layers
        dict(name="path_4", op="path", dtype="bf16", layers=32, batch=4, tree=16, path=4, ctx_lo=50, ctx_hi=900,
             heads_kv=8, dim=128, page=16),
        # the same after a wide draft of many requests
        dict(name="path_128", op="path", dtype="fp16", layers=16, batch=128, tree=64, path=9, ctx_lo=10, ctx_hi=300,
             heads_kv=8, dim=128, page=32),
        # one token of each of 4 requests: decoding, where latency counts
        dict(name="decode_4", op="tree", dtype="bf16", batch=4, q_lo=1, q_hi=1, ctx_lo=500, ctx_hi=4000, heads=32,
             heads_kv=8, dim=128, page=16, masked=False),
        # drafted trees of 32 requests with contexts from short to long
        dict(name="tree_32", op="tree", dtype="bf16", batch=32, q_lo=5, q_hi=32, ctx_lo=200, ctx_hi=24000, heads=32,
             heads_kv=8, dim=128, page=32, masked=True),
        # the reference benchmark's element type and head size: fp32, 64 wide, 16384 keys
        dict(name="tree_fp32_16k", op="tree", dtype="fp32", batch=3, q_lo=3, q_hi=8, ctx_lo=4096, ctx_hi=16384,
             heads=8, heads_kv=8, dim=64, page=64, masked=True),
        # a chunk of a long prompt over what is cached of it: causal, bound by the tensor cores
        dict(name="chunk_32k", op="tree", dtype="fp16", batch=1, q_lo=1000, q_hi=1000, ctx_lo=32000, ctx_hi=32000,
             heads=32, heads_kv=8, dim=128, page=128, masked=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "append", "copy", "path", "tree", "tree"])
    dtype = rng.choice(["bf16", "fp16"])
    dim = rng.choice([64, 128])
    heads_kv, group = rng.choice([(1, 8), (2, 7), (4, 4), (8, 4), (8, 1), (8, 8), (5, 3)])
    page = rng.choice([16, 32, 64, 128])
    if op == "rotary":
        return dict(op=op, dtype=rng.choice(["bf16", "fp16", "fp32"]), tokens=_log(rng, 1, 8000), heads=heads_kv * group,
                    heads_kv=heads_kv, dim=dim, rotary=rng.choice([dim, dim // 2]), interleaved=rng.random() < 0.5,
                    far=_log(rng, 100, 1 << 22), base=rng.choice([10000.0, 500000.0]), scale=rng.choice([1.0, 1.25]),
                    grad=rng.random() < 0.5)
    if op == "append":
        hi = _log(rng, 1, 900)
        return dict(op=op, dtype=rng.choice(["bf16", "fp16", "fp32"]), batch=_log(rng, 1, 20), q_lo=rng.randint(1, hi),
                    q_hi=hi, ctx_lo=0, ctx_hi=_log(rng, 10, 3000), heads=heads_kv * group, heads_kv=heads_kv, dim=dim,
                    page=page, rotary=dim, interleaved=rng.random() < 0.5, base=10000.0)
    if op == "copy":
        pages = _log(rng, 20, 400)
        return dict(op=op, dtype=dtype, layers=rng.randint(1, 32), pages=pages, pairs=rng.randint(1, pages // 2),
                    heads_kv=heads_kv, dim=dim, page=min(page, 32))
    if op == "path":
        tree = _log(rng, 2, 64)
        return dict(op=op, dtype=dtype, layers=rng.randint(1, 16), batch=_log(rng, 1, 100), tree=tree,
                    path=rng.randint(1, min(tree, 12)), ctx_lo=0, ctx_hi=_log(rng, 10, 200), heads_kv=heads_kv, dim=dim,
                    page=page)
    if rng.random() < 0.2:
        heads_kv = rng.choice([1, 2, 8])
        return dict(op=op, dtype="fp32", batch=_log(rng, 1, 6), q_lo=1, q_hi=_log(rng, 1, 8), ctx_lo=0,
                    ctx_hi=_log(rng, 50, 12000), heads=heads_kv * rng.choice([1, 2]), heads_kv=heads_kv, dim=dim,
                    page=page, masked=rng.random() < 0.7)
    masked = rng.random() < 0.7
    hi = _log(rng, 1, 64) if masked else _log(rng, 1, 400)
    batch = _log(rng, 1, 24) if masked else _log(rng, 1, 6)
    return dict(op=op, dtype=dtype, batch=batch, q_lo=rng.randint(1, hi), q_hi=hi, ctx_lo=0, ctx_hi=_log(rng, 30, 16000),
                heads=heads_kv * group, heads_kv=heads_kv, dim=dim, page=page, masked=masked)


# --------------------------------------------------------------------------- what a case holds
def _spread(lo, hi, n):
    """n whole numbers from lo to hi, in an order that is not their size's."""
    at = [(b * 7919) % n for b in range(n)] if n % 7919 else list(range(n))
    return [lo + (hi - lo) * a // max(1, n - 1) for a in at] if n > 1 else [hi]


def _path(tree, n):
    """The places in the drafted tree of an accepted path of n tokens: the first and the last, and what lies between."""
    return [i + (i * (tree - n)) // max(1, n - 1) for i in range(n)] if n > 1 else [tree - 1]


def _frequencies(rotary, base):
    p = torch.arange(rotary // 2, dtype=torch.float64)
    return base ** (-2.0 * p / rotary)


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(shape, dtype, g, std=1.0):
    return (torch.randn(shape, device="cuda", dtype=torch.float32, generator=g) * std).to(dtype)


def _ragged(case):
    """Tokens already cached and tokens of this pass, per request."""
    return _spread(case["ctx_lo"], case["ctx_hi"], case["batch"]), _spread(case["q_lo"], case["q_hi"], case["batch"])[::-1]


def _table(lens, page, g):
    """A page table over a pool in which every request's pages lie anywhere; the pool has some pages that nobody holds."""
    need = [-(-n // page) for n in lens]
    pool = sum(need) + 3
    order = torch.randperm(pool, device="cuda", generator=g)
    start = torch.tensor([0] + need).cumsum(0)[:-1].cuda()
    wide = torch.arange(max(need), device="cuda")
    at = (start[:, None] + wide).clamp(max=pool - 1)
    table = torch.where(wide < torch.tensor(need).cuda()[:, None], order[at], torch.zeros_like(at))
    return table.to(torch.int32), pool


def _int32(v):
    return torch.tensor(v, dtype=torch.int32).cuda()


def _borders(counts):
    return _int32([0] + counts).cumsum(0).to(torch.int32)


def prepare(case, seed):
    g, dt, op = _gen(seed), _DTYPES[case["dtype"]], case["op"]
    s = dict(case=case)
    if op == "rotary":
        T, H, Hk, D = case["tokens"], case["heads"], case["heads_kv"], case["dim"]
        qkv = _normal((T, H + 2 * Hk, D), dt, g)  # one projection's output: q, k and v lie side by side
        s["q"], s["k"] = qkv[:, :H], qkv[:, H:H + Hk]
        far = case["far"]
        s["positions"] = (torch.randint(0, far, (T,), device="cuda", generator=g) if T < 256 else
                          torch.randint(0, far, (1,), device="cuda", generator=g) + torch.arange(T, device="cuda"))
        s["inv_freq"] = _frequencies(case["rotary"], case["base"]).cuda()
        if case["grad"]:
            s["q"], s["k"] = s["q"].requires_grad_(), s["k"].requires_grad_()
            s["gq"], s["gk"] = _normal((T, H, D), dt, g), _normal((T, Hk, D), dt, g)
        return s
    if op == "append":
        ctx, n = _ragged(case)
        T, H, Hk, D, page = sum(n), case["heads"], case["heads_kv"], case["dim"], case["page"]
        s["table"], pool = _table([c + m for c, m in zip(ctx, n)], page, g)
        qkv = _normal((T, H + 2 * Hk, D), dt, g)
        s["q"], s["k"], s["v"] = qkv[:, :H], qkv[:, H:H + Hk], qkv[:, H + Hk:]
        s["k_pages"], s["v_pages"] = (_normal((pool, Hk, page, D), dt, g) for _ in "kv")
        s["ctx"], s["cu_q"] = _int32(ctx), _borders(n)
        s["inv_freq"] = _frequencies(case["rotary"], case["base"]).cuda()
        return s
    if op == "copy":
        L, P, Hk, D, page = case["layers"], case["pages"], case["heads_kv"], case["dim"], case["page"]
        s["k_pages"], s["v_pages"] = (_normal((L, P, Hk, page, D), dt, g) for _ in "kv")
        order = torch.randperm(P, device="cuda", generator=g).cpu().to(torch.int32)
        # what a scheduler holds on the host: which pages go where; a page may be copied to several places
        n = case["pairs"]
        s["dst"], s["src"] = order[:n].clone(), order[n:][torch.arange(n) % max(1, min(n, P - n) // 2 + 1)].clone()
        return s
    if op == "path":
        ctx = _spread(case["ctx_lo"], case["ctx_hi"], case["batch"])
        L, Hk, D, page = case["layers"], case["heads_kv"], case["dim"], case["page"]
        s["table"], pool = _table([c + case["tree"] for c in ctx], page, g)
        s["k_pages"], s["v_pages"] = (_normal((L, pool, Hk, page, D), dt, g) for _ in "kv")
        s["ctx"] = _int32(ctx)
        s["path"] = _int32([_path(case["tree"], case["path"])] * case["batch"])
        s["path_lens"] = _int32([max(1, case["path"] - b % 3) for b in range(case["batch"])])
        return s
    ctx, n = _ragged(case)
    T, H, Hk, D, page = sum(n), case["heads"], case["heads_kv"], case["dim"], case["page"]
    s["table"], pool = _table([c + m for c, m in zip(ctx, n)], page, g)
    s["q"] = _normal((T, H, D), dt, g)
    s["k_pages"], s["v_pages"] = _normal((pool, Hk, page, D), dt, g), _normal((pool, Hk, page, D), dt, g)
    s["ctx"], s["cu_q"], s["max_q"] = _int32(ctx), _borders(n), max(n)
    s["mask"] = None
    if case["masked"]:
        # a drafted tree of each request: every token's parent is one of the tokens before it, the first is the root;
        # a token sees its ancestors and itself, as bits of 32-bit words
        w = max(n)
        parent = (torch.rand((case["batch"], w), device="cuda", generator=g) * torch.arange(w, device="cuda")).long()
        sees = torch.eye(w, device="cuda", dtype=torch.bool).repeat(case["batch"], 1, 1)
        each = torch.arange(case["batch"], device="cuda")
        for i in range(1, w):
            sees[:, i] |= sees[each, parent[:, i]]
        words = -(-w // 32)
        bits = torch.nn.functional.pad(sees.long(), (0, words * 32 - w)).view(case["batch"], w, words, 32)
        packed = (bits << torch.arange(32, device="cuda")).sum(-1)
        packed = torch.where(packed >= 1 << 31, packed - (1 << 32), packed).to(torch.int32)
        row = torch.arange(w, device="cuda") < torch.tensor(n).cuda()[:, None]
        s["mask"] = packed[row].contiguous()
    return s


# --------------------------------------------------------------------------- the operators
def run(s):
    return _OWN[s["case"]["op"]](s) if own else _PLAIN[s["case"]["op"]](s)


def _own_rotary(s):
    from ring_attention_benchmark_b200.ops.rotary import apply_rotary

    c = s["case"]
    out = apply_rotary(s["q"], s["k"], s["positions"], s["inv_freq"], interleaved=c["interleaved"], scale=c["scale"])
    if c["grad"]:
        return out + torch.autograd.grad(out, (s["q"], s["k"]), (s["gq"], s["gk"]))
    return out


def _own_append(s):
    from ring_attention_benchmark_b200.ops.paged import append_kv

    q = append_kv(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["ctx"], s["cu_q"], q=s["q"],
                  inv_freq=s["inv_freq"], interleaved=s["case"]["interleaved"])
    return q, s["k_pages"], s["v_pages"]


def _own_copy(s):
    from ring_attention_benchmark_b200.ops.paged import copy_pages

    copy_pages(s["k_pages"], s["v_pages"], s["src"], s["dst"])
    return s["k_pages"], s["v_pages"]


def _own_path(s):
    from ring_attention_benchmark_b200.ops.paged import compact_path

    compact_path(s["k_pages"], s["v_pages"], s["table"], s["ctx"], s["path"], s["path_lens"])
    return s["k_pages"], s["v_pages"]


def _own_tree(s):
    from ring_attention_benchmark_b200.ops.paged import tree_attention

    return tree_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["ctx"], s["cu_q"], max_q=s["max_q"],
                          mask=s["mask"], return_lse=True)


def _rotate(x, positions, inv_freq, interleaved, scale):
    angle = positions.double()[:, None] * inv_freq  # 64 bits: far positions
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    r, xf = 2 * inv_freq.numel(), x.float()
    if interleaved:
        a, b = xf[..., 0:r:2], xf[..., 1:r:2]
    else:
        a, b = xf[..., :r // 2], xf[..., r // 2:r]
    y = ((a * cos - b * sin) * scale, (b * cos + a * sin) * scale)
    y = torch.stack(y, -1).flatten(-2) if interleaved else torch.cat(y, -1)
    return torch.cat((y, xf[..., r:]), -1).to(x.dtype)


def _plain_rotary(s):
    c = s["case"]
    out = tuple(_rotate(s[x], s["positions"], s["inv_freq"], c["interleaved"], c["scale"]) for x in "qk")
    if c["grad"]:
        return out + torch.autograd.grad(out, (s["q"], s["k"]), (s["gq"], s["gk"]))
    return out


def _places(s, total):
    """Request, place in the cache, page and offset of each packed token."""
    token = torch.arange(total, device="cuda")
    request = torch.searchsorted(s["cu_q"], token, right=True) - 1
    at = s["ctx"][request] + token - s["cu_q"][request]
    page = s["case"]["page"]
    return at, s["table"][request, at // page].long(), at % page


def _plain_append(s):
    at, page, off = _places(s, s["k"].shape[0])
    inter = s["case"]["interleaved"]
    s["k_pages"][page, :, off] = _rotate(s["k"], at, s["inv_freq"], inter, 1.0)
    s["v_pages"][page, :, off] = s["v"]
    return _rotate(s["q"], at, s["inv_freq"], inter, 1.0), s["k_pages"], s["v_pages"]


def _plain_copy(s):
    src, dst = s["src"].cuda().long(), s["dst"].cuda().long()
    s["k_pages"][:, dst] = s["k_pages"][:, src]
    s["v_pages"][:, dst] = s["v_pages"][:, src]
    return s["k_pages"], s["v_pages"]


def _plain_path(s):
    page, n = s["case"]["page"], s["path"].shape[1]
    step = torch.arange(n, device="cuda").expand_as(s["path"])
    kept = step < s["path_lens"][:, None]
    request = torch.arange(kept.shape[0], device="cuda")[:, None].expand_as(kept)[kept]
    frm, to = (s["ctx"][:, None] + s["path"])[kept], (s["ctx"][:, None] + step)[kept]
    src, dst = s["table"][request, frm // page].long(), s["table"][request, to // page].long()
    s["k_pages"][:, dst, :, to % page] = s["k_pages"][:, src, :, frm % page]
    s["v_pages"][:, dst, :, to % page] = s["v_pages"][:, src, :, frm % page]
    return s["k_pages"], s["v_pages"]


def _plain_tree(s):
    q, cu, ctx, page, w = s["q"], s["cu_q"].long(), s["ctx"].long(), s["case"]["page"], s["max_q"]
    T, H, D = q.shape
    B, Hk = ctx.numel(), s["k_pages"].shape[1]
    count = cu[1:] - cu[:-1]
    width = s["table"].shape[1] * page
    key = torch.arange(width, device="cuda")
    # the requests' keys and values side by side, queries padded to the widest request
    pages = s["table"].long()
    k = s["k_pages"][pages].permute(0, 2, 1, 3, 4).reshape(B, Hk, width, D).float()
    v = s["v_pages"][pages].permute(0, 2, 1, 3, 4).reshape(B, Hk, width, D).float()
    token = torch.arange(T, device="cuda")
    request = torch.searchsorted(cu, token, right=True) - 1
    place = token - cu[request]
    qp = q.new_zeros(B, w, H, D, dtype=torch.float32)
    qp[request, place] = q.float()
    qp = qp.view(B, w, Hk, H // Hk, D).permute(0, 2, 1, 3, 4).reshape(B, Hk, w * (H // Hk), D)
    rel = key - ctx[:, None]  # a key's place among the request's new tokens
    row = torch.arange(w, device="cuda")[:, None]
    if s["mask"] is None:
        sees = rel[:, None] <= row
    else:
        bits = torch.zeros(B, w, s["mask"].shape[1], dtype=torch.int64, device="cuda")
        bits[request, place] = s["mask"].long()
        new = (rel >= 0) & (rel < count[:, None])
        at = rel.clamp(0, w - 1)[:, None].expand(B, w, width)
        sees = (rel < 0)[:, None] | (new[:, None] & ((bits.gather(2, at >> 5) >> (at & 31)) & 1).bool())
    sees = sees[:, None, :, None].expand(B, 1, w, H // Hk, width).reshape(B, 1, w * (H // Hk), width)
    score = (qp @ k.transpose(-1, -2)).mul_(D ** -0.5).masked_fill_(~sees, -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-1e30)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p @ v) / total.clamp(min=1e-38)
    lse = (top + total.log()).squeeze(-1)
    o = o.view(B, Hk, w, H // Hk, D).permute(0, 2, 1, 3, 4).reshape(B, w, H, D)[request, place]
    lse = lse.view(B, Hk, w, H // Hk).permute(0, 2, 1, 3).reshape(B, w, H)[request, place]
    return o.to(q.dtype), lse


_OWN = dict(rotary=_own_rotary, append=_own_append, copy=_own_copy, path=_own_path, tree=_own_tree)
_PLAIN = dict(rotary=_plain_rotary, append=_plain_append, copy=_plain_copy, path=_plain_path, tree=_plain_tree)


# --------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    e, D, op = _BYTES[case["dtype"]], case["dim"], case["op"]
    if op == "rotary":
        T, h = case["tokens"], case["heads"] + case["heads_kv"]
        passes = 2 if case["grad"] else 1
        return {"bytes": passes * 2 * T * h * D * e + 8 * T, "flops": passes * 3 * T * h * case["rotary"]}
    if op == "append":
        T, h = sum(_ragged(case)[1]), case["heads"] + 2 * case["heads_kv"]
        return {"bytes": 2 * T * h * D * e, "flops": 3 * T * (case["heads"] + case["heads_kv"]) * case["rotary"]}
    if op == "copy":
        n = case["pairs"]
        read = min(n, max(1, min(n, case["pages"] - n) // 2 + 1))  # source pages, each read once
        return {"bytes": (n + read) * case["layers"] * 2 * case["heads_kv"] * case["page"] * D * e, "flops": 0}
    if op == "path":
        moved = sum(sum(i != j for j, i in enumerate(_path(case["tree"], case["path"])[:max(1, case["path"] - b % 3)]))
                    for b in range(case["batch"]))
        return {"bytes": 2 * moved * case["layers"] * 2 * case["heads_kv"] * D * e + 4 * case["batch"], "flops": 0}
    ctx, n = _ragged(case)
    keys = sum(c + m for c, m in zip(ctx, n))
    seen = sum(m * c + m * (m + 1) // 2 for c, m in zip(ctx, n))
    if case["masked"]:  # at most that many: what a tree's tokens see of one another is small beside the context
        seen = sum(m * c + m for c, m in zip(ctx, n))
    return {"bytes": 2 * keys * case["heads_kv"] * D * e + 2 * sum(n) * case["heads"] * D * e,
            "flops": 4 * seen * case["heads"] * D}


# --------------------------------------------------------------------------- the definition, in 64 bits
def _turned(x, positions, inv_freq, interleaved, scale):
    """x as complex numbers, each turned by its angle."""
    r = 2 * inv_freq.numel()
    y = x.detach().double().clone()
    z = torch.polar(torch.full_like(angle := torch.outer(positions.double(), inv_freq), scale), angle)[:, None, :]
    if interleaved:
        y[..., :r] = torch.view_as_real(torch.view_as_complex(y[..., :r].unflatten(-1, (-1, 2)).contiguous()) * z).flatten(-2)
    else:
        t = torch.complex(y[..., :r // 2].contiguous(), y[..., r // 2:r].contiguous()) * z
        y[..., :r // 2], y[..., r // 2:r] = t.real, t.imag
    return y


def _token_places(case, s):
    ctx, n = _ragged(case)
    return torch.cat([torch.arange(c, c + m) for c, m in zip(ctx, n)]).cuda()


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "rotary":
        args = (s["positions"], s["inv_freq"], case["interleaved"], case["scale"])
        out = _turned(s["q"], *args), _turned(s["k"], *args)
        if case["grad"]:  # the transposed rotation
            back = (-s["positions"],) + args[1:]
            out += _turned(s["gq"], *back), _turned(s["gk"], *back)
        return out
    if op == "append":
        at = _token_places(case, s)
        args = (at, s["inv_freq"], case["interleaved"], 1.0)
        kt, (kp, vp) = _turned(s["k"], *args), (s[x].double() for x in ("k_pages", "v_pages"))
        ctx, n = _ragged(case)
        first, page = 0, case["page"]
        for b, m in enumerate(n):
            pos = at[first:first + m]
            pg = s["table"][b].long()[pos // page]
            kp[pg, :, pos % page], vp[pg, :, pos % page] = kt[first:first + m], s["v"][first:first + m].double()
            first += m
        return _turned(s["q"], *args), kp, vp
    if op == "copy":
        out = [s["k_pages"].double(), s["v_pages"].double()]
        for x, old in zip(out, ("k_pages", "v_pages")):
            for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
                x[:, b] = s[old][:, a].double()
        return tuple(out)
    if op == "path":
        out, page = [s["k_pages"].double(), s["v_pages"].double()], case["page"]
        ctx, table = s["ctx"].tolist(), s["table"].tolist()
        keep, lens = s["path"].tolist(), s["path_lens"].tolist()
        for x, old in zip(out, ("k_pages", "v_pages")):
            for b in range(case["batch"]):
                for i in range(lens[b]):
                    f, t = ctx[b] + keep[b][i], ctx[b] + i
                    x[:, table[b][t // page], :, t % page] = s[old][:, table[b][f // page], :, f % page].double()
        return tuple(out)
    ctx, n = _ragged(case)
    page, H, Hk, D = case["page"], case["heads"], case["heads_kv"], case["dim"]
    o = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    first, scale = 0, 1.0 / math.sqrt(D)
    for b, (c, m) in enumerate(zip(ctx, n)):
        pg = s["table"][b, :-(-(c + m) // page)].long()
        hidden = torch.ones(m, m, dtype=torch.bool, device="cuda").triu(1)
        if s["mask"] is not None:
            words = s["mask"][first:first + m].long()
            j = torch.arange(m, device="cuda")
            hidden = ((words[:, j // 32] >> (j % 32)) & 1) == 0
        for h in range(Hk):
            k, v = (s[x][pg, h].reshape(-1, D)[:c + m].double() for x in ("k_pages", "v_pages"))
            heads = slice(h * (H // Hk), (h + 1) * (H // Hk))
            z = torch.einsum("thd,kd->htk", s["q"][first:first + m, heads].double(), k) * scale
            z[:, :, c:].masked_fill_(hidden, -math.inf)
            lse[first:first + m, heads] = torch.logsumexp(z, -1).T
            o[first:first + m, heads] = torch.einsum("htk,kd->thd", torch.softmax(z, -1), v)
        first += m
    return o, lse
