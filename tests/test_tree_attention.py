"""Attention of drafted trees, single tokens and chunks over a paged cache, against 64 bits."""
import math

import pytest
import torch

import _paged_oracle as O
from ring_attention_benchmark_b200.ops.attention import DeviceTimeout, check_status, new_status
from ring_attention_benchmark_b200.ops.paged import pack_mask, tree_attention, tree_mask

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _case(ctx, counts, H, Hk, D, page, dtype, seed=0, extra=0, spread=1.0, fill=None):
    """Inputs on the CPU; unused rows of the pool hold `fill` (a stale cache holds anything)."""
    g = torch.Generator().manual_seed(seed)
    T = sum(counts)
    q = (torch.randn(T + extra, H, D, generator=g) * spread).to(dtype)
    need = [-(-(c + m) // page) for c, m in zip(ctx, counts)]
    pool = sum(need) + 2
    order = torch.randperm(pool, generator=g).tolist()
    table = torch.zeros(len(ctx), max(max(need), 1) + 1, dtype=torch.int32)
    kp, vp = (torch.full((pool, Hk, page, D), 0.0 if fill is None else fill).to(dtype) for _ in "kv")
    for b, n in enumerate(need):
        for i in range(n):
            table[b, i] = order.pop()
        for j in range(ctx[b] + counts[b]):
            kp[table[b, j // page], :, j % page] = torch.randn(Hk, D, generator=g).to(dtype)
            vp[table[b, j // page], :, j % page] = torch.randn(Hk, D, generator=g).to(dtype)
    return q, kp, vp, table


def _run(q, kp, vp, table, ctx, counts, uniform=False, **kw):
    cu = None if uniform else torch.tensor([0] + counts).cumsum(0).int().cuda()
    return tree_attention(q.cuda(), kp.cuda(), vp.cuda(), table.cuda(),
                          torch.tensor(ctx, dtype=torch.int32).cuda(), cu, return_lse=True, **kw)


def _check(got, lse, case, ctx, counts, masks=None, scale=None):
    q, kp, vp, table = case
    T = sum(counts)
    ref, rlse, mag, smax = O.attention(q[:T], kp, vp, table, ctx, counts, masks, scale)
    keys = max([c + m for c, m in zip(ctx, counts)] + [1])
    bo, bl = O.attention_bound(ref, mag, smax, q.dtype, keys, q.shape[2])
    g, gl = got[:T].cpu().double(), lse[:T].cpu().double()
    empty = rlse == -math.inf
    assert torch.equal(gl == -math.inf, empty)
    assert (g[empty] == 0).all()
    d = (g - ref).abs()
    assert (d <= bo).all(), ((d - bo).max().item(), d.max().item())
    dl = (gl - rlse).abs()[~empty]
    assert (dl <= (bl + 2.0 ** -22 * rlse.abs())[~empty]).all(), dl.max().item()


def _trees(counts, seed=0):
    g = torch.Generator().manual_seed(seed)
    parents, masks, depths = [], [], []
    for m in counts:
        p = [-1 if i == 0 or torch.rand(1, generator=g).item() < 0.1
             else int(torch.randint(0, i, (1,), generator=g)) for i in range(m)]
        mask, depth = O.ancestors(p)
        parents += p
        masks.append(mask)
        depths += depth
    w = max(counts)
    rows = torch.zeros(sum(counts), w, dtype=torch.bool)
    first = 0
    for m, mask in zip(counts, masks):
        rows[first:first + m, :m] = mask
        first += m
    return parents, masks, rows, depths


# ------------------------------------------------------------------ refusals (CPU)
def _args(**kw):
    a = dict(q=torch.zeros(2, 4, 64), k_pages=torch.zeros(3, 2, 16, 64),
             v_pages=torch.zeros(3, 2, 16, 64), block_table=torch.zeros(1, 2, dtype=torch.int32),
             context_lens=torch.zeros(1, dtype=torch.int32))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw, what", [
    (dict(), "CUDA"),
    (dict(q=torch.zeros(2, 4, 32), k_pages=torch.zeros(3, 2, 16, 32), v_pages=torch.zeros(3, 2, 16, 32)), "64 or 128"),
    (dict(q=torch.zeros(2, 4, 128)), "head dim"),
    (dict(q=torch.zeros(2, 3, 64)), "multiple"),
    (dict(q=torch.zeros(2, 4, 64).half()), "share a dtype"),
    (dict(k_pages=torch.zeros(3, 2, 24, 64), v_pages=torch.zeros(3, 2, 24, 64)), "page size"),
    (dict(k_pages=torch.zeros(3, 2, 8, 64), v_pages=torch.zeros(3, 2, 8, 64)), "page size"),
    (dict(k_pages=torch.zeros(3, 2, 512, 64), v_pages=torch.zeros(3, 2, 512, 64)), "page size"),
    (dict(mask=torch.zeros(3, 2, dtype=torch.bool)), "row for each"),
    (dict(mask=torch.zeros(2, 2)), "bool, or int32"),
    (dict(mask=torch.zeros(2, 0, dtype=torch.bool)), "columns"),
    (dict(scale=math.nan), "finite"),
    (dict(max_q=0), "max_q"),
    (dict(out=torch.zeros(2, 4, 128)), "shape"),
    (dict(out=torch.zeros(2, 4, 64).half()), "dtype"),
    (dict(out=torch.zeros(1, 4, 64).expand(2, 4, 64)), "shares memory"),
    (dict(out=torch.zeros(2, 4, 66)[:, :, :64]), "aligned"),
    (dict(timeout_s=0.0), "timeout_s"),
    (dict(context_lens=torch.zeros(1, dtype=torch.int64)), "int32"),
    (dict(context_lens=torch.zeros(3, dtype=torch.int32), block_table=torch.zeros(3, 2, dtype=torch.int32)), "evenly"),
])
def test_refusals(ext, kw, what):
    with pytest.raises(RuntimeError, match=what):
        tree_attention(**_args(**kw))


@pytest.mark.parametrize("kw, what", [
    (dict(parents=torch.zeros(4, dtype=torch.int32), max_q=4), "CUDA"),
    (dict(parents=torch.zeros(4), max_q=4), "int32"),
    (dict(parents=torch.zeros(4, dtype=torch.int32), max_q=0), "max_q"),
    (dict(parents=torch.zeros(4, dtype=torch.int32), max_q=4, batch=3), "evenly"),
])
def test_tree_mask_refusals(ext, kw, what):
    with pytest.raises(RuntimeError, match=what):
        tree_mask(**kw)


def test_pack_mask_refusals(ext):
    for m in (torch.zeros(2, 2), torch.zeros(2, 0, dtype=torch.bool), torch.zeros(2, 2, dtype=torch.bool)):
        with pytest.raises(RuntimeError, match="bool|columns|CUDA"):
            pack_mask(m)


# ------------------------------------------------------------------ masks (GPU)
def _bits(words, cols):
    j = torch.arange(cols)
    return ((words.cpu().long()[:, j // 32] >> (j % 32)) & 1).bool()


@pytest.mark.gpu
@pytest.mark.parametrize("counts", [[1], [1, 0, 5], [33, 64, 2], [70, 7]])
def test_tree_mask(ext, cuda_device, counts):
    parents, _, rows, depths = _trees([c for c in counts])
    w = max(counts)
    cu = torch.tensor([0] + counts).cumsum(0).int().cuda()
    st = new_status("cuda")
    mask, depth = tree_mask(torch.tensor(parents, dtype=torch.int32).cuda(), cu, max_q=w, status=st)
    check_status(st)
    assert mask.shape == (sum(counts), -(-w // 32))
    assert torch.equal(_bits(mask, w), rows) and depth.cpu().tolist() == depths
    assert torch.equal(pack_mask(rows.cuda()), mask)
    narrow, _ = tree_mask(torch.tensor(parents, dtype=torch.int32).cuda(), cu, max_q=1)
    assert torch.equal(_bits(narrow, min(w, 32)), rows[:, :32])


@pytest.mark.gpu
def test_tree_mask_uniform_and_bad_parents(ext, cuda_device):
    st = new_status("cuda")
    p = torch.tensor([-1, 0, 1, -1, 0, 0], dtype=torch.int32).cuda()
    mask, depth = tree_mask(p, batch=2, max_q=3, status=st)
    check_status(st)
    assert mask.flatten().tolist() == [1, 3, 7, 1, 3, 5] and depth.tolist() == [0, 1, 2, 0, 1, 1]
    mask, _ = tree_mask(torch.tensor([-1, 1, 5, -2], dtype=torch.int32).cuda(), batch=1, max_q=4, status=st)
    assert mask.flatten().tolist() == [1, 2, 4, 8]  # a token whose parent is no token before it is a root
    with pytest.raises(DeviceTimeout, match="code=2"):
        check_status(st)


# ------------------------------------------------------------------ values (GPU)
SHAPES = [
    # ctx, counts, heads, kv heads, dim, page
    ([0], [1], 1, 1, 64, 16),
    ([1, 0, 127, 128, 129], [1, 1, 1, 1, 1], 8, 2, 128, 16),
    ([300, 5, 64], [7, 1, 16], 7, 1, 64, 32),
    ([33, 0, 200], [3, 0, 40], 4, 4, 128, 64),
    ([0, 0], [130, 64], 2, 1, 64, 128),
    ([255, 256, 900], [2, 33, 5], 16, 2, 128, 256),
    ([70], [65], 24, 8, 64, 16),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ctx, counts, H, Hk, D, page", SHAPES)
def test_causal_values(ext, cuda_device, dtype, ctx, counts, H, Hk, D, page):
    case = _case(ctx, counts, H, Hk, D, page, dtype)
    st = new_status("cuda")
    out, lse = _run(*case, ctx, counts, status=st)
    check_status(st)
    _check(out, lse, case, ctx, counts)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ctx, counts, H, Hk, D, page", SHAPES)
def test_tree_values(ext, cuda_device, dtype, ctx, counts, H, Hk, D, page):
    case = _case(ctx, counts, H, Hk, D, page, dtype, seed=1)
    parents, masks, rows, _ = _trees(counts)
    st = new_status("cuda")
    out, lse = _run(*case, ctx, counts, mask=rows.cuda(), max_q=max(counts), status=st)
    _check(out, lse, case, ctx, counts, masks)
    words, _ = tree_mask(torch.tensor(parents, dtype=torch.int32).cuda(),
                         torch.tensor([0] + counts).cumsum(0).int().cuda(), max_q=max(counts))
    out2, lse2 = _run(*case, ctx, counts, mask=words, max_q=1, status=st)  # the hint only steers
    check_status(st)
    _check(out2, lse2, case, ctx, counts, masks)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("rows", [8, 9, 15, 16, 17, 24, 32, 33])
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_around_the_widths_of_a_unit(ext, cuda_device, dtype, rows, D):
    """Row counts about the widths that units have, whole and in pieces, alone and beside shorter requests."""
    for ctx, counts in (([5000], [rows]), ([70, 0, 300], [rows, 1, rows - 1])):
        case = _case(ctx, counts, 2, 2, D, 32, dtype, seed=rows)
        st = new_status("cuda")
        out, lse = _run(*case, ctx, counts, status=st)
        _check(out, lse, case, ctx, counts)
        _, masks, seen, _ = _trees(counts, seed=rows)
        out, lse = _run(*case, ctx, counts, mask=seen.cuda(), max_q=max(counts), status=st)
        check_status(st)
        _check(out, lse, case, ctx, counts, masks)
        again, lse2 = _run(*case, ctx, counts, mask=seen.cuda(), max_q=max(counts), status=st)
        assert torch.equal(out, again) and torch.equal(lse, lse2)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("tokens, ctx", [(5, 37), (12, 130), (30, 4000)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_values_that_are_not_finite_reach_their_rows(ext, cuda_device, dtype, tokens, ctx, D):
    """An infinite V of a new token is in the results of the rows that see it, and in no others."""
    case = _case([ctx], [tokens], 1, 1, D, 16, dtype, seed=tokens)
    q, kp, vp, table = case
    j = ctx + 2
    vp[table[0, j // 16], 0, j % 16, D - 3] = math.inf
    mask = torch.ones(tokens, tokens, dtype=torch.bool).tril()
    mask[4, 2] = False
    out, lse = _run(*case, [ctx], [tokens], mask=mask.cuda())
    sees = mask[:, 2]
    out = out.cpu()
    assert (out[sees, 0, D - 3] == math.inf).all() and torch.isfinite(out[~sees]).all()
    clean = (q, kp, vp.nan_to_num(posinf=0.0), table)
    ref, _, mag, smax = O.attention(*clean, [ctx], [tokens], [mask])
    bo, _ = O.attention_bound(ref, mag, smax, dtype, ctx + tokens, D)
    good = torch.ones(out.shape, dtype=torch.bool)
    good[sees, 0, D - 3] = False
    assert ((out.double() - ref).abs() <= bo)[good].all()


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("tokens", [10, 24, 150])
@pytest.mark.parametrize("dtype", DTYPES)
def test_scales_empty_rows_and_large_scores_at_every_width(ext, cuda_device, dtype, tokens, D):
    """Requests of few, some and many rows: any scale, rows that see nothing, scores of some hundreds."""
    ctx, counts = [90, 0, 33], [tokens, tokens - 1, 2]
    case = _case(ctx, counts, 2, 2, D, 16, dtype, seed=tokens)
    for scale in (0.03, -0.5, 0.0):
        out, lse = _run(*case, ctx, counts, scale=scale)
        _check(out, lse, case, ctx, counts, scale=scale)
    _, masks, _, _ = _trees(counts, seed=tokens)
    for m in masks:
        m[m.shape[0] // 2] = False
        m[-1] = False
    width = max(m.shape[1] for m in masks)
    masks = [torch.nn.functional.pad(m, (0, width - m.shape[1])) for m in masks]
    out, lse = _run(*case, ctx, counts, mask=torch.cat(masks).cuda())
    _check(out, lse, case, ctx, counts, masks)
    assert (lse.reshape(-1, 2)[tokens + tokens - 2] == -math.inf).all()
    case = _case(ctx, counts, 2, 2, D, 16, dtype, seed=tokens + 1, spread=40.0)
    out, lse = _run(*case, ctx, counts)
    _check(out, lse, case, ctx, counts)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_uniform_borders_scale_and_out(ext, cuda_device, dtype):
    ctx, counts = [40, 41, 7], [2, 2, 2]
    case = _case(ctx, counts, 4, 2, 64, 16, dtype, seed=2)
    big = torch.full((6, 6, 64), 5.0, dtype=dtype, device="cuda")
    out, lse = _run(*case, ctx, counts, uniform=True, scale=0.03, out=big[:, 1:5])
    _check(out, lse, case, ctx, counts, scale=0.03)
    assert (big[:, 0] == 5.0).all() and (big[:, 5] == 5.0).all()
    out, lse = _run(*case, ctx, counts, uniform=True, scale=-0.5)
    _check(out, lse, case, ctx, counts, scale=-0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_that_see_nothing(ext, cuda_device, dtype):
    """An empty mask row without context gives 0 and -inf; with context it sees the context."""
    ctx, counts = [0, 50, 0], [4, 4, 3]
    case = _case(ctx, counts, 4, 2, 128, 16, dtype, seed=3)
    masks = [torch.zeros(m, 4, dtype=torch.bool) for m in counts]
    masks[0][1, 0] = masks[2][2, 2] = masks[1][0, 3] = True
    out, lse = _run(*case, ctx, counts, mask=torch.cat(masks).cuda())
    _check(out, lse, case, ctx, counts, masks)
    narrow = [m[:, :1] for m in masks]  # columns beyond the mask are not seen
    out, lse = _run(*case, ctx, counts, mask=torch.cat(narrow).cuda())
    _check(out, lse, case, ctx, counts, narrow)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_masked_places_may_hold_anything(ext, cuda_device, dtype, bad):
    """Stale rows of the pool, and a new token that some rows see and others do not."""
    ctx, counts = [37, 130], [5, 9]
    for where in ("pool", "k", "v"):
        case = _case(ctx, counts, 4, 2, 64, 32, dtype, seed=4, fill=bad if where == "pool" else None)
        q, kp, vp, table = case
        masks = [torch.ones(m, 9, dtype=torch.bool).tril() for m in counts]
        for m in masks:
            m[4, 2] = False  # row 4 does not see token 2, row 3 does
        if where != "pool":
            for b in range(2):
                j = ctx[b] + 2
                (kp if where == "k" else vp)[table[b, j // 32], 1, j % 32, 5] = bad
        out, lse = _run(*case, ctx, counts, mask=torch.cat(masks).cuda())
        out, lse = out.cpu(), lse.cpu()
        blind = torch.tensor([t for t in range(14) if t in (0, 1, 4, 5, 6, 9)])
        keep = torch.arange(14) if where == "pool" else blind
        clean = (q, kp.nan_to_num(0.0, 0.0, 0.0), vp.nan_to_num(0.0, 0.0, 0.0), table)
        ref, rlse, mag, smax = O.attention(*clean, ctx, counts, masks)
        bo, bl = O.attention_bound(ref, mag, smax, dtype, 139, 64)
        assert ((out.double() - ref).abs() <= bo)[keep].all(), where
        assert ((lse.double() - rlse).abs() <= bl + 2.0 ** -22 * rlse.abs())[keep].all(), where
        if where == "v":  # a row that sees it has it in its own column, and only there
            seen = torch.tensor([t for t in range(14) if t not in blind.tolist()])
            got = out[seen][:, 2:].float()  # the heads of kv head 1
            assert (got[..., 5].isnan() if math.isnan(bad) else got[..., 5] == bad).all()
            rest = torch.arange(64) != 5
            assert torch.isfinite(got[..., rest]).all() and torch.isfinite(out[seen][:, :2]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_behind_the_last_request_are_left(ext, cuda_device, dtype):
    ctx, counts = [10, 20], [3, 2]
    case = _case(ctx, counts, 4, 2, 64, 16, dtype, extra=4)
    q = case[0].clone()
    q[5:] = math.nan
    out = torch.full(q.shape, 2.5, dtype=dtype, device="cuda")
    got, lse = _run(q, *case[1:], ctx, counts, out=out)
    _check(got, lse, case, ctx, counts)
    assert (out[5:] == 2.5).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_large_and_small_scores(ext, cuda_device, dtype):
    """Scores of some hundreds, where one key takes all the weight, and of zero."""
    ctx, counts = [200, 90], [4, 1]
    case = _case(ctx, counts, 4, 1, 128, 16, dtype, seed=6, spread=40.0)
    out, lse = _run(*case, ctx, counts)
    _check(out, lse, case, ctx, counts)
    zero = (case[0] * 0, *case[1:])
    out, lse = _run(*zero, ctx, counts)
    _check(out, lse, zero, ctx, counts)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_long_contexts_are_split_and_joined(ext, cuda_device, dtype):
    """One request over every SM, alone and beside short ones; a repeat gives the same bits."""
    for ctx, counts in (([9001], [1]), ([6000, 3, 1500], [9, 1, 2])):
        case = _case(ctx, counts, 4, 2, 64, 64, dtype, seed=7)
        out, lse = _run(*case, ctx, counts)
        _check(out, lse, case, ctx, counts)
        out2, lse2 = _run(*case, ctx, counts)
        assert torch.equal(out, out2) and torch.equal(lse, lse2)


@pytest.mark.gpu
def test_many_requests(ext, cuda_device):
    """More requests than threads in a block, most of them without tokens."""
    n = 700
    counts = [1 if b % 3 == 0 else 0 for b in range(n)]
    ctx = [(b * 37) % 90 for b in range(n)]
    case = _case(ctx, counts, 2, 1, 64, 16, torch.bfloat16, seed=8)
    out, lse = _run(*case, ctx, counts)
    _check(out, lse, case, ctx, counts)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_queries_and_pools(ext, cuda_device, dtype):
    """Queries that are a slice of a projection (aligned and not), a pool that is one layer's slice."""
    ctx, counts = [100], [3]
    q, kp, vp, table = _case(ctx, counts, 4, 2, 64, 16, dtype, seed=9)
    pool = torch.zeros(kp.shape[0], 2, *kp.shape[1:], dtype=dtype)
    pool[:, 0], pool[:, 1] = kp, vp
    dev = pool.cuda()
    want = tree_attention(q.cuda(), kp.cuda(), vp.cuda(), table.cuda(), torch.tensor([100], dtype=torch.int32).cuda())
    for shift in (0, 1):
        flat = torch.zeros(3, 4 * 64 + 72, dtype=dtype, device="cuda")
        flat[:, shift:shift + 256] = q.flatten(1).cuda()
        got = tree_attention(flat[:, shift:shift + 256].unflatten(1, (4, 64)), dev[:, 0], dev[:, 1],
                             table.cuda(), torch.tensor([100], dtype=torch.int32).cuda())
        assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_bad_pages_and_lengths_are_reported(ext, cuda_device, dtype):
    """A page outside the pool reads as zeros, a context longer than the table ends with it; neither faults."""
    ctx, counts = [60, 60], [2, 2]
    q, kp, vp, table = _case(ctx, counts, 2, 1, 64, 16, dtype, seed=10)
    good = table.clone()
    table[0, 1] = 10 ** 6
    table[1, 2] = -3
    st = new_status("cuda")
    out, _ = _run(q, kp, vp, table, ctx, counts, status=st)
    with pytest.raises(DeviceTimeout, match="code=2"):
        check_status(st)
    assert torch.isfinite(out).all()
    out, lse = _run(q, kp, vp, good[:, :4], [63, 2 ** 31 - 5], counts)  # the table has room for 64
    assert torch.isfinite(out).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_streams_and_graphs(ext, cuda_device, dtype):
    """Two captured calls replayed at the same time, and a call on a side stream."""
    ctx, counts = [700, 30], [3, 6]
    cases = [_case(ctx, counts, 8, 2, 128, 16, dtype, seed=s) for s in (11, 12)]
    cu = torch.tensor([0] + counts).cumsum(0).int().cuda()
    ctx_t = torch.tensor(ctx, dtype=torch.int32).cuda()
    dev = [[x.cuda() for x in c] for c in cases]
    want = [tree_attention(*d, ctx_t, cu) for d in dev]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in dev]
    graphs, outs = [], []
    for d, s in zip(dev, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(tree_attention(*d, ctx_t, cu))
        graphs.append(g)
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w)
    with torch.cuda.stream(streams[0]):
        got = tree_attention(*dev[1], ctx_t, cu)
    streams[0].synchronize()
    assert torch.equal(got, want[1])


@pytest.mark.gpu
def test_empty_call(ext, cuda_device):
    case = _case([5], [0], 2, 1, 64, 16, torch.bfloat16)
    out, lse = _run(*case, [5], [0])
    assert out.shape == (0, 2, 64) and lse.shape == (0, 2)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_replayed_call_follows_its_lengths(ext, cuda_device, dtype):
    """Lengths, borders, pages and masks are read on the GPU: one captured call serves
    every later step of the same shapes, filled in place."""
    ctx, counts = [300, 40], [5, 3]
    case = _case(ctx, counts, 4, 2, 64, 16, dtype, seed=13)
    q, kp, vp, table = (x.cuda() for x in case)
    ctx_t = torch.tensor(ctx, dtype=torch.int32).cuda()
    cu = torch.tensor([0] + counts).cumsum(0).int().cuda()
    mask = torch.zeros(8, 1, dtype=torch.int32, device="cuda")
    tree_attention(q, kp, vp, table, ctx_t, cu, mask=mask)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = tree_attention(q, kp, vp, table, ctx_t, cu, mask=mask, return_lse=True)
    for ctx2, counts2, seed in (([300, 40], [5, 3], 1), ([7, 290], [1, 7], 2), ([0, 100], [8, 0], 3)):
        _, masks, rows, _ = _trees([max(c, 1) for c in counts2], seed)
        rows = torch.cat([torch.nn.functional.pad(m[:c], (0, 32 - m.shape[1]))
                          for m, c in zip(masks, counts2)])
        ctx_t.copy_(torch.tensor(ctx2, dtype=torch.int32))
        cu.copy_(torch.tensor([0] + counts2).cumsum(0).int())
        mask.copy_(pack_mask(rows.cuda()))
        graph.replay()
        torch.cuda.synchronize()
        tab = torch.nn.functional.pad(case[3], (0, 4))
        # the table has room for the first request's 305 places in both rows
        if ctx2[1] > 40:
            table.copy_(case[3][[0, 0]])
            graph.replay()
            torch.cuda.synchronize()
            tab = tab[[0, 0]]
        _check(out, lse, (case[0], case[1], case[2], tab), ctx2, counts2,
               [m[:c, :c] for m, c in zip(masks, counts2)])
        table.copy_(case[3])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [16, 256])
def test_a_million_tokens(ext, cuda_device, dtype, page):
    """2^20 cached tokens of one request that are 2048 keys 512 times over: the outputs
    are theirs, and the sums 512 times as large."""
    keys, times, D = 2048, 512, 128
    case = _case([keys], [2], 4, 2, D, page, dtype, seed=14)
    q, kp, vp, table = case
    n = keys // page
    long = torch.cat((table[0, :n].repeat(times), table[0, n:n + 2])).view(1, -1)
    out, lse = tree_attention(q.cuda(), kp.cuda(), vp.cuda(), long.cuda(),
                              torch.tensor([keys * times], dtype=torch.int32).cuda(), return_lse=True,
                              mask=torch.zeros(2, 1, dtype=torch.bool, device="cuda"))
    blank = [torch.zeros(2, 2, dtype=torch.bool)]
    ref, rlse, mag, smax = O.attention(q, kp, vp, table, [keys], [2], blank)
    rlse = rlse + math.log(times)
    bo, bl = O.attention_bound(ref, mag, smax, dtype, keys * times, D)
    assert ((out.cpu().double() - ref).abs() <= bo).all()
    assert ((lse.cpu().double() - rlse).abs() <= bl + 2.0 ** -22 * rlse.abs()).all()
    # the sums of so many keys are bounded loosely; a wrong key would show here
    assert ((out.cpu().double() - ref).abs().max() <= (2.0 ** -16 + 2 * O.half_step(dtype)) * mag.max())


@pytest.mark.gpu
def test_pools_past_two_to_the_31(ext, cuda_device):
    """Pages whose elements lie beyond 2^31: written, copied, compacted and attended to."""
    from ring_attention_benchmark_b200.ops.paged import append_kv, compact_path, copy_pages

    pages, Hk, page, D = 33000, 8, 128, 64  # 2.16e9 elements, 4.3 GB a pool
    kp = torch.empty(pages, Hk, page, D, dtype=torch.bfloat16, device="cuda")
    vp = torch.empty_like(kp)
    ids = [pages - 1, 5, pages - 7, pages - 2]
    q, k, v = (torch.randn(300, h, D, generator=torch.Generator().manual_seed(h)).bfloat16() for h in (8, 8, 8))
    v = v + 1
    table = torch.tensor([ids[:3]], dtype=torch.int32).cuda()
    zero = torch.zeros(1, dtype=torch.int32).cuda()
    append_kv(k.cuda(), v.cuda(), kp, vp, table, zero)
    copy_pages(kp, vp, [ids[2]], [ids[3]])
    table[0, 2] = ids[3]
    ctx = torch.tensor([290], dtype=torch.int32).cuda()
    compact_path(kp, vp, table, ctx, torch.tensor([[2, 5, 9]], dtype=torch.int32).cuda(),
                 torch.tensor([3], dtype=torch.int32).cuda())
    out, lse = tree_attention(q[:1].cuda(), kp, vp, table, torch.tensor([292], dtype=torch.int32).cuda(),
                              return_lse=True)
    keep = list(range(290)) + [292, 295, 299]
    one = lambda x: x[keep].permute(1, 0, 2).reshape(1, Hk, len(keep), D)  # noqa: E731
    ref, rlse, mag, smax = O.attention(q[:1], one(k), one(v), torch.zeros(1, 1, dtype=torch.int32), [292], [1])
    bo, bl = O.attention_bound(ref, mag, smax, torch.bfloat16, 293, D)
    assert ((out.cpu().double() - ref).abs() <= bo).all()
    assert ((lse.cpu().double() - rlse).abs() <= bl + 2.0 ** -22 * rlse.abs()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_an_event_between_overlapped_launches_is_waited_for(ext, cuda_device, dtype):
    """A launch may start while its predecessor in the stream runs, but not before an
    event of another stream that it was told to wait for."""
    from ring_attention_benchmark_b200.ops.paged import append_kv, copy_pages

    ctx, counts = [150], [4]
    q, kp, vp, table = (x.cuda() for x in _case(ctx, counts, 4, 2, 64, 16, dtype, seed=15))
    ctx_t = torch.tensor(ctx, dtype=torch.int32).cuda()
    want = tree_attention(q, kp, vp, table, ctx_t)
    side, main = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        late, pool = torch.zeros_like(q), torch.zeros_like(kp)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(2_000_000)  # about a millisecond
            late.copy_(q)
            pool.copy_(kp)
            ready = side.record_event()
        with torch.cuda.stream(main):
            copy_pages(kp, vp, [], [])
            scratch = torch.zeros_like(kp)
            append_kv(torch.zeros(4, 2, 64, dtype=dtype, device="cuda"),
                      torch.zeros(4, 2, 64, dtype=dtype, device="cuda"), scratch,
                      torch.zeros_like(vp), table, ctx_t)
            main.wait_event(ready)
            got = tree_attention(late, pool, vp, table, ctx_t)
            late.zero_()  # an ordinary launch behind the overlapped ones
        torch.cuda.synchronize()
        assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 12, 40, 150])
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_bad_request_leaves_the_others_whole(ext, cuda_device, dtype, tokens):
    """A page outside the pool and a context longer than its table are reported, and every
    row of the healthy request beside them is right; so is a later call that is given the
    status word with the report still in it."""
    ctx, counts = [60, 60, 3000], [tokens, 1, tokens]
    case = _case(ctx, counts, 2, 1, 64, 16, dtype, seed=20)
    q, kp, vp, table = case
    broken = table.clone()
    broken[0, 1] = 10 ** 6
    at = torch.tensor(ctx, dtype=torch.int32)
    at[1] = 2 ** 31 - 7
    cu = torch.tensor([0] + counts).cumsum(0).int().cuda()
    ref, rlse, mag, smax = O.attention(q, kp, vp, table, ctx, counts)
    bo, bl = O.attention_bound(ref, mag, smax, dtype, 3000 + tokens, 64)
    st = new_status("cuda")
    good = slice(sum(counts[:2]), None)
    for tab, lens, rows in ((broken, at, good), (table, torch.tensor(ctx, dtype=torch.int32), slice(None))):
        out = torch.full(q.shape, 77.0, dtype=dtype, device="cuda")
        got, lse = tree_attention(q.cuda(), kp.cuda(), vp.cuda(), tab.cuda(), lens.cuda(), cu, out=out,
                                  max_q=tokens, return_lse=True, status=st)
        with pytest.raises(DeviceTimeout, match="code=2"):
            check_status(st)
        assert ((got.cpu().double() - ref).abs() <= bo)[rows].all()
        assert ((lse.cpu().double() - rlse).abs() <= bl + 2.0 ** -22 * rlse.abs())[rows].all()
        assert (got != 77.0).any(-1).all()  # every row was written


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 3, 12, 40, 150])
@pytest.mark.parametrize("dtype", DTYPES)
def test_queries_at_odd_places_in_memory(ext, cuda_device, dtype, tokens):
    """Contiguous queries whose first element is not on a 16-byte boundary, and rows cut from
    a wider tensor at every offset, give what aligned ones give."""
    ctx, H, D = [100], 2, 64
    q, kp, vp, table = (x.cuda() for x in _case(ctx, [tokens], H, 2, D, 16, dtype, seed=40))
    ctx_t = torch.tensor(ctx, dtype=torch.int32).cuda()
    want = tree_attention(q, kp, vp, table, ctx_t)
    n = q.numel()
    for shift in range(1, 9):
        flat = torch.zeros(n + 16, dtype=dtype, device="cuda")
        at = flat[shift:shift + n].view(tokens, H, D)
        at.copy_(q)
        assert at.is_contiguous()
        assert torch.equal(tree_attention(at, kp, vp, table, ctx_t), want)
        wide = torch.zeros(tokens, H * D + 16, dtype=dtype, device="cuda")
        rows = wide[:, shift:shift + H * D].unflatten(1, (H, D))
        rows.copy_(q)
        assert torch.equal(tree_attention(rows, kp, vp, table, ctx_t), want)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_pieces_of_one_tile_behind_longer_ones(ext, cuda_device, dtype, D):
    """Units of many tiles and of one in turn, on every SM: a piece's results take both
    chains' halves, whatever the next piece has.  Repeats give the same bits."""
    n = 600
    counts = [20 + b % 3 for b in range(n)]
    ctx = [(700, 5, 60, 1300, 0)[b % 5] for b in range(n)]
    some = list(range(0, n, 37))
    T, page = sum(counts), 64
    g = torch.Generator().manual_seed(41)
    q = torch.randn(T, 1, D, generator=g).to(dtype)
    kp, vp = (torch.randn(50, 1, page, D, generator=g).to(dtype) for _ in "kv")
    table = torch.randint(0, 50, (n, 22), generator=g, dtype=torch.int32)  # pages are shared and only read
    first = [0]
    for c in counts:
        first.append(first[-1] + c)
    got = [_run(q, kp, vp, table, ctx, counts, max_q=22) for _ in range(3)]
    for out, lse in got[1:]:
        assert torch.equal(out, got[0][0]) and torch.equal(lse, got[0][1])
    out, lse = got[0]
    for b in some:
        rows = slice(first[b], first[b + 1])
        _check(out[rows], lse[rows], (q[rows], kp, vp, table[b:b + 1]), [ctx[b]], [counts[b]])


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 12, 40, 150])
@pytest.mark.parametrize("dtype", DTYPES)
def test_split_units_of_every_request_are_joined(ext, cuda_device, dtype, tokens):
    """Whichever request of a batch the SMs share out, its pieces are joined: the long one
    stands first, in the middle and last, behind requests without tokens too."""
    for at in (0, 2, 5):
        ctx = [2500 if b == at else 9 * b for b in range(6)]
        counts = [0 if b == 1 else tokens if b == at else 1 for b in range(6)]
        case = _case(ctx, counts, 1, 1, 64, 64, dtype, seed=42 + at)
        out, lse = _run(*case, ctx, counts, max_q=tokens)
        _check(out, lse, case, ctx, counts)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("tokens", [1, 12, 24, 150])
@pytest.mark.parametrize("dtype", DTYPES)
def test_infinities_among_the_cached_keys(ext, cuda_device, dtype, tokens, D):
    """An infinite V of a cached key is in its own column of every row's result; an infinite
    K takes all weight from its key where the product is -inf, and makes the row NaN where
    it is +inf.  Everything else is as without them."""
    ctx, at, col = 500, (40, 333), 7
    case = _case([ctx], [tokens], 1, 1, D, 16, dtype, seed=30 + tokens)
    q, kp, vp, table = case
    ref, _, mag, smax = O.attention(*case, [ctx], [tokens])
    bo, _ = O.attention_bound(ref, mag, smax, dtype, ctx + tokens, D)
    rest = torch.arange(D) != col
    for signs, want in (((1, 1), math.inf), ((-1, -1), -math.inf), ((1, -1), math.nan)):
        bad = vp.clone()
        for j, s in zip(at, signs):
            bad[table[0, j // 16], 0, j % 16, col] = s * math.inf
        got = _run(q, kp, bad, table, [ctx], [tokens])[0].cpu().double()
        assert ((got - ref).abs() <= bo)[..., rest].all()
        c = got[..., col]
        assert (c.isnan() if math.isnan(want) else c == want).all()
    bad = kp.clone()
    for j in at:
        bad[table[0, j // 16], 0, j % 16, col] = math.inf
    got, lse = (x.cpu().double() for x in _run(q, bad, vp, table, [ctx], [tokens]))
    low = q[:, 0, col] < 0
    assert got[~low].isnan().all() and lse[~low].isnan().all()
    ref2, rlse2, mag2, _ = O.attention(q, bad, vp, table, [ctx], [tokens])
    bo2, bl2 = O.attention_bound(ref2, mag2, smax, dtype, ctx + tokens, D)  # sizes of the finite scores
    assert ((got - ref2).abs() <= bo2)[low].all()
    assert ((lse - rlse2).abs() <= bl2 + 2.0 ** -22 * rlse2.abs())[low].all()


@pytest.mark.gpu
@pytest.mark.parametrize("tokens, n", [(1, 1 << 20), (12, 1 << 18), (20, 1 << 17), (130, 1 << 17)])
def test_many_small_weights_in_fp16(ext, cuda_device, tokens, n):
    """Keys whose weights lie 2^-26 below the largest add up over a long context.

    As many requests as there are SMs, so that hardly a unit is cut; all share the same pages:
    first one whose keys j % 16 == 0 score 0 with a V of zero, then the same page over and
    over, of keys that score -18 with a V of one.  A weight below 2^-14 is held to steps of
    2^-24, after a factor of 2^7 at least over the row's largest: off by 2^-32 of that each,
    n of them over a sum of 8.  fp32 sums: n terms of 2^-24 relative, and the exponential 2^-21.
    """
    D, page, few = 64, 128, 8
    batch = torch.cuda.get_device_properties(0).multi_processor_count
    kp, vp = torch.zeros(3, 1, page, D).half(), torch.zeros(3, 1, page, D).half()
    kp[:2, 0, :, 0] = -18.0
    kp[0, 0, ::16, 0] = 0.0
    vp[:2] = 1.0
    vp[0, 0, ::16] = 0.0
    table = torch.ones(n // page + 2, dtype=torch.int32)
    table[0], table[-2:] = 0, 2
    q = torch.zeros(batch * tokens, 1, D).half()
    q[..., 0] = 1.0
    ctx = torch.full((batch,), n, dtype=torch.int32)
    blank = torch.zeros(batch * tokens, 1, dtype=torch.bool)
    out, lse = tree_attention(q.cuda(), kp.cuda(), vp.cuda(), table.cuda().expand(batch, -1), ctx.cuda(),
                              mask=blank.cuda(), scale=1.0, return_lse=True)
    small = (n - few) * math.exp(-18.0)
    want = small / (few + small)
    tol = want * (O.half_step(torch.float16) * 2 + n * 2.0 ** -24 + 2.0 ** -20) + n * 2.0 ** -32 / few
    assert tol < want / 4
    assert (out.cpu().double() - want).abs().max().item() <= tol
    assert (lse.cpu().double() - math.log(few + small)).abs().max().item() <= n * 2.0 ** -24 + 2.0 ** -20


def test_outputs_that_overlap_are_refused(ext):
    a = _args()
    wide = torch.zeros(2, 8, 64)
    for q, out, what in ((a["q"], a["q"], "CUDA"), (wide[:, :4], wide[:, 4:], "CUDA"),
                         (wide[:, :4], wide[:, 2:6], "out shares memory with q"),
                         (a["q"], a["k_pages"][0, 0, :8].view(2, 4, 64), "with k_pages"),
                         (a["q"], a["v_pages"][1, 0, :8].view(2, 4, 64), "with v_pages")):
        with pytest.raises(RuntimeError, match=what):
            tree_attention(**dict(a, q=q, out=out))


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 12, 40, 150])
@pytest.mark.parametrize("dtype", DTYPES)
def test_the_result_may_take_the_place_of_the_queries(ext, cuda_device, dtype, tokens):
    ctx, counts = [900, 3], [tokens, tokens]
    q, kp, vp, table = (x.cuda() for x in _case(ctx, counts, 4, 2, 64, 16, dtype, seed=43))
    ctx_t = torch.tensor(ctx, dtype=torch.int32).cuda()
    want = tree_attention(q, kp, vp, table, ctx_t)
    assert torch.equal(tree_attention(q, kp, vp, table, ctx_t, out=q), want) and torch.equal(q, want)


@pytest.mark.parametrize("scale", [1e39, -1e300, 3e38, math.inf])
def test_scales_beyond_fp32_are_refused(ext, scale):
    """Scores are scaled in fp32, in base-2 units; a scale that is infinite there gives NaN."""
    with pytest.raises(RuntimeError, match="scale must be finite"):
        tree_attention(**_args(scale=scale))


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 12, 20, 130])
@pytest.mark.parametrize("step", [1, 2, 4, 8, 16])
@pytest.mark.parametrize("dtype", DTYPES)
def test_scores_that_fp32_holds_in_whole_steps(ext, cuda_device, dtype, step, tokens):
    """Scores of 1.25 * 2^23 * step in base-2 units, which fp32 holds to a step, and 16 to 48
    more from tile to tile: weights are powers of two whatever the running maximum.

    The scores are exact, so are their distances; the exponential is good to 2^-21, the sums
    to 2^-24 a term, and a weight that is 2^-16 of the largest or more is exact in every type.
    """
    D, page, n = 64, 128, 40 * 128
    g = torch.Generator().manual_seed(step)
    more = torch.randint(0, 4, (n // page,), generator=g) * 16
    more[0], more[-1] = 0, 48
    kp, vp = torch.zeros(n // page + 2, 1, page, D), torch.randn(n // page + 2, 1, page, D, generator=g)
    kp[:-2, 0, :, 0], kp[:-2, 0, :, 1] = 2048.0 * step, more[:, None].float()
    vp = vp.to(dtype)
    q = torch.zeros(tokens, 1, D)
    q[:, 0, 0], q[:, 0, 1] = 5120.0, 1.0
    table = torch.arange(n // page + 2, dtype=torch.int32).view(1, -1)
    out, lse = tree_attention(q.to(dtype).cuda(), kp.to(dtype).cuda(), vp.cuda(), table.cuda(),
                              torch.tensor([n], dtype=torch.int32).cuda(), scale=math.log(2.0),
                              mask=torch.zeros(tokens, 1, dtype=torch.bool, device="cuda"), return_lse=True)
    w = torch.exp2((more - 48).double()).repeat_interleave(page)
    v = vp[:-2, 0].reshape(n, D).double()
    want, mag = w @ v / w.sum(), w @ v.abs() / w.sum()
    tol = mag * (2.0 ** -20 + n * 2.0 ** -23) + O.half_step(dtype) * want.abs()
    # weights 2^-32 and 2^-48 below the largest may vanish in 16 bits: their share is below 2^-31
    assert ((out.cpu().double()[:, 0] - want).abs() <= tol + 2.0 ** -31 * 8).all()
    ref = (5120.0 * 2048.0 * step + 48 + math.log2(w.sum().item())) * math.log(2.0)
    assert (lse.cpu().double() - ref).abs().max().item() <= 2 * 2.0 ** -24 * ref + 2.0 ** -20


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_one_row_of_an_odd_stride(ext, cuda_device, dtype):
    """A single token or head may be a slice of any width, queries and results alike."""
    from ring_attention_benchmark_b200.ops.rotary import apply_rotary, rotary_frequencies

    ctx, D = [40], 64
    for T, H in ((1, 4), (3, 1), (1, 1)):
        q, kp, vp, table = (x.cuda() for x in _case(ctx, [T], H, 1, D, 16, dtype, seed=44))
        ctx_t = torch.tensor(ctx, dtype=torch.int32).cuda()
        want = tree_attention(q, kp, vp, table, ctx_t)
        pos, inv = torch.arange(T).cuda(), rotary_frequencies(D)[0].cuda()
        turned = apply_rotary(q, None, pos, inv)
        for st, sh in ((H * D + 1, D), (H * D + 8, D + 1)):
            if (T > 1 and st % 8) or (H > 1 and sh % 8):
                continue
            flat_q, flat_o = (torch.full((T * st + 64 * H,), 3.0, dtype=dtype, device="cuda") for _ in "qo")
            odd, out = (x.as_strided((T, H, D), (st, sh, 1)) for x in (flat_q, flat_o))
            odd.copy_(q)
            assert torch.equal(tree_attention(odd, kp, vp, table, ctx_t, out=out), want) and torch.equal(out, want)
            apply_rotary(odd, None, pos, inv, out=(out, None))
            assert torch.equal(out, turned)
            left = torch.ones(flat_o.numel(), dtype=torch.bool, device="cuda")
            left.as_strided((T, H, D), (st, sh, 1)).fill_(False)
            assert (flat_o[left] == 3.0).all()
