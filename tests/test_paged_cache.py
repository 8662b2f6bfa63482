"""Writing, copying and compacting pages of a cache, against plain 64-bit indexing."""
import pytest
import torch

import _paged_oracle as O
from ring_attention_benchmark_b200.ops.attention import DeviceTimeout, check_status, new_status
from ring_attention_benchmark_b200.ops.paged import append_kv, compact_path, copy_pages
from ring_attention_benchmark_b200.ops.rotary import rotary_frequencies

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _pool(pages, hk, page, d, dtype, seed=0, layers=None):
    g = torch.Generator().manual_seed(seed)
    shape = (pages, hk, page, d) if layers is None else (layers, pages, hk, page, d)
    return torch.randn(shape, generator=g).to(dtype), torch.randn(shape, generator=g).to(dtype)


def _table(lens, page, seed=0, width=None):
    """Shuffled pages, unused entries -1."""
    need = [-(-n // page) for n in lens]
    order = torch.randperm(sum(need) + 2, generator=torch.Generator().manual_seed(seed)).tolist()
    t = torch.full((len(lens), width or max(max(need), 1)), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        for i in range(n):
            t[b, i] = order.pop()
    return t, sum(need) + 2


def _cu(counts):
    return torch.tensor([0] + counts).cumsum(0).int()


# ------------------------------------------------------------------ refusals (CPU)
def _append_args(**kw):
    kp, vp = _pool(4, 2, 16, 64, torch.float32)
    a = dict(k=torch.zeros(3, 2, 64), v=torch.zeros(3, 2, 64), k_pages=kp, v_pages=vp,
             block_table=torch.zeros(1, 2, dtype=torch.int32),
             context_lens=torch.zeros(1, dtype=torch.int32))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw, what", [
    (dict(), "CUDA"),
    (dict(k=torch.zeros(3, 2, 32), v=torch.zeros(3, 2, 32)), "for this cache"),
    (dict(v=torch.zeros(3, 1, 64)), "k's shape"),
    (dict(k=torch.zeros(3, 2, 64).half(), v=torch.zeros(3, 2, 64).half()), "share a dtype"),
    (dict(k_pages=torch.zeros(4, 2, 64)), "k_pages must be"),
    (dict(k_pages=torch.zeros(1, 4, 2, 16, 64), v_pages=torch.zeros(1, 4, 2, 16, 64)), "k_pages must be"),
    (dict(v_pages=torch.zeros(4, 2, 32, 64)), "k_pages' shape"),
    (dict(k_pages=torch.zeros(4, 16, 2, 64).transpose(1, 2)), "contiguous"),
    (dict(v_pages=torch.zeros(1, 2, 16, 64).expand(4, 2, 16, 64)), "shares memory"),
    (dict(block_table=torch.zeros(2, 2, dtype=torch.int32)), "rows"),
    (dict(block_table=torch.zeros(1, 2)), "int32"),
    (dict(block_table=torch.zeros(1, 0, dtype=torch.int32)), "no columns"),
    (dict(context_lens=torch.zeros(0, dtype=torch.int32)), "empty"),
    (dict(context_lens=torch.zeros(2, dtype=torch.int32), block_table=torch.zeros(2, 2, dtype=torch.int32)), "evenly"),
    (dict(cu_q=torch.zeros(3, dtype=torch.int32)), "cu_q"),
    (dict(positions=torch.arange(3)), "no use"),
    (dict(q=torch.zeros(3, 4, 64)), "no use"),
    (dict(q=torch.zeros(2, 4, 64), inv_freq=rotary_frequencies(64)[0]), "same tokens"),
    (dict(inv_freq=rotary_frequencies(66)[0]), "head dim"),
    (dict(status=torch.zeros(4, dtype=torch.int32)), "CUDA"),
])
def test_append_refusals(ext, kw, what):
    with pytest.raises(RuntimeError, match=what):
        append_kv(**_append_args(**kw))


@pytest.mark.parametrize("src, dst, what", [
    ([0], [1], "CUDA"),
    ([0, 1], [2], "names 2 pages, dst 1"),
    ([0, 1], [2, 2], "twice"),
    ([0], [0], "both in src and in dst"),
    ([0, 2], [2, 3], "both in src and in dst"),
    ([4], [0], "no page"),
    ([-1], [0], "no page"),
    ([0], [4], "no page"),
    ([0], [-1], "no page"),
    (torch.tensor([0.0]), [1], "int32 or int64"),
    (torch.tensor([[0]]), [1], "int32 or int64"),
])
def test_copy_refusals(ext, src, dst, what):
    kp, vp = _pool(4, 2, 16, 64, torch.float32)
    with pytest.raises(RuntimeError, match=what):
        copy_pages(kp, vp, src, dst)


@pytest.mark.parametrize("kw, what", [
    (dict(), "CUDA"),
    (dict(path=torch.zeros(2, 3, dtype=torch.int32)), "a row for each"),
    (dict(path=torch.zeros(1, 3)), "int32"),
    (dict(path_lens=torch.zeros(2, dtype=torch.int32)), "a row for each"),
    (dict(path=torch.zeros(3, 1, dtype=torch.int32).t().expand(1, 3)[:, ::2]), "contiguous"),
])
def test_compact_refusals(ext, kw, what):
    kp, vp = _pool(4, 2, 16, 64, torch.float32)
    a = dict(k_pages=kp, v_pages=vp, block_table=torch.zeros(1, 2, dtype=torch.int32),
             context_lens=torch.zeros(1, dtype=torch.int32),
             path=torch.zeros(1, 3, dtype=torch.int32), path_lens=torch.ones(1, dtype=torch.int32))
    a.update(kw)
    with pytest.raises(RuntimeError, match=what):
        compact_path(**a)


# ------------------------------------------------------------------ append (GPU)
def _append_oracle(k, v, kp, vp, table, ctx, counts, inv=None, inter=False, positions=None):
    """The pools after the call in 64 bits, and which rows were written from which token."""
    at = torch.cat([torch.arange(c, c + m) for c, m in zip(ctx, counts)])
    pos = at if positions is None else positions
    n = at.numel()
    kr = O.rotate(k[:n], pos[:n], inv, inter) if inv is not None else k[:n].double()
    ko, vo = kp.double().clone(), vp.double().clone()
    page, first = kp.shape[2], 0
    for b, m in enumerate(counts):
        for i in range(m):
            p = int(at[first + i])
            ko[table[b, p // page], :, p % page] = kr[first + i]
            vo[table[b, p // page], :, p % page] = v[first + i].double()
        first += m
    return ko, vo, pos


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("ctx, counts, H, Hk, D, page, r", [
    ([0], [1], 1, 1, 64, 16, 64),
    ([5, 0, 31, 16], [1, 0, 3, 33], 8, 2, 128, 16, 64),
    ([100, 7, 0], [0, 17, 0], 3, 3, 64, 32, 32),
    ([3, 15], [20, 1], 6, 2, 80, 5, 10),
    ([0, 9, 2, 700], [1200, 0, 1, 1700], 2, 1, 64, 16, 32),  # many tokens of few heads
])
def test_append_values(ext, cuda_device, dtype, inter, ctx, counts, H, Hk, D, page, r):
    T, extra = sum(counts), 2
    g = torch.Generator().manual_seed(4)
    q, k, v = (torch.randn(T + extra, h, D, generator=g).to(dtype) for h in (H, Hk, Hk))
    table, pages = _table([c + m for c, m in zip(ctx, counts)], page)
    kp, vp = _pool(pages, Hk, page, D, dtype)
    inv = rotary_frequencies(r)[0]
    kd, vd = kp.cuda(), vp.cuda()
    st = new_status("cuda")
    q_out = torch.full(q.shape, 9.0, dtype=dtype, device="cuda")
    ctx_t = torch.tensor(ctx, dtype=torch.int32)
    got = append_kv(k.cuda(), v.cuda(), kd, vd, table.cuda(), ctx_t.cuda(), _cu(counts).cuda(),
                    inv_freq=inv.cuda(), interleaved=inter, q=q.cuda(), q_out=q_out, status=st)
    check_status(st)
    assert got.data_ptr() == q_out.data_ptr()
    ko, vo, pos = _append_oracle(k, v, kp, vp, table, ctx, counts, inv, inter)
    assert torch.equal(vd.cpu().double(), vo)
    bound = O.rotate_bound(k[:T], inv, inter, 1.0, dtype, pos).amax() if T else 0.0
    assert (kd.cpu().double() - ko).abs().max() <= bound
    untouched = ko == kp.double()
    assert torch.equal(kd.cpu()[untouched].double(), kp[untouched].double()) or bool(
        ((kd.cpu().double() - ko).abs() <= bound)[untouched].all())
    d = (got[:T].cpu().double() - O.rotate(q[:T], pos, inv, inter)).abs()
    assert (d <= O.rotate_bound(q[:T], inv, inter, 1.0, dtype, pos)).all()
    assert (got[T:] == 9.0).all()  # rows behind the last request


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_append_without_rotation_and_with_positions(ext, cuda_device, dtype):
    ctx, counts, Hk, D, page = [4, 40], [3, 3], 2, 64, 16
    g = torch.Generator().manual_seed(6)
    k, v = (torch.randn(6, Hk, D, generator=g).to(dtype) for _ in "kv")
    table, pages = _table([7, 43], page, width=9)
    kp, vp = _pool(pages, Hk, page, D, dtype)
    ctx_t = torch.tensor(ctx, dtype=torch.int32).cuda()
    kd, vd = kp.cuda(), vp.cuda()
    assert append_kv(k.cuda(), v.cuda(), kd, vd, table.cuda(), ctx_t) is None  # 3 tokens each
    ko, vo, _ = _append_oracle(k, v, kp, vp, table, ctx, counts)
    assert torch.equal(kd.cpu().double(), ko) and torch.equal(vd.cpu().double(), vo)
    pos = torch.tensor([4, 5, 5, 40, 41, 41])  # a tree's tokens share depths
    inv = rotary_frequencies(64)[0]
    kd, vd = kp.cuda(), vp.cuda()
    append_kv(k.cuda(), v.cuda(), kd, vd, table.cuda(), ctx_t, positions=pos.cuda(), inv_freq=inv.cuda())
    ko, vo, _ = _append_oracle(k, v, kp, vp, table, ctx, counts, inv, False, pos)
    assert (kd.cpu().double() - ko).abs().max() <= O.rotate_bound(k, inv, False, 1.0, dtype, pos).amax()
    assert torch.equal(vd.cpu().double(), vo)


@pytest.mark.gpu
def test_append_skips_and_reports_bad_places(ext, cuda_device):
    """A page outside the pool and a place outside the table are skipped, the rest is written."""
    Hk, D, page = 1, 64, 16
    k, v = torch.randn(3, Hk, D), torch.randn(3, Hk, D)
    kp, vp = _pool(3, Hk, page, D, torch.float32)
    table = torch.tensor([[0], [7], [1]], dtype=torch.int32)
    ctx = torch.tensor([2, 2, 16], dtype=torch.int32)  # the last lies behind its table
    kd, vd = kp.cuda(), vp.cuda()
    st = new_status("cuda")
    append_kv(k.cuda(), v.cuda(), kd, vd, table.cuda(), ctx.cuda(), status=st)
    with pytest.raises(DeviceTimeout, match="code=2"):
        check_status(st)
    kp[0, :, 2], vp[0, :, 2] = k[0], v[0]
    assert torch.equal(kd.cpu(), kp) and torch.equal(vd.cpu(), vp)


@pytest.mark.gpu
def test_append_of_many_tokens_skips_bad_places(ext, cuda_device):
    """As above where one block holds many tokens: q is turned all the same."""
    T, D, page = 2400, 64, 16
    g = torch.Generator().manual_seed(8)
    q, k, v = (torch.randn(T + 3, 1, D, generator=g) for _ in range(3))
    inv = rotary_frequencies(64)[0]
    kp, vp = _pool(200, 1, page, D, torch.float32)
    table = torch.arange(140).int().view(1, 140).clone()  # room for 2240 places
    table[0, 7] = 200
    kd, vd = kp.cuda(), vp.cuda()
    st = new_status("cuda")
    qo = torch.full_like(q, 4.0).cuda()
    append_kv(k.cuda(), v.cuda(), kd, vd, table.cuda(), torch.zeros(1, dtype=torch.int32).cuda(),
              _cu([T]).cuda(), inv_freq=inv.cuda(), q=q.cuda(), q_out=qo, status=st)
    with pytest.raises(DeviceTimeout, match="code=2"):
        check_status(st)
    pos = torch.arange(T)
    assert ((qo[:T].cpu().double() - O.rotate(q[:T], pos, inv, False)).abs()
            <= O.rotate_bound(q[:T], inv, False, 1.0, torch.float32, pos)).all()
    assert (qo[T:] == 4.0).all()
    kept = [i for i in range(2240) if i // page != 7]
    vp[torch.tensor(kept) // page, 0, torch.tensor(kept) % page] = v[kept, 0]
    assert torch.equal(vd.cpu(), vp)


# ------------------------------------------------------------------ copies (GPU)
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layers", [None, 3])
@pytest.mark.parametrize("hk, page, d", [(1, 1, 8), (2, 16, 64), (8, 16, 128), (5, 48, 72)])
def test_copy_pages(ext, cuda_device, dtype, layers, hk, page, d):
    kp, vp = _pool(9, hk, page, d, dtype, layers=layers)
    kd, vd = kp.cuda(), vp.cuda()
    src, dst = [3, 3, 8, 0], [1, 7, 2, 5]
    copy_pages(kd, vd, src, dst)
    for x, got in ((kp, kd), (vp, vd)):
        ref = x.clone()
        ref[..., dst, :, :, :] = x[..., src, :, :, :]
        assert torch.equal(got.cpu(), ref)


@pytest.mark.gpu
def test_copy_many_pages_and_strided_pools(ext, cuda_device):
    """More pairs than one launch takes, in a pool whose K and V share a tensor."""
    pool = torch.randn(2, 2, 2600, 1, 1, 16, device="cuda").half()  # layers, K and V, pages
    ref = pool.clone()
    order = torch.randperm(2600, generator=torch.Generator().manual_seed(1))
    src, dst = order[:1234], order[1300:2534].int()
    copy_pages(pool[:, 0], pool[:, 1], src, dst)
    ref[:, :, dst.long()] = ref[:, :, src]
    assert torch.equal(pool, ref)
    copy_pages(pool[:, 0], pool[:, 1], [], [])
    assert torch.equal(pool, ref)


@pytest.mark.gpu
def test_captured_copy(ext, cuda_device):
    kp, vp = (x.cuda() for x in _pool(4, 1, 16, 64, torch.float16))
    copy_pages(kp, vp, [0], [1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        copy_pages(kp, vp, [2], [3])
    kp[2].fill_(3.0)
    graph.replay()
    torch.cuda.synchronize()
    assert (kp[3] == 3.0).all() and torch.equal(vp[3], vp[2])


# ------------------------------------------------------------------ accepted path (GPU)
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layers", [None, 2])
@pytest.mark.parametrize("hk, page, d", [(1, 16, 64), (8, 16, 128), (3, 32, 64), (2, 7, 24)])
def test_compact_path(ext, cuda_device, dtype, layers, hk, page, d):
    ctx = [0, 15, 16, 100, 3, 9]
    paths = [[0], [1, 3], [0, 1, 2, 3], list(range(0, 40, 2)), [], [31]]
    w = max(len(p) for p in paths)
    path = torch.full((len(ctx), w), -5, dtype=torch.int32)
    for b, p in enumerate(paths):
        path[b, :len(p)] = torch.tensor(p, dtype=torch.int32)
    lens = torch.tensor([len(p) for p in paths], dtype=torch.int32)
    table, pages = _table([c + 40 for c in ctx], page)
    kp, vp = _pool(pages, hk, page, d, dtype, layers=layers)
    kd, vd = kp.cuda(), vp.cuda()
    st = new_status("cuda")
    compact_path(kd, vd, table.cuda(), torch.tensor(ctx, dtype=torch.int32).cuda(), path.cuda(),
                 lens.cuda(), status=st)
    check_status(st)
    for x, got in ((kp, kd), (vp, vd)):
        ref = x.clone()
        for b, p in enumerate(paths):
            for i, j in enumerate(p):
                s, t = ctx[b] + j, ctx[b] + i
                ref[..., table[b, t // page], :, t % page, :] = x[..., table[b, s // page], :, s % page, :]
        assert torch.equal(got.cpu(), ref)


@pytest.mark.gpu
@pytest.mark.parametrize("path, n, ctx, table", [
    ([2, 2, 3], 3, 0, [0, 1]),      # the same place twice
    ([3, 1, 4], 3, 0, [0, 1]),      # not increasing
    ([-1, 1, 2], 3, 0, [0, 1]),
    ([1, 2, 3], 4, 0, [0, 1]),      # longer than its row
    ([1, 2, 40], 3, 0, [0, 1]),     # behind the table
    ([1, 2, 3], 3, 14, [0, 5]),     # no such page
    ([1, 2, 3], 3, -1, [0, 1]),
])
def test_compact_reports_bad_paths_and_moves_nothing(ext, cuda_device, path, n, ctx, table):
    kp, vp = _pool(3, 1, 16, 64, torch.float32)
    kd, vd = kp.cuda(), vp.cuda()
    st = new_status("cuda")
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    compact_path(kd, vd, i32([table]), i32([ctx]), i32([path]), i32([n]), status=st)
    with pytest.raises(DeviceTimeout, match="code=2"):
        check_status(st)
    assert torch.equal(kd.cpu(), kp) and torch.equal(vd.cpu(), vp)


@pytest.mark.gpu
def test_written_tensors_change_their_version(ext, cuda_device):
    """Pools and outputs that a call writes count as changed in place."""
    from ring_attention_benchmark_b200.ops.paged import tree_attention

    kp, vp = (x.cuda() for x in _pool(4, 1, 16, 64, torch.float16))
    table = torch.tensor([[0, 1]], dtype=torch.int32).cuda()
    ctx = torch.tensor([3], dtype=torch.int32).cuda()
    q, k, v = (torch.randn(2, 1, 64, device="cuda").half() for _ in range(3))
    path, n = torch.tensor([[1]], dtype=torch.int32).cuda(), torch.tensor([1], dtype=torch.int32).cuda()
    out = torch.empty_like(q)
    for call, written in (
            (lambda: append_kv(k, v, kp, vp, table, ctx, inv_freq=rotary_frequencies(64)[0].cuda(), q=q, q_out=out),
             (kp, vp, out)),
            (lambda: copy_pages(kp, vp, [0], [2]), (kp, vp)),
            (lambda: compact_path(kp, vp, table, ctx, path, n), (kp, vp)),
            (lambda: tree_attention(q, kp, vp, table, ctx, out=out), (out,))):
        before = [t._version for t in written]
        call()
        assert all(t._version > x for t, x in zip(written, before))


def test_written_tensors_that_learn_are_refused(ext):
    """Writing past autograd into a tensor that requires a gradient is refused, as torch does."""
    kp, vp = _pool(4, 2, 16, 64, torch.float32)
    one = torch.ones(1, dtype=torch.int32)
    for a, b in ((kp.clone().requires_grad_(), vp), (kp, vp.clone().requires_grad_())):
        with pytest.raises(RuntimeError, match="require a gradient"):
            append_kv(**_append_args(k_pages=a, v_pages=b))
        with pytest.raises(RuntimeError, match="require a gradient"):
            copy_pages(a, b, [0], [1])
        with pytest.raises(RuntimeError, match="require a gradient"):
            compact_path(a, b, torch.zeros(1, 2, dtype=torch.int32), one, torch.zeros(1, 3, dtype=torch.int32), one)
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
        copy_pages(kp.clone().requires_grad_(), vp, [0], [1])


def test_pools_and_outputs_that_overlap_are_refused(ext):
    inv, one = rotary_frequencies(64)[0], torch.ones(1, dtype=torch.int32)
    kp, vp = _pool(4, 2, 16, 64, torch.float32)
    both = torch.zeros(4, 2, 2, 16, 64)  # K and V of a page side by side
    big = torch.zeros(5, 2, 16, 64)
    q = torch.zeros(3, 2, 64)
    flat = torch.zeros(4, 2, 64)
    table, path = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, 3, dtype=torch.int32)
    for a, b, what in ((kp, vp, "CUDA"), (both[:, 0], both[:, 1], "CUDA"), (kp, kp, "shares memory"),
                       (big[:4], big[1:], "shares memory"), (both[:, 0], both[:, 0], "shares memory")):
        with pytest.raises(RuntimeError, match=what):
            append_kv(**_append_args(k_pages=a, v_pages=b))
        with pytest.raises(RuntimeError, match=what):
            compact_path(a, b, table, one, path, one)
        with pytest.raises(RuntimeError, match="CUDA" if a is b or a.data_ptr() == b.data_ptr() else what):
            copy_pages(a, b, [0], [1])
    thin = torch.zeros(4 * 2048).as_strided((4, 2, 16, 64), (1024, 1024, 64, 1))  # pages overlap
    with pytest.raises(RuntimeError, match="between its pages"):
        append_kv(**_append_args(k_pages=thin))
    args = _append_args(inv_freq=inv, q=q)
    for out, what in ((q, "CUDA"), (torch.zeros(3, 2, 64), "CUDA"), (args["k"], "shares memory with k"),
                      (args["v"], "shares memory with v"), (args["k_pages"][0, 0, :6].view(3, 2, 64), "k_pages"),
                      (args["v_pages"][1, 1, 3:9].view(3, 2, 64), "v_pages")):
        with pytest.raises(RuntimeError, match=what):
            append_kv(**args, q_out=out)
    with pytest.raises(RuntimeError, match="q_out shares memory with q"):
        append_kv(**_append_args(inv_freq=inv, q=flat[:3]), q_out=flat[1:])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("ctx, counts, Hk, D, page", [
    ([5, 0, 31, 16], [1, 0, 3, 33], 2, 128, 16),
    ([0, 9, 2, 700], [1200, 0, 1, 1700], 1, 64, 16),  # many tokens of few heads
])
def test_append_holds_each_element_to_its_own_bound(ext, cuda_device, dtype, inter, ctx, counts, Hk, D, page):
    """K within its own element's bound where it was written, and every other row as it was."""
    T = sum(counts)
    g = torch.Generator().manual_seed(9)
    k, v = (torch.randn(T, Hk, D, generator=g).to(dtype) for _ in "kv")
    table, pages = _table([c + m for c, m in zip(ctx, counts)], page)
    kp, vp = _pool(pages, Hk, page, D, dtype)
    inv = rotary_frequencies(D // 2)[0]
    kd, vd = kp.cuda(), vp.cuda()
    append_kv(k.cuda(), v.cuda(), kd, vd, table.cuda(), torch.tensor(ctx, dtype=torch.int32).cuda(),
              _cu(counts).cuda(), inv_freq=inv.cuda(), interleaved=inter)
    pos = torch.cat([torch.arange(c, c + m) for c, m in zip(ctx, counts)])
    req = torch.repeat_interleave(torch.arange(len(counts)), torch.tensor(counts))
    page_of, off = table[req, pos // page].long(), pos % page
    got, ref = kd.cpu(), O.rotate(k, pos, inv, inter)
    bound = O.rotate_bound(k, inv, inter, 1.0, dtype, pos)
    assert ((got[page_of, :, off].double() - ref).abs() <= bound).all()
    assert torch.equal(vd.cpu()[page_of, :, off], v)
    other = torch.ones(pages, page, dtype=torch.bool)
    other[page_of, off] = False
    for x, y in ((got, kp), (vd.cpu(), vp)):
        assert torch.equal(x.transpose(1, 2)[other], y.transpose(1, 2)[other])


@pytest.mark.gpu
def test_single_entries_of_any_stride(ext, cuda_device):
    """One request's lengths, pages, borders and path may be slices of wider tensors: the stride
    of a single element means nothing."""
    from ring_attention_benchmark_b200.ops.paged import tree_attention

    kp, vp = _pool(3, 1, 16, 64, torch.float32)
    wide = torch.tensor([[2, 9], [1, 9], [1, 9]], dtype=torch.int32).cuda()
    table, one = wide[:1, :1], wide[1:2, 0]  # page 2; one
    ctx = torch.tensor([[5, 9]], dtype=torch.int32).cuda()[:, 0]
    assert one.stride(0) == 2 and ctx.stride(0) == 2
    k, v = torch.randn(2, 1, 64), torch.randn(2, 1, 64)
    kd, vd = kp.cuda(), vp.cuda()
    append_kv(k.cuda(), v.cuda(), kd, vd, table, ctx)
    kp[2, 0, 5:7], vp[2, 0, 5:7] = k[:, 0], v[:, 0]
    assert torch.equal(kd.cpu(), kp) and torch.equal(vd.cpu(), vp)
    q = torch.randn(2, 1, 64).cuda()
    assert torch.equal(tree_attention(q, kd, vd, table, ctx),
                       tree_attention(q, kd, vd, table.contiguous().clone(), ctx.clone()))
    compact_path(kd, vd, table, ctx, one.view(1, 1), one)
    kp[2, 0, 5], vp[2, 0, 5] = k[1, 0], v[1, 0]
    assert torch.equal(kd.cpu(), kp) and torch.equal(vd.cpu(), vp)
