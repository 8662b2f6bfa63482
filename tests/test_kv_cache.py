"""The cache's bookkeeping on the host, and prompts, forks, drafted trees and
defragmentation together on the GPU, against a plain model of both."""
import random

import pytest
import torch

import _paged_oracle as O
from ring_attention_benchmark_b200 import PagedKVCache, RingAttention, Rotary
from ring_attention_benchmark_b200.models.kv_cache import OutOfPages, PageTable


# ------------------------------------------------------------------ bookkeeping (CPU)
def _check(t):
    held = {}
    for s in t.sequences():
        pages = t.pages(s)
        assert len(set(pages)) == len(pages)
        assert len(pages) * t.page_size >= t.length(s)
        for p in pages:
            held[p] = held.get(p, 0) + 1
    assert t.free_pages == t.num_pages - len(held)
    assert sorted(t._free) == [p for p in range(t.num_pages) if p not in held]
    assert [t._holders[p] for p in range(t.num_pages)] == [held.get(p, 0) for p in range(t.num_pages)]


def test_random_operations_keep_the_tokens():
    """Random steps, forks, truncations, frees and compactions; a dict of what each
    place of the pool holds stands in for the GPU."""
    rng = random.Random(3)
    t = PageTable(40, 4)
    pool, want, stamp = {}, {}, 0

    def move(src, dst):
        assert not set(src) & set(dst) and len(set(dst)) == len(dst)
        old = {p: [pool.get((p, i)) for i in range(4)] for p in src}
        for a, b in zip(src, dst):
            for i in range(4):
                pool[b, i] = old[a][i]

    for _ in range(3000):
        seqs = t.sequences()
        op = rng.random()
        if not seqs or op < 0.1:
            want[t.new()] = []
        elif op < 0.2:
            s = rng.choice(seqs)
            want[t.fork(s)] = list(want[s])
        elif op < 0.3:
            s = rng.choice(seqs)
            t.free(s)
            del want[s]
        elif op < 0.4:
            s = rng.choice(seqs)
            n = rng.randint(0, t.length(s))
            t.truncate(s, n)
            want[s] = want[s][:n]
        elif op < 0.45:
            move(*t.compact())
            used = t.num_pages - t.free_pages
            assert all(p < used for s in t.sequences() for p in t.pages(s))
        else:
            some = rng.sample(seqs, rng.randint(1, len(seqs)))
            counts = [rng.choice([0, 1, 1, 2, 5, 9]) for _ in some]
            before = {s: t.pages(s) for s in seqs}
            try:
                move(*t.reserve(some, counts))
            except OutOfPages:
                assert {s: t.pages(s) for s in seqs} == before
                continue
            for s, n in zip(some, counts):
                keep = rng.randint(0, n)
                for i in range(n):
                    p = t.length(s) + i
                    page = t.pages(s)[p // 4]
                    assert t._holders[page] == 1  # nobody else's
                    stamp += 1
                    pool[page, p % 4] = stamp
                    if i < keep:
                        want[s].append(stamp)
                t.grow(s, keep)
        _check(t)
        for s in t.sequences():
            assert [pool[t.pages(s)[i // 4], i % 4] for i in range(t.length(s))] == want[s]


def test_table_refusals():
    t = PageTable(4, 16, max_len=40)
    s = t.new()
    with pytest.raises(KeyError):
        t.length(99)
    with pytest.raises(ValueError, match="twice"):
        t.reserve([s, s], [1, 1])
    with pytest.raises(ValueError, match="counts"):
        t.reserve([s], [1, 1])
    with pytest.raises(ValueError, match="40"):
        t.reserve([s], [41])
    with pytest.raises(ValueError):
        t.reserve([s], [-1])
    with pytest.raises(ValueError, match="not reserved"):
        t.grow(s, 1)
    t.reserve([s], [40])
    t.grow(s, 40)
    with pytest.raises(ValueError):
        t.truncate(s, 41)
    with pytest.raises(OutOfPages):
        t.reserve([t.new()], [17])
    with pytest.raises(KeyError):
        t.free(99)
    for kw in (dict(num_pages=0, page_size=16), dict(num_pages=4, page_size=0),
               dict(num_pages=4, page_size=16, max_len=0)):
        with pytest.raises(ValueError):
            PageTable(**kw)


@pytest.mark.parametrize("kw", [dict(layers=0), dict(heads_kv=0), dict(head_dim=32),
                                dict(page_size=20), dict(dtype=torch.float64)])
def test_cache_refusals(kw):
    a = dict(layers=1, num_pages=4, heads_kv=1, head_dim=64, device="cpu")
    a.update(kw)
    with pytest.raises(ValueError):
        PagedKVCache(**a)


def test_step_tensors_and_refusals():
    cache = PagedKVCache(2, 8, 1, 64, page_size=16, device="cpu")
    a, b = cache.new_sequence(), cache.new_sequence()
    step = cache.step([a, b], [17, 3])
    assert step.context_lens.tolist() == [0, 0] and step.cu_q.tolist() == [0, 17, 20]
    assert step.block_table.shape == (2, 2) and step.max_q == 17
    step.commit()
    assert cache.length(a) == 17 and cache.length(b) == 3
    with pytest.raises(RuntimeError, match="committed"):
        step.commit()
    step = cache.step([b, a], [2, 4])
    assert step.context_lens.tolist() == [3, 17]
    assert step.positions(torch.tensor([0, 1, 0, 1, 1, 2], dtype=torch.int32)).tolist() == [3, 4, 17, 18, 18, 19]
    with pytest.raises(ValueError, match="parent"):
        step.tree([[-1, 1], [-1, 0, 0, 0]])
    with pytest.raises(ValueError, match="parent"):
        step.tree([[-1], [-1, 0, 0, 0]])
    for bad in ([[0]], [[0, 0], []], [[1, 0], []], [[2], []], [[-1], []]):
        with pytest.raises(ValueError):
            step.accept(bad)
    step.accept([[0, 1], []])  # a path from the start needs no move
    assert cache.length(b) == 5 and cache.length(a) == 17
    with pytest.raises(ValueError):
        cache.step([], [])


def test_one_open_step_per_sequence():
    cache = PagedKVCache(1, 8, 1, 64, page_size=16, device="cpu")
    a, b = cache.new_sequence(), cache.new_sequence()
    step = cache.step([a], [20])
    for call in (lambda: cache.step([b, a], [1, 1]), lambda: cache.free(a),
                 lambda: cache.truncate(a, 0), cache.defragment):
        with pytest.raises(RuntimeError, match="step"):
            call()
    assert cache.table.free_pages == 6  # the refused calls took nothing
    fork = cache.fork(a)  # holds what is committed: nothing
    assert cache.length(fork) == 0 and cache.table.pages(fork) == ()
    step.cancel()
    step.cancel()  # again: nothing
    assert cache.table.free_pages == 8 and cache.length(a) == 0
    with pytest.raises(RuntimeError, match="committed"):
        step.commit()
    cache.step([a], [3])  # dropped without a word: it does not block the sequence
    step = cache.step([a], [5])
    step.commit()
    assert cache.length(a) == 5 and cache.defragment() == 1
    cache.free(a)


# ------------------------------------------------------------------ together (GPU)
class _Plain:
    """What each sequence holds, layer by layer, as lists of 64-bit rows."""

    def __init__(self, layers):
        self.k = [torch.zeros(0) for _ in range(layers)]
        self.v = [torch.zeros(0) for _ in range(layers)]

    def copy(self):
        other = _Plain(0)
        other.k, other.v = [x.clone() for x in self.k], [x.clone() for x in self.v]
        return other


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, d", [(torch.bfloat16, 128), (torch.float32, 64)])
def test_prompt_fork_trees_and_defragmentation(ext, cuda_device, dtype, d):
    """A prompt through the ring and into the cache, a fork, two rounds of drafted
    trees with accepted paths, frees and a defragmentation; every attention is held
    to the plain model, and the cache at the end to what was written."""
    H, Hk, L, S = 4, 2, 2, 256
    g = torch.Generator().manual_seed(0)
    rand = lambda n, h: torch.randn(n, h, d, generator=g).to(dtype)  # noqa: E731
    rot = Rotary(d, base=500000.0, interleaved=True, device="cuda")
    inv = rot.inv_freq.cpu()
    cache = PagedKVCache(L, 40, Hk, d, page_size=16, dtype=dtype)
    other = cache.new_sequence()  # lies in front of the prompt and is freed later
    seq = cache.new_sequence()
    plain = {seq: _Plain(L)}

    def close(got, lse, q, pos, model, layer, vis, first):
        """`got` against attention of rotated q over the model's rows and the new ones."""
        n = q.shape[0]
        kr, vr = model.k[layer], model.v[layer]
        keys = kr.shape[0]
        # the kernel's own rotation of q and K is held elsewhere: one page here, 64 bits beside it
        pool_k = kr.permute(1, 0, 2).reshape(1, Hk, keys, d)
        pool_v = vr.permute(1, 0, 2).reshape(1, Hk, keys, d)
        qr = first  # already rotated on the GPU
        ref, rlse, mag, smax = O.attention(qr, pool_k, pool_v, torch.zeros(1, 1, dtype=torch.int32),
                                           [keys - n], [n], [vis])
        bo, bl = O.attention_bound(ref, mag, smax, dtype, keys, d)
        assert ((got.cpu().double() - ref).abs() <= bo).all()
        assert ((lse.cpu().double() - rlse).abs() <= bl + 2.0 ** -22 * rlse.abs()).all()

    def run(step, seqs, mask, vis, positions):
        news = []
        for layer in range(L):
            q, k, v = rand(step.tokens, H), rand(step.tokens, Hk), rand(step.tokens, Hk)
            qr = step.append(layer, k.cuda(), v.cuda(), rotary=rot, q=q.cuda(), positions=positions)
            out, lse = step.attend(layer, qr, mask=mask, return_lse=True)
            pos = positions.cpu() if positions is not None else torch.cat(
                [torch.arange(c, c + n) for c, n in zip(step.lengths, step.counts)])
            kr = O.rotate(k, pos, inv, True)
            bound = O.rotate_bound(k, inv, True, 1.0, dtype, pos)
            at = 0
            for b, s in enumerate(seqs):
                n, m = step.counts[b], plain[s]
                rows = slice(at, at + n)
                # the cache's own rounded K stands in the model (checked against 64 bits)
                place = [(int(step.block_table[b, (step.lengths[b] + i) // 16]), (step.lengths[b] + i) % 16)
                         for i in range(n)]
                held = torch.stack([cache.k[layer, p, :, o] for p, o in place]).cpu()
                assert ((held.double() - kr[rows]).abs() <= bound[rows]).all()
                m.k[layer] = torch.cat((m.k[layer].reshape(-1, Hk, d).to(dtype), held))
                m.v[layer] = torch.cat((m.v[layer].reshape(-1, Hk, d).to(dtype), v[rows]))
                close(out[rows], lse[rows], q[rows], pos[rows], m, layer, vis[b], qr[rows].cpu())
                at += n
            news.append(out)
        return news

    # other traffic in front, then the prompt: the ring's own result beside the cache's
    st = cache.step([other], [40])
    plain[other] = _Plain(L)
    run(st, [other], None, [torch.ones(40, 40, dtype=torch.bool).tril()], None)
    st.commit()
    q, k, v = rand(S, H), rand(S, Hk), rand(S, Hk)
    st = cache.step([seq], [S])
    with RingAttention(S, heads=H, head_dim=d, heads_kv=Hk, dtype=dtype, causal=True, rotary=rot) as ring:
        want = ring(q.cuda(), k.cuda(), v.cuda())
    for layer in range(L):
        qr = st.append(layer, k.cuda(), v.cuda(), rotary=rot, q=q.cuda())
        got = st.attend(layer, qr)
        # two kernels of the same rounded inputs, each off by half a step for the rounded
        # weights and half for the result, and fp32 sums (5: four and what those need);
        # the ring's fp32 products carry 2^-21 each and D of them a score
        tol = 5 * O.half_step(dtype) if dtype != torch.float32 else 2 * 2.0 ** -21 * d
        assert (got.float() - want.float()).abs().max().item() <= tol * v.abs().max().item()
        held = torch.stack([cache.k[layer, int(st.block_table[0, i // 16]), :, i % 16] for i in range(S)]).cpu()
        plain[seq].k[layer], plain[seq].v[layer] = held, v.clone()
    st.commit()

    two = cache.fork(seq)
    plain[two] = plain[seq].copy()
    cache.truncate(two, S - 5)  # into the middle of a shared page
    for layer in range(L):
        plain[two].k[layer], plain[two].v[layer] = plain[two].k[layer][:S - 5], plain[two].v[layer][:S - 5]
    cache.free(other)
    for rnd in range(2):
        parents = [[-1, 0, 0, 1, 1, 2, 5], [-1, 0, 1, 0]]
        vis = [O.ancestors(p)[0] for p in parents]
        before = [cache.length(seq), cache.length(two)]
        st = cache.step([seq, two], [7, 4])
        mask, depth = st.tree(parents)
        run(st, [seq, two], mask, vis, st.positions(depth))
        paths = [[0, 2, 5, 6], [0, 3]] if rnd == 0 else [[0, 1], []]
        st.accept(paths)
        for s, n0, p in zip((seq, two), before, paths):
            assert cache.length(s) == n0 + len(p)
            for x in (plain[s].k, plain[s].v):
                for layer in range(L):
                    x[layer] = torch.cat((x[layer][:n0], x[layer][n0:][p]))
        assert cache.defragment() == cache.table.num_pages - cache.table.free_pages
    for s in (seq, two):
        for layer in range(L):
            for pool, rows in ((cache.k, plain[s].k[layer]), (cache.v, plain[s].v[layer])):
                pages = cache.table.pages(s)
                held = torch.stack([pool[layer, pages[i // 16], :, i % 16] for i in range(cache.length(s))])
                assert torch.equal(held.cpu(), rows)
    cache.free(seq)
    cache.free(two)
    assert cache.table.free_pages == 40


def test_steps_refuse_too_few_rows(ext):
    """A step's tensors hold all of its tokens: a missing one would leave stale rows in the
    cache that a commit then counts.  More rows are a padded batch."""
    cache = PagedKVCache(1, 8, 1, 64, page_size=16, device="cpu")
    step = cache.step([cache.new_sequence(), cache.new_sequence()], [3, 2])
    full, short = torch.zeros(5, 1, 64).bfloat16(), torch.zeros(4, 1, 64).bfloat16()
    rot = Rotary(64, device="cpu")
    for k, v, q in ((short, short, None), (full, short, None), (full, full, short)):
        with pytest.raises(ValueError, match="4 rows, the step 5 tokens"):
            step.append(0, k, v, rotary=rot, q=q)
    with pytest.raises(ValueError, match="4 rows, the step 5 tokens"):
        step.attend(0, short)
    for rows in (5, 8):  # on to the operators, which want a GPU
        x = torch.zeros(rows, 1, 64).bfloat16()
        with pytest.raises(RuntimeError, match="CUDA"):
            step.append(0, x, x)
        with pytest.raises(RuntimeError, match="CUDA"):
            step.attend(0, x)


@pytest.mark.gpu
def test_a_drafted_step_does_not_wait_for_the_gpu(ext, cuda_device):
    """Tables, trees, positions and paths are handed over without a synchronisation."""
    cache = PagedKVCache(1, 32, 1, 64, page_size=16)
    a, b = cache.new_sequence(), cache.new_sequence()
    prompt = cache.step([a, b], [5, 9])
    prompt.append(0, *(torch.randn(14, 1, 64, device="cuda").bfloat16() for _ in "kv"))
    prompt.commit()
    parents = [[-1, 0, 0, 1], [-1, 0, 1]]
    k = torch.randn(7, 1, 64, device="cuda").bfloat16()
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        step = cache.step([a, b], [4, 3])
        mask, depth = step.tree(parents)
        pos = step.positions(depth)
        step.append(0, k, k)
        out = step.attend(0, k, mask=mask)
        step.accept([[0, 2], [0, 1, 2]])
    finally:
        torch.cuda.set_sync_debug_mode("default")
    assert pos.dtype == torch.int32 and pos.tolist() == [5, 6, 6, 7, 9, 10, 11]
    assert out.isfinite().all() and cache.length(a) == 7 and cache.length(b) == 12
    none = cache.step([a, b], [0, 0])  # nothing drafted
    mask, depth = none.tree([[], []])
    assert none.positions(depth).numel() == 0 and mask.shape[0] == 0


@pytest.mark.gpu
def test_uploads_inside_a_capture_are_refused(ext, cuda_device):
    """A replay would copy from host memory that is long someone else's."""
    cache = PagedKVCache(1, 32, 1, 64, page_size=16)
    seq, other = cache.new_sequence(), cache.new_sequence()
    step = cache.step([seq], [3])
    x = torch.zeros(3, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = x + 1
        for call in (lambda: step.tree([[-1, 0, 0]]), lambda: step.accept([[0, 2]]),
                     lambda: cache.step([other], [1])):
            with pytest.raises(RuntimeError, match="outside a capture"):
                call()
    graph.replay()
    assert (y == 1).all()
    assert cache.table.pages(other) == () and cache.length(seq) == 0
    step.accept([[0]])  # still open
    assert cache.length(seq) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("parents, path", [([-1, 0, 0, 1, 2, 2], [0, 2, 5]), ([-1, 0, 0], [0, 2]),
                                           ([-1, -1], [1]), ([-1, 0], []), ([-1], [0])])
def test_one_sequence_from_prompt_to_defragmentation(ext, cuda_device, parents, path):
    """The whole course with a single sequence: a prompt, a drafted tree whose path is accepted,
    single tokens, a fork, a free and a defragmentation; the cache holds what was kept."""
    L, Hk, D, n = 2, 2, 64, 21
    g = torch.Generator().manual_seed(len(parents))
    rot = Rotary(D, device="cuda")
    cache = PagedKVCache(L, 16, Hk, D, page_size=16)
    seq = cache.new_sequence()
    kept = [torch.zeros(0, Hk, D).bfloat16() for _ in range(L)]

    def write(step, keep, mask=None, positions=None):
        for layer in range(L):
            q, k, v = (torch.randn(step.tokens, h, D, generator=g).bfloat16() for h in (4, Hk, Hk))
            q = step.append(layer, k.cuda(), v.cuda(), rotary=rot, q=q.cuda(), positions=positions)
            assert step.attend(layer, q, mask=mask).isfinite().all()
            kept[layer] = torch.cat((kept[layer], v[keep]))

    step = cache.step([seq], [n])
    write(step, list(range(n)))
    step.commit()
    step = cache.step([seq], [len(parents)])
    mask, depth = step.tree([parents])
    write(step, path, mask, step.positions(depth))
    step.accept([path])
    for _ in range(3):
        step = cache.step([seq], [1])
        write(step, [0])
        step.commit()
    best = cache.fork(seq)
    cache.free(seq)
    assert cache.defragment() == len(cache.table.pages(best))
    assert cache.length(best) == n + len(path) + 3
    pages = cache.table.pages(best)
    for layer in range(L):
        held = torch.stack([cache.v[layer, pages[i // 16], :, i % 16] for i in range(cache.length(best))])
        assert torch.equal(held.cpu(), kept[layer])


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(6))
def test_a_random_course_of_a_cache(ext, cuda_device, seed):
    """Steps (prompts, single tokens, trees, none), paths, forks, truncations, frees and
    defragmentations at random: V of every sequence stays what was kept, K too, and every
    attention is that of the rows that its sequence holds."""
    rng, g = random.Random(seed), torch.Generator().manual_seed(seed)
    D, L = rng.choice([(64, 2), (128, 1)])
    Hk, group, page = rng.choice([1, 2, 3]), rng.choice([1, 2, 5]), rng.choice([16, 32])
    dtype = [torch.bfloat16, torch.float16, torch.float32][seed % 3]
    cache = PagedKVCache(L, 24, Hk, D, page_size=page, dtype=dtype)
    held = {}

    def rand(n, h):
        return torch.randn(n, h, D, generator=g).to(dtype)

    for _ in range(60):
        op, seqs = rng.random(), cache.table.sequences()
        if not seqs or op < 0.1:
            held[cache.new_sequence()] = [[torch.zeros(0, Hk, D).to(dtype)] * 2] * L
        elif op < 0.2:
            s = rng.choice(seqs)
            held[cache.fork(s)] = held[s]
        elif op < 0.3 and len(seqs) > 2:
            s = rng.choice(seqs)
            cache.free(s)
            del held[s]
        elif op < 0.38:
            s = rng.choice(seqs)
            n = rng.randint(0, cache.length(s))
            cache.truncate(s, n)
            held[s] = [[x[:n] for x in kv] for kv in held[s]]
        elif op < 0.45:
            cache.defragment()
        else:
            some = rng.sample(seqs, rng.randint(1, len(seqs)))
            counts = [rng.choice([0, 1, 1, 2, 7, 30]) for _ in some]
            try:
                step = cache.step(some, counts)
            except OutOfPages:
                continue
            tree = rng.random() < 0.5
            parents = [[-1 if i == 0 else rng.randint(-1, i - 1) for i in range(n)] for n in counts]
            mask, depth = step.tree(parents) if tree else (None, None)
            masks = [O.ancestors(p)[0] for p in parents] if tree else None
            new = [[] for _ in some]
            pad = rng.choice([0, 0, 3])
            for layer in range(L):
                q, k, v = rand(step.tokens + pad, Hk * group), rand(step.tokens + pad, Hk), rand(step.tokens + pad, Hk)
                step.append(layer, k.cuda(), v.cuda())
                m = mask if mask is None or not pad else torch.cat((mask, mask.new_zeros(pad, mask.shape[1])))
                out, lse = step.attend(layer, q.cuda(), mask=m, return_lse=True)
                at = 0
                for b, (s, n) in enumerate(zip(some, counts)):
                    rows, was = slice(at, at + n), held[s][layer]
                    kk, vv = torch.cat((was[0], k[rows])), torch.cat((was[1], v[rows]))
                    new[b].append((k[rows], v[rows]))
                    at += n
                    if n == 0:
                        continue
                    pool = [x.permute(1, 0, 2).reshape(1, Hk, len(x), D) for x in (kk, vv)]
                    ref, rlse, mag, smax = O.attention(q[rows], *pool, torch.zeros(1, 1, dtype=torch.int32),
                                                       [len(kk) - n], [n], masks and [masks[b]])
                    bo, bl = O.attention_bound(ref, mag, smax, dtype, len(kk), D)
                    assert ((out[rows].cpu().double() - ref).abs() <= bo).all()
                    assert ((lse[rows].cpu().double() - rlse).abs() <= bl + 2.0 ** -22 * rlse.abs()).all()
            if rng.random() < 0.15:
                paths = [[] for _ in some]
                step.cancel()
            elif tree:
                paths = [sorted(rng.sample(range(n), rng.randint(0, n))) for n in counts]
                step.accept(paths)
            else:
                paths = [list(range(n)) for n in counts]
                step.commit()
            for s, kv, p in zip(some, new, paths):
                held[s] = [[torch.cat((x, y[p])) for x, y in zip(held[s][layer], kv[layer])] for layer in range(L)]
        for s in cache.table.sequences():
            n, pages = cache.length(s), torch.tensor(cache.table.pages(s), dtype=torch.long)
            i = torch.arange(n)
            for layer in range(L):
                for pool, rows in zip((cache.k, cache.v), held[s][layer]):
                    assert torch.equal(pool[layer].cpu()[pages[i // page], :, i % page], rows)
