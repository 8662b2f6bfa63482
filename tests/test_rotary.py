"""Rotary positions: both layouts, part of the head, odd sizes, strides, far
positions, scaled frequencies, gradients and refusals, against 64 bits."""
import math

import pytest
import torch

import _paged_oracle as O
from ring_attention_benchmark_b200 import RingAttention
from ring_attention_benchmark_b200.ops.rotary import (Rotary, SCALINGS, apply_rotary,
                                                      rotary_frequencies)

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


# ------------------------------------------------------------------ frequencies (CPU)
def test_plain_frequencies():
    inv, scale = rotary_frequencies(8, base=10000.0)
    assert inv.dtype == torch.float64 and scale == 1.0
    assert inv.tolist() == pytest.approx([1.0, 0.1, 0.01, 0.001], rel=1e-14)


def test_linear_and_ntk_frequencies():
    plain, _ = rotary_frequencies(64)
    lin, _ = rotary_frequencies(64, scaling="linear", factor=4.0)
    assert torch.equal(lin, plain / 4)
    ntk, _ = rotary_frequencies(64, scaling="ntk", factor=4.0)
    assert ntk[0] == plain[0]  # the fastest pair is kept
    assert ntk[-1].item() == pytest.approx(plain[-1].item() / 4, rel=1e-12)


@pytest.mark.parametrize("scaling", ["yarn", "bands"])
def test_banded_frequencies(scaling):
    plain, _ = rotary_frequencies(128, base=500000.0)
    inv, scale = rotary_frequencies(128, base=500000.0, scaling=scaling, factor=8.0,
                                    original_length=8192, fast=32.0, slow=1.0)
    turns = 8192 * plain / (2 * math.pi)
    ratio = plain / inv
    assert (ratio >= 1 - 1e-12).all() and (ratio <= 8 + 1e-9).all()
    assert torch.all(ratio[1:] >= ratio[:-1] - 1e-9)  # slower pairs are stretched at least as much
    if scaling == "bands":
        assert torch.equal(inv[turns > 32], plain[turns > 32])
        assert scale == 1.0
    else:
        assert torch.equal(inv[turns > 40], plain[turns > 40])
        assert scale == pytest.approx(0.1 * math.log(8) + 1)
    assert ratio[turns < 0.5].tolist() == pytest.approx([8.0] * int((turns < 0.5).sum()), rel=1e-9)


def test_factor_one_changes_nothing():
    plain, _ = rotary_frequencies(32)
    for scaling in SCALINGS:
        inv, scale = rotary_frequencies(32, scaling=scaling, factor=1.0, original_length=512)
        assert inv.tolist() == pytest.approx(plain.tolist(), rel=1e-14) and scale == 1.0


@pytest.mark.parametrize("kw", [dict(rotary_dim=3), dict(rotary_dim=0), dict(rotary_dim=8, base=1.0),
                                dict(rotary_dim=8, factor=0.5), dict(rotary_dim=8, scaling="x"),
                                dict(rotary_dim=8, scaling="yarn"), dict(rotary_dim=2, scaling="ntk"),
                                dict(rotary_dim=8, scaling="bands", original_length=9, fast=1.0, slow=2.0),
                                dict(rotary_dim=8, base=math.nan)])
def test_frequency_refusals(kw):
    with pytest.raises(ValueError):
        rotary_frequencies(**kw)


# ------------------------------------------------------------------ refusals (CPU)
def _args(**kw):
    a = dict(q=torch.zeros(4, 2, 16), k=torch.zeros(4, 1, 16), positions=torch.arange(4),
             inv_freq=rotary_frequencies(16)[0])
    a.update(kw)
    return a


@pytest.mark.parametrize("kw, what", [
    (dict(), "CUDA"),
    (dict(q=torch.zeros(4, 16)), "tokens, heads, dim"),
    (dict(q=torch.zeros(4, 2, 16, dtype=torch.float64)), "bfloat16"),
    (dict(q=torch.zeros(4, 16, 2).transpose(1, 2)), "last dimension"),
    (dict(k=torch.zeros(3, 1, 16)), "same tokens"),
    (dict(k=torch.zeros(4, 1, 8)), "same tokens"),
    (dict(k=torch.zeros(4, 1, 16, dtype=torch.float16)), "dtype"),
    (dict(positions=torch.arange(3)), "positions"),
    (dict(positions=torch.zeros(4)), "int64 or int32"),
    (dict(inv_freq=torch.ones(8)), "float64"),
    (dict(inv_freq=torch.ones(9, dtype=torch.float64)), "head dim"),
    (dict(scale=math.inf), "finite"),
    (dict(out=(torch.zeros(4, 2, 8), None)), "shape"),
    (dict(out=(torch.zeros(1, 2, 16).expand(4, 2, 16), None)), "shares memory"),
])
def test_refusals(ext, kw, what):
    a = _args(**kw)
    with pytest.raises(RuntimeError, match=what):
        apply_rotary(a.pop("q"), a.pop("k"), a.pop("positions"), a.pop("inv_freq"), **a)


# ------------------------------------------------------------------ values (GPU)
def _inputs(T, H, Hk, D, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(T, H, D, generator=g).to(dtype), torch.randn(T, Hk, D, generator=g).to(dtype)


def _close(got, x, positions, inv, inter, scale, inverse=False):
    ref = O.rotate(x, positions, inv, inter, scale, inverse)
    bound = O.rotate_bound(x, inv, inter, scale, got.dtype, positions)
    d = (got.cpu().double() - ref).abs()
    assert (d <= bound).all(), (d - bound).max().item()
    r = 2 * inv.numel()
    assert torch.equal(got.cpu()[..., r:], x[..., r:])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("T,H,Hk,D,r", [(1, 1, 1, 64, 64), (7, 8, 2, 128, 128), (33, 3, 1, 128, 64),
                                        (5, 2, 2, 80, 32), (3, 5, 1, 96, 10), (2, 2, 1, 63, 2),
                                        (1025, 4, 4, 64, 48), (2, 1, 1, 512, 512), (3, 40, 17, 64, 64),
                                        # many tokens of few heads: all operands of a token in one block
                                        (3001, 1, 1, 64, 64), (2500, 3, 2, 128, 64), (2400, 1, 1, 512, 512),
                                        (9999, 2, 1, 64, 32)])
def test_rotary_values(ext, cuda_device, dtype, inter, T, H, Hk, D, r):
    q, k = _inputs(T, H, Hk, D, dtype)
    inv, _ = rotary_frequencies(r)
    pos = torch.randint(0, 1 << 20, (T,), generator=torch.Generator().manual_seed(1))
    dev = cuda_device
    qo, ko = apply_rotary(q.to(dev), k.to(dev), pos.to(dev), inv.to(dev), interleaved=inter,
                          scale=1.25)
    _close(qo, q, pos, inv, inter, 1.25)
    _close(ko, k, pos, inv, inter, 1.25)
    alone = apply_rotary(q.to(dev), None, pos.to(dev).int(), inv.to(dev), interleaved=inter, scale=1.25)
    assert torch.equal(alone, qo)
    back = apply_rotary(q.to(dev), None, pos.to(dev), inv.to(dev), interleaved=inter, inverse=True)
    _close(back, q, pos, inv, inter, 1.0, inverse=True)


@pytest.mark.gpu
def test_far_and_negative_positions(ext, cuda_device):
    pos = torch.tensor([0, 1, -1, 2 ** 31 - 1, 2 ** 31, 2 ** 33 + 12345, -(2 ** 32) - 7])
    q, _ = _inputs(7, 2, 1, 64, torch.float32)
    inv, _ = rotary_frequencies(64)
    got = apply_rotary(q.cuda(), None, pos.cuda(), inv.cuda())
    _close(got, q, pos, inv, False, 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shift", [0, 1])
def test_strided_inputs_and_outputs(ext, cuda_device, dtype, shift):
    """Slices of one projection, at an aligned and at an odd place, into strided outputs."""
    T, H, Hk, D = 9, 4, 2, 64
    g = torch.Generator().manual_seed(3)
    flat = torch.randn(T, (H + 2 * Hk) * D + 8, generator=g).to(dtype).cuda()
    q = flat[:, shift:shift + H * D].unflatten(1, (H, D))
    k = flat[:, shift + H * D:shift + (H + Hk) * D].unflatten(1, (Hk, D))
    pos = torch.arange(T).cuda() * 1000
    inv = rotary_frequencies(32)[0].cuda()
    big = torch.full((T, H + 1, D), 7.0, dtype=dtype, device="cuda")
    qo, ko = apply_rotary(q, k, pos, inv, out=(big[:, :H], torch.empty_like(k)))
    _close(qo, q.cpu(), pos.cpu(), inv.cpu(), False, 1.0)
    _close(ko, k.cpu(), pos.cpu(), inv.cpu(), False, 1.0)
    assert (big[:, H] == 7.0).all()
    before = q.cpu().clone()
    apply_rotary(q, None, pos, inv, out=(q, None))  # in place
    _close(q, before, pos.cpu(), inv.cpu(), False, 1.0)
    assert torch.equal(k.cpu(), flat[:, shift + H * D:shift + (H + Hk) * D].unflatten(1, (Hk, D)).cpu())


@pytest.mark.gpu
def test_empty(ext, cuda_device):
    inv = rotary_frequencies(64)[0].cuda()
    q = torch.zeros(0, 4, 64, device="cuda")
    qo, ko = apply_rotary(q, torch.zeros(0, 0, 64, device="cuda"), torch.zeros(0, dtype=torch.long, device="cuda"), inv)
    assert qo.shape == q.shape and ko.shape == (0, 0, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_gradient_is_the_transposed_rotation(ext, cuda_device, inter, dtype):
    T, H, Hk, D, r = 11, 3, 2, 64, 48
    q, k = _inputs(T, H, Hk, D, dtype, 5)
    gq, gk = _inputs(T, H, Hk, D, dtype, 6)
    pos, inv = torch.arange(T) * 977, rotary_frequencies(r)[0]
    ql, kl = q.cuda().requires_grad_(), k.cuda().requires_grad_()
    out = apply_rotary(ql, kl, pos.cuda(), inv.cuda(), interleaved=inter, scale=1.5)
    dq, dk = torch.autograd.grad(out, (ql, kl), (gq.cuda(), gk.cuda()))
    _close(dq, gq, pos, inv, inter, 1.5, inverse=True)
    _close(dk, gk, pos, inv, inter, 1.5, inverse=True)


@pytest.mark.gpu
def test_gradient_against_differences(ext, cuda_device):
    """Central differences of a smooth function of the result, in fp32 with a step
    of 2^-6: the function is cubic in q, so the difference is off by h^2 / 6 times
    its third derivative (6 |w| scale^3 ...), and by rounding 2^-23 |f| / h."""
    T, D = 2, 16
    g = torch.Generator().manual_seed(9)
    q = torch.randn(T, 1, D, generator=g).cuda()
    w = torch.randn(T, 1, D, generator=g).cuda()
    pos, inv = torch.tensor([3, 100]).cuda(), rotary_frequencies(12)[0].cuda()
    f = lambda x: (apply_rotary(x, None, pos, inv, interleaved=True).double() * w.double()).sum()  # noqa: E731
    ql = q.clone().requires_grad_()
    grad, = torch.autograd.grad(f(ql), ql)
    h = 2.0 ** -6
    for i in range(D):
        e = torch.zeros_like(q)
        e[1, 0, i] = h
        d = (f(q + e) - f(q - e)) / (2 * h)  # f is linear: no error but rounding
        size = (q.abs().amax() + 1) * w.abs().sum()
        assert abs(d.item() - grad[1, 0, i].item()) <= size.item() * 8 * 2.0 ** -23 / h


@pytest.mark.gpu
def test_gradients_of_shared_expanded_and_single_inputs(ext, cuda_device):
    T, D = 6, 64
    pos, inv = torch.arange(T).cuda(), rotary_frequencies(64)[0].cuda()
    base = torch.randn(T, 1, D, device="cuda", requires_grad=True)
    q, k = apply_rotary(base.expand(T, 4, D), base, pos, inv)  # one key head read by four
    (q.sum() + k.sum()).backward()  # expanded gradients
    ones = torch.ones(T, 1, D)
    ref = 5 * O.rotate(ones, pos.cpu(), inv.cpu(), False, 1.0, inverse=True)
    # five sums of values of at most 2: a few fp32 roundings each
    assert (base.grad.cpu().double() - ref).abs().max() <= 5 * 2 * 16 * 2.0 ** -24
    only_k = torch.randn(T, 1, D, device="cuda", requires_grad=True)
    _, k2 = apply_rotary(torch.randn(T, 2, D, device="cuda"), only_k, pos, inv)
    k2.sum().backward()
    assert (only_k.grad.cpu().double() - ref / 5).abs().max() <= 2 * 16 * 2.0 ** -24
    a = torch.randn(T, 1, D, device="cuda", requires_grad=True)
    y = apply_rotary(a, None, pos, inv)
    g1, = torch.autograd.grad((y ** 3).sum(), a, create_graph=True)
    g2, = torch.autograd.grad(g1.sum(), a)  # the backward's own gradient
    y64 = O.rotate(a.detach().cpu(), pos.cpu(), inv.cpu(), False)
    back = O.rotate(ones, pos.cpu(), inv.cpu(), False)  # R applied to ones
    ref2 = O.rotate(6 * y64 * back, pos.cpu(), inv.cpu(), False, inverse=True)
    assert (g2.cpu().double() - ref2).abs().max() <= ref2.abs().max() * 64 * 2.0 ** -24
    with pytest.raises(ValueError, match="gradient"):
        apply_rotary(a, None, pos, inv, out=(torch.empty_like(a), None))


@pytest.mark.gpu
def test_captured_forward_and_backward(ext, cuda_device):
    T, D = 8, 64
    pos, inv = torch.arange(T).cuda(), rotary_frequencies(64)[0].cuda()
    x = torch.randn(T, 2, D, device="cuda", requires_grad=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(apply_rotary(x, None, pos, inv).sum(), x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = apply_rotary(x, None, pos, inv)
        g, = torch.autograd.grad(y, x, torch.ones_like(y))
    with torch.no_grad():
        x.copy_(torch.randn_like(x))
    graph.replay()
    torch.cuda.synchronize()
    _close(y.detach(), x.detach().cpu(), pos.cpu(), inv.cpu(), False, 1.0)
    _close(g, torch.ones(T, 2, D), pos.cpu(), inv.cpu(), False, 1.0, inverse=True)


@pytest.mark.gpu
def test_ring_attention_rotates_its_shard(ext, cuda_device):
    """RingAttention(rotary=...) equals rotating q and k by the rank's positions first."""
    S, H, Hk, D = 256, 4, 2, 64
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(S, h, D, generator=g).bfloat16().cuda() for h in (H, Hk, Hk))
    rot = Rotary(64, base=500000.0, interleaved=True, device="cuda")
    with RingAttention(S, heads=H, head_dim=D, heads_kv=Hk, dtype=torch.bfloat16, causal=True,
                       rotary=rot) as attn:
        got = attn(q, k, v)
        graph, out = attn.capture(q, k, v)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, got)
        pos = attn.positions()
    assert torch.equal(pos.cpu(), torch.arange(S))  # one rank: its zigzag shard is the sequence
    q2, k2 = rot(q, k, pos)
    with RingAttention(S, heads=H, head_dim=D, heads_kv=Hk, dtype=torch.bfloat16, causal=True) as attn:
        assert torch.equal(attn(q2, k2, v), got)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [3, 2367, 2368, 3000])
@pytest.mark.parametrize("dtype", DTYPES)
def test_operands_without_heads(ext, cuda_device, dtype, T):
    """q or k may have no heads, at any number of tokens; the other is rotated."""
    g = torch.Generator().manual_seed(5)
    x = torch.randn(T, 1, 64, generator=g).to(dtype)
    none = torch.zeros(T, 0, 64, dtype=dtype, device="cuda")
    pos, inv = torch.arange(T), rotary_frequencies(64)[0]
    qo, ko = apply_rotary(none, x.cuda(), pos.cuda(), inv.cuda())
    assert qo.shape == none.shape
    _close(ko, x, pos, inv, False, 1.0)
    qo, ko = apply_rotary(x.cuda(), none, pos.cuda(), inv.cuda())
    assert ko.shape == none.shape
    _close(qo, x, pos, inv, False, 1.0)
    qo, ko = apply_rotary(none, none, pos.cuda(), inv.cuda())
    assert qo.shape == ko.shape == none.shape
    learns = x.cuda().requires_grad_()
    _, ko = apply_rotary(none, learns, pos.cuda(), inv.cuda())
    grad, = torch.autograd.grad(ko, learns, torch.ones_like(ko))
    _close(grad, torch.ones(T, 1, 64, dtype=dtype), pos, inv, False, 1.0, inverse=True)


@pytest.mark.gpu
def test_rotating_in_place_is_an_in_place_operation(ext, cuda_device):
    """A tensor that a backward pass still needs may not be rotated in place unseen, as
    with torch's own in-place operations."""
    pos, inv = torch.arange(5).cuda(), rotary_frequencies(64)[0].cuda()
    x = torch.randn(5, 2, 64, device="cuda", requires_grad=True)
    for which in (0, 1):
        y = x * 2
        z = (y * y).sum()  # saves y
        with torch.no_grad():
            before = y._version
            other = torch.randn_like(y)
            pair = (y, other) if which == 0 else (other, y)
            apply_rotary(*pair, pos, inv, out=pair)
            assert y._version > before
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            z.backward()
    with pytest.raises(ValueError, match="gradient"):  # into a leaf that learns
        apply_rotary(x.detach(), None, pos, inv, out=(x, None))
    with torch.inference_mode():
        t = torch.randn(5, 2, 64, device="cuda")
        apply_rotary(t, None, pos, inv, out=(t, None))
    want = O.rotate(t.cpu(), pos.cpu(), inv.cpu(), False)
    apply_rotary(t, None, pos, inv, out=(t, None))  # an inference tensor keeps no versions
    assert (t.cpu().double() - want).abs().max() <= O.rotate_bound(
        want, inv.cpu(), False, 1.0, torch.float32, pos.cpu()).max() * 2


def test_forward_mode_is_refused(ext):
    """A tangent is never dropped without a word, whether or not the primal learns."""
    import torch.autograd.forward_ad as fw

    a = _args()
    for name in ("q", "k"):
        for learns in (False, True):
            with fw.dual_level():
                b = dict(a)
                b[name] = fw.make_dual(a[name].clone().requires_grad_(learns), torch.ones_like(a[name]))
                with pytest.raises(RuntimeError, match="forward-mode"):
                    apply_rotary(**b)


@pytest.mark.parametrize("dim, length", [(64, 131072), (128, 65536), (128, 1 << 20), (64, 1 << 24)])
def test_yarn_ramp_ends_where_its_turns_do(dim, length):
    """Where even the last pair turns more than `slow` times within the original length,
    the ramp ends behind it: no such pair is stretched by the whole factor, and the ramp
    is linear in the pair index up to the index of `slow` turns."""
    base, factor, fast, slow = 10000.0, 4.0, 32.0, 1.0
    plain, _ = rotary_frequencies(dim, base=base)
    inv, _ = rotary_frequencies(dim, base=base, scaling="yarn", factor=factor, original_length=length,
                                fast=fast, slow=slow)
    turns = length * plain / (2 * math.pi)
    assert turns[-1] > slow
    index = lambda t: dim * math.log(length / (2 * math.pi * t)) / (2 * math.log(base))  # noqa: E731
    lo, hi = math.floor(index(fast)), min(math.ceil(index(slow)), dim - 1)
    assert hi > dim // 2 - 1
    for p in range(dim // 2):
        keep = min(1.0, max(0.0, 1.0 - (p - lo) / (hi - lo)))
        assert keep > 0
        want = plain[p].item() * (keep + (1.0 - keep) / factor)
        assert inv[p].item() == pytest.approx(want, rel=1e-12)


def test_outputs_that_overlap_are_refused(ext):
    """An output may be its own input or lie between other slices; any other shared element
    would be read and written at the same time."""
    pos, inv = torch.arange(4), rotary_frequencies(16)[0]
    flat = torch.zeros(200)
    rows = lambda at, h=1: flat[at:at + 4 * h * 16].view(4, h, 16)  # noqa: E731
    qkv = torch.zeros(4, 6, 16)  # heads of q, k and v side by side
    pair = torch.zeros(4, 2, 2, 16)  # q's and k's heads in turn
    far = torch.zeros(4, 2, 16)
    cases = [  # q, k, q_out, k_out, refused
        (rows(0), None, rows(16), None, "q_out shares memory with q"),       # a token further on
        (rows(0), None, rows(1), None, "q_out shares memory with q"),
        (rows(0), None, rows(64), None, None),
        (rows(0), rows(64), rows(64), torch.zeros(4, 1, 16), "q_out shares memory with k"),
        (rows(0), rows(64), torch.zeros(4, 1, 16), rows(0), "k_out shares memory with q"),
        (rows(0), rows(64), far[:, :1], far[:, :1], "q_out shares memory with k_out"),
        (rows(0), rows(64), far[:, :1], far[:, 1:], None),
        (rows(0), rows(0), rows(0), torch.zeros(4, 1, 16), "q_out shares memory with k"),
        (qkv[:, :3], qkv[:, 3:5], qkv[:, :3], qkv[:, 3:5], None),            # in place, both
        (qkv[:, :3], qkv[:, 3:5], qkv[:, :3], qkv[:, 4:6], "k_out shares memory with k"),
        (qkv[:, :3], None, qkv[:, 3:], None, None),
        (pair[:, :, 0], pair[:, :, 1], pair[:, :, 0], pair[:, :, 1], None),
        (far, None, flat.as_strided((4, 2, 16), (24, 16, 1)), None, "shares memory between"),
        (far, None, flat.as_strided((4, 2, 16), (16, 16, 1)), None, "shares memory between"),
        (far, None, flat.as_strided((4, 2, 16), (16, 64, 1)), None, None),   # heads outside
    ]
    for q, k, qo, ko, what in cases:
        with pytest.raises(RuntimeError, match=what or "CUDA"):
            apply_rotary(q, k, pos, inv, out=(qo, ko))


@pytest.mark.parametrize("scale", [1e39, -1e300, math.nan])
def test_scales_beyond_fp32_are_refused(ext, scale):
    with pytest.raises(RuntimeError, match="scale must be finite"):
        apply_rotary(**_args(scale=scale))
