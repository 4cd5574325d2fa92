"""Rotary positions against complex products in 64 bits, forward and backward, and what they refuse."""
import ctypes
import math

import pytest
import torch

import mindspeed_rl_amd as mrl
from mindspeed_rl_amd import _lib
from mindspeed_rl_amd.positions import RotarySide

U = 2.0 ** -24                                      # half a step of fp32
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}      # least steps
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def turned(x, positions, inv_freq, interleaved, start, scale, back=False):
    """The result in 64 bits and a bound for each entry.

    Angle: what is left of it is rounded to fp32 and multiplied by pi/2 (rounded too): 2.4 U at most at pi/4; its series add 1 U
    and what is cut off 0.05 U; slopes are at most one: sine and cosine are off by 5 U amply, and by three roundings in 64 bits of the whole
    angle, which the reference's own share.  The pair's sum: that times |a| + |b|, and three roundings of each product."""
    part, d = 2 * inv_freq.shape[0], x.shape[-1]
    begin = start if start >= 0 else d + start
    at = torch.arange(part, device=x.device) + begin
    one, two = (at[0::2], at[1::2]) if interleaved else (at[:part // 2], at[part // 2:])
    angle = positions.double()[..., None, None] * inv_freq.double()
    z = x.double()
    a, b = z[..., one], z[..., two]
    w = torch.complex(a, b) * torch.polar(torch.full_like(angle, abs(scale)), -angle if back else angle) * (1 if scale >= 0 else -1)
    y, e = z.clone(), torch.zeros_like(z)
    off = (a.abs() + b.abs()) * abs(scale) * (9 * U + 4 * 2.0 ** -53 * angle.abs())
    for place, v in ((one, w.real), (two, w.imag)):
        y[..., place] = v
        e[..., place] = off + HALF[x.dtype] * v.abs() + TINY[x.dtype]
    return y, e


def turned_wide(x, positions, inv_freq):
    """x of 64 bits, halves, turned as a matrix would."""
    angle = positions.double()[:, None, None] * inv_freq
    a, b = x.chunk(2, -1)
    return torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()], -1)


def within(got, want):
    value, bound = want
    off = (got.double() - value).abs() - bound * 1.01
    assert off.numel() == 0 or (off <= 0).all(), "off by %g more than the bound at %s" % (off.max().item(), off.argmax().item())


# ------------------------------------------------------------------------------------ CPU
def test_frequencies():
    inv, scale = mrl.rotary_frequencies(8, base=10000.0)
    assert inv.dtype is torch.float64 and scale == 1.0
    assert torch.allclose(inv, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-14)
    lin, scale = mrl.rotary_frequencies(8, scaling="linear", factor=4.0)
    assert torch.allclose(lin, inv / 4, rtol=1e-14) and scale == 1.0
    # pairs that turn often stay, those that hardly turn are stretched, in between neither
    for scaling in ("yarn", "bands"):
        own, _ = mrl.rotary_frequencies(128, base=1e6)
        got, scale = mrl.rotary_frequencies(128, base=1e6, scaling=scaling, factor=4.0, trained=32768)
        turns = 32768 * own / (2 * math.pi)
        ratio = got / own
        assert (ratio <= 1 + 1e-12).all() and (ratio >= 0.25 - 1e-12).all() and (ratio.diff() <= 1e-12).all()
        assert torch.allclose(ratio[turns > 64], torch.ones(1, dtype=torch.float64)) and torch.allclose(
            ratio[turns < 0.5], torch.full((1,), 0.25, dtype=torch.float64))
        assert scale == (0.1 * math.log(4.0) + 1.0 if scaling == "yarn" else 1.0)
    got, _ = mrl.rotary_frequencies(64, scaling="bands", factor=8.0, trained=8192, fast=4.0, slow=1.0)
    own, _ = mrl.rotary_frequencies(64)
    share = ((8192 * own / (2 * math.pi) - 1) / 3).clamp(0, 1)
    assert torch.allclose(got, own * share + own / 8 * (1 - share), rtol=1e-13)
    assert all(torch.equal(mrl.rotary_frequencies(64, scaling=s, factor=1.0, trained=100)[0], own) or
               torch.allclose(mrl.rotary_frequencies(64, scaling=s, factor=1.0, trained=100)[0], own, rtol=1e-14) for s in ("yarn", "bands"))
    for kw in (dict(part=7), dict(part=0), dict(base=1.0), dict(factor=0.5), dict(scaling="yarn"), dict(scaling="other"),
               dict(scaling="bands", trained=100, fast=1.0, slow=1.0)):
        with pytest.raises(ValueError):
            mrl.rotary_frequencies(**{"part": 8, **kw})


def test_refused_arguments():
    q, k, pos = torch.zeros(5, 2, 8), torch.zeros(5, 1, 8), torch.zeros(5, dtype=torch.int64)
    inv, _ = mrl.rotary_frequencies(8)
    for kw, error in [(dict(q=q.double()), TypeError), (dict(k=k.half()), TypeError), (dict(q=q[0]), ValueError),
                      (dict(k=k[:4]), ValueError), (dict(k=k[None]), ValueError), (dict(inv_freq=inv[None]), TypeError),
                      (dict(inv_freq=inv.half()), TypeError), (dict(inv_freq=inv[:0]), TypeError), (dict(start=1), ValueError), (dict(start=-7), ValueError),
                      (dict(start=-9), ValueError), (dict(scale=float("nan")), ValueError), (dict(position_ids=pos.float()), TypeError),
                      (dict(position_ids=pos[:4]), ValueError), (dict(position_ids=pos.expand(2, 5)), ValueError),
                      (dict(q=q.expand(3, 5, 2, 8), k=None, position_ids=pos.expand(2, 5)), ValueError),
                      (dict(q=q[:, :0]), ValueError), (dict(inv_freq=torch.cat([inv, inv])), ValueError), (dict(), RuntimeError)]:
        with pytest.raises(error):
            mrl.rotary(**{"q": q, "k": k, "position_ids": pos, "inv_freq": inv, **kw})


def test_entry_point_refuses_and_launches_nothing():
    lib = _lib.load()
    buf = (ctypes.c_char * 4096)()
    p = (ctypes.addressof(buf) + 15) // 16 * 16

    def call(q=None, k=None, dtype=_lib.F32, pos=p, pdtype=_lib.I64, outer=1, inner=2, inv=p, part=8, scale=1.0, **side):
        fields = dict(x=p, out=p + 1024, heads=2, dim=8, start=0, stride_outer=0, stride_inner=16, stride_head=8)
        s = RotarySide(**{**fields, **side})
        return lib.mrl_rotary(ctypes.addressof(s) if q is None else q, ctypes.addressof(s) if k is None else None, dtype, pos, pdtype, 0, 1,
                              outer, inner, inv, part, 0, scale, 0, None)

    for rc, kw in [(-2, dict(dtype=_lib.I32)), (-2, dict(pdtype=_lib.F32)), (-1, dict(outer=-1)), (-1, dict(inner=-1)),
                   (-2, dict(inner=1 << 26)), (-2, dict(outer=1 << 40, inner=1 << 40)), (-1, dict(part=7)), (-1, dict(part=0)),
                   (-2, dict(part=4096, dim=4096)), (-1, dict(part=10)), (-1, dict(start=1)), (-1, dict(start=-1)), (-1, dict(heads=0)),
                   (-2, dict(heads=1 << 24)), (-1, dict(scale=float("inf"))), (-1, dict(x=None)), (-1, dict(out=None)), (-1, dict(pos=None)),
                   (-1, dict(inv=None)), (-3, dict(x=p + 2)), (-3, dict(pos=p + 4)), (-3, dict(inv=p + 4)), (0, dict(inner=0, x=None))]:
        assert call(**kw) == rc, kw
    assert lib.mrl_rotary(None, None, _lib.F32, p, _lib.I64, 0, 1, 1, 1, p, 8, 0, 1.0, 0, None) == -1


# ------------------------------------------------------------------------------------ GPU
@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    torch.cuda.set_device(0)
    return torch.device("cuda:0")


def make(dev, tokens, heads, dims, dtype, seed, far=1 << 20):
    g = torch.Generator(device=dev).manual_seed(seed)
    xs = [torch.randn(tokens, h, d, generator=g, device=dev).to(dtype) for h, d in zip(heads, dims)]
    grads = [torch.randn(x.shape, generator=g, device=dev).to(dtype) for x in xs]
    return xs, grads, torch.randint(0, far, (tokens,), generator=g, device=dev)


# heads, dims of q and k, the turned part, where it starts
LAYOUTS = [((2, 1), (2, 2), 2, 0), ((3, 1), (8, 8), 8, 0), ((28, 4), (128, 128), 128, 0), ((4, 4), (64, 64), 32, 0), ((5, 1), (80, 80), 20, 0),
           ((4, 2), (96, 96), 96, 0), ((3, 2), (72, 72), 72, 0), ((16, 1), (192, 64), 64, -64), ((2, 1), (10, 10), 6, 3), ((2, 2), (100, 100), 50, 25),
           ((7, 1), (256, 256), 64, 192), ((1, 1), (34, 34), 34, 0), ((2, 1), (1024, 1024), 1024, 0), ((70, 3), (24, 24), 8, 8)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=lambda t: str(t).split(".")[-1])
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "pairs"])
@pytest.mark.parametrize("heads,dims,part,start", LAYOUTS, ids=lambda v: str(v).replace(" ", ""))
def test_forward_and_backward(dev, heads, dims, part, start, interleaved, dtype):
    inv, _ = mrl.rotary_frequencies(part, base=1e4, device=dev)
    for tokens, scale in ((1, 1.0), (37, 1.25), (2100, 1.0)):
        (q, k), grads, pos = make(dev, tokens, heads, dims, dtype, tokens)
        q.requires_grad_(), k.requires_grad_()
        out = mrl.rotary(q, k, pos, inv, interleaved=interleaved, start=start, scale=scale)
        got = torch.autograd.grad(out, [q, k], grads)
        for x, y, g, d in zip((q, k), out, grads, got):
            assert y.dtype is dtype and y.shape == x.shape and d.dtype is dtype and d.shape == x.shape
            within(y.detach(), turned(x.detach(), pos, inv, interleaved, start, scale))
            within(d, turned(g, pos, inv, interleaved, start, scale, back=True))
            # what is not turned is copied
            begin = start % x.shape[-1]
            rest = [slice(0, begin), slice(begin + part, None)]
            assert all(torch.equal(y[..., s], x[..., s]) and torch.equal(d[..., s], g[..., s]) for s in rest)
        alone, none = mrl.rotary(q.detach(), None, pos, inv, interleaved=interleaved, start=start, scale=scale)
        assert none is None and torch.equal(alone, out[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_strides_batches_and_positions(dev, dtype):
    """Views of one projection's output, [s, b] batches, heads apart from one another, entries apart; positions of 32 bits, shared
    by a batch, in a column, expanded: as the dense tensors'."""
    b, s, hq, hk, d = 3, 7, 6, 2, 64
    inv, _ = mrl.rotary_frequencies(d, device=dev)
    g = torch.Generator(device=dev).manual_seed(1)
    whole = torch.randn(b, s, (hq + 2 * hk) * d + 3, generator=g, device=dev).to(dtype)
    pos = torch.randint(0, 100000, (b, s), generator=g, device=dev)
    for off in (0, 1, 3):
        q = whole[..., off:off + hq * d].unflatten(-1, (hq, d))
        k = whole[..., off + hq * d:off + (hq + hk) * d].unflatten(-1, (hk, d))
        for p in (pos, pos.int(), pos[:1], pos[1], pos.t().contiguous().t(), pos[:, :1].expand(b, s)):
            out = mrl.rotary(q, k, p, inv)
            for x, y in zip((q, k), out):
                assert y.is_contiguous()
                within(y, turned(x, p.expand(b, s), inv, False, 0, 1.0))
        for way in (lambda t: t.transpose(0, 1).contiguous().transpose(0, 1), lambda t: t.transpose(1, 2).contiguous().transpose(1, 2),
                    lambda t: t.transpose(2, 3).contiguous().transpose(2, 3), lambda t: t[:, :, :1].expand(t.shape), lambda t: t.flip(1)):
            vq, vk = (way(t).detach().requires_grad_() for t in (q, k))
            out = mrl.rotary(vq, vk, pos, inv, interleaved=True)
            ups = [way(torch.randn(x.shape, generator=g, device=dev).to(dtype)) for x in out]
            for x, y, u, gr in zip((vq, vk), out, ups, torch.autograd.grad(out, [vq, vk], ups)):
                within(y.detach(), turned(x.detach(), pos, inv, True, 0, 1.0))
                within(gr, turned(u, pos, inv, True, 0, 1.0, back=True))
    # packed: [1, tokens] of position ids
    flat = q.reshape(b * s, hq, d)
    assert torch.equal(mrl.rotary(flat, None, pos.reshape(1, -1), inv)[0], mrl.rotary(q, None, pos, inv)[0].view(flat.shape))
    # fp32 frequencies are taken as they are
    within(mrl.rotary(flat, None, pos.reshape(-1), inv.float())[0], turned(flat, pos.reshape(-1), inv.float(), False, 0, 1.0))


@pytest.mark.gpu
def test_far_and_negative_positions(dev):
    """Where fp32 angles would have lost all their digits; positions of both signs; whole and half turns."""
    inv, _ = mrl.rotary_frequencies(64, base=1e6, device=dev)
    pos = torch.tensor([0, 1, -1, 2 ** 20, 2 ** 24 + 1, 2 ** 31 - 1, -2 ** 31, 2 ** 36 + 5, 99999], device=dev)
    q = torch.randn(len(pos), 3, 64, device=dev)
    within(mrl.rotary(q, None, pos, inv)[0], turned(q, pos, inv, False, 0, 1.0))
    few = pos[:7]
    assert torch.equal(mrl.rotary(q[:7], None, few.int(), inv)[0], mrl.rotary(q[:7], None, few, inv)[0])
    assert torch.equal(mrl.rotary(q[:1], None, pos[:1], inv)[0], q[:1])
    # quarter turns come out exactly
    quarter = torch.tensor([math.pi / 2], dtype=torch.float64, device=dev)
    x = torch.tensor([[[3.0, 5.0]]], device=dev).expand(8, 1, 2).contiguous()
    y = mrl.rotary(x, None, torch.arange(8, device=dev), quarter)[0].view(8, 2).cpu()
    want = torch.tensor([[3, 5], [-5, 3], [-3, -5], [5, -3]] * 2, dtype=torch.float32)
    assert (y - want).abs().max() <= 8 * 9 * U
    # turned there and back is where it was, but for roundings
    there = mrl.rotary(q, None, pos, inv)[0]
    assert (mrl.rotary(there, None, -pos, inv)[0] - q).abs().max() <= 60 * U * q.abs().max()


@pytest.mark.gpu
def test_values_that_are_not_finite_stay_in_their_pair(dev):
    inv, _ = mrl.rotary_frequencies(16, device=dev)
    q = torch.randn(4, 2, 24, device=dev)
    pos = torch.arange(4, device=dev) + 5
    want = mrl.rotary(q, None, pos, inv)[0]
    bad = q.clone()
    bad[1, 0, 3], bad[2, 1, 20] = float("nan"), float("inf")       # a pair's first entry, and one that is copied
    got = mrl.rotary(bad, None, pos, inv)[0]
    assert torch.isnan(got[1, 0, [3, 11]]).all() and got[2, 1, 20] == float("inf")
    got[1, 0, [3, 11]], got[2, 1, 20] = want[1, 0, [3, 11]], want[2, 1, 20]
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_asked_gradients_and_differences(dev):
    """Gradients of q alone, of k alone, of a part of an expanded k; the derivative along a direction by a difference."""
    inv, _ = mrl.rotary_frequencies(32, device=dev)
    (q, k), (gq, gk), pos = make(dev, 9, (4, 1), (32, 32), F32, 3, far=100)
    for need in ((1, 0), (0, 1), (1, 1)):
        ts = [t.clone().requires_grad_(bool(n)) for t, n in zip((q, k), need)]
        out = mrl.rotary(*ts, pos, inv)
        (out[0] * gq).sum().add((out[1] * gk).sum()).backward()
        for t, g, n in zip(ts, (gq, gk), need):
            assert (t.grad is not None) == bool(n)
            if n:
                within(t.grad, turned(g, pos, inv, False, 0, 1.0, back=True))
    # only one of the results is used
    ts = [t.clone().requires_grad_() for t in (q, k)]
    mrl.rotary(*ts, pos, inv)[1].backward(gk)
    assert ts[0].grad is None or not ts[0].grad.any()
    within(ts[1].grad, turned(gk, pos, inv, False, 0, 1.0, back=True))
    # one key head for all query heads
    one = k.clone().requires_grad_()
    shared, _ = mrl.rotary(one.expand(9, 4, 32), None, pos, inv)
    (g,) = torch.autograd.grad(shared, [one], gq)
    y, e = turned(gq, pos, inv, False, 0, 1.0, back=True)
    within(g, (y.sum(1, keepdim=True), e.sum(1, keepdim=True) + 4 * U * y.abs().sum(1, keepdim=True)))
    # a central difference of the formula: the map is linear, so only the roundings of 64 bits are left
    way = torch.randn(q.shape, device=dev)
    ql = q.clone().requires_grad_()
    (g,) = torch.autograd.grad(mrl.rotary(ql, None, pos, inv)[0], [ql], gq)
    f = lambda t: (turned_wide(q.double() + t * way.double(), pos, inv) * gq.double()).sum()  # noqa: E731
    slope = (f(0.5) - f(-0.5)).item()
    bound = (turned(gq, pos, inv, False, 0, 1.0, back=True)[1] * way.double().abs()).sum()
    assert abs((g.double() * way.double()).sum() - slope) <= bound * 1.01 + 1e-9


@pytest.mark.gpu
def test_empty_streams_graphs_and_second_derivatives(dev):
    inv, _ = mrl.rotary_frequencies(64, device=dev)
    e = torch.zeros(0, 2, 64, device=dev, requires_grad=True)
    y, _ = mrl.rotary(e, None, torch.zeros(0, dtype=torch.int64, device=dev), inv)
    y.sum().backward()
    assert y.shape == e.shape == e.grad.shape
    e4 = torch.zeros(2, 0, 3, 64, device=dev)
    assert mrl.rotary(e4, e4, torch.zeros(2, 0, dtype=torch.int64, device=dev), inv)[1].shape == e4.shape

    def new(seed):
        (q, k), grads, pos = make(dev, 150, (6, 2), (64, 64), BF16, seed)
        return [q, k, *grads, pos]

    def step(q, k, gq, gk, pos):
        ts = [t.detach().requires_grad_() for t in (q, k)]
        out = mrl.rotary(*ts, pos, inv)
        return (*(t.detach() for t in out), *torch.autograd.grad(out, ts, [gq, gk]))

    static = [t.clone() for t in new(1)]
    want = step(*static)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(*static)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(*static)
    for k in range(4):
        fresh = new(20 + k)
        for t, n in zip(static, fresh):
            t.copy_(n)
        eager = step(*fresh)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(captured, eager))
    ql = static[0].float().requires_grad_()
    (g,) = torch.autograd.grad(mrl.rotary(ql, None, static[4], inv)[0].square().sum(), [ql], create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    with pytest.raises(ValueError, match="inv_freq"):
        mrl.rotary(ql, None, static[4], inv.clone().requires_grad_())


@pytest.mark.gpu
def test_nothing_is_written_outside(dev):
    """Outputs of every layout keep what lies around them; tokens in front of and behind the last are as they were."""
    for (hq, hk), (dq, dk), part, start in LAYOUTS:
        inv, _ = mrl.rotary_frequencies(part, device=dev)
        for dtype in (F32, BF16):
            (q, k), _, pos = make(dev, 11, (hq, hk), (dq, dk), dtype, 2)
            sides, wholes = [], []
            for x in (q, k):
                whole = torch.full((x.numel() + 129,), 77, dtype=dtype, device=dev)
                out = whole[65:65 + x.numel()]
                begin = start % x.shape[-1]
                sides.append(RotarySide(x.data_ptr(), out.data_ptr(), x.shape[1], x.shape[2], begin, 0, x.stride(0), x.stride(1)))
                wholes.append((whole, out.view(x.shape), x))
            _lib.call("mrl_rotary", ctypes.addressof(sides[0]), ctypes.addressof(sides[1]), _lib.dtype_code(q), pos.data_ptr(), _lib.I64, 0, 1,
                      1, 11, inv.data_ptr(), part, 1, 1.0, 0, _lib.stream(dev))
            for whole, out, x in wholes:
                within(out, turned(x, pos, inv, True, start, 1.0))
                assert (whole[:65] == 77).all() and (whole[65 + x.numel():] == 77).all()


@pytest.mark.gpu
def test_more_entries_than_31_bits(dev):
    """Tokens behind 2^31 entries: the bits that those tokens alone have."""
    inv, _ = mrl.rotary_frequencies(128, device=dev)
    tokens = 2 ** 31 // (28 * 128) + 1000
    q = torch.zeros(tokens, 28, 128, dtype=BF16, device=dev)
    (tail, _), _, pos = make(dev, 64, (28, 1), (128, 128), BF16, 4)
    q[-64:] = tail
    positions = torch.zeros(tokens, dtype=torch.int64, device=dev)
    positions[-64:] = pos
    y, _ = mrl.rotary(q, None, positions, inv)
    assert torch.equal(y[-64:], mrl.rotary(tail, None, pos, inv)[0]) and not y[:-64].any()


def test_entry_point_refuses_launches_that_do_not_fit():
    """A wavefront a token of more than 32 units, four in a workgroup of 256 threads: from 2^26 - 3 tokens on that is 2^32 threads.  In front of
    any launch, so the buffers may be anything."""
    lib = _lib.load()
    buf = (ctypes.c_char * 64)()
    p = (ctypes.addressof(buf) + 15) // 16 * 16
    for heads, dim, part in ((33, 2, 2), (64, 2, 2), (65, 2, 2), (40, 128, 128)):
        side = RotarySide(p, p, heads, dim, 0, 0, heads * dim, dim)
        for tokens in (2 ** 26 - 3, 2 ** 26 - 1):
            for dtype in (_lib.F32, _lib.BF16):
                for shape in ((1, tokens), (tokens, 1)):
                    rc = lib.mrl_rotary(ctypes.addressof(side), None, dtype, p, _lib.I64, 0, 1, *shape, p, part, 0, 1.0, 0, None)
                    assert rc == -2 and b"threads" in lib.mrl_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,heads", [(2 ** 26 - 1, 2), (2 ** 26 - 4, 33)])
def test_as_many_tokens_as_a_launch_holds(dev, tokens, heads):
    """The last tokens have the bits that they alone have; one more of many heads is refused."""
    inv, _ = mrl.rotary_frequencies(2, device=dev)
    q = torch.zeros(tokens, heads, 2, dtype=BF16, device=dev)
    (tail, _), _, pos = make(dev, 5, (heads, 1), (2, 2), BF16, 6)
    q[-5:] = tail
    positions = torch.zeros(tokens, dtype=torch.int32, device=dev)
    positions[-5:] = pos
    y, _ = mrl.rotary(q, None, positions, inv)
    assert torch.equal(y[-5:], mrl.rotary(tail, None, pos, inv)[0]) and not y[:-5].any()
    if heads > 32:
        with pytest.raises(_lib.MrlError, match="threads"):
            mrl.rotary(q[:1].expand(tokens + 1, heads, 2), None, positions[:1].expand(tokens + 1), inv)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,interleaved,heads,dim,part,start", [(BF16, True, (32, 2), 128, 128, 0), (F16, False, (7, 1), 256, 128, 128), (F32, False, (2, 2), 64, 64, 0),
                                                                    (F32, True, (9, 2), 96, 64, 32)], ids=str)
def test_much_data(dev, dtype, interleaved, heads, dim, part, start):
    """Past the caches: more than 256 MiB read and written, heads of whole lines; many heads and few, both layouts, there and back."""
    size = torch.finfo(dtype).bits // 8
    tokens = (256 << 20) // (2 * sum(heads) * dim * size) + 301
    inv, _ = mrl.rotary_frequencies(part, base=1e4, device=dev)
    (q, k), grads, pos = make(dev, tokens, heads, (dim, dim), dtype, 7)
    q.requires_grad_(), k.requires_grad_()
    out = mrl.rotary(q, k, pos, inv, interleaved=interleaved, start=start, scale=1.25)
    got = torch.autograd.grad(out, [q, k], grads)
    for x, y, g, d in zip((q, k), out, grads, got):
        within(y.detach(), turned(x.detach(), pos, inv, interleaved, start, 1.25))
        within(d, turned(g, pos, inv, interleaved, start, 1.25, back=True))


def test_frequencies_have_their_schemes_own_borders():
    """Unless it is given, a pair stays from 32 turns on ("yarn") or from 4 on ("bands")."""
    for scaling, fast in (("yarn", 32.0), ("bands", 4.0)):
        kw = dict(base=5e5, scaling=scaling, factor=8.0, trained=8192)
        inv, scale = mrl.rotary_frequencies(128, **kw)
        want, wanted_scale = mrl.rotary_frequencies(128, fast=fast, slow=1.0, **kw)
        assert torch.equal(inv, want) and scale == wanted_scale
    own, _ = mrl.rotary_frequencies(128, base=5e5)
    bands, _ = mrl.rotary_frequencies(128, base=5e5, scaling="bands", factor=8.0, trained=8192)
    turns = 8192 * own / (2 * math.pi)
    assert torch.equal(bands[turns >= 4], own[turns >= 4]) and ((turns >= 4) & (turns < 32)).any()
