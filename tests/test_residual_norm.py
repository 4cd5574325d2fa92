"""RMS norm with the residual's addition, and with an output in 8 bits, against the formula in 64 bits, and what they refuse."""
import ctypes

import pytest
import torch

import mindspeed_rl_amd as mrl
from mindspeed_rl_amd import _lib

U = 2.0 ** -24                                      # half a step of fp32
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}      # least steps
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def formula(x, r, w, eps, dy=None, dh=None):
    """h, y, d, dw in 64 bits and a bound for each entry of what fp32 arithmetic and one rounding may be off by.

    h: the sum of two numbers is rounded to fp32 and from there to the stream's type, by both: no bound.  A sum of n fp32 terms
    whose chains have at most D additions is off by at most D U sum|terms|.  Rows: D = H / 64 + 16 (at least 64 lanes share
    a row, 16 for their joining).  Columns: D = R / 128 + 272 (slabs of rows, then their sums).  mean h^2 is off by (D + 2) U of itself, its
    root's reciprocal by half of that and three roundings: n by (D + 10) U |n| amply."""
    h = x if r is None else (x.float() + r.float()).to(r.dtype)
    half, tiny, whalf, wtiny = HALF[x.dtype], TINY[x.dtype], HALF[w.dtype], TINY[w.dtype]
    z, w = h.double(), w.double()
    rows, n = z.reshape(-1, z.shape[-1]).shape
    d, dr = n / 64 + 16, rows / 128 + 272
    s = (z.square().mean(-1, keepdim=True) + eps).sqrt()
    n = z / s
    en = n.abs() * (d + 10) * U
    y = n * w
    exact = w.abs() * en + 4 * U * y.abs()
    out = {"h": h, "y": (y, exact + half * y.abs() + tiny), "wide": (y, exact)}
    if dy is None:
        return out
    dy, dh = dy.double(), torch.zeros_like(z) if dh is None else dh.double()
    g = dy * w
    mgn = (g * n).mean(-1, keepdim=True)
    emgn = (d + 4) * U * (g * n).abs().mean(-1, keepdim=True) + (g.abs() * en).mean(-1, keepdim=True)
    inner = (g - n * mgn) / s
    total = inner + dh
    # products and differences, the sum's error, n's, r's; then the addition of dh
    e = (3 * U * (g.abs() + (n * mgn).abs()) + n.abs() * emgn + en * mgn.abs()) / s * 1.01 + inner.abs() * (d + 10) * U + U * total.abs()
    out["dx"] = (total, e + half * total.abs() + tiny)
    out["dr"] = (total, e + HALF[h.dtype] * total.abs() + TINY[h.dtype])
    col = lambda t: t.reshape(-1, t.shape[-1]).sum(0)  # noqa: E731
    dw = col(dy * n)
    out["dw"] = (dw, col(dy.abs() * en) + (dr + 3) * U * col((dy * n).abs()) + whalf * dw.abs() * 1.01 + wtiny)
    return out


def within(got, want):
    value, bound = want
    assert torch.isfinite(got).all()
    off = (got.double() - value).abs() - bound * 1.01
    assert off.numel() == 0 or (off <= 0).all(), "off by %g more than the bound at %s" % (off.max().item(), off.argmax().item())


def check_codes(q, scale, wide, block):
    """q scale is y to the nearest code: half a step of e4m3 is 2^-4 of the value, or 2^-10 of the scale below the least normal number.
    The scale is the largest |y| over 448, of which y's own error and two roundings."""
    y, e = wide
    parts = lambda t: t.unflatten(-1, (-1, block or t.shape[-1]))  # noqa: E731
    y, e, q = parts(y), parts(e), parts(q.double())
    s = scale.double().unsqueeze(-1)
    want = (y.abs().amax(-1, keepdim=True) / 448).clamp(min=2.0 ** -126)
    assert ((s - want).abs() <= (e.amax(-1, keepdim=True) / 448 + 3 * U * want) * 1.01).all()
    assert (q.abs() <= 448).all()
    off = (q * s - y).abs()
    assert (off <= (e + torch.maximum(2.0 ** -4 * (y.abs() + e), 2.0 ** -10 * s)) * (1 + 4 * U) * 1.001).all()


def make(dev, shape, dtype, rtype, wdtype, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    h = shape[-1]
    return (n(*shape).to(dtype), (n(*shape) * 2 + 0.3).to(rtype), (1 + 0.3 * n(h)).to(wdtype), n(*shape).to(dtype), n(*shape).to(rtype))


# ------------------------------------------------------------------------------------ refusals (CPU)
def test_refused_arguments():
    x, w = torch.zeros(2, 128), torch.ones(128)
    for bad, error in [(lambda: mrl.add_rms_norm(x.double(), x, w), TypeError), (lambda: mrl.add_rms_norm(x, x.half(), w), TypeError),
                       (lambda: mrl.add_rms_norm(x, x, w.half()), TypeError), (lambda: mrl.add_rms_norm(x, x[:1], w), ValueError),
                       (lambda: mrl.add_rms_norm(x, x, w[:7]), ValueError), (lambda: mrl.add_rms_norm(x, x, w[None]), ValueError),
                       (lambda: mrl.add_rms_norm(torch.zeros(2, 0), torch.zeros(2, 0), torch.ones(0)), ValueError),
                       (lambda: mrl.add_rms_norm(x, x, w, eps=0.0), ValueError), (lambda: mrl.add_rms_norm(x, x, w, eps=float("nan")), ValueError),
                       (lambda: mrl.add_rms_norm(x, x, w), RuntimeError), (lambda: mrl.rms_norm_fp8(x, w), RuntimeError)]:
        with pytest.raises(error):
            bad()


def test_entry_points_refuse_and_launch_nothing():
    lib = _lib.load()
    buf = (ctypes.c_char * 8192)()
    p = (ctypes.addressof(buf) + 15) // 16 * 16
    most = 1 << 20

    def fwd(x=p, dtype=_lib.F32, xs=8, r=p, rtype=_lib.F32, rs=8, rows=2, hidden=8, w=p, wdtype=_lib.F32, eps=1e-5, h=p, y=p):
        return lib.mrl_add_norm_fwd(x, dtype, xs, r, rtype, rs, rows, hidden, w, wdtype, eps, h, y, None, None)

    for rc, kw in [(-2, dict(dtype=_lib.I32)), (-2, dict(wdtype=_lib.BF16)), (-2, dict(rtype=_lib.BF16)), (-1, dict(rows=-1)),
                   (-1, dict(hidden=0)), (-2, dict(hidden=most + 1, xs=most + 1, rs=most + 1)), (-2, dict(rows=1 << 24)),
                   (-2, dict(rows=1 << 62)), (-2, dict(rows=1 << 22, hidden=8192, xs=8192, rs=8192)), (-1, dict(xs=7)), (-1, dict(rs=7)), (-1, dict(eps=0.0)), (-1, dict(eps=float("nan"))),
                   (-1, dict(x=None)), (-1, dict(r=None)), (-1, dict(h=None)), (-1, dict(r=None, h=None)), (-1, dict(w=None)),
                   (-1, dict(y=None)), (-3, dict(x=p + 2)), (-3, dict(y=p + 1)), (-3, dict(h=p + 2)), (0, dict(rows=0, x=None))]:
        assert fwd(**kw) == rc, kw

    def fp8(r=None, h=None, hidden=128, block=128, scale=p, q=p, stride=128):
        return lib.mrl_norm_fp8_fwd(p, _lib.F32, stride, r, _lib.F32, stride, 2, hidden, p, _lib.F32, 1e-5, block, h, q, scale, None)

    for rc, kw in [(-2, dict(block=64)), (-2, dict(hidden=120)), (-1, dict(r=p)), (-1, dict(h=p)), (-1, dict(scale=None)),
                   (-1, dict(q=None)), (-3, dict(scale=p + 2)), (-1, dict(stride=100))]:
        assert fp8(**kw) == rc, kw
    need = lib.mrl_add_norm_bwd_workspace_bytes(2, 8)
    assert need > 0 and lib.mrl_add_norm_bwd_workspace_bytes(0, 8) == 0 and lib.mrl_add_norm_bwd_workspace_bytes(2, most + 1) == 0

    def bwd(dy=p, dys=8, dh=p, dhs=8, h=p, rtype=_lib.F32, dtype=_lib.F32, rows=2, hidden=8, w=p, wdtype=_lib.F32, rstd=p, dx=p, dr=None,
            dw=p, ws=p, n=need):
        return lib.mrl_add_norm_bwd(dy, dys, dh, dhs, h, rtype, dtype, rows, hidden, w, wdtype, rstd, dx, dr, dw, ws, n, None)

    for rc, kw in [(-2, dict(dtype=_lib.I64)), (-2, dict(wdtype=_lib.F16)), (-2, dict(rtype=_lib.F16)), (-1, dict(dys=7)), (-1, dict(dhs=7)),
                   (-1, dict(dy=None)), (-1, dict(h=None)), (-1, dict(w=None)), (-1, dict(rstd=None)), (-1, dict(ws=None)),
                   (-1, dict(n=need - 1)), (-3, dict(ws=p + 4)), (-3, dict(dx=p + 2)), (-3, dict(dr=p + 2)), (-3, dict(rstd=p + 2)),
                   (0, dict(rows=0, dw=None))]:
        assert bwd(**kw) == rc, kw


def test_loss_objects_refuse_a_residual_that_is_not_added():
    fn = mrl.LossFuncFactory.get_instance("ray_grpo", "actor")
    fn.add_loss_meta_info({"clip_ratio": 0.2, "kl_ctrl": mrl.FixedKLController(0.0), "kl_penalty": "low_var_kl", "entropy_coeff": 0.0})
    batch = {"responses": torch.zeros(1, 2), "response_length": torch.ones(1, 1), "prompt_length": torch.ones(1, 1),
             "labels": torch.zeros(1, 4, dtype=torch.int64), "advantages": torch.zeros(1, 2)}
    hidden, w, head = torch.zeros(1, 4, 8), torch.ones(8), torch.zeros(16, 8)
    for forward_only in (False, True):
        with pytest.raises(ValueError, match="lm_head_weight"):
            fn.compute_loss(hidden, batch, forward_only=forward_only, final_norm_residual=hidden)
        for kw in (dict(), dict(final_norm_type="layer", final_norm_weight=w)):
            with pytest.raises(ValueError, match="final_norm_residual"):
                fn.compute_loss(hidden, batch, forward_only=forward_only, lm_head_weight=head, final_norm_residual=hidden, **kw)


# ------------------------------------------------------------------------------------ GPU
@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    torch.cuda.set_device(0)
    return torch.device("cuda:0")


SHAPES = [(1, 1), (1, 2), (3, 7), (1, 64), (2, 63), (5, 257), (33, 512), (4, 1000), (31, 1343), (9, 2048), (64, 3584), (7, 4104),
          (5, 8192), (3, 16384), (2, 16392), (2, 20011), (3, 70001), (1000, 96), (2500, 72), (1, 3584), (700, 8), (513, 128), (3, 32768)]
TYPES = [(F32, F32, F32), (BF16, BF16, BF16), (F16, F16, F16), (BF16, F32, F32), (F16, F32, F16), (BF16, BF16, F32), (BF16, F32, BF16)]
names = lambda t: str(t).split(".")[-1]  # noqa: E731


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,rtype,wdtype", TYPES, ids=names)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_forward_and_backward(dev, shape, dtype, rtype, wdtype):
    eps = 1e-5
    x, r, w, dy, dh = make(dev, shape, dtype, rtype, wdtype, 1)
    want = formula(x, r, w, eps, dy, dh)
    leaves = [t.requires_grad_() for t in (x, r, w)]
    y, h = mrl.add_rms_norm(x, r, w, eps)
    assert y.shape == x.shape and y.dtype is dtype and h.shape == x.shape and h.dtype is rtype
    assert torch.equal(h, want["h"])
    within(y.detach(), want["y"])
    grads = torch.autograd.grad([y, h], leaves, [dy, dh])
    for name, g, leaf in zip(("dx", "dr", "dw"), grads, leaves):
        assert g.dtype is leaf.dtype and g.shape == leaf.shape
        within(g, want[name])
    # the same call gives the same bits, without gradients too
    with torch.no_grad():
        again = mrl.add_rms_norm(x, r, w, eps)
    assert torch.equal(again[0], y) and torch.equal(again[1], h)
    again = torch.autograd.grad(mrl.add_rms_norm(x, r, w, eps), leaves, [dy, dh])
    assert all(torch.equal(p, q) for p, q in zip(again, grads))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,rtype,wdtype", TYPES, ids=names)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_eight_bits(dev, shape, dtype, rtype, wdtype):
    x, r, w, _, _ = make(dev, shape, dtype, rtype, wdtype, 2)
    for res in (None, r):
        for block in (None, 128) if shape[-1] % 128 == 0 else (None,):
            got = mrl.rms_norm_fp8(x, w, 1e-5, residual=res, block=block)
            want = formula(x, res, w, 1e-5)
            assert got[0].dtype is torch.float8_e4m3fn and got[0].shape == x.shape and got[1].dtype is F32
            assert got[1].shape == (*shape[:-1], shape[-1] // 128 if block else 1)
            check_codes(got[0].float(), got[1], want["wide"], block)
            assert len(got) == (2 if res is None else 3) and (res is None or torch.equal(got[2], want["h"]))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,rtype,rows,hidden", [(BF16, BF16, 26001, 1343), (F32, F32, 30000, 616), (F16, F32, 33000, 1032)], ids=str)
def test_much_data(dev, dtype, rtype, rows, hidden):
    x, r, w, dy, dh = make(dev, (rows, hidden), dtype, rtype, dtype, 13)
    want = formula(x, r, w, 1e-5, dy, dh)
    leaves = [t.requires_grad_() for t in (x, r, w)]
    y, h = mrl.add_rms_norm(x, r, w, 1e-5)
    assert torch.equal(h, want["h"])
    within(y.detach(), want["y"])
    grads = torch.autograd.grad([y, h], leaves, [dy, dh])
    for name, g in zip(("dx", "dr", "dw"), grads):
        within(g, want[name])
    again = torch.autograd.grad(mrl.add_rms_norm(x, r, w, 1e-5), leaves, [dy, dh])
    assert all(torch.equal(p, q) for p, q in zip(again, grads))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,rtype", [(F32, F32), (BF16, BF16), (BF16, F32)], ids=names)
def test_strides_and_places(dev, dtype, rtype):
    """Rows apart, rows that start off a vector, a transposed batch, columns apart, a residual and upstream gradients that are
    expanded: as the dense tensors'."""
    for h, off in ((512, 0), (512, 1), (1343, 3), (40, 5), (128, 8)):
        x, r, w, dy, dh = make(dev, (24, h), dtype, rtype, dtype, 2)

        def wide(t):
            o = torch.full((24, h + 24), float("nan"), dtype=t.dtype, device=dev)
            o[:, off:off + h] = t
            return o[:, off:off + h]

        ways = [wide, lambda t: t.view(4, 6, h).transpose(0, 1), lambda t: t.t().contiguous().t(), lambda t: t.view(2, 3, 4, h),
                lambda t: t[:1].expand(24, h)]
        for way in ways:
            vx, vr, vdy, vdh = (way(t) for t in (x, r, dy, dh))
            leaves = [vx.detach().requires_grad_(), vr.detach().requires_grad_(), w.clone().requires_grad_()]
            y, hs = mrl.add_rms_norm(*leaves, 1e-5)
            want = formula(vx, vr, w, 1e-5, vdy, vdh)
            assert torch.equal(hs, want["h"])
            within(y.detach(), want["y"])
            for name, g in zip(("dx", "dr", "dw"), torch.autograd.grad([y, hs], leaves, [vdy, vdh])):
                within(g, want[name])
            got = mrl.rms_norm_fp8(vx, w, 1e-5, residual=vr)
            check_codes(got[0].float(), got[1], formula(vx, vr, w, 1e-5)["wide"], None)


@pytest.mark.gpu
@pytest.mark.parametrize("rtype", [BF16, F32], ids=names)
def test_asked_gradients(dev, rtype):
    """Only what is asked for, from either output or both; a weight shared by two norms; the stream through two layers."""
    x, r, w, dy, dh = make(dev, (40, 136), BF16, rtype, BF16, 3)
    for up in ((1, 1), (1, 0), (0, 1)):
        want = formula(x, r, w, 1e-5, dy if up[0] else torch.zeros_like(dy), dh if up[1] else None)
        for need in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 0), (1, 1, 1)):
            ts = [t.detach().clone().requires_grad_(bool(n)) for t, n in zip((x, r, w), need)]
            y, h = mrl.add_rms_norm(*ts, 1e-5)
            outs = [(o, g) for o, g, u in zip((y, h), (dy, dh), up) if u]
            torch.autograd.backward([o for o, _ in outs], [g for _, g in outs])
            for t, name, n in zip(ts, ("dx", "dr", "dw"), need):
                assert (t.grad is not None) == bool(n)
                if n:
                    within(t.grad, want[name])
    # gradients that meet: x and the residual one tensor
    t, wl = r.detach().clone().requires_grad_(), w.float().requires_grad_()
    if rtype is BF16:
        y, h = mrl.add_rms_norm(t, t, wl, 1e-5)
        (g,) = torch.autograd.grad([y, h], [t], [dy, dh])
        d, e = formula(t.detach(), t.detach(), wl.detach(), 1e-5, dy, dh)["dx"]
        within(g, (2 * d, 2 * e + 2.0 ** -8 * (2 * d).abs()))
    # empty batches
    e = torch.zeros(0, 5, 136, device=dev, requires_grad=True)
    y, h = mrl.add_rms_norm(e, e, wl)
    assert y.shape == h.shape == (0, 5, 136)
    y.sum().backward()
    assert e.grad.shape == e.shape and torch.equal(wl.grad, torch.zeros_like(wl))
    q, s = mrl.rms_norm_fp8(e.detach(), wl.detach())
    assert q.shape == (0, 5, 136) and s.shape == (0, 5, 1)


@pytest.mark.gpu
def test_against_differences(dev):
    """The derivative along a direction of a function of both outputs, formed in 64 bits by a central difference."""
    x, r, w, dy, dh = make(dev, (6, 200), F32, F32, F32, 4)
    leaves = [t.requires_grad_() for t in (x, r, w)]
    grads = torch.autograd.grad(mrl.add_rms_norm(*leaves, 1e-5), leaves, [dy, dh])
    want = formula(x.detach(), r.detach(), w.detach(), 1e-5, dy, dh)
    g = torch.Generator(device=dev).manual_seed(5)
    ways = [torch.randn(t.shape, generator=g, device=dev).double() for t in leaves]

    def at(t):
        a, b, c = (p.detach().double() + t * v for p, v in zip(leaves, ways))
        h = a + b
        return ((h / (h.square().mean(-1, keepdim=True) + 1e-5).sqrt() * c) * dy.double()).sum() + (h * dh.double()).sum()

    slope = (at(1e-5) - at(-1e-5)) / 2e-5
    got = sum((p.double() * v).sum() for p, v in zip(grads, ways))
    bound = sum((want[k][1] * v.abs()).sum() for k, v in zip(("dx", "dr", "dw"), ways))
    # h is rounded to fp32 by the call and not by the difference: n moves by U |h| / s in each entry, and y's share of the slope
    # by that times second derivatives of the order of one: U times the sum of all terms, amply by 10
    terms = sum((p.double() * v).abs().sum() for p, v in zip(grads, ways))
    assert abs(got - slope) <= bound + 10 * U * terms + 1e-6 * abs(slope)


@pytest.mark.gpu
@pytest.mark.parametrize("rtype", [F32, BF16], ids=names)
def test_values_where_it_can_go_wrong(dev, rtype):
    """Rows of zeros and of one value, tiny and huge ones, sums that cancel; what is not finite stays in its row (its block)."""
    n = 1024
    x, r, w, dy, dh = make(dev, (12, n), rtype, rtype, rtype, 6)
    x[1], r[1] = 7.25, 0.0
    x[2], r[2] = 0.0, 0.0
    x[3] = -r[3]
    x[4], r[4] = x[4] * 1e-18, r[4] * 1e-18
    x[6], r[6] = x[6] * 1e15, r[6] * 1e15
    want = formula(x, r, w, 1e-5, dy, dh)
    leaves = [t.clone().requires_grad_() for t in (x, r, w)]
    y, h = mrl.add_rms_norm(*leaves, 1e-5)
    grads = torch.autograd.grad([y, h], leaves, [dy, dh])
    assert torch.equal(h, want["h"])
    within(y.detach(), want["y"])
    within(grads[0], want["dx"])
    q, s, _ = mrl.rms_norm_fp8(x, w, 1e-5, residual=r)
    check_codes(q.float(), s, want["wide"], None)
    assert not q[2].float().any() and s[2].item() == 2.0 ** -126
    qb, sb, _ = mrl.rms_norm_fp8(x, w, 1e-5, residual=r, block=128)
    check_codes(qb.float(), sb, want["wide"], 128)
    bad = x.clone()
    bad[5, 3], bad[7, n - 1], bad[9, 0] = float("nan"), float("inf"), float("-inf")
    fine = [i for i in range(12) if i not in (5, 7, 9)]
    bl = bad.clone().requires_grad_()
    y2, h2 = mrl.add_rms_norm(bl, r, w, 1e-5)
    (dx2,) = torch.autograd.grad([y2, h2], [bl], [dy, dh])
    assert torch.equal(y2[fine], y[fine]) and torch.equal(dx2[fine], grads[0][fine])
    z = (bad.float() + r.float()).to(rtype).double()
    ref = z / (z.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w.double()
    assert torch.equal(torch.isnan(y2), torch.isnan(ref)) and torch.isnan(dx2[[5, 7, 9]]).any(1).all()
    q2, s2, _ = mrl.rms_norm_fp8(bad, w, 1e-5, residual=r)
    assert torch.equal(q2[fine].float(), q[fine].float()) and torch.equal(s2[fine], s[fine])
    assert not torch.isfinite(s2[[5, 7, 9]]).any()


@pytest.mark.gpu
def test_rows_at_the_end_of_the_range(dev):
    """3 584 squares of at most 2.9e17 add up inside fp32; of twice as large entries they do not: zeros, and the stream's gradient alone."""
    for n in (3584, 40000):
        x, r, w, dy, dh = make(dev, (4, n), F32, F32, F32, 15)
        top = 2.9e17 * (3584 / n) ** 0.5
        x = torch.sign(x) * top * torch.linspace(0.5, 1.0, n, device=dev) - r
        want = formula(x, r, w, 1e-5, dy, dh)
        leaves = [x.requires_grad_(), r.requires_grad_()]
        y, h = mrl.add_rms_norm(*leaves, w, 1e-5)
        within(y.detach(), want["y"])
        within(torch.autograd.grad([y, h], [x], [dy, dh])[0], want["dx"])
        far = [(2 * x).detach().requires_grad_(), (2 * r).detach()]
        y, h = mrl.add_rms_norm(*far, w, 1e-5)
        assert not y.any() and torch.equal(torch.autograd.grad([y, h], far[:1], [dy, dh])[0], dh)


@pytest.mark.gpu
def test_nothing_is_written_outside(dev):
    """Outputs of every width keep what lies around them, and the workspace what lies behind it."""
    pad = 64
    for rows, n in ((1, 1), (3, 7), (5, 64), (9, 257), (40, 1343), (3, 3584), (2, 20011), (130, 128)):
        x, r, w, dy, dh = make(dev, (rows, n), BF16, F32, BF16, 7)
        want = formula(x, r, w, 1e-5, dy, dh)

        def guarded(count, dtype):
            t = torch.full((count + 2 * pad + 1,), 77, dtype=dtype, device=dev)
            return t, t[pad + 1:pad + 1 + count]            # starts off a vector

        sizes = dict(h=(rows * n, F32), y=(rows * n, BF16), rstd=(rows, F32), dx=(rows * n, BF16), dr=(rows * n, F32), dw=(n, BF16),
                     q=(rows * n, torch.uint8), h2=(rows * n, F32), scale=(rows, F32))
        bufs = {k: guarded(*v) for k, v in sizes.items()}
        p = {k: v[1].data_ptr() for k, v in bufs.items()}
        s = _lib.stream(dev)
        _lib.call("mrl_add_norm_fwd", x.data_ptr(), _lib.BF16, n, r.data_ptr(), _lib.F32, n, rows, n, w.data_ptr(), _lib.BF16, 1e-5, p["h"],
                  p["y"], p["rstd"], s)
        _lib.call("mrl_norm_fp8_fwd", x.data_ptr(), _lib.BF16, n, r.data_ptr(), _lib.F32, n, rows, n, w.data_ptr(), _lib.BF16, 1e-5, 0,
                  p["h2"], p["q"], p["scale"], s)
        size = _lib.load().mrl_add_norm_bwd_workspace_bytes(rows, n)
        ws = torch.full((size + 64,), 77, dtype=torch.uint8, device=dev)
        _lib.call("mrl_add_norm_bwd", dy.data_ptr(), n, dh.data_ptr(), n, p["h"], _lib.F32, _lib.BF16, rows, n, w.data_ptr(), _lib.BF16,
                  p["rstd"], p["dx"], p["dr"], p["dw"], ws.data_ptr(), size, s)
        for name in ("y", "dx", "dr", "dw"):
            within(bufs[name][1].view(want[name][0].shape), want[name])
        assert torch.equal(bufs["h"][1].view(rows, n), want["h"]) and torch.equal(bufs["h2"][1].view(rows, n), want["h"])
        check_codes(bufs["q"][1].view(torch.float8_e4m3fn).view(rows, n).float(), bufs["scale"][1].view(rows, 1), want["wide"], None)
        assert (ws[size:] == 77).all()
        for whole, part in bufs.values():
            assert (whole[:pad + 1] == 77).all() and (whole[pad + 1 + part.numel():] == 77).all()


@pytest.mark.gpu
def test_streams_and_graphs(dev):
    """On another stream, and captured with its backward and replayed with new inputs between eager passes."""
    def new(seed):
        return make(dev, (200, 256), BF16, F32, BF16, seed)

    static = [t.clone() for t in new(8)]
    side = torch.cuda.Stream()

    def step(x, r, w, dy, dh):
        ts = [t.detach().requires_grad_() for t in (x, r, w)]
        y, h = mrl.add_rms_norm(*ts)
        q, s, _ = mrl.rms_norm_fp8(x, w, residual=r, block=128)
        return (y.detach(), h.detach(), q.float(), s, *torch.autograd.grad([y, h], ts, [dy, dh]))

    want = step(*static)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(*static)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    del want, got
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


@pytest.mark.gpu
def test_once_differentiable_and_without_gradients_in_eight_bits(dev):
    x, r, w, dy, _ = make(dev, (3, 128), F32, F32, F32, 9)
    xl = x.clone().requires_grad_()
    y, _ = mrl.add_rms_norm(xl, r, w)
    (g,) = torch.autograd.grad(y, [xl], dy, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    for kw in (dict(x=xl, weight=w), dict(x=x, weight=w.clone().requires_grad_()), dict(x=x, weight=w, residual=xl)):
        with pytest.raises(RuntimeError, match="no gradient"):
            mrl.rms_norm_fp8(**kw)
        with torch.no_grad():
            mrl.rms_norm_fp8(**kw)
    for bad in (dict(block=64), dict(block=0.5), dict(block=128, x=x[:, :100], weight=w[:100])):
        with pytest.raises(ValueError):
            mrl.rms_norm_fp8(**{"x": x, "weight": w, **bad})


@pytest.mark.gpu
def test_more_entries_than_31_bits(dev):
    """Rows behind 2^31 entries: the bits that those rows alone have."""
    rows, n = 600001, 3584
    x, r, w, dy, dh = make(dev, (64, n), BF16, BF16, BF16, 10)
    big = [torch.zeros(rows, n, dtype=BF16, device=dev) for _ in range(2)]
    for b, t in zip(big, (x, r)):
        b[-64:] = t
    y, h = mrl.add_rms_norm(*big, w)
    few = mrl.add_rms_norm(x, r, w)
    assert torch.equal(y[-64:], few[0]) and torch.equal(h[-64:], few[1]) and not y[:-64].any() and not h[:-64].any()
    del y, h
    for b, t in zip(big, (x, r)):
        b[-64:] = t
    q, s, _ = mrl.rms_norm_fp8(big[0], w, residual=big[1])
    q1, s1, _ = mrl.rms_norm_fp8(x, w, residual=r)
    assert torch.equal(q[-64:].view(torch.uint8), q1.view(torch.uint8)) and torch.equal(s[-64:], s1)


@pytest.mark.gpu
@pytest.mark.parametrize("hidden", [4, 256, 512, 1024, 4096, 65536])
@pytest.mark.parametrize("dtype,rtype", [(BF16, None), (F16, F32), (BF16, BF16), (F32, F32), (F32, None)], ids=lambda t: str(t).split(".")[-1])
def test_codes_are_quotients(dev, dtype, rtype, hidden):
    """Rows of 1 and -1, whose norm is +- the weight itself, so that y is known to the bit: the scale is max |y| times 1/448, one rounding,
    and a code the nearest to the fp32 quotient y / scale, ties to even.  Weights lie at and right beside the middle between two codes."""
    gen = torch.Generator().manual_seed(hidden)
    for block in (None, 128):
        if block and hidden % block:
            continue
        size = block or hidden
        most = 1 + torch.rand(hidden // size, 1, generator=gen)
        s = most * (1 / 448)
        # 8 to 15 and a half, in the binades below 448
        middle = (torch.randint(8, 16, (hidden // size, size), generator=gen) + 0.5) * torch.exp2(torch.randint(-12, 5, (hidden // size, size), generator=gen).float())
        w = (middle * s).clamp(max=most)
        beside = torch.randint(-1, 2, w.shape, generator=gen)
        w = torch.where(beside == 0, w, torch.nextafter(w, torch.where(beside > 0, most, 0.0)))
        w[:, -1:] = most
        want = (w / s).to(torch.float8_e4m3fn).float().view(-1)
        ones = torch.randint(0, 2, (5, hidden), generator=gen) * 2.0 - 1
        x = ones.to(dev, dtype)
        kw = {} if rtype is None else dict(residual=(2 * x).to(rtype))
        q, scale, *h = mrl.rms_norm_fp8(-x if kw else x, w.view(-1).to(dev), eps=1e-30, block=block, **kw)
        assert all(torch.equal(t.float(), x.float()) for t in h)
        assert torch.equal(scale.cpu(), s.view(1, -1).expand(5, -1))
        assert torch.equal(q.cpu().float(), want * ones)


@pytest.mark.gpu
@pytest.mark.parametrize("hidden", [256, 4096, 65536])
def test_codes_of_zeros_and_under_an_infinite_scale(dev, hidden):
    """Numbers over infinity are zeros, infinity over it is NaN; a zero keeps its sign."""
    w = torch.ones(hidden, device=dev)
    w[1], w[2] = 0.0, -0.0
    x = torch.ones(2, hidden, device=dev)
    for block in (None, 128):
        q, scale = mrl.rms_norm_fp8(x, w, eps=1e-30, block=block)
        assert torch.isfinite(scale).all() and (q.view(torch.uint8)[:, 1] == 0).all() and (q.view(torch.uint8)[:, 2] == 0x80).all()
        bad = w.clone()
        bad[0] = float("inf")
        q, scale = mrl.rms_norm_fp8(x, bad, eps=1e-30, block=block)
        end = block or hidden
        assert torch.isinf(scale[:, 0]).all() and torch.isnan(q[:, 0].float()).all() and not q[:, 1:end].float().any()
        assert torch.isfinite(scale[:, 1:]).all() and (q[:, end:].float() == 448).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,rtype,rows,hidden", [(BF16, BF16, 32800, 2048), (BF16, BF16, 16500, 4091), (F16, F16, 17000, 3840), (F32, F32, 33001, 1022),
                                                     (F32, F32, 16400, 2048), (F16, F32, 32790, 1024), (BF16, F32, 16401, 2045)], ids=str)
def test_much_data_in_teams_of_two_vectors(dev, dtype, rtype, rows, hidden):
    """128 MiB of rows that two vectors a lane hold, whole and not, with and without a gradient of the sum."""
    x, r, w, dy, dh = make(dev, (rows, hidden), dtype, rtype, dtype, 15)
    leaves = [t.requires_grad_() for t in (x, r, w)]
    for up in (dh, None):
        y, h = mrl.add_rms_norm(x, r, w, 1e-5)
        grads = torch.autograd.grad([y] if up is None else [y, h], leaves, [dy] if up is None else [dy, up])
        with torch.no_grad():
            want = formula(x, r, w, 1e-5, dy, up)
            assert torch.equal(h, want["h"])
            within(y.detach(), want["y"])
            for name, g in zip(("dx", "dr", "dw"), grads):
                within(g, want[name])
        del want, y, h, grads


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,rtype,rows,hidden", [(BF16, BF16, 13001, 1024), (BF16, BF16, 101, 128 * 1024), (F16, F32, 8300, 1024), (F32, F32, 50000, 128), (BF16, BF16, 26001, 512)],
                         ids=str)
def test_much_data_in_eight_bits(dev, dtype, rtype, rows, hidden):
    """Past the caches: more than 96 MiB read and written."""
    x, r, w, _, _ = make(dev, (rows, hidden), dtype, rtype, dtype, 16)
    for res in (r, None):
        for block in (None, 128):
            want = formula(x, res, w, 1e-5)
            got = mrl.rms_norm_fp8(x, w, 1e-5, residual=res, block=block)
            check_codes(got[0].float(), got[1], want["wide"], block)
            assert res is None or torch.equal(got[2], want["h"])


@pytest.mark.gpu
def test_gradients_behind_31_bits(dev):
    """Rows behind 2^31 entries have the gradients that they alone have; the weight's is off by the order of its sums alone."""
    rows, n = 600001, 3584
    few = make(dev, (64, n), BF16, BF16, BF16, 17)
    x, r, dy, dh = (torch.zeros(rows, n, dtype=BF16, device=dev) for _ in range(4))
    for b, t in zip((x, r, dy, dh), (few[0], few[1], few[3], few[4])):
        b[-64:] = t
    x, r, w = (t.requires_grad_() for t in (x, r, few[2]))
    y, h = mrl.add_rms_norm(x, r, w)
    dx, dw = torch.autograd.grad([y, h], [x, w], [dy, dh])
    fx, fr = few[0].requires_grad_(), few[1].requires_grad_()
    small = torch.autograd.grad(mrl.add_rms_norm(fx, fr, w), [fx], [few[3], few[4]])
    assert torch.equal(dx[-64:], small[0]) and not dx[:-64].any()
    del y, h, dx
    with torch.no_grad():
        within(dw, formula(fx, fr, w, 1e-6, few[3], few[4])["dw"])
