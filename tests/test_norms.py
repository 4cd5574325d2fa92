"""Layer norm and RMS norm against the formula in 64 bits, forward and backward, and what they refuse."""
import ctypes

import pytest
import torch

import mindspeed_rl_amd as mrl
from mindspeed_rl_amd import _lib

U = 2.0 ** -24                                      # half a step of fp32
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}      # least steps


def formula(x, w, b, eps, layer, dy=None):
    """y, dx, dw, db in 64 bits and a bound for each entry of what fp32 arithmetic and one rounding may be off by.

    A sum of n fp32 terms whose chains have at most D additions is off by at most D U sum|terms|.  Rows: D = H / 64 + 16
    (at least 64 lanes share a row, 16 for their joining).  Columns: D = R / 128 + 272 (slabs of rows, then their sums).
    With a = mean|x| and s = sqrt(var + eps): mu is off by D U a; n = (x - mu) / s by (D + 10) U |n| + (D + 2) U a / s, where
    the mean's error enters var only in second order, ((D U a) / s)^2 relative."""
    half, tiny = HALF[x.dtype], TINY[x.dtype]
    whalf, wtiny = HALF[w.dtype], TINY[w.dtype]
    x, w = x.double(), w.double()
    b = None if b is None else b.double()
    rows, h = x.reshape(-1, x.shape[-1]).shape
    d, dr = h / 64 + 16, rows / 128 + 272
    a = x.abs().mean(-1, keepdim=True)
    c = x - x.mean(-1, keepdim=True) if layer else x
    s = (c.square().mean(-1, keepdim=True) + eps).sqrt()
    n = c / s
    shift = (d + 2) * U * a / s if layer else 0.0 * a
    en = n.abs() * ((d + 10) * U + shift.square()) + shift
    y = n * w + (0 if b is None else b)
    ey = w.abs() * en + 4 * U * ((n * w).abs() + (0 if b is None else b.abs())) + half * y.abs() + tiny
    out = {"y": (y, ey)}
    if dy is None:
        return out
    dy = dy.double()
    g = dy * w
    mg = g.mean(-1, keepdim=True) if layer else torch.zeros_like(a)
    mgn = (g * n).mean(-1, keepdim=True)
    emg = (d + 2) * U * g.abs().mean(-1, keepdim=True) if layer else 0.0
    emgn = (d + 4) * U * (g * n).abs().mean(-1, keepdim=True) + (g.abs() * en).mean(-1, keepdim=True)
    dx = (g - mg - n * mgn) / s
    edx = (3 * U * (g.abs() + mg.abs() + (n * mgn).abs()) + emg + n.abs() * emgn + en * mgn.abs()) / s * 1.01
    out["dx"] = (dx, edx + dx.abs() * ((d + 10) * U + shift.square() + half) + tiny)
    r = lambda t: t.reshape(-1, h).sum(0)  # noqa: E731
    dw, db = r(dy * n), r(dy)
    out["dw"] = (dw, r(dy.abs() * en) + (dr + 3) * U * r((dy * n).abs()) + whalf * dw.abs() * 1.01 + wtiny)
    out["db"] = (db, dr * U * r(dy.abs()) + whalf * db.abs() * 1.01 + wtiny)
    return out


def within(got, want):
    value, bound = want
    assert torch.isfinite(got).all()
    off = (got.double() - value).abs() - bound * 1.01
    assert (off <= 0).all(), "off by %g more than the bound at %s" % (off.max().item(), off.argmax().item())


def apply(kind, x, w, b, eps):
    return mrl.layer_norm(x, w, b, eps=eps) if kind == "layer" else mrl.rms_norm(x, w, eps=eps)


def make(dev, shape, dtype, wdtype, seed, bias=True):
    g = torch.Generator(device=dev).manual_seed(seed)
    h = shape[-1]
    x = (torch.randn(*shape, generator=g, device=dev) * 2 + 0.3).to(dtype)
    w = (1 + 0.3 * torch.randn(h, generator=g, device=dev)).to(wdtype)
    b = (0.2 * torch.randn(h, generator=g, device=dev)).to(wdtype) if bias else None
    return x, w, b, torch.randn(*shape, generator=g, device=dev).to(dtype)


# ------------------------------------------------------------------------------------ refusals (CPU)
def test_refused_arguments():
    x, w = torch.zeros(2, 8), torch.ones(8)
    for bad, error in [(lambda: mrl.layer_norm(x.double(), w), TypeError), (lambda: mrl.layer_norm(x, w.half()), TypeError),
                       (lambda: mrl.layer_norm(x, torch.ones(7)), ValueError),
                       (lambda: mrl.layer_norm(x, torch.ones(1, 8)), ValueError),
                       (lambda: mrl.layer_norm(x, w, torch.ones(7)), ValueError),
                       (lambda: mrl.layer_norm(x, w, w.half()), ValueError),
                       (lambda: mrl.layer_norm(torch.zeros(2, 0), torch.ones(0)), ValueError),
                       (lambda: mrl.layer_norm(torch.tensor(1.0), torch.ones(1)), ValueError),
                       (lambda: mrl.rms_norm(x, w, eps=0.0), ValueError),
                       (lambda: mrl.rms_norm(x, w, eps=float("nan")), ValueError),
                       (lambda: mrl.rms_norm(x, w, eps=float("inf")), ValueError),
                       (lambda: mrl.rms_norm(x, w), RuntimeError), (lambda: mrl.layer_norm(x, w, w), RuntimeError)]:
        with pytest.raises(error):
            bad()


def test_entry_points_refuse_and_launch_nothing():
    lib = _lib.load()
    buf = (ctypes.c_char * 4096)()
    p = (ctypes.addressof(buf) + 15) // 16 * 16
    most = 1 << 20

    def fwd(x=p, dtype=_lib.F32, rows=2, hidden=8, stride=8, w=p, b=None, wdtype=_lib.F32, layer=1, eps=1e-5, y=p):
        return lib.mrl_norm_fwd(x, dtype, rows, hidden, stride, w, b, wdtype, layer, eps, y, None, None, None)

    for rc, kw in [(-2, dict(dtype=_lib.I32)), (-2, dict(wdtype=_lib.BF16)), (-1, dict(rows=-1)), (-1, dict(hidden=0)),
                   (-2, dict(hidden=most + 1, stride=most + 1)), (-2, dict(rows=1 << 31)), (-2, dict(rows=(1 << 28), hidden=8)), (-1, dict(stride=7)),
                   (-1, dict(eps=0.0)), (-1, dict(eps=float("nan"))), (-1, dict(b=p, layer=0)), (-1, dict(x=None)),
                   (-1, dict(w=None)), (-1, dict(y=None)), (-3, dict(x=p + 2)), (-3, dict(y=p + 1)), (0, dict(rows=0, x=None))]:
        assert fwd(**kw) == rc, kw
    need = lib.mrl_norm_bwd_workspace_bytes(2, 8)
    assert need > 0 and lib.mrl_norm_bwd_workspace_bytes(0, 8) == 0 and lib.mrl_norm_bwd_workspace_bytes(2, most + 1) == 0

    def bwd(dy=p, dys=8, x=p, xs=8, dtype=_lib.F32, rows=2, hidden=8, w=p, wdtype=_lib.F32, rstd=p, dx=p, dw=p, ws=p, n=need):
        return lib.mrl_norm_bwd(dy, dys, x, xs, dtype, rows, hidden, w, wdtype, None, rstd, dx, dw, None, ws, n, None)

    for rc, kw in [(-2, dict(dtype=_lib.I64)), (-2, dict(wdtype=_lib.F16)), (-1, dict(dys=7)), (-1, dict(xs=7)),
                   (-1, dict(dy=None)), (-1, dict(x=None)), (-1, dict(w=None)), (-1, dict(rstd=None)), (-1, dict(ws=None)),
                   (-1, dict(n=need - 1)), (-3, dict(ws=p + 4)), (-3, dict(dx=p + 2)), (-3, dict(rstd=p + 2)),
                   (0, dict(rows=0, dw=None))]:
        assert bwd(**kw) == rc, kw


def test_workspace_of_few_rows():
    """Two sums of a column for every row, and for no more than the most workgroups."""
    size = _lib.load().mrl_norm_bwd_workspace_bytes
    for h in (1, 1000, 1 << 20):
        assert size(1, h) == 8 * h and size(4, h) == 32 * h
        assert all(size(n, h) <= size(n + 1, h) <= size(1 << 20, h) <= 512 * 8 * h for n in (1, 15, 16, 17, 255, 256, 511, 512, 513, 4096))


def test_loss_objects_refuse_a_norm_that_is_not_applied():
    fn = mrl.LossFuncFactory.get_instance("ray_grpo", "actor")
    fn.add_loss_meta_info({"clip_ratio": 0.2, "kl_ctrl": mrl.FixedKLController(0.0), "kl_penalty": "low_var_kl",
                           "entropy_coeff": 0.0})
    batch = {"responses": torch.zeros(1, 2), "response_length": torch.ones(1, 1), "prompt_length": torch.ones(1, 1),
             "labels": torch.zeros(1, 4, dtype=torch.int64), "advantages": torch.zeros(1, 2)}
    w, head = torch.ones(8), torch.zeros(16, 8)
    with pytest.raises(ValueError, match="lm_head_weight"):
        fn.compute_loss(torch.zeros(1, 4, 8), batch, final_norm_weight=w)
    with pytest.raises(ValueError, match="lm_head_weight"):
        fn.compute_loss(torch.zeros(1, 4, 8), batch, forward_only=True, final_norm_weight=w)
    for kw in (dict(final_norm_type="group", final_norm_weight=w), dict(final_norm_bias=w),
               dict(final_norm_bias=w, final_norm_weight=w)):
        for forward_only in (False, True):
            with pytest.raises(ValueError, match="final_norm"):
                fn.compute_loss(torch.zeros(1, 4, 8), batch, forward_only=forward_only, lm_head_weight=head, **kw)


# ------------------------------------------------------------------------------------ GPU
@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    torch.cuda.set_device(0)
    return torch.device("cuda:0")


SHAPES = [(1, 1), (1, 2), (3, 7), (1, 64), (2, 63), (5, 257), (33, 512), (4, 1000), (31, 1343), (9, 2048), (64, 3584), (7, 4104),
          (5, 8192), (3, 16384), (2, 16392), (2, 20011), (3, 70001), (1000, 96), (2500, 72), (1, 3584)]
TYPES = [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
         (torch.bfloat16, torch.float32), (torch.float16, torch.float32)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("dtype,wdtype", TYPES, ids=lambda t: str(t).split(".")[-1])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_forward_and_backward(dev, shape, dtype, wdtype, kind):
    eps = 1e-5
    x, w, b, dy = make(dev, shape, dtype, wdtype, 1, kind == "layer")
    want = formula(x, w, b, eps, kind == "layer", dy)
    leaves = [t.requires_grad_() for t in (x, w, b) if t is not None]
    y = apply(kind, x, w, b, eps)
    assert y.shape == x.shape and y.dtype is dtype
    grads = torch.autograd.grad(y, leaves, dy)
    within(y.detach(), want["y"])
    for name, g, leaf in zip(("dx", "dw", "db"), grads, leaves):
        assert g.dtype is leaf.dtype and g.shape == leaf.shape
        within(g, want[name])
    # the same call gives the same bits, without gradients too
    with torch.no_grad():
        assert torch.equal(apply(kind, x, w, b, eps), y)
    again = torch.autograd.grad(apply(kind, x, w, b, eps), leaves, dy)
    assert all(torch.equal(p, q) for p, q in zip(again, grads))


@pytest.mark.gpu
@pytest.mark.parametrize("kind,dtype,rows,hidden", [("layer", torch.bfloat16, 26001, 1343), ("rms", torch.float32, 30000, 616),
                                                    ("rms", torch.float16, 33000, 1032)])
def test_much_data(dev, kind, dtype, rows, hidden):
    """Rows of 64 MiB and more, whose backward deals them out differently."""
    x, w, b, dy = make(dev, (rows, hidden), dtype, dtype, 13, kind == "layer")
    want = formula(x, w, b, 1e-5, kind == "layer", dy)
    leaves = [t.requires_grad_() for t in (x, w, b) if t is not None]
    y = apply(kind, x, w, b, 1e-5)
    grads = torch.autograd.grad(y, leaves, dy)
    within(y.detach(), want["y"])
    for name, g in zip(("dx", "dw", "db"), grads):
        within(g, want[name])
    again = torch.autograd.grad(apply(kind, x, w, b, 1e-5), leaves, dy)
    assert all(torch.equal(p, q) for p, q in zip(again, grads))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_strides_and_places(dev, dtype, kind):
    """Rows apart, rows that start off a vector, a transposed batch, columns apart: as the dense tensor's."""
    for h, off in ((512, 0), (512, 1), (1343, 3), (40, 5)):
        x, w, b, dy = make(dev, (24, h), dtype, dtype, 2, kind == "layer")
        wide = torch.full((24, h + 24), float("nan"), dtype=dtype, device=dev)
        wide_dy = wide.clone()
        wide[:, off:off + h], wide_dy[:, off:off + h] = x, dy
        views = [(wide[:, off:off + h], wide_dy[:, off:off + h])]
        views.append((x.view(4, 6, h).transpose(0, 1), dy.view(4, 6, h).transpose(0, 1)))
        views.append((x.t().contiguous().t(), dy.t().contiguous().t()))
        views.append((x.view(2, 3, 4, h), dy.view(2, 3, 4, h)))
        for v, vdy in views:
            v = v.detach().requires_grad_()
            wl = w.clone().requires_grad_()
            y = apply(kind, v, wl, b, 1e-5)
            dx, dw = torch.autograd.grad(y, [v, wl], vdy)
            want = formula(v.detach(), w, b, 1e-5, kind == "layer", vdy)
            within(y.detach(), want["y"])
            within(dx, want["dx"])
            within(dw, want["dw"])


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_narrow_wide_and_frozen_rows(dev, dtype, kind):
    """Rows of less than a vector, many of them; rows that no team holds, apart from one another; the vectors' gradients alone."""
    for rows, h in ((3001, 3), (700, 7), (21, 20011), (40, 16396)):
        x, w, b, dy = make(dev, (rows, h), dtype, dtype, 7, kind == "layer")
        wide = torch.full((rows, h + 3), float("nan"), dtype=dtype, device=dev)
        wide[:, 1:1 + h] = x
        want = formula(x, w, b, 1e-5, kind == "layer", dy)
        leaves = [wide[:, 1:1 + h].detach().requires_grad_()] + [t.requires_grad_() for t in (w, b) if t is not None]
        y = apply(kind, leaves[0], w, b, 1e-5)
        within(y.detach(), want["y"])
        for name, g in zip(("dx", "dw", "db"), torch.autograd.grad(y, leaves, dy)):
            within(g, want[name])
        y = apply(kind, x, w, b, 1e-5)
        for name, g in zip(("dw", "db"), torch.autograd.grad(y, leaves[1:], dy)):
            within(g, want[name])


@pytest.mark.gpu
def test_asked_gradients_and_broadcast_upstream(dev):
    """Only what is asked for is computed; an upstream gradient of one value; a vector shared by two norms."""
    x, w, b, _ = make(dev, (40, 136), torch.float32, torch.float32, 3)
    ones = torch.ones_like(x)
    want = formula(x, w, b, 1e-5, True, ones)
    for need in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1), (1, 1, 1)):
        ts = [t.clone().requires_grad_(bool(n)) for t, n in zip((x, w, b), need)]
        mrl.layer_norm(*ts, eps=1e-5).sum().backward()
        for t, name, n in zip(ts, ("dx", "dw", "db"), need):
            assert (t.grad is not None) == bool(n)
            if n:
                within(t.grad, want[name])
    wl = w.clone().requires_grad_()
    (mrl.rms_norm(x, wl, eps=1e-5).sum() + mrl.rms_norm(x[:8], wl, eps=1e-5).sum()).backward()
    one, two = formula(x, w, None, 1e-5, False, ones)["dw"], formula(x[:8], w, None, 1e-5, False, ones[:8])["dw"]
    within(wl.grad, (one[0] + two[0], one[1] + two[1] + U * (one[0] + two[0]).abs()))
    # without a bias, and empty batches
    y = mrl.layer_norm(x, w)
    within(y, formula(x, w, None, 1e-5, True)["y"])
    e = torch.zeros(0, 5, 136, device=dev, requires_grad=True)
    wl = w.clone().requires_grad_()
    y = mrl.layer_norm(e, wl, b)
    assert y.shape == (0, 5, 136)
    y.sum().backward()
    assert e.grad.shape == e.shape and torch.equal(wl.grad, torch.zeros_like(w))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_values_where_it_can_go_wrong(dev, kind):
    """A large common offset, rows of one value, rows of zeros, tiny rows, and what is not finite stays in its row."""
    h = 1000
    x, w, b, dy = make(dev, (12, h), torch.float32, torch.float32, 4, kind == "layer")
    x[0] += 300.0
    x[1] = 7.25
    x[2] = 0.0
    x[3] *= 1e-12
    x[4] *= 1e15
    want = formula(x, w, b, 1e-5, kind == "layer", dy)
    xl = x.clone().requires_grad_()
    y = apply(kind, xl, w, b, 1e-5)
    (dx,) = torch.autograd.grad(y, [xl], dy)
    within(y.detach(), want["y"])
    within(dx, want["dx"])
    bad = x.clone()
    bad[5, 3], bad[7, 999], bad[9, 0] = float("nan"), float("inf"), float("-inf")
    bl, wl = bad.requires_grad_(), w.clone().requires_grad_()
    y2 = apply(kind, bl, wl, b, 1e-5)
    dx2, dw2 = torch.autograd.grad(y2, [bl, wl], dy)
    fine = [r for r in range(12) if r not in (5, 7, 9)]
    assert torch.equal(y2[fine], y[fine]) and torch.equal(dx2[fine], dx[fine])
    plain = bad.detach().double()
    if kind == "layer":
        plain = plain - plain.mean(-1, keepdim=True)
    ref = plain / (plain.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w.double() + (0 if b is None else b.double())
    assert torch.equal(torch.isnan(y2), torch.isnan(ref)) and torch.isnan(dw2).any()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_gradient_against_differences(dev, kind):
    """The directional derivative of sum(y dy) by central differences of the formula in 64 bits.  Truncation is of third
    order in the step: below 1e-7 of the values here at 1e-4; what the kernel may be off by is its bound, entry by entry."""
    x, w, b, dy = make(dev, (6, 200), torch.float32, torch.float32, 5, kind == "layer")
    leaves = [t.requires_grad_() for t in (x, w, b) if t is not None]
    grads = torch.autograd.grad(apply(kind, x, w, b, 1e-5), leaves, dy)
    bounds = formula(x.detach(), w.detach(), None if b is None else b.detach(), 1e-5, kind == "layer", dy)
    g = torch.Generator(device=dev).manual_seed(6)

    def value(ts):
        xs, ws = ts[0], ts[1]
        c = xs - xs.mean(-1, keepdim=True) if kind == "layer" else xs
        y = c / (c.square().mean(-1, keepdim=True) + 1e-5).sqrt() * ws + (ts[2] if kind == "layer" else 0)
        return (y * dy.double()).sum()

    for k, name in enumerate(("dx", "dw", "db")[:len(leaves)]):
        v = torch.randn(leaves[k].shape, generator=g, device=dev, dtype=torch.float64)
        ends = []
        for step in (1e-4, -1e-4):
            ts = [t.detach().double() for t in leaves]
            ts[k] = ts[k] + step * v
            ends.append(value(ts))
        slope = (ends[0] - ends[1]) / 2e-4
        got = (grads[k].double() * v).sum()
        assert abs(got - slope) <= (bounds[name][1] * v.abs()).sum() + 1e-6 * (grads[k].double() * v).abs().sum()


@pytest.mark.gpu
def test_differentiated_once(dev):
    """Under create_graph the first gradient is the usual one and a second differentiation is refused; a vector alone;
    rows overwritten before the backward are noticed."""
    x, w, b, dy = make(dev, (6, 40), torch.float32, torch.float32, 12)
    xl = x.clone().requires_grad_()
    (plain,) = torch.autograd.grad(mrl.layer_norm(xl, w, b), [xl], dy)
    up = dy.clone().requires_grad_()
    (dx,) = torch.autograd.grad(mrl.layer_norm(xl, w, b), [xl], up, create_graph=True)
    assert torch.equal(dx, plain)
    with pytest.raises(RuntimeError):
        dx.sum().backward()
    assert torch.equal(mrl.rms_norm(x[2], w), mrl.rms_norm(x, w)[2])
    h = xl * 2
    y = mrl.rms_norm(h, w)
    h.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@pytest.mark.gpu
def test_two_streams_at_once(dev):
    """Steps that overlap in time, each with its own memory: the bits of a step alone."""
    sets = [make(dev, (3000, 1024), torch.bfloat16, torch.bfloat16, 30 + k) for k in range(2)]

    def step(x, w, b, dy):
        ts = [t.detach().requires_grad_() for t in (x, w, b)]
        y = mrl.layer_norm(*ts)
        return (y.detach(), *torch.autograd.grad(y, ts, dy))

    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                got[k].append(step(*sets[k]))
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(p, q) for g in got[k] for p, q in zip(g, want[k]))


@pytest.mark.gpu
def test_memory_around_the_outputs(dev):
    """Through the C ABI: nothing outside y, mean, rstd, dx, dweight and dbias is written, odd sizes and places."""
    for rows, h in ((3, 7), (5, 1343), (2, 2049), (9, 64), (1, 9000), (3, 17001)):
        x, w, b, dy = make(dev, (rows, h), torch.bfloat16, torch.bfloat16, 7)
        want = formula(x, w, b, 1e-5, True, dy)
        pad = 16

        def guarded(n, dtype):
            t = torch.full((n + 2 * pad + 1,), 77.0, dtype=dtype, device=dev)
            return t, t[pad + 1:pad + 1 + n]            # starts off a vector

        sizes = dict(y=(rows * h, torch.bfloat16), mean=(rows, torch.float32), rstd=(rows, torch.float32),
                     dx=(rows * h, torch.bfloat16), dw=(h, torch.bfloat16), db=(h, torch.bfloat16))
        bufs = {k: guarded(*v) for k, v in sizes.items()}
        p = {k: v[1].data_ptr() for k, v in bufs.items()}
        s = _lib.stream(dev)
        _lib.call("mrl_norm_fwd", x.data_ptr(), _lib.BF16, rows, h, h, w.data_ptr(), b.data_ptr(), _lib.BF16, 1, 1e-5, p["y"],
                  p["mean"], p["rstd"], s)
        n = _lib.load().mrl_norm_bwd_workspace_bytes(rows, h)
        ws, inner = torch.full((n + 64,), 77, dtype=torch.uint8, device=dev), None
        inner = ws[:n]
        _lib.call("mrl_norm_bwd", dy.data_ptr(), h, x.data_ptr(), h, _lib.BF16, rows, h, w.data_ptr(), _lib.BF16, p["mean"],
                  p["rstd"], p["dx"], p["dw"], p["db"], inner.data_ptr(), n, s)
        for name in ("y", "dx", "dw", "db"):
            within(bufs[name][1].view(want[name][0].shape), want[name])
        assert (ws[n:] == 77).all()
        for whole, part in bufs.values():
            assert (whole[:pad + 1] == 77).all() and (whole[pad + 1 + part.numel():] == 77).all()


@pytest.mark.gpu
def test_streams_and_graphs(dev):
    """On another stream, and captured with its backward and replayed with new inputs between eager passes."""
    x, w, b, dy = make(dev, (200, 264), torch.bfloat16, torch.bfloat16, 8)
    static = [t.clone() for t in (x, w, b, dy)]
    side = torch.cuda.Stream()

    def step(xs, ws, bs, d):
        ts = [t.detach().requires_grad_() for t in (xs, ws, bs)]
        y = mrl.layer_norm(*ts)
        return (y.detach(), *torch.autograd.grad(y, ts, d))

    want = step(x, w, b, dy)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(*static)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(*static)
    for k in range(4):
        nx, nw, nb, ndy = make(dev, (200, 264), torch.bfloat16, torch.bfloat16, 20 + k)
        for t, n in zip(static, (nx, nw, nb, ndy)):
            t.copy_(n)
        eager = step(nx, nw, nb, ndy)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(captured, eager))


@pytest.mark.gpu
def test_more_entries_than_31_bits(dev):
    """Rows behind 2^31 entries, forward and backward: the same bits as those rows alone have."""
    rows, h = 600001, 3584
    x = torch.zeros(rows, h, dtype=torch.bfloat16, device=dev)
    tail, w, _, dy_tail = make(dev, (64, h), torch.bfloat16, torch.bfloat16, 9)
    x[-64:] = tail
    dy = torch.zeros_like(x)
    dy[-64:] = dy_tail
    x.requires_grad_()
    y = mrl.rms_norm(x, w)
    (dx,) = torch.autograd.grad(y, [x], dy)
    want = formula(tail, w, None, 1e-6, False, dy_tail)
    within(y[-64:].detach(), want["y"])
    within(dx[-64:], want["dx"])
    assert not y[:-64].any() and not dx[:-64].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_rms_norm_with_the_gradient_of_a_bias(dev, dtype):
    """Through the C ABI: dbias is the columns' sum of dy without a mean too, whatever else is asked for, in rows of every kind,
    and what is asked for beside it has the bits that it has alone.  The workspace holds NaN where nothing was written."""
    code = _lib.dtype_code(torch.empty(0, dtype=dtype))
    for rows, h in ((1, 64), (3, 3), (5, 64), (40, 136), (700, 1000), (2500, 1024), (33, 3584), (9, 20011)):
        x, w, _, dy = make(dev, (rows, h), dtype, dtype, 14)
        want = formula(x, w, None, 1e-5, False, dy)
        y, rstd, s = torch.empty_like(x), torch.empty(rows, device=dev), _lib.stream(dev)
        _lib.call("mrl_norm_fwd", x.data_ptr(), code, rows, h, h, w.data_ptr(), None, code, 0, 1e-5, y.data_ptr(), None,
                  rstd.data_ptr(), s)
        n = _lib.load().mrl_norm_bwd_workspace_bytes(rows, h)

        def backward(need):
            out = {k: torch.full_like(like, float("nan")) for k, like, on in zip(("dx", "dw", "db"), (x, w, w), need) if on}
            ws = torch.full((n,), 255, dtype=torch.uint8, device=dev)
            _lib.call("mrl_norm_bwd", dy.data_ptr(), h, x.data_ptr(), h, code, rows, h, w.data_ptr(), code, None, rstd.data_ptr(),
                      *[out[k].data_ptr() if k in out else None for k in ("dx", "dw", "db")], ws.data_ptr(), n, s)
            return out

        for need in ((1, 1), (1, 0), (0, 1), (0, 0)):
            got = backward(need + (1,))
            for name, g in got.items():
                within(g, want[name])
            if any(need):
                assert all(torch.equal(g, got[name]) for name, g in backward(need + (0,)).items())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_rows_at_the_end_of_the_range(dev, dtype, kind):
    """3 584 squares of at most 2.9e17 add up to at most 3.02e38, inside fp32; of twice as large entries they do not: zeros, and
    the bias."""
    for h in (3584, 20011):
        x, w, b, dy = make(dev, (4, h), dtype, dtype, 15, kind == "layer")
        top = 2.9e17 * (3584 / h) ** 0.5
        x = (torch.sign(x.float()) * top * torch.linspace(0.5, 1.0, h, device=dev)).to(dtype)
        want = formula(x, w, b, 1e-5, kind == "layer", dy)
        xl = x.clone().requires_grad_()
        y = apply(kind, xl, w, b, 1e-5)
        within(y.detach(), want["y"])
        within(torch.autograd.grad(y, [xl], dy)[0], want["dx"])
        far = (x * 2).requires_grad_()
        y = apply(kind, far, w, b, 1e-5)
        assert torch.equal(y.detach(), torch.zeros_like(x) if b is None else b.expand(4, h))
        assert not torch.autograd.grad(y, [far], dy)[0].any()
