"""AdamW over many tensors against the formula in 64 bits, its moments in 8 bits against the rule of their rounding, and what it refuses."""
import ctypes
import math

import pytest
import torch

import mindspeed_rl_amd as mrl
from mindspeed_rl_amd import _lib

U = 2.0 ** -24                                      # half a step of fp32
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}      # least steps
BF16, F16, F32, E4M3 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn
HYPER = dict(lr=3e-3, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)


def held(code, scale):
    """What codes and scales stand for, in 64 bits."""
    c = code.double().reshape(-1)
    return (c * scale.double().repeat_interleave(128)[:c.numel()]).view(code.shape)


def formula(p, g, m, v, t, factor=1.0, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01):
    """p, m, v, sqrt(v) of step t in 64 bits and bounds of what fp32 arithmetic may be off by, before p is rounded to its own type.

    g' has one rounding (and the factor's: two).  m: constants, products and sum: 5 U of the terms' magnitudes.  v: 8 U.  Its root: 5 U.  The
    quotient's divisor: the root, sqrt(1 - b2^t) and two roundings: 9 U; the quotient, the rate and their product 3 U more; p (1 - lr wd): 2 U; a last one."""
    b1, b2 = betas
    p, g, m, v = (x.double() for x in (p, g, m, v))
    g = g * factor
    m1, v1 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    em = 5 * U * (b1 * m.abs() + (1 - b1) * g.abs()) + 2.0 ** -126
    ev = 8 * U * v1 + 2.0 ** -126
    root = v1.sqrt()
    er = 5 * U * root + 2.0 ** -63
    rate, second = lr / (1 - b1 ** t), 1 / math.sqrt(1 - b2 ** t)
    div = root * second + eps
    q = m1 / div * rate
    eq = rate / div * em + q.abs() * (12 * U + 2.0 ** -63 * second / div) * 1.01
    new = p * (1 - lr * weight_decay) - q
    ep = eq + 2 * U * p.abs() + U * (p.abs() + q.abs())
    return {"p": (new, ep), "m": (m1, em), "v": (v1, ev), "root": (root, er)}


def within(got, want, dtype=F32):
    value, bound = want
    assert torch.isfinite(got.float()).all()
    bound = bound if dtype is F32 else bound + HALF[dtype] * (value.abs() + bound) + TINY[dtype]
    off = (got.double() - value).abs() - bound * 1.01
    assert off.numel() == 0 or (off <= 0).all(), "off by %g more than the bound at %s" % (off.max().item(), off.argmax().item())


def dither(t, n, device):
    """16 bits for each of n entries, from the hash of the step and the pair."""
    x = torch.arange((n + 1) // 2, device=device) ^ ((t * 0x9E3779B9) & 0xffffffff)
    x = ((x ^ (x >> 16)) * 0x7feb352d) & 0xffffffff
    x = ((x ^ (x >> 15)) * 0x846ca68b) & 0xffffffff
    x = x ^ (x >> 16)
    return torch.stack([x & 0xffff, x >> 16], 1).view(-1)[:n]


def codes(x, bits, root):
    """The rule of the rounding, on values of fp32: codes (as numbers) and scales."""
    flat = x.reshape(-1)
    rows = torch.nn.functional.pad(flat, (0, -flat.numel() % 128)).view(-1, 128)
    scale = (rows.abs().amax(1) * (1 / 448)).clamp(min=2.0 ** -126)
    size = (rows * scale.reciprocal()[:, None]).view(-1)[:flat.numel()].abs().clamp(max=448.0).double()
    if root:
        size = torch.where(flat > 0, size.clamp(min=2.0 ** -9), 0.0)
    step = torch.exp2(torch.floor(torch.log2(size.clamp(min=2.0 ** -6))) - 3)
    return (torch.floor(size / step + bits * 2.0 ** -16) * step * torch.sign(flat)).view(x.shape), scale


def fp32_moments(g, m, v, factor, b1, b2):
    """m and v as fp32 arithmetic rounds them, one operation at a time."""
    g = g.float() * factor
    return m * b1 + g * (1 - b1), v * b2 + (g * g) * (1 - b2)


def factor_of(norm, limit):
    """As torch gives it: a number over a tensor is the number times the tensor's reciprocal, two roundings."""
    return torch.clamp(limit / (norm + 1e-6), max=1.0).item()


def make(dev, shapes, dtype, gdtype, seed, bits=32, master=True, scale=1e-2):
    """Parameters, gradients and a state that some steps have been taken on; some gradients are zero, some rows have none."""
    gen = torch.Generator(device=dev).manual_seed(seed)
    n = lambda s: torch.randn(s, generator=gen, device=dev)  # noqa: E731
    params = [n(s).mul(0.1).to(dtype) for s in shapes]
    grads = [(n(s) * scale * torch.exp(n(s)) * (n(s) > -1)).to(gdtype) for s in shapes]
    state = mrl.adamw_state(params, bits=bits, master=master)
    state["step"].fill_(7)
    for k, s in enumerate(shapes):
        m, d = n(s) * scale, n(s).abs() * scale * (n(s) > -1.5)
        if bits == 32:
            state["exp_avg"][k].copy_(m)
            state["exp_avg_sq"][k].copy_(d * d)
            continue
        for name, x in (("exp_avg", m), ("exp_avg_sq", d)):
            c, sc = codes(x, torch.full((x.numel(),), 32768, device=dev), name == "exp_avg_sq")
            state[name][k].copy_(c.float())
            state[name + "_scale"][k].copy_(sc)
    return params, grads, state


def clone(params, state):
    copy = lambda v: [None if t is None else t.clone() for t in v] if isinstance(v, list) else v.clone()  # noqa: E731
    return [p.clone() for p in params], {k: copy(v) for k, v in state.items()}


def check(params, grads, state, old_params, old, factor=1.0, hyper=None):
    """Every tensor of a step that was taken on (old_params, old)."""
    hyper = {**HYPER, **(hyper or {})}
    t = int(old["step"].item()) + 1
    assert state["step"].item() == t
    small = "exp_avg_scale" in old
    for k, g in enumerate(grads):
        if g is None:
            assert torch.equal(params[k], old_params[k]) and torch.equal(state["exp_avg"][k].float(), old["exp_avg"][k].float())
            continue
        w = (old.get("master") or [None] * len(grads))[k]
        if small:
            m, v = held(old["exp_avg"][k], old["exp_avg_scale"][k]), held(old["exp_avg_sq"][k], old["exp_avg_sq_scale"][k]) ** 2
        else:
            m, v = old["exp_avg"][k], old["exp_avg_sq"][k]
        want = formula(old_params[k] if w is None else w, g, m, v, t, factor, **hyper)
        if w is None:
            within(params[k], want["p"], params[k].dtype)
        else:
            within(state["master"][k], want["p"])
            assert torch.equal(params[k], state["master"][k].to(params[k].dtype))
        if not small:
            within(state["exp_avg"][k], want["m"])
            within(state["exp_avg_sq"][k], want["v"])
            continue
        # the rule to the bit, from the moments as fp32 rounds them; and at most a step of the 64-bit formula's
        fm = (m.float(), held(old["exp_avg_sq"][k], old["exp_avg_sq_scale"][k]).float().square())
        fm = fp32_moments(g, *fm, factor, *hyper["betas"])
        for name, x, root, key in (("exp_avg", fm[0], False, "m"), ("exp_avg_sq", fm[1].sqrt(), True, "root")):
            c, s = codes(x, dither(t, x.numel(), x.device), root)
            assert torch.equal(state[name + "_scale"][k], s)
            assert torch.equal(state[name][k].double(), c)
            value, bound = want[key]
            sc = s.double().repeat_interleave(128)[:x.numel()].view(x.shape)
            off = (held(state[name][k], s) - value).abs()
            assert (off <= bound + 2.0 ** -3 * (value.abs() + bound) * (1 + 4 * U) + 2.0 ** -9 * sc).all()


# ------------------------------------------------------------------------------------ refusals (CPU)
def test_refused_arguments():
    p, g = [torch.zeros(3, 4)], [torch.zeros(3, 4)]
    s = {"exp_avg": [torch.zeros(3, 4)], "exp_avg_sq": [torch.zeros(3, 4)], "step": torch.zeros((), dtype=torch.int64)}
    h = [torch.zeros(3, 4, dtype=BF16)]
    leaf = [torch.zeros(3, 4, requires_grad=True)]
    for kw, error in [(dict(params=[1.0]), TypeError), (dict(params=[p[0].double()]), TypeError), (dict(params=[p[0].t()]), ValueError),
                      (dict(params=p * 2), ValueError), (dict(grads=[]), ValueError), (dict(grads=[g[0][:2]]), ValueError),
                      (dict(grads=h), ValueError), (dict(params=h, grads=[g[0].half()]), ValueError), (dict(exp_avg=h), ValueError),
                      (dict(exp_avg_sq=[p[0].view(-1)]), ValueError), (dict(exp_avg=[torch.zeros(4, 3).t()]), ValueError), (dict(exp_avg=leaf), ValueError),
                      (dict(master=[p[0]]), ValueError), (dict(params=h, grads=h, master=h), ValueError), (dict(exp_avg_scale=[torch.ones(1)]), ValueError),
                      (dict(exp_avg_scale=[torch.ones(1)], exp_avg_sq_scale=[torch.ones(1)]), ValueError),
                      (dict(step=torch.zeros(())), TypeError), (dict(step=0), TypeError), (dict(lr=-1.0), ValueError), (dict(lr=float("nan")), ValueError),
                      (dict(lr=torch.zeros(2)), TypeError), (dict(eps=0.0), ValueError), (dict(weight_decay=-0.1), ValueError),
                      (dict(betas=(1.0, 0.9)), ValueError), (dict(betas=(0.9, -0.1)), ValueError), (dict(max_norm=1.0), ValueError),
                      (dict(grad_norm=torch.ones(())), ValueError), (dict(grad_norm=1.0, max_norm=1.0), TypeError),
                      (dict(grad_norm=torch.ones(()), max_norm=-1.0), ValueError), (dict(grad_norm=torch.ones(()), max_norm=float("nan")), ValueError),
                      (dict(), RuntimeError)]:
        with pytest.raises(error):
            mrl.adamw_(**{"params": p, "grads": g, "lr": 1e-3, **s, **kw})
    for kw, error in [(dict(params=[]), ValueError), (dict(bits=16), ValueError), (dict(params=[p[0].t()]), ValueError), (dict(), RuntimeError)]:
        with pytest.raises(error):
            mrl.adamw_state(**{"params": p, **kw})


class Tensor(ctypes.Structure):
    """struct mrl_adamw_tensor"""
    _fields_ = [(n, ctypes.c_void_p) for n in ("param", "grad", "master", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")] + [
        ("n", ctypes.c_int64), ("dtype", ctypes.c_int32), ("grad_dtype", ctypes.c_int32)]


def test_entry_point_refuses_and_launches_nothing():
    lib = _lib.load()
    buf = (ctypes.c_char * 65536)()
    p = (ctypes.addressof(buf) + 15) // 16 * 16
    at = lambda k: p + 1024 * k  # noqa: E731

    def call(count=1, bits=32, step=at(20), lr=1e-3, lr_at=None, b1=0.9, b2=0.99, eps=1e-8, wd=0.0, norm=None, most=1.0, ws=at(21), second=None, **t):
        fields = dict(param=at(0), grad=at(1), master=None, exp_avg=at(3), exp_avg_sq=at(4), exp_avg_scale=None, exp_avg_sq_scale=None, n=16,
                      dtype=_lib.F32, grad_dtype=_lib.F32)
        list_ = (Tensor * 2)(Tensor(**{**fields, **t}), Tensor(**{**fields, **(second or {})}))
        return lib.mrl_adamw_step(ctypes.addressof(list_), count, bits, step, lr, lr_at, b1, b2, eps, wd, norm, most, ws, None)

    apart = dict(param=at(10), grad=at(11), exp_avg=at(13), exp_avg_sq=at(14))
    for rc, kw in [(-1, dict(count=-1)), (-2, dict(count=16385)), (-2, dict(bits=16)), (-1, dict(step=None)), (-1, dict(ws=None)),
                   (-1, dict(lr=-1.0)), (-1, dict(lr=float("nan"))), (-1, dict(eps=0.0)), (-1, dict(eps=1e-60)), (-1, dict(wd=-1.0)), (-1, dict(b1=1.0)),
                   (-1, dict(b2=-0.1)), (-1, dict(norm=at(22), most=-1.0)), (-1, dict(norm=at(22), most=float("nan"))), (-3, dict(step=at(20) + 4)),
                   (-3, dict(ws=at(21) + 8)), (-3, dict(norm=at(22) + 2)), (-2, dict(dtype=_lib.I32)), (-2, dict(grad_dtype=_lib.BF16)),
                   (-1, dict(n=-1)), (-2, dict(n=(1 << 33) + 1)), (-1, dict(master=at(2))), (-1, dict(param=None)), (-1, dict(grad=None)),
                   (-1, dict(exp_avg=None)), (-1, dict(bits=8)), (-3, dict(param=at(0) + 2)), (-3, dict(exp_avg=at(3) + 2)),
                   # what is written meets something else: the parameter its gradient, a moment, the other tensor's, the step, the workspace
                   (-1, dict(grad=at(0))), (-1, dict(exp_avg=at(0) + 60)), (-1, dict(exp_avg=at(4))), (-1, dict(count=2)),
                   (-1, dict(count=2, second=dict(apart, param=at(1) + 32))), (-1, dict(count=2, second=dict(apart, exp_avg=at(0) + 32))),
                   (-1, dict(step=at(0))), (-1, dict(ws=at(3))), (-1, dict(ws=at(20) - 16)), (-1, dict(norm=at(0), most=1.0)), (-1, dict(lr_at=at(3) + 4)),
                   (-1, dict(bits=8, exp_avg_scale=at(3), exp_avg_sq_scale=at(6)))]:
        assert call(**kw) == rc, kw


# ------------------------------------------------------------------------------------ GPU
@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    torch.cuda.set_device(0)
    return torch.device("cuda:0")


SHAPES = [(1,), (3,), (0,), (127,), (128,), (129,), (2049,), (5, 7), (256, 64), (33, 1343), (4096,), (), (8, 16, 8), (100, 2048)]
TYPES = [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)]
names = lambda t: str(t).split(".")[-1]  # noqa: E731


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("master", [True, False], ids=["main", "alone"])
@pytest.mark.parametrize("dtype,gdtype", TYPES, ids=names)
def test_three_steps(dev, dtype, gdtype, master, bits):
    params, grads, state = make(dev, SHAPES, dtype, gdtype, 1, bits, master)
    for k in range(3):
        old_params, old = clone(params, state)
        if k == 1:                          # without a gradient
            grads[4] = grads[9] = None
        mrl.adamw_(params, grads, **state, **HYPER)
        check(params, grads, state, old_params, old)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_clipping_on_the_way(dev, bits):
    """The factor that clip_grad_norm_ multiplies by, above and below the limit; a norm that is none."""
    params, grads, state = make(dev, SHAPES, BF16, F32, 2, bits)
    norm = mrl.global_grad_norm(grads)
    for limit in (0.3 * norm.item(), 10 * norm.item(), 0.0):
        old_params, old = clone(params, state)
        copies = clone(params, state)
        mrl.adamw_(params, grads, **state, grad_norm=norm, max_norm=limit, **HYPER)
        check(params, grads, state, old_params, old, factor_of(norm, limit))
        # the same bits as from gradients that torch's operations have clipped
        clipped = [g * torch.clamp(limit / (norm + 1e-6), max=1.0) for g in grads]
        mrl.adamw_(copies[0], clipped, **copies[1], **HYPER)
        assert all(torch.equal(a, b) for a, b in zip(params, copies[0]))
        assert all(torch.equal(a.float(), b.float()) for a, b in zip(state["exp_avg"], copies[1]["exp_avg"]))
        # and as clip_grad_norm_ scales them, whose factor is one rounding of the quotient: a step and a half of it apart
        mrl.clip_grad_norm_(grads, limit, out=clipped)
        for c, g in zip(clipped, grads):
            assert ((c - g * factor_of(norm, limit)).abs() <= 5 * U * c.abs() + 2.0 ** -149).all()
    mrl.adamw_(params, grads, **state, grad_norm=torch.full((), float("nan"), device=dev), max_norm=1.0, **HYPER)
    assert all(torch.isnan(p).all() for p in params)


@pytest.mark.gpu
def test_the_factor_has_the_bits_of_torch(dev):
    """Of many norms and limits: the first moment of a first step is (1 - b1) g factor, rounded operation by operation."""
    gen = torch.Generator().manual_seed(13)
    g = torch.linspace(0.5, 2.0, 64, device=dev)
    for _ in range(100):
        norm = torch.rand((), generator=gen).mul(10).exp().to(dev)
        limit = float(torch.rand((), generator=gen, dtype=torch.float64)) * norm.item()
        p = [torch.zeros_like(g)]
        state = mrl.adamw_state(p)
        mrl.adamw_(p, [g], **state, lr=1e-3, grad_norm=norm, max_norm=limit)
        assert torch.equal(state["exp_avg"][0], g * torch.clamp(limit / (norm + 1e-6), max=1.0) * (1 - 0.9))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_settings(dev, bits):
    """No decay, no momentum, a rate on the device, the first step of all, large and small eps."""
    for hyper in (dict(weight_decay=0.0), dict(betas=(0.0, 0.9)), dict(betas=(0.9, 0.0)), dict(betas=(0.9, 0.999), eps=1e-3), dict(lr=0.0),
                  dict(lr=1.0, weight_decay=1.0), dict(eps=1e-15)):
        for first in (False, True):
            params, grads, state = make(dev, [(3, 130), (257,)], F32, F32, 3, bits)
            if first:
                state = mrl.adamw_state(params, bits=bits)
            old_params, old = clone(params, state)
            twin = clone(params, state)
            mrl.adamw_(params, grads, **state, **{**HYPER, **hyper})
            check(params, grads, state, old_params, old, hyper=hyper)
            rate = torch.tensor({**HYPER, **hyper}["lr"], dtype=F32, device=dev)
            mrl.adamw_(twin[0], grads, **twin[1], **{**HYPER, **hyper, "lr": rate})
            hyper32 = {**hyper, "lr": rate.item()}
            check(twin[0], grads, twin[1], old_params, old, hyper=hyper32)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors_of_all_kinds(dev, bits):
    """More than a launch holds, types mixed, views of one flat buffer that start anywhere, strided gradients."""
    gen = torch.Generator(device=dev).manual_seed(4)
    sizes = [int(s) for s in torch.randint(1, 5000, (150,), generator=torch.Generator().manual_seed(5))]
    flat = torch.randn(sum(sizes), generator=gen, device=dev) * 0.1
    params, grads = [], []
    for k, piece in enumerate(flat.split(sizes)):
        params.append(piece if k % 3 == 0 else piece.to((BF16, F16)[k % 2]))
        g = torch.randn(sizes[k], generator=gen, device=dev) * 1e-2
        grads.append(g if k % 2 else g.to(params[-1].dtype))
        if k % 7 == 0:
            grads[-1] = torch.stack([grads[-1], grads[-1]], 1)[:, 0]            # every other entry
        if k % 11 == 0:
            grads[-1] = grads[-1][:1].expand(sizes[k])
    state = mrl.adamw_state(params, bits=bits)
    assert [w is None for w in state["master"]] == [p.dtype is F32 for p in params]
    for _ in range(2):
        old_params, old = clone(params, state)
        mrl.adamw_(params, grads, **state, **HYPER)
        check(params, grads, state, old_params, old)


@pytest.mark.gpu
def test_eight_bits_move_as_they_should_on_average(dev):
    """Changes of a fiftieth of a step per update: to the nearest the codes would stay.  One entry in each block keeps the scale.
    After n steps m is b1^n m0 (no gradients); its mean over N entries is off by at most n rounding errors, each of at most a step
    with mean zero: within 5 standard deviations of sqrt(n / N) steps."""
    n, b1 = 128 * 4096, 0.999
    p, g = [torch.zeros(n, device=dev)], [torch.zeros(n, device=dev)]
    state = mrl.adamw_state(p, bits=8)
    start = torch.full((n,), 104.0, device=dev)          # a code; its neighbours are 8 apart
    state["exp_avg"][0].copy_(start)
    state["exp_avg_sq"][0].copy_(start)
    state["exp_avg_scale"][0].fill_(1.0)
    state["exp_avg_sq_scale"][0].fill_(1.0)
    # an entry in 128 stays at 448 by its gradient: m = v' = 448 and g = 448
    state["exp_avg"][0][::128], state["exp_avg_sq"][0][::128] = 448.0, 448.0
    g[0][::128] = 448.0
    steps = 40
    for _ in range(steps):
        mrl.adamw_(p, g, **state, lr=1e-3, betas=(b1, 0.998), weight_decay=0.0)
    rest = torch.ones(n, dtype=torch.bool, device=dev)
    rest[::128] = False
    for name, want in (("exp_avg", 104 * b1 ** steps), ("exp_avg_sq", 104 * 0.998 ** (steps / 2))):
        got = held(state[name][0], state[name + "_scale"][0])[rest]
        assert abs(got.mean().item() - want) <= 5 * 8 * math.sqrt(steps / got.numel())
        assert got.std() > 0


@pytest.mark.gpu
def test_values_where_it_can_go_wrong(dev):
    """Zeros everywhere, tiny and huge gradients, blocks with one large entry, gradients that are not finite."""
    n = 1024
    for bits in (32, 8):
        params, grads, state = make(dev, [(n,)], F32, F32, 6, bits)
        g = grads[0]
        g[:128] = 0.0
        state["exp_avg"][0].view(torch.uint8 if bits == 8 else F32)[:128] = 0
        state["exp_avg_sq"][0].view(torch.uint8 if bits == 8 else F32)[:128] = 0
        g[128:256] = 1e-25
        g[256:384] *= 1e10
        g[384] = 1e6
        old_params, old = clone(params, state)
        mrl.adamw_(params, grads, **state, **HYPER)
        check(params, grads, state, old_params, old)
        # below a sqrt(v) that is not zero there is always a code
        if bits == 8:
            assert (held(state["exp_avg_sq"][0], state["exp_avg_sq_scale"][0])[385:512] > 0).any()
        bad, old = clone(params, state)
        good = clone(params, state)
        worse = [g.clone()]
        worse[0][600], worse[0][900] = float("nan"), float("inf")
        mrl.adamw_(bad, worse, **old, **HYPER)
        mrl.adamw_(good[0], grads, **good[1], **HYPER)
        hit = torch.zeros(n, dtype=torch.bool, device=dev)
        hit[[600, 900]] = True
        assert torch.isnan(bad[0][hit]).all() and torch.equal(bad[0][~hit], good[0][0][~hit])
        mrl.adamw_(bad, grads, **old, **HYPER)
        mrl.adamw_(good[0], grads, **good[1], **HYPER)
        if bits == 8:
            hit[512:640] = hit[896:1024] = True
        assert torch.isnan(bad[0][[600, 900]]).all() and torch.equal(bad[0][~hit], good[0][0][~hit])


@pytest.mark.gpu
def test_autograd_sees_the_writes(dev):
    """Leaves that require gradients are taken as they are; a graph that kept a parameter notices; what cannot be written is refused."""
    w = torch.randn(4, 8, device=dev, requires_grad=True)
    x = torch.randn(3, 4, device=dev, requires_grad=True)
    state = mrl.adamw_state([w])
    loss = (x @ w).square().sum()
    (g,) = torch.autograd.grad(loss, [w], retain_graph=True)
    before = w.detach().clone()
    mrl.adamw_([w], [g], **state, lr=1e-2)
    assert w.requires_grad and w.is_leaf and not torch.equal(w, before)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(loss, [x])
    for kw in (dict(params=[w, w], grads=[g, g], exp_avg=[g.clone(), g.clone()], exp_avg_sq=[g.abs(), g.abs()], master=None),
               dict(exp_avg=[state["exp_avg_sq"][0]]), dict(grads=[w.detach()]), dict(exp_avg=[w.detach()])):
        kept = w.detach().clone()
        with pytest.raises(_lib.MrlError, match="shares memory"):
            mrl.adamw_(**{"params": [w], "grads": [g], **state, "lr": 1e-2, **kw})
        assert torch.equal(w, kept)


@pytest.mark.gpu
def test_tensors_of_inference_mode_and_empty_lists(dev):
    """They have no version to count up; a step without a gradient is counted."""
    params, grads, state = make(dev, [(300,)], F32, F32, 12)
    twin, twin_state = clone(params, state)
    with torch.inference_mode():
        inner, inner_state = clone(params, state)
        mrl.adamw_(inner, grads, **inner_state, **HYPER)
    mrl.adamw_(twin, grads, **twin_state, **HYPER)
    assert torch.equal(inner[0], twin[0]) and inner_state["step"].item() == twin_state["step"].item() == 8
    mrl.adamw_(twin, [None], **twin_state, **HYPER)
    assert torch.equal(inner[0], twin[0]) and twin_state["step"].item() == 9
    step = torch.zeros((), dtype=torch.int64, device=dev)
    mrl.adamw_([], [], [], [], step, lr=1e-3)
    assert step.item() == 1


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_streams_graphs_and_saved_states(dev, bits):
    """On another stream; captured with the norm in front and replayed, the step counted on the device; saved and loaded."""
    import io
    shapes = [(300, 129), (77,), (5000,)]
    params, grads, state = make(dev, shapes, BF16, F32, 8, bits)
    eager, eager_state = clone(params, state)
    rate = torch.full((), 1e-3, device=dev)

    def step(ps, gs, st):
        mrl.adamw_(ps, gs, **st, grad_norm=mrl.global_grad_norm(gs), max_norm=0.5, **{**HYPER, "lr": rate})

    side = torch.cuda.Stream()
    step(eager, grads, eager_state)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(params, grads, state)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(params, grads, state)
    gen = torch.Generator(device=dev).manual_seed(9)
    for k in range(4):
        rate.fill_(1e-3 * (k + 1))
        for g in grads:
            g.copy_(torch.randn(g.shape, generator=gen, device=dev) * 1e-2)
        step(eager, grads, eager_state)
        graph.replay()
        torch.cuda.synchronize()
        assert state["step"].item() == eager_state["step"].item() == 9 + k
        assert all(torch.equal(a, b) for a, b in zip(params, eager))
        for name, v in state.items():
            if isinstance(v, list):
                assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(v, eager_state[name]) if a is not None)
    file = io.BytesIO()
    torch.save(state, file)
    file.seek(0)
    loaded = torch.load(file, weights_only=True)
    mrl.adamw_(params, grads, **loaded, **HYPER)
    mrl.adamw_(eager, grads, **eager_state, **HYPER)
    assert all(torch.equal(a, b) for a, b in zip(params, eager))


@pytest.mark.gpu
def test_nothing_is_written_outside(dev):
    """Tensors in the middle of buffers keep what lies around them."""
    for n in (1, 7, 8, 127, 129, 2047, 2049, 5003):
        for bits in (32, 8):
            params, grads, state = make(dev, [(n,)], BF16, BF16, 10, bits)
            old_params, old = clone(params, state)
            wholes = []

            def inside(t):
                raw = torch.full((t.numel() + 131,), 77, dtype=F32, device=dev).to(t.dtype)
                wholes.append((raw, t.numel()))
                raw[65:65 + t.numel()] = t
                return raw[65:65 + t.numel()]

            params = [inside(params[0])]
            state = {k: [inside(v[0])] if isinstance(v, list) else v for k, v in state.items()}
            mrl.adamw_(params, grads, **state, **HYPER)
            check(params, grads, state, old_params, old)
            for raw, count in wholes:
                edge = torch.tensor(77.0).to(raw.dtype).float().to(dev)
                assert (raw[:65].float() == edge).all() and (raw[65 + count:].float() == edge).all()


@pytest.mark.gpu
def test_more_entries_than_31_bits(dev):
    """Entries behind 2^31 of one tensor: the 8-bit moments' blocks and the dither's places count on."""
    n = 2 ** 31 + 4096 + 5
    p = torch.zeros(n, dtype=BF16, device=dev)
    g = torch.zeros(n, dtype=BF16, device=dev)
    tail, tail_g, _ = make(dev, [(4096 + 5,)], BF16, BF16, 11)
    p[2 ** 31:], g[2 ** 31:] = tail[0], tail_g[0]
    state = mrl.adamw_state([p], bits=8, master=False)
    mrl.adamw_([p], [g], **state, **HYPER)
    want = formula(tail[0], tail_g[0], torch.zeros(4101, device=dev), torch.zeros(4101, device=dev), 1, **HYPER)
    within(p[2 ** 31:], want["p"], BF16)
    assert not p[:2 ** 31].any()
    m, v = fp32_moments(tail_g[0], 0.0, 0.0, 1.0, *HYPER["betas"])
    x = (torch.arange(2051, device=dev) + 2 ** 30) ^ 0x9E3779B9      # pairs from 2^30 on
    x = ((x ^ (x >> 16)) * 0x7feb352d) & 0xffffffff
    x = ((x ^ (x >> 15)) * 0x846ca68b) & 0xffffffff
    x = x ^ (x >> 16)
    bits = torch.stack([x & 0xffff, x >> 16], 1).view(-1)[:4101]
    for name, x, root in (("exp_avg", m, False), ("exp_avg_sq", v.sqrt(), True)):
        c, s = codes(x, bits, root)
        assert torch.equal(state[name][0][2 ** 31:].double(), c) and torch.equal(state[name + "_scale"][0][2 ** 24:], s)


@pytest.mark.gpu
@pytest.mark.parametrize("worst", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("n", [129, 255, 257, 3 * 1024 + 5, 1024 + 128 + 4])
def test_a_block_that_is_not_finite_stays_alone(dev, n, worst):
    """A gradient that is not finite in the first block of a tensor that ends inside its last one, or in the last block itself: after every step all
    other blocks, the last and not whole one among them, have the bits that they have without it."""
    for at in (5, n - 1):
        params, grads, state = make(dev, [(n,), (70,)], BF16, F32, 14, 8)
        twin, twin_state = clone(params, state)
        worse = [g.clone() for g in grads]
        worse[0][at] = worst
        hit = torch.zeros(-(-n // 128), dtype=torch.bool, device=dev)
        hit[at // 128] = True
        rest = ~hit.repeat_interleave(128)[:n]
        for step in range(3):
            mrl.adamw_(params, worse if step == 0 else grads, **state, **HYPER)
            mrl.adamw_(twin, grads, **twin_state, **HYPER)
            assert torch.isnan(params[0][at]) and not torch.isfinite(state["exp_avg_scale"][0][hit]).any()
            for mine, other, keep in ((params, twin, rest), *((state[k], twin_state[k], rest) for k in ("master", "exp_avg", "exp_avg_sq")),
                                      *((state[k], twin_state[k], ~hit) for k in ("exp_avg_scale", "exp_avg_sq_scale"))):
                assert torch.equal(mine[0][keep].float(), other[0][keep].float()) and torch.equal(mine[1].float(), other[1].float())
                assert torch.isfinite(other[0].float()).all()


def test_parameters_that_a_graph_has_computed_are_refused():
    """A write to one would change what its graph gives; leaves and detached views of them are looked at further."""
    leaf = torch.zeros(4, 6, requires_grad=True)
    held = lambda: [torch.zeros(4, 6)]  # noqa: E731
    for p in (leaf * 1, leaf.view(4, 6), leaf[:]):
        with pytest.raises(ValueError, match="graph"):
            mrl.adamw_([p], held(), held(), held(), torch.zeros((), dtype=torch.int64), lr=1e-3)
        with pytest.raises(ValueError, match="graph"):
            mrl.adamw_state([p])
    for p in (leaf, leaf.detach().view(4, 6)):
        with pytest.raises(RuntimeError, match="GPU only"):
            mrl.adamw_([p], held(), held(), held(), torch.zeros((), dtype=torch.int64), lr=1e-3)


@pytest.mark.gpu
def test_no_root_above_zero_is_lost(dev):
    """Beside one large entry every sqrt(v) above zero keeps a code, in whole blocks and in the last; a zero stays one."""
    n = 3 * 128 + 77
    params, grads, state = make(dev, [(n,)], F32, F32, 18, 8)
    g = grads[0]
    g[::128] = 1e6                          # one in each block
    g[1::5] = 0.0
    state["exp_avg_sq"][0].zero_()
    mrl.adamw_(params, grads, **state, **HYPER)
    v = fp32_moments(g, 0.0, 0.0, 1.0, *HYPER["betas"])[1]
    kept = held(state["exp_avg_sq"][0], state["exp_avg_sq_scale"][0])
    assert (v == 0).any() and torch.equal(kept > 0, v > 0)


@pytest.mark.gpu
@pytest.mark.parametrize("b2,steps", [(0.95, 300), (0.999, 6000)])
def test_eight_bits_hold_v_too_large_by_less_than_their_step(dev, b2, steps):
    """Independent normal gradients g of variance 1.  A root r, held as a code, moves by d = sqrt(b2 r^2 + (1 - b2) g^2) - r and goes to one of two codes, a step
    s <= r / 8 apart: the mean of r moves by d, that of its square by d (2 r + d) and, of the dither, by at most |d| s, where |d| <= (1 - b2) |g^2 - r^2| / (r (1 +
    sqrt(b2))).  What is added goes by (1 - b2) a step, so the mean of v is above 1 by 0 <= e <= E|g^2 - v| / (8 (1 + sqrt(b2))) <= (2 + e) / (8 (1 + sqrt(b2))), below
    0.14; 0.01 for the mean over entries and steps, whose deviation is below 0.001."""
    n = 128 * 512
    gen = torch.Generator(device=dev).manual_seed(19)
    p, g = [torch.zeros(n, device=dev)], [torch.empty(n, device=dev)]
    state = mrl.adamw_state(p, bits=8)
    means = []
    for k in range(steps):
        g[0].normal_(generator=gen)
        mrl.adamw_(p, g, **state, lr=0.0, betas=(0.9, b2), weight_decay=0.0)
        if k >= steps * 3 // 4 and k % 10 == 0:
            means.append(held(state["exp_avg_sq"][0], state["exp_avg_sq_scale"][0]).square().mean() / (1 - b2 ** (k + 1)))
    above = torch.stack(means).mean().item() - 1
    print("v is held too large by %.4f" % above)
    assert -0.01 <= above <= 0.14 + 0.01
