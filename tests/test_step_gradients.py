"""The global norm of gradients and clipping against 64-bit sums, what they refuse, and the operators around the lm_head step
together: token table, final norm, loss from the hidden states, a shared table's gradient, clipping."""
import ctypes
import math
import random

import pytest
import torch

import mindspeed_rl_amd as mrl
from mindspeed_rl_amd import _lib

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def plain_norm(grads):
    return math.sqrt(sum(g.double().square().sum().item() for g in grads))


def check_norm(got, grads):
    """Squares and sums in 64 bits (n entries: n 2^-53 relative, halved by the root), rounded once to fp32."""
    want = plain_norm(grads)
    n = sum(g.numel() for g in grads)
    assert got.dtype is torch.float32 and got.dim() == 0
    assert abs(got.item() - want) <= want * (U + n * 2.0 ** -53) + 2.0 ** -149, (got.item(), want)
    return want


def check_scaled(got, grad, norm, limit):
    """norm, norm + 1e-6, the quotient and the product: a rounding to fp32 each; then one to the output's type."""
    factor = min(1.0, limit / (norm + 1e-6))
    want = grad.double() * factor
    bound = want.abs() * (5 * U + HALF[got.dtype] * 1.01) + TINY[got.dtype]
    assert ((got.double() - want).abs() <= bound).all()


def make(dev, sizes, dtypes, seed, scale=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return [(torch.randn(s, generator=g, device=dev) * scale).to(dtypes[k % len(dtypes)]) for k, s in enumerate(sizes)]


# ------------------------------------------------------------------------------------ refusals (CPU)
def test_refused_arguments():
    a, b = torch.zeros(4), torch.zeros(5)
    for bad, error in [(lambda: mrl.global_grad_norm([]), ValueError), (lambda: mrl.global_grad_norm([None]), ValueError),
                       (lambda: mrl.global_grad_norm([a.double()]), TypeError), (lambda: mrl.global_grad_norm([a.to_sparse()]), TypeError),
                       (lambda: mrl.global_grad_norm([1.0]), TypeError), (lambda: mrl.global_grad_norm([a]), RuntimeError),
                       (lambda: mrl.clip_grad_norm_([a], -1.0), ValueError), (lambda: mrl.clip_grad_norm_([a], float("nan")), ValueError),
                       (lambda: mrl.clip_grad_norm_([], 1.0), ValueError), (lambda: mrl.clip_grad_norm_([a], 1.0, out=[]), ValueError),
                       (lambda: mrl.clip_grad_norm_([a], 1.0, out=[b]), ValueError),
                       (lambda: mrl.clip_grad_norm_([a], 1.0, out=[None]), ValueError),
                       (lambda: mrl.clip_grad_norm_([a], 1.0, out=[a.half()]), ValueError),
                       (lambda: mrl.clip_grad_norm_([a.half()], 1.0, out=[a.bfloat16()]), ValueError),
                       (lambda: mrl.clip_grad_norm_([a], 1.0, out=[b[:4]]), RuntimeError)]:
        with pytest.raises(error):
            bad()


def test_clipping_writes_to_no_part_of_a_graph():
    """Parameters in the place of their gradients, gradients that are differentiated on: refused and left as they were."""
    p = torch.full((4,), 3.0, requires_grad=True)
    (g,) = torch.autograd.grad(p.square().sum(), [p], create_graph=True)
    kept = (p * 2, p.detach() * 2)
    for bad in (lambda: mrl.clip_grad_norm_([p], 1.0), lambda: mrl.clip_grad_norm_([kept[1], g], 1.0), lambda: mrl.clip_grad_norm_(kept[0], 1.0),
                lambda: mrl.clip_grad_norm_([kept[1]], 1.0, out=[p]), lambda: mrl.clip_grad_norm_([p.unfold(0, 2, 2).t()], 1.0)):
        with pytest.raises(ValueError, match="part of a graph"):
            bad()
    assert (p == 3).all()
    # what is only read may be
    with pytest.raises(RuntimeError, match="GPU only"):
        mrl.clip_grad_norm_([g], 1.0, out=[torch.zeros(4)])


def test_shared_memory_of_spaced_tensors():
    """Entries apart: what is written and meets something else is refused, also where the entry point would get copies; what
    lies between one another's entries is not (and is refused for its device here)."""
    a, z = torch.zeros(6, 8), lambda *s: torch.zeros(s)  # noqa: E731
    flat = torch.zeros(200)
    shared = [([a[:, ::2], a[:, ::2]], None), ([a[:, :5], a[:, 4:]], None), ([a[:, 3:], a[2]], None), ([a[1:, 2:4], a.t()[3:]], None),
              ([a[::2, :3], a[::4, 2:]], None), ([a[:, 3], a[4, 3:4]], None), ([flat.as_strided((5, 2), (21, 1)), flat[85:87]], None),
              ([flat.as_strided((5, 2), (21, 1)), flat.as_strided((9, 1), (17, 1), 5)], None),      # 21 + 1 = 5 + 17
              ([a[:, :4]], [a[:, 2:6]]), ([a[:, :4]], [a[:, 1:].t()[:4].t()]), ([z(6, 4), z(6, 5)], [a[:, :4], a[:, 3:]]),
              ([z(6, 4), a[:, 3:5]], [a[:, :4], z(6, 2)]), ([z(6, 4), a[1, 3].expand(5, 4)], [a[:, :4], z(5, 4)]),
              ([z(6, 6), a[:6, :6]], [z(6, 6), a[:6, :6].t()])]
    apart = [([a[:, ::2], a[:, 1::2]], None), ([a[:, :3], a[:, 3:]], None), ([a[::2, :3], a[1::2, :3]], None), ([a[:, 3:], a[2, :3]], None),
             ([a[::2, 3:], a[1]], None), ([a[:, 7], a[4, :7], a[0, :7]], None), ([a[:, :4]], [a[:, :4]]), ([a[:, :4], a[:, :4]], [z(6, 4), z(6, 4)]),
             ([flat.as_strided((5, 2), (21, 1)), flat.as_strided((9, 1), (17, 1), 6)], None),
             ([a[:, :4], a[1, :2].expand(5, 2)], [a[:, 4:], z(5, 2)]), ([a[:0, :4], a[:, :4]], None)]
    for lists, error in ((shared, ValueError), (apart, RuntimeError)):
        for grads, outs in lists:
            for order in (1, -1):
                with pytest.raises(error, match="shares memory" if error is ValueError else "GPU only"):
                    mrl.clip_grad_norm_(grads[::order], 1.0, out=outs and outs[::order])


def test_which_entries_share_memory():
    """Against the sets of bytes, over views of one buffer in two types: any steps, expanded and overlapping ones among them."""
    from mindspeed_rl_amd.gradients import _meet, _places
    rng, base = random.Random(1), torch.zeros(300)

    def view():
        b = base if rng.random() < 0.7 else base.view(torch.bfloat16)
        shape = [rng.randint(1, 5) for _ in range(rng.randint(0, 3))]
        steps = [rng.choice([0, 1, 1, 2, 3, 4, 5, 7, 10, 14, 20, 35]) for _ in shape]
        return b.as_strided(shape, steps, rng.randint(0, b.numel() // 3))

    def touched(t):
        places = [t.data_ptr()]
        for st, n in zip(t.stride(), t.shape):
            places = [p + st * i * t.element_size() for p in places for i in range(n)]
        return {p + k for p in places for k in range(t.element_size())}

    seen = [0, 0]
    for _ in range(4000):
        try:
            p, q = view(), view()
        except RuntimeError:                    # behind the buffer's end
            continue
        want = bool(touched(p) & touched(q))
        assert _meet(_places(p), _places(q)) == _meet(_places(q), _places(p)) == want
        seen[want] += 1
    assert min(seen) > 100


class Grad(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("out", ctypes.c_void_p), ("n", ctypes.c_int64), ("dtype", ctypes.c_int32),
                ("out_dtype", ctypes.c_int32)]


def test_entry_points_refuse_and_launch_nothing():
    lib = _lib.load()
    buf = (ctypes.c_char * 8192)()
    p = (ctypes.addressof(buf) + 15) // 16 * 16
    w = p + 4096
    F32, BF16 = _lib.F32, _lib.BF16

    def clip(*entries, limit=1.0, norm=w, ws=w + 8, n=None):
        table = (Grad * max(1, len(entries)))(*[Grad(*e) for e in entries])
        return lib.mrl_grad_clip(ctypes.addressof(table), len(entries) if n is None else n, limit, norm, ws, None)

    ok = (p, p, 4, F32, F32)
    for rc, entries, kw in [(-2, [(p, p, 4, _lib.I32, F32)], {}), (-2, [(p, p, 4, F32, BF16)], {}), (-1, [(p, p, -1, F32, F32)], {}),
                            (-2, [(p, p, (1 << 33) + 1, F32, F32)], {}), (-1, [(None, p, 4, F32, F32)], {}),
                            (-1, [(p, None, 4, F32, F32)], {}), (-3, [(p + 2, p + 2, 4, F32, F32)], {}),
                            (-3, [(p, p + 65, 4, BF16, BF16)], {}), (-1, [(p, p, 4, BF16, F32)], {}), (-1, [ok], dict(limit=-1.0)),
                            (-1, [ok], dict(limit=float("nan"))), (-1, [ok], dict(norm=None)), (-1, [ok], dict(ws=None)),
                            (-3, [ok], dict(ws=w + 4)), (-2, [ok], dict(n=16385)), (-1, [ok], dict(n=-1))]:
        assert clip(*entries, **kw) == rc, (entries, kw)
    # what is written meets something else in the list
    for entries in ([ok, ok], [ok, (p + 8, p + 8, 4, F32, F32)], [(p, p + 8, 4, F32, F32)], [(p, p + 64, 4, F32, F32), (p + 64, p + 128, 4, F32, F32)],
                    [(p, p + 64, 4, F32, F32), (p + 32, p + 64, 4, F32, F32)], [(p, p + 64, 8, BF16, F32), (p + 94, p + 256, 2, BF16, F32)],
                    [(p + 256, p + 256, 100, BF16, BF16), (p, p + 64, 4, F32, F32), (p + 300, p + 300, 1, F32, F32)]):
        for order in (entries, entries[::-1]):
            assert clip(*order) == -1 and b"shares memory" in lib.mrl_last_error(), order
    table = (Grad * 1)(Grad(p, None, 4, _lib.F64, 0))
    assert lib.mrl_grad_norm(ctypes.addressof(table), 1, w, w + 8, None) == -2
    assert lib.mrl_grad_norm(None, 1, w, w + 8, None) == -1


# ------------------------------------------------------------------------------------ GPU
@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    torch.cuda.set_device(0)
    return torch.device("cuda:0")


LISTS = [[1], [0, 3, 0], [7, 8, 9], [8191, 8192, 8193], [65536 * 3 + 5], [1000003, 17, 4096], list(range(1, 131)),
         [33] * 113, [2] * 1500, [5000000, 1]]


@pytest.mark.gpu
@pytest.mark.parametrize("dtypes", [[torch.float32], [torch.bfloat16], [torch.float16],
                                    [torch.bfloat16, torch.float32, torch.float16]], ids=["f32", "bf16", "f16", "mixed"])
@pytest.mark.parametrize("sizes", LISTS, ids=lambda s: "%dx%d" % (len(s), max(s)))
def test_norm_and_clip(dev, sizes, dtypes):
    grads = make(dev, sizes, dtypes, 1)
    got = mrl.global_grad_norm(grads)
    norm = check_norm(got, grads)
    assert torch.equal(got, mrl.global_grad_norm(iter(grads + [None])))
    for limit in (norm * 2 + 1, norm * 0.37, 0.0):
        mine = [g.clone() for g in grads]
        assert torch.equal(mrl.clip_grad_norm_(mine, limit), got)
        for m, g in zip(mine, grads):
            assert torch.equal(m, g) if limit > norm else True
            check_scaled(m, g, norm, limit)
        for otype in (None, torch.float32):
            outs = [torch.full(g.shape, float("nan"), dtype=otype or g.dtype, device=dev) for g in grads]
            kept = [g.clone() for g in grads]
            assert torch.equal(mrl.clip_grad_norm_(kept, limit, out=outs), got)
            for k, g, o in zip(kept, grads, outs):
                assert torch.equal(k, g)
                check_scaled(o, g, norm, limit)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_views_of_one_buffer(dev, dtype):
    """Gradients that lie back to back at odd places of a flat buffer: scaled there, and nothing around them."""
    sizes = [5, 4099, 1, 16384 * 3 + 7, 30, 777]
    flat = make(dev, [sum(sizes) + 9], [dtype], 2)[0]
    want = flat.clone()
    for skip in (1, 2, 3, 8):
        mine = flat.clone()
        views = list(mine[skip:skip + sum(sizes)].split(sizes))
        norm = plain_norm([v.clone() for v in views])
        out = torch.full((sum(sizes) + 9,), 77.0, device=dev)
        outs = list(out[skip + 1:skip + 1 + sum(sizes)].split(sizes))
        check_norm(mrl.clip_grad_norm_(views, 0.25 * norm, out=outs), views)
        check_scaled(out[skip + 1:skip + 1 + sum(sizes)], want[skip:skip + sum(sizes)], norm, 0.25 * norm)
        assert (out[:skip + 1] == 77).all() and (out[skip + 1 + sum(sizes):] == 77).all()
        mrl.clip_grad_norm_(views, 0.25 * norm)
        check_scaled(mine[skip:skip + sum(sizes)], want[skip:skip + sum(sizes)], norm, 0.25 * norm)
        assert torch.equal(mine[:skip], want[:skip]) and torch.equal(mine[skip + sum(sizes):], want[skip + sum(sizes):])


@pytest.mark.gpu
def test_strides(dev):
    """Permuted and spaced gradients, in place and into outputs of another order; what shares memory is refused."""
    g = torch.Generator(device=dev).manual_seed(3)
    base = torch.randn(40, 70, generator=g, device=dev)
    for view in (lambda t: t.t(), lambda t: t[:, 3:40], lambda t: t[::2], lambda t: t.view(4, 10, 70).permute(2, 0, 1)):
        mine = base.clone()
        v = view(mine)
        norm = plain_norm([v.clone()])
        check_norm(mrl.global_grad_norm(v), [v])
        want = v.clone()
        mrl.clip_grad_norm_([v], 0.5 * norm)
        check_scaled(v, want, norm, 0.5 * norm)
        left = mine.clone()
        view(left).copy_(want)
        assert torch.equal(left, base)                  # entries between them are as they were
        out = torch.full(v.shape, float("nan"), device=dev)
        check_norm(mrl.clip_grad_norm_([v], 0.25 * norm, out=[out]), [v])
        check_scaled(out, v, plain_norm([v]), 0.25 * norm)
        wide = torch.full((*v.shape[:-1], v.shape[-1] + 3), 77.0, device=dev)
        mrl.clip_grad_norm_(v, 0.25 * norm, out=wide[..., 2:-1])
        check_scaled(wide[..., 2:-1], v, plain_norm([v]), 0.25 * norm)
        assert (wide[..., :2] == 77).all() and (wide[..., -1] == 77).all()
    one = torch.ones(5, device=dev)
    check_norm(mrl.global_grad_norm(one.expand(6, 5)), [one.expand(6, 5)])
    for bad in ([one.expand(6, 5)], [one, one], [one[:3], one[2:]]):
        with pytest.raises((ValueError, _lib.MrlError)):
            mrl.clip_grad_norm_(bad, 1.0)
    with pytest.raises(_lib.MrlError):
        mrl.clip_grad_norm_([base.view(-1)[:2000]], 1.0, out=[base.view(-1)[700:2700]])
    check_norm(mrl.global_grad_norm([one, one]), [one, one])
    # what is written counts as written to: autograd refuses a backward that kept it
    leaf = torch.ones(5, device=dev, requires_grad=True)
    kept = leaf * 2
    y = kept.square().sum()
    mrl.clip_grad_norm_([kept.detach()], 1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@pytest.mark.gpu
def test_spaced_tensors_between_one_another(dev):
    """Columns and rows of one matrix that share no entry, in place and into one another's gaps; what is refused is untouched."""
    g = torch.Generator(device=dev).manual_seed(7)
    base = torch.randn(30, 40, generator=g, device=dev)
    for cut in (lambda t: [t[:, ::2], t[:, 1::2]], lambda t: [t[:, :13], t[:, 13:]], lambda t: [t[::2, :9], t[1::2, :9], t[:, 9:].t()]):
        mine = base.clone()
        parts = cut(mine)
        norm = plain_norm(cut(base))
        check_norm(mrl.clip_grad_norm_(parts, 0.5 * norm), cut(base))
        for p, q in zip(parts, cut(base)):
            check_scaled(p, q, norm, 0.5 * norm)
    mine = base.clone()
    check_norm(mrl.clip_grad_norm_([mine[:, ::2]], 1.0, out=[mine[:, 1::2]]), [base[:, ::2]])
    assert torch.equal(mine[:, ::2], base[:, ::2])
    check_scaled(mine[:, 1::2], base[:, ::2], plain_norm([base[:, ::2]]), 1.0)
    mine = base.clone()
    with pytest.raises(ValueError, match="shares memory"):
        mrl.clip_grad_norm_([mine[:, ::2], mine[:, ::2]], 1.0)
    assert torch.equal(mine, base)


@pytest.mark.gpu
def test_extreme_values(dev):
    """Entries whose squares leave fp32 on either side, and what is not finite, as the formula has it."""
    for dtype, big, small in ((torch.float32, 3.0e38, 1e-40), (torch.bfloat16, 3.0e38, 1e-38), (torch.float16, 6e4, 1e-7)):
        for value in (big / 64, small):
            t = torch.full((999,), value, device=dev).to(dtype)
            check_norm(mrl.global_grad_norm(t), [t])
        huge = torch.full((4096,), big / 2, device=dev).to(dtype)
        keep = huge.clone()
        norm = mrl.clip_grad_norm_(huge, 1.0)
        want = plain_norm([keep])
        if want < 3.4e38:
            check_scaled(huge, keep, want, 1.0)
        else:                                           # the norm leaves fp32: the factor is 0
            assert torch.isinf(norm) and not huge.any()
        for bad in (float("nan"), float("inf")):
            t = torch.ones(3000, device=dev).to(dtype)
            t[1234] = bad
            other = torch.ones(7, device=dev)
            plain = [t.float(), other.clone()]
            norm = mrl.clip_grad_norm_([t, other], 1.0)
            assert torch.isnan(norm) if math.isnan(bad) else torch.isinf(norm)
            factor = torch.clamp(1.0 / (norm + 1e-6), max=1.0)
            for m, q in zip((t, other), plain):
                assert torch.equal(torch.nan_to_num(m.float(), nan=-5.0), torch.nan_to_num((q * factor).to(m.dtype).float(), nan=-5.0))


@pytest.mark.gpu
def test_streams_and_graphs(dev):
    """On another stream; clipping captured into two graphs and replayed in turn with new gradients."""
    sizes = [300, 70001, 5] + [64] * 120
    static = make(dev, sizes, [torch.bfloat16, torch.float32], 4)
    outs = [[torch.empty(g.shape, device=dev) for g in static] for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = mrl.global_grad_norm(static)
    torch.cuda.current_stream().wait_stream(side)
    check_norm(got, static)
    graphs, norms = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph, out in zip(graphs, outs):
        with torch.cuda.graph(graph):
            norms.append(mrl.clip_grad_norm_(static, 10.0, out=out))
    for k in range(4):
        for s, n in zip(static, make(dev, sizes, [torch.bfloat16, torch.float32], 10 + k, 0.01 if k == 2 else 1.0)):
            s.copy_(n)
        eager = [torch.empty(g.shape, device=dev) for g in static]
        want = mrl.clip_grad_norm_(static, 10.0, out=eager)
        for graph, out, norm in zip(graphs, outs, norms):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(norm, want) and all(torch.equal(a, b) for a, b in zip(out, eager))


@pytest.mark.gpu
def test_more_entries_than_31_bits(dev):
    t = torch.zeros((1 << 31) + 4099, dtype=torch.bfloat16, device=dev)
    t[-5:] = torch.tensor([3.0, 0, 4.0, 0, 12.0], device=dev)
    assert mrl.clip_grad_norm_(t, 6.5).item() == 13.0
    factor = torch.tensor(6.5) / (torch.tensor(13.0) + 1e-6)
    assert torch.equal(t[-5:].cpu(), (torch.tensor([3.0, 0, 4.0, 0, 12.0]) * factor).bfloat16())


# ------------------------------------------------------------------------------------ together
def _batch(dev, g, vocab):
    plen, rlen = [3, 1, 5, 2], [20, 9, 1, 33]
    n, width, total = len(plen), max(rlen), sum(plen) + sum(rlen)
    seqlens = torch.tensor([p + r for p, r in zip(plen, rlen)], dtype=torch.int32, device=dev)
    cu = torch.zeros(n + 1, dtype=torch.int32, device=dev)
    cu[1:] = torch.cumsum(seqlens, 0)
    live = torch.arange(width, device=dev)[None, :] < torch.tensor(rlen, device=dev)[:, None]
    ids = torch.randint(0, vocab, (1, total), generator=g, device=dev)
    ids[0, ::3] = 11                                    # one token that is everywhere
    batch = {"labels": torch.roll(ids, -1, 1), "responses": torch.zeros(n, width, dtype=torch.int64, device=dev),
             "prompt_length": torch.tensor(plen, dtype=torch.int32, device=dev)[:, None],
             "response_length": torch.tensor(rlen, dtype=torch.int32, device=dev)[:, None],
             "advantages": torch.randn(n, 1, generator=g, device=dev) * live,
             "old_log_prob": -8 + torch.randn(n, width, generator=g, device=dev) * 0.1,
             "ref_log_prob": -8 + torch.randn(n, width, generator=g, device=dev) * 0.1}
    kw = dict(use_remove_padding=True, seqlens_in_batch=seqlens, cu_seqlens_padded=cu, seq_len=max(p + r for p, r in zip(plen, rlen)))
    return ids, batch, kw


def _loss_object(kind="ray_grpo"):
    fn = mrl.LossFuncFactory.get_instance(kind, "actor")
    fn.add_loss_meta_info({"clip_ratio": 0.2, "kl_ctrl": mrl.FixedKLController(0.01), "kl_penalty": "low_var_kl",
                           "entropy_coeff": 0.001, "token_level_loss": True, "clip_higher_enable": True, "clip_ratio_low": 0.2,
                           "clip_ratio_high": 0.28})
    return fn


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["ray_grpo", "ray_dapo", "ray_ppo"])
@pytest.mark.parametrize("norm", ["rms", "layer"])
def test_loss_objects_take_the_final_norm(dev, kind, norm):
    """final_norm_weight= is the norm in front of the same call: the same loss, gradients and scores, bit for bit."""
    g = torch.Generator(device=dev).manual_seed(5)
    vocab, h = 1000, 128
    _, batch, kw = _batch(dev, g, vocab)
    hidden = torch.randn(1, batch["labels"].shape[1], h, generator=g, device=dev).to(torch.bfloat16).requires_grad_()
    head = (torch.randn(vocab, h, generator=g, device=dev) * 0.1).to(torch.bfloat16).requires_grad_()
    w = (1 + 0.1 * torch.randn(h, generator=g, device=dev)).to(torch.bfloat16).requires_grad_()
    b = (0.1 * torch.randn(h, generator=g, device=dev)).to(torch.bfloat16).requires_grad_() if norm == "layer" else None
    extra = dict(final_norm_weight=w, final_norm_type=norm, final_norm_eps=1e-4, **({"final_norm_bias": b} if b is not None else {}))
    leaves = [t for t in (hidden, head, w, b) if t is not None]
    fn = _loss_object(kind)

    def normed():
        return mrl.rms_norm(hidden, w, eps=1e-4) if norm == "rms" else mrl.layer_norm(hidden, w, b, eps=1e-4)

    loss, stats = fn.compute_loss(hidden, batch, lm_head_weight=head, **extra, **kw)
    grads = torch.autograd.grad(loss, leaves)
    want_loss, want_stats = _loss_object(kind).compute_loss(normed(), batch, lm_head_weight=head, **kw)
    want = torch.autograd.grad(want_loss, leaves)
    assert torch.equal(loss, want_loss) and dict(stats) == dict(want_stats)
    assert all(torch.equal(p, q) for p, q in zip(grads, want)) and all(q.abs().max() > 0 for q in want)
    score = fn.compute_loss(hidden, batch, forward_only=True, lm_head_weight=head, **extra, **kw)
    with torch.no_grad():
        assert torch.equal(score, fn.compute_loss(normed(), batch, forward_only=True, lm_head_weight=head, **kw))


@pytest.mark.gpu
def test_a_step_with_a_shared_table(dev):
    """Token table in, final norm, the same table as lm_head, backward, the tokens' gradient added to the lm_head's, clipping
    into fp32: each stage against 64-bit arithmetic on what the stage before handed over."""
    from test_token_embedding import plain_grad, within as within_sums
    g = torch.Generator(device=dev).manual_seed(6)
    vocab, h = 504, 192
    ids, batch, kw = _batch(dev, g, vocab)
    table = (torch.randn(vocab, h, generator=g, device=dev) * 0.1).to(torch.bfloat16).requires_grad_()
    w = (1 + 0.1 * torch.randn(h, generator=g, device=dev)).to(torch.bfloat16).requires_grad_()
    x = mrl.token_embedding(ids, table, scale=h ** 0.5)
    leaf = x.detach().requires_grad_()
    loss, stats = _loss_object().compute_loss(leaf, batch, lm_head_weight=table, final_norm_weight=w, **kw)
    dx, dtable, dw = torch.autograd.grad(loss, [leaf, table, w])
    main = dtable.float()
    value, bound, _ = plain_grad(ids, dx, vocab, float(torch.tensor(h ** 0.5)), 0, torch.float32, main)
    mrl.token_embedding_grad(ids, dx, main, scale=h ** 0.5, accumulate=True)
    within_sums(main, value, bound)
    # the same through autograd, which adds the two gradients of the table in its own type: two roundings to it and their sum's
    (whole,) = torch.autograd.grad(mrl.token_embedding(ids, table, scale=h ** 0.5), [table], dx)
    both = (whole + dtable).double()
    assert ((both - value).abs() <= 2.0 ** -8 * 1.01 * (whole.double().abs() + both.abs()) + 2 * bound).all()
    grads, outs = [main, dw], [torch.empty_like(main), torch.empty(h, device=dev)]
    norm = plain_norm(grads)
    check_norm(mrl.clip_grad_norm_(grads, 0.1 * norm, out=outs), grads)
    for o, q in zip(outs, grads):
        check_scaled(o, q, norm, 0.1 * norm)
    # and as a training loop writes it, through the leaves' .grad
    for p in (table, w):
        p.grad = None
    loss, _ = _loss_object().compute_loss(mrl.token_embedding(ids, table, scale=h ** 0.5), batch, lm_head_weight=table,
                                          final_norm_weight=w, **kw)
    loss.backward()
    assert torch.equal(w.grad, dw) and torch.equal(table.grad, dtable + whole)
    before = [p.grad.clone() for p in (table, w)]
    norm = plain_norm(before)
    check_norm(mrl.clip_grad_norm_([p.grad for p in (table, w)], 0.5 * norm), before)
    for p, q in zip((table, w), before):
        check_scaled(p.grad, q, norm, 0.5 * norm)
