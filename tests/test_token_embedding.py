"""The token table's lookup and its gradient by sorted tokens against plain 64-bit sums, and what they refuse."""
import ctypes

import pytest
import torch

import mindspeed_rl_amd as mrl
from mindspeed_rl_amd import _lib

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def rows_of(ids, vocab, start):
    local = ids.long().reshape(-1) - start
    return torch.where((local >= 0) & (local < vocab), local, vocab)


def plain_grad(ids, dy, vocab, scale, start, dtype, old=None):
    """The sums in 64 bits and what fp32 sums with one rounding may be off by: a row that c tokens name is a chain of at
    most c additions, off by c U sum|dy|; the scale and what was there cost a rounding each."""
    row = rows_of(ids, vocab, start)
    d = dy.reshape(-1, dy.shape[-1]).double()
    sums, size = (torch.zeros(vocab + 1, d.shape[1], dtype=torch.float64, device=d.device) for _ in range(2))
    sums.index_add_(0, row, d)
    size.index_add_(0, row, d.abs())
    count = torch.bincount(row, minlength=vocab + 1)[:vocab, None]
    value, size = sums[:vocab] * scale, size[:vocab] * abs(scale)
    bound = (count + 3) * U * size
    if old is not None:
        value = value + old.double()
        bound = bound + U * (value.abs() + bound)
    return value, bound + HALF[dtype] * value.abs() * 1.01 + TINY[dtype] * (count > 0), count


def within(got, value, bound):
    assert torch.isfinite(got).all()
    off = (got.double() - value).abs() - bound * 1.01
    assert (off <= 0).all(), "off by %g more than the bound at %s" % (off.max().item(), off.argmax().item())


def make_ids(dev, n, vocab, how, seed, dtype=torch.int64):
    g = torch.Generator(device=dev).manual_seed(seed)
    if how == "uniform":
        ids = torch.randint(0, vocab, (n,), generator=g, device=dev)
    elif how == "one":
        ids = torch.full((n,), vocab // 2, device=dev)
    elif how == "hot":                          # half of them one token, the rest few others
        ids = torch.randint(0, max(1, min(vocab, 9)), (n,), generator=g, device=dev)
        ids = torch.where(torch.rand(n, generator=g, device=dev) < 0.5, vocab - 1, ids)
    elif how == "order":
        ids = torch.arange(n, device=dev) % vocab
    else:                                       # two thirds outside, on both sides
        ids = torch.randint(-vocab, 2 * vocab, (n,), generator=g, device=dev)
    return ids.to(dtype)


# ------------------------------------------------------------------------------------ refusals (CPU)
def test_refused_arguments():
    w, ids = torch.zeros(10, 8), torch.zeros(3, dtype=torch.int64)
    grad, out = torch.zeros(3, 8), torch.zeros(10, 8)
    for bad, error in [(lambda: mrl.token_embedding(ids.float(), w), TypeError),
                       (lambda: mrl.token_embedding(ids.bool(), w), TypeError),
                       (lambda: mrl.token_embedding(ids, w.double()), TypeError),
                       (lambda: mrl.token_embedding(ids, w[0]), ValueError),
                       (lambda: mrl.token_embedding(ids, w[:0]), ValueError),
                       (lambda: mrl.token_embedding(ids, w[:, :0]), ValueError),
                       (lambda: mrl.token_embedding(ids, w, scale=float("nan")), ValueError),
                       (lambda: mrl.token_embedding(ids, w, vocab_start=-1), ValueError),
                       (lambda: mrl.token_embedding(ids, w, vocab_start=1 << 64), ValueError),
                       (lambda: mrl.token_embedding(ids, w), RuntimeError),
                       (lambda: mrl.token_embedding_grad(ids, grad[:2], out), ValueError),
                       (lambda: mrl.token_embedding_grad(ids, grad[:, :4], out), ValueError),
                       (lambda: mrl.token_embedding_grad(ids, grad.double(), out), TypeError),
                       (lambda: mrl.token_embedding_grad(ids, grad, out.half()), TypeError),
                       (lambda: mrl.token_embedding_grad(ids, grad, torch.zeros(8, 10).t()), ValueError),
                       (lambda: mrl.token_embedding_grad(ids, grad, out.clone().requires_grad_()), ValueError),
                       (lambda: mrl.token_embedding_grad(ids.float(), grad, out), TypeError),
                       (lambda: mrl.token_embedding_grad(ids, grad, out), RuntimeError)]:
        with pytest.raises(error):
            bad()


def test_entry_points_refuse_and_launch_nothing():
    lib = _lib.load()
    buf = (ctypes.c_char * 4096)()
    p = (ctypes.addressof(buf) + 15) // 16 * 16

    def fwd(ids=p, it=_lib.I64, n=2, start=0, table=p, dtype=_lib.F32, vocab=4, hidden=8, scale=1.0, out=p):
        return lib.mrl_embedding_fwd(ids, it, n, start, table, dtype, vocab, hidden, scale, out, None)

    for rc, kw in [(-2, dict(it=_lib.F32)), (-2, dict(dtype=_lib.I32)), (-1, dict(n=-1)), (-1, dict(start=-1)), (-1, dict(vocab=0)),
                   (-1, dict(hidden=0)), (-2, dict(vocab=(1 << 31) - 1)), (-2, dict(n=1 << 26)), (-2, dict(hidden=(1 << 20) + 1)),
                   (-1, dict(scale=float("inf"))), (-1, dict(ids=None)), (-1, dict(table=None)), (-1, dict(out=None)),
                   (-3, dict(ids=p + 4)), (-3, dict(table=p + 2)), (-3, dict(out=p + 2)), (0, dict(n=0, ids=None))]:
        assert fwd(**kw) == rc, kw
    need = lib.mrl_embedding_bwd_workspace_bytes(2, 4, 8)
    assert need > 0 and lib.mrl_embedding_bwd_workspace_bytes(0, 4, 8) == 0

    def bwd(ids=p, it=_lib.I64, n=2, start=0, dy=p, dtype=_lib.BF16, vocab=4, hidden=8, scale=1.0, out=p, ot=_lib.F32, ws=p,
            size=need):
        return lib.mrl_embedding_bwd(ids, it, n, start, dy, dtype, vocab, hidden, scale, out, ot, 0, ws, size, None)

    for rc, kw in [(-2, dict(it=_lib.U8)), (-2, dict(dtype=_lib.F64)), (-2, dict(ot=_lib.F16)), (-1, dict(n=-1)), (-2, dict(n=1 << 26)),
                   (-2, dict(vocab=1 << 30, hidden=16, size=1 << 40)), (-2, dict(vocab=(1 << 30) - 1, hidden=16, size=1 << 40)),
                   (-1, dict(vocab=0)), (-1, dict(dy=None)), (-1, dict(out=None)), (-1, dict(ws=None)), (-1, dict(size=need - 1)),
                   (-3, dict(ws=p + 8)), (-3, dict(dy=p + 1)), (-3, dict(out=p + 2)), (-1, dict(scale=float("nan")))]:
        assert bwd(**kw) == rc, kw


# ------------------------------------------------------------------------------------ GPU
@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    torch.cuda.set_device(0)
    return torch.device("cuda:0")


TYPES = [torch.float32, torch.bfloat16, torch.float16]
SIZES = [(1, 1, 1), (1, 1000, 64), (2, 7, 5), (31, 511, 33), (33, 512, 64), (64, 32003, 136), (511, 2, 40), (513, 1000, 257),
         (4097, 50000, 24), (5000, 300000, 16), (9000, 152064, 8), (70001, 1000, 12), (700, 900, 3584), (300, 64, 8200)]
HOWS = ["uniform", "one", "hot", "order", "outside"]


@pytest.mark.gpu
@pytest.mark.parametrize("how", HOWS)
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_lookup_and_gradient(dev, size, how):
    n, vocab, h = size
    dtype = TYPES[(n + h) % 3]
    ids = make_ids(dev, n, vocab, how, 1, torch.int64 if n % 2 else torch.int32)
    g = torch.Generator(device=dev).manual_seed(2)
    w = torch.randn(vocab, h, generator=g, device=dev).to(dtype).requires_grad_()
    dy = torch.randn(n, h, generator=g, device=dev).to(dtype)
    scale = 1.0 if n % 3 == 0 else 1.7
    y = mrl.token_embedding(ids, w, scale=scale)
    # One product: rounded to fp32 (U) and then to the type (half a step), or, where the instruction that converts to fp16
    # takes the product itself, once.  -0.7080078125 * fp32(1.7) = -1.2036133150 is such a value: above the middle
    # -1.20361328125 of its fp16 neighbours, so -1.2041 is next to it, but its fp32 rounding is that middle, which goes to -1.2031.
    row = rows_of(ids, vocab, 0)
    exact = torch.cat([w.detach().double(), torch.zeros(1, h, dtype=torch.float64, device=dev)])[row]
    if scale == 1.0:
        assert torch.equal(y.detach().double(), exact)
    within(y.detach(), exact * float(torch.tensor(scale)), (exact * scale).abs() * (U + HALF[dtype]) * 1.01 + TINY[dtype])
    assert not y.detach()[row == vocab].any()
    (dw,) = torch.autograd.grad(y, [w], dy)
    value, bound, count = plain_grad(ids, dy, vocab, scale, 0, dtype)
    assert dw.dtype is dtype
    within(dw, value, bound)
    assert not dw[(count == 0)[:, 0]].any()
    (again,) = torch.autograd.grad(mrl.token_embedding(ids, w, scale=scale), [w], dy)
    assert torch.equal(again, dw)


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["uniform", "hot", "outside"])
@pytest.mark.parametrize("dtype,otype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                         (torch.bfloat16, torch.float32), (torch.float16, torch.float16),
                                         (torch.float16, torch.float32)], ids=lambda t: str(t).split(".")[-1])
def test_added_gradient(dev, dtype, otype, how):
    """Added to what is there; rows that no token names keep their bits, NaN among them; and written whole without."""
    for n, vocab, h, start in ((100, 37, 72, 0), (2050, 500, 129, 500), (40, 4000, 1024, 8000), (600, 40, 2056, 3)):
        ids = make_ids(dev, n, vocab, how, 3) + start
        g = torch.Generator(device=dev).manual_seed(4)
        dy = torch.randn(n, h, generator=g, device=dev).to(dtype)
        old = torch.randn(vocab, h, generator=g, device=dev).to(otype)
        value, bound, count = plain_grad(ids, dy, vocab, 0.5, start, otype, old)
        untouched = (count == 0)[:, 0]
        old[untouched] = float("nan")
        out = old.clone()
        assert mrl.token_embedding_grad(ids, dy, out, scale=0.5, vocab_start=start, accumulate=True) is out
        assert torch.isnan(out[untouched]).all()
        within(out[~untouched], value[~untouched], bound[~untouched])
        fresh = torch.full_like(old, float("nan"))
        mrl.token_embedding_grad(ids, dy, fresh, scale=0.5, vocab_start=start)
        within(fresh, *plain_grad(ids, dy, vocab, 0.5, start, otype)[:2])


@pytest.mark.gpu
def test_shapes_strides_and_places(dev):
    """Scalars and batches of ids, other integer types, strided ids and gradients, a transposed table, empty batches."""
    g = torch.Generator(device=dev).manual_seed(5)
    w = torch.randn(50, 30, generator=g, device=dev)
    assert torch.equal(mrl.token_embedding(torch.tensor(7, device=dev), w), w[7])
    ids = torch.randint(0, 50, (4, 6), generator=g, device=dev)
    for view in (ids, ids.t(), ids.to(torch.int16), ids.to(torch.uint8), ids[:, ::2], ids.view(2, 2, 6)):
        assert torch.equal(mrl.token_embedding(view, w), w[view.long()])
    assert torch.equal(mrl.token_embedding(ids, w.t().contiguous().t()), w[ids])
    odd = torch.empty(50 * 30 + 1, device=dev)[1:].view(50, 30).copy_(w)
    assert torch.equal(mrl.token_embedding(ids, odd, scale=2.0), w[ids] * 2)
    # an upstream gradient of one value, and one whose rows lie apart
    wl = w.clone().requires_grad_()
    mrl.token_embedding(ids, wl).sum().backward()
    assert torch.equal(wl.grad, torch.bincount(ids.reshape(-1), minlength=50)[:, None].float().expand(50, 30))
    wide = torch.randn(4, 6, 64, generator=g, device=dev)
    out = torch.empty(50, 30, device=dev)
    mrl.token_embedding_grad(ids.t(), wide.transpose(0, 1)[..., 3:33], out)
    within(out, *plain_grad(ids, wide[..., 3:33], 50, 1.0, 0, torch.float32)[:2])
    none = ids[:0]
    wl = w.clone().requires_grad_()
    y = mrl.token_embedding(none, wl)
    assert y.shape == (0, 6, 30)
    y.sum().backward()
    assert torch.equal(wl.grad, torch.zeros_like(w))
    keep = w.clone()
    mrl.token_embedding_grad(none, torch.empty(0, 6, 30, device=dev), keep, accumulate=True)
    assert torch.equal(keep, w)


@pytest.mark.gpu
def test_parts_of_a_table_add_up(dev):
    """Two ranks' parts: lookups add up to the whole table's, gradients are its rows."""
    g = torch.Generator(device=dev).manual_seed(6)
    w = torch.randn(1000, 48, generator=g, device=dev)
    ids = torch.randint(-3, 1003, (3000,), generator=g, device=dev)
    dy = torch.randn(3000, 48, generator=g, device=dev)
    parts = [w[:600].clone().requires_grad_(), w[600:].clone().requires_grad_()]
    whole = w.clone().requires_grad_()
    y = mrl.token_embedding(ids, whole, scale=3.0)
    ys = [mrl.token_embedding(ids, p, scale=3.0, vocab_start=s) for p, s in zip(parts, (0, 600))]
    assert torch.equal(ys[0] + ys[1], y)
    (dw,) = torch.autograd.grad(y, [whole], dy)
    dparts = [torch.autograd.grad(a, [p], dy)[0] for a, p in zip(ys, parts)]
    value, bound, _ = plain_grad(ids, dy, 1000, 3.0, 0, torch.float32)
    within(torch.cat(dparts), value, bound)
    within(dw, value, bound)


@pytest.mark.gpu
def test_ids_at_the_ends_of_their_types(dev):
    """The largest and smallest integers are outside any table, and the rows next to its ends are not."""
    w = torch.arange(1.0, 6.0, device=dev)[:, None].expand(5, 4).contiguous()
    for dtype in (torch.int64, torch.int32):
        i = torch.iinfo(dtype)
        ids = torch.tensor([i.min, i.min + 1, -1, 0, 9, 10, 14, 15, i.max - 1, i.max], dtype=dtype, device=dev)
        want = torch.tensor([0., 0, 0, 0, 0, 1, 5, 0, 0, 0], device=dev)
        assert torch.equal(mrl.token_embedding(ids, w, vocab_start=10)[:, 0], want)
        out = torch.empty(5, 4, device=dev)
        mrl.token_embedding_grad(ids, torch.ones(10, 4, device=dev), out, vocab_start=10)
        assert out[:, 0].tolist() == [1, 0, 0, 0, 1]
    top = (1 << 62) + 5
    ids = torch.tensor([top - 1, top, top + 4, top + 5], device=dev)
    assert mrl.token_embedding(ids, w, vocab_start=top)[:, 0].tolist() == [0, 1, 5, 0]


@pytest.mark.gpu
def test_gradient_against_differences(dev):
    """sum(y dy) is linear in the table: its difference along a direction is the product with the gradient, exactly but for
    the gradient's own bound."""
    g = torch.Generator(device=dev).manual_seed(7)
    ids = torch.randint(-2, 40, (300,), generator=g, device=dev)
    w = torch.randn(30, 20, generator=g, device=dev).requires_grad_()
    dy = torch.randn(300, 20, generator=g, device=dev)
    (dw,) = torch.autograd.grad(mrl.token_embedding(ids, w, scale=0.7), [w], dy)
    v = torch.randn(30, 20, generator=g, device=dev, dtype=torch.float64)
    row = rows_of(ids, 30, 0)

    def value(table):
        return (torch.cat([table, torch.zeros(1, 20, dtype=torch.float64, device=dev)])[row] * 0.7 * dy.double()).sum()

    slope = (value(w.detach().double() + v) - value(w.detach().double() - v)) / 2
    _, bound, _ = plain_grad(ids, dy, 30, 0.7, 0, torch.float32)
    # the scale itself is rounded to fp32: half a step of every product
    assert abs((dw.double() * v).sum() - slope) <= (bound * v.abs()).sum() * 1.01 + U * (dw.double() * v).abs().sum() + 1e-12


@pytest.mark.gpu
def test_differentiated_once_and_written_in_place(dev):
    """A second differentiation is refused; a gradient that is added to counts as written to."""
    w = torch.randn(9, 12, device=dev).requires_grad_()
    ids = torch.tensor([3, 3, 0], device=dev)
    dy = torch.randn(3, 12, device=dev).requires_grad_()
    (dw,) = torch.autograd.grad(mrl.token_embedding(ids, w), [w], dy, create_graph=True)
    assert torch.equal(dw[3], dy[0] + dy[1])
    with pytest.raises(RuntimeError):
        dw.sum().backward()
    out = torch.zeros(9, 12, device=dev)
    before = out._version
    mrl.token_embedding_grad(ids, dy.detach(), out, accumulate=True)
    assert out._version > before
    with torch.inference_mode():
        assert torch.equal(mrl.token_embedding(ids, w), w[ids])


@pytest.mark.gpu
def test_two_streams_at_once(dev):
    """Gradients that overlap in time, each with its own workspace: the bits of one alone."""
    g = torch.Generator(device=dev).manual_seed(11)
    sets = [(torch.randint(-9, 3000, (9000,), generator=g, device=dev), torch.randn(9000, 256, generator=g, device=dev)) for _ in range(2)]

    def step(ids, dy):
        return mrl.token_embedding_grad(ids, dy, torch.empty(3000, 256, device=dev))

    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                got[k].append(step(*sets[k]))
    torch.cuda.synchronize()
    assert all(torch.equal(p, want[k]) for k in range(2) for p in got[k])


@pytest.mark.gpu
def test_memory_around_the_outputs(dev):
    for n, vocab, h in ((5, 3, 7), (700, 65, 129), (40, 40, 2049)):
        ids = make_ids(dev, n, vocab, "hot", 8)
        g = torch.Generator(device=dev).manual_seed(9)
        dy = torch.randn(n, h, generator=g, device=dev).to(torch.bfloat16)
        w = torch.randn(vocab, h, generator=g, device=dev).to(torch.bfloat16)
        need = _lib.load().mrl_embedding_bwd_workspace_bytes(n, vocab, h)
        ws = torch.full((need + 64,), 77, dtype=torch.uint8, device=dev)
        for otype, code in ((torch.bfloat16, _lib.BF16), (torch.float32, _lib.F32)):
            whole = torch.full((vocab * h + 33,), 77.0, dtype=otype, device=dev)
            out = whole[17:17 + vocab * h]
            _lib.call("mrl_embedding_bwd", ids.data_ptr(), _lib.I64, n, 0, dy.data_ptr(), _lib.BF16, vocab, h, 2.0, out.data_ptr(),
                      code, 0, ws.data_ptr(), need, _lib.stream(dev))
            within(out.view(vocab, h), *plain_grad(ids, dy, vocab, 2.0, 0, otype)[:2])
            assert (whole[:17] == 77).all() and (whole[17 + vocab * h:] == 77).all() and (ws[need:] == 77).all()
        whole = torch.full((n * h + 33,), 77.0, dtype=torch.bfloat16, device=dev)
        out = whole[17:17 + n * h]
        _lib.call("mrl_embedding_fwd", ids.data_ptr(), _lib.I64, n, 0, w.data_ptr(), _lib.BF16, vocab, h, 1.0, out.data_ptr(),
                  _lib.stream(dev))
        assert torch.equal(out.view(n, h), w[ids])
        assert (whole[:17] == 77).all() and (whole[17 + n * h:] == 77).all()


@pytest.mark.gpu
def test_streams_and_graphs(dev):
    """On another stream; two graphs, replayed in turn with new tokens, against eager passes."""
    g = torch.Generator(device=dev).manual_seed(10)
    w = torch.randn(700, 72, generator=g, device=dev).to(torch.bfloat16)
    batches = [(torch.randint(-5, 700, (1500,), generator=g, device=dev),
                torch.randn(1500, 72, generator=g, device=dev).to(torch.bfloat16)) for _ in range(5)]
    static = [t.clone() for t in batches[0]]

    def step(ids, dy):
        t = w.detach().requires_grad_()
        y = mrl.token_embedding(ids, t, scale=2.0)
        sums = torch.zeros(700, 72, device=dev)
        mrl.token_embedding_grad(ids, dy, sums, accumulate=True)
        return (y.detach(), *torch.autograd.grad(y, [t], dy), sums)

    want = step(*batches[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(*static)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    captured = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            captured.append(step(*static))
    for ids, dy in batches:
        static[0].copy_(ids)
        static[1].copy_(dy)
        eager = step(ids, dy)
        for graph, got in zip(graphs, captured):
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(got, eager))


@pytest.mark.gpu
@pytest.mark.parametrize("hidden", [4, 64, 257, 520])
def test_runs_that_cross_shares(dev, hidden):
    """Tokens that are there 1 to 1 100 times, around every multiple of 8 of them at which a sum is taken another way.  Gradients of
    small whole numbers: their sums are exact in whatever order, so equal bits are wanted."""
    lengths = [8 * k + off for k in (1, 2, 3, 14, 15, 16, 17, 18, 31, 32, 33, 63, 64, 65, 79, 80, 81, 82, 136) for off in (-1, 0, 1, 9)]
    vocab = len(lengths) + 3
    g = torch.Generator(device=dev).manual_seed(8)
    ids = torch.repeat_interleave(torch.arange(len(lengths), device=dev), torch.tensor(lengths, device=dev))
    for left_out in (0, 1, 5):                      # the list's places against the shares' move
        some = torch.cat([ids[left_out:], torch.full((100,), vocab + 7, device=dev)])
        some = some[torch.randperm(some.numel(), generator=g, device=dev)]
        dy = torch.randint(-2, 3, (some.numel(), hidden), generator=g, device=dev).float()
        inside = some < vocab
        want = torch.zeros(vocab, hidden, device=dev).index_add_(0, some[inside], dy[inside])
        out = torch.full((vocab, hidden), float("nan"), device=dev)
        assert torch.equal(mrl.token_embedding_grad(some, dy, out), want)
        assert torch.equal(mrl.token_embedding_grad(some, dy, out, scale=-3.0, accumulate=True), want - 3.0 * want)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1500, 30000])
def test_the_largest_table(dev, n):
    """2^31 - 2 rows, of one entry: row numbers of 31 bits, and the largest of them next to the ids that are outside."""
    vocab = (1 << 31) - 2
    ids = torch.randint(0, vocab + 1, (n,), device=dev)
    ids[:40], ids[40:80] = vocab - 1, vocab
    ids[80:90], ids[90:100] = 0, -1
    table = torch.zeros(vocab, 1, dtype=torch.bfloat16, device=dev)
    table[-1], table[0] = 3.0, 5.0
    y = mrl.token_embedding(ids, table)
    assert (y[:40] == 3).all() and not y[40:80].any() and (y[80:90] == 5).all() and not y[90:100].any()
    mrl.token_embedding_grad(ids, torch.ones(n, 1, dtype=torch.bfloat16, device=dev), table, accumulate=True)
    rows, counts = ids[(ids >= 0) & (ids < vocab)].unique(return_counts=True)
    want = counts.float() + 3.0 * (rows == vocab - 1) + 5.0 * (rows == 0)
    assert torch.equal(table[rows, 0].float(), want)            # whole numbers below 256
    table[rows] = 0
    assert not table.any()


@pytest.mark.gpu
def test_more_entries_than_31_bits(dev):
    """A table of more than 2^31 entries, and a gradient of as many."""
    vocab, h = 600011, 3584
    w = torch.zeros(vocab, h, dtype=torch.bfloat16, device=dev)
    w[-40:] = torch.randn(40, h, device=dev)
    ids = torch.tensor([vocab - 1, 3, vocab - 40, vocab - 2, vocab - 1], device=dev)
    assert torch.equal(mrl.token_embedding(ids, w), w[ids])
    dy = torch.randn(5, h, device=dev).to(torch.bfloat16)
    out = torch.full_like(w, float("nan"))
    mrl.token_embedding_grad(ids, dy, out)
    assert torch.equal(out[-1], (dy[0].float() + dy[4].float()).bfloat16())
    assert torch.equal(out[[3, vocab - 40, vocab - 2]], dy[[1, 2, 3]])
    out[ids] = 0
    assert not out.any()
    del w, out
    n = 600001
    ids = torch.full((n,), 9, device=dev)
    ids[-3:] = torch.tensor([0, 1, 0], device=dev)
    table = torch.randn(10, h, device=dev).to(torch.bfloat16)
    y = mrl.token_embedding(ids, table)
    assert torch.equal(y[-3:], table[[0, 1, 0]]) and torch.equal(y[:100], table[9].expand(100, h))
    y.zero_()
    y[-3:] = dy[:3]
    sums = torch.empty(10, h, device=dev)
    mrl.token_embedding_grad(ids, y, sums)
    assert torch.equal(sums[0], dy[0].float() + dy[2].float()) and torch.equal(sums[1], dy[1].float()) and not sums[2:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,h", [(torch.bfloat16, 8), (torch.float32, 4), (torch.bfloat16, 3)], ids=["8xbf16", "4xf32", "3xbf16"])
def test_the_most_tokens(dev, dtype, h):
    """2^26 - 1 tokens, three more than a launch holds wavefronts in workgroups of four: all of them looked up, and summed.
    The gradient of ones: counts below 2^24, exact in fp32."""
    n, vocab = (1 << 26) - 1, 50
    g = torch.Generator(device=dev).manual_seed(12)
    table = torch.randn(vocab, h, generator=g, device=dev).to(dtype)
    ids = torch.randint(0, vocab, (n,), generator=g, device=dev, dtype=torch.int32)
    for some in (ids, ids[:-2], ids[:-3]):              # one launch holds the last of them
        y = mrl.token_embedding(some, table)
        assert all(torch.equal(part, table[i.long()]) for part, i in zip(y.split(1 << 23), some.split(1 << 23)))
        del y
    out = torch.empty(vocab, h, device=dev)
    mrl.token_embedding_grad(ids, torch.ones(n, h, dtype=dtype, device=dev), out)
    counts = torch.bincount(ids, minlength=vocab)
    assert counts.max() < 1 << 24 and torch.equal(out, counts.float()[:, None].expand(vocab, h))
