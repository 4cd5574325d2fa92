"""The operators of a decoder layer and of the update's last step together, as a training loop would use them."""
import pytest
import torch

import mindspeed_rl_amd as mrl

BF16, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    torch.cuda.set_device(0)
    return torch.device("cuda:0")


@pytest.mark.gpu
@pytest.mark.parametrize("stream", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("kind", ["ray_grpo", "ray_dapo", "ray_ppo"])
def test_loss_objects_add_the_residual(dev, kind, stream):
    """final_norm_residual= is add_rms_norm in front of the same call: the same loss, gradients and scores, bit for bit."""
    from test_step_gradients import _batch, _loss_object
    g = torch.Generator(device=dev).manual_seed(5)
    vocab, h = 1000, 128
    _, batch, kw = _batch(dev, g, vocab)
    hidden = torch.randn(1, batch["labels"].shape[1], h, generator=g, device=dev).to(BF16).requires_grad_()
    residual = torch.randn(hidden.shape, generator=g, device=dev).to(stream).requires_grad_()
    head = (torch.randn(vocab, h, generator=g, device=dev) * 0.1).to(BF16).requires_grad_()
    w = (1 + 0.1 * torch.randn(h, generator=g, device=dev)).to(BF16).requires_grad_()
    extra = dict(final_norm_weight=w, final_norm_eps=1e-4, final_norm_residual=residual)
    leaves = [hidden, residual, head, w]
    fn = _loss_object(kind)
    loss, stats = fn.compute_loss(hidden, batch, lm_head_weight=head, **extra, **kw)
    grads = torch.autograd.grad(loss, leaves)
    want_loss, want_stats = _loss_object(kind).compute_loss(mrl.add_rms_norm(hidden, residual, w, 1e-4)[0], batch, lm_head_weight=head, **kw)
    want = torch.autograd.grad(want_loss, leaves)
    assert torch.equal(loss, want_loss) and dict(stats) == dict(want_stats)
    assert all(torch.equal(p, q) for p, q in zip(grads, want)) and all(q.abs().max() > 0 for q in want)
    score = fn.compute_loss(hidden, batch, forward_only=True, lm_head_weight=head, **extra, **kw)
    with torch.no_grad():
        assert torch.equal(score, fn.compute_loss(mrl.add_rms_norm(hidden, residual, w, 1e-4)[0], batch, forward_only=True,
                                                  lm_head_weight=head, **kw))


# ------------------------------------------------------------------------------------ a small decoder
VOCAB, H, HEADS, KV, DIM, INNER, LAYERS = 256, 64, 4, 2, 16, 96, 2


def weights(dev, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    layer = lambda: [1 + 0.1 * n(H), n((HEADS + 2 * KV) * DIM, H) / 8, n(H, HEADS * DIM) / 8, 1 + 0.1 * n(H), n(INNER, H) / 8, n(H, INNER) / 10]  # noqa: E731
    return [n(VOCAB, H) * 0.5] + [t for _ in range(LAYERS) for t in layer()] + [1 + 0.1 * n(H), n(VOCAB, H) / 8]


def packed(dev):
    """Two prompts of different lengths as preprocess_packed_seqs lays them out, and who may look at whom."""
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(0, VOCAB, (2, 24), generator=g).to(dev)
    mask = mrl.generate_mask(ids, torch.tensor([[24], [17]], dtype=torch.int32, device=dev))
    flat, positions, labels, seqlens, _ = mrl.preprocess_packed_seqs(ids, torch.roll(ids, -1, 1), mask, 1)
    owner = torch.repeat_interleave(torch.arange(2, device=dev), seqlens.long())
    at = torch.arange(owner.numel(), device=dev)
    sees = (owner[:, None] == owner[None, :]) & (at[None, :] <= at[:, None])
    return flat, positions, labels, sees


def attention(q, k, v, sees):
    k, v = (t.repeat_interleave(HEADS // KV, 1) for t in (k, v))
    scores = torch.matmul(q.transpose(0, 1), k.permute(1, 2, 0).contiguous()) * DIM ** -0.5
    return torch.matmul(scores.masked_fill(~sees, float("-inf")).softmax(-1), v.transpose(0, 1).contiguous()).transpose(0, 1).reshape(q.shape[0], -1)


def forward(ws, data, ops):
    """The mean log-probability of the labels."""
    embed, norm, add_norm, rotary, logprob = ops
    flat, positions, labels, sees = data
    table, *layers, last, head = ws
    h = embed(flat, table)[0]
    x = None
    for k in range(LAYERS):
        w1, qkv, out, w2, up, down = layers[6 * k:6 * k + 6]
        y, h = (norm(h, w1), h) if x is None else add_norm(x, h, w1)
        heads = (y @ qkv.t()).view(-1, HEADS + 2 * KV, DIM)
        q, key = rotary(heads[:, :HEADS], heads[:, HEADS:HEADS + KV], positions)
        x = attention(q, key, heads[:, HEADS + KV:], sees) @ out.t()
        y, h = add_norm(x, h, w2)
        x = torch.tanh(y @ up.t()) @ down.t()
    y, _ = add_norm(x, h, last)
    return logprob(y @ head.t(), labels[0]).mean()


def own(dev):
    inv, scale = mrl.rotary_frequencies(DIM, device=dev)
    return (mrl.token_embedding, mrl.rms_norm, mrl.add_rms_norm, lambda q, k, p: mrl.rotary(q, k, p, inv, scale=scale),
            lambda z, lab: mrl.vocab_logprob_entropy(z, lab)[0])


def plain(dev):
    """The same in elementary operations, for 64 bits."""
    inv = 10000.0 ** (-torch.arange(0, DIM, 2, device=dev, dtype=torch.float64) / DIM)

    def norm(x, w):
        return x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w

    def turn(x, p):
        t = (p[0].double()[:, None] * inv)[:, None, :]
        a, b = x.chunk(2, -1)
        return torch.cat([a * t.cos() - b * t.sin(), b * t.cos() + a * t.sin()], -1)

    return (lambda i, t: t[i], norm, lambda x, r, w: (norm(x + r, w), x + r), lambda q, k, p: (turn(q, p), turn(k, p)),
            lambda z, lab: torch.log_softmax(z, -1).gather(-1, lab[:, None].long())[:, 0])


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_three_updates(dev, bits):
    """Forward, backward, norm and step, three times: the loss and its gradients against the whole in 64 bits, each step of the weights
    and moments against the formula from the gradients that came out.

    The chain has 8 products forward and twice as many back, over at most 256 terms: 256 U each of the terms' magnitudes, and norms,
    softmax and attention between them that pass relative errors on by factors of a few.  24 x 256 U x 4 = 1.5e-3 of a tensor's norm."""
    from test_optimizer_step import check, clone, factor_of
    data = packed(dev)
    params = weights(dev, 2)
    state = mrl.adamw_state(params, bits=bits)
    hyper = dict(lr=1e-2, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)
    bound = 24 * 256 * U * 4
    for _ in range(3):
        leaves = [p.detach().requires_grad_() for p in params]
        loss = -forward(leaves, data, own(dev))
        grads = torch.autograd.grad(loss, leaves)
        wide = [p.double().requires_grad_() for p in params]
        want = -forward(wide, data, plain(dev))
        assert abs(loss.item() - want.item()) <= bound * abs(want.item())
        for g, w in zip(grads, torch.autograd.grad(want, wide)):
            assert w.norm() > 0 and (g.double() - w).norm() <= bound * w.norm()
        norm = mrl.global_grad_norm(grads)
        limit = 0.5 * norm.item()
        old_params, old = clone(params, state)
        mrl.adamw_(params, grads, **state, grad_norm=norm, max_norm=limit, **hyper)
        check(params, grads, state, old_params, old, factor_of(norm, limit), hyper)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_an_update_captured_and_replayed(dev, bits):
    """The whole update in one graph: after each replay weights, moments and loss have the bits of the eager update's."""
    data = packed(dev)
    ops = own(dev)

    def update(params, state):
        leaves = [p.detach().requires_grad_() for p in params]
        loss = -forward(leaves, data, ops)
        grads = torch.autograd.grad(loss, leaves)
        mrl.adamw_(params, grads, **state, lr=3e-3, grad_norm=mrl.global_grad_norm(grads), max_norm=0.1)
        return loss.detach()

    sides = []
    for _ in range(2):
        params = weights(dev, 3)
        sides.append((params, mrl.adamw_state(params, bits=bits)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        update(*sides[0])
        update(*sides[1])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = update(*sides[0])
    for _ in range(4):
        want = update(*sides[1])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(loss, want)
        flat = [[*p, *(t for v in s.values() for t in (v if isinstance(v, list) else [v]) if t is not None)] for p, s in sides]
        for a, b in zip(*flat):
            assert torch.equal(a.view(torch.uint8) if a.dtype is torch.float8_e4m3fn else a, b.view(torch.uint8) if b.dtype is torch.float8_e4m3fn else b)


@pytest.mark.gpu
def test_a_scoring_layer_in_eight_bits(dev):
    """add_rms_norm's 8-bit form in front of a product: what q and scale stand for, times a weight, within the codes' half steps of the
    product that bf16 rows give: 2^-4 of each entry at most, summed up with the weight's magnitudes."""
    g = torch.Generator(device=dev).manual_seed(4)
    x, r = (torch.randn(40, 256, generator=g, device=dev).to(BF16) for _ in range(2))
    w, product = (1 + 0.1 * torch.randn(256, generator=g, device=dev)).to(BF16), torch.randn(32, 256, generator=g, device=dev)
    y, h = mrl.add_rms_norm(x, r, w)
    for block in (None, 128):
        q, scale, h8 = mrl.rms_norm_fp8(x, w, residual=r, block=block)
        assert torch.equal(h, h8)
        stands = (q.double().view(40, -1, block or 256) * scale.double()[..., None]).view(40, 256)
        got, want = stands @ product.double().t(), y.double() @ product.double().t()
        half = (2.0 ** -4 * 1.01 + 2.0 ** -8) * y.double().abs() + 2.0 ** -10 * scale.double().amax(-1, keepdim=True)
        assert ((got - want).abs() <= half @ product.double().abs().t()).all()


def _parts(dev, seed):
    """What one call of each operator takes, and the call."""
    g = torch.Generator(device=dev).manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    x, r, dy, dh, w = n(700, 520).to(BF16), n(700, 520), n(700, 520).to(BF16), n(700, 520), 1 + 0.1 * n(520)
    q, k, gq, gk = n(300, 6, 64).to(BF16), n(300, 2, 64).to(BF16), n(300, 6, 64).to(BF16), n(300, 2, 64).to(BF16)
    pos = torch.randint(0, 5000, (300,), generator=g, device=dev)
    inv, _ = mrl.rotary_frequencies(64, device=dev)
    params, grads = [n(900, 33), n(5000).to(BF16)], [n(900, 33), n(5000)]
    state = mrl.adamw_state(params, bits=8)

    def call():
        ts = [t.detach().requires_grad_() for t in (x, r, w)]
        y, h = mrl.add_rms_norm(*ts)
        got = [y.detach(), h.detach(), *torch.autograd.grad([y, h], ts, [dy, dh])]
        ts = [t.detach().requires_grad_() for t in (q, k)]
        out = mrl.rotary(*ts, pos, inv)
        got += [*(t.detach() for t in out), *torch.autograd.grad(out, ts, [gq, gk])]
        codes, scale = mrl.rms_norm_fp8(x, w)
        mrl.adamw_(params, grads, **state, lr=1e-3, grad_norm=mrl.global_grad_norm(grads), max_norm=1.0)
        return [*got, codes.float(), scale, *params, *(t.float() for t in state["exp_avg"] + state["exp_avg_sq"])]

    return call


@pytest.mark.gpu
def test_two_streams_at_once(dev):
    """Calls that overlap in time, each with a workspace of its own: the bits that they give one after the other."""
    want = [[[t.clone() for t in call()] for _ in range(6)] for call in (_parts(dev, 1), _parts(dev, 2))]
    calls, streams = [_parts(dev, 1), _parts(dev, 2)], [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(6):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                got[k].append([t.clone() for t in calls[k]()])
    torch.cuda.synchronize()
    for k in range(2):
        for a, b in zip(got[k], want[k]):
            assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.gpu
def test_two_graphs_of_one_pool(dev):
    """Captured one behind the other into one pool of memory and replayed in turn: the bits of the eager calls."""
    eager, calls = [_parts(dev, 3), _parts(dev, 4)], [_parts(dev, 3), _parts(dev, 4)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for call in (*eager, *calls):
            call()
    torch.cuda.current_stream().wait_stream(side)
    graphs, captured = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for k, graph in enumerate(graphs):
        with torch.cuda.graph(graph, pool=graphs[0].pool() if k else None):
            captured.append(calls[k]())
    for _ in range(4):
        for k in range(2):
            want = eager[k]()
            graphs[k].replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(captured[k], want))
