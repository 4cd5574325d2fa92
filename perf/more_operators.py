"""Performance cases of the operators that surround a decoder layer's products, and of the update's last step: RMS norm with the
residual's addition (also to 8 bits), rotary positions, and AdamW over a list of parameters.

``run`` computes them in their plain form, by elementary torch operations in 32 bits (64 for angles and for values next to a
border between two codes), or, where ``own`` is true, by the framework's entry points.  A case is a dict of plain values; its
inputs follow from it and a seed.

* ``addnorm``  ``h = x + residual``, rounded to the residual's type, and the RMS norm of ``h``; forward only, or forward and backward
               with gradients arriving at both outputs
* ``normfp8``  the norm's output as e4m3 with a scale for each row or for each 128 entries, with or without a residual
* ``rotary``   queries and keys (views of one projection's output) turned by their positions; forward only, or with the backward
* ``adamw``    one step over many tensors, clipped by a norm that is there already; moments in 32 or in 8 bits

Moments in 8 bits: blocks of 128 entries of a tensor hold e4m3 codes of ``m / s`` and of ``sqrt(v) / s``, with an fp32 scale ``s =
max(largest / 448, 2^-126)`` each.  ``|x|`` in steps of its binade goes down to ``floor(|x| / step + u)``, ``u`` the 16 bits
that :func:`_dither` makes of the step's number and the entry's place; a ``sqrt(v)`` that is not zero keeps at least the least code.
"""
import math
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.getcwd(), "mindspeed-rl_amd"))       # imported with the repository's root as working folder

own = False

_DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32, "f16": torch.float16}
_BYTES = {"bf16": 2, "f32": 4, "f16": 2}
_E4M3, _MOST, _LEAST = torch.float8_e4m3fn, 448.0, 2.0 ** -126
_BLOCK = 128
_ADAM = dict(lr=3e-4, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)


# ------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one sequence's new token between two layers: latency alone
        dict(name="addnorm_token", op="addnorm", dtype="bf16", stream="bf16", rows=1, hidden=3584, step=False),
        # an update's micro-batch of 32 k tokens
        dict(name="addnorm_step", op="addnorm", dtype="bf16", stream="bf16", rows=32768, hidden=3584, step=True),
        # an odd number of rows of an odd width, fp16 beside a residual stream in fp32
        dict(name="addnorm_odd_step", op="addnorm", dtype="f16", stream="f32", rows=9477, hidden=1343, step=True),
        # a scoring pass of 64 k tokens, in front of a product in 8 bits with a scale per 128 entries
        dict(name="normfp8_score", op="normfp8", dtype="bf16", stream="bf16", rows=65536, hidden=5120, residual=True, block=128),
        # a small batch without a residual, a scale per row
        dict(name="normfp8_rows", op="normfp8", dtype="bf16", stream="bf16", rows=2500, hidden=1343, residual=False, block=0),
        # the tokens that 64 long sequences have just drawn
        dict(name="rotary_tokens", op="rotary", dtype="bf16", rows=64, q_heads=28, k_heads=4, head=128, part=128, start=0,
             interleaved=False, far=131072, step=False),
        # the update's packed micro-batch, forward and backward
        dict(name="rotary_step", op="rotary", dtype="bf16", rows=32768, q_heads=28, k_heads=4, head=128, part=128, start=0,
             interleaved=False, far=8192, step=True),
        # an odd number of tokens, pairs side by side in the last part of wider heads, one key head for all
        dict(name="rotary_part", op="rotary", dtype="f16", rows=9477, q_heads=16, k_heads=1, head=192, part=64, start=-64,
             interleaved=True, far=32768, step=False),
        # a small model in fp32 with odd sizes: many tensors, latency
        dict(name="adamw_small", op="adamw", dtype="f32", grad="f32", bits=32, master=False, layers=2, hidden=255, vocab=4001, clip=True),
        # bf16 weights with fp32 main weights, gradients and moments
        dict(name="adamw_step", op="adamw", dtype="bf16", grad="f32", bits=32, master=True, layers=12, hidden=2048, vocab=32000,
             clip=True),
        # the same update with moments in 8 bits and bf16 gradients, two wider layers
        dict(name="adamw_8bit", op="adamw", dtype="bf16", grad="bf16", bits=8, master=True, layers=2, hidden=3584, vocab=32000,
             clip=True),
        # a critic's few layers in fp32 with moments in 8 bits, widths that end inside a block
        dict(name="adamw_8bit_odd", op="adamw", dtype="f32", grad="f32", bits=8, master=False, layers=3, hidden=1023, vocab=1001,
             clip=False),
    ]


def _log_uniform(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def _draw_width(rng, lo, hi, whole):
    w = int(_log_uniform(rng, lo, hi))
    return max(lo, w // whole * whole if rng.random() < 0.6 else w)


def draw(rng):
    op = rng.choice(["addnorm", "normfp8", "rotary", "adamw"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op in ("addnorm", "normfp8"):
        block = rng.choice([0, 128]) if op == "normfp8" else 0
        hidden = _draw_width(rng, 64, 8192, 64)
        hidden = max(128, hidden // 128 * 128) if block else hidden
        stream = rng.choice([dtype, dtype, "f32"])
        most = 32768 * 3584 * 2 // (hidden * _BYTES[stream])
        case = dict(op=op, dtype=dtype, stream=stream, rows=max(1, int(_log_uniform(rng, 1, min(most, 65536)))), hidden=hidden)
        if op == "addnorm":
            return dict(case, step=rng.random() < 0.7)
        return dict(case, residual=rng.random() < 0.6, block=block)
    if op == "rotary":
        head = rng.choice([64, 72, 80, 96, 128, 128, 192, 256])
        part = rng.choice([head, head, head // 2, head // 4 // 2 * 2])
        kv = rng.choice([1, 2, 4, 8])
        q = kv * rng.choice([1, 2, 4, 7])
        most = 32768 * 32 * 128 * 2 // ((q + kv) * head * _BYTES[dtype])
        return dict(op=op, dtype=dtype, rows=max(1, int(_log_uniform(rng, 1, min(most, 65536)))), q_heads=q, k_heads=kv, head=head,
                    part=part, start=rng.choice([0, 0, -part]), interleaved=rng.random() < 0.4, far=int(_log_uniform(rng, 1000, 1 << 20)),
                    step=rng.random() < 0.6)
    bits = rng.choice([32, 8])
    return dict(op=op, dtype=dtype, grad=rng.choice([dtype, "f32"]), bits=bits, master=dtype != "f32" and rng.random() < 0.7,
                layers=rng.randint(1, 6), hidden=_draw_width(rng, 64, 2048 if bits == 32 else 1500, 64),
                vocab=int(_log_uniform(rng, 1000, 32000)), clip=rng.random() < 0.7)


def _shapes(case):
    """The parameters of a decoder of `layers` layers: products of attention and feed-forward, two norms each, table and last norm."""
    h, f = case["hidden"], case["hidden"] * 7 // 2
    layer = [(h,), (h, h), (h // 4, h), (h // 4, h), (h, h), (h,), (f, h), (f, h), (h, f)]
    return [(case["vocab"], h)] + layer * case["layers"] + [(h,)]


def work(case):
    size = _BYTES[case["dtype"]]
    if case["op"] in ("addnorm", "normfp8"):
        n, h, wide = case["rows"] * case["hidden"], case["hidden"], _BYTES[case["stream"]]
        if case["op"] == "normfp8":
            scales = case["rows"] * (h // case["block"] if case["block"] else 1) * 4
            return {"bytes": n * (size + 1 + (2 * wide if case["residual"] else 0)) + scales + h * size, "flops": 8 * n}
        # x and the residual in, h and y out
        moved = n * (2 * size + 2 * wide) + h * size
        if not case["step"]:
            return {"bytes": moved, "flops": 7 * n}
        # dy and dh in, the gradient of the sum out, in each type once, and the weight's; h stays what the forward wrote
        return {"bytes": moved + n * (size + wide + wide + (size if wide != size else 0)) + 2 * h * size, "flops": 20 * n}
    if case["op"] == "rotary":
        n = case["rows"] * (case["q_heads"] + case["k_heads"]) * case["head"]
        passes = 2 if case["step"] else 1
        return {"bytes": passes * (2 * n * size) + case["rows"] * 8, "flops": passes * 6 * n}
    n = sum(math.prod(s) for s in _shapes(case))
    blocks = sum(-(-math.prod(s) // _BLOCK) for s in _shapes(case))
    moments = 16 * n if case["bits"] == 32 else 4 * n + 16 * blocks
    weights = (size + 8 if case["master"] else 2 * size) * n
    return {"bytes": weights + _BYTES[case["grad"]] * n + moments, "flops": 16 * n}


# ------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = _DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=gen, device=dev) * scale

    state = dict(case)
    if case["op"] in ("addnorm", "normfp8"):
        r, h, wide = case["rows"], case["hidden"], _DTYPES[case["stream"]]
        # a residual stream has a few columns that are much larger than the others; a layer's output is smaller
        column = torch.exp(normal(h, scale=0.5))
        state["x"] = (normal(r, h, scale=0.5) * torch.exp(normal(r, 1, scale=0.3))).to(dt)
        state["weight"] = (1 + normal(h, scale=0.2)).to(dt)
        if case["op"] == "addnorm" or case["residual"]:
            state["stream_"] = (normal(r, h) * column + 0.1 * column).to(wide)
        if case.get("step"):
            state["dy"] = (normal(r, h, scale=1e-2) * torch.exp(normal(r, 1))).to(dt)
            state["dh"] = normal(r, h, scale=1e-2).to(wide)
            state["inputs"] = [state[k].requires_grad_() for k in ("x", "stream_", "weight")]
        return state
    if case["op"] == "rotary":
        t, q, k, d, part = case["rows"], case["q_heads"], case["k_heads"], case["head"], case["part"]
        # queries, keys and values of a token lie together, as the projection wrote them
        whole = normal(t, (q + 2 * k) * d).to(dt)
        state["q"] = whole[:, :q * d].view(t, q, d)
        state["k"] = whole[:, q * d:(q + k) * d].view(t, k, d)
        # packed sequences: positions count up from where a sequence begins; of single tokens, wherever each one is
        if t < 256:
            state["positions"] = torch.randint(0, case["far"], (t,), generator=gen, device=dev)
        else:
            begins = torch.rand(t, generator=gen, device=dev) < 4.0 / min(t, case["far"])
            at = torch.arange(t, device=dev)
            first = torch.where(begins, at, 0).cummax(0).values
            state["positions"] = (at - first + torch.randint(0, case["far"], (1,), generator=gen, device=dev)) % case["far"]
        state["inv_freq"] = 1e6 ** (-torch.arange(0, part, 2, device=dev, dtype=torch.float64) / part)
        state["scale"] = 1.0 if case["start"] == 0 else 1.2       # stretched to longer contexts: the logits' temperature
        if case["step"]:
            state["inputs"] = [state[n].detach().requires_grad_() for n in ("q", "k")]
            state["grads"] = [normal(t, n, d, scale=1e-2).to(dt) for n in (q, k)]
        return state
    shapes = _shapes(case)
    sizes = [math.prod(s) for s in shapes]
    n, blocks = sum(sizes), [-(-s // _BLOCK) for s in sizes]
    weights = torch.empty(n, device=dev).normal_(0, 0.02, generator=gen)
    flat = {"param": weights.to(dt), "grad": torch.empty(n, dtype=_DTYPES[case["grad"]], device=dev)}
    if case["master"]:
        flat["master"] = weights
    small = case["bits"] == 8
    flat["m"] = torch.empty(n, dtype=_E4M3 if small else torch.float32, device=dev)
    flat["v"] = torch.empty(n, dtype=_E4M3 if small else torch.float32, device=dev)
    if small:
        flat["m_scale"] = torch.empty(sum(blocks), device=dev)
        flat["v_scale"] = torch.empty(sum(blocks), device=dev)
    lists = {name: [p.view(s) for p, s in zip(f.split(blocks if name.endswith("scale") else sizes),
                                              [(b,) for b in blocks] if name.endswith("scale") else shapes)]
             for name, f in flat.items()}
    squares = torch.zeros((), dtype=torch.float64, device=dev)
    for k, s in enumerate(shapes):
        # rows of different size; rows of the table that no token named have none
        row = torch.exp(normal(s[0], *[1] * (len(s) - 1)))
        row = row * (torch.rand(row.shape, generator=gen, device=dev) < (0.4 if k == 0 else 1.0))
        g = normal(*s, scale=1e-3) * row
        lists["grad"][k].copy_(g)
        squares += lists["grad"][k].double().square().sum()
        m, d = normal(*s, scale=2e-4) * row, torch.exp(normal(*s, scale=0.5)) * 8e-4 * row
        if small:
            for name, x in (("m", m), ("v", d)):
                code, scale = _nearest_codes(x)
                lists[name][k].copy_(code)
                lists[name + "_scale"][k].copy_(scale)
        else:
            lists["m"][k].copy_(m)
            lists["v"][k].copy_(d.square())
    state["flat"], state["lists"] = flat, lists
    state["steps"] = torch.full((), 20 + seed % 100, dtype=torch.int64, device=dev)     # steps that were taken
    state["norm"] = squares.sqrt().float()
    state["limit"] = 0.5e-3 * math.sqrt(n)                                              # lies below the norm
    return state


def _rows_of_blocks(x):
    """A tensor's entries in rows of 128, zeros behind the last."""
    x = x.reshape(-1)
    return torch.nn.functional.pad(x, (0, -x.numel() % _BLOCK)).view(-1, _BLOCK)


def _nearest_codes(x):
    b = _rows_of_blocks(x)
    scale = (b.abs().amax(1) * (1 / _MOST)).clamp(min=_LEAST)
    code = (b / scale[:, None]).clamp(-_MOST, _MOST)
    return code.reshape(-1)[:x.numel()].view(x.shape).to(_E4M3), scale


# ------------------------------------------------------------------------------------------ one pass
def run(state):
    return _RUN[state["op"]](state) if own else _PLAIN[state["op"]](state)


def _run_addnorm(state):
    import mindspeed_rl_amd as mrl
    y, h = mrl.add_rms_norm(state["x"], state["stream_"], state["weight"], eps=1e-6)
    if not state["step"]:
        return {"y": y, "h": h}
    return {"y": y.detach(), "h": h.detach(), "grads": torch.autograd.grad([y, h], state["inputs"], [state["dy"], state["dh"]])}


def _run_normfp8(state):
    import mindspeed_rl_amd as mrl
    return mrl.rms_norm_fp8(state["x"], state["weight"], eps=1e-6, residual=state.get("stream_"), block=state["block"] or None)


def _run_rotary(state):
    import mindspeed_rl_amd as mrl
    q, k = state["inputs"] if state["step"] else (state["q"], state["k"])
    out = mrl.rotary(q, k, state["positions"], state["inv_freq"], interleaved=state["interleaved"], start=state["start"],
                     scale=state["scale"])
    if not state["step"]:
        return out
    return tuple(t.detach() for t in out) + tuple(torch.autograd.grad(out, state["inputs"], state["grads"]))


def _run_adamw(state):
    import mindspeed_rl_amd as mrl
    t = state["lists"]
    mrl.adamw_(t["param"], t["grad"], t["m"], t["v"], state["steps"], master=t.get("master"), exp_avg_scale=t.get("m_scale"),
               exp_avg_sq_scale=t.get("v_scale"), grad_norm=state["norm"] if state["clip"] else None,
               max_norm=state["limit"] if state["clip"] else None, **_ADAM)
    return _updated(state)


def _updated(state):
    return {"steps": state["steps"], **{k: v for k, v in state["flat"].items() if k != "grad"}}


_RUN = {"addnorm": _run_addnorm, "normfp8": _run_normfp8, "rotary": _run_rotary, "adamw": _run_adamw}


# ------------------------------------------------------------------------------------------ the plain forms
def _plain_addnorm(state):
    with torch.no_grad():
        # the stream as the next layer finds it is what is normalised
        h = (state["x"].float() + state["stream_"].float()).to(state["stream_"].dtype)
        z, w = h.float(), state["weight"].float()
        r = torch.rsqrt(z.square().mean(-1, keepdim=True) + 1e-6)
        n = z * r
        y = (n * w).to(state["x"].dtype)
        if not state["step"]:
            return {"y": y, "h": h}
        dy = state["dy"].float()
        g = dy * w
        d = (g - n * (g * n).mean(-1, keepdim=True)) * r + state["dh"].float()
        return {"y": y, "h": h, "grads": (d.to(state["x"].dtype), d.to(h.dtype), (dy * n).sum(0).to(state["weight"].dtype))}


def _plain_normfp8(state):
    with torch.no_grad():
        x, h = state["x"], None
        if state["residual"]:
            h = (x.float() + state["stream_"].float()).to(state["stream_"].dtype)
        z = (x if h is None else h).float()
        y = z * torch.rsqrt(z.square().mean(-1, keepdim=True) + 1e-6) * state["weight"].float()
        groups = y.view(y.shape[0], -1, state["block"] or y.shape[1])
        scale = (groups.abs().amax(-1, keepdim=True) * (1 / _MOST)).clamp(min=_LEAST)
        q = (groups / scale).clamp(-_MOST, _MOST).to(_E4M3).view(y.shape)
        scale = scale.view(y.shape[0], -1)
        return (q, scale) if h is None else (q, scale, h)


def _turned(x, cos, sin, state):
    begin = state["start"] % x.shape[-1]
    part = x[..., begin:begin + state["part"]].float()
    half = state["part"] // 2
    a, b = (part[..., 0::2], part[..., 1::2]) if state["interleaved"] else (part[..., :half], part[..., half:])
    both = a * cos - b * sin, b * cos + a * sin
    part = torch.stack(both, -1).flatten(-2) if state["interleaved"] else torch.cat(both, -1)
    return torch.cat([x[..., :begin], part.to(x.dtype), x[..., begin + state["part"]:]], -1)


def _plain_rotary(state):
    with torch.no_grad():
        angle = (state["positions"].double()[:, None] * state["inv_freq"])[:, None, :]
        cos, sin = (angle.cos() * state["scale"]).float(), (angle.sin() * state["scale"]).float()
        out = _turned(state["q"], cos, sin, state), _turned(state["k"], cos, sin, state)
        if not state["step"]:
            return out
        return out + tuple(_turned(g, cos, -sin, state) for g in state["grads"])


def _dither(steps, n):
    """16 bits for each of n entries: a mixed 32-bit word for each pair, its lower half for the first."""
    key = (steps * 0x9E3779B9) & 0xffffffff
    x = torch.arange((n + 1) // 2, device=steps.device) ^ key
    x = ((x ^ (x >> 16)) * 0x7feb352d) & 0xffffffff
    x = ((x ^ (x >> 15)) * 0x846ca68b) & 0xffffffff
    x = x ^ (x >> 16)
    return torch.stack([x & 0xffff, x >> 16], 1).view(-1)[:n]


def _dithered(x, bits, least):
    """(e4m3 codes of a tensor of fp32, scales): |x| in steps of its binade, up or down by the dither."""
    rows = _rows_of_blocks(x)
    scale = (rows.abs().amax(1) * (1 / _MOST)).clamp(min=_LEAST)
    rows = (rows * scale.reciprocal()[:, None]).clamp(-_MOST, _MOST)
    size = rows.abs().view(-1)[:x.numel()].double()
    if least:
        size = torch.where(x.reshape(-1) > 0, size.clamp(min=2.0 ** -9), 0.0)
    step = torch.ldexp(torch.ones_like(size), (torch.frexp(size).exponent - 4).clamp(min=-9))
    size = torch.floor(size / step + bits * 2.0 ** -16) * step
    return torch.copysign(size.float(), x.reshape(-1)).to(_E4M3).view(x.shape), scale


def _held(code, scale):
    """What codes and scales stand for."""
    return (_rows_of_blocks(code.float()) * scale[:, None]).view(-1)[:code.numel()].view(code.shape)


def _plain_tensor(factor, rate, second, decay, steps, p, g, master, m, v, m_scale, v_scale):
    b1, b2 = _ADAM["betas"]
    g = g.float() * factor
    old_m, old_v = (m, v) if m_scale is None else (_held(m, m_scale), _held(v, v_scale).square())
    new_m = old_m * b1 + g * (1 - b1)
    new_v = old_v * b2 + (g * g) * (1 - b2)
    root = new_v.sqrt()
    new_p = (p.float() if master is None else master) * decay - new_m / (root * second + _ADAM["eps"]) * rate
    p.copy_(new_p)
    if master is not None:
        master.copy_(new_p)
    if m_scale is None:
        m.copy_(new_m)
        v.copy_(new_v)
        return
    bits = _dither(steps, g.numel())
    for x, code, scale, least in ((new_m, m, m_scale, False), (root, v, v_scale, True)):
        c, s = _dithered(x, bits, least)
        code.copy_(c)
        scale.copy_(s)


def _plain_adamw(state):
    with torch.no_grad():
        t, b1, b2 = state["lists"], *_ADAM["betas"]
        steps = state["steps"].add_(1)
        factor = torch.clamp(state["limit"] / (state["norm"] + 1e-6), max=1.0) if state["clip"] else 1.0
        rate = (_ADAM["lr"] / (1 - b1 ** steps.double())).float()
        second = (1 / torch.sqrt(1 - b2 ** steps.double())).float()
        nothing = [None] * len(t["param"])
        columns = [t.get(k, nothing) for k in ("param", "grad", "master", "m", "v", "m_scale", "v_scale")]
        [_plain_tensor(factor, rate, second, 1 - _ADAM["lr"] * _ADAM["weight_decay"], steps, *x) for x in zip(*columns)]
        return _updated(state)


_PLAIN = {"addnorm": _plain_addnorm, "normfp8": _plain_normfp8, "rotary": _plain_rotary, "adamw": _plain_adamw}


# ------------------------------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"addnorm": _exact_norm, "normfp8": _exact_norm, "rotary": _exact_rotary, "adamw": _exact_adamw}[case["op"]](s)


def _exact_norm(s):
    """The backward pass as the product with the Jacobian's transpose, written out from the sums over a row."""
    x, w, hidden = s["x"], s["weight"].double(), s["hidden"]
    h = (x.double() + s["stream_"].double()).to(s["stream_"].dtype) if "stream_" in s else None
    z = x.double() if h is None else h.double()
    size = torch.sqrt((z * z).sum(1, keepdim=True) / hidden + 1e-6)
    y = z / size * w
    if s["op"] == "normfp8":
        parts = y.unflatten(1, (-1, s["block"] or hidden))
        scale = torch.clamp(parts.abs().amax(2, keepdim=True) / 448, min=2.0 ** -126)
        units = parts / scale
        step = torch.exp2(torch.floor(torch.log2(units.abs().clamp(min=2.0 ** -6))) - 3)
        q = (torch.round(units / step) * step).flatten(1)
        return (q, scale.squeeze(2)) if h is None else (q, scale.squeeze(2), h.double())
    out = {"y": y, "h": h.double()}
    if s["step"]:
        dy = s["dy"].double()
        dn = dy * w
        d = dn / size - z * (dn * z).sum(1, keepdim=True) / (hidden * size ** 3) + s["dh"].double()
        out["grads"] = (d, d, (dy * z / size).sum(0))
    return out


def _exact_rotary(s):
    """Pairs as complex numbers, turned by a product."""
    d, part = s["head"], s["part"]
    begin, angle = s["start"] % d, s["positions"].double()[:, None, None] * s["inv_freq"]
    at = torch.arange(part, device=angle.device) + begin
    first, second = (at[0::2], at[1::2]) if s["interleaved"] else (at[:part // 2], at[part // 2:])

    def turn(x, angle):
        y = x.detach().double().clone()
        z = torch.complex(y[..., first], y[..., second]) * torch.polar(torch.full_like(angle, s["scale"]), angle)
        y[..., first], y[..., second] = z.real, z.imag
        return y

    out = turn(s["q"], angle), turn(s["k"], angle)
    return out + tuple(turn(g, -angle) for g in s["grads"]) if s["step"] else out


def _exact_adamw(s):
    """Moments in 8 bits: what lies between two codes has no value in 64 bits but for the rounding's own rule, so the scales alone."""
    (b1, b2), t, small = _ADAM["betas"], s["lists"], s["bits"] == 8
    count = s["steps"].item() + 1
    factor = min(1.0, s["limit"] / (s["norm"].item() + 1e-6)) if s["clip"] else 1.0
    names = ["param"] + ["master"] * s["master"] + (["m_scale", "v_scale"] if small else ["m", "v"])
    got = {n: [] for n in names}
    for k, g in enumerate(t["grad"]):
        g = g.double().reshape(-1) * factor
        m, v = t["m"][k].double().reshape(-1), t["v"][k].double().reshape(-1)
        if small:
            m = m * t["m_scale"][k].double().repeat_interleave(128)[:m.numel()]
            v = (v * t["v_scale"][k].double().repeat_interleave(128)[:v.numel()]) ** 2
        m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g ** 2
        p = t["master" if s["master"] else "param"][k].double().reshape(-1)
        p = p - _ADAM["lr"] * (_ADAM["weight_decay"] * p + m / (1 - b1 ** count) / (torch.sqrt(v / (1 - b2 ** count)) + _ADAM["eps"]))
        got["param"].append(p)
        if s["master"]:
            got["master"].append(p)
        for name, x in (("m", m), ("v", torch.sqrt(v) if small else v)):
            if small:
                tail = torch.nn.functional.pad(x.abs(), (0, -x.numel() % 128)).view(-1, 128)
                got[name + "_scale"].append(torch.clamp(tail.amax(1) / 448, min=2.0 ** -126))
            else:
                got[name].append(x)
    out = {n: torch.cat(v) for n, v in got.items()}
    return {n: out.get(n) for n in s["flat"] if n != "grad"}
