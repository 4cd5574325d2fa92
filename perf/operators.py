"""Performance cases of the operators around the lm_head step: normalisation of hidden states, the token table's lookup and
gradient, and the global norm of gradients with clipping.

``run`` computes them in their plain form, by elementary torch operations in 32 bits (64 where sums are long), or, where ``own``
is true, by the framework's entry points.  A case is a dict of plain values; its inputs follow from it and a seed.

* ``norm``   layer norm or RMS norm of ``[rows, hidden]``: forward only, or forward and backward (dx, dweight, dbias)
* ``embed``  rows of a ``[vocab, hidden]`` table: the lookup alone, with the dense gradient, or a gradient that is added to
             fp32 sums that are there already (a tied table's, or those of earlier micro-batches)
* ``grads``  the global norm of a list of gradients: alone, with a limit that is not reached, or clipped into other tensors
"""
import math
import os
import random
import sys

import torch

sys.path.insert(0, os.path.join(os.getcwd(), "mindspeed-rl_amd"))       # imported with the repository's root as working folder

own = False

_DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32, "f16": torch.float16}
_BYTES = {"bf16": 2, "f32": 4, "f16": 2}


# ------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one sequence's new token, whose hidden state goes to the lm_head: latency alone
        dict(name="norm_token", op="norm", kind="rms", dtype="bf16", rows=1, hidden=3584, step=False),
        # a small critic in fp32, a micro-batch of short responses
        dict(name="norm_small_step", op="norm", kind="layer", dtype="f32", rows=2500, hidden=1024, step=True),
        # an odd number of rows of an odd width, fp16
        dict(name="norm_odd_step", op="norm", kind="layer", dtype="f16", rows=9477, hidden=1343, step=True),
        # the final norm of an update's micro-batch of 32 k tokens
        dict(name="norm_step", op="norm", kind="rms", dtype="bf16", rows=32768, hidden=3584, step=True),
        # a scoring pass at the forward budget of 64 k tokens, wider hidden states
        dict(name="norm_score", op="norm", kind="rms", dtype="bf16", rows=65536, hidden=5120, step=False),
        # the tokens that 64 sequences have just drawn
        dict(name="embed_tokens", op="embed", kind="lookup", dtype="bf16", ids="i64", tokens=64, vocab=152064, hidden=3584,
             pad=0.0, parts=1),
        # a prompt batch of 64 k tokens
        dict(name="embed_prompts", op="embed", kind="lookup", dtype="bf16", ids="i64", tokens=65536, vocab=152064, hidden=3584,
             pad=0.0, parts=1),
        # the update's micro-batch: lookup, and the dense gradient of the whole table
        dict(name="embed_step", op="embed", kind="step", dtype="bf16", ids="i64", tokens=32768, vocab=152064, hidden=3584,
             pad=0.0, parts=1),
        # padded rows, one rank's quarter of a table, its gradient added to fp32 sums; most tokens are the padding
        # token or another rank's
        dict(name="embed_added", op="embed", kind="added", dtype="bf16", ids="i32", tokens=49152, vocab=32320, hidden=2048,
             pad=0.4, parts=4),
        # the gradients of a small model in fp32, clipped into other tensors; odd sizes in one flat buffer
        dict(name="grads_small", op="grads", kind="clip", dtype="f32", out="f32", layers=2, hidden=255, vocab=4001, bucket=True),
        # bf16 gradients of four layers and the table, the limit not reached
        dict(name="grads_kept", op="grads", kind="kept", dtype="bf16", out="bf16", layers=4, hidden=3584, vocab=152064,
             bucket=False),
        # the optimizer's fp32 gradients from bf16 ones, clipped on the way
        dict(name="grads_clip", op="grads", kind="clip", dtype="bf16", out="f32", layers=12, hidden=2048, vocab=32000, bucket=True),
    ]


def _log_uniform(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def _draw_width(rng, lo, hi):
    w = int(_log_uniform(rng, lo, hi))
    return max(lo, w // 64 * 64 if rng.random() < 0.6 else w)


def draw(rng):
    op = rng.choice(["norm", "embed", "grads"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "norm":
        hidden = _draw_width(rng, 64, 8192)
        most = 32768 * 3584 * 2 // (hidden * _BYTES[dtype])
        return dict(op=op, kind=rng.choice(["rms", "layer"]), dtype=dtype, rows=max(1, int(_log_uniform(rng, 1, min(most, 65536)))),
                    hidden=hidden, step=rng.random() < 0.7)
    if op == "embed":
        kind = rng.choice(["lookup", "step", "added"])
        hidden = _draw_width(rng, 64, 5120)
        parts = rng.choice([1, 1, 2, 8])
        table = 152064 * 3584 // (1 if kind == "lookup" else 2) // hidden
        tokens = max(1, int(_log_uniform(rng, 1, min(65536 if kind == "lookup" else 32768, 65536 * 3584 // (hidden * _BYTES[dtype])))))
        return dict(op=op, kind=kind, dtype=dtype, ids=rng.choice(["i64", "i32"]), tokens=tokens,
                    vocab=int(_log_uniform(rng, 1000, min(152064, table))), hidden=hidden, pad=rng.choice([0.0, 0.0, 0.3]), parts=parts)
    kind = rng.choice(["norm", "kept", "clip", "clip"])
    hidden = _draw_width(rng, 64, 2048)
    return dict(op=op, kind=kind, dtype=dtype, out=rng.choice([dtype, "f32"]) if kind == "clip" else dtype, layers=rng.randint(1, 6),
                hidden=hidden, vocab=int(_log_uniform(rng, 1000, 32000)), bucket=rng.choice([True, False]))


def _shapes(case):
    """The gradients of a decoder of `layers` layers: products of attention and feed-forward, two norms each, table and last norm."""
    h, f = case["hidden"], case["hidden"] * 7 // 2
    layer = [(h,), (h, h), (h // 4, h), (h // 4, h), (h, h), (h,), (f, h), (f, h), (h, f)]
    return [(case["vocab"], h)] + layer * case["layers"] + [(h,)]


def _entries(case):
    return sum(math.prod(s) for s in _shapes(case))


def work(case):
    size = _BYTES[case["dtype"]]
    if case["op"] == "norm":
        n, h = case["rows"] * case["hidden"], case["hidden"]
        # x in, y out; x and dy in, dx and the vectors' gradients out
        vectors = h * size * (1 if case["kind"] == "rms" else 2)
        if not case["step"]:
            return {"bytes": 2 * n * size + vectors, "flops": 6 * n}
        return {"bytes": 4 * n * size + 2 * vectors, "flops": 18 * n}
    if case["op"] == "embed":
        t, v, h = case["tokens"], case["vocab"], case["hidden"]
        inside = t * _share(case)
        rows = _different(case)
        ids = t * (8 if case["ids"] == "i64" else 4)
        if case["kind"] == "lookup":
            return {"bytes": ids + rows * h * size + t * h * size, "flops": t * h}
        if case["kind"] == "step":
            return {"bytes": ids + rows * h * size + t * h * size + inside * h * size + v * h * size, "flops": 2 * t * h}
        return {"bytes": ids + inside * h * size + 2 * rows * h * 4, "flops": inside * h}
    n = _entries(case)
    return {"bytes": n * size + (n * _BYTES[case["out"]] if case["kind"] == "clip" else 0), "flops": 2 * n}


def _share(case):
    """The share of the tokens that lie in this part of the table: all, or part 1 of several (where the padding token is)."""
    v, p = case["vocab"], case["parts"]
    if p == 1:
        return 1.0
    return case["pad"] + (1 - case["pad"]) * (math.log(2) / math.log(v * p))


def _different(case):
    """About how many rows of the table the tokens name: ids have density 1 / (id ln V), so id v comes n / (v ln V) times."""
    v, p = case["vocab"], case["parts"]
    n = case["tokens"] * (1 - case["pad"])
    top = math.log(v * p)
    lo, hi = (1, v + 1) if p == 1 else (v, 2 * v)
    once = n / top                              # ids below this are named about once or more
    full = min(max(once, lo), hi)
    return max(1.0, min((full - lo) + once * math.log(hi / full), case["tokens"] * _share(case)))


# ------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = _DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=gen, device=dev) * scale

    state = dict(case)
    if case["op"] == "norm":
        r, h = case["rows"], case["hidden"]
        # hidden states have a few columns that are much larger than the others, and rows of different size
        column = torch.exp(normal(h, scale=0.5))
        state["x"] = (normal(r, h) * column * torch.exp(normal(r, 1, scale=0.3)) + 0.1 * column).to(dt)
        state["weight"] = (1 + normal(h, scale=0.2)).to(dt)
        state["bias"] = normal(h, scale=0.1).to(dt) if case["kind"] == "layer" else None
        if case["step"]:
            state["dy"] = (normal(r, h, scale=1e-2) * torch.exp(normal(r, 1))).to(dt)
            state["inputs"] = [t.requires_grad_() for t in (state["x"], state["weight"], state["bias"]) if t is not None]
        return state
    if case["op"] == "embed":
        t, v, h = case["tokens"], case["vocab"], case["hidden"]
        everything = v * case["parts"]
        state["start"] = v if case["parts"] > 1 else 0          # part 1 of several
        state["scale"] = 1.0 if case["kind"] == "lookup" else math.sqrt(h)
        # the rank of a word by frequency: density 1 / rank
        ids = torch.exp(torch.rand(t, generator=gen, device=dev, dtype=torch.float64) * math.log(everything)).to(torch.int64) - 1
        ids = ids.clamp(0, everything - 1)
        padding = state["start"] + v // 2
        ids = torch.where(torch.rand(t, generator=gen, device=dev) < case["pad"], padding, ids)
        state["ids_"] = ids.to(torch.int64 if case["ids"] == "i64" else torch.int32)
        if case["kind"] != "added":
            state["table"] = torch.empty(v, h, dtype=dt, device=dev).normal_(0, 0.02, generator=gen)
        if case["kind"] != "lookup":
            state["dy"] = normal(t, h, scale=1e-2).to(dt)
        if case["kind"] == "step":
            state["table"].requires_grad_()
        if case["kind"] == "added":
            state["sums"] = torch.empty(v, h, device=dev).normal_(0, 1e-2, generator=gen)
        return state
    shapes = _shapes(case)
    flat = torch.empty(_entries(case), dtype=dt, device=dev)
    at, grads = 0, []
    for k, s in enumerate(shapes):
        n = math.prod(s)
        part = flat[at:at + n].view(s)
        part.normal_(0, 1e-3 * (1 + k % 5), generator=gen)
        grads.append(part if case["bucket"] else part.clone())
        at += n
    state["grads"] = grads
    if case["bucket"]:
        state["flat"] = flat
    # an ordinary step's norm lies below the limit, a clipped one's about three times above
    state["limit"] = 1e-3 * math.sqrt(at) * (10.0 if case["kind"] == "kept" else 1.0)
    if case["kind"] == "clip":
        state["result"] = torch.empty(at, dtype=_DTYPES[case["out"]], device=dev)
        state["parts_"] = [p.view(s) for p, s in zip(state["result"].split([math.prod(s) for s in shapes]), shapes)]
    return state


# ------------------------------------------------------------------------------------------ one pass
def run(state):
    return _RUN[state["op"]](state) if own else _PLAIN[state["op"]](state)


def _run_norm(state):
    import mindspeed_rl_amd as mrl
    x, w, b = state["x"], state["weight"], state["bias"]
    y = mrl.rms_norm(x, w, eps=1e-6) if state["kind"] == "rms" else mrl.layer_norm(x, w, b, eps=1e-5)
    if not state["step"]:
        return {"y": y}
    return {"y": y.detach(), "grads": torch.autograd.grad(y, state["inputs"], state["dy"])}


def _run_embed(state):
    import mindspeed_rl_amd as mrl
    ids = state["ids_"]
    if state["kind"] == "added":
        return {"sums": mrl.token_embedding_grad(ids, state["dy"], state["sums"], scale=state["scale"], vocab_start=state["start"],
                                                 accumulate=True)}
    y = mrl.token_embedding(ids, state["table"], scale=state["scale"], vocab_start=state["start"])
    if state["kind"] == "lookup":
        return {"y": y}
    return {"y": y.detach(), "grads": torch.autograd.grad(y, [state["table"]], state["dy"])}


def _run_grads(state):
    import mindspeed_rl_amd as mrl
    if state["kind"] == "norm":
        return {"norm": mrl.global_grad_norm(state["grads"])}
    if state["kind"] == "kept":
        return {"norm": mrl.clip_grad_norm_(state["grads"], state["limit"]), "grads": state.get("flat", state["grads"])}
    return {"norm": mrl.clip_grad_norm_(state["grads"], state["limit"], out=state["parts_"]), "result": state["result"]}


_RUN = {"norm": _run_norm, "embed": _run_embed, "grads": _run_grads}


# ------------------------------------------------------------------------------------------ the plain forms
def _plain_norm(state):
    with torch.no_grad():
        x, w = state["x"].float(), state["weight"].float()
        rms = state["kind"] == "rms"
        centred = x if rms else x - x.mean(-1, keepdim=True)
        r = torch.rsqrt(centred.square().mean(-1, keepdim=True) + (1e-6 if rms else 1e-5))
        n = centred * r
        y = n * w if rms else n * w + state["bias"].float()
        y = y.to(state["x"].dtype)
        if not state["step"]:
            return {"y": y}
        dy = state["dy"].float()
        g = dy * w
        dx = g - n * (g * n).mean(-1, keepdim=True)
        if not rms:
            dx = dx - g.mean(-1, keepdim=True)
        grads = [(dx * r).to(state["x"].dtype), (dy * n).sum(0).to(state["weight"].dtype)]
        if not rms:
            grads.append(dy.sum(0).to(state["bias"].dtype))
        return {"y": y, "grads": tuple(grads)}


def _plain_embed(state):
    with torch.no_grad():
        v, scale = state["vocab"], state["scale"]
        local = state["ids_"].to(torch.int64) - state["start"]
        inside = ((local >= 0) & (local < v)).unsqueeze(1)
        row = local.clamp(0, v - 1)
        if state["kind"] == "added":
            return {"sums": state["sums"].index_add_(0, row, torch.where(inside, state["dy"].float() * scale, 0.0))}
        table = state["table"]
        y = torch.where(inside, table[row].float() * scale, 0.0).to(table.dtype)
        if state["kind"] == "lookup":
            return {"y": y}
        sums = torch.zeros(table.shape, dtype=torch.float32, device=table.device)
        sums.index_add_(0, row, torch.where(inside, state["dy"].float() * scale, 0.0))
        return {"y": y, "grads": (sums.to(table.dtype),)}


def _plain_grads(state):
    grads = state["grads"]
    # squares and their sums of a tensor in 32 bits, by torch's tree; the tensors' sums in 64
    norm = torch.stack([g.float().square().sum() for g in grads]).double().sum().sqrt().float()
    if state["kind"] == "norm":
        return {"norm": norm}
    factor = torch.clamp(state["limit"] / (norm + 1e-6), max=1.0)
    if state["kind"] == "kept":
        [g.copy_(g.float() * factor) for g in grads]
        return {"norm": norm, "grads": state.get("flat", grads)}
    [p.copy_(g.float() * factor) for p, g in zip(state["parts_"], grads)]
    return {"norm": norm, "result": state["result"]}


_PLAIN = {"norm": _plain_norm, "embed": _plain_embed, "grads": _plain_grads}


# ------------------------------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"norm": _exact_norm, "embed": _exact_embed, "grads": _exact_grads}[case["op"]](s)


def _exact_norm(s):
    """The backward pass as the product with the Jacobian's transpose, written out from the sums over a row."""
    w, x = s["weight"].double(), s["x"].double()
    layer, h = s["kind"] == "layer", s["hidden"]
    if layer:
        x = x - x.sum(1, keepdim=True) / h
    size = torch.sqrt((x * x).sum(1, keepdim=True) / h + (1e-5 if layer else 1e-6))
    y = x / size * w
    out = {"y": y + s["bias"].double() if layer else y}
    if s["step"]:
        dy = s["dy"].double()
        dn = dy * w
        dx = dn / size - x * (dn * x).sum(1, keepdim=True) / (h * size ** 3)
        dw = (dy * x / size).sum(0)
        out["grads"] = (dx - dx.sum(1, keepdim=True) / h, dw, dy.sum(0)) if layer else (dx, dw)
    return out


def _exact_embed(s):
    """The table with a row of zeros behind it, which every token outside this part names."""
    v = s["vocab"]
    ids = s["ids_"].long() - s["start"]
    ids[(ids < 0) | (ids >= v)] = v
    out = {}
    if s["kind"] != "added":
        y = torch.zeros(s["tokens"], s["hidden"], dtype=torch.float64, device=ids.device)
        y[ids < v] = s["table"].detach()[ids[ids < v]].double() * s["scale"]
        out["y"] = y
    if s["kind"] == "lookup":
        return out
    sums = torch.zeros(v + 1, s["hidden"], dtype=torch.float64, device=ids.device)
    sums.index_add_(0, ids, s["dy"].double() * s["scale"])
    if s["kind"] == "added":
        return {"sums": s["sums"].double() + sums[:v]}
    out["grads"] = (sums[:v],)
    return out


def _exact_grads(s):
    norm = sum(g.double().pow(2).sum() for g in s["grads"]) ** 0.5
    if s["kind"] == "norm":
        return {"norm": norm}
    factor = min(1.0, s["limit"] / (norm.item() + 1e-6))
    if s["kind"] == "kept":
        whole = s["flat"].double() * factor if "flat" in s else [g.double() * factor for g in s["grads"]]
        return {"norm": norm, "grads": whole}
    return {"norm": norm, "result": torch.cat([g.double().reshape(-1) * factor for g in s["grads"]])}
