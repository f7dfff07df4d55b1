"""What a model that is trained on its own answers needs of its output layer besides the loss, as cases that can be timed: the logits and
logsumexps of given tokens with gradients for any upstream gradient, the logits of an 8-bit copy of the weight, and the clipping of
many tensors' gradients by their common norm.

A case is a dict of plain values.  `what` names the operator:

  "tokens"  logit and logsumexp of one token a row, hidden states x (N, H) against a weight (H, V), and both gradients
            N, H, V      token rows, hidden size, columns of the weight
            dtype        of x and the weight ("bf16", "f16", "f32")
            tied         True: the weight is an embedding stored (V, H), handed over as ``weight.t()``; else (H, V)
            drop         share of the rows without a token (prompts, padding)
            pieces       the vocabulary is cut into so many weights of V columns, of which this is the middle one
            grads        False: scores alone (a reference model, an evaluation)
            scale        factor of the logits
  "int8"    logits of N rows from int8 weights with a scale for each column, the rows quantised within the call
            N, H, V, dtype, tied, scale   as above; the logits have the type of x
            fresh        True: the weight has changed and is quantised within the call as well
  "clip"    gradients of a model of `layers` layers of hidden size H under a head of V columns, scaled to a norm of at most 1
            dtype, out   types of the gradients and of what comes out (the float32 ones that an optimizer reads, or the same)
            norm         norm of the gradients, about: above 1 they are scaled
            divisor      the factor that the loss was multiplied by
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
# float16 training multiplies the loss by such a factor before the backward, so that small gradients survive
LOSS_SCALE = 4096.0
IGNORE = -100


def _tokens(N, H, V, dtype, tied=False, drop=0.0, pieces=1, grads=True, scale=1.0):
    return dict(what="tokens", N=N, H=H, V=V, dtype=dtype, tied=tied, drop=drop, pieces=pieces, grads=grads, scale=scale)


def _int8(N, H, V, dtype, tied=False, fresh=False, scale=1.0):
    return dict(what="int8", N=N, H=H, V=V, dtype=dtype, tied=tied, fresh=fresh, scale=scale)


def _clip(H, V, layers, dtype, out, norm=4.0, divisor=1.0):
    return dict(what="clip", H=H, V=V, layers=layers, dtype=dtype, out=out, norm=norm, divisor=divisor)


def listed():
    cases = {
        # one short answer through a toy model: launches and host work are all there is
        "tokens_tiny": _tokens(64, 256, 4096, "bf16", drop=0.25),
        # sizes that are multiples of nothing, the middle third of a vocabulary
        "tokens_ragged": _tokens(1999, 500, 10007, "f16", drop=0.1, pieces=3),
        # float32 throughout: a small model, or a check against a 16-bit run
        "tokens_f32": _tokens(2048, 1024, 16384, "f32", drop=0.05),
        # scores under the frozen model that a policy is compared with: the output layer of a small GPT-2, tied, no gradients
        "tokens_score": _tokens(8192, 768, 50257, "bf16", tied=True, drop=0.25, grads=False),
        # a batch of answers at the sizes of the headline workload of the loss, a quarter of it prompts
        "tokens_policy": _tokens(16384, 2048, 131072, "bf16", drop=0.25),
        # the next token of one conversation
        "int8_one": _int8(1, 2048, 131072, "bf16"),
        # a serving batch, odd sizes, float32 logits
        "int8_odd": _int8(37, 777, 50257, "f32", scale=0.5),
        # one step of some hundred rollouts at once
        "int8_rollouts": _int8(256, 4096, 128256, "bf16", tied=True),
        # all rows of some prompts, as for log-probabilities of them
        "int8_prompts": _int8(2048, 4096, 32000, "f16"),
        # the first step after an update of the weight, which is quantised anew
        "int8_fresh": _int8(64, 2048, 131072, "bf16", fresh=True),
        # a toy model's gradients: launches and host work
        "clip_small": _clip(64, 1003, 2, "f32", "f32"),
        # the gradients of a small model under a large head, for an optimizer in float32
        "clip_large": _clip(2048, 131072, 4, "bf16", "f32"),
    }
    return [dict(case, name=name) for name, case in cases.items()]


def draw(rng):
    """One more case: sizes spread over their logarithms, about a third of them odd, options as users set them."""
    most = {what: max(_cost(c) for c in listed() if c["what"] == what) for what in ("tokens", "int8", "clip")}

    def size(low, high, multiple):
        v = math.exp(rng.uniform(math.log(low), math.log(high)))
        if rng.random() < 0.35:
            return max(low, min(high, int(v) | 1))
        return max(min(multiple, high), low, min(high, int(round(v / multiple)) * multiple))

    while True:
        what = rng.choice(["tokens", "tokens", "int8", "int8", "clip"])
        dtype = rng.choice(["bf16", "bf16", "bf16", "f16", "f16", "f32"])
        if what == "tokens":
            case = _tokens(size(1, 16384, 8), size(64, 4096, 64), size(1024, 131072, 128), dtype,
                           tied=dtype != "f32" and rng.random() < 0.4, drop=rng.choice([0.0, 0.05, 0.25, 0.5]),
                           pieces=rng.choice([1, 1, 1, 2, 3]), grads=rng.random() < 0.75, scale=rng.choice([1.0, 1.0, 0.5]))
        elif what == "int8":
            case = _int8(size(1, 4096, 1), size(64, 8192, 64), size(1000, 262144, 128), dtype, tied=rng.random() < 0.4,
                         fresh=rng.random() < 0.3, scale=rng.choice([1.0, 1.0, 0.5]))
        else:
            case = _clip(size(16, 4096, 16), size(256, 131072, 128), rng.randint(0, 24), dtype, rng.choice([dtype, "f32"]),
                         norm=rng.choice([0.5, 2.0, 4.0, 100.0]), divisor=LOSS_SCALE if dtype == "f16" else 1.0)
        if _cost(case) <= most[what]:
            return case


def _shapes(case):
    """Shapes of a "clip" case's gradients: the head, and of each layer two norms, a bias and four matrices."""
    H, V = case["H"], case["V"]
    return [(H, V)] + case["layers"] * [(H,), (3 * H, H), (3 * H,), (H, H), (H,), (4 * H, H), (H, 4 * H)]


def _elements(case):
    return sum(math.prod(shape) for shape in _shapes(case))


def _rows(case):
    """Rows of a "tokens" case that have a token."""
    return max(1, case["N"] - int(case["drop"] * case["N"]))


def _cost(case):
    if case["what"] == "clip":
        return float(_elements(case))
    # (float32 products cost several times a 16-bit one; a pass over the weight counts however few the rows are)
    cost = float(case["N"] + 64) * case["H"] * case["V"]
    return cost * (6.0 if case["what"] == "tokens" and case["dtype"] == "f32" else 1.0)


def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    if case["what"] == "clip":
        return {"bytes": float(_elements(case) * (es + (4 if case["out"] == "f32" else 2)) + 4), "flops": 3.0 * _elements(case)}
    N, H, V = case["N"], case["H"], case["V"]
    if case["what"] == "tokens":
        # (a token of 8 bytes, a logit and an lse of 4 a row; two upstream gradients of 4, gradients as large as what they belong to)
        size = (N * H + H * V) * es
        return {"bytes": float((2 if case["grads"] else 1) * size + N * (24 if case["grads"] else 16)),
                "flops": (6.0 if case["grads"] else 2.0) * _rows(case) * H * V}
    weight = H * V * es if case["fresh"] else H * V + 4 * V
    return {"bytes": float(weight + N * (H + V) * es), "flops": 2.0 * N * H * V}


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _weight(case, gen):
    H, V = case["H"], case["V"]
    std = 1.0 / math.sqrt(H)
    shape = (V, H) if case["tied"] else (H, V)
    return torch.nn.init.trunc_normal_(torch.empty(shape, device=gen.device), mean=0.0, std=std, a=-3 * std, b=3 * std,
                                       generator=gen).to(DTYPES[case["dtype"]])


def _prepare_tokens(case, gen):
    dev = gen.device
    N, V, pieces = case["N"], case["V"], case["pieces"]
    weight = _weight(case, gen)
    x = torch.randn((N, case["H"]), generator=gen, device=dev)
    # mostly frequent tokens, of the whole vocabulary
    rank = (V * pieces * torch.rand(N, generator=gen, device=dev, dtype=torch.float64) ** 4).long()
    tokens = torch.randperm(V * pieces, generator=gen, device=dev)[rank.clamp_(max=V * pieces - 1)]
    first = V * (pieces // 2)
    # the answers are the model's own: their tokens stand 0 ... 8 above the others' middle
    at = (tokens - first).clamp(0, V - 1)
    columns = weight[at] if case["tied"] else weight[:, at].t()
    x += columns.float() * (torch.rand((N, 1), generator=gen, device=dev) * (8.0 / case["scale"]))
    tokens[torch.randperm(N, generator=gen, device=dev)[:N - _rows(case)]] = IGNORE
    state = {"case": case, "x": x.to(DTYPES[case["dtype"]]), "weight": weight, "tokens": tokens, "first": first}
    if case["grads"]:
        # of a policy's objective: an advantage for each token over their number; of a piece's lse the share that the piece
        # has of the whole sum
        factor = LOSS_SCALE if case["dtype"] == "f16" else 1.0
        state["g_logits"] = torch.randn(N, generator=gen, device=dev) * (factor / _rows(case))
        share = torch.rand(N, generator=gen, device=dev) if pieces > 1 else 1.0
        state["g_lse"] = -state["g_logits"] * share
        state["x"].requires_grad_(True)
        weight.requires_grad_(True)
    return state


def _prepare_int8(case, gen):
    dev = gen.device
    weight = _weight(case, gen)
    x = torch.randn((case["N"], case["H"]), generator=gen, device=dev)
    # some hidden units are much larger than the others throughout
    x *= 1.0 + 9.0 * (torch.rand(case["H"], generator=gen, device=dev) < 0.01)
    state = {"case": case, "x": x.to(DTYPES[case["dtype"]])}
    At = weight.t() if case["tied"] else weight
    if case["fresh"]:
        state["At"] = At
    elif own:
        from linear_cross_entropy_loss_amd import quantize_weight

        state["weight"] = quantize_weight(At)
    else:
        state["weight"] = _plain_quantize(At.t())
    return state


def prepare(case, seed):
    gen = _generator(seed)
    if case["what"] == "tokens":
        return _prepare_tokens(case, gen)
    if case["what"] == "int8":
        return _prepare_int8(case, gen)
    shapes = _shapes(case)
    # the layers' gradients differ in size
    each = [math.exp(2.0 * float(v)) for v in torch.randn(len(shapes), generator=torch.Generator().manual_seed(seed))]
    whole = math.sqrt(sum(s * s * math.prod(shape) for s, shape in zip(each, shapes)))
    factor = case["norm"] * case["divisor"] / whole
    grads = [torch.randn(shape, generator=gen, device=gen.device).mul_(s * factor).to(DTYPES[case["dtype"]])
             for s, shape in zip(each, shapes)]
    return {"case": case, "grads": grads, "out": [torch.empty_like(g, dtype=DTYPES[case["out"]]) for g in grads]}


# The plain forms: elementary operations in 32 bits, or in 64 where a value lies next to a border or a sum is long.


def _plain_tokens(x, At, tokens, first, scale, g_logits=None, g_lse=None):
    x, w = x.float(), At.float()
    z = torch.mm(x, w).mul_(scale)
    top = z.amax(1, keepdim=True)
    lse = top + (z - top).exp_().sum(1, keepdim=True).log_()
    rows = (tokens != IGNORE).unsqueeze(1)
    at = (tokens - first).unsqueeze(1)
    here = rows & (at >= 0) & (at < w.shape[1])
    at = at.clamp(0, w.shape[1] - 1)
    logits = torch.where(here, z.gather(1, at), 0.0)[:, 0]
    if g_logits is None:
        return logits, torch.where(rows, lse, 0.0)[:, 0]
    dz = z.sub_(lse).exp_().mul_(torch.where(rows, g_lse.unsqueeze(1), 0.0))
    dz.scatter_add_(1, at, torch.where(here, g_logits.unsqueeze(1), 0.0)).mul_(scale)
    return logits, torch.where(rows, lse, 0.0)[:, 0], torch.mm(dz, w.t()), torch.mm(x.t(), dz)


def _plain_quantize(t):
    """Whole numbers of -127 ... 127 for each row of t, and what one of them stands for."""
    top = t.abs().amax(1, keepdim=True).double()
    q = torch.where(top > 0, torch.round(t.double() * 127.0 / torch.where(top > 0, top, 1.0)), 0.0)
    return q.to(torch.int8), (top[:, 0] / 127.0).float()


def _plain_int8(x, weight, scale):
    q, scales = _plain_quantize(x)
    z = torch.mm(q.float(), weight[0].float().t())
    return z.mul_(scales.unsqueeze(1) * scale).mul_(weight[1]).to(x.dtype)


def _plain_clip(grads, max_norm, divisor, out):
    norm = sum(g.double().square().sum() for g in grads).sqrt() / divisor
    factor = (torch.clamp(max_norm / norm, max=1.0) / divisor).float()
    for g, o in zip(grads, out):
        o.copy_(g.float() * factor)
    return norm.float()


def run(state):
    case = state["case"]
    if case["what"] == "tokens":
        x, weight, V = state["x"], state["weight"], case["V"]
        At = weight.t() if case["tied"] else weight
        grads = (state["g_logits"], state["g_lse"]) if case["grads"] else ()
        if own:
            from linear_cross_entropy_loss_amd import linear_token_logits

            logits, lse = linear_token_logits(x, At, state["tokens"], ignore_index=IGNORE, logit_scale=case["scale"],
                                              vocab_start=state["first"], vocab_size=V * case["pieces"])
            if not grads:
                return {"logits": logits, "lse": lse}
            dx, dw = torch.autograd.grad((logits, lse), (x, weight), grads)
            return {"logits": logits.detach(), "lse": lse.detach(), "dx": dx, "dw": dw}
        with torch.no_grad():
            done = _plain_tokens(x, At, state["tokens"], state["first"], case["scale"], *grads)
            if not grads:
                return {"logits": done[0], "lse": done[1]}
            dw = done[3].t() if case["tied"] else done[3]
            return {"logits": done[0], "lse": done[1], "dx": done[2].to(x.dtype), "dw": dw.to(weight.dtype).contiguous()}
    if case["what"] == "int8":
        if own:
            from linear_cross_entropy_loss_amd import quantize_weight, quantized_logits

            weight = quantize_weight(state["At"]) if case["fresh"] else state["weight"]
            return {"logits": quantized_logits(state["x"], weight, logit_scale=case["scale"])}
        weight = _plain_quantize(state["At"].t()) if case["fresh"] else state["weight"]
        return {"logits": _plain_int8(state["x"], weight, case["scale"])}
    if own:
        from linear_cross_entropy_loss_amd import clip_gradients

        norm = clip_gradients(state["grads"], 1.0, divisor=case["divisor"], out=state["out"])
    else:
        norm = _plain_clip(state["grads"], 1.0, case["divisor"], state["out"])
    return {"norm": norm, "out": state["out"]}


def exact(case, seed):
    """The same from the definitions in 64 bits, a block of rows at a time."""
    if case["what"] == "clip":
        grads = [g.double() for g in prepare(case, seed)["grads"]]
        norm = math.sqrt(math.fsum(float((g * g).sum()) for g in grads)) / case["divisor"]
        factor = min(1.0, 1.0 / norm) / case["divisor"]
        return {"norm": torch.tensor(norm, dtype=torch.float64, device=grads[0].device), "out": [g.mul_(factor) for g in grads]}
    gen = _generator(seed)
    if case["what"] == "int8":
        # (the weight as it was before it was quantised)
        state = _prepare_int8(dict(case, fresh=True), gen)
        w = state["At"].t()

        def whole(t):
            step = t.double().abs().max(dim=1, keepdim=True).values / 127
            return (t.double() / step).nan_to_num_(0.0).round_(), step

        qx, sx = whole(state["x"])
        parts = []
        for rows in w.split(16384):
            qw, sw = whole(rows)
            parts.append((qx @ qw.t()) * sx * sw.t() * case["scale"])
        return {"logits": torch.cat(parts, 1)}
    state = _prepare_tokens(case, gen)
    x, weight, tokens, first = state["x"].detach(), state["weight"].detach(), state["tokens"], state["first"]
    w = (weight.t() if case["tied"] else weight).double() * case["scale"]
    N, V = case["N"], case["V"]
    logits = torch.zeros(N, dtype=torch.float64, device=x.device)
    lse = torch.zeros_like(logits)
    dx = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    dw = torch.zeros(w.shape, dtype=torch.float64, device=x.device)
    for rows in (tokens != IGNORE).nonzero()[:, 0].split(1024):
        xs = x[rows].double()
        z = xs @ w
        lse[rows] = torch.logsumexp(z, 1)
        at = tokens[rows] - first
        mine = ((at >= 0) & (at < V)).nonzero()[:, 0]
        logits[rows[mine]] = z[mine, at[mine]]
        if case["grads"]:
            dz = torch.softmax(z, 1) * state["g_lse"][rows].double().unsqueeze(1)
            dz[mine, at[mine]] += state["g_logits"][rows[mine]].double()
            dx[rows] = dz @ w.t()
            dw += xs.t() @ dz
    if not case["grads"]:
        return {"logits": logits, "lse": lse}
    dw *= case["scale"]
    return {"logits": logits, "lse": lse, "dx": dx, "dw": dw.t().contiguous() if case["tied"] else dw}
