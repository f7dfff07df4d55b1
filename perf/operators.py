"""The operators around the output layer of a language model besides its loss, as cases that can be timed: distillation
from a teacher's top logits with both gradients, the top logits of a row, and sampling from given random numbers.

A case is a dict of plain values.  `what` names the operator:

  "distill"  loss and gradients of a student's hidden states x (N, H) and weight against K teacher logits a token
             N, H, V, K   token rows, hidden size, vocabulary, teacher logits a row
             dtype        of x and the weight ("bf16", "f16", "f32")
             tied         True: the weight is an embedding stored (V, H), handed over as ``weight.t()``; else (H, V)
             empty        share of the rows without any teacher logit (prompts, padding)
             short        share of the other rows whose teacher kept fewer than K logits (the rest of the slots is -1)
             T, scale     temperature of both distributions, factor of the student's logits
  "top"      the K largest of V logits of N rows, their columns and the rows' logsumexp
             masked       share of the columns that are minus infinity throughout
  "sample"   one token for each of N rows of V logits
             how          "nucleus": temperature and top-p, numbers for the whole batch; "plain": temperature alone;
                          "short": temperature, top-k, top-p and min-p, numbers for the whole batch; "mixed": a tensor of
                          each with one entry a row, greedy rows among them
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
# float16 training multiplies the loss by such a factor before the backward, so that small gradients survive
LOSS_SCALE = 4096.0


def _distill(N, H, V, K, dtype, tied=False, empty=0.0, short=0.0, T=1.0, scale=1.0):
    return dict(what="distill", N=N, H=H, V=V, K=K, dtype=dtype, tied=tied, empty=empty, short=short, T=T, scale=scale)


def _top(N, V, K, dtype, masked=0.0):
    return dict(what="top", N=N, V=V, K=K, dtype=dtype, masked=masked)


def _sample(N, V, dtype, how, masked=0.0):
    return dict(what="sample", N=N, V=V, dtype=dtype, how=how, masked=masked)


def listed():
    cases = {
        # one short sequence through a toy model: launches and host work are all there is
        "distill_tiny": _distill(256, 256, 4096, 8, "bf16", empty=0.05),
        # sizes that are multiples of nothing, softened distributions, teachers cut off at a share of their mass
        "distill_ragged": _distill(1999, 500, 10007, 20, "f16", empty=0.1, short=0.5, T=2.0),
        # the output layer of a small GPT-2 with its tied embedding (its vocabulary is odd); a quarter of the tokens are prompts
        "distill_gpt2": _distill(8192, 768, 50257, 32, "bf16", tied=True, empty=0.25, short=0.3),
        # float32 throughout: a small model, or a check against a 16-bit run
        "distill_f32": _distill(2048, 2048, 16384, 64, "f32", T=1.5),
        # the sizes of the headline workload of the loss
        "distill_headline": _distill(16384, 2048, 131072, 64, "bf16", empty=0.05, short=0.2),
        # the alternatives shown beside one short answer
        "top_answer": _top(48, 50304, 20, "bf16"),
        # a teacher's pass over a batch, kept for a student; columns beyond the tokenizer's are masked
        "top_teacher": _top(8192, 50257, 32, "bf16", masked=0.01),
        # float32 logits of a large vocabulary
        "top_f32": _top(2048, 131072, 100, "f32"),
        # the next token of one conversation
        "sample_one": _sample(1, 131072, "bf16", "nucleus"),
        # a serving batch in which every request has its own settings
        "sample_batch": _sample(256, 131072, "bf16", "mixed", masked=0.02),
        # float32 logits with every filter on
        "sample_f32": _sample(61, 50257, "f32", "short"),
        # one step of many rollouts at once, from the whole distribution
        "sample_rollouts": _sample(2048, 32000, "f16", "plain"),
    }
    return [dict(case, name=name) for name, case in cases.items()]


def draw(rng):
    """One more case: sizes spread over their logarithms, about a third of them odd, options as users set them."""
    most = {what: max(_cost(c) for c in listed() if c["what"] == what) for what in ("distill", "top", "sample")}

    def size(low, high, multiple):
        v = math.exp(rng.uniform(math.log(low), math.log(high)))
        if rng.random() < 0.35:
            return max(low, min(high, int(v) | 1))
        return max(multiple, min(high, int(round(v / multiple)) * multiple))

    while True:
        what = rng.choice(["distill", "distill", "top", "sample"])
        dtype = rng.choice(["bf16", "bf16", "bf16", "f16", "f16", "f32"])
        if what == "distill":
            case = _distill(size(64, 16384, 64), size(64, 4096, 64), size(1024, 131072, 128), size(1, 128, 4), dtype,
                            tied=dtype != "f32" and rng.random() < 0.4, empty=rng.choice([0.0, 0.05, 0.25, 0.5]),
                            short=rng.choice([0.0, 0.0, 0.3, 0.6]), T=rng.choice([1.0, 1.0, 1.5, 2.0]),
                            scale=rng.choice([1.0, 1.0, 0.5]))
        elif what == "top":
            V = size(1000, 262144, 128)
            case = _top(size(1, 8192, 8), V, size(1, 256, 4), dtype, masked=rng.choice([0.0, 0.0, 0.01, 0.1]))
        else:
            case = _sample(size(1, 4096, 8), size(1000, 262144, 128), dtype, rng.choice(["nucleus", "plain", "short", "mixed"]),
                           masked=rng.choice([0.0, 0.0, 0.02]))
        # (float32 products cost several times a 16-bit one)
        if _cost(case) <= most[what]:
            return case


def _rows(case):
    """Rows of a "distill" case that have a teacher."""
    return max(1, case["N"] - int(case["empty"] * case["N"]))


def _cost(case):
    if case["what"] == "distill":
        return 6.0 * case["N"] * case["H"] * case["V"] * (6.0 if case["dtype"] == "f32" else 1.0)
    return float(case["N"]) * case["V"]


def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    N, V = case["N"], case["V"]
    if case["what"] == "distill":
        H, K = case["H"], case["K"]
        # (an index of 8 bytes and a logit of 4 for every slot; gradients as large as what they belong to)
        return {"bytes": float(2 * (N * H + H * V) * es + N * K * 12 + 4), "flops": 6.0 * _rows(case) * H * V}
    if case["what"] == "top":
        return {"bytes": float(N * V * es + N * case["K"] * (8 + es) + 4 * N), "flops": 0.0}
    return {"bytes": float(N * V * es + 12 * N), "flops": 0.0}


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _model_logits(N, V, dtype, masked, gen):
    """Logits as a language model gives them: most of the vocabulary in a wide bell, some dozens of tokens well above it, by
    an amount that varies from row to row (from a certain next token to an open one)."""
    dev = gen.device
    z = torch.randn((N, V), generator=gen, device=dev).mul_(2.0)
    few = min(V, 64)
    step = 1 + (torch.rand((N, 1), generator=gen, device=dev) * (V // few - 1)).long()
    at = (torch.randint(0, V, (N, 1), generator=gen, device=dev) + step * torch.arange(few, device=dev)) % V  # (different ones)
    lift = torch.empty((N, few), device=dev).exponential_(1.0, generator=gen) * (torch.rand((N, 1), generator=gen, device=dev) * 4.0)
    z.scatter_add_(1, at, lift + 4.0)
    if masked > 0:
        z[:, torch.rand(V, generator=gen, device=dev) < masked] = -math.inf
    return z.to(dtype)


def _prepare_distill(case, gen):
    dev = gen.device
    N, H, V, K, dtype = case["N"], case["H"], case["V"], case["K"], DTYPES[case["dtype"]]
    std = 1.0 / math.sqrt(H)
    weight = torch.nn.init.trunc_normal_(torch.empty((V, H) if case["tied"] else (H, V), device=dev), mean=0.0, std=std,
                                         a=-3 * std, b=3 * std, generator=gen).to(dtype)
    # K different tokens a row, mostly frequent ones: the k-th in the k-th part of the ranks, which are denser at the front
    part = (torch.arange(K, device=dev, dtype=torch.float64) + torch.rand((N, K), generator=gen, device=dev, dtype=torch.float64)) / K
    rank = torch.arange(K, device=dev) + ((V - K) * part ** 4).long()
    index = torch.randperm(V, generator=gen, device=dev)[rank.clamp_(max=V - 1)]
    index = index.gather(1, torch.rand((N, K), generator=gen, device=dev).argsort(1))
    # the teacher's logits fall from its first choice on, faster or slower from row to row
    steps = torch.empty((N, K), device=dev).exponential_(1.0, generator=gen) * (0.05 + torch.rand((N, 1), generator=gen, device=dev))
    logits = 15.0 - torch.cumsum(steps, 1)
    x = torch.randn((N, H), generator=gen, device=dev)
    # the student has learned something: the teacher's first choice stands 0 ... 8 above the others' middle
    first = index[:, 0]
    columns = weight[first] if case["tied"] else weight[:, first].t()
    x += columns.float() * (torch.rand((N, 1), generator=gen, device=dev) * (8.0 / case["scale"]))
    if case["short"] > 0:
        kept = 1 + (torch.rand((N, 1), generator=gen, device=dev) * (K - 1)).long()
        cut = (torch.rand((N, 1), generator=gen, device=dev) < case["short"]) & (torch.arange(K, device=dev) >= kept)
        index[cut] = -1
    empty = torch.randperm(N, generator=gen, device=dev)[:N - _rows(case)]
    index[empty] = -1
    weight.requires_grad_(True)
    return {"x": x.to(dtype).requires_grad_(True), "weight": weight, "index": index, "logits": logits}


def prepare(case, seed):
    gen = _generator(seed)
    if case["what"] == "distill":
        return dict(_prepare_distill(case, gen), case=case)
    N, V = case["N"], case["V"]
    state = {"case": case, "logits": _model_logits(N, V, DTYPES[case["dtype"]], case["masked"], gen)}
    if case["what"] == "sample":
        state["u"] = torch.rand(N, generator=gen, device=gen.device)
        state["settings"] = _settings(case, gen)
    return state


def _settings(case, gen):
    N, how = case["N"], case["how"]
    if how == "plain":
        return {"temperature": 1.0}
    if how == "nucleus":
        return {"temperature": 0.8, "top_p": 0.9}
    if how == "short":
        return {"temperature": 0.7, "top_k": 50, "top_p": 0.95, "min_p": 0.02}

    def pick(values, dtype):
        at = torch.randint(0, len(values), (N,), generator=gen, device=gen.device)
        return torch.tensor(values, dtype=dtype, device=gen.device)[at]

    return {"temperature": pick([0.0, 0.6, 0.8, 1.0, 1.3], torch.float32), "top_k": pick([0, 0, 0, 20, 50, 400], torch.int64),
            "top_p": pick([1.0, 0.95, 0.9, 0.5], torch.float32), "min_p": pick([0.0, 0.0, 0.02, 0.1], torch.float32)}


# The plain forms: elementary operations in 32 bits, or in 64 where a sum decides on which side of a border a token falls.


def _plain_distill(x, At, index, logits, temperature, scale):
    x, w = x.float(), At.float()
    c = scale / temperature
    z = torch.mm(x, w).mul_(c)
    top = z.amax(1, keepdim=True)
    lse = top + (z - top).exp_().sum(1, keepdim=True).log_()
    present = (index >= 0) & (logits > -math.inf)
    rows = present.any(1, keepdim=True)
    t = torch.where(present, logits.float() / temperature, -math.inf)
    e = torch.where(present, torch.exp(t - torch.where(rows, t.amax(1, keepdim=True), 0.0)), 0.0)
    q = e / torch.where(rows, e.sum(1, keepdim=True), 1.0)
    at = index.clamp(min=0)
    terms = torch.where(q > 0, q * (torch.log(torch.where(q > 0, q, 1.0)) - z.gather(1, at) + lse), 0.0)
    count = rows.sum()
    loss = (terms.double().sum() / count).float()
    dz = z.sub_(lse).exp_().scatter_add_(1, at, -q).mul_(rows * (c / count))
    return loss, torch.mm(dz, w.t()), torch.mm(x.t(), dz)


def _plain_top(logits, k):
    z = logits.float()
    order = torch.sort(z, dim=1, descending=True, stable=True)
    top = order.values[:, :1]
    lse = top + (z - top).exp_().sum(1, keepdim=True).log_()
    return order.values[:, :k].to(logits.dtype), order.indices[:, :k].contiguous(), lse[:, 0]


def _plain_sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    z = logits.double()
    N, V = z.shape

    def column(v):
        return torch.as_tensor(v, device=z.device).to(torch.float32).double().expand(N).reshape(N, 1)

    temperature, top_k, top_p, min_p = column(temperature), column(top_k), column(top_p), column(min_p)
    order = torch.sort(z, dim=1, descending=True, stable=True)
    greedy = temperature <= 0
    w = torch.exp((order.values - order.values[:, :1]) / torch.where(greedy, 1.0, temperature))
    place = torch.arange(V, device=z.device)
    w = torch.where((top_k <= 0) | (place < top_k), w, 0.0)
    before = torch.cumsum(w, 1) - w
    stays = (place == 0) | (((top_p >= 1) | (before < top_p * w.sum(1, keepdim=True))) & (w >= min_p) & ~greedy)
    w = torch.where(stays, w, 0.0)
    upto = torch.cumsum(w, 1)
    first = (upto > u.double().reshape(N, 1) * upto[:, -1:]).to(torch.uint8).argmax(1, keepdim=True)
    return order.indices.gather(1, first)[:, 0]


def run(state):
    case = state["case"]
    if case["what"] == "distill":
        x, weight = state["x"], state["weight"]
        At = weight.t() if case["tied"] else weight
        factor = LOSS_SCALE if case["dtype"] == "f16" else 1.0
        if own:
            from linear_cross_entropy_loss_amd import linear_distillation

            loss = linear_distillation(x, At, state["index"], state["logits"], temperature=case["T"], logit_scale=case["scale"])
            dx, dw = torch.autograd.grad(loss * factor if factor != 1.0 else loss, (x, weight))
            return {"loss": loss.detach(), "dx": dx, "dw": dw}
        with torch.no_grad():
            loss, dx, dw = _plain_distill(x, At, state["index"], state["logits"], case["T"], case["scale"])
            dw = dw.t() if case["tied"] else dw
            return {"loss": loss, "dx": dx.mul_(factor).to(x.dtype), "dw": dw.mul(factor).to(weight.dtype).contiguous()}
    if case["what"] == "top":
        if own:
            from linear_cross_entropy_loss_amd import top_logits

            values, columns, lse = top_logits(state["logits"], case["K"])
        else:
            values, columns, lse = _plain_top(state["logits"], case["K"])
        return {"values": values, "columns": columns, "lse": lse}
    if own:
        from linear_cross_entropy_loss_amd import sample_logits

        return {"tokens": sample_logits(state["logits"], state["u"], **state["settings"])}
    return {"tokens": _plain_sample(state["logits"], state["u"], **state["settings"])}


def exact(case, seed):
    """The same from the definitions in 64 bits, a block of rows at a time."""
    if case["what"] == "sample":
        return None  # (whole numbers)
    state = prepare(case, seed)
    if case["what"] == "top":
        lse = torch.cat([torch.logsumexp(rows.double(), 1) for rows in state["logits"].split(256)])
        return {"values": torch.topk(state["logits"].float(), case["K"], dim=1).values.double(), "columns": None, "lse": lse}
    factor = LOSS_SCALE if case["dtype"] == "f16" else 1.0
    x, weight = state["x"].detach(), state["weight"].detach()
    w = (weight.t() if case["tied"] else weight).double()
    index, given = state["index"], state["logits"].double()
    kept = ((index >= 0).sum(1) > 0).nonzero()[:, 0]
    dx = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    dw = torch.zeros(w.shape, dtype=torch.float64, device=x.device)
    loss = torch.zeros((), dtype=torch.float64, device=x.device)
    for rows in kept.split(1024):
        here = x[rows].double()
        at = index[rows]
        # the teacher's distribution over the whole vocabulary; what is absent goes to a column behind the last
        teacher = torch.full((len(rows), w.shape[1] + 1), -math.inf, dtype=torch.float64, device=x.device)
        teacher.scatter_(1, torch.where(at < 0, w.shape[1], at), given[rows] / case["T"])
        teacher = torch.softmax(teacher[:, :-1], 1)
        student = torch.log_softmax(here @ w * (case["scale"] / case["T"]), 1)
        loss += torch.special.xlogy(teacher, teacher).sum() - (teacher * student).sum()
        dz = (student.exp() - teacher) * (case["scale"] / case["T"] / len(kept))
        dx[rows] = dz @ w.t()
        dw += here.t() @ dz
    return {"loss": loss / len(kept), "dx": dx * factor, "dw": (dw.t() if case["tied"] else dw).contiguous() * factor}
