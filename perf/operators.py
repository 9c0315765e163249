"""Measured cases of the operators that answer with, and learn from, the logits of whole candidate rows:

  score    logits of query rows against a table of candidates held in 8 bits (e4m3) with one power-of-two scale for each
           block of 128 columns of a row; the queries arrive in 16 or 32 bits and are quantised in the same way on the way in
  top      the k largest logits of each row, their candidates, and the row's softmax statistics
  distill  the Kullback-Leibler divergence of a student's softmax over all candidates from a teacher's top logits, with its
           gradient with respect to the student's logits

Shapes are rows x candidates, the candidates being the nodes of a graph: 10 312 (a blog network), 99 991 (a ragged one),
1 000 000 (the benchmark graph); columns are the embedding dimension."""
import math

import torch

own = False

DEVICE = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BLOCK = 128  # columns that share a scale
LARGEST = 448.0  # the largest e4m3 number
DIMS = (32, 64, 96, 128, 256, 512)


def _score(name, rows, cols, dim, query, out):
    return {"name": name, "op": "score", "rows": rows, "cols": cols, "dim": dim, "in": query, "out": out}


def _top(name, rows, cols, k, logits, temperature):
    return {"name": name, "op": "top", "rows": rows, "cols": cols, "k": k, "in": logits, "temperature": temperature}


def _distill(name, pass_, rows, cols, k, logits, temperature, whole, weighted):
    return {"name": name, "op": "distill", "pass": pass_, "rows": rows, "cols": cols, "k": k, "in": logits,
            "temperature": temperature, "whole": whole, "weighted": weighted}


def listed():
    return [
        # one node asks for its links, small graph: latency
        _score("score 1x10312 d128", 1, 10312, 128, "f32", "f32"),
        # one node asks for its links, benchmark graph: the table is read once
        _score("score 1x1000000 d128", 1, 1000000, 128, "f32", "f32"),
        # an odd batch on an odd graph, a dimension below the block, 16-bit queries and logits
        _score("score 777x99991 d96", 777, 99991, 96, "bf16", "f16"),
        # a teacher's batch over the whole benchmark graph, logits in 32 bits: the answer is what moves
        _score("score 1024x1000000 d128", 1024, 1000000, 128, "f32", "f32"),
        # four blocks of columns, 16-bit logits: the most arithmetic per answer
        _score("score 4096x65536 d512", 4096, 65536, 512, "f32", "bf16"),
        # the ten best links of a handful of nodes
        _top("top 10 of 7x10312", 7, 10312, 10, "f32", 1.0),
        # an odd batch, a long list, a temperature
        _top("top 100 of 333x99991", 333, 99991, 100, "f32", 2.0),
        # a teacher's batch over the benchmark graph; 16-bit logits tie
        _top("top 64 of 1024x1000000", 1024, 1000000, 64, "bf16", 1.0),
        # a small training step: loss and gradient
        _distill("distill step 50x10312", "step", 50, 10312, 10, "f32", 1.0, False, False),
        # validation: the loss alone
        _distill("distill loss 500x99991", "loss", 500, 99991, 100, "f16", 2.0, False, False),
        # a training step on the benchmark graph in 16 bits, rows weighted
        _distill("distill step 512x1000000", "step", 512, 1000000, 64, "bf16", 2.0, True, True),
        # the backward pass alone, its loss weighted by what follows it
        _distill("distill grad 256x1000000", "grad", 256, 1000000, 32, "f32", 1.0, True, True),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("score", "top", "distill"))
    cols = _spread(rng, 1000, 1000000)
    if op == "score":
        dim = rng.choice(DIMS) if rng.random() < 0.6 else rng.randint(20, 512)
        rows = _spread(rng, 1, min(4096, 2 ** 30 // cols))
        return {"op": op, "rows": rows, "cols": cols, "dim": dim, "in": rng.choice(list(TYPES)), "out": rng.choice(list(TYPES))}
    k = min(_spread(rng, 1, 128), cols // 4)
    case = {"op": op, "cols": cols, "k": k, "in": rng.choice(list(TYPES)), "temperature": rng.choice((0.5, 1.0, 2.0, 4.0))}
    if op == "top":
        return dict(case, rows=_spread(rng, 1, min(1024, 2 ** 30 // cols)))
    return {**case, "rows": _spread(rng, 1, min(1024, 2 ** 28 // cols)), "pass": rng.choice(("step", "loss", "grad")),
            "whole": rng.random() < 0.5, "weighted": rng.random() < 0.5}


# ---- inputs -----------------------------------------------------------------------------------------------------------------

def _embeddings(g, rows, dim):
    """Trained rows: normal, their lengths falling from the hubs to the leaves."""
    size = 0.1 + 1.5 * torch.rand(rows, 1, generator=g, device=DEVICE) ** 3
    return torch.randn(rows, dim, generator=g, device=DEVICE) * size


def _quantise(x):
    """float32 [rows, dim] -> (e4m3 values [rows, dim rounded up to 32], the rest 0, exponents [rows, blocks] + 127): the least power of two that
    brings a block's largest magnitude to 448 or below."""
    rows, dim = x.shape
    blocks = -(-dim // BLOCK)
    x = torch.nn.functional.pad(x, (0, blocks * BLOCK - dim)).view(rows, blocks, BLOCK)
    fraction, power = torch.frexp(x.abs().amax(-1))  # fraction in [0.5, 1)
    power = torch.where(fraction > LARGEST / 512, power - 8, power - 9).clamp(-127, 127)
    power = torch.where(fraction == 0, 0, power)
    values = torch.ldexp(x, -power[..., None]).to(torch.float8_e4m3fn).view(rows, blocks * BLOCK)
    return values[:, :-(-dim // 32) * 32].contiguous(), (power + 127).to(torch.uint8)


def _unquantise(values, exponents, dim):
    blocks = exponents.shape[1]
    x = torch.nn.functional.pad(values.float(), (0, blocks * BLOCK - values.shape[1])).view(len(values), blocks, BLOCK)
    return torch.ldexp(x, exponents[..., None].int() - 127).view(len(values), -1)[:, :dim]


def prepare(case, seed):
    g = torch.Generator(DEVICE)
    g.manual_seed(seed)
    rows, cols = case["rows"], case["cols"]
    state = {"case": case}
    if case["op"] == "score":  # the queries, and the table a serving program holds
        state["query"] = _embeddings(g, rows, case["dim"]).to(TYPES[case["in"]])
        state["values"], state["exponents"] = _quantise(_embeddings(g, cols, case["dim"]))
        return state
    logits = torch.randn(rows, cols, generator=g, device=DEVICE)
    logits.mul_(2.0)
    # known links of a row are no candidates: one in five hundred
    logits.masked_fill_(torch.randint(0, 512, (rows, cols), generator=g, device=DEVICE, dtype=torch.int16) == 0, -math.inf)
    if case["op"] == "top":
        state["logits"] = logits.to(TYPES[case["in"]])
        return state
    k = case["k"]
    # a teacher's list: k candidates from all over the row, its logits falling; some lists are shorter, a few are empty
    place = torch.rand(rows, k, generator=g, device=DEVICE, dtype=torch.float64)
    index = ((torch.arange(k, device=DEVICE) + place) * (cols / k)).long().clamp_(max=cols - 1)
    index = index.gather(1, torch.rand(rows, k, generator=g, device=DEVICE).argsort(1))
    state["teacher"] = (6 + 2 * torch.randn(rows, k, generator=g, device=DEVICE)).sort(1, descending=True)[0].contiguous()
    logits.scatter_(1, index, state["teacher"] - 1 + 1.5 * torch.randn(rows, k, generator=g, device=DEVICE))
    length = torch.where(torch.rand(rows, 1, generator=g, device=DEVICE) < 0.1, torch.rand(rows, 1, generator=g, device=DEVICE) * k, float(k))
    state["index"] = torch.where(torch.arange(k, device=DEVICE) < length.long(), index, -1).int().contiguous()
    state["logits"] = logits.to(TYPES[case["in"]])
    state["teacher_stats"] = state["weight"] = state["stats"] = None
    if case["whole"]:  # the list holds 0.5 to 0.95 of the teacher's whole row
        share = 0.5 + 0.45 * torch.rand(rows, generator=g, device=DEVICE)
        total = ((state["teacher"] - state["teacher"][:, :1]) / case["temperature"]).exp().sum(1)
        state["teacher_stats"] = torch.stack([state["teacher"][:, 0], (total / share).log()], 1).contiguous()
    if case["weighted"]:
        state["weight"] = torch.rand(rows, generator=g, device=DEVICE) / rows
    if case["pass"] == "grad":  # what the forward pass left
        z = state["logits"].float()
        top = z.amax(1)
        state["stats"] = torch.stack([top, ((z - top[:, None]) / case["temperature"]).exp().sum(1, dtype=torch.float64).log().float()], 1).contiguous()
    return state


# ---- plain forms ------------------------------------------------------------------------------------------------------------

def _plain_score(state):
    case = state["case"]
    query = _unquantise(*_quantise(state["query"].float()), case["dim"])
    table = _unquantise(state["values"], state["exponents"], case["dim"])
    return (query @ table.t()).to(TYPES[case["out"]])


def _softmax_parts(z, temperature):
    """max [rows], exp((z - max) / temperature) and its sum"""
    top = z.amax(1)
    e = ((z - top[:, None]) / temperature).exp()
    return top, e, e.sum(1)


def _plain_top(state):
    case, logits = state["case"], state["logits"].float()
    cols = logits.shape[1]
    top, _, total = _softmax_parts(logits, case["temperature"])
    # one whole number orders (logit, lower candidate first)
    bits = (logits + 0.0).view(torch.int32)
    bits = torch.where(bits < 0, bits ^ 0x7fffffff, bits).long()
    key = (bits << 32) | (cols - 1 - torch.arange(cols, device=logits.device))
    index = cols - 1 - (key.topk(case["k"], dim=1)[0] & 0xffffffff)
    return {"values": logits.gather(1, index), "index": index.int(), "stats": torch.stack([top, total.log()], 1)}


def _teacher(state):
    """(probabilities, their logarithms) of the list: of the whole row's softmax where the teacher's statistics are given, else of the list's own"""
    temperature, t = state["case"]["temperature"], state["teacher"]
    listed_ = state["index"] >= 0
    if state["teacher_stats"] is not None:
        log_q = (t - state["teacher_stats"][:, :1]) / temperature - state["teacher_stats"][:, 1:]
    else:
        shifted = (t - torch.where(listed_, t, -math.inf).amax(1, keepdim=True).clamp(min=-1e30)) / temperature
        total = torch.where(listed_, shifted.exp(), 0.0).sum(1, keepdim=True)
        log_q = shifted - torch.where(total > 0, total, 1.0).log()
    return torch.where(listed_, log_q.exp(), 0.0), log_q, state["index"].clamp(min=0).long()


def _plain_distill(state):
    case, logits = state["case"], state["logits"].float()
    temperature = case["temperature"]
    q, log_q, index = _teacher(state)
    if case["pass"] == "grad":
        top, log_total = state["stats"][:, 0], state["stats"][:, 1]
        p = ((logits - top[:, None]) / temperature - log_total[:, None]).exp()
    else:
        top, e, total = _softmax_parts(logits, temperature)
        log_total = total.log()
        log_p = (logits.gather(1, index) - top[:, None]) / temperature - log_total[:, None]
        out = {"loss": torch.where(q > 0, q * (log_q - log_p), 0.0).sum(1), "stats": torch.stack([top, log_total], 1)}
        if case["pass"] == "loss":
            return out
        p = e / total[:, None]
    grad = p * q.sum(1, keepdim=True)
    grad.scatter_add_(1, index, -q)
    grad *= (1.0 if state["weight"] is None else state["weight"][:, None]) / temperature
    grad = grad.to(TYPES[case["in"]])
    return {"grad": grad} if case["pass"] == "grad" else dict(out, grad=grad)


# ---- the framework's calls --------------------------------------------------------------------------------------------------

def _kernels():
    from graphvite_amd.kernels import HipKernels
    return HipKernels()


def _own_score(state):
    from graphvite_amd.kernels import BlockTable
    case = state["case"]
    table = BlockTable(state["values"], state["exponents"], case["dim"])
    logits = torch.empty(case["rows"], case["cols"], dtype=TYPES[case["out"]], device=DEVICE)
    _kernels().block_logits(state["query"], table, logits)
    return logits


def _own_top(state):
    case = state["case"]
    values = torch.empty(case["rows"], case["k"], device=DEVICE)
    index = torch.empty(case["rows"], case["k"], dtype=torch.int32, device=DEVICE)
    stats = torch.empty(case["rows"], 2, device=DEVICE)
    _kernels().top_logits(state["logits"], values, index, stats, temperature=case["temperature"])
    return {"values": values, "index": index, "stats": stats}


def _own_distill(state):
    case, rows = state["case"], state["case"]["rows"]
    given = dict(teacher_stats=state["teacher_stats"], temperature=case["temperature"])
    grad = None if case["pass"] == "loss" else torch.empty_like(state["logits"])
    if case["pass"] == "grad":
        _kernels().distill_grad(state["logits"], state["index"], state["teacher"], state["stats"], grad, weight=state["weight"], **given)
        return {"grad": grad}
    loss, stats = torch.empty(rows, device=DEVICE), torch.empty(rows, 2, device=DEVICE)
    _kernels().distill(state["logits"], state["index"], state["teacher"], loss, stats, grad=grad, weight=state["weight"], **given)
    out = {"loss": loss, "stats": stats}
    return out if grad is None else dict(out, grad=grad)


def run(state):
    plain = {"score": _plain_score, "top": _plain_top, "distill": _plain_distill}
    kernels = {"score": _own_score, "top": _own_top, "distill": _own_distill}
    return (kernels if own else plain)[state["case"]["op"]](state)


# ---- what a pass cannot do without --------------------------------------------------------------------------------------------

def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2}
    rows, cols = case["rows"], case["cols"]
    if case["op"] == "score":
        blocks = -(-case["dim"] // BLOCK)
        moved = cols * (case["dim"] + blocks) + rows * case["dim"] * size[case["in"]] + rows * cols * size[case["out"]]
        return {"bytes": moved, "flops": 2 * rows * cols * case["dim"]}
    plane, lists = rows * cols * size[case["in"]], rows * case["k"] * 8
    if case["op"] == "top":
        return {"bytes": plane + lists + rows * 8, "flops": 4 * rows * cols}
    passes = 1 if case["pass"] == "loss" else 2
    return {"bytes": passes * plane + lists + rows * 12, "flops": 4 * passes * rows * cols}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------------------

def _exact_rounded(x):
    """float64 -> the values its e4m3 blocks stand for: steps of 2^-3 of a number's own power of two, of 2^-9 below 2^-6, ties to even."""
    rows, dim = x.shape
    parts = []
    for start in range(0, dim, BLOCK):
        part = x[:, start:start + BLOCK]
        largest = part.abs().amax(1, keepdim=True)
        scale = torch.exp2(torch.ceil(torch.log2(torch.where(largest > 0, largest, 1.0) / LARGEST)))
        scale = torch.where(largest > scale * LARGEST, scale * 2, torch.where(largest <= scale / 2 * LARGEST, scale / 2, scale))
        part = part / scale
        step = torch.exp2(torch.floor(torch.log2(part.abs().clamp(min=2.0 ** -6))) - 3)
        parts.append(torch.round(part / step) * step * scale)
    return torch.cat(parts, 1)


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "score":
        scale = torch.exp2(state["exponents"].double() - 127).repeat_interleave(BLOCK, 1)[:, :case["dim"]]
        table = state["values"][:, :case["dim"]].double() * scale
        return _exact_rounded(state["query"].double()) @ table.t()
    z = state["logits"].double()
    temperature = case["temperature"]
    if case["op"] == "top":
        values, index, stats = [], [], []
        for at in range(0, len(z), 64):
            v, i = z[at:at + 64].sort(dim=1, descending=True, stable=True)
            values.append(v[:, :case["k"]].clone())
            index.append(i[:, :case["k"]].int())
            stats.append(torch.stack([v[:, 0], torch.logsumexp((v - v[:, :1]) / temperature, 1)], 1))
        return {"values": torch.cat(values), "index": torch.cat(index), "stats": torch.cat(stats)}
    listed_ = state["index"] >= 0
    t = state["teacher"].double().masked_fill(~listed_, -math.inf)
    if state["teacher_stats"] is None:
        q = torch.softmax(t / temperature, 1).nan_to_num(0.0)
    else:
        q = torch.exp((t - state["teacher_stats"][:, :1].double()) / temperature - state["teacher_stats"][:, 1:].double())
    index = torch.where(listed_, state["index"], 0).long()
    if case["pass"] == "grad":  # with the statistics that the forward pass left
        log_p = (z - state["stats"][:, :1].double()) / temperature - state["stats"][:, 1:].double()
    else:
        log_p = torch.log_softmax(z / temperature, 1)
    out = {}
    if case["pass"] != "grad":
        at = log_p.gather(1, index)
        out["loss"] = (torch.special.xlogy(q, q) - torch.where(q > 0, q * at, 0.0)).sum(1)
        top = z.amax(1)
        out["stats"] = torch.stack([top, torch.logsumexp((z - top[:, None]) / temperature, 1)], 1)
    if case["pass"] != "loss":
        out["grad"] = (log_p.exp() * q.sum(1, keepdim=True)).scatter_add(1, index, -q) / temperature
        if state["weight"] is not None:
            out["grad"] = out["grad"] * state["weight"].double()[:, None]
    return out
