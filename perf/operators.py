"""The operators of a dropless-MoE layer around its block-sparse products, as a user's program calls them.

gate     router logits -> the top-k experts of every token and their weights, with the gradient of the logits
sort     expert choices -> placement in padded expert bins; token rows copied there, with the gradient of the rows
unsort   the experts' rows back in token order, weighted and summed, with the gradients of the rows and the weights
int4     the experts' two-layer MLP on few tokens, from 4-bit weights with a scale for each group of inputs
"""
import math

import torch

own = False

BLOCK = 128
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # gate.  One decoding batch; the router of the 64-expert layer on its whole batch, weights as they come out
        # of the softmax; many experts, an odd number of tokens of which the last ones are padding, sigmoid scores.
        dict(name="gate_decode", op="gate", tokens=16, experts=64, top_k=2, dtype="f32", score="softmax",
             normalize=True, masked=0, grad=False),
        dict(name="gate_train_e64", op="gate", tokens=131072, experts=64, top_k=2, dtype="f32", score="softmax",
             normalize=False, masked=0, grad=True),
        dict(name="gate_train_sigmoid", op="gate", tokens=10007, experts=160, top_k=6, dtype="bf16", score="sigmoid",
             normalize=True, masked=301, grad=True),
        # sort.  A short prompt; the 8-expert layer with one choice per token and as many rows as the batch needs (the
        # host reads their number back); the 16-expert layer with uneven experts.  fixed: the number of rows is settled
        # in advance (no read-back: the step can be captured).
        dict(name="sort_prompt", op="sort", tokens=64, hidden=1024, experts=8, top_k=2, dtype="f16", skew=0.0,
             masked=0, fixed=True, grad=False),
        dict(name="sort_train_e8", op="sort", tokens=16384, hidden=1024, experts=8, top_k=1, dtype="f16", skew=0.0,
             masked=0, fixed=False, grad=True),
        dict(name="sort_train_e16", op="sort", tokens=32768, hidden=2048, experts=16, top_k=2, dtype="bf16", skew=1.2,
             masked=0, fixed=True, grad=True),
        # unsort.  A short prompt; the 64-expert layer's share of one of eight GPUs; odd sizes in 32 bits, more
        # choices, padding tokens.
        dict(name="unsort_prompt", op="unsort", tokens=100, hidden=1024, experts=8, top_k=2, dtype="f16", skew=0.0,
             masked=0, grad=False),
        dict(name="unsort_train_e64", op="unsort", tokens=16384, hidden=4096, experts=64, top_k=2, dtype="bf16",
             skew=0.0, masked=0, grad=True),
        dict(name="unsort_train_odd", op="unsort", tokens=5003, hidden=1001, experts=24, top_k=4, dtype="f32",
             skew=0.7, masked=77, grad=True),
        # int4.  One token; a decoding batch on the largest layer's experts of one of eight GPUs; a larger batch with
        # zero points and a shorter group.
        dict(name="int4_one_token", op="int4", tokens=1, hidden=1024, ffn=4096, experts=8, top_k=2, dtype="f16",
             group=128, zeros=False, masked=0),
        dict(name="int4_decode_xl", op="int4", tokens=16, hidden=4096, ffn=14336, experts=8, top_k=2, dtype="bf16",
             group=128, zeros=False, masked=0),
        dict(name="int4_decode_64", op="int4", tokens=64, hidden=2048, ffn=8192, experts=16, top_k=2, dtype="bf16",
             group=64, zeros=True, masked=3),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["gate", "sort", "unsort", "int4"])
    if op == "gate":
        tokens, experts = _log(rng, 1, 131072), _log(rng, 2, 256)
        if tokens * experts > 131072 * 64:
            tokens = 131072 * 64 // experts
        return dict(op=op, tokens=tokens, experts=experts, top_k=rng.randint(1, min(8, experts)),
                    dtype=rng.choice(["f16", "bf16", "f32"]), score=rng.choice(["softmax", "sigmoid"]),
                    normalize=rng.random() < 0.5, masked=rng.choice([0, tokens // 7]), grad=rng.random() < 0.7)
    if op in ("sort", "unsort"):
        experts = _log(rng, 1, 128)
        top_k = rng.randint(1, min(6, experts))
        dtype = rng.choice(["f16", "bf16", "f32"])
        tokens, hidden = _log(rng, 1, 32768), _log(rng, 64, 4096)
        if rng.random() < 0.7:                       # mostly whole 16-byte vectors, as in practice; odd widths too
            hidden = max(8, hidden // 8 * 8)
        most = 16384 * 4096 // (2 if dtype == "f32" else 1)
        if tokens * top_k * hidden > most:
            tokens = max(1, most // (top_k * hidden))
        case = dict(op=op, tokens=tokens, hidden=hidden, experts=experts, top_k=top_k, dtype=dtype,
                    skew=rng.choice([0.0, 0.7, 1.2]), masked=rng.choice([0, tokens // 9]), grad=rng.random() < 0.7)
        if op == "sort":
            case["fixed"] = top_k > 1 or rng.random() < 0.5
        return case
    group = rng.choice([32, 64, 128])
    hidden, ffn = group * _log(rng, 2, 4096 // group), group * _log(rng, 2, 14336 // group)
    experts = rng.randint(2, 16)
    if experts * hidden * ffn > 8 * 4096 * 14336:
        experts = max(2, 8 * 4096 * 14336 // (hidden * ffn))
    top_k = rng.randint(1, min(4, experts))
    tokens = min(_log(rng, 1, 64), max(1, 64 * 2 * 2048 * 8192 // (top_k * hidden * ffn)))
    return dict(op=op, tokens=tokens, hidden=hidden, ffn=ffn, experts=experts, top_k=top_k,
                dtype=rng.choice(["f16", "bf16"]), group=group, zeros=rng.random() < 0.5,
                masked=rng.choice([0, tokens // 5]))


# ------------------------------------------------------------------------------ inputs
def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _choices(g, case):
    """int32 [T, k]: k different experts for every token, expert e with the share (e + 1)^-skew; -1 for the last
    `masked` tokens, which are padding."""
    tokens, experts = case["tokens"], case["experts"]
    share = -case.get("skew", 0.0) * torch.log(torch.arange(1, experts + 1, device="cuda", dtype=torch.float32))
    if not case.get("fixed", True):                    # one choice each; how many choose an expert, and so the number
        live = tokens - case["masked"]                 # of rows, is the case's and not the seed's
        ends = torch.round(torch.cumsum(torch.softmax(share.double(), 0), 0) * live)
        who = torch.searchsorted(ends, torch.arange(live, device="cuda", dtype=torch.float64), right=True)
        who = who.clamp(max=experts - 1)[torch.randperm(live, generator=g, device="cuda")]
        return torch.nn.functional.pad(who, (0, case["masked"]), value=-1).to(torch.int32)[:, None]
    noise = -torch.log(-torch.log(torch.rand((tokens, experts), generator=g, device="cuda").clamp(1e-20, 1 - 1e-6)))
    ids = torch.topk(share + noise, case["top_k"], dim=1).indices.to(torch.int32)
    if case["masked"]:
        ids[tokens - case["masked"]:] = -1
    return ids


def _bits(g, experts, n, k, group, dtype, zeros):
    """4-bit weights [E, N, K] as they come out of a checkpoint: two codes a byte (the lower one first), a scale and,
    optionally, a zero point for each row and group."""
    codes = torch.randn(experts * n * k, generator=g, device="cuda").mul_(2.6).add_(7.5).round_().clamp_(0, 15)
    codes = codes.to(torch.uint8).view(experts, n, k // 2, 2)
    packed = codes[..., 0] | (codes[..., 1] << 4)
    scales = (0.0077 * (0.5 + torch.rand((experts, n, k // group), generator=g, device="cuda"))).to(dtype)
    zero = torch.randint(5, 11, (experts, n, k // group), generator=g, device="cuda").to(torch.uint8) if zeros else None
    return packed, scales, zero


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, tokens = DTYPES[case["dtype"]], case["tokens"]
    if case["op"] == "gate":
        s = dict(logits=_randn(g, tokens, case["experts"]).to(dtype), mask=None)
        if case["masked"]:
            s["mask"] = torch.arange(tokens, device="cuda") < tokens - case["masked"]
        if case["grad"]:
            s["dweights"] = _randn(g, tokens, case["top_k"])
        return s
    s = dict(ids=_choices(g, case))
    if case["op"] == "int4":
        s["x"] = _randn(g, tokens, case["hidden"]).to(dtype)
        s["weights"] = torch.softmax(_randn(g, tokens, case["top_k"]), dim=1)
        s["w1"] = _bits(g, case["experts"], case["ffn"], case["hidden"], case["group"], dtype, case["zeros"])
        s["w2"] = _bits(g, case["experts"], case["hidden"], case["ffn"], case["group"], dtype, case["zeros"])
        return s
    index, position, _ = _placement(s["ids"], case["experts"], case.get("fixed", True))
    rows = index.numel()
    if case["op"] == "sort":
        s["x"] = _randn(g, tokens, case["hidden"]).to(dtype)
        if case["grad"]:
            s["drows"] = _randn(g, rows, case["hidden"]).to(dtype)
        return s
    s["index"], s["position"] = index, position
    s["rows"] = _randn(g, rows, case["hidden"]).to(dtype)
    s["weights"] = torch.softmax(_randn(g, tokens, case["top_k"]), dim=1)
    if case["grad"]:
        s["dout"] = _randn(g, tokens, case["hidden"]).to(dtype)
    return s


def prepare(case, seed):
    s = dict(_inputs(case, seed), case=case)
    if own:
        from stk_b200 import dmoe
        if case["op"] == "int4":                       # the weights in the layout that a serving program keeps
            s["w1"] = dmoe.pack_int4(*s["w1"])
            s["w2"] = dmoe.pack_int4(*s["w2"])
        if case["op"] == "unsort":                     # the placement that the rows were sorted with
            s["plan"] = dmoe.plan_tokens(s["ids"], case["experts"], rows=s["rows"].shape[0])
    if case.get("grad"):                               # what the gradients are asked of
        for name in {"gate": ("logits",), "sort": ("x",), "unsort": ("rows", "weights")}[case["op"]]:
            s[name].requires_grad_()
    return s


# ------------------------------------------------------------------------------ plain forms
def _bound(slots, experts):
    """Most rows that `slots` choices can take in padded bins: every bin in use may end in an incomplete block."""
    return (slots + min(experts, slots) * (BLOCK - 1)) // BLOCK * BLOCK


def _placement(ids, experts, fixed):
    """(index [rows]: the slot in each row of the bins or -1; position [T * k]: the row of each slot or -1; bin_rows:
    blocks of each expert).  Slots stay in order within an expert.  fixed: as many rows as any batch of this size can
    need, the last expert's bin taking those that are left."""
    flat = ids.reshape(-1).long()
    slots = flat.numel()
    key = torch.where(flat >= 0, flat, torch.full_like(flat, experts))
    order = torch.sort(key, stable=True).indices
    counts = (key[:, None] == torch.arange(experts + 1, device=ids.device)).sum(0)
    blocks = (counts[:experts] + BLOCK - 1) // BLOCK
    rows = _bound(slots, experts) if fixed else int(blocks.sum()) * BLOCK
    bin_start = torch.cumsum(blocks, 0) * BLOCK - blocks * BLOCK
    slot_start = torch.cumsum(counts, 0) - counts
    sorted_key = key[order]
    rank = torch.arange(slots, device=ids.device) - slot_start[sorted_key]
    place = torch.where(sorted_key < experts, bin_start[sorted_key.clamp(max=experts - 1)] + rank, torch.full_like(rank, -1))
    position = torch.empty_like(flat)
    position[order] = place
    index = torch.full((rows + 1,), -1, dtype=torch.int64, device=ids.device)
    index[torch.where(position >= 0, position, torch.full_like(position, rows))] = torch.arange(slots, device=ids.device)
    if fixed:
        blocks = blocks.clone()
        blocks[-1] += rows // BLOCK - blocks.sum()
    return index[:rows].to(torch.int32), position.to(torch.int32), blocks.to(torch.int32)


def _plain_gate(s, case):
    k = case["top_k"]
    logits = s["logits"].detach().float()
    ids = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :k]
    if case["score"] == "softmax":
        scores = torch.exp(logits - logits.amax(1, keepdim=True))
        scores = scores / scores.sum(1, keepdim=True)
    else:
        scores = 1 / (1 + torch.exp(-logits))
    chosen = torch.gather(scores, 1, ids)
    total = chosen.sum(1, keepdim=True)
    weights = chosen / total if case["normalize"] else chosen
    alive = torch.ones_like(weights[:, :1], dtype=torch.bool) if s["mask"] is None else s["mask"][:, None]
    out = dict(weights=torch.where(alive, weights, torch.zeros_like(weights)),
               ids=torch.where(alive, ids, torch.full_like(ids, -1)).to(torch.int32))
    if case["grad"]:
        dw = s["dweights"]
        dchosen = (dw - (dw * weights).sum(1, keepdim=True)) / total if case["normalize"] else dw
        dscores = torch.zeros_like(scores).scatter(1, ids, dchosen)
        if case["score"] == "softmax":
            dlogits = scores * (dscores - (dscores * scores).sum(1, keepdim=True))
        else:
            dlogits = dscores * scores * (1 - scores)
        out["dlogits"] = torch.where(alive, dlogits, torch.zeros_like(dlogits)).to(s["logits"].dtype)
    return out


def _plain_sort(s, case):
    index, position, bin_rows = _placement(s["ids"], case["experts"], case["fixed"])
    k, x = case["top_k"], s["x"].detach()
    rows = torch.where((index >= 0)[:, None], x[index.clamp(min=0).long() // k], torch.zeros((), dtype=x.dtype, device=x.device))
    out = dict(rows=rows, index=index, position=position, bin_rows=bin_rows)
    if case["grad"]:
        if rows.shape[0] == 0:
            out["dx"] = torch.zeros_like(x)
        else:
            back = s["drows"].float()[position.clamp(min=0).long()] * (position >= 0)[:, None]
            out["dx"] = back.view(case["tokens"], k, -1).sum(1).to(x.dtype)
    return out


def _plain_unsort(s, case):
    index, position, k = s["index"].long(), s["position"].long(), case["top_k"]
    rows, weights = s["rows"].detach(), s["weights"].detach()
    y = (rows.float()[position.clamp(min=0)] * (position >= 0)[:, None]).view(case["tokens"], k, -1)
    out = dict(out=(weights[:, :, None] * y).sum(1).to(rows.dtype))
    if case["grad"]:
        dout = s["dout"].float()
        slot = index.clamp(min=0)
        out["drows"] = (weights.reshape(-1)[slot][:, None] * dout[slot // k] * (index >= 0)[:, None]).to(rows.dtype)
        out["dweights"] = (dout[:, None] * y).sum(2)
    return out


def _values(bits, dtype, pick=None):
    """The numbers that 4-bit weights stand for, [E, N, K], or those of the experts `pick`."""
    packed, scales, zero = bits if pick is None else [None if t is None else t[pick] for t in bits]
    e, n, half = packed.shape
    codes = torch.stack((packed & 15, packed >> 4), dim=3).view(e, n, scales.shape[2], -1).to(dtype)
    codes = codes - (8 if zero is None else zero.to(dtype)[..., None])
    return (codes * scales.to(dtype)[..., None]).view(e, n, 2 * half)


def _plain_int4(s, case):
    ids, tokens, k = s["ids"].long(), case["tokens"], case["top_k"]
    alive, x = ids >= 0, s["x"].float()
    if tokens * k <= case["experts"]:                  # the chosen experts alone, a matrix for each choice
        pick = ids.clamp(min=0).reshape(-1)
        h = torch.matmul(_values(s["w1"], torch.float32, pick), x.repeat_interleave(k, 0)[:, :, None])
        h = 0.5 * h * (1 + torch.erf(h * math.sqrt(0.5)))
        y = torch.matmul(_values(s["w2"], torch.float32, pick), h).view(tokens, k, -1)
    else:                                              # every expert on every token, and then the chosen ones
        h = torch.matmul(x, _values(s["w1"], torch.float32).transpose(1, 2))
        h = 0.5 * h * (1 + torch.erf(h * math.sqrt(0.5)))
        y = torch.matmul(h, _values(s["w2"], torch.float32).transpose(1, 2))
        y = y[ids.clamp(min=0), torch.arange(tokens, device=ids.device)[:, None]]
    return dict(out=((s["weights"] * alive)[:, :, None] * y).sum(1).to(s["x"].dtype))


# ------------------------------------------------------------------------------ the framework's operators
def _own_run(s, case):
    from stk_b200 import dmoe
    if case["op"] == "gate":
        weights, ids = dmoe.top_k_gate(s["logits"], case["top_k"], score=case["score"], normalize=case["normalize"],
                                       token_mask=s["mask"])
        out = dict(weights=weights.detach(), ids=ids)
        if case["grad"]:
            out["dlogits"], = torch.autograd.grad(weights, s["logits"], s["dweights"])
        return out
    if case["op"] == "sort":
        rows = dmoe.plan_rows(s["ids"].numel(), case["experts"]) if case["fixed"] else None
        plan = dmoe.plan_tokens(s["ids"], case["experts"], rows=rows)
        sorted_rows = dmoe.sort_tokens(s["x"], plan)
        out = dict(rows=sorted_rows.detach(), index=plan.index, position=plan.position, bin_rows=plan.bin_rows)
        if case["grad"]:
            out["dx"], = torch.autograd.grad(sorted_rows, s["x"], s["drows"])
        return out
    if case["op"] == "unsort":
        y = dmoe.unsort_tokens(s["rows"], s["weights"], s["plan"])
        out = dict(out=y.detach())
        if case["grad"]:
            out["drows"], out["dweights"] = torch.autograd.grad(y, (s["rows"], s["weights"]), s["dout"])
        return out
    return dict(out=dmoe.expert_mlp_int4(s["x"], s["ids"], s["weights"], s["w1"], s["w2"]))


def run(s):
    case = s["case"]
    if own:
        return _own_run(s, case)
    return {"gate": _plain_gate, "sort": _plain_sort, "unsort": _plain_unsort, "int4": _plain_int4}[case["op"]](s, case)


# ------------------------------------------------------------------------------ work and exact values
def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    tokens, k, experts = case["tokens"], case["top_k"], case["experts"]
    slots = tokens * k
    if case["op"] == "gate":
        passes = 2 if case["grad"] else 1              # the logits, and their gradient
        return dict(bytes=passes * tokens * experts * size + slots * (8 + (4 if case["grad"] else 0)),
                    flops=(10 if case["grad"] else 5) * tokens * experts)
    if case["op"] in ("sort", "unsort"):
        live = (tokens - case["masked"]) * k
        rows = _bound(slots, experts) if case.get("fixed", True) else live + min(experts, live) * BLOCK // 2
        width = case["hidden"] * size
        token_rows = (tokens - case["masked"]) * width
        if case["op"] == "sort":
            moved = token_rows + rows * width + 4 * (2 * slots + rows)
            back = live * width + tokens * width + 4 * slots
            return dict(bytes=moved + (back if case["grad"] else 0), flops=(live * case["hidden"] if case["grad"] else 0))
        moved = live * width + tokens * width + 8 * slots
        back = token_rows + rows * width + 4 * (slots + rows)
        return dict(bytes=moved + (back if case["grad"] else 0), flops=(5 if case["grad"] else 2) * live * case["hidden"])
    live = tokens - case["masked"]
    used = experts * (1 - (1 - k / experts) ** live)   # experts that some token chose, on average
    matrix = case["hidden"] * case["ffn"]
    bits = matrix / 2 + matrix / case["group"] * (size + (1 if case["zeros"] else 0))
    return dict(bytes=2 * used * bits + 2 * tokens * case["hidden"] * size + 8 * slots, flops=4 * live * k * matrix)


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "gate":
        return _exact_gate(s, case)
    if case["op"] == "int4":
        return _exact_int4(s, case)
    tokens, k = case["tokens"], case["top_k"]
    if case["op"] == "sort":
        index, position, _ = _placement(s["ids"], case["experts"], case["fixed"])
        place = position.view(tokens, k)
        rows = torch.zeros((index.numel(), case["hidden"]), dtype=torch.float64, device="cuda")
        out = dict(rows=rows, index=None, position=None, bin_rows=None)
        if case["grad"]:
            out["dx"] = torch.zeros(s["x"].shape, dtype=torch.float64, device="cuda")
        for j in range(k):
            on = place[:, j] >= 0
            rows[place[on, j].long()] = s["x"][on].double()
            if case["grad"]:
                out["dx"][on] += s["drows"][place[on, j].long()].double()
        return out
    place, weights = s["position"].view(tokens, k).long(), s["weights"].double()
    hidden = case["hidden"]
    y = torch.zeros((tokens, hidden), dtype=torch.float64, device="cuda")
    out = dict(out=y)
    if case["grad"]:
        dout = s["dout"].double()
        drows = torch.zeros(s["rows"].shape, dtype=torch.float64, device="cuda")
        dweights = torch.zeros((tokens, k), dtype=torch.float64, device="cuda")
        out.update(drows=drows, dweights=dweights)
    for j in range(k):
        on = place[:, j] >= 0
        at = place[on, j]
        part = s["rows"][at].double()
        y[on] += weights[on, j, None] * part
        if case["grad"]:
            drows[at] = weights[on, j, None] * dout[on]
            dweights[on, j] = torch.linalg.vecdot(dout[on], part)
    return out


def _exact_gate(s, case):
    """Gradients by the log-derivative: d log(weight j) / d logit i."""
    logits, k = s["logits"].double(), case["top_k"]
    top, ids = torch.sort(logits, dim=1, descending=True, stable=True)
    top, ids = top[:, :k], ids[:, :k]
    soft = case["score"] == "softmax"
    log_score = (lambda v: v - torch.logsumexp(logits, 1, keepdim=True)) if soft else torch.nn.functional.logsigmoid
    chosen = log_score(top)
    log_weight = chosen - torch.logsumexp(chosen, 1, keepdim=True) if case["normalize"] else chosen
    weights = torch.exp(log_weight)
    out = dict(weights=weights, ids=None)
    if case["grad"]:
        flow = s["dweights"].double() * weights        # dL / d log(weight)
        if case["normalize"]:
            flow = flow - weights * flow.sum(1, keepdim=True)
        dlogits = torch.zeros_like(logits)
        if soft:
            dlogits.scatter_(1, ids, flow)
            dlogits -= torch.softmax(logits, 1) * flow.sum(1, keepdim=True)
        else:
            dlogits.scatter_(1, ids, flow * torch.sigmoid(-top))
        out["dlogits"] = dlogits
    if s["mask"] is not None:
        for name in ("weights", "dlogits"):
            if name in out:
                out[name] = out[name] * s["mask"][:, None]
    return out


def _exact_int4(s, case):
    out = torch.zeros((case["tokens"], case["hidden"]), dtype=torch.float64, device="cuda")
    x = s["x"].double()
    for e in range(case["experts"]):
        token, choice = torch.nonzero(s["ids"] == e, as_tuple=True)
        if token.numel() == 0:
            continue
        first, second = (_values([None if t is None else t[e:e + 1] for t in s[w]], torch.float64)[0] for w in ("w1", "w2"))
        hidden = torch.nn.functional.gelu(x[token] @ first.t())
        out.index_add_(0, token, s["weights"][token, choice, None].double() * (hidden @ second.t()))
    return dict(out=out)
