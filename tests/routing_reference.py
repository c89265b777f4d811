"""Plain 64-bit statements of the gate, the token placement and the rows' ways, for the tests of stk_b200.routing."""
import torch

# One rounding to 32 bits is off by 2^-24 at most, relative to the value.
U32 = 2.0 ** -24
# Smallest step of the 16-bit formats near zero, halved (float32's is far below everything here).
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 0.0}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def gate(logits, top_k, score, normalize, mask=None):
    """(weights, ids, valid) in 64 bits, by lists: every token on its own.  Differentiable in `logits` (float64)."""
    weights, ids = [], []
    for t, row in enumerate(logits):
        values = row.tolist()
        order = sorted(range(len(values)), key=lambda e: (-values[e], e))[:top_k]
        picked = [e for e in order if values[e] != -float("inf")]
        if mask is not None and not bool(mask[t]):
            picked = []
        rest = top_k - len(picked)
        if picked:
            chosen = row[picked]
            if score == "softmax":
                w = torch.softmax(chosen if normalize else row, 0)
                w = w if normalize else w[picked]
            else:
                w = torch.sigmoid(chosen)
                w = torch.softmax(torch.nn.functional.logsigmoid(chosen), 0) if normalize else w
        else:
            w = row.new_zeros(0)
        weights.append(torch.cat([w, row.new_zeros(rest)]))
        ids.append(picked + [-1] * rest)
    return torch.stack(weights), torch.tensor(ids, dtype=torch.int32)


def placement(ids, experts, block, rows=None):
    """(index, position, bin_rows) by a plain loop over the slots."""
    flat = [int(e) for e in ids.reshape(-1)]
    bins = [[s for s, e in enumerate(flat) if e == x] for x in range(experts)]
    index, position, blocks = [], [-1] * len(flat), []
    for slots in bins:
        for i, s in enumerate(slots):
            position[s] = len(index) + i
        n = -(-len(slots) // block)
        index += slots + [-1] * (n * block - len(slots))
        blocks.append(n)
    if rows is not None:
        blocks[-1] += (rows - len(index)) // block
        index += [-1] * (rows - len(index))
    return tuple(torch.tensor(v, dtype=torch.int32) for v in (index, position, blocks))


def sort_rows(x, position, top_k, rows):
    out = torch.zeros((rows, x.shape[1]), dtype=x.dtype)
    for s, r in enumerate(position.tolist()):
        if r >= 0:
            out[r] = x[s // top_k]
    return out


def sum_rows(rows, position, weights, tokens, top_k):
    """(out, sum of magnitudes) in 64 bits; weights None: ones."""
    out = torch.zeros((tokens, rows.shape[1]), dtype=torch.float64)
    size = torch.zeros_like(out)
    for s, r in enumerate(position.tolist()):
        if r >= 0:
            w = 1.0 if weights is None else weights.reshape(-1)[s].double()
            out[s // top_k] += w * rows[r].double()
            size[s // top_k] += (w * rows[r].double()).abs()
    return out, size
