"""The trainable way of the tokens through a dMoE layer: the router's gate, the placement of the chosen (token, choice)
slots in padded expert bins, the copy of the token rows there and the weighted sum of the experts' rows back, each
with its gradient.  Public as stk_b200.dmoe.top_k_gate / plan_rows / plan_tokens / sort_tokens / unsort_tokens:

    weights, ids = dmoe.top_k_gate(x @ w_router, top_k)
    plan = dmoe.plan_tokens(ids, num_experts)
    topo = dmoe.topology_from_bins(plan.bin_rows, plan.block_rows, ffn, x.dtype, x.device, materialize=False)
    y = dmoe.expert_mlp(dmoe.sort_tokens(x, plan), w1, w2, topo)
    out = dmoe.unsort_tokens(y, weights, plan)             # differentiable in x, w_router, w1 and w2

On CUDA tensors everything runs as kernels of libstk_b200.so.  Host tensors take plain torch operations (as in
stk_b200.dmoe: for tests, not for production use).  The reference is a matmul library and has no counterpart.
"""
import threading

import torch
from torch.autograd.function import once_differentiable

from stk_b200.backend import lib as _lib

BLOCK = 128
MAX_EXPERTS = 1024     # of the gate and of a plan
MAX_TOP_K = 32         # of the gate
_SCORES = {"softmax": 0, "sigmoid": 1}


def _rows(t):
    """`t`, or a copy, as rows that are contiguous in themselves.  (Rows that are one row repeated, with a stride of 0,
    are fine: they are only read.)"""
    return t if t.shape[1] <= 1 or t.stride(1) == 1 else t.contiguous()


def _ld(t):
    return t.stride(0) if t.shape[0] > 1 else max(t.shape[1], 1)


def _same_device(what, *tensors):
    devices = {t.device for t in tensors if t is not None}
    if len(devices) > 1:
        raise ValueError(f"{what}: all tensors must be on one device, got " + ", ".join(sorted(map(str, devices))))


# ------------------------------------------------------------------------------ gate
class _TopKGate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, mask, top_k, score, normalize):
        tokens, experts = logits.shape
        dev = logits.device
        weights = torch.empty((tokens, top_k), dtype=torch.float32, device=dev)
        ids = torch.empty((tokens, top_k), dtype=torch.int32, device=dev)
        dense = score == 0 and not normalize           # the gradient reaches every logit
        stats = torch.empty((tokens, 2), dtype=torch.float32, device=dev) if dense and ctx.needs_input_grad[0] else None
        rows = _rows(logits)
        with _lib.on_device(dev):
            rc = _lib.load().stk_b200_top_k_gate(
                _lib.ptr(rows), _ld(rows), tokens, experts, top_k, score, int(normalize), _lib.ptr(mask),
                _lib.ptr(weights), _lib.ptr(ids), _lib.ptr(stats), _lib.row_dtype_code(logits.dtype),
                _lib.stream_ptr(dev))
        _lib.check(rc, "stk_b200_top_k_gate")
        ctx.mark_non_differentiable(ids)
        ctx.set_materialize_grads(False)
        # (the normalized softmax weights alone give their gradient)
        ctx.save_for_backward(logits if dense or score == 1 else None, weights, ids, stats)
        ctx.like = (logits.shape, logits.dtype)
        ctx.kind = (score, normalize)
        return weights, ids

    @staticmethod
    @once_differentiable
    def backward(ctx, dweights, _):
        if dweights is None:
            return None, None, None, None, None
        logits, weights, ids, stats = ctx.saved_tensors
        (tokens, experts), dtype = ctx.like
        dev = weights.device
        dweights = dweights.contiguous()
        dlogits = torch.empty((tokens, experts), dtype=dtype, device=dev)
        rows = dlogits if logits is None else _rows(logits)
        with _lib.on_device(dev):
            rc = _lib.load().stk_b200_top_k_gate_backward(
                _lib.ptr(rows), _ld(rows), tokens, experts, weights.shape[1], ctx.kind[0],
                int(ctx.kind[1]), _lib.ptr(weights), _lib.ptr(ids), _lib.ptr(stats), _lib.ptr(dweights),
                _lib.ptr(dlogits), _lib.row_dtype_code(dtype), _lib.stream_ptr(dev))
        _lib.check(rc, "stk_b200_top_k_gate_backward")
        return dlogits, None, None, None, None


def _host_gate(logits, mask, top_k, score, normalize):
    values = logits.float()
    nan = values.detach().isnan()
    ids = torch.sort(values.detach().masked_fill(nan, torch.inf), dim=1, descending=True, stable=True).indices[:, :top_k]
    top = torch.gather(values, 1, ids)
    valid = top.detach() != -torch.inf
    if mask is not None:
        valid = valid & mask[:, None]
    top = top.masked_fill(~valid, -torch.inf)
    if score == 0:
        some = valid.any(1, keepdim=True)
        if normalize:
            weights = torch.softmax(top.masked_fill(~some, 0.0), 1)
        else:
            whole = values.masked_fill(~some, 0.0)
            weights = torch.gather(torch.softmax(whole, 1), 1, ids)
    elif normalize:
        some = valid.any(1, keepdim=True)
        logs = torch.nn.functional.logsigmoid(top.masked_fill(~valid, 0.0)).masked_fill(~valid & some, -torch.inf)
        weights = torch.softmax(logs, 1)
    else:
        weights = torch.sigmoid(top)
    weights = weights + torch.zeros(()).masked_fill(nan.any(1, keepdim=True), torch.nan)
    return weights.masked_fill(~valid, 0.0), ids.masked_fill(~valid, -1).to(torch.int32)


def top_k_gate(logits, top_k, score="softmax", normalize=True, token_mask=None):
    """The router's choice: (weights float32 [T, k], expert_ids int32 [T, k]) of the k largest logits of every token,
    the largest first, differentiable in `logits` through the weights.

    logits: [T, E] float16, bfloat16 or float32, E <= 1024; k <= min(E, 32).  score: "softmax" (over all E logits) or
    "sigmoid"; normalize: the k weights of a token are scaled to add up to 1.  Equal logits go to the lower expert, and
    an expert whose logit is -inf is never chosen.  A choice that is left without an expert (fewer than k logits above
    -inf, or token_mask[t] False: bool [T], padding tokens) has id -1 and weight 0 and passes no gradient; plan_tokens
    gives it no row.  A NaN counts as +inf among the logits and makes the token's weights NaN."""
    if logits.dim() != 2:
        raise ValueError(f"top_k_gate: logits must be [tokens, experts], got {tuple(logits.shape)}")
    if score not in _SCORES:
        raise ValueError(f"top_k_gate: score must be one of {sorted(_SCORES)}, got {score!r}")
    tokens, experts = logits.shape
    _lib.row_dtype_code(logits.dtype)
    if not 1 <= experts <= MAX_EXPERTS or not 1 <= top_k <= min(experts, MAX_TOP_K):
        raise ValueError(f"top_k_gate: 1 <= top_k <= min(experts, {MAX_TOP_K}) and experts <= {MAX_EXPERTS}, got "
                         f"top_k = {top_k}, {experts} experts")
    if token_mask is not None:
        if token_mask.dtype != torch.bool or tuple(token_mask.shape) != (tokens,):
            raise ValueError(f"top_k_gate: token_mask must be bool [{tokens}], got {token_mask.dtype} "
                             f"{tuple(token_mask.shape)}")
        _same_device("top_k_gate", logits, token_mask)
        token_mask = token_mask.contiguous()
    if not logits.is_cuda:
        return _host_gate(logits, token_mask, top_k, _SCORES[score], normalize)
    return _TopKGate.apply(logits, token_mask, int(top_k), _SCORES[score], bool(normalize))


# ------------------------------------------------------------------------------ placement
class TokenPlan:
    """Where the slots of one routed batch (slot = token * top_k + choice) sit in padded expert bins; made by
    plan_tokens and not to be changed.

    index     int32 [rows]       slot in the row, -1: padding
    position  int32 [T * top_k]  row of the slot, -1: a slot without an expert
    bin_rows  int32 [E]          blocks of every expert's bin, as topology_from_bins takes them
    rows, block_rows             rows of all bins, and the same in blocks (host ints)"""

    __slots__ = ("index", "position", "bin_rows", "rows", "block_rows", "tokens", "top_k", "num_experts", "block")

    def __init__(self, index, position, bin_rows, rows, tokens, top_k, num_experts, block):
        self.index, self.position, self.bin_rows = index, position, bin_rows
        self.rows, self.block_rows = rows, rows // block
        self.tokens, self.top_k, self.num_experts, self.block = tokens, top_k, num_experts, block


def plan_rows(slots, num_experts, block=BLOCK):
    """Most rows that `slots` choices can take in bins padded to a multiple of `block`, whatever the choices are."""
    return (slots + min(slots, num_experts) * (block - 1)) // block * block


_pinned = threading.local()


def _host_word():
    """Pinned int64 of this thread, which a kernel writes and the thread waits for: never in two uses at once."""
    word = getattr(_pinned, "word", None)
    if word is None:
        word = _pinned.word = torch.zeros(1, dtype=torch.int64).pin_memory()
    return word


def plan_tokens(expert_ids, num_experts, block=BLOCK, rows=None):
    """TokenPlan of expert_ids ([T] or [T, k], integers; a negative id: no expert): every expert's slots in order, its
    bin padded to a multiple of `block` rows.

    rows None: as many rows as this batch needs - the one read-back of the step (the call waits for the stream).
    rows = plan_rows(slots, num_experts) or more, a multiple of `block`: that many, the surplus as padding at the end
    of the last expert's bin; nothing waits for the device, and the step can be captured in a CUDA graph."""
    if expert_ids.dim() not in (1, 2) or expert_ids.dtype not in (torch.int16, torch.int32, torch.int64):
        raise ValueError(f"plan_tokens: expert_ids must be integers [T] or [T, k], got {expert_ids.dtype} "
                         f"{tuple(expert_ids.shape)}")
    if not 1 <= num_experts <= MAX_EXPERTS:
        raise ValueError(f"plan_tokens: 1 to {MAX_EXPERTS} experts, got {num_experts}")
    if block < 1:
        raise ValueError(f"plan_tokens: block must be positive, got {block}")
    tokens = expert_ids.shape[0]
    top_k = 1 if expert_ids.dim() == 1 else expert_ids.shape[1]
    if top_k < 1:
        raise ValueError("plan_tokens: no choices")
    flat = expert_ids.reshape(-1)
    slots, need = flat.numel(), plan_rows(flat.numel(), num_experts, block)
    if need > 2 ** 31 - 1:
        raise ValueError(f"plan_tokens: {slots} slots are beyond what 32-bit row numbers name")
    if rows is not None and (rows < need or rows % block or rows > 2 ** 31 - 1):
        raise ValueError(f"plan_tokens: rows must be a multiple of {block} and at least plan_rows(...) = {need}, got {rows}")
    if not flat.is_cuda:
        index, position, bin_rows = _host_plan(flat.long(), num_experts, block, rows)
        return TokenPlan(index, position, bin_rows, index.numel(), tokens, top_k, num_experts, block)
    dev = flat.device
    if rows is None and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("plan_tokens: reading the number of rows back cannot be captured; pass rows=plan_rows(...)")
    flat = flat.to(torch.int32).contiguous()
    length = need if rows is None else rows
    index = torch.empty(length, dtype=torch.int32, device=dev)
    position = torch.empty(slots, dtype=torch.int32, device=dev)
    bin_rows = torch.empty(num_experts, dtype=torch.int32, device=dev)
    lib = _lib.load()
    ws_bytes = lib.stk_b200_place_workspace_bytes(slots, num_experts)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None
    word = _host_word() if rows is None else None
    with _lib.on_device(dev):
        rc = lib.stk_b200_place_tokens(
            _lib.ptr(flat), slots, num_experts, block, length, int(rows is not None), _lib.ptr(index),
            _lib.ptr(position), _lib.ptr(bin_rows), _lib.ptr(word), _lib.ptr(ws), ws_bytes, _lib.stream_ptr(dev))
    _lib.check(rc, "stk_b200_place_tokens")
    if rows is None:
        torch.cuda.current_stream(dev).synchronize()
        length = int(word)
        index = index[:length]
    return TokenPlan(index, position, bin_rows, length, tokens, top_k, num_experts, block)


def _host_plan(flat, num_experts, block, rows):
    if bool((flat >= num_experts).any()):
        raise ValueError(f"plan_tokens: expert ids reach {int(flat.max())}, there are {num_experts} experts")
    live = torch.nonzero(flat >= 0).view(-1)
    order = live[torch.argsort(flat[live], stable=True)]
    counts = torch.bincount(flat[live], minlength=num_experts)
    blocks = (counts + block - 1) // block
    used = int(blocks.sum()) * block
    starts = (torch.cumsum(blocks, 0) - blocks) * block
    first = torch.cumsum(counts, 0) - counts
    experts = flat[order]
    place = starts[experts] + torch.arange(order.numel()) - first[experts]
    position = torch.full((flat.numel(),), -1, dtype=torch.int32)
    position[order] = place.to(torch.int32)
    index = torch.full((used if rows is None else rows,), -1, dtype=torch.int32)
    index[place] = order.to(torch.int32)
    if rows is not None:
        blocks[-1] += (rows - used) // block
    return index, position, blocks.to(torch.int32)


# ------------------------------------------------------------------------------ rows there and back
def _sum_rows(rows, weights, plan):
    rows = _rows(rows)
    out = torch.empty((plan.tokens, rows.shape[1]), dtype=rows.dtype, device=rows.device)
    with _lib.on_device(rows.device):
        rc = _lib.load().stk_b200_sum_rows(
            _lib.ptr(rows), _ld(rows), _lib.ptr(plan.position), _lib.ptr(weights), _lib.ptr(out), plan.tokens,
            plan.top_k, rows.shape[1], _lib.row_dtype_code(rows.dtype), _lib.stream_ptr(rows.device))
    _lib.check(rc, "stk_b200_sum_rows")
    return out


class _SortTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, plan):
        ctx.plan = plan
        x = _rows(x)
        rows = torch.empty((plan.rows, x.shape[1]), dtype=x.dtype, device=x.device)
        with _lib.on_device(x.device):
            rc = _lib.load().stk_b200_sort_rows(
                _lib.ptr(x), _ld(x), _lib.ptr(rows), _lib.ptr(plan.index), _lib.ptr(plan.position), plan.tokens,
                plan.top_k, plan.rows, x.shape[1], _lib.row_dtype_code(x.dtype), _lib.stream_ptr(x.device))
        _lib.check(rc, "stk_b200_sort_rows")
        return rows

    @staticmethod
    @once_differentiable
    def backward(ctx, drows):
        return _sum_rows(drows, None, ctx.plan), None


class _UnsortTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, plan):
        ctx.plan = plan
        need_weights = weights is not None and ctx.needs_input_grad[1]
        ctx.save_for_backward(rows if need_weights else None, weights)
        ctx.like = (rows.shape, rows.dtype)
        return _sum_rows(rows, weights, plan)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        rows, weights = ctx.saved_tensors
        plan, (shape, dtype) = ctx.plan, ctx.like
        dout = _rows(dout)
        drows = dweights = None
        if ctx.needs_input_grad[0]:
            drows = torch.empty(shape, dtype=dtype, device=dout.device)
        if rows is not None:
            rows = _rows(rows)
            dweights = torch.empty_like(weights)
        with _lib.on_device(dout.device):
            rc = _lib.load().stk_b200_unsort_backward(
                _lib.ptr(dout), _ld(dout), _lib.ptr(rows), 0 if rows is None else _ld(rows), _lib.ptr(weights),
                _lib.ptr(plan.index), _lib.ptr(plan.position), _lib.ptr(drows), _lib.ptr(dweights), plan.tokens,
                plan.top_k, plan.rows, shape[1], _lib.row_dtype_code(dtype), _lib.stream_ptr(dout.device))
        _lib.check(rc, "stk_b200_unsort_backward")
        return drows, dweights, None


def _check_rows(what, t, n, name, plan):
    if t.dim() != 2 or t.shape[0] != n:
        raise ValueError(f"{what}: expected {n} rows ({name}), got {tuple(t.shape)}")
    _lib.row_dtype_code(t.dtype)
    _same_device(what, t, plan.position)


def sort_tokens(x, plan):
    """The token rows x [T, h] (float16, bfloat16 or float32) in the padded expert order of `plan`: [plan.rows, h],
    zeros in padding rows.  Differentiable: the gradient of a token is the sum of those of its rows, added up in
    32 bits."""
    _check_rows("sort_tokens", x, plan.tokens, "tokens of the plan", plan)
    if x.is_cuda:
        return _SortTokens.apply(x, plan)
    valid = plan.index >= 0
    out = x.new_zeros((plan.rows, x.shape[1]))
    return out.index_put((torch.nonzero(valid).view(-1),),
                         x[torch.div(plan.index[valid].long(), plan.top_k, rounding_mode="floor")])


def unsort_tokens(rows, weights, plan):
    """The way back: out[t] = sum_j weights[t, j] * rows[row of slot t * k + j], [T, h], added up in 32 bits and rounded
    once.  rows [plan.rows, h]; weights [T, k] (or [T] for k = 1) float32 or a 16-bit float, None: all ones.  Slots
    without an expert contribute nothing.  Differentiable in `rows` (padding rows get zeros) and in `weights` (a slot
    without an expert gets 0)."""
    _check_rows("unsort_tokens", rows, plan.rows, "rows of the plan", plan)
    if weights is not None:
        if weights.numel() != plan.tokens * plan.top_k or weights.shape[:1] != (plan.tokens,):
            raise ValueError(f"unsort_tokens: weights must be [{plan.tokens}, {plan.top_k}], got {tuple(weights.shape)}")
        _lib.row_dtype_code(weights.dtype)
        _same_device("unsort_tokens", rows, weights)
        weights = weights.reshape(plan.tokens, plan.top_k).float().contiguous()
    if rows.is_cuda:
        return _UnsortTokens.apply(rows, weights, plan)
    position = plan.position.long()
    # (a gather of at least one row, so that an empty plan needs no case of its own)
    padded = torch.cat([rows.float(), torch.zeros((1, rows.shape[1]))])
    y = padded[torch.where(position >= 0, position, torch.full_like(position, plan.rows))]
    y = y.view(plan.tokens, plan.top_k, rows.shape[1])
    if weights is not None:
        y = y * weights[:, :, None]
    return y.sum(1).to(rows.dtype)
