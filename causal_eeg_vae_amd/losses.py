"""Losses at the end of a training step: the token cross entropy behind a vocabulary product (the reference's `recon_loss`,
scripts/gpt2.py:1080-1084 and scripts/models.py:34, over the hidden states of the caller's language decoder) and the balance loss over an
assignment to codes or experts.  The kernels are ceeg_linear_ce_fwd / _bwd and ceeg_balance_fwd / _bwd (include/ceeg.h)."""
import torch
import torch.autograd.forward_ad as _forward

from . import _lib

_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


def _dtype(t, what):
    if t.dtype == torch.float32:
        return _lib.CEEG_F32
    if t.dtype == torch.bfloat16:
        return _lib.CEEG_BF16
    raise TypeError(f"{what} must be float32 or bfloat16, got {t.dtype}")


def _same_device(*tensors):
    _lib.require_cuda(*tensors)
    if len({t.get_device() for t in tensors if t is not None}) > 1:
        raise ValueError(f"all tensors must be on one device, got {[str(t.device) for t in tensors if t is not None]}")


def _came_back(t, shape, dtype, dev):
    """A saved tensor comes back through a hook with its values in other strides, perhaps; as something else it is refused: its memory would be read as the old one's."""
    if t.shape != shape or t.dtype != dtype or t.device != dev:
        raise ValueError(f"a saved tensor came back as {t.dtype} {tuple(t.shape)} on {t.device}, not as {dtype} {tuple(shape)} on {dev}")


def _has_tangent(*tensors):
    """Inside a level of forward mode (where there is none, nothing has one): whether one of them carries a tangent."""
    return _forward._current_level >= 0 and any(_forward.unpack_dual(t).tangent is not None for t in tensors)


def _weight_rows(weight, dtype):
    """(weight, row stride) as the entries take it: a copy where its strides or its alignment do not allow to read it in place."""
    V, H = weight.shape
    if weight.stride(1) != 1 or (V > 1 and not H <= weight.stride(0) <= 1 << 22) or (dtype == _lib.CEEG_BF16 and (weight.data_ptr() % 16 or not weight.is_contiguous())):
        weight = weight.clone(memory_format=torch.contiguous_format)
    return weight, H if weight.is_contiguous() else weight.stride(0)


def _linear_ce(hidden, weight, target, ignore_index, reduction):
    """The loss, and what the backward takes back."""
    L = _lib.lib()
    dtype = _dtype(hidden, "hidden")
    (T, H), V = hidden.shape, weight.shape[0]
    dev = hidden.device
    if hidden.stride(1) != 1 or (T > 1 and hidden.stride(0) < H):
        hidden = hidden.contiguous()
    weight, ldw = _weight_rows(weight, dtype)
    target = target.contiguous()
    ldh = max(hidden.stride(0), H)
    with _lib.on(dev):
        loss = torch.empty(T if reduction == 0 else (), dtype=torch.float32, device=dev)
        # one buffer for what the backward takes back: the packed rows, lse [T], tokens [3 T + 1]
        rows = L.ceeg_linear_ce_packed_bytes(T, H, dtype)
        kept = _lib.workspace(rows + 16 * T + 4, dev)
        packed = kept.data_ptr()
        lse, tokens = packed + rows, packed + rows + 4 * T
        ws = _lib.workspace(L.ceeg_linear_ce_fwd_ws_bytes(T, H, V, dtype), dev)
        with _lib.timed("linear_ce_fwd"):
            _lib.check(L.ceeg_linear_ce_fwd(hidden.data_ptr(), ldh, weight.data_ptr(), ldw, target.data_ptr(), T, H, V, dtype, ignore_index, reduction,
                                            loss.data_ptr(), lse, tokens, packed, ws.data_ptr(), ws.numel(), _lib.stream()),
                       "ceeg_linear_ce_fwd")
    return loss, kept, weight, (T, H, V, dtype, reduction, rows)


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, target, ignore_index, reduction):
        loss, kept, weight, ctx.sizes = _linear_ce(hidden, weight, target, ignore_index, reduction)
        ctx.save_for_backward(kept, weight)
        ctx.saved_as = kept.shape, weight.shape, weight.dtype, weight.device
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        kept, weight = ctx.saved_tensors
        T, H, V, dtype, reduction, rows = ctx.sizes
        L = _lib.lib()
        # saved tensors may come back through a hook as other tensors of the same values: strides and alignment are theirs, not those of the forward
        kept_shape, shape, saved_type, dev = ctx.saved_as
        _came_back(kept, kept_shape, torch.uint8, dev)
        _came_back(weight, shape, saved_type, dev)
        weight, ldw = _weight_rows(weight, dtype)
        if kept.data_ptr() % 256 or not kept.is_contiguous():
            kept = kept.clone(memory_format=torch.contiguous_format)
        need_h, need_w = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        with _lib.on(dev):
            g = g.to(torch.float32).contiguous()
            packed = kept.data_ptr()
            dh = torch.empty(T, H, dtype=weight.dtype, device=dev) if need_h else None
            dw = torch.empty(V, H, dtype=weight.dtype, device=dev) if need_w else None
            ws = _lib.workspace(L.ceeg_linear_ce_bwd_ws_bytes(T, H, V, dtype), dev)
            with _lib.timed("linear_ce_bwd"):
                _lib.check(L.ceeg_linear_ce_bwd(packed, weight.data_ptr(), ldw, T, H, V, dtype, reduction, g.data_ptr(), packed + rows,
                                                packed + rows + 4 * T, _lib.ptr(dh), _lib.ptr(dw), ws.data_ptr(), ws.numel(), _lib.stream()),
                           "ceeg_linear_ce_bwd")
        return dh, dw, None, None, None


def linear_cross_entropy(hidden, weight, target, ignore_index=-100, reduction="mean"):
    """Cross entropy of `hidden @ weight.T` against `target` without the logits in memory, forward and backward.

    hidden [..., H], weight [V, H] (both float32 or both bfloat16), target [...] int64 of hidden's leading shape.  Tokens whose target is
    `ignore_index` (padding) take no part, whatever their hidden row holds.  reduction: "mean" over the tokens that count (0 where none does),
    "sum", or "none" (target's shape, 0 where ignored).  The loss is float32; the gradients have their inputs' types, all sums are float32.
    bfloat16: the gradient of the logits is rounded to bfloat16 before the two products that it enters (2^-8 of a value at most), and the gradients are
    rounded again.  A probability in the backward is off by about 2^-24 |log sum exp| of itself.
    A target outside [0, V) makes the loss and the gradients it reaches NaN: an error would need a host read of the targets.
    There is no forward mode: a tangent is a NotImplementedError."""
    if not all(isinstance(t, torch.Tensor) for t in (hidden, weight, target)):
        raise TypeError("hidden, weight and target must be tensors")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be 'none', 'mean' or 'sum', got {reduction!r}")
    if hidden.dim() < 1 or weight.dim() != 2 or hidden.shape[-1] != weight.shape[1] or target.shape != hidden.shape[:-1]:
        raise ValueError(f"hidden [..., H], weight [V, H] and target [...] expected; got {tuple(hidden.shape)}, {tuple(weight.shape)} and {tuple(target.shape)}")
    if target.dtype != torch.int64:
        raise TypeError(f"target must be int64, got {target.dtype}")
    _dtype(hidden, "hidden")
    if hidden.dtype != weight.dtype:
        raise TypeError(f"hidden and weight must have one type, got {hidden.dtype} and {weight.dtype}")
    if weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError(f"weight must have a class and a column at least, got {tuple(weight.shape)}")
    _same_device(hidden, weight, target)
    if target.numel() == 0:  # no token: nothing to launch, the gradients are zero
        none = hidden.float().sum(-1) + weight[:0].float().sum()
        return none if reduction == "none" else none.sum()
    if hidden.dim() != 2:   # rows of a matrix go in as they are: a view would be another node of the graph
        hidden = hidden.reshape(-1, hidden.shape[-1])
    args = hidden, weight, target.reshape(-1), int(ignore_index), _REDUCTIONS[reduction]
    if torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad) or _has_tangent(hidden, weight):
        loss = _LinearCrossEntropy.apply(*args)   # which refuses forward mode
    else:  # nothing comes back: autograd's part of the call is left out
        loss = _linear_ce(*args)[0]
    return loss.view(target.shape) if reduction == "none" else loss


def _score_rows(scores):
    """(scores, row stride) as the entries take them."""
    T, E = scores.shape
    row, column = scores.stride()
    if column != 1 or (T > 1 and row < E):
        scores = scores.contiguous()
        row = scores.stride(0)
    return scores, max(row, E)


class _Balance(torch.autograd.Function):
    @staticmethod
    def forward(ctx, scores, indices, mask):
        L = _lib.lib()
        dtype = _dtype(scores, "scores")
        (T, E), K = scores.shape, indices.shape[1]
        dev = scores.device
        scores, ld = _score_rows(scores)
        indices = indices.contiguous()
        mask = None if mask is None else mask.contiguous()
        with _lib.on(dev):
            loss = torch.empty((), dtype=torch.float32, device=dev)
            counts = torch.empty(E, dtype=torch.int64, device=dev)
            stats = torch.empty(E + 1, dtype=torch.float32, device=dev)
            ws = _lib.workspace(L.ceeg_balance_ws_bytes(T, E), dev)
            with _lib.timed("balance_fwd"):
                _lib.check(L.ceeg_balance_fwd(scores.data_ptr(), ld, dtype, indices.data_ptr(), indices.element_size(), T, E, K, _lib.ptr(mask),
                                              loss.data_ptr(), counts.data_ptr(), stats.data_ptr(), ws.data_ptr(), ws.numel(), _lib.stream()),
                           "ceeg_balance_fwd")
        ctx.save_for_backward(scores, mask)
        ctx.sizes, ctx.stats = (T, E, dtype), stats
        ctx.saved_as = scores.shape, scores.dtype, dev
        ctx.mark_non_differentiable(counts)
        return loss, counts

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g, _g_counts):
        scores, mask = ctx.saved_tensors
        (T, E, dtype), stats = ctx.sizes, ctx.stats
        # saved tensors may come back through a hook as other tensors of the same values: strides are theirs, not those of the forward
        shape, saved_type, dev = ctx.saved_as
        _came_back(scores, shape, saved_type, dev)
        scores, ld = _score_rows(scores)
        if mask is not None:
            _came_back(mask, (T,), torch.bool, dev)
            mask = mask.contiguous()
        with _lib.on(dev):
            g = g.to(torch.float32).contiguous()
            ds = torch.empty(T, E, dtype=scores.dtype, device=dev)
            with _lib.timed("balance_bwd"):
                _lib.check(_lib.lib().ceeg_balance_bwd(scores.data_ptr(), ld, dtype, T, E, _lib.ptr(mask), stats.data_ptr(), g.data_ptr(), ds.data_ptr(),
                                                       _lib.stream()), "ceeg_balance_bwd")
        return ds, None, None


def balance_loss(scores, indices, mask=None):
    """(loss, counts): E * sum_e f_e P_e with f the share of the assignments that code (or expert) e got and P its mean softmax probability - 1 where the
    codes are used evenly, more where few of them get both - and the assignments per code, int64 [E].

    scores [T, E] float32 or bfloat16, indices [T] or [T, K] int32 / int64 (-1: no assignment), mask [T] bool (False: the row does not
    count).  The gradient flows to the scores through P.  No row that counts: loss 0.  A code outside [-1, E) makes the loss NaN.  E <= 4096."""
    if not all(isinstance(t, torch.Tensor) for t in (scores, indices)) or not (mask is None or isinstance(mask, torch.Tensor)):
        raise TypeError("scores, indices and mask must be tensors")
    if indices.dim() == 1:
        indices = indices[:, None]
    if scores.dim() != 2 or indices.dim() != 2 or indices.shape[0] != scores.shape[0]:
        raise ValueError(f"scores [T, E] and indices [T] or [T, K] expected; got {tuple(scores.shape)} and {tuple(indices.shape)}")
    T, E = scores.shape
    if not 1 <= E <= 4096 or not 1 <= indices.shape[1] <= E:
        raise ValueError(f"1 <= E <= 4096 and 1 <= K <= E expected, got E = {E}, K = {indices.shape[1]}")
    if indices.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"indices must be int32 or int64, got {indices.dtype}")
    if mask is not None and (mask.dtype != torch.bool or mask.shape != (T,)):
        raise ValueError(f"mask must be bool [{T}], got {mask.dtype} {tuple(mask.shape)}")
    _dtype(scores, "scores")
    _same_device(scores, indices, mask)
    if T == 0:  # no row: nothing to launch, the gradient is empty
        return scores.float().sum() * 0.0, torch.zeros(E, dtype=torch.int64, device=scores.device)
    return _Balance.apply(scores, indices, mask)
