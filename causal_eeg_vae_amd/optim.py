"""AdamW over many tensors in one launch (ceeg_adamw_step, include/ceeg.h), moments in 32 bits or in 8.  The reference trains with Adam
(scripts/run.py:56); `Trainer(optimizer="adamw")` takes this one."""
import array
import operator

import torch

from . import _lib

BLOCK = 256                 # elements that share a scale of an 8-bit state
_SPREAD = 0x9E3779B97F4A7C15  # between the random streams of two steps
_DTYPES = {torch.float32: _lib.CEEG_F32, torch.bfloat16: _lib.CEEG_BF16}


def block_state(like):
    """A zero 8-bit moment of a parameter: (codes float8_e4m3fn of its shape, scales float32, one per 256 consecutive elements)."""
    return (torch.zeros(like.shape, dtype=torch.float8_e4m3fn, device=like.device),
            torch.zeros(-(-like.numel() // BLOCK), dtype=torch.float32, device=like.device))


def block_values(state, square=False):
    """What an 8-bit moment stands for, in float32; `square` for the second one, which is held as its root."""
    codes, scales = state
    x = codes.reshape(-1).float() * scales.repeat_interleave(BLOCK)[:codes.numel()]
    return (x * x if square else x).view(codes.shape)


_dtype_of = operator.attrgetter("dtype")


def _addresses(tensors):
    return list(map(torch.Tensor.data_ptr, tensors))


def _scalar(x, name, dev):
    if isinstance(x, torch.Tensor):
        if x.dtype != torch.float32 or x.numel() != 1 or x.device != dev:
            raise ValueError(f"{name}: a float32 tensor of one element on {dev} expected, got {x.dtype} {tuple(x.shape)} on {x.device}")
        return x
    return None


def adamw_step_(params, grads, exp_avgs, exp_avg_sqs, step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, seed=0):
    """One AdamW step over lists of tensors, in place.

    params and grads: all float32 or all bfloat16, contiguous, one device, each gradient of its parameter's shape.  exp_avgs and exp_avg_sqs: float32 tensors, or pairs
    (codes, scales) as `block_state` makes them, which hold m and sqrt(v) in 8 bits (all tensors alike).  step: the number of this step, from 1.
    step and lr may be float32 tensors of one element on the device, which a captured graph reads anew at every replay.  seed: of the random
    numbers that round 8-bit moments; take another one for every step (with a step tensor it changes by itself)."""
    n = len(params)
    if not n == len(grads) == len(exp_avgs) == len(exp_avg_sqs):
        raise ValueError(f"lists of one length expected, got {n}, {len(grads)}, {len(exp_avgs)} and {len(exp_avg_sqs)}")
    if n == 0:
        return
    if not isinstance(params[0], torch.Tensor):
        raise TypeError(f"parameters must be tensors, got {type(params[0]).__name__}")
    dtype, dev = params[0].dtype, params[0].device
    if dtype not in _DTYPES:
        raise TypeError(f"parameters must be float32 or bfloat16, got {dtype}")
    T = torch.Tensor
    held = not isinstance(exp_avgs[0], T)
    scales = None
    if held:
        try:
            (ms, m_scales), (vs, v_scales) = zip(*exp_avgs), zip(*exp_avg_sqs)
        except (TypeError, ValueError):
            raise TypeError("exp_avgs and exp_avg_sqs must be all tensors or all pairs (codes, scales)") from None
        scales = m_scales + v_scales
        try:
            scale_sizes = list(map(T.numel, scales))
        except TypeError:
            raise TypeError("exp_avgs and exp_avg_sqs must be all tensors or all pairs (codes, scales)") from None
    else:
        ms, vs = exp_avgs, exp_avg_sqs
    state = torch.float8_e4m3fn if held else torch.float32
    every = (("params", params, dtype), ("grads", grads, dtype), ("exp_avgs", ms, state), ("exp_avg_sqs", vs, state))
    try:   # a call goes through hundreds of small tensors: mapped methods, no loop of attributes
        sizes = list(map(T.numel, params))
        at = params[0].get_device()
        shapes = list(map(T.size, params))   # a gradient of as many elements in another shape is not this parameter's
        for what, tensors, want in every:
            fits = list(map(T.size, tensors)) == shapes if tensors is grads else tensors is params or list(map(T.numel, tensors)) == sizes
            if not fits or not all(map(T.is_contiguous, tensors)) or set(map(_dtype_of, tensors)) != {want} or set(map(T.get_device, tensors)) != {at}:
                raise ValueError(f"{what}: contiguous {want} tensors of the parameters' sizes on {dev} expected, got " +
                                 ", ".join(f"{t.dtype} {tuple(t.shape)} on {t.device}" for t in tensors[:4]))
    except TypeError:
        raise ValueError("params, grads, exp_avgs and exp_avg_sqs: tensors expected") from None
    if held:
        if scale_sizes != [-(-k // BLOCK) for k in sizes] * 2 or not all(map(T.is_contiguous, scales)) or \
                set(map(_dtype_of, scales)) != {torch.float32} or set(map(T.get_device, scales)) != {at}:
            raise ValueError(f"scales: contiguous float32 tensors of one element per {BLOCK} on {dev} expected, got " +
                             ", ".join(f"{t.dtype} {tuple(t.shape)} on {t.device}" for t in scales[:4]))
    _lib.require_cuda(params[0])
    pp, mp, vp = _addresses(params), _addresses(ms), _addresses(vs)
    sp = _addresses(scales) if held else []
    where = pp + mp + vp + sp
    if len(set(where)) < len(where) and len(set(where) - {0}) < len(where) - where.count(0):   # an empty tensor has no address
        raise ValueError("a tensor that the step writes is given twice")
    b1, b2 = betas
    step_t, lr_t = _scalar(step, "step", dev), _scalar(lr, "lr", dev)
    if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0 and eps >= 0.0 and (step_t is not None or step >= 1)):
        raise ValueError(f"betas in [0, 1), eps >= 0 and step >= 1 expected, got {betas}, {eps} and {step}")
    if step_t is None and torch.cuda.is_current_stream_capturing():
        raise ValueError("a captured step needs its number as a tensor on the device: an int would be the same at every replay")
    # host arrays of addresses, alive for the call
    lists = [array.array("q", sizes)] + [array.array("Q", x) for x in (pp, _addresses(grads), mp, vp, sp[:n], sp[n:])]
    sizes_at, p_at, g_at, m_at, v_at, ms_at, vs_at = (x.buffer_info()[0] for x in lists)
    with _lib.on(dev):
        _lib.check(_lib.lib().ceeg_adamw_step(
            n, sizes_at, p_at, g_at, m_at, v_at, ms_at if held else None, vs_at if held else None, _DTYPES[dtype], 8 if held else 32,
            0.0 if lr_t is not None else float(lr), float(b1), float(b2), float(eps), float(weight_decay), 1 if step_t is not None else int(step),
            _lib.ptr(lr_t), _lib.ptr(step_t), int(seed) & (2**64 - 1), _lib.stream()), "ceeg_adamw_step")
    torch.autograd.graph.increment_version(params)   # a graph that saved a parameter notices


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW's update with one launch for (up to 56) tensors, and, with state_bits=8, moments of one byte an element (+ 4 per 256):
    an optimizer state of a quarter of the size.  Tensors of fewer than `min_8bit_size` elements keep theirs in 32 bits.

    capturable=True keeps the step counts on the device, so that `step()` can be captured into a graph and replayed (with gradients of the same
    parameters every time; the first step, which makes the moments, is taken before); lr may then be a float32 tensor on the device too.  Parameters: float32 or bfloat16 on the GPU, contiguous, gradients of the same type."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, min_8bit_size=4096, seed=0, capturable=False):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0 and eps >= 0.0 and weight_decay >= 0.0):
            raise ValueError(f"betas in [0, 1), eps >= 0 and weight_decay >= 0 expected, got {betas}, {eps} and {weight_decay}")
        if not isinstance(lr, torch.Tensor) and lr < 0.0:
            raise ValueError(f"lr >= 0 expected, got {lr}")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits, min_8bit_size=min_8bit_size,
                                      seed=seed, capturable=capturable))

    def _new_state(self, p, group):
        held = group["state_bits"] == 8 and p.numel() >= group["min_8bit_size"]
        new = block_state if held else lambda t: torch.zeros_like(t, dtype=torch.float32, memory_format=torch.contiguous_format)  # noqa: E731
        return dict(exp_avg=new(p), exp_avg_sq=new(p))

    def load_state_dict(self, state_dict):
        """As torch's, with the moments in the types that they were saved in (torch casts them to the parameter's)."""
        if not all("state_bits" in saved for saved in state_dict["param_groups"]):
            raise ValueError("the state of another optimizer")
        super().load_state_dict(state_dict)
        kept = lambda x, dev: tuple(t.detach().to(dev, copy=True) for t in x) if isinstance(x, tuple) else x.detach().to(dev, copy=True)  # noqa: E731
        for group, saved in zip(self.param_groups, state_dict["param_groups"]):
            counts = {}  # parameters that have taken as many steps share their count again
            for p, i in zip(group["params"], saved["params"]):
                if i in state_dict["state"]:
                    held = state_dict["state"][i]
                    st = {k: kept(x, p.device) for k, x in held.items() if k != "step"}
                    n = int(held["step"])
                    if group["capturable"]:
                        if (n, p.device) not in counts:
                            counts[n, p.device] = torch.full((), n, dtype=torch.float32, device=p.device)
                        n = counts[n, p.device]
                    st["step"] = n
                    self.state[p] = st

    def _count(self, group, taking):
        """One step more for the parameters in `taking`; on the device one count serves all that have taken the same steps."""
        if not group["capturable"]:
            for p in taking:
                self.state[p]["step"] += 1
            return
        now, counts = set(taking), {}
        for p in group["params"]:
            st = self.state.get(p)
            if st:
                counts.setdefault(id(st["step"]), (st["step"], [], []))[1 if p in now else 2].append(p)
        for count, with_grad, without in counts.values():
            if with_grad and without:
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("AdamW: a captured step must take the parameters of the step before it")
                count = count.clone()
                for p in with_grad:
                    self.state[p]["step"] = count
            if with_grad:
                count += 1

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        ordinal = 0
        for group in self.param_groups:
            taking = [p for p in group["params"] if p.grad is not None]
            fresh = {}
            for p in taking:
                st = self.state[p]
                if not st:
                    if p.is_cuda and torch.cuda.is_current_stream_capturing():
                        raise RuntimeError("AdamW: take a step before capturing one: moments made inside a graph would start anew at every replay")
                    st.update(self._new_state(p, group))
                    if group["capturable"] and p.device not in fresh:
                        fresh[p.device] = torch.zeros((), dtype=torch.float32, device=p.device)
                    st["step"] = fresh[p.device] if group["capturable"] else 0
            self._count(group, taking)
            lists = {}  # one call takes tensors of one type, one device, one form of state and one number of steps
            for p in taking:
                st = self.state[p]
                lists.setdefault((p.dtype, p.device, isinstance(st["exp_avg"], tuple), id(st["step"]) if group["capturable"] else st["step"]), []).append(p)
            for ps in lists.values():
                step = self.state[ps[0]]["step"]
                seed = group["seed"] + (ordinal << 32)  # another stream for every list
                ordinal += 1
                if not group["capturable"]:
                    seed += step * _SPREAD
                adamw_step_(ps, [p.grad if p.grad.is_contiguous() else p.grad.contiguous() for p in ps], [self.state[p]["exp_avg"] for p in ps],
                            [self.state[p]["exp_avg_sq"] for p in ps], step, lr=group["lr"], betas=group["betas"], eps=group["eps"],
                            weight_decay=group["weight_decay"], seed=seed)
        return loss
