"""Cases of the training-step operators: the token cross entropy behind a vocabulary product, the balance loss over code (or expert) assignments
and the multi-tensor AdamW step, with the same operators in plain torch operations beside the framework's calls.

`run` makes the framework's calls where `own` is true and computes the plain forms otherwise; both work on what `prepare` made."""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
BLOCK = 256              # consecutive elements of a tensor that share one scale of an 8-bit state
TOP = 448.0              # largest number of an 8-bit state
TINY = 2.0 ** -100       # a block whose largest magnitude is below this is held as zeros
TAG = 0x41444D57         # third counter word of the rounding's random numbers (the fourth is the tensor's place in the list)
IGNORE = -100


def listed():
    return [
        # the smallest call: latents of a few graphs scored against a codebook of 512 codes, forward and backward; launches are what it costs
        dict(name="ce_code_head_f32", op="ce", tokens=97, width=64, classes=512, dtype="f32", grad=True, ignored=0.1),
        # the next code of a sequence predicted over the largest codebook, in the framework's own 32 bits
        dict(name="ce_codebook_f32", op="ce", tokens=16384, width=256, classes=4096, dtype="f32", grad=True, ignored=0.0),
        # 32 headlines of 60 tokens, padded ones ignored, against a language decoder's odd vocabulary
        dict(name="ce_text_bf16", op="ce", tokens=1920, width=768, classes=50257, dtype="bf16", grad=True, ignored=0.4),
        # the largest: a long batch against a large vocabulary
        dict(name="ce_large_bf16", op="ce", tokens=8192, width=1024, classes=131072, dtype="bf16", grad=True, ignored=0.1),
        # validation: the loss of every token, no gradient
        dict(name="ce_eval_bf16", op="ce", tokens=5000, width=768, classes=50257, dtype="bf16", grad=False, ignored=0.3),
        # one token scored against the vocabulary while text is generated
        dict(name="ce_one_token_bf16", op="ce", tokens=1, width=768, classes=50257, dtype="bf16", grad=False, ignored=0.0),
        # a router's few rows, some masked, some assignments dropped
        dict(name="balance_small_bf16", op="balance", rows=61, classes=16, picks=2, dtype="bf16", masked=0.3),
        # the code of every node of a large graph against 512 codes
        dict(name="balance_codes_f32", op="balance", rows=262144, classes=512, picks=1, dtype="f32", masked=0.0),
        # the graph model's own few parameters: one launch is what it costs
        dict(name="adamw_model_f32", op="adamw", tensors=7, elements=262144, dtype="f32", bits=32),
        # a language decoder's parameters, matrices and vectors, many of them of odd sizes
        dict(name="adamw_many_f32", op="adamw", tensors=148, elements=66_000_000, dtype="f32", bits=32),
        dict(name="adamw8_many_f32", op="adamw", tensors=148, elements=66_000_000, dtype="f32", bits=8),
        dict(name="adamw8_many_bf16", op="adamw", tensors=40, elements=50_000_000, dtype="bf16", bits=8),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("ce", "ce", "balance", "adamw"))
    dtype = rng.choice(("f32", "bf16"))
    if op == "ce":
        tokens, width = _log(rng, 1, 8192), _log(rng, 8, 1024)
        # in 32 bits the code heads' range: up to the largest codebook's work of the listed case
        classes = _log(rng, 64, 131072 if dtype == "bf16" else max(64, min(50257, (1 << 34) // (tokens * width))))
        return dict(op=op, tokens=tokens, width=width, classes=classes, dtype=dtype, grad=rng.random() < 0.7, ignored=rng.choice((0.0, 0.1, 0.4)))
    if op == "balance":
        classes = _log(rng, 2, 4096)
        return dict(op=op, rows=_log(rng, 1, (1 << 27) // classes), classes=classes, picks=rng.randint(1, min(8, classes)), dtype=dtype,
                    masked=rng.choice((0.0, 0.3)))
    tensors = _log(rng, 1, 160)
    return dict(op=op, tensors=tensors, elements=_log(rng, 64 * tensors, 66_000_000), dtype=dtype, bits=rng.choice((8, 32)))


def _sizes(case):
    """Elements of every tensor: every fourth a matrix, the others vectors of odd lengths; together about case["elements"]."""
    n = case["tensors"]
    small = [17 + 61 * (i % 13) for i in range(n)]
    big = [i for i in range(n) if i % 4 == 0]
    left = max(case["elements"] - sum(small), 0)
    return [small[i] + (left // len(big) + (i * 37) % 101 if i % 4 == 0 else 0) for i in range(n)]


def _views(flat, sizes, step=256):
    at, out = 0, []
    for n in sizes:
        out.append(flat[at:at + n])
        at += -(-n // step) * step
    return out


def prepare(case, seed):
    dev, dt = torch.device("cuda"), DTYPES[case["dtype"]]
    g = torch.Generator(device=dev).manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    uniform = lambda *s: torch.rand(*s, generator=g, device=dev)  # noqa: E731
    if case["op"] == "ce":
        T, H, V = case["tokens"], case["width"], case["classes"]
        h = normal(T, H).to(dt)                                            # behind a layer norm
        w = (normal(V, H) * (2.5 / math.sqrt(H))).to(dt)                   # logits of deviation 2.5
        y = (V ** uniform(T).double() - 1).long().clamp_(0, V - 1)         # words by their rank: the first ones are the frequent ones
        y = torch.where(uniform(T) < case["ignored"], torch.full_like(y, IGNORE), y)
        return dict(case=case, h=h.requires_grad_(case["grad"]), w=w.requires_grad_(case["grad"]), y=y)
    if case["op"] == "balance":
        T, E, K = case["rows"], case["classes"], case["picks"]
        s = normal(T, E)
        s += 1.5 * normal(E)                                               # some codes are used much more than others
        i = s.topk(K, dim=1).indices
        if case["masked"]:
            i = torch.where(uniform(T, K) < 0.05, torch.full_like(i, -1), i)   # dropped assignments
        m = uniform(T) >= case["masked"] if case["masked"] else None
        return dict(case=case, s=s.to(dt).requires_grad_(True), i=i.contiguous(), m=m)
    sizes = _sizes(case)
    total = sum(-(-n // 256) * 256 for n in sizes)
    p, gr = (0.05 * normal(total)).to(dt), (1e-3 * normal(total) * torch.exp(normal(total))).to(dt)
    m, v = 5e-4 * normal(total), (1e-3 * torch.exp(normal(total))) ** 2
    gaps = torch.ones(total, dtype=torch.bool, device=dev)
    for a in _views(gaps, sizes):
        a.fill_(False)
    for a in (p, gr, m, v):
        a.masked_fill_(gaps, 0)
    st = dict(case=case, sizes=sizes, p=p, g=gr, ps=_views(p, sizes), gs=_views(gr, sizes), step=137, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, wd=1e-2,
              seed=seed % (1 << 31))
    if case["bits"] == 32:
        return dict(st, m=m, v=v, ms=_views(m, sizes), vs=_views(v, sizes))
    for key, x in (("m", m), ("v", v.sqrt())):
        scale = x.view(-1, BLOCK).abs().amax(1) / TOP                      # a block holds one element of a tensor at least: not 0
        codes = (x.view(-1, BLOCK) / scale[:, None]).to(torch.float8_e4m3fn).view(-1)
        blocks = [-(-n // BLOCK) for n in sizes]
        st.update({key: codes, key + "_scale": scale, key + "s": list(zip(_views(codes, sizes), _views(scale, blocks, 1)))})
    return st


def run(state):
    return {"ce": _ce, "balance": _balance, "adamw": _adamw}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------ token cross entropy
def _ce(s):
    grad = s["case"]["grad"]
    if own:
        from causal_eeg_vae_amd import linear_cross_entropy
        loss = linear_cross_entropy(s["h"], s["w"], s["y"], ignore_index=IGNORE, reduction="mean" if grad else "none")
        return (loss.detach(),) + torch.autograd.grad(loss, (s["h"], s["w"])) if grad else loss
    h, w, y = s["h"].detach().float(), s["w"].detach().float(), s["y"]
    keep = y != IGNORE
    at = torch.where(keep, y, torch.zeros_like(y))[:, None]
    logits = h @ w.t()
    top = logits.amax(1, keepdim=True)
    p = (logits - top).exp_()
    total = p.sum(1, keepdim=True)
    loss = torch.where(keep, (top + total.log() - logits.gather(1, at))[:, 0], torch.zeros_like(top[:, 0]))
    if not grad:
        return loss
    del logits
    n = keep.sum().clamp(min=1)
    p /= total
    p.scatter_add_(1, at, torch.full_like(top, -1.0))
    p *= (keep / n)[:, None]
    return loss.sum() / n, (p @ w).to(s["h"].dtype), (p.t() @ h).to(s["w"].dtype)


# ------------------------------------------------------------------------------------------ balance loss
def _balance(s):
    if own:
        from causal_eeg_vae_amd import balance_loss
        loss, counts = balance_loss(s["s"], s["i"], mask=s["m"])
        return loss.detach(), counts, torch.autograd.grad(loss, s["s"])[0]
    x, idx = s["s"].detach().float(), s["i"]
    (T, E), K = x.shape, idx.shape[1]
    keep = torch.ones(T, dtype=torch.bool, device=x.device) if s["m"] is None else s["m"]
    n = keep.sum().clamp(min=1)
    slot = torch.where(keep[:, None] & (idx >= 0), idx, torch.full_like(idx, E)).reshape(-1)
    counts = torch.zeros(E + 1, dtype=torch.int64, device=x.device).scatter_add_(0, slot, torch.ones_like(slot))[:E]
    p = (x - x.amax(1, keepdim=True)).exp_()
    p *= (keep / p.sum(1))[:, None]
    f = counts.float() / (n * K)
    loss = E * (f * (p.sum(0) / n)).sum()
    ds = p * (f - (p * f).sum(1, keepdim=True)) * (E / n)      # rows of p that do not count are zero
    return loss, counts, ds.to(s["s"].dtype)


# ------------------------------------------------------------------------------------------ AdamW
def _adamw(s):
    """The plain forms step the whole buffers at once: what lies between two tensors is zero and stays so."""
    if own:
        from causal_eeg_vae_amd import adamw_step_
        adamw_step_(s["ps"], s["gs"], s["ms"], s["vs"], step=s["step"], lr=s["lr"], betas=s["betas"], eps=s["eps"], weight_decay=s["wd"], seed=s["seed"])
    elif s["case"]["bits"] == 32:
        _moved(s, s["m"].mul_(s["betas"][0]).add_(s["g"].float() * (1 - s["betas"][0])),
               s["v"].mul_(s["betas"][1]).add_(s["g"].float().square() * (1 - s["betas"][1])))
    else:
        _adamw8(s)
    if s["case"]["bits"] == 32:
        return s["p"], s["m"], s["v"]
    return s["p"], s["m"], s["m_scale"], s["v"], s["v_scale"]


def _moved(s, m, v):
    c1, c2 = 1 - s["betas"][0] ** s["step"], 1 - s["betas"][1] ** s["step"]
    by = m / (v.sqrt().div_(math.sqrt(c2)).add_(s["eps"]))
    s["p"].copy_((s["p"].float() * (1 - s["lr"] * s["wd"])).add_(by, alpha=-s["lr"] / c1))


def _low_high(a, c):
    """Low and high 32 bits of a * c, both below 2^32, in 64-bit integers."""
    low, high = a * (c & 0xFFFF), a * (c >> 16)
    whole = (low >> 16) + high                              # bits 16 and up of the product
    return ((whole << 16) | (low & 0xFFFF)) & 0xFFFFFFFF, whole >> 16


def _rounds(c, k0, k1, left):
    if left == 0:
        return c
    l0, h0 = _low_high(c[0], 0xD2511F53)
    l1, h1 = _low_high(c[2], 0xCD9E8D57)
    return _rounds([h1 ^ c[1] ^ k0, l1, h0 ^ c[3] ^ k1, l0], (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF, left - 1)


def _random_words(s):
    """Philox 4x32-10 with the seed as key: element i of a tensor takes word i % 4 of the counter (i / 4, tag, tensor)."""
    dev = s["p"].device
    room = torch.tensor([-(-n // BLOCK) * (BLOCK // 4) for n in s["sizes"]], device=dev)
    total = s["p"].numel() // 4
    tensor = torch.repeat_interleave(torch.arange(len(s["sizes"]), device=dev), room, output_size=total)
    q = torch.arange(total, device=dev) - torch.repeat_interleave(room.cumsum(0) - room, room, output_size=total)
    c = _rounds([q & 0xFFFFFFFF, q >> 32, torch.full_like(q, TAG), tensor], s["seed"] & 0xFFFFFFFF, s["seed"] >> 32, 10)
    return torch.stack(c, 1).view(-1)


def _held(x, r16, keep_positive):
    """x in 8 bits: e4m3 numbers times one scale a block, each rounded up with the probability of what rounding down leaves out."""
    x = x.view(-1, BLOCK)
    top = x.abs().amax(1)
    none = top < TINY
    scale = torch.where(none, torch.zeros_like(top), top / TOP)
    y = torch.where(none[:, None], torch.zeros_like(x), x.abs() / scale[:, None]).clamp_(max=TOP).view(-1)
    normal = ((y.view(torch.int32) + (r16 << 4)) >> 20) - (120 << 3)
    small = torch.floor(y * 512 + r16.float() / 65536).int()
    code = torch.where(y >= 2.0 ** -6, normal, small)
    if keep_positive:
        code = torch.where((y > 0) & (code == 0), torch.ones_like(code), code)
    code = code | (torch.signbit(x).view(-1).int() << 7)
    return code.to(torch.uint8).view(torch.float8_e4m3fn), scale


def _adamw8(s):
    b1, b2 = s["betas"]
    g = s["g"].float()
    wide = lambda q, scale: (q.float().view(-1, BLOCK) * scale[:, None]).view(-1)  # noqa: E731
    m = b1 * wide(s["m"], s["m_scale"]) + (1 - b1) * g
    u = wide(s["v"], s["v_scale"])
    v = b2 * (u * u) + (1 - b2) * (g * g)
    _moved(s, m, v)
    r = _random_words(s)
    for x, key, r16, positive in ((m, "m", r & 0xFFFF, False), (v.sqrt(), "v", r >> 16, True)):
        code, scale = _held(x, r16.int(), positive)
        s[key].copy_(code)
        s[key + "_scale"].copy_(scale)


# ------------------------------------------------------------------------------------------ work
def work(case):
    b = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "ce":
        T, H, V = case["tokens"], case["width"], case["classes"]
        if case["grad"]:
            return dict(bytes=2.0 * b * H * (T + V) + 8 * T + 4, flops=6.0 * T * H * V)
        return dict(bytes=1.0 * b * H * (T + V) + 8 * T + 4 * T, flops=2.0 * T * H * V)
    if case["op"] == "balance":
        T, E, K = case["rows"], case["classes"], case["picks"]
        return dict(bytes=2.0 * b * T * E + 8 * T * K + (T if case["masked"] else 0) + 8 * E + 4, flops=8.0 * T * E)
    n = sum(_sizes(case))
    held = 16 if case["bits"] == 32 else 4 + 16 / BLOCK
    return dict(bytes=1.0 * n * (3 * b + held), flops=20.0 * n)


# ------------------------------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "ce":
        return _exact_ce(s)
    if case["op"] == "balance":
        return _exact_balance(s)
    return _exact_adamw(s)


def _exact_ce(s):
    h, w, y = s["h"].detach().double(), s["w"].detach().double(), s["y"]
    rows = torch.nonzero(y != IGNORE)[:, 0]
    losses = torch.zeros(y.numel(), dtype=torch.float64, device=h.device)
    dh, dw = torch.zeros_like(h), torch.zeros_like(w)
    for at in rows.split(1024):
        z = h[at] @ w.t()
        lse = torch.logsumexp(z, 1)
        losses[at] = lse - z[torch.arange(at.numel(), device=z.device), y[at]]
        if s["case"]["grad"]:
            d = torch.exp(z - lse[:, None])
            d[torch.arange(at.numel(), device=z.device), y[at]] -= 1
            d /= rows.numel()
            dh[at] = d @ w
            dw += d.t() @ h[at]
    return (losses.sum() / max(rows.numel(), 1), dh, dw) if s["case"]["grad"] else losses


def _exact_balance(s):
    x, idx = s["s"].detach().double(), s["i"]
    rows = torch.arange(x.shape[0], device=x.device) if s["m"] is None else torch.nonzero(s["m"])[:, 0]
    E, n = x.shape[1], max(rows.numel(), 1)
    given = idx[rows].reshape(-1)
    counts = torch.bincount(given[given >= 0], minlength=E)
    p = torch.softmax(x[rows], 1)
    f = counts.double() / (n * idx.shape[1])
    ds = torch.zeros_like(x)
    ds[rows] = p * (f - (p @ f)[:, None]) * E / n
    return E * torch.dot(f, p.sum(0) / n), counts, ds


def _exact_words(n, seed, tensor):
    mask = np.uint64(0xFFFFFFFF)
    q = np.arange(-(-n // 4), dtype=np.uint64)
    c = [q & mask, q >> np.uint64(32), np.full_like(q, TAG), np.full_like(q, tensor)]
    k = [np.uint64(seed & 0xFFFFFFFF), np.uint64(seed >> 32)]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ k[0], b & mask, (a >> np.uint64(32)) ^ c[3] ^ k[1], a & mask]
        k = [(k[0] + np.uint64(0x9E3779B9)) & mask, (k[1] + np.uint64(0xBB67AE85)) & mask]
    return np.stack(c, 1).reshape(-1)[:n].astype(np.int64)


def _exact_adamw(s):
    b1, b2 = s["betas"]
    c1, c2 = 1 - b1 ** s["step"], 1 - b2 ** s["step"]
    small = s["case"]["bits"] == 8
    p, m, v = (s[k].double() for k in "pmv")
    scales = {k: s[k + "_scale"].double() for k in "mv"} if small else {}
    places = list(zip(*(_views(x, s["sizes"]) for x in (p, s["g"].double(), m, v))))
    blocks = [-(-n // BLOCK) for n in s["sizes"]]
    held = list(zip(*(_views(scales[k], blocks, 1) for k in "mv"))) if small else [None] * len(places)
    # the numbers of e4m3 that are not negative, in order: a magnitude lies between two neighbours
    grid = torch.arange(127, dtype=torch.uint8, device=p.device).view(torch.float8_e4m3fn).double()
    for j, ((pj, gj, mj, vj), sc) in enumerate(zip(places, held)):
        n = pj.numel()
        if small:
            mj_, uj_ = mj * sc[0].repeat_interleave(BLOCK)[:n], vj * sc[1].repeat_interleave(BLOCK)[:n]
            vj_ = uj_ ** 2
        else:
            mj_, vj_ = mj, vj
        mn, vn = mj_ + (1 - b1) * (gj - mj_), vj_ + (1 - b2) * (gj ** 2 - vj_)
        pj -= s["lr"] * (s["wd"] * pj + (mn / c1) / ((vn / c2).sqrt() + s["eps"]))
        if not small:
            mj.copy_(mn)
            vj.copy_(vn)
            continue
        words = torch.from_numpy(_exact_words(n, s["seed"], j)).to(p.device)
        for x, q, scale, r in ((mn, mj, sc[0], words % 65536), (vn.sqrt(), vj, sc[1], words // 65536)):
            top = torch.nn.functional.pad(x.abs(), (0, -n % BLOCK)).view(-1, BLOCK).amax(1)
            scale.copy_(torch.where(top < TINY, torch.zeros_like(top), top / TOP))
            wide = scale.repeat_interleave(BLOCK)[:n]
            y = torch.where(wide > 0, x.abs() / wide, torch.zeros_like(x)).clamp(max=TOP)
            low = (torch.searchsorted(grid, y, right=True) - 1).clamp(0, 125)
            up = (y - grid[low]) / (grid[low + 1] - grid[low]) + r.double() / 65536 >= 1
            code = low + up.long()
            if q is vj:
                code = torch.where((y > 0) & (code == 0), torch.ones_like(code), code)
            q.copy_(grid[code] * torch.where(x < 0, -1.0, 1.0))
    if not small:
        return p, m, v
    return p, m, scales["m"], v, scales["v"]
