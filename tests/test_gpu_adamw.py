"""GPU: adamw_step_ and AdamW (ceeg_adamw_step) against the formula in 64 bits, and the 8-bit moments against a restatement of their rounding in numpy.

Bounds, with u = 2^-24: m and v are two products and a sum of fp32 numbers (3 u of the magnitudes); the update is m's error, a root, two
products and a division (8 u of it) and what an error of m left in a difference is worth; p adds 2 u of itself, a bf16 parameter half a step (2^-8)."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HYPER = dict(step=7, lr=2e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)


def _tensors(sizes, dtype, seed=0, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda n: torch.randn(n, generator=g, device="cuda")  # noqa: E731
    p = [rnd(n).to(dtype) for n in sizes]
    gr = [(rnd(n) * torch.exp(spread * rnd(n))).to(dtype) for n in sizes]
    return p, gr, [rnd(n) * 0.3 for n in sizes], [rnd(n) ** 2 for n in sizes]


def _formula(p, g, m, v, step, lr, betas, eps, weight_decay):
    p, g, m, v = (x.double() for x in (p, g, m, v))
    m1 = betas[0] * m + (1 - betas[0]) * g
    v1 = betas[1] * v + (1 - betas[1]) * g * g
    den = (v1 / (1 - betas[1] ** step)).sqrt() + eps
    up = lr / (1 - betas[0] ** step) / den
    e_m = 3 * U * (betas[0] * m.abs() + (1 - betas[0]) * g.abs())
    p1 = p * (1 - lr * weight_decay) - up * m1
    return p1, m1, v1, e_m, 3 * U * v1, 4 * U * p.abs() + up * (e_m + 10 * U * m1.abs()) + 1e-42


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("sizes", [[1], [3, 0, 255, 256, 257, 1024, 1025], [4097, 5], [1 + 13 * i for i in range(130)], [70001, 0]], ids=str)
def test_32_bit_moments(sizes, dtype):
    from causal_eeg_vae_amd import adamw_step_
    p, g, m, v = _tensors(sizes, dtype)
    want = [_formula(*x, **HYPER) for x in zip(p, g, m, v)]
    assert adamw_step_(p, g, m, v, **HYPER) is None
    for a, b, c, (p1, m1, v1, e_m, e_v, e_p) in zip(p, m, v, want):
        assert bool(((b.double() - m1).abs() <= e_m + 1e-45).all()) and bool(((c.double() - v1).abs() <= e_v + 1e-45).all())
        half = 2.0 ** -8 * p1.abs() if dtype == torch.bfloat16 else 0.0
        assert bool(((a.double() - p1).abs() <= e_p + half).all())


def test_large_lists_take_the_wide_workgroups():
    """From 2^23 elements a workgroup takes four times as many: the same numbers as the same tensors one by one."""
    from causal_eeg_vae_amd import adamw_step_
    sizes = [(1 << 23) + 1001, 4095, 77]
    a, b = _tensors(sizes, torch.float32, seed=4), _tensors(sizes, torch.float32, seed=4)
    adamw_step_(*a, **HYPER)
    for j in range(3):
        adamw_step_(*[x[j].split(1 << 20) for x in b], **HYPER)
    for x, y in zip(a, b):
        assert all(torch.equal(s, t) for s, t in zip(x, y))


def _philox_words(n, seed, tensor):
    mask = np.uint64(0xFFFFFFFF)
    q = np.arange(-(-n // 4), dtype=np.uint64)
    c = [q & mask, q >> np.uint64(32), np.full_like(q, 0x41444D57), np.full_like(q, tensor)]
    k = [np.uint64(seed & 0xFFFFFFFF), np.uint64(seed >> 32)]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ k[0], b & mask, (a >> np.uint64(32)) ^ c[3] ^ k[1], a & mask]
        k = [(k[0] + np.uint64(0x9E3779B9)) & mask, (k[1] + np.uint64(0xBB67AE85)) & mask]
    return np.stack(c, 1).reshape(-1)[:n].astype(np.int64)


GRID = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).float().numpy()   # the numbers of e4m3 that are not negative


def _held(x, r16, second):
    """x (fp32) in 8 bits, operation by operation in fp32: (codes, scales)."""
    codes, scales = np.empty(x.size, np.uint8), []
    for b in range(0, x.size, 256):
        y, r = x[b:b + 256], r16[b:b + 256].astype(np.float32)
        fine = np.abs(y)[np.isfinite(y)]
        top = fine.max() if fine.size else np.float32(0)
        scale = np.float32(0) if top < 2.0 ** -100 else np.float32(top * (np.float32(1) / np.float32(448)))
        scales.append(scale)
        z = np.minimum(np.abs(y) / scale, np.float32(448)) if scale > 0 else np.zeros_like(y)
        z = np.where(np.isfinite(y), z, np.float32(0))
        c = np.clip(np.searchsorted(GRID, z, side="right") - 1, 0, 126)
        low = GRID[c]
        step = (GRID[np.minimum(c + 1, 126)] - low).astype(np.float32)
        step = np.where(step == 0, np.float32(32), step)
        share = (z - low) / step
        if second:
            share = share * (z + low) / (low + low + step)
        c = c + (share * np.float32(65536) + r >= 65536)
        if second:
            c = np.where((z > 0) & (c == 0), 1, c)
        c = np.where(np.isfinite(y), c, 127)
        codes[b:b + 256] = c | (np.signbit(y) << 7)
    return codes, np.array(scales, np.float32)


def _states(values):
    """8-bit states near given fp32 values."""
    from causal_eeg_vae_amd.optim import BLOCK, block_state
    out = []
    for x in values:
        q, s = block_state(x)
        pad = torch.nn.functional.pad(x, (0, -x.numel() % BLOCK)).view(-1, BLOCK)
        s.copy_(pad.abs().amax(1) / 448)
        q.copy_((pad / s.clamp(min=1e-30)[:, None]).view(-1)[:x.numel()].to(torch.float8_e4m3fn))
        out.append((q, s))
    return out


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("sizes", [[1], [3, 0, 255, 256, 257, 1024, 1025], [5000, 2], [40 + i for i in range(70)]], ids=str)
def test_8_bit_moments_bit_for_bit(sizes, dtype):
    from causal_eeg_vae_amd import adamw_step_
    from causal_eeg_vae_amd.optim import block_values
    p, g, m, v = _tensors(sizes, dtype, spread=3.0)      # magnitudes over the whole range of a block
    m, v = _states(m), _states([x.sqrt() for x in v])
    seed = 0x123456789ABCDEF
    mf, vf = [block_values(x) for x in m], [block_values(x, square=True) for x in v]
    want = [_formula(*x, **HYPER) for x in zip(p, g, mf, vf)]
    b1, b2 = (np.float32(b) for b in HYPER["betas"])
    o1, o2 = (np.float32(1 - b) for b in HYPER["betas"])
    expect = []
    for j, n in enumerate(sizes):
        gf, a, b = (x.float().cpu().numpy() for x in (g[j], mf[j], vf[j]))
        w = _philox_words(n, seed, j)
        expect.append((_held(b1 * a + o1 * gf, w & 0xFFFF, False), _held(np.sqrt(b2 * b + o2 * (gf * gf)), w >> 16, True)))
    adamw_step_(p, g, m, v, seed=seed, **HYPER)
    for j, n in enumerate(sizes):
        for (codes, scales), (c, s) in zip((m[j], v[j]), expect[j]):
            np.testing.assert_array_equal(codes.view(torch.uint8).cpu().numpy(), c, err_msg=f"tensor {j}")
            np.testing.assert_array_equal(scales.cpu().numpy(), s if n else scales.cpu().numpy())
        p1, _, _, _, _, e_p = want[j]
        half = 2.0 ** -8 * p1.abs() if dtype == torch.bfloat16 else 0.0
        assert bool(((p[j].double() - p1).abs() <= e_p + half).all())


def test_8_bit_moments_follow_a_constant_gradient():
    """With 1 - b2 = 2^-7 a step moves v by less than a tenth of an 8-bit step; the rounding keeps the expectation, so the mean over n elements that
    start at the same v follows b2^t v0 + (1 - b2^t) g^2.  A rounding up happens with probability c / s (change c, step s of v <= 0.27 v), so its
    variance is at most c s <= (1 - b2) max(g^2, v) 0.27 v a step; over t <= 200 steps, for the mean of n = 65536: 6 deviations are 0.02 of v's range."""
    from causal_eeg_vae_amd import adamw_step_
    from causal_eeg_vae_amd.optim import block_state, block_values
    n, b2 = 1 << 16, 1 - 2.0 ** -7
    for v0, gr in ((1.0, 0.25), (0.0625, 1.0)):
        p, g = [torch.zeros(n, device="cuda")], [torch.full((n,), gr, device="cuda")]
        # one element of each block holds the scale still
        m, v = [block_state(p[0])], _states([torch.full((n,), v0 ** 0.5, device="cuda")])
        g[0][::256] = max(v0, gr * gr) ** 0.5
        v[0][0].view(-1)[::256] = 448.0
        v[0][1].fill_(max(v0, gr * gr) ** 0.5 / 448)
        inside = torch.arange(n, device="cuda") % 256 != 0
        v[0][0][inside] = torch.tensor(v0 ** 0.5 / float(v[0][1][0]), device="cuda").to(torch.float8_e4m3fn)
        start = float(block_values(v[0], square=True)[inside].double().mean())
        mids = []
        for t in range(1, 201):
            adamw_step_(p, g, m, v, step=t, betas=(0.9, b2), lr=1e-3, seed=1000 + t)
            if t % 50 == 0:
                mean = float(block_values(v[0], square=True)[inside].double().mean())
                want = b2 ** t * start + (1 - b2 ** t) * gr * gr
                assert abs(mean - want) <= 0.02 * max(v0, gr * gr), (t, mean, want)
                mids.append(float(block_values(m[0])[inside].double().mean()))
        assert abs(mids[-1] - gr) <= 0.02 * gr * 3


def test_gradients_that_are_not_finite_stay_where_they_are():
    from causal_eeg_vae_amd import adamw_step_
    from causal_eeg_vae_amd.optim import block_values
    for bits in (32, 8):
        p, g, m, v = _tensors([600], torch.float32)
        if bits == 8:
            m, v = _states(m), _states([x.sqrt() for x in v])
        clean = [[x.clone() for x in p], [x.clone() for x in g]] + [[(a.clone(), b.clone()) for a, b in z] if bits == 8 else [a.clone() for a in z] for z in (m, v)]
        adamw_step_(*clean, seed=3, **HYPER)
        bad = torch.tensor([5, 300, 599], device="cuda")
        # the scale of a block is its largest finite magnitude: an element that does not set it goes, the others stay as they are
        g[0][bad] = torch.tensor([float("nan"), float("inf"), float("-inf")], device="cuda")
        adamw_step_(p, g, m, v, seed=3, **HYPER)
        ok = torch.ones(600, dtype=torch.bool, device="cuda")
        ok[bad] = False
        assert torch.equal(p[0][ok], clean[0][0][ok]) and not bool(torch.isfinite(p[0][bad]).any() & torch.isnan(p[0][bad[0]]).logical_not())
        if bits == 8:
            x = block_values(m[0])
            assert bool(torch.isnan(x[bad]).all()) and bool(torch.isfinite(x[ok]).all())


def test_zero_moments_and_zero_gradients():
    from causal_eeg_vae_amd import adamw_step_
    from causal_eeg_vae_amd.optim import block_state
    p = [torch.ones(700, device="cuda")]
    st = [[block_state(p[0])], [block_state(p[0])]]
    adamw_step_(p, [torch.zeros(700, device="cuda")], *st, step=1, lr=0.5, weight_decay=0.5)
    assert torch.equal(p[0], torch.full((700,), 0.75, device="cuda"))
    assert not any(bool(t.view(torch.uint8).any()) for q in st for t in q[0])


@pytest.mark.parametrize("bits", [32, 8])
def test_unaligned_views(bits):
    """Views of one flat buffer at odd offsets: the numbers of the separate tensors, and nothing beside the views is touched."""
    from causal_eeg_vae_amd import adamw_step_
    sizes, at = [301, 77, 1030], [3, 310, 391]
    for dtype in (torch.float32, torch.bfloat16):
        p, g, m, v = _tensors(sizes, dtype, seed=8)
        if bits == 8:
            m, v = _states(m), _states([x.sqrt() for x in v])
        flat = []
        for xs in (p, g, [x[0] if bits == 8 else x for x in m], [x[0] if bits == 8 else x for x in v]):
            f = torch.full((1500,), 2.0, device="cuda").to(xs[0].dtype)
            for x, o in zip(xs, at):
                f[o:o + x.numel()] = x
            flat.append(f)
        views = [[f[o:o + n] for o, n in zip(at, sizes)] for f in flat]
        if bits == 8:
            views[2] = [(q, s[1].clone()) for q, s in zip(views[2], m)]
            views[3] = [(q, s[1].clone()) for q, s in zip(views[3], v)]
        adamw_step_(p, g, m, v, seed=2, **HYPER)
        adamw_step_(*views, seed=2, **HYPER)
        inside = torch.zeros(1500, dtype=torch.bool, device="cuda")
        for o, n in zip(at, sizes):
            inside[o:o + n] = True
        for f in flat:
            assert bool((f[~inside].float() == 2.0).all())
        for j in range(3):
            assert torch.equal(p[j], views[0][j])
            for a, b in ((m[j], views[2][j]), (v[j], views[3][j])):
                for x, y in zip(a, b) if bits == 8 else ((a, b),):
                    assert torch.equal(x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x, y.view(torch.uint8) if y.dtype == torch.float8_e4m3fn else y)


def _model(dtype=torch.float32):
    torch.manual_seed(0)
    return torch.nn.Sequential(torch.nn.Linear(40, 300), torch.nn.Tanh(), torch.nn.Linear(300, 7)).to("cuda", dtype)


def test_optimizer_against_torch():
    """Ten steps of the class against torch.optim.AdamW in fp64 on the same gradients; each step is off by 2^-18 of lr (8 u of the update and u of p)."""
    from causal_eeg_vae_amd import AdamW
    a = _model()
    b = _model().double()
    b.load_state_dict(a.state_dict())
    oa = AdamW([dict(params=a[0].parameters(), lr=3e-3), dict(params=a[2].parameters(), weight_decay=0.3)])
    ob = torch.optim.AdamW([dict(params=b[0].parameters(), lr=3e-3), dict(params=b[2].parameters(), weight_decay=0.3)])
    g = torch.Generator(device="cuda").manual_seed(2)
    for _ in range(10):
        for x, y in zip(a.parameters(), b.parameters()):
            x.grad = torch.randn(x.shape, generator=g, device="cuda")
            y.grad = x.grad.double()
        oa.step(), ob.step()
    for x, y in zip(a.parameters(), b.parameters()):
        assert float((x.double() - y).abs().max()) <= 10 * (3e-3 * 2.0 ** -18 + 2 * U)


def test_optimizer_with_8_bit_states_and_its_state_dict():
    from causal_eeg_vae_amd import AdamW
    runs = []
    for resume in (False, True):
        model = _model()
        opt = AdamW(model.parameters(), state_bits=8, min_8bit_size=300, seed=5)
        g = torch.Generator(device="cuda").manual_seed(2)
        for k in range(6):
            for x in model.parameters():
                x.grad = torch.randn(x.shape, generator=g, device="cuda")
            opt.step()
            if resume and k == 2:
                saved = {n: t.clone() for n, t in model.state_dict().items()}, opt.state_dict()
                model = _model()
                model.load_state_dict(saved[0])
                opt = AdamW(model.parameters(), state_bits=8, min_8bit_size=300, seed=5)
                opt.load_state_dict(saved[1])
        st = [opt.state[x]["exp_avg"] for x in model.parameters()]
        assert [isinstance(s, tuple) for s in st] == [True, True, True, False]     # 12000, 300, 2100 and 7 elements
        assert st[0][0].dtype == torch.float8_e4m3fn and st[0][1].dtype == torch.float32
        runs.append([x.detach().clone() for x in model.parameters()])
    for x, y in zip(*runs):
        assert torch.equal(x, y)


@pytest.mark.parametrize("bits", [32, 8])
def test_step_captured_into_a_graph(bits):
    """Replays of a captured step equal eager steps: the count and the learning rate are read on the device."""
    from causal_eeg_vae_amd import AdamW
    models, opts = [_model() for _ in range(2)], []
    for k, model in enumerate(models):
        lr = torch.tensor(1e-2, device="cuda")
        opts.append(AdamW(model.parameters(), lr=lr, state_bits=bits, seed=9, capturable=True))
        for x in model.parameters():
            x.grad = torch.zeros_like(x)
    grads = [[torch.randn(x.shape, device="cuda") for x in models[0].parameters()] for _ in range(6)]

    def feed(model, k):
        for x, gr in zip(model.parameters(), grads[k]):
            x.grad.copy_(gr)

    for model, opt in zip(models, opts):
        feed(model, 0)
        opt.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opts[0].step()
    for k in range(1, 6):
        for opt in opts:
            opt.param_groups[0]["lr"].fill_(1e-2 / k)
        feed(models[0], k), feed(models[1], k)
        graph.replay()
        opts[1].step()
        torch.cuda.synchronize()
        for x, y in zip(models[0].parameters(), models[1].parameters()):
            assert torch.equal(x, y), k


def test_captures_that_would_replay_wrongly_are_refused():
    from causal_eeg_vae_amd import AdamW, adamw_step_
    p = [torch.ones(10, device="cuda")]
    x = [torch.zeros(10, device="cuda") for _ in range(3)]
    model = _model()
    for q in model.parameters():
        q.grad = torch.zeros_like(q)
    opt = AdamW(model.parameters(), capturable=True)
    for error, call in ((ValueError, lambda: adamw_step_(p, x[:1], x[1:2], x[2:], step=3)), (RuntimeError, opt.step)):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            p[0].mul_(1.0)
            with pytest.raises(error):
                call()
    assert torch.equal(p[0], torch.ones(10, device="cuda"))


def test_a_graph_that_saved_a_parameter_notices():
    from causal_eeg_vae_amd import adamw_step_
    w = torch.ones(8, device="cuda", requires_grad=True)
    loss = (w * w).sum()
    x = [torch.zeros(8, device="cuda") for _ in range(3)]
    adamw_step_([w], x[:1], x[1:2], x[2:], step=1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_on_another_stream():
    from causal_eeg_vae_amd import adamw_step_
    a, b = _tensors([70001, 300], torch.float32, seed=4), _tensors([70001, 300], torch.float32, seed=4)
    adamw_step_(*a, **HYPER)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        b[1][0].mul_(1.0)        # the step follows what its own stream holds
        adamw_step_(*b, **HYPER)
    s.synchronize()
    for x, y in zip(a, b):
        assert all(torch.equal(s, t) for s, t in zip(x, y))


def test_capturable_equals_plain():
    """The count on the device and the count on the host give the same stream of random numbers; the factors differ by a rounding."""
    from causal_eeg_vae_amd import AdamW
    out = []
    for capturable in (False, True):
        model = _model()
        opt = AdamW(model.parameters(), state_bits=8, min_8bit_size=1, seed=3, capturable=capturable)
        g = torch.Generator(device="cuda").manual_seed(2)
        for _ in range(3):
            for x in model.parameters():
                x.grad = torch.randn(x.shape, generator=g, device="cuda")
            opt.step()
        out.append([x.detach() for x in model.parameters()] + [opt.state[x]["exp_avg"][0].view(torch.uint8) for x in model.parameters()])
    for x, y in zip(*out):
        assert torch.equal(x, y) if x.dtype == torch.uint8 else float((x - y).abs().max()) <= 1e-7


def test_mixed_types_and_missing_gradients():
    from causal_eeg_vae_amd import AdamW
    a = torch.nn.Parameter(torch.ones(5000, device="cuda"))
    b = torch.nn.Parameter(torch.ones(5000, device="cuda", dtype=torch.bfloat16))
    c = torch.nn.Parameter(torch.ones(10, device="cuda"))
    opt = AdamW([a, b, c], lr=0.5, weight_decay=0.0, state_bits=8)
    a.grad = torch.ones(100, 50, device="cuda").t().reshape(-1)
    b.grad = torch.full((5000,), -2.0, device="cuda", dtype=torch.bfloat16)
    opt.step()
    assert float((a.detach() - 0.5).abs().max()) <= 1e-6 and bool((b.detach() == 1.5).all()) and bool((c.detach() == 1.0).all()) and not opt.state[c]


@pytest.mark.parametrize("capturable", [False, True])
def test_each_parameter_counts_its_own_steps(capturable):
    """Gradients that come late or stay away: the bias corrections are those of the parameter's own steps, through a saved state as well.
    Rounding: about 8 operations of half a step each on numbers below 2 in every one of 6 steps of at most 0.1."""
    from causal_eeg_vae_amd import AdamW
    mine = [torch.nn.Parameter(torch.ones(300, device="cuda")) for _ in range(3)]
    ref = [torch.nn.Parameter(torch.ones(300, dtype=torch.float64)) for _ in range(3)]
    new = lambda: AdamW(mine, lr=0.1, capturable=capturable)  # noqa: E731
    a, b = new(), torch.optim.AdamW(ref, lr=0.1)
    g = torch.Generator().manual_seed(5)
    for k, on in enumerate(((0,), (0, 1), (0, 1, 2), (1, 2), (0, 1, 2), (2,))):
        for j in range(3):
            grad = torch.randn(300, generator=g)
            mine[j].grad, ref[j].grad = (grad.cuda(), grad.double()) if j in on else (None, None)
        a.step()
        b.step()
        if k == 3:
            state = a.state_dict()
            a = new()
            a.load_state_dict(state)
    for x, y in zip(mine, ref):
        assert float((x.detach().cpu().double() - y.detach()).abs().max()) <= 6 * 8 * 2.0 ** -24
    assert [int(a.state[x]["step"]) for x in mine] == [4, 4, 4]


def test_a_captured_step_takes_the_parameters_of_the_one_before():
    from causal_eeg_vae_amd import AdamW
    p = [torch.nn.Parameter(torch.ones(10, device="cuda")) for _ in range(2)]
    opt = AdamW(p, capturable=True)
    for x in p:
        x.grad = torch.ones_like(x)
    opt.step()
    p[1].grad = None
    before = [x.detach().clone() for x in p]
    work = torch.zeros(4, device="cuda")
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        work.add_(1.0)
        with pytest.raises(RuntimeError, match="parameters of the step before"):
            opt.step()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(p, before))
