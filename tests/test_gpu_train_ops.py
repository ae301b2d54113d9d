"""GPU: the cross entropy, the balance loss and AdamW together, as a training step uses them, and through the models and the trainer."""
import os

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


class _Headline(torch.nn.Module):
    """A small conditional model around the quantiser: states -> latent -> code -> token states, with a vocabulary head."""

    def __init__(self, width=64, latent=16, codes=32, classes=500):
        super().__init__()
        from causal_eeg_vae_amd import VectorQuantizer
        self.to_latent = torch.nn.Linear(width, latent)
        self.vq = VectorQuantizer(codes, latent, 0.25, return_one_hot=False)
        self.back = torch.nn.Linear(latent, width)
        self.head = torch.nn.Parameter(torch.randn(classes, width) / width ** 0.5)
        torch.nn.init.normal_(self.vq.embedding.weight, std=0.5)


def _step(model, x, target):
    from causal_eeg_vae_amd import linear_cross_entropy
    z = model.to_latent(x)
    vq_loss, z_q, _, _, idx = model.vq(z)
    bal, counts = model.vq.balance(z, idx, temperature=2.0)
    rec = linear_cross_entropy(torch.tanh(model.back(z_q)) + x, model.head, target, ignore_index=-1)
    return rec + vq_loss + 0.1 * bal, idx, counts


def _step64(model, x, target, idx):
    """The same loss in 64 bits with the codes given; straight through the quantiser."""
    z = model.to_latent(x)
    w = model.vq.embedding.weight
    e = w[idx[:, 0]]
    vq_loss = ((e.detach() - z) ** 2).mean() + 0.25 * ((e - z.detach()) ** 2).mean()   # beta on the codebook's term, as scripts/quantizer.py:57-58
    z_q = z + (e - z).detach()
    f = torch.bincount(idx[:, 0], minlength=w.shape[0]).double() / z.shape[0]
    p = torch.softmax(-((z[:, None] - w[None]) ** 2).sum(-1) / 2.0, 1)
    logits = (torch.tanh(model.back(z_q)) + x) @ model.head.t()
    return torch.nn.functional.cross_entropy(logits, target, ignore_index=-1) + vq_loss + 0.1 * w.shape[0] * (f * p.mean(0)).sum()


def test_a_step_of_all_three():
    """Loss and gradients against 64 bits (rtol 1e-5 as every parity test of this package, atol 1e-5 of the tensor's largest), then the update."""
    import copy
    from causal_eeg_vae_amd import AdamW
    torch.manual_seed(0)
    model = _Headline().cuda()
    x = torch.randn(120, 64, device="cuda")
    target = torch.randint(0, 500, (120,), device="cuda")
    target[::5] = -1
    opt = AdamW(model.parameters(), lr=1e-2, state_bits=8, min_8bit_size=1000)
    for _ in range(3):
        ref = copy.deepcopy(model).double()
        before = [p.detach().double() for p in model.parameters()]
        opt.zero_grad()
        loss, idx, counts = _step(model, x, target)
        loss.backward()
        want = _step64(ref, x.double(), target, idx)
        want.backward()
        assert abs(float(loss.detach()) - float(want.detach())) <= 1e-5 * abs(float(want.detach()))
        assert torch.equal(counts, torch.bincount(idx[:, 0], minlength=32))
        for a, b in zip(model.parameters(), ref.parameters()):
            assert float((a.grad.double() - b.grad).abs().max()) <= 1e-5 * float(b.grad.abs().max())
        opt.step()
        for a, b in zip(model.parameters(), before):   # every element moved by about lr at most, none stayed where its gradient was not zero
            moved = (a.detach().double() - b * (1 - 1e-4)).abs()
            assert float(moved.max()) <= 1e-2 * 4 and bool((moved[a.grad != 0] > 0).all())


def _graph(N, E, seed):
    from causal_eeg_vae_amd import EventGraph
    from causal_eeg_vae_amd.synth import synth_event_graph
    return EventGraph(synth_event_graph(N, E, seed=seed).cuda(), N)


@pytest.mark.parametrize("negatives", ["sigma", "uniform"])
def test_balance_in_the_graph_model(negatives):
    """VGAEVQ(balance=w): the loss grows by w times the balance loss, and its gradient is that of the two parts."""
    from causal_eeg_vae_amd import VGAEVQ
    N = 1500
    graph, x = _graph(N, 12000, 1), torch.randn(N, 16, device="cuda")
    eps = torch.randn(N, 16, device="cuda")
    grads, losses, auxs = [], [], []
    for w in (0.0, 0.5):
        torch.manual_seed(3)
        model = VGAEVQ(16, 16, 32, 0.25, negatives=negatives, balance=w, balance_temperature=0.7).cuda()
        loss, aux = model(x, graph, step=2, eps=eps)
        loss.backward()
        grads.append({n: p.grad.double() for n, p in model.named_parameters()}), losses.append(loss.detach()), auxs.append(aux)
    assert "balance" not in auxs[0] and torch.equal(auxs[0]["idx"], auxs[1]["idx"])
    bal = auxs[1]["balance"].detach()
    assert torch.equal(losses[1], losses[0] + 0.5 * bal)
    assert torch.equal(auxs[1]["code_counts"], torch.bincount(auxs[1]["idx"].view(-1), minlength=32))
    torch.manual_seed(3)
    model = VGAEVQ(16, 16, 32, 0.25, negatives=negatives, balance=0.5, balance_temperature=0.7).cuda()
    _, aux = model(x, graph, step=2, eps=eps)
    z, w = aux["z"].detach().double(), model.vector_quantization.embedding.weight.detach().double().requires_grad_(True)
    f = aux["code_counts"].double() / N
    p = torch.softmax(-((z[:, None] - w[None]) ** 2).sum(-1) / 0.7, 1)
    want = 32 * (f * p.mean(0)).sum()
    (dw,) = torch.autograd.grad(want, w)
    assert abs(float(bal) - float(want.detach())) <= 1e-5 * float(want.detach())
    name = "vector_quantization.embedding.weight"
    diff = grads[1][name] - grads[0][name]
    assert float((diff - 0.5 * dw).abs().max()) <= 1e-5 * float(grads[1][name].abs().max())
    # the encoder is reached too
    assert any(float((grads[1][n] - grads[0][n]).abs().max()) > 0 for n in grads[0] if n != name)


@pytest.mark.parametrize("bits", [32, 8])
def test_trainer_with_adamw(bits):
    from causal_eeg_vae_amd import AdamW, VGAEVQ
    from causal_eeg_vae_amd.trainer import Trainer
    N = 1200
    graph, x = _graph(N, 9000, 2), torch.randn(N, 64, device="cuda")
    runs = []
    for _ in range(2):
        torch.manual_seed(1)
        model = VGAEVQ(64, 64, 64, 0.25, balance=0.01).cuda()
        trainer = Trainer(model, lr=1e-2, optimizer="adamw", weight_decay=0.0, state_bits=bits)
        assert isinstance(trainer.opt, AdamW)
        runs.append([float(trainer.step(x, graph)[0]) for _ in range(5)])
        trainer.end_epoch(runs[-1][-1])
    assert runs[0] == runs[1] and all(v == v for v in runs[0])
    held = [isinstance(trainer.opt.state[p]["exp_avg"], tuple) for p in model.parameters()]
    assert any(held) == (bits == 8)


def test_training_from_csv_with_all_three(tmp_path):
    from causal_eeg_vae_amd.run_csv import main
    nodes, edges = tmp_path / "nodes.csv", tmp_path / "edges.csv"
    _write_csv(nodes, edges)
    assert main([str(nodes), str(edges), "--epochs", "1", "--steps-per-epoch", "2", "--optimizer", "adamw", "--state-bits", "8", "--balance", "0.1"]) == 0


def _write_csv(nodes, edges):
    import numpy as np
    rng = np.random.default_rng(0)
    with open(nodes, "w") as f:
        f.write("title,text,publish_date,url,id\n")
        for k in range(40):
            f.write(f"t{k},words {k},2020-01-{1 + k % 28:02d},u{k},{k}\n")
    with open(edges, "w") as f:
        f.write("old_id,new_id,entity,entity_type,date_diff\n")
        for _ in range(200):
            a, b = sorted(rng.choice(40, 2, replace=False))
            f.write(f"{a},{b},e,ORG,1\n")


def test_two_graphs_with_their_own_workspaces():
    """Two captured graphs of the losses, replayed in turn and then at once on two streams: each keeps its results."""
    from causal_eeg_vae_amd import balance_loss, linear_cross_entropy
    made = []
    for k in range(2):
        g = torch.Generator(device="cuda").manual_seed(k)
        h = torch.randn(150 + 70 * k, 64, generator=g, device="cuda").bfloat16().requires_grad_(True)
        w = (torch.randn(900 + 300 * k, 64, generator=g, device="cuda") / 8).bfloat16().requires_grad_(True)
        y = torch.randint(0, 900, (150 + 70 * k,), generator=g, device="cuda")
        s = torch.randn(150 + 70 * k, 48, generator=g, device="cuda").requires_grad_(True)

        def both(h=h, w=w, y=y, s=s):
            loss = linear_cross_entropy(h, w, y)
            bal, counts = balance_loss(s, y % 48)
            return [loss.detach(), bal.detach(), counts] + list(torch.autograd.grad(loss + bal, (h, w, s)))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            both()
        torch.cuda.current_stream().wait_stream(side)
        want = both()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = both()
        made.append((graph, out, want, both))   # a graph reads its inputs again: they are kept with it
    streams = [torch.cuda.Stream() for _ in made]
    for turn in range(3):
        for (graph, out, *_), st in zip(made, streams):
            for t in out:
                t.zero_()
            torch.cuda.synchronize()
        for (graph, *_), st in zip(made, streams):
            if turn == 0:
                graph.replay()
            else:
                with torch.cuda.stream(st):
                    graph.replay()
        torch.cuda.synchronize()
        for _, out, want, _ in made:
            for a, b in zip(out, want):
                assert torch.equal(a, b)
