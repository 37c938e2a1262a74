"""The framework's own paths over the training / serving operators on a real
MI355X: value nets of any hidden size (forward and as search leaves), the
trainer with clipping and fused layers, and a policy step over the option rows
of searched trees.  Bounds as in test_gpu_ops.py."""
import copy
import math

import numpy as np
import pytest
import torch

from citadels_self_play_amd import models, ops, train

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def chain_bound(net, x):
    """64-bit logits of the folded layers and how far fp32 sums of them can be: each layer adds (K + 4) u of its
    terms' sizes to what its inputs were off by."""
    x = x.double().cpu()
    off = torch.zeros_like(x)
    for k, (w, b) in enumerate(zip(net.host[::2], net.host[1::2])):
        w, b = w.double(), b.double()
        off = off @ w.abs() + (w.shape[0] + 4) * U * ((x.abs() + off) @ w.abs() + b.abs())
        x = x @ w + b
        if k < 3:
            x = x.clamp(min=0)
    return x, off


@pytest.mark.parametrize("hidden", [64, 96, 512, 1000])
@pytest.mark.parametrize("rows", [1, 37, 1500])
def test_value_net_of_any_hidden_size(hidden, rows):
    torch.manual_seed(hidden)
    m = models.ValueOnlyNN(418, hidden)
    m.bn1.running_mean.normal_()
    m.bn2.running_var.uniform_(0.5, 2.0)
    net = models.ValueNet(m, "cuda")
    x = torch.randint(-3, 6, (rows, 418)).float().cuda()
    probs, logits = net.forward(x, logits=True)
    want, off = chain_bound(net, x)
    assert bool(((logits.double().cpu() - want).abs() <= off).all())
    lg = logits.double().cpu()
    exact = lg.square() / lg.square().sum(1, keepdim=True)
    assert bool(((probs.double().cpu() - exact).abs() <= 16 * U).all())
    if hidden != 512:
        assert net.packed is None and net.wave is None
        for kw in ({"fused": True}, {"wave": True}):
            with pytest.raises(ValueError, match="built for"):
                net.forward(x, **kw)


def test_fused_layers_match_the_module():
    """Train and eval mode, forward and gradients, against the same module in 64 bits."""
    torch.manual_seed(3)
    plain = models.ValueOnlyNN(418, 128).cuda()
    plain.dropout1.p = plain.dropout2.p = 0.0
    fused = copy.deepcopy(plain)
    fused.fused = True
    exact = copy.deepcopy(plain).double()
    assert set(fused.state_dict()) == set(plain.state_dict())
    x = torch.randint(-3, 6, (200, 418)).float().cuda()
    for mode in (True, False):
        got, ref = [], exact.train(mode)(x.double())
        scale = float(ref.detach().abs().max())
        for m in (plain, fused):
            m.train(mode)
            y = m(x)
            got.append(float((y.detach().double() - ref.detach()).abs().max()) / scale)
        # the fused sums are bounded like torch's: both are fp32 of the same terms (418 of them at most)
        assert got[1] <= max(4 * got[0], 418 * U), got
    grads = []
    for m in (exact, plain, fused):
        m.train()
        m.zero_grad()
        m(x.to(m.fc1.weight.dtype)).square().sum().backward()
        grads.append([p.grad.double() for p in m.parameters()])
    for w, p, f in zip(*grads):
        size = float(w.norm())
        a, b = float((p - w).norm()), float((f - w).norm())
        assert b <= max(4 * a, 418 * U * max(size, 1.0)), (a, b, size)


def test_search_with_a_net_of_another_size():
    """cfr_pred with leaves from a 128-wide net: rounds on one stream and on three give the same trees and decisions,
    and the search kernel's own leaves are refused."""
    from citadels_self_play_amd.engine import GameBatch
    torch.manual_seed(5)
    net = models.ValueNet(models.ValueOnlyNN(418, 128), "cuda")
    out = []
    for groups in (1, 3):
        b = GameBatch(list(range(24)), preset=True)
        b.advance_random(5, 60)
        chosen, stats, rounds = b.cfr_pred(60, net, groups=groups)
        assert rounds > 0
        out.append((chosen.cpu(), stats[:, 1:4].clone()))
    assert torch.equal(out[0][0], out[1][0]) and torch.equal(out[0][1], out[1][1])
    with pytest.raises(ValueError, match="fused=False"):
        b.cfr_pred(10, net, fused=True)


def targets(seed, n):
    g = torch.Generator().manual_seed(seed)
    x = torch.randint(-3, 6, (n, 418), generator=g).float()
    return x, torch.rand(n, 6, generator=g, dtype=torch.float64)


@pytest.mark.parametrize("fused", [False, True])
def test_trainer_with_clipping(tmp_path, fused):
    """A clipped step by the trainer's own path leaves gradients of norm max_grad_norm; a bound no step reaches changes
    nothing (the gradients are left as they are, bit for bit)."""
    seen = []
    clip = train.clip_grad_norm

    def spy(grads, limit):
        norm = clip(grads, limit)
        seen.append((float(norm), float(ops.grad_norm(grads))))
        return norm
    train.clip_grad_norm = spy
    try:
        kw = dict(epochs=2, lr=0.01, hidden_size=64, gamma=0.9, batch_size=32, parent_folder=str(tmp_path), fused=fused)
        train.train_node_value_only(targets(0, 96), targets(1, 32), seed=1, max_grad_norm=0.05, **kw)
    finally:
        train.clip_grad_norm = clip
    assert len(seen) == 6
    for before, after in seen:
        want = before if before <= 0.05 else 0.05 * before / (before + 1e-6)
        assert abs(after - want) <= 4 * U * want + 1e-12, (before, after)
    assert any(before > 0.05 for before, _ in seen)
    if not fused:
        a = train.train_node_value_only(targets(0, 96), targets(1, 32), seed=1, **kw)[2]
        b = train.train_node_value_only(targets(0, 96), targets(1, 32), seed=1, max_grad_norm=1e9, **kw)[2]
        assert abs(a["train"][0] - b["train"][0]) <= 1e-3 * abs(a["train"][0])


def test_policy_step_over_searched_options():
    """cfr_targets' ragged option rows through a scoring net and policy_loss, its gradients clipped: loss and gradients
    against 64 bits over the same rows."""
    from citadels_self_play_amd.engine import GameBatch, pool_caps
    b = GameBatch(list(range(6)), preset=True)
    b.random_position(100)
    b.seed_numpy()
    nc, ec = pool_caps(2000)
    _, stats = b.cfr_decide(2000, node_cap=nc, edge_cap=ec)
    t = b.cfr_targets(stats[:, 0])
    offsets = train.option_offsets(t)
    lengths = (offsets[1:] - offsets[:-1]).cpu()
    assert lengths.tolist() == t["meta"][:, 3].cpu().tolist() and int(offsets[-1]) == t["dist"].shape[0]
    rows, n = t["opt_feat"].shape[0], len(lengths)
    torch.manual_seed(0)
    x = torch.cat([t["opt_feat"], t["feat"].repeat_interleave(lengths.cuda(), 0)], 1)
    w1 = (torch.randn(64, x.shape[1], device="cuda") * 0.02).requires_grad_()
    b1, w2 = torch.zeros(64, device="cuda", requires_grad=True), (torch.randn(1, 64, device="cuda") * 0.1).requires_grad_()
    ref = torch.log(t["dist"].clamp(min=0) + 1e-3).float()              # the search's own strategy, smoothed
    g = torch.Generator().manual_seed(2)
    actions = (torch.rand(n, generator=g) * lengths).long().clamp(max=lengths - 1).cuda()
    adv = torch.randn(n, generator=g).cuda()
    params = [w1, b1, w2]

    def scores(w1, b1, w2, lib):
        if lib:
            return ops.linear(ops.linear(x, w1, b1, activation="silu"), w2)[:, 0]
        h = x.double() @ w1.t() + b1
        return (h * torch.sigmoid(h) @ w2.t())[:, 0]

    d = [p.detach().double().requires_grad_() for p in params]
    logits = scores(*d, False)
    lp = [torch.log_softmax(logits[offsets[i]:offsets[i + 1]], 0) for i in range(n)]
    lq = [torch.log_softmax(ref[offsets[i]:offsets[i + 1]].double(), 0) for i in range(n)]
    taken = torch.stack([lp[i][actions[i]] for i in range(n)])
    old = (taken.detach() - 0.05).float()                               # rho 1.05: inside the clipping borders
    ratio = torch.exp(taken - old.double())
    kl = torch.stack([(p.exp() * (p - q)).sum() for p, q in zip(lp, lq)])
    want = (-torch.minimum(ratio * adv, ratio.clamp(0.8, 1.2) * adv) + 0.1 * kl).mean()
    wgrads = torch.autograd.grad(want, d)
    got = train.policy_loss(scores(*params, True), actions, old, adv, ref_logits=ref, offsets=offsets, kl_coef=0.1)
    grads = torch.autograd.grad(got.loss, params)
    # three fp32 products of at most 549 terms, a softmax of at most 60, a mean
    tol = 600 * U
    assert abs(float(got.loss.detach()) - float(want.detach())) <= tol * (1 + float(kl.detach().mean()))
    assert bool(((got.kl.double() - kl).abs() <= tol * (1 + kl)).all())
    for p, q in zip(grads, wgrads):
        assert float((p.double() - q).norm()) <= 4 * tol * float(q.norm()) + tol * 0.01
    norm = math.sqrt(sum(float(q.square().sum()) for q in wgrads))
    assert abs(float(ops.clip_grad_norm(grads, norm / 3)) - norm) <= 4 * tol * norm
    assert abs(float(ops.grad_norm(grads)) - norm / 3) <= 8 * tol * norm
