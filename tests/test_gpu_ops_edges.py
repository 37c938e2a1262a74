"""Edges of the training / serving operators (citadels_self_play_amd/ops.py) on a
real MI355X that test_gpu_ops.py leaves out.  Tolerances are counted as there: u =
2^-24 is half a step of fp32, a device exp or log is off by at most 4 u of its
value, every rounding by half a step of its type."""
import math

import pytest
import torch

from citadels_self_play_amd import ops
from test_gpu_ops import (DT, U, call_policy, linear_inputs, linear_want, policy_rows, policy_want, rounded, tiny,
                          within)

pytestmark = pytest.mark.gpu


# ---- policy loss ------------------------------------------------------------------

def even_rows(rows, width, dt=torch.float32):
    """Rows whose entries are all alike: every exp(l - max) is 1 and their sum exact, so log p is -log width to 64 bits."""
    return {"logits": torch.full((rows, width), 0.75, dtype=dt, device="cuda"), "ref": None, "mask": None, "offsets": None,
            "actions": (torch.arange(rows) * 7 % width).cuda(), "old": torch.full((rows,), -math.log(width), device="cuda"),
            "adv": torch.ones(rows, device="cuda"), "weights": torch.ones(rows, device="cuda")}


@pytest.mark.parametrize("widths", [range(2, 65), range(65, 257, 3), (300, 1000, 2049, 3000, 9001, 16383), (20001, 65537)],
                         ids=lambda w: "%d-%d" % (w[0], w[-1]))
def test_policy_gradient_of_even_rows(widths):
    """dloss/dl_j = rho (1 / n - 1[j = a]).  rho is 64-bit (in 32 bits where a row has one wave: a logarithm of log n, an
    exponential); it, 1 / n, their product and the result round once each."""
    for n in widths:
        a = even_rows(3, n)
        l = a["logits"].requires_grad_()
        grad = torch.autograd.grad(call_policy(a, (0.2, 0.2), 0.0, l).loss, l)[0].double()
        rho = math.exp(-math.log(n) - float(a["old"][0].double()))
        want = torch.full((3, n), rho / n, dtype=torch.float64, device="cuda")
        tol = 4 * U * want
        at = a["actions"][:, None]
        want.scatter_add_(1, at, torch.full_like(want, -rho)[:, :1])
        tol.scatter_(1, at, 6 * U * want.gather(1, at).abs())
        if 64 < n <= 1024:
            tol += want.abs() * (4 * math.log(n) + 4) * U
        within(grad, want, tol, "width %d" % n)


@pytest.mark.parametrize("rows,width,dtype", [(512, 50, "fp32"), (256, 4000, "fp32"), (512, 50001, "bf16"), (128, 20001, "bf16"), (4, 20001, "fp32")])
def test_policy_loss_that_cancels(rows, width, dtype):
    """A signed mean a thousand times smaller than its terms, and more, keeps its digits: rows' values and their sum are 64-bit (1e-13 of
    the terms allowed for them), the weights powers of two, the result rounds once."""
    a = even_rows(rows, width, DT[dtype])
    g = torch.Generator().manual_seed(2)
    a["old"] = (a["old"].cpu() + 0.1 * torch.randn(rows, generator=g).clamp(-1, 1)).cuda()
    rho = torch.exp(-math.log(width) - a["old"].double())
    adv = torch.randn(rows, generator=g).cuda()
    adv[rows // 2:] = (-adv[:rows // 2].double() * rho[:rows // 2] / rho[rows // 2:]).float()
    adv[0] *= 1 + 2.0 ** -10
    a["adv"], a["weights"] = adv, None
    terms = -rho * adv.double()
    want = float(terms.mean())
    assert 1e-9 < abs(want) < 1e-3 * float(terms.abs().mean())
    for ref in (None, a["logits"]):
        got = call_policy(dict(a, ref=ref), (0.2, 0.2), 0.0)
        assert abs(float(got.loss) - want) <= U * abs(want) + 1e-13 * float(terms.abs().mean()), (float(got.loss), want)


def test_policy_gradient_belongs_to_its_pass():
    """A forward and a backward pass of two captures, or one eager and one captured: each replay gives the gradient of
    what it finds, in memory that nothing else has."""
    s = torch.cuda.Stream()
    a = policy_rows([4, 9, 30, 64], torch.float32)
    l = a["logits"].requires_grad_()
    up = torch.ones((), device="cuda")

    def want(v):
        c = l.detach().clone().requires_grad_()
        return torch.autograd.grad(call_policy(a, (0.2, 0.2), 0.1, c).loss, c, torch.tensor(v, device="cuda"))[0]

    want(1.0)
    torch.cuda.synchronize()
    # both captured, each for itself: the second one replayed again, its result changed in between
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(first, stream=s):
        loss = call_policy(a, (0.2, 0.2), 0.1, l).loss
    with torch.cuda.graph(second, stream=s):
        grad = torch.autograd.grad(loss, l, up, retain_graph=True)[0]
    for _ in range(3):
        l.data.mul_(0.9)
        first.replay()
        for v in (0.5, 1.0, 1.0, -2.0):
            up.fill_(v)
            second.replay()
            torch.cuda.synchronize()
            assert torch.equal(grad, want(v)), v
            grad.mul_(3.0)
            torch.cuda.synchronize()
    # captured, then an eager backward pass: its gradient is the caller's, and stays
    with torch.cuda.stream(s):
        mine = torch.autograd.grad(loss, l, retain_graph=True)[0]
    torch.cuda.synchronize()
    kept = want(1.0)
    assert torch.equal(mine, kept)
    l.data.mul_(0.9)
    for _ in range(2):
        first.replay()
        torch.cuda.synchronize()
        assert torch.equal(mine, kept)
    # eager, then a captured backward pass through logits that are no leaf: what the allocator gives out meanwhile is not
    # written to
    with torch.cuda.stream(s):
        leaf = l.detach().clone().requires_grad_()
        eager = call_policy(a, (0.2, 0.2), 0.1, leaf * 1.0).loss
    torch.cuda.synchronize()
    third = torch.cuda.CUDAGraph()
    with torch.cuda.graph(third, stream=s):
        grad = torch.autograd.grad(eager, leaf, up, retain_graph=True)[0]
    with torch.cuda.stream(s):
        others = [torch.full_like(leaf, 7.0) for _ in range(64)]
    torch.cuda.synchronize()
    for v in (1.0, 0.5, 1.0):
        up.fill_(v)
        third.replay()
        torch.cuda.synchronize()
        assert torch.equal(grad, want(v)), v
        assert all(bool((t == 7.0).all()) for t in others)
    # the same node once more, eager: the gradient that its forward pass made
    with torch.cuda.stream(s):
        again = torch.autograd.grad(eager, leaf)[0]
    torch.cuda.synchronize()
    assert torch.equal(again, want(1.0))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("shape", [(3, 64), (3, 200), (3, 1000), (3, 4000), (3, 9001), (130, 16500), (130, 17001), (130, 19999), (3, 20001)], ids=str)
def test_policy_kl_of_a_sure_reference(shape, dtype):
    """An even policy, a reference with all but e^-18 of the weight on one entry.  The policy's sum is exact; of the two
    others' terms a lane has at most 20 (of 16-bit types 40), then 6 shuffles and 16 waves: so many half steps of 17,
    a few of 18, and those of the logarithm of the sums' ratio, 4 of each of its units."""
    rows, n = shape
    l, r = torch.full(shape, 0.75, device="cuda"), torch.zeros(shape, device="cuda")
    at = torch.arange(rows, device="cuda") * 31 % n
    r.scatter_(1, at[:, None], 18.0)
    zero = torch.zeros(rows, device="cuda")
    got = ops.policy_loss(l.to(DT[dtype]), at, zero, zero, ref_logits=r.to(DT[dtype]))
    lp, lq = torch.log_softmax(l.double(), 1), torch.log_softmax(r.double(), 1)
    terms = (20 if dtype == "fp32" else 40) + 22
    tol = U * (17 * (terms + 2) + 3 * 18 + 4 * math.log(n) + 10)
    within(got.kl, (lp.exp() * (lp - lq)).sum(1), torch.full((rows,), tol), "kl")


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("dense", [(5, 12), (5, 200), (4, 1500), (3, 9001), (3, 20001)], ids=str)
def test_policy_kl_watched_only(dense, dtype):
    """kl_coef 0 with a reference that rules out what the policy plays, or leaves nothing: KL says so, loss and
    gradient are those without a reference."""
    a = policy_rows(None, DT[dtype], dense=dense)
    a["ref"][0, int(a["actions"][0])] = -math.inf
    a["ref"][1] = -math.inf
    a["ref"][2, 3] = math.nan
    want = policy_want(dict(a, ref=None), (0.2, 0.2), 0.0)
    l = a["logits"].detach().requires_grad_()
    for leaf in (a["logits"], l):
        got = call_policy(a, (0.2, 0.2), 0.0, leaf)
        within(got.loss.detach(), *want[0], what="loss")
        within(got.logp, *want[1], what="logp")
        assert float(got.kl[0]) == math.inf and bool(got.kl[1:3].isnan().all())
    for up in (1.0, 0.5):
        grad = torch.autograd.grad(got.loss, l, torch.tensor(up, device="cuda"), retain_graph=True)[0]
        v, t = want[3]
        within(grad, v * up, (t + U * v.abs()) * up + tiny(DT[dtype]), what="grad")


# ---- linear ------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("size", [(70, 96, 88), (2100, 131, 300)], ids=str)
@pytest.mark.parametrize("res", [False, True])
def test_linear_relu_passes_not_a_number_on(size, dtype, res):
    """relu's gradient where the pre-activation is NaN is dy, as torch has it: a NaN does not hide in a 0."""
    dt = DT[dtype]
    x, w, b, r, dy = linear_inputs(*size, dt, "relu", True, res)
    x[13, 5], x[29, 95] = math.nan, math.nan
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = ops.linear(x, w, b, residual=r, activation="relu")
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    z = x.detach().double() @ w.detach().double().t() + b.detach().double()
    assert bool(z[[13, 29]].isnan().all()) and bool(y[[13, 29]].isnan().all())
    dz = dy.double() * ~(z <= 0)
    M, N = size[0], size[2]
    # dz is dy or 0, exactly; the sums and their rounding
    wd = w.detach().double()
    want = dz @ wd
    within(dx, want, rounded((N + 2) * U * (dz.abs() @ wd.abs()), want, dt), "dx")
    want = dz.sum(0)
    within(db, want, rounded((M + 2) * U * dz.abs().sum(0), want, dt), "db")
    assert bool(dw[:, [5, 95]].isnan().any(0).all()) and not bool(dw[:, :5].isnan().any())


def test_linear_rows_past_a_grid_of_direct_loads():
    """2^24 tiles of 256 threads are one grid dimension's most: fp32 over more rows than that takes."""
    M, N = (1 << 30) + 1000, 33
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 4 * M * (N + 1) + (8 << 30):
        pytest.skip("needs 154 GB of free memory on the GPU")
    x, w = torch.empty(M, 1, device="cuda"), torch.randn(N, 1, device="cuda")
    x.normal_()
    y = ops.linear(x, w)
    for at in (0, (1 << 27) - 3000, (1 << 29) + 77, (1 << 30) - 3000, M - 5000):
        assert torch.equal(y[at:at + 5000], x[at:at + 5000] * w.t()), at   # one product each, rounded once
    del x, y
    torch.cuda.empty_cache()


def test_linear_gradient_is_the_slope():
    """Along the gradient's own direction v (|v| = 1) the slope is the gradient's norm.  (F(+h) - F(-h)) / 2h differs
    from it by h^2 / 6 sum |dy| |dz/ds|^3 0.8 (|gelu'''| < 0.78), by the values' rounding / h, and by that of the points."""
    x, w, b, r, dy = linear_inputs(20, 30, 25, torch.float32, "gelu", True, True)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(ops.linear(x, w, b, residual=r, activation="gelu"), leaves, dy)
    h = 2.0 ** -4
    d = dy.double()
    for k, along in enumerate((lambda v: v @ w.detach().double().t(), lambda v: x.detach().double() @ v.t(), lambda v: v.expand(20, 25))):
        slope = float(grads[k].double().norm())
        v = grads[k].double() / slope
        noise = 0.0

        def at(s):
            nonlocal noise
            a = [(t.detach().double() + (s * h * v if i == k else 0)).float() for i, t in enumerate(leaves)]
            noise += float((d.abs().cpu() * linear_want(*a, r, dy, "gelu")[0][1]).sum())
            return float((ops.linear(*a, residual=r, activation="gelu").double() * d).sum())

        got = (at(1) - at(-1)) / (2 * h)
        third = 0.8 * float((d.abs() * along(v).abs() ** 3).sum()) * h * h / 6
        points = float((grads[k].double().abs() * U * (leaves[k].detach().double().abs() + h * v.abs())).sum()) * 1.5 / h
        tol = third + noise / (2 * h) + points
        assert tol <= 0.02 * slope, (k, third, noise, slope)       # so that a wrong gradient fails
        assert abs(got - slope) <= tol, (k, got, slope, third, noise)


# ---- gradient norm ------------------------------------------------------------------

def test_clip_of_tensors_that_hold_nothing():
    for n in (1, 3, 200):
        grads = [torch.empty((0, 3), device="cuda") for _ in range(n)]
        assert float(ops.grad_norm(grads)) == 0.0 and float(ops.clip_grad_norm(grads, 1.0)) == 0.0
        assert float(ops.clip_grad_norm(grads, 1.0, out=[t.clone() for t in grads])) == 0.0


# ---- together ---------------------------------------------------------------------------

def test_two_streams_with_every_workspace():
    """Two layers on two streams at once, other inputs each, of sizes that take copies, dz, column sums and split sums:
    each has what it has alone."""
    inputs = [linear_inputs(16500, 131, 523, torch.bfloat16, "gelu", True, True, seed=s) for s in (1, 2)]
    inputs += [linear_inputs(1000, 8201, 1100, torch.float32, "silu", True, False, seed=s) for s in (3, 4)]

    def step(k):
        x, w, b, r, dy = inputs[k]
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        y = ops.linear(*leaves, residual=r, activation="gelu" if k < 2 else "silu")
        return [y.detach()] + list(torch.autograd.grad(y, leaves, dy))

    want = []
    for k in range(4):
        want.append(step(k))
        torch.cuda.synchronize()
    assert not torch.equal(want[0][0], want[1][0])
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for pair in (0, 2):
        for _ in range(3):
            for i, s in enumerate(streams):
                with torch.cuda.stream(s):
                    got.append((pair + i, step(pair + i)))
    torch.cuda.synchronize()
    for k, g in got:
        assert all(torch.equal(p, q) for p, q in zip(g, want[k])), k


def test_tensors_without_memory_are_refused():
    """vmap's, torch.func's and batches of gradients: an error that says so, and the graph is as it was."""
    x, w, b, r, dy = linear_inputs(37, 50, 41, torch.float32, "silu", True, True)
    with pytest.raises(ValueError, match="torch.func or vmap"):
        torch.vmap(lambda t: ops.linear(t, w))(x.view(37, 1, 50))
    with pytest.raises(ValueError, match="torch.func or vmap"):
        torch.func.grad(lambda t: ops.linear(x, t).sum())(w)
    leaves = [t.requires_grad_() for t in (x, w, b, r)]
    y = ops.linear(*leaves, activation="silu")
    with pytest.raises(RuntimeError, match="not a batch"):
        torch.autograd.grad(y, leaves, torch.stack([dy, dy]), is_grads_batched=True, retain_graph=True)
    got = torch.autograd.grad(y, leaves, dy)
    want = torch.autograd.grad(ops.linear(*leaves, activation="silu"), leaves, dy)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    a = policy_rows([4, 9, 30], torch.float32)
    with pytest.raises(ValueError, match="torch.func or vmap"):
        torch.func.grad(lambda t: call_policy(a, (0.2, 0.2), 0.1, t).loss)(a["logits"])
    l = a["logits"].requires_grad_()
    loss = call_policy(a, (0.2, 0.2), 0.1, l).loss
    with pytest.raises(RuntimeError, match="not a batch"):
        torch.autograd.grad(loss, l, torch.ones(3, device="cuda"), is_grads_batched=True, retain_graph=True)
    assert torch.equal(torch.autograd.grad(loss, l)[0], torch.autograd.grad(call_policy(a, (0.2, 0.2), 0.1, l).loss, l)[0])
    with pytest.raises(ValueError, match="dense tensor"):
        torch.vmap(lambda t: ops.clip_grad_norm([t], 1.0))(w.detach())


def test_graphed_callable():
    """torch's own graphs of a module: the forward pass in one, the backward pass in another, each replayed with new inputs
    and upstream gradients.  (A warm-up's graph would be alive beside the capture.)"""
    a = policy_rows([4, 9, 30, 64], torch.float32)
    x, w, b, _, _ = linear_inputs(107, 50, 40, torch.float32, "gelu", True, False)

    class Step(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.w1, self.b1 = torch.nn.Parameter(w.clone()), torch.nn.Parameter(b.clone())
            self.w2 = torch.nn.Parameter(w[:1, :40].clone())

        def forward(self, x):
            logits = ops.linear(ops.linear(x, self.w1, self.b1, activation="gelu"), self.w2)[:, 0]
            return call_policy(a, (0.2, 0.2), 0.1, logits).loss

    plain, graphed = Step(), torch.cuda.make_graphed_callables(Step(), (x.clone(),), num_warmup_iters=0)
    for k in range(4):
        x = x * 0.9
        loss, want = graphed(x), plain(x)
        assert torch.equal(loss, want)
        up = torch.tensor((1.0, 0.5, -2.0, 1.0)[k], device="cuda")
        got = torch.autograd.grad(loss, list(graphed.parameters()), up)
        want = torch.autograd.grad(want, list(plain.parameters()), up)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want)), k
