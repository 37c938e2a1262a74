"""The training / serving operators (citadels_self_play_amd/ops.py) on a real
MI355X against plain formulas in 64 bits.

Tolerances are error bounds, not fits.  u = 2^-24 is half a step of fp32, e
half a step of the result's type (eps / 2), tiny its smallest step.  A sum of
n terms in fp32, in any order, is off by at most (n + 2) u sum |terms|; a
device exp, log or erfc by 4 u of its value (2 ulp); every rounding to the
element type by e of the value or half of tiny."""
import math
import threading

import pytest
import torch
import torch.utils.checkpoint

from citadels_self_play_amd import ops

pytestmark = pytest.mark.gpu
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
U = 2.0 ** -24


def half_step(dt):
    return torch.finfo(dt).eps / 2


def tiny(dt):
    return torch.finfo(dt).smallest_normal * torch.finfo(dt).eps


def rounded(tol, value, dt):
    """`tol` of a value before it is rounded to dt, with that rounding."""
    return tol + half_step(dt) * (value.abs() + tol) + tiny(dt) / 2


def within(got, want, tol, what):
    got, want, tol = got.double().cpu(), want.double().cpu(), tol.double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got - want).abs()
    bad = ~(off <= tol)
    assert not bool(bad.any()), "%s: %d of %d off, the worst %.3g of its tolerance (got %r, want %r)" % (
        what, int(bad.sum()), bad.numel(), float((off / tol)[bad].max()), float(got[bad][0]), float(want[bad][0]))


# ---- linear --------------------------------------------------------------------

ACT = {  # f, f', and bounds of |f'|, |f''|
    "none": (lambda z: z, torch.ones_like, 1.0, 0.0),
    "relu": (lambda z: z.clamp(min=0), lambda z: (z > 0).double(), 1.0, 0.0),
    "gelu": (lambda z: z * torch.special.ndtr(z),
             lambda z: torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi), 1.13, 0.8),
    "silu": (lambda z: z * torch.sigmoid(z), lambda z: torch.sigmoid(z) * (1 + z * (1 - torch.sigmoid(z))), 1.1, 0.5),
}


def linear_inputs(M, K, N, dt, act, bias, res, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=g)
    w = torch.randn(N, K, generator=g) / math.sqrt(max(K, 1))
    b = torch.randn(N, generator=g) * 0.3
    if act == "relu":              # z on a grid, half a step off 0: its sign is no matter of rounding
        x, w = torch.randint(-4, 5, (M, K), generator=g).float(), torch.randint(-8, 9, (N, K), generator=g) / 64.0
        b = (torch.randint(-20, 20, (N,), generator=g) + 0.5) / 64.0
        if not bias and K:
            x[:, 0], w[:, 0] = 1.0, b
    r = torch.randn(M, N, generator=g)
    dy = torch.randn(M, N, generator=g)
    return [None if t is None else t.to(dt).cuda() for t in (x, w, b if bias else None, r if res else None, dy)]


def linear_want(x, w, b, r, dy, act):
    """(values, tolerances) of y, dx, dw, db in 64 bits on the CPU."""
    dt = x.dtype
    x, w, b, r, dy = (None if t is None else t.detach().double().cpu() for t in (x, w, b, r, dy))
    M, K, N = x.shape[0], x.shape[1], w.shape[0]
    f, df, c1, c2 = ACT[act]
    z = x @ w.t() + (0 if b is None else b)
    zt = (K + 4) * U * (x.abs() @ w.abs().t() + (0 if b is None else b.abs()))
    y = f(z)
    yt = c1 * zt + 16 * U * (y.abs() + z.abs())
    if r is not None:
        y, yt = y + r, yt + 2 * U * (y.abs() + r.abs())
    kept = zt if dt == torch.float32 else rounded(zt, z, dt)         # the pre-activation as the backward pass has it
    d = df(z)
    dz = dy * d
    dt_f = dy.abs() * (c2 * kept + 24 * U * (1 + z.abs())) if act in ("gelu", "silu") else 2 * U * dz.abs()
    if act == "none":
        dt_f = torch.zeros_like(dz)
    dzt = dt_f if act == "none" else rounded(dt_f, dz, dt)
    size = dz.abs() + dzt
    dx, dw, db = dz @ w, dz.t() @ x, dz.sum(0)
    dxt = dzt @ w.abs() + (N + 2) * U * (size @ w.abs())
    dwt = dzt.t() @ x.abs() + (M + 2) * U * (size.t() @ x.abs())
    dbt = dt_f.sum(0) + (M + 2) * U * size.sum(0)
    return [(v, rounded(t, v, dt)) for v, t in ((y, yt), (dx, dxt), (dw, dwt), (db, dbt))]


def check_linear(x, w, b, r, dy, act, what=""):
    want = linear_want(x, w, b, r, dy, act)
    y0 = ops.linear(x, w, b, residual=r, activation=act)
    within(y0, *want[0], what + " y (no grad)")
    leaves = [t.detach().requires_grad_() for t in (x, w, b, r) if t is not None]
    it = iter(leaves)
    x, w, b, r = (None if t is None else next(it) for t in (x, w, b, r))
    y = ops.linear(x, w, b, residual=r, activation=act)
    assert torch.equal(y.detach(), y0)
    got = list(torch.autograd.grad(y, leaves, dy))
    within(got[0], *want[1], what + " dx")
    within(got[1], *want[2], what + " dw")
    if b is not None:
        within(got[2], *want[3], what + " db")
    if r is not None:
        assert torch.equal(got[-1], dy)


SIZES = [(1, 1, 1), (1, 7, 5), (2, 64, 16), (3, 65, 17), (16, 32, 64), (17, 33, 130), (64, 418, 512), (65, 64, 64),
         (100, 128, 96), (130, 200, 70), (1, 1024, 300), (5, 2000, 33), (257, 72, 264), (300, 515, 129)]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_linear_sizes(size, dtype):
    for act, bias, res in (("relu", True, False), ("gelu", True, True), ("none", False, False)):
        check_linear(*linear_inputs(*size, DT[dtype], act, bias, res), act, "%s %s %s" % (size, dtype, act))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("act", list(ACT))
@pytest.mark.parametrize("bias,res", [(False, False), (True, False), (False, True), (True, True)])
def test_linear_epilogues(act, bias, res, dtype):
    check_linear(*linear_inputs(70, 96, 88, DT[dtype], act, bias, res), act)
    check_linear(*linear_inputs(3, 160, 72, DT[dtype], act, bias, res, seed=1), act)


@pytest.mark.parametrize("dtype", list(DT))
def test_linear_long_reductions(dtype):
    """Few outputs over a long reduction (split sums), each way round."""
    for size in ((8, 5003, 40), (2100, 40, 24), (24, 48, 3001)):
        check_linear(*linear_inputs(*size, DT[dtype], "silu", True, True), "silu", str(size))


@pytest.mark.parametrize("dtype", list(DT))
def test_linear_large(dtype):
    """Sizes of the throughput kernels, tile edges on every side."""
    for size in ((1024, 512, 768), (777, 1000, 520)):
        check_linear(*linear_inputs(*size, DT[dtype], "gelu", True, True), "gelu", str(size))


# (rows, in, out): few outputs over a long reduction (dw over the rows, y over `in`), shared out by tiles of 64 and 128,
# with and without whole chunks; many outputs in each of the larger tiles, with a part of a tile at either end; odd rows
# of a product large enough to be copied first
SHARED = [(4100, 520, 130), (9000, 264, 520), (16400, 768, 776), (32768, 64, 512), (16390, 130, 259), (40001, 67, 130),
          (128, 8200, 520), (100, 16392, 264), (520, 4104, 1032), (1030, 8192, 1000), (16500, 131, 523), (130, 520, 8200), (1000, 8201, 1100)]
LARGE = [(4000, 801, 1023), (4200, 801, 1023), (2570, 520, 5000), (4100, 1032, 2310), (6150, 516, 3010), (9000, 520, 1030), (4001, 1001, 2003)]


# one to a few rows: reductions that end inside a lane's chunk, shared by 1 to 8 waves, outputs that end inside a wave's
FEW = [(1, 512, 64), (1, 513, 1003), (2, 4100, 77), (3, 2051, 130), (4, 5001, 33), (1, 40003, 5), (2, 16384, 64),
       (1, 4096, 3000), (4, 260, 9000), (1, 256, 8200), (3, 300, 1), (5, 4096, 300)]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("size", FEW, ids=str)
def test_linear_few_rows(size, dtype):
    check_linear(*linear_inputs(*size, DT[dtype], "silu", True, True), "silu", "%s %s" % (size, dtype))
    x, w, b, r, _ = linear_inputs(*size, DT[dtype], "gelu", True, True)
    pad = lambda t: torch.cat([t, t.new_full((t.shape[0], 3), math.nan)], 1)[:, :t.shape[1]]  # noqa: E731
    want = ops.linear(x, w, b, residual=r, activation="gelu")
    assert torch.equal(ops.linear(pad(x), pad(w), b, residual=pad(r), activation="gelu"), want)

# odd rows through registers in each of the three products, by one or two halves of a workgroup
ODD = [(2100, 131, 1100), (1030, 259, 1030), (3000, 700, 201), (2500, 700, 201), (200, 1501, 1500), (200, 1101, 1100)]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("size", SHARED + LARGE + ODD, ids=str)
def test_linear_tiles(size, dtype):
    check_linear(*linear_inputs(*size, DT[dtype], "gelu", True, True), "gelu", "%s %s" % (size, dtype))
    if size[0] == 16500:           # dy itself copied to padded rows
        check_linear(*linear_inputs(*size, DT[dtype], "none", False, False), "none", "%s %s" % (size, dtype))


@pytest.mark.parametrize("dtype", list(DT))
def test_linear_strides_and_alignment(dtype):
    """Rows further apart than their width, storage that starts at any element, transposed and expanded tensors."""
    dt = DT[dtype]
    x, w, b, r, dy = linear_inputs(70, 96, 88, dt, "gelu", True, True)
    def view(t, pad, off):
        buf = torch.full((t.shape[0] * (t.shape[1] + pad) + off,), float("nan"), dtype=dt, device="cuda")
        v = buf[off:].view(t.shape[0], t.shape[1] + pad)[:, :t.shape[1]]
        v.copy_(t)
        return v
    for pad, off in ((8, 0), (1, 0), (3, 5), (0, 1)):
        check_linear(view(x, pad, off), view(w, pad, off), b, view(r, pad, off), view(dy, pad, off), "gelu", str((pad, off)))
    check_linear(x.t().contiguous().t(), w.t().contiguous().t(), b, r.t().contiguous().t(), dy.t().contiguous().t(), "gelu")
    check_linear(x[:1].expand(70, 96), w, b, r[:, :1].expand(70, 88), dy[:1, :1].expand(70, 88), "gelu", "expanded")


@pytest.mark.parametrize("dtype", list(DT))
def test_linear_rows_far_apart(dtype):
    """Rows over 8 MB apart, past what a tile's 32-bit offsets reach."""
    dt = DT[dtype]
    x, w, b, r, dy = linear_inputs(300, 72, 3400, dt, "silu", True, True)
    far = torch.empty(300, (1 << 23) // x.element_size() + 8, dtype=dt, device="cuda")[:, :72]
    check_linear(far.copy_(x), w, b, r, dy, "silu", "far rows")


def test_linear_leading_dimensions_and_empty():
    x, w, b, r, dy = linear_inputs(24, 40, 56, torch.bfloat16, "gelu", True, True)
    y = ops.linear(x, w, b, residual=r, activation="gelu")
    assert torch.equal(ops.linear(x.view(2, 3, 4, 40), w, b, residual=r.view(2, 3, 4, 56), activation="gelu").view(24, 56), y)
    assert torch.equal(ops.linear(x[0], w, b, activation="silu"), ops.linear(x[:1], w, b, activation="silu")[0])
    for M, K, N in ((0, 8, 4), (3, 8, 0), (3, 0, 4)):
        leaves = [torch.randn(s, device="cuda", requires_grad=True) for s in ((M, K), (N, K), (N,), (M, N))]
        y = ops.linear(*leaves[:3], residual=leaves[3], activation="relu")
        assert y.shape == (M, N)
        if K == 0:
            assert torch.equal(y, leaves[2].relu().expand(M, N) + leaves[3])
        grads = torch.autograd.grad(y, leaves, torch.ones_like(y))
        assert [g.shape for g in grads] == [t.shape for t in leaves]
        if not M:
            assert all(not bool(g.any()) for g in grads)
        if K == 0:
            assert torch.equal(grads[2], (leaves[2] > 0).float() * M)


@pytest.mark.parametrize("act", list(ACT))
def test_linear_not_a_number_stays_in_its_row(act):
    x, w, b, r, dy = linear_inputs(70, 96, 88, torch.float32, act, True, False)
    clean = ops.linear(x, w, b, activation=act)
    x = x.clone()
    x[13, 5], x[29, 95] = math.nan, math.nan
    y = ops.linear(x, w, b, activation=act)
    hit = torch.zeros(70, dtype=torch.bool, device="cuda")
    hit[[13, 29]] = True
    assert bool(y[hit].isnan().all()) and torch.equal(y[~hit], clean[~hit])
    # memory beside the matrices is never part of a sum
    wide = torch.full((71, 131), math.nan, device="cuda")
    wide[:70, :96] = linear_inputs(70, 96, 88, torch.float32, act, True, False)[0]
    assert torch.equal(ops.linear(wide[:70, :96], w, b, activation=act), clean)


def test_linear_fp16_edges():
    """Pre-activations past fp16's range or below its smallest step keep a right gradient."""
    x = torch.tensor([[60000.0], [2.0 ** -14]], device="cuda").half()
    w = torch.tensor([[4.0], [-4.0], [2.0 ** -14]], device="cuda").half()
    for act in ("gelu", "silu", "relu"):
        for res in (None, torch.zeros(2, 3, device="cuda").half()):
            xx, ww = x.clone().requires_grad_(), w.clone().requires_grad_()
            y = ops.linear(xx, ww, residual=res, activation=act)
            assert float(y[0, 0].detach()) == math.inf and float(y[1, 2].detach().abs()) < 1e-7
            dw = torch.autograd.grad(y, ww, torch.tensor([[0.0] * 3, [1.0] * 3], device="cuda").half())[0]
            slope = 1.0 if act == "relu" else 0.5
            assert abs(float(dw[2, 0]) / 2.0 ** -14 - slope) < 1e-3
            dx = torch.autograd.grad(ops.linear(xx, ww, residual=res, activation=act), xx,
                                     torch.tensor([[1.0, 1.0, 0.0], [0.0] * 3], device="cuda").half())[0]
            assert float(dx[0, 0]) == 4.0


def test_linear_partial_gradients():
    x, w, b, r, dy = linear_inputs(33, 40, 24, torch.float32, "silu", True, True)
    leaves = [t.detach().requires_grad_() for t in (x, w, b, r)]
    full = torch.autograd.grad(ops.linear(*leaves[:3], residual=leaves[3], activation="silu"), leaves, dy)
    for k in range(4):
        only = [t.detach().requires_grad_(i == k) for i, t in enumerate((x, w, b, r))]
        got = torch.autograd.grad(ops.linear(*only[:3], residual=only[3], activation="silu"), only[k], dy)[0]
        assert torch.equal(got, full[k]), k


def test_linear_gradient_against_differences():
    """Along a direction v, (F(+h) - F(-h)) / 2h differs from grad . v by h^2 / 6 |F'''| and the values' rounding / h."""
    x, w, b, r, dy = linear_inputs(20, 30, 25, torch.float32, "gelu", True, True)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(ops.linear(x, w, b, residual=r, activation="gelu"), leaves, dy)
    h = 2.0 ** -7
    g = torch.Generator().manual_seed(3)
    for k in range(3):
        v = torch.randn(leaves[k].shape, generator=g).cuda()
        v = v / v.norm()
        def at(s):
            a = [t.detach() + (s * h * v if i == k else 0) for i, t in enumerate(leaves)]
            return float((ops.linear(*a, residual=r, activation="gelu").double() * dy.double()).sum())
        slope, want = (at(1) - at(-1)) / (2 * h), float((grads[k].double() * v.double()).sum())
        # |dz| <= h |x| |v|; gelu''' <= 2; rounding: 40 u of each value, dy-weighted
        third = 2.0 * float(dy.abs().double().sum()) * max(float(x.detach().abs().max()), 1.0) ** 3 * h * h / 6
        noise = 80 * U * float((dy.abs() * (r.abs() + 4)).double().sum()) / h
        assert abs(slope - want) <= third + noise, (k, slope, want, third, noise)


# ---- policy loss ------------------------------------------------------------------

def policy_rows(lengths, dt, seed=0, spread=2.0, masked=0.0, ref=True, dense=None):
    """Inputs on the GPU: ragged rows of these lengths, or with dense = (rows, width) a table."""
    g = torch.Generator().manual_seed(seed)
    n = sum(lengths) if dense is None else dense[0] * dense[1]
    N = len(lengths) if dense is None else dense[0]
    if dense is not None:
        lengths = [dense[1]] * N
    a = {"logits": (torch.randn(n, generator=g) * spread).to(dt)}
    a["ref"] = (a["logits"].float() + 0.3 * torch.randn(n, generator=g)).to(dt) if ref else None
    a["mask"] = torch.rand(n, generator=g) >= masked if masked else None
    off = [0]
    for k in lengths:
        off.append(off[-1] + k)
    acts, old = [], []
    for i, k in enumerate(lengths):
        legal = [j for j in range(k) if a["mask"] is None or bool(a["mask"][off[i] + j])]
        act = legal[int(torch.randint(len(legal), (1,), generator=g))] if legal else 0
        acts.append(act)
        if legal:
            l = a["logits"][off[i]:off[i + 1]].double()[legal]
            old.append(float(a["logits"][off[i] + act].double() - torch.logsumexp(l, 0)))
        else:
            old.append(0.0)
    a["actions"] = torch.tensor(acts, dtype=torch.int64)
    noise = torch.randn(N, generator=g) * 0.15
    noise[(noise.abs() - 0.215).abs() < 0.045] = 0.0   # not next to a clipping border (log 1.2 .. 1.28 = 0.18 .. 0.25, -log 0.8 = 0.22)
    a["old"] = (torch.tensor(old, dtype=torch.float64) - noise).float()
    a["adv"] = torch.randn(N, generator=g)
    a["weights"] = torch.rand(N, generator=g)
    a["offsets"] = torch.tensor(off) if dense is None else None
    if dense is not None:
        for k in ("logits", "ref", "mask"):
            a[k] = None if a[k] is None else a[k].view(dense)
    return {k: None if v is None else v.cuda() for k, v in a.items()}


def policy_want(a, clip, beta):
    """(loss, logp, kl, grad) with tolerances, row by row in 64 bits on the CPU."""
    a = {k: None if v is None else v.detach().cpu() for k, v in a.items()}
    dt = a["logits"].dtype
    N = len(a["actions"])
    flat = {k: None if a[k] is None else a[k].reshape(-1) for k in ("logits", "ref", "mask")}
    width = 0 if a["offsets"] is not None else a["logits"].shape[1]
    off = a["offsets"].tolist() if a["offsets"] is not None else [i * width for i in range(N + 1)]
    w_all = a["weights"].double() if a["weights"] is not None else torch.full((N,), float(torch.tensor(1.0 / max(N, 1))))
    logp, kls, tl, tk = (torch.zeros(N, dtype=torch.float64) for _ in range(4))
    grad, tg = torch.zeros_like(flat["logits"], dtype=torch.float64), torch.zeros_like(flat["logits"], dtype=torch.float64)
    loss = loss_t = size = 0.0
    for i in range(N):
        l = flat["logits"][off[i]:off[i + 1]].double()
        ok = torch.ones(len(l), dtype=torch.bool) if flat["mask"] is None else flat["mask"][off[i]:off[i + 1]].clone()
        ok &= l > -math.inf
        w = float(w_all[i])
        if w == 0 or not bool(ok.any()):
            continue
        l = torch.where(ok, l, -math.inf)
        n = int(ok.sum())
        lp = l - torch.logsumexp(l, 0)
        p = torch.exp(lp)
        # the log sum: n terms of 4 u each, summed; the row's entries and it are rounded where they are subtracted
        err = (2 * n + 40) * U + 4 * U * float(l[ok].abs().max())
        act = int(a["actions"][i])
        logp[i], tl[i] = lp[act], err
        kl, klt = 0.0, 0.0
        d = torch.zeros_like(lp)
        if flat["ref"] is not None:
            q = torch.where(ok, flat["ref"][off[i]:off[i + 1]].double(), -math.inf)
            err_q = (2 * n + 40) * U + 4 * U * float(q[ok].abs().max())
            d = torch.where(ok, lp - (q - torch.logsumexp(q, 0)), 0.0)
            pq = torch.where(ok, torch.exp(q - torch.logsumexp(q, 0)), 0.0)
            kl = float((p * d).sum())
            # The kernel sums p f(x), f(x) = x + exp(-x) - 1, around x = d + L, L the difference of the log sums less
            # that of the maxima, and takes L + exp(-L) - 1 off again, which is what the shift added:
            # sum p f(d + L) = KL + L - 1 + exp(-L).  So its sum's error counts on KL + f(L), and an entry's own error
            # (err, err_q in the exponents) moves its term by |p - q|, or by p + q where |x| >= 1/2.  What is taken off
            # has the slope 1 - exp(-L) in the ratio of the two sums.
            L = abs(float((l.max() - q.max()) - (torch.logsumexp(l, 0) - torch.logsumexp(q, 0)))) + 2e-4
            shifted = math.exp(L) - L - 1                            # f(-L) >= f(L) for L > 0
            far = d.abs() + L >= 0.5
            klt = float(((p - pq).abs() * (err + err_q)).sum()) + (abs(kl) + shifted + math.exp(L) - 1) * (err + err_q + (n + 20) * U) \
                + float((4 * U * (p * d.abs() + p + pq) + (err + err_q) * (p + pq))[far].sum())
            kls[i], tk[i] = kl, klt
        adv, ratio = float(a["adv"][i]), math.exp(float(lp[act]) - float(a["old"][i]))
        free, held = ratio * adv, min(max(ratio, 1 - clip[0]), 1 + clip[1]) * adv
        assert min(abs(ratio - 1 + clip[0]), abs(ratio - 1 - clip[1])) > 1e-3
        rt = ratio * (err + 2 * U * abs(float(lp[act]) - float(a["old"][i])) + 8 * U) * abs(adv)
        value, vt = -min(free, held), max(rt, 4 * U * abs(held))
        g1 = -free if free <= held else 0.0
        loss += w * (value + beta * kl)
        loss_t += abs(w) * (vt + beta * (klt + 4 * U * abs(kl)) + 4 * U * abs(value))
        size += abs(w) * (abs(value) + beta * abs(kl))
        one = torch.zeros_like(p)
        one[act] = 1.0
        g = w * (g1 * (one - p) + torch.where(ok, beta * p * (d - kl), 0.0))
        pt = p * (err + 8 * U)
        gt = abs(w) * (rt * (one + p) + abs(g1) * pt + beta * (pt * (d - kl).abs() + p * (2 * err + klt + 4 * U * (d.abs() + abs(kl))))
                       + 8 * U * (abs(g1) * (one + p) + beta * p * (d - kl).abs()))
        grad[off[i]:off[i + 1]] = torch.where(ok, g, 0.0)
        tg[off[i]:off[i + 1]] = torch.where(ok, gt, 0.0)
    live = grad != 0
    tg = torch.where(live, rounded(tg, grad, dt), tg)
    shape = a["logits"].shape
    loss = torch.tensor(loss)
    return (loss, rounded(torch.tensor(loss_t + 4 * U * size), loss, torch.float32)), (logp, tl + 2 * U * logp.abs()), \
        (kls, tk + 2 * U * kls.abs()), (grad.view(shape), tg.view(shape))


def call_policy(a, clip, beta, logits=None):
    return ops.policy_loss(a["logits"] if logits is None else logits, a["actions"], a["old"], a["adv"],
                           ref_logits=a["ref"], offsets=a["offsets"], mask=a["mask"], weights=a["weights"], clip=clip,
                           kl_coef=beta)


def check_policy(a, clip=(0.2, 0.2), beta=0.1, what=""):
    if a["ref"] is None:
        beta = 0.0
    want = policy_want(a, clip, beta)
    got = call_policy(a, clip, beta)
    logits = a["logits"].detach().requires_grad_()
    with_grad = call_policy(a, clip, beta, logits)
    for x, y in zip(got, with_grad):
        assert torch.equal(x, y.detach()), what
    for name, x, (v, t) in zip(("loss", "logp", "kl"), got, want):
        within(x, v, t, what + " " + name)
    grad = torch.autograd.grad(with_grad.loss, logits, retain_graph=True)[0]
    within(grad, *want[3], what=what + " grad")
    # another upstream gradient, and the same graph once more
    for up in (0.375, 1.0, -3.0):
        again = torch.autograd.grad(with_grad.loss, logits, torch.tensor(up, device="cuda"), retain_graph=True)[0]
        v, t = want[3]
        within(again, v * up, (t + U * v.abs()) * abs(up) + tiny(a["logits"].dtype), what + " grad of upstream %g" % up)
    return got, grad


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("ref", [True, False], ids=["kl", "plain"])
def test_policy_ragged(dtype, ref):
    g = torch.Generator().manual_seed(9)
    lengths = torch.randint(1, 61, (150,), generator=g).tolist() + [1, 1, 2, 63, 64, 65, 128, 129, 257, 1000, 3, 1]
    check_policy(policy_rows(lengths, DT[dtype], ref=ref), what="ragged")
    check_policy(policy_rows(lengths[-20:], DT[dtype], masked=0.5, ref=ref, seed=4), what="ragged and masked")
    check_policy(policy_rows([1], DT[dtype], ref=ref), what="one row of one")


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("dense", [(1, 1), (3, 2), (37, 10), (5, 64), (9, 255), (4, 1000), (3, 4097), (2, 20011), (1, 70003)], ids=str)
def test_policy_dense(dtype, dense):
    check_policy(policy_rows(None, DT[dtype], dense=dense), what="dense")
    check_policy(policy_rows(None, DT[dtype], dense=dense, ref=False, seed=2), what="dense, no reference")
    if dense[1] > 4:
        check_policy(policy_rows(None, DT[dtype], dense=dense, masked=0.4, seed=1), clip=(0.2, 0.28), what="dense and masked")


@pytest.mark.parametrize("dtype", list(DT))
def test_policy_rows_that_count_nothing(dtype):
    """No options, all masked, all -inf, weight 0 over NaN: zeros, and nothing of them anywhere else."""
    a = policy_rows([5, 0, 7, 6, 4, 3], DT[dtype])
    off = a["offsets"]
    a["mask"] = torch.ones_like(a["logits"], dtype=torch.bool)
    a["mask"][off[2]:off[3]] = False
    a["logits"][off[3]:off[4]] = -math.inf
    a["logits"][off[4]:off[5]] = math.nan
    a["weights"][4] = 0.0
    a["actions"][1] = -1
    got, grad = check_policy(a)
    assert got.logp[1:5].tolist() == [0.0] * 4 and got.kl[1:5].tolist() == [0.0] * 4
    assert not bool(grad[off[1]:off[5]].any())
    # the same rows as a table, one that a workgroup a row takes and one whose rows are taken in parts
    for width in (2000, 20000):
        b = policy_rows(None, DT[dtype], dense=(4, width))
        b["mask"] = torch.ones_like(b["logits"], dtype=torch.bool)
        b["mask"][0] = False
        b["logits"][1] = -math.inf
        b["logits"][2] = math.nan
        b["weights"][2] = 0.0
        got, grad = check_policy(b)
        assert not bool(grad[:3].any()) and got.logp[:3].tolist() == [0.0] * 3


def test_policy_long_rows_with_everything_in_one_part():
    """Rows in parts where one part holds all that is legal, or all of the reference's mass."""
    for where in (slice(0, 4000), slice(30000, 34000)):
        a = policy_rows(None, torch.float32, dense=(2, 65536))
        a["mask"] = torch.zeros_like(a["logits"], dtype=torch.bool)
        a["mask"][:, where] = True
        a["actions"] = torch.full((2,), where.start + 7, device="cuda")
        l = torch.where(a["mask"], a["logits"].double(), -math.inf)
        a["old"] = (l.gather(1, a["actions"][:, None])[:, 0] - torch.logsumexp(l, 1) + 0.05).float()
        check_policy(a)
        b = dict(a, mask=None, logits=a["logits"].clone(), ref=a["ref"].clone())
        b["logits"][~a["mask"]] = -math.inf
        b["ref"][:, where] += 9.0                    # the reference's mass moves there; outside it keeps some
        l = b["logits"].double()
        b["old"] = (l.gather(1, a["actions"][:, None])[:, 0] - torch.logsumexp(l, 1) + 0.05).float()
        got = call_policy(b, (0.2, 0.2), 0.1)
        q = torch.log_softmax(b["ref"].double(), 1)
        lp = torch.log_softmax(l, 1)
        kl = (lp.exp() * torch.where(lp > -math.inf, lp - q, 0.0)).sum(1)
        # sums of 4,000 terms with logits of at most 20: see policy_want
        tol = (2 * 4000 + 200) * U
        assert bool(((got.kl.double() - kl).abs() <= tol * (1 + kl)).all())


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("width", [12, 1500, 20001])
def test_policy_infinities_and_lowest_values(dtype, width):
    """-inf and the type's lowest value as masks inside a row; NaN and infinities under the mask."""
    dt = DT[dtype]
    a = policy_rows(None, dt, dense=(3, width))
    keep = a["actions"].clone()
    a["mask"] = torch.ones_like(a["logits"], dtype=torch.bool)
    for i in range(3):
        at = [j for j in range(0, width, 3) if j != int(keep[i])]
        a["mask"][i, at] = False
        a["logits"][i, at] = [math.nan, math.inf, -math.inf][i]
        a["ref"][i, at] = math.nan
    at = [j for j in range(1, width, 3) if all(j != int(k) for k in keep)]
    a["logits"][:, at] = -math.inf
    a["ref"][:, at] = torch.finfo(dt).min
    legal = a["mask"] & (a["logits"] > -math.inf)
    l = torch.where(legal, a["logits"].double(), -math.inf)
    a["old"] = (l.gather(1, keep[:, None])[:, 0] - torch.logsumexp(l, 1) + 0.05).float()
    check_policy(a)
    # the lowest value in place of -inf says the same
    same = dict(a, logits=torch.where(a["logits"] == -math.inf, torch.finfo(dt).min, a["logits"]))
    one, two = call_policy(a, (0.2, 0.2), 0.1), call_policy(same, (0.2, 0.2), 0.1)
    assert all(torch.equal(x, y) for x, y in zip(one, two))
    # a reference that rules out what the policy plays: KL is infinite there, other rows keep theirs
    a["ref"][0, int(keep[0])] = -math.inf
    three = call_policy(a, (0.2, 0.2), 0.1)
    assert float(three.kl[0]) == math.inf and torch.equal(three.kl[1:], one.kl[1:])


@pytest.mark.parametrize("width", [8, 3000, 20001])
def test_policy_bad_rows_are_loud(width):
    a = policy_rows(None, torch.float32, dense=(4, width))
    good = call_policy(a, (0.2, 0.2), 0.1)
    for bad in (-1, width, 2 ** 40):
        b = dict(a, actions=a["actions"].clone())
        b["actions"][2] = bad
        got = call_policy(b, (0.2, 0.2), 0.1)
        assert math.isnan(float(got.loss)) and math.isnan(float(got.logp[2]))
        assert torch.equal(got.logp[[0, 1, 3]], good.logp[[0, 1, 3]])
    r = policy_rows([3, 4, 5], torch.float32)
    for at, v in ((1, -3), (3, 13), (2, 2), (0, -1), (3, 2 ** 40)):
        b = dict(r, offsets=r["offsets"].clone())
        b["offsets"][at] = v
        logits = b["logits"].detach().requires_grad_()
        got = call_policy(b, (0.2, 0.2), 0.1, logits)
        assert math.isnan(float(got.loss.detach())), (at, v)
        torch.autograd.grad(got.loss, logits)
    # a masked action is one that cannot be played: rho is 0
    m = dict(a, mask=torch.ones_like(a["logits"], dtype=torch.bool), adv=torch.ones_like(a["adv"]))
    m["mask"][1, int(a["actions"][1])] = False
    got = call_policy(m, (0.2, 0.2), 0.0)
    assert float(got.logp[1]) == -math.inf and math.isfinite(float(got.loss))


def test_policy_entries_of_no_row():
    """Entries before the first row and behind the last: not read, gradient 0."""
    a = policy_rows([3, 70, 5], torch.float32)
    pad = lambda t: torch.cat([t.new_full((4,), math.nan), t, t.new_full((300,), math.nan)])  # noqa: E731
    b = dict(a, logits=pad(a["logits"]), ref=pad(a["ref"]), offsets=a["offsets"] + 4)
    la, lb = a["logits"].requires_grad_(), b["logits"].requires_grad_()
    # (the list's mean row length picks the kernel's shape, so the two lists' sums have other orders: both are held to
    # the bounds of the same rows)
    want = policy_want(a, (0.2, 0.2), 0.1)
    for l, c in ((la, a), (lb, b)):
        got = call_policy(c, (0.2, 0.2), 0.1, l)
        g = torch.autograd.grad(got.loss, l)[0]
        for name, x, (v, t) in zip(("loss", "logp", "kl"), got, want):
            within(x.detach(), v, t, name)
        if c is b:
            assert not bool(g[:4].any()) and not bool(g[82:].any())
            g = g[4:82]
        within(g, *want[3], what="grad")
    none = ops.policy_loss(lb, a["actions"][:0], a["old"][:0], a["adv"][:0], offsets=a["offsets"][:1])
    assert float(none.loss.detach()) == 0.0 and none.logp.shape == (0,)
    assert not bool(torch.autograd.grad(none.loss, lb)[0].any())
    assert float(ops.policy_loss(la.detach().view(1, -1)[:0], a["actions"][:0], a["old"][:0], a["adv"][:0]).loss) == 0.0


def kl_want(l, q):
    """(KL of the softmaxes of rows l against q, gradient of it in l, their tolerances), in 64 bits.

    An entry's exponential is off by e = (8 max|l| + 3) u: two differences and the product with log2 e round, |l - max|
    <= 2 max|l|.  A sum adds 100 u: at most 64 entries a lane, then 6 shuffles and 16 waves.  With x = d + L, L the log
    of the sums' ratio (off by 2 e + 2 * 100 u + 5 u |L|), the two sums that KL comes from are off by e and 100 u of
    sum p (|x| + 2), and by what e makes of x itself, e (1 + sum q / sum p <= 3)."""
    lp, lq = torch.log_softmax(l, 1), torch.log_softmax(q, 1)
    p = lp.exp()
    d = torch.where(p > 0, lp - lq, 0.0)
    kl = (p * d).sum(1)
    real = torch.where(p > 0, l, 0.0)
    e = (8 * torch.maximum(real.abs().amax(1), q.abs().amax(1)) + 3) * U
    top = l.amax(1) - q.amax(1)
    big = (top - (torch.logsumexp(l, 1) - torch.logsumexp(q, 1))).abs()
    err_l = 2 * e + (200 + 5 * big) * U
    err = (2 * e + 100 * U) * (4 + (p * d.abs()).sum(1) + 2 * big) + 2 * err_l
    grad = p * (d - kl[:, None])
    err_g = p * (2 * e + 100 * U)[:, None] * (d - kl[:, None]).abs() + p * (err_l + err)[:, None] + 8 * U * p * (d.abs() + kl[:, None])
    return kl, grad, err, err_g


def check_kl(logits, ref, want=None):
    rows = logits.shape[0]
    l = logits.clone().requires_grad_()
    zero = torch.zeros(rows, device="cuda")
    got = ops.policy_loss(l, zero.long(), zero, zero, ref_logits=ref, weights=zero + 1.0, kl_coef=1.0)
    grad = torch.autograd.grad(got.loss, l)[0]
    kl, g, err, err_g = want or kl_want(logits.double(), ref.double())
    within(got.kl, kl, rounded(err, kl, torch.float32), "kl")
    within(grad, g, rounded(err_g, g, logits.dtype), "grad")


KL_SHAPES = [(3, 40), (3, 200), (3, 1500), (3, 6001), (130, 16500), (3, 20001), (2, 70001)]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("shape", KL_SHAPES, ids=str)
def test_policy_reference_much_flatter(shape, dtype):
    """A policy that is sure of one option, a reference that is of none."""
    g = torch.Generator().manual_seed(3)
    l = torch.randn(shape, generator=g)
    l[:, shape[1] // 2] = 18.0
    r = 0.1 * torch.randn(shape, generator=g)
    check_kl(l.to(DT[dtype]).cuda(), r.to(DT[dtype]).cuda())
    check_kl(r.to(DT[dtype]).cuda(), l.to(DT[dtype]).cuda())


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("shape", KL_SHAPES, ids=str)
def test_policy_entries_far_below_the_others(shape, dtype):
    """Stretches of a row, whole parts of a long one among them, that have no weight in it, with and without the
    reference's: what they hold is a number, and counts nothing."""
    dt = DT[dtype]
    g = torch.Generator().manual_seed(4)
    l, r = torch.randn(shape, generator=g).to(dt).cuda(), torch.randn(shape, generator=g).to(dt).cuda()
    half = shape[1] // 2
    for low in (-720.0, -1000.0, torch.finfo(dt).min):
        a = l.clone()
        a[:, half:] = low
        kl, grad, err, err_g = kl_want(torch.where(a < -700, -math.inf, a.double()), r.double())
        check_kl(a, r, (kl, grad, err, err_g))
        b = r.clone()
        b[:, half:] = -math.inf                      # ruled out by the reference too
        want = kl_want(a[:, :half].double(), b[:, :half].double())
        pad = lambda t: torch.cat([t, t.new_zeros(shape[0], shape[1] - half)], 1)  # noqa: E731
        if low < -800:                               # (exp(-720) is no 0 to a row in parts)
            check_kl(a, b, (want[0], pad(want[1]), want[2], pad(want[3])))


def test_policy_strides_and_types():
    a = policy_rows(None, torch.float32, dense=(6, 700), masked=0.3)
    want = call_policy(a, (0.2, 0.2), 0.1)
    wide = lambda t, pad: torch.cat([t, t.new_zeros(6, pad)], 1)[:, :700]  # noqa: E731
    b = dict(a, logits=wide(a["logits"], 9), ref=wide(a["ref"], 3), mask=wide(a["mask"], 1), actions=a["actions"].int())
    assert all(torch.equal(x, y) for x, y in zip(want, call_policy(b, (0.2, 0.2), 0.1)))
    c = dict(a, logits=a["logits"].t().contiguous().t(), ref=a["ref"].t().contiguous().t())
    assert all(torch.equal(x, y) for x, y in zip(want, call_policy(c, (0.2, 0.2), 0.1)))
    d = dict(a, weights=None)
    e = dict(a, weights=torch.full((6,), 1 / 6, device="cuda"))
    assert torch.equal(call_policy(d, 0.2, 0.1).loss, call_policy(e, 0.2, 0.1).loss)


def test_policy_gradient_against_differences():
    a = policy_rows([5, 30, 64, 200, 2], torch.float32)
    l = a["logits"].requires_grad_()
    grad = torch.autograd.grad(call_policy(a, (0.2, 0.2), 0.3, l).loss, l)[0].double()
    g = torch.Generator().manual_seed(1)
    h = 2.0 ** -6
    for _ in range(4):
        v = torch.randn(l.shape, generator=g).cuda()
        v = v / v.abs().max()
        up, down = (float(call_policy(a, (0.2, 0.2), 0.3, l.detach() + s * h * v).loss) for s in (1, -1))
        # the third derivative along v (|v| <= 1) is at most 8 sum w (|A| rho + beta (2 + KL)); the loss is 2^-21 exact
        third = 8 * float((a["weights"] * (a["adv"].abs() * 1.3 + 1.0)).sum()) * h * h / 6
        assert abs((up - down) / (2 * h) - float((grad * v.double()).sum())) <= third + 2.0 ** -21 * 4 / h


# ---- gradient norm ------------------------------------------------------------------

def clip_want(grads, max_norm, out_types):
    d = [g.detach().double().cpu() for g in grads]
    norm = math.sqrt(sum(float((t * t).sum()) for t in d))
    c = min(1.0, max_norm / (norm + 1e-6))
    # c is one fp32 number (u) of a sum in fp64; a product of fp32 (u), rounded to its type
    return norm, [(t * c, rounded(4 * U * (t * c).abs(), t * c, o)) for t, o in zip(d, out_types)]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("sizes", [[1], [3, 0, 5], [4096, 1, 2047, 8, 33], [100003], [17] * 230, [70000, 12, 3_000_001]], ids=lambda s: "%dx%d" % (len(s), s[0]))
def test_clip_sizes(dtype, sizes):
    dt = DT[dtype]
    g = torch.Generator().manual_seed(5)
    grads = [(torch.randn(n, generator=g) * 0.1).to(dt).cuda() for n in sizes]
    full = math.sqrt(sum(float(t.double().square().sum()) for t in grads))
    for max_norm in (0.3 * full, 2 * full, math.inf):
        norm, want = clip_want(grads, max_norm, [dt] * len(sizes))
        got = [t.clone() for t in grads]
        n = ops.clip_grad_norm(got, max_norm)
        assert abs(float(n) - norm) <= 2 * U * norm
        assert torch.equal(n, ops.grad_norm(grads))
        for x, (v, t) in zip(got, want):
            within(x, v, t, "in place")
        if max_norm > full:
            assert all(torch.equal(x, y) for x, y in zip(got, grads))
        flat = torch.full((sum(sizes) + 2,), math.nan, device="cuda")
        out = list(flat[1:-1].split(sizes))
        assert torch.equal(ops.clip_grad_norm(grads, max_norm, out=out), n)
        norm, want = clip_want(grads, max_norm, [torch.float32] * len(sizes))
        for x, (v, t) in zip(out, want):
            within(x, v, t, "into fp32")
        assert math.isnan(float(flat[0])) and math.isnan(float(flat[-1]))


def test_clip_mixed_types_and_alignment():
    g = torch.Generator().manual_seed(6)
    grads = []
    for i, n in enumerate([5, 1000, 77, 4099, 260]):
        base = torch.randn(n + 8, generator=g).to(list(DT.values())[i % 3]).cuda()
        grads.append(base[i + 1:i + 1 + n])
    norm, want = clip_want(grads, 3.0, [t.dtype for t in grads])
    got = [torch.cat([t.new_zeros(3), t])[3:] for t in grads]
    assert abs(float(ops.clip_grad_norm(got, 3.0)) - norm) <= 2 * U * norm
    for x, (v, t) in zip(got, want):
        within(x, v, t, "mixed")


def test_clip_strided_gradients():
    a, b = torch.randn(40, 30, device="cuda"), torch.randn(9, 16, device="cuda")
    grads = [a.t(), b[:, ::2], torch.ones(1, device="cuda").expand(50)]
    norm, want = clip_want(grads, 1.0, [torch.float32] * 3)
    out = [torch.empty(t.shape, device="cuda") for t in grads]
    assert abs(float(ops.clip_grad_norm(grads, 1.0, out=out)) - norm) <= 2 * U * norm
    for x, (v, t) in zip(out, want):
        within(x, v, t, "out")
    rest = b[:, 1::2].clone()
    norm, want = clip_want(grads[:2], 1.0, [torch.float32] * 2)
    ops.clip_grad_norm(grads[:2], 1.0)
    for x, (v, t) in zip(grads, want):
        within(x, v, t, "in place")
    assert torch.equal(b[:, 1::2], rest)


def test_clip_range():
    """Squares past fp32's range on either side; infinities and NaN as torch's clip_grad_norm_ treats them."""
    for s in (1e30, 1e-30):
        t = [torch.full((300,), s, device="cuda"), torch.full((100,), s, device="cuda").bfloat16()]
        norm, want = clip_want(t, s, [torch.float32, torch.bfloat16])
        assert abs(float(ops.clip_grad_norm(t, s)) - norm) <= 2 * U * norm
        if s > 1:
            within(t[0], *want[0], what="large")
    for v in (math.inf, math.nan):
        t = torch.ones(70, device="cuda")
        t[3] = v
        p = torch.nn.Parameter(torch.zeros(70, device="cuda"))
        p.grad = t.clone()
        torch.nn.utils.clip_grad_norm_([p], 1.0)
        with pytest.raises(RuntimeError, match="not finite"):
            ops.clip_grad_norm([t], 1.0, error_if_nonfinite=True)
        assert float(t[0]) == 1.0
        ops.clip_grad_norm([t], 1.0)
        assert torch.equal(t.isnan(), p.grad.isnan()) and torch.equal(t.nan_to_num(), p.grad.nan_to_num())
    t = torch.ones(4, device="cuda")
    ops.clip_grad_norm([t], 0.0)
    assert not bool(t.any())


def test_clip_same_from_run_to_run():
    g = [torch.randn(1_000_003, device="cuda"), torch.randn(77, device="cuda")]
    assert len({float(ops.grad_norm(g)) for _ in range(5)}) == 1


def test_many_short_rows():
    """More rows than one workgroup sums: the loss is their weighted sum all the same."""
    n = 300_001
    g = torch.Generator().manual_seed(0)
    l = (torch.randn(n, 3, generator=g) * 2).cuda()
    act = torch.randint(0, 3, (n,), generator=g).cuda()
    old = torch.log_softmax(l.double(), 1).gather(1, act[:, None])[:, 0].float() + 0.05
    adv = torch.randn(n, generator=g).cuda()
    got = ops.policy_loss(l, act, old, adv)
    lp = torch.log_softmax(l.double(), 1).gather(1, act[:, None])[:, 0]
    ratio = torch.exp(lp - old.double())
    value = -torch.minimum(ratio * adv, ratio.clamp(0.8, 1.2) * adv)
    # each row's ratio is off by what its log probability is (3 exponentials, logits of at most 12), the weight 1 / n by u
    tol = float(((200 * U + U) * value.abs()).sum()) / n + U * abs(float(value.mean()))
    assert abs(float(got.loss) - float(value.mean())) <= tol


def test_no_second_derivatives():
    """Asked for, they are refused: never left out in silence."""
    x, w, b, r, dy = linear_inputs(5, 6, 7, torch.float32, "gelu", True, False)
    y = ops.linear(x.requires_grad_(), w, b, activation="gelu")
    with pytest.raises(RuntimeError, match="first derivatives only"):
        torch.autograd.grad(y.sum(), x, create_graph=True)
    a = policy_rows([4, 5], torch.float32)
    l = a["logits"].requires_grad_()
    with pytest.raises(RuntimeError, match="first derivatives only"):
        torch.autograd.grad(call_policy(a, (0.2, 0.2), 0.1, l).loss, l, create_graph=True)


def test_offsets_past_32_bits():
    """Elements behind the 2^31st: the last rows of long inputs against the same rows alone."""
    M, K, N = 540_000, 4096, 24
    x = torch.zeros(M, K, dtype=torch.bfloat16, device="cuda")
    w, tail = torch.randn(N, K, device="cuda").bfloat16(), torch.randn(300, K, device="cuda").bfloat16()
    x[-300:] = tail
    want = tail.double() @ w.double().t()
    tol = rounded((K + 4) * U * (tail.double().abs() @ w.double().abs().t()), want, torch.bfloat16)
    y = ops.linear(x, w)
    within(y[-300:], want, tol, "linear")
    assert not bool(y[:-300].any())
    ws = w.clone().requires_grad_()
    dy = torch.zeros(M, N, dtype=torch.bfloat16, device="cuda")
    dy[-1] = 1.0
    dw = torch.autograd.grad(ops.linear(x, ws), ws, dy)[0]
    assert torch.equal(dw, tail[-1:].expand(N, K))
    del x, y, dy
    a = policy_rows(None, torch.bfloat16, dense=(3, 32768))
    l = torch.zeros(66_000, 32768, dtype=torch.bfloat16, device="cuda")
    l[-3:] = a["logits"]
    wide = dict(a, logits=l, ref=None, mask=None, weights=torch.zeros(66_000, device="cuda"))
    wide["weights"][-3:] = a["weights"]
    for k in ("actions", "old", "adv"):
        wide[k] = torch.zeros(66_000, dtype=a[k].dtype, device="cuda")
        wide[k][-3:] = a[k]
    want = policy_want(dict(a, ref=None), (0.2, 0.2), 0.0)
    l.requires_grad_()
    got = call_policy(wide, (0.2, 0.2), 0.0, l)
    within(got.loss.detach(), *want[0], what="loss")
    within(got.logp[-3:], *want[1], what="logp")
    g = torch.autograd.grad(got.loss, l)[0]
    within(g[-3:], *want[3], what="grad")
    assert not bool(g[:-3].any())
    del l, g, got, wide
    t = torch.zeros(2 ** 31 + 5000, dtype=torch.bfloat16, device="cuda")
    t[-1], t[-4000] = 3.0, 4.0
    assert float(ops.clip_grad_norm([t], 1.0)) == 5.0
    assert abs(float(t[-1]) - 0.6) <= 0.6 * 2 ** -8 and abs(float(t[-4000]) - 0.8) <= 0.8 * 2 ** -8
    assert not bool(t[:-4000].any())


def test_clip_by_an_infinite_norm():
    """max_norm inf clips nothing, and an infinite norm against it makes NaN, as torch's clip_grad_norm_ has it."""
    for v in (1.0, math.inf, math.nan):
        t = torch.ones(70, device="cuda")
        t[3] = v
        p = torch.nn.Parameter(torch.zeros(70, device="cuda"))
        p.grad = t.clone()
        torch.nn.utils.clip_grad_norm_([p], math.inf)
        ops.clip_grad_norm([t], math.inf)
        assert torch.equal(t.isnan(), p.grad.isnan()) and torch.equal(t.nan_to_num(), p.grad.nan_to_num())


def test_more_workgroups_than_one_dimension_takes():
    """Past 2^21 workgroups a launch goes on in its grid's next dimension."""
    M = (1 << 26) + 100
    x = torch.randn(M, 1, device="cuda").bfloat16()
    for N in (1, 131):                               # 32 x 32 tiles, 64 x 64 tiles
        w = torch.randn(N, 1, device="cuda").bfloat16()
        y = ops.linear(x, w)
        for at in (0, (1 << 26) - 4000, M - 5000):   # a product of two bf16 numbers is exact in fp32
            rows = slice(at, at + 5000)
            assert torch.equal(y[rows], (x[rows].float() * w.float().t()).bfloat16())
        del y
    del x
    N = (1 << 25) + 1000
    g = torch.Generator(device="cuda").manual_seed(0)
    l = torch.randn(N, 2, generator=g, device="cuda").half()
    act = torch.randint(0, 2, (N,), generator=g, device="cuda")
    zero = torch.zeros(N, device="cuda")
    one = torch.full((N,), 2.0 ** -10, device="cuda")
    l.requires_grad_()
    got = ops.policy_loss(l, act, zero, zero + 1.0, weights=one, clip=(1.0, 1.0))
    grad = torch.autograd.grad(got.loss, l)[0]
    total = 0.0
    for at in range(0, N, 1 << 22):
        rows = slice(at, min(N, at + (1 << 22)))
        p = torch.softmax(l[rows].detach().double(), 1).gather(1, act[rows][:, None])[:, 0]
        total += float(p.sum())
        # two exponentials, a logarithm of their sum, logits of at most 8
        assert bool(((got.logp[rows].double() - p.log()).abs() <= 100 * U).all())
        want = 2.0 ** -10 * p * (1 - p)              # rho = p (old 0): -w p (1 - p) where chosen, w p (1 - p) where not
        sign = torch.ones(len(p), 2, device="cuda", dtype=torch.float64).scatter_(1, act[rows][:, None], -1.0)
        want = want[:, None] * sign
        assert bool(((grad[rows].double() - want).abs() <= want.abs() * (2.0 ** -11 + 300 * U) + 2.0 ** -25).all())
    assert abs(float(got.loss.detach()) + total * 2.0 ** -10) <= 150 * U * total * 2.0 ** -10


def test_autograd_manners():
    """What torch's own nodes keep to: a graph used twice, saved tensors written over, hooks that move them to the host,
    undefined gradients, backward passes on two threads at once, no forward mode."""
    x, w, b, r, dy = linear_inputs(37, 50, 41, torch.float32, "silu", True, True)
    leaves = [t.requires_grad_() for t in (x, w, b, r)]
    want = torch.autograd.grad(ops.linear(*leaves, activation="silu"), leaves, dy)
    a = policy_rows([4, 9, 30], torch.float32)
    l = a["logits"].requires_grad_()
    want_l = torch.autograd.grad(call_policy(a, (0.2, 0.2), 0.1, l).loss, l)[0]
    # once without retain_graph
    for make, of, up in ((lambda: ops.linear(*leaves, activation="silu"), leaves, dy),
                         (lambda: call_policy(a, (0.2, 0.2), 0.1, l).loss, [l], None)):
        y = make()
        torch.autograd.grad(y, of, up)
        with pytest.raises(RuntimeError, match="second time"):
            torch.autograd.grad(y, of, up)
    # what a node saved, written over: y itself for relu, x and w, the logits
    y = ops.linear(x, w, b, activation="relu")
    y.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, w, dy)
    for at in (0, 1):
        given = [t.detach().clone().requires_grad_() for t in (x, w)]
        y = ops.linear(*given)
        with torch.no_grad():
            given[at].add_(1.0)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(y, given[1 - at], dy)
    m = l.detach().clone().requires_grad_()
    loss = call_policy(a, (0.2, 0.2), 0.1, m).loss
    with torch.no_grad():
        m.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(loss, m)
    # saved on the host meanwhile
    with torch.autograd.graph.save_on_cpu():
        y, loss = ops.linear(*leaves, activation="silu"), call_policy(a, (0.2, 0.2), 0.1, l).loss
    assert all(torch.equal(g, v) for g, v in zip(torch.autograd.grad(y, leaves, dy), want))
    assert torch.equal(torch.autograd.grad(loss, l)[0], want_l)
    # a checkpointed segment works its forward pass out again
    y = torch.utils.checkpoint.checkpoint(lambda *t: ops.linear(*t, activation="silu"), *leaves, use_reentrant=False)
    assert all(torch.equal(g, v) for g, v in zip(torch.autograd.grad(y, leaves, dy), want))
    # the statistics have no gradient; one of several outputs unused
    got = call_policy(a, (0.2, 0.2), 0.1, l)
    assert got.loss.requires_grad and not got.logp.requires_grad and not got.kl.requires_grad
    assert torch.equal(torch.autograd.grad(got.loss + ops.linear(x, w).sum() * 0.0, l)[0], want_l)
    # one graph, two threads
    y, loss = ops.linear(*leaves, activation="silu"), call_policy(a, (0.2, 0.2), 0.1, l).loss
    out = [None] * 8

    def back(i):
        out[i] = torch.autograd.grad(y, leaves, dy, retain_graph=True) + torch.autograd.grad(loss, l, retain_graph=True)

    threads = [threading.Thread(target=back, args=(i,)) for i in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    torch.cuda.synchronize()
    assert all(g is not None and all(torch.equal(p, q) for p, q in zip(g, want + (want_l,))) for g in out)
    # leaves accumulate
    for t in leaves:
        t.grad = None
    for _ in range(2):
        ops.linear(*leaves, activation="silu").backward(dy)
    assert all(torch.equal(t.grad, 2 * v) for t, v in zip(leaves, want))
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x.detach(), torch.ones_like(x))
        with pytest.raises(RuntimeError, match="no forward-mode"):
            ops.linear(dual, w)
    with torch.inference_mode():
        y = ops.linear(*leaves, activation="silu")
        assert y.is_inference() and not y.requires_grad
        t = torch.ones(30, device="cuda")
        assert abs(float(ops.clip_grad_norm([t], 1.0)) - math.sqrt(30.0)) <= 4 * U * 6 and float(t[0]) < 1.0
    # a clipped gradient's version goes up, and a graph that saved it notices
    t = torch.ones(30, device="cuda")
    y = (torch.ones(30, device="cuda", requires_grad=True) * t).sum()
    ops.clip_grad_norm([t], 1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


# ---- together ---------------------------------------------------------------------------

def step_of_a_policy(params, x, opts, a, max_norm, lib):
    """Two layers with a residual, the policy loss over ragged options, gradients, clipping: (loss, norm, gradients)."""
    w1, b1, w2, b2 = params
    h = lib.linear(x, w1, b1, activation="silu")
    h = lib.linear(h, w1, b1, residual=h, activation="gelu")
    logits = lib.linear(h, w2, b2)[:, 0]
    got = lib.policy_loss(logits, a["actions"], a["old"], a["adv"], ref_logits=a["ref"], offsets=a["offsets"], clip=0.2, kl_coef=0.2)
    grads = torch.autograd.grad(got.loss, params)
    return got.loss.detach(), lib.clip_grad_norm(grads, max_norm), grads


class Plain:
    """The same calls in 64 bits."""

    @staticmethod
    def linear(x, w, b, residual=None, activation="none"):
        y = ACT[activation][0](x @ w.t() + b) if activation != "none" else x @ w.t() + b
        return y if residual is None else y + residual

    @staticmethod
    def policy_loss(logits, actions, old, adv, ref_logits, offsets, clip, kl_coef):
        import types
        off, loss = offsets.tolist(), 0.0
        for i in range(len(actions)):
            lp = torch.log_softmax(logits[off[i]:off[i + 1]], 0)
            lq = torch.log_softmax(ref_logits[off[i]:off[i + 1]].double(), 0)
            r = torch.exp(lp[actions[i]] - old[i].double())
            A = adv[i].double()
            loss = loss - torch.minimum(r * A, r.clamp(1 - clip, 1 + clip) * A) + kl_coef * (lp.exp() * (lp - lq)).sum()
        return types.SimpleNamespace(loss=loss / len(actions))

    @staticmethod
    def clip_grad_norm(grads, max_norm):
        norm = math.sqrt(sum(float(g.square().sum()) for g in grads))
        for g in grads:
            g *= min(1.0, max_norm / (norm + 1e-6))
        return torch.tensor(norm)


def step_inputs(dt):
    g = torch.Generator().manual_seed(11)
    a = policy_rows([4, 9, 1, 30, 17, 60, 2, 11], torch.float32)
    n = a["logits"].shape[0]
    x = torch.randn(n, 40, generator=g).cuda().to(dt)
    params = [(torch.randn(s, generator=g) * c).cuda().to(dt) for s, c in (((40, 40), 0.15), ((40,), 0.1), ((1, 40), 0.15), ((1,), 0.1))]
    a["ref"] = (0.3 * torch.randn(n, generator=g)).cuda().to(dt)
    w1, b1, w2, b2 = (p.double() for p in params)
    h = Plain.linear(x.double(), w1, b1, activation="silu")
    h = Plain.linear(h, w1, b1, residual=h, activation="gelu")
    l, off = Plain.linear(h, w2, b2)[:, 0], a["offsets"].tolist()
    lp = torch.stack([torch.log_softmax(l[off[i]:off[i + 1]], 0)[a["actions"][i]] for i in range(8)])
    a["old"] = (lp + torch.tensor([0.05, -0.05, 0.1, -0.1, 0.3, -0.3, 0.02, 0.0]).cuda()).float()
    return params, x, a


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_training_step_together(dtype):
    """Norm-wise: each of the ~6 roundings to the type on a gradient's way costs at most one half step of its own
    size, times the products' condition (|w| |x| against |w x|: at most 4 here, checked in 64 bits below)."""
    params, x, a = step_inputs(DT[dtype])
    leaves = [p.clone().requires_grad_() for p in params]
    loss, norm, grads = step_of_a_policy(leaves, x, None, a, 0.05, ops)
    exact = [p.double().requires_grad_() for p in params]
    want, wnorm, wgrads = step_of_a_policy(exact, x.double(), None, a, 0.05, Plain)
    e = 64 * half_step(DT[dtype]) if dtype == "bf16" else 512 * U
    assert float(wnorm) > 0.05
    assert abs(float(loss) - float(want)) <= e * (1 + abs(float(want)))
    assert abs(float(norm) - float(wnorm)) <= e * float(wnorm)
    for g, w in zip(grads, wgrads):
        assert float((g.double() - w).norm()) <= e * float(w.norm()) + e * 0.05


def test_training_step_in_a_graph():
    """Captured once and replayed with new inputs, eager work between the replays; an eager graph of the same leaves stays alive."""
    params, x, a = step_inputs(torch.float32)
    leaves = [p.clone().requires_grad_() for p in params]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step_of_a_policy(leaves, x, None, a, 0.05, ops)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step_of_a_policy(leaves, x, None, a, 0.05, ops)
    for k in range(3):
        with torch.no_grad():
            x.mul_(0.9)
            leaves[2].mul_(1.05)
        want = step_of_a_policy(leaves, x, None, a, 0.05, ops)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        for p, q in zip(got[2], want[2]):
            assert torch.equal(p, q), k


def test_capture_beside_an_eager_graph_is_refused():
    x, w, b, r, dy = linear_inputs(37, 50, 41, torch.float32, "silu", True, False)
    a = policy_rows([4, 9, 30], torch.float32)
    w.requires_grad_()
    l = a["logits"].requires_grad_()
    want = torch.autograd.grad(ops.linear(x, w, b), w, dy)[0]
    eager = ops.linear(x, w), call_policy(a, (0.2, 0.2), 0.1, l).loss
    torch.cuda.synchronize()
    for back in (lambda: torch.autograd.grad(ops.linear(x, w, b), w, dy),
                 lambda: torch.autograd.grad(call_policy(a, (0.2, 0.2), 0.1, l).loss, l)):
        with pytest.raises(RuntimeError, match="eager graph of the same leaves"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                back()
        torch.cuda.synchronize()
    del eager
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(ops.linear(x, w, b), w, dy)[0]
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_two_streams_at_once():
    """Two steps on two streams, one after another from the host, each with its own workspaces."""
    params, x, a = step_inputs(torch.float32)
    leaves = [p.clone().requires_grad_() for p in params]
    want = step_of_a_policy(leaves, x, None, a, 0.05, ops)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(step_of_a_policy(leaves, x, None, a, 0.05, ops))
    torch.cuda.synchronize()
    for g in got:
        assert torch.equal(g[0], want[0]) and all(torch.equal(p, q) for p, q in zip(g[2], want[2]))
