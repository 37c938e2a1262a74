"""Measured cases of the training and serving operators (citadels_self_play_amd.ops):
the linear layer with its epilogue, the clipped policy loss and the global
gradient norm.  Plain forms are elementary torch operations in 32 bits."""
import math
import random

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
# ValueOnlyNN(418, 512)'s parameters in module order (weights and biases of fc1, bn1, fc2, bn2, fc3, fc4)
VALUE_NET = [512 * 418, 512, 512, 512, 256 * 512, 256, 256, 256, 128 * 256, 128, 6 * 128, 6]


# ---- cases --------------------------------------------------------------------

def linear_case(M, K, N, dtype, act, bias, residual, train, **more):
    return dict(op="linear", M=M, K=K, N=N, dtype=dtype, act=act, bias=bias, residual=residual, train=train, **more)


def rows_case(rows, longest, dtype, ref, train, **more):
    return dict(op="policy", layout="ragged", rows=rows, longest=longest, dtype=dtype, ref=ref, mask=False,
                weights=False, train=train, **more)


def dense_case(rows, width, dtype, ref, mask, weights, train, **more):
    return dict(op="policy", layout="dense", rows=rows, width=width, dtype=dtype, ref=ref, mask=mask,
                weights=weights, train=train, **more)


def clip_case(tensors, elements, dtype, out, **more):
    return dict(op="clip", tensors=tensors, elements=elements, dtype=dtype, out=out, **more)


def listed():
    return [
        # the value net's first layer in its trainer's default batch of 64: latency of a training step
        linear_case(64, 418, 512, "fp32", "relu", True, False, True, name="fc1 train, batch 64"),
        # the same layer over the leaf rows of 4,096 searches: serving
        linear_case(4096, 418, 512, "fp32", "relu", True, False, False, name="fc1 serve, 4096 rows"),
        # the second layer in the self-play loop's batches of 2,048
        linear_case(2048, 512, 256, "fp32", "relu", True, False, True, name="fc2 train, batch 2048"),
        # a wide block's product with its residual, a long batch of tokens: throughput of a training step
        linear_case(8192, 4096, 4096, "bf16", "gelu", True, True, True, name="block train, bf16"),
        # one token through a wide layer: the weight's bytes are what there is to do
        linear_case(1, 4096, 16384, "bf16", "silu", True, False, False, name="one token, bf16"),
        # nothing a multiple of anything: 2-byte rows that start off every alignment
        linear_case(1023, 2051, 1537, "fp16", "silu", True, True, True, name="odd sizes, fp16"),
        # a trainer's batch of 64 positions, up to 60 legal options each: latency
        rows_case(64, 60, "fp32", True, True, name="options, 64 positions"),
        # the options of a whole self-play round in one step
        rows_case(65536, 60, "fp32", True, True, name="options, 65536 positions"),
        # rows of a large action table, padded batch, reference policy beside: throughput of a training step
        dense_case(4096, 32768, "bf16", True, False, True, True, name="tokens train, bf16"),
        # an odd width with illegal entries masked, evaluated only
        dense_case(509, 50001, "bf16", False, True, False, False, name="masked eval, odd width"),
        # the value net's own gradients: latency
        clip_case(len(VALUE_NET), sum(VALUE_NET), "fp32", "fp32", net=True, name="value net gradients"),
        # many 16-bit gradients into flat 32-bit masters, which start at any element
        clip_case(290, 400_000_000, "bf16", "fp32", net=False, name="290 tensors to masters"),
    ]


def spread(rng, low, high):
    """A whole number of [low, high], even over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5)))))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "policy", "policy", "clip"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if kind == "linear":
        M, K, N = spread(rng, 1, 8192), spread(rng, 64, 4096), spread(rng, 6, 16384)
        while M * K * N > 8192 * 4096 * 4096:
            M = max(1, M // 2)
        return linear_case(M, K, N, dtype, rng.choice(["none", "relu", "gelu", "silu"]), rng.random() < 0.8,
                           rng.random() < 0.4, rng.random() < 0.6)
    if kind == "policy" and rng.random() < 0.4:
        return rows_case(spread(rng, 1, 65536), spread(rng, 2, 60), dtype, rng.random() < 0.7, rng.random() < 0.7)
    if kind == "policy":
        rows, width = spread(rng, 1, 8192), spread(rng, 16, 131072)
        while rows * width > 4096 * 32768:
            rows = max(1, rows // 2)
        return dense_case(rows, width, dtype, rng.random() < 0.6, rng.random() < 0.4, rng.random() < 0.5,
                          rng.random() < 0.7)
    return clip_case(spread(rng, 1, 400), spread(rng, 10_000, 400_000_000), dtype, rng.choice(["fp32", dtype]),
                     net=False)


def tensor_sizes(case):
    """The element counts of a clip case's tensors: matrices of many sizes with small vectors between."""
    if case["net"]:
        return list(VALUE_NET)
    n, total = case["tensors"], case["elements"]
    rng = random.Random(n * 1_000_003 + total)
    share = [rng.random() ** 2 + 0.05 if k % 3 == 0 else 0.002 * rng.random() for k in range(n)]
    sizes = [max(1, int(total * s / sum(share))) for s in share]
    sizes[0] += max(0, total - sum(sizes))
    return sizes


def row_lengths(case):
    """The ragged rows' option counts: most short, none empty in a batch that is trained on."""
    rng = random.Random(case["rows"] * 1009 + case["longest"])
    return [min(case["longest"], 1 + int(rng.expovariate(4.0 / case["longest"]))) for _ in range(case["rows"])]


# ---- inputs -------------------------------------------------------------------

def prepare_linear(case, gen):
    M, K, N, dt = case["M"], case["K"], case["N"], DTYPES[case["dtype"]]
    r = dict(device="cuda", generator=gen)
    bound = 1.0 / math.sqrt(K)
    x = torch.randn(M, K, **r)
    w = (torch.rand(N, K, **r) * 2 - 1) * bound
    b = (torch.rand(N, **r) * 2 - 1) * bound if case["bias"] else None
    if case["act"] == "relu":
        # relu's gradient jumps at z = 0, where the order of a sum decides.  Game features are small whole numbers;
        # with weights on a grid (and the bias half a step off it) every z is exact in 32 bits and none is 0.
        x = torch.randint(0, 9, (M, K), **r).float() * (torch.rand(M, K, **r) < 0.5)
        w = torch.round(w * 4096) / 4096
        b = (torch.round(b * 4096).clamp(-60, 60) + 0.5) / 4096 if b is not None else None   # 8 bits hold these
        if b is None:
            x[:, 0], w[:, 0] = 1.0, (torch.round(w[:, 0] * 4096).clamp(-60, 60) + 0.5) / 4096
    s = {"x": x.to(dt), "w": w.to(dt), "b": None if b is None else b.to(dt), "act": case["act"], "train": case["train"],
         "res": torch.randn(M, N, **r).to(dt) if case["residual"] else None,
         "dy": (torch.randn(M, N, **r) * 0.01).to(dt) if case["train"] else None}
    if case["train"]:
        s["leaves"] = [t.requires_grad_() for t in (s["x"], s["w"], s["b"], s["res"]) if t is not None]
    return s


def prepare_policy(case, gen):
    N, dt = case["rows"], DTYPES[case["dtype"]]
    r = dict(device="cuda", generator=gen)
    s = {"clip": (0.2, 0.2), "kl_coef": 0.05 if case["ref"] else 0.0, "train": case["train"], "mask": None, "ref": None,
         "offsets": None, "weights": None, "longest": case.get("longest")}
    if case["layout"] == "ragged":
        offsets = torch.zeros(N + 1, dtype=torch.int64)
        offsets[1:] = torch.tensor(row_lengths(case)).cumsum(0)
        s["offsets"] = offsets.cuda()
        shape = (int(offsets[-1]),)
    else:
        shape = (N, case["width"])
    logits = torch.randn(shape, **r) * 2
    s["logits"] = logits.to(dt)
    if case["ref"]:
        s["ref"] = (logits + 0.3 * torch.randn(shape, **r)).to(dt)
    del logits
    if case["mask"]:
        s["mask"] = torch.rand(shape, **r) < 0.7
        s["mask"][:, 3] = True
    x, legal = padded(s, s["logits"])
    x = torch.where(legal, x.float(), -math.inf)
    noise = torch.rand(x.shape, **r).clamp_(1e-7, 1 - 1e-7)
    s["actions"] = (x - torch.log(-torch.log(noise))).argmax(1)          # a draw from the softmax
    lp = x.gather(1, s["actions"][:, None])[:, 0].double() - torch.logsumexp(x.double(), 1)
    old = (lp + 0.15 * torch.randn(N, **r)).float()
    ratio = torch.exp(lp - old.double())
    # the gradient jumps where the ratio crosses a clipping border: a row closer to one than the sums' rounding says nothing
    near = ((ratio - 0.8).abs() < 2e-3) | ((ratio - 1.2).abs() < 2e-3)
    s["old"] = torch.where(near, lp.float(), old)
    s["adv"] = torch.randn(N, **r)
    if case["weights"]:                                                  # a padded batch: an eighth of the rows is padding
        live = torch.rand(N, **r) >= 0.125
        s["weights"] = live.float() / N
    if case["train"]:
        s["logits"].requires_grad_()
    return s


def prepare_clip(case, gen):
    sizes, dt, out = tensor_sizes(case), DTYPES[case["dtype"]], DTYPES[case["out"]]
    flat = torch.randn(sum(sizes), device="cuda", generator=gen).to(dt)
    scale = 10.0 ** (torch.rand(len(sizes), device="cuda", generator=gen) * 2 - 3)
    grads = [t.clone() * c.to(dt) for t, c in zip(flat.split(sizes), scale)]
    buffer = torch.empty(sum(sizes), dtype=out, device="cuda")
    return {"grads": grads, "flat": buffer, "out": list(buffer.split(sizes)), "max_norm": 0.3 * 1e-2 * math.sqrt(sum(sizes))}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return dict({"linear": prepare_linear, "policy": prepare_policy, "clip": prepare_clip}[case["op"]](case, gen),
                op=case["op"])


# ---- one pass -----------------------------------------------------------------

def run(state):
    if own:
        return {"linear": own_linear, "policy": own_policy, "clip": own_clip}[state["op"]](state)
    with torch.no_grad():
        return {"linear": plain_linear, "policy": plain_policy, "clip": plain_clip}[state["op"]](state)


def own_linear(s):
    from citadels_self_play_amd import ops
    y = ops.linear(s["x"], s["w"], s["b"], residual=s["res"], activation=s["act"])
    if not s["train"]:
        return [y]
    return [y.detach()] + list(torch.autograd.grad(y, s["leaves"], s["dy"]))


def own_policy(s):
    from citadels_self_play_amd import ops
    got = ops.policy_loss(s["logits"], s["actions"], s["old"], s["adv"], ref_logits=s["ref"], offsets=s["offsets"],
                          mask=s["mask"], weights=s["weights"], clip=s["clip"], kl_coef=s["kl_coef"])
    if not s["train"]:
        return [got.loss, got.logp, got.kl]
    return [got.loss.detach(), got.logp, got.kl, torch.autograd.grad(got.loss, s["logits"])[0]]


def own_clip(s):
    from citadels_self_play_amd import ops
    return [ops.clip_grad_norm(s["grads"], s["max_norm"], out=s["out"]), s["flat"]]


# ---- plain forms --------------------------------------------------------------

def plain_linear(s):
    dt = s["x"].dtype
    x, w = s["x"].float(), s["w"].float()
    z = x @ w.t()
    if s["b"] is not None:
        z = z + s["b"].float()
    act = s["act"]
    if act == "relu":
        y = torch.where(z > 0, z, 0.0)
    elif act == "gelu":
        cdf = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        y = z * cdf
    elif act == "silu":
        cdf = 1 / (1 + torch.exp(-z))
        y = z * cdf
    else:
        y = z
    if s["res"] is not None:
        y = y + s["res"].float()
    y = y.to(dt)
    if not s["train"]:
        return [y]
    dz = s["dy"].float()
    if act == "relu":
        dz = torch.where(z > 0, dz, 0.0)
    elif act == "gelu":
        dz = dz * (cdf + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi)))
    elif act == "silu":
        dz = dz * (cdf * (1 + z * (1 - cdf)))
    got = [y, (dz @ w).to(dt), (dz.t() @ x).to(dt)]
    if s["b"] is not None:
        got.append(dz.sum(0).to(dt))
    if s["res"] is not None:
        got.append(s["dy"])
    return got


def row_places(s, n):
    """The places of ragged rows' entries in a padded table, and which of them there are."""
    at = s["offsets"][:-1, None] + torch.arange(s["longest"], device="cuda")
    there = at < s["offsets"][1:, None]
    return torch.where(there, at, n), there


def padded(s, t):
    """[rows][widest] entries of `t` and which of them are legal."""
    if s["offsets"] is None:
        return t, torch.ones_like(t, dtype=torch.bool) if s["mask"] is None else s["mask"]
    at, there = row_places(s, t.shape[0])
    return torch.cat([t.detach(), t.new_zeros(1)])[at], there


def plain_policy(s):
    x, legal = padded(s, s["logits"])
    every = s["offsets"] is None and s["mask"] is None
    x = x.float()
    if not every:
        x = torch.where(legal, x, -math.inf)
    top = x.max(1, keepdim=True).values
    lse = top + torch.log(torch.exp(x - top).sum(1, keepdim=True))
    lp = x - lse
    p = torch.exp(lp)
    at = s["actions"][:, None]
    logp = lp.gather(1, at)[:, 0]
    ratio = torch.exp(logp - s["old"])
    low, high = s["clip"]
    adv = s["adv"]
    free, held = ratio * adv, ratio.clamp(1 - low, 1 + high) * adv
    per_row = -torch.minimum(free, held)
    dlogp = torch.where(free <= held, -free, 0.0)
    kl = torch.zeros_like(logp)
    if s["ref"] is not None:
        q = padded(s, s["ref"])[0].float()
        if not every:
            q = torch.where(legal, q, -math.inf)
        top = q.max(1, keepdim=True).values
        d = lp - (q - (top + torch.log(torch.exp(q - top).sum(1, keepdim=True))))
        if not every:
            d = torch.where(legal, d, 0.0)
        kl = (p * (d + torch.expm1(-d))).sum(1)          # sum p d, written so that no term is negative
        per_row = per_row + s["kl_coef"] * kl
    w = s["weights"] if s["weights"] is not None else torch.full_like(logp, 1.0 / logp.shape[0])
    live = w != 0
    loss = torch.where(live, w * per_row, 0.0).sum()
    logp, kl = torch.where(live, logp, 0.0), torch.where(live, kl, 0.0)
    if not s["train"]:
        return [loss, logp, kl]
    g = -p * dlogp[:, None]
    g.scatter_add_(1, at, dlogp[:, None])
    if s["ref"] is not None:
        g = g + s["kl_coef"] * (p * (d - kl[:, None]))
    g = torch.where(live[:, None], w[:, None] * g, 0.0)
    if s["offsets"] is not None:
        n = s["logits"].shape[0]
        places = row_places(s, n)[0]
        g = g.new_zeros(n + 1).scatter_(0, places.reshape(-1), g.reshape(-1))[:n]
    return [loss, logp, kl, g.to(s["logits"].dtype)]


def plain_clip(s):
    squares = torch.stack([g.float().square().sum() for g in s["grads"]])
    norm = squares.double().sum().sqrt()
    c = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
    return [norm.float(), torch.cat([(g.float() * c).to(s["flat"].dtype) for g in s["grads"]])]


# ---- what a pass cannot do without ----------------------------------------------

def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        n = M * K + N * K + (N if case["bias"] else 0) + M * N * (2 if case["residual"] else 1)
        if case["train"]:
            n += M * N + M * K + N * K + (N if case["bias"] else 0)
        return {"bytes": e * n, "flops": (6 if case["train"] else 2) * M * N * K}
    if case["op"] == "policy":
        n = sum(row_lengths(case)) if case["layout"] == "ragged" else case["rows"] * case["width"]
        live = 0.875 if case["weights"] else 1.0
        per = live * (e * (2 if case["ref"] else 1) + (1 if case["mask"] else 0)) + (e if case["train"] else 0)
        rows = case["rows"] * (8 + 4 + 4 + 8 + (4 if case["weights"] else 0) + (8 if case["layout"] == "ragged" else 0))
        return {"bytes": n * per + rows, "flops": n * (12 if case["ref"] else 5)}
    n = sum(tensor_sizes(case))
    return {"bytes": n * (e + BYTES[case["out"]]), "flops": 3 * n}


# ---- the definition in 64 bits ----------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"linear": exact_linear, "policy": exact_policy, "clip": exact_clip}[case["op"]](s)


def exact_linear(s):
    x, w, b, res = (None if t is None else t.detach().double().requires_grad_(s["train"])
                    for t in (s["x"], s["w"], s["b"], s["res"]))
    y = torch.addmm(torch.zeros(w.shape[0], dtype=torch.float64, device="cuda") if b is None else b, x, w.t())
    if s["act"] == "relu":
        y = y.clamp(min=0)
    elif s["act"] == "gelu":
        y = y * torch.special.ndtr(y)
    elif s["act"] == "silu":
        y = y * torch.sigmoid(y)
    if res is not None:
        y = y + res
    if not s["train"]:
        return [y]
    return [y.detach()] + list(torch.autograd.grad(y, [t for t in (x, w, b, res) if t is not None], s["dy"].double()))


def exact_policy(s):
    logits = s["logits"].detach().double().requires_grad_(s["train"])
    if s["offsets"] is None:
        x, legal = logits, s["mask"]
        q = None if s["ref"] is None else s["ref"].double()
    else:
        at, legal = row_places(s, logits.shape[0])
        pad = lambda t: torch.cat([t, t.new_zeros(1)])[at]  # noqa: E731
        x, q = pad(logits), None if s["ref"] is None else pad(s["ref"].double())
    if legal is not None:
        x = x.masked_fill(~legal, -math.inf)
        q = None if q is None else q.masked_fill(~legal, -math.inf)
    lp = x - torch.logsumexp(x, 1, keepdim=True)
    logp = lp.gather(1, s["actions"][:, None])[:, 0]
    adv = s["adv"].double()
    ratio = torch.exp(logp - s["old"].double())
    value = -torch.minimum(ratio * adv, ratio.clamp(1 - s["clip"][0], 1 + s["clip"][1]) * adv)
    kl = torch.zeros_like(logp)
    if q is not None:
        d = lp - (q - torch.logsumexp(q, 1, keepdim=True))
        if legal is not None:
            lp, d = lp.masked_fill(~legal, 0.0), d.masked_fill(~legal, 0.0)
        kl = (torch.exp(lp) * d).sum(1)
        value = value + s["kl_coef"] * kl
    w = torch.full_like(adv, 1.0 / len(adv)) if s["weights"] is None else s["weights"].double()
    live = w != 0
    loss = (w * value)[live].sum()
    got = [loss.detach(), torch.where(live, logp, 0.0).detach(), torch.where(live, kl, 0.0).detach()]
    if s["train"]:
        got.append(torch.autograd.grad(loss, logits)[0])
    return got


def exact_clip(s):
    flat = torch.cat([g.double() for g in s["grads"]])
    norm = torch.linalg.vector_norm(flat)
    return [norm, flat * min(1.0, s["max_norm"] / (float(norm) + 1e-6))]
