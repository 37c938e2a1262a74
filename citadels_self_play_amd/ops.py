"""Operators of a net's training step and of serving it, as hand-written HIP
kernels (csrc/cit_linear.hip, cit_policy.hip, cit_gradnorm.hip):

* `linear`         - act(x W^T + b) + residual, with its gradients;
* `policy_loss`    - the clipped policy loss with a KL term over rows of
                     option logits (ragged, dense or masked), with its gradient;
* `clip_grad_norm` - the global norm of many gradients, and their clipping
                     (`grad_norm`: the norm alone).

Tensors are fp32, bf16 or fp16 on one GPU.  Every call runs on the current
stream of its tensors' device, takes its workspace from torch's caching
allocator, waits for nothing and can be captured into a HIP graph.  Wrong
arguments raise ValueError before anything is launched.
"""
import collections
import ctypes as C
import math

import torch
from torch.autograd.function import once_differentiable

from . import _lib

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}
_MOST = 2 ** 31 - 1


def _need(ok, what):
    if not ok:
        raise ValueError(what)


def _tensor(name, t, like=None):
    _need(isinstance(t, torch.Tensor), "%s must be a tensor, not %s" % (name, type(t).__name__))
    _need(t.layout == torch.strided, "%s must be a dense tensor" % name)
    if like is not None:
        _need(t.device == like.device, "%s is on %s, the first tensor on %s" % (name, t.device, like.device))


def _gpu(t):
    _need(t.is_cuda, "tensors must be on the GPU (there is no CPU path), not on %s" % t.device)


class _on:
    """The tensors' device as the current one (nothing where it is already); gives the current stream's handle."""

    def __init__(self, t):
        self.device = t.device
        self.guard = None if t.device.index == torch.cuda.current_device() else torch.cuda.device(t.device)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()
        return torch.cuda.current_stream(self.device).cuda_stream

    def __exit__(self, *a):
        if self.guard is not None:
            self.guard.__exit__(*a)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _work(n, like):
    return torch.empty(n, dtype=torch.uint8, device=like.device) if n else None


def _rows(t, width):
    """`t` [rows][width] with its entries side by side, and the elements between rows."""
    if t.shape[0] == 1 and (width <= 1 or t.stride(1) == 1):
        return t, width
    if (width > 1 and t.stride(1) != 1) or t.stride(0) < width:
        t = t.contiguous()
    return t, max(width, t.stride(0))


# ---- linear ---------------------------------------------------------------------

def _linear_forward(x, w, b, r, act, keep):
    """(y, z): z is the pre-activation for the backward pass where `keep` asks for it."""
    M, K, N = x.shape[0], x.shape[1], w.shape[0]
    lib = _lib.load()
    y = torch.empty((M, N), dtype=x.dtype, device=x.device)
    z = torch.empty_like(y) if keep else None
    if not y.numel():
        return y, z
    t = TYPES[x.dtype]
    x, ldx = _rows(x, K)
    w, ldw = _rows(w, K)
    ldr = N
    if r is not None:
        r, ldr = _rows(r, N)
    with _on(x) as stream:
        n = int(lib.cit_linear_forward_work_bytes(M, N, K, t))
        work = _work(n, x)
        _lib.check(lib.cit_linear_forward(x.data_ptr(), ldx, w.data_ptr(), ldw, _ptr(b), _ptr(r), ldr, y.data_ptr(),
                                          _ptr(z), M, N, K, t, act, _ptr(work), n, stream), "cit_linear_forward")
    return y, z


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b, r, act):
        # relu without a residual leaves its sign in y (fp16 aside, where a small y rounds to 0); other activations
        # need the pre-activation
        own_y = act == ACTIVATIONS["relu"] and r is None and x.dtype != torch.float16
        x2 = x.reshape(-1, w.shape[1]) if w.shape[1] else x.reshape(math.prod(x.shape[:-1]), 0)
        y, z = _linear_forward(x2, w, b, None if r is None else r.reshape(x2.shape[0], w.shape[0]), act,
                               act != ACTIVATIONS["none"] and not own_y)
        out = y.reshape(x.shape[:-1] + (w.shape[0],))
        ctx.act = act
        need_x, need_w = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        ctx.save_for_backward(x if need_w else None, w if need_x else None, out if own_y else z)
        ctx.dims = (x.shape, w.shape)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w, z = ctx.saved_tensors
        (xs, (N, K)), (nx, nw, nb, nr) = ctx.dims, ctx.needs_input_grad[:4]
        M = math.prod(xs[:-1])
        dx = dw = db = None
        if nx or nw or nb:
            make = torch.empty if M and N else torch.zeros
            new = lambda *s: make(s, dtype=dy.dtype, device=dy.device)  # noqa: E731
            dx, dw, db = new(M, K) if nx else None, new(N, K) if nw else None, new(N) if nb else None
        if (nx or nw or nb) and M and N:
            lib, t = _lib.load(), TYPES[dy.dtype]
            d2, ldy = _rows(dy.reshape(M, N), N)
            ldx = ldw = K
            if nw:
                x, ldx = _rows(x.reshape(M, K), K)
            if nx:
                w, ldw = _rows(w, K)
            if z is not None:
                z = z.reshape(M, N)
                z = z if z.is_contiguous() else z.contiguous()
            with _on(dy) as stream:
                n = int(lib.cit_linear_backward_work_bytes(M, N, K, t, ctx.act))
                work = _work(n, dy)
                _lib.check(lib.cit_linear_backward(d2.data_ptr(), ldy, _ptr(z), _ptr(x) if nw else None, ldx,
                                                   _ptr(w) if nx else None, ldw, _ptr(dx), _ptr(dw), _ptr(db), M, N, K,
                                                   t, ctx.act, _ptr(work), n, stream), "cit_linear_backward")
        return (dx.reshape(xs) if nx else None, dw, db, dy if nr else None, None)


def linear(x, weight, bias=None, residual=None, activation="none"):
    """activation(x @ weight.T + bias) + residual, rounded once to x's type.

    x [..., K], weight [N, K] (nn.Linear's layout), bias [N], residual [..., N],
    all of one type; activation "none", "relu", "gelu" (by erf) or "silu".
    Sums are fp32.  Differentiable in every tensor; under no_grad nothing is
    kept.  The gradient of the pre-activation is rounded to the type before the
    two products that use it (bias gradients are summed before that)."""
    _tensor("x", x)
    _need(x.dtype in TYPES, "x must be fp32, bf16 or fp16, not %s" % x.dtype)
    _need(activation in ACTIVATIONS, "activation must be one of %s, not %r" % (sorted(ACTIVATIONS), activation))
    _need(x.dim() >= 1, "x must be [..., K]")
    _tensor("weight", weight, x)
    _need(weight.dim() == 2 and weight.shape[1] == x.shape[-1],
          "weight must be [N, %d] for x %s, not %s" % (x.shape[-1], tuple(x.shape), tuple(weight.shape)))
    out = x.shape[:-1] + (weight.shape[0],)
    for name, t, shape in (("bias", bias, (weight.shape[0],)), ("residual", residual, out)):
        if t is not None:
            _tensor(name, t, x)
            _need(tuple(t.shape) == tuple(shape), "%s must be %s, not %s" % (name, tuple(shape), tuple(t.shape)))
    for name, t in (("weight", weight), ("bias", bias), ("residual", residual)):
        _need(t is None or t.dtype == x.dtype, "%s is %s, x %s" % (name, t is not None and t.dtype, x.dtype))
    M = math.prod(x.shape[:-1])
    _need(max(M, x.shape[-1], weight.shape[0]) <= _MOST, "a dimension is over %d" % _MOST)
    _gpu(x)
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    act = ACTIVATIONS[activation]
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)
                                    or (residual is not None and residual.requires_grad)):
        return _Linear.apply(x, weight, bias, residual, act)
    y, _ = _linear_forward(x.reshape(M, x.shape[-1]), weight, bias,
                           None if residual is None else residual.reshape(M, weight.shape[0]), act, False)
    return y.reshape(out)


# ---- policy loss ------------------------------------------------------------------

PolicyLoss = collections.namedtuple("PolicyLoss", "loss logp kl")


def _policy_args(logits, ref, mask, offsets, actions, old, adv, weights, low, high, beta):
    rows = actions.shape[0]
    if offsets is None:
        width = logits.shape[1]
        logits, ld = _rows(logits, width)
        ref, ld_ref = (None, width) if ref is None else _rows(ref, width)
        mask, ld_mask = (None, width) if mask is None else _rows(mask, width)
        total = 0
    else:
        width = ld = ld_ref = ld_mask = 0
        total = logits.shape[0]
        logits, ref, mask = (None if t is None else t.contiguous() for t in (logits, ref, mask))
    keep = (logits, ref, mask)
    return keep, (_ptr(logits), ld, _ptr(ref), ld_ref, _ptr(mask), ld_mask, _ptr(offsets), total, rows, width,
                  actions.data_ptr(), old.data_ptr(), adv.data_ptr(), _ptr(weights), low, high, beta,
                  TYPES[logits.dtype])


def _policy_forward(given, want_grad):
    logits, actions = given[0], given[4]
    lib = _lib.load()
    dev, rows = logits.device, actions.shape[0]
    loss = torch.empty((), dtype=torch.float32, device=dev)
    stats = torch.empty((2, rows), dtype=torch.float32, device=dev)
    grad = None
    if want_grad:
        grad = torch.empty(logits.shape, dtype=logits.dtype, device=dev)
        if not rows:
            grad.zero_()
    with _on(logits) as stream:
        keep, args = _policy_args(*given)
        n = int(lib.cit_policy_loss_work_bytes(rows))
        work = _work(n, logits)
        _lib.check(lib.cit_policy_loss(*args, loss.data_ptr(), stats[0].data_ptr(), stats[1].data_ptr(), _ptr(grad),
                                       _ptr(work), n, stream), "cit_policy_loss")
    return loss, stats[0], stats[1], grad


class _PolicyLoss(torch.autograd.Function):
    """The forward kernel has a row's probabilities in hand, so it writes the
    gradient for an upstream gradient of 1 in the same pass over the logits;
    the backward kernel reads the upstream gradient on the device and computes
    the gradient again only where it is something else."""

    @staticmethod
    def forward(ctx, *given):
        loss, logp, kl, grad = _policy_forward(given, ctx.needs_input_grad[0])
        ctx.mark_non_differentiable(logp, kl)
        ctx.save_for_backward(*given[:8])
        ctx.scalars = given[8:]
        ctx.held = [(grad, torch.cuda.is_current_stream_capturing())]
        return loss, logp, kl

    @staticmethod
    @once_differentiable
    def backward(ctx, up, _logp, _kl):
        given = ctx.saved_tensors + ctx.scalars
        logits, rows = given[0], given[4].shape[0]
        try:
            grad, captured = ctx.held.pop()
        except IndexError:                       # a second backward pass: the first one's gradient is its owner's
            grad = None
        # a graph replayed on its own may find the forward pass's gradient used up
        fresh = grad is None or (torch.cuda.is_current_stream_capturing() and not captured)
        if grad is None:
            grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        if not rows:
            return (grad.zero_(),) + (None,) * 10
        up = up.to(torch.float32).contiguous()
        lib = _lib.load()
        with _on(logits) as stream:
            keep, args = _policy_args(*given)
            _lib.check(lib.cit_policy_loss_backward(*args, up.data_ptr(), 0 if fresh else 1, grad.data_ptr(), stream),
                       "cit_policy_loss_backward")
        return (grad,) + (None,) * 10


def policy_loss(logits, actions, old_logp, advantages, *, ref_logits=None, offsets=None, mask=None, weights=None,
                clip=0.2, kl_coef=0.0):
    """The clipped policy loss with a KL term over N positions; gives
    PolicyLoss(loss, logp [N], kl [N]).

    logits: [N, width], or with `offsets` (N + 1 ascending whole numbers) one
    list whose entries offsets[i] .. offsets[i + 1] - 1 are position i's options
    (engine.GameBatch.cfr_targets' option rows).  mask (bool, as logits): the
    legal entries.  actions [N]: the chosen entry, counted from the row's first.
    Over a row's legal entries, with rho = exp(logp[action] - old_logp),

        loss = sum_i weights_i (-min(rho A, clip(rho, 1 - low, 1 + high) A) + kl_coef KL(p || p_ref))

    weights [N] default to 1 / N; clip is one number or (low, high); p_ref is the
    softmax of ref_logits (as logits) over the same entries.  Only `logits` has
    a gradient.  Rows of weight 0 are not read, rows with no legal entry (or
    nothing over -inf) count nothing: both give logp 0, kl 0 and a gradient of 0.
    A masked action has rho 0; an action outside its row, or offsets that
    leave the list, give NaN.  KL is infinite where p_ref is 0 and p is not."""
    _tensor("logits", logits)
    _need(logits.dtype in TYPES, "logits must be fp32, bf16 or fp16, not %s" % logits.dtype)
    _need(logits.dim() == (2 if offsets is None else 1),
          "logits must be [N, width], or one list with offsets, not %s" % (tuple(logits.shape),))
    low, high = (clip, clip) if isinstance(clip, (int, float)) else clip
    low, high, kl_coef = float(low), float(high), float(kl_coef)
    _need(low >= 0 and high >= 0, "clip must be two numbers >= 0, not %r" % (clip,))
    _need(0 <= kl_coef < math.inf, "kl_coef must be a finite number >= 0, not %r" % kl_coef)
    _need(kl_coef == 0 or ref_logits is not None, "a KL term needs ref_logits")
    _tensor("actions", actions, logits)
    _need(actions.dim() == 1 and actions.dtype in (torch.int64, torch.int32), "actions must be [N] whole numbers")
    N = actions.shape[0]
    if offsets is None:
        _need(logits.shape[0] == N, "%d rows of logits, %d actions" % (logits.shape[0], N))
        _need(logits.shape[1] <= _MOST, "a row is over %d entries" % _MOST)
    else:
        _tensor("offsets", offsets, logits)
        _need(offsets.dim() == 1 and offsets.dtype in (torch.int64, torch.int32) and offsets.shape[0] == N + 1,
              "offsets must be [N + 1] whole numbers for %d actions" % N)
    for name, t in (("old_logp", old_logp), ("advantages", advantages), ("weights", weights)):
        if t is not None:
            _tensor(name, t, logits)
            _need(t.shape == (N,) and t.dtype.is_floating_point, "%s must be [N] floating point numbers" % name)
    if ref_logits is not None:
        _tensor("ref_logits", ref_logits, logits)
        _need(ref_logits.shape == logits.shape and ref_logits.dtype == logits.dtype,
              "ref_logits must be as logits (%s %s)" % (logits.dtype, tuple(logits.shape)))
    if mask is not None:
        _tensor("mask", mask, logits)
        _need(mask.shape == logits.shape and mask.dtype == torch.bool,
              "mask must be bool and as logits %s" % (tuple(logits.shape),))
    _gpu(logits)
    f32 = lambda t: None if t is None else t.detach().to(torch.float32).contiguous()  # noqa: E731
    given = (logits, None if ref_logits is None else ref_logits.detach(), mask,
             None if offsets is None else offsets.to(torch.int64).contiguous(),
             actions.to(torch.int64).contiguous(), f32(old_logp), f32(advantages), f32(weights), low, high, kl_coef)
    if torch.is_grad_enabled() and logits.requires_grad:
        return PolicyLoss(*_PolicyLoss.apply(*given))
    return PolicyLoss(*_policy_forward(given, False)[:3])


# ---- gradient norm ------------------------------------------------------------------

def _overlap(outs, others=()):
    """Whether a tensor of `outs` shares memory with another one of them or with one of `others`."""
    spans = [(t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(), k) for k, ts in ((1, outs), (0, others))
             for t in ts if t.numel()]
    end = [0, 0]                                 # of the spans of others and of outs so far
    for a, b, k in sorted(spans):
        if a < end[1] or (k and a < end[0]):
            return True
        end[k] = max(end[k], b)
    return False


def _listed(grads):
    grads = [grads] if isinstance(grads, torch.Tensor) else list(grads)
    for t in grads:
        _tensor("a gradient", t, grads[0])
        _need(t.dtype in TYPES, "gradients must be fp32, bf16 or fp16, not %s" % t.dtype)
    return [t.detach() for t in grads]


def _norm(flat, max_norm=math.inf, outs=None):
    """cit_clip_grad_norm over contiguous tensors (outs: None, `flat` itself or as many others)."""
    _gpu(flat[0])
    lib, n = _lib.load(), len(flat)
    norm = torch.empty((), dtype=torch.float32, device=flat[0].device)
    ptrs = (C.c_void_p * n)(*[t.data_ptr() for t in flat])
    sizes = (C.c_int64 * n)(*[t.numel() for t in flat])
    types = (C.c_int32 * n)(*[TYPES[t.dtype] for t in flat])
    to, to_types = (None, None) if outs is None else (ptrs, types)
    if outs is not None and outs is not flat:
        to = (C.c_void_p * n)(*[t.data_ptr() for t in outs])
        to_types = (C.c_int32 * n)(*[TYPES[t.dtype] for t in outs])
    with _on(norm) as stream:
        size = int(lib.cit_clip_grad_norm_work_bytes(n))
        work = _work(size, norm)
        _lib.check(lib.cit_clip_grad_norm(ptrs, to, sizes, types, to_types, n, max_norm, norm.data_ptr(),
                                          work.data_ptr(), size, stream), "cit_clip_grad_norm")
    return norm


def grad_norm(grads):
    """sqrt of the sum of all squares of a list of gradients (fp32 scalar on the device; no tensors: 0)."""
    grads = _listed(grads)
    return _norm([t.contiguous() for t in grads]) if grads else torch.zeros(())


def clip_grad_norm(grads, max_norm, out=None, error_if_nonfinite=False):
    """Scales a list of gradients by min(1, max_norm / (norm + 1e-6)) and gives
    their global norm (fp32 scalar on the device; no tensors: 0).

    In place, or into the tensors of `out` (contiguous, the gradients' type or
    fp32: 16-bit gradients into flat fp32 masters).  Squares are summed in fp64
    in a fixed order.  An infinite or NaN norm scales as torch's
    clip_grad_norm_ does; error_if_nonfinite waits for the norm and raises
    RuntimeError before anything is scaled."""
    max_norm = float(max_norm)
    _need(max_norm >= 0, "max_norm must be a number >= 0, not %r" % max_norm)
    grads = _listed(grads)
    flat = [t if t.is_contiguous() else t.contiguous() for t in grads]
    if out is None:
        outs = flat
        _need(all(s > 0 or n <= 1 for t in grads if not t.is_contiguous() for n, s in zip(t.shape, t.stride())),
              "a gradient whose elements share memory cannot be clipped in place: give out=")
        at = [t.data_ptr() for t in grads if t.numel()]
        _need(len(set(at)) == len(at) and not _overlap(flat), "a gradient is listed twice, or two share memory")
    else:
        outs = [t.detach() for t in ([out] if isinstance(out, torch.Tensor) else out)]
        _need(len(outs) == len(grads), "%d gradients, %d tensors in out" % (len(grads), len(outs)))
        for g, o in zip(grads, outs):
            _tensor("an out tensor", o, g)
            _need(o.shape == g.shape and o.dtype in (g.dtype, torch.float32) and o.is_contiguous(),
                  "an out tensor must be contiguous, of its gradient's shape, and of its type or fp32")
        _need(not _overlap(outs, [f for f, o in zip(flat, outs) if f.data_ptr() != o.data_ptr() or f.dtype != o.dtype]),
              "out tensors share memory with one another or with other gradients")
    if not grads:
        return torch.zeros(())
    if error_if_nonfinite and not math.isfinite(float(_norm(flat))):
        raise RuntimeError("the gradients' global norm is not finite: nothing was clipped")
    norm = _norm(flat, max_norm, outs)
    torch.autograd.graph.increment_version(outs)
    if out is None:
        for t, c in zip(grads, flat):
            if c.data_ptr() != t.data_ptr():
                t.copy_(c)
    return norm
