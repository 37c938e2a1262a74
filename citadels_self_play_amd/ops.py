"""Operators of a net's training step and of serving it, as hand-written HIP
kernels (csrc/cit_linear.hip, cit_policy.hip, cit_gradnorm.hip):

* `linear`         - act(x W^T + b) + residual, with its gradients;
* `policy_loss`    - the clipped policy loss with a KL term over rows of
                     option logits (ragged, dense or masked), with its gradient;
* `clip_grad_norm` - the global norm of many gradients, and their clipping
                     (`grad_norm`: the norm alone).

Tensors are fp32, bf16 or fp16 on one GPU.  Every call runs on the current
stream of its tensors' device, takes its workspace from torch's caching
allocator and waits for nothing.  Calls can be captured into a HIP graph (a
backward pass too, while no eager graph of the same leaves is alive: torch's
autograd engine would join the two graphs' streams; RuntimeError).  A backward
pass captured apart from its forward pass needs retain_graph=True, and the
forward pass's outputs alive as long as it is replayed.  (torch.cuda.
make_graphed_callables: with num_warmup_iters=0, since a warm-up's graph stays
alive beside its captures.)
Wrong arguments raise ValueError before anything is launched, tensors of
torch.func and vmap among them; a batch of gradients (is_grads_batched) raises
RuntimeError.

The checks are written out rather than shared: at a trainer's batch of 64 a
call's time is the host's.  What follows them, autograd included, is
csrc/cit_torch.cpp.
"""
import collections
import math

import torch

from . import _lib

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}
# a matrix's sides; a row's entries; rows (the kernels' indexes are 32 bits)
_MOST, _LONGEST, _ROWS = 2 ** 31 - 1024, 2 ** 30, 2 ** 30 - 1
_NORM, _CHECK, _CLIP = 0, 1, 2                  # cit_torch.cpp's clip_grad_norm
_calls = _lib.torch_calls


def _same_place(first, **others):
    """Every tensor a strided one on the first one's device, and that a GPU; None is left out."""
    for name, t in others.items():
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise ValueError("%s must be a tensor, not %s" % (name, type(t).__name__))
        if t.layout != torch.strided or t.is_neg():
            raise ValueError("%s must be a dense tensor" % name)
        if t.device != first.device:
            raise ValueError("%s is on %s, the first tensor on %s" % (name, t.device, first.device))


def _gpu(t):
    if not t.is_cuda:
        raise ValueError("tensors must be on the GPU (there is no CPU path), not on %s" % t.device)


# ---- linear ---------------------------------------------------------------------

def linear(x, weight, bias=None, residual=None, activation="none"):
    """activation(x @ weight.T + bias) + residual, rounded once to x's type.

    x [..., K], weight [N, K] (nn.Linear's layout), bias [N], residual [..., N],
    all of one type; activation "none", "relu", "gelu" (by erf) or "silu".
    Sums are fp32.  Differentiable in every tensor; under no_grad nothing is
    kept; there are no second derivatives (create_graph=True raises RuntimeError).
    For the backward pass the pre-activation is kept in the type, and its
    gradient is rounded to it before the two products that use it (bias gradients
    are summed before that); relu passes the gradient on where it is NaN."""
    _same_place(x if isinstance(x, torch.Tensor) else torch.empty(0), x=x, weight=weight, bias=bias, residual=residual)
    dt, shape, ws = x.dtype, x.shape, weight.shape
    if dt not in TYPES:
        raise ValueError("x must be fp32, bf16 or fp16, not %s" % dt)
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError("activation must be one of %s, not %r" % (sorted(ACTIVATIONS), activation))
    if not shape:
        raise ValueError("x must be [..., K]")
    if len(ws) != 2 or ws[1] != shape[-1]:
        raise ValueError("weight must be [N, %d] for x %s, not %s" % (shape[-1], tuple(shape), tuple(ws)))
    if weight.dtype != dt:
        raise ValueError("weight is %s, x %s" % (weight.dtype, dt))
    if bias is not None:
        if bias.shape != ws[:1]:
            raise ValueError("bias must be [%d], not %s" % (ws[0], tuple(bias.shape)))
        if bias.dtype != dt:
            raise ValueError("bias is %s, x %s" % (bias.dtype, dt))
    if residual is not None:
        if residual.shape != shape[:-1] + ws[:1]:
            raise ValueError("residual must be %s, not %s" % (tuple(shape[:-1] + ws[:1]), tuple(residual.shape)))
        if residual.dtype != dt:
            raise ValueError("residual is %s, x %s" % (residual.dtype, dt))
    _gpu(x)
    M = shape[0] if len(shape) == 2 else math.prod(shape[:-1])
    if max(M, shape[-1], ws[0]) > _MOST:
        raise ValueError("a dimension is over %d" % _MOST)
    return _calls().linear(x, weight, bias, residual, act)


# ---- policy loss ------------------------------------------------------------------

PolicyLoss = collections.namedtuple("PolicyLoss", "loss logp kl")


def _f32(name, t, N):
    if t.shape != (N,) or not t.dtype.is_floating_point:
        raise ValueError("%s must be [%d] floating point numbers" % (name, N))
    if t.dtype != torch.float32:
        t = t.float()
    if not t.is_contiguous():
        t = t.contiguous()
    return t.detach() if t.requires_grad else t


def _whole(t):
    if t.dtype != torch.int64:
        t = t.long()
    return t if t.is_contiguous() else t.contiguous()


def policy_loss(logits, actions, old_logp, advantages, *, ref_logits=None, offsets=None, mask=None, weights=None,
                clip=0.2, kl_coef=0.0):
    """The clipped policy loss with a KL term over N positions; gives
    PolicyLoss(loss, logp [N], kl [N]).

    logits: [N, width], or with `offsets` (N + 1 ascending whole numbers) one
    list whose entries offsets[i] .. offsets[i + 1] - 1 are position i's options
    (engine.GameBatch.cfr_targets' option rows).  mask (bool, as logits): the
    legal entries.  actions [N]: the chosen entry, counted from the row's first.
    Lists are for rows of like lengths: the lanes that share a row go by twice
    the mean length, and one that is far longer takes its time in proportion.
    Over a row's legal entries, with rho = exp(logp[action] - old_logp),

        loss = sum_i weights_i (-min(rho A, clip(rho, 1 - low, 1 + high) A) + kl_coef KL(p || p_ref))

    weights [N] default to 1 / N; clip is one number or (low, high); p_ref is the
    softmax of ref_logits (as logits) over the same entries.  Only `logits` has
    a gradient, and no second one.  Rows of weight 0 are not read, rows with no legal entry (or
    nothing over -inf) count nothing: both give logp 0, kl 0 and a gradient of 0.
    A masked action has rho 0; an action outside its row, or offsets that
    leave the list, give NaN (what gradient the entries of no row then have is
    not defined).  KL is infinite where p_ref is 0 and p is not, and
    NaN where the reference leaves nothing of a row; with kl_coef 0 it is
    told, whatever it is, and is no part of the loss."""
    _same_place(logits if isinstance(logits, torch.Tensor) else torch.empty(0), logits=logits, actions=actions,
                old_logp=old_logp, advantages=advantages, ref_logits=ref_logits, offsets=offsets, mask=mask,
                weights=weights)
    dt, shape = logits.dtype, logits.shape
    if dt not in TYPES:
        raise ValueError("logits must be fp32, bf16 or fp16, not %s" % dt)
    if len(shape) != (2 if offsets is None else 1):
        raise ValueError("logits must be [N, width], or one list with offsets, not %s" % (tuple(shape),))
    low, high = (clip, clip) if isinstance(clip, (int, float)) else clip
    low, high, kl_coef = float(low), float(high), float(kl_coef)
    if not (low >= 0 and high >= 0):
        raise ValueError("clip must be two numbers >= 0, not %r" % (clip,))
    if not 0 <= kl_coef < math.inf:
        raise ValueError("kl_coef must be a finite number >= 0, not %r" % kl_coef)
    if kl_coef and ref_logits is None:
        raise ValueError("a KL term needs ref_logits")
    if actions.dim() != 1 or actions.dtype not in (torch.int64, torch.int32):
        raise ValueError("actions must be [N] whole numbers")
    N = actions.shape[0]
    if N > _ROWS:
        raise ValueError("over %d positions" % _ROWS)
    if offsets is None:
        if shape[0] != N:
            raise ValueError("%d rows of logits, %d actions" % (shape[0], N))
        if shape[1] > _LONGEST:
            raise ValueError("a row is over %d entries" % _LONGEST)
    else:
        if offsets.dtype not in (torch.int64, torch.int32) or offsets.shape != (N + 1,):
            raise ValueError("offsets must be [N + 1] whole numbers for %d actions" % N)
        offsets = _whole(offsets)
    old_logp, advantages = _f32("old_logp", old_logp, N), _f32("advantages", advantages, N)
    if weights is not None:
        weights = _f32("weights", weights, N)
    if ref_logits is not None and (ref_logits.shape != shape or ref_logits.dtype != dt):
        raise ValueError("ref_logits must be as logits (%s %s)" % (dt, tuple(shape)))
    if mask is not None and (mask.shape != shape or mask.dtype != torch.bool):
        raise ValueError("mask must be bool and as logits %s" % (tuple(shape),))
    _gpu(logits)
    return PolicyLoss(*_calls().policy_loss(logits, ref_logits, mask, offsets, _whole(actions), old_logp, advantages,
                                            weights, low, high, kl_coef))


# ---- gradient norm ------------------------------------------------------------------

def _listed(tensors):
    return [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)


def grad_norm(grads):
    """sqrt of the sum of all squares of a list of gradients (fp32 scalar on the device; no tensors: 0)."""
    grads = _listed(grads)
    return _calls().clip_grad_norm(grads, math.inf, None, _NORM) if grads else torch.zeros(())


def clip_grad_norm(grads, max_norm, out=None, error_if_nonfinite=False):
    """Scales a list of gradients by min(1, max_norm / (norm + 1e-6)) and gives
    their global norm (fp32 scalar on the device; no tensors: 0).

    In place, or into the tensors of `out` (contiguous, the gradients' type or
    fp32: 16-bit gradients into flat fp32 masters).  Squares are summed in fp64
    in a fixed order.  An infinite or NaN norm scales as torch's
    clip_grad_norm_ does; error_if_nonfinite waits for the norm and raises
    RuntimeError before anything is scaled."""
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError("max_norm must be a number >= 0, not %r" % max_norm)
    grads, out = _listed(grads), None if out is None else _listed(out)
    if not grads:
        if out:
            raise ValueError("0 gradients, %d tensors in out" % len(out))
        return torch.zeros(())
    call = _calls().clip_grad_norm
    if error_if_nonfinite and not math.isfinite(float(call(grads, max_norm, out, _CHECK))):
        raise RuntimeError("the gradients' global norm is not finite: nothing was clipped")
    return call(grads, max_norm, out, _CLIP)
