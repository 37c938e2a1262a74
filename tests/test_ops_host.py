"""Refusals of the training / serving operators (citadels_self_play_amd/ops.py
and their C entry points): wrong arguments end in ValueError or -1 before a
launch, so all of this runs without a GPU."""
import ctypes as C
import math

import pytest
import torch

from citadels_self_play_amd import _lib, ops


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


T = torch.zeros


@pytest.mark.parametrize("args,kw,says", [
    ((T(3, 4), T(5, 3)), {}, "weight must be"),
    ((T(3, 4), T(5, 4, 1)), {}, "weight must be"),
    ((T(3, 4), T(5, 4), T(4)), {}, "bias must be"),
    ((T(3, 4), T(5, 4), T(5), T(3, 4)), {}, "residual must be"),
    ((T(3, 4), T(5, 4).half()), {}, "weight is torch.float16"),
    ((T(3, 4).double(), T(5, 4).double()), {}, "x must be fp32"),
    ((T(3, 4), T(5, 4)), {"activation": "tanh"}, "activation must be"),
    ((T(3, 4), [1.0]), {}, "weight must be a tensor"),
    ((T(3, 4), T(5, 4)), {}, "must be on the GPU"),
    ((T(()), T(5, 1)), {}, "x must be"),
])
def test_linear_refuses(args, kw, says):
    with pytest.raises(ValueError, match=says):
        ops.linear(*args, **kw)


def policy(**kw):
    a = dict(logits=T(3, 4), actions=T(3, dtype=torch.int64), old_logp=T(3), advantages=T(3))
    a.update(kw)
    return ops.policy_loss(a.pop("logits"), a.pop("actions"), a.pop("old_logp"), a.pop("advantages"), **a)


@pytest.mark.parametrize("kw,says", [
    (dict(logits=T(12)), "logits must be"),
    (dict(offsets=T(4, dtype=torch.int64)), "logits must be"),
    (dict(logits=T(12), offsets=T(3, dtype=torch.int64)), "offsets must be"),
    (dict(logits=T(12), offsets=T(4)), "offsets must be"),
    (dict(logits=T(2, 4)), "2 rows of logits"),
    (dict(logits=T(3, 4).double()), "logits must be fp32"),
    (dict(actions=T(3)), "actions must be"),
    (dict(actions=T(3, 1, dtype=torch.int64)), "actions must be"),
    (dict(old_logp=T(4)), "old_logp must be"),
    (dict(advantages=T(3, dtype=torch.int64)), "advantages must be"),
    (dict(weights=T(2)), "weights must be"),
    (dict(mask=T(3, 4)), "mask must be"),
    (dict(mask=T(3, 5, dtype=torch.bool)), "mask must be"),
    (dict(ref_logits=T(3, 5)), "ref_logits must be"),
    (dict(ref_logits=T(3, 4).half()), "ref_logits must be"),
    (dict(kl_coef=0.1), "needs ref_logits"),
    (dict(kl_coef=math.nan), "kl_coef must be"),
    (dict(kl_coef=-1.0, ref_logits=T(3, 4)), "kl_coef must be"),
    (dict(clip=-0.1), "clip must be"),
    (dict(clip=(0.1, math.nan)), "clip must be"),
    (dict(), "must be on the GPU"),
])
def test_policy_loss_refuses(kw, says):
    with pytest.raises(ValueError, match=says):
        policy(**kw)


def test_clip_refuses():
    g = T(6)
    two = [T(6), T(4)]
    for args, says in [
        (([g.long()], 1.0), "gradients must be"),
        (([g], -1.0), "max_norm"),
        (([g], math.nan), "max_norm"),
        (([g, g], 1.0), "listed twice"),
        (([g[:4], g[2:]], 1.0), "share memory"),
        (([T(1).expand(6)], 1.0), "give out="),
        ((two, 1.0, [T(6)]), "2 gradients, 1 tensors"),
        ((two, 1.0, [T(6), T(5)]), "an out tensor must be"),
        ((two, 1.0, [T(6), T(4).half()]), "an out tensor must be"),
        ((two, 1.0, [T(6), T(8)[::2]]), "an out tensor must be"),
        (([g, T(6)], 1.0, [T(6), g]), "share memory"),
        (([T(4), T(4)], 1.0, list(T(7).as_strided((2, 4), (3, 1)))), "share memory"),
        (([g, g], 1.0, [T(6), T(6)]), "must be on the GPU"),
        (([g], 1.0, [g]), "must be on the GPU"),
        ((two, 1.0), "must be on the GPU"),
    ]:
        with pytest.raises(ValueError, match=says):
            ops.clip_grad_norm(*args)
    with pytest.raises(ValueError, match="must be on the GPU"):
        ops.grad_norm([g])
    assert float(ops.grad_norm([])) == 0.0 and float(ops.clip_grad_norm([], 1.0)) == 0.0


def test_entry_points_refuse(lib):
    """Null or short buffers, unknown types, strides under a row: -1 before any launch."""
    b = C.create_string_buffer(1 << 17)
    p = (C.addressof(b) + 255) // 256 * 256
    fw = lib.cit_linear_forward
    assert fw(p, 8, p, 8, None, None, 0, p, None, 4, 4, 8, 3, 0, None, 0, None) == -1
    assert fw(p, 8, p, 8, None, None, 0, p, None, 4, 4, 8, 0, 4, None, 0, None) == -1
    assert fw(p, 7, p, 8, None, None, 0, p, None, 4, 4, 8, 0, 0, None, 0, None) == -1
    assert fw(p, 8, p, 7, None, None, 0, p, None, 4, 4, 8, 0, 0, None, 0, None) == -1
    assert fw(p, 8, p, 8, None, p, 3, p, None, 4, 4, 8, 0, 0, None, 0, None) == -1
    assert fw(p, 8, p, 8, None, None, 0, None, None, 4, 4, 8, 0, 0, None, 0, None) == -1
    assert fw(p, 8, p, 8, None, None, 0, p, None, -1, 4, 8, 0, 0, None, 0, None) == -1
    assert fw(p, 2 ** 31 - 1, p, 2 ** 31 - 1, None, None, 0, p, None, 4, 4, 2 ** 31 - 1, 0, 0, None, 0, None) == -1
    assert fw(p, 8, p, 8, None, None, 0, p, None, 2 ** 31 - 1, 4, 8, 0, 0, None, 0, None) == -1
    assert fw(None, 8, None, 8, None, None, 0, None, None, 0, 4, 8, 0, 0, None, 0, None) == 0
    need = lib.cit_linear_backward_work_bytes(p, 4000, p, 4000, p, p, p, 4000, 4000, 4000, 1, 1)
    assert need > 0
    bw = lib.cit_linear_backward
    assert bw(p, 4000, p, p, 4000, p, 4000, p, p, p, 4000, 4000, 4000, 1, 1, p, need - 1, None) == -1
    assert bw(p, 4, None, p, 8, p, 8, p, p, p, 4, 4, 8, 1, 1, p, need, None) == -1
    assert bw(p, 3, p, p, 8, p, 8, p, p, p, 4, 4, 8, 1, 1, p, need, None) == -1
    assert bw(p, 4000, p, p, 4000, p, 4000, p, p, p, 4000, 4000, 4000, 1, 1, p + 8, need, None) == -1
    pl = lib.cit_policy_loss
    ok = [p, 4, None, 0, None, 0, None, 0, 3, 4, p, p, p, None, 0.2, 0.2, 0.0, 0, p, p, p, None, p, 1 << 16, None]
    for at, bad in [(0, None), (1, 3), (8, -1), (9, -1), (10, None), (14, -1.0), (16, math.nan), (17, 3), (18, None),
                    (19, None), (22, None), (22, p + 4), (23, 0), (9, 2 ** 31 - 1)]:
        a = list(ok)
        a[at] = bad
        assert pl(*a) == -1, (at, bad)
    cl = lib.cit_clip_grad_norm
    need = lib.cit_clip_grad_norm_work_bytes(1)
    ptr, null = (C.c_void_p * 1)(p), (C.c_void_p * 1)(None)
    n, neg = (C.c_int64 * 1)(4), (C.c_int64 * 1)(-4)
    t32, t16, t9 = ((C.c_int32 * 1)(v) for v in (0, 1, 9))
    assert cl(ptr, ptr, n, t32, t32, 1, 1.0, p, p, need - 1, None) == -1
    assert cl(ptr, ptr, n, t32, t32, 1, 1.0, p, p + 8, need, None) == -1
    assert cl(null, ptr, n, t32, t32, 1, 1.0, p, p, need, None) == -1
    assert cl(ptr, null, n, t32, t32, 1, 1.0, p, p, need, None) == -1
    assert cl(ptr, ptr, neg, t32, t32, 1, 1.0, p, p, need, None) == -1
    assert cl(ptr, ptr, n, t9, t32, 1, 1.0, p, p, need, None) == -1
    assert cl(ptr, ptr, n, t32, t16, 1, 1.0, p, p, need, None) == -1
    assert cl(ptr, ptr, n, t32, t32, 1, math.nan, p, p, need, None) == -1
    assert cl(ptr, ptr, n, t32, t32, 1, 1.0, None, p, need, None) == -1


def test_lazily_negated_tensors_refused():
    """Their memory holds the values before the sign changed."""
    n = torch._neg_view(T(3, 4))
    with pytest.raises(ValueError, match="x must be a dense tensor"):
        ops.linear(n, T(5, 4))
    with pytest.raises(ValueError, match="logits must be a dense tensor"):
        policy(logits=n)
    with pytest.raises(ValueError, match="a gradient must be a dense tensor"):
        ops.clip_grad_norm([n], 1.0)


def test_missing_extension_is_loud(monkeypatch):
    import sys
    monkeypatch.setattr(_lib, "_torch_calls", None)
    monkeypatch.setitem(sys.modules, "citadels_self_play_amd._cit_torch", None)
    monkeypatch.delattr("citadels_self_play_amd._cit_torch", raising=False)
    with pytest.raises(_lib.NativeError, match="_cit_torch.so"):
        _lib.torch_calls()


def test_copies_and_split_sums_have_room_of_their_own(lib):
    """A forward product of odd rows whose operands are copied and whose long reduction is shared out as well."""
    M, N, K = 1000, 1100, 8201
    for dtype, size in ((0, 4), (1, 2), (2, 2)):
        row = -(-K * size // 16) * 16
        assert lib.cit_linear_forward_work_bytes(M, N, K, dtype) >= (M + N) * row + 2 * M * N * 4
