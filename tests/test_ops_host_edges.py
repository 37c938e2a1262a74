"""Edges of the training / serving operators (citadels_self_play_amd/ops.py and
their C entry points) that end on the host."""
import os
import subprocess
import sys

import pytest
import torch

from citadels_self_play_amd import ops

CLIP_EMPTY = """
import ctypes as C
from citadels_self_play_amd import _lib
lib = _lib.load()
b = C.create_string_buffer(1 << 17)
p = (C.addressof(b) + 255) // 256 * 256
none, sizes, types = (C.c_void_p * 3)(), (C.c_int64 * 3)(), (C.c_int32 * 3)()
need = lib.cit_clip_grad_norm_work_bytes(3)
for out in (none, None):
    rc = lib.cit_clip_grad_norm(none, out, sizes, types, types, 3, 1.0, p, p, need, None)
    assert rc not in (0, -1), rc
"""


@pytest.mark.skipif(torch.cuda.is_available(), reason="the buffers are the host's: only for where there is no device to launch on")
def test_clip_of_tensors_that_hold_nothing_ends():
    """Every tensor of the list empty: on to the launch, which has no device here."""
    subprocess.run([sys.executable, "-c", CLIP_EMPTY], check=True, timeout=60,
                   cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))


def test_clip_refuses_tensors_without_memory():
    """What vmap hands a function stands for a batch of tensors."""
    with pytest.raises(ValueError, match="a gradient must be a dense tensor"):
        torch.vmap(lambda t: ops.clip_grad_norm([t], 1.0))(torch.ones(3, 4))


def test_policy_refuses_more_rows_than_it_counts():
    n = 1 << 30
    one = torch.zeros(1)
    with pytest.raises(ValueError, match="over 1073741823 positions"):
        ops.policy_loss(one.view(1, 1).expand(n, 1), one.long().expand(n), one.expand(n), one.expand(n))
    with pytest.raises(ValueError, match="over 1073741823 positions"):
        ops.policy_loss(one, one.long().expand(n), one.expand(n), one.expand(n), offsets=one.long().expand(n + 1))
