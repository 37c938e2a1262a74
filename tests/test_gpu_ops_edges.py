"""Edges of the training / serving operators (citadels_self_play_amd/ops.py) on a
real MI355X that test_gpu_ops.py leaves out.  Tolerances are counted as there: u =
2^-24 is half a step of fp32, a device exp or log is off by at most 4 u of its
value, every rounding by half a step of its type."""
import math

import pytest
import torch

from test_gpu_ops import DT, U, call_policy

pytestmark = pytest.mark.gpu


# ---- policy loss ------------------------------------------------------------------

def even_rows(rows, width, dt=torch.float32):
    """Rows whose entries are all alike: every exp(l - max) is 1 and their sum exact, so log p is -log width to 64 bits."""
    return {"logits": torch.full((rows, width), 0.75, dtype=dt, device="cuda"), "ref": None, "mask": None, "offsets": None,
            "actions": (torch.arange(rows) * 7 % width).cuda(), "old": torch.full((rows,), -math.log(width), device="cuda"),
            "adv": torch.ones(rows, device="cuda"), "weights": torch.ones(rows, device="cuda")}


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
