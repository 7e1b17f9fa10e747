"""verify / verify_parity of the tuning ops' HIP cards on the GPU."""
from __future__ import annotations

import pytest

from xkernels_amd import verify, verify_parity

pytestmark = pytest.mark.gpu
OPS = ["moe_balance_loss", "moe_router_backward", "lora_projection", "lora_projection_backward", "act_checkpoint",
       "act_restore"]


@pytest.mark.parametrize("op", OPS)
def test_verify_hip_card(op, dev):
    r = verify(f"{op}.hip@1.0.0", arch="amd_cdna4", measure_perf=True)
    assert r["compiled"], r["artifacts"]
    assert r["correctness"]["passed"], r["correctness"]
    assert r["determinism_check"] and r["perf"]["ms"] > 0


@pytest.mark.parametrize("op", OPS)
def test_verify_parity_hip_vs_reference(op, dev):
    r = verify_parity(f"{op}@1.0.0", archs=["amd_cdna4"])
    assert r["n_runnable"] == 2, r["errors"]
    assert r["agree"] is True, r["diverging"]
