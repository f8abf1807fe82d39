"""Plans used on a second GPU of the same process. A kernel's dynamic
shared-memory limit belongs to a device: a launch that relies on another
device's fails."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "flashengine.cpp_b200", "csrc")
# raised per device there: allow_smem, and the table of the allocation-free path
PER_DEVICE = {"fe_common.cuh": 1, "fe_decode.cu": 1}


def test_limits_are_raised_per_device():
    """No launch keeps "done once" for the whole process (needs no GPU)."""
    seen = {}
    for name in sorted(os.listdir(CSRC)):
        with open(os.path.join(CSRC, name)) as f:
            text = f.read()
        n = len(re.findall(r"\bcudaFuncSetAttribute\s*\(", text))
        if n:
            seen[name] = n
    assert seen == PER_DEVICE
    with open(os.path.join(CSRC, "fe_decode.cu")) as f:
        assert "d.attr_set[ti][hi]" in f.read()  # d: the current device's entry


def devices():
    import torch
    return torch.cuda.device_count() if torch.cuda.is_available() else 0


@pytest.mark.gpu
@pytest.mark.skipif(devices() < 2, reason="needs two GPUs")
@pytest.mark.parametrize("kind", ["SharedPlan", "ScoredPlan", "AttentionPlan"])
@pytest.mark.parametrize("dim", [128, 256])
def test_each_device_in_turn(dim, kind):
    import fekv
    import torch
    from test_gpu_shared_attention import Step, ones
    outs = []
    for device in (0, 1):
        with torch.cuda.device(device):
            layout = [(24, ones(*range(1, 61)))] if kind == "SharedPlan" else [(0, ones(5, 33, 700))]
            if kind == "AttentionPlan":
                layout[0][1].append((300, 300))
            s = Step(layout, 16, 2, dim, 16, "bfloat16")
            more = {"max_keys": 1000} if kind == "ScoredPlan" else {}
            plan = s.plan(getattr(fekv, kind), **more)
            plan.prepare(*s.meta())
            out = torch.empty_like(s.q)
            if kind == "ScoredPlan":
                plan.attention(s.q, s.k, s.v, torch.zeros(2, s.k.shape[0], device="cuda"), out)
            else:
                plan.attention(s.q, s.k, s.v, out, True)
            s.check(out, True)
            assert fekv.device_errors() == 0
            outs.append(out.cpu())
    assert torch.equal(*outs)
