"""A call that returns an error of the CUDA runtime leaves none behind: the next
call, and what else the program does on the GPU, does not fail for it."""
import pytest

pytestmark = pytest.mark.gpu


def test_a_plan_that_does_not_fit_the_gpu():
    """One terabyte of raw scores: the allocation fails, nothing else does."""
    import fekv
    import torch
    from fekv import _lib
    x = torch.arange(8, device="cuda")
    draft = torch.zeros(3, 2, dtype=torch.int64, device="cuda")
    verify, out = (torch.zeros(3, n, dtype=torch.int64, device="cuda") for n in (3, 4))
    free = torch.cuda.mem_get_info()[0]
    for _ in range(2):
        with pytest.raises(fekv.FeError, match="workspace") as e:
            fekv.ScoredPlan(32, 8, 128, 16, 4, 64, True, 99, max_keys=1 << 33)
        assert e.value.status == _lib.FE_ERR_CUDA
        # the next call's own check of its launch
        fekv.accept(draft, verify, out)
        assert (x + 1).sum().item() == 36
        torch.cuda.synchronize()
    assert torch.cuda.mem_get_info()[0] > free - (1 << 28)  # what was allocated is freed
