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


def test_scores_between_their_elements():
    import ctypes
    import fekv
    import torch
    from fekv import _lib
    from test_gpu_scored_attention import scored_plan
    from test_gpu_shared_attention import Step, ones
    s = Step([(0, ones(5, 33))], 8, 2, 128, 16, "bfloat16")
    plan = scored_plan(s)
    plan.prepare(*s.meta())
    scores, out = torch.zeros(2, s.k.shape[0] + 16, device="cuda"), torch.zeros_like(s.q)
    at = [ctypes.c_void_p(x.data_ptr()) for x in (s.q, s.k, s.v)]
    rc = fekv.load().fe_scored_attn_run(plan.handle, *at, ctypes.c_void_p(scores.data_ptr() + 2),
                                        ctypes.c_void_p(out.data_ptr()), None)
    assert rc == _lib.FE_ERR_INVALID_ARGUMENT and b"aligned" in fekv.load().fe_last_error()
    assert not scores.any() and not out.any()
