"""max_len of select_tokens at its limits: it sizes the launch, and any value
serves any lengths."""
import numpy as np
import pytest

import evict_ref as ref
from test_gpu_evict import layout, run_select

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("said", [0, 1, (1 << 31) - 33, (1 << 31) - 32, (1 << 31) - 1])
@pytest.mark.parametrize("seqs", [1, 40])
def test_any_max_len(seqs, said):
    lens = [37 * i % 900 + 1 for i in range(seqs)]
    tables, slots = layout(lens, 16, 1)
    x = np.random.default_rng(0).random((8, slots)).astype(np.float32)
    want = ref.select(x, tables, lens, 16, 32, 2, 3)
    np.testing.assert_array_equal(run_select(x, tables, lens, 16, 32, 2, 3, said), want)
