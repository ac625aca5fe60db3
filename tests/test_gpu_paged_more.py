"""More of the paged-pool operators against 64 bits: workspaces of larger batches, infinities, values of rows
that others do not see, and prefixes long enough that every ring of the tensor-core kernel goes round."""
import math

import pytest
from test_gpu_paged import KINDS, Batch, T  # noqa: F401 (T is a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("large,small", [((129, 8192), (128, 8192)), ((64, 2432), (64, 2304)),
                                         ((65, 2432), (64, 2304))])
def test_a_larger_batchs_workspace(T, q3lib, large, small):  # noqa: F811
    """A workspace sized for more rows or a longer prefix serves fewer, and nothing behind it changes."""
    b = Batch(T, q3lib, "e4m3", "bf16", 8, 2, 128, [1 + i % 5 for i in range(small[0])], [1] * small[0],
              prefix=small[1], seed=51, spare_rows=0)
    size = q3lib.paged_attn_workspace_size(b.pool.handle, 16, large[0], large[0], 1, large[1])
    b.ws = T.full((size + (16 << 20),), 0xFF, dtype=T.uint8, device="cuda")
    b.call()
    b.check()
    assert bool((b.ws[size:] == 0xFF).all())
