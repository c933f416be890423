"""The matrix product's kernels one by one: every tile size, depth split and
output path against float64, exact by integers (see integers)."""

import pytest
import torch

from forgetune_b200 import fp8_linear

from . import fp8_reference as ref
from .test_fp8_gpu import TYPES, f64, integers

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,offset", [(4000, 2320, 0), (4000, 2304, 1), (2600, 4112, 0)])
def test_residual_boxes_after_boxes_stored_by_rows(m, n, offset, dtype):
    """Residual rows on 16-byte boundaries come in by TMA through the box that the output leaves by rows: at the
    right edge, or everywhere where the output is off the boundaries.  Several tiles per pair."""
    a, av = integers(m, 128, 1, seed=1)
    w, wv = integers(n, 128, 128, seed=2)
    res = (torch.arange(m * n).reshape(m, n) % 19 - 9).to(dtype).cuda()
    want, _ = ref.linear(av, wv, None, True, f64(res))
    out = torch.full((m, n + 8), 7.0, dtype=dtype, device="cuda")
    for _ in range(3):
        fp8_linear(a, w, relu=True, residual=res, out_dtype=dtype, out=out[:, offset:n + offset])
        assert torch.equal(out[:, offset:n + offset].cpu(), torch.from_numpy(want).float().to(dtype))
    assert bool((out[:, :offset] == 7).all()) and bool((out[:, n + offset:] == 7).all())
