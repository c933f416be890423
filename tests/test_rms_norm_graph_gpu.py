"""RMSNORM in compiled graphs on the GPU against float64 and PyTorch."""

import numpy as np
import pytest
import torch
import torch.nn as nn

from forgetune_b200 import compile_model
from forgetune_b200.frontend import export_to_ir
from forgetune_b200.ir_json import evaluate

from .test_rms_norm_graph_cpu import Block

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("gpu_kernel", ["auto", "simt", "simt_exact"])
@pytest.mark.parametrize("width,fusion", [(48, True), (512, True), (33, False)])
def test_norm_block_matches(width, fusion, gpu_kernel, tmp_path):
    torch.manual_seed(width)
    model = nn.Sequential(nn.Linear(width, width), Block(width), nn.ReLU(), Block(width, affine=False, eps=1e-3),
                          nn.RMSNorm(width), nn.Linear(width, 10)).eval()
    cm = compile_model(model, (torch.randn(2, width),), output_dir=str(tmp_path), autotune=False,
                       enable_fusion=fusion, dynamic_batch=True, max_batch_size=5000, gpu_kernel=gpu_kernel)
    ir = export_to_ir(model, (torch.randn(2, width),), dynamic_batch=True, max_batch_size=5000)
    for rows in (1, 7, 64, 5000):
        x = np.random.default_rng(rows).standard_normal((rows, width)).astype(np.float32)
        want = evaluate(ir, x)
        got = cm.run(x)
        assert np.allclose(got, want, atol=1e-4, rtol=1e-4), float(np.max(np.abs(got - want)))
        dev = cm.run_device(torch.from_numpy(x).cuda())
        assert np.array_equal(dev.cpu().numpy(), got)
    cm.close()


def test_norm_as_the_output_static_batch_and_zero_rows(tmp_path):
    model = nn.Sequential(nn.Linear(64, 32), nn.RMSNorm(32)).eval()
    x = torch.randn(6, 64)
    cm = compile_model(model, (x,), output_dir=str(tmp_path), autotune=False)
    with torch.no_grad():
        want = model(x).numpy()
    assert np.allclose(cm.run(x), want, atol=1e-4, rtol=1e-4)
    cm.close()
    only = nn.Sequential(nn.RMSNorm(20)).eval()
    x = torch.randn(4, 20)
    x[1] = 0
    x[2, 3] = float("nan")
    cm = compile_model(only, (torch.randn(4, 20),), output_dir=str(tmp_path / "b"), autotune=False)
    y = cm.run(x)
    with torch.no_grad():
        assert np.allclose(y, only(x).numpy(), atol=1e-6, rtol=1e-6, equal_nan=True)
    assert np.all(y[1] == 0) and np.all(np.isnan(y[2]))
    cm.close()
