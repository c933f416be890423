"""RMSNORM in compiled graphs, without a GPU: lowering, planning, refusals."""

import numpy as np
import pytest
import torch
import torch.nn as nn

from forgetune_b200 import UnsupportedOpError, _native, export_to_ir, to_graph_json
from forgetune_b200.errors import ForgeTuneRuntimeError
from forgetune_b200.graph_blob import serialize
from forgetune_b200.ir_json import evaluate


class Block(nn.Module):
    def __init__(self, n=48, affine=True, eps=None):
        super().__init__()
        self.norm = nn.RMSNorm(n, eps=eps, elementwise_affine=affine)
        self.fc = nn.Linear(n, n)
        if affine:
            nn.init.normal_(self.norm.weight, 1.0, 0.2)

    def forward(self, x):
        return x + self.fc(self.norm(x))


def lowered(model, shape=(3, 48), dynamic=True):
    torch.manual_seed(0)
    x = torch.randn(shape)
    return export_to_ir(model.eval(), (x,), dynamic_batch=dynamic, max_batch_size=64), x


@pytest.mark.parametrize("dynamic", [True, False])
@pytest.mark.parametrize("affine,eps", [(True, None), (True, 1e-3), (False, 1e-5)])
def test_lowering_and_plan(affine, eps, dynamic):
    model = Block(affine=affine, eps=eps)
    ir, x = lowered(model, dynamic=dynamic)
    with torch.no_grad():
        assert np.allclose(evaluate(ir, x.numpy()), model(x).numpy(), atol=1e-5, rtol=1e-5)
    desc = _native.describe_blob(serialize(ir, enable_fusion=True, bias_first_fused=True))
    assert [s["kind"] for s in desc["steps"]] == [13, 0]  # the norm, then the Linear with bias and residual folded
    assert [n["op"] for n in desc["nodes"]].count("RMSNORM") == 1


def test_refusals():
    with pytest.raises(UnsupportedOpError):
        lowered(nn.Sequential(nn.RMSNorm([4, 4])), (2, 3, 4, 4), dynamic=False)
    ir, _ = lowered(Block())
    with pytest.raises(UnsupportedOpError):
        to_graph_json(ir)
    for eps in (-1.0, float("nan"), float("inf")):
        for n in ir.nodes:
            if n.op == "RMSNORM":
                n.eps = eps
        with pytest.raises(ForgeTuneRuntimeError, match="eps"):
            _native.describe_blob(serialize(ir, enable_fusion=True, bias_first_fused=True))
