"""The few-token NVFP4 operators on the paths that tests of other sizes do not
take: FP16, strided rows and tokens that are not finite through the conversion
ahead of the products, the resident blocks and the router of many tokens; and
arguments that only a GPU tensor can carry."""
from __future__ import annotations

import pytest

import nvfp4_reference as ref
from test_moe_nvfp4_gpu import Layer

pytestmark = pytest.mark.gpu


def _gen(cuda, seed):
    import torch

    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    return g


def test_layer_without_a_workspace_is_refused(gplk, cuda):
    import torch

    layer = Layer(4, 128, 64, torch.bfloat16, _gen(cuda, 1), cuda)
    x = torch.zeros(2, 128, dtype=torch.bfloat16, device=cuda)
    with pytest.raises(gplk.GplkError):
        layer.run(gplk, x, 2, workspace=None)
