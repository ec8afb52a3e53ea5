"""The operators around a recurrence in traced models: what their custom operators say of their outputs is what they return, the
gradient of heads comes back in the heads' layout, inference keeps nothing for a backward, and steps write the buffer they are given."""

import numpy as np
import pytest
import torch

import mlstm_kernels_b200 as mk
from mlstm_kernels_b200 import _lib
from util_layers import make

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
OPS = torch.ops.mlstm_b200


def layouts(rng, D=40):
    """x (2, 5, 3, D) in several layouts."""
    return {"plain": make(rng, 2, 5, 3, D, dtype=BF16), "heads": make(rng, 2, 3, 5, D, dtype=BF16).transpose(1, 2),
            "slice": make(rng, 2, 5, 3, 100, dtype=BF16)[..., 8:8 + D], "expanded": make(rng, 1, 5, 3, D, dtype=BF16).expand(2, 5, 3, D),
            "last_axis": make(rng, 2, 5, D, 3, dtype=BF16).transpose(2, 3), "permuted": make(rng, 3, 2, 5, D, dtype=BF16).permute(1, 2, 0, 3)}


@pytest.mark.parametrize("how", ["plain", "heads", "slice", "expanded", "last_axis", "permuted"])
def test_norm_says_what_it_returns(how):
    rng = np.random.default_rng(1)
    x = layouts(rng)[how]
    w = make(rng, 3, 40)
    test = ("test_schema", "test_faketensor")
    torch.library.opcheck(OPS.layer_norm, (x, w, w, 1e-6), test_utils=test)
    _, mean, rstd = OPS.layer_norm(x, w, w, 1e-6)
    args = (x, w, mean, rstd, make(rng, 2, 5, 3, 40, dtype=BF16), True, torch.float32)
    torch.library.opcheck(OPS.layer_norm_bw, args, test_utils=test)
    if how in ("plain", "heads", "permuted"):
        assert OPS.layer_norm_bw(*args)[0].stride() == x.stride()


def test_heads_gradient_in_their_layout():
    rng = np.random.default_rng(2)
    h, w = make(rng, 2, 3, 50, 64, dtype=BF16, grad=True), make(rng, 3, 64, grad=True)
    dy = make(rng, 2, 50, 3, 64, dtype=BF16)
    fn = lambda h, w: mk.layer_norm__b200(h.transpose(1, 2), w)  # noqa: E731
    eager = torch.autograd.grad(fn(h, w), (h, w), dy)
    traced = torch.autograd.grad(torch.compile(fn, fullgraph=True)(h, w), (h, w), dy)
    assert traced[0].is_contiguous()
    for a, b in zip(eager, traced):
        assert torch.equal(a, b)
