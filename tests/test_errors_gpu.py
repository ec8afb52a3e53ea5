"""A call that a CUDA function refuses raises, and is over with that: the next call, this package's or PyTorch's, does not find its error."""

import numpy as np
import pytest
import torch

import mlstm_kernels_b200 as mk
from util_layers import make

pytestmark = pytest.mark.gpu


def test_a_refused_call_leaves_no_error_behind():
    """A step whose operands need more shared memory than an SM has: the limit is refused, and nothing is launched."""
    rng = np.random.default_rng(1)
    q, k, v = make(rng, 1, 1, 40000), make(rng, 1, 1, 40000), make(rng, 1, 1, 32)
    i, f, m = (make(rng, 1, 1, 1) for _ in range(3))
    c, n = make(rng, 1, 1, 40000, 32), make(rng, 1, 1, 40000)
    x, h = make(rng, 2, 64), make(rng, 2, 64)
    for after in (lambda: mk.gated_step__b200(x, x, h)[0], lambda: x * 2):   # both ask for the last error behind their launch
        with pytest.raises(RuntimeError, match="cudaErrorInvalidValue"):
            mk.mlstm_recurrent_step__b200(q, k, v, i, f, c, n, m)
        assert torch.isfinite(after()).all()
    torch.cuda.synchronize()
