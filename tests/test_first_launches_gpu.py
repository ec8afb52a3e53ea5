"""First launches of kernels that have just been loaded: their warps stand still for instructions at places where they never do later, and
hand-overs between the roles of a CTA must hold all the same.  Every repetition loads a copy of the library of its own."""

import ctypes
import shutil

import pytest
import torch

from mlstm_kernels_b200 import _lib, build

pytestmark = pytest.mark.gpu


def fresh_library(path):
    shutil.copy(build.LIB, path)
    lib = ctypes.CDLL(str(path))
    for name in ("mlstm_b200_chunkwise_fw", "mlstm_b200_set_unit_split", "mlstm_b200_device_status"):
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = _lib.SIGNATURES[name]
    path.unlink()   # (it stays mapped)
    return lib


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_forward_in_segments(tmp_path, dtype):
    """The recurrence with 128-column tiles beside the intra-chunk kernel, both launched for the first time: the same bits as in one piece."""
    B, NH, S, DHQK, DHHV = 1, 8, 90000, 256, 512
    NC = -(-S // 128)
    g = torch.Generator("cuda").manual_seed(1)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    new = lambda *s, dt=torch.float32: torch.empty(*s, device="cuda", dtype=dt)  # noqa: E731
    q, k, v = (rnd(B, NH, S, d).to(dtype) for d in (DHQK, DHQK, DHHV))
    i, f = rnd(B, NH, S), rnd(B, NH, S) + 4.0
    out = [new(B, NH, S, DHHV, dt=dtype), new(B, NH, S), new(B, NH, S), new(B, NH, NC + 1, DHQK, DHHV, dt=dtype), new(B, NH, NC + 1, DHQK), new(B, NH, NC + 1)]
    ws = new(1 << 30, dt=torch.uint8)

    def run(lib, split):
        lib.mlstm_b200_set_unit_split(split)
        rc = lib.mlstm_b200_chunkwise_fw(*(t.data_ptr() for t in (q, k, v, i, f)), None, None, None, *(t.data_ptr() for t in out), None, None, None,
                                         ws.data_ptr(), ws.numel(), B, NH, S, DHQK, DHHV, 128, _lib.dtype_code(dtype), _lib.F32, _lib.EXP, 0, 1e-6,
                                         torch.cuda.current_stream().cuda_stream)
        assert rc == 0
    want = None
    for n in range(24):
        lib = fresh_library(tmp_path / f"lib{n}.so")
        run(lib, 0)
        if want is None:
            want = [t.clone() for t in out]
        keep = [t.clone() for t in (out[0], out[3], out[3])]   # the GPU has something to do while kernels are loaded
        del keep
        run(lib, 1)
        for a, b in zip(want, out):
            assert torch.equal(a, b), n
        assert lib.mlstm_b200_device_status(1) == 0
