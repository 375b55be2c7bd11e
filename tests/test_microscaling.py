"""What the 4-bit operators refuse without a GPU, and the plain formats they are tested against."""
import numpy as np
import pytest
import torch

import plain_microscaling as plain
from rust_deeplearning_b200.kernels import ops
from rust_deeplearning_b200.kernels.library import KernelError
from rust_deeplearning_b200.parts.model import WEIGHT_FORMATS


def test_there_is_no_cpu_path():
    x = torch.zeros(4, 64)
    for call in (lambda: ops.pack_mx8(x), lambda: ops.norm_mx8(x), lambda: ops.pack_mx4(x), lambda: ops.Mx4Weight(4, 64, False, "cpu"),
                 lambda: ops.mx8_rows(x.to(torch.float8_e4m3fn), torch.zeros(4, 2, dtype=torch.uint8)),
                 lambda: ops.mx4_weight(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8), 64),
                 lambda: ops.linear_mx4(x, x), lambda: ops.linear_gated_mx4(x, x, "silu"), lambda: ops.linear_gated_mx4(x, x, "tanh")):
        with pytest.raises(KernelError):
            call()


def test_sizes_are_checked_before_anything_else():
    for rows, columns, gated in ((0, 64, False), (4, 0, False), (3, 64, True)):
        with pytest.raises(KernelError, match="4-bit weight"):
            ops.Mx4Weight(rows, columns, gated, "cuda:0")


def test_the_plain_formats():
    """The values of both formats, every one a fixed point of its own rounding; ties go to the even code."""
    assert len(plain.E4M3) == 127 and plain.E4M3[-1] == 448 and plain.E4M3[1] == 2.0 ** -9
    for grid in (plain.E2M1, plain.E4M3):
        assert np.array_equal(plain.nearest(grid, grid), np.arange(len(grid)))
        mid = (grid[1:] + grid[:-1]) / 2
        assert np.array_equal(plain.nearest(mid, grid), np.arange(len(mid)) + np.arange(len(mid)) % 2)
    v = torch.linspace(-460, 460, 4001).clamp(-448, 448).double()        # float32 values: a cast from wider ones would round twice
    want = v.to(torch.float32).to(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(plain.E4M3[plain.nearest(v.numpy(), plain.E4M3)] * np.sign(v.numpy()), want)


def test_the_smallest_scale_that_cuts_nothing_off():
    v = np.zeros((4, 32))
    v[0, 3], v[1, 3], v[2, 3], v[3, 3] = 6.0, 6.0001, -3.0, 2.0 ** -140
    q, codes = plain.quantise(v, plain.E2M1)
    assert codes[:, 0].tolist() == [127, 128, 126, 0] and q[0, 3] == 6.0 and q[2, 3] == -3.0


def test_weight_formats_are_named():
    assert WEIGHT_FORMATS == ("mx4", "mx4+head")


def test_the_stream_without_torchs_short_cut(monkeypatch):
    """torch builds that lack the raw-stream function: the stream's number comes the long way."""
    import importlib.util
    import types
    monkeypatch.delattr(torch._C, "_cuda_getCurrentRawStream", raising=False)
    spec = importlib.util.spec_from_file_location("rust_deeplearning_b200.kernels.ops_again", ops.__file__)
    again = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(again)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda index: types.SimpleNamespace(cuda_stream=100 + index))
    assert again._raw_stream(3) == 103
