"""The forms that linear's products take, by rka_describe_linear (host only)."""
import ctypes

import pytest

F32, BF16 = 0, 1
THREADS = {"rows": 512, "columns": 512}


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("outputs,inputs", [(1, 1), (16, 16), (8, 24), (16, 64), (32, 16)])
def test_every_number_of_rows_has_a_launch(hip_lib, outputs, inputs, dtype):
    """A launch has fewer than 2^32 threads: rows past what few columns' kernel may have go
    to tiles, and past what small tiles may have to larger ones."""
    from rnn_kernel_amd import _lib

    for rows in (2 ** 20, 2 ** 27 - 16, 2 ** 27, 2 ** 28 + 1, 2 ** 30, 2 ** 31 - 512):
        d = _lib.describe_linear("y", rows, outputs, inputs, dtype)
        threads = THREADS.get(d["form"], 512 if d["edge"] == 256 else 256)
        assert d["workgroups"] * threads < 2 ** 32, (rows, d)
    assert _lib.describe_linear("y", 2 ** 27 - 16, 16, 16, BF16)["form"] == "columns"
    assert _lib.describe_linear("y", 2 ** 27, 16, 16, BF16)["form"] == "tiles"


def test_describe_refuses(hip_lib):
    out = (ctypes.c_int * 4)()
    assert hip_lib.rka_describe_linear(3, 4, 4, 4, 0, 1, out, 4) == 1001
    assert hip_lib.rka_describe_linear(0, 4, 4, 4, 0, 1, None, 4) == 1001
    assert hip_lib.rka_describe_linear(0, 0, 4, 4, 0, 1, out, 4) == 1001
    assert hip_lib.rka_describe_linear(0, 4, 4, 4, 2, 1, out, 4) == 1001


@pytest.mark.gpu
def test_rows_past_what_few_columns_kernel_may_have(gpu):
    """2^27 rows (4 GiB), the same 4096 over and over."""
    import torch

    from rnn_kernel_amd import linear

    gen = torch.Generator().manual_seed(0)
    x, w = torch.randn(4096, 16, generator=gen).bfloat16(), (torch.randn(16, 16, generator=gen) / 4).bfloat16()
    y = linear(x.to(gpu).repeat(2 ** 15, 1), w.to(gpu)).view(2 ** 15, 4096, 16)
    want = x.double() @ w.double().t()
    # one rounding to 8 bits, and room for a float32 sum of 16
    assert ((y[-1].double().cpu() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-5).all()
    assert torch.equal(y, y[-1:].expand_as(y))
