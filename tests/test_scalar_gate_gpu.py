"""Gates of one element: their gradient is one sum, rounded once."""
import pytest
import torch

import residual_oracle as ro
from test_residual_calls_gpu import routes  # noqa: F401

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,C", [(1000, 2), (1000, 16), (700, 1003), (5, 4096)])
def test_columns_that_cancel(routes, dtype, rows, C):  # noqa: F811
    """Columns of 100 and -100 that sum to 100 but for one element: whole numbers below 2^24, so that float32 sums are exact in any order, while a
    column of 1000 rows is beyond float16 and no multiple of bfloat16's step."""
    from spiky_b200 import residual

    def gradient():
        f, gate = torch.ones(rows, C, device=DEV, dtype=dtype), torch.ones(1, device=DEV, dtype=dtype, requires_grad=True)
        up = torch.full((rows, C), 100.0, device=DEV, dtype=dtype)
        up[:, 1::2] = -100.0
        if C % 2:
            up[:, -1] = 0.0
        up[0, 1] = 0.0
        g, = torch.autograd.grad(residual.residual_join(f, f, gate=gate), gate, up)
        assert g.dtype == dtype and g.shape == (1,) and g.item() == 100.0

    routes(gradient)


@pytest.mark.parametrize("shape", [(), (1,), (1, 1, 1, 1)])
@pytest.mark.parametrize("C", [1, 5, 64])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_shapes_of_one_element(routes, shape, C, dtype):  # noqa: F811
    from spiky_b200 import residual

    def one():
        gen = torch.Generator().manual_seed(C)
        x, f = (torch.randn(4, 3, C, generator=gen).to(dtype).to(DEV) for _ in range(2))
        gate, up = torch.full(shape, 0.75, device=DEV, dtype=dtype, requires_grad=True), torch.randn(4, 3, C, generator=gen).to(dtype).to(DEV)
        h = residual.residual_join(x, f, gate=gate)
        g, = torch.autograd.grad(h, gate, up)
        x64, f64, up64 = (t.cpu().double() for t in (x, f, up))
        ro.assert_near(h, x64 + 0.75 * f64, x64.abs() + f64.abs(), "h")
        ro.assert_near(g, (up64 * f64).sum().reshape(shape), (up64 * f64).abs().sum().reshape(shape), "gate")

    routes(one)
