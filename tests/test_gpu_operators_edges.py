"""GPU tests of the training-side operators at the edge of what their entry points allow: layer norm without an eps.  Definitions, bounds and fixtures are
test_gpu_operators.py's."""
import pytest
import torch

from test_gpu_operators import BF16, F16, F32, dev, ln_check   # noqa: F401  (dev is a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("shape,rows", [((2, 8, 65), False), ((2, 8, 1000), False), ((1, 16, 52), False), ((2, 32, 12), False), ((2, 64, 1921), False), ((1, 20, 100), False),
                                        ((1, 3, 100), False), ((1, 100, 17), False), ((1, 300, 40), False), ((2, 520, 3), False), ((1, 8, 1024), False), ((5, 20), True),
                                        ((7, 5), True), ((3, 300), True), ((2, 2048), True)])
def test_layer_norm_without_an_eps(dev, shape, rows, dtype):   # noqa: F811
    """eps = 0: a thread without a position has no spread to divide by; nothing of it reaches the weight gradient."""
    g = torch.Generator().manual_seed(sum(shape))
    C = shape[-1] if rows else shape[1]
    x = (torch.randn(shape, generator=g) * 1.7 + 0.6).to(dtype)
    ln_check(dev, x, torch.rand(C, generator=g) + 0.5, torch.randn(C, generator=g) * 0.3, torch.randn(shape, generator=g).to(dtype), eps=0.0, channels_last=rows)
