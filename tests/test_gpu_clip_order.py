"""What the norm of a clipping call may depend on besides the values: counts, types, where a tensor begins within a line of 32 bytes (16 in
bf16), and the GPU's number of SMs say in which order the squares are added.

The squares of fp32 and bf16 values are exact in 64 bits and are added there: by at most 2^21 additions in any order, each off by
2^-53 of a partial sum of positive terms, so two orders differ by less than 2^-31 of the sum, and of the norm by half as much; rounding
it to fp32 leaves them equal or neighbours (2^-23)."""
import pytest
import torch

from geeps_b200.ops import functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def norm_of(tensors):
    r = torch.zeros(2, device=DEV)
    F.clip_gradients(tensors, float("inf"), r)
    return r[0].item()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [31, 5000, 300_001, 2_000_000])
def test_norms_at_every_alignment(n, dtype):
    values = torch.randn(n, generator=torch.Generator(device=DEV).manual_seed(n), device=DEV).to(dtype)
    exact = values.double().square().sum().sqrt().item()
    norms = []
    for shift in range(16):
        flat = torch.full((n + 32,), 1e4, dtype=dtype, device=DEV)
        flat[shift:shift + n] = values
        norms.append(norm_of([flat[shift:shift + n]]))
        assert norms[-1] == norm_of([flat[shift:shift + n]])                       # the same call repeats bit for bit
        assert abs(norms[-1] - exact) <= (2.0 ** -24 + 2.0 ** -30) * exact
    line = 8                                                                        # values to the next such line
    assert norms[:line] == norms[line:]
    assert max(norms) - min(norms) <= 2.0 ** -23 * max(norms)
