"""Newton-Schulz at the ends of fp32's range: G times a power of two has the same result where eps is 0."""
import pytest
import torch

import cudatransformer_amd as ct


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 1), (2, 3), (64, 200), (200, 64), (3, 96, 96), (1024, 1100)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("power", [-125, -118, -60, 60, 118, 125])
def test_powers_of_two(power, dtype, shape):
    g = torch.Generator().manual_seed(shape[-1])
    # 8 significant bits and no magnitude below 2^-6, so that no element loses a bit as a subnormal number.
    x = torch.randn(shape, generator=g).clamp_(-3.5, 3.5)
    x = torch.where(x.abs() < 2.0 ** -6, 0.25, x).to(torch.bfloat16).to(dtype).cuda()
    y = torch.ldexp(x, torch.tensor(power, device="cuda")).to(dtype)
    assert bool(torch.isfinite(y).all()) and bool((y != 0).all())
    if power < -100 and dtype == torch.bfloat16:  # bf16's own subnormal numbers have fewer bits
        x = torch.ldexp(y.float(), torch.tensor(-power, device="cuda")).to(dtype)
    want = ct.newton_schulz(x, eps=0.0)
    assert bool(torch.isfinite(want).all())
    assert torch.equal(ct.newton_schulz(y, eps=0.0), want)


@pytest.mark.gpu
def test_zeros():
    x = torch.zeros((40, 70), device="cuda")
    assert bool((ct.newton_schulz(x) == 0).all())
    assert bool(ct.newton_schulz(x, eps=0.0).isnan().all())  # 0 / 0
