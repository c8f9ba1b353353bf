"""The cosine and sine of a rotation's angles: rows of (1, 0) turn into them."""
import pytest
import torch

from gomlx_hip import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("inverse", [False, True])
def test_cosines_and_sines(cuda, inverse):
    """Rounded to fp32 once, from values that are off by less than 2^-40 (the sine's Taylor sum to r^13
    by 2^-45, the cosine's to r^12 by 2^-41), so within half a step and 2^-40 of what they are.
    The products of positions and frequencies are exact in 64 bits (15 and 24 bits)."""
    S, half = 1 << 15, 128
    g = torch.Generator(device=cuda).manual_seed(0)
    freqs = 0.5 + 0.5 * torch.rand(half, generator=g, device=cuda)
    x = torch.zeros((1, 1, S, 2 * half), device=cuda)
    x[..., 0::2] = 1.0
    pos = torch.arange(S, dtype=torch.int32, device=cuda)[None]
    got = ops.rope(x, pos, freqs, interleaved=True, inverse=inverse)[0, 0].double()
    angle = pos[0].double()[:, None] * freqs.double()
    for at, want in ((0, torch.cos(angle)), (1, -torch.sin(angle) if inverse else torch.sin(angle))):
        half_step = torch.exp2(torch.floor(torch.log2(want.abs().clamp_min(2.0 ** -100))) - 24)
        assert ((got[:, at::2] - want).abs() <= half_step + 2.0 ** -40).all()
