"""lb_rotary's cosines and sines by themselves: rows of pairs (1, 0) become (cos, sin) of their angles.

Each is right to 2^-21 of itself, however near a multiple of a quarter turn the angle lies: 2 ulp of the function (2^-22) and three
roundings to 32 bits (what is left of the angle, its product, the sum; 2^-24 each), and the angle's own error in 64 bits, three roundings
of it: 2^-51 |position frequency|.  A part of a turn rounded to 32 bits would be off by 2^-24 of a turn there, whatever is left of the sine."""
import numpy as np
import pytest
import torch

import lowbit_hip as lb
from conftest import announce

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('pairs', ['half', 'neighbours'])
@pytest.mark.parametrize('back', [False, True], ids=['on', 'back'])
def test_small_sines(device, pairs, back):
    announce('rotary angles', pairs, back)
    n, rows = 256, 2000
    g = torch.Generator().manual_seed(1)
    f = torch.rand(n, generator=g, dtype=torch.float64) * 3
    f[:16] = torch.arange(16, dtype=torch.float64) * (np.pi / 8) * (1 + 2.0 ** -30)       # near eighths of a turn
    x = torch.zeros((1, rows, 1, 2 * n), device=device)
    at = (slice(0, n), slice(n, 2 * n)) if pairs == 'half' else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    x[..., at[0]] = 1
    position = torch.randint(-131072, 131072, (1, rows), generator=g)
    position[0, :3] = torch.tensor([0, 8, -4])
    out = lb.rotary(x, position.to(device), lb.Rotary(f.to(device), pairs=pairs), back=back)[0, :, 0].double().cpu().numpy()
    angle = position[0][:, None].numpy().astype(np.float64) * f.numpy()
    for got, want in ((out[:, at[0]], np.cos(angle)), (out[:, at[1]], np.sin(angle) * (-1 if back else 1))):
        limit = 2.0 ** -21 * np.abs(want) + 2.0 ** -51 * np.abs(angle) + 2.0 ** -126
        worst = float(np.max(np.abs(got - want) / limit))
        assert worst <= 1, worst
