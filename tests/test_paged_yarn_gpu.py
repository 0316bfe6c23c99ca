"""YaRN with a factor up to 1: cosine and sine keep their size."""
import math

import pytest

from paged_reference import HALF_STEP
from test_paged_rope_gpu import BATCH, Rope, frequencies

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


@pytest.mark.parametrize("factor", [1.0, 0.5, 2.0 ** -16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("R", [64, 62])
def test_a_factor_that_stretches_nothing(torch, R, interleaved, factor):
    """Frequencies as for any factor; the results' tolerance is that of
    test_paged_rope_gpu with a magnitude of 1.  Angles reach 300 x 2^16 radians,
    3 10^6 turns, whose rate is off by 64 roundings of 2^-53: 2^-23 radians,
    within the 2^-20 that is counted."""
    params = dict(scaling="yarn", factor=factor, original_max_len=256, low=1.0, high=32.0)
    r = Rope(torch, BATCH, 4, 2, 64, 16, "fp32", rotary_dim=R, interleaved=interleaved, **params).run()
    f, _ = frequencies(R, **params)
    f = torch.tensor(f, dtype=torch.float64, device="cuda")
    u, half = HALF_STEP["bf16"], R // 2
    first = torch.arange(half, device="cuda") * (2 if interleaved else 1)
    second = first + (1 if interleaved else half)
    for s, (n, length) in enumerate(r.c.seqs):
        pos = torch.arange(length - n, length, device="cuda")
        angle = (pos.double()[:, None] * f)[:, None]
        rows = slice(r.c.starts[s], r.c.starts[s] + n)
        page = r.c.table[s].long()[pos // 16]
        for x, got in ((r.q[rows], r.q_out[rows]), (r.kn[rows], r.c.k[page, :, pos % 16])):
            x, got = x.double(), got.double()
            a, b = x[..., first], x[..., second]
            slack = (a.abs() + b.abs()) * 2.0 ** -20
            for want, at in ((a * angle.cos() - b * angle.sin(), first), (b * angle.cos() + a * angle.sin(), second)):
                assert bool(((got[..., at] - want).abs() <= slack + u * (want.abs() + slack)).all()), (s, factor)
            assert math.isclose(float(got[..., at].norm()), float(want.norm()), rel_tol=0.02)
