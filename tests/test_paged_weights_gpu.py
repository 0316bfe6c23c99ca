"""infernt_paged_attention where most of a row's weights are small beside its
largest ones, as over long caches: 2^15 keys of 2^-26 to 2^-24 of the largest
weight are 2^-10 of the row together, two half-steps of fp16."""
import math

import pytest

import infernt_b200 as ib
from paged_reference import HALF_STEP, Case, new_workspace

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


@pytest.fixture(scope="module")
def ws(torch):
    return new_workspace(torch)


def light_weights(torch, seqs, D, dtype, seed):
    """Every 16th key has score 0 and value 0; the others have scores of
    -26 ln 2 to -24 ln 2 and values near 1000, so that a row's result is the
    small weights' alone.  The scores are K's first column (q is 8 there and 0
    elsewhere, the scale 1/8): exact in FP32."""
    c = Case(torch, seqs, 2, 2, D, 64, dtype, seed=seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    c.q.zero_()
    c.q[:, :, 0] = 8.0
    c.k.zero_()
    shape = c.k.shape[:3]
    c.k[..., 0] = (-(24.0 + 2.0 * torch.rand(shape, device="cuda", generator=g)) * math.log(2.0)).to(c.dtype)
    c.v.copy_(1000.0 * (1.0 + 0.1 * torch.randn(c.v.shape, device="cuda", generator=g)))
    c.k[:, :, 5::16] = 0.0
    c.v[:, :, 5::16] = 0.0
    return c


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("seqs", [[(1, 32768)], [(1, 9001)] * 40, [(70, 32768)], [(300, 5000), (1, 9001)]])
def test_light_weights_are_kept(torch, ws, seqs, D, dtype):
    """A weight w (the largest is 1) is held to half a step u, relative, and
    where fp16 runs out of normal numbers to 2^-29: the largest is stored as
    2^4, and half of fp16's last step is 2^-25.  The result adds u.  2^x is off
    by 2^-22; the FP32 sums add 16 keys at a time in the products and 32 in the
    denominator, each off by 2^-22 at most."""
    c = light_weights(torch, seqs, D, dtype, len(seqs))
    ib.paged_attention(c.out, c.q, c.cache(), c.batch(), ws, scale=0.125, lse=c.lse, err=c.err)
    torch.cuda.synchronize()
    assert int(c.err) == 0
    u, least = HALF_STEP[dtype], 2.0 ** -29 if dtype == "fp16" else 0.0
    for s, (new, n) in enumerate(seqs):
        k, v = c.dense(c.k, s)[..., 0], c.dense(c.v, s)
        for i in {0, new // 2, new - 1}:
            seen = n - new + i + 1
            w = k[:seen].exp()
            l = w.sum(0)[:, None]
            want = torch.einsum("ph,phd->hd", w, v[:seen]) / l
            sums = (seen / 16 + 64) * 2.0 ** -22
            tol = want * (2 * u + sums) + least * v[:seen].sum(0) / l
            far = (c.out[c.starts[s] + i].double() - want).abs()
            assert bool((far <= tol).all()), (s, i, float((far / want).amax()), float((tol / want).amin()))
            # the weights of a row that sees n / 16 ones: log of a sum of that size
            far = (c.lse[c.starts[s] + i].double() - l[:, 0].log()).abs()
            assert bool((far <= sums + 2.0 ** -21 * l[:, 0].log().abs()).all()), (s, i, float(far.amax()))
