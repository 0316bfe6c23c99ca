"""The bounds of paged_bounds tell a right row from a wrong one: rows computed
as the kernels do (weights in 16 bits, FP32 sums) pass; zeros, a tile of V that
is lost, one that is taken twice, one from another page, a part that was not
joined, a denominator without a tile do not."""
import math

import pytest

from paged_bounds import holds
from paged_reference import HALF_STEP, dtypes

torch = pytest.importorskip("torch")
SHIFT = {"bf16": -13, "fp16": 4}


def token(n, nkv, G, D, kind, seed, peak=1.0):
    g = torch.Generator().manual_seed(seed)
    t = dtypes(torch)[kind]
    q = (torch.randn(nkv, G, D, generator=g) * peak).to(t).double()
    k, v = (torch.randn(n, nkv, D, generator=g).to(t).double() for _ in range(2))
    scale = 1.0 / math.sqrt(D)
    s = torch.einsum("hgd,phd->hgp", q, k) * scale
    big = float(torch.einsum("hgd,phd->hgp", q.abs(), k.abs()).amax())
    w = torch.softmax(s, -1)
    return dict(kind=kind, D=D, w=w, v=v, out=torch.einsum("hgp,phd->hgd", w, v), big=big, scale=scale), s


def computed(case, s, v=None, keys=slice(None), counted=slice(None)):
    """A row as the kernels have it, of `keys`, the denominator of `counted`."""
    v, t = case["v"] if v is None else v, dtypes(torch)[case["kind"]]
    p = torch.exp(s - s.amax(-1, keepdim=True)).float() * 2.0 ** SHIFT[case["kind"]]
    l = p[..., counted].sum(-1)
    o = torch.einsum("hgp,phd->hgd", p.to(t).float()[..., keys], v[keys].float())
    return (o / l[..., None]).to(t).double()


CASES = [(65, 2, 4, 64), (300, 2, 1, 128), (2000, 1, 4, 64), (9000, 1, 4, 128), (70001, 1, 8, 128)]


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("n,nkv,G,D", CASES)
def test_right_rows_pass(n, nkv, G, D, kind):
    for seed, peak in ((0, 1.0), (1, 2.0), (2, 8.0), (3, 0.0)):
        case, s = token(n, nkv, G, D, kind, seed, peak)
        assert holds(got=computed(case, s), **case), (seed, peak)


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("n,nkv,G,D", CASES)
def test_wrong_rows_do_not(n, nkv, G, D, kind):
    case, s = token(n, nkv, G, D, kind, 5)
    assert holds(got=computed(case, s), **case)
    assert not holds(got=torch.zeros_like(case["out"]), **case)
    at = torch.arange(n)
    for first in {0, n // 2 // 64 * 64, (n - 1) // 64 * 64}:
        tile = (at >= first) & (at < first + 64)
        if int(tile.sum()) < 16 or int(tile.sum()) == n:
            continue
        v = case["v"].clone()
        v[tile] = 0
        assert not holds(got=computed(case, s, v), **case), ("lost", first)
        v[tile] = 2 * case["v"][tile]
        assert not holds(got=computed(case, s, v), **case), ("twice", first)
        v[tile] = case["v"][(at >= first - 32) & (at < first - 32 + int(tile.sum()))] if first else -case["v"][tile]
        assert not holds(got=computed(case, s, v), **case), ("another page", first)
        assert not holds(got=computed(case, s, keys=~tile, counted=~tile), **case), ("not joined", first)
    part = at < n // 2
    assert not holds(got=computed(case, s, keys=part, counted=part), **case)
    # a denominator without a tile moves a row by 64 / n of itself, and two roundings are allowed 2 sqrt(2) u (the
    # log of the denominator, which calls return too, is held to 2^-22 terms)
    if 64 / n > 3 * HALF_STEP[kind]:
        assert not holds(got=computed(case, s, counted=at >= 64), **case)
