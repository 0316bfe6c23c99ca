"""verify_drafts where the temperature is tiny beside the logits, or the logits
are far from 0: the drawn token is the formula's own, and no token of
probability 0 is ever drawn."""
import math

import pytest

import test_verify_gpu as verify

pytestmark = pytest.mark.gpu

LOWEST = -3.4028234663852886e38


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


class Sharp(verify.Step):
    """Rows of the largest logit `top`, a few logits up to six FP32 steps below it, the rest some 5 % lower, a
    fifth of the tokens at -infinity; drafts that are mostly not the likeliest tokens."""

    def __init__(self, torch, top, t, draft, dtype="float32", V=1001, seed=0):
        super().__init__(torch, [1, 2, 2, 3, 1, 2] * 5, V, draft=False, seed=seed, banned=False)
        g = torch.Generator(device="cuda").manual_seed(seed + 1)
        rows = self.rows

        def rand(*shape):
            return torch.rand(*shape, generator=g, device="cuda")

        x = torch.full((rows, V), top, dtype=torch.float32, device="cuda")
        x = x - (0.02 + 0.08 * rand(rows, V)) * max(abs(top), 1e-3)
        x = torch.where(x < LOWEST, LOWEST, x)
        step = torch.full((rows, 1), top, dtype=torch.float32, device="cuda")
        for i in range(7):  # 0 to 6 steps below, at places of their own, two of each
            for _ in range(2):
                x.scatter_(1, torch.randint(V, (rows, 1), generator=g, device="cuda"), step)
            step = torch.nextafter(step, torch.full_like(step, LOWEST))
        x.scatter_(1, torch.randint(V, (rows, 1), generator=g, device="cuda"), top)
        keep = torch.arange(V, device="cuda") % 5 != 3
        keep[0] = False  # a number of 0 draws no token that may not be
        x = torch.where(keep | (x == top), x, -math.inf)
        x[:, 0] = -math.inf
        self.target = x.to(getattr(torch, dtype)).contiguous()
        self.temps = [t] * len(self.counts)
        self.temperature = torch.tensor(self.temps, device="cuda")
        if draft:
            q = rand(rows, V)
            q = 0.5 * q / q.sum(-1, keepdim=True)
            q.scatter_add_(1, torch.randint(V, (rows, 1), generator=g, device="cuda"), torch.full((rows, 1), 0.5, device="cuda"))
            self.draft = q
        best = self.target.double().argmax(-1)
        other = torch.randint(1, V, (rows,), generator=g, device="cuda")
        d = torch.where(rand(rows) < 0.3, best, other).to(torch.int32)
        self.tokens = torch.cat((d[:1] * 0, d[:-1]))
        self.u = rand(rows).clamp(min=1e-3)
        last = torch.tensor(self.starts[1:], device="cuda") - 1
        self.u[last[::3]] = 0.0
        self.u[last[1::3]] = 1.0 - 2.0 ** -24

    def row(self, r, t):
        """Weights of 2^-990 of the largest and below are 0."""
        p, best, fine = super().row(r, t)
        if t > 0 and fine:
            p = self.torch.where(p > p.amax() * 2.0 ** -990, p, 0.0)
        return p, best, fine

    def check_sharp(self):
        assert self.check(2) == 0
        for s, n in enumerate(self.counts):
            a, acc = self.starts[s], int(self.accepted[s])
            token = int(self.out[a + acc])
            assert 0 <= token < self.V and float(self.target[a + acc, token]) > -math.inf, (s, token)


@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("top", [0.5, 20.1, -20.1, 1000.0, 0.0])
@pytest.mark.parametrize("t", [1e-3, 1e-5, 1e-6, 1e-7, 1e-8, 1e-9, 1e-12, 1e-20, 1e-30, 1e-38])
def test_tiny_temperatures(torch, t, top, draft):
    s = Sharp(torch, top, t, draft, seed=int(-10 * math.log10(t) + abs(top)))
    s.run()
    s.check_sharp()


@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("t", [1.0, 0.7, 30.0, 1e-9])
@pytest.mark.parametrize("top", [-1e4, -1e9, -1e10, -1e20, LOWEST, 1e10, 3e38])
def test_logits_far_from_zero(torch, top, t, draft):
    """Rows of which all that is allowed lies at a mask's value, the type's
    lowest among them."""
    s = Sharp(torch, top, t, draft, seed=int(abs(math.log10(abs(top)))))
    s.run()
    s.check_sharp()


@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("dtype,top", [("bfloat16", -3.3895313892515355e38), ("bfloat16", 12.0), ("float16", -65504.0),
                                       ("float16", 12.0)])
@pytest.mark.parametrize("t", [1.0, 1e-9])
def test_sixteen_bits(torch, dtype, top, t, draft):
    s = Sharp(torch, top, t, draft, dtype=dtype, V=5000, seed=7)
    s.run()
    s.check_sharp()
