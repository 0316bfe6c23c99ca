"""infernt_paged_rope_append against 64 bits: rotary layouts, parts of the
head, scalings, types, far positions, ragged batches, strides, bad device
data, graphs.

A result is x cos - y sin in FP32, rounded once: cosine and sine are off by
2^-22 at most (the fraction of a turn enters in FP32: 2 pi 2^-26, and
sincospif by 2 ulp), the products and the sum by 2^-23 each, so
|off| <= m (|x| + |y|) 2^-20 + u |result|, u half a step of the type.  What
is copied is the rounding of its source."""
import math

import pytest

import infernt_b200 as ib
from paged_reference import HALF_STEP, Case, dtypes

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def frequencies(R, theta=10000.0, scaling="none", original_max_len=0, factor=1.0, low=1.0, high=4.0, **_):
    out, much = [], 1.0
    for i in range(R // 2):
        f = theta ** (-2.0 * i / R)
        turns = original_max_len * f / (2 * math.pi)
        if scaling == "linear":
            f /= factor
        elif scaling == "llama3":
            if turns < low:
                f /= factor
            elif turns <= high:
                mix = (turns - low) / (high - low)
                f = (1 - mix) * f / factor + mix * f
        elif scaling == "yarn":
            def at(t):
                return R * math.log(original_max_len / (t * 2 * math.pi)) / (2 * math.log(theta))
            lo, hi = max(math.floor(at(high)), 0), min(math.ceil(at(low)), R - 1)
            mix = min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0)
            f = f / factor * mix + f * (1 - mix)
            much = 0.1 * math.log(factor) + 1.0
        out.append(f)
    return out, much


class Rope:
    def __init__(self, torch, seqs, nq, nkv, D, page, src="bf16", dtype="bf16", seed=0, spare_rows=0, **params):
        self.torch, self.src = torch, src
        self.c = Case(torch, seqs, nq, nkv, D, page, dtype, seed=seed, spare_rows=spare_rows)
        g = torch.Generator(device="cuda").manual_seed(seed + 100)
        t = dtypes(torch)[src]
        rows = self.c.rows
        self.q = torch.randn(rows, nq, D, device="cuda", generator=g).to(t)
        self.kn = torch.randn(rows, nkv, D, device="cuda", generator=g).to(t)
        self.vn = torch.randn(rows, nkv, D, device="cuda", generator=g).to(t)
        self.q_out = torch.full((rows, nq, D), 7.0, device="cuda").to(self.c.dtype)
        self.params = dict(rotary_dim=D)
        self.params.update(params)
        self.k0, self.v0 = self.c.k.clone(), self.c.v.clone()

    def run(self, stream=None):
        ib.paged_rope_append(self.q_out, self.q, self.kn, self.vn, self.c.cache(), self.c.batch(),
                             ib.RopeParams(**self.params), err=self.c.err, stream=stream)
        self.torch.cuda.synchronize()
        return self

    def turn(self, x, pos):
        """(value, tolerance) of rows x [n][heads][D] at positions pos [n], in 64 bits."""
        torch, p, D = self.torch, self.params, x.shape[-1]
        R, u = p["rotary_dim"], HALF_STEP[self.c.kind]
        f, much = frequencies(R, **{k: v for k, v in p.items() if k != "rotary_dim"})
        angle = (pos.double()[:, None] * torch.tensor(f, dtype=torch.float64, device="cuda"))[:, None]
        x = x.double()
        out, tol = x.clone(), x.abs() * u
        a, b = ((slice(0, R, 2), slice(1, R, 2)) if p.get("interleaved") else (slice(0, R // 2), slice(R // 2, R)))
        out[..., a] = much * (x[..., a] * angle.cos() - x[..., b] * angle.sin())
        out[..., b] = much * (x[..., b] * angle.cos() + x[..., a] * angle.sin())
        slack = much * (x[..., a].abs() + x[..., b].abs()) * 2.0 ** -20
        tol[..., a] = slack + u * (out[..., a].abs() + slack)
        tol[..., b] = slack + u * (out[..., b].abs() + slack)
        # fp16 results below its normal range step by 2^-24
        return out, tol + (2.0 ** -25 if self.c.kind == "fp16" else 0.0)

    def check(self, q=True, k=True):
        torch, c = self.torch, self.c
        want_k, want_v = self.k0.double(), self.v0.double()
        tol_k = torch.zeros_like(want_k)
        hit = torch.zeros(c.k.shape[0], c.page, dtype=torch.bool, device="cuda")
        for s, (n, length) in enumerate(c.seqs):
            a = c.starts[s]
            pos = torch.arange(length - n, length, device="cuda")
            ok = pos >= 0
            if n and q:
                out, tol = self.turn(self.q[a:a + n], pos)
                far = (self.q_out[a:a + n].double() - out).abs()
                assert bool((far <= tol)[ok].all()), ("q", s, float((far - tol)[ok].amax()))
                assert bool((self.q_out[a:a + n][~ok] == 7).all())
            if n and k and bool(ok.any()):
                p = pos[ok]
                page = c.table[s].long()[p // c.page]
                kk, tol = self.turn(self.kn[a:a + n][ok], p)
                want_k[page, :, p % c.page] = kk
                tol_k[page, :, p % c.page] = tol
                want_v[page, :, p % c.page] = self.vn[a:a + n][ok].to(c.dtype).double()
                hit[page, p % c.page] = True
        far = (c.k.double() - want_k).abs()
        assert bool((far <= tol_k).all()), ("k", float((far - tol_k).amax()))
        assert bool((c.v.double() == want_v).all())
        assert bool((self.q_out[c.starts[-1]:] == 7).all())


BATCH = [(1, 1), (5, 5), (1, 300), (40, 100), (3, 16), (1, 17)]


@pytest.mark.parametrize("src,dtype", [("fp32", "bf16"), ("bf16", "bf16"), ("fp16", "fp16"), ("fp32", "fp16"),
                                       ("fp16", "bf16"), ("bf16", "fp16")])
@pytest.mark.parametrize("interleaved", [False, True])
def test_types(torch, src, dtype, interleaved):
    Rope(torch, BATCH, 8, 2, 128, 16, src, dtype, interleaved=interleaved, spare_rows=3).run().check()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,R", [(64, 64), (64, 32), (64, 16), (64, 2), (64, 62), (64, 6), (128, 128), (128, 64),
                                 (128, 126), (128, 100), (128, 24), (128, 8)])
def test_parts_of_the_head(torch, D, R, interleaved):
    for src in ("bf16", "fp32"):
        Rope(torch, BATCH, 6, 3, D, 16, src, rotary_dim=R, interleaved=interleaved).run().check()


SCALINGS = [dict(theta=500000.0), dict(scaling="linear", factor=4.0),
            dict(theta=500000.0, scaling="llama3", factor=8.0, original_max_len=8192, low=1.0, high=4.0),
            dict(scaling="yarn", factor=16.0, original_max_len=4096, low=1.0, high=32.0),
            dict(theta=100.0, scaling="yarn", factor=2.0, original_max_len=64, low=1.0, high=32.0),
            dict(theta=10.0, scaling="llama3", factor=2.0, original_max_len=16, low=1.0, high=4.0)]


@pytest.mark.parametrize("params", SCALINGS)
@pytest.mark.parametrize("R", [64, 48])
def test_scalings(torch, params, R):
    Rope(torch, BATCH + [(7, 5000)], 4, 2, 64, 32, "fp32", rotary_dim=R, **params).run().check()


@pytest.mark.parametrize("length", [131072, 1000003, (1 << 24) + 5])
def test_far_positions(torch, length):
    """Angles of 10^5 to 10^7 radians; the table points all pages before the
    last at one page."""
    r = Rope(torch, [(9, 9)], 4, 2, 128, 16, "fp32", "fp16")
    c = r.c
    width = -(-length // 16)
    table = torch.zeros(1, width, dtype=torch.int32, device="cuda")
    table[0, -1], table[0, -2] = 1, 2
    c.table, c.seqs = table, [(9, length)]
    c.kv_len.fill_(length)
    r.run().check()


@pytest.mark.parametrize("seqs", [[(1, 1)], [(2, 1), (1, 0), (0, 9), (40, 10)], [(0, 0), (0, 5), (3, 3), (0, 7)]])
def test_negative_positions_and_empty_sequences(torch, seqs):
    r = Rope(torch, seqs, 4, 2, 64, 16, spare_rows=2).run()
    r.check()
    assert int(r.c.err) == 0


@pytest.mark.parametrize("n", [31, 32, 33, 64, 1000, 1100])
def test_many_sequences(torch, n):
    Rope(torch, [(i % 3, 1 + i % 50 + i % 3) for i in range(n)], 2, 1, 64, 8).run().check()


@pytest.mark.parametrize("page", [1, 5, 24, 100, 256])
def test_page_sizes(torch, page):
    Rope(torch, BATCH, 4, 2, 64, page).run().check()


def test_rotation_only_and_append_only(torch):
    r = Rope(torch, BATCH, 8, 2, 64, 16)
    p, cache, batch = ib.RopeParams(**r.params), r.c.cache(), r.c.batch()
    ib.paged_rope_append(r.q_out, r.q, None, None, cache, batch, p)
    torch.cuda.synchronize()
    assert bool((r.c.k == r.k0).all()) and bool((r.c.v == r.v0).all())
    first = r.q_out.clone()
    r.q_out.fill_(7)
    ib.paged_rope_append(None, None, r.kn, r.vn, cache, batch, p)
    torch.cuda.synchronize()
    assert bool((r.q_out == 7).all())
    r.check(q=False)
    r.q_out.copy_(first)
    r.check()


@pytest.mark.parametrize("src", ["bf16", "fp32"])
def test_stacked_rows_and_odd_strides(torch, src):
    """q, k and v slices of stacked rows; then rows an odd number of values
    apart from an odd address, where no wide load fits."""
    for pad, shift in ((0, 0), (64, 0), (3, 1)):
        r = Rope(torch, BATCH, 6, 2, 64, 16, src)
        t, n = r.q.dtype, r.c.rows
        ld = 10 * 64 + pad
        flat = torch.zeros(n * ld + shift + 8, device="cuda", dtype=t)
        view = flat[shift:shift + n * ld].view(n, ld)[:, :640].view(n, 10, 64)
        view[:, :6], view[:, 6:8], view[:, 8:] = r.q, r.kn, r.vn
        r.q, r.kn, r.vn = view[:, :6], view[:, 6:8], view[:, 8:]
        out = torch.full((n * (6 * 64 + pad) + 8,), 7.0, device="cuda").to(r.c.dtype)
        r.q_out = out[shift:shift + n * (384 + pad)].view(n, 384 + pad)[:, :384].view(n, 6, 64)
        r.run().check()
        if pad:
            assert bool((out[shift:shift + n * (384 + pad)].view(n, -1)[:, 384:] == 7).all())


@pytest.mark.parametrize("R,interleaved", [(64, False), (64, True), (32, False), (62, True)])
def test_in_place(torch, R, interleaved):
    r = Rope(torch, BATCH, 8, 2, 64, 16, rotary_dim=R, interleaved=interleaved)
    q0 = r.q.clone()
    r.q_out = r.q
    r.run()
    r.q = q0
    r.check()


def test_bad_pages_and_lengths(torch):
    r = Rope(torch, [(4, 40), (3, 20), (2, 30)], 4, 2, 64, 16)
    c = r.c
    c.table[0, 2] = 1000          # positions 32..39 of sequence 0
    c.kv_len[1] = 16 * c.table.shape[1] + 1
    r.run()
    assert int(c.err) == (1 << 3) | (1 << 4)
    # sequence 0 is rotated and not appended, sequence 1 skipped, sequence 2 whole
    assert bool((r.q_out[4:7] == 7).all())
    out, tol = r.turn(r.q[:4], torch.arange(36, 40, device="cuda"))
    assert bool(((r.q_out[:4].double() - out).abs() <= tol).all())
    c.seqs[0], c.seqs[1] = (0, 0), (0, 0)
    r.check()


def test_offsets_past_32_bits(torch):
    r = Rope(torch, [(3, 40)], 4, 8, 128, 64)
    c = r.c
    pages = (1 << 31) // (8 * 64 * 128) + 10
    big_k = torch.empty(pages, 8, 64, 128, device="cuda", dtype=c.dtype)
    big_v = torch.empty_like(big_k)
    p = c.pages[0][0]
    big_k[-1], big_v[-1] = c.k[p], c.v[p]
    small = (c.k, c.v)
    c.k, c.v = big_k, big_v
    c.table.fill_(pages - 1)
    r.run()
    small[0][p], small[1][p] = big_k[-1], big_v[-1]
    c.k, c.v = small
    c.table.fill_(p)
    r.check()


def test_captured_call_and_side_stream(torch):
    r = Rope(torch, [(2, 20), (1, 30)], 4, 2, 64, 16)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        r.run(stream=st.cuda_stream).check()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        ib.paged_rope_append(r.q_out, r.q, r.kn, r.vn, r.c.cache(), r.c.batch(), ib.RopeParams(**r.params),
                             err=r.c.err, stream=st.cuda_stream)
    r.c.kv_len.copy_(torch.tensor([25, 7], dtype=torch.int32))
    r.c.seqs = [(2, 25), (1, 7)]
    r.k0, r.v0 = r.c.k.clone(), r.c.v.clone()
    g.replay()
    torch.cuda.synchronize()
    r.check()


def test_host_memory_is_refused(torch):
    r = Rope(torch, [(2, 20)], 4, 2, 64, 16)
    cache, batch, p = r.c.cache(), r.c.batch(), ib.RopeParams(**r.params)
    for q_out, q, k, v in ((r.q_out.cpu(), r.q, r.kn, r.vn), (r.q_out, r.q.cpu(), r.kn, r.vn),
                           (r.q_out, r.q, r.kn.cpu(), r.vn), (r.q_out, r.q, r.kn, r.vn.cpu())):
        with pytest.raises(ib.InferntError):
            ib.paged_rope_append(q_out, q, k, v, cache, batch, p)
    r.run().check()
