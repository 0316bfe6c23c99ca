"""paged4_rope_append against 64 bits: what the pages stand for, the codes, q;
and paged4_unpack."""
import math

import pytest

import infernt_b200 as ib
import paged4_reference as ref4
import paged_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def turned(torch, x, pos, rotary, theta, interleaved):
    """x [rows][heads][D] in 64 bits, turned at the rows' positions."""
    x = x.double().clone()
    i = torch.arange(rotary // 2, device="cuda", dtype=torch.float64)
    angle = pos.double()[:, None, None] * theta ** (-2 * i / rotary)
    a, b = (slice(0, rotary, 2), slice(1, rotary, 2)) if interleaved else (slice(0, rotary // 2),
                                                                           slice(rotary // 2, rotary))
    u, v = x[..., a].clone(), x[..., b].clone()
    x[..., a], x[..., b] = u * angle.cos() - v * angle.sin(), v * angle.cos() + u * angle.sin()
    return x


class Append:
    def __init__(self, torch, seqs, nq, nkv, D, page, dtype, source, seed=0, spare=0, offset=0, scale=1.0):
        self.torch, self.kind = torch, dtype
        self.case = ref4.Case4(torch, seqs, nq, nkv, D, page, dtype, seed=seed, spare_rows=spare)
        c = self.case
        g = torch.Generator(device="cuda").manual_seed(seed + 100)
        width = (nq + 2 * nkv) * D + 2 * offset
        qkv = (torch.randn(c.rows, width, device="cuda", generator=g) * scale).to(ref.dtypes(torch)[source])
        self.q, self.kn, self.vn = (qkv[:, a:b].view(-1, h, D) if offset == 0 else
                                    qkv.as_strided((c.rows, h, D), (width, D, 1), a)
                                    for a, b, h in ((offset, offset + nq * D, nq),
                                                    (offset + nq * D, offset + (nq + nkv) * D, nkv),
                                                    (offset + (nq + nkv) * D, offset + (nq + 2 * nkv) * D, nkv)))
        self.q_out = torch.full((c.rows, nq, D), 7.0, device="cuda").to(c.dtype)
        self.before = [x.clone() for x in (c.kc, c.vc, c.scales)]

    def run(self, rope, **kw):
        c = self.case
        ib.paged4_rope_append(self.q_out, self.q, self.kn, self.vn, c.cache(), c.batch(), rope, err=c.err, **kw)
        self.torch.cuda.synchronize()

    def places(self):
        """(rows, sequence's page, row of the page) of the rows that are written."""
        c, rows, pages, at, pos = self.case, [], [], [], []
        for s, (n, length) in enumerate(c.seqs):
            for i in range(n):
                p = length - n + i
                if p >= 0:
                    rows.append(c.starts[s] + i)
                    pages.append(c.pages[s][p // c.page])
                    at.append(p % c.page)
                    pos.append(p)
        return (self.torch.tensor(x, device="cuda", dtype=self.torch.long) for x in (rows, pages, at, pos))

    def check(self, rotary, theta, interleaved):
        torch, c = self.torch, self.case
        rows, pages, at, pos = self.places()
        want_q = turned(torch, self.q[rows], pos, rotary, theta, interleaved)
        u = ref.HALF_STEP[self.kind]
        # FP32 sine, cosine and products: 2^-21 of the pair's size
        size = want_q.abs() + self.q[rows].double().abs().amax()
        assert bool(((self.q_out[rows].double() - want_q).abs() <= u * want_q.abs() + 2.0 ** -21 * size + 2.0 ** -25).all())
        kw, vw = ref4.split_words(c.scales)
        for x, codes, w in ((turned(torch, self.kn[rows], pos, rotary, theta, interleaved), c.kc, kw),
                            (self.vn[rows].double(), c.vc, vw)):
            x = x.float()  # rounded once
            got_w, got = w[pages, :, at], ref4.values(torch, codes[pages, :, at], w[pages, :, at])
            want_c, s, zero = ref4.quantise(torch, x, self.kind)
            # a value (or a range) within FP32's rounding of a border may be on either side of it; at most one in 10^4
            ratio = (x.double() / s[..., None]).abs()
            border = ((ratio - ratio.floor() - 0.5).abs() < 2.0 ** -20) | (
                ((x.double().amax(-1).clamp(min=0) - x.double().amin(-1).clamp(max=0)) / 15 / s - 1).abs() < 2.0 ** -22)[..., None]
            same = ref4.pack(want_c) == codes[pages, :, at]
            either = border[..., 0::2] | border[..., 1::2]
            assert bool((same | either).all()) and int((~same).sum()) <= same.numel() // 10000 + 1
            words = ref4.word(torch, s, zero)
            assert int((words != got_w).sum()) <= words.numel() // 10000
            # half a step, or a whole one where the type ends; the step is at most 9 / 8 of what the range needs
            step = torch.ldexp((8 + ((got_w >> 4) & 7)).double(), ((got_w >> 7) & 255) - 130)
            assert bool(((got - x.double()).abs() <= (0.5 + 2.0 ** -20) * step[..., None]).all())
            spread = (x.double().amax(-1).clamp(min=0) - x.double().amin(-1).clamp(max=0)) / 15
            assert bool((step >= spread * (1 - 2.0 ** -22)).all())
            assert bool((step <= (spread * 1.125 * (1 + 2.0 ** -22)).clamp(min=ref4.LEAST[self.kind])).all())
        # nothing else has moved
        keep = torch.ones(c.kc.shape[0], c.page, dtype=torch.bool, device="cuda")
        keep[pages, at] = False
        for now, old in zip((c.kc, c.vc, c.scales), self.before):
            assert bool((now.transpose(1, 2)[keep] == old.transpose(1, 2)[keep]).all())
        left = torch.ones(c.rows, dtype=torch.bool, device="cuda")
        left[rows] = False
        assert bool((self.q_out[left] == 7).all())


@pytest.mark.parametrize("D,rotary", [(64, 64), (64, 32), (64, 62), (128, 128), (128, 96), (128, 2)])
@pytest.mark.parametrize("source,dtype", [("fp32", "bf16"), ("bf16", "bf16"), ("fp32", "fp16"), ("fp16", "fp16")])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rows(torch, D, rotary, source, dtype, interleaved):
    a = Append(torch, [(1, 1), (5, 300), (0, 40), (2, 1), (130, 131)], 6, 3, D, 24, dtype, source, seed=rotary, spare=3)
    a.run(ib.RopeParams(theta=10000.0, rotary_dim=rotary, interleaved=interleaved))
    assert int(a.case.err) == 0
    a.check(rotary, 10000.0, interleaved)


@pytest.mark.parametrize("offset", [1, 4, 8])
def test_rows_that_start_anywhere(torch, offset):
    a = Append(torch, [(3, 50), (1, 9)], 4, 2, 128, 16, "bf16", "fp32", offset=offset)
    a.run(ib.RopeParams(theta=500000.0, rotary_dim=128))
    a.check(128, 500000.0, False)


@pytest.mark.parametrize("heads", [(1, 1), (71, 1), (40, 20)])
def test_head_counts(torch, heads):
    a = Append(torch, [(2, 5), (1, 17)], *heads, 64, 16, "fp16", "fp16")
    a.run(ib.RopeParams(theta=10000.0, rotary_dim=64))
    a.check(64, 10000.0, False)


def test_far_positions(torch):
    """Codes at positions past 10^6 are those of 64-bit angles."""
    page = 1 << 16
    a = Append(torch, [(3, 20 * page + 7)], 2, 1, 64, page, "bf16", "fp32")
    a.run(ib.RopeParams(theta=10000.0, rotary_dim=64))
    a.check(64, 10000.0, False)


def test_a_page_does_not_depend_on_who_wrote_it(torch):
    """The same rows as one prompt, token by token, and as FP32 or bf16 sources
    on the wide and on the plain path: the same bits."""
    first = None
    for source, offset, step in (("bf16", 0, 40), ("bf16", 0, 1), ("bf16", 3, 40), ("fp32", 0, 8), ("fp32", 1, 40)):
        base = Append(torch, [(40, 40)], 4, 2, 128, 16, "bf16", "bf16", seed=5)
        a = Append(torch, [(40, 40)], 4, 2, 128, 16, "bf16", source, seed=5, offset=offset)
        a.q.copy_(base.q), a.kn.copy_(base.kn), a.vn.copy_(base.vn)
        c = a.case
        for at in range(0, 40, step):
            batch = ib.RaggedBatch(torch.tensor([0, step], dtype=torch.int32, device="cuda"),
                                   torch.tensor([at + step], dtype=torch.int32, device="cuda"), c.table, step, step)
            ib.paged4_rope_append(None, None, a.kn[at:at + step], a.vn[at:at + step], c.cache(), batch,
                                  ib.RopeParams(theta=10000.0, rotary_dim=128))
        torch.cuda.synchronize()
        kept = [x.clone() for x in (c.kc, c.vc, c.scales)]
        first = first or kept
        assert all(bool((x == y).all()) for x, y in zip(first, kept))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_values_that_are_not_finite(torch, dtype):
    """Their vectors are NaN, the others as ever; fp16 has no 10^5."""
    a = Append(torch, [(6, 6)], 2, 2, 64, 8, dtype, "fp32")
    a.kn[1, 0, 3], a.kn[2, 1, 63], a.vn[3, 0, 0], a.vn[4, 1, 7] = math.nan, math.inf, -math.inf, 1.0e5
    a.run(ib.RopeParams(theta=10000.0, rotary_dim=32))
    kw, vw = ref4.split_words(a.case.scales)
    rows, pages, at, pos = a.places()
    k_none, v_none = (w[pages, :, at] == ref4.NONE for w in (kw, vw))
    want_k, want_v = torch.zeros_like(k_none), torch.zeros_like(v_none)
    want_k[1, 0] = want_k[2, 1] = want_v[3, 0] = True
    want_v[4, 1] = dtype == "fp16"
    assert bool((k_none == want_k).all()) and bool((v_none == want_v).all())
    assert bool(torch.isnan(ref4.values(torch, a.case.kc, kw)[pages[1], 0, at[1]]).all())


@pytest.mark.parametrize("dtype,big", [("bf16", 3.3895313892515355e38), ("fp16", 65504.0)])
def test_largest_least_and_zero(torch, dtype, big):
    """At the type's ends: no value becomes infinite, a vector of zeros is zeros,
    a tiny one keeps half of the least step."""
    a = Append(torch, [(6, 6)], 2, 1, 64, 8, dtype, "fp32")
    v = a.vn
    v[0] = torch.linspace(-big, big, 64, device="cuda", dtype=torch.float64).float().clamp(-big, big)
    v[1] = big
    v[2], v[2, 0, 0] = 0, -big
    v[3] = 0
    v[4] = v[5] * ref4.LEAST[dtype]
    v[5] = torch.linspace(0.92, 1.0, 64, device="cuda") * big
    a.run(ib.RopeParams(theta=10000.0, rotary_dim=64))
    rows, pages, at, pos = a.places()
    kw, vw = ref4.split_words(a.case.scales)
    got = ref4.values(torch, a.case.vc, vw)[pages, :, at]
    step = torch.ldexp((8 + ((vw >> 4) & 7)).double(), ((vw >> 7) & 255) - 130)[pages, :, at][..., None]
    assert bool((got.abs() <= big).all()) and bool((vw[pages, :, at] != ref4.NONE).all())
    off = (got - v[rows].double()).abs() / step
    assert bool((off <= 1.0 + 2.0 ** -20).all())
    assert bool((off[[2, 3, 4]] <= 0.5 + 2.0 ** -20).all()) and not bool(got[3].any())


@pytest.mark.parametrize("rotary", [64, 62])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_ties_go_to_the_even_code(torch, dtype, rotary):
    """Values halfway between two of the scale's steps, and some last places of
    FP32 to either side of it: every code is that of the exact quotient."""
    n = 400
    a = Append(torch, [(n, n)], 2, 1, 64, 16, dtype, "fp32")
    g = torch.Generator(device="cuda").manual_seed(8)
    m, e = (torch.randint(lo, hi, (n, 1), generator=g, device="cuda") for lo, hi in ((8, 16), (-15, 4)))
    s = torch.ldexp(m.double(), e)
    zero = torch.randint(0, 16, (n, 1), generator=g, device="cuda")
    k = torch.randint(0, 15, (n, 64), generator=g, device="cuda") - zero
    x = ((k + 0.5) * s).float()
    x = (x.view(torch.int32) + torch.randint(-2, 3, x.shape, generator=g, device="cuda", dtype=torch.int32)).view(torch.float32)
    x[:, 0], x[:, 1] = (-zero * s)[:, 0].float(), ((15 - zero) * s)[:, 0].float()  # the range: 15 s
    a.vn[:, 0] = x
    a.run(ib.RopeParams(theta=10000.0, rotary_dim=rotary))
    rows, pages, at, pos = a.places()
    kw, vw = ref4.split_words(a.case.scales)
    want, want_s, want_zero = ref4.quantise(torch, x, dtype)
    assert bool((want_s == s[:, 0]).all()) and bool((want_zero == zero[:, 0]).all())
    assert bool((vw[pages, 0, at] == ref4.word(torch, want_s, want_zero)).all())
    assert bool((a.case.vc[pages, 0, at] == ref4.pack(want)).all())


def test_only_q_and_only_k(torch):
    a = Append(torch, [(3, 40)], 4, 2, 64, 16, "bf16", "bf16")
    c = a.case
    ib.paged4_rope_append(a.q_out, a.q, None, None, c.cache(), c.batch(), ib.RopeParams(rotary_dim=64))
    torch.cuda.synchronize()
    assert all(bool((x == y).all()) for x, y in zip((c.kc, c.vc, c.scales), a.before))
    ib.paged4_rope_append(None, None, a.kn, a.vn, c.cache(), c.batch(), ib.RopeParams(rotary_dim=64))
    torch.cuda.synchronize()
    a.check(64, 10000.0, False)


@pytest.mark.parametrize("rotary", [64, 30])
def test_q_in_place(torch, rotary):
    a = Append(torch, [(3, 40)], 4, 2, 64, 16, "bf16", "bf16")
    want = a.q_out.clone()
    c, rope = a.case, ib.RopeParams(rotary_dim=rotary)
    ib.paged4_rope_append(want, a.q, None, None, c.cache(), c.batch(), rope)
    q = a.q.contiguous().clone()
    ib.paged4_rope_append(q, q, a.kn, a.vn, c.cache(), c.batch(), rope)
    torch.cuda.synchronize()
    # cosines of 32 and of 64 bits differ in the last bit: two roundings of the type apart at most
    assert float((q.double() - want.double()).abs().amax()) <= 2 * ref.HALF_STEP["bf16"] * float(want.abs().amax())


def test_bad_pages_and_sequences(torch):
    a = Append(torch, [(2, 20), (2, 40), (3, 10)], 4, 2, 64, 16, "bf16", "bf16")
    c = a.case
    c.table[0, 1] = c.kc.shape[0]
    c.kv_len[1] = 1000
    a.run(ib.RopeParams(rotary_dim=64))
    assert int(c.err) == 8 | 16
    assert bool((a.q_out[2:4] == 7).all()) and not bool((a.q_out[:2] == 7).any())
    pages = torch.tensor(c.pages[2][:1], device="cuda")
    for now, old in zip((c.kc, c.vc, c.scales), a.before):
        same = (now == old).flatten(1).all(-1)
        same[pages] = True
        assert bool(same.all())


# ---------------------------------------------------------------- unpack


@pytest.mark.parametrize("nkv,page,D", [(1, 1, 64), (3, 5, 128), (8, 32, 128), (2, 300, 64)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_unpack(torch, nkv, page, D, dtype):
    case = ref4.Case4(torch, [(1, 7 * page)], nkv, nkv, D, page, dtype, seed=page)
    n = case.kc.shape[0]
    kw, vw = case.words
    kw[1], vw[2] = ref4.NONE, ref4.NONE
    case.set_words(kw, vw)
    pools = [torch.full((n + 2, nkv, page, D), 7.0, device="cuda").to(case.dtype) for _ in range(2)]
    src = torch.tensor([3, 1, 2, 3, n - 1, n, -1, 0], dtype=torch.int32, device="cuda")
    dst = torch.tensor([n + 1, 0, 5, 4, n, 1, 1, n + 2], dtype=torch.int32, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    ib.paged4_unpack(case.cache(), ib.PagedCache(*pools), src, dst, err=err)
    torch.cuda.synchronize()
    assert int(err) == 8
    for pool, values in zip(pools, (case.k, case.v)):
        want = torch.full(pool.shape, 7.0, device="cuda", dtype=torch.float64)
        for a, b in zip(src.tolist()[:5], dst.tolist()[:5]):
            want[b] = values[a]
        assert bool(((pool.double() == want) | (torch.isnan(want) & torch.isnan(pool))).all())


def test_unpack_of_many_pages(torch):
    case = ref4.Case4(torch, [(1, 70000)], 1, 1, 64, 1, "fp16")
    n = case.kc.shape[0]
    assert n > 65535
    pools = [torch.zeros(n, 1, 1, 64, device="cuda", dtype=case.dtype) for _ in range(2)]
    order = torch.randperm(n, device="cuda").to(torch.int32)
    ib.paged4_unpack(case.cache(), ib.PagedCache(*pools), order, order.flip(0).contiguous())
    torch.cuda.synchronize()
    for pool, values in zip(pools, (case.k, case.v)):
        assert bool((pool[order.flip(0).long()].double() == values[order.long()]).all())
