"""Pages of 4 bits for the tests: the format restated in 64 bits (no code
shared with the library), and ragged batches over such pages."""
import infernt_b200 as ib
import paged_reference as ref

LARGEST = {"bf16": 3.3895313892515355e38, "fp16": 65504.0}
LEAST = {"bf16": 2.0 ** -100, "fp16": 2.0 ** -21}


def quantise(torch, x, kind):
    """(codes 0..15 [..., D] int64, scale [...] float64, zero [...] int64) of
    vectors x in their last dimension (64-bit arithmetic)."""
    x = x.double()
    hi, lo = x.amax(-1).clamp(min=0), x.amin(-1).clamp(max=0)
    m, e = torch.frexp((hi - lo) / 15)
    s = torch.ldexp(torch.ceil(m * 16) / 16, e).clamp(min=LEAST[kind])
    zero = torch.round(-lo / s).clamp(0, 15)
    k = torch.round(x / s[..., None])
    k = torch.where((k * s[..., None]).abs() > LARGEST[kind], k - k.sign(), k)
    return (k + zero[..., None]).clamp(0, 15).long(), s, zero.long()


def pack(codes):
    return (codes[..., 0::2] | codes[..., 1::2] << 4).to(codes.new_zeros(0).byte().dtype)


def word(torch, s, zero):
    """16-bit words: the upper twelve bits of s as a bf16, zero below."""
    return ((s.float().view(torch.int32) >> 16) & 0xFFF0).long() | zero


NONE = 0x7FF0  # the word of a vector that is not finite


def scales(torch, k_word, v_word):
    w = k_word | v_word << 16
    return torch.where(w >= 2 ** 31, w - 2 ** 32, w).to(torch.int32)


def split_words(scales_):
    w = scales_.long() & 0xFFFFFFFF
    return w & 0xFFFF, w >> 16


def values(torch, packed, w):
    """64-bit values of packed codes and their words."""
    c = torch.stack((packed & 15, packed >> 4), -1).flatten(-2).double()
    e, m = (w >> 7) & 255, (w >> 4) & 7
    s = torch.ldexp((8 + m).double(), e - 130)
    s = torch.where(e == 255, torch.full_like(s, float("nan")), s)
    return (c - (w & 15).double()[..., None]) * s[..., None]


class Case4(ref.Case):
    """A Case whose k and v are what its 4-bit pages stand for.  k_scale and
    v_scale: factors of each position's vectors ([positions] callables of an
    index tensor), none: 1."""

    def __init__(self, torch, seqs, nq, nkv, D, page, dtype="bf16", hide=False, stretch=None, **kw):
        super().__init__(torch, seqs, nq, nkv, D, page, dtype, **kw)
        k, v = self.k.double(), self.v.double()
        if stretch is not None:
            k, v = stretch(k, v)
        kc, ks, kz = quantise(torch, k, dtype)
        vc, vs, vz = quantise(torch, v, dtype)
        self.kc, self.vc = pack(kc).contiguous(), pack(vc).contiguous()
        kw_, vw = word(torch, ks, kz), word(torch, vs, vz)
        if hide:  # rows that no sequence has written: vectors of NaN
            keep = torch.zeros(k.shape[0], page, dtype=torch.bool, device="cuda")
            for r, (_, n) in zip(self.pages, seqs):
                for p in range(n):
                    keep[r[p // page], p % page] = True
            kw_.masked_fill_(~keep[:, None], NONE)
            vw.masked_fill_(~keep[:, None], NONE)
        self.set_words(kw_, vw)

    def set_words(self, kw, vw):
        torch = self.torch
        self.words = kw, vw
        self.scales = scales(torch, kw, vw).contiguous()
        self.k, self.v = values(torch, self.kc, kw), values(torch, self.vc, vw)

    def cache(self):
        return ib.PagedCache4(self.kc, self.vc, self.scales, self.dtype)
