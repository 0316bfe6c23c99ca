"""Ragged batches over paged caches for the tests, and the operators' 64-bit
values restated row by row (no code shared with the library)."""
import math
import random

import infernt_b200 as ib

# half a step of each type, relative to the value
HALF_STEP = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11, "fp32": 2.0 ** -24}


def dtypes(torch):
    return {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


class Case:
    """Sequences (new tokens, length) over shuffled pages of a pool."""

    def __init__(self, torch, seqs, nq, nkv, D, page, dtype="bf16", seed=0, spare_rows=0, q_scale=1.0, spare_pages=2,
                 fill=None):
        self.torch, self.seqs, self.nq, self.nkv, self.D, self.page = torch, seqs, nq, nkv, D, page
        self.kind, self.dtype = dtype, dtypes(torch)[dtype]
        g = torch.Generator(device="cuda").manual_seed(seed)
        counts = [-(-n // page) for _, n in seqs]
        total = sum(counts) + spare_pages
        order = list(range(total))
        random.Random(seed).shuffle(order)
        width = max(counts + [1])
        rows, at = [], 0
        for c in counts:
            rows.append(order[at:at + c] + [-1] * (width - c))
            at += c
        self.pages = rows
        self.table = torch.tensor(rows, dtype=torch.int32, device="cuda").view(len(seqs), width)
        shape = (total, nkv, page, D)
        self.k = torch.randn(shape, device="cuda", generator=g).to(self.dtype)
        self.v = torch.randn(shape, device="cuda", generator=g).to(self.dtype)
        starts = [0]
        for n, _ in seqs:
            starts.append(starts[-1] + n)
        self.starts = starts
        self.rows = starts[-1] + spare_rows
        self.q_start = torch.tensor(starts, dtype=torch.int32, device="cuda")
        self.kv_len = torch.tensor([n for _, n in seqs], dtype=torch.int32, device="cuda")
        self.max_q = max(n for n, _ in seqs)
        self.q = (torch.randn(self.rows, nq, D, device="cuda", generator=g) * q_scale).to(self.dtype)
        self.out = torch.full((self.rows, nq, D), 7.0, device="cuda").to(self.dtype)
        self.lse = torch.full((self.rows, nq), 7.0, device="cuda")
        self.err = torch.zeros(1, dtype=torch.int32, device="cuda")
        if fill is not None:  # what no sequence has written
            keep = torch.zeros(total, page, dtype=torch.bool, device="cuda")
            for r, (_, n) in zip(rows, seqs):
                for p in range(n):
                    keep[r[p // page], p % page] = True
            self.k.masked_fill_(~keep[:, None, :, None], fill)
            self.v.masked_fill_(~keep[:, None, :, None], fill)

    def cache(self):
        return ib.PagedCache(self.k, self.v)

    def batch(self):
        return ib.RaggedBatch(self.q_start, self.kv_len, self.table, self.rows, self.max_q)

    def dense(self, pool, s):
        """[length][nkv][D] of sequence s in 64 bits."""
        n = self.seqs[s][1]
        if n == 0:
            return pool.new_zeros(0, self.nkv, self.D).double()
        pages = self.torch.tensor(self.pages[s][:-(-n // self.page)], device="cuda")
        return pool[pages].transpose(1, 2).reshape(-1, self.nkv, self.D)[:n].double()


def new_workspace(torch):
    return torch.zeros(ib.paged_attention_workspace_bytes(), dtype=torch.uint8, device="cuda")


def attention_row(case, q, k, v, pos, window, sinks, scale):
    """(out [nq][D], lse [nq], largest sum |q_i k_i|, largest |V|) of one token over the keys that it sees."""
    torch, G = case.torch, case.nq // case.nkv
    seen = [p for p in range(0, pos + 1) if window == 0 or p > pos - window or p < sinks]
    if not seen:
        return (torch.zeros(case.nq, case.D, dtype=torch.float64, device="cuda"),
                torch.full((case.nq,), -math.inf, dtype=torch.float64, device="cuda"), 0.0, 0.0)
    if len(seen) < pos + 1:
        at = torch.tensor(seen, device="cuda")
        k, v = k[at], v[at]
    else:
        k, v = k[:pos + 1], v[:pos + 1]
    qg = q.double().view(case.nkv, G, case.D)
    s = torch.einsum("hgd,phd->hgp", qg, k) * scale
    big = torch.einsum("hgd,phd->hgp", qg.abs(), k.abs()).amax()
    w = torch.softmax(s, -1)
    out = torch.einsum("hgp,phd->hgd", w, v).reshape(case.nq, case.D)
    return out, torch.logsumexp(s, -1).reshape(case.nq), float(big), float(v.abs().amax())


def check_attention(case, window=0, sinks=0, scale=0.0, rows=None, lse=True):
    """Every row (or `rows` of each sequence) against 64 bits.

    out = round(sum round(p) V / l): each probability and the result are off
    by half a step u of the type, relative, so 2 u max|V|.  A score is a sum
    of D products in FP32 (each step off by 2^-23 of the sum of magnitudes at
    most) scaled: e_s = (D + 2) 2^-23 scale max sum|q k|; it moves a
    probability and l by e_s each, relative.  The sums over n keys and 2^x
    (2^-22) add (n + 64) 2^-22.  lse: e_s, the sum of n terms, and the
    rounding of its own value."""
    torch = case.torch
    u, sc = HALF_STEP[case.kind], scale or 1.0 / math.sqrt(case.D)
    for s, (n, length) in enumerate(case.seqs):
        k, v = case.dense(case.k, s), case.dense(case.v, s)
        for i in (range(n) if rows is None else [x for x in rows if x < n]):
            r, pos = case.starts[s] + i, length - n + i
            out, want, big, vmax = attention_row(case, case.q[r], k, v, pos, window, sinks, sc)
            got = case.out[r].double()
            es = (case.D + 2) * 2.0 ** -23 * abs(sc) * big
            tol = vmax * (2 * u + 4 * es + (pos + 65) * 2.0 ** -22)
            if math.isfinite(tol):
                far = float((got - out).abs().amax())
                assert far <= tol, ("out", s, i, pos, far, tol)
            if lse:
                got = case.lse[r].double()
                if pos < 0:
                    assert bool((got == -math.inf).all()), ("lse", s, i, got)
                elif math.isfinite(tol):
                    far = (got - want).abs()
                    tol = es + (pos + 9) * 2.0 ** -22 + 2.0 ** -21 * want.abs()
                    assert bool((far <= tol).all()), ("lse", s, i, float(far.amax()), float(tol.amin()))
    behind = case.out[case.starts[-1]:]
    assert bool((behind == 7.0).all()) and bool((case.lse[case.starts[-1]:] == 7.0).all())
