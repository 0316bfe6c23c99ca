"""How far a row of the attention over pages may be off, column by column and
over the row: bounds that shrink with the row's own sums, so that a lost tile or
part shows however long the cache is."""
import math

from paged_reference import HALF_STEP

# the smallest difference that is kept of a weight, of the row's largest (fp16: half of its last step, 2^-25, at 2^4)
LEAST = {"bf16": 0.0, "fp16": 2.0 ** -29}


def row_bounds(kind, D, w, v, out, big, scale):
    """(per column, root mean square over the row) for one token.

    w [nkv][G][n]: its weights, summing to 1; v [n][nkv][D]; out [nkv][G][D]
    their product; big: largest sum |q_i k_i|; all in 64 bits.

    A weight is rounded to the type (half a step u, relative, or LEAST of the
    largest weight), the result too.  A score is off by e = (D + 2) 2^-23 scale
    big, which moves a weight and the denominator by e each, relative (and 2^x
    by as much again); FP32 sums add 16 keys at a time, each step off by 2^-22
    of the sum.  So per column
      u sum w|V| + u |out| + (4 e + (n / 16 + 64) 2^-22) sum w|V| + LEAST max w sum |V|.
    Over the row's columns the roundings of different keys are independent: the
    root of sum w^2 V^2 takes the place of sum w|V| (and the root of D that of D
    in a score, that of n that of n), twice that for the chance of it.  A
    result below fp16's normal numbers steps by 2^-24."""
    u, n, least = HALF_STEP[kind], w.shape[-1], LEAST[kind] * float(w.amax())
    near = 2.0 ** -25 if kind == "fp16" else 0.0
    sums = (n / 16 + 64) * 2.0 ** -22
    e, e_row = ((x + 2) * 2.0 ** -23 * abs(scale) * big for x in (D, math.sqrt(D)))
    total = v.new_zeros(out.shape)
    square = v.new_zeros(out.shape)
    for h in range(w.shape[0]):
        total[h] = w[h] @ v[:, h].abs()
        square[h] = (w[h] ** 2) @ (v[:, h] ** 2)
    column = u * total + u * out.abs() + (4 * e + sums) * total + least * v.abs().sum(0)[:, None] + near
    row = 2 * math.sqrt(float(((u * u + 4 * e_row * e_row) * square + u * u * out ** 2).mean()))
    row += sums * math.sqrt(float((square + out ** 2).mean()))
    row += 2 * least * math.sqrt(float((v ** 2).sum(0).mean())) + near
    return column, row


def holds(kind, D, w, v, out, big, scale, got):
    """Whether got [nkv][G][D] is within both bounds of out."""
    column, row = row_bounds(kind, D, w, v, out, big, scale)
    far = (got - out).abs()
    return bool((far <= column).all()) and math.sqrt(float((far ** 2).mean())) <= row


def check_rows(case, window=0, sinks=0, scale=0.0, rows=None):
    """Every row (or `rows` of each sequence) of a paged_reference.Case against both bounds."""
    torch, G, sc = case.torch, case.nq // case.nkv, scale or 1.0 / math.sqrt(case.D)
    for s, (n, length) in enumerate(case.seqs):
        k, v = case.dense(case.k, s), case.dense(case.v, s)
        at = torch.arange(length, device=v.device)
        for i in (range(n) if rows is None else [x for x in rows if x < n]):
            r, pos = case.starts[s] + i, length - n + i
            got = case.out[r].double().view(case.nkv, G, case.D)
            seen = at <= pos
            if window:
                seen &= (at > pos - window) | (at < sinks)
            kk, vv = k[seen], v[seen]
            if not kk.shape[0]:
                assert bool((got == 0).all()), (s, i)
                continue
            q = case.q[r].double().view(case.nkv, G, case.D)
            w = torch.softmax(torch.einsum("hgd,phd->hgp", q, kk) * sc, -1)
            big = float(torch.einsum("hgd,phd->hgp", q.abs(), kk.abs()).amax())
            out = torch.einsum("hgp,phd->hgd", w, vv)
            column, row = row_bounds(case.kind, case.D, w, vv, out, big, sc)
            far = (got - out).abs()
            assert bool((far <= column).all()), ("column", s, i, pos, float((far / column).amax()))
            rms = math.sqrt(float((far ** 2).mean()))
            assert rms <= row, ("row", s, i, pos, rms, row)
