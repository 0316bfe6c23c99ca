"""Cases of the operators of a drafting step over paged caches held in 4 bits, with their plain forms.

Five operators, as such a step calls them: block tables, lengths and slots from what each request holds and wants;
rotary positions with the append of K and V rows in 4 bits, and the pages' values in 16 bits again; attention of a
ragged batch of new tokens over such pages; verification of drafted tokens against the target's distributions.  A case
names its operator and its sizes; lengths are spread evenly between the case's bounds and dealt to the sequences by
the seed.

The 4 bits: a vector x of a KV head at a position is held as whole numbers k = round(x / s), s k being the value, with
s the range of x and 0 over 15, rounded up to four significant bits, and codes c = k + zero in 0..15.  s k has eight
significant bits, so a value is a number of bf16 and of fp16 as it is.
"""
import math

import torch

own = False

# The attention's workspace: a fixed size, zeroed once by its owner.
WORKSPACE_BYTES = 64 << 20

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
LARGEST = {"bf16": 3.3895313892515355e38, "fp16": 65504.0}
LEAST_SCALE = {"bf16": 2.0 ** -100, "fp16": 2.0 ** -21}

ROPE = {
    # plain: the 1.1B shape's; llama3: the 8B shape's theta with the scaling of its long-context successor;
    # yarn: another scaling in common use
    "plain": dict(theta=10000.0, scaling="none", factor=1.0, low=1.0, high=4.0, original=2048),
    "llama3": dict(theta=500000.0, scaling="llama3", factor=8.0, low=1.0, high=4.0, original=8192),
    "yarn": dict(theta=10000.0, scaling="yarn", factor=16.0, low=1.0, high=32.0, original=4096),
}


def attention(name, seqs, chunks, chunk, rest, lo, hi, nq, nkv, dim, page, window=0, sinks=0, dtype="bf16"):
    """`chunks` of the `seqs` sequences bring `chunk` new tokens each, the others `rest`; lengths lo..hi."""
    return dict(name=name, op="attention", seqs=seqs, chunks=chunks, chunk=chunk, rest=rest, lo=lo, hi=hi, nq=nq,
                nkv=nkv, dim=dim, page=page, window=window, sinks=sinks, dtype=dtype)


def append(name, seqs, chunk, lo, hi, nq, nkv, dim, page, rotary, interleaved, scaling, source, dtype):
    return dict(name=name, op="append", seqs=seqs, chunks=0, chunk=chunk, rest=chunk, lo=lo, hi=hi, nq=nq, nkv=nkv,
                dim=dim, page=page, rotary=rotary, interleaved=interleaved, scaling=scaling, source=source,
                dtype=dtype)


def verify(name, seqs, lo, hi, vocab, kind, dtype, draft, greedy):
    """lo..hi drafted tokens a sequence; kind: logits or probs; draft: their distributions are given; every
    `greedy`-th sequence has temperature 0 (0: none)."""
    return dict(name=name, op="verify", seqs=seqs, lo=lo, hi=hi, vocab=vocab, kind=kind, dtype=dtype, draft=draft,
                greedy=greedy)


def plan(name, seqs, lo, hi, new_lo, new_hi, page, spare, then):
    """Sequences that hold lo..hi positions and want new_lo..new_hi more, `spare` hundredths of the pages that these
    need being free; then: "trim" to what is kept of them, or "free" all."""
    return dict(name=name, op="plan", seqs=seqs, lo=lo, hi=hi, new_lo=new_lo, new_hi=new_hi, page=page, spare=spare,
                then=then)


def listed():
    return [
        # the first tokens of one chat on the 1.1B shape: latency
        attention("attention_one", 1, 0, 1, 1, 37, 37, 32, 4, 64, 16),
        # 16 long documents on the 8B shape: the whole cache is read once
        attention("attention_long", 16, 0, 1, 1, 32768, 32768, 32, 8, 128, 32),
        # four drafted tokens and the last one of 64 sequences of the 1.1B shape, at the batched benchmark's contexts
        attention("attention_drafts", 64, 0, 5, 5, 512, 2048, 32, 4, 64, 32),
        # one chunk of a long prompt on the 8B shape: the tensor cores' work
        attention("attention_chunk", 1, 1, 4096, 1, 12288, 12288, 32, 8, 128, 32),
        # a step of continuous batching, fp16: a prompt's chunk among drafts, odd pages, a window and first tokens
        attention("attention_mixed", 16, 1, 509, 3, 700, 4001, 32, 8, 128, 24, window=1500, sinks=4, dtype="fp16"),
        # the step of 64 sequences with four drafted tokens each on the 8B shape, FP32 projection rows
        append("append_drafts", 64, 5, 60, 300, 32, 8, 128, 32, 128, False, "llama3", "fp32", "bf16"),
        # a prompt on the 8B shape
        append("append_prompt", 1, 8192, 8192, 8192, 32, 8, 128, 32, 128, False, "llama3", "bf16", "bf16"),
        # one chat of the 1.1B shape's vocabulary with four drafts: latency
        verify("verify_one", 1, 4, 4, 32000, "logits", "fp32", True, 0),
        # 64 sequences of four drafts with the 8B shape's vocabulary
        verify("verify_batch", 64, 4, 4, 128256, "logits", "fp32", True, 0),
        # drafts found in the prompt, which have no distribution, 0 to 7 of them; every third request is greedy
        verify("verify_ragged", 100, 0, 7, 32000, "logits", "bf16", False, 3),
        # the step of 256 requests with up to 8 drafts, most of which are given back
        plan("plan_step", 256, 100, 4000, 1, 9, 16, 100, "trim"),
        # 100 prompts admitted at once, for which the pool does not quite suffice, and their end
        plan("plan_prompts", 100, 0, 0, 17, 8192, 32, 95, "free"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "append", "verify", "verify", "plan"])
    nkv = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 8])
    dim = rng.choice([64, 128])
    page = rng.choice([1, 8, 16, 24, 32, 64, 100, 128, 256])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "attention":
        chunk = rng.choice([1, _log(rng, 2, 16), _log(rng, 2, 16), _log(rng, 16, 3000)])
        rest = rng.choice([1, min(chunk, rng.randint(1, 6))])
        hi = max(chunk, _log(rng, 16, 32768))
        if chunk > 16:  # the plain form's scores: seqs x chunk x heads x hi floats
            hi = max(chunk, min(hi, 8192))
            seqs = max(1, min(_log(rng, 1, 16), int(1.2e9 / (chunk * nkv * group * hi))))
            if seqs == 1:
                hi = max(chunk, min(hi, int(1.2e9 / (chunk * nkv * group))))
        else:
            seqs = max(1, min(_log(rng, 1, 96), int(4.0e8 / (hi * nkv * dim)), int(1.2e9 / (chunk * nkv * group * hi))))
        window = rng.choice([0, 0, _log(rng, 1, max(2, hi))])
        sinks = rng.choice([0, 1, 4, 64, 200]) if window else 0
        c = attention("", seqs, rng.randint(1, seqs), chunk, rest, max(1, chunk, hi // rng.randint(1, 8)), hi,
                      nkv * group, nkv, dim, page, window, sinks, dtype)
    elif op == "append":
        chunk = _log(rng, 1, 4000)
        seqs = max(1, min(_log(rng, 1, 64), 8000 // chunk))
        hi = max(chunk, min(_log(rng, 16, 32768), 30000 // seqs))
        rotary = rng.choice([dim, dim // 2, dim // 4, dim - 2])
        c = append("", seqs, chunk, max(chunk, hi // 3), hi, nkv * group, nkv, dim, page, rotary, rng.random() < 0.5,
                   rng.choice(sorted(ROPE)), rng.choice(["fp32", dtype]), dtype)
    elif op == "verify":
        vocab, hi = _log(rng, 11, 152000), rng.choice([0, 1, 2, 4, 8])
        seqs = max(1, min(_log(rng, 1, 256), int(4.0e7 / (vocab * (hi + 1)))))
        kind = rng.choice(["logits", "logits", "probs"])
        c = verify("", seqs, rng.randint(0, hi), hi, vocab, kind, "fp32" if kind == "probs" else
                   rng.choice(["fp32", "bf16", "fp16"]), rng.random() < 0.6, rng.choice([0, 0, 1, 2, 5]))
    else:
        seqs, page = _log(rng, 1, 3000), rng.choice([8, 16, 24, 32, 64, 100, 128])
        then = rng.choice(["trim", "trim", "free"])
        new = rng.randint(1, 9) if then == "trim" else _log(rng, 1, max(2, min(8192, 700000 // seqs)))
        hi = _log(rng, 1, 8000)
        c = plan("", seqs, rng.randint(0, hi), hi, rng.randint(0, new), new, page, rng.choice([60, 95, 100, 100, 130]),
                 then)
    del c["name"]
    return c


# ---------------------------------------------------------------- the 4 bits


def _quantise(x, kind):
    """Codes (two a byte, the even element low) and the scale word (16 bits: scale, zero in the low four) of FP32
    vectors in the last dimension."""
    hi, lo = x.amax(-1).clamp(min=0), x.amin(-1).clamp(max=0)
    # in 32 bits, correctly rounded: a code goes by which side of a border a value is on
    s = (hi - lo) / torch.full_like(hi, 15)
    s = ((s.view(torch.int32) + 0xFFFFF) & ~0xFFFFF).view(torch.float32).clamp(min=LEAST_SCALE[kind])
    k = torch.round(x / s[..., None])
    k = torch.where((k * s[..., None]).abs() > LARGEST[kind], k - k.sign(), k)
    zero = torch.round(-lo / s).clamp(0, 15)
    c = (k + zero[..., None]).clamp(0, 15).to(torch.uint8)
    word = ((s.view(torch.int32) >> 16) & 0xFFF0) | zero.to(torch.int32)
    return c[..., 0::2] | (c[..., 1::2] << 4), word


def _words(k, v):
    """The K vector's word in the low half, the V vector's in the high half."""
    return k | (v << 16)


def _values(codes, word):
    """FP32 values that codes and their 16-bit words stand for."""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float()
    scale = ((word & 0xFFF0) << 16).view(torch.float32)
    return (c - (word & 15).float()[..., None]) * scale[..., None]


def _k_word(scales):
    return scales & 0xFFFF


def _v_word(scales):
    return (scales >> 16) & 0xFFFF


# ---------------------------------------------------------------- inputs


def _lengths(case):
    """(new tokens, positions in the cache after them) of each sequence, before they are dealt."""
    n = case["seqs"]
    new = [case["chunk"] if i < case["chunks"] else case["rest"] for i in range(n)]
    step = (case["hi"] - case["lo"]) / max(1, n - 1)
    return new, [max(new[i], int(round(case["hi"] - step * i))) for i in range(n)]


def _spread(lo, hi, n):
    return [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)]


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _starts(counts):
    return _ints([0] + torch.tensor(counts).cumsum(0).tolist())


def _tables(counts, pages, width, g, fill):
    """Pages of each sequence in the order of a used pool, and that order."""
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    counts = torch.tensor(counts, device="cuda")
    first = torch.cumsum(counts, 0) - counts
    at = torch.arange(width, device="cuda")
    return torch.where(at < counts[:, None], order[(first[:, None] + at).clamp(max=pages - 1)], fill), order


def _cache(case, g):
    """Lengths, block table and 4-bit pools of the sequences of a case."""
    new, kv = _lengths(case)
    deal = torch.randperm(len(new), generator=g, device="cuda").tolist()
    new, kv = [new[i] for i in deal], [kv[i] for i in deal]
    page, nkv, dim, kind = case["page"], case["nkv"], case["dim"], case["dtype"]
    counts = [-(-n // page) for n in kv]
    pages = sum(counts) + 3
    table, _ = _tables(counts, pages, max(counts), g, 0)
    s = {"case": dict(case), "table": table.contiguous(), "q_start": _starts(new), "kv_len": _ints(kv),
         "rows": sum(new), "max_q": max(new),
         "k": torch.empty(pages, nkv, page, dim // 2, dtype=torch.uint8, device="cuda"),
         "v": torch.empty(pages, nkv, page, dim // 2, dtype=torch.uint8, device="cuda"),
         "scales": torch.empty(pages, nkv, page, dtype=torch.int32, device="cuda")}
    step = max(1, (1 << 25) // (nkv * page * dim))
    for a in range(0, pages, step):
        b = min(pages, a + step)
        words = []
        for name in ("k", "v"):
            x = torch.empty(b - a, nkv, page, dim, device="cuda").normal_(generator=g)
            s[name][a:b], w = _quantise(x, kind)
            words.append(w)
        s["scales"][a:b] = _words(*words)
    return s


def _prepare_verify(case, g):
    n, vocab = case["seqs"], case["vocab"]
    drafts = _spread(case["lo"], case["hi"], n)
    deal = torch.randperm(n, generator=g, device="cuda").tolist()
    counts = [drafts[i] + 1 for i in deal]
    rows = sum(counts)
    q_start = _starts(counts)
    seq = torch.repeat_interleave(torch.arange(n, device="cuda"), torch.tensor(counts, device="cuda"))
    temperature = 0.6 + 0.7 * torch.rand(n, generator=g, device="cuda")
    if case["greedy"]:
        temperature[::case["greedy"]] = 0.0
    warm = torch.where(temperature > 0, temperature, torch.ones_like(temperature))[seq, None]
    logits = torch.empty(rows, vocab, device="cuda").normal_(generator=g) * 2.5
    logits[:, 5::97] = -math.inf  # tokens that are not allowed
    logits = logits.to(DTYPES[case["dtype"]])
    # the draft model's opinion is near the target's; a greedy sequence's draft is mostly the target's choice
    noise = torch.empty(rows, vocab, device="cuda").normal_(generator=g) * 0.7
    q = torch.softmax((logits.float() + noise) / warm, -1)
    picked = torch.multinomial(q, 1, generator=g).squeeze(1).to(torch.int32)
    best = logits.float().argmax(-1).to(torch.int32)
    agree = torch.rand(rows, generator=g, device="cuda") < 0.7
    picked = torch.where((temperature[seq] <= 0) & agree, best, picked)
    tokens = torch.cat((torch.zeros(1, dtype=torch.int32, device="cuda"), picked[:-1]))  # row r's logits judge token r + 1
    if case["kind"] == "probs":
        logits = torch.softmax(logits.float() / warm, -1)
    return {"case": dict(case), "target": logits, "draft": q if case["draft"] else None, "tokens": tokens,
            "q_start": q_start, "seqs": n, "rows": rows, "temperature": temperature,
            "u": torch.rand(rows, generator=g, device="cuda"),
            "kv_len": torch.randint(10, 5000, (n,), generator=g, device="cuda", dtype=torch.int32) + q_start.diff(),
            "out": torch.zeros(rows, dtype=torch.int32, device="cuda"),
            "accepted": torch.zeros(n, dtype=torch.int32, device="cuda"),
            "kept": torch.zeros(n, dtype=torch.int32, device="cuda"),
            "workspace": torch.zeros(512 * rows + 128 * n + 65536, dtype=torch.uint8, device="cuda")}


def _plan_sizes(case):
    """(positions held, positions wanted, pages held, pages wanted more) of each sequence, before they are dealt."""
    n, page = case["seqs"], case["page"]
    lens, new = _spread(case["lo"], case["hi"], n), _spread(case["new_lo"], case["new_hi"], n)
    new = [new[(i * 7) % n] for i in range(n)] if n % 7 else new
    held = [-(-x // page) for x in lens]
    more = [-(-(x + w) // page) - h for x, w, h in zip(lens, new, held)]
    return lens, new, held, more


def _prepare_plan(case, g):
    lens, new, held, more = _plan_sizes(case)
    deal = torch.randperm(len(lens), generator=g, device="cuda").tolist()
    lens, new, held, more = ([x[i] for i in deal] for x in (lens, new, held, more))
    free = max(1, sum(more) * case["spare"] // 100)
    pages = sum(held) + free
    width = max(h + m for h, m in zip(held, more)) + 1
    table, order = _tables(held, pages, width, g, -1)
    ring = torch.cat((order[sum(held):], torch.zeros(sum(held), dtype=torch.int32, device="cuda")))
    n, rows = len(lens), max(1, sum(new))
    lens, new = _ints(lens), _ints(new)
    if case["then"] == "trim":  # one token is sure, some of the drafts are kept
        share = torch.rand(n, generator=g, device="cuda")
        kept = lens + torch.minimum(new, 1 + (share * new).to(torch.int32))
    else:
        kept = torch.zeros_like(lens)
    return {"case": dict(case), "table": table.to(torch.int32).contiguous(), "held": _ints(held), "free": ring,
            "state": _ints([0, free, 0, 0]), "lens": lens, "new": new, "kept": kept, "none": torch.zeros_like(new),
            "q_start": torch.zeros(n + 1, dtype=torch.int32, device="cuda"), "kv_len": torch.zeros_like(lens),
            "positions": torch.zeros(rows, dtype=torch.int32, device="cuda"),
            "slots": torch.zeros(rows, dtype=torch.int32, device="cuda"),
            "q_start_then": torch.zeros(n + 1, dtype=torch.int32, device="cuda"), "kv_len_then": torch.zeros_like(lens)}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    if case["op"] == "verify":
        return _prepare_verify(case, g)
    if case["op"] == "plan":
        return _prepare_plan(case, g)
    dtype = DTYPES[case["dtype"]]
    s = _cache(case, g)
    nq, nkv, dim = case["nq"], case["nkv"], case["dim"]
    if case["op"] == "attention":
        s["q"] = torch.empty(s["rows"], nq, dim, device="cuda", dtype=dtype).normal_(generator=g) * 2
        s["out"] = torch.zeros(s["rows"], nq, dim, device="cuda", dtype=dtype)
        s["lse"] = torch.zeros(s["rows"], nq, device="cuda")
        s["workspace"] = torch.zeros(WORKSPACE_BYTES, dtype=torch.uint8, device="cuda")
        return s
    # the rows of one projection: q | k | v
    qkv = torch.empty(s["rows"], nq + 2 * nkv, dim, device="cuda", dtype=DTYPES[case["source"]]).normal_(generator=g)
    s["q"], s["k_new"], s["v_new"] = qkv[:, :nq], qkv[:, nq:nq + nkv], qkv[:, nq + nkv:]
    s["q_out"] = torch.zeros(s["rows"], nq, dim, device="cuda", dtype=dtype)
    # where the pages' values go: pools of 16 bits with pages of the same numbers
    s["all"] = torch.arange(s["k"].shape[0], dtype=torch.int32, device="cuda")
    for name in ("k16", "v16"):
        s[name] = torch.zeros(*s["k"].shape[:3], dim, device="cuda", dtype=dtype)
    return s


# ---------------------------------------------------------------- plain forms


def _rows(s):
    """Sequence, token within it and position of every new token."""
    r = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(s["q_start"].long(), r, right=True) - 1
    token = r - s["q_start"][seq]
    new = s["q_start"][1:] - s["q_start"][:-1]
    return seq, token, (s["kv_len"] - new)[seq] + token


def _visible(pos, keys, case):
    seen = keys <= pos
    if case["window"]:
        seen = seen & ((keys > pos - case["window"]) | (keys < case["sinks"]))
    return seen


def _plain_attention(s):
    case = s["case"]
    n, group = case["seqs"], case["nq"] // case["nkv"]
    nkv, dim, most = case["nkv"], case["dim"], s["max_q"]

    def gather(pool, word):  # [sequence][KV head][position][dim]
        return _values(pool[s["table"]], word[s["table"]]).transpose(1, 2).reshape(n, nkv, -1, dim)

    k, v = gather(s["k"], _k_word(s["scales"])), gather(s["v"], _v_word(s["scales"]))
    seq, token, _ = _rows(s)
    at = (s["q_start"][:-1, None] + torch.arange(most, device="cuda")).clamp(max=s["rows"] - 1)
    q = s["q"][at].float().view(n, most, nkv, group, dim).permute(0, 2, 3, 1, 4).reshape(n, nkv, group * most, dim)
    new = s["q_start"][1:] - s["q_start"][:-1]
    pos = (s["kv_len"] - new)[:, None] + torch.arange(most, device="cuda")
    keys = torch.arange(k.shape[2], device="cuda")
    seen = _visible(pos[:, :, None], keys, case)[:, None, None] & (keys < s["kv_len"][:, None, None, None, None])
    scores = torch.matmul(q, k.transpose(2, 3)).view(n, nkv, group, most, -1).mul_(1.0 / math.sqrt(dim))
    scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(n, nkv, group * most, -1), v).view(n, nkv, group, most, dim)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    lse = (top + total.log()).squeeze(-1)
    s["out"].copy_(o.permute(0, 3, 1, 2, 4)[seq, token].reshape(s["rows"], -1, dim))
    s["lse"].copy_(lse.permute(0, 3, 1, 2)[seq, token].reshape(s["rows"], -1))
    return {"out": s["out"], "lse": s["lse"]}


def _frequencies(case):
    """Radians a position of every rotated pair, in 64 bits, and what cosine and sine are multiplied by."""
    c, r = ROPE[case["scaling"]], case["rotary"]
    i = torch.arange(r // 2, device="cuda", dtype=torch.float64)
    f = c["theta"] ** (-2.0 * i / r)
    if c["scaling"] == "llama3":
        turns = c["original"] * f / (2 * math.pi)
        keep = ((turns - c["low"]) / (c["high"] - c["low"])).clamp(0, 1)
        f = f * (keep + (1 - keep) / c["factor"])
    if c["scaling"] == "yarn":
        def border(turns):
            return r * math.log(c["original"] / (turns * 2 * math.pi)) / (2 * math.log(c["theta"]))

        lo = max(0, math.floor(border(c["high"])))
        hi = min(r - 1, math.ceil(border(c["low"])))
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        f = f * (1 - ramp + ramp / c["factor"])
    return f, 0.1 * math.log(c["factor"]) + 1 if c["scaling"] == "yarn" else 1.0


def _plain_append(s):
    case = s["case"]
    seq, _, pos = _rows(s)
    f, much = _frequencies(case)
    angle = pos.double()[:, None] * f
    cos, sin = (angle.cos() * much)[:, None], (angle.sin() * much)[:, None]
    r = case["rotary"]

    def turned(x):  # in 64 bits: k's values lie next to the borders of their codes
        x = x.double()
        a, b = (x[..., 0:r:2], x[..., 1:r:2]) if case["interleaved"] else (x[..., :r // 2], x[..., r // 2:r])
        u, w = a * cos - b * sin, b * cos + a * sin
        front = torch.stack((u, w), -1).flatten(-2) if case["interleaved"] else torch.cat((u, w), -1)
        return torch.cat((front, x[..., r:]), -1).float()

    s["q_out"].copy_(turned(s["q"]))
    page, row = s["table"][seq, pos // case["page"]].long(), pos % case["page"]
    s["k"][page, :, row], k_word = _quantise(turned(s["k_new"]), case["dtype"])
    s["v"][page, :, row], v_word = _quantise(s["v_new"].float(), case["dtype"])
    s["scales"][page, :, row] = _words(k_word, v_word)
    s["k16"].copy_(_values(s["k"], _k_word(s["scales"])))
    s["v16"].copy_(_values(s["v"], _v_word(s["scales"])))
    return {"q": s["q_out"], "k": s["k16"], "v": s["v16"]}


def _plain_verify(s):
    n, rows, vocab = s["seqs"], s["rows"], s["case"]["vocab"]
    r = torch.arange(rows, device="cuda")
    start = s["q_start"].long()
    seq = torch.searchsorted(start, r, right=True) - 1
    last = start[1:] - 1
    greedy = s["temperature"] <= 0
    x = s["target"].double()
    ids = torch.arange(vocab, device="cuda")
    best = torch.where(x == x.amax(-1, keepdim=True), ids, vocab).amin(-1)  # the lowest of equal ones
    if s["case"]["kind"] == "probs":
        p = x
    else:
        x = x / torch.where(greedy, 1.0, s["temperature"].double())[seq, None]
        p = (x - x.amax(-1, keepdim=True)).exp()
        p = p / p.sum(-1, keepdim=True)
    drafted = torch.cat((s["tokens"][1:], s["tokens"][:1])).long()
    drafted = torch.where(r == last[seq], 0, drafted)
    at = p.gather(1, drafted[:, None]).squeeze(1)
    q = 1.0 if s["draft"] is None else s["draft"].gather(1, drafted[:, None]).squeeze(1).double()
    good = torch.where(greedy[seq], drafted == best, s["u"].double() * q < at) & (r != last[seq])
    stop = torch.full((n,), rows, device="cuda").scatter_reduce(0, seq, torch.where(good, rows, r), "amin")
    rest = p[stop]
    if s["draft"] is None:
        minus = torch.zeros_like(rest).scatter_(1, drafted[stop][:, None], 2.0)
    else:
        minus = s["draft"][stop].double()
    left = (rest - torch.where((stop == last)[:, None], 0.0, minus)).clamp(min=0)
    left = torch.where(left.sum(-1, keepdim=True) > 0, left, rest)
    upto = left.cumsum(-1)
    drawn = (upto <= s["u"][last].double()[:, None] * upto[:, -1:]).sum(-1)
    drawn = torch.minimum(drawn, torch.where(left > 0, ids, 0).amax(-1))
    drawn = torch.where(greedy, best[stop], drawn).to(torch.int32)
    accepted = (stop - start[:-1]).to(torch.int32)
    i = (r - start[seq]).to(torch.int32)
    s["accepted"].copy_(accepted)
    s["out"].copy_(torch.where(i < accepted[seq], drafted.to(torch.int32),
                               torch.where(i == accepted[seq], drawn[seq], -1)))
    s["kept"].copy_(s["kv_len"] - (last - stop).to(torch.int32))
    return {"out": s["out"], "accepted": s["accepted"], "kept": s["kept"]}


def _plain_tables(s, lens, new, q_start, kv_len, positions, slots):
    page, table, held, ring = s["case"]["page"], s["table"], s["held"].long(), s["free"]
    width, pages = table.shape[1], ring.numel()
    head, count = s["state"][0].long(), s["state"][1].long()
    lens, new = lens.long(), new.long()
    need = (lens + new + page - 1) // page
    more = (need - held).clamp(min=0)
    granted = ((more == 0) | (more.cumsum(0) <= count))
    if positions is not None:
        granted &= (new == 0) | (new.cumsum(0) <= positions.numel())
    new = torch.where(granted, new, 0)
    need = torch.where(granted, need, held)
    more, less = (need - held).clamp(min=0), (held - need).clamp(min=0)
    at = torch.arange(width, device="cuda")
    taking = (at >= held[:, None]) & (at < need[:, None])
    giving = (at >= need[:, None]) & (at < held[:, None])
    from_ = (head + (more.cumsum(0) - more - held)[:, None] + at) % pages
    to = (head + count + (less.cumsum(0) - less - need)[:, None] + at) % pages
    taken = ring[from_]
    wider = torch.cat((ring, ring[:1]))  # a place behind the ring for what is not given back
    wider.scatter_(0, torch.where(giving, to, pages).flatten(), table.flatten())
    ring.copy_(wider[:pages])
    table.copy_(torch.where(taking, taken, torch.where(giving, -1, table)))
    s["state"][0] = ((head + more.sum()) % pages).to(torch.int32)
    s["state"][1] = (count - more.sum() + less.sum()).to(torch.int32)
    s["held"].copy_(need)
    q_start[1:] = new.cumsum(0)
    kv_len.copy_(lens + new)
    if positions is not None:
        r = torch.arange(positions.numel(), device="cuda")
        seq = (torch.searchsorted(q_start.long(), r, right=True) - 1).clamp(max=lens.numel() - 1)
        there = r < q_start[-1]
        pos = torch.where(there, lens[seq] + r - q_start[seq], 0)
        slot = table[seq, pos // page] * page + pos % page
        positions.copy_(torch.where(there, pos, positions))
        slots.copy_(torch.where(there, slot, slots))


def _plain_plan(s):
    _plain_tables(s, s["lens"], s["new"], s["q_start"], s["kv_len"], s["positions"], s["slots"])
    _plain_tables(s, s["kept"], s["none"], s["q_start_then"], s["kv_len_then"], None, None)
    return _plan_outputs(s)


def _plan_outputs(s):
    return {x: s[x] for x in ("table", "held", "free", "state", "q_start", "kv_len", "positions", "slots",
                              "q_start_then", "kv_len_then")}


# ---------------------------------------------------------------- the framework's calls


def _own(s):
    import infernt_b200 as ib

    case = s["case"]
    if case["op"] == "plan":
        tables = ib.PageTables(s["table"], s["held"], s["free"], s["state"], case["page"])
        ib.plan_batch(tables, s["lens"], s["new"], s["q_start"], s["kv_len"], s["positions"], s["slots"])
        ib.plan_batch(tables, s["kept"], s["none"], s["q_start_then"], s["kv_len_then"])
        return _plan_outputs(s)
    if case["op"] == "verify":
        ib.verify_drafts(s["out"], s["accepted"], s["target"], s["tokens"], s["q_start"], s["u"], s["workspace"],
                         draft_probs=s["draft"], temperature=s["temperature"],
                         probabilities=case["kind"] == "probs", kv_len=s["kv_len"], kept=s["kept"])
        return {"out": s["out"], "accepted": s["accepted"], "kept": s["kept"]}
    cache = ib.PagedCache4(s["k"], s["v"], s["scales"], DTYPES[case["dtype"]])
    batch = ib.RaggedBatch(s["q_start"], s["kv_len"], s["table"], s["rows"], s["max_q"])
    if case["op"] == "attention":
        ib.paged4_attention(s["out"], s["q"], cache, batch, s["workspace"], window=case["window"],
                            sinks=case["sinks"], lse=s["lse"])
        return {"out": s["out"], "lse": s["lse"]}
    c = ROPE[case["scaling"]]
    params = ib.RopeParams(theta=c["theta"], rotary_dim=case["rotary"], interleaved=case["interleaved"],
                           scaling=c["scaling"], factor=c["factor"], low=c["low"], high=c["high"],
                           original_max_len=c["original"])
    ib.paged4_rope_append(s["q_out"], s["q"], s["k_new"], s["v_new"], cache, batch, params)
    ib.paged4_unpack(cache, ib.PagedCache(s["k16"], s["v16"]), s["all"], s["all"])
    return {"q": s["q_out"], "k": s["k16"], "v": s["v16"]}


def run(state):
    if own:
        return _own(state)
    return {"attention": _plain_attention, "append": _plain_append, "verify": _plain_verify,
            "plan": _plain_plan}[state["case"]["op"]](state)


# ---------------------------------------------------------------- work and exact values


def _seen_count(pos, window, sinks):
    """Keys that a token at `pos` sees."""
    if not window or pos + 1 <= window:
        return pos + 1
    return window + min(sinks, pos + 1 - window)


def work(case):
    if case["op"] == "plan":
        lens, new, held, more = _plan_sizes(case)
        moved = sum(more)  # pages: out of the ring into the table, and, when given back, the other way
        return {"bytes": 4 * (10 * len(lens) + 2 * sum(new) + 4 * moved), "flops": 0}
    if case["op"] == "verify":
        rows = sum(x + 1 for x in _spread(case["lo"], case["hi"], case["seqs"]))
        size = 4 if case["dtype"] == "fp32" else 2
        draft = case["seqs"] * case["vocab"] * 4 if case["draft"] else 0  # the row of one stop a sequence
        if case["kind"] == "probs":  # only what is drafted, and the rows where sequences stop
            return {"bytes": case["seqs"] * case["vocab"] * size + draft + 40 * rows,
                    "flops": 2 * case["seqs"] * case["vocab"]}
        return {"bytes": rows * case["vocab"] * size + draft + 40 * rows, "flops": 4 * rows * case["vocab"]}
    new, kv = _lengths(case)
    rows, dim = sum(new), case["dim"]
    if case["op"] == "append":
        pool = (sum(-(-n // case["page"]) for n in kv) + 3) * case["page"] * case["nkv"]
        values = rows * (case["nq"] + 2 * case["nkv"]) * dim * (4 if case["source"] == "fp32" else 2)
        return {"bytes": values + rows * (case["nq"] * dim * 2 + case["nkv"] * (dim + 4)) + pool * (dim + 4 + 4 * dim),
                "flops": 3 * rows * (case["nq"] + case["nkv"]) * case["rotary"]}
    w, k = case["window"], case["sinks"]
    keys = seen = 0
    for n, t in zip(new, kv):
        # keys that any of the new tokens sees, and the sum over the tokens
        lo = max(0, t - n - w + 1) if w else 0
        keys += t - lo + (min(k, lo) if w else 0)
        seen += sum(_seen_count(p, w, k) for p in range(t - n, t))
    return {"bytes": keys * case["nkv"] * (dim + 4) + rows * case["nq"] * (dim * 4 + 4),
            "flops": 4 * dim * case["nq"] * seen}


def _exact_values(codes, word):
    """The same numbers in 64 bits, by another way: a table of the sixteen products."""
    word = word.long()
    scale = torch.ldexp((8 + ((word >> 4) & 7)).double(), ((word >> 7) & 255) - 130)
    c = torch.empty(*codes.shape[:-1], 2 * codes.shape[-1], dtype=torch.long, device=codes.device)
    c[..., 0::2], c[..., 1::2] = codes.long() % 16, codes.long() // 16
    sixteen = torch.arange(16, device=codes.device) - (word % 16)[..., None]
    return torch.gather(sixteen * scale[..., None], -1, c)


def _exact_attention(s):
    case = s["case"]
    group, dim = case["nq"] // case["nkv"], case["dim"]
    starts, lens = s["q_start"].tolist(), s["kv_len"].tolist()
    out = torch.zeros(s["rows"], case["nq"], dim, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["rows"], case["nq"], dtype=torch.float64, device="cuda")
    for i, length in enumerate(lens):
        a, b = starts[i], starts[i + 1]
        pages = s["table"][i, :-(-length // case["page"])].long()
        pos = torch.arange(length - (b - a), length, device="cuda")[:, None]
        key = torch.arange(length, device="cuda")[None]
        hidden = key > pos
        if case["window"]:
            hidden |= (pos - key >= case["window"]) & (key >= case["sinks"])
        for h in range(case["nkv"]):
            word = s["scales"][pages, h].reshape(-1)[:length]
            k = _exact_values(s["k"][pages, h].reshape(-1, dim // 2)[:length], word & 0xFFFF)
            v = _exact_values(s["v"][pages, h].reshape(-1, dim // 2)[:length], (word >> 16) & 0xFFFF)
            for j in range(h * group, (h + 1) * group):
                w = (s["q"][a:b, j].double() @ k.T) / math.sqrt(dim)
                w[hidden] = -math.inf
                out[a:b, j] = torch.softmax(w, 1) @ v
                lse[a:b, j] = torch.logsumexp(w, 1)
    return {"out": out, "lse": lse}


def _exact_append(s):
    case, c = s["case"], ROPE[s["case"]["scaling"]]
    r, half = case["rotary"], case["rotary"] // 2
    freq, much = [], 1.0
    for i in range(half):
        f = math.exp(-2 * i / r * math.log(c["theta"]))
        if c["scaling"] == "llama3":
            wave = 2 * math.pi / f
            if wave > c["original"] / c["low"]:
                f /= c["factor"]
            elif wave >= c["original"] / c["high"]:
                mix = (c["original"] / wave - c["low"]) / (c["high"] - c["low"])
                f = (1 - mix) * f / c["factor"] + mix * f
        elif c["scaling"] == "yarn":
            dims = [r * math.log(c["original"] / (b * 2 * math.pi)) / (2 * math.log(c["theta"])) for b in (c["high"], c["low"])]
            lo, hi = max(0, math.floor(dims[0])), min(r - 1, math.ceil(dims[1]))
            mix = min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001)))
            f = f / c["factor"] * mix + f * (1 - mix)
            much = 1 + 0.1 * math.log(c["factor"])
        freq.append(f)
    first = [2 * i if case["interleaved"] else i for i in range(half)]
    second = [2 * i + 1 if case["interleaved"] else half + i for i in range(half)]
    freq = torch.tensor(freq, dtype=torch.float64, device="cuda")
    q, k, v = s["q"].double(), s["k_new"].double(), s["v_new"].double()
    turned_q, turned_k = q.clone(), k.clone()
    word = s["scales"]
    out = {"k": _exact_values(s["k"], word & 0xFFFF), "v": _exact_values(s["v"], (word >> 16) & 0xFFFF)}

    def stored(x):
        """x as it is held: whole steps of the range of x and 0 over 15, rounded up to four significant bits."""
        lo, hi = torch.clamp(x.min(-1).values, max=0), torch.clamp(x.max(-1).values, min=0)
        mantissa, exponent = torch.frexp((hi - lo) / 15)
        step = torch.ldexp(torch.ceil(mantissa * 16) / 16, exponent)[..., None]
        zero = torch.round(-lo[..., None] / step)
        return (torch.clamp(torch.round(x / step) + zero, 0, 15) - zero) * step

    starts, lens = s["q_start"].tolist(), s["kv_len"].tolist()
    for i, length in enumerate(lens):
        a, b = starts[i], starts[i + 1]
        pos = torch.arange(length - (b - a), length, device="cuda")
        turn = torch.polar(torch.full((b - a, half), much, dtype=torch.float64, device="cuda"), pos[:, None] * freq)[:, None]
        for x, y in ((q, turned_q), (k, turned_k)):
            z = torch.complex(x[a:b][..., first], x[a:b][..., second]) * turn
            y[a:b, :, first], y[a:b, :, second] = z.real, z.imag
        page = s["table"][i].long()[pos // case["page"]]
        out["k"][page, :, pos % case["page"]] = stored(turned_k[a:b])
        out["v"][page, :, pos % case["page"]] = stored(v[a:b])
    out["q"] = turned_q
    return out


def exact(case, seed):
    if case["op"] in ("verify", "plan"):  # whole numbers
        return None
    s = prepare(case, seed)
    return _exact_attention(s) if case["op"] == "attention" else _exact_append(s)
