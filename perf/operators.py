"""Cases of the operators over paged KV caches, with their plain forms.

Four operators: rotary positions with the append of K and V rows into pages;
attention of a ragged batch of new tokens over a paged cache; the same with a
sliding window and sinks; copies of pages in every pool of a model.  A case
names its operator and its sizes; sequence lengths are spread evenly between
the case's bounds and dealt to the sequences by the seed.
"""
import math

import torch

own = False

# The attention's workspace: a fixed size, zeroed once by its owner.
WORKSPACE_BYTES = 64 << 20

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}

ROPE = {
    # plain: the 1.1B shape's; llama3: the 8B shape's theta with the scaling of its long-context successor;
    # linear and yarn: the two other scalings in common use
    "plain": dict(theta=10000.0, scaling="none", factor=1.0, low=1.0, high=4.0, original=2048),
    "llama3": dict(theta=500000.0, scaling="llama3", factor=8.0, low=1.0, high=4.0, original=8192),
    "linear": dict(theta=10000.0, scaling="linear", factor=4.0, low=1.0, high=4.0, original=2048),
    "yarn": dict(theta=10000.0, scaling="yarn", factor=16.0, low=1.0, high=32.0, original=4096),
}


def attention(name, seqs, chunks, chunk, lo, hi, nq, nkv, dim, page, window=0, sinks=0, dtype="bf16"):
    """`chunks` of the `seqs` sequences bring `chunk` new tokens each, the others one; lengths lo..hi."""
    return dict(name=name, op="attention", seqs=seqs, chunks=chunks, chunk=chunk, lo=lo, hi=hi, nq=nq, nkv=nkv,
                dim=dim, page=page, window=window, sinks=sinks, dtype=dtype)


def rope(name, seqs, chunk, lo, hi, nq, nkv, dim, page, rotary, interleaved, scaling, source, dtype):
    return dict(name=name, op="rope", seqs=seqs, chunks=seqs, chunk=chunk, lo=lo, hi=hi, nq=nq, nkv=nkv, dim=dim,
                page=page, rotary=rotary, interleaved=interleaved, scaling=scaling, source=source, dtype=dtype)


def copy(name, layers, pages, moves, nkv, dim, page, dtype="bf16"):
    return dict(name=name, op="copy", layers=layers, pages=pages, moves=moves, nkv=nkv, dim=dim, page=page, dtype=dtype)


def listed():
    return [
        # the first tokens of one chat on the 1.1B shape: latency
        attention("decode_one", 1, 0, 1, 37, 37, 32, 4, 64, 16),
        # 64 sequences of the 1.1B shape at the batched benchmark's contexts
        attention("decode_ragged", 64, 0, 1, 512, 2048, 32, 4, 64, 32),
        # 16 long documents on the 8B shape: the whole cache is read once
        attention("decode_long", 16, 0, 1, 32768, 32768, 32, 8, 128, 32),
        # one chunk of a long prompt on the 8B shape: the tensor cores' work
        attention("chunk_long", 1, 1, 4096, 12288, 12288, 32, 8, 128, 32),
        # a step of continuous batching: odd lengths, one prompt's chunk among decodes, fp16
        attention("mixed_step", 16, 1, 509, 700, 4001, 32, 8, 128, 16, dtype="fp16"),
        # chats far past their window, whose first tokens stay visible
        attention("window_decode", 32, 0, 1, 9000, 20011, 32, 8, 128, 64, window=4096, sinks=4),
        # two prompts with a short window on the 1.1B shape's heads
        attention("window_chunk", 2, 2, 2039, 2039, 8111, 32, 4, 64, 64, window=1000, sinks=5),
        # the step of 64 decoding sequences on the 8B shape, FP32 projection rows
        rope("rope_step", 64, 1, 512, 8192, 32, 8, 128, 32, 128, False, "llama3", "fp32", "bf16"),
        # a long prompt's chunk on the 8B shape
        rope("rope_chunk", 1, 8192, 32768, 32768, 32, 8, 128, 32, 128, False, "llama3", "bf16", "bf16"),
        # far positions, interleaved pairs on half of the head, odd counts, fp16
        rope("rope_far", 3, 501, 90001, 131072, 16, 4, 64, 16, 32, True, "yarn", "fp16", "fp16"),
        # a fork's one partly filled page in every layer of the 8B shape
        copy("copy_fork", 32, 256, 1, 8, 128, 32),
        # compaction of a pool of the 1.1B shape
        copy("copy_compact", 22, 1024, 301, 4, 64, 32),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "rope", "copy"])
    nkv = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 8])
    dim = rng.choice([64, 128])
    page = rng.choice([8, 16, 24, 32, 64, 100, 128, 256])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "attention":
        chunk = rng.choice([1, 1, _log(rng, 2, 16), _log(rng, 16, 3000)])
        hi = max(chunk, _log(rng, 16, 32768))
        if chunk > 16:  # the plain form's scores: seqs x chunk x heads x hi floats
            hi = max(chunk, min(hi, 8192))
            seqs = max(1, min(_log(rng, 1, 16), int(1.2e9 / (chunk * nkv * group * hi))))
            if seqs == 1:
                hi = max(chunk, min(hi, int(1.2e9 / (chunk * nkv * group))))
        else:
            seqs = max(1, min(_log(rng, 1, 96), int(4.0e8 / (hi * nkv * dim))))
        chunks = 0 if chunk == 1 else rng.randint(1, seqs)
        window = rng.choice([0, 0, _log(rng, 1, max(2, hi))])
        sinks = rng.choice([0, 1, 4, 64, 200]) if window else 0
        c = attention("", seqs, chunks, chunk, max(1, chunk, hi // rng.randint(1, 8)), hi, nkv * group, nkv, dim, page,
                      window, sinks, dtype)
    elif op == "rope":
        chunk = _log(rng, 1, 4000)
        hi = max(chunk, _log(rng, 16, 131072))
        seqs = max(1, min(_log(rng, 1, 64), 8000 // chunk, 3000000 // hi))
        rotary = rng.choice([dim, dim // 2, dim // 4, dim - 2])
        c = rope("", seqs, chunk, max(chunk, hi // 3), hi, nkv * group, nkv, dim, page, rotary, rng.random() < 0.5,
                 rng.choice(sorted(ROPE)), rng.choice(["fp32", dtype]), dtype)
    else:
        pages, layers, page = _log(rng, 4, 600), rng.randint(1, 32), rng.choice([8, 16, 24, 32, 64])
        most = max(1, int(1.0e9 / (8 * layers * nkv * page * dim)))  # a gigabyte read and written
        c = copy("", layers, pages, min(most, rng.randint(1, pages // 2)), nkv, dim, page, dtype)
    del c["name"]
    return c


# ---------------------------------------------------------------- inputs


def _lengths(case):
    """(new tokens, positions in the cache after them) of each sequence, before they are dealt."""
    n = case["seqs"]
    new = [case["chunk"] if i < case["chunks"] else 1 for i in range(n)]
    step = (case["hi"] - case["lo"]) / max(1, n - 1)
    return new, [max(new[i], int(round(case["hi"] - step * i))) for i in range(n)]


def _cache(case, g, dtype):
    """Lengths, block table and pools of the sequences of a case; pages in the order of a used pool."""
    new, kv = _lengths(case)
    deal = torch.randperm(len(new), generator=g, device="cuda").tolist()
    new, kv = [new[i] for i in deal], [kv[i] for i in deal]
    page = case["page"]
    width = max(-(-n // page) for n in kv)
    counts = torch.tensor([-(-n // page) for n in kv], device="cuda")
    total = sum(-(-n // page) for n in kv)
    pages = total + 3
    order = torch.randperm(pages, generator=g, device="cuda")[:total].to(torch.int32)
    first = torch.cumsum(counts, 0) - counts
    at = torch.arange(width, device="cuda")
    table = torch.where(at < counts[:, None], order[(first[:, None] + at).clamp(max=total - 1)], 0).to(torch.int32)
    shape = (pages, case["nkv"], page, case["dim"])
    s = {
        "k": torch.empty(shape, device="cuda", dtype=dtype).normal_(generator=g),
        "v": torch.empty(shape, device="cuda", dtype=dtype).normal_(generator=g),
        "table": table.contiguous(),
        "q_start": torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32, device="cuda"),
        "kv_len": torch.tensor(kv, dtype=torch.int32, device="cuda"),
        "rows": sum(new), "max_q": max(new), "case": dict(case),
    }
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "copy":
        shape = (2 * case["layers"], case["pages"], case["nkv"], case["page"], case["dim"])
        order = torch.randperm(case["pages"], generator=g, device="cuda").tolist()
        n = case["moves"]
        return {"case": dict(case), "pools": torch.empty(shape, device="cuda", dtype=dtype).normal_(generator=g),
                "src": order[:n], "dst": order[n:2 * n]}
    s = _cache(case, g, dtype)
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
    return s


# ---------------------------------------------------------------- plain forms


def _rows(s):
    """Sequence, token within it and position of every new token."""
    r = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(s["q_start"], r, right=True) - 1
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

    def gather(pool):  # [sequence][KV head][position][dim]
        return pool[s["table"]].transpose(1, 2).reshape(n, nkv, -1, dim).float()

    k, v = gather(s["k"]), gather(s["v"])
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
    if c["scaling"] == "linear":
        f = f / c["factor"]
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


def _plain_rope(s):
    case = s["case"]
    seq, _, pos = _rows(s)
    f, much = _frequencies(case)
    angle = pos.double()[:, None] * f
    cos, sin = (angle.cos() * much).float()[:, None], (angle.sin() * much).float()[:, None]
    r = case["rotary"]

    def turned(x):
        x = x.float()
        a, b = (x[..., 0:r:2], x[..., 1:r:2]) if case["interleaved"] else (x[..., :r // 2], x[..., r // 2:r])
        u, w = a * cos - b * sin, b * cos + a * sin
        front = torch.stack((u, w), -1).flatten(-2) if case["interleaved"] else torch.cat((u, w), -1)
        return torch.cat((front, x[..., r:]), -1)

    s["q_out"].copy_(turned(s["q"]))
    page = s["table"][seq, pos // case["page"]].long()
    s["k"][page, :, pos % case["page"]] = turned(s["k_new"]).to(s["k"].dtype)
    s["v"][page, :, pos % case["page"]] = s["v_new"].to(s["v"].dtype)
    return {"q": s["q_out"], "k": s["k"], "v": s["v"]}


def _plain_copy(s):
    s["pools"][:, s["dst"]] = s["pools"][:, s["src"]]
    return {"pools": s["pools"]}


# ---------------------------------------------------------------- the framework's calls


def _own(s):
    import infernt_b200 as ib

    case = s["case"]
    if case["op"] == "copy":
        ib.copy_pages(s["pools"], s["src"], s["dst"])
        return {"pools": s["pools"]}
    cache = ib.PagedCache(s["k"], s["v"])
    batch = ib.RaggedBatch(s["q_start"], s["kv_len"], s["table"], s["rows"], s["max_q"])
    if case["op"] == "attention":
        ib.paged_attention(s["out"], s["q"], cache, batch, s["workspace"], window=case["window"], sinks=case["sinks"],
                           lse=s["lse"])
        return {"out": s["out"], "lse": s["lse"]}
    c = ROPE[case["scaling"]]
    params = ib.RopeParams(theta=c["theta"], rotary_dim=case["rotary"], interleaved=case["interleaved"],
                           scaling=c["scaling"], factor=c["factor"], low=c["low"], high=c["high"],
                           original_max_len=c["original"])
    ib.paged_rope_append(s["q_out"], s["q"], s["k_new"], s["v_new"], cache, batch, params)
    return {"q": s["q_out"], "k": s["k"], "v": s["v"]}


def run(state):
    if own:
        return _own(state)
    return {"attention": _plain_attention, "rope": _plain_rope, "copy": _plain_copy}[state["case"]["op"]](state)


# ---------------------------------------------------------------- work and exact values


def _seen_count(pos, window, sinks):
    """Keys that a token at `pos` sees."""
    if not window or pos + 1 <= window:
        return pos + 1
    return window + min(sinks, pos + 1 - window)


def work(case):
    if case["op"] == "copy":
        page = case["nkv"] * case["page"] * case["dim"] * 2
        return {"bytes": 2 * 2 * case["layers"] * case["moves"] * page, "flops": 0}
    new, kv = _lengths(case)
    rows, dim = sum(new), case["dim"]
    if case["op"] == "rope":
        values = rows * (case["nq"] + 2 * case["nkv"]) * dim
        return {"bytes": values * ((4 if case["source"] == "fp32" else 2) + 2),
                "flops": 3 * rows * (case["nq"] + case["nkv"]) * case["rotary"]}
    w, k = case["window"], case["sinks"]
    keys = seen = 0
    for n, t in zip(new, kv):
        # keys that any of the new tokens sees, and the sum over the tokens
        lo = max(0, t - n - w + 1) if w else 0
        keys += t - lo + (min(k, lo) if w else 0)
        seen += sum(_seen_count(p, w, k) for p in range(t - n, t))
    return {"bytes": keys * case["nkv"] * dim * 2 * 2 + rows * case["nq"] * (dim * 4 + 4),
            "flops": 4 * dim * case["nq"] * seen}


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
            k = s["k"][pages, h].reshape(-1, dim)[:length].double()
            v = s["v"][pages, h].reshape(-1, dim)[:length].double()
            for j in range(h * group, (h + 1) * group):
                w = (s["q"][a:b, j].double() @ k.T) / math.sqrt(dim)
                w[hidden] = -math.inf
                out[a:b, j] = torch.softmax(w, 1) @ v
                lse[a:b, j] = torch.logsumexp(w, 1)
    return {"out": out, "lse": lse}


def _exact_rope(s):
    case, c = s["case"], ROPE[s["case"]["scaling"]]
    r, half = case["rotary"], case["rotary"] // 2
    freq, much = [], 1.0
    for i in range(half):
        f = math.exp(-2 * i / r * math.log(c["theta"]))
        if c["scaling"] == "linear":
            f /= c["factor"]
        elif c["scaling"] == "llama3":
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
    out = {"q": q.clone(), "k": s["k"].double(), "v": s["v"].double()}
    starts, lens = s["q_start"].tolist(), s["kv_len"].tolist()
    k2 = k.clone()
    for i, length in enumerate(lens):
        a, b = starts[i], starts[i + 1]
        pos = torch.arange(length - (b - a), length, device="cuda")
        turn = torch.polar(torch.full((b - a, half), much, dtype=torch.float64, device="cuda"), pos[:, None] * freq)[:, None]
        for x, y in ((q, out["q"]), (k, k2)):
            z = torch.complex(x[a:b][..., first], x[a:b][..., second]) * turn
            y[a:b, :, first], y[a:b, :, second] = z.real, z.imag
        page = s["table"][i].long()[pos // case["page"]]
        out["k"][page, :, pos % case["page"]] = k2[a:b]
        out["v"][page, :, pos % case["page"]] = v[a:b]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "copy":
        for a, b in zip(s["src"], s["dst"]):
            s["pools"][:, b].copy_(s["pools"][:, a])
        return {"pools": s["pools"]}
    return _exact_attention(s) if case["op"] == "attention" else _exact_rope(s)
