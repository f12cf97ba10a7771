"""The operators of a speculative serving pass over a paged cache, case by case, in plain form and as the runtime's calls.

  attn    causal GQA attention of every sequence's rows over its pages of a cache held in 4 bits
  append  new K/V rows into the pages of that cache; what comes back is the rows as the cache holds them
  fork    branches of one sequence that share its pages, each with the last, partly filled page as its own
  compact pages of ended sequences given back, the others' pages moved to the lowest ids, sequences copied
  verify  drafted tokens accepted or refused against the target's logits from given random numbers, one more token sampled

The cache in 4 bits: groups of 32 values of a (token, kv head) have a scale d (an f16 of at most 7 significant bits) and a zero
point z in 0 .. 15, and a code c in 0 .. 15 stands for d (c - z). d is the smallest such f16 with 15 d >= max(x, 0) - min(x, 0),
z = rint(-min(x, 0) / d), c = rint(x / d) + z cut to 0 .. 15. A group's header is the 16 bits of d with z in the low four.
A page of one kv head, P positions of hd dims, is its code words (u32, element 2 i of eight at bits 4 i, element 2 i + 1 at bits
16 + 4 i) and then its headers:
  K  words [P][4][hd / 32], word (g, u) being dims 32 u + 8 g .. + 7; headers [P][hd / 32]
  V  words [P / 8][hd], a word being eight positions of one dim; headers [P / 8][hd / 32][8]; dim d's word stands at
     ((d // 16 w) * 16 + d % 16) * w + d // 16 % w, w = 4 where hd is a multiple of 64, else 2
"""
import math

import numpy as np
import torch

own = False

PAGE = 64
VOCAB = 248320


def listed():
    qwen = dict(heads=24, kv_heads=4, hd=256, page=PAGE)
    return [
        # a lone request's decode step early in its context: latency
        dict(qwen, name="attn 1 sequence, 500", op="attn", seqs=1, rows=1, ctx=500),
        # continuous batching: a decode step of sequences of mixed length
        dict(qwen, name="attn 16 sequences, 8192", op="attn", seqs=16, rows=1, ctx=8192),
        # one long document
        dict(qwen, name="attn 1 sequence, 131071", op="attn", seqs=1, rows=1, ctx=131071),
        # the verify pass of three drafted tokens of eight sequences, 128-dim heads
        dict(name="attn 8 verified by 4", op="attn", heads=32, kv_heads=8, hd=128, page=16, seqs=8, rows=4, ctx=4100),
        # the last chunk of a prompt
        dict(qwen, name="attn prompt 512 of 2048", op="attn", seqs=1, rows=512, ctx=2048),
        # what a decode step writes
        dict(qwen, name="append 16 sequences", op="append", seqs=16, rows=1, ctx=4099),
        # what a long prompt chunk writes
        dict(qwen, name="append prompt 4001", op="append", seqs=1, rows=4001, ctx=4004),
        # a prompt sampled four times over
        dict(qwen, name="fork into 4", op="fork", branches=4, length=1003, pools=8),
        # half of a pool of sequences ends
        dict(qwen, name="compact 32 sequences", op="compact", seqs=16, length=2000, pools=4),
        # a lone request's drafts, from a greedy draft model
        dict(name="verify 1 of 3", op="verify", seqs=1, drafted=3, vocab=VOCAB, probs=False, temp=0.7),
        # a batch whose draft model samples, ragged drafts, some requests greedy
        dict(name="verify 16 of 4, sampled", op="verify", seqs=16, drafted=4, vocab=VOCAB, probs=True, temp=0.8),
        # a decode step's sampling without drafts
        dict(name="sample 64", op="verify", seqs=64, drafted=0, vocab=VOCAB, probs=False, temp=1.0),
    ]


HEADS = [(24, 4, 256), (32, 8, 128), (16, 16, 128), (64, 8, 64), (6, 2, 96), (8, 1, 160), (5, 5, 32)]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attn", "attn", "attn", "append", "fork", "compact", "verify", "verify"])
    heads, kv_heads, hd = rng.choice(HEADS)
    cache = dict(heads=heads, kv_heads=kv_heads, hd=hd, page=rng.choice([16, 24, 32, 64, 256]))
    if op == "attn":
        rows = rng.choice([1, 1, rng.randint(2, 8), _log_int(rng, 9, 500)])
        seqs = _log_int(rng, 1, 16) if rows <= 8 else rng.randint(1, 2)
        return dict(cache, op=op, seqs=seqs, rows=rows, ctx=_log_int(rng, rows + 8, 8000 if rows <= 8 else 2048))
    if op == "append":
        rows = rng.choice([1, rng.randint(2, 8), _log_int(rng, 9, 2000)])
        return dict(cache, op=op, seqs=_log_int(rng, 1, 16) if rows <= 8 else 1, rows=rows, ctx=rows + rng.randint(0, 2000))
    if op == "fork":
        return dict(cache, op=op, branches=rng.randint(1, 12), length=_log_int(rng, 20, 3000), pools=rng.randint(1, 8))
    if op == "compact":
        return dict(cache, op=op, seqs=rng.randint(1, 12), length=_log_int(rng, 20, 2000), pools=rng.randint(1, 4))
    return dict(op=op, seqs=_log_int(rng, 1, 16), drafted=rng.randint(0, 7), vocab=_log_int(rng, 1000, 151000),
                probs=rng.random() < 0.5, temp=rng.choice([0.0, 0.3, 0.7, 1.0, 1.6]))


def _contexts(case):
    """Positions each sequence holds after the pass: from a quarter of ctx to ctx."""
    n, c, r = case["seqs"], case["ctx"], case["rows"]
    return [max(r, c - (3 * c * i) // (4 * n)) for i in range(n)]


def _drafted(case):
    """Drafted tokens of each sequence: every third one or two fewer."""
    return [max(0, case["drafted"] - i % 3) for i in range(case["seqs"])]


def _temperatures(case):
    """The case's temperature, higher for every third sequence; every fourth of a larger batch is greedy."""
    return [0.0 if i % 4 == 3 else case["temp"] * (1.25 if i % 3 == 1 else 1.0) for i in range(case["seqs"])]


# ---- the cache in 4 bits -------------------------------------------------------------------------------------


def _quantise(x):
    """Codes, scales and zero points of x [..., hd] in groups of 32: int32 [..., hd / 32, 32], float64 and int32 [..., hd / 32].
    64 bits: a value at the border of two codes goes to the even one only if it is exactly there."""
    g = x.unflatten(-1, (-1, 32)).double()
    mn, mx = g.amin(-1).clamp(max=0.0), g.amax(-1).clamp(min=0.0)
    step15 = (mx - mn) / 15
    step = torch.exp2((torch.frexp(step15)[1] - 7).clamp(min=-20).double())
    d = (torch.ceil(step15 / step) * step).clamp(max=4352.0)
    by = torch.where(d > 0, d, torch.ones_like(d))
    z = torch.round(-mn / by).clamp(max=15.0)
    c = (torch.round(g / by[..., None]) + z[..., None]).clamp(0.0, 15.0)
    return c.int(), d, z.int()


def _shifts(device):
    e = torch.arange(8, device=device, dtype=torch.int32)
    return 4 * (e // 2) + 16 * (e % 2)


def _words(c):
    """Codes [..., 8] -> int32 words."""
    return (c << _shifts(c.device)).sum(-1, dtype=torch.int32)


def _headers(d, z):
    return (d.half().view(torch.int16).int() | z).to(torch.int16)


def _v_order(hd, device):
    """Where the word of each dim stands among a V slab's hd words."""
    d, w = torch.arange(hd, device=device), 4 if hd % 64 == 0 else 2
    return ((d // (16 * w)) * 16 + d % 16) * w + d // 16 % w


def _pack(x, values):
    """The bytes [blocks, ...] of K (values False) or V pages from x [blocks, P, hd]."""
    n, p, hd = x.shape
    c, d, z = _quantise(x)
    if values:
        c = c.reshape(n, p // 8, 8, hd).transpose(2, 3)
        words = torch.empty(n, p // 8, hd, dtype=torch.int32, device=x.device)
        words[:, :, _v_order(hd, x.device)] = _words(c)
        heads = _headers(d, z).reshape(n, p // 8, 8, hd // 32).transpose(2, 3)
    else:
        words = _words(c.reshape(n, p, hd // 32, 4, 8)).transpose(2, 3)
        heads = _headers(d, z)
    return torch.cat([words.contiguous().view(torch.uint8).reshape(n, -1), heads.contiguous().view(torch.uint8).reshape(n, -1)], 1)


def _unpack(blocks, p, hd, values):
    """float32 [..., P, hd] of blocks [..., bytes]; exact, a value having at most 11 significant bits."""
    lead, cut = blocks.shape[:-1], p * hd // 2
    words = blocks[..., :cut].contiguous().view(torch.int32)
    head = blocks[..., cut:].contiguous().view(torch.int16).int()
    d, z = (head & -16).to(torch.int16).view(torch.float16).float(), (head & 15).float()
    if values:
        words = words.view(*lead, p // 8, hd)[..., _v_order(hd, blocks.device)]
        c = ((words[..., None] >> _shifts(blocks.device)) & 15).float().transpose(-1, -2)  # [..., P / 8, 8, hd]
        d, z = (t.view(*lead, p // 8, hd // 32, 8).transpose(-1, -2).reshape(*lead, p, hd // 32, 1) for t in (d, z))
        c = c.reshape(*lead, p, hd // 32, 32)
    else:
        c = ((words.view(*lead, p, 4, hd // 32, 1) >> _shifts(blocks.device)) & 15).float()
        c = c.transpose(-2, -3).reshape(*lead, p, hd // 32, 32)
        d, z = (t.view(*lead, p, hd // 32, 1) for t in (d, z))
    return (d * (c - z)).reshape(*lead, p, hd)


# ---- inputs --------------------------------------------------------------------------------------------------


def _gen(seed, tag):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1009 + tag)
    return g


def _randn(seed, tag, *shape):
    return torch.randn(*shape, device="cuda", generator=_gen(seed, tag))


def _keys(seed, tag, *shape):
    """K as a model has it: some dims many times larger than the others."""
    big = torch.rand(shape[-1], device="cuda", generator=_gen(seed, tag + 50)) < 0.04
    return _randn(seed, tag, *shape) * torch.where(big, 6.0, 1.0)


def prepare(case, seed):
    return {"attn": _prepare_attn, "append": _prepare_append, "fork": _prepare_pages, "compact": _prepare_pages,
            "verify": _prepare_verify}[case["op"]](case, seed)


def _runtime(buffers):
    """A runtime whose fp32 buffers hold the tensors given by name (32-bit whole numbers by their bits)."""
    from vinf_3080ti_amd.runtime import HipWeightRuntime

    rt = HipWeightRuntime()
    for name, t in buffers.items():
        rt.alloc(name, t.numel())
        rt.buffer_tensor(name).copy_(t.reshape(-1).view(torch.float32))
    return rt


def _paged(case, seed):
    """Contexts, pages of a sequence and the table of a pool whose pages are dealt at random."""
    ctxs = _contexts(case)
    pps = -(-max(ctxs) // case["page"])
    deal = torch.randperm(len(ctxs) * pps, device="cuda", generator=_gen(seed, 1)).to(torch.int32)
    return ctxs, pps, deal.view(len(ctxs), pps)


def _prepare_attn(case, seed):
    ctxs, pps, table = _paged(case, seed)
    n, p, hd, kvh = len(ctxs), case["page"], case["hd"], case["kv_heads"]
    s = {"case": case, "table": table, "ctxs": torch.tensor(ctxs, device="cuda"),
         "q": _randn(seed, 2, n * case["rows"], case["heads"], hd),
         "kc": _pack(_keys(seed, 3, n * pps * kvh, p, hd), False), "vc": _pack(_randn(seed, 4, n * pps * kvh, p, hd), True)}
    if own:
        rt = s["rt"] = _runtime({"q": s["q"], "table": table})
        for name in ("kc", "vc"):
            rt.alloc_kv4(name, n * pps * kvh, p, hd)
            rt.buffer_tensor(name).copy_(s[name].reshape(-1))
        rt.alloc("o", s["q"].numel())
        rt.set_paging("table", p, pps, n)
        rt.set_segments([(i, c - case["rows"], case["rows"]) for i, c in enumerate(ctxs)])
        s["o"] = rt.buffer_tensor("o").view(s["q"].shape)
    return s


def _prepare_append(case, seed):
    ctxs, pps, table = _paged(case, seed)
    n, shape = len(ctxs), (len(ctxs) * case["rows"], case["kv_heads"], case["hd"])
    s = {"case": case, "k": _keys(seed, 2, *shape), "v": _randn(seed, 3, *shape)}
    if own:
        rt = s["rt"] = _runtime({"k": s["k"], "v": s["v"], "table": table})
        for name in ("kc", "vc"):
            rt.alloc_kv4(name, n * pps * case["kv_heads"], case["page"], case["hd"])
        rt.alloc("k4", s["k"].numel())
        rt.alloc("v4", s["v"].numel())
        rt.set_paging("table", case["page"], pps, n)
        rt.set_segments([(i, c - case["rows"], case["rows"]) for i, c in enumerate(ctxs)])
        s["out"] = {name: rt.buffer_tensor(name + "4").view(shape) for name in ("k", "v")}
    return s


def _prepare_pages(case, seed):
    """fork: pages 0 .. 2 are free, the sequence has the next ones. compact: the pages of `seqs` sequences, then those of as
    many others. fp16 pools."""
    p, per = case["page"], max(3, -(-(case["length"] + 1) // case["page"]))
    held = -(-case["length"] // p)
    if case["op"] == "fork":
        slots, pages = 2 + case["branches"], 3 + held + 2 * case["branches"]
    else:
        slots, pages = 2 * case["seqs"], 2 * case["seqs"] * held
    shape = (pages, case["kv_heads"], p, case["hd"])
    pools = [_randn(seed, 10 + i, *shape).half() for i in range(case["pools"])]
    table = torch.zeros(slots, per, dtype=torch.int32, device="cuda")
    if case["op"] == "fork":
        table[0, :held] = torch.arange(3, 3 + held, device="cuda")
    else:
        table[:, :held] = torch.arange(slots * held, device="cuda").view(slots, held)
    s = {"case": case, "held": held, "pools": pools, "table": table}
    if own:
        rt = s["rt"] = _runtime({"table": torch.zeros_like(table)})
        names = ["pool%d" % i for i in range(len(pools))]
        for name, t in zip(names, pools):
            rt.alloc(name, t.numel(), 2)
            rt.buffer_tensor(name).copy_(t.reshape(-1))
        rt.set_paging("table", p, per, slots)
        rt.set_page_pools(names, pages)
        if case["op"] == "fork":
            last = slots - 1
            rt.pages_reserve([(last, 0, 3 * p), (0, 0, case["length"])])
            rt.pages_free([last])
            rt.buffer_tensor("table").view(slots, per)[last] = 0
        else:
            rt.pages_reserve([(i, 0, case["length"]) for i in range(slots)])
        s["pools"] = [rt.buffer_tensor(name).view(shape) for name in names]
        s["table"] = rt.buffer_tensor("table").view(torch.int32).view(slots, per)
    return s


def _prepare_verify(case, seed):
    drafted, vocab = _drafted(case), case["vocab"]
    rows, d = sum(drafted) + len(drafted), sum(drafted)
    logits = 2.0 * _randn(seed, 1, rows, vocab)
    top = torch.randint(vocab, (rows, 24), device="cuda", generator=_gen(seed, 2))
    logits.scatter_(1, top, 12.0 + 3.0 * _randn(seed, 3, rows, 24))
    rank = torch.tensor([j for k in drafted for j in range(k + 1)], device="cuda")  # row's place in its sequence
    seq = torch.tensor([i for i, k in enumerate(drafted) for _ in range(k + 1)], device="cuda")
    k_of = torch.tensor(drafted, device="cuda")
    temps = _temperatures(case)
    temp = torch.tensor(temps, dtype=torch.float64, device="cuda")
    at = torch.nonzero(rank < k_of[seq])[:, 0]  # rows that a drafted token follows
    guess = logits[at] + 0.7 * _randn(seed, 4, d, vocab)  # the draft model's logits
    if case["probs"] and d:
        probs = torch.softmax(guess / temp[seq[at], None].clamp(min=0.25).float(), 1)
        draft = torch.multinomial(probs, 1, generator=_gen(seed, 5))[:, 0].to(torch.int32)
    else:
        probs, draft = None, guess.argmax(1).to(torch.int32) if d else torch.zeros(0, dtype=torch.int32, device="cuda")
    u = torch.rand(rows, 2, device="cuda", generator=_gen(seed, 6))
    first = torch.cumsum(k_of + 1, 0) - k_of - 1
    s = {"case": case, "logits": logits, "draft": draft, "probs": probs, "u": u, "rank": rank, "seq": seq, "k": k_of,
         "first": first, "at": at, "temp": temp}
    if own:
        whole = torch.zeros(max(d, 1), dtype=torch.int32, device="cuda")
        whole[:d] = draft
        bufs = {"logits": logits, "draft": whole, "u": u}
        if probs is not None:
            bufs["probs"] = probs
        rt = s["rt"] = _runtime(bufs)
        for name, n in (("tokens", rows), ("counts", len(drafted)), ("logprobs", rows)):
            rt.alloc(name, n)
        s["call"] = (drafted, temps)
        s["out"] = {"tokens": rt.buffer_tensor("tokens").view(torch.int32), "counts": rt.buffer_tensor("counts").view(torch.int32),
                    "logprobs": rt.buffer_tensor("logprobs")}
    return s


# ---- one pass ------------------------------------------------------------------------------------------------


def run(state):
    if own:
        return _run_own(state)
    return {"attn": _plain_attn, "append": _plain_append, "fork": _plain_fork, "compact": _plain_compact,
            "verify": _plain_verify}[state["case"]["op"]](state)


def _run_own(s):
    rt, case = s["rt"], s["case"]
    op = case["op"]
    if op == "attn":
        rt.attention_seg("q", "kc", "vc", "o", case["heads"], case["kv_heads"], case["hd"])
        return s["o"]
    if op == "append":
        rt.kv_append_seg("k", "v", "kc", "vc", case["kv_heads"], case["hd"])
        rt.kv4_read_seg("kc", "vc", "k4", "v4", case["kv_heads"], case["hd"])
        return s["out"]
    if op == "verify":
        drafted, temps = s["call"]
        rt.verify_draft("logits", "draft", "u", "tokens", "counts", case["vocab"], drafted, temperature=temps,
                        probs="probs" if s["probs"] is not None else None, logprobs="logprobs")
        return s["out"]
    n, length = case.get("branches") or case["seqs"], case["length"]
    if op == "fork":  # the branches of the pass before end first
        rt.pages_free(range(1, n + 1))
        rt.pages_fork(0, range(1, n + 1), length)
        rt.pages_reserve([(i, length, 1) for i in range(1, n + 1)])
    else:
        low, high = range(n), range(n, 2 * n)
        for gone, kept in ((low, high), (high, low)):
            rt.pages_free(gone)
            rt.pages_compact()
            rt.pages_copy([(a, b, length) for a, b in zip(kept, gone)])
    return {"pools": s["pools"], "table": s["table"]}


def _plain_attn(s):
    case, table = s["case"], s["table"].long()
    (n, pps), p, hd, kvh, rows = table.shape, case["page"], case["hd"], case["kv_heads"], case["rows"]
    per = case["heads"] // kvh
    k, v = (_unpack(s[name].view(-1, kvh, s[name].shape[-1])[table], p, hd, name == "vc").transpose(1, 2).reshape(n, kvh, pps * p, hd)
            for name in ("kc", "vc"))
    q = s["q"].view(n, rows, kvh, per, hd).permute(0, 2, 1, 3, 4).reshape(n, kvh, rows * per, hd)
    score = torch.matmul(q, k.transpose(-1, -2)).view(n, kvh, rows, per, -1) / math.sqrt(hd)
    sees = s["ctxs"][:, None] - rows + 1 + torch.arange(rows, device=q.device)  # positions each row sees
    hidden = torch.arange(pps * p, device=q.device) >= sees[..., None]
    score.masked_fill_(hidden[:, None, :, None, :], -math.inf)
    w = torch.exp(score - score.amax(-1, keepdim=True))
    out = torch.matmul(w.view(n, kvh, rows * per, -1), v).view(n, kvh, rows, per, hd) / w.sum(-1, keepdim=True)
    return out.permute(0, 2, 1, 3, 4).reshape(n * rows, case["heads"], hd)


def _plain_append(s):
    def held(x):
        c, d, z = _quantise(x)
        return (d[..., None] * (c - z[..., None])).flatten(-2).float()

    return {"k": held(s["k"]), "v": held(s["v"])}


def _plain_fork(s):
    n, held, p, length, table = s["case"]["branches"], s["held"], s["case"]["page"], s["case"]["length"], s["table"]
    free = torch.cat([torch.arange(3, device="cuda"), torch.arange(3 + held, 3 + held + n, device="cuda")])[:n]
    table[1:n + 1, :held] = table[:1, :held]
    if length % p:
        last = table[0, held - 1].long()
        for pool in s["pools"]:
            pool[free] = pool[last].clone()
    table[1:n + 1, length // p] = free.to(torch.int32)
    return {"pools": s["pools"], "table": table}


def _plain_compact(s):
    n, held, table = s["case"]["seqs"], s["held"], s["table"]
    half = n * held
    for gone, kept in ((slice(0, n), slice(n, None)), (slice(n, None), slice(0, n))):
        table[kept, :held] -= half
        table[gone, :held] = table[kept, :held] + half
        src, dst = table[kept, :held].reshape(-1).long(), table[gone, :held].reshape(-1).long()
        for pool in s["pools"]:
            pool[src] = pool[src + half]
            pool[dst] = pool[src]
    return {"pools": s["pools"], "table": table}


def _plain_verify(s):
    logits, draft, u, at, seq, first, k = (s[n] for n in ("logits", "draft", "u", "at", "seq", "first", "k"))
    # In 64 bits: of 248320 tokens many have less than 1e-8 of the mass, and a random number falls between their borders.
    top, best = logits.max(1)
    t = s["temp"][seq, None]
    p = torch.exp((logits - top[:, None]).double() / torch.where(t > 0, t, torch.ones_like(t)))
    p /= p.sum(1, keepdim=True)
    one = torch.zeros_like(p).scatter_(1, best[:, None], 1.0)
    p = torch.where(t > 0, p, one)
    x = draft.long()
    px = p[at, x]
    qx = s["probs"].gather(1, x[:, None])[:, 0].double() if s["probs"] is not None else torch.ones_like(px)
    ok = torch.zeros(k.numel(), int(s["case"]["drafted"]) + 1, dtype=torch.int64, device=k.device)
    ok[seq[at], s["rank"][at]] = (u[at, 0].double() * qx < px).long()
    count = ok.cumprod(1).sum(1)  # accepted tokens of each sequence
    stop = first + count
    rest = p[stop]
    place = torch.full_like(seq, -1)  # a row's place among the drafted ones
    place[at] = torch.arange(at.numel(), device=k.device)
    refused = torch.nonzero(count < k)[:, 0]
    from_ = place[stop[refused]]
    if s["probs"] is not None:
        rest[refused] -= s["probs"][from_].double()
    else:
        rest[refused, x[from_]] = 0.0
    rest.clamp_(min=0.0)
    rest = torch.where(rest.sum(1, keepdim=True) > 0, rest, p[stop])
    run_ = rest.cumsum(1)
    token = (run_ > u[stop, 1, None].double() * run_[:, -1:]).int().argmax(1)
    tokens = torch.full_like(seq, -1)
    tokens[at] = torch.where(s["rank"][at] < count[seq[at]], x, tokens[at])
    tokens[stop] = token
    shown = tokens >= 0
    logprobs = torch.where(shown, torch.log(p.gather(1, tokens.clamp(min=0)[:, None])[:, 0]), torch.zeros_like(p[:, 0]))
    return {"tokens": tokens.to(torch.int32), "counts": count.to(torch.int32), "logprobs": logprobs.float()}


def work(case):
    op = case["op"]
    if op in ("attn", "append"):
        ctxs, rows, hd = _contexts(case), case["rows"], case["hd"]
        if op == "append":
            n = len(ctxs) * rows * case["kv_heads"] * hd * 2
            return {"bytes": n * (4 + 9 / 16 + 9 / 16 + 4), "flops": 0}  # fp32 in, the cache written and read, fp32 out
        pairs = sum(rows * (c - rows) + rows * (rows + 1) // 2 for c in ctxs)
        return {"bytes": sum(ctxs) * 2 * case["kv_heads"] * hd * 9 // 16 + len(ctxs) * rows * case["heads"] * hd * 8,
                "flops": 4 * pairs * case["heads"] * hd}
    if op == "verify":
        n, d = case["seqs"] + sum(_drafted(case)), sum(_drafted(case))
        refused = case["seqs"] if case["probs"] and d else 0  # the draft's probabilities where a token is refused
        return {"bytes": 4 * case["vocab"] * (n + refused), "flops": 0}
    page = case["page"] * case["kv_heads"] * case["hd"] * 2 * case["pools"]
    if op == "fork":
        return {"bytes": 2 * page * case["branches"] + 4 * case["branches"] * -(-case["length"] // case["page"]), "flops": 0}
    return {"bytes": 8 * page * case["seqs"] * -(-case["length"] // case["page"]), "flops": 0}


# ---- the same in 64 bits, from the definitions -----------------------------------------------------------------


def exact(case, seed):
    if case["op"] == "attn":
        return _exact_attn(case, prepare(case, seed))
    if case["op"] == "append":
        s = prepare(case, seed)
        return {name: _exact_held(s[name]) for name in ("k", "v")}
    if case["op"] == "verify":
        return _exact_verify(case, prepare(case, seed))
    return None  # bytes moved: nothing is computed


def _exact_position(block, hd, page, pos, values):
    """Values [kv_heads, positions, hd] of the blocks [kv_heads, positions, bytes] at places pos [positions] of their pages."""
    dim = np.arange(hd)
    nibble = lambda e: e // 2 + 4 * (e % 2)  # noqa: E731  place of element e among a word's eight nibbles
    pos = np.asarray(pos)[:, None]
    if values:
        w = 4 if hd % 64 == 0 else 2
        word = (pos // 8) * hd + (dim // (16 * w) * 16 + dim % 16) * w + dim // 16 % w
        nib = nibble(pos % 8) + 0 * dim
        head = ((pos // 8) * (hd // 32) + dim // 32) * 8 + pos % 8
    else:
        word = pos * (hd // 8) + (dim % 32 // 8) * (hd // 32) + dim // 32
        nib = nibble(dim % 8) + 0 * pos
        head = pos * (hd // 32) + dim // 32
    up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(block.device).expand(block.shape[0], -1, -1)  # noqa: E731
    pick = lambda a: torch.gather(block, 2, up(a)).int()  # noqa: E731
    code = (pick(4 * word + nib // 2) >> up(4 * (nib % 2))) & 15
    at = page * hd // 2 + 2 * head
    bits = pick(at) | (pick(at + 1) << 8)
    expo, mant = bits >> 10, ((bits >> 4) & 63) << 4
    d = torch.where(expo > 0, (1024 + mant).double() * torch.exp2(expo.double() - 25), mant.double() * 2.0 ** -24)
    return d * (code - (bits & 15)).double()


def _exact_attn(case, s):
    hd, page, kvh, rows, heads = case["hd"], case["page"], case["kv_heads"], case["rows"], case["heads"]
    if sum(_contexts(case)) * rows * heads > 2 ** 31:
        return None
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for i, ctx in enumerate(_contexts(case)):
        pos = np.arange(ctx)
        pages = s["table"][i].cpu().numpy().astype(np.int64)[pos // page]
        kv = [torch.empty(kvh, ctx, hd, dtype=torch.float64, device=out.device) for _ in range(2)]
        for j in range(0, ctx, 4096):  # the blocks of 4096 positions at a time
            part = slice(j, min(ctx, j + 4096))
            where = torch.from_numpy(pages[part]).to(out.device)
            for name, to in zip(("kc", "vc"), kv):
                blocks = s[name].view(-1, kvh, s[name].shape[-1])
                used, back = torch.unique(where, return_inverse=True)
                held = blocks[used].transpose(0, 1)
                for a in range(0, back.numel(), 256):
                    to[:, part][:, a:a + 256] = _exact_position(held[:, back[a:a + 256]], hd, page, pos[part][a:a + 256] % page,
                                                                name == "vc")
        q = s["q"][i * rows:(i + 1) * rows].double()
        for h in range(heads):
            sc = q[:, h] @ kv[0][h * kvh // heads].T / math.sqrt(hd)
            for t in range(rows):
                sc[t, ctx - rows + t + 1:] = -math.inf
            out[i * rows:(i + 1) * rows, h] = torch.softmax(sc, 1) @ kv[1][h * kvh // heads]
    return out


def _exact_held(x):
    """What the cache holds of x: on the host, scales found by trying the f16 values of 7 significant bits in turn."""
    a = x.double().cpu().numpy().reshape(-1, 32)
    bits = np.arange(0, 0x7C00, 16, dtype=np.uint16)
    grid = bits.view(np.float16).astype(np.float64)
    grid = grid[grid <= 4352]
    lo, hi = np.minimum(a.min(1), 0), np.maximum(a.max(1), 0)
    d = grid[np.minimum(np.searchsorted(15 * grid, hi - lo), grid.size - 1)][:, None]
    some = np.where(d > 0, d, 1.0)
    z = np.minimum(np.rint(-lo[:, None] / some), 15)
    return torch.from_numpy((d * (np.clip(np.rint(a / some) + z, 0, 15) - z)).reshape(tuple(x.shape)))


def _exact_verify(case, s):
    """The log-probabilities; tokens and counts are whole numbers and have no other value. Sequence by sequence, on the host."""
    u, draft = s["u"].double().cpu().numpy(), s["draft"].cpu().numpy()
    found, row, d = [], 0, 0
    for k, t in zip(_drafted(case), _temperatures(case)):
        done = False
        for j in range(k + 1):
            if done:
                found.append(0.0)
                continue
            a = s["logits"][row + j].double().cpu().numpy()
            if t == 0:
                logp = np.where(np.arange(a.size) == a.argmax(), 0.0, -np.inf)
            else:
                b = a / t
                logp = b - (b.max() + np.log(np.exp(b - b.max()).sum()))
            p, take = np.exp(logp), None
            if j < k:
                x = draft[d + j]
                q = s["probs"][d + j].double().cpu().numpy() if s["probs"] is not None else np.eye(1, a.size, x)[0]
                if u[row + j, 0] * q[x] < p[x]:
                    take = x
                else:
                    left = np.maximum(p - q, 0)
                    p = left if left.sum() > 0 else p
            if take is None:
                c = np.cumsum(p)
                take, done = np.searchsorted(c, u[row + j, 1] * c[-1], side="right"), True
            found.append(float(logp[take]))
        row, d = row + k + 1, d + k
    return {"tokens": None, "counts": None, "logprobs": torch.tensor(found, dtype=torch.float64)}
