"""The operators of a decoding loop with drafted tokens over a paged cache, each as a user calls it: norm, RoPE and store of several new
tokens per sequence; attention of those tokens over their sequences' pages; verification of drafted tokens; reassigning and compacting pages.

`listed` names the cases, `draw` gives others of the same ranges, `prepare` makes what a program has in hand before the call, `run` is one
pass (plain torch, or the framework's operators where `own` is true), `work` is what it cannot do without, `exact` the same in 64 bits."""

import math
import random

import torch

own = False

PAGE = 16  # positions of a page
D = 128    # values of a head
EPS = 1e-6
THETA = 1e6


def listed():
    return [
        # one sequence decoding alone over its pages: latency
        dict(name="attend-one-token", kind="attend", kv="f16", precision="f32", hq=32, hkv=8, few=1, few_tokens=1, past=700, past_spread=0, lengths=1),
        # a serving step with four drafted tokens for each of 64 sequences
        dict(name="attend-drafts-64", kind="attend", kv="f16", precision="f16", hq=32, hkv=8, few=64, few_tokens=5, past=2600, past_spread=900, lengths=2),
        # a prompt's next portion beside decoding sequences, 8-bit cache
        dict(name="attend-mixed-q8", kind="attend", kv="q8_0", precision="f16", hq=64, hkv=8, few=24, few_tokens=3, past=4000, past_spread=2500, many=1, many_tokens=1000,
             many_past=9000, lengths=3),
        # admitted prompts of very different lengths, in one run; two of them go on from a cached prefix
        dict(name="attend-prompts", kind="attend", kv="f16", precision="f16", hq=32, hkv=8, many=14, many_tokens=4000, many_past=500, lengths=4),
        # a small model in 32 bits: short prompts and single tokens
        dict(name="attend-small-f32", kind="attend", kv="f32", precision="f32", hq=6, hkv=2, few=9, few_tokens=2, past=300, past_spread=200, many=5, many_tokens=211,
             many_past=40, lengths=5),
        # the new tokens of that serving step on their way into the cache
        dict(name="store-drafts-64", kind="store", kv="q8_0", hq=32, hkv=8, few=64, few_tokens=5, past=150, past_spread=100, lengths=6),
        # and of admitted prompts
        dict(name="store-prompts", kind="store", kv="f16", hq=32, hkv=8, many=9, many_tokens=2500, many_past=100, lengths=7),
        # one sequence's drafts, proposed by a lookup (no probabilities of their own): latency
        dict(name="verify-lookup-1", kind="verify", seqs=1, drafts=6, vocab=151936, proposal=False, lengths=8),
        # a serving step's drafts against the draft model's probabilities
        dict(name="verify-64", kind="verify", seqs=64, drafts=4, vocab=151936, proposal=True, lengths=9),
        # after verification: every sequence keeps what was accepted and gets room for the next step
        dict(name="pages-step-64", kind="reassign", kv="f16", hkv=8, layers=36, rows=64, past=300, fork=1, room=5, max_pages=256, lengths=10),
        # every prompt sampled several times: the rows of a prompt share its pages, each with a copy of the last one
        dict(name="pages-fork-48", kind="reassign", kv="q8_0", hkv=8, layers=36, rows=48, past=300, fork=6, room=40, max_pages=128, lengths=11),
        # half of the sequences have gone: the rest move to the front of the pool
        dict(name="pages-compact", kind="compact", kv="f16", hkv=8, layers=24, rows=40, past=220, gone=0.5, max_pages=64, lengths=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "store", "verify", "reassign", "compact"])
    case = dict(kind=kind, lengths=rng.randint(100, 10 ** 6))
    if kind == "verify":
        return dict(case, seqs=_log(rng, 1, 96), drafts=rng.randint(0, 8), vocab=_log(rng, 300, 152000), proposal=rng.random() < 0.7)
    hkv = rng.choice([1, 2, 4, 8])
    case.update(kv=rng.choice(["f16", "f16", "q8_0", "f32"] if kind in ("attend", "store") else ["f16", "q8_0"]), hkv=hkv)
    if kind == "compact":
        return dict(case, layers=_log(rng, 1, 32), rows=_log(rng, 1, 48), past=_log(rng, 1, 300), gone=rng.choice([0.1, 0.5, 0.8]), max_pages=rng.randint(40, 100))
    if kind == "reassign":
        return dict(case, layers=_log(rng, 1, 36), rows=_log(rng, 1, 64), past=_log(rng, 1, 300), fork=rng.randint(1, 8), room=_log(rng, 1, 64), max_pages=rng.randint(64, 300))
    case["hq"] = hkv * rng.choice([1, 2, 3, 4, 5, 7, 8])
    shape = rng.choice(["few", "many", "both"])
    if shape != "many":
        past = _log(rng, 1, 6000) if kind == "attend" else _log(rng, 1, 400)
        case.update(few=_log(rng, 1, 64), few_tokens=rng.randint(1, 8), past=past, past_spread=rng.randint(0, past))
    if shape != "few":
        most = 1500 if case["kv"] == "f32" else 2500
        case.update(many=rng.randint(1, 8), many_tokens=_log(rng, 9, most), many_past=_log(rng, 1, 2000) if kind == "attend" else _log(rng, 1, 300))
    if kind == "attend":
        case["precision"] = "f32" if case["kv"] == "f32" else rng.choice(["f16", "f16", "f16", "f32"] if shape == "few" else ["f16"])
    return case


# ---- what a program has in hand -----------------------------------------------------------------------------------------


def _lengths(c):
    """(new tokens, positions before them) of every sequence, by the case alone."""
    rng = random.Random(c["lengths"])
    seqs = []
    for _ in range(c.get("many", 0)):
        seqs.append((max(1, round(c["many_tokens"] * rng.random() ** 2) if seqs else c["many_tokens"]), rng.choice([0, 0, 0, rng.randint(0, c["many_past"])]) if seqs else c["many_past"]))
    for i in range(c.get("few", 0)):
        seqs.append((c["few_tokens"] if i == 0 else rng.randint(max(1, c["few_tokens"] - 3), c["few_tokens"]), c["past"] + rng.randint(-c["past_spread"], c["past_spread"])))
    seqs = [(n, max(0, p)) for n, p in seqs]
    rng.shuffle(seqs)
    return seqs


_CTX = []


def _framework():
    import brasa_b200 as B

    if not _CTX:
        ctx = B.Context(0)
        _CTX.extend([B, ctx, B.Kernels(ctx)])
    return _CTX


class _Bytes:
    """A buffer of the framework that torch can look into, given back with the last tensor that does."""

    def __init__(self, n):
        _, ctx, _ = _framework()
        self.buffer = ctx.buffer(n)
        ctx.sync()
        self.__cuda_array_interface__ = dict(shape=(n,), typestr="|u1", data=(self.buffer.ptr, False), version=3)

    def __del__(self):
        self.buffer.free()


class _State:
    """Tensors by name; where the framework runs, each lies in one of its buffers (`held`)."""

    def __init__(self, case):
        self.case, self.held = case, {}

    def put(self, name, t):
        if own:
            held = _Bytes(max(16, t.numel() * t.element_size()))
            view = torch.as_tensor(held, device="cuda")[:t.numel() * t.element_size()].view(t.dtype).view(t.shape)
            view.copy_(t)
            self.held[name], t = held.buffer, view
        setattr(self, name, t)


def _rng(seed):
    return torch.Generator("cuda").manual_seed(seed)


def _row_shape(kv):
    return {"f16": (D, torch.float16), "f32": (D, torch.float32), "q8_0": (136, torch.uint8)}[kv]


def _randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _quantize(x):
    """Rows of 128 values as 128 8-bit codes and four 16-bit scales."""
    b = x.float().unflatten(-1, (4, 32))
    d = (b.abs().amax(-1, keepdim=True) / 127).half()
    f = d.float()
    q = torch.where(f == 0, 0.0, (b / torch.where(f == 0, 1.0, f)).round().clamp(-127, 127)).to(torch.int8)
    return torch.cat([q.flatten(-2).view(torch.uint8), d.squeeze(-1).contiguous().view(torch.uint8)], -1)


def _values(rows, kv, to=torch.float32):
    """Rows of a cache as the values that they stand for."""
    if kv != "q8_0":
        return rows.to(to)
    rows = rows.contiguous()
    return (rows[..., :128].view(torch.int8).to(to).unflatten(-1, (4, 32)) * rows[..., 128:].contiguous().view(torch.float16).to(to)[..., None]).flatten(-2)


def _pool(g, shape, kv, scale):
    """Pages of random rows; in parts, so that large pools need no larger scratch."""
    width, dtype = _row_shape(kv)
    pool = torch.empty(*shape, width, device="cuda", dtype=dtype)
    for part in pool.flatten(0, -3).split(65536):
        x = _randn(g, *part.shape[:-1], D) * scale
        part.copy_(_quantize(x) if kv == "q8_0" else x)
    return pool


def _pages(c, g, s):
    """Pools, page table, lengths and the run's starts for the sequences of an attention or store case."""
    seqs = _lengths(c)
    counts = [-(-(n + p) // PAGE) for n, p in seqs]
    pages, most = sum(counts), max(counts)
    s.seqs, s.num_pages, s.max_pages, s.longest, s.lengths = len(seqs), pages + 3, most + 1, max(n for n, _ in seqs), seqs
    order = torch.randperm(s.num_pages, generator=torch.Generator().manual_seed(c["lengths"]))
    table, at = torch.zeros(len(seqs), s.max_pages, dtype=torch.int32), 0
    for i, n in enumerate(counts):
        table[i, :n] = order[at:at + n]
        at += n
    starts = torch.tensor([0] + [n for n, _ in seqs]).cumsum(0).int()
    s.tokens = int(starts[-1])
    s.put("table", table.cuda())
    s.put("lens", torch.tensor([p for _, p in seqs], dtype=torch.int32).cuda())
    s.put("starts", starts.cuda())
    # keys of unit norm times sqrt(128), as a norm of the heads leaves them; a few dimensions stand out
    s.put("kpool", _pool(g, (s.num_pages, PAGE, c["hkv"]), c["kv"], 1.0 + 2.0 * (torch.arange(D, device="cuda") % 37 == 5)))
    s.put("vpool", _pool(g, (s.num_pages, PAGE, c["hkv"]), c["kv"], 0.7))


def _table_rows(c):
    """Page table and lengths of the rows that page operators start from, by the case alone: groups of `fork` rows of which the first holds a prompt."""
    rng = random.Random(c["lengths"])
    most = c["max_pages"] * PAGE
    lens = [min(most - 1, max(1, round(c["past"] * rng.uniform(0.3, 1.7)))) for _ in range(c["rows"])]
    if c["kind"] == "reassign":
        lens = [n if r % c["fork"] == 0 else 0 for r, n in enumerate(lens)]
    counts = [-(-n // PAGE) for n in lens]
    need = sum(counts)
    if c["kind"] == "reassign":
        need += c["rows"] * (2 + -(-c["room"] // PAGE))
    num = need + 5
    order = list(range(num))
    rng.shuffle(order)
    table, at = [], 0
    for n in counts:
        table.append(order[at:at + n] + [-1] * (c["max_pages"] - n))
        at += n
    pinned = [0] * num
    for p in order[-3:]:
        pinned[p] = 1
    return rng, lens, table, num, pinned


def prepare(case, seed):
    c, g, s = case, _rng(seed), _State(case)
    if c["kind"] == "verify":
        rng = random.Random(c["lengths"])
        n = [c["drafts"] if i == 0 else rng.randint(0, c["drafts"]) for i in range(c["seqs"])]
        starts = torch.tensor([0] + [k + 1 for k in n]).cumsum(0).int()
        s.rows, s.seqs = int(starts[-1]), c["seqs"]
        last = torch.zeros(s.rows, dtype=torch.bool)
        last[(starts[1:] - 1).long()] = True
        # logits of a language model: a long tail and a few clear candidates; the draft model's are near the target's
        shape = -1.1 * torch.log(1 + torch.arange(c["vocab"], device="cuda", dtype=torch.float32))
        logits = shape[torch.argsort(torch.rand(c["vocab"], device="cuda", generator=g))] + _randn(g, s.rows, c["vocab"])
        s.put("p", torch.softmax(logits, -1))
        drafted = logits[~last.cuda()] + 0.5 * _randn(g, s.rows - c["seqs"], c["vocab"])
        if c["proposal"]:
            s.put("q", torch.softmax(drafted, -1))
        noise = -torch.log(-torch.log(torch.rand(drafted.shape, device="cuda", generator=g, dtype=torch.float64).clamp(min=1e-12)))
        s.put("drafts", torch.argmax(drafted + noise, -1).int() if len(drafted) else torch.zeros(0, dtype=torch.int32, device="cuda"))
        s.put("u", torch.rand(s.rows, device="cuda", generator=g))
        s.put("starts", starts.cuda())
        s.put("out", torch.zeros(s.rows, dtype=torch.int32, device="cuda"))
        s.put("accepted", torch.zeros(c["seqs"], dtype=torch.int32, device="cuda"))
    elif c["kind"] in ("reassign", "compact"):
        rng, lens, table, s.num_pages, pinned = _table_rows(c)
        if c["kind"] == "reassign":
            s.put("source", torch.tensor([r - r % c["fork"] for r in range(c["rows"])], dtype=torch.int32).cuda())
            cut = [rng.randint(0, 5) for _ in range(c["rows"])]
            s.put("keep", torch.tensor([max(0, lens[r - r % c["fork"]] - (cut[r] if c["fork"] == 1 else 0)) for r in range(c["rows"])], dtype=torch.int32).cuda())
            s.put("room", torch.full((c["rows"],), c["room"], dtype=torch.int32, device="cuda"))
            s.put("lens_out", torch.zeros(c["rows"], dtype=torch.int32, device="cuda"))
        else:
            for r in range(c["rows"]):
                if rng.random() < c["gone"]:
                    lens[r], table[r] = 0, [-1] * c["max_pages"]
            s.put("moved", torch.zeros(s.num_pages, dtype=torch.int32, device="cuda"))
        s.put("table", torch.tensor(table, dtype=torch.int32).cuda())
        s.put("lens", torch.tensor(lens, dtype=torch.int32).cuda())
        s.put("pinned", torch.tensor(pinned, dtype=torch.int32).cuda())
        s.put("table_out", torch.zeros_like(s.table))
        s.put("result", torch.zeros(4, dtype=torch.int32, device="cuda"))
        for name in ("kpool", "vpool"):
            s.put(name, _pool(g, (c["layers"], s.num_pages, PAGE, c["hkv"]), c["kv"], 1.0))
    else:
        _pages(c, g, s)
        s.put("q", 1.5 * _randn(g, s.tokens, c["hq"], D))
        if c["kind"] == "store":
            s.put("k", 3.0 * _randn(g, s.tokens, c["hkv"], D))
            s.put("v", _randn(g, s.tokens, c["hkv"], D))
            s.put("q_norm", 1.0 + 0.2 * _randn(g, D))
            s.put("k_norm", 1.0 + 0.2 * _randn(g, D))
            s.put("q_out", torch.zeros(s.tokens, c["hq"], D, device="cuda"))
            angle = torch.arange(s.max_pages * PAGE, device="cuda").double()[:, None] * THETA ** (-2.0 * torch.arange(D // 2, device="cuda").double() / D)
            s.put("cos", angle.cos().float())
            s.put("sin", angle.sin().float())
        else:
            s.put("o", torch.zeros(s.tokens, c["hq"], D, device="cuda", dtype=torch.float16 if c["precision"] == "f16" else torch.float32))
    if own:  # one command for many calls, as a program's step has
        B, ctx, s.kernels = _framework()
        s.cmd, b = ctx.command(), s.held
        kv = {"f16": B.KvType.F16, "q8_0": B.KvType.Q8_0, "f32": B.KvType.F32}.get(c.get("kv"))
        if c["kind"] in ("attend", "store"):
            s.paged = B.Kernels.paged_kv(b["kpool"], b["vpool"], b["table"], b["lens"], s.seqs, s.max_pages, s.num_pages, kv)
            s.packed = B.Kernels.packed_run(b["starts"], s.tokens, s.longest)
            if c["kind"] == "store":
                s.rope = B.RopeTable(ctx, THETA, D, s.max_pages * PAGE)
        elif c["kind"] != "verify":
            s.pool = B.Kernels.page_pool(b["kpool"], b["vpool"], b["table"], b["lens"], b["pinned"], c["rows"], c["max_pages"], s.num_pages, c["layers"], c["hkv"],
                                         kv)
        torch.cuda.synchronize()
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------------


def run(state):
    s, c = state, state.case
    return {"attend": _attend, "store": _store, "verify": _verify, "reassign": _reassign, "compact": _compact}[c["kind"]](s, c)


def _softmax_rows(scores, hidden):
    scores = scores.masked_fill_(hidden, -math.inf)
    scores = (scores - scores.amax(-1, keepdim=True)).exp_()
    return scores.div_(scores.sum(-1, keepdim=True))


def _attend(s, c):
    if own:
        b = s.held
        B = _framework()[0]
        s.kernels.attention_packed(s.cmd, b["q"], s.paged, s.packed, b["o"], c["hq"], c["hkv"], B.PrefillPrecision.F16 if c["precision"] == "f16" else B.PrefillPrecision.F32)
        return s.o
    G = c["hq"] // c["hkv"]
    out = torch.empty_like(s.o)
    kpool, vpool = s.kpool.flatten(0, 1), s.vpool.flatten(0, 1)
    few = [i for i, (n, _) in enumerate(s.lengths) if n <= 8]
    if few:  # sequences of few tokens together, padded
        at = torch.tensor(few, device="cuda")
        n, past, first = (s.starts[1:] - s.starts[:-1])[at], s.lens[at], s.starts[:-1][at]
        N, L = max(s.lengths[i][0] for i in few), max(sum(s.lengths[i]) for i in few)
        pos, j = torch.arange(L, device="cuda"), torch.arange(N, device="cuda")
        slot = s.table[at][:, pos // PAGE].clamp(min=0).long() * PAGE + pos % PAGE
        k, v = (_values(p[slot], c["kv"]).permute(0, 2, 1, 3) for p in (kpool, vpool))  # [sequence, key head, position, 128]
        live = j[None] < n[:, None]
        token = (first[:, None] + torch.where(live, j[None], 0)).long()
        q = s.q[token].unflatten(2, (c["hkv"], G)).permute(0, 2, 1, 3, 4).flatten(2, 3)
        hidden = (pos[None, None] > (past[:, None] + j[None])[..., None])[:, None, :, None].expand(-1, -1, -1, G, -1).flatten(2, 3)
        o = _softmax_rows(q @ k.transpose(2, 3) / math.sqrt(D), hidden) @ v
        o = o.unflatten(2, (N, G)).permute(0, 2, 1, 3, 4).flatten(2, 3)
        out[token[live]] = o[live].to(out.dtype)
    for i, (n, past) in enumerate(s.lengths):  # the others one by one
        if n > 8:
            pos = torch.arange(past + n, device="cuda")
            slot = s.table[i][pos // PAGE].long() * PAGE + pos % PAGE
            k, v = (_values(p[slot], c["kv"]).permute(1, 0, 2) for p in (kpool, vpool))
            a = s.starts[i].long() + torch.arange(n, device="cuda")
            q = s.q[a].unflatten(1, (c["hkv"], G)).permute(1, 0, 2, 3).flatten(1, 2)
            hidden = (pos[None] > past + torch.arange(n, device="cuda")[:, None]).repeat_interleave(G, 0)
            o = _softmax_rows(q @ k.transpose(1, 2) / math.sqrt(D), hidden) @ v
            out[a] = o.unflatten(1, (n, G)).permute(1, 0, 2, 3).flatten(1, 2).to(out.dtype)
    return out


def _store(s, c):
    if own:
        b = s.held
        s.kernels.qk_norm_rope_store_packed(s.cmd, b["q"], b["k"], b["v"], b["q_norm"], b["k_norm"], EPS, s.rope, s.paged, s.packed, b["q_out"], c["hq"], c["hkv"])
        q = s.q_out
    else:
        t = torch.arange(s.tokens, device="cuda")
        seq = torch.searchsorted(s.starts[1:].contiguous(), t.int(), right=True)
        pos = (s.lens[seq] + t - s.starts[seq]).long()
        slot = s.table[seq, pos // PAGE].long() * PAGE + pos % PAGE
        cos, sin = s.cos[pos][:, None], s.sin[pos][:, None]

        def normed(x, w):
            y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w
            a, b = y[..., :D // 2], y[..., D // 2:]
            return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        q, k = normed(s.q, s.q_norm), normed(s.k, s.k_norm)
        for pool, x in ((s.kpool, k), (s.vpool, s.v)):
            pool.view(-1, *pool.shape[2:])[slot] = _quantize(x) if c["kv"] == "q8_0" else x.to(pool.dtype)
    if c["kv"] != "q8_0":
        return dict(q=q, k=s.kpool, v=s.vpool)
    if own:  # the framework's stream ends before torch's reads the codes
        torch.cuda.current_stream().wait_stream(torch.cuda.ExternalStream(_framework()[1].stream))
    return dict(q=q, k=_values(s.kpool, "q8_0", torch.float16), v=_values(s.vpool, "q8_0", torch.float16))


def _verify(s, c):
    if own:
        b = s.held
        s.kernels.verify_drafts(s.cmd, b["p"], b["q"] if c["proposal"] else None, b["drafts"], b["u"], b["starts"], s.seqs, s.rows, c["vocab"], b["out"], b["accepted"])
        return dict(tokens=s.out, accepted=s.accepted)
    first, n = s.starts[:-1].long(), (s.starts[1:] - s.starts[:-1] - 1).long()
    row = torch.arange(s.rows, device="cuda")
    seq = torch.searchsorted(s.starts[1:].contiguous(), row.int(), right=True)
    is_last = row == s.starts[1:].long()[seq] - 1
    at = (row - seq)[~is_last]  # of the drafted rows
    tok = s.drafts.long()
    pt = s.p[row[~is_last], tok].double()
    qt = s.q[at, tok].double() if c["proposal"] else torch.ones_like(pt)
    refused = torch.ones(s.rows, dtype=torch.bool, device="cuda")
    refused[~is_last] = ~(s.u[~is_last].double() * qt < pt)
    stop = torch.full((s.seqs,), s.rows, device="cuda", dtype=torch.long).scatter_reduce(0, seq[refused], row[refused], "amin")
    accepted = stop - first
    full = accepted == n
    p = s.p[stop].double()
    drafted = torch.zeros(s.rows, dtype=torch.long, device="cuda")
    drafted[~is_last] = tok
    if c["proposal"]:
        qrow = (stop - torch.arange(s.seqs, device="cuda")).clamp(max=max(0, len(s.q) - 1))
        mass = p if not len(s.q) else torch.where(full[:, None], p, (p - s.q[qrow].double()).clamp(min=0))
    else:
        mass = torch.where(~full[:, None] & (torch.arange(c["vocab"], device="cuda")[None] == drafted[stop][:, None]), 0.0, p)
    total = mass.cumsum(-1)
    point = s.u[s.starts[1:].long() - 1].double() * total[:, -1]
    extra = torch.searchsorted(total, point[:, None], right=True).squeeze(-1)
    out = torch.where(row < stop[seq], drafted, torch.where(row == stop[seq], extra[seq], 0)).int()
    return dict(tokens=out, accepted=accepted.int())


def _copied(s, src, dst):
    for pool in (s.kpool, s.vpool):
        pool[:, dst] = pool[:, src]


def _reassign(s, c):
    if own:
        b = s.held
        s.kernels.pages_reassign(s.cmd, s.pool, b["source"], b["keep"], b["room"], b["table_out"], b["lens_out"], b["result"])
        return dict(table=s.table_out, lens=s.lens_out, result=s.result, k=s.kpool, v=s.vpool)
    R, P, N = c["rows"], c["max_pages"], s.num_pages
    row, page = torch.arange(R, device="cuda"), torch.arange(P, device="cuda")
    source = s.source.long()
    keep = torch.minimum(s.keep, s.lens[source]).long()
    ends = torch.minimum(keep + s.room, torch.full_like(keep, P * PAGE))
    have, want, whole = (keep + PAGE - 1) // PAGE, (ends + PAGE - 1) // PAGE, keep // PAGE
    old = s.table[source].long()
    table = torch.where(page[None] < have[:, None], old, -1)
    ragged = keep % PAGE > 0
    tail = old.gather(1, whole.clamp(max=P - 1)[:, None]).squeeze(1)
    shared = torch.zeros(N + 1, dtype=torch.bool, device="cuda")
    shared[torch.where(page[None] < whole[:, None], old, N).flatten()] = True
    shared[:N] |= s.pinned > 0
    owner = torch.full((N + 1,), R, device="cuda").scatter_reduce(0, torch.where(ragged, tail, N), row, "amin")
    copied = ragged & (shared[tail] | (owner[tail] != row))
    used = s.pinned > 0
    used[table[(table >= 0)]] = True
    free = torch.nonzero(~used).squeeze(1)
    need = copied.long() + want - have
    first = need.cumsum(0) - need
    place = first[:, None] + copied[:, None].long() + page[None] - have[:, None]
    fresh = (page[None] >= have[:, None]) & (page[None] < want[:, None])
    table = torch.where(fresh, free[place.clamp(0, len(free) - 1)], table)
    dst = free[first.clamp(max=len(free) - 1)]
    table = torch.where(copied[:, None] & (page[None] == whole[:, None]), dst[:, None], table)
    short = (need.sum() - len(free)).clamp(min=0)
    if short == 0:
        _copied(s, tail[copied], dst[copied])
    else:
        table, keep, need, copied = s.table.long(), s.lens.long(), need * 0, copied & False
        used = s.pinned > 0
        used[table[(table >= 0)]] = True
    in_use = used.sum() + need.sum()
    result = torch.stack([in_use, copied.sum(), N - in_use, short])
    return dict(table=table.int(), lens=keep.int(), result=result.int(), k=s.kpool, v=s.vpool)


def _compact(s, c):
    if own:
        b = s.held
        s.kernels.pages_compact(s.cmd, s.pool, b["table_out"], b["moved"], b["result"])
        return dict(table=s.table_out, moved=s.moved, result=s.result, k=s.kpool, v=s.vpool)
    N = s.num_pages
    used = torch.zeros(N, dtype=torch.bool, device="cuda")
    used[s.table[s.table >= 0].long()] = True
    used |= s.pinned > 0
    holes, movers = torch.nonzero(~used).squeeze(1), torch.nonzero(used & (s.pinned == 0)).squeeze(1).flip(0)
    n = min(len(holes), len(movers))
    holes, movers = holes[:n], movers[:n]
    moves = holes < movers
    holes, movers = holes[moves], movers[moves]
    _copied(s, movers, holes)
    moved = torch.where(used, torch.arange(N, device="cuda"), -1)
    moved[movers] = holes
    used[movers], used[holes] = False, True
    table = torch.where(s.table >= 0, moved[s.table.clamp(min=0).long()], -1)
    end = (torch.nonzero(used).squeeze(1).max() + 1) if bool(used.any()) else torch.zeros((), dtype=torch.long, device="cuda")
    result = torch.stack([used.sum(), torch.tensor(len(holes), device="cuda"), end, torch.zeros((), dtype=torch.long, device="cuda")])
    return dict(table=table.int(), moved=moved.int(), result=result.int(), k=s.kpool, v=s.vpool)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------


def work(case):
    c = case
    if c["kind"] == "verify":
        return dict(bytes=c["seqs"] * c["vocab"] * 4 * (1 + c["proposal"]), flops=0)
    row = {"f16": 256, "f32": 512, "q8_0": 136}[c["kv"]] * c["hkv"]
    if c["kind"] == "compact":
        rng, lens, table, num, pinned = _table_rows(c)
        left = set()
        for r in range(c["rows"]):
            if not rng.random() < c["gone"]:
                left |= {p for p in table[r] if p >= 0}
        pins = {p for p in range(num) if pinned[p]}
        holes, movers = [p for p in range(num) if p not in left | pins], sorted(left - pins, reverse=True)
        moves = sum(h < m for h, m in zip(holes, movers))
        return dict(bytes=moves * 4 * PAGE * row * c["layers"] + c["rows"] * c["max_pages"] * 8, flops=0)
    if c["kind"] == "reassign":
        _, lens, _, _, _ = _table_rows(c)
        copies = sum(lens[r - r % c["fork"]] % PAGE > 0 for r in range(c["rows"]) if r % c["fork"])
        return dict(bytes=copies * 4 * PAGE * row * c["layers"] + c["rows"] * c["max_pages"] * 8, flops=0)
    seqs = _lengths(c)
    tokens = sum(n for n, _ in seqs)
    if c["kind"] == "store":
        return dict(bytes=tokens * ((2 * c["hq"] + 2 * c["hkv"]) * D * 4 + 2 * row), flops=0)
    keys = sum(n + p for n, p in seqs)
    pairs = sum(n * p + n * (n + 1) // 2 for n, p in seqs)
    return dict(bytes=2 * keys * row + tokens * c["hq"] * D * (4 + (2 if c["precision"] == "f16" else 4)), flops=4 * D * c["hq"] * pairs)


# ---- the same in 64 bits, from the definitions ----------------------------------------------------------------------------


def _stands64(rows, kv):
    """What rows of a cache stand for, in 64 bits."""
    if kv != "q8_0":
        return rows.double()
    codes, scales = rows[..., :128].contiguous().view(torch.int8).double(), rows[..., 128:].contiguous().view(torch.float16).double()
    return codes * scales.repeat_interleave(32, -1)


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    c = case
    if c["kind"] == "attend":
        out, at = torch.zeros(s.tokens, c["hq"], D, device="cuda", dtype=torch.float64), 0
        for i, (n, past) in enumerate(s.lengths):
            pos = torch.arange(past + n, device="cuda")
            page = s.table[i, pos // PAGE].long()
            for h in range(c["hkv"]):
                k, v = (_stands64(pool[page, pos % PAGE, h], c["kv"]) for pool in (s.kpool, s.vpool))
                for e in range(0, n, 512):
                    m = min(512, n - e)
                    seen = past + e + m
                    keep = pos[None, :seen] <= past + e + torch.arange(m, device="cuda")[:, None]
                    for g in range(h * c["hq"] // c["hkv"], (h + 1) * c["hq"] // c["hkv"]):
                        w = s.q[at + e:at + e + m, g].double() @ k[:seen].T * D ** -0.5
                        w = torch.where(keep, w, -math.inf)
                        w = torch.exp(w - torch.logsumexp(w, 1, keepdim=True))
                        out[at + e:at + e + m, g] = w @ v[:seen]
            at += n
        return out
    if c["kind"] == "store":
        where = torch.tensor([p + j for n, p in s.lengths for j in range(n)], device="cuda")
        owner = torch.tensor([i for i, (n, _) in enumerate(s.lengths) for _ in range(n)], device="cuda")
        angle = where.double()[:, None] * THETA ** (-2.0 * torch.arange(D // 2, device="cuda").double() / D)
        turn = torch.polar(torch.ones_like(angle), angle)[:, None]

        def rotated(x, w):
            x = x.double()
            x = x / (x.pow(2).sum(-1, keepdim=True) / D + EPS).sqrt() * w.double()
            z = torch.complex(x[..., :D // 2], x[..., D // 2:]) * turn
            return torch.cat([z.real, z.imag], -1)
        pools = []
        for pool, x in ((s.kpool, rotated(s.k, s.k_norm)), (s.vpool, s.v.double())):
            stands = _stands64(pool, c["kv"])
            if c["kv"] == "q8_0":
                b = x.unflatten(-1, (4, 32))
                d = (b.abs().amax(-1, keepdim=True) / 127).half().double()
                x = (torch.where(d > 0, torch.round(b / d.clamp(min=1e-30)).clamp(-127, 127), 0) * d).flatten(-2)
            stands[s.table[owner, where // PAGE].long(), where % PAGE] = x
            pools.append(stands)
        return dict(q=rotated(s.q, s.q_norm), k=pools[0], v=pools[1])
    return None
