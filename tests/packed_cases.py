"""Inputs and 64-bit references for the operators over packed runs: caches whose pages lie scattered in a pool, and what a run over them gives."""
import numpy as np

import oracle as O

PAGE, D = 16, 128
ROW = {"f32": 512, "f16": 256, "q8_0": 136}


def to_bytes(rows, kv):
    """f32 [..., 128] -> the cache's bytes [..., ROW]."""
    if kv == "f32":
        return np.ascontiguousarray(rows, np.float32).view(np.uint8)
    if kv == "f16":
        return rows.astype(np.float16).view(np.uint8)
    return np.frombuffer(np.ascontiguousarray(O.quantize_kv_q8(np.ascontiguousarray(rows, np.float32).reshape(-1))).tobytes(), np.uint8).reshape(*rows.shape[:-1], 136).copy()


def from_bytes(raw, kv):
    if kv == "f32":
        return np.ascontiguousarray(raw).view(np.float32).astype(np.float64)
    if kv == "f16":
        return np.ascontiguousarray(raw).view(np.float16).astype(np.float64)
    d = np.ascontiguousarray(raw[..., 128:]).view(np.float16).astype(np.float64)
    return np.ascontiguousarray(raw[..., :128]).view(np.int8).astype(np.float64) * np.repeat(d, 32, -1)


class Run:
    """Sequences (new tokens, positions before them), their pages in a random order, rows of the pool that nobody reached full of NaN."""

    def __init__(self, seqs, hq, hkv, kv, seed=0, spare_tokens=0, scale=1.0):
        g = np.random.default_rng(seed)
        self.seqs, self.hq, self.hkv, self.kv = seqs, hq, hkv, kv
        counts = [-(-(n + p) // PAGE) for n, p in seqs]
        self.max_pages = max(counts) + 1
        self.num_pages = sum(counts) + 2
        order = g.permutation(self.num_pages)
        self.table = np.zeros((len(seqs), self.max_pages), np.int32)
        at = 0
        for s, c in enumerate(counts):
            self.table[s, :c] = order[at:at + c]
            at += c
        self.lens = np.array([p for _, p in seqs], np.uint32)
        self.starts = np.concatenate([[0], np.cumsum([n for n, _ in seqs])]).astype(np.uint32)
        self.tokens = int(self.starts[-1]) + spare_tokens
        self.longest = max(1, max(n for n, _ in seqs))
        self.q = (scale * g.standard_normal((self.tokens, hq, D))).astype(np.float32)
        fill = np.full((self.num_pages, PAGE, hkv, ROW[kv]), 0xFF, np.uint8)  # NaN in every type (in 8 bits: a NaN scale)
        self.k, self.v = fill.copy(), fill.copy()
        for s, (n, p) in enumerate(seqs):
            for pool in (self.k, self.v):
                rows = to_bytes(g.standard_normal((n + p, hkv, D)).astype(np.float32), kv)
                for i in range(n + p):
                    pool[self.table[s, i // PAGE], i % PAGE] = rows[i]

    def rows(self, pool, s, upto):
        """(values [upto, hkv, 128], which positions have a page)."""
        out, there = np.zeros((upto, self.hkv, D)), np.zeros(upto, bool)
        for i in range(upto):
            page = self.table[s, i // PAGE]
            if 0 <= page < self.num_pages:
                out[i], there[i] = from_bytes(pool[page, i % PAGE], self.kv), True
        return out, there

    def attention(self, half, kv=None):
        """o in 64 bits, and how far a result may be off. With s the scores, o = sum p v: do = sum p ds (v - o) to first order, and
        kv: the cache that the rows came from, if not this one.
        half: q rounded to f16, 2^-11 of every factor, independent (six standard deviations of the sum); P to f16, 2^-11 of each; o to f16; an
        8-bit cache's rows, whose values d * code have up to 19 bits, to f16 as well.
        both: sums of 128 terms in 32 bits, where a tensor core may cut instead of round, and products of terms of 2^-22: 2^-22 * 130 of sum |q k|;
        sums over the keys and the exponentials, 2^-22 * (keys + 8) of sum p |v|."""
        out, tol = np.zeros((self.tokens, self.hq, D)), np.zeros((self.tokens, self.hq, D))
        G = self.hq // self.hkv
        for s, (n, past) in enumerate(self.seqs):
            k, there = self.rows(self.k, s, n + past)
            v, _ = self.rows(self.v, s, n + past)
            for j in range(n):
                see = there[:past + j + 1]
                if not see.any():
                    continue
                t = int(self.starts[s]) + j
                for h in range(self.hq):
                    kk, vv, qq = k[:past + j + 1, h // G][see], v[:past + j + 1, h // G][see], self.q[t, h].astype(np.float64)
                    a = kk @ qq / np.sqrt(D)
                    p = np.exp(a - a.max())
                    p /= p.sum()
                    o = p @ vv
                    spread = p @ np.abs(vv - o)
                    ds = 2.0 ** -22 * 130 * (np.abs(kk) @ np.abs(qq)).max() / np.sqrt(D)
                    e = ds * spread + 2.0 ** -22 * (len(p) + 8) * (p @ np.abs(vv))
                    if (kv or self.kv) != "f32":  # weights enter a product as f16 terms, whose last step is 2^-24 of the largest weight: at most 2^-25 off, or lost below that
                        e = e + np.minimum(2.0 ** -25, p) @ np.abs(vv)
                    if half:
                        dq = 6 * 2.0 ** -11 / np.sqrt(3) * np.sqrt((kk ** 2) @ (qq ** 2)).max() / np.sqrt(D)
                        if (kv or self.kv) == "q8_0":  # k too, independent of q: the root of two; v: 2^-11 of each, sum p |v| of them at most
                            dq, e = dq * np.sqrt(2), e + 2.0 ** -11 * (p @ np.abs(vv))
                        e = e + (dq + 2.0 ** -11) * spread + 2.0 ** -11 * np.abs(o) + 2.0 ** -24
                    out[t, h], tol[t, h] = o, e
        return out, tol


def norm_rope(x, w, eps, theta, pos):
    """RMS norm and NeoX RoPE of rows x [..., 128] at one position, in 64 bits."""
    x = x.astype(np.float64)
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    a = pos * theta ** (-2.0 * np.arange(64) / 128)
    c, s = np.cos(a), np.sin(a)
    return np.concatenate([y[..., :64] * c - y[..., 64:] * s, y[..., 64:] * c + y[..., :64] * s], -1)


def verify(p, q, drafts, u, starts, tokens, accepted):
    """brasa_k_verify_drafts, id by id; tokens and accepted are written like its buffers."""
    at = 0
    for s in range(len(accepted)):
        first, end = int(starts[s]), int(starts[s + 1])
        accepted[s] = 0
        if end == first:
            continue
        n = end - first - 1
        stop = n
        for i in range(n):
            x = int(drafts[at + i])
            ok = x < p.shape[1] and float(u[first + i]) * (1.0 if q is None else float(q[at + i, x])) < float(p[first + i, x])
            if not ok:
                stop = i
                break
        row = p[first + stop].astype(np.float64)
        mass = row.copy()
        if stop < n:
            if q is not None:
                mass = row - q[at + stop].astype(np.float64)
            elif drafts[at + stop] < p.shape[1]:
                mass[drafts[at + stop]] = 0

        def clean(m):
            return np.where(np.isfinite(m) & (m > 0), m, 0.0)
        mass = clean(mass)
        if mass.sum() == 0:
            mass = clean(row)
        token = 0
        if mass.sum() > 0:
            run = np.cumsum(mass)
            over = np.nonzero((run > float(u[end - 1]) * run[-1]) & (mass > 0))[0]
            token = over[0] if len(over) else np.nonzero(mass > 0)[0][-1]
        accepted[s] = stop
        tokens[first:end] = 0
        tokens[first:first + stop] = drafts[at:at + stop]
        tokens[first + stop] = token
        at += n


def reassign(table, lens, pinned, num_pages, source, keep, room, accepted=None):
    """(table, lens, result, copies) of brasa_k_pages_reassign."""
    R, P = table.shape
    valid = np.where((table >= 0) & (table < num_pages), table, -1)
    new, whole, tails, ends = [], set(), {}, []
    for r in range(R):
        s = int(source[r])
        holds = int(lens[s]) + (0 if accepted is None else int(accepted[s]) + 1) if 0 <= s < R else 0
        k = min(holds if keep is None else int(keep[r]), holds, P * PAGE)
        have = -(-k // PAGE)
        row = list(valid[s][:have]) if have else []
        whole |= {p for p in row[:k // PAGE] if p >= 0}
        if k % PAGE and row[-1] >= 0:
            tails.setdefault(row[-1], r)
        new.append((k, row))
        ends.append(-(-min(k + int(room[r]), P * PAGE) // PAGE))
    pins = {p for p in range(num_pages) if pinned is not None and pinned[p]}
    used = pins | {p for _, row in new for p in row if p >= 0}
    free = [p for p in range(num_pages) if p not in used]
    out, copies, need, handed = np.full((R, P), -1, np.int32), [], 0, iter(free)
    plan = []
    for r, (k, row) in enumerate(new):
        copy = bool(k % PAGE) and row[-1] >= 0 and (row[-1] in whole or row[-1] in pins or tails[row[-1]] != r)
        plan.append(copy)
        need += copy + ends[r] - len(row)
    if need > len(free):
        used = pins | {p for p in valid.flatten() if p >= 0}
        return valid, lens.copy(), [len(used), 0, num_pages - len(used), need - len(free)], []
    for r, (k, row) in enumerate(new):
        if plan[r]:
            to = next(handed)
            copies.append((row[-1], to))
            row = row[:-1] + [to]
        row = row + [next(handed) for _ in range(ends[r] - len(row))]
        out[r, :len(row)] = row
    in_use = len(used) + need
    return out, np.array([k for k, _ in new], np.uint32), [in_use, len(copies), num_pages - in_use, 0], copies


def compact(table, pinned, num_pages):
    """(table, moved, result, moves) of brasa_k_pages_compact."""
    valid = np.where((table >= 0) & (table < num_pages), table, -1)
    pins = {p for p in range(num_pages) if pinned is not None and pinned[p]}
    used = pins | {p for p in valid.flatten() if p >= 0}
    holes, movers = [p for p in range(num_pages) if p not in used], sorted(used - pins, reverse=True)
    moves = [(m, h) for h, m in zip(holes, movers) if h < m]
    to = {p: p for p in used} | dict(moves)
    moved = np.array([to.get(p, -1) for p in range(num_pages)], np.int32)
    return np.where(valid >= 0, moved[np.maximum(valid, 0)], -1).astype(np.int32), moved, [len(used), len(moves), max(to.values(), default=-1) + 1, 0], moves
