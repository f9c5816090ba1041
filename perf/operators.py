"""Cases of the candidate operators: pages of a K/V cache that sequences share (fork, copy, release,
compact), attention over such a cache with a common prefix computed once, and the log
probabilities of given tokens.  `own` selects the plain torch form or the calls of the library."""
import math
import os
import random
import sys

import numpy as np
import torch

own = False
PAGE = 64
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gpt-sovits.cpp_b200")


def _t2sx():
    if PKG not in sys.path:
        sys.path.insert(0, PKG)
    import t2sx
    return t2sx


# ---- the cases -----------------------------------------------------------------------------------

def listed():
    at = dict(op="attend", dtype="f16", heads=16, kv_heads=16, dim=32, new=1)
    pg = dict(dtype="f16", layers=24, kv_heads=16, dim=32)
    lp = dict(op="logprobs", dtype="f32")
    return [
        # one layer of one decode step of four candidates drawn from one 350-position prompt: latency
        dict(at, name="attend 4 of one prompt", prompts=1, each=4, prefix=350, tail=60),
        # a full serving batch of the decode workload: 2048 ragged sequences, 32 to a prompt
        dict(at, name="attend 2048, 32 a prompt", prompts=64, each=32, prefix=350, tail=1000),
        # many candidates of one long prompt, grouped heads: the shared part is matrix work
        dict(at, name="attend 256 of one long prompt", dtype="bf16", heads=32, kv_heads=8, dim=128,
             prompts=1, each=256, prefix=16384, tail=256),
        # one token against one very long sequence: the long axis has to be split
        dict(at, name="attend one long sequence", dtype="bf16", heads=32, kv_heads=8, dim=128,
             prompts=1, each=1, prefix=65531, tail=37),
        # a prompt's rows taken in a chunk over what is cached (odd counts, causal inside the chunk)
        dict(at, name="attend chunk of 509", heads=16, kv_heads=4, dim=64, prompts=4, each=1, prefix=1000,
             tail=509, new=509),
        # one prompt to four candidates, the model's 24 layers: latency
        dict(pg, op="fork", name="fork 1 to 4", prompts=1, each=4, length=350),
        # a batch of prompts to 16 candidates each
        dict(pg, op="fork", name="fork 32 to 512", prompts=32, each=16, length=350),
        # finished sequences leave holes: every second one is rewritten elsewhere, released, the pool compacted
        dict(op="compact", name="compact half of 64", dtype="bf16", layers=8, kv_heads=8, dim=128, seqs=64, length=1350),
        # the scores of one step of eight candidates (the model's 1025 tokens)
        dict(lp, name="logprobs 8 x 1025", rows=8, vocab=1025, top=5),
        # the scores of a full batch's step
        dict(lp, name="logprobs 2048 x 1025", rows=2048, vocab=1025, top=15),
        # a wide vocabulary of odd size, rows off the 16-byte grid
        dict(lp, name="logprobs 2048 x 100003", dtype="bf16", rows=2048, vocab=100003, top=20),
        # few rows of a wide vocabulary: each row has to be shared out
        dict(lp, name="logprobs 4 x 131072", dtype="f16", rows=4, vocab=131072, top=20),
    ]


def _spread(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


MOST_BYTES, MOST_FLOPS = 4.0e9, 7.0e10


def draw(rng):
    while True:
        op = rng.choice(["attend", "attend", "attend", "fork", "compact", "logprobs", "logprobs"])
        if op == "attend":
            kv, group, dim = rng.choice([(16, 1, 32), (4, 4, 64), (8, 4, 128), (1, 8, 64), (2, 7, 128), (8, 1, 64), (3, 2, 32)])
            case = dict(op=op, dtype=rng.choice(["f16", "bf16"]), heads=kv * group, kv_heads=kv, dim=dim,
                        prompts=_spread(rng, 1, 64), each=_spread(rng, 1, 256), prefix=_spread(rng, 1, 65536),
                        tail=_spread(rng, 1, 1000), new=1)
            if rng.random() < 0.25:
                case["new"] = _spread(rng, 2, 600)
                case["each"] = _spread(rng, 1, 8)
                case["tail"] = max(case["tail"], case["new"])
        elif op == "fork":
            case = dict(op=op, dtype=rng.choice(["f16", "bf16"]), layers=rng.randint(1, 24), kv_heads=rng.choice([1, 4, 8, 16]),
                        dim=rng.choice([32, 64, 128]), prompts=_spread(rng, 1, 64), each=_spread(rng, 1, 32),
                        length=_spread(rng, 1, 2000))
        elif op == "compact":
            case = dict(op=op, dtype=rng.choice(["f16", "bf16"]), layers=rng.randint(1, 24), kv_heads=rng.choice([1, 4, 8, 16]),
                        dim=rng.choice([32, 64, 128]), seqs=_spread(rng, 2, 256), length=_spread(rng, 3, 2000))
        else:
            case = dict(op=op, dtype=rng.choice(["f32", "f16", "bf16"]), rows=_spread(rng, 1, 4096),
                        vocab=_spread(rng, 33, 140000), top=rng.randint(0, 32))
        w = work(case)
        if 0 < w["bytes"] <= MOST_BYTES and w["flops"] <= MOST_FLOPS and _held(case) <= 6.0e9:
            return case


# ---- sizes that follow from a case ------------------------------------------------------------------

def _lengths(case):
    """Ragged lengths, a function of the case alone: of prompts and of what each sequence adds, or of the sequences."""
    r = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    if case["op"] == "attend":
        n = case["prompts"]
        prefix = [case["prefix"]] + [r.randint((case["prefix"] + 1) // 2, case["prefix"]) for _ in range(n - 1)]
        tails = [r.randint(case["new"], case["tail"]) for _ in range(n * case["each"])]
        tails[0] = case["tail"]
        return prefix, tails
    if case["op"] == "fork":
        n = case["prompts"]
        return [case["length"]] + [r.randint((case["length"] + 1) // 2, case["length"]) for _ in range(n - 1)]
    n = case["seqs"]
    return [case["length"]] + [r.randint(max(1, case["length"] // 4), case["length"]) for _ in range(n - 1)]


def _pages(length):
    return -(-length // PAGE)


def _n_pages(case):
    """Pages of the pool: what the sequences need at most at one time."""
    if case["op"] == "attend":
        prefix, tails = _lengths(case)
        e = case["each"]
        if e == 1:
            return sum(_pages(p + t) for p, t in zip(prefix, tails))
        return sum(_pages(p) + sum(_pages(p % PAGE + t) for t in tails[i * e:(i + 1) * e]) for i, p in enumerate(prefix))
    lens = _lengths(case)
    if case["op"] == "fork":
        return sum(_pages(n) + (case["each"] if n % PAGE else 0) for n in lens)
    return sum(_pages(n) for n in lens) + sum(_pages(n) for n in lens[1::2])


def _held(case):
    """Bytes of a state."""
    if case["op"] == "logprobs":
        return case["rows"] * case["vocab"] * (4 if case["dtype"] == "f32" else 2)
    return _n_pages(case) * case.get("layers", 1) * 2 * case["kv_heads"] * PAGE * case["dim"] * 2


def work(case):
    if case["op"] == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (4 if case["dtype"] == "f32" else 2) + case["rows"] * (4 * 4 + 8 * case["top"]), "flops": 6 * n}
    pos = case.get("layers", 1) * 2 * case["kv_heads"] * case["dim"] * 2   # bytes of a position's K and V
    lens = _lengths(case)
    if case["op"] == "fork":
        return {"bytes": sum(n % PAGE for n in lens) * (1 + case["each"]) * pos, "flops": 0}
    if case["op"] == "compact":
        # the sequences written anew, then moved: both read and write each position once
        return {"bytes": 4 * sum(lens[1::2]) * pos, "flops": 0}
    prefix, tails = lens
    new, e, rows = case["new"], case["each"], len(tails) * case["new"]
    held = sum(prefix) + sum(tails)
    # a row sees the positions up to its own
    seen = sum(new * (prefix[i // e] + t) - new * (new - 1) // 2 for i, t in enumerate(tails))
    return {"bytes": held * pos + rows * (2 * case["heads"] * case["dim"] * 2 + case["heads"] * 4 + pos),
            "flops": 4 * case["dim"] * case["heads"] * seen}


# ---- page bookkeeping of the plain form: lowest free page first, pages counted by their users --------

class Pages:
    def __init__(self, n_pages):
        self.users = np.zeros(n_pages, dtype=np.int64)
        self.tables, self.lens = {}, {}

    def _take(self, n):
        ids = np.flatnonzero(self.users == 0)[:n]
        self.users[ids] += 1
        return ids

    def extend(self, seq, count):
        had = self.tables.get(seq, np.zeros(0, dtype=np.int64))
        self.lens[seq] = self.lens.get(seq, 0) + count
        self.tables[seq] = np.concatenate([had, self._take(_pages(self.lens[seq]) - len(had))])

    def share(self, src, dst, full):
        """dst := src with its first `full` pages shared and the others its own; (from, to) of the own ones."""
        table = self.tables[src]
        self.users[table[:full]] += 1
        mine = self._take(len(table) - full)
        self.tables[dst], self.lens[dst] = np.concatenate([table[:full], mine]), self.lens[src]
        return table[full:], mine

    def release(self, seqs):
        for s in seqs:
            self.users[self.tables.pop(s)] -= 1
            del self.lens[s]

    def fills(self, seq):
        return np.minimum(PAGE, self.lens[seq] - PAGE * np.arange(len(self.tables[seq])))

    def compact(self):
        """(from, to, filled positions) of the pages that move."""
        live = np.flatnonzero(self.users)
        n = len(live)
        src, dst = live[live >= n], np.flatnonzero(self.users[:n] == 0)
        to = np.arange(len(self.users))
        to[src] = dst
        fill = np.zeros(len(self.users), dtype=np.int64)
        for s, t in self.tables.items():
            fill[t] = self.fills(s)
            self.tables[s] = to[t]
        self.users[dst] = self.users[src]
        self.users[src] = 0
        return src, dst, fill[src]

    def table(self, seqs):
        got = np.full((len(seqs), max(len(self.tables[s]) for s in seqs)), -1, dtype=np.int32)
        for i, s in enumerate(seqs):
            got[i, :len(self.tables[s])] = self.tables[s]
        return got


# ---- inputs ------------------------------------------------------------------------------------------

def _store(case):
    shape = (case.get("layers", 1), _n_pages(case), case["kv_heads"], PAGE, case["dim"])
    return (torch.empty(shape, dtype=DTYPES[case["dtype"]], device="cuda"),
            torch.empty(shape, dtype=DTYPES[case["dtype"]], device="cuda"))


def _inputs(case, seed, k=None, v=None):
    """The tensors of a case, from the seed alone; the cache's values go into k and v."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    if case["op"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        x = torch.randn((rows, vocab), generator=gen, device="cuda").mul_(2.5)
        x[:, vocab - 1] = float("-inf")   # the end token is masked, as in a decode of a fixed number of steps
        tokens = torch.randint(0, vocab, (rows,), generator=gen, device="cuda", dtype=torch.int32)
        x[torch.arange(rows, device="cuda"), tokens.long()] += 6.0   # drawn tokens are likely ones
        return dict(x=x.to(dt), tokens=tokens)
    k.normal_(generator=gen)
    v.normal_(generator=gen)
    got = dict(k=k, v=v)
    if case["op"] == "attend":
        rows = case["prompts"] * case["each"] * case["new"]
        for name, heads, size in (("q", case["heads"], 1.5), ("k_new", case["kv_heads"], 1.0), ("v_new", case["kv_heads"], 1.0)):
            got[name] = torch.randn((rows, heads, case["dim"]), generator=gen, device="cuda").mul_(size).to(dt)
    return got


def _build(case, pages):
    """Makes the case's sequences in the plain bookkeeping (no data moves: the storage is filled afterwards);
    the ids that take part."""
    lens = _lengths(case)
    if case["op"] != "attend":
        for i, n in enumerate(lens):
            pages.extend(i, n)
        return list(range(len(lens)))
    prefix, tails = lens
    n, e = case["prompts"], case["each"]
    if e == 1:
        for i in range(n):
            pages.extend(i, prefix[i] + tails[i])
        return list(range(n))
    for i in range(n):
        pages.extend(i, prefix[i])
    for i in range(n * e):
        pages.share(i // e, n + i, prefix[i // e] // PAGE)
        pages.extend(n + i, tails[i])
    return list(range(n, n + n * e))


def _build_own(case, k, v):
    """The same sequences in the library's pool over the storage k, v."""
    t2sx = _t2sx()
    most = 2 * case["seqs"] if case["op"] == "compact" else case["prompts"] * (1 + case["each"])
    pool = t2sx.PagePool(t2sx.F16 if case["dtype"] == "f16" else t2sx.BF16, k.shape[0], k.shape[1], case["kv_heads"],
                         case["dim"], most, k.data_ptr(), v.data_ptr())
    lens = _lengths(case)
    if case["op"] != "attend":
        pool.extend(list(range(len(lens))), lens)
        return pool, list(range(len(lens)))
    prefix, tails = lens
    n, e = case["prompts"], case["each"]
    if e == 1:
        pool.extend(list(range(n)), [p + t for p, t in zip(prefix, tails)])
        return pool, list(range(n))
    pool.extend(list(range(n)), prefix)
    for i in range(n * e):
        pool.fork([i // e], [n + i], _stream())
        pool.extend([n + i], [tails[i]])
    return pool, list(range(n, n + n * e))


def _stream():
    return torch.cuda.current_stream().cuda_stream


def prepare(case, seed):
    s = dict(case)
    if case["op"] == "logprobs":
        s.update(_inputs(case, seed))
        rows, top = case["rows"], case["top"]
        s["logprob"], s["entropy"] = (torch.empty(rows, dtype=torch.float32, device="cuda") for _ in range(2))
        s["rank"] = torch.empty(rows, dtype=torch.int32, device="cuda")
        s["ids"] = torch.empty((rows, top), dtype=torch.int32, device="cuda")
        s["values"] = torch.empty((rows, top), dtype=torch.float32, device="cuda")
        return s
    k, v = _store(case)
    if own:
        s["pool"], seqs = _build_own(case, k, v)
    else:
        s["pages"] = Pages(k.shape[1])
        seqs = _build(case, s["pages"])
    s.update(_inputs(case, seed, k, v))
    if case["op"] == "attend":
        s["scale"] = 1.0 / math.sqrt(case["dim"])
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(s["q"].shape[:2], dtype=torch.float32, device="cuda")
        if own:
            # a step's plan serves the calls of all its layers
            s["plan"] = s["pool"].plan(case["heads"])
            s["plan"].update(seqs, [case["new"]] * len(seqs), _stream())
        else:
            s.update(_plain_plan(case, s["pages"], seqs))
    if case["op"] == "fork":
        n, e = case["prompts"], case["each"]
        s["src"], s["dst"] = [i // e for i in range(n * e)], list(range(n, n + n * e))
    if case["op"] == "compact":
        # the sequences that are rewritten, and the ids that they are rewritten to
        s["all"], s["from"], s["to"] = seqs, seqs[1::2], [i + case["seqs"] for i in seqs[1::2]]
    return s


def _plain_plan(case, pages, seqs):
    """Index tensors: the pages that a prompt's candidates share, each sequence's other pages, where the new rows go."""
    prefix, _ = _lengths(case)
    e, new = case["each"], case["new"]
    full = np.array([p // PAGE if e > 1 else 0 for p in prefix])
    tables = [pages.tables[q] for q in seqs]
    lens = np.array([pages.lens[q] for q in seqs])
    shared = np.zeros((len(prefix), full.max()), dtype=np.int64)
    rest = np.zeros((len(seqs), max(len(t) - full[i // e] for i, t in enumerate(tables))), dtype=np.int64)
    for i, n in enumerate(full):
        shared[i, :n] = tables[i * e][:n]
    for i, t in enumerate(tables):
        rest[i, :len(t) - full[i // e]] = t[full[i // e]:]
    limit = lens[:, None] - new + 1 + np.arange(new)[None, :]     # positions that a row sees
    at = limit - 1                                                # its own
    page = np.stack([t[a // PAGE] for t, a in zip(tables, at)])
    start = full.repeat(e) * PAGE
    got = dict(shared=shared, rest=rest, shared_len=full * PAGE, limit=limit - start[:, None], page=page.reshape(-1),
               at=(at % PAGE).reshape(-1))
    return {name: torch.as_tensor(a, device="cuda") for name, a in got.items()}


# ---- one pass ----------------------------------------------------------------------------------------

def _cache(s):
    """The cache as it stands, its values as the bits they are: they move, and nothing rounds them."""
    return {"k": s["k"].view(torch.int16), "v": s["v"].view(torch.int16)}


def run(state):
    return {"attend": _attend, "fork": _fork, "compact": _compact, "logprobs": _logprobs}[state["op"]](state)


def _attend(s):
    if own:
        s["plan"].attend(0, s["q"].data_ptr(), s["out"].data_ptr(), s["scale"], k_new_ptr=s["k_new"].data_ptr(),
                         v_new_ptr=s["v_new"].data_ptr(), lse_ptr=s["lse"].data_ptr(), stream=_stream())
        return {"out": s["out"], "lse": s["lse"], **_cache(s)}
    n, e, new, kv, dim = s["prompts"], s["each"], s["new"], s["kv_heads"], s["dim"]
    k, v = s["k"][0], s["v"][0]
    k[s["page"], :, s["at"]] = s["k_new"]
    v[s["page"], :, s["at"]] = s["v_new"]
    q = s["q"].float().view(n, e, new, kv, -1, dim).permute(0, 3, 1, 2, 4, 5) * s["scale"]   # prompt, kv head, seq, token, group, dim
    dev, shape = q.device, q.shape

    def dense(store, table):
        return store[table].float().transpose(1, 2).flatten(2, 3)   # [tables, kv head, position, dim]

    k2, v2 = (dense(x, s["rest"]).unflatten(0, (n, e)).transpose(1, 2) for x in (k, v))   # prompt, kv head, seq, position, dim
    s2 = (q.flatten(3, 4) @ k2.transpose(-1, -2)).view(*shape[:-1], -1)
    unseen = torch.arange(s2.shape[-1], device=dev) >= s["limit"].view(n, 1, e, new, 1, 1)
    s2 = s2.masked_fill_(unseen, float("-inf"))
    m = s2.amax(-1, keepdim=True)
    if s["shared"].shape[1]:
        k1, v1 = (dense(x, s["shared"]) for x in (k, v))   # prompt, kv head, position, dim
        s1 = (q.flatten(2, 4) @ k1.transpose(-1, -2)).view(*shape[:-1], -1)
        s1 = s1.masked_fill_(torch.arange(s1.shape[-1], device=dev) >= s["shared_len"].view(n, 1, 1, 1, 1, 1), float("-inf"))
        m = torch.maximum(m, s1.amax(-1, keepdim=True))
        p1 = s1.sub_(m).exp_()
    p2 = s2.sub_(m).exp_()
    l = p2.sum(-1, keepdim=True)
    o = (p2.flatten(3, 4) @ v2).view(shape)
    if s["shared"].shape[1]:
        l = l + p1.sum(-1, keepdim=True)
        o = o + (p1.flatten(2, 4) @ v1).view(shape)
    out = (o / l).permute(0, 2, 3, 1, 4, 5).reshape(s["q"].shape).to(s["q"].dtype)
    lse = (m + l.log()).permute(0, 2, 3, 1, 4, 5).reshape(s["q"].shape[:2])
    return {"out": out, "lse": lse, **_cache(s)}


def _move(store, src, dst, fill):
    """The first fill[i] positions of page src[i] of every layer and head into page dst[i]."""
    src, dst, fill = (torch.as_tensor(np.ascontiguousarray(a), device=store.device) for a in (src, dst, fill))
    keep = torch.arange(PAGE, device=store.device)[None, :] < fill[:, None]
    store[:, dst] = torch.where(keep[None, :, None, :, None], store[:, src], store[:, dst])


def _fork(s):
    if own:
        pool = s["pool"]
        pool.fork(s["src"], s["dst"], _stream())
        table = pool.table(s["dst"])
        pool.release(s["dst"])
        return {"table": table, **_cache(s)}
    pages = s["pages"]
    moves = [pages.share(a, b, pages.lens[a] // PAGE) for a, b in zip(s["src"], s["dst"])]
    src, dst = (np.concatenate(x) for x in zip(*moves))
    fill = np.concatenate([pages.fills(b)[pages.lens[b] // PAGE:] for b in s["dst"]])
    for store in (s["k"], s["v"]):
        _move(store, src, dst, fill)
    table = pages.table(s["dst"])
    pages.release(s["dst"])
    return {"table": table, **_cache(s)}


def _compact(s):
    """Every second sequence is copied to pages of its own, released, and the pool compacted; its new id is the
    next pass's old one, and pages, tables and values end where they were."""
    live = s["all"][:]
    live[1::2] = s["to"]
    if own:
        pool = s["pool"]
        pool.copy(s["from"], s["to"], _stream())
        pool.release(s["from"])
        pool.compact(_stream())
        table = pool.table(live)
    else:
        pages = s["pages"]
        moves = [pages.share(a, b, 0) for a, b in zip(s["from"], s["to"])]
        src, dst = (np.concatenate(x) for x in zip(*moves))
        fill = np.concatenate([pages.fills(b) for b in s["to"]])
        for store in (s["k"], s["v"]):
            _move(store, src, dst, fill)
        pages.release(s["from"])
        src, dst, fill = pages.compact()
        for store in (s["k"], s["v"]):
            _move(store, src, dst, fill)
        table = pages.table(live)
    s["from"], s["to"] = s["to"], s["from"]
    return {"table": table, **_cache(s)}


def _logprobs(s):
    x, tokens, top = s["x"], s["tokens"], s["top"]
    if own:
        t2sx = _t2sx()
        t2sx.token_logprobs({"f32": t2sx.F32, "f16": t2sx.F16, "bf16": t2sx.BF16}[s["dtype"]], s["rows"], s["vocab"],
                            x.data_ptr(), tokens.data_ptr(), s["logprob"].data_ptr(), entropy_ptr=s["entropy"].data_ptr(),
                            rank_ptr=s["rank"].data_ptr(), top_k=top, top_ids_ptr=s["ids"].data_ptr(),
                            top_logprobs_ptr=s["values"].data_ptr(), stream=_stream())
        return {name: s[name] for name in ("logprob", "entropy", "rank", "ids", "values")}
    x = x.float()
    m = x.amax(-1, keepdim=True)
    d = x - m
    p = d.exp()
    z = p.sum(-1, keepdim=True)
    lse = m + z.log()
    t = tokens.long()[:, None]
    xt = x.gather(1, t)
    entropy = z.log()[:, 0] - torch.where(p > 0, p * d, 0.0).sum(-1) / z[:, 0]
    before = torch.arange(x.shape[1], device=x.device) < t
    rank = ((x > xt) | ((x == xt) & before)).sum(-1).to(torch.int32)
    ids = _top(x, top)
    return {"logprob": (xt - lse)[:, 0], "entropy": entropy, "rank": rank, "ids": ids.to(torch.int32),
            "values": x.gather(1, ids) - lse}


def _top(x, k):
    """Indices of the k largest of each row, ties to the lowest index: the sort's key has the value's bits in an
    order that integers keep, above the index."""
    bits = (x + 0.0).view(torch.int32)   # one zero
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    key = (key << 32) | (0xFFFFFFFF - torch.arange(x.shape[1], device=x.device))
    return 0xFFFFFFFF - (key.topk(k, dim=1).values & 0xFFFFFFFF)


# ---- the definition, in 64 bits ------------------------------------------------------------------------

def exact(case, seed):
    if case["op"] == "logprobs":
        s = _inputs(case, seed)
        got = dict(logprob=[], entropy=[], values=[])
        for x, t in zip(s["x"].split(256), s["tokens"].split(256)):
            lp = x.double().log_softmax(-1)
            got["logprob"].append(lp[torch.arange(len(t), device=lp.device), t.long()])
            got["entropy"].append(-torch.special.xlogy(lp.exp(), lp.exp()).sum(-1))
            got["values"].append(lp.topk(case["top"], dim=1).values)
        return dict({name: torch.cat(x) for name, x in got.items()}, rank=None, ids=None)
    if case["op"] != "attend":
        return None   # nothing is computed: values move
    pages = Pages(_n_pages(case))
    seqs = _build(case, pages)
    k, v = _store(case)
    s = _inputs(case, seed, k, v)
    new, kv, dim = case["new"], case["kv_heads"], case["dim"]
    outs, lses = [], []
    for i, q in enumerate(s["q"].split(new)):
        table, n = torch.as_tensor(pages.tables[seqs[i]], device="cuda"), pages.lens[seqs[i]]
        # the sequence's keys and values in order of position, the new rows last
        kk, vv = (torch.cat([x[0][table].movedim(1, 2).reshape(-1, kv, dim)[:n - new], y[i * new:(i + 1) * new]]).double().movedim(0, 1)
                  for x, y in ((k, s["k_new"]), (v, s["v_new"])))
        a = torch.einsum("nhgd,hld->hgnl", q.double().unflatten(1, (kv, -1)), kk) / math.sqrt(dim)
        if new > 1:
            a += torch.full((new, n), float("-inf"), device="cuda", dtype=torch.float64).triu_(n - new + 1)
        lse = a.logsumexp(-1)
        outs.append(torch.einsum("hgnl,hld->nhgd", (a - lse[..., None]).exp_(), vv).flatten(1, 2))
        lses.append(lse.permute(2, 0, 1).flatten(1, 2))
    return {"out": torch.cat(outs), "lse": torch.cat(lses), "k": None, "v": None}
