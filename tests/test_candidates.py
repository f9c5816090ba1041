"""Shared cache pages, attention over them and token log probabilities, against plain 64-bit forms.

Tolerances (u = half a unit in the last place of the 16-bit type: 2^-11 for f16, 2^-8 for bf16):
attention: with a = sum_j p_j |v_j|, rounding the softmax weights moves an output by at most u a and rounding
the output by u |out|; a score of up to 128 products accumulated in f32, its exponential, and sums
of up to 2^17 terms in f32 parts leave less than 2^-14 a.  Absolute log-sum-exp error: 2^-14 likewise.
Log probabilities: sums of f32 terms in blocks, 2^-17 of the values' scale (the largest |x - max|, at
least 1).  Ids, ranks, tables and moved values are equal."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu
PAGE = 64
TORCH = {1: torch.float16, 30: torch.bfloat16, 0: torch.float32}
UNIT = {1: 2.0 ** -11, 30: 2.0 ** -8}


def _need_gpu():
    if not torch.cuda.is_available():
        pytest.fail("CUDA device required for -m gpu tests")


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _store(dtype, layers, pages, kv, dim, fill=float("nan")):
    shape = (layers, pages, kv, PAGE, dim)
    return [torch.full(shape, fill, dtype=TORCH[dtype], device="cuda") for _ in range(2)]


class Cache:
    """A pool, its storage, and for each sequence what its positions must hold ([layers][len][kv][dim], K and V)."""

    def __init__(self, t2sx, dtype, layers, pages, kv, dim, seqs, seed=0):
        self.k, self.v = _store(dtype, layers, pages, kv, dim)
        self.pool = t2sx.PagePool(dtype, layers, pages, kv, dim, seqs, self.k.data_ptr(), self.v.data_ptr())
        self.gen = torch.Generator(device="cuda").manual_seed(seed)
        self.want = {s: [torch.empty((layers, 0, kv, dim), dtype=TORCH[dtype], device="cuda")] * 2 for s in range(seqs)}

    def at(self, seq):
        pages = torch.as_tensor(self.pool.table([seq])[0], device="cuda").long()
        n = self.pool.length(seq)
        return [x[:, pages].movedim(2, 3).flatten(1, 2)[:, :n] for x in (self.k, self.v)]

    def extend(self, seq, count, write=True):
        had = self.pool.length(seq)
        self.pool.extend([seq], [count])
        table = torch.as_tensor(self.pool.table([seq])[0], device="cuda").long()
        pos = torch.arange(had, had + count, device="cuda")
        for i, x in enumerate((self.k, self.v)):
            rows = torch.randn((x.shape[0], count, x.shape[2], x.shape[4]), generator=self.gen, device="cuda").to(x.dtype)
            if write and count:
                x[:, table[pos // PAGE], :, pos % PAGE] = rows.movedim(1, 0)
            self.want[seq] = self.want[seq][:i] + [torch.cat([self.want[seq][i], rows], 1)] + self.want[seq][i + 1:]

    def derive(self, op, srcs, dsts):
        getattr(self.pool, op)(srcs, dsts, _stream())
        for a, b in zip(srcs, dsts):
            self.want[b] = list(self.want[a])

    def release(self, seqs):
        self.pool.release(seqs)
        for s in seqs:
            self.want[s] = [x[:, :0] for x in self.want[s]]

    def check(self):
        users = {}
        for s, want in self.want.items():
            assert self.pool.length(s) == want[0].shape[1]
            for got, x in zip(self.at(s), want):
                assert torch.equal(got.view(torch.int16), x.contiguous().view(torch.int16)), s
            for j, page in enumerate(self.pool.table([s])[0]):
                users.setdefault(int(page), set()).add((s, j))
        assert self.pool.available() == self.pool.n_pages - len(users)
        for held in users.values():   # shared pages are full in each of their sequences
            if len(held) > 1:
                assert all((j + 1) * PAGE <= self.pool.length(s) for s, j in held)
        return set(users)


# ---- pages ---------------------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("dtype,layers,kv,dim", [(1, 3, 2, 32), (30, 1, 1, 128), (1, 2, 5, 64)])
def test_pool_random_life(t2sx_mod, dtype, layers, kv, dim):
    """Random extend, fork, copy, release and compact calls against the values that sequences must hold."""
    _need_gpu()
    rng = np.random.default_rng(dim + layers)
    c = Cache(t2sx_mod, dtype, layers, 120, kv, dim, 12)
    for step in range(160):
        live = [s for s in c.want if c.pool.length(s)]
        free = [s for s in c.want if not c.pool.length(s)]
        op = rng.choice(["extend", "fork", "copy", "release", "compact"], p=[0.35, 0.25, 0.1, 0.2, 0.1])
        try:
            if op == "extend":
                c.extend(int(rng.choice(12)), int(rng.choice([0, 1, 5, 63, 64, 65, 200])))
            elif op in ("fork", "copy") and live and free:
                n = int(rng.integers(1, len(free) + 1))
                c.derive(op, rng.choice(live, n).tolist(), rng.choice(free, n, replace=False).tolist())
            elif op == "release" and live:
                c.release(rng.choice(live, int(rng.integers(1, len(live) + 1)), replace=False).tolist())
            elif op == "compact":
                before = c.check()
                moved = c.pool.compact(_stream())
                assert moved == sum(p >= len(before) for p in before)
                assert c.check() == set(range(len(before)))
        except t2sx_mod.T2SXError as e:
            assert e.code == t2sx_mod.ERR_OOM
        c.check()


@gpu
def test_pool_lowest_free_page_first(t2sx_mod):
    _need_gpu()
    c = Cache(t2sx_mod, 1, 1, 70, 1, 32, 6)
    c.pool.extend([0, 1, 2], [130, 1, 64])
    assert c.pool.table([0, 1, 2]).tolist() == [[0, 1, 2], [3, -1, -1], [4, -1, -1]]
    c.pool.fork([0], [3], _stream())
    assert c.pool.table([3]).tolist() == [[0, 1, 5]]
    c.pool.release([0, 1])
    c.pool.extend([4], [66 * PAGE])   # 64 pages are free above, and 2 and 3
    assert c.pool.table([4])[0].tolist() == [2, 3] + list(range(6, 70))
    assert c.pool.available() == 0
    with pytest.raises(t2sx_mod.T2SXError) as e:
        c.pool.extend([1], [1])
    assert e.value.code == t2sx_mod.ERR_OOM and c.pool.length(1) == 0


@gpu
def test_pool_many_moves(t2sx_mod):
    """More page copies than one launch's list holds."""
    _need_gpu()
    n = 700
    c = Cache(t2sx_mod, 1, 1, n + 2, 1, 32, n + 1)
    c.extend(0, 70)
    c.derive("fork", [0] * n, list(range(1, n + 1)))
    c.check()
    c.release(list(range(0, n, 2)))
    assert c.pool.compact(_stream()) > 0
    c.check()


@gpu
def test_pool_refusals(t2sx_mod):
    _need_gpu()
    k, v = _store(1, 1, 8, 1, 32)
    make = lambda **kw: t2sx_mod.PagePool(*[{**dict(dtype=1, layers=1, pages=8, kv=1, dim=32, seqs=4, k=k.data_ptr(), v=v.data_ptr()), **kw}[n]
                                            for n in ("dtype", "layers", "pages", "kv", "dim", "seqs", "k", "v")])
    for kw in (dict(dtype=0), dict(layers=0), dict(pages=0), dict(kv=0), dict(dim=48), dict(seqs=0), dict(k=0),
               dict(k=k.data_ptr() + 2), dict(pages=(1 << 26) + 1)):
        with pytest.raises(t2sx_mod.T2SXError) as e:
            make(**kw)
        assert e.value.code == t2sx_mod.ERR_INVALID, kw
    pool = make()
    pool.extend([0], [65])
    for call, code in ((lambda: pool.fork([0], [0]), t2sx_mod.ERR_STATE), (lambda: pool.fork([0, 0], [1, 1]), t2sx_mod.ERR_INVALID),
                       (lambda: pool.fork([4], [1]), t2sx_mod.ERR_INVALID), (lambda: pool.copy([0], [-1]), t2sx_mod.ERR_INVALID),
                       (lambda: pool.extend([1, 1], [1, 1]), t2sx_mod.ERR_INVALID), (lambda: pool.extend([1], [-1]), t2sx_mod.ERR_INVALID),
                       (lambda: pool.extend([1], [1 << 40]), t2sx_mod.ERR_INVALID), (lambda: pool.release([9]), t2sx_mod.ERR_INVALID),
                       (lambda: pool.length(4), t2sx_mod.ERR_INVALID), (lambda: pool.plan(0), t2sx_mod.ERR_INVALID),
                       (lambda: pool.copy([0, 0, 0, 0], [1, 2, 3, 3]), t2sx_mod.ERR_INVALID),
                       (lambda: pool.extend([1], [7 * 64]), t2sx_mod.ERR_OOM)):
        with pytest.raises(t2sx_mod.T2SXError) as e:
            call()
        assert e.value.code == code
    assert pool.available() == 6 and pool.length(0) == 65
    plan = pool.plan(3)
    for seqs, new in (([0], [66]), ([0, 0], [1, 1]), ([7], [1]), ([0], [-1]), ([1], [1])):
        with pytest.raises(t2sx_mod.T2SXError) as e:
            plan.update(seqs, new)
        assert e.value.code == t2sx_mod.ERR_INVALID
    x = torch.zeros((1, 3, 32), dtype=torch.float16, device="cuda")
    with pytest.raises(t2sx_mod.T2SXError) as e:
        plan.attend(0, x.data_ptr(), x.data_ptr(), 1.0)
    assert e.value.code == t2sx_mod.ERR_STATE
    plan.update([0], [1], _stream())
    for kw in (dict(layer=1), dict(layer=-1), dict(q_ptr=None), dict(q_ptr=x.data_ptr() + 2), dict(q_stride=88), dict(q_stride=100),
               dict(k_new_ptr=x.data_ptr()), dict(scale=float("nan")), dict(out_ptr=None), dict(lse_ptr=x.data_ptr() + 2)):
        with pytest.raises(t2sx_mod.T2SXError) as e:
            plan.attend(**{**dict(layer=0, q_ptr=x.data_ptr(), out_ptr=x.data_ptr(), scale=1.0), **kw})
        assert e.value.code == t2sx_mod.ERR_INVALID, kw
    pool.extend([1], [1])
    pool.release([1])
    with pytest.raises(t2sx_mod.T2SXError) as e:
        plan.attend(0, x.data_ptr(), x.data_ptr(), 1.0)
    assert e.value.code == t2sx_mod.ERR_STATE
    with pytest.raises(t2sx_mod.T2SXError):
        pool.plan(1 << 20)
    torch.cuda.synchronize()


def test_refusals_without_device(t2sx_mod):
    """Arguments are checked before any device work."""
    import ctypes as C
    L, h, one = t2sx_mod.lib(), C.c_void_p(), 4096
    assert L.t2sx_pool_create(0, 2, 1, 1, 1, 32, 1, one, one, C.byref(h)) == t2sx_mod.ERR_INVALID and not h.value
    assert b"f16 or bf16" in L.t2sx_last_error()
    assert L.t2sx_pool_create(0, 1, 1, 1, 1, 32, 1, one, one, None) == t2sx_mod.ERR_INVALID
    assert L.t2sx_plan_create(None, 1, C.byref(h)) == t2sx_mod.ERR_INVALID
    assert L.t2sx_pool_fork(None, 0, None, None, None) == t2sx_mod.ERR_INVALID
    assert L.t2sx_pool_length(None, 0) == -1
    assert L.t2sx_plan_attend(None, 0, one, 32, None, None, 0, 1.0, one, 32, None, None) == t2sx_mod.ERR_INVALID
    L.t2sx_pool_free(None)
    L.t2sx_plan_free(None)
    bad = lambda **kw: L.t2sx_token_logprobs(*{**dict(dev=0, type=0, rows=1, vocab=8, x=one, stride=8, t=one, k=2, lp=one, h=None, r=None,
                                                      ids=one, top=one, st=None), **kw}.values())
    for kw in (dict(type=2), dict(rows=-1), dict(vocab=0), dict(stride=7), dict(k=33), dict(k=-1), dict(x=None), dict(t=None), dict(lp=None),
               dict(ids=None), dict(top=None), dict(x=one + 2), dict(type=1, x=one + 1), dict(h=one + 2)):
        assert bad(**kw) == t2sx_mod.ERR_INVALID, kw
    assert bad(rows=0) == t2sx_mod.OK


# ---- attention -----------------------------------------------------------------------------------------

def _reference(c, layer, seqs, n_new, q, heads, scale):
    """out, sum p |v| and log-sum-exp in 64 bits, from what the sequences must hold."""
    kv = c.k.shape[2]
    out, mag, lse, at = [], [], [], 0
    for s, n in zip(seqs, n_new):
        k, v = (x[layer].double().repeat_interleave(heads // kv, 1) for x in c.want[s])
        a = torch.einsum("nhd,lhd->hnl", q[at:at + n].double(), k) * scale
        length = k.shape[0]
        pos = torch.arange(length, device="cuda")[None] > torch.arange(length - n, length, device="cuda")[:, None]
        a = a.masked_fill(pos[None], float("-inf"))
        z = a.logsumexp(-1, keepdim=True)
        p = (a - z).exp()
        out.append(torch.einsum("hnl,lhd->nhd", p, v))
        mag.append(torch.einsum("hnl,lhd->nhd", p, v.abs()))
        lse.append(z[..., 0].T)
        at += n
    return torch.cat(out), torch.cat(mag), torch.cat(lse)


def _attend(c, dtype, layer, seqs, n_new, heads, scale=None, q_scale=1.5, write=False, pad=0, seed=1):
    """attend() against the reference; write: the rows' keys and values are passed to the call."""
    kv, dim = c.k.shape[2], c.k.shape[4]
    scale = 1.0 / math.sqrt(dim) if scale is None else scale
    rows = sum(n_new)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    row = heads * dim + pad
    q = (torch.randn((rows, row), generator=gen, device="cuda") * q_scale).to(TORCH[dtype])
    out = torch.full((rows, row), 7.0, dtype=TORCH[dtype], device="cuda")
    lse = torch.full((rows, heads), 7.0, device="cuda")
    kn = vn = None
    if write:
        kn, vn = (torch.cat([c.want[s][i][layer, c.want[s][i].shape[1] - n:] for s, n in zip(seqs, n_new)]) for i in (0, 1))
        kn, vn = (torch.nn.functional.pad(x.flatten(1), (0, 8)).contiguous() for x in (kn, vn))
    plan = c.pool.plan(heads)
    plan.update(seqs, n_new, _stream())
    assert plan.rows == rows
    call = lambda: plan.attend(layer, q.data_ptr(), out.data_ptr(), scale, lse_ptr=lse.data_ptr(), q_stride=row, out_stride=row,
                               k_new_ptr=kn.data_ptr() if write else None, v_new_ptr=vn.data_ptr() if write else None,
                               kv_stride=kv * dim + 8, stream=_stream())
    call()
    first = out.clone()
    call()   # the same plan again: the same bits
    assert torch.equal(first.view(torch.int16), out.view(torch.int16))
    ref, mag, zref = _reference(c, layer, seqs, n_new, q[:, :heads * dim].unflatten(1, (heads, dim)), heads, scale)
    assert (out[:, heads * dim:] == 7.0).all()
    got = out[:, :heads * dim].unflatten(1, (heads, dim)).double()
    u = UNIT[dtype]
    err = (got - ref).abs() - (u * (mag + ref.abs()) + 2.0 ** -14 * mag + 2.0 ** -24)
    assert torch.isfinite(got).all() and (err <= 0).all(), (float((got - ref).abs().max()), int((err > 0).sum()))
    assert ((lse.double() - zref).abs() <= 2.0 ** -14 * (1 + zref.abs())).all()
    plan.close()


SHAPES = [(1, 16, 16, 32), (30, 8, 2, 64), (30, 8, 1, 128), (1, 14, 2, 128), (1, 6, 3, 32), (30, 20, 1, 64)]


@gpu
@pytest.mark.parametrize("dtype,heads,kv,dim", SHAPES)
@pytest.mark.parametrize("length", [1, 2, 63, 64, 65, 127, 128, 129, 700])
def test_attend_lengths(t2sx_mod, dtype, heads, kv, dim, length):
    """One token, alone, at lengths around the page; what stands beyond the length is NaN."""
    _need_gpu()
    c = Cache(t2sx_mod, dtype, 2, 40, kv, dim, 3)
    c.extend(0, 3)
    c.extend(1, length)
    _attend(c, dtype, 1, [1], [1], heads)
    _attend(c, dtype, 0, [1, 0], [1, 1], heads, write=True)


@gpu
@pytest.mark.parametrize("dtype,heads,kv,dim", SHAPES)
@pytest.mark.parametrize("prompt,each", [(350, 5), (64, 3), (63, 20), (1000, 40), (130, 150)])
def test_attend_forked(t2sx_mod, dtype, heads, kv, dim, prompt, each):
    """Candidates of two prompts, ragged, in a shuffled order, one of them still of the prompt's length."""
    _need_gpu()
    rng = np.random.default_rng(prompt + each)
    c = Cache(t2sx_mod, dtype, 1, 2 * (prompt // PAGE + 1) + 8 * each, kv, dim, 2 + 2 * each)
    c.extend(0, prompt)
    c.extend(1, max(1, prompt - 40))
    cand = list(range(2, 2 + 2 * each))
    c.derive("fork", [i % 2 for i in cand], cand)
    for s in cand[1:]:
        c.extend(s, int(rng.integers(1, 200)))
    grown = cand[1:]
    rng.shuffle(cand)
    rng.shuffle(grown)
    _attend(c, dtype, 0, cand, [1] * len(cand), heads)
    _attend(c, dtype, 0, grown, [1] * len(grown), heads, write=True, pad=8)


@gpu
@pytest.mark.parametrize("dtype,heads,kv,dim", SHAPES)
def test_attend_forks_of_forks(t2sx_mod, dtype, heads, kv, dim):
    """Three generations; sequences of no rows, a prompt beside its candidates, chunks of several rows."""
    _need_gpu()
    rng = np.random.default_rng(dim)
    c = Cache(t2sx_mod, dtype, 1, 260, kv, dim, 40)
    c.extend(0, 200)
    c.derive("fork", [0] * 3, [1, 2, 3])
    for s in (1, 2, 3):
        c.extend(s, int(rng.integers(60, 200)))
    c.derive("fork", [1] * 4 + [2] * 4, list(range(4, 12)))
    for s in range(4, 12):
        c.extend(s, int(rng.integers(1, 130)))
    c.derive("fork", [5] * 12, list(range(12, 24)))
    for s in range(12, 24):
        c.extend(s, int(rng.integers(0, 70)))
    c.extend(30, 77)
    seqs = rng.permutation(list(range(24)) + [30]).tolist()
    new = [int(rng.choice([0, 1, 1, 2, 9])) for _ in seqs]
    new[0] = 1
    _attend(c, dtype, 0, seqs, new, heads)
    # a row in a page of several sequences is not written; the rows behind those pages are
    users = np.zeros(c.pool.n_pages, dtype=int)
    for s in c.want:
        users[c.pool.table([s])[0]] += 1
    with pytest.raises(t2sx_mod.T2SXError) as e:
        _attend(c, dtype, 0, [0, 1], [150, 1], heads, write=True)
    assert e.value.code == t2sx_mod.ERR_STATE
    own = [c.pool.length(s) - PAGE * int((users[c.pool.table([s])[0]] > 1).sum()) for s in seqs]
    _attend(c, dtype, 0, seqs, [min(n, o) for n, o in zip(new, own)], heads, write=True)


@gpu
@pytest.mark.parametrize("dtype,heads,kv,dim", SHAPES)
@pytest.mark.parametrize("cached,new", [(0, 1), (0, 2), (0, 64), (0, 65), (37, 130), (300, 200), (63, 129), (1, 517)])
def test_attend_chunk(t2sx_mod, dtype, heads, kv, dim, cached, new):
    """Rows of a prompt over what is cached, causal, two ragged prompts in a call."""
    _need_gpu()
    c = Cache(t2sx_mod, dtype, 1, 40, kv, dim, 3)
    c.extend(0, cached + new, write=False)
    c.extend(1, 5, write=False)
    for s in (0, 1):   # the rows come with the call; only what is cached is there before
        t = torch.as_tensor(c.pool.table([s])[0], device="cuda").long()
        pos = torch.arange(cached if s == 0 else 2, device="cuda")
        for i, x in enumerate((c.k, c.v)):
            x[:, t[pos // PAGE], :, pos % PAGE] = c.want[s][i][:, :len(pos)].movedim(1, 0)
    _attend(c, dtype, 0, [0, 1], [new, 3], heads, write=True)
    c.check()


@gpu
@pytest.mark.parametrize("dtype,heads,kv,dim", SHAPES)
def test_attend_long_and_peaked(t2sx_mod, dtype, heads, kv, dim):
    """A long axis with few rows; scores of several hundreds, rising and falling along it; a zero scale."""
    _need_gpu()
    c = Cache(t2sx_mod, dtype, 1, 330, kv, dim, 4)
    c.extend(0, 20000)
    c.derive("fork", [0, 0], [1, 2])
    c.extend(1, 70)
    _attend(c, dtype, 0, [0], [1], heads)
    _attend(c, dtype, 0, [0, 1, 2], [1, 3, 1], heads)
    _attend(c, dtype, 0, [0, 1, 2], [1, 3, 1], heads, scale=0.0)
    # keys that grow along the sequence: the running maximum keeps changing
    x = c.want[0][0]
    x.mul_(torch.linspace(0.0, 12.0, x.shape[1], device="cuda", dtype=x.dtype)[None, :, None, None])
    t = torch.as_tensor(c.pool.table([0])[0], device="cuda").long()
    pos = torch.arange(c.pool.length(0), device="cuda")
    c.k[:, t[pos // PAGE], :, pos % PAGE] = x.movedim(1, 0)
    # the bound of 2^-14 on what scores leave holds for scores up to about 2^6: the scale keeps them there
    _attend(c, dtype, 0, [0], [1], heads, scale=0.25 / math.sqrt(dim))


@gpu
def test_attend_other_stream(t2sx_mod):
    """Calls on two streams in turn take effect in the order of the calls."""
    _need_gpu()
    c = Cache(t2sx_mod, 1, 1, 3000, 4, 64, 60)
    c.extend(0, 3000)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in range(1, 40):
        with torch.cuda.stream(streams[s % 2]):
            c.derive("copy", [s - 1], [s])   # each reads what the other stream's call wrote
    torch.cuda.synchronize()
    c.check()
    with torch.cuda.stream(streams[0]):
        c.derive("fork", [39], [50])
        c.release(list(range(39)))
        with torch.cuda.stream(streams[1]):
            c.pool.compact(_stream())
        _attend(c, 1, 0, [39, 50], [2, 2], 8)
    torch.cuda.synchronize()
    c.check()


@gpu
def test_plan_outlives_pool_and_updates_grow(t2sx_mod):
    _need_gpu()
    c = Cache(t2sx_mod, 1, 1, 400, 2, 32, 200)
    plan = c.pool.plan(4)
    q = torch.randn((400, 4, 32), device="cuda").half()
    out = torch.empty_like(q)
    plan.update([], [], _stream())
    plan.attend(0, q.data_ptr(), out.data_ptr(), 0.2, stream=_stream())
    for n in (1, 30, 180, 7):
        for s in range(n):
            c.extend(s, 1 + s % 3)
        plan.update(list(range(n)), [1] * n, _stream())
        plan.attend(0, q.data_ptr(), out.data_ptr(), 0.2, stream=_stream())
        ref, mag, _ = _reference(c, 0, list(range(n)), [1] * n, q[:n], 4, 0.2)
        assert ((out[:n].double() - ref).abs() <= 2.0 ** -11 * (mag + ref.abs()) + 2.0 ** -14 * mag + 2.0 ** -24).all()
    c.pool.close()
    with pytest.raises(t2sx_mod.T2SXError):
        plan.attend(0, q.data_ptr(), out.data_ptr(), 0.2, stream=_stream())
    plan.close()


@gpu
@pytest.mark.parametrize("dtype,heads,kv,dim", SHAPES)
def test_attend_again_and_again(t2sx_mod, dtype, heads, kv, dim):
    """Many rows of shared and of own pages, one to three pages to a tile: every call gives the same bits, also
    with other work between the calls."""
    _need_gpu()
    c = Cache(t2sx_mod, dtype, 1, 400, kv, dim, 90)
    c.extend(0, 190)
    c.derive("fork", [0] * 80, list(range(1, 81)))
    for s in range(1, 81):
        c.extend(s, 1 + s * 7 % 90)
    c.extend(85, 170)
    seqs, new = list(range(1, 81)) + [85], [1] * 80 + [130]
    gen = torch.Generator(device="cuda").manual_seed(2)
    q = torch.randn((sum(new), heads, dim), generator=gen, device="cuda").to(TORCH[dtype])
    plan = c.pool.plan(heads)
    plan.update(seqs, new, _stream())
    outs = []
    for i in range(12):
        out = torch.full_like(q, 7.0)
        plan.attend(0, q.data_ptr(), out.data_ptr(), 0.2, stream=_stream())
        outs.append(out)
        if i % 3 == 0:
            torch.empty(1 << 26, device="cuda").fill_(1.0)   # what the caches held is gone
    ref, mag, _ = _reference(c, 0, seqs, new, q, heads, 0.2)
    u = UNIT[dtype]
    for out in outs:
        assert torch.equal(out.view(torch.int16), outs[0].view(torch.int16))
        assert ((out.double() - ref).abs() <= u * (mag + ref.abs()) + 2.0 ** -14 * mag + 2.0 ** -24).all()
    plan.sync()


@gpu
@pytest.mark.parametrize("dim", [32, 64, 128])
def test_attend_wait_timeout_reported_and_recovered(t2sx_mod, dim):
    """A wait that nothing ends runs out: NaN outputs and a status, and the next calls are right again."""
    _need_gpu()
    c = Cache(t2sx_mod, 1, 1, 40, 8, dim, 3)
    c.extend(0, 700)
    q = torch.randn((300, 16, dim), device="cuda").half()
    out = torch.zeros_like(q)
    plan = c.pool.plan(16)
    plan.update([0], [300], _stream())
    call = lambda: plan.attend(0, q.data_ptr(), out.data_ptr(), 0.1, stream=_stream())
    try:
        t2sx_mod.test_set_tc_wait_cycles(100_000)
        call()
        with pytest.raises(t2sx_mod.T2SXError) as e:
            plan.sync()
        assert e.value.code == t2sx_mod.ERR_TIMEOUT
        assert out.isnan().any()
        call()
        torch.cuda.synchronize()
        with pytest.raises(t2sx_mod.T2SXError) as e:
            call()
        assert e.value.code == t2sx_mod.ERR_TIMEOUT
    finally:
        t2sx_mod.test_set_tc_wait_cycles(0)
    for _ in range(2):
        call()
        plan.sync()
        ref, mag, _ = _reference(c, 0, [0], [300], q, 16, 0.1)
        assert ((out.double() - ref).abs() <= 2.0 ** -11 * (mag + ref.abs()) + 2.0 ** -14 * mag + 2.0 ** -24).all()


# ---- log probabilities -----------------------------------------------------------------------------------

def _scores(t2sx, x, tokens, top, stream=None):
    rows, vocab = x.shape
    dtype = {torch.float32: t2sx.F32, torch.float16: t2sx.F16, torch.bfloat16: t2sx.BF16}[x.dtype]
    lp, h = (torch.full((rows,), 7.0, device="cuda") for _ in range(2))
    rank = torch.full((rows,), 7, dtype=torch.int32, device="cuda")
    ids = torch.full((rows, top), 7, dtype=torch.int32, device="cuda")
    tl = torch.full((rows, top), 7.0, device="cuda")
    t2sx.token_logprobs(dtype, rows, vocab, x.data_ptr(), tokens.data_ptr(), lp.data_ptr(), h.data_ptr(), rank.data_ptr(), top,
                        ids.data_ptr() if top else None, tl.data_ptr() if top else None, stride=x.stride(0), stream=_stream())
    return lp, h, rank, ids, tl


def _check_scores(t2sx, x, tokens, top):
    got = [a.cpu() for a in _scores(t2sx, x, tokens, top)]
    x, tokens = x.double().cpu(), tokens.cpu().long()
    lp, h, rank, ids, tl = got
    ref = x.log_softmax(-1)
    span = (x.amax(-1, keepdim=True) - x).masked_fill(x == float("-inf"), 0).amax(-1).clamp(min=1)
    tol = 2.0 ** -17 * span
    want = ref.gather(1, tokens[:, None])[:, 0]
    same = (lp.double() == want) | ((lp.double() - want).abs() <= tol)
    assert same.all(), (lp.double() - want).abs().max()
    href = -torch.special.xlogy(ref.exp(), ref.exp()).sum(-1)
    assert ((h.double() - href).abs() <= tol).all(), (h.double() - href).abs().max()
    xt = x.gather(1, tokens[:, None])
    before = (x > xt) | ((x == xt) & (torch.arange(x.shape[1])[None] < tokens[:, None]))
    assert torch.equal(rank.long(), before.sum(-1))
    order = torch.sort(x, dim=1, descending=True, stable=True)
    k = min(top, x.shape[1])
    listed = order.values[:, :k] > float("-inf")
    assert torch.equal(ids[:, :k].long(), torch.where(listed, order.indices[:, :k], -1))
    assert (ids[:, k:] == -1).all() and (tl[:, k:] == float("-inf")).all()
    tref = ref.gather(1, order.indices[:, :k])
    assert ((tl[:, :k].double() == tref) | ((tl[:, :k].double() - tref).abs() <= tol[:, None])).all()


@gpu
@pytest.mark.parametrize("dtype", [0, 1, 30])
@pytest.mark.parametrize("rows,vocab,top,pad", [(1, 1, 1, 0), (3, 2, 5, 0), (1, 31, 32, 1), (5, 33, 0, 3), (8, 1025, 5, 0), (2, 1025, 32, 7),
                                                (257, 1024, 15, 0), (1, 4097, 20, 0), (2, 70001, 20, 0), (300, 70001, 20, 1),
                                                (40, 131072, 32, 0), (1, 140001, 1, 0), (3000, 200, 3, 5)])
def test_logprobs(t2sx_mod, dtype, rows, vocab, top, pad):
    """Sizes from one token to wide, strided rows, masked tokens (the given one among them), many ties in 16 bits."""
    _need_gpu()
    gen = torch.Generator(device="cuda").manual_seed(rows + vocab)
    x = (torch.randn((rows, vocab + pad), generator=gen, device="cuda") * 2.5).to(TORCH[dtype])
    x[:, vocab:] = float("nan")
    x = x[:, :vocab]
    tokens = torch.randint(0, vocab, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    if vocab > 2:
        x[:, torch.randint(0, vocab, (vocab // 5,), generator=gen, device="cuda")] = float("-inf")
        x[::3, 1:][x[::3, 1:] > 3.0] = float("-inf")
        x[:, 0] = 1.0   # one token at least is open
    _check_scores(t2sx_mod, x, tokens, top)


@gpu
@pytest.mark.parametrize("dtype", [0, 1, 30])
@pytest.mark.parametrize("vocab", [700, 50000])
def test_logprobs_orders(t2sx_mod, dtype, vocab):
    """Rows that rise, fall, are all equal, have one open token, or few distinct values: every list is hard somewhere."""
    _need_gpu()
    j = torch.arange(vocab, device="cuda", dtype=torch.float32)
    rows = [j / vocab * 9, -j / vocab * 9, torch.zeros_like(j), torch.where(j == vocab - 3, 2.0, float("-inf")), (j * 7919 % 5) - 2,
            torch.where(j % 1000 == 999, 5.0, 0.0), torch.where(j >= vocab - 40, j / vocab, -3.0), -1e4 + j % 3, (j % 2) * -0.0]
    x = torch.stack(rows).to(TORCH[dtype])
    tokens = torch.tensor([0, vocab - 1, vocab // 2, vocab - 3, 4, 5, vocab - 40, 2, 3], device="cuda", dtype=torch.int32)
    _check_scores(t2sx_mod, x, tokens, 32)


@gpu
@pytest.mark.parametrize("dtype", [0, 1, 30])
@pytest.mark.parametrize("rows,vocab", [(8, 300), (8, 90001), (600, 1025)])
def test_logprobs_empty_rows_and_padding(t2sx_mod, dtype, rows, vocab):
    _need_gpu()
    inf, nan = float("inf"), float("nan")
    x = torch.randn((rows, vocab), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).to(TORCH[dtype])
    x[0] = -inf
    x[1, vocab // 2] = nan
    x[2, vocab - 1] = inf
    tokens = torch.full((rows,), 5, dtype=torch.int32, device="cuda")
    tokens[3], tokens[4], tokens[5] = -1, vocab, -7
    lp, h, rank, ids, tl = (a.cpu() for a in _scores(t2sx_mod, x, tokens, 4))
    assert lp[0] == -inf and h[0] == 0 and rank[0] == 5 and (ids[0] == -1).all() and (tl[0] == -inf).all()
    for r in (1, 2):
        assert lp[r].isnan() and h[r].isnan() and tl[r].isnan().all()
    assert ids[2, 0] == vocab - 1 and vocab // 2 not in ids[1].tolist()
    assert torch.equal(ids[1, :4].long(), torch.sort(x[1].nan_to_num(nan=-inf).double().cpu(), descending=True, stable=True).indices[:4])
    assert lp[3] == 0 and rank[3] == -1 and h[3].isfinite()
    assert lp[4].isnan() and lp[5].isnan() and rank[4] == rank[5] == -1
    assert torch.isfinite(lp[6:]).all() and (ids[3:] >= 0).all()


@gpu
@pytest.mark.parametrize("dtype", [0, 1, 30])
@pytest.mark.parametrize("vocab", [900, 40000])
def test_logprobs_ends_of_the_range(t2sx_mod, dtype, vocab):
    """Tokens masked with the type's lowest value: some, all, all but masked ones, beside -inf; values near the
    greatest one; values around -10000, whose differences count."""
    _need_gpu()
    low = torch.finfo(TORCH[dtype]).min
    gen = torch.Generator(device="cuda").manual_seed(vocab)
    x = (torch.randn((7, vocab), generator=gen, device="cuda") * 2).to(TORCH[dtype])
    x[0, ::2] = low
    x[1] = low
    x[2] = low
    x[2, 1::3] = float("-inf")
    x[3, : vocab - 9] = low
    x[4] = -low
    x[4, ::2] = -low * 0.5
    x[5] = -10000 + x[5] * 8
    x[6] = low
    x[6, vocab // 3 :] = low * 0.998
    tokens = torch.tensor([1, 7, 0, vocab - 1, 3, 2, vocab // 2], device="cuda", dtype=torch.int32)
    got = [a.cpu() for a in _scores(t2sx_mod, x, tokens, 8)]
    ref = x.double().log_softmax(-1).cpu()
    lp, h, rank, ids, tl = got
    # (differences of up to twice the type's range: compared where the weight is not 0)
    want = ref.gather(1, tokens.cpu().long()[:, None])[:, 0]
    near = want > -1e3
    assert near.sum() >= 5 and ((lp.double() - want).abs()[near] <= 2.0 ** -17 * want.abs().clamp(min=1)[near]).all()
    href = -torch.special.xlogy(ref.exp(), ref.exp()).sum(-1)
    assert ((h.double() - href).abs() <= 2.0 ** -17 * 16).all(), (h, href)
    order = torch.sort(x.double().cpu(), dim=1, descending=True, stable=True)
    assert torch.equal(ids.long(), order.indices[:, :8])
    tref = ref.gather(1, order.indices[:, :8])
    assert ((tl.double() - tref).abs()[tref > -1e3] <= 2.0 ** -17 * 16).all()


@gpu
def test_logprobs_optional_outputs(t2sx_mod):
    _need_gpu()
    x = torch.randn((4, 50), device="cuda")
    t = torch.zeros(4, dtype=torch.int32, device="cuda")
    lp = torch.empty(4, device="cuda")
    t2sx_mod.token_logprobs(0, 4, 50, x.data_ptr(), t.data_ptr(), lp.data_ptr(), stream=_stream())
    assert ((lp.double() - x.double().log_softmax(-1)[:, 0]).abs() < 2.0 ** -14).all()


@gpu
def test_candidates_together(t2sx_mod):
    """candidates.draw(): scores of what it draws against a plain forward pass in 64 bits over each whole sequence.
    Six roundings to f16 in each of two layers, of activations and as many of weights, independent of one another, move a
    row by sqrt(24) 2^-12 of its length, and a logit by that share of its spread (0.02 x 512 / sqrt(512) = 0.45): 0.0006.
    2^-8 is six times that."""
    _need_gpu()
    import candidates
    import synth
    tensors = [(n, a) for n, a in synth.tensor_values(3, n_layer=2)]
    dec = candidates.Decoder(tensors)
    rng = np.random.default_rng(5)
    prompts = [rng.integers(0, candidates.EOS, m).tolist() for m in (130, 64, 1)]
    found = candidates.draw(dec, prompts, each=5, steps=9, seed=1)
    again = candidates.draw(dec, prompts, each=5, steps=9, seed=1)
    assert found == again
    w = {n: torch.tensor(a).double() for n, a in tensors}

    def scores(tokens):
        n, d = len(tokens), 512
        freq = torch.exp(torch.arange(0, d, 2).double() * (-math.log(10000.0) / d))
        angle = torch.arange(n).double()[:, None] * freq
        x = w["encoder.audio_embedding"][tokens] + torch.stack([angle.sin(), angle.cos()], 2).flatten(1)
        for i in range(2):
            g = lambda name: w[f"attention.{i}.{name}"]
            q, k, v = ((x @ g("qkv_w").T + g("qkv_b")).view(n, 3, 16, 32).permute(1, 2, 0, 3))
            s = (q @ k.transpose(1, 2)) * 32 ** -0.5
            s = s.masked_fill(torch.ones(n, n, dtype=torch.bool).triu(1), -math.inf).softmax(-1)
            a = (s @ v).transpose(0, 1).reshape(n, d)
            x = torch.nn.functional.layer_norm(x + a @ g("out_proj_w").T + g("out_proj_b"), (d,), g("ln1_w"), g("ln1_b"))
            up = (x @ g("ffn_up_w").T + g("ffn_up_b")).relu()
            x = torch.nn.functional.layer_norm(x + up @ g("ffn_down_w").T + g("ffn_down_b"), (d,), g("ln2_w"), g("ln2_b"))
        return (x @ w["sampler.lm_head_w"].T).log_softmax(-1)

    for prompt, kept in zip(prompts, found):
        assert len(kept) == 3 and [c[0] for c in kept] == sorted((c[0] for c in kept), reverse=True)
        for mean, drawn in kept:
            assert 1 <= len(drawn) <= 9 and (len(drawn) == 9 or drawn[-1] == candidates.EOS)
            lp = scores(prompt + drawn)[len(prompt) - 1:-1].gather(1, torch.tensor(drawn)[:, None])
            assert abs(mean - lp.mean().item()) <= 2.0 ** -8, (mean, lp)


# ---- layers, peaks, alignments -----------------------------------------------------------------------------

def _forget(c, layer, seq, count):
    """Zeros in place of the sequence's last positions in one layer: a call that writes them has to."""
    t = torch.as_tensor(c.pool.table([seq])[0], device="cuda").long()
    n = c.pool.length(seq)
    pos = torch.arange(n - count, n, device="cuda")
    for x in (c.k, c.v):
        x[layer, t[pos // PAGE], :, pos % PAGE] = 0


@gpu
@pytest.mark.parametrize("dtype,heads,kv,dim", SHAPES)
def test_attend_layers(t2sx_mod, dtype, heads, kv, dim):
    """Layers above the first in every form of the attention: many rows over shared pages (the tcgen05 kernel, warp tiles
    and joins), chunks (rows written by a launch of their own), one long sequence in parts.  Rows go to
    the call's layer and nowhere else."""
    _need_gpu()
    rng = np.random.default_rng(heads + dim)
    c = Cache(t2sx_mod, dtype, 3, 700, kv, dim, 150)
    c.extend(0, 1000)
    c.extend(1, 130)
    cand = list(range(2, 122))
    c.derive("fork", [i % 2 for i in cand], cand)
    for s in cand:
        c.extend(s, int(rng.integers(1, 150)))
    c.extend(130, 500)
    c.extend(131, 9000)
    for layer in (2, 1):
        _attend(c, dtype, layer, cand, [1] * len(cand), heads)
        for seqs, new in ((cand, [1] * len(cand)), ([130, 5], [333, 1]), ([131], [1])):
            for s, n in zip(seqs, new):
                _forget(c, layer, s, n)
            _attend(c, dtype, layer, seqs, new, heads, write=True)
            c.check()


@gpu
@pytest.mark.parametrize("dtype", [1, 30])
@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("rows", [100, 200])
@pytest.mark.parametrize("step", [2.5, 8.0])
def test_attend_rising_and_falling(t2sx_mod, dtype, dim, rows, step):
    """Scores whose level rises by `step` from page to page, eight times, and falls again, over and over: the maximum that weights
    refer to moves several times inside an item, at once or after weights have grown.  One and two tiles of rows of
    the tcgen05 kernel.  Scores stay below 2^6, which the tolerance needs."""
    _need_gpu()
    heads, kv = 8, 2
    each = rows // (heads // kv)
    c = Cache(t2sx_mod, dtype, 1, 60 + 2 * each, kv, dim, 1 + each)
    gen = torch.Generator(device="cuda").manual_seed(dim + rows)
    length = 60 * PAGE
    c.extend(0, length)
    page = torch.arange(length, device="cuda") // PAGE % 16
    level = step * torch.minimum(page, 16 - page)            # 0 .. 8 and down
    level = level * min(1.0, 56.0 / float(level.max()))
    sign = torch.randint(0, 2, (dim,), generator=gen, device="cuda") * 2.0 - 1.0
    noise = torch.randn(c.want[0][0].shape, generator=gen, device="cuda") * 0.3
    c.want[0][0] = (level[None, :, None, None] / math.sqrt(dim) * sign + noise).to(TORCH[dtype])
    t = torch.as_tensor(c.pool.table([0])[0], device="cuda").long()
    pos = torch.arange(length, device="cuda")
    c.k[:, t[pos // PAGE], :, pos % PAGE] = c.want[0][0].movedim(1, 0)
    seqs = list(range(1, 1 + each))
    c.derive("fork", [0] * each, seqs)
    for s in seqs:
        c.extend(s, 1 + s % 70)
    q = (sign + torch.randn((each, heads, dim), generator=gen, device="cuda") * 0.05).to(TORCH[dtype])
    out = torch.full_like(q, 7.0)
    lse = torch.full((each, heads), 7.0, device="cuda")
    scale = 1.0 / math.sqrt(dim)
    plan = c.pool.plan(heads)
    plan.update(seqs, [1] * each, _stream())
    plan.attend(0, q.data_ptr(), out.data_ptr(), scale, lse_ptr=lse.data_ptr(), stream=_stream())
    ref, mag, zref = _reference(c, 0, seqs, [1] * each, q, heads, scale)
    assert 8 < float(zref.min()) and float(zref.max()) < 70
    err = (out.double() - ref).abs() - (UNIT[dtype] * (mag + ref.abs()) + 2.0 ** -14 * mag + 2.0 ** -24)
    assert (err <= 0).all(), (float((out.double() - ref).abs().max()), int((err > 0).sum()))
    assert ((lse.double() - zref).abs() <= 2.0 ** -14 * (1 + zref.abs())).all()
    plan.sync()


@gpu
@pytest.mark.parametrize("dtype", [0, 1, 30])
@pytest.mark.parametrize("level", [0.0, 100.0, -1000.0, 10000.0, 50000.0])
@pytest.mark.parametrize("vocab,pad", [(3, 0), (5, 2), (9, 0), (41, 0), (300, 1), (1025, 0)])
def test_logprobs_level(t2sx_mod, dtype, level, vocab, pad):
    """Rows at every alignment whose logits stand far from zero: what counts is their differences, also for the
    elements before and after a row's whole vectors, which are the likely tokens here."""
    _need_gpu()
    gen = torch.Generator(device="cuda").manual_seed(vocab)
    rows = 16
    x = torch.randn((rows, vocab + pad), generator=gen, device="cuda") * 2
    for e in (0, 1, 2, -3, -2, -1):
        x[:, :vocab][:, max(e, -vocab) if e < 0 else min(e, vocab - 1)] += 4
    x = (x + level).to(TORCH[dtype])[:, :vocab]
    tokens = torch.arange(rows, device="cuda", dtype=torch.int32) % vocab
    _check_scores(t2sx_mod, x, tokens, min(5, vocab))


@gpu
@pytest.mark.parametrize("dtype,rows,vocab", [(0, 700, 1025), (0, 3000, 333), (1, 40, 5001), (30, 12, 100003), (30, 2000, 1023)])
def test_logprobs_equal_rows(t2sx_mod, dtype, rows, vocab):
    """The same row again and again in a call: the same bits where its address is the same modulo 16, and the same within
    the sums' error (twice 2^-17 of the span) where it is not."""
    _need_gpu()
    gen = torch.Generator(device="cuda").manual_seed(vocab)
    one = (torch.randn(vocab, generator=gen, device="cuda") * 2.5).to(TORCH[dtype])
    x = one.repeat(rows, 1)
    tokens = torch.full((rows,), vocab // 3, dtype=torch.int32, device="cuda")
    got = _scores(t2sx_mod, x, tokens, 9)
    span = float((one.max() - one.min()).double())
    place = [r * vocab * x.element_size() % 16 for r in range(rows)]
    first = [place.index(p) for p in place]
    assert len(set(first)) > 3
    for a in got:
        assert torch.equal(a.view(torch.int32), a[first].view(torch.int32))
        assert ((a.double() - a[:1].double()).abs() <= (2.0 ** -16 * span if a.dtype == torch.float32 else 0)).all()
