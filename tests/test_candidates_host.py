"""The host side of the candidate operators (page lists, plans, launch shapes, the order of device work) on a fake
CUDA runtime: nothing here needs or touches a GPU."""
import ctypes as C
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOURCES = ("t2sx_pool.cu", "t2sx_prefix_attn.cu", "t2sx_prefix_tc.cu", "t2sx_logprobs.cu")
K_STORE, V_STORE, Q = 1 << 20, 1 << 21, 1 << 22   # addresses: nothing reads what stands there


@pytest.fixture(scope="module")
def fake_lib(tmp_path_factory):
    import build
    import t2sx
    tmp = tmp_path_factory.mktemp("fake_cuda")
    jobs = []
    for name in SOURCES:
        cmd = [build.nvcc(), *build.NVCC_FLAGS, "-I", os.path.join(ROOT, "include"), "-c", os.path.join(build.CSRC, name), "-o", str(tmp / (name + ".o"))]
        jobs.append((name, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
    for name, job in jobs:
        out = job.communicate()[0]
        assert job.returncode == 0, (name, out)
    gxx = shutil.which("g++")
    assert gxx, "g++ is required"
    so = str(tmp / "libfake.so")
    cuda = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(build.nvcc()))), "include")
    r = subprocess.run([gxx, "-std=c++17", "-O2", "-shared", "-fPIC", "-fvisibility=hidden", "-Wl,-Bsymbolic", "-I", cuda, os.path.join(ROOT, "tests", "cpp", "fake_cuda.cpp"),
                        *[str(tmp / (n + ".o")) for n in SOURCES], "-o", so], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    lib = C.CDLL(so)
    for name, (res, args) in t2sx.SIGNATURES.items():
        if name.startswith(("t2sx_pool_", "t2sx_plan_")) or name in ("t2sx_token_logprobs", "t2sx_last_error"):
            getattr(lib, name).restype, getattr(lib, name).argtypes = res, args
    for name in ("fake_launches", "fake_grid_x", "fake_synced", "fake_recorded"):
        getattr(lib, name).restype = C.c_longlong
    lib.fake_recorded.argtypes, lib.fake_fail_launch.argtypes = [C.c_void_p], [C.c_longlong]
    return lib


@pytest.fixture
def host(fake_lib, monkeypatch):
    """The binding on the fake runtime."""
    import t2sx
    monkeypatch.setattr(t2sx, "_lib", fake_lib)
    fake_lib.fake_reset()
    yield t2sx
    while OPEN:   # while the binding still has the library that they come from
        OPEN.pop().close()


OPEN = []


def _pool(t2sx, pages, seqs, dim=32, kv=1, layers=1):
    OPEN.append(t2sx.PagePool(t2sx.F16, layers, pages, kv, dim, seqs, K_STORE, V_STORE))
    return OPEN[-1]


def _state(pool):
    return pool.available(), [pool.length(s) for s in range(pool.max_seqs)], [pool.table([s]).tolist() for s in range(pool.max_seqs)]


def _refused(t2sx, code, call):
    with pytest.raises(t2sx.T2SXError) as e:
        call()
    assert e.value.code == code, e.value


@pytest.mark.parametrize("op", ["fork", "copy"])
def test_source_among_the_destinations(host, fake_lib, op):
    """A sequence that a call fills is not a source of that call: its pages would be copied while they are
    written, and they are not counted.  Refused before anything changes, whatever the order of the pairs."""
    pool = _pool(host, pages=40, seqs=6)
    pool.extend([0], [70])
    derive = getattr(pool, op)
    before = _state(pool)
    for srcs, dsts in (([0, 1], [1, 2]), ([1, 0], [2, 1]), ([0, 1, 2], [1, 2, 3]), ([0, 3, 1], [1, 2, 3]), ([4], [4])):
        _refused(host, host.ERR_INVALID, lambda: derive(srcs, dsts))
        assert _state(pool) == before and fake_lib.fake_launches() == 0
    # as many pages as one copy needs: the second one's were taken from beyond the list of free pages
    small = _pool(host, pages=3 if op == "fork" else 4, seqs=4)
    small.extend([0], [70])
    before = _state(small)
    _refused(host, host.ERR_INVALID, lambda: getattr(small, op)([0, 1], [1, 2]))
    assert _state(small) == before
    # ids of the refused calls are free for others; the same source for several is no such case
    derive([0, 0, 5], [1, 2, 3])
    assert [pool.length(s) for s in range(6)] == [70, 70, 70, 0, 0, 0]


def _plan(pool, heads):
    OPEN.append(pool.plan(heads))
    return OPEN[-1]


def _attend(plan, new=False, layer=0, stream=0):
    plan.attend(layer, Q, Q, 1.0, k_new_ptr=Q if new else None, v_new_ptr=Q if new else None, stream=stream)


def test_fork_between_update_and_attend(host, fake_lib):
    """A fork that comes to share the page of a plan's row: the row's keys and values are not written there any
    more; attending without writing them goes on, and so do rows in pages that are still their sequence's own."""
    pool = _pool(host, pages=40, seqs=6)
    pool.extend([0, 1], [64, 70])
    plan, other = _plan(pool, 1), _plan(pool, 1)
    plan.update([0, 1], [1, 1])
    other.update([1], [1])
    _attend(plan, new=True)
    pool.fork([1], [2])   # shares the first page of 1; its row is in the second one
    _attend(plan, new=True)
    pool.fork([0], [3])
    fake_lib.fake_reset()
    for _ in range(2):
        _refused(host, host.ERR_STATE, lambda: _attend(plan, new=True))
    assert fake_lib.fake_launches() == 0
    _attend(plan)
    _attend(other, new=True)
    # the row after that page is the sequence's own again
    pool.extend([0], [1])
    plan.update([0, 1], [1, 1])
    _attend(plan, new=True)
    plan.update([0, 1], [2, 1])
    _refused(host, host.ERR_STATE, lambda: _attend(plan, new=True))
    pool.release([3])
    plan.update([0, 1], [2, 1])
    _attend(plan, new=True)


def test_failed_call_leaves_its_device_work_known(host, fake_lib):
    """Where a later launch of a call fails, the earlier ones are the pool's last work: the next call on another stream
    waits for them.  A call whose first launch fails leaves none."""
    pool = _pool(host, pages=2000, seqs=900, kv=16)
    pool.extend([0], [70])
    fake_lib.fake_fail_launch(2)
    _refused(host, host.ERR_CUDA, lambda: pool.fork([0] * 700, list(range(1, 701)), 11))   # two launches of 512 copies at most
    pool.fork([0], [801], 12)
    assert fake_lib.fake_recorded(11) == 1
    fake_lib.fake_fail_launch(1)
    _refused(host, host.ERR_CUDA, lambda: pool.fork([0], [802], 13))
    pool.fork([0], [803], 12)
    assert fake_lib.fake_recorded(13) == 0 and fake_lib.fake_recorded(12) == 1   # for the call on 13 that failed
    pool.fork([0], [804], 14)
    assert fake_lib.fake_recorded(12) == 2

    shared = _pool(host, pages=600, seqs=130, kv=16)
    shared.extend([0], [64])
    shared.fork([0] * 128, list(range(1, 129)))
    seqs = list(range(1, 129))
    shared.extend(seqs, [1] * 128)
    plan = _plan(shared, 16)
    plan.update(seqs, [1] * 128, 21)
    fake_lib.fake_reset()
    _attend(plan, stream=21)
    launches = fake_lib.fake_launches()
    assert launches > 1
    for nth in range(1, launches + 1):
        fake_lib.fake_reset()
        fake_lib.fake_fail_launch(nth)
        _refused(host, host.ERR_CUDA, lambda: _attend(plan, stream=100 + nth))
        _attend(plan, stream=200 + nth)
        assert fake_lib.fake_recorded(100 + nth) == (nth > 1)


def test_failed_copies_change_nothing(host, fake_lib):
    """fork, copy and compact whose launches fail leave lists, lengths and free pages as they were."""
    pool = _pool(host, pages=1500, seqs=1210)
    pool.extend([0, 1], [70, 3])
    pool.fork([0] * 600, list(range(2, 602)))
    for op, n, launches in (("fork", 1, 1), ("fork", 600, 2), ("copy", 1, 1), ("copy", 400, 2)):
        for nth in range(1, launches + 1):
            before = _state(pool)
            fake_lib.fake_fail_launch(nth)
            _refused(host, host.ERR_CUDA, lambda: getattr(pool, op)([0] * n, list(range(602, 602 + n))))
            assert _state(pool) == before
    before = _state(pool)
    pool.fork([0] * 600, list(range(602, 1202)))
    assert pool.available() == before[0] - 600
    pool.release(list(range(602, 1202)))
    assert _state(pool) == before

    pool = _pool(host, pages=2500, seqs=2400)
    pool.extend(list(range(2399)), [1] * 2399)
    pool.extend([2399], [130])
    pool.release(list(range(1200)))
    pool.fork([2399], [0])   # pages of two users move, too
    before = _state(pool)
    for nth in (1, 2, 3):
        fake_lib.fake_fail_launch(nth)
        _refused(host, host.ERR_CUDA, lambda: pool.compact())
        assert _state(pool) == before
    held = len({p for t in before[2] for row in t for p in row})
    assert pool.compact() == sum(p >= held for p in {p for t in before[2] for row in t for p in row})
    after = _state(pool)
    assert after[:2] == before[:2] and {p for t in after[2] for row in t for p in row} == set(range(held))
    assert after[2][0][0][:2] == after[2][2399][0][:2]
    pool.extend([1], [1])
    assert pool.table([1])[0].tolist() == [held]


def test_free_waits(host, fake_lib):
    """The pool's end waits for its device work, also where plans still hold the pool: the caller may free the
    storage then."""
    for plans in (0, 1):
        pool = _pool(host, pages=8, seqs=4)
        pool.extend([0], [70])
        if plans:
            plan = _plan(pool, 1)
        pool.fork([0], [1], 5)
        fake_lib.fake_reset()
        pool.close()
        assert fake_lib.fake_synced() == 1 and fake_lib.fake_recorded(5) == 1
    _refused(host, host.ERR_INVALID, lambda: plan.update([], []))
    plan.close()   # the stream may be gone by now
    assert fake_lib.fake_recorded(5) == 1


@pytest.mark.parametrize("n", [4, 60])
def test_update_time_does_not_follow_the_pool(host, n):
    """A step's plan costs what the step's sequences cost, however many pages the pool has (its first update may
    prepare something for each of them)."""
    import time

    def best(pages):
        pool = _pool(host, pages=pages, seqs=n + 1, kv=16)
        pool.extend([0], [640])
        seqs = list(range(1, n + 1))
        pool.fork([0] * n, seqs)
        pool.extend(seqs, [1] * n)
        plan = _plan(pool, 16)
        took = []
        for _ in range(40):
            t0 = time.perf_counter()
            plan.update(seqs, [1] * n)
            took.append(time.perf_counter() - t0)
        return min(took)

    small, large = best(4096), best(1 << 24)
    assert large < 8 * small + 100e-6, (small, large)


@pytest.mark.parametrize("vocab,rows_of_a_cta", [(1, 4), (1025, 4), (5000, 1)])
@pytest.mark.parametrize("rows", [2000, 2001, 2 ** 31 - 1, 2 ** 31 - 2])
def test_logprobs_grid(host, fake_lib, vocab, rows_of_a_cta, rows):
    """As many blocks as the rows need, up to the greatest number of rows."""
    host.token_logprobs(host.F32, rows, vocab, Q, Q, Q)
    assert fake_lib.fake_grid_x() == -(-rows // rows_of_a_cta)


def test_update_refuses_what_its_lists_cannot_hold(host):
    """A chunk of 2^24 rows over pages that 17 sequences leave one after the other: each shared run lists the rows anew."""
    pages, forks = 1 << 18, 17
    pool = _pool(host, pages=pages + 2 * forks, seqs=forks + 1)
    others = list(range(1, forks + 1))
    for s in others:
        pool.extend([0], [64])
        pool.fork([0], [s])
    pool.extend([0], [(1 << 24) - 64 * forks])
    pool.extend(others, [1] * forks)
    plan = _plan(pool, 1)
    plan.update(others, [1] * forks)
    rows = (1 << 24) - forks
    _refused(host, host.ERR_INVALID, lambda: plan.update([0] + others, [rows] + [1] * forks))
    _refused(host, host.ERR_STATE, lambda: _attend(plan))
    plan.update([0] + others, [1] * (forks + 1))
    _attend(plan)


def test_ids_that_do_not_fit(host):
    """Arrays of ids are taken for what they hold, as lists are: what is no 32-bit integer (a count: 64-bit) is not cut down to one."""
    import numpy as np
    pool = _pool(host, pages=8, seqs=4)
    for ids in ([2 ** 32], np.array([2 ** 32]), np.array([2 ** 32 + 1], dtype=np.uint64), np.array([-2 ** 32])):
        with pytest.raises(OverflowError):
            pool.extend(ids, [1])
    for ids in ([0.5], np.array([0.5]), np.array([1.0])):
        with pytest.raises(TypeError):
            pool.extend(ids, [1])
    with pytest.raises(OverflowError):
        pool.extend([0], np.array([2 ** 64 - 1], dtype=np.uint64))
    assert [pool.length(s) for s in range(4)] == [0, 0, 0, 0]
    for ids in ([0, 3], (0, 3), np.array([0, 3]), np.array([0, 9, 3], dtype=np.uint8)[::2], range(0, 4, 3), np.array([[0], [3]], dtype=np.int32)):
        pool.extend(ids, np.array([1, 2]))
    pool.extend(np.array([]), [])
    pool.extend(np.int64(1), 5)
    assert [pool.length(s) for s in range(4)] == [6, 5, 0, 12]


def test_draw_refuses_an_empty_prompt(host, fake_lib):
    """A prompt without tokens has no last row to draw from; it is refused before any work."""
    import types
    import candidates
    dec = types.SimpleNamespace(device=0, layers=1, vocab=1025, d=512)
    for prompts in ([[]], [[1, 2], []]):
        with pytest.raises(ValueError):
            candidates.draw(dec, prompts, each=2, steps=3)
    assert fake_lib.fake_launches() == 0
