"""tmg_op_logprobs against numpy in 64 bits.

Tolerances, from the arithmetic: the sum of exponentials and the weighted
sum are sums of non-negative terms in f32, at most n = ceil(V / 512) + 40
additions deep, each term a few roundings and 2^-21 (exp2) off, so the log of
the sum is off by at most (n + 16) * 2^-24, a log probability by that plus two
roundings of its own size, and the entropy by that times (1 + the mean |y|)
twice over (the weighted sum's own error, and the quotient's).  Ids are
compared exactly.
"""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover - CPU box
    pytest.skip("needs a GPU", allow_module_level=True)

from tinyminigo_b200._lib import TmgError, check, lib  # noqa: E402

U = 2.0 ** -24


@pytest.fixture(scope="module")
def ctx():
    h = ctypes.c_void_p()
    check(lib().tmg_create(0, None, ctypes.byref(h)))
    yield h
    lib().tmg_destroy(h)


def P(t, off=0):
    return None if t is None else ctypes.c_void_p(t.data_ptr() + off)


def score(ctx, x, targets, n_top, ld=None, off=0, entropy=True):
    """x [rows, V] numpy, laid out `ld` floats a row from `off` floats into a buffer."""
    rows, V = x.shape
    ld = ld or V
    buf = torch.full((off + rows * ld + 8,), float("nan"), device="cuda")
    view = buf[off:off + rows * ld].view(rows, ld)
    view[:, :V] = torch.from_numpy(x).cuda()
    t = None if targets is None else torch.from_numpy(
        np.asarray(targets, np.uint32).view(np.int32)).cuda()
    lp = None if targets is None else torch.full((rows,), -7.0, device="cuda")
    h = torch.full((rows,), -7.0, device="cuda") if entropy else None
    ids = torch.full((rows, n_top), -7, device="cuda", dtype=torch.int32) if n_top else None
    tlp = torch.full((rows, n_top), -7.0, device="cuda") if n_top else None
    torch.cuda.synchronize()
    check(lib().tmg_op_logprobs(ctx, P(buf, 4 * off), ld, rows, V, P(t), n_top, P(lp), P(h),
                                P(ids), P(tlp)), ctx)
    check(lib().tmg_sync(ctx), ctx)
    return [None if a is None else a.cpu().numpy() for a in (lp, h, ids, tlp)]


def expect(x, targets, n_top):
    x = x.astype(np.float64)
    V = x.shape[1]
    with np.errstate(all="ignore"):
        y = x - x.max(1, keepdims=True)
        e = np.exp(y)
        z = np.log(e.sum(1, keepdims=True))
        logp = y - z
        p = np.exp(logp)
        mean_y = (p * np.where(p > 0, np.abs(y), 0)).sum(1)
        h = z[:, 0] - (p * np.where(p > 0, y, 0)).sum(1)
    order = np.argsort(-np.where(np.isnan(x), -np.inf, x), axis=1, kind="stable")[:, :n_top]
    lp = None if targets is None else np.take_along_axis(logp, np.asarray(targets)[:, None], 1)[:, 0]
    n = -(-V // 512) + 56
    return lp, h, order, np.take_along_axis(logp, order, 1), n * U, 2 * n * U * (1 + mean_y)


def check_rows(ctx, x, targets, n_top, **kw):
    lp, h, ids, tlp = score(ctx, x, targets, n_top, **kw)
    rlp, rh, rids, rtlp, tol, htol = expect(x, targets, n_top)

    def near(a, b, t):
        fin = np.isfinite(b)
        assert np.array_equal(np.isnan(a), np.isnan(b)) and np.array_equal(a[~fin & ~np.isnan(b)],
                                                                            b[~fin & ~np.isnan(b)])
        assert np.all(np.abs(a - b)[fin] <= (t + 4 * U * np.abs(b))[fin]), np.abs(a - b)[fin].max()

    if targets is not None:
        near(lp, rlp, tol)
    if h is not None:
        near(h, rh, htol)
    if n_top:
        assert np.array_equal(ids.view(np.uint32), rids.astype(np.uint32))
        near(tlp, rtlp, tol)
    return lp, h, ids, tlp


@pytest.mark.parametrize("rows,V,n_top", [
    (1, 1, 1), (1, 2, 1), (3, 3, 3), (5, 64, 64), (2, 65, 64), (7, 255, 5), (4, 513, 20),
    (1, 2047, 64), (33, 2049, 1), (1, 32000, 20), (16, 32003, 64), (1, 128256, 5),
    (2, 128256, 64), (300, 1000, 8), (150, 5003, 3), (80, 20000, 10), (40, 9999, 0)])
def test_scores(ctx, rows, V, n_top):
    rng = np.random.default_rng(rows * 13 + V + n_top)
    x = rng.normal(0, 3, (rows, V)).astype(np.float32)
    x[rng.random((rows, V)) < 0.01] = -np.inf
    x[:, rng.integers(0, V)] = 4.0  # every row keeps a finite logit
    check_rows(ctx, x, rng.integers(0, V, rows), n_top)


@pytest.mark.parametrize("off,pad", [(0, 1), (1, 0), (2, 3), (3, 6), (1, 4)])
def test_unaligned_rows(ctx, off, pad):
    rng = np.random.default_rng(off * 10 + pad)
    x = rng.normal(0, 2, (5, 1003)).astype(np.float32)
    check_rows(ctx, x, rng.integers(0, 1003, 5), 7, ld=1003 + pad, off=off)


@pytest.mark.parametrize("V", [5, 700, 40001])
def test_ties_go_to_the_lowest_index(ctx, V):
    rng = np.random.default_rng(V)
    k = min(V, 64)
    x = np.zeros((4, V), np.float32)
    x[1] = rng.integers(-2, 3, V)
    x[2] = -0.0
    x[2, ::2] = 0.0
    x[3] = np.finfo(np.float32).min  # the type's lowest value everywhere: uniform
    lp, h, ids, _ = check_rows(ctx, x, rng.integers(0, V, 4), k)
    assert np.array_equal(ids[0], np.arange(k)) and np.array_equal(ids[2], np.arange(k))
    assert np.array_equal(ids[3], np.arange(k))
    assert np.allclose(h[[0, 3]], np.log(V), rtol=1e-5)


def test_clustered_large_values(ctx):
    # the large logits where few threads read them: at the front, and at
    # every multiple of the threads' stride (the bound on the n_top-th is then
    # poor and thousands of elements lie above it)
    V = 128256
    rng = np.random.default_rng(3)
    x = rng.normal(0, 1, (4, V)).astype(np.float32)
    x[0, :400] += 30
    for s in (2048, 4096, 16384):
        i = np.arange(0, V, s)
        for j in range(4):
            x[1, np.minimum(i + j, V - 1)] += 50
    x[2] = np.sort(x[2])
    x[3] = np.sort(x[3])[::-1]
    for n_top in (1, 20, 64):
        check_rows(ctx, x, rng.integers(0, V, 4), n_top)


@pytest.mark.parametrize("n_top", [20, 64])
def test_a_few_threads_hold_everything_large(ctx, n_top):
    # 4 floats a thread, 512 threads: the elements of the first n_top + 3
    # threads are all larger than any other's, for every slice of the row
    V = 512 * 4 * 128
    rng = np.random.default_rng(n_top)
    x = rng.normal(0, 1, (2, V)).astype(np.float32)
    at = np.arange(V) // 4 % 512 < n_top + 3
    x[0, at] += 100
    x[1, at] = 50
    check_rows(ctx, x, [5, V - 1], n_top)


def test_rows_without_a_distribution(ctx):
    rng = np.random.default_rng(1)
    x = rng.normal(0, 1, (5, 3001)).astype(np.float32)
    x[0] = -np.inf
    x[1, 2500] = np.nan
    x[2, 7] = np.inf
    x[3, :] = np.nan
    lp, h, ids, tlp = score(ctx, x, [1, 2, 3, 4, 5], 4)
    assert np.isnan(lp[:4]).all() and np.isnan(h[:4]).all() and np.isnan(tlp[:4]).all()
    assert np.isfinite(lp[4]) and np.isfinite(h[4]) and np.isfinite(tlp[4]).all()
    assert ids[0].tolist() == [0, 1, 2, 3] == ids[3].tolist()
    order = np.argsort(-np.where(np.isnan(x[1]), -np.inf, x[1]), kind="stable")[:4]
    assert np.array_equal(ids[1], order)
    assert ids[2][0] == 7


def test_ruled_out_targets_and_alternatives(ctx):
    # fewer finite logits than alternatives wanted: the rest is -inf, in order
    x = np.full((2, 500), -np.inf, np.float32)
    x[0, [400, 30]] = [1.0, 2.0]
    x[1, 77] = -3.0
    lp, h, ids, tlp = check_rows(ctx, x, [0, 77], 5)
    assert lp[0] == -np.inf and lp[1] == 0.0 and h[1] == 0.0
    assert ids[0].tolist() == [30, 400, 0, 1, 2] and ids[1].tolist() == [77, 0, 1, 2, 3]
    assert np.all(tlp[0, 2:] == -np.inf)


def test_extreme_logits(ctx):
    rng = np.random.default_rng(12)
    x = rng.normal(0, 1, (3, 4001)).astype(np.float32)
    x[0] *= 1e4
    x[1] = np.finfo(np.float32).min
    x[1, 9] = 3.0
    x[2, ::2] = np.finfo(np.float32).max
    x[2, 1::2] = np.finfo(np.float32).min
    check_rows(ctx, x, [17, 9, 4], 6)


def test_parts_on_their_own(ctx):
    rng = np.random.default_rng(2)
    x = rng.normal(0, 1, (3, 1000)).astype(np.float32)
    full = score(ctx, x, [1, 2, 3], 4)
    a = score(ctx, x, [1, 2, 3], 0, entropy=False)
    b = score(ctx, x, None, 4, entropy=False)
    c = score(ctx, x, None, 0)
    assert np.array_equal(a[0], full[0]) and np.array_equal(c[1], full[1])
    assert np.array_equal(b[2], full[2]) and np.array_equal(b[3], full[3])


def test_target_outside_the_vocabulary(ctx):
    x = np.zeros((2, 100), np.float32)
    t = torch.tensor([100, 5], dtype=torch.int32, device="cuda")
    lp = torch.zeros(2, device="cuda")
    xd = torch.from_numpy(x).cuda()
    torch.cuda.synchronize()
    check(lib().tmg_op_logprobs(ctx, P(xd), 100, 2, 100, P(t), 0, P(lp), None, None, None), ctx)
    with pytest.raises(TmgError) as e:
        check(lib().tmg_sync(ctx), ctx)
    assert e.value.code == -1 and "vocabulary" in str(e.value)
    lp = lp.cpu().numpy()
    assert np.isnan(lp[0]) and abs(lp[1] + np.log(100)) < 1e-5


def test_refusals(ctx):
    x = torch.zeros((4, 100), device="cuda")
    o = torch.full((4, 64), 3.0, device="cuda")
    ids = torch.zeros((4, 64), dtype=torch.int32, device="cuda")
    f = lib().tmg_op_logprobs
    for args in ((None, 100, 4, 100, P(ids), 0, P(o), None, None, None),
                 (P(x), 99, 4, 100, P(ids), 0, P(o), None, None, None),
                 (P(x), 100, -1, 100, P(ids), 0, P(o), None, None, None),
                 (P(x), 100, 4, 0, P(ids), 0, P(o), None, None, None),
                 (P(x, 2), 100, 4, 100, P(ids), 0, P(o), None, None, None),
                 (P(x), 100, 4, 100, None, 0, P(o), None, None, None),
                 (P(x), 100, 4, 100, P(ids), 0, None, P(o), None, None),
                 (P(x), 100, 4, 100, None, 65, None, None, P(ids), P(o)),
                 (P(x), 100, 4, 3, None, 4, None, None, P(ids), P(o)),
                 (P(x), 100, 4, 100, None, 4, None, None, None, P(o)),
                 (P(x), 100, 4, 100, None, 0, None, None, None, None)):
        assert f(ctx, *args) == -1
        assert b"logprobs" in lib().tmg_last_error(ctx)
    assert f(ctx, P(x), 100, 0, 100, P(ids), 0, P(o), None, None, None) == 0  # no rows
    check(lib().tmg_sync(ctx), ctx)
    assert bool((o == 3.0).all())


@pytest.mark.parametrize("rows,V,n_top", [(1, 40000, 8), (500, 3001, 20)])
def test_captured_and_replayed_on_two_contexts(ctx, rows, V, n_top):
    # two contexts' graphs in flight at once, each over its own buffers, replayed
    # for new logits: the results of calls one by one
    other = ctypes.c_void_p()
    check(lib().tmg_create(0, None, ctypes.byref(other)))
    rng = np.random.default_rng(rows)
    sets = []
    for c in (ctx, other):
        b = dict(c=c, x=torch.zeros((rows, V), device="cuda"),
                 t=torch.zeros(rows, dtype=torch.int32, device="cuda"),
                 lp=torch.zeros(rows, device="cuda"), h=torch.zeros(rows, device="cuda"),
                 ids=torch.zeros((rows, n_top), dtype=torch.int32, device="cuda"),
                 tlp=torch.zeros((rows, n_top), device="cuda"),
                 s=torch.cuda.ExternalStream(lib().tmg_stream(c)), g=torch.cuda.CUDAGraph())
        torch.cuda.synchronize()
        with torch.cuda.graph(b["g"], stream=b["s"]):
            for _ in range(2):  # the second call finds the first one's results in place
                check(lib().tmg_op_logprobs(c, P(b["x"]), V, rows, V, P(b["t"]), n_top, P(b["lp"]),
                                            P(b["h"]), P(b["ids"]), P(b["tlp"])), c)
        sets.append(b)
    for _ in range(3):
        host = []
        for b in sets:
            x = rng.normal(0, 3, (rows, V)).astype(np.float32)
            t = rng.integers(0, V, rows)
            b["x"].copy_(torch.from_numpy(x))
            b["t"].copy_(torch.from_numpy(t.astype(np.int32)))
            host.append((x, t))
        torch.cuda.synchronize()
        for _ in range(3):
            for b in sets:
                with torch.cuda.stream(b["s"]):
                    b["g"].replay()
        for b in sets:
            check(lib().tmg_sync(b["c"]), b["c"])
        for b, (x, t) in zip(sets, host):
            one = score(ctx, x, t, n_top)
            for name, want in zip(("lp", "h", "ids", "tlp"), one):
                assert np.array_equal(b[name].cpu().numpy(), want)
    for b in sets:
        del b["g"]
    lib().tmg_destroy(other)


def test_offsets_beyond_32_bits(ctx):
    # rows further apart than 2^32 bytes in all: the last ones, and a long row
    rows, V, ld = 40, 1003, 1 << 25
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB free")
    assert (rows - 1) * ld * 4 > 1 << 32
    rng = np.random.default_rng(9)
    x = rng.normal(0, 2, (rows, V)).astype(np.float32)
    check_rows(ctx, x, rng.integers(0, V, rows), 5, ld=ld)
    n = 1 << 24  # one row of 16M
    x = rng.normal(0, 2, (1, n)).astype(np.float32)
    x[0, n - 1] = 20.0
    check_rows(ctx, x, [n - 1], 3)
