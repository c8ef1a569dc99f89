"""The 4-bit KV cache (tmg_op_kv4_append, tmg_op_kv4_read) and the decode
attention over it (tmg_op_attn_decode_kv4) against numpy in 64 bits
(kv4_ref.py).

Codes and parameters are compared bit for bit: the format fixes every
rounding.  Values read back are one f32 rounding of m + code * s, so exact
too.

Attention tolerance, from the arithmetic: with A the largest sum of |q_i
k_i| / sqrt(d) behind a score, a score is off by at most 40 * 2^-24 * A (at
most 24 truncated or rounded partial sums and a few products of a
two-part operand with 22 bits), its probability by that much relative (and
2^-21 for exp2), which moves a weighted mean of v by at most twice that
times max |v|; the sums over positions add one rounding of 2^-24 for each
of at most 64 partial results.  Hence (80 A + 128) * 2^-24 * max |v|.
"""
import ctypes

import numpy as np
import pytest

import kv4_ref as R

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover - CPU box
    pytest.skip("needs a GPU", allow_module_level=True)

from tinyminigo_b200._lib import Kv4View, TmgError, check, lib  # noqa: E402

INVALID, CAPACITY = -1, -4
NAN_WORD = 0x7FC07FC0


@pytest.fixture(scope="module")
def ctx():
    h = ctypes.c_void_p()
    check(lib().tmg_create(0, None, ctypes.byref(h)))
    yield h
    lib().tmg_destroy(h)


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def P(t, off=0):
    return None if t is None else ctypes.c_void_p(t.data_ptr() + off)


class Cache:
    """Buffers of a 4-bit cache filled with a pattern, and their view."""

    def __init__(self, M, n_kv, d, cap, fill=0xA5, guard=64):
        g = min(d, 32)
        self.shape = (M, n_kv, cap)
        self.M, self.n_kv, self.d, self.cap, self.g = M, n_kv, d, cap, g
        self.guard = guard
        n = M * n_kv * cap

        def make(count, dtype, value):
            return torch.full((count + guard,), value, dtype=dtype, device="cuda")

        self.kc, self.vc = make(n * d // 2, torch.uint8, fill), make(n * d // 2, torch.uint8, fill)
        self.kp = make(n * d // g, torch.int32, NAN_WORD)
        self.vp = make(n * d // g, torch.int32, NAN_WORD)
        self.view = Kv4View(self.kc.data_ptr(), self.kp.data_ptr(), self.vc.data_ptr(),
                            self.vp.data_ptr(), M, n_kv, d, cap)

    def ref(self):
        return ctypes.byref(self.view)

    def host(self):
        """codes [M, n_kv, cap, d], params [M, n_kv, cap, d / g] of keys and values."""
        out = []
        for c, p in ((self.kc, self.kp), (self.vc, self.vp)):
            n = np.prod(self.shape)
            cc = c[:n * self.d // 2].cpu().numpy().reshape(*self.shape, self.d // 2)
            pp = p[:n * self.d // self.g].cpu().numpy().view(np.uint32)
            out.append((R.unpack(cc), pp.reshape(*self.shape, self.d // self.g)))
        return out

    def guards_intact(self, fill=0xA5):
        return bool((self.kc[-self.guard:] == fill).all() and (self.vc[-self.guard:] == fill).all()
                    and (self.kp[-self.guard:] == NAN_WORD).all()
                    and (self.vp[-self.guard:] == NAN_WORD).all())


def rows(rng, M, T, n_kv, d, extra=0):
    ld = 2 * n_kv * d + extra
    x = rng.normal(0, 1, (M, T, ld)).astype(np.float32)
    x[..., :n_kv * d] *= np.exp(rng.normal(0, 1, n_kv * d)).astype(np.float32)
    return x


def append(ctx, c, x, pos, count):
    w = c.n_kv * c.d
    xd, pd = dev(x), dev(np.asarray(pos, np.int32))
    cd = None if count is None else dev(np.asarray(count, np.int32))
    torch.cuda.synchronize()
    check(lib().tmg_op_kv4_append(ctx, c.ref(), P(xd), P(xd, 4 * w), x.shape[-1], x.shape[1],
                                  P(pd), P(cd)), ctx)
    check(lib().tmg_sync(ctx), ctx)


def read(ctx, c, pos, count, T, extra=0, want=(True, True)):
    ld = c.n_kv * c.d + extra
    out = [torch.full((c.M, T, ld), -7.0, device="cuda") if w else None for w in want]
    pd = dev(np.asarray(pos, np.int32))
    cd = None if count is None else dev(np.asarray(count, np.int32))
    torch.cuda.synchronize()
    check(lib().tmg_op_kv4_read(ctx, c.ref(), P(pd), P(cd), T, P(out[0]), P(out[1]), ld), ctx)
    check(lib().tmg_sync(ctx), ctx)
    return [None if o is None else o.cpu().numpy() for o in out]


@pytest.mark.parametrize("M,T,n_kv,d,cap,extra", [
    (1, 1, 1, 16, 4, 0), (1, 1, 8, 64, 64, 0), (3, 5, 2, 32, 16, 4), (2, 17, 3, 16, 40, 0),
    (4, 33, 2, 64, 100, 8), (2, 9, 3, 128, 24, 0), (1, 300, 8, 128, 300, 0), (16, 1, 8, 64, 32, 0)])
def test_append_and_read_bit_exact(ctx, M, T, n_kv, d, cap, extra):
    rng = np.random.default_rng(M * 1000 + T * 10 + d)
    x = rows(rng, M, T, n_kv, d, extra)
    pos = rng.integers(0, cap - T + 1, M)
    count = rng.integers(0, T + 1, M)
    count[0] = T
    c = Cache(M, n_kv, d, cap)
    append(ctx, c, x, pos, count)
    got = c.host()
    assert c.guards_intact()
    back = read(ctx, c, pos, count, T, extra)
    w = n_kv * d
    for i in range(2):
        codes, params = got[i]
        want_c = np.full((M, n_kv, cap, d), 5, np.uint8)
        want_c[..., 1::2] = 0xA
        want_p = np.full((M, n_kv, cap, d // c.g), NAN_WORD, np.uint32)
        want_v = np.full((M, T, w + extra), -7.0, np.float32)
        for m in range(M):
            n = count[m]
            xi = x[m, :n, i * w:(i + 1) * w].reshape(n, n_kv, d).transpose(1, 0, 2)
            qc, qp = R.quantise(xi)
            want_c[m, :, pos[m]:pos[m] + n] = qc
            want_p[m, :, pos[m]:pos[m] + n] = qp
            v = R.values(qc, qp)
            want_v[m, :n, :w] = v.transpose(1, 0, 2).reshape(n, w).astype(np.float32)
            half = np.repeat(R.steps(qp), c.g, -1).astype(np.float64) / 2
            assert np.all(np.abs(v - xi) <= half * (1 + 2.0 ** -20))
        assert np.array_equal(codes, want_c)
        assert np.array_equal(params, want_p)
        assert np.array_equal(back[i], want_v)


def test_append_special_values(ctx):
    # groups that are constant, zero, subnormal, huge, on ties, with NaN / inf
    rng = np.random.default_rng(4)
    d, n = 64, 64
    x = rng.normal(0, 1, (1, n, 2 * d)).astype(np.float32)
    x[0, 0, :32] = 0.0
    x[0, 1, :32] = -0.0
    x[0, 2, :32] = 100.3
    x[0, 3, :32] = -100.3
    x[0, 4, :32] *= np.float32(1e-40)
    x[0, 5, :32] *= np.float32(1e-45)
    x[0, 6, :32] *= np.float32(1e37)
    x[0, 7, 5] = np.nan
    x[0, 8, 40] = np.inf
    x[0, 9, 40] = -np.inf
    x[0, 10, 0], x[0, 10, 1] = 3e38, -3e38  # wider than f32
    x[0, 11, 0] = -np.finfo(np.float32).max  # no bf16 below it
    x[0, 12, :32] = np.arange(32, dtype=np.float32) * 0.5  # ties: codes at .5
    x[0, 13, :32] = np.arange(32, dtype=np.float32) / 2 - 7.5
    x[0, 14, :32] = 1e-30
    x[0, 14, 3] = -15.0
    x[0, 15, :32] = np.float32(1e-20) * rng.normal(0, 1, 32)
    x[0, 15, 7] = 5.0
    for i in range(16, 40):  # near ties: quotients a few ulps from .5
        s = np.float32(2.0 ** rng.integers(-4, 5))
        k = rng.integers(0, 15, 32) + np.float32(0.5)
        x[0, i, :32] = np.nextafter(k * s, np.float32(rng.choice([-1e9, 1e9]))).astype(np.float32)
        x[0, i, 0], x[0, i, 1] = 0.0, 15.0 * s
    c = Cache(1, 1, d, n)
    append(ctx, c, x, [0], None)
    (kc, kp), (vc, vp) = c.host()
    for got_c, got_p, part in ((kc, kp, x[0, :, :d]), (vc, vp, x[0, :, d:])):
        qc, qp = R.quantise(part)
        assert np.array_equal(got_p[0, 0], qp)
        assert np.array_equal(got_c[0, 0], qc)
    k, _ = read(ctx, c, [0], None, n)
    bad = np.isnan(k[0]).reshape(n, 2, 32).all(-1)
    assert [tuple(i) for i in np.argwhere(bad)] == [(7, 0), (8, 1), (9, 1), (10, 0), (11, 0)]
    assert np.isnan(k[0]).sum() == 5 * 32
    # a constant between two bf16: the group's step covers its distance to the lower
    assert np.all(np.abs(k[0, 2, :32] - np.float32(100.3)) <= R.steps(kp[0, 0, 2, 0]) / 2)
    assert np.all(k[0, :2, :32] == 0)


def test_read_one_side_and_ragged_positions(ctx):
    rng = np.random.default_rng(8)
    c = Cache(2, 2, 32, 64)
    x = rows(rng, 2, 64, 2, 32)
    append(ctx, c, x, [0, 0], None)
    k, v = read(ctx, c, [10, 3], [4, 0], 7, want=(True, False))
    assert v is None and np.all(k[1] == -7.0) and np.all(k[0, 4:] == -7.0)
    qc, qp = R.quantise(x[0, 10:14, :64].reshape(4, 2, 32))
    assert np.array_equal(k[0, :4], R.values(qc, qp).reshape(4, 64).astype(np.float32))


def test_positions_outside_the_cache(ctx):
    # skipped, reported by tmg_sync, the other rows written; counts beyond T
    # or below 0 are the nearer bound
    rng = np.random.default_rng(9)
    c = Cache(3, 2, 64, 8)
    x = rows(rng, 3, 4, 2, 64)
    with pytest.raises(TmgError) as e:
        append(ctx, c, x, [6, -2, 4], [4, 4, 99])
    assert e.value.code == CAPACITY
    check(lib().tmg_sync(ctx), ctx)  # reported once
    (kc, kp), _ = c.host()
    assert c.guards_intact()
    written = (kp != NAN_WORD).all((1, 3))
    assert written.tolist() == [[False] * 6 + [True] * 2, [True] * 2 + [False] * 6,
                                [False] * 4 + [True] * 4]
    with pytest.raises(TmgError) as e:
        read(ctx, c, [6, 0, 4], [3, -5, 0], 4)
    assert e.value.code == CAPACITY


def test_large_offsets(ctx):
    # a cache whose codes lie beyond 2^32 bytes: the last stream's rows
    M, n_kv, d, cap = 9, 8, 128, 1 << 20
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip("needs 30 GB free")
    c = Cache(M, n_kv, d, cap)
    assert (M - 1) * n_kv * cap * d // 2 >= 1 << 32
    rng = np.random.default_rng(2)
    x = rows(rng, M, 3, n_kv, d)
    pos, count = [0] * (M - 1) + [cap - 3], [0] * (M - 1) + [3]
    append(ctx, c, x, pos, count)
    back = read(ctx, c, pos, count, 3)
    for i in range(2):
        xi = x[M - 1, :, i * n_kv * d:(i + 1) * n_kv * d].reshape(3, n_kv, d)
        want = R.values(*R.quantise(xi)).astype(np.float32).reshape(3, -1)
        assert np.array_equal(back[i][M - 1], want)
    assert c.guards_intact()


def test_more_rows_than_a_grid_has_blocks(ctx):
    # 65535 blocks of 32 rows (heads of 128) and some: the blocks go round
    T, d = 65535 * 32 + 75, 128
    if torch.cuda.mem_get_info()[0] < 20 << 30:
        pytest.skip("needs 20 GB free")
    cap = (T + 3) // 4 * 4
    c = Cache(1, 1, d, cap)
    x = torch.randn(T, 2 * d, generator=torch.Generator(device="cuda").manual_seed(3),
                    device="cuda")
    out = torch.full((2, T, d), -7.0, device="cuda")
    pos = torch.zeros(1, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    check(lib().tmg_op_kv4_append(ctx, c.ref(), P(x), P(x, 4 * d), 2 * d, T, P(pos), None), ctx)
    check(lib().tmg_op_kv4_read(ctx, c.ref(), P(pos), None, T, P(out[0]), P(out[1]), d), ctx)
    check(lib().tmg_sync(ctx), ctx)
    assert c.guards_intact() and not bool((out == -7.0).any())
    for at in (0, 65535 * 16, 65535 * 32 - 5, T - 80):
        part = x[at:at + 80].cpu().numpy()
        for i in range(2):
            want = R.values(*R.quantise(part[:, i * d:(i + 1) * d])).astype(np.float32)
            assert np.array_equal(out[i, at:at + 80].cpu().numpy(), want)


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------
def filled(rng, M, n_kv, d, cap, lens, loud=1.0):
    """A cache whose rows below lens hold keys and values and whose other rows
    hold NaN parameters and arbitrary codes."""
    c = Cache(M, n_kv, d, cap)
    for codes, params, scale in ((c.kc, c.kp, loud), (c.vc, c.vp, 1.0)):
        x = (rng.normal(0, scale, (M, n_kv, cap, d))).astype(np.float32)
        qc, qp = R.quantise(x)
        for m in range(M):
            qp[m, :, lens[m]:] = NAN_WORD
        n = M * n_kv * cap
        codes[:n * d // 2] = dev(R.pack(qc).reshape(-1))
        params[:n * d // c.g] = dev(qp.reshape(-1).view(np.int32))
    return c


def workspace(ctx, c, n_q):
    b = ctypes.c_int64()
    check(lib().tmg_op_attn_decode_kv4_ws(ctx, c.ref(), n_q, ctypes.byref(b)), ctx)
    # filled with NaN patterns: its contents are of no matter
    return torch.full((b.value + 16,), 0xFF, dtype=torch.uint8, device="cuda"), b.value


def attend(ctx, c, q, lens, max_len=None, extra=0, ws=None):
    M, n_q, d = q.shape
    ld = n_q * d + extra
    qd = torch.full((M, ld), float("nan"), device="cuda")
    qd[:, :n_q * d] = dev(q.reshape(M, n_q * d))
    out = torch.full((M, ld), -7.0, device="cuda")
    ln = dev(np.asarray(lens, np.int32))
    buf, n = ws or workspace(ctx, c, n_q)
    torch.cuda.synchronize()
    check(lib().tmg_op_attn_decode_kv4(ctx, c.ref(), P(qd), ld, P(ln),
                                       c.cap if max_len is None else max_len, n_q, P(out), ld,
                                       P(buf), n), ctx)
    check(lib().tmg_sync(ctx), ctx)
    assert bool((buf[n:] == 0xFF).all())
    out = out.cpu().numpy()
    assert np.all(out[:, n_q * d:] == -7.0)
    return out[:, :n_q * d].reshape(M, n_q, d)


def expect(c, q, lens):
    (kc, kp), (vc, vp) = c.host()
    refs, tols = [], []
    for m in range(c.M):
        n = lens[m]
        k = R.values(kc[m, :, :n], kp[m, :, :n]).transpose(1, 0, 2)
        v = R.values(vc[m, :, :n], vp[m, :, :n]).transpose(1, 0, 2)
        o, A = R.attention(q[m], k, v)
        refs.append(o)
        tols.append((80 * A + 128) * 2.0 ** -24 * (np.abs(v).max() if n else 0.0))
    return refs, tols


def check_attention(ctx, c, q, lens, **kw):
    out = attend(ctx, c, q, lens, **kw)
    refs, tols = expect(c, q, lens)
    for m in range(c.M):
        err = np.abs(out[m] - refs[m]).max()
        assert err <= tols[m], (m, lens[m], err, tols[m])
    return out


@pytest.mark.parametrize("d", [16, 32, 64, 128])
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 200, 517])
def test_attention_lengths(ctx, d, n):
    rng = np.random.default_rng(n * 7 + d)
    cap = (n + 3) // 4 * 4
    c = filled(rng, 1, 2, d, cap, [n])
    q = rng.normal(0, 1.5, (1, 8, d)).astype(np.float32)
    check_attention(ctx, c, q, [n])


@pytest.mark.parametrize("d", [16, 32, 64, 128])
@pytest.mark.parametrize("n_kv,group", [(1, 1), (3, 2), (2, 3), (8, 4), (1, 5), (2, 7), (2, 8),
                                        (1, 9), (3, 16)])
def test_attention_heads_and_ragged_lengths(ctx, d, n_kv, group):
    rng = np.random.default_rng(d + n_kv * 100 + group)
    cap = 700
    lens = [700, 0, 1, 333, 64, 699, 5]
    c = filled(rng, len(lens), n_kv, d, cap, lens)
    q = rng.normal(0, 1.5, (len(lens), n_kv * group, d)).astype(np.float32)
    out = check_attention(ctx, c, q, lens, extra=4)
    assert np.all(out[1] == 0.0)


@pytest.mark.parametrize("M,n_kv,group,d,n", [(1, 8, 4, 64, 20000), (1, 1, 4, 128, 9001),
                                              (1, 2, 16, 32, 5000), (5, 1, 1, 64, 4099),
                                              (1, 1, 1, 16, 3001)])
def test_attention_long(ctx, M, n_kv, group, d, n):
    rng = np.random.default_rng(n + d)
    lens = [n] + [int(v) for v in rng.integers(0, n, M - 1)]
    c = filled(rng, M, n_kv, d, (n + 3) // 4 * 4, lens)
    q = rng.normal(0, 1.0, (M, n_kv * group, d)).astype(np.float32)
    a = check_attention(ctx, c, q, lens)
    b = attend(ctx, c, q, lens)
    assert np.array_equal(a, b)  # sums have a fixed order


def test_attention_many_short_streams(ctx):
    rng = np.random.default_rng(77)
    M, n_kv, d = 300, 2, 64
    lens = [int(v) for v in rng.integers(0, 40, M)]
    c = filled(rng, M, n_kv, d, 40, lens)
    q = rng.normal(0, 1.0, (M, 8, d)).astype(np.float32)
    out = check_attention(ctx, c, q, lens)
    for m in range(M):
        if lens[m] == 0:
            assert np.all(out[m] == 0.0)


@pytest.mark.parametrize("d", [32, 64, 128])
def test_attention_value_ranges(ctx, d):
    # loud keys (one position takes all the weight), queries and values over
    # the range of f32 exponents, one position with a far larger step
    rng = np.random.default_rng(d)
    lens = [150]
    for qs, vs in ((30.0, 1.0), (1.0, 1e30), (1e-3, 1e-30), (1e20, 1.0)):
        c = filled(rng, 1, 2, d, 152, lens)
        x = (rng.normal(0, 1, (1, 2, 152, d)) * vs).astype(np.float32)
        x[0, :, 40] *= np.float32(1e4)
        qc, qp = R.quantise(x)
        c.vc[:qc.size // 2] = dev(R.pack(qc).reshape(-1))
        c.vp[:qp.size] = dev(qp.reshape(-1).view(np.int32))
        q = rng.normal(0, qs, (1, 8, d)).astype(np.float32)
        if qs == 1e20:
            q = (q * 0 + rng.normal(0, 1, q.shape)).astype(np.float32)
            q[0, 0] *= np.float32(1e-20)  # one head far quieter than the others
        check_attention(ctx, c, q, lens)


@pytest.mark.parametrize("d", [16, 32, 64, 128])
@pytest.mark.parametrize("n,at", [(150, 3), (150, 149), (5000, 4321)])
@pytest.mark.parametrize("low", [False, True])
def test_attention_far_scores(ctx, d, n, at, low):
    # scores of up to +-1e37, one position ahead of all others by more than any
    # rounding: its value comes back.  Tolerance: p s in two f16 parts (2^-22)
    # against codes of up to 8 steps, p (m + 8 s) and the division with a few
    # roundings of 2^-24, of numbers up to 3 max |v|: 2^-19 max |v|
    rng = np.random.default_rng(d + n + at)
    cap = (n + 3) // 4 * 4
    for scale in (1e3, 1e7, 1e15, 1e30, 1e36):
        q = (rng.normal(0, 1, (1, 8, d)) * scale).astype(np.float32)
        q[0, 1] = rng.normal(0, 1, d)  # heads of one kv head far apart
        c = filled(rng, 1, 4, d, cap, [n])
        x = rng.normal(0, 1, (1, 4, cap, d))
        along = np.sign(q[0, ::2])  # the first of a kv head's two heads
        if low:
            x = 0.1 * x - 8 * along[None, :, None]
            x[0, :, at] = -2 * along
        else:
            x[0, :, at] = 8 * along
        qc, qp = R.quantise(x.astype(np.float32))
        qp[0, :, n:] = NAN_WORD
        c.kc[:qc.size // 2] = dev(R.pack(qc).reshape(-1))
        c.kp[:qp.size] = dev(qp.reshape(-1).view(np.int32))
        out = attend(ctx, c, q, [n])
        refs, tols = expect(c, q, [n])
        (kc, kp), (vc, vp) = c.host()
        v = R.values(vc[0, :, at], vp[0, :, at])
        vmax = np.abs(R.values(vc[0, :, :n], vp[0, :, :n])).max()
        assert np.abs(refs[0][::2] - v).max() <= 1e-9  # the premise
        assert np.abs(out[0, ::2] - v).max() <= 2.0 ** -19 * vmax
        k0 = R.values(kc[0, :1, :n], kp[0, :1, :n]).transpose(1, 0, 2)
        o, A = R.attention(q[0, 1:2], k0, R.values(vc[0, :1, :n], vp[0, :1, :n]).transpose(1, 0, 2))
        assert np.abs(out[0, 1] - o[0]).max() <= (80 * A + 128) * 2.0 ** -24 * vmax
        assert np.isfinite(out).all()


@pytest.mark.parametrize("d", [32, 128])
def test_attention_queries_near_the_end_of_f32(ctx, d):
    # |q| of 1e36 against keys of 1e-36: ordinary scores
    rng = np.random.default_rng(d)
    c = filled(rng, 1, 2, d, 300, [300], loud=2e-36)
    q = (rng.normal(0, 1, (1, 8, d)) * 1e36).astype(np.float32)
    q[0, 3] *= np.float32(1e-36)
    check_attention(ctx, c, q, [300])


@pytest.mark.parametrize("M", [31, 32, 33, 512, 513, 1024])
@pytest.mark.parametrize("group", [4, 8])
def test_attention_numbers_of_streams(ctx, M, group):
    rng = np.random.default_rng(M)
    lens = [int(v) for v in rng.integers(0, 200, M)]
    lens[-1], lens[0] = 200, 0
    c = filled(rng, M, 1, 32, 200, lens)
    q = rng.normal(0, 1.0, (M, group, 32)).astype(np.float32)
    out = check_attention(ctx, c, q, lens)
    assert np.all(out[0] == 0.0)


@pytest.mark.parametrize("M", [3, 40, 1024])
def test_attention_of_empty_streams(ctx, M):
    c = Cache(M, 2, 64, 4096)  # nothing written: NaN parameters
    q = np.random.default_rng(M).normal(0, 1, (M, 4, 64)).astype(np.float32)
    assert np.all(attend(ctx, c, q, [0] * M) == 0.0)


@pytest.mark.parametrize("d,tiles", [(64, 64), (128, 32)])
@pytest.mark.parametrize("n_kv,group", [(1, 16), (5, 8), (80, 2), (148, 1), (149, 1),
                                        (197, 1), (198, 1)])
def test_attention_around_the_split(ctx, d, tiles, n_kv, group):
    # bounds of 32 and 64 tiles a head group, with and without a join
    rng = np.random.default_rng(n_kv + d)
    for n in (32 * tiles, 32 * tiles + 4, 64 * tiles, 64 * tiles + 4):
        if n_kv > 80 and n > 32 * tiles + 4:
            continue
        c = filled(rng, 1, n_kv, d, n, [n])
        q = rng.normal(0, 1.0, (1, n_kv * group, d)).astype(np.float32)
        check_attention(ctx, c, q, [n])


def test_attention_beyond_32_bit_offsets(ctx):
    # the last streams of a cache whose codes lie beyond 2^32 bytes
    M, n_kv, d, cap = 9, 8, 128, 1 << 20
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB free")
    small = filled(np.random.default_rng(1), 1, n_kv, d, 2000, [2000])
    c = Cache(M, n_kv, d, cap)
    for big, part, w in ((c.kc, small.kc, d // 2), (c.vc, small.vc, d // 2),
                         (c.kp, small.kp, d // 32), (c.vp, small.vp, d // 32)):
        n = n_kv * cap * w
        to = big[(M - 1) * n:M * n].view(n_kv, cap, w)
        to[:, :2000] = part[:n_kv * 2000 * w].view(n_kv, 2000, w)
    q = np.random.default_rng(2).normal(0, 1, (M, 16, d)).astype(np.float32)
    out = attend(ctx, c, q, [0] * (M - 1) + [2000])
    refs, tols = expect(small, q[M - 1:], [2000])
    assert np.abs(out[M - 1] - refs[0]).max() <= tols[0]
    assert np.all(out[:M - 1] == 0.0)


def test_attention_nan_rows_stay_in_their_head(ctx):
    rng = np.random.default_rng(5)
    d, lens = 64, [100, 100]
    c = filled(rng, 2, 2, d, 100, lens)
    # a NaN key group of stream 0's kv head 1; a NaN value group of stream 1's
    # kv head 0 (its second group)
    c.kp[(0 * 2 + 1) * 100 * 2 + 50 * 2] = NAN_WORD
    c.vp[(1 * 2 + 0) * 100 * 2 + 20 * 2 + 1] = NAN_WORD
    q = rng.normal(0, 1, (2, 8, d)).astype(np.float32)
    out = attend(ctx, c, q, lens)
    nan = np.isnan(out)
    assert nan[0, 4:].all() and not nan[0, :4].any()
    assert nan[1, :4, 32:].all() and not nan[1, :4, :32].any() and not nan[1, 4:].any()


@pytest.mark.parametrize("n", [92, 6000])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_attention_bad_queries_stay_in_their_head(ctx, n, value):
    rng = np.random.default_rng(n)
    for d, group in ((64, 4), (128, 8)):
        c = filled(rng, 2, 2, d, n, [n, n])
        q = rng.normal(0, 1, (2, 2 * group, d)).astype(np.float32)
        clean = attend(ctx, c, q, [n, n])
        q[1, 1, 7] = value
        out = attend(ctx, c, q, [n, n])
        refs, tols = expect(c, np.where(np.isfinite(q), q, 0), [n, n])
        assert np.isnan(out[1, 1]).all() and np.array_equal(out[0], clean[0])
        rest = [h for h in range(2 * group) if h != 1]
        assert np.abs(out[1, rest] - refs[1][rest]).max() <= tols[1]


def test_attention_over_its_own_query(ctx):
    # out may be q: a head group's query is read before its output is written
    rng = np.random.default_rng(3)
    for M, n, d in ((2, 300, 64), (3, 20000, 64), (40, 700, 128)):
        lens = [int(v) for v in rng.integers(0, n, M)]
        lens[0] = n
        c = filled(rng, M, 2, d, (n + 3) // 4 * 4, lens)
        q = rng.normal(0, 1, (M, 8, d)).astype(np.float32)
        want = attend(ctx, c, q, lens)
        x, ln = dev(q.reshape(M, 8 * d)), dev(np.asarray(lens, np.int32))
        ws, size = workspace(ctx, c, 8)
        torch.cuda.synchronize()
        check(lib().tmg_op_attn_decode_kv4(ctx, c.ref(), P(x), 8 * d, P(ln), c.cap, 8, P(x), 8 * d,
                                           P(ws), size), ctx)
        check(lib().tmg_sync(ctx), ctx)
        assert np.array_equal(x.cpu().numpy().reshape(M, 8, d), want)


def test_attention_length_out_of_range(ctx):
    rng = np.random.default_rng(6)
    c = filled(rng, 2, 2, 64, 64, [64, 64])
    q = rng.normal(0, 1, (2, 4, 64)).astype(np.float32)
    for lens, bound in (([65, 3], 64), ([-1, 3], 64), ([33, 3], 32)):
        with pytest.raises(TmgError) as e:
            attend(ctx, c, q, lens, max_len=bound)
        assert e.value.code == INVALID
    out = attend(ctx, c, q, [0, 0], max_len=0)
    assert np.all(out == 0.0)


@pytest.mark.parametrize("bad", ["head_dim", "capacity", "streams", "group", "ld", "ws", "align",
                                 "null", "max_len"])
def test_refusals(ctx, bad):
    # nothing is enqueued: the outputs keep their contents
    c = Cache(2, 2, 64, 64)
    x = torch.zeros((2, 4, 256), device="cuda")
    pos = torch.zeros(2, dtype=torch.int32, device="cuda")
    q, out = torch.zeros((2, 256), device="cuda"), torch.full((2, 256), 3.0, device="cuda")
    ws, n = workspace(ctx, c, 4)
    v = Kv4View.from_buffer_copy(c.view)
    n_q, ld, off, wsb, max_len, T, row_ld = 4, 256, 0, n, 64, 4, 256
    if bad == "head_dim":
        v.head_dim = 48
    elif bad == "capacity":
        v.capacity = 62
    elif bad == "streams":
        v.n_streams = 0
    elif bad == "group":
        n_q = 5
    elif bad == "ld":
        ld = row_ld = 255
    elif bad == "ws":
        wsb = n - 1
        if n == 0:
            pytest.skip("this shape needs no workspace")
    elif bad == "align":
        off = 4
    elif bad == "null":
        v.v_params = None
    elif bad == "max_len":
        max_len, T = 65, 65
    r = ctypes.byref(v)
    torch.cuda.synchronize()
    rc = lib().tmg_op_attn_decode_kv4(ctx, r, P(q, off), ld, P(pos), max_len, n_q, P(out), ld,
                                      P(ws), wsb)
    assert rc == INVALID and b"attn_decode_kv4" in lib().tmg_last_error(ctx)
    if bad not in ("group", "ws"):
        assert lib().tmg_op_kv4_append(ctx, r, P(x, off), P(x, 512), row_ld, T, P(pos),
                                       None) == INVALID
        assert b"kv4_append" in lib().tmg_last_error(ctx)
        assert lib().tmg_op_kv4_read(ctx, r, P(pos), None, T, P(x, off), None, row_ld) == INVALID
        assert b"kv4_read" in lib().tmg_last_error(ctx)
    check(lib().tmg_sync(ctx), ctx)
    assert bool((out == 3.0).all()) and c.guards_intact() and bool((c.kc == 0xA5).all())


def test_captured_and_replayed(ctx):
    # a step (append, attend) captured into a graph on the context's stream
    # and replayed on other inputs and lengths gives the eager calls' bits
    rng = np.random.default_rng(31)
    M, n_kv, n_q, d, cap = 3, 2, 8, 64, 400
    lens = [399, 17, 250]
    c = filled(rng, M, n_kv, d, cap, lens)
    w = n_kv * d
    x = torch.zeros((M, 1, 2 * w), device="cuda")
    q = torch.zeros((M, n_q * d), device="cuda")
    out = torch.zeros((M, n_q * d), device="cuda")
    pos = torch.zeros(M, dtype=torch.int32, device="cuda")
    now = torch.zeros(M, dtype=torch.int32, device="cuda")
    ws, n = workspace(ctx, c, n_q)

    def step():
        check(lib().tmg_op_kv4_append(ctx, c.ref(), P(x), P(x, 4 * w), 2 * w, 1, P(pos), None),
              ctx)
        check(lib().tmg_op_attn_decode_kv4(ctx, c.ref(), P(q), n_q * d, P(now), cap, n_q, P(out),
                                           n_q * d, P(ws), n), ctx)

    stream = torch.cuda.ExternalStream(lib().tmg_stream(ctx))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    for i in range(3):
        x.copy_(dev(rng.normal(0, 1, tuple(x.shape)).astype(np.float32)))
        q.copy_(dev(rng.normal(0, 1, tuple(q.shape)).astype(np.float32)))
        pos.copy_(dev(np.asarray([lens[0] - i, lens[1] + i, lens[2]], np.int32)))
        now.copy_(pos + 1)
        out.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        check(lib().tmg_sync(ctx), ctx)
        got = out.clone()
        torch.cuda.synchronize()
        out.zero_()
        torch.cuda.synchronize()
        step()
        check(lib().tmg_sync(ctx), ctx)
        assert torch.equal(got, out)
        refs, tols = expect(c, q.cpu().numpy().reshape(M, n_q, d), now.cpu().tolist())
        for m in range(M):
            assert np.abs(got[m].cpu().numpy().reshape(n_q, d) - refs[m]).max() <= tols[m]
    del graph


def test_captured_behind_other_work(ctx):
    # a copy and a kernel of the caller's before the calls, in one graph, and
    # the lengths read from what that copy brings
    rng = np.random.default_rng(32)
    M, n_kv, n_q, d, cap = 2, 2, 8, 128, 4096
    lens = [4096, 2500]
    c = filled(rng, M, n_kv, d, cap, lens)
    src = torch.zeros((M, n_q * d), device="cuda")
    q = torch.zeros_like(src)
    now, new = (torch.zeros(M, dtype=torch.int32, device="cuda") for _ in range(2))
    out = torch.zeros_like(src)
    ws, n = workspace(ctx, c, n_q)
    stream = torch.cuda.ExternalStream(lib().tmg_stream(ctx))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        torch.mul(src, 0.5, out=q)
        now.copy_(new)
        check(lib().tmg_op_attn_decode_kv4(ctx, c.ref(), P(q), n_q * d, P(now), cap, n_q, P(out),
                                           n_q * d, P(ws), n), ctx)
        out.mul_(2.0)
    for lens in ([4096, 2500], [3, 2222], [0, 2049]):
        src.copy_(dev(rng.normal(0, 2, tuple(src.shape)).astype(np.float32)))
        new.copy_(dev(np.asarray(lens, np.int32)))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
            graph.replay()
        check(lib().tmg_sync(ctx), ctx)
        refs, tols = expect(c, q.cpu().numpy().reshape(M, n_q, d), lens)
        for m in range(M):
            assert np.abs(out[m].cpu().numpy().reshape(n_q, d) / 2 - refs[m]).max() <= tols[m]
    del graph


def test_two_contexts_at_once(ctx):
    # two contexts (two streams) over one cache, a workspace each
    h = ctypes.c_void_p()
    check(lib().tmg_create(0, None, ctypes.byref(h)))
    try:
        rng = np.random.default_rng(41)
        n = 6000
        c = filled(rng, 1, 8, 64, n, [n])
        qs = [dev(rng.normal(0, 1, (1, 32 * 64)).astype(np.float32)) for _ in range(2)]
        ln = dev(np.asarray([n], np.int32))
        outs = [torch.zeros(1, 32 * 64, device="cuda") for _ in range(2)]
        ws = [workspace(ctx, c, 32) for _ in range(2)]
        torch.cuda.synchronize()
        for _ in range(20):
            for i, cx in enumerate((ctx, h)):
                check(lib().tmg_op_attn_decode_kv4(cx, c.ref(), P(qs[i]), 2048, P(ln), n, 32,
                                                   P(outs[i]), 2048, P(ws[i][0]), ws[i][1]), cx)
        check(lib().tmg_sync(ctx), ctx)
        check(lib().tmg_sync(h), h)
        for i in range(2):
            refs, tols = expect(c, qs[i].cpu().numpy().reshape(1, 32, 64), [n])
            assert np.abs(outs[i].cpu().numpy().reshape(32, 64) - refs[0]).max() <= tols[0]
    finally:
        lib().tmg_destroy(h)
