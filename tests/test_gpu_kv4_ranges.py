"""Decode attention over the 4-bit cache where the magnitudes of its values
differ: constant groups (step 0), groups and positions far apart, values next
to the end of f32 (tmg_op_attn_decode_kv4 against kv4_ref.py in 64 bits).

The tolerance is each output's own.  With b_t the largest magnitude that the
16 codes of a position's group stand for, max(|m|, |m + 15 s|), and p the
probabilities, W = sum_t p_t b_t is what the group's columns are made of.  A
score is off by at most 40 * 2^-24 * A (A: the largest sum of |q_i k_i| /
sqrt(d) behind one) and a probability by that and 2^-21 (exp2) relative,
which moves a weighted mean by at most twice that times W.  A product p s
has two f16 parts: 2^-21 of p s (|c - 8| <= 8 and s <= 2 b / 15 make that
2^-20 W) and, for parts below f16's normal range, 2^-25 of the largest, n
times and times 8 steps of at most 2 b / 15: n 2^-24 W.  Sums: at most 200
roundings of 2^-24 (a lane's positions of a warp, slots, partial results).
Hence (80 A + 256 + n) 2^-24 W, and 2^-148 where f32 ends.
"""
import ctypes

import numpy as np
import pytest

import kv4_ref as R

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover - CPU box
    pytest.skip("needs a GPU", allow_module_level=True)

from test_gpu_kv4 import Cache, attend, dev, filled  # noqa: E402

from tinyminigo_b200._lib import check, lib  # noqa: E402


@pytest.fixture(scope="module")
def ctx():
    h = ctypes.c_void_p()
    check(lib().tmg_create(0, None, ctypes.byref(h)))
    yield h
    lib().tmg_destroy(h)


def bf16_bits(x):
    """The pattern of a bf16 number."""
    b = np.asarray(x, np.float32).view(np.uint32)
    assert np.all(b & 0xFFFF == 0)
    return b >> 16


def set_values(c, codes=None, params=None, keys=False):
    """Codes [M, n_kv, cap, d] and params [M, n_kv, cap, d / g] of the values."""
    cc, pp = (c.kc, c.kp) if keys else (c.vc, c.vp)
    if codes is not None:
        cc[:codes.size // 2] = dev(R.pack(codes).reshape(-1))
    if params is not None:
        pp[:params.size] = dev(np.ascontiguousarray(params).reshape(-1).view(np.int32))


def compare(ctx, c, q, lens, copies=1):
    """The attention against 64 bits, each output within its own tolerance; of `copies`
    of the heads the first, which the others equal."""
    out = attend(ctx, c, q, lens)
    again = out.reshape(out.shape[0], copies, -1)
    assert np.array_equal(again, np.broadcast_to(again[:, :1], again.shape))
    (kc, kp), (vc, vp) = c.host()
    M, n_q, d = q.shape
    per = n_q // c.n_kv
    for m in range(M):
        n = lens[m]
        if n == 0:
            assert np.all(out[m] == 0.0)
            continue
        k = R.values(kc[m, :, :n], kp[m, :, :n])
        v = R.values(vc[m, :, :n], vp[m, :, :n])
        low = R.bf16_value(vp[m, :, :n] >> np.uint32(16)).astype(np.float64)
        b = np.maximum(np.abs(low), np.abs(low + 15.0 * R.steps(vp[m, :, :n])))
        for h in range(n_q // copies):
            kv = h // per
            x = k[kv] @ q[m, h].astype(np.float64) / np.sqrt(d)
            A = (np.abs(k[kv]) @ np.abs(q[m, h].astype(np.float64))).max() / np.sqrt(d)
            p = np.exp(x - x.max())
            p /= p.sum()
            tol = np.repeat((80 * A + 256 + n) * 2.0 ** -24 * (p @ b[kv]), c.g) + 2.0 ** -148
            err = np.abs(out[m, h] - p @ v[kv])
            assert np.all(err <= tol), (m, h, np.nanmax(err / np.where(tol > 0, tol, 1e-300)))
    return out


CONSTANTS = [1.0, -1024.0, 2.0 ** 28, -float(R.bf16_value(R.bf16_down(np.float32(1e38))))]


@pytest.mark.parametrize("d", [16, 32, 64, 128])
@pytest.mark.parametrize("n", [1, 64, 131072])
@pytest.mark.parametrize("equal", [True, False])
def test_constant_value_groups(ctx, d, n, equal):
    # every group of every row one number, exact in bf16: that number comes back
    # (p adds up to 1 within the sums' roundings), with and without a split
    rng = np.random.default_rng(d + n)
    cap = (n + 3) // 4 * 4
    c = filled(rng, 1, 1, d, cap, [n])
    q = rng.normal(0, 0.0 if equal else 1.0, (1, 4, d)).astype(np.float32)
    for value in CONSTANTS:
        word = np.uint32(int(bf16_bits(value)) << 16)
        params = np.full((1, 1, cap, d // c.g), word, np.uint32)
        params[:, :, n:] = 0x7FC07FC0
        set_values(c, params=params)
        out = attend(ctx, c, q, [n])
        assert np.all(np.abs(out - value) <= 256 * 2.0 ** -24 * abs(value)), (value, out)


@pytest.mark.parametrize("d,group", [(16, 4), (32, 8), (64, 4), (64, 16), (128, 4), (128, 8)])
@pytest.mark.parametrize("n", [150, 2500])
@pytest.mark.parametrize("value", [1.0, 4096.0, 1e9, 1e30])
def test_constant_groups_beside_others(ctx, d, group, n, value):
    # one kv head's first group constant, the others ordinary and small; and some
    # constant rows among ordinary ones
    rng = np.random.default_rng(n + d)
    cap = (n + 3) // 4 * 4
    x = rng.normal(0, 1, (1, 2, cap, d)).astype(np.float32)
    x[0, 0, :, :min(d, 32)] = R.bf16_value(R.bf16_down(np.float32(value)))
    x[0, 0, :, 32:] *= np.float32(1e-3)
    x[0, 1, 5:n:7] = -R.bf16_value(R.bf16_down(np.float32(value)))
    c = filled(rng, 1, 2, d, cap, [n])
    codes, params = R.quantise(x)
    params[:, :, n:] = 0x7FC07FC0
    set_values(c, codes, params)
    q = rng.normal(0, 1, (1, 2 * group, d)).astype(np.float32)
    compare(ctx, c, q, [n])


def along(rng, n_kv, group, d):
    """Queries [1, n_kv * group, d], nearly the same for the heads of a kv head, and
    their directions [n_kv, d] (the score of direction * x is about x)."""
    base = rng.normal(0, 1, (n_kv, 1, d))
    q = base + rng.normal(0, 0.05, (n_kv, group, d))
    way = base[:, 0] * np.sqrt(d) / (base[:, 0] ** 2).sum(-1, keepdims=True)
    return q.reshape(1, n_kv * group, d).astype(np.float32), way


def put(rng, d, n, n_kv, group, values, scores=None, copies=1):
    """A cache of n positions with the values [1, n_kv, n, d]; keys of size 1, at the
    positions of `scores` along the queries, and the queries.  All of it `copies` times."""
    cap = (n + 3) // 4 * 4
    c = Cache(1, n_kv * copies, d, cap)
    q, way = along(rng, n_kv, group, d)
    k = rng.normal(0, 0.3, (1, n_kv, cap, d))
    for at, x in (scores or {}).items():
        k[0, :, at] = way * x
    x = np.zeros((1, n_kv, cap, d))
    x[:, :, :n] = values
    for part, keys in ((k, True), (x, False)):
        codes, params = R.quantise(part.astype(np.float32))
        params[:, :, n:] = 0x7FC07FC0
        set_values(c, np.tile(codes, (1, copies, 1, 1)), np.tile(params, (1, copies, 1, 1)), keys)
    return c, np.tile(q, (1, copies, 1))


@pytest.mark.parametrize("d", [16, 32, 64, 128])
@pytest.mark.parametrize("group", [1, 4, 5, 16])
@pytest.mark.parametrize("n", [1, 17, 64, 65, 517, 5000])
def test_each_output_within_its_own_tolerance(ctx, d, group, n):
    rng = np.random.default_rng(n + d + group)
    c = filled(rng, 1, 2, d, (n + 3) // 4 * 4, [n])
    q = rng.normal(0, 1, (1, 2 * group, d)).astype(np.float32)
    compare(ctx, c, q, [n])


@pytest.mark.parametrize("d,group", [(64, 4), (64, 8), (128, 4), (128, 16)])
@pytest.mark.parametrize("n", [150, 2500])
@pytest.mark.parametrize("e", [-100, -36, 10, 20, 30, 36, 60, 100])
def test_one_group_far_from_the_others(ctx, d, group, n, e):
    rng = np.random.default_rng(n + d + abs(e))
    v = rng.normal(0, 1, (1, 2, n, d))
    v[0, 1, :, 32:64] *= 2.0 ** e
    c, q = put(rng, d, n, 2, group, v)
    compare(ctx, c, q, [n])


@pytest.mark.parametrize("d,group", [(16, 4), (32, 16), (64, 4), (128, 4), (128, 8)])
@pytest.mark.parametrize("n,at", [(150, 3), (150, 130), (2500, 1300)])
@pytest.mark.parametrize("e", [13, 20, 30, 36, 60])
def test_a_wide_position_of_little_weight(ctx, d, group, n, at, e):
    # one position 2^e wider than the others, whose probability is about 2^-87
    rng = np.random.default_rng(n + d + e)
    v = rng.normal(0, 1, (1, 1, n, d))
    v[0, 0, at] *= 2.0 ** e
    c, q = put(rng, d, n, 1, group, v, {at: -60.0})
    compare(ctx, c, q, [n])


@pytest.mark.parametrize("d,group", [(16, 4), (32, 16), (64, 4), (128, 4), (128, 8)])
@pytest.mark.parametrize("n,at", [(150, 3), (150, 130), (2500, 1300)])
@pytest.mark.parametrize("e", [None, -13, -20, -30, -60])
def test_a_sink_of_small_values(ctx, d, group, n, at, e):
    # one position has nearly all the weight, the others 2^-36 each, and its values
    # are zeros or 2^e of the others'
    rng = np.random.default_rng(n + d + at)
    v = rng.normal(0, 1, (1, 1, n, d))
    v[0, 0, at] *= 0.0 if e is None else 2.0 ** e
    c, q = put(rng, d, n, 1, group, v, {at: 25.0})
    compare(ctx, c, q, [n])


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n", [150, 2500])
def test_groups_of_zeros(ctx, d, n):
    # a group of zeros throughout (heads padded to d): zeros come back; one that is
    # zero up to a position that has nearly all the weight, and not behind it
    rng = np.random.default_rng(n + d)
    v = rng.normal(0, 1, (1, 3, n, d))
    v[0, 0, :, d - 32:] = 0.0
    v[0, 1, :n // 2, :32] = 0.0
    v[0, 2, n // 2:, :32] = 0.0
    c, q = put(rng, d, n, 3, 4, v, {n // 2 - 1: 25.0})
    out = compare(ctx, c, q, [n])
    assert np.all(out[0, :4, d - 32:] == 0.0)
    assert np.all(compare(ctx, *put(rng, d, n, 3, 4, 0 * v), [n]) == 0.0)


@pytest.mark.parametrize("d", [16, 32, 64, 128])
@pytest.mark.parametrize("scale", [1e-38, 1e-30, 1e-12, 1e-7, 1e5, 1e12, 1e30, 1e37])
def test_values_of_any_size(ctx, d, scale):
    rng = np.random.default_rng(d)
    for n, group in ((1, 4), (200, 4), (200, 9), (3000, 4)):
        c, q = put(rng, d, n, 2, group, np.clip(rng.normal(0, 1, (1, 2, n, d)), -4, 4) * scale)
        compare(ctx, c, q, [n])


@pytest.mark.parametrize("d,group", [(16, 1), (32, 4), (64, 4), (64, 16), (128, 2), (128, 8)])
def test_steps_all_over(ctx, d, group):
    # every group of every position of its own size, over streams that several
    # CTAs share; the same bits twice
    rng = np.random.default_rng(d * group)
    lens, cap, n_kv = [9000, 0, 301, 64], 9000, 2
    x = rng.normal(0, 1, (4, n_kv, cap, d // min(d, 32), min(d, 32)))
    x *= 2.0 ** rng.integers(-60, 61, x.shape[:-1] + (1,))
    x[2] *= 2.0 ** -40
    c = filled(rng, 4, n_kv, d, cap, lens)
    codes, params = R.quantise(x.reshape(4, n_kv, cap, d).astype(np.float32))
    for m, n in enumerate(lens):
        params[m, :, n:] = 0x7FC07FC0
    set_values(c, codes, params)
    q = rng.normal(0, 1, (4, n_kv * group, d)).astype(np.float32)
    a = compare(ctx, c, q, lens)
    assert np.array_equal(a, attend(ctx, c, q, lens))


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("n", [150, 5000])
def test_far_scores_over_far_values(ctx, d, n):
    # scores of up to 1e30 (the weight is one position's), values 2^60 apart: the
    # position's values come back, each group within its own rounding
    rng = np.random.default_rng(n + d)
    at = n // 3
    v = rng.normal(0, 1, (1, 2, n, d))
    v[0, 0, ::5] *= 2.0 ** 60
    v[0, 1, :, :32] *= 2.0 ** -50
    c, q = put(rng, d, n, 2, 4, v, {at: 40.0})
    (_, _), (vc, vp) = c.host()
    want = R.values(vc[0, :, at], vp[0, :, at])
    low = R.bf16_value(vp[0, :, at] >> np.uint32(16)).astype(np.float64)
    b = np.repeat(np.maximum(np.abs(low), np.abs(low + 15.0 * R.steps(vp[0, :, at]))), 32, -1)
    out = attend(ctx, c, q * np.float32(1e30), [n])[0].reshape(2, 4, d)
    assert np.all(np.abs(out - want[:, None]) <= 64 * 2.0 ** -24 * b[:, None])


def test_nan_groups_stay_in_their_columns(ctx):
    rng = np.random.default_rng(12)
    d, n = 64, 300
    v = rng.normal(0, 1, (1, 2, n, d))
    v[0, :, 50] *= 2.0 ** 40
    c, q = put(rng, d, n, 2, 4, v)
    clean = attend(ctx, c, q, [n])
    for at in (0, 50, 120, 299):
        c, q2 = put(np.random.default_rng(12), d, n, 2, 4, v)
        c.vp[(1 * n + at) * 2 + 1] = 0x7FC07FC0
        out = attend(ctx, c, q, [n])
        assert np.isnan(out[0, 4:, 32:]).all()
        assert not np.isnan(out[0, 4:, :32]).any() and not np.isnan(out[0, :4]).any()
    assert np.isfinite(clean).all()


@pytest.mark.parametrize("d,group", [(16, 4), (32, 9), (64, 4), (128, 4), (128, 8)])
@pytest.mark.parametrize("base,e,score", [(0, 12, -15.0), (-15, 30, -25.0), (-15, 34, -30.0),
                                          (-18, 15, -12.0), (3, 17, -14.0)])
def test_a_wide_stretch_of_little_weight(ctx, d, group, base, e, score):
    # whole tiles of positions 2^e wider than those before and behind, each with so
    # much less weight that they make up about as much of the result.  So many head
    # groups that each stays on one SM: a warp takes 4 tiles (of 64 positions, of 32
    # for heads of 128) in a row.
    rng = np.random.default_rng(d + e)
    tile, copies = 32 if d == 128 else 64, 40 if group <= 8 else 20
    n = 64 * tile
    at = np.arange(n) // tile % 4 // 2 == 1 if e % 2 else np.arange(n) // tile % 4 == 1
    v = rng.normal(0, 2.0 ** base, (1, 2, n, d))
    v[0, :, at] *= 2.0 ** e
    c, q = put(rng, d, n, 2, group, v, {int(i): score for i in np.flatnonzero(at)}, copies)
    compare(ctx, c, q, [n], copies)


@pytest.mark.parametrize("d,group", [(16, 4), (64, 4), (64, 9), (128, 4)])
@pytest.mark.parametrize("e", [-30, -8, 8, 14, 30, 50])
def test_sizes_that_change_on_the_way(ctx, d, group, e):
    # stretches of one size, the other, constants and zeros, in a row of one warp
    rng = np.random.default_rng(d + abs(e))
    tile, copies = 32 if d == 128 else 64, 40 if group <= 8 else 20
    n = 64 * tile
    v = rng.normal(0, 1, (1, 2, n, d))
    kind = np.arange(n) // (tile // 2 + 5) % 11
    v[:, :, kind == 3] *= 2.0 ** e
    v[:, :, kind == 5] = 2.0 ** e
    v[:, :, kind == 8] *= 2.0 ** -e
    v[:, 1, kind == 9] = 0.0
    c, q = put(rng, d, n, 2, group, v, copies=copies)
    compare(ctx, c, q, [n], copies)


@pytest.mark.parametrize("d,group", [(16, 4), (64, 4), (64, 9), (128, 4)])
@pytest.mark.parametrize("scale", [1e-25, 1e-7, 1e-5, 1e-3, 1e3])
@pytest.mark.parametrize("score", [1e7, 1e12])
def test_scores_that_go_far_on_the_way(ctx, d, group, scale, score):
    # ordinary scores, and in the third tile of a warp one beyond all others: its
    # values come back, whatever their size
    rng = np.random.default_rng(d + group)
    tile, copies = 32 if d == 128 else 64, 40 if group <= 8 else 20
    n = 64 * tile
    at = 10 * tile + 5
    c, q = put(rng, d, n, 2, group, rng.normal(0, scale, (1, 2, n, d)), {at: score}, copies)
    (_, _), (vc, vp) = c.host()
    want = R.values(vc[0, :, at], vp[0, :, at])
    low = R.bf16_value(vp[0, :, at] >> np.uint32(16)).astype(np.float64)
    b = np.repeat(np.maximum(np.abs(low), np.abs(low + 15.0 * R.steps(vp[0, :, at]))), c.g, -1)
    out = attend(ctx, c, q, [n])[0].reshape(2 * copies, group, d)
    assert np.all(np.abs(out - want[:, None]) <= 64 * 2.0 ** -24 * b[:, None])
