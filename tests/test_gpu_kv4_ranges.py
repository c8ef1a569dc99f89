"""Decode attention over the 4-bit cache where the magnitudes of its values
differ: constant groups (step 0), groups and positions far apart, values next
to the end of f32 (tmg_op_attn_decode_kv4 against kv4_ref.py in 64 bits).

The tolerance is each output's own.  With b_t the largest magnitude that the
16 codes of a position's group stand for, max(|m|, |m + 15 s|), and p the
probabilities, W = sum_t p_t b_t is what the group's columns are made of.  A
score is off by at most 40 * 2^-24 * A (A: the largest sum of |q_i k_i| /
sqrt(d) behind one) and a probability by that and 2^-21 (exp2) relative,
which moves a weighted mean by at most twice that times W.  A product p s
has two f16 parts: 2^-21 of p s (|c - 8| <= 8 and s <= 2 b / 15 make that 2^-20 W) and,
for parts below f16's normal range, 2^-25 of the largest, n times and times 8
steps of at most 2 b / 15: n 2^-24 W.  Sums: at most 200 roundings of 2^-24
(a lane's positions of a warp, slots, partial results).  Hence
(80 A + 256 + n) 2^-24 W.
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


def compare(ctx, c, q, lens):
    """The attention against 64 bits, each output within its own tolerance."""
    out = attend(ctx, c, q, lens)
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
        for h in range(n_q):
            kv = h // per
            x = k[kv] @ q[m, h].astype(np.float64) / np.sqrt(d)
            A = (np.abs(k[kv]) @ np.abs(q[m, h].astype(np.float64))).max() / np.sqrt(d)
            p = np.exp(x - x.max())
            p /= p.sum()
            tol = np.repeat((80 * A + 256 + n) * 2.0 ** -24 * (p @ b[kv]), c.g)
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
