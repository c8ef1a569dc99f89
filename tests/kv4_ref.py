"""The 4-bit KV cache in numpy, in 64 bits: the format and arithmetic that
include/tmg_cuda.h states for tmg_kv4 (test infrastructure only)."""
import numpy as np


def bf16_down(x):
    """The largest bf16 <= x, as its pattern (finite f32)."""
    b = np.asarray(x, np.float32).view(np.uint32)
    t = b & np.uint32(0xFFFF0000)
    return np.where((b >> 31 == 1) & (t != b), t + np.uint32(0x10000), t) >> 16


def bf16_value(h):
    return (np.asarray(h, np.uint32) << 16).view(np.float32)


def quantise(x):
    """x [..., d] f32 -> codes [..., d] uint8, params [..., d / g] uint32."""
    x = np.asarray(x, np.float32)
    d = x.shape[-1]
    g = min(d, 32)
    x = x.reshape(*x.shape[:-1], d // g, g)
    ok = np.isfinite(x).all(-1)
    x = np.where(ok[..., None], x, np.float32(0))
    lo, hi = x.min(-1), x.max(-1)
    m = bf16_down(lo)
    with np.errstate(over="ignore", invalid="ignore"):
        # hi - m without an error: want + rest (Knuth's two-sum)
        a, b = hi.astype(np.float64), -bf16_value(m).astype(np.float64)
        want = a + b
        rest = (a - (want - (want - a))) + (b - (want - a))
        s = (want / 15).astype(np.float32).view(np.uint32) >> 16  # at most one below
        for _ in range(2):
            p = 15 * bf16_value(s).astype(np.float64)
            s = np.where((p < want) | ((p == want) & (rest > 0)), s + np.uint32(1), s)
        sv = bf16_value(s)
        ok &= np.isfinite(bf16_value(m)) & np.isfinite(sv) & (want <= np.finfo(np.float32).max)
        div = np.where(ok & (sv > 0), sv, np.float32(1)).astype(np.float64)
        base = np.where(ok, bf16_value(m), np.float32(0)).astype(np.float64)
        c = np.rint((x.astype(np.float64) - base[..., None]) / div[..., None])
    c = np.where((ok & (sv > 0))[..., None], c, 0)
    assert np.all((c >= 0) & (c <= 15))
    params = np.where(ok, (m << 16) | s, np.uint32(0x7FC07FC0)).astype(np.uint32)
    return c.astype(np.uint8).reshape(*x.shape[:-2], d), params


def pack(codes):
    return (codes[..., 0::2] | (codes[..., 1::2] << 4)).astype(np.uint8)


def unpack(packed):
    c = np.empty((*packed.shape[:-1], packed.shape[-1] * 2), np.uint8)
    c[..., 0::2], c[..., 1::2] = packed & 15, packed >> 4
    return c


def steps(params):
    return bf16_value(params & np.uint32(0xFFFF))


def values(codes, params):
    """What codes [..., d] stand for, in 64 bits (before the one f32 rounding)."""
    d = codes.shape[-1]
    g = min(d, 32)
    c = codes.reshape(*codes.shape[:-1], d // g, g).astype(np.float64)
    m = bf16_value(params >> np.uint32(16)).astype(np.float64)
    s = steps(params).astype(np.float64)
    return (c * s[..., None] + m[..., None]).reshape(codes.shape)


def attention(q, k, v):
    """Decode attention of q [n_q, d] over k, v [n, n_kv, d] in 64 bits; also
    the largest sum of |q_i k_i| / sqrt(d) a score is made of."""
    n_q, d = q.shape
    n, n_kv, _ = k.shape
    if n == 0:
        return np.zeros((n_q, d)), 0.0
    q = q.astype(np.float64).reshape(n_kv, n_q // n_kv, d)
    x = np.einsum("hgd,nhd->hgn", q, k) / np.sqrt(d)
    a = np.einsum("hgd,nhd->hgn", np.abs(q), np.abs(k)) / np.sqrt(d)
    p = np.exp(x - x.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    return np.einsum("hgn,nhd->hgd", p, v).reshape(n_q, d), float(a.max())
