"""The operators of the 4-bit KV cache and of token scoring, as cases to time.

`run` makes one pass through an operator.  With `own` false it computes the
operator in plain torch (32 bits, 64 where a rounding decides); with `own`
true it makes the calls of this library (include/tmg_cuda.h) that a serving
program makes.  The operators:

  append    rows of keys and values quantised to 4 bits as they are written
            into the cache, and the same rows read back
  read      a long stretch of the cache read back to f32 rows
  attn      decode attention (one query row a stream) over the 4-bit cache
  logprobs  log probabilities of given tokens, the entropy of their
            distributions and the top alternatives

The cache.  Codes [n_streams, n_kv, capacity, head_dim / 2] bytes, element 2i
of a row in the low half of byte i; one 32-bit word of parameters for each
group of g = min(head_dim, 32) elements of a row, [n_streams, n_kv, capacity,
head_dim / g]: the bf16 minimum in its high half, the bf16 step in its low
half.  For a group x: m = the largest bf16 <= min(x); s = the smallest bf16
with 15 s >= max(x) - m; code = rint((x - m) / s), 0 where s = 0; the value it
stands for is m + code * s.
"""
import ctypes
import math

import torch

own = False

_HANDLE = []


def _library():
    """The library's ctypes table and an op-only context (own form only)."""
    if not _HANDLE:
        from tinyminigo_b200 import _lib

        ctx = ctypes.c_void_p()
        _lib.check(_lib.lib().tmg_create(0, None, ctypes.byref(ctx)))
        _HANDLE.extend([_lib, _lib.lib(), ctx])
    return _HANDLE


# --------------------------------------------------------------------------
# Cases
# --------------------------------------------------------------------------
def listed():
    return [
        # one decode step of 16 streams of a 1B-class model: 16 rows written
        dict(name="append step 16x8x64", op="append", streams=16, rows=1, n_kv=8, d=64,
             capacity=2048),
        # a prompt's chunk of a long prefill, padded: 1 stream, 8B-class heads
        dict(name="append chunk 4000x8x128", op="append", streams=1, rows=4000, n_kv=8, d=128,
             capacity=4096),
        # a batch of short prompts of different lengths, small model
        dict(name="append ragged 7x333x2x32", op="append", streams=7, rows=333, n_kv=2, d=32,
             capacity=1024),
        # a short prefix read back, and a long context read back for a prefill
        dict(name="read 777x8x64", op="read", streams=1, rows=777, n_kv=8, d=64, capacity=1024),
        dict(name="read 65536x8x128", op="read", streams=1, rows=65536, n_kv=8, d=128,
             capacity=65536),
        # one stream early in its generation: the smallest call, its latency
        dict(name="attn 1x333 32/8x64", op="attn", streams=1, length=333, n_q=32, n_kv=8, d=64,
             ragged=False),
        # a batch of streams of different lengths, one empty, 8B-class heads
        dict(name="attn ragged 16x8191 32/8x128", op="attn", streams=16, length=8191, n_q=32,
             n_kv=8, d=128, ragged=True),
        # one long stream; and the long-context batch of the benchmark
        dict(name="attn 1x131072 32/8x64", op="attn", streams=1, length=131072, n_q=32, n_kv=8,
             d=64, ragged=False),
        dict(name="attn 16x32768 32/8x64", op="attn", streams=16, length=32768, n_q=32, n_kv=8,
             d=64, ragged=False),
        # one row (a single stream's step), a step of 16 streams, a prompt
        dict(name="logprobs 1x128256 top 5", op="logprobs", rows=1, vocab=128256, pad=0, top=5),
        dict(name="logprobs 16x32003 top 20", op="logprobs", rows=16, vocab=32003, pad=5, top=20),
        dict(name="logprobs 2047x128256 top 8", op="logprobs", rows=2047, vocab=128256, pad=0,
             top=8),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "read", "attn", "attn", "logprobs", "logprobs"])
    d = rng.choice([16, 32, 64, 64, 128, 128])
    n_kv = rng.choice([1, 2, 3, 4, 8, 8])
    if op in ("append", "read"):
        streams = _log(rng, 1, 16) if op == "append" or rng.random() < 0.5 else 1
        rows = _log(rng, 1, max(1, 4000 * 1024 // (streams * n_kv * d)))
        return dict(op=op, streams=streams, rows=rows, n_kv=n_kv, d=d,
                    capacity=(rows + rng.randrange(1, 500) + 3) // 4 * 4)
    if op == "attn":
        group = rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 16])
        streams = _log(rng, 1, 16)
        length = _log(rng, 1, min(131072, 16 * 32768 * 512 // (streams * n_kv * d)))
        return dict(op=op, streams=streams, length=length, n_q=n_kv * group, n_kv=n_kv, d=d,
                    ragged=rng.random() < 0.6)
    vocab = rng.choice([_log(rng, 100, 128256), 32000, 128256])
    rows = _log(rng, 1, min(2048, max(2, 2047 * 128256 // (4 * vocab))))
    return dict(op=op, rows=rows, vocab=vocab, pad=rng.choice([0, 0, 1, 5, 8]),
                top=rng.choice([0, 1, 5, 20, 64]))


# --------------------------------------------------------------------------
# What a program has in hand
# --------------------------------------------------------------------------
def _dims(case):
    g = min(case["d"], 32)
    return g, case["d"] // g


def _ptr(t):
    return ctypes.c_void_p(t.data_ptr())


class _View(ctypes.Structure):
    """tmg_kv4 of include/tmg_cuda.h."""

    _fields_ = [("k_codes", ctypes.c_void_p), ("k_params", ctypes.c_void_p),
                ("v_codes", ctypes.c_void_p), ("v_params", ctypes.c_void_p),
                ("n_streams", ctypes.c_int32), ("n_kv", ctypes.c_int32),
                ("head_dim", ctypes.c_int32), ("capacity", ctypes.c_int64)]


def _view(st, streams, n_kv, d, capacity):
    return _View(st["kc"].data_ptr(), st["kp"].data_ptr(), st["vc"].data_ptr(),
                 st["vp"].data_ptr(), streams, n_kv, d, capacity)


def _cache(gen, shape, d):
    """A filled cache as a generation leaves it: random codes, steps and
    minima of the size that keys (some channels louder) or values have."""
    g = min(d, 32)
    codes = torch.randint(0, 256, (*shape, d // 2), generator=gen, device="cuda",
                          dtype=torch.uint8)
    step = torch.rand((*shape, d // g), generator=gen, device="cuda") * 0.35 + 0.1
    low = -step * (6.0 + 3.0 * torch.rand((*shape, d // g), generator=gen, device="cuda"))
    s = step.bfloat16().view(torch.int16).int() & 0xffff
    m = low.bfloat16().view(torch.int16).int() << 16
    return codes, m | s


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    op = case["op"]
    if op == "logprobs":
        rows, V = case["rows"], case["vocab"]
        ld = V + case["pad"]
        logits = torch.randn((rows, ld), generator=gen, device="cuda") * 2.5
        # a few likely tokens a row, and tokens that a program has ruled out
        peak = torch.randint(0, V, (rows, 4), generator=gen, device="cuda")
        logits.scatter_add_(1, peak, torch.rand((rows, 4), generator=gen, device="cuda") * 12.0)
        out = torch.randint(0, V, (rows, max(1, V // 200)), generator=gen, device="cuda")
        logits.scatter_(1, out, -math.inf)
        targets = torch.where(torch.rand(rows, generator=gen, device="cuda") < 0.5, peak[:, 0],
                              torch.randint(0, V, (rows,), generator=gen, device="cuda"))
        f = dict(device="cuda", dtype=torch.float32)
        return dict(case=case, logits=logits, targets=targets.int(),
                    logprob=torch.zeros(rows, **f), entropy=torch.zeros(rows, **f),
                    top_ids=torch.zeros((rows, case["top"]), device="cuda", dtype=torch.int32),
                    top_logprobs=torch.zeros((rows, case["top"]), **f))
    M, n_kv, d = case["streams"], case["n_kv"], case["d"]
    if op == "attn":
        capacity = (case["length"] + 3) // 4 * 4
    else:
        capacity = case["capacity"]
    st = dict(case=case, capacity=capacity)
    st["kc"], st["kp"] = _cache(gen, (M, n_kv, capacity), d)
    st["vc"], st["vp"] = _cache(gen, (M, n_kv, capacity), d)
    st["view"] = _view(st, M, n_kv, d, capacity)
    if op == "attn":
        lens = torch.full((M,), case["length"], device="cuda", dtype=torch.int32)
        if case["ragged"]:
            lens = torch.randint(0, case["length"] + 1, (M,), generator=gen, device="cuda",
                                 dtype=torch.int32)
            lens[0] = case["length"]
            if M > 2:
                lens[M // 2] = 0
        st["lens"] = lens
        st["q"] = torch.randn((M, case["n_q"] * d), generator=gen, device="cuda") * 1.2
        st["out"] = torch.zeros((M, case["n_q"] * d), device="cuda")
        # partial results of split rows: a generous fixed size, zero is not needed
        st["ws"] = torch.empty(32 << 20, device="cuda", dtype=torch.uint8)
        return st
    R = case["rows"]
    # the projections' rows: keys and values side by side, as one GEMM writes
    # them; some channels of the keys are louder, as they are in a decoder
    ld = 2 * n_kv * d
    x = torch.randn((M, R, ld), generator=gen, device="cuda")
    x[:, :, :n_kv * d] *= torch.exp(torch.randn(n_kv * d, generator=gen, device="cuda"))
    st["rows"] = x
    room = capacity - R
    st["pos"] = torch.randint(0, room + 1, (M,), generator=gen, device="cuda", dtype=torch.int32)
    count = torch.full((M,), R, device="cuda", dtype=torch.int32)
    if M > 1 and R > 1:
        count = torch.randint(0, R + 1, (M,), generator=gen, device="cuda", dtype=torch.int32)
    st["count"] = count
    st["k"] = torch.zeros((M, R, n_kv * d), device="cuda")
    st["v"] = torch.zeros((M, R, n_kv * d), device="cuda")
    return st


# --------------------------------------------------------------------------
# The plain forms
# --------------------------------------------------------------------------
def _down(x):
    """The largest bf16 <= x (f32 tensors of finite values)."""
    b = x.view(torch.int32)
    t = b & -65536
    return torch.where((b < 0) & (b != t), t + 65536, t).view(torch.float32)


def _quantise(x, g):
    """x [..., d] to (codes [..., d] int32, m [..., d/g], s [..., d/g])."""
    x = x.unflatten(-1, (-1, g))
    lo, hi = x.amin(-1), x.amax(-1)
    m = _down(lo)
    # hi - m as a sum of two 64-bit values, then the smallest s
    a, b = hi.double(), -m.double()
    r = a + b
    e = (a - (r - (r - a))) + (b - (r - a))
    low = (r / 15).float().view(torch.int32) & -65536
    p = 15 * low.view(torch.float32).double()
    enough = (p > r) | ((p == r) & (e <= 0))
    s = torch.where(enough, low, low + 65536).view(torch.float32)
    s = torch.where(r > 0, s, torch.zeros_like(s))
    bad = ~torch.isfinite(x).all(-1) | ~torch.isfinite(m) | ~torch.isfinite(s) | ~torch.isfinite(
        r.float())
    t = (x.double() - m.double()[..., None]) / s.double()[..., None]
    code = torch.where((s > 0)[..., None] & ~bad[..., None], torch.round(t), torch.zeros_like(t))
    nan = torch.full_like(m, math.nan)
    return code.int().flatten(-2), torch.where(bad, nan, m), torch.where(bad, nan, s)


def _values(codes, m, s, g):
    """The values that codes [..., d] stand for."""
    c = codes.unflatten(-1, (-1, g)).double()
    return (c * s.double()[..., None] + m.double()[..., None]).float().flatten(-2)


def _unpack(codes, params):
    """Cache codes and parameters to int codes and f32 (m, s)."""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    return c, (params & -65536).view(torch.float32), (params << 16).view(torch.float32)


def _pack(codes, m, s):
    lo, hi = codes[..., 0::2], codes[..., 1::2]
    p = (m.view(torch.int32) & -65536) | ((s.view(torch.int32) >> 16) & 65535)
    return (lo | (hi << 4)).to(torch.uint8), p


def _places(st):
    """(stream, row) pairs that are no padding, and their cache positions."""
    R = st["case"]["rows"]
    t = torch.arange(R, device="cuda")
    keep = t[None, :] < st["count"][:, None]
    at, row = keep.nonzero(as_tuple=True)
    return at, row, st["pos"][at].long() + row


def _plain_append(st):
    c = st["case"]
    n_kv, d = c["n_kv"], c["d"]
    g, _ = _dims(c)
    at, row, pos = _places(st)
    x = st["rows"][at, row].unflatten(-1, (2, n_kv, d))
    codes, params = _pack(*_quantise(x, g))
    st["kc"][at, :, pos], st["kp"][at, :, pos] = codes[:, 0], params[:, 0]
    st["vc"][at, :, pos], st["vp"][at, :, pos] = codes[:, 1], params[:, 1]
    return _plain_read(st)


def _plain_read(st):
    g, _ = _dims(st["case"])
    at, row, pos = _places(st)
    k, v = _unpack(st["kc"][at, :, pos], st["kp"][at, :, pos]), _unpack(
        st["vc"][at, :, pos], st["vp"][at, :, pos])
    st["k"][at, row] = _values(*k, g).flatten(1)
    st["v"][at, row] = _values(*v, g).flatten(1)
    return {"k": st["k"], "v": st["v"]}


def _plain_attn(st):
    c = st["case"]
    M, n_kv, d, n_q = c["streams"], c["n_kv"], c["d"], c["n_q"]
    g, _ = _dims(c)
    L = c["length"]

    def rows(codes, params):
        i, m, s = _unpack(codes[:, :, :L], params[:, :, :L])
        i = i.unflatten(-1, (-1, g)).float()
        return torch.addcmul(m[..., None], i, s[..., None]).flatten(-2)

    q = st["q"].view(M, n_kv, n_q // n_kv, d)
    x = (q @ rows(st["kc"], st["kp"]).transpose(2, 3)) * (1.0 / math.sqrt(d))
    seen = torch.arange(L, device="cuda")[None, :] < st["lens"][:, None]
    x = x.masked_fill(~seen[:, None, None, :], -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    st["out"].copy_((p @ rows(st["vc"], st["vp"])).reshape(M, n_q * d))
    return {"out": st["out"]}


def _plain_logprobs(st):
    V, k = st["case"]["vocab"], st["case"]["top"]
    x = st["logits"][:, :V]
    top = x.amax(-1, keepdim=True)
    y = x - top
    e = torch.exp(y)
    total = e.sum(-1)
    lse = torch.log(total)
    at = y.gather(1, st["targets"].long()[:, None])[:, 0]
    weighed = torch.where(e > 0, e * y, torch.zeros_like(e)).sum(-1)
    st["logprob"].copy_(at - lse)
    st["entropy"].copy_(lse - weighed / total)
    out = {"logprob": st["logprob"], "entropy": st["entropy"]}
    if k:
        # order by value, ties to the lowest index: both in one whole number
        b = (x + 0.0).view(torch.int32) if x.is_contiguous() else (x + 0.0).contiguous().view(
            torch.int32)
        b = torch.where(b < 0, b ^ 0x7fffffff, b).long()
        key = (b << 32) | (V - 1 - torch.arange(V, device="cuda"))
        best = V - 1 - (torch.topk(key, k, dim=1, sorted=True).values & 0xffffffff)
        st["top_ids"].copy_(best)
        st["top_logprobs"].copy_(y.gather(1, best) - lse[:, None])
        out.update(top_ids=st["top_ids"], top_logprobs=st["top_logprobs"])
    return out


# --------------------------------------------------------------------------
# One pass
# --------------------------------------------------------------------------
def run(st):
    op = st["case"]["op"]
    if not own:
        return {"append": _plain_append, "read": _plain_read, "attn": _plain_attn,
                "logprobs": _plain_logprobs}[op](st)
    lib, L, ctx = _library()
    c = st["case"]
    if op == "logprobs":
        k = c["top"]
        lib.check(L.tmg_op_logprobs(ctx, _ptr(st["logits"]), st["logits"].stride(0), c["rows"],
                                    c["vocab"], _ptr(st["targets"]), k, _ptr(st["logprob"]),
                                    _ptr(st["entropy"]), _ptr(st["top_ids"]) if k else None,
                                    _ptr(st["top_logprobs"]) if k else None), ctx)
        out = {"logprob": st["logprob"], "entropy": st["entropy"]}
        if k:
            out.update(top_ids=st["top_ids"], top_logprobs=st["top_logprobs"])
        return out
    kv = ctypes.byref(st["view"])
    if op == "attn":
        w = c["n_q"] * c["d"]
        lib.check(L.tmg_op_attn_decode_kv4(ctx, kv, _ptr(st["q"]), w, _ptr(st["lens"]),
                                           c["length"], c["n_q"], _ptr(st["out"]), w,
                                           _ptr(st["ws"]), st["ws"].numel()), ctx)
        return {"out": st["out"]}
    w = c["n_kv"] * c["d"]
    if op == "append":
        rows = st["rows"]
        lib.check(L.tmg_op_kv4_append(ctx, kv, _ptr(rows),
                                      ctypes.c_void_p(rows.data_ptr() + 4 * w), 2 * w, c["rows"],
                                      _ptr(st["pos"]), _ptr(st["count"])), ctx)
    lib.check(L.tmg_op_kv4_read(ctx, kv, _ptr(st["pos"]), _ptr(st["count"]), c["rows"],
                                _ptr(st["k"]), _ptr(st["v"]), w), ctx)
    return {"k": st["k"], "v": st["v"]}


def work(case):
    """Bytes that a pass has to read and write, and its multiply-adds."""
    op = case["op"]
    if op == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4.0 * n + case["rows"] * (12 + 8 * case["top"]), "flops": 5.0 * n}
    M, n_kv, d = case["streams"], case["n_kv"], case["d"]
    g, groups = _dims(case)
    packed = 2.0 * n_kv * (d / 2 + 4 * groups)  # a position's keys and values
    wide = 2.0 * n_kv * d * 4
    if op == "attn":
        n = M * case["length"] * (0.5 if case["ragged"] and M > 1 else 1.0)
        return {"bytes": n * packed + 8.0 * M * case["n_q"] * d, "flops": 4.0 * n * case["n_q"] * d}
    n = M * case["rows"] * (0.5 if M > 1 and case["rows"] > 1 else 1.0)
    both = 2 if op == "append" else 1
    return {"bytes": both * n * (packed + wide), "flops": both * 2.0 * n * 2 * n_kv * d}


# --------------------------------------------------------------------------
# In 64 bits
# --------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "logprobs":
        return _exact_logprobs(case, st)
    if op == "attn":
        return _exact_attn(case, st)
    M, R, n_kv, d = case["streams"], case["rows"], case["n_kv"], case["d"]
    g = min(d, 32)
    out = {"k": torch.zeros((M, R, n_kv * d), dtype=torch.float64, device="cuda"),
           "v": torch.zeros((M, R, n_kv * d), dtype=torch.float64, device="cuda")}
    for name, i in (("k", 0), ("v", 1)):
        codes, params = st[name + "c"], st[name + "p"]
        for a in range(M):
            n, p = int(st["count"][a]), int(st["pos"][a])
            if op == "append":
                x = st["rows"][a, :n, i * n_kv * d:(i + 1) * n_kv * d].double()
                x = x.reshape(n, n_kv * d // g, g)
                low, high = x.min(-1).values, x.max(-1).values
                m = _bf16_toward(low, torch.floor)
                s = _bf16_toward((high - m) / 15, torch.ceil)
                t = torch.round((x - m[..., None]) / torch.where(s > 0, s, 1.0)[..., None])
                y = m[..., None] + t * s[..., None]
            else:
                b = codes[a, :, p:p + n].long()
                t = torch.empty((n_kv, n, d), dtype=torch.float64, device="cuda")
                t[..., 0::2], t[..., 1::2] = (b % 16).double(), (b // 16).double()
                w = params[a, :, p:p + n].long() & 0xffffffff
                m, s = _bf16_value(w // 65536), _bf16_value(w % 65536)
                y = m[..., None] + t.reshape(n_kv, n, d // g, g) * s[..., None]
                y = y.reshape(n_kv, n, d).transpose(0, 1)
            out[name][a, :n] = y.reshape(n, n_kv * d)
    return out


def _bf16_toward(x, step):
    """x (64 bits) to a multiple of the bf16 spacing of its size, by `step`."""
    e = torch.frexp(x).exponent.double()
    unit = torch.exp2(e - 8)
    return step(x / unit) * unit


def _bf16_value(h):
    """What a bf16 pattern (normal or zero) stands for, in 64 bits."""
    e, f = (h // 128) % 256, (h % 128).double()
    x = torch.where(e > 0, (1 + f / 128) * torch.exp2(e.double() - 127), f * 2.0 ** -133)
    return torch.where(h >= 32768, -x, x)


def _exact_attn(case, st):
    M, n_kv, d, n_q = case["streams"], case["n_kv"], case["d"], case["n_q"]
    g = min(d, 32)
    out = torch.zeros((M, n_q, d), dtype=torch.float64, device="cuda")
    for a in range(M):
        n = int(st["lens"][a])
        if n == 0:
            continue
        for h in range(n_kv):
            wide = []
            for codes, params in ((st["kc"], st["kp"]), (st["vc"], st["vp"])):
                b = codes[a, h, :n].long()
                t = torch.empty((n, d), dtype=torch.float64, device="cuda")
                t[:, 0::2], t[:, 1::2] = (b % 16).double(), (b // 16).double()
                w = params[a, h, :n].long() & 0xffffffff
                m, s = _bf16_value(w // 65536), _bf16_value(w % 65536)
                wide.append(t * s.repeat_interleave(g, 1) + m.repeat_interleave(g, 1))
            G = n_q // n_kv
            q = st["q"][a].view(n_q, d)[h * G:(h + 1) * G].double()
            x = q @ wide[0].T / math.sqrt(d)
            p = torch.exp(x - x.max(1, keepdim=True).values)
            out[a, h * G:(h + 1) * G] = (p @ wide[1]) / p.sum(1, keepdim=True)
    return {"out": out.view(M, n_q * d)}


def _exact_logprobs(case, st):
    rows, V, k = case["rows"], case["vocab"], case["top"]
    out = {"logprob": [], "entropy": []}
    if k:
        out.update(top_ids=[], top_logprobs=[])
    for at in range(0, rows, 128):
        x = st["logits"][at:at + 128, :V].double()
        lse = torch.logsumexp(x, 1, keepdim=True)
        z = x - lse
        p = torch.exp(z)
        out["logprob"].append(torch.gather(z, 1, st["targets"][at:at + 128].long()[:, None])[:, 0])
        out["entropy"].append(-(p * torch.where(p > 0, z, 0.0)).sum(1))
        if k:
            ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k]
            out["top_ids"].append(ids.int())
            out["top_logprobs"].append(torch.gather(z, 1, ids))
    return {name: torch.cat(v) for name, v in out.items()}
