"""The operators of a paged serving step through the C ABI, and what they compute, in 64 bits with NumPy."""
import numpy as np

from axono_amd import _lib
from axono_amd.device import DeviceBuffer, check, synchronize

F16, F32, I32, I64 = 4, 5, 2, 3
CODE = {np.dtype(np.float16): F16, np.dtype(np.float32): F32, np.dtype(np.int32): I32, np.dtype(np.int64): I64}
PAGE = 128
U = {np.dtype(np.float16): 2.0 ** -11, np.dtype(np.float32): 2.0 ** -24}   # half a step, relative to the value
TINY = {np.dtype(np.float16): 2.0 ** -25, np.dtype(np.float32): 2.0 ** -149}


def lib():
    return _lib.load()


def dev(a):
    return None if a is None else DeviceBuffer.from_numpy(np.ascontiguousarray(a))


def ptr(b):
    return None if b is None else b.ptr


def pages_for(n, start, rng, spare=2):
    """page table [B, max_pages] handed out at random, -1 behind a sequence's pages; pages in the pool"""
    held = [max(0, (s + m + PAGE - 1) // PAGE) for s, m in zip(start, n)]
    order = rng.permutation(sum(held) + spare)
    table = np.full((len(n), max(max(held), 1)), -1, np.int32)
    at = 0
    for b, h in enumerate(held):
        table[b, :h] = order[at:at + h]
        at += h
    return table, len(order)


def cu_of(n):
    return np.concatenate([[0], np.cumsum(n)]).astype(np.int32)


# ---- rotation --------------------------------------------------------------------------------------------------------
def turned(x, pos, freq, rd, interleaved, scale, axis=None):
    """x [rows, heads, d] in 64 bits with the first rd elements of every head rotated; (result, size of what was added)"""
    x = np.asarray(x, np.float64)
    pos = np.asarray(pos, np.int64).reshape(-1, x.shape[0])
    axis = np.zeros(rd // 2, np.int64) if axis is None else axis
    turns = pos[axis].T.astype(np.longdouble) * np.asarray(freq, np.float32).astype(np.longdouble)
    c = (np.cos(turns) * np.float32(scale)).astype(np.float64)[:, None, :]
    s = (np.sin(turns) * np.float32(scale)).astype(np.float64)[:, None, :]
    i = np.arange(rd // 2)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rd // 2)
    y, size = x.copy(), np.zeros_like(x)
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    size[..., a] = size[..., b] = (np.abs(x[..., a]) + np.abs(x[..., b])) * scale
    return y, size


def mrope_axis(rd, h_sec, w_sec):
    i = np.arange(rd // 2)
    return np.where((i % 3 == 1) & (i < 3 * h_sec), 1, np.where((i % 3 == 2) & (i < 3 * w_sec), 2, 0))


# of cosine and sine: the angle, below half a turn, rounds to fp32 (pi 2^-24), sincosf is good to 2 ulp (2^-22 near 1), the
# scale rounds once; two products and a sum round three times more: all relative to |x0| + |x1|
ROTATION = np.pi * 2.0 ** -24 + 2.0 ** -22 + 2.0 ** -24 + 3 * 2.0 ** -24


def rotary_qk(q, k, pos, freq, scale, interleaved, rd, q_stride=None, k_stride=None):
    rows, hq, d = q.shape
    hk = 0 if k is None else k.shape[1]
    qs, ks = q_stride or hq * d, k_stride or max(hk * d, 1)

    def padded(x, stride):
        if x is None:
            return None
        flat = np.full((rows, stride), 7.0, x.dtype)
        flat[:, :x.shape[1] * d] = x.reshape(rows, -1)
        return flat

    dq, dk = dev(padded(q, qs)), dev(padded(k, ks))
    dp, df = dev(np.asarray(pos, np.int64)), dev(np.asarray(freq, np.float32))
    oq, ok = DeviceBuffer(q.nbytes), None if k is None else DeviceBuffer(k.nbytes)
    check(lib().axhip_rotary_qk(dq.ptr, qs, ptr(dk), ks, dp.ptr, df.ptr, scale, int(interleaved), rd, oq.ptr, ptr(ok),
                                CODE[q.dtype], rows, hq, hk, d, None), "rotary_qk")
    synchronize()
    return oq.download(q.dtype, q.shape), None if k is None else ok.download(k.dtype, k.shape)


# ---- append ------------------------------------------------------------------------------------------------------------
def append_want(qkv, hq, hk, w, eps, norm, pos, freq, scale, interleaved, rd, axis, n, start, table, k_pool, v_pool):
    """(q, k_pool, v_pool) in 64 bits and how far a right result may be off: norm of a head = (4 sqrt(D) + 4) 2^-24 (a sum of
    squares in another order, root, quotient, two products), the rotation, one rounding to the cache's type"""
    d, ct = qkv.shape[2], k_pool.dtype
    x = qkv.astype(np.float64)
    cu = cu_of(n)
    rel = 0.0
    heads = [x[:, :hq], x[:, hq:hq + hk]]
    if norm:
        rel = (4 * np.sqrt(d) + 4) * 2.0 ** -24
        for i in range(2):
            heads[i] = heads[i] / np.sqrt((heads[i] ** 2).mean(-1, keepdims=True) + np.float32(eps))
            if w[i] is not None:
                heads[i] = heads[i] * w[i].astype(np.float64)
    got = [turned(h, pos, freq, rd, interleaved, scale, axis) for h in heads]
    tol = [np.abs(y) * (U[ct] + rel) + size * (ROTATION + rel) + TINY[ct] for y, size in got]
    kp, vp = k_pool.astype(np.float64), v_pool.astype(np.float64)
    ktol, vtol = np.zeros_like(kp), np.zeros_like(vp)
    for b in range(len(n)):
        for i in range(n[b]):
            p, t = int(start[b]) + i, cu[b] + i
            if p < 0 or p // PAGE >= table.shape[1] or not 0 <= table[b, p // PAGE] < kp.shape[0]:
                continue
            at = (table[b, p // PAGE], slice(None), p % PAGE)
            kp[at], ktol[at] = got[1][0][t], tol[1][t]
            vp[at] = x[t, hq + hk:]
            vtol[at] = np.abs(x[t, hq + hk:]) * U[ct] + TINY[ct]
    return (got[0][0], kp, vp), (tol[0], ktol, vtol)


def append(qkv, hq, hk, w, eps, norm, pos, axes, freq, scale, interleaved, rd, sections, cu, start, table, k_pool, v_pool,
           q_fill=9.0, tokens=None):
    T, _, d = qkv.shape
    size, width = qkv.dtype.itemsize, (hq + 2 * hk) * d
    bufs = [dev(a) for a in (qkv, w[0], w[1], pos, freq, cu, np.asarray(start, np.int32), table, k_pool, v_pool)]
    dx, dqw, dkw, dp, df, dcu, dst, dt_, dk, dv = bufs
    q = np.full((T, hq, d), q_fill, k_pool.dtype)
    dq = dev(q)
    wd = CODE[w[0].dtype] if w[0] is not None else F32
    check(lib().axhip_rotary_append_paged(dx.ptr, width, dx.ptr + hq * d * size, width, dx.ptr + (hq + hk) * d * size, width,
                                          CODE[qkv.dtype], ptr(dqw), ptr(dkw), wd, eps, int(norm), ptr(dp), axes, df.ptr, scale,
                                          int(interleaved), rd, sections[0], sections[1], dcu.ptr, dst.ptr, dt_.ptr, dq.ptr,
                                          dk.ptr, dv.ptr, CODE[k_pool.dtype], T if tokens is None else tokens, len(cu) - 1, hq,
                                          hk, d, table.shape[1], k_pool.shape[0], None), "rotary_append_paged")
    synchronize()
    return (dq.download(q.dtype, q.shape), dk.download(k_pool.dtype, k_pool.shape), dv.download(v_pool.dtype, v_pool.shape))


# ---- attention -----------------------------------------------------------------------------------------------------------
def chunk_want(q, k_pool, v_pool, table, n, start, max_len, lost=2.0 ** -25):
    """softmax over the keys that a token sees, in 64 bits; and the bound of a right result's error:
    - a score is a sum of D products in fp32: D 2^-24 sum |q k| scale; the argument of the exponential, of size A, rounds twice
      and the exponential itself is good to 2^-22: every probability is off by d = that sum, relative;
    - fp16: a probability rounds to fp16, 2^-11 relative, or `lost` absolute where it is tiny (the largest is at least 1; 2^-25 where
      it is held as it is, 2^-35 where the largest is held at 2^10 at least);
    - numerator and denominator are sums of n terms in fp32: n 2^-24 each;
    - the result rounds once.  With W = sum p |v| / sum p the error is at most W (2 d + 2 u + 2 n 2^-24) + n lost max |v|
      (fp16 only; the maximum over the keys of that element) + |out| u."""
    T, hq, d = q.shape
    hk, g = k_pool.shape[1], hq // k_pool.shape[1]
    t_ = q.dtype
    half = t_ == np.float16
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    cu, scale = cu_of(n), 1 / np.sqrt(d)
    for b in range(len(n)):
        last = min(int(start[b]) + int(n[b]), max_len)
        if n[b] == 0 or last <= 0:
            continue
        pages = np.clip(table[b, :(last + PAGE - 1) // PAGE], 0, k_pool.shape[0] - 1)
        for h in range(hk):
            K = k_pool[pages, h].reshape(-1, d)[:last].astype(np.float64)
            V = v_pool[pages, h].reshape(-1, d)[:last].astype(np.float64)
            for i in range(n[b]):
                m = min(int(start[b]) + i, max_len - 1) + 1
                if m <= 0:
                    continue
                x = q[cu[b] + i, h * g:(h + 1) * g].astype(np.float64)
                with np.errstate(invalid="ignore", over="ignore"):
                    s = x @ K[:m].T * scale
                    top = s.max(-1, keepdims=True)
                    p = np.exp(s - top)
                    l = p.sum(-1, keepdims=True)
                    o = p @ V[:m] / l
                    W = p @ np.abs(V[:m]) / l
                    delta = d * 2.0 ** -24 * (np.abs(x) @ np.abs(K[:m]).T).max() * scale + \
                        2 * np.abs(s - top).max() * 2.0 ** -24 * 1.5 + np.abs(top).max() * 2.0 ** -23 + 2.0 ** -22
                    e = W * (2 * delta + 2 * m * 2.0 ** -24 + (2 * U[t_] if half else 0)) + np.abs(o) * U[t_] + TINY[t_]
                    if half:
                        e = e + m * lost * np.abs(V[:m]).max(0)
                out[cu[b] + i, h * g:(h + 1) * g] = o
                tol[cu[b] + i, h * g:(h + 1) * g] = e
    return out, tol


def chunk(q, k_pool, v_pool, table, cu, start, max_q, max_len, fill=9.0, tokens=None, dirty=True):
    T, hq, d = q.shape
    B, hk = len(cu) - 1, k_pool.shape[1]
    T = T if tokens is None else tokens
    dq, dk, dv, dt_, dcu, dst = (dev(a) for a in (q, k_pool, v_pool, table, np.asarray(cu, np.int32), np.asarray(start, np.int32)))
    out = dev(np.full(q.shape, fill, q.dtype))
    sizes = (CODE[q.dtype], T, B, hq, hk, d, max_q, max_len)
    nbytes = lib().axhip_chunk_attention_paged_workspace_bytes(*sizes)
    ws = dev(np.full(max(nbytes, 16), 0xff if dirty else 0, np.uint8))   # NaN in every word: nothing may be read unwritten
    check(lib().axhip_chunk_attention_paged(dq.ptr, dk.ptr, dv.ptr, dt_.ptr, dcu.ptr, dst.ptr, out.ptr, ws.ptr, nbytes, *sizes,
                                            table.shape[1], k_pool.shape[0], None), "chunk_attention_paged")
    synchronize()
    return out.download(q.dtype, q.shape)


# Inputs whose results are whole numbers over whole numbers, so that one key too few, too many, taken twice or taken from another
# place shows: K holds 0 and -240, V 1 and -1, a query 8 in one place and 0 elsewhere.  The keys that have 0 in that place weigh 1, the
# others 2^-170 and less, which is nothing in either type: a row's result is the sum of its keys' values over their number.
def picking(n, start, hq, hk, d, dtype, seed=0):
    rng = np.random.default_rng(seed)
    table, n_pages = pages_for(n, start, rng)
    T = sum(n)
    q = np.zeros((T, hq, d), dtype)
    row = np.arange(T * hq)
    q.reshape(-1, d)[row, (7 * row + row // d) % d] = 8
    k = (-240 * rng.integers(0, 2, (n_pages, hk, 128, d))).astype(dtype)
    v = (2 * rng.integers(0, 2, (n_pages, hk, 128, d)) - 1).astype(dtype)
    return q, k, v, table


def picking_want(q, k_pool, v_pool, table, n, start, keys_of=None):
    """(sums [T, hq, d], numbers of keys [T, hq]); keys_of(b, m): the keys that a row with m visible ones takes (an oracle with a
    mistake in it), all m by default"""
    T, hq, d = q.shape
    hk, g = k_pool.shape[1], hq // k_pool.shape[1]
    sums, numbers = np.zeros((T, hq, d)), np.zeros((T, hq))
    cu = cu_of(n)
    for b in range(len(n)):
        pages = table[b, :(int(start[b]) + int(n[b]) + PAGE - 1) // PAGE]
        for h in range(hk):
            K, V = (p[pages, h].reshape(-1, d).astype(np.float32) for p in (k_pool, v_pool))
            for i in range(n[b]):
                m = int(start[b]) + i + 1
                at = np.arange(m) if keys_of is None else keys_of(b, m)
                x = q[cu[b] + i, h * g:(h + 1) * g].argmax(-1)
                taken = (K[at][:, x] == 0).T
                taken[~taken.any(-1)] = True            # they all weigh the same then
                sums[cu[b] + i, h * g:(h + 1) * g] = taken.astype(np.float32) @ V[at]
                numbers[cu[b] + i, h * g:(h + 1) * g] = taken.sum(-1)
    return sums, numbers


def picking_error(got, sums, numbers):
    """largest distance of result * number from the sum: under 1 / 4 for a right result in fp16 too, whose rounding of sums up to
    500 is half a step, 500 * 2^-11"""
    assert np.abs(sums).max() <= 500
    return np.abs(got.astype(np.float64) * numbers[..., None] - sums).max()


# ---- logits ----------------------------------------------------------------------------------------------------------------
def logits_want(x, hist, hist_len, prompt_len, rep, pres, freq, bias_ids, bias, allowed):
    """(result in 64 bits, bound): each of the up to four steps in fp32 rounds at most twice, a sum of biases once per entry,
    all relative to the largest value that occurs; one rounding to the type of the logits"""
    B, V = x.shape
    out, size = x.astype(np.float64), np.abs(x.astype(np.float64))
    steps = np.full(x.shape, 0.0)
    for b in range(B):
        if hist is not None:
            ids = np.asarray(hist[b][:hist_len[b]], np.int64)
            ok = (ids >= 0) & (ids < V)
            said = ids[int(prompt_len[b]):][ok[int(prompt_len[b]):]]
            seen = np.unique(ids[ok])
            r = np.float64(rep[b]) if rep is not None else 1.0
            v = out[b, seen]
            out[b, seen] = np.where(v > 0, v / r, v * r)
            size[b, seen] = np.maximum(size[b, seen], np.abs(out[b, seen]))
            steps[b, seen] += 1
            which, times = np.unique(said, return_counts=True)
            f = np.float64(freq[b]) if freq is not None else 0.0
            p = np.float64(pres[b]) if pres is not None else 0.0
            out[b, which] -= f * times + p
            size[b, which] += np.abs(f) * times + np.abs(p)
            steps[b, which] += 3
        if bias_ids is not None:
            for i, w in zip(bias_ids[b], bias[b]):
                if 0 <= i < V:
                    out[b, i] += np.float64(w)
                    size[b, i] += abs(np.float64(w))
                    steps[b, i] += 2
        if allowed is not None:
            bits = np.unpackbits(allowed[b].view(np.uint8), bitorder="little")[:V]
            out[b, bits == 0] = -np.inf
    with np.errstate(invalid="ignore"):
        tol = size * steps * 2.0 ** -24 + np.where(np.isfinite(out), np.abs(out), 0) * (U[x.dtype] if x.dtype == np.float16 else 0) + \
            (TINY[x.dtype] if x.dtype == np.float16 else 0)
    return out, tol


def logits(x, hist, hist_len, prompt_len, rep, pres, freq, bias_ids, bias, allowed, by_step=False, stride=None, in_place=False):
    B, V = x.shape
    stride = stride or V
    flat = np.full((B, stride), 3.0, x.dtype)
    flat[:, :V] = x
    dx = dev(flat)
    do = dx if in_place else dev(np.full((B, stride), 5.0, x.dtype))
    h = None if hist is None else np.ascontiguousarray(hist.T if by_step else hist)
    H = 0 if hist is None else hist.shape[1]
    rs, ts = (1, B) if by_step else (H, 1)
    bufs = [dev(a) for a in (h, None if hist_len is None else np.asarray(hist_len, np.int32),
                             None if prompt_len is None else np.asarray(prompt_len, np.int32), rep, pres, freq, bias_ids, bias, allowed)]
    dh, dl, dpl, dr, dp, df, dbi, dbv, da = bufs
    check(lib().axhip_logits_process(dx.ptr, stride, CODE[x.dtype], ptr(dh), CODE[hist.dtype] if hist is not None else I32, rs, ts, H,
                                     ptr(dl), ptr(dpl), ptr(dr), ptr(dp), ptr(df), ptr(dbi), ptr(dbv),
                                     0 if bias_ids is None else bias_ids.shape[1], ptr(da), 0 if allowed is None else allowed.shape[1],
                                     do.ptr, stride, B, V, None), "logits_process")
    synchronize()
    got = do.download(x.dtype, (B, stride))
    assert np.all(got[:, V:] == (3.0 if in_place else 5.0))   # what lies behind a row stays
    return got[:, :V]


def assert_within(got, want, tol):
    got = got.astype(np.float64)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    np.testing.assert_array_equal(np.isinf(got) * np.sign(np.nan_to_num(got)), np.isinf(want) * np.sign(np.nan_to_num(want)))
    fine = np.isfinite(want)
    err, tol = np.abs(got[fine] - want[fine]), np.broadcast_to(tol, want.shape)[fine]
    worst = float((err - tol).max(initial=-1.0))
    assert worst <= 0, (worst, float(err.max()), int((err > tol).sum()))
