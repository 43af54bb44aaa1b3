"""The operators of a paged serving step, each in its plain form and as the framework's call, over the sizes they run at.

    rotary   rotation of q and k by a frequency table: half or interleaved pairs, part of the head, scaled tables
    append   q/k/v rows of a ragged batch of new tokens: norm of each head, rotation, keys and values into the pages
    chunk    attention of a ragged batch of new tokens over the paged cache that holds them and what came before
    logits   penalties for repeated tokens, biases and grammar masks on the logits of a step

`own` false computes them with elementary torch operations in 32 bits (angles in 64), `own` true calls libaxhip.so.
A ragged batch of B sequences is T rows in a line: the rows of sequence b are cu[b] .. cu[b + 1], and its first new token
sits at position start[b] of its cache.  A page holds 128 consecutive keys of one sequence.
"""
import math

import numpy as np
import torch

own = False

PAGE = 128
F16, F32, I32, I64 = 4, 5, 2, 3  # the type numbers of the C boundary
TORCH = {"f16": torch.float16, "f32": torch.float32}
CODE = {"f16": F16, "f32": F32}


def listed():
    return [
        # one decode step of the 32-sequence benchmark batch: 24 heads a row, everything is latency
        {"name": "rotary decode 32 rows", "op": "rotary", "rows": 32, "hq": 16, "hk": 8, "d": 128, "rd": 128, "inter": False,
         "table": "plain", "type": "f16", "far": 8192},
        # a long prefill in 32 bits: interleaved pairs, half of each head, a table stretched for long contexts
        {"name": "rotary prefill 33001 rows", "op": "rotary", "rows": 33001, "hq": 16, "hk": 8, "d": 128, "rd": 64,
         "inter": True, "table": "yarn", "type": "f32", "far": 131072},
        # one token of each of 16 sequences at a context of 4096: the projection's 32-bit rows, norms, three position axes
        {"name": "append decode 16 rows", "op": "append", "batch": 16, "kind": "single", "rows": 16, "ctx": 4096, "hq": 16,
         "hk": 8, "d": 128, "rd": 128, "inter": False, "norm": True, "axes": 3, "type": "f32", "cache": "f16"},
        # a prompt's chunk of 501 rows beside 31 decoding sequences, 16-bit rows, a quarter of each head rotated
        {"name": "append mixed 532 rows", "op": "append", "batch": 32, "kind": "mixed", "rows": 532, "ctx": 4096, "hq": 32,
         "hk": 8, "d": 128, "rd": 32, "inter": False, "norm": False, "axes": 1, "type": "f16", "cache": "f16"},
        # the prefill of the decode benchmark: 16 prompts of 4096 tokens in one pass
        {"name": "append prefill 65536 rows", "op": "append", "batch": 16, "kind": "even", "rows": 65536, "ctx": 0, "hq": 16,
         "hk": 8, "d": 128, "rd": 128, "inter": False, "norm": True, "axes": 3, "type": "f32", "cache": "f16"},
        # four drafted tokens of each of 32 sequences checked at once, contexts of 512 to 8192
        {"name": "chunk drafts 32x4", "op": "chunk", "batch": 32, "kind": "even", "rows": 128, "ctx": 8192, "hq": 32, "hk": 8,
         "d": 128, "type": "f16"},
        # short prompts of odd lengths in 32 bits with heads of 64
        {"name": "chunk f32 5 prompts", "op": "chunk", "batch": 5, "kind": "ragged", "rows": 643, "ctx": 1500, "hq": 16,
         "hk": 8, "d": 64, "type": "f32"},
        # a prompt's chunk of 1024 beside 15 decoding sequences at a context of 4096
        {"name": "chunk mixed 15+1024", "op": "chunk", "batch": 16, "kind": "mixed", "rows": 1039, "ctx": 4096, "hq": 16,
         "hk": 8, "d": 128, "type": "f16"},
        # the prefill of the decode benchmark through the pages
        {"name": "chunk prefill 16x4096", "op": "chunk", "batch": 16, "kind": "even", "rows": 65536, "ctx": 0, "hq": 16,
         "hk": 8, "d": 128, "type": "f16"},
        # the last chunk of 2048 of a prompt of 131072 tokens
        {"name": "chunk 2048 at 129024", "op": "chunk", "batch": 1, "kind": "even", "rows": 2048, "ctx": 129024, "hq": 16,
         "hk": 8, "d": 128, "type": "f16"},
        # one row of 16-bit logits: the latency of a single sequence
        {"name": "logits 1 row", "op": "logits", "batch": 1, "vocab": 151936, "hist": 700, "bias": 8, "mask": True,
         "type": "f16", "ids": "i32"},
        # a step of 64 sequences with histories of up to 8192 tokens, kept as the decode loop's log keeps them
        {"name": "logits 64 rows", "op": "logits", "batch": 64, "vocab": 151936, "hist": 8192, "bias": 64, "mask": True,
         "type": "f32", "ids": "i64"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "append", "chunk", "chunk", "logits"])
    hk = rng.choice([1, 2, 4, 8])
    hq = hk * rng.choice([1, 2, 4, 8] if hk < 8 else [1, 2, 4])
    if op == "rotary":
        d = rng.choice([64, 80, 96, 128, 256])
        rows = min(_log(rng, 1, 33001), 33001 * 24 * 128 // ((hq + hk) * d))
        return {"op": op, "rows": rows, "hq": hq, "hk": hk, "d": d, "rd": rng.choice([d, d // 2, d // 4]),
                "inter": rng.random() < 0.5, "table": rng.choice(["plain", "linear", "ntk", "yarn"]),
                "type": rng.choice(["f16", "f32"]), "far": _log(rng, 64, 1 << 20)}
    if op == "append":
        d = rng.choice([64, 128, 256])
        batch = _log(rng, 1, 64)
        kind = rng.choice(["single", "mixed", "ragged", "even"])
        rows = batch if kind == "single" else min(batch * _log(rng, 1, 2048), 65536 * 32 * 128 // ((hq + 2 * hk) * d))
        rows = max(rows, batch)
        rows = rows // batch * batch if kind == "even" else rows
        return {"op": op, "batch": batch, "kind": kind, "rows": rows, "ctx": _log(rng, 1, 8192), "hq": hq, "hk": hk, "d": d,
                "rd": rng.choice([d, d // 2, d // 4]), "inter": rng.random() < 0.5, "norm": rng.random() < 0.5,
                "axes": rng.choice([1, 3]), "type": rng.choice(["f16", "f32"]), "cache": rng.choice(["f16", "f16", "f32"])}
    if op == "chunk":
        d = rng.choice([64, 128, 128])
        batch = _log(rng, 1, 32)
        kind = rng.choice(["single", "mixed", "ragged", "even"])
        ctx = _log(rng, 1, 32768)
        rows = batch if kind == "single" else max(batch, min(batch * _log(rng, 1, 2048), 16384))
        longest = 1 if kind == "single" else rows  # of one sequence, at most
        while batch * hq * longest * (ctx + longest) > (1 << 31) and rows > batch:
            rows = max(batch, rows // 2)
            longest = rows
        rows = rows // batch * batch if kind == "even" else rows
        return {"op": op, "batch": batch, "kind": kind, "rows": rows, "ctx": ctx, "hq": hq, "hk": hk, "d": d,
                "type": rng.choice(["f16", "f16", "f32"])}
    batch = _log(rng, 1, 64)
    return {"op": op, "batch": batch, "vocab": _log(rng, 1000, 151936), "hist": _log(rng, 1, 8192),
            "bias": rng.choice([0, 1, 7, 64, 300]), "mask": rng.random() < 0.7, "type": rng.choice(["f16", "f32"]),
            "ids": rng.choice(["i32", "i64"])}


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _frequencies(rd, table):
    """inverse frequencies of the pairs and the factor on cosine and sine: theta^(-2i/rd), positions divided (linear),
    the base raised (ntk), or the slow frequencies divided and the fast ones kept (yarn), for contexts 4 times as long"""
    theta, factor, trained = 1e6, 4.0, 32768
    i = np.arange(0, rd, 2, dtype=np.float64) / rd
    if table == "ntk":
        theta *= factor ** (rd / (rd - 2)) if rd > 2 else factor
    f = theta ** -i
    if table == "linear":
        f = f / factor
    if table == "yarn":
        turns = trained * f / (2 * math.pi)                    # of a pair over the trained context
        keep = np.clip((turns - 1) / (32 - 1), 0, 1)           # 1: fast, kept; 0: slow, divided
        f = f * keep + f / factor * (1 - keep)
    return f.astype(np.float32), 0.1 * math.log(factor) + 1 if table == "yarn" else 1.0


def _batch(case, rng):
    """rows of each sequence and the positions of their first ones"""
    B, T, ctx, kind = case["batch"], case["rows"], case["ctx"], case["kind"]
    if kind in ("single", "even"):
        n = np.full(B, T // B)
    elif kind == "mixed":  # one prompt's chunk, the others decode
        n = np.ones(B, np.int64)
        n[rng.integers(B)] += T - B
    else:
        cuts = np.sort(rng.integers(0, T - B + 1, B - 1))
        n = np.diff(np.concatenate([[0], cuts, [T - B]])) + 1
    start = np.full(B, ctx) if B == 1 or ctx == 0 else rng.integers(ctx // 16, ctx + 1, B)
    return n.astype(np.int64), start.astype(np.int64)


def _pages(case, n, start, rng):
    """a page table whose sequences hold the pages they need, handed out in a random order from a pool that has enough
    for any batch of the case; -1 behind them"""
    held = (start + n + PAGE - 1) // PAGE
    table = np.full((len(n), int(held.max())), -1, np.int32)
    order = rng.permutation((case["batch"] * case["ctx"] + case["rows"]) // PAGE + 2 * case["batch"])
    at = 0
    for b, h in enumerate(held):
        table[b, :h] = order[at:at + h]
        at += h
    return table, len(order)


def prepare(case, seed):
    rng = np.random.default_rng(seed)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def randn(*shape, type="f32", scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(TORCH[type])

    def dev(a):
        return torch.from_numpy(np.ascontiguousarray(a)).cuda()

    s = dict(case)
    if case["op"] == "rotary":
        f, scale = _frequencies(case["rd"], case["table"])
        s |= {"q": randn(case["rows"], case["hq"], case["d"], type=case["type"]),
              "k": randn(case["rows"], case["hk"], case["d"], type=case["type"]),
              "pos": dev(rng.integers(0, case["far"], case["rows"])), "freq": dev(f), "scale": scale}
        return s
    if case["op"] == "logits":
        B, V, H = case["batch"], case["vocab"], case["hist"]
        ids = np.minimum(rng.zipf(1.3, (B, H)), V) - 1          # some tokens come often, most never
        ids = (ids * 7919 + seed) % V
        ids = ids.astype(np.int32 if case["ids"] == "i32" else np.int64)
        length = rng.integers(H // 2, H + 1, B)
        s["ids_by_step"] = case["ids"] == "i64"                 # the decode loop's log: [steps, batch]
        s |= {"logits": randn(B, V, type=case["type"], scale=4.0), "hist_ids": dev(ids.T if s["ids_by_step"] else ids),
              "hist_len": dev(length.astype(np.int32)), "prompt_len": dev((length // 3).astype(np.int32)),
              "repetition": dev(rng.uniform(1.0, 1.4, B).astype(np.float32)),
              "presence": dev(rng.uniform(-0.5, 1.0, B).astype(np.float32)),
              "frequency": dev(rng.uniform(0.0, 0.3, B).astype(np.float32)),
              "bias_ids": None, "bias": None, "allowed": None}
        if case["bias"]:
            at = np.stack([rng.choice(V, case["bias"], replace=False) for _ in range(B)]).astype(np.int32)
            s |= {"bias_ids": dev(at), "bias": dev(rng.uniform(-8, 8, at.shape).astype(np.float32))}
        if case["mask"]:                                        # a grammar allows few tokens in some states, most in others
            share = rng.choice([0.02, 0.9], B)[:, None]
            bits = np.zeros((B, (V + 31) // 32 * 32), bool)
            bits[:, :V] = rng.random((B, V)) < share
            s["allowed"] = dev(np.packbits(bits, axis=1, bitorder="little").view(np.int32))
        return s
    n, start = _batch(case, rng)
    table, n_pages = _pages(case, n, start, rng)
    cu = np.concatenate([[0], np.cumsum(n)])
    hq, hk, d, T = case["hq"], case["hk"], case["d"], int(cu[-1])
    s |= {"cu": dev(cu.astype(np.int32)), "start": dev(start.astype(np.int32)), "page_table": dev(table), "T": T,
          "n_pages": n_pages, "max_q": int(n.max()), "max_len": int((start + n).max())}
    if case["op"] == "chunk":
        s |= {"q": randn(T, hq, d, type=case["type"]), "k_pool": randn(n_pages, hk, PAGE, d, type=case["type"]),
              "v_pool": randn(n_pages, hk, PAGE, d, type=case["type"])}
        return s
    f, scale = _frequencies(case["rd"], "plain")
    pos = np.concatenate([p + np.arange(m) for p, m in zip(start, n)])
    if case["axes"] == 3:                                       # the second and third axis of an image's tokens lag behind
        pos = np.stack([pos, pos - pos % 3, pos - pos % 5])
    s |= {"qkv": randn(T, hq + 2 * hk, d, type=case["type"]), "pos": dev(pos), "freq": dev(f), "scale": scale,
          "qw": dev((1 + 0.1 * rng.standard_normal(d)).astype(np.float32)) if case["norm"] else None,
          "kw": dev((1 + 0.1 * rng.standard_normal(d)).astype(np.float32)) if case["norm"] else None,
          "section": (rng.integers(0, case["rd"] // 6 + 1), rng.integers(0, case["rd"] // 6 + 1)),
          "k_pool": randn(n_pages, hk, PAGE, d, type=case["cache"]), "v_pool": randn(n_pages, hk, PAGE, d, type=case["cache"])}
    return s


# ---- plain forms ----------------------------------------------------------------------------------------------------
def _angles(pos, freq, section, real):
    """cosine and sine [rows, pairs] of position times frequency, formed in 64 bits"""
    if pos.ndim == 1:
        a = pos.double()[:, None] * freq.double()
    else:  # pairs 1, 4, 7, .. below 3 h turn by the second axis, pairs 2, 5, 8, .. below 3 w by the third
        i = torch.arange(freq.numel(), device=freq.device)
        axis = torch.where((i % 3 == 1) & (i < 3 * section[0]), 1, torch.where((i % 3 == 2) & (i < 3 * section[1]), 2, 0))
        a = pos[axis].t().double() * freq.double()
    return a.cos().to(real), a.sin().to(real)


def _rotate(x, c, s, rd, inter, scale):
    """x [rows, heads, d] rotated by c, s [rows, rd / 2]"""
    c, s = (c * scale)[:, None, :], (s * scale)[:, None, :]
    if inter:
        a, b = x[..., 0:rd:2], x[..., 1:rd:2]
        y = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = x[..., :rd // 2], x[..., rd // 2:rd]
        y = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([y, x[..., rd:]], -1)


def _rotary(s):
    c, n = _angles(s["pos"], s["freq"], None, torch.float32)
    return [_rotate(x.float(), c, n, s["rd"], s["inter"], s["scale"]).to(x.dtype) for x in (s["q"], s["k"])]


def _rows(s):
    """sequence of every row, and its position in that sequence's cache"""
    t = torch.arange(s["T"], device="cuda")
    b = torch.searchsorted(s["cu"][1:].long(), t, right=True)
    return b, s["start"].long()[b] + t - s["cu"].long()[b]


def _append(s):
    hq, hk = s["hq"], s["hk"]
    b, at = _rows(s)
    c, n = _angles(s["pos"], s["freq"], s["section"], torch.float32)
    x = s["qkv"].float()
    q, k, v = x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]
    if s["norm"]:
        q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + 1e-6) * s["qw"]
        k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + 1e-6) * s["kw"]
    q = _rotate(q, c, n, s["rd"], s["inter"], s["scale"])
    k = _rotate(k, c, n, s["rd"], s["inter"], s["scale"])
    page, row = s["page_table"].long()[b, at // PAGE], at % PAGE
    s["k_pool"][page, :, row] = k.to(s["k_pool"].dtype)
    s["v_pool"][page, :, row] = v.to(s["v_pool"].dtype)
    return [q.to(s["k_pool"].dtype), s["k_pool"], s["v_pool"]]


def _chunk(s):
    hq, hk, d, S = s["hq"], s["hk"], s["d"], s["max_q"]
    g, P = hq // hk, (s["max_len"] + PAGE - 1) // PAGE
    b, at = _rows(s)
    off = torch.arange(s["T"], device="cuda") - s["cu"].long()[b]
    B, L = s["batch"], P * PAGE
    q = torch.zeros(B, S, hk, g, d, device="cuda")
    q[b, off] = s["q"].float().view(-1, hk, g, d)
    q = (q * d ** -0.5).permute(0, 2, 3, 1, 4).reshape(B * hk, g * S, d)
    pages = s["page_table"].long()[:, :P].clamp_min(0)
    k = s["k_pool"][pages].float().permute(0, 2, 4, 1, 3).reshape(B * hk, d, L).contiguous()
    v = s["v_pool"][pages].float().permute(0, 2, 1, 3, 4).reshape(B * hk, L, d).contiguous()
    p = torch.bmm(q, k).view(B, hk * g, S, L)
    last = torch.full((B, S), -1, device="cuda", dtype=torch.long)
    last[b, off] = at
    p.masked_fill_((torch.arange(L, device="cuda") > last[..., None])[:, None], float("-inf"))
    m = p.amax(-1, keepdim=True).clamp_min(-1e30)
    p.sub_(m).exp_()
    total = p.sum(-1).clamp_min(1e-30)
    o = torch.bmm(p.view(B * hk, g * S, L), v).view(B, hk * g, S, d) / total[..., None]
    return o.permute(0, 2, 1, 3)[b, off].to(s["q"].dtype)


def _logits(s):
    B, V = s["logits"].shape
    x = s["logits"].float()
    ids = s["hist_ids"].long()
    ids = ids.t() if s["ids_by_step"] else ids
    t = torch.arange(ids.shape[1], device="cuda")
    one = torch.ones((), device="cuda").expand(ids.shape)
    seen = torch.zeros(B, V + 1, device="cuda").scatter_add_(1, torch.where(t < s["hist_len"][:, None], ids, V), one)[:, :V]
    said = (t < s["hist_len"][:, None]) & (t >= s["prompt_len"][:, None])
    count = torch.zeros(B, V + 1, device="cuda").scatter_add_(1, torch.where(said, ids, V), one)[:, :V]
    r = s["repetition"][:, None]
    x = torch.where(seen > 0, torch.where(x > 0, x / r, x * r), x)
    x = x - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0)
    if s["bias"] is not None:
        x = x + torch.zeros_like(x).scatter_add_(1, s["bias_ids"].long(), s["bias"])
    if s["allowed"] is not None:
        bits = (s["allowed"][:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
        x = x.masked_fill(bits.flatten(1)[:, :V] == 0, float("-inf"))
    return x.to(s["logits"].dtype)


# ---- the framework's calls ------------------------------------------------------------------------------------------
def _done(status):
    if status:
        raise RuntimeError("libaxhip status %d" % status)


def _at(t):
    return None if t is None else t.data_ptr()


def _own(s):
    from axono_amd import _lib
    lib, stream, op = _lib.load(), torch.cuda.current_stream().cuda_stream, s["op"]
    if op == "rotary":
        q, k, d = s["q"], s["k"], s["d"]
        yq, yk = torch.empty_like(q), torch.empty_like(k)
        _done(lib.axhip_rotary_qk(q.data_ptr(), s["hq"] * d, k.data_ptr(), s["hk"] * d, s["pos"].data_ptr(), s["freq"].data_ptr(),
                                  s["scale"], int(s["inter"]), s["rd"], yq.data_ptr(), yk.data_ptr(), CODE[s["type"]], s["rows"],
                                  s["hq"], s["hk"], d, stream))
        return [yq, yk]
    if op == "append":
        x, hq, hk, d = s["qkv"], s["hq"], s["hk"], s["d"]
        q = torch.empty(s["T"], hq, d, dtype=s["k_pool"].dtype, device="cuda")
        base, size, width = x.data_ptr(), x.element_size(), (hq + 2 * hk) * d
        _done(lib.axhip_rotary_append_paged(base, width, base + hq * d * size, width, base + (hq + hk) * d * size, width,
                                            CODE[s["type"]], _at(s["qw"]), _at(s["kw"]), F32, 1e-6, int(s["norm"]),
                                            s["pos"].data_ptr(), s["axes"], s["freq"].data_ptr(), s["scale"], int(s["inter"]),
                                            s["rd"], int(s["section"][0]), int(s["section"][1]), s["cu"].data_ptr(),
                                            s["start"].data_ptr(), s["page_table"].data_ptr(), q.data_ptr(),
                                            s["k_pool"].data_ptr(), s["v_pool"].data_ptr(), CODE[s["cache"]], s["T"],
                                            s["batch"], hq, hk, d, s["page_table"].shape[1], s["n_pages"], stream))
        return [q, s["k_pool"], s["v_pool"]]
    if op == "chunk":
        q, sizes = s["q"], (s["T"], s["batch"], s["hq"], s["hk"], s["d"], s["max_q"], s["max_len"])
        out = torch.empty_like(q)
        space = torch.empty(lib.axhip_chunk_attention_paged_workspace_bytes(CODE[s["type"]], *sizes), dtype=torch.uint8, device="cuda")
        _done(lib.axhip_chunk_attention_paged(q.data_ptr(), s["k_pool"].data_ptr(), s["v_pool"].data_ptr(),
                                              s["page_table"].data_ptr(), s["cu"].data_ptr(), s["start"].data_ptr(),
                                              out.data_ptr(), space.data_ptr(), space.numel(), CODE[s["type"]], *sizes,
                                              s["page_table"].shape[1], s["n_pages"], stream))
        return out
    x, ids = s["logits"], s["hist_ids"]
    y = torch.empty_like(x)
    by_row, by_step = (1, ids.shape[1]) if s["ids_by_step"] else (ids.shape[1], 1)
    _done(lib.axhip_logits_process(x.data_ptr(), x.shape[1], CODE[s["type"]], ids.data_ptr(), I64 if s["ids"] == "i64" else I32,
                                   by_row, by_step, s["hist"], s["hist_len"].data_ptr(), s["prompt_len"].data_ptr(),
                                   s["repetition"].data_ptr(), s["presence"].data_ptr(), s["frequency"].data_ptr(),
                                   _at(s["bias_ids"]), _at(s["bias"]), _width(s["bias_ids"]), _at(s["allowed"]),
                                   _width(s["allowed"]), y.data_ptr(), x.shape[1], x.shape[0], x.shape[1],
                                   stream))
    return y


def _width(t):
    return 0 if t is None else t.shape[1]


def run(state):
    if own:
        return _own(state)
    return {"rotary": _rotary, "append": _append, "chunk": _chunk, "logits": _logits}[state["op"]](state)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case):
    size = {"f16": 2, "f32": 4}
    if case["op"] == "rotary":
        n = case["rows"] * (case["hq"] + case["hk"]) * case["d"]
        return {"bytes": 2 * n * size[case["type"]] + 8 * case["rows"], "flops": 3 * n}
    if case["op"] == "append":
        n = case["rows"] * (case["hq"] + 2 * case["hk"]) * case["d"]
        return {"bytes": n * (size[case["type"]] + size[case["cache"]]) + 8 * case["axes"] * case["rows"],
                "flops": n * (7 if case["norm"] else 3)}
    if case["op"] == "logits":
        B, V = case["batch"], case["vocab"]
        return {"bytes": 2 * B * V * size[case["type"]] + B * (V // 8 if case["mask"] else 0)
                + B * case["hist"] * (4 if case["ids"] == "i32" else 8) + 8 * B * case["bias"], "flops": 4 * B * V}
    B, hq, hk, d = case["batch"], case["hq"], case["hk"], case["d"]
    if case["kind"] == "mixed":
        n, k = case["rows"] - B + 1, B - 1
        ctx = case["ctx"] if B == 1 else case["ctx"] * 17 / 32   # the middle of what start is drawn from
        pairs, keys = n * (ctx + (n + 1) / 2) + k * (ctx + 1), n + k + B * ctx
    else:
        n, ctx = case["rows"] / B, case["ctx"] if B == 1 else case["ctx"] * 17 / 32
        pairs, keys = B * n * (ctx + (n + 1) / 2), B * (ctx + n)
    return {"bytes": size[case["type"]] * (2 * case["rows"] * hq * d + 2 * keys * hk * d), "flops": 4 * hq * d * pairs}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------
def _turned(x, pos, freq, rd, inter, scale, axis=None):
    """every pair of x [rows, heads, d] as a complex number, multiplied by scale * e^(i * position * frequency)"""
    rows = pos.shape[-1]
    p = pos.double().view(1, rows) if pos.ndim == 1 else pos.double()
    axis = torch.zeros(rd // 2, dtype=torch.long, device="cuda") if axis is None else axis
    turn = torch.polar(torch.full((rows, rd // 2), float(scale), dtype=torch.float64, device="cuda"), p[axis].t() * freq.double())
    first = torch.arange(rd // 2, device="cuda") * (2 if inter else 1)
    second = first + (1 if inter else rd // 2)
    z = torch.complex(x[..., first], x[..., second]) * turn[:, None]
    y = x.clone()
    y[..., first], y[..., second] = z.real, z.imag
    return y


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        return [_turned(s[n].double(), s["pos"], s["freq"], s["rd"], s["inter"], s["scale"]) for n in ("q", "k")]
    if case["op"] == "logits":
        out = s["logits"].double()
        ids = s["hist_ids"].cpu().numpy()
        ids = ids.T if s["ids_by_step"] else ids
        for b in range(case["batch"]):
            n, p = int(s["hist_len"][b]), int(s["prompt_len"][b])
            every = torch.from_numpy(np.unique(ids[b, :n])).long().cuda()
            r = float(s["repetition"][b])
            v = out[b, every]
            out[b, every] = torch.where(v > 0, v / r, v * r)
            which, times = np.unique(ids[b, p:n], return_counts=True)
            out[b, torch.from_numpy(which).long().cuda()] -= (torch.from_numpy(times).cuda().double() * float(s["frequency"][b])
                                                              + float(s["presence"][b]))
            if s["bias"] is not None:
                out[b, s["bias_ids"][b].long()] += s["bias"][b].double()
            if s["allowed"] is not None:
                bits = np.unpackbits(s["allowed"][b].cpu().numpy().view(np.uint8), bitorder="little")[:case["vocab"]]
                out[b, torch.from_numpy(bits == 0).cuda()] = -math.inf
        return out
    cu, start, table = (s[n].cpu().numpy() for n in ("cu", "start", "page_table"))
    if case["op"] == "append":
        hq, hk = case["hq"], case["hk"]
        i = np.arange(case["rd"] // 2)
        axis = np.zeros(len(i), np.int64)
        if case["axes"] == 3:
            axis[(i % 3 == 1) & (i < 3 * s["section"][0])] = 1
            axis[(i % 3 == 2) & (i < 3 * s["section"][1])] = 2
        x = s["qkv"].double()
        heads = []
        for part, w in ((x[:, :hq], s["qw"]), (x[:, hq:hq + hk], s["kw"])):
            if case["norm"]:
                part = part / torch.sqrt((part ** 2).sum(-1, keepdim=True) / case["d"] + 1e-6) * w.double()
            heads.append(_turned(part, s["pos"], s["freq"], case["rd"], case["inter"], s["scale"], torch.from_numpy(axis).cuda()))
        pools = [s["k_pool"].double(), s["v_pool"].double()]
        for b in range(case["batch"]):
            p = start[b] + np.arange(cu[b + 1] - cu[b])
            page, row = torch.from_numpy(table[b, p // PAGE]).long().cuda(), torch.from_numpy(p % PAGE).long().cuda()
            for pool, new in zip(pools, (heads[1], x[:, hq + hk:])):
                pool.transpose(1, 2)[page, row] = new[cu[b]:cu[b + 1]]
        return [heads[0], *pools]
    g, d = case["hq"] // case["hk"], case["d"]
    out = torch.zeros(s["T"], case["hq"], d, dtype=torch.float64, device="cuda")
    for b in range(case["batch"]):
        n, L = int(cu[b + 1] - cu[b]), int(start[b] + cu[b + 1] - cu[b])
        pages = torch.from_numpy(table[b, :(L + PAGE - 1) // PAGE]).long().cuda()
        hidden = torch.arange(L, device="cuda") > int(start[b]) + torch.arange(n, device="cuda")[:, None]
        for h in range(case["hk"]):
            k = s["k_pool"][pages, h].reshape(-1, d)[:L].double()
            v = s["v_pool"][pages, h].reshape(-1, d)[:L].double()
            for j in range(h * g, h * g + g):
                score = (s["q"][cu[b]:cu[b + 1], j].double() @ k.t().contiguous()) / math.sqrt(d)
                score[hidden] = -math.inf
                out[cu[b]:cu[b + 1], j] = torch.softmax(score, -1) @ v
    return out
