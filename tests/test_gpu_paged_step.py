"""The operators of a paged serving step together, as the decoder, the cache and a captured step use them."""
import numpy as np
import pytest

from axono_amd import DataType, HIPGraph, Tensor, libaxono as L, nn
from axono_amd.device import AxhipError
from axono_amd.examples.qwen3vl_text import Qwen3VLTextDecoder, TextConfig, random_weights
from oracle.decode_step import OracleDecoder

import paged_step_util as ps

pytestmark = pytest.mark.gpu

CFG = TextConfig(num_hidden_layers=3, hidden_size=256, num_attention_heads=4, num_key_value_heads=2, head_dim=128,
                 intermediate_size=512, vocab_size=1000)


def hip(a):
    return Tensor.from_numpy_ref(np.ascontiguousarray(a)).to("hip:0")


def decoders(B, max_len, seed=0):
    w = random_weights(CFG, seed)
    rng = np.random.default_rng(seed + 1)
    for k in w:
        if k.endswith("norm.weight"):
            w[k] = (1 + 0.1 * rng.standard_normal(w[k].shape)).astype(np.float32)
    order = rng.permutation(B * ((max_len + 127) // 128)).tolist()
    gpu = Qwen3VLTextDecoder(CFG, w, B, max_len, "hip:0", paged=True)
    gpu._cache = nn.PagedKVCache(CFG.num_hidden_layers, B, 2, 128, len(order), max_len, DataType.FLOAT16, "hip:0", page_order=order)
    return gpu, OracleDecoder(CFG, w, B, max_len), rng


@pytest.mark.parametrize("chunks", [[150], [1, 149], [64, 64, 22], [128, 1, 1, 20]])
def test_prefill_in_chunks_gives_the_logits_of_the_whole_prompt(chunks):
    """against the oracle's prefill, at the bar of the model tests (2e-3: fp16 data formats inside)"""
    gpu, cpu, rng = decoders(3, 256)
    ids = rng.integers(0, CFG.vocab_size, (3, sum(chunks)))
    at = 0
    for c in chunks:
        logits, nxt = gpu.prefill_chunk(list(ids[:, at:at + c]))
        at += c
    want, _ = cpu.prefill(ids)
    assert np.abs(logits.to_numpy() - want).max() <= 2e-3
    np.testing.assert_array_equal(nxt.to_numpy(), logits.to_numpy().argmax(-1))
    np.testing.assert_array_equal(gpu.cache.seq_lens.to_numpy(), [150] * 3)


def test_chunks_beside_decoding_sequences():
    """one sequence decodes token by token while the others are prefilled in uneven chunks, some steps without them"""
    gpu, cpu, rng = decoders(3, 256, seed=2)
    ids = rng.integers(0, CFG.vocab_size, (3, 140))
    plan = [(10, 130, 0), (1, 0, 1), (1, 5, 126), (0, 0, 0), (128, 5, 13)]
    at = np.zeros(3, int)
    last = {}
    for step in plan:
        logits, _ = gpu.prefill_chunk([ids[b, at[b]:at[b] + step[b]] for b in range(3)])
        if sum(step) == 0:
            assert logits is None
            continue
        for row, b in enumerate([b for b in range(3) if step[b]]):
            last[b] = logits.to_numpy()[row]
        at += step
    assert list(at) == [140] * 3
    want, _ = cpu.prefill(ids)
    for b in range(3):
        assert np.abs(last[b] - want[b]).max() <= 2e-3


@pytest.mark.parametrize("use_graph", [False, True])
def test_decode_after_chunked_prefill(use_graph):
    gpu, cpu, rng = decoders(2, 256, seed=4)
    ids = rng.integers(0, CFG.vocab_size, (2, 130))
    for c in (ids[:, :100], ids[:, 100:]):
        _, nxt = gpu.prefill_chunk(list(c))
    cpu.prefill(ids)
    first, pos = nxt.to_numpy(), np.full((3, 2), 130, np.int64)
    gpu.start_decode(first, pos, 5)
    if use_graph:
        gpu.capture()
    toks = gpu.generate(5, use_graph=use_graph)
    cur = first
    for s in range(5):
        logits, _ = cpu.decode_step(cur, pos + s)
        assert np.all(logits[np.arange(2), toks[s]] >= logits.max(-1) - 4e-3)
        cur = toks[s]


def test_sampling_of_a_decode_loop():
    """the captured loop with penalties, biases and a mask: the eager loop's tokens, and what they forbid never comes"""
    B, V, steps = 2, CFG.vocab_size, 12
    rng = np.random.default_rng(7)
    allowed = np.zeros((B, (V + 31) // 32), np.uint32)
    may = np.sort(rng.choice(V, (B, 40), replace=False), axis=1)
    for b in range(B):
        for t in may[b]:
            allowed[b, t // 32] |= np.uint32(1 << (t % 32))
    never = may[:, 3:4].astype(np.int32)
    sampling = dict(presence=hip(np.full(B, 1e4, np.float32)), bias_ids=hip(never), bias=hip(np.full((B, 1), -1e6, np.float32)),
                    allowed=hip(allowed.view(np.int32)))
    got = []
    for use_graph in (False, True):
        gpu, _, r = decoders(B, 256, seed=9)
        ids = r.integers(0, V, (B, 20))
        _, nxt = gpu.prefill_chunk(list(ids))
        gpu.start_decode(nxt.to_numpy(), np.full((3, B), 20, np.int64), steps, sampling=sampling)
        if use_graph:
            gpu.capture()
        got.append(gpu.generate(steps, use_graph=use_graph))
    np.testing.assert_array_equal(got[0], got[1])
    for b in range(B):
        assert set(got[0][:, b]) <= set(may[b]) - {never[b, 0]}
        assert len(set(got[0][:, b])) == steps            # presence: no token twice


def test_captured_append_and_attention_follow_lengths_on_the_device():
    """a graph of append + attention + the lengths' increment, replayed: every replay against the eager calls on a copy, with eager
    work and synchronizations between the replays"""
    B, hq, hk, d, steps = 3, 4, 2, 64, 6
    rng = np.random.default_rng(3)
    n = np.array([2, 1, 2])
    cu = hip(ps.cu_of(n))
    table, _ = L.rotary_inv_freq(d, 1e6, device="hip:0")
    caches = [nn.PagedKVCache(1, B, hk, d, 12, 300, DataType.FLOAT16, "hip:0") for _ in range(2)]
    for c in caches:
        c.reserve(np.array([100, 250, 128]) + 4 * steps)
        c._lens = np.array([100, 250, 125])
        c.seq_lens.copy_from_numpy(c._lens.astype(np.int32))
        for pool in c.get(0):
            pool.copy_from_numpy(np.random.default_rng(5).standard_normal(pool.shape).astype(np.float16))
    qkv = hip(rng.standard_normal((5, (hq + 2 * hk) * d)).astype(np.float32))

    def body(c):
        q = c.append_chunk(0, qkv, hq, table, cu, eps=1e-6)
        return c.attend_chunk(0, q, cu, 2, max_len=300)

    g = HIPGraph()
    out = []
    g.capture(lambda: out.append(body(caches[0])))
    graph_out = out[-1]
    for s in range(steps):
        x = rng.standard_normal(qkv.shape).astype(np.float32)
        qkv.copy_from_numpy(x)
        g.replay()
        eager = body(caches[1])
        L.synchronize()
        np.testing.assert_array_equal(graph_out.to_numpy(), eager.to_numpy())
        for a, b in zip(caches[0].get(0), caches[1].get(0)):
            np.testing.assert_array_equal(a.to_numpy(), b.to_numpy())
        for c in caches:
            c.advance_each(n)


def test_graphs_with_workspaces_of_their_own_run_side_by_side():
    rng = np.random.default_rng(6)
    n, start = [3, 1], [2000, 700]
    made = []
    for k in range(2):
        table, n_pages = ps.pages_for(n, start, rng)
        q = rng.standard_normal((4, 8, 64)).astype(np.float16)
        pools = [rng.standard_normal((n_pages, 2, 128, 64)).astype(np.float16) for _ in range(2)]
        args = [hip(a) for a in (q, *pools, table, ps.cu_of(n), np.array(start, np.int32))]
        g, out = HIPGraph(), []
        g.capture(lambda: out.append(L.chunk_attention_paged(*args, 3, 2003)))
        made.append((g, out, args, ps.chunk_want(q, *pools, table, n, start, 2003)))
    for _ in range(5):
        for g, *_ in made:
            g.launch_async()
        for g, *_ in made:
            g.sync()
        for _, out, _, (want, tol) in made:
            ps.assert_within(out[-1].numpy(), want, tol)


def test_surface_functions_and_their_refusals():
    rng = np.random.default_rng(8)
    q, k = rng.standard_normal((5, 4, 64)).astype(np.float32), rng.standard_normal((5, 2, 64)).astype(np.float32)
    pos = rng.integers(0, 500, 5)
    f, scale = L.rotary_inv_freq(32, 1e4, "yarn", factor=8.0, trained_len=256, device="hip:0")
    got = L.rotary_qk(hip(q), hip(k), hip(pos), f, scale, interleaved=True)
    for x, y in zip((q, k), got):
        want, size = ps.turned(x, pos, f.to_numpy(), 32, True, scale)
        ps.assert_within(y.numpy(), want, size * ps.ROTATION + np.abs(want) * 2.0 ** -24)
    bad = [lambda: L.rotary_qk(hip(q), hip(k[:4]), hip(pos), f), lambda: L.rotary_qk(hip(q), None, hip(pos[:4]), f),
           lambda: L.rotary_qk(hip(q), hip(k.astype(np.float16)), hip(pos), f), lambda: L.rotary_qk(hip(q), None, hip(pos.astype(np.int32)), f),
           lambda: L.rotary_qk(hip(q), None, hip(pos), hip(np.ones(40, np.float32))),
           lambda: L.rotary_qk(Tensor.from_numpy_ref(q), None, hip(pos), f)]
    n, start = [2, 3], [0, 100]
    table, n_pages = ps.pages_for(n, start, rng)
    pools = [hip(np.zeros((n_pages, 2, 128, 64), np.float16)) for _ in range(2)]
    cu, st, tb = hip(ps.cu_of(n)), hip(np.array(start, np.int32)), hip(table)
    qkv = hip(rng.standard_normal((5, 8 * 64)).astype(np.float32))
    ok = (qkv, 4, f, cu, st, *pools, tb)
    assert L.rotary_append_paged(*ok).shape == [5, 4, 64]
    bad += [lambda: L.rotary_append_paged(qkv, 5, f, cu, st, *pools, tb), lambda: L.rotary_append_paged(qkv, 4, f, st, st, *pools, tb),
            lambda: L.rotary_append_paged(*ok, pos=hip(pos[:4])), lambda: L.rotary_append_paged(*ok, pos=hip(pos.astype(np.int32))),
            lambda: L.rotary_append_paged(*ok, q_weight=hip(np.ones(64, np.float32))),
            lambda: L.rotary_append_paged(qkv, 4, f, cu, st, pools[0], hip(np.zeros((n_pages, 2, 128, 64), np.float32)), tb)]
    qh = hip(rng.standard_normal((5, 4, 64)).astype(np.float16))
    assert L.chunk_attention_paged(qh, *pools, tb, cu, st, 3, 103).shape == [5, 4, 64]
    bad += [lambda: L.chunk_attention_paged(hip(q), *pools, tb, cu, st, 3, 103), lambda: L.chunk_attention_paged(qh, *pools, tb, cu, st, 3, 1 << 20),
            lambda: L.chunk_attention_paged(qh, *pools, tb, st, st, 3, 103),
            lambda: L.chunk_attention_paged(qh, *pools, tb, cu, st, 3, 103, out=hip(np.zeros((5, 4, 64), np.float32)))]
    x = hip(rng.standard_normal((2, 100)).astype(np.float32))
    ids = hip(np.zeros((2, 7), np.int32))
    assert L.logits_process(x, ids, repetition=hip(np.ones(2, np.float32))).shape == [2, 100]
    bad += [lambda: L.logits_process(x, ids, by_step=True), lambda: L.logits_process(x, bias_ids=ids),
            lambda: L.logits_process(x, ids, presence=hip(np.ones(3, np.float32))),
            lambda: L.logits_process(x, allowed=hip(np.zeros((2, 3), np.int32))), lambda: L.logits_process(x, out=qh)]
    for f_ in bad:
        with pytest.raises(AxhipError):
            f_()
    with pytest.raises(ValueError):
        L.rotary_inv_freq(32, kind="other")
    with pytest.raises(ValueError):
        decoders(1, 128)[0].prefill_chunk([[1], [2]])


def test_advance_each_needs_the_pages():
    cache = nn.PagedKVCache(1, 2, 1, 64, 6, 512, device="hip:0")
    cache.reserve([100, 300])
    cache.advance_each([100, 300])
    for bad in ([29, 0], [0, 85], [-1, 0]):
        with pytest.raises(ValueError):
            cache.advance_each(bad)
    cache.advance_each([28, 84])
    assert cache.seq_lens.to_numpy().tolist() == [128, 384]


def test_pages_beyond_four_gigabytes():
    """the same pages at the end of a pool of 4.3 GB and in a small one: the same bits"""
    hq, hk, d, far = 8, 8, 128, 16500
    rng = np.random.default_rng(11)
    n, start, where = [3, 1], [254, 5], [far - 1, 7, 16390, far - 3]
    near_table = np.array([[0, 1, 2], [3, -1, -1]], np.int32)
    far_table = np.array([where[:3], [where[3], -1, -1]], np.int32)
    page_bytes = hk * 128 * d * 2
    table, _ = L.rotary_inv_freq(d, 1e6, device="hip:0")
    cu, st = hip(ps.cu_of(n)), hip(np.array(start, np.int32))
    qkv = hip(rng.standard_normal((4, (hq + 2 * hk) * d)).astype(np.float32))
    old = [hip(rng.standard_normal((4, hk, 128, d)).astype(np.float16)) for _ in range(2)]
    pools = [Tensor(DataType.FLOAT16, [far, hk, 128, d], "hip:0", _zero=False) for _ in range(2)]
    for small, large in zip(old, pools):
        for i, p in enumerate(where):
            L.copy_bytes(large, p * page_bytes, small, i * page_bytes, page_bytes)
    results = []
    for ks, tb in ((old, near_table), (pools, far_table)):
        q = L.rotary_append_paged(qkv, hq, table, cu, st, *ks, hip(tb), eps=1e-6)
        results.append(L.chunk_attention_paged(q, *ks, hip(tb), cu, st, 3, 257).to_numpy())
    np.testing.assert_array_equal(results[0], results[1])
    for small, large in zip(old, pools):
        back = Tensor(DataType.FLOAT16, [4, hk, 128, d], "hip:0")
        for i, p in enumerate(where):
            L.copy_bytes(back, i * page_bytes, large, p * page_bytes, page_bytes)
        np.testing.assert_array_equal(back.to_numpy(), small.to_numpy())


def test_bounds_wider_than_an_int_do_not_wrap():
    """max_q of 2^32 bounds nothing; a max_len that the page table does not hold is refused, whatever its low bits say"""
    n, start = [3, 1], [200, 5]
    q, k, v, table = ps.picking(n, start, 4, 2, 64, np.float16)
    args = [hip(a) for a in (q, k, v, table, ps.cu_of(n), np.array(start, np.int32))]
    want = L.chunk_attention_paged(*args, 3, 203).numpy()
    for max_q in (1 << 32, (1 << 40) + 1, 1 << 31):
        out = hip(np.full(q.shape, 9, np.float16))
        np.testing.assert_array_equal(L.chunk_attention_paged(*args, max_q, 203, out=out).numpy(), want)
    for bad in ((3, 1 << 32), (3, (1 << 32) + 203), (3, -1), (-1, 203), (-(1 << 32), 203)):
        with pytest.raises(AxhipError):
            L.chunk_attention_paged(*args, *bad)
