"""The decode loop with penalties, biases and masks: what its history holds, and what it leaves behind."""
import numpy as np
import pytest

from axono_amd import Tensor
from axono_amd.examples.qwen3vl_text import Qwen3VLTextDecoder, TextConfig, random_weights

import paged_step_util as ps

pytestmark = pytest.mark.gpu

CFG = TextConfig(num_hidden_layers=2, hidden_size=256, num_attention_heads=4, num_key_value_heads=2, head_dim=128,
                 intermediate_size=512, vocab_size=1000)
B, V = 3, CFG.vocab_size


def hip(a):
    return Tensor.from_numpy_ref(np.ascontiguousarray(a)).to("hip:0")


def prompts(seed):
    rng = np.random.default_rng(seed)
    return [rng.integers(0, V, n) for n in (23, 1, 140)]


def started(seed=0):
    """a decoder that holds the prompts, and their next tokens"""
    gpu = Qwen3VLTextDecoder(CFG, random_weights(CFG, seed), B, 256, "hip:0", paged=True)
    ids = prompts(seed)
    gpu.prefill_chunk([ids[0][:10], [], ids[2][:139]])
    _, nxt = gpu.prefill_chunk([[], ids[1], []])
    middle = nxt.to_numpy()[0]
    _, nxt = gpu.prefill_chunk([ids[0][10:], [], ids[2][139:]])
    return gpu, ids, np.array([nxt.to_numpy()[0], middle, nxt.to_numpy()[1]])


def positions(ids):
    return np.tile(np.array([len(x) for x in ids], np.int64), (3, 1))


def penalties(repetition=2.0, presence=0.5, frequency=0.25):
    """by row: all three, without repetition, without the others"""
    row = lambda *x: hip(np.array(x, np.float32))  # noqa: E731
    return dict(repetition=row(repetition, 1, repetition), presence=row(presence, presence, 0), frequency=row(frequency, frequency, 0))


@pytest.mark.parametrize("use_graph", [False, True])
def test_penalties_see_the_prompt_the_first_token_and_every_step(use_graph):
    """the logits of every step against the formula, made from the logits of a loop without penalties that is fed the same tokens;
    bar of the model tests (2e-3), times the repetition penalty"""
    steps = 8
    gpu, ids, first = started()
    plain, _, _ = started()
    gpu.start_decode(first, positions(ids), steps, sampling=penalties())
    if use_graph:
        gpu.capture()
    rep, pres, freq = (penalties()[n].to_numpy() for n in ("repetition", "presence", "frequency"))
    said = [[int(t)] for t in first]
    cur, pos = first.astype(np.int64), positions(ids)
    for s in range(steps):
        plain.cache.reserve(1)
        raw, _ = plain.decode_forward(hip(cur), hip(pos + s), gpu._decode_bound)
        plain.cache.advance(1)
        hist = np.full((B, 200), -1, np.int64)
        for b in range(B):
            hist[b, :len(ids[b]) + len(said[b])] = [*ids[b], *said[b]]
        n = [len(i) + len(t) for i, t in zip(ids, said)]
        want, tol = ps.logits_want(raw.to_numpy(), hist, n, [len(i) for i in ids], rep, pres, freq, None, None, None)
        if use_graph:
            gpu._graph.replay()
            logits, nxt = gpu._graph_out
        else:
            logits, nxt = gpu._step_fn()
        assert np.abs(logits.to_numpy() - want).max() <= 4e-3, s
        cur = nxt.to_numpy().copy()
        for b in range(B):
            said[b].append(int(cur[b]))


@pytest.mark.parametrize("use_graph", [False, True])
def test_the_first_token_does_not_come_again(use_graph):
    """presence takes 1e4 off what was said, the first token among it, which a bias of 100 would bring back at once"""
    gpu, ids, first = started(1)
    sampling = dict(presence=hip(np.full(B, 1e4, np.float32)), bias_ids=hip(first[:, None].astype(np.int32)),
                    bias=hip(np.full((B, 1), 100, np.float32)))
    gpu.start_decode(first, positions(ids), 6, sampling=sampling)
    if use_graph:
        gpu.capture()
    toks = gpu.generate(6, use_graph=use_graph)
    assert not np.any(toks == first)


@pytest.mark.parametrize("use_graph", [False, True])
def test_a_loop_in_two_parts_is_the_loop_in_one(use_graph):
    got = []
    for parts in ((12,), (5, 7)):
        gpu, ids, first = started(2)
        gpu.start_decode(first, positions(ids), 12, sampling=penalties(50.0, 8.0, 1.0))
        if use_graph:
            gpu.capture()
        got.append(np.concatenate([gpu.generate(n, use_graph=use_graph) for n in parts]))
        assert got[-1].shape == (12, B)
    np.testing.assert_array_equal(got[0], got[1])


def test_a_loop_that_is_rewound_gives_the_same_tokens():
    gpu, ids, first = started(2)
    gpu.start_decode(first, positions(ids), 6, sampling=penalties(50.0, 8.0, 1.0))
    gpu.capture()
    got = []
    for _ in range(2):
        got.append(gpu.generate(6))
        gpu._ids.copy_from_numpy(first.astype(np.int64))
        gpu._pos.copy_from_numpy(positions(ids))
        gpu.cache.set_lengths([len(i) for i in ids])
    np.testing.assert_array_equal(got[0], got[1])
    gpu.cache.set_lengths([1, 1, 1])
    with pytest.raises(RuntimeError, match="start_decode"):
        gpu.generate(1)


def test_prompts_can_be_given_and_have_to_be_where_they_are_not_known():
    got = []
    for given in (False, True):
        gpu, ids, first = started(3)
        more = [[int(t)] for t in first] if given else first[:, None]
        if given:                                   # tokens that the decoder did not see: written behind its back
            gpu, ids, first = started(3)
            gpu.start_decode(first, positions(ids), 4)
            gpu.generate(1, use_graph=False)
            with pytest.raises(ValueError, match="prompt_ids"):
                gpu.start_decode(gpu._ids.numpy(), gpu._pos.numpy(), 4, sampling=penalties())
            gpu.start_decode(gpu._ids.numpy(), gpu._pos.numpy(), 4, sampling=dict(presence=penalties()["presence"]))  # no need of it
            gpu.start_decode(gpu._ids.numpy(), gpu._pos.numpy(), 4, sampling=penalties(), prompt_ids=[[*i, *m] for i, m in zip(ids, more)])
            got.append(gpu.generate(4, use_graph=False))
        else:                                       # the same tokens through prefill_chunk
            _, nxt = gpu.prefill_chunk(list(more))
            gpu.start_decode(nxt.to_numpy(), positions(ids) + 1, 4, sampling=penalties())
            got.append(gpu.generate(4, use_graph=False))
    np.testing.assert_array_equal(got[0], got[1])
    with pytest.raises(ValueError, match="prompt_ids"):
        gpu.start_decode(first, positions(ids), 4, sampling=penalties(), prompt_ids=[[1], [2]])


def test_a_dense_prefill_is_known_too():
    gpu = Qwen3VLTextDecoder(CFG, random_weights(CFG, 5), B, 64, "hip:0")
    ids = np.random.default_rng(5).integers(0, V, (B, 20))
    got = []
    for prompt in (None, list(ids)):
        _, nxt = gpu.prefill(ids)
        gpu.start_decode(nxt.to_numpy(), np.full((3, B), 20, np.int64), 1, sampling=penalties(), prompt_ids=prompt)
        got.append(gpu._step_fn()[0].to_numpy().copy())
    np.testing.assert_array_equal(got[0], got[1])
    _, nxt = gpu.prefill(ids)
    gpu.start_decode(nxt.to_numpy(), np.full((3, B), 20, np.int64), 1, sampling=penalties(), prompt_ids=[[]] * B)
    other = gpu._step_fn()[0].to_numpy()
    np.testing.assert_array_equal(other[1], got[0][1])            # the row without a repetition penalty
    for b in (0, 2):
        assert set(np.nonzero(other[b] != got[0][b])[0]) == set(ids[b]) - {nxt.to_numpy()[b]}


@pytest.mark.parametrize("key", ["history", "history_len", "prompt_len", "by_step", "out", "temperature"])
def test_what_the_loop_keeps_itself_or_does_not_know_is_refused(key):
    gpu, ids, first = started(4)
    with pytest.raises(ValueError, match=key):
        gpu.start_decode(first, positions(ids), 4, sampling={**penalties(), key: hip(np.zeros(B, np.int32))})


@pytest.mark.parametrize("use_graph", [False, True])
def test_a_step_behind_a_sampled_loop_gives_plain_logits(use_graph):
    """decode_forward and forward take no penalties and masks from a loop that was started before"""
    def tokens():
        return hip(np.arange(B, dtype=np.int64)), hip(positions(ids))

    gpu, ids, first = started(6)
    want = gpu.decode_forward(*tokens())[0].to_numpy().copy()
    gpu.start_decode(first, positions(ids), 4, sampling=dict(allowed=hip(np.full((B, 32), 5, np.int32)), **penalties()))
    if use_graph:
        gpu.capture()
    assert np.isinf((gpu._graph.replay() and gpu._graph_out if use_graph else gpu._step_fn())[0].to_numpy()).any()
    gpu.cache.set_lengths([len(i) for i in ids])
    for step in (gpu.decode_forward, gpu.forward):
        np.testing.assert_array_equal(step(*tokens())[0].to_numpy(), want)


def test_a_new_loop_needs_a_capture_of_its_own():
    """the graph of the loop before applies that loop's penalties and writes to its log"""
    gpu, ids, first = started(7)
    gpu.start_decode(first, positions(ids), 4)
    with pytest.raises(RuntimeError, match="capture"):
        gpu.generate(4)
    old = gpu.capture()
    gpu.start_decode(first, positions(ids), 4, sampling=dict(allowed=hip(np.full((B, 32), 5, np.int32))))
    with pytest.raises(RuntimeError, match="capture"):
        gpu.generate(4)
    assert gpu.generate(0, use_graph=False).shape == (0, B)
    gpu.capture()
    log = gpu._log.to_numpy().copy()
    old.replay()                                    # into its own log
    np.testing.assert_array_equal(gpu._log.to_numpy(), log)
    gpu._ids.copy_from_numpy(first.astype(np.int64))
    gpu._pos.copy_from_numpy(positions(ids))
    gpu.cache.set_lengths([len(i) for i in ids])
    toks = gpu.generate(4)
    assert np.all((5 >> (toks % 32)) & 1)
