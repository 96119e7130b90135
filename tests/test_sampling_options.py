"""Options of a request's sampling: what they refuse, how allowed tokens are packed, that a preempted request keeps them."""
import math

import numpy as np
import pytest

from kv_cache_optimization_for_llm_amd.cache.manager import CacheError, CacheManager
from kv_cache_optimization_for_llm_amd.engine.scheduler import Request, Scheduler
from kv_cache_optimization_for_llm_amd.parts.base import attention_cache_spec
from kv_cache_optimization_for_llm_amd.sampling.options import AllowedWords, SampleOptions, pack_allowed


@pytest.mark.parametrize("bad", [
    dict(top_k=-1), dict(top_k=1.5), dict(top_k=1 << 31), dict(top_p=0.0), dict(top_p=1.01), dict(top_p=math.nan), dict(min_p=-0.1),
    dict(min_p=1.5), dict(min_p=math.nan), dict(repetition_penalty=0.0), dict(repetition_penalty=math.inf), dict(presence_penalty=math.nan),
    dict(frequency_penalty=math.inf), dict(logit_bias={-1: 0.0}), dict(logit_bias={1.5: 0.0}), dict(logit_bias={3: math.nan}),
    dict(logit_bias={3: math.inf}), dict(grammar=[1, 2])])
def test_options_refuse(bad):
    with pytest.raises(ValueError):
        SampleOptions(**bad)


def test_options_say_what_they_ask_for():
    assert not SampleOptions().truncates and not SampleOptions().penalizes
    assert SampleOptions(top_k=1).truncates and SampleOptions(top_p=0.9).truncates and SampleOptions(min_p=0.1).truncates
    assert SampleOptions(repetition_penalty=1.1).penalizes and SampleOptions(presence_penalty=-1.0).penalizes
    assert not SampleOptions(repetition_penalty=1.0, logit_bias={3: -math.inf}).penalizes


@pytest.mark.parametrize("vocab", [1, 31, 32, 33, 100])
def test_pack_allowed(vocab):
    rng = np.random.default_rng(vocab)
    for share in (0.0, 0.3, 1.0):
        free = rng.random(vocab) < share
        ids = np.nonzero(free)[0]
        for given in (free, ids, ids.tolist(), set(ids.tolist()), np.repeat(ids, 2), free.tolist()):
            words = pack_allowed(given, vocab)
            assert words.dtype == np.int32 and words.shape == ((vocab + 31) // 32,)
            assert [bool(int(words[t // 32]) >> (t % 32) & 1) for t in range(vocab)] == free.tolist()
        assert np.array_equal(pack_allowed(words, vocab), words) and np.array_equal(pack_allowed(words.view(np.uint32), vocab), words)
    assert pack_allowed(None, vocab) is None
    for bad in ([vocab], [-1], [0.5], np.zeros(vocab + 1, bool), np.zeros((2, 2), int)):
        with pytest.raises(ValueError):
            pack_allowed(bad, vocab)


def cache(pages=64, max_len=64):
    return CacheManager([(attention_cache_spec(2, 16), [0, 1])], {}, page_size=4, num_pages=pages, max_seqs=4, max_seq_len=max_len)


def test_a_preempted_request_keeps_its_options():
    s = Scheduler(cache(pages=6), max_batch_tokens=64)
    options = [SampleOptions(top_k=3), SampleOptions(min_p=0.5)]
    for i, o in enumerate(options):
        s.add(Request(i, list(range(8, 17)), 20, options=o))
    events = []
    while not any(e.kind == "preempted" for e in events):
        plan = s.plan()
        events += plan.events
        for e in plan.entries:
            assert s.cache.grow(e.seq.seat, e.start + len(e.tokens))
        events += s.complete(plan, [9] * sum(e.sample for e in plan.entries))
    assert s.waiting[0].preempted and s.waiting[0].options is options[s.waiting[0].id]
    assert s.running[0].request.options is options[s.running[0].request.id]


def test_positions_without_a_page_are_refused():
    m = cache()
    seat = m.admit("a")
    assert m.grow(seat, 10)
    m.check_mapped(seat, 0, 12, 0)
    m.check_mapped(seat, 11, 1, 0)
    m.check_mapped(seat, 12, 0, 0)
    with pytest.raises(CacheError):
        m.check_mapped(seat, 0, 13, 0)
    with pytest.raises(CacheError):
        m.check_mapped(seat, 12, 1, 0)
    m.flush_tables()                    # (no device: nothing to bring up to date)
    assert not m.groups[0].dirty


@pytest.mark.parametrize("bad", [dict(logit_bias={3: 1e39}), dict(presence_penalty=1e39), dict(frequency_penalty=-1e39), dict(repetition_penalty=1e-50),
                                 dict(repetition_penalty=1e39), dict(logit_bias={3: float("nan")})])
def test_numbers_that_32_bits_do_not_hold_are_refused(bad):
    with pytest.raises(ValueError):
        SampleOptions(**bad)


def test_a_ban_may_be_as_low_as_it_likes():
    assert SampleOptions(logit_bias={3: -1e300, 4: -float("inf")}).logit_bias[4] == -float("inf")


@pytest.mark.parametrize("dtype", [np.int8, np.int16, np.int32, np.uint32, np.int64])
def test_ids_of_any_type_and_number_are_ids(dtype):
    """Also exactly as many as there are words of 32 tokens."""
    for vocab, ids in ((20, [3]), (64, [3, 5]), (100, [0, 1, 2, 99]), (128, [3, 5, 7, 9]), (128, [1, 1, 2, 127])):
        want = pack_allowed(sorted(set(ids)), vocab)
        assert len(ids) == len(want) and np.array_equal(pack_allowed(np.asarray(ids, dtype), vocab), want)


def test_words_say_that_they_are():
    words = np.asarray([0b1010, -2], np.int32)
    free = [t in (1, 3) or 33 <= t for t in range(64)]
    for given in (AllowedWords(words), AllowedWords(words.view(np.uint32)), AllowedWords(np.repeat(words, 2)[::2])):
        assert np.array_equal(pack_allowed(given, 64), pack_allowed(free, 64))
    for vocab in (32, 65):
        with pytest.raises(ValueError):
            pack_allowed(AllowedWords(words), vocab)
    with pytest.raises(ValueError):
        pack_allowed(AllowedWords(words).astype(np.int64), 64)
    for bad in (words.astype(np.int64), words[None], [1.5, 2]):
        with pytest.raises(ValueError):
            AllowedWords(bad)


def test_positions_outside_the_table_are_refused():
    m = cache(max_len=62)               # 16 blocks of 4
    seat = m.admit("a")
    assert m.grow(seat, 62)
    m.check_mapped(seat, 0, 64, 0)
    m.check_mapped(seat, 63, 1, 0)
    m.check_mapped(seat, 64, 0, 0)
    for start, count in ((60, 5), (60, 10), (64, 1), (100, 3), (-1, 1), (-1, 64), (-8, 2), (0, 1 << 40)):
        with pytest.raises(CacheError):
            m.check_mapped(seat, start, count, 0)
