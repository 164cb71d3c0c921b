"""Forks of requests through the engine: what a parent has not run is not handed on."""

import pytest
import torch

from helpers import TINY, seeded_tokens

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def engine_of(tmp_models):
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from stride_b200 import Engine, config_from_dict, preset, write_random_model

    def make(name, **options):
        cfg = TINY[name] if name in TINY else preset(name)
        folder = write_random_model(config_from_dict(cfg), seed=3, out_dir=str(tmp_models / f"fork-{name}"), stored_dtype="float32", std=0.08, vector_jitter=0.1)
        return Engine(folder, dtype="float32", block_size=8, num_blocks=40, max_model_len=128, max_batch_seqs=4, check_invariants=True, **options)
    return make


@pytest.mark.parametrize("cache_dtype", [None, "int4"])
def test_tokens_that_have_not_run_are_not_forked(engine_of, cache_dtype):
    engine = engine_of("A", cache_dtype=cache_dtype)
    tokens = seeded_tokens(40, engine.model.vocab, 1)
    engine.cache.open(1)
    engine.cache.ensure(1, 64, 0)                           # pages for more than is run
    engine.forward([(1, tokens[:10], 0, [])])
    live = engine.cache.stats()["live"]
    for count in (11, 32, 64, 100):
        with pytest.raises(ValueError, match="has run 10 tokens"):
            engine.fork(1, 2, count)
    assert not engine.cache.has(2) and engine.cache.stats()["live"] == live
    engine.fork(1, 2, 10)
    engine.cache.ensure(2, 20, 0)
    want = engine.forward([(1, tokens[10:20], 10, range(10))]).clone()
    assert torch.equal(want, engine.forward([(2, tokens[10:20], 10, range(10))]))
    engine.fork(2, 3, 17)                                   # of a fork, within what it has run
    engine.cache.check_invariants()


def test_a_state_is_forked_where_it_stands(engine_of):
    engine = engine_of("nidilix-tiny")
    tokens = seeded_tokens(30, engine.model.vocab, 2)
    engine.cache.open(1)
    engine.cache.ensure(1, 30, 0)
    engine.forward([(1, tokens[:21], 0, [])])
    for count in (5, 20):
        with pytest.raises(ValueError, match="keep a state"):
            engine.fork(1, 2, count)
    with pytest.raises(ValueError, match="has run 21"):
        engine.fork(1, 2, 22)
    engine.fork(1, 2, 21)
    engine.fork(1, 3, 0)                                    # from the beginning
    for key in (2, 3):
        engine.cache.ensure(key, 30, 0)
    want = engine.forward([(1, tokens[21:], 21, range(9))]).clone()
    assert torch.equal(want, engine.forward([(2, tokens[21:], 21, range(9))]))
    fresh = engine.forward([(3, tokens[:21], 0, [20])]).clone()
    engine.cache.close(2)
    engine.cache.open(4)
    engine.cache.ensure(4, 21, 0)
    assert torch.equal(fresh, engine.forward([(4, tokens[:21], 0, [20])]))
