"""What portions expand out of a cache in 4 bits: one buffer of a bounded size, whatever a step holds."""

import pytest
import torch

from helpers import TINY, seeded_tokens

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def folder(tmp_models):
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from stride_b200 import config_from_dict, write_random_model
    return write_random_model(config_from_dict(TINY["D"]), seed=3, out_dir=str(tmp_models / "portions-D"), stored_dtype="bfloat16", std=0.08, vector_jitter=0.2)


def engine_of(folder, **options):
    from stride_b200 import Engine
    return Engine(folder, dtype="bfloat16", cache_dtype="int4", block_size=16, num_blocks=256, max_model_len=512, check_invariants=True, **options)


def test_requests_expanded_in_groups_have_the_results_of_all_at_once(folder, monkeypatch):
    from stride_b200.parts.attention import PagedAttention
    lens = [300, 40, 1, 200, 90, 7, 150, 1, 1]               # the last two: single tokens behind the portions
    tokens = [seeded_tokens(n + 60, 515, 10 + i) for i, n in enumerate(lens)]

    def logits(limit):
        monkeypatch.setattr(PagedAttention, "MAX_EXPANDED_BYTES", limit)
        engine = engine_of(folder, max_batch_tokens=1024, max_batch_seqs=16)
        for i in range(len(lens)):
            engine.cache.open(i)
            engine.cache.ensure(i, lens[i] + 60, 0)
            engine.forward([(i, tokens[i][:60], 0, [])])
        out = engine.forward([(i, tokens[i][60:], 60, [n - 1]) for i, n in enumerate(lens)]).clone()
        bytes_of = [b.numel() * 4 for key, b in engine.model.rt._buffers.items() if "int4_expanded" in key]
        return out, bytes_of, engine
    whole, (all_bytes,), _ = logits(1 << 28)
    parts, (bytes_,), engine = logits(1)
    assert torch.equal(whole, parts)
    assert bytes_ == engine.model.expanded_bytes(512, 16) < all_bytes


def test_growing_requests_leave_one_buffer(folder):
    from stride_b200 import SamplingParams
    engine = engine_of(folder, max_batch_tokens=512, max_batch_seqs=8)
    engine.runner.CONTEXT_BUCKET_BASE = 64                   # (many buckets for a short model)
    params = SamplingParams(temperature=0.0, max_tokens=3, ignore_eos=True)
    engine.generate([seeded_tokens(5, 515, 1), seeded_tokens(30, 515, 2)], params)
    first = next(b for key, b in engine.model.rt._buffers.items() if "int4_expanded" in key)
    engine.generate([seeded_tokens(500, 515, 3)], params)
    for i in range(8):
        engine.cache.open(1000 + i)
        engine.cache.ensure(1000 + i, 500, 0)
        engine.forward([(1000 + i, seeded_tokens(450, 515, 4), 0, [])])
    engine.forward([(1000 + i, seeded_tokens(50, 515, 5), 450, []) for i in range(8)])      # 4000 keys
    assert next(b for key, b in engine.model.rt._buffers.items() if "int4_expanded" in key) is first
    assert first.dtype == torch.int32 and not any(b.dtype == torch.int32 and b.numel() >= 1024 for b in engine.model.rt._retired)
    assert first.numel() * 4 == engine.model.expanded_bytes(512, 8)
