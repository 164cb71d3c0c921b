"""Models served from a cache in 4 bits, and with norms on query and key heads, through the engine."""

import pytest
import torch

import plain_int4
import plain_llama as plain
from helpers import TINY, compare_logits, read_model_dir, seeded_tokens

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


def model_dir(tmp_models, name, dtype, qk_norm=False):
    from stride_b200 import config_from_dict, write_random_model
    cfg = dict(TINY[name], **({"qk_norm": True} if qk_norm else {}))
    return write_random_model(config_from_dict(cfg), seed=3, out_dir=str(tmp_models / f"int4-{name}-{dtype}-{qk_norm}"), stored_dtype=dtype, std=0.08,
                              vector_jitter=0.2)


def plain_forward(cfg, state, tokens, four, monkeypatch):
    """The plain model in float64 with head norms where the weights have them, keys and values through 4 bits where asked."""
    state = {k: v.double() for k, v in state.items()}

    def block(x, w, prefix, cfg, cos, sin, window=None):
        nq, nkv, hd = cfg["num_attention_heads"], cfg["num_key_value_heads"], cfg["head_dim"]
        q, k, v = (x @ w[f"{prefix}.self_attn.{n}_proj.weight"].T for n in "qkv")
        q, k, v = q.view(-1, nq, hd), k.view(-1, nkv, hd), v.view(-1, nkv, hd)
        if f"{prefix}.self_attn.q_norm.weight" in w:
            q, k = (plain.rms_norm(t, w[f"{prefix}.self_attn.{n}_norm.weight"], cfg["rms_norm_eps"]) for t, n in ((q, "q"), (k, "k")))
        q, k = plain.apply_rope(q, cos, sin), plain.apply_rope(k, cos, sin)
        if four:
            k, v = (plain_int4.unpack(n, plain_int4.pack(n, *plain_int4.quantise(t.float())), hd) for n, t in (("k", k), ("v", v)))
        return plain.causal_attention(q, k, v, hd ** -0.5, window).reshape(-1, nq * hd) @ w[f"{prefix}.self_attn.o_proj.weight"].T
    monkeypatch.setattr(plain, "attention_block", block)
    return plain.forward(cfg, state, tokens, torch.float64)


def logits_of(engine, tokens, cuts, key=1):
    """Logits of every token, the tokens brought in pieces of the lengths ``cuts``."""
    out, at = [], 0
    engine.cache.open(key)
    for n in cuts:
        assert engine.cache.ensure(key, at + n, 0)
        out.append(engine.forward([(key, tokens[at:at + n], at, range(n))]).cpu())
        at += n
    engine.cache.close(key)
    return torch.cat(out)


@pytest.mark.parametrize("name", ["A", "B", "C", "D"])
@pytest.mark.parametrize("qk_norm", [False, True])
def test_float32_has_the_same_bits_however_it_is_cut(gpu, tmp_models, monkeypatch, name, qk_norm):
    from stride_b200 import Engine
    folder = model_dir(tmp_models, name, "float32", qk_norm)
    cfg, state = read_model_dir(folder)
    tokens = seeded_tokens(83, cfg["vocab_size"], 5)
    for cache_dtype in (None, "int4"):
        engine = Engine(folder, dtype="float32", cache_dtype=cache_dtype, block_size=8, num_blocks=40, max_model_len=128, check_invariants=True)
        whole = logits_of(engine, tokens, [83])
        assert torch.equal(whole, logits_of(engine, tokens, [40] + [1] * 13 + [30])) and torch.equal(whole, logits_of(engine, tokens, [1, 81, 1]))
        want = plain_forward(cfg, state, tokens, cache_dtype == "int4", monkeypatch)
        if cache_dtype is None:
            ok, message = compare_logits(whole, want, "float32")
            assert ok, message
        else:
            # a number may fall to the other side of a border than in float64 and is then one step off: as far as one step of one entry
            # reaches, and a few such entries
            cosine = torch.nn.functional.cosine_similarity(whole.double(), want, dim=-1)
            assert float(cosine.min()) > 0.999, float(cosine.min())
            assert float(cosine.median()) > 0.999999


@pytest.mark.parametrize("qk_norm,cache_dtype", [(True, None), (False, "int4"), (True, "int4")])
def test_bfloat16_against_the_plain_model(gpu, tmp_models, monkeypatch, qk_norm, cache_dtype):
    from stride_b200 import Engine
    folder = model_dir(tmp_models, "D", "bfloat16", qk_norm)
    cfg, state = read_model_dir(folder)
    tokens = seeded_tokens(300, cfg["vocab_size"], 6)
    engine = Engine(folder, dtype="bfloat16", cache_dtype=cache_dtype, block_size=16, num_blocks=64, max_model_len=512, check_invariants=True)
    want = plain_forward(cfg, state, tokens, cache_dtype == "int4", monkeypatch)
    other = plain_forward(cfg, state, tokens, cache_dtype != "int4", monkeypatch)
    for cuts in ([300], [200] + [1] * 20 + [80], [17, 283]):
        got = logits_of(engine, tokens, cuts).double()
        cosine = torch.nn.functional.cosine_similarity(got, want, dim=-1)
        # bfloat16 noise moves entries over the borders of their numbers: the floor is the one that 4 bits themselves keep
        floor = 0.9995 if cache_dtype is None else float(torch.nn.functional.cosine_similarity(other, want, dim=-1).min())
        assert float(cosine.min()) > floor, (float(cosine.min()), floor)
    mean = lambda a, b: float(((a - b).norm(dim=-1) / b.norm(dim=-1)).mean())  # noqa: E731
    assert mean(got, want) < mean(got, other)           # it is the model with (or without) the 4 bits that it computes


def test_generation_graphs_prefixes_and_metrics(gpu, tmp_models):
    """Decode steps replayed from graphs, portions that fill the budget replayed too, a shared prefix: the tokens of an eager engine."""
    from stride_b200 import Engine, SamplingParams
    folder = model_dir(tmp_models, "D", "bfloat16", True)
    prompts = [seeded_tokens(150, 515, 1), seeded_tokens(9, 515, 2), seeded_tokens(64, 515, 3) + seeded_tokens(5, 515, 4), seeded_tokens(64, 515, 3) + [1, 2]]
    params = SamplingParams(temperature=0.0, max_tokens=12, ignore_eos=True)
    found = []
    for graphs in (True, False):
        engine = Engine(folder, dtype="bfloat16", cache_dtype="int4", block_size=16, num_blocks=64, max_model_len=512, max_batch_tokens=64, max_batch_seqs=4,
                        cuda_graphs=graphs, check_invariants=True)
        assert engine.device_cache.pages[0].dtype == torch.uint8
        found.append([o.tokens for o in engine.generate(prompts, params)])
        assert all(len(t) == 12 for t in found[-1])
        again = engine.generate(prompts[3:], params)[0]
        assert again.cached_prompt_tokens == 64 and (engine.metrics()["graph_replays"] > 0) == graphs
    assert found[0] == found[1]


@pytest.mark.parametrize("cache_dtype", [None, "int4"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_forked_request_goes_on_as_the_first_one_would(gpu, tmp_models, dtype, cache_dtype):
    from stride_b200 import Engine
    folder = model_dir(tmp_models, "D", dtype)
    engine = Engine(folder, dtype=dtype, cache_dtype=cache_dtype, block_size=16, num_blocks=32, max_model_len=256, check_invariants=True)
    tokens = seeded_tokens(60, 515, 8)
    cache = engine.cache
    cache.open(1)
    cache.ensure(1, 45, 0)
    engine.forward([(1, tokens[:45], 0, [])])
    engine.fork(1, 2, 41)                               # in the middle of a page, and before the parent's end
    cache.check_invariants()
    assert cache.table(2)[:2] == cache.table(1)[:2] and cache.table(2)[2] != cache.table(1)[2]
    cache.ensure(2, 50, 0)
    forked = engine.forward([(2, tokens[50:59], 41, range(9))]).clone()          # other tokens than the parent's
    cache.ensure(1, 60, 0)
    parent = engine.forward([(1, tokens[45:], 45, range(15))]).clone()
    for key, tail, got in ((3, tokens[41:], parent), (4, tokens[50:59], forked)):
        cache.open(key)
        cache.ensure(key, 41 + len(tail), 0)
        engine.forward([(key, tokens[:41], 0, [])])
        want = engine.forward([(key, tail, 41, range(len(tail)))])[-got.shape[0]:]
        if dtype == "float32":
            assert torch.equal(got, want)
        else:
            assert float(torch.nn.functional.cosine_similarity(got, want, dim=-1).min()) > 0.999
    for key in (1, 2, 3, 4):
        cache.close(key)
    cache.check_invariants()


def test_a_fork_copies_the_state_of_recurrent_layers(gpu, tmp_models):
    from stride_b200 import Engine, config_from_dict, preset, write_random_model
    folder = write_random_model(config_from_dict(preset("nidilix-tiny")), seed=2, out_dir=str(tmp_models / "fork-nidilix"), stored_dtype="float32", std=0.08,
                                vector_jitter=0.1)
    engine = Engine(folder, dtype="float32", block_size=8, num_blocks=32, max_batch_seqs=4, max_model_len=128, check_invariants=True)
    vocab = engine.model.vocab
    tokens = seeded_tokens(30, vocab, 8)
    engine.cache.open(1)
    engine.cache.ensure(1, 30, 0)
    engine.forward([(1, tokens[:21], 0, [])])
    engine.fork(1, 2, 21)
    engine.cache.ensure(2, 30, 0)
    first = engine.forward([(1, tokens[21:], 21, range(9))]).clone()
    assert torch.equal(first, engine.forward([(2, tokens[21:], 21, range(9))]))
    engine.cache.check_invariants()
