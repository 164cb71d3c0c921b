"""The cache in 4 bits, on the host: its layout in the planner and the groups, what refuses it, forks of requests, refused calls."""

import pytest
import torch

import plain_int4
from stride_b200.cache import CacheManager, plan_groups, runtime
from stride_b200.config import EngineConfig, PlanError, config_from_dict, plan_memory, preset


def model_for(cfg, dtype=torch.bfloat16, cache_dtype="int4"):
    from stride_b200.parts import DecoderModel, Runtime
    return DecoderModel(cfg.to_model_spec(), Runtime("meta", dtype, 1, 1, cache_dtype))


@pytest.mark.parametrize("hd", [16, 32, 48, 64, 80, 128, 256])
def test_rows_round_trip(hd):
    x = torch.randn(7, hd, generator=torch.Generator().manual_seed(hd)) * 3 + 1
    n, s, c = plain_int4.quantise(x)
    for which in "kv":
        rows = plain_int4.pack(which, n, s, c)
        assert rows.shape[-1] == 20 * plain_int4.groups(hd)
        of = torch.arange(hd) // 32
        assert torch.equal(plain_int4.unpack(which, rows, hd), c.double()[..., of] + s.double()[..., of] * (n - 8))
    # half a step; what 15 steps of s, rounded by 2^-8 at most, fall short of the range; what c is rounded by; and 32 bits
    limit = s[..., of] * (0.5 + 15 * 2.0 ** -8) + 2.0 ** -8 * c[..., of].abs() + 1e-6
    assert bool(((plain_int4.unpack("k", plain_int4.pack("k", n, s, c), hd) - x).abs() <= limit).all())


def test_pages_and_the_planner_count_five_bits_an_entry():
    cfg = config_from_dict(preset("llama3.1-8b"))
    model = model_for(cfg)
    group, = plan_groups(model.cache_requests())
    assert group.dtype == torch.uint8 and group.layout == (("k", 8, 80), ("v", 8, 80))
    assert group.bytes_per_page(16, 2) == 32 * 16 * 2 * 8 * 80
    wide, four = plan_memory(cfg), plan_memory(cfg, cache_dtype="int4")
    assert wide.kv_bytes_per_token == 32 * 2 * 8 * 128 * 2 and four.kv_bytes_per_token * 16 == wide.kv_bytes_per_token * 5
    assert four.num_blocks > 3 * wide.num_blocks


@pytest.mark.parametrize("name", ["nidilix-tiny", "netusun-tiny", "dopudra-tiny", "negotar-tiny"])
def test_layers_that_keep_something_else_refuse(name):
    with pytest.raises(ValueError, match="4 bits|int4"):
        model_for(config_from_dict(preset(name)))
    with pytest.raises(PlanError):
        plan_memory(config_from_dict(preset(name)), cache_dtype="int4")


def test_what_takes_it():
    for name in ("tiny-a", "tiny-b", "tiny-d"):
        assert all(r.dtype == torch.uint8 for r, _s in model_for(config_from_dict(preset(name))).cache_requests())
    with pytest.raises(ValueError, match="cache_dtype"):
        EngineConfig(cache_dtype="int8")
    from stride_b200.parts import Runtime
    with pytest.raises(ValueError, match="int4"):
        Runtime("meta", torch.float32, 1, 1, "fp4")


def test_head_norms_in_a_llama_config():
    raw = dict(preset("tiny-d"), qk_norm=True)
    cfg = config_from_dict(raw)
    assert cfg.qk_norm and config_from_dict(cfg.to_dict()) == cfg and not config_from_dict(preset("tiny-d")).qk_norm
    declared = model_for(cfg, cache_dtype=None).declare()
    assert declared["model.layers.0.self_attn.q_norm.weight"].shape == (128,) == declared["model.layers.1.self_attn.k_norm.weight"].shape
    from stride_b200.config.llama import LlamaConfig
    assert LlamaConfig.complete_from_checkpoint({}, {"model.layers.0.self_attn.q_norm.weight"})["qk_norm"]
    assert not LlamaConfig.complete_from_checkpoint({}, {"model.layers.0.self_attn.q_proj.weight"})["qk_norm"]


# ------------------------------------------------------------------------------------------------------------------- forks
def test_a_fork_shares_whole_pages_and_copies_the_last():
    cache = CacheManager(4, [(12, 0)], 3, False)
    cache.open(1, "tenant")
    assert cache.ensure(1, 11, 0)
    copies, (a, b) = cache.fork(1, 2, 11)
    table, child = cache.table(1), cache.table(2)
    assert child[:2] == table[:2] and child[2] != table[2] and copies == [(0, table[2], child[2])]
    assert (a, b) == (cache.state_slot(1), cache.state_slot(2)) and a != b
    cache.check_invariants()
    assert cache.stats()["live"] == 4
    copies, _ = cache.fork(2, 3, 8)                 # whole pages alone: nothing to copy; of a fork, too
    assert copies == [] and cache.table(3) == table[:2]
    cache.close(1)
    cache.check_invariants()
    assert cache.ensure(3, 9, 0) and cache.table(3)[2] not in child
    cache.close(2), cache.close(3)
    cache.check_invariants()
    assert cache.stats()["live"] == 0


def test_a_fork_of_nothing_and_of_part_of_a_request():
    cache = CacheManager(4, [(6, 0)], 4, False)
    cache.open(1)
    cache.ensure(1, 10, 0)
    assert cache.fork(1, 2, 0)[0] == [] and cache.table(2) == []
    copies, _ = cache.fork(1, 3, 5)
    assert len(cache.table(3)) == 2 and copies == [(0, cache.table(1)[1], cache.table(3)[1])]
    cache.check_invariants()


def test_refused_forks_change_nothing():
    cache = CacheManager(4, [(3, 0)], 2, False)
    cache.open(1)
    cache.ensure(1, 10, 0)
    with pytest.raises(ValueError, match="fewer"):
        cache.fork(1, 2, 13)
    with pytest.raises(ValueError, match="holds no cache"):
        cache.fork(5, 2, 1)
    with pytest.raises(ValueError, match="already"):
        cache.fork(1, 1, 4)
    with pytest.raises(runtime().OutOfPages):
        cache.fork(1, 2, 10)                        # no page is left for the copy
    assert cache.num_requests == 1 and cache.free_slots == 1
    cache.check_invariants()
    cache.fork(1, 2, 8)
    with pytest.raises(runtime().OutOfPages):
        cache.fork(1, 3, 8)                         # no state slot is left
    cache.check_invariants()
    assert cache.num_requests == 2


def test_forks_under_a_window():
    cache = CacheManager(4, [(20, 0), (20, 6)], 4, False)
    cache.open(1)
    cache.ensure(1, 22, 0)
    cache.trim(1, 22)
    assert cache.table(1, 1)[:4] == [-1] * 4
    copies, _ = cache.fork(1, 2, 22)
    assert [c[0] for c in copies] == [0, 1] and cache.table(2, 1)[:4] == [-1] * 4 and cache.table(2, 1)[4] == cache.table(1, 1)[4]
    with pytest.raises(ValueError, match="given back"):
        cache.fork(1, 3, 15)                        # its next query reads keys 10 to 15, whose page is gone
    cache.check_invariants()
    cache.ensure(2, 30, 0)
    cache.trim(2, 30)
    cache.check_invariants()
    cache.close(1)
    cache.check_invariants()


def test_a_fork_of_a_shared_prefix():
    cache = CacheManager(4, [(8, 0)], 3, True)
    tokens = list(range(8))
    cache.open(1)
    cache.ensure(1, 8, 0)
    cache.publish(1, tokens, 8)
    cache.fork(1, 2, 8)
    cache.close(1)
    cache.check_invariants()
    assert cache.stats()["live"] == 2
    cache.close(2)
    assert cache.stats()["cached"] == 2
    cache.check_invariants()


# --------------------------------------------------------------------------------------------------------------- refusals
def rows(tokens=3, nq=4, nkv=2, hd=64, page=8, pages=5, dtype=torch.bfloat16, bits4=True):
    made = dict(qkv=torch.zeros(tokens, (nq + 2 * nkv) * hd, dtype=dtype), bias=None, q_norm=None, k_norm=None, eps=1e-5,
                positions=torch.zeros(tokens, dtype=torch.int32), slot_mapping=torch.zeros(tokens, dtype=torch.int32),
                cos=torch.zeros(16, hd // 2), sin=torch.zeros(16, hd // 2), nq=nq, nkv=nkv, hd=hd, page_size=page)
    width, kind = (20 * plain_int4.groups(hd), torch.uint8) if bits4 else (hd, dtype)
    made.update(k_pages=torch.zeros(pages, nkv, page, width, dtype=kind), v_pages=torch.zeros(pages, nkv, page, width, dtype=kind))
    return made


@pytest.mark.parametrize("bits4", [False, True])
@pytest.mark.parametrize("change", [
    dict(nq=3), dict(nkv=1), dict(hd=0), dict(page_size=16), dict(q_norm=torch.ones(64)), dict(positions=torch.zeros(2, dtype=torch.int32)),
    dict(slot_mapping=torch.zeros(2, dtype=torch.int32)), dict(cos=torch.zeros(16, 31)), dict(k_pages=torch.zeros(5, 2, 8, 63, dtype=torch.uint8)),
    dict(v_pages=torch.zeros(4, 2, 8, 40, dtype=torch.uint8)), 
    dict(qkv=torch.zeros(3, 512, dtype=torch.float16)), dict()])
def test_refused_writes(bits4, change):
    from stride_b200.csrc import ops
    write = ops.rope_kv_write_int4 if bits4 else ops.qk_norm_rope_write
    with pytest.raises(ops.KernelError):            # the last case: nothing is wrong but that the tensors live on the host
        write(**{**rows(bits4=bits4), **change})


def attention_call(kind, tokens=3, nq=4, nkv=2, hd=64, page=8, pages=5):
    width = 20 * plain_int4.groups(hd)
    made = dict(q=torch.zeros(tokens, nq * hd, dtype=torch.bfloat16), q_stride=nq * hd, out=torch.zeros(tokens, nq * hd, dtype=torch.bfloat16),
                k_pages=torch.zeros(pages, nkv, page, width, dtype=torch.uint8), v_pages=torch.zeros(pages, nkv, page, width, dtype=torch.uint8),
                block_table=torch.zeros(2, 3, dtype=torch.int32), nq=nq, nkv=nkv, hd=hd, page_size=page, scale=0.125, window=0)
    index = torch.zeros(tokens, dtype=torch.int32)
    if kind == "portion":
        made.update(q_start=index, q_len=index, ctx_len=index, scratch=torch.zeros(1 << 20, dtype=torch.int32), num_seqs=2, keys=20)
    else:
        made.update(seq_of_token=index, positions=index)
        if kind == "decode":
            made.update(scratch=torch.zeros(1 << 20), max_context=24)
    return made


@pytest.mark.parametrize("kind", ["exact", "decode", "portion"])
@pytest.mark.parametrize("change", [
    dict(nq=3), dict(nkv=3), dict(hd=32), dict(page_size=16), dict(q_stride=200), dict(q=torch.zeros(2, 256, dtype=torch.bfloat16)),
    dict(out=torch.zeros(3, 128, dtype=torch.bfloat16)), dict(out=torch.zeros(3, 256)), dict(window=-1), dict(softcap=-1.0),
    dict(block_table=torch.zeros(6, dtype=torch.int32)), dict(k_pages=torch.zeros(0, 2, 8, 40, dtype=torch.uint8)), dict()])
def test_refused_attention(kind, change):
    from stride_b200.csrc import ops
    call = {"exact": ops.paged_attention_int4, "decode": ops.paged_attention_decode_int4, "portion": ops.paged_attention_prefill_int4}[kind]
    with pytest.raises(ops.KernelError):
        call(**{**attention_call(kind), **change})


def test_refused_copies():
    from stride_b200.csrc import ops
    pool = torch.zeros(2, 6, 3)
    for src, dst in (([1], [2, 3]), ([0, 1], [2, 2]), ([0, 2], [2, 3]), ([0], [0]), ([6], [1]), ([1], [-1])):
        with pytest.raises(ops.KernelError, match="copy_pages"):
            ops.copy_pages([pool], src, dst)
    with pytest.raises(ops.KernelError, match="pool is"):
        ops.copy_pages([pool[0]], [0], [1])
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.copy_pages([pool], [0], [1])


def test_records_are_as_long_as_the_launchers_read():
    """sizeof of the C records, which the sources assert."""
    from stride_b200.csrc import ops
    assert {n: r.size for n, r in ops._RECORDS.items()} == {"stride_head_write": 160, "stride_int4_read": 80, "stride_int4_prefill": 176,
                                                            "stride_attention_int4_exact": 152, "stride_decode_int4": 160}


@pytest.mark.parametrize("number", [2 ** 31, -2 ** 31 - 1])
def test_numbers_that_no_launch_holds_are_refused(number):
    from stride_b200.csrc import ops
    with pytest.raises(ops.KernelError, match="read_int4: a number does not fit"):
        ops._launch("stride_int4_read", "read_int4", 0, 0, 0, 0, 0, 0, 0, number, 1, 64, 16, 1, 0)


# ------------------------------------------------------------------------------------- what portions expand out of the cache
def mixer_of(name="llama3.1-8b"):
    return [p for p in model_for(config_from_dict(preset(name))).layers[0].parts() if hasattr(p, "expanded_keys")][0]


def test_what_portions_expand_is_bounded():
    mixer = mixer_of()
    of_key = 2 * 8 * 128 * 2
    for longest, requests in ((8192, 256), (131072, 256), (131072, 1), (300, 4), (65536, 2), (1, 1)):
        keys = mixer.expanded_keys(longest, requests)
        assert longest <= keys <= longest * requests            # one request always fits, and no more than a step can hold
        assert keys * of_key <= max(mixer.MAX_EXPANDED_BYTES, longest * of_key)
        # the buffer: pages in quarters of an octave, a table and a record a page
        assert mixer.expanded_bytes(longest, requests) <= 1.25 * (keys + 64 * requests) * of_key * 1.02 + 32 * 64 * of_key
    assert model_for(config_from_dict(preset("tiny-a")), torch.float32).expanded_bytes(8192, 16) == 0


def test_requests_are_expanded_in_groups_that_fit():
    from types import SimpleNamespace
    mixer = mixer_of()

    def groups(held, room):
        items = [(i, 0, 5, n - 5, 0) for i, n in enumerate(held)] + [(99, 0, 1, 700, 0)] * 3       # and single tokens behind them
        return mixer._portion_groups(SimpleNamespace(portion_keys=sum(held), decode_tail_seq=len(held), host_items=items), room)
    assert groups([50, 60, 70], 180) == [(0, 3, 180)]
    assert groups([50, 60, 70], 179) == [(0, 2, 110), (2, 3, 70)]
    assert groups([100, 100, 100], 100) == [(0, 1, 100), (1, 2, 100), (2, 3, 100)]
    for room in range(40, 200):
        found = groups([40, 7, 33, 39, 12, 12, 40], room)
        assert [g[0] for g in found][1:] == [g[1] for g in found][:-1] and found[0][0] == 0 and found[-1][1] == 7
        assert all(g[2] <= max(room, 40) for g in found) and sum(g[2] for g in found) == 183


def test_the_planner_sets_aside_what_portions_expand():
    cfg = config_from_dict(preset("llama3.1-8b"))
    four = plan_memory(cfg, cache_dtype="int4", max_requests=64)
    wide = plan_memory(cfg, max_requests=64)
    expanded = model_for(cfg).expanded_bytes(cfg.max_position_embeddings, 64)
    assert expanded > 0 and four.activation_reserve_bytes - wide.activation_reserve_bytes == expanded == wide.kv_bytes - four.kv_bytes
