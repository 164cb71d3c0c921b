"""Attention over a cache held in 4 bits where sizes differ: groups of a row, rows of a cache, queries."""

import pytest
import torch

import plain_int4 as plain

pytestmark = pytest.mark.gpu
BF16, F64 = torch.bfloat16, torch.float64
HALF_STEP = 2.0 ** -8                   # of a bfloat16 result, relative


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from stride_b200.csrc import ops
    ops.check_kernel_status()
    yield ops
    ops.check_kernel_status()


def cache_of(keys, values, page):
    """Pages of one request's keys and values [n, nkv, hd], its table, and what the pages stand for (float64)."""
    n, nkv, hd = keys.shape
    count = -(-n // page)
    pages, stored = [], []
    for which, x in (("k", keys), ("v", values)):
        rows = plain.pack(which, *plain.quantise(x.float()))
        stored.append(plain.unpack(which, rows, hd))
        full = torch.full((count * page, nkv, rows.shape[-1]), 255, dtype=torch.uint8)
        full[:n] = rows
        pages.append(full.view(count, page, nkv, -1).transpose(1, 2).contiguous().cuda())
    return pages, torch.arange(count, dtype=torch.int32, device="cuda")[None], stored


def decode(ops, q, pages, table, n, nq, nkv, hd, page, scale=None):
    out = torch.empty(q.shape[0], nq * hd, dtype=BF16, device="cuda")
    at = torch.full((q.shape[0],), n - 1, dtype=torch.int32, device="cuda")
    scratch = torch.zeros(ops.decode_int4_scratch_floats(q.shape[0], nq, nkv, hd, n), device="cuda")
    ops.paged_attention_decode_int4(q.cuda(), nq * hd, out, *pages, table, torch.zeros_like(at), at, scratch, nq, nkv, hd, page,
                                    hd ** -0.5 if scale is None else scale, 0, n)
    return out.view(-1, nq, hd).double().cpu()


def group_errors(got, want):
    """Of every group of 32 of every head: the error's norm over the result's."""
    return ((got - want).unflatten(-1, (-1, 32)).norm(dim=-1) / want.unflatten(-1, (-1, 32)).norm(dim=-1)).amax()


def positive(g, *shape):
    """Values that do not cancel: a sum of them with weights is as large as they are."""
    return 0.5 + torch.rand(*shape, generator=g)


SHAPES = [(8, 2, 128, 16), (16, 1, 64, 16), (3, 1, 128, 5), (4, 1, 64, 32)]


@pytest.mark.parametrize("large", [0, 1])
@pytest.mark.parametrize("log_ratio", [4, 9, 12, 16, 20, 24, 40])
@pytest.mark.parametrize("nq,nkv,hd,page", SHAPES)
def test_decode_of_values_whose_groups_differ_in_size(ops, nq, nkv, hd, page, log_ratio, large):
    n, g = 500, torch.Generator().manual_seed(hd + log_ratio)
    values = positive(g, n, nkv, hd)
    values[..., 32 * large:32 * large + 32] *= 2.0 ** log_ratio
    pages, table, (k, v) = cache_of(torch.randn(n, nkv, hd, generator=g), values, page)
    q = torch.randn(2, nq * hd, generator=g).to(BF16)
    want, _l, _v = plain.attention(q.view(2, nq, hd), [k], [v], torch.tensor([n - 1] * 2), torch.tensor([0, 0]), hd ** -0.5)
    # the result's rounding; a weight's, 2^-11 of its product with a scale, and what it drops below 2^-24 of the largest such product, times
    # the numbers up to 15, where a row's groups are so near in size that 16-bit floating point takes them (a factor of 64)
    floor = 15 * n * 2.0 ** (log_ratio - 25) if log_ratio <= 6 else 0.0
    assert group_errors(decode(ops, q, pages, table, n, nq, nkv, hd, page), want) <= HALF_STEP + 2.0 ** -10 + floor
    ops.check_kernel_status()


@pytest.mark.parametrize("weight", [0.0, 3.0])
@pytest.mark.parametrize("at", [0, 3, 130, 299])
@pytest.mark.parametrize("nq,nkv,hd,page", SHAPES)
def test_decode_beside_one_token_with_a_group_that_stands_out(ops, nq, nkv, hd, page, at, weight):
    """One value's first group is 2^20 times the others'; what the rest of the head holds comes from all tokens."""
    n, g = 300, torch.Generator().manual_seed(hd + at)
    keys, values = 0.3 * torch.randn(n, nkv, hd, generator=g), positive(g, n, nkv, hd)
    values[at, :, :32] *= 2.0 ** 20
    q = torch.randn(1, nq * hd, generator=g).to(BF16)
    keys[at] += weight * q.float().view(nkv, nq // nkv, hd).mean(1) / hd ** 0.5
    pages, table, (k, v) = cache_of(keys, values, page)
    want, _l, _v = plain.attention(q.view(1, nq, hd), [k], [v], torch.tensor([n - 1]), torch.tensor([0]), hd ** -0.5)
    assert group_errors(decode(ops, q, pages, table, n, nq, nkv, hd, page), want) <= HALF_STEP + 2.0 ** -10
    ops.check_kernel_status()


def portion(ops, q, pages, table, n, nq, nkv, hd, page, scale=None, **rules):
    """The last q.shape[0] tokens of a request of n keys."""
    p = q.shape[0]
    ints = lambda x: torch.tensor([x], dtype=torch.int32, device="cuda")  # noqa: E731
    out = torch.full((p, nq * hd), 9.0, dtype=BF16, device="cuda")
    scratch = torch.full((ops.prefill_int4_scratch_ints(1, n, nkv, hd),), -1, dtype=torch.int32, device="cuda")
    ops.paged_attention_prefill_int4(q.cuda(), nq * hd, out, *pages, table, ints(0), ints(p), ints(n), scratch, 1, n, nq, nkv, hd, page,
                                     hd ** -0.5 if scale is None else scale, 0, **rules)
    return out.view(p, nq, hd).double().cpu()


def rows_of(n, p):
    return torch.arange(n - p, n), torch.zeros(p, dtype=torch.int32)


@pytest.mark.parametrize("large", [0, 1])
@pytest.mark.parametrize("log_ratio", [12, 20, 24])
@pytest.mark.parametrize("nq,nkv,hd,page", SHAPES)
def test_portions_of_values_whose_groups_differ_in_size(ops, nq, nkv, hd, page, log_ratio, large):
    n, p, g = 300, 5, torch.Generator().manual_seed(hd + log_ratio)
    values = positive(g, n, nkv, hd)
    values[..., 32 * large:32 * large + 32] *= 2.0 ** log_ratio
    pages, table, (k, v) = cache_of(0.3 * torch.randn(n, nkv, hd, generator=g), values, page)
    q = torch.randn(p, nq * hd, generator=g).to(BF16)
    want, largest, _v = plain.attention(q.view(p, nq, hd), [k], [v], *rows_of(n, p), hd ** -0.5)
    # the result's rounding, a weight's and a value's of 2^-11, a key's of 2^-11 in every product of a score; of the largest value 2^-40
    limit = HALF_STEP + 2 * 2.0 ** -11 + 2 * 2.0 ** -11 * largest + 2.0 ** (log_ratio - 40)
    assert group_errors(portion(ops, q, pages, table, n, nq, nkv, hd, page), want) <= limit
    ops.check_kernel_status()


SIZES = [(1e-6, 1.0, 1.0), (1e-8, 1.0, 1.0), (1e-30, 1e-3, 1e3), (1e5, 1.0, 1.0), (1e15, 1e6, 1e-6), (1.0, 1e-20, 1e20), (3.0, 1e15, 1e-15), (1.0, 1.0, 1e-30),
         (1e-33, 1e-33, 1e33)]


@pytest.mark.parametrize("rules", [dict(), dict(softcap=4.0, precise_cap=True), dict(slopes=True), dict(softcap=4.0, precise_cap=True, slopes=True, sinks=True)], ids=str)
@pytest.mark.parametrize("of_values,of_keys,of_queries", SIZES)
@pytest.mark.parametrize("nq,nkv,hd,page", SHAPES[:2])
def test_portions_of_keys_values_and_queries_of_any_size(ops, nq, nkv, hd, page, of_values, of_keys, of_queries, rules):
    """Rows of queries of very different sizes beside one another, tokens of different sizes in one head, scores of the usual size."""
    n, p, g = 200, 130, torch.Generator().manual_seed(7)
    keys = torch.randn(n, nkv, hd, generator=g, dtype=F64) * of_keys
    values = positive(g, n, nkv, hd).double() * of_values * torch.logspace(-2, 0, n, dtype=F64)[:, None, None]
    pages, table, (k, v) = cache_of(keys, values, page)
    q = torch.randn(p, nq * hd, generator=g, dtype=F64) * of_queries * 0.3
    q[::2] *= 2.0 ** -20                                    # rows whose scores are all alike
    q = q.to(BF16)
    sinks = torch.randn(nq, generator=g) if rules.get("sinks") else None
    slopes = torch.full((nq,), 0.01) if rules.get("slopes") else None
    want, largest, _v = plain.attention(q.view(p, nq, hd), [k], [v], *rows_of(n, p), hd ** -0.5, softcap=rules.get("softcap", 0.0), sinks=sinks, slopes=slopes)
    given = dict(rules, sinks=None if sinks is None else sinks.cuda(), slopes=None if slopes is None else slopes.cuda())
    got = portion(ops, q, pages, table, n, nq, nkv, hd, page, **given)
    # as above; the penalty of up to 200 positions of 0.01 in 32 bits counts nothing, the capped score's tanh a few 2^-24 of the cap
    assert group_errors(got, want) <= HALF_STEP + 2 * 2.0 ** -11 + 2 * 2.0 ** -11 * largest
    ops.check_kernel_status()


def test_a_portion_reads_entries_beyond_the_16_bit_range_as_they_are(ops):
    """The first token sees itself alone: its result is its value. (The largest number of 16-bit floating point is 65504.)"""
    n, nq, nkv, hd, page, g = 40, 4, 1, 64, 16, torch.Generator().manual_seed(5)
    values = torch.randn(n, nkv, hd, generator=g) * 3e4
    values[0, 0, :4] = torch.tensor([84760.0, -1e5, 1e6, 7e4])
    pages, table, (k, v) = cache_of(torch.randn(n, nkv, hd, generator=g), values, page)
    got = portion(ops, torch.randn(n, nq * hd, generator=g).to(BF16), pages, table, n, nq, nkv, hd, page)
    assert bool(((got[0] - v[0]).abs() <= (HALF_STEP + 2.0 ** -10) * v[0].abs()).all())
    ops.check_kernel_status()


# ------------------------------------------------------------------------------------------------------- keys without a page
def without(q, k, v, pos, keep, scale):
    """Attention of every row to those of its keys that ``keep`` names; zeros where there are none."""
    p, nq, hd = q.shape
    nkv = k.shape[1]
    out = torch.zeros(p, nq, hd, dtype=F64)
    for t in range(p):
        on = keep & (torch.arange(k.shape[0]) <= int(pos[t]))
        for h in range(nq if bool(on.any()) else 0):
            kv = h // (nq // nkv)
            out[t, h] = torch.softmax(k[on, kv] @ q[t, h].double() * scale, 0) @ v[on, kv]
    return out


GONE = [[2], [0, 1], [4, 9], "last", "all"]


def with_holes(page, gone, entry):
    n, nq, nkv, hd, g = 190, 4, 2, 64, torch.Generator().manual_seed(page)
    pages, table, (k, v) = cache_of(torch.randn(n, nkv, hd, generator=g), positive(g, n, nkv, hd), page)
    at = [table.shape[1] - 1] if gone == "last" else list(range(table.shape[1])) if gone == "all" else sorted({i % table.shape[1] for i in gone})
    keep = torch.ones(n, dtype=torch.bool)
    for i in at:
        table[0, i] = entry
        keep[i * page:(i + 1) * page] = False
    q = torch.randn(6, nq * hd, generator=g).to(BF16)
    want = without(q.view(6, nq, hd), k, v, torch.arange(n - 6, n), keep, hd ** -0.5)
    return n, nq, nkv, hd, pages, table, q, want


def close(got, want):
    # values between 0.5 and 1.5: the result's rounding, and some 2^-9 for weights and scores of 11 bits
    assert bool(((got - want).abs() <= HALF_STEP * want.abs() + 2.0 ** -8 * (want != 0)).all()), float((got - want).abs().max())


@pytest.mark.parametrize("entry", [-1, 9999])
@pytest.mark.parametrize("gone", GONE, ids=str)
@pytest.mark.parametrize("page", [1, 5, 8, 16, 48, 64])
def test_decode_leaves_out_keys_without_a_page(ops, page, gone, entry):
    n, nq, nkv, hd, pages, table, q, want = with_holes(page, gone, entry)
    out = torch.full((6, nq * hd), 9.0, dtype=BF16, device="cuda")
    at, seq = torch.arange(n - 6, n, dtype=torch.int32, device="cuda"), torch.zeros(6, dtype=torch.int32, device="cuda")
    scratch = torch.zeros(ops.decode_int4_scratch_floats(6, nq, nkv, hd, n), device="cuda")
    ops.paged_attention_decode_int4(q.cuda(), nq * hd, out, *pages, table, seq, at, scratch, nq, nkv, hd, page, hd ** -0.5, 0, n)
    with pytest.raises(ops.KernelError, match="names no page"):
        ops.check_kernel_status()
    close(out.view(6, nq, hd).double().cpu(), want)


@pytest.mark.parametrize("entry", [-1, 9999])
@pytest.mark.parametrize("gone", GONE, ids=str)
@pytest.mark.parametrize("page", [1, 5, 8, 16, 48, 64])
def test_portions_leave_out_keys_without_a_page(ops, page, gone, entry):
    n, nq, nkv, hd, pages, table, q, want = with_holes(page, gone, entry)
    got = portion(ops, q, pages, table, n, nq, nkv, hd, page)
    with pytest.raises(ops.KernelError, match="names no page"):
        ops.check_kernel_status()
    close(got, want)


@pytest.mark.parametrize("gone", GONE, ids=str)
@pytest.mark.parametrize("page", [5, 16])
def test_the_exact_kernel_leaves_out_keys_without_a_page(ops, page, gone):
    n, nq, nkv, hd, pages, table, q, want = with_holes(page, gone, -1)
    out = torch.full((6, nq * hd), 9.0, dtype=BF16, device="cuda")
    at, seq = torch.arange(n - 6, n, dtype=torch.int32, device="cuda"), torch.zeros(6, dtype=torch.int32, device="cuda")
    ops.paged_attention_int4(q.cuda(), nq * hd, out, *pages, table, seq, at, nq, nkv, hd, page, hd ** -0.5)
    with pytest.raises(ops.KernelError, match="names no page"):
        ops.check_kernel_status()
    close(out.view(6, nq, hd).double().cpu(), want)


@pytest.mark.parametrize("held", [2 ** 31 - 1, 2 ** 30, 64 * 32 + 1])
def test_a_portion_of_a_request_beyond_the_room_for_its_keys_is_reported_and_not_run(ops, held):
    n, nq, nkv, hd, pages, table, q, _want = with_holes(16, "last", -1)
    ints = lambda x: torch.tensor([x], dtype=torch.int32, device="cuda")  # noqa: E731
    out = torch.full((6, nq * hd), 9.0, dtype=BF16, device="cuda")
    scratch = torch.zeros(ops.prefill_int4_scratch_ints(1, n, nkv, hd), dtype=torch.int32, device="cuda")       # 32 pages of 64
    ops.paged_attention_prefill_int4(q.cuda(), nq * hd, out, *pages, table, ints(0), ints(6), ints(held), scratch, 1, n, nq, nkv, hd, 16, 0.125, 0)
    with pytest.raises(ops.KernelError, match="more keys|names no page"):       # (both are so; the first report stays)
        ops.check_kernel_status()
    assert bool((out == 9.0).all())


# --------------------------------------------------------------------------------------------------- where pages may begin
@pytest.mark.parametrize("nq,nkv,hd,page,pages_of", [(4, 1, 64, 5, 41), (6, 3, 64, 1, 201), (4, 1, 64, 16, 13), (2, 1, 128, 5, 41), (2, 2, 128, 16, 13)])
def test_every_layer_of_an_odd_pool_is_read(ops, nq, nkv, hd, page, pages_of):
    """A layer's pages begin behind the layer before: heads of 64 have rows of 40 bytes, so that is any multiple of 8. Pages of 16 are moved to one, too."""
    n, g = 200, torch.Generator().manual_seed(page)
    pages, table, (k, v) = cache_of(torch.randn(n, nkv, hd, generator=g), positive(g, n, nkv, hd), page)
    shift = 8 if page == 16 and hd == 64 else 0
    moved = []
    for t in pages:
        pool = torch.zeros(2 * pages_of * t[0].numel() + shift, dtype=torch.uint8, device="cuda")[shift:].view(2, pages_of, *t.shape[1:])
        pool[1, :t.shape[0]] = t
        moved.append(pool[1])
    if hd == 64:
        assert moved[0].data_ptr() % 16 == 8
    q = torch.randn(3, nq * hd, generator=g).to(BF16)
    want, largest, _v = plain.attention(q.view(3, nq, hd), [k], [v], torch.tensor([n - 1] * 3), torch.zeros(3, dtype=torch.int32), hd ** -0.5)
    got = decode(ops, q, moved, table, n, nq, nkv, hd, page)
    assert group_errors(got, want) <= HALF_STEP + 2.0 ** -10
    assert torch.equal(got, decode(ops, q, pages, table, n, nq, nkv, hd, page)) or page == 16       # (of the same copies: the same bits)
    q = q.repeat(4, 1)
    want, largest, _v = plain.attention(q.view(12, nq, hd), [k], [v], *rows_of(n, 12), hd ** -0.5)
    assert group_errors(portion(ops, q, moved, table, n, nq, nkv, hd, page), want) <= HALF_STEP + 2 * 2.0 ** -11 + 2 * 2.0 ** -11 * largest
    exact = torch.empty(12, nq * hd, dtype=BF16, device="cuda")
    at, seq = (x.int().cuda() for x in rows_of(n, 12))
    ops.paged_attention_int4(q.cuda(), nq * hd, exact, *moved, table, seq, at, nq, nkv, hd, page, hd ** -0.5)
    assert group_errors(exact.view(12, nq, hd).double().cpu(), want) <= HALF_STEP + 2.0 ** -12
    ops.check_kernel_status()


def test_decode_over_pages_at_odd_addresses_is_refused(ops):
    n, nq, nkv, hd, page, g = 60, 4, 1, 64, 5, torch.Generator().manual_seed(1)
    pages, table, _stored = cache_of(torch.randn(n, nkv, hd, generator=g), positive(g, n, nkv, hd), page)
    moved = []
    for t in pages:
        pool = torch.zeros(t.numel() + 4, dtype=torch.uint8, device="cuda")[4:].view(t.shape)
        moved.append(pool)
    with pytest.raises(ops.KernelError):
        decode(ops, torch.zeros(1, nq * hd, dtype=BF16), moved, table, n, nq, nkv, hd, page)


# ------------------------------------------------------------------------------------------------------------ how near to 64 bits
# A bfloat16 result has 8 bits: a rounding is off by up to 2^-8 of the power of two below the value, evenly, 2^-8 / sqrt(3) of it in the mean square,
# and a value's mean square is 2.16 of that power's where mantissas are spread as logarithms are: 1.53e-3 in the norm, up to 1.7e-3 for
# sums of random values. What 11 bits of weights, keys and values (2^-11 / sqrt(3) / 1.47 = 1.9e-4 each) and 16 of a centre's weights add
# stays below 8e-4 together, and sqrt(1.7^2 + 0.8^2) = 1.9. Keys, values or a centre's weights in 8 bits come to 2.4e-3 and more.
NEAR = 2.1e-3


def norm_error(got, want):
    return float((got - want).norm() / want.norm())


@pytest.mark.parametrize("nq,nkv,hd,page", [(32, 8, 128, 16), (16, 4, 64, 16), (16, 1, 128, 8)])
def test_decode_is_as_near_as_its_result_can_be(ops, nq, nkv, hd, page):
    n, g = 1500, torch.Generator().manual_seed(hd)
    pages, table, (k, v) = cache_of(torch.randn(n, nkv, hd, generator=g), torch.randn(n, nkv, hd, generator=g), page)
    q = torch.randn(4, nq * hd, generator=g).to(BF16)
    want, _l, _v = plain.attention(q.view(4, nq, hd), [k], [v], torch.tensor([n - 1] * 4), torch.zeros(4, dtype=torch.int32), hd ** -0.5)
    assert norm_error(decode(ops, q, pages, table, n, nq, nkv, hd, page), want) < NEAR


@pytest.mark.parametrize("nq,nkv,hd,page", [(8, 2, 128, 16), (12, 4, 64, 16), (3, 1, 128, 8)])
def test_portions_are_as_near_as_their_result_can_be(ops, nq, nkv, hd, page):
    n, p, g = 700, 60, torch.Generator().manual_seed(hd)
    pages, table, (k, v) = cache_of(torch.randn(n, nkv, hd, generator=g), torch.randn(n, nkv, hd, generator=g), page)
    q = torch.randn(p, nq * hd, generator=g).to(BF16)
    want, _l, _v = plain.attention(q.view(p, nq, hd), [k], [v], *rows_of(n, p), hd ** -0.5)
    assert norm_error(portion(ops, q, pages, table, n, nq, nkv, hd, page), want) < NEAR


def test_calls_on_the_same_inputs_have_the_same_bits(ops):
    """Parts of a request are merged in the order of its keys, whichever CTA comes last."""
    nq, nkv, hd, page, g = 32, 8, 128, 16, torch.Generator().manual_seed(3)
    lengths = [3000, 1, 700, 1200]
    kept = [cache_of(torch.randn(n, nkv, hd, generator=g), torch.randn(n, nkv, hd, generator=g), page)[0] for n in lengths]
    pages = [torch.cat([made[w] for made in kept]) for w in (0, 1)]
    table = torch.full((4, -(-3000 // page)), -1, dtype=torch.int32)
    first = 0
    for r, n in enumerate(lengths):
        table[r, :-(-n // page)] = torch.arange(first, first - (-n // page))
        first -= -n // page
    table = table.cuda()
    q = torch.randn(4, nq * hd, generator=g).to(BF16).cuda()
    at, seq = torch.tensor([n - 1 for n in lengths], dtype=torch.int32, device="cuda"), torch.arange(4, dtype=torch.int32, device="cuda")
    scratch = torch.zeros(ops.decode_int4_scratch_floats(4, nq, nkv, hd, 3000), device="cuda")
    outs = []
    for _ in range(20):
        outs.append(torch.empty(4, nq * hd, dtype=BF16, device="cuda"))
        ops.paged_attention_decode_int4(q, nq * hd, outs[-1], *pages, table, seq, at, scratch, nq, nkv, hd, page, hd ** -0.5, 0, 3000)
    assert all(torch.equal(outs[0], o) for o in outs)
    ops.check_kernel_status()


# sizes of the values of the pages, one after another over and over
MIXES = [(0.0, 1e15), (1e15, 0.0), (1e-25, 1e10), (1e18, 1e-25, 0.0, 1.0), (0.0, 1e-28), (1e-28, 0.0, 1e-24)]


@pytest.mark.parametrize("run", [16, 64, 128])
@pytest.mark.parametrize("mix", MIXES, ids=str)
@pytest.mark.parametrize("call", ["decode", "portion"])
def test_pages_of_values_of_very_different_sizes(ops, call, mix, run):
    """The sum of the weights is that of all tokens, whatever their values' size."""
    n, nq, nkv, hd, page, g = 520, 4, 2, 64, 16, torch.Generator().manual_seed(run)
    size = torch.tensor([mix[i // run % len(mix)] for i in range(n)], dtype=F64)
    pages, table, (k, v) = cache_of(0.3 * torch.randn(n, nkv, hd, generator=g), positive(g, n, nkv, hd) * size[:, None, None], page)
    q = torch.randn(7, nq * hd, generator=g).to(BF16)
    if call == "decode":
        want, largest, _v = plain.attention(q.view(7, nq, hd), [k], [v], torch.tensor([n - 1] * 7), torch.zeros(7, dtype=torch.int32), hd ** -0.5)
        got = decode(ops, q, pages, table, n, nq, nkv, hd, page)
    else:
        want, largest, _v = plain.attention(q.view(7, nq, hd), [k], [v], *rows_of(n, 7), hd ** -0.5)
        got = portion(ops, q, pages, table, n, nq, nkv, hd, page)
    assert group_errors(got, want) <= HALF_STEP + 2 * 2.0 ** -11 + 2 * 2.0 ** -11 * largest
    ops.check_kernel_status()


@pytest.mark.parametrize("call", ["decode", "portion"])
def test_large_values_that_weigh_nothing_do_not_drown_the_others(ops, call):
    n, nq, nkv, hd, page, g = 320, 2, 2, 64, 16, torch.Generator().manual_seed(4)
    far = (torch.arange(n) // 64) % 2 == 1                   # tokens whose scores are about -280 below the others'
    q = torch.full((5, nq * hd), 2.0).to(BF16)
    keys = 0.05 * torch.randn(n, nkv, hd, generator=g) - 17.5 * far[:, None, None]
    values = positive(g, n, nkv, hd) * torch.where(far, 1e12, 1e-3)[:, None, None]
    pages, table, (k, v) = cache_of(keys, values, page)
    rows = rows_of(n, 5) if call == "portion" else (torch.tensor([n - 1] * 5), torch.zeros(5, dtype=torch.int32))
    want, _l, _v = plain.attention(q.view(5, nq, hd), [k], [v], *rows, hd ** -0.5)
    got = (portion if call == "portion" else decode)(ops, q, pages, table, n, nq, nkv, hd, page)
    # keys near -17.5 are of no weight; the others' scores, of up to 0.2 times 16 in all, are off by 2^-11 of that
    assert group_errors(got, want) <= HALF_STEP + 2 * 2.0 ** -11 + 4 * 2.0 ** -11
    ops.check_kernel_status()


@pytest.mark.parametrize("scale", [0.0, -0.125, float("nan")])
@pytest.mark.parametrize("call", [decode, portion])
def test_scales_that_are_not_positive_are_refused(ops, call, scale):
    """The largest score is looked for before the scale, and a masked one is -inf."""
    n, nq, nkv, hd, page, g = 60, 4, 2, 64, 16, torch.Generator().manual_seed(2)
    pages, table, _stored = cache_of(torch.randn(n, nkv, hd, generator=g), positive(g, n, nkv, hd), page)
    with pytest.raises(ops.KernelError, match="positive"):
        call(ops, torch.zeros(6, nq * hd, dtype=BF16), pages, table, n, nq, nkv, hd, page, scale)
    ops.check_kernel_status()


@pytest.mark.parametrize("scale", [0.0, -0.125, 1e-40])
def test_the_exact_kernel_takes_any_scale(ops, scale):
    n, nq, nkv, hd, page, g = 190, 4, 2, 64, 16, torch.Generator().manual_seed(2)
    pages, table, (k, v) = cache_of(torch.randn(n, nkv, hd, generator=g), positive(g, n, nkv, hd), page)
    q = torch.randn(6, nq * hd, generator=g).to(BF16)
    want, _l, _v = plain.attention(q.view(6, nq, hd), [k], [v], *rows_of(n, 6), scale)
    at, seq = (x.int().cuda() for x in rows_of(n, 6))
    out = torch.full((6, nq * hd), 9.0, dtype=BF16, device="cuda")
    ops.paged_attention_int4(q.cuda(), nq * hd, out, *pages, table, seq, at, nq, nkv, hd, page, scale)
    assert group_errors(out.view(6, nq, hd).double().cpu(), want) <= HALF_STEP + 2.0 ** -10
    ops.check_kernel_status()


@pytest.mark.parametrize("call", [decode, portion])
def test_the_smallest_scales_and_queries(ops, call):
    """Scores below any number: every token weighs the same, and masked ones nothing."""
    n, nq, nkv, hd, page, g = 190, 4, 2, 64, 16, torch.Generator().manual_seed(2)
    pages, table, (k, v) = cache_of(torch.randn(n, nkv, hd, generator=g), positive(g, n, nkv, hd), page)
    q = (torch.randn(6, nq * hd, generator=g) * 1e-36).to(BF16)
    rows = rows_of(n, 6) if call is portion else (torch.tensor([n - 1] * 6), torch.zeros(6, dtype=torch.int32))
    want, _l, _v = plain.attention(q.view(6, nq, hd), [k], [v], *rows, 1e-38)
    assert group_errors(call(ops, q, pages, table, n, nq, nkv, hd, page, 1e-38), want) <= HALF_STEP + 2.0 ** -10
    ops.check_kernel_status()
