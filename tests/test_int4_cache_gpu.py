"""The cache in 4 bits on the GPU: what is written into the rows, and attention over them, against a plain implementation in float64."""

import math

import pytest
import torch

import plain_int4 as plain

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
HALF = {F32: 2.0 ** -24, BF16: 2.0 ** -8}       # a rounding of a value, at most, relative to it


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from stride_b200.csrc import ops
    ops.check_kernel_status()
    yield ops
    ops.check_kernel_status()


def made_rows(seed, tokens, nq, nkv, hd, dtype, bias, norms, positions=4096):
    g = torch.Generator().manual_seed(seed)
    width = (nq + 2 * nkv) * hd
    rows = (torch.randn(tokens, width, generator=g) * (0.3 + torch.rand(width, generator=g))).to(dtype)
    f = 10000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)
    angles = torch.outer(torch.arange(positions, dtype=torch.float64), f)
    return dict(rows=rows, bias=torch.randn(width, generator=g) * 0.2 if bias else None,
                q_norm=1 + 0.3 * torch.randn(hd, generator=g) if norms else None, k_norm=1 + 0.3 * torch.randn(hd, generator=g) if norms else None,
                positions=torch.randint(0, positions, (tokens,), generator=g, dtype=torch.int32), cos=angles.cos().float(), sin=angles.sin().float())


def on_gpu(d):
    return {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in d.items()}


def write(ops, made, slots, pages, nq, nkv, hd, page, bits4, rotate=True, eps=1e-5, **more):
    d = on_gpu(made)
    call = ops.rope_kv_write_int4 if bits4 else ops.qk_norm_rope_write
    call(d["rows"], d["bias"], d["q_norm"], d["k_norm"], eps, d["positions"], slots, d["cos"], d["sin"], *pages, nq, nkv, hd, page, rotate, **more)
    return d["rows"]


SHAPES = [  # tokens, nq, nkv, hd, page
    (1, 4, 1, 128, 16), (37, 32, 8, 128, 16), (5, 3, 1, 64, 8), (64, 8, 8, 64, 32), (9, 12, 4, 96, 8), (11, 6, 2, 80, 5), (6, 5, 5, 48, 1),
    (7, 4, 2, 16, 16), (3, 2, 2, 32, 64), (4, 2, 1, 256, 16), (130, 7, 1, 128, 16), (3, 2, 1, 20, 4), (4, 3, 3, 192, 7)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("norms", [False, True])
@pytest.mark.parametrize("tokens,nq,nkv,hd,page", SHAPES)
def test_head_norms_rotation_and_pages(ops, tokens, nq, nkv, hd, page, norms, dtype):
    made = made_rows(tokens + hd, tokens, nq, nkv, hd, dtype, tokens % 2 == 1, norms)
    count = -(-tokens // page) + 2
    slots = torch.randperm(count * page, generator=torch.Generator().manual_seed(1))[:tokens].int()
    if tokens > 4:
        slots[3] = -1                                       # a padded token: its queries are turned, nothing is stored
    pages = [torch.full((count, nkv, page, hd), math.nan, dtype=dtype, device="cuda") for _ in "kv"]
    out = write(ops, made, slots.cuda(), pages, nq, nkv, hd, page, False).cpu()
    q, k, v = plain.prepare_heads(made["rows"], made["bias"], made["q_norm"], made["k_norm"], 1e-5, made["positions"], made["cos"], made["sin"], nq, nkv, hd)
    # 32 bits between load and store: the sum of squares hd roundings, the norm four, the rotation three, of terms as large as the pair
    pair = lambda t: torch.sqrt(t.square() + t.roll(hd // 2, -1).square()) * 1.5  # noqa: E731
    for got, want in ((out[:, :nq * hd].view(tokens, nq, hd), q),):
        assert bool(((got.double() - want).abs() <= HALF[dtype] * want.abs() + (hd + 16) * 2.0 ** -24 * pair(want) + 1e-30).all())
    untouched = made["rows"][:, nq * hd:]
    assert torch.equal(out[:, nq * hd:], untouched)         # the projection's keys and values stay
    seen = torch.zeros(count * page, dtype=torch.bool)
    for name, t, want in (("k", pages[0], k), ("v", pages[1], v)):
        flat = t.cpu().transpose(1, 2).reshape(count * page, nkv, hd)
        for i, s in enumerate(slots.tolist()):
            if s < 0:
                continue
            seen[s] = True
            limit = HALF[dtype] * want[i].abs() + (hd + 16) * 2.0 ** -24 * pair(want[i]) + 1e-30
            assert bool(((flat[s].double() - want[i]).abs() <= limit).all()), (name, i)
        assert bool(flat[~seen].isnan().all())              # the other slots were left alone
    ops.check_kernel_status()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rotate", [True, False])
@pytest.mark.parametrize("tokens,nq,nkv,hd,page", SHAPES)
def test_rows_in_4_bits_bit_by_bit(ops, tokens, nq, nkv, hd, page, rotate, dtype):
    """Without norms every step from the projection to a number is one 32-bit operation, the same on any machine."""
    made = made_rows(tokens + hd, tokens, nq, nkv, hd, dtype, tokens % 2 == 0, False)
    count = -(-tokens // page) + 2
    slots = torch.randperm(count * page, generator=torch.Generator().manual_seed(2))[:tokens].int()
    pages = [torch.full((count, nkv, page, ops.int4_row_bytes(hd)), 255, dtype=torch.uint8, device="cuda") for _ in "kv"]
    q_out = torch.full((tokens, nq * hd + 8), 7.0, dtype=dtype, device="cuda")[:, :nq * hd]          # rows of another length
    rows = write(ops, made, slots.cuda(), pages, nq, nkv, hd, page, True, rotate, q_out=q_out)
    assert torch.equal(rows.cpu(), made["rows"])
    q, k, v = plain.prepare_heads(made["rows"], made["bias"], None, None, 0, made["positions"], made["cos"], made["sin"], nq, nkv, hd, rotate, F32)
    assert torch.equal(q_out.cpu(), q.reshape(tokens, -1).to(dtype))
    for which, t, x in (("k", pages[0], k), ("v", pages[1], v)):
        flat = t.cpu().transpose(1, 2).reshape(count * page, nkv, -1)
        assert torch.equal(flat[slots.long()], plain.pack(which, *plain.quantise(x)))
        others = torch.ones(count * page, dtype=torch.bool)
        others[slots.long()] = False
        assert bool((flat[others] == 255).all())
    read = [torch.empty(tokens + 1, nkv, hd, dtype=F32, device="cuda") for _ in "kv"]
    ops.read_int4(*pages, torch.cat([slots, torch.tensor([-1], dtype=torch.int32)]).cuda(), *read, nkv, hd, page)
    for which, t, got in (("k", pages[0], read[0]), ("v", pages[1], read[1])):
        flat = t.cpu().transpose(1, 2).reshape(count * page, nkv, -1)
        assert torch.equal(got[:-1].cpu(), plain.unpack(which, flat[slots.long()], hd).float()) and not bool(got[-1].any())
    ops.check_kernel_status()


@pytest.mark.parametrize("tokens,nq,nkv,hd,page", SHAPES)
def test_rows_in_4_bits_behind_norms(ops, tokens, nq, nkv, hd, page):
    made = made_rows(tokens + hd, tokens, nq, nkv, hd, BF16, True, True)
    count = -(-tokens // page) + 1
    slots = torch.randperm(count * page, generator=torch.Generator().manual_seed(3))[:tokens].int().cuda()
    pages = [torch.full((count, nkv, page, ops.int4_row_bytes(hd)), 255, dtype=torch.uint8, device="cuda") for _ in "kv"]
    write(ops, made, slots, pages, nq, nkv, hd, page, True)
    _q, k, v = plain.prepare_heads(made["rows"], made["bias"], made["q_norm"], made["k_norm"], 1e-5, made["positions"], made["cos"], made["sin"], nq, nkv, hd)
    read = [torch.empty(tokens, nkv, hd, dtype=F32, device="cuda") for _ in "kv"]
    ops.read_int4(*pages, slots, *read, nkv, hd, page)
    for got, want in ((read[0], k), (read[1], v)):
        for lo in range(0, hd, 32):
            part = want[..., lo:lo + 32]
            low, high = part.amin(-1, keepdim=True), part.amax(-1, keepdim=True)
            step = (high - low) / 15
            limit = step * (0.5 * (1 + 2.0 ** -8) + 15 * 2.0 ** -8) + 2.0 ** -8 * (low + 8 * step).abs() + hd * 2.0 ** -22 * part.abs().amax(-1, keepdim=True)
            assert bool(((got[..., lo:lo + 32].cpu().double() - part).abs() <= limit).all())


def test_groups_without_a_range_and_tokens_that_are_no_numbers(ops):
    nq, nkv, hd, page, tokens = 2, 2, 64, 8, 8
    rows = torch.randn(tokens, (nq + 2 * nkv) * hd, generator=torch.Generator().manual_seed(5))
    k, v = rows[:, nq * hd:(nq + nkv) * hd].view(tokens, nkv, hd), rows[:, (nq + nkv) * hd:].view(tokens, nkv, hd)
    k[0, 0, :32], v[0, 1] = 3.0, 0.0                        # groups of one value
    k[1, 0, 5], v[2, 1, 40], k[3, 1, 63] = math.nan, math.inf, -math.inf
    k[4, 0, 0], k[4, 0, 1] = 3e38, -3e38                    # a range that is no 32-bit number
    v[5, 0] = 1e-39                                         # below the smallest normal number
    v[6, 0, :32] = torch.linspace(1e-30, 2e-30, 32)
    made = dict(rows=rows, bias=None, q_norm=None, k_norm=None, positions=torch.zeros(tokens, dtype=torch.int32), cos=torch.ones(1, 32), sin=torch.zeros(1, 32))
    pages = [torch.zeros(1, nkv, page, 40, dtype=torch.uint8, device="cuda") for _ in "kv"]
    slots = torch.arange(tokens, dtype=torch.int32, device="cuda")
    write(ops, made, slots, pages, nq, nkv, hd, page, True, False)
    kr, vr = (torch.empty(tokens, nkv, hd, device="cuda") for _ in "kv")
    ops.read_int4(*pages, slots, kr, vr, nkv, hd, page)
    kr, vr = kr.cpu(), vr.cpu()
    bad = {(1, 0), (2, 1), (3, 1), (4, 0)}
    for t in range(tokens):
        for h in range(nkv):
            if (t, h) in bad:                               # every entry of the key is no number, the value nothing
                assert bool(kr[t, h].isnan().all()) and not bool(vr[t, h].any())
            else:
                assert bool(kr[t, h].isfinite().all()) and bool(vr[t, h].isfinite().all())
    assert bool((kr[0, 0, :32] == 3.0).all()) and not bool(vr[0, 1].any())
    assert bool((vr[5, 0] - 1e-39).abs().max() <= 1e-40)
    assert bool((vr[6, 0, :32] - v[6, 0, :32]).abs().max() <= 1e-30 / 15 * 0.6)
    ops.check_kernel_status()


@pytest.mark.parametrize("bits4", [False, True])
@pytest.mark.parametrize("columns", [(64, 320), (256, 512)])
def test_rows_for_queries_among_those_of_the_call_are_refused(ops, bits4, columns):
    """A block of qkv other than its queries is still to be read when queries are written."""
    nq, nkv, hd, page = 4, 2, 64, 4
    qkv = torch.zeros(3, (nq + 2 * nkv) * hd, dtype=BF16, device="cuda")
    row = ops.int4_row_bytes(hd) if bits4 else hd
    pages = [torch.zeros(2, nkv, page, row, dtype=torch.uint8 if bits4 else BF16, device="cuda") for _ in "kv"]
    at = torch.zeros(3, dtype=torch.int32, device="cuda")
    angles = torch.zeros(8, hd // 2, device="cuda")
    call = ops.rope_kv_write_int4 if bits4 else ops.qk_norm_rope_write
    with pytest.raises(ops.KernelError, match="lie apart"):
        call(qkv, None, None, None, 1e-5, at, None, angles, angles, *pages, nq, nkv, hd, page, q_out=qkv[:, columns[0]:columns[1]])
    call(qkv, None, None, None, 1e-5, at, None, angles, angles, *pages, nq, nkv, hd, page, q_out=qkv[:, :nq * hd])
    ops.check_kernel_status()


@pytest.mark.parametrize("bits4", [False, True])
@pytest.mark.parametrize("q_out", [torch.zeros(3, 255, dtype=BF16), torch.zeros(3, 256), torch.zeros(2, 256, dtype=BF16), torch.zeros(256, 3, dtype=BF16).t(),
                                   torch.zeros(3, 2, 128, dtype=BF16)])
def test_refused_rows_for_queries(ops, bits4, q_out):
    made = made_rows(1, 3, 4, 2, 64, BF16, False, False)
    pages = [torch.zeros(2, 2, 4, 40 if bits4 else 64, dtype=torch.uint8 if bits4 else BF16, device="cuda") for _ in "kv"]
    slots = torch.arange(3, dtype=torch.int32, device="cuda")
    for bad in (q_out.cuda(), torch.zeros(3, 256, dtype=BF16)):            # the last on the host
        with pytest.raises(ops.KernelError):
            write(ops, made, slots, pages, 4, 2, 64, 4, bits4, q_out=bad)


def test_slots_and_positions_out_of_range_are_reported(ops):
    made = made_rows(1, 3, 2, 1, 64, BF16, False, False, positions=50)
    for bits4 in (False, True):
        pages = [torch.full((2, 1, 4, 40 if bits4 else 64), 9, dtype=torch.uint8 if bits4 else BF16, device="cuda") for _ in "kv"]
        slots = torch.tensor([1, 8, 2], dtype=torch.int32, device="cuda")
        write(ops, made, slots, pages, 2, 1, 64, 4, bits4)
        with pytest.raises(ops.KernelError, match="slot"):
            ops.check_kernel_status()
        assert bool((pages[0][0, 0, 0] == 9).all()) and not bool((pages[0][0, 0, 1:3] == 9).all(-1).any())
        bad = dict(made, positions=torch.tensor([3, 50, -1], dtype=torch.int32))
        out = write(ops, bad, torch.tensor([1, 3, 0], dtype=torch.int32, device="cuda"), pages, 2, 1, 64, 4, bits4)
        with pytest.raises(ops.KernelError, match="position"):
            ops.check_kernel_status()
        assert torch.equal(out[1:].cpu(), made["rows"][1:]) and bool((pages[0][0, 0, 3] == 9).all())
    k, v = (torch.full((2, 1, 64), 5.0, device="cuda") for _ in "kv")
    ops.read_int4(*pages, torch.tensor([1, 8], dtype=torch.int32, device="cuda"), k, v, 1, 64, 4)
    with pytest.raises(ops.KernelError, match="slot"):
        ops.check_kernel_status()
    assert not bool(k[1].any())


# --------------------------------------------------------------------------------------------------------------- attention
def made_cache(seed, lengths, nkv, hd, page, spread=1.0, hole=0):
    """Pages of random keys and values, their values per request (float64), a table, and everything else full of 255 (no numbers)."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lengths]
    total = sum(need) + 2
    order = torch.randperm(total, generator=g).tolist()
    width = plain.groups(hd) * 20
    pages = [torch.full((total, nkv, page, width), 255, dtype=torch.uint8) for _ in "kv"]
    table = torch.full((len(lengths), max(need)), -1, dtype=torch.int32)
    values = [[], []]
    for r, n in enumerate(lengths):
        ids = [order.pop() for _ in range(need[r])]
        table[r, :need[r]] = torch.tensor(ids, dtype=torch.int32)
        for w, which in enumerate("kv"):
            x = torch.randn(n, nkv, hd, generator=g) * spread
            rows = plain.pack(which, *plain.quantise(x))
            values[w].append(plain.unpack(which, rows, hd))
            for i in range(n):
                pages[w][ids[i // page], :, i % page] = rows[i]
        for gone in range(hole):
            table[r, gone] = -1                             # pages that a window has passed
    return [p.cuda() for p in pages], table.cuda(), values


def score_error(hd, largest):
    """A score in 32 bits: hd products and sums, the value's own two operations, scale, cap and slope."""
    return (hd + 8) * 2.0 ** -24 * largest


def check(got, want, ds, keys, value, dtype, weight_error=0.0, value_error=0.0):
    """A weight is off by 2 ds (its own score's and the maximum's) and a few roundings of the exponential, a sum of `keys` terms by as many."""
    relative = 2 * math.expm1(2 * ds) + (keys + 32) * 2.0 ** -23 + weight_error
    limit = HALF[dtype] * want.abs() + (relative + value_error) * value
    worst = float(((got.double().cpu() - want).abs() - limit).max())
    assert bool((got.double().cpu() - want).isfinite().all()) and worst <= 0, (worst, float((got.double().cpu() - want).abs().max()))


RULES = [dict(), dict(window=7), dict(softcap=5.0), dict(sinks=True), dict(slopes=True), dict(window=40, softcap=3.0, sinks=True, slopes=True)]


def rule_args(rules, nq, seed=0):
    g = torch.Generator().manual_seed(seed)
    sinks = torch.randn(nq, generator=g) if rules.get("sinks") else None
    slopes = torch.tensor([2.0 ** (-8 * (h + 1) / nq) for h in range(nq)]) if rules.get("slopes") else None
    return rules.get("window", 0), rules.get("softcap", 0.0), sinks, slopes


def gpu(t):
    return None if t is None else t.cuda()


@pytest.mark.parametrize("rules", RULES, ids=str)
@pytest.mark.parametrize("nq,nkv,hd,page", [(4, 2, 64, 16), (3, 1, 32, 8), (5, 5, 48, 5), (2, 1, 256, 16), (8, 1, 128, 64), (4, 4, 16, 1)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_exact_attention(ops, nq, nkv, hd, page, rules, dtype):
    lengths = [1, 90, 33]
    pages, table, (k, v) = made_cache(7 + hd, lengths, nkv, hd, page)
    at = [(0, 0), (1, 0), (1, 31), (1, 32), (1, 89), (2, 32), (-1, 0), (2, 5)]
    seq, pos = (torch.tensor(c, dtype=torch.int32) for c in zip(*at))
    q = torch.randn(len(at), nq * hd + 3, generator=torch.Generator().manual_seed(2)).to(dtype)
    window, softcap, sinks, slopes = rule_args(rules, nq)
    out = torch.full((len(at), nq * hd), 9.0, dtype=dtype, device="cuda")
    ops.paged_attention_int4(q.cuda(), nq * hd + 3, out, *pages, table, seq.cuda(), pos.cuda(), nq, nkv, hd, page, hd ** -0.5, window, softcap, gpu(sinks),
                             gpu(slopes))
    want, largest, value = plain.attention(q[:, :nq * hd].view(-1, nq, hd), k, v, pos, seq, hd ** -0.5, window, softcap, sinks, slopes)
    check(out.view(-1, nq, hd), want, score_error(hd, largest + 90), 90, value, dtype)
    again = torch.full_like(out, 9.0)
    ops.paged_attention_int4(q.cuda(), nq * hd + 3, again, *pages, table, seq.cuda(), pos.cuda(), nq, nkv, hd, page, hd ** -0.5, window, softcap, gpu(sinks),
                             gpu(slopes), neighbours=True)
    assert torch.equal(out, again)                          # rows of several requests side by side: only the time differs
    for neighbours in (False, True):
        for bound in (1, 5000):                             # one CTA for a row's keys, eight of them
            again = torch.full_like(out, 9.0)
            ops.paged_attention_int4(q.cuda(), nq * hd + 3, again, *pages, table, seq.cuda(), pos.cuda(), nq, nkv, hd, page, hd ** -0.5, window, softcap,
                                     gpu(sinks), gpu(slopes), neighbours, bound)
            assert torch.equal(out, again)
    ops.check_kernel_status()


def test_exact_attention_of_a_long_prompt_has_the_bits_of_its_portions(ops):
    """1190 rows of 16 key heads: enough for eight rows a CTA; a last tile of six; against portions of other sizes and rows alone."""
    nq, nkv, hd, page, n = 16, 16, 64, 16, 1190
    pages, table, (k, v) = made_cache(12, [n], nkv, hd, page)
    q = torch.randn(n, nq * hd, generator=torch.Generator().manual_seed(8)).cuda()
    pos, seq = torch.arange(n, dtype=torch.int32, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda")

    def run(lo, hi, **cut):
        into = torch.full((hi - lo, nq * hd), 9.0, device="cuda")
        ops.paged_attention_int4(q[lo:hi], nq * hd, into, *pages, table, seq[lo:hi], pos[lo:hi], nq, nkv, hd, page, hd ** -0.5, **cut)
        return into

    out = run(0, n)
    for lo, hi in ((0, 37), (500, 503), (1100, n)):
        assert torch.equal(run(lo, hi), out[lo:hi])
        assert torch.equal(run(lo, hi, neighbours=False, context_bound=1), out[lo:hi])
    some = [0, 31, 32, 255, 256, 257, 700, n - 1]
    want, largest, value = plain.attention(q.cpu()[some].view(-1, nq, hd), k, v, pos.cpu()[some], seq.cpu()[some], hd ** -0.5)
    check(out[some].view(-1, nq, hd), want, score_error(hd, largest), n, value, torch.float32)
    ops.check_kernel_status()


@pytest.mark.parametrize("window", [0, 300])
@pytest.mark.parametrize("hd", [64, 112, 160, 200, 256])
@pytest.mark.parametrize("dtype", [torch.float32, BF16], ids=str)
def test_exact_attention_over_rounds_of_streams(ops, dtype, hd, window):
    """1900 keys: each of the eight streams comes round more than seven times; a portion of 70 rows, and rows of two requests in one tile."""
    nq, nkv, page = 10, 2, 48
    lengths = [1900, 517]
    pages, table, (k, v) = made_cache(9, lengths, nkv, hd, page)
    at = [(0, p) for p in range(1830, 1900)] + [(1, 516), (0, 255), (0, 256), (1, 0), (-1, 0), (1, 300)]
    seq, pos = (torch.tensor(c, dtype=torch.int32) for c in zip(*at))
    q = torch.randn(len(at), nq * hd, generator=torch.Generator().manual_seed(5)).to(dtype)
    sinks = torch.randn(nq, generator=torch.Generator().manual_seed(6))
    outs = []
    for neighbours in (False, True):
        for bound in (1, 5000):
            outs.append(torch.full((len(at), nq * hd), 9.0, dtype=dtype, device="cuda"))
            ops.paged_attention_int4(q.cuda(), nq * hd, outs[-1], *pages, table, seq.cuda(), pos.cuda(), nq, nkv, hd, page, hd ** -0.5, window, 0.0,
                                     sinks.cuda(), None, neighbours, bound)
    want, largest, value = plain.attention(q.view(-1, nq, hd), k, v, pos, seq, hd ** -0.5, window, 0.0, sinks, None)
    check(outs[0].view(-1, nq, hd), want, score_error(hd, largest), 1900, value, dtype)
    assert all(torch.equal(outs[0], o) for o in outs[1:])
    ops.check_kernel_status()


def test_exact_attention_has_the_same_bits_however_the_work_is_cut(ops):
    nq, nkv, hd, page = 6, 2, 64, 8
    pages, table, _values = made_cache(3, [75], nkv, hd, page)
    pages2 = [torch.cat([p, p]) for p in pages]
    q = torch.randn(75, nq * hd, generator=torch.Generator().manual_seed(4)).cuda()
    pos, seq = torch.arange(75, dtype=torch.int32, device="cuda"), torch.zeros(75, dtype=torch.int32, device="cuda")

    def run(lo, hi, pages, table):
        out = torch.empty(hi - lo, nq * hd, device="cuda")
        ops.paged_attention_int4(q[lo:hi], nq * hd, out, *pages, table, seq[lo:hi], pos[lo:hi], nq, nkv, hd, page, 0.125)
        return out
    whole = run(0, 75, pages, table)
    moved = torch.where(table < 0, table, table + pages[0].shape[0])
    assert torch.equal(whole, torch.cat([run(0, 13, pages, table), run(13, 14, pages, table), run(14, 75, pages2, moved)]))


def run_decode(ops, q, stride, out, pages, table, seq, pos, nq, nkv, hd, page, window, softcap, sinks, slopes, bound, scratch=None):
    if scratch is None:
        scratch = torch.zeros(ops.decode_int4_scratch_floats(out.shape[0], nq, nkv, hd, bound), device="cuda")
    ops.paged_attention_decode_int4(q, stride, out, *pages, table, seq, pos, scratch, nq, nkv, hd, page, hd ** -0.5, window, bound, softcap, gpu(sinks),
                                    gpu(slopes))
    return scratch


def check_decode(got, want, hd, largest, keys, value):
    # 16-bit weights: 2^-11 of a weight and of its product with a scale, for what a centre is multiplied by 2^-8; below the normal 16-bit
    # numbers 2^-25 of the largest product, 15 times for the largest number, a key
    check(got, want, score_error(hd, largest), keys, value, BF16, weight_error=2 * 2.0 ** -11 + 2.0 ** -8 + 15 * keys * 2.0 ** -25)


DECODE_SHAPES = [(4, 1, 128, 16), (32, 8, 128, 16), (8, 1, 128, 16), (7, 1, 64, 16), (2, 2, 64, 32), (16, 1, 128, 64), (12, 4, 64, 8), (6, 2, 128, 5), (3, 3, 128, 1),
                 (13, 1, 64, 48)]


@pytest.mark.parametrize("rules", RULES + [dict(window=1), dict(window=16), dict(window=100)], ids=str)
@pytest.mark.parametrize("nq,nkv,hd,page", DECODE_SHAPES)
def test_decode_attention(ops, nq, nkv, hd, page, rules):
    lengths = [1, 2, 16, 17, 64, 131, 300]
    pages, table, (k, v) = made_cache(11 + hd + nq, lengths, nkv, hd, page)
    seq = torch.tensor([6, 0, 1, 2, -1, 3, 4, 5, 6], dtype=torch.int32)
    pos = torch.tensor([299, 0, 1, 15, 0, 16, 63, 130, 200], dtype=torch.int32)
    stride = nq * hd + 8
    q = torch.randn(len(seq), stride, generator=torch.Generator().manual_seed(6)).to(BF16)
    window, softcap, sinks, slopes = rule_args(rules, nq)
    want, largest, value = plain.attention(q[:, :nq * hd].view(-1, nq, hd), k, v, pos, seq, hd ** -0.5, window, softcap, sinks, slopes)
    out = torch.full((len(seq) + 1, nq * hd), 9.0, dtype=BF16, device="cuda")
    scratch = None
    for bound in (300, 301, 4096, 300):
        out.fill_(9.0)
        fresh = None if scratch is None or scratch.numel() < ops.decode_int4_scratch_floats(len(seq), nq, nkv, hd, bound) else scratch
        scratch = run_decode(ops, q.cuda(), stride, out[:-1], pages, table, seq.cuda(), pos.cuda(), nq, nkv, hd, page, window, softcap, sinks, slopes, bound, fresh)
        check_decode(out[:-1].view(-1, nq, hd), want, hd, largest + 300, 300, value)
        assert bool((out[-1] == 9.0).all())
    ops.check_kernel_status()


@pytest.mark.parametrize("nq,nkv,hd", [(32, 8, 128), (4, 1, 64), (16, 1, 128)])
def test_decode_attention_over_a_long_context(ops, nq, nkv, hd):
    """Many splits, uneven requests; the reference here in float64 on the GPU, head by head."""
    page, lengths = 16, [20000, 4097, 513]
    g = torch.Generator(device="cuda").manual_seed(1)
    total = sum(-(-n // page) for n in lengths)
    small, _t, (ks, vs) = made_cache(9, [160], nkv, hd, page)        # ten pages, used over and over
    ids = torch.randint(0, 10, (total,), generator=g, device="cuda").int()
    own = _t[0]
    table = torch.full((3, 1250), -1, dtype=torch.int32, device="cuda")
    at = 0
    out = torch.empty(3, nq * hd, dtype=BF16, device="cuda")
    q = (2 * torch.randn(3, nq * hd, generator=g, device="cuda")).to(BF16)
    pick = []
    for r, n in enumerate(lengths):
        need = -(-n // page)
        pick.append(ids[at:at + need].long())
        table[r, :need] = own[pick[-1]]
        at += need
    pos = torch.tensor([n - 1 for n in lengths], dtype=torch.int32, device="cuda")
    run_decode(ops, q, nq * hd, out, small, table, torch.arange(3, dtype=torch.int32, device="cuda"), pos, nq, nkv, hd, page, 0, 0.0, None, None, 20000)
    k10, v10 = (t[0].cuda().view(10, page, nkv, hd) for t in (ks, vs))
    for r, n in enumerate(lengths):
        k, v = (t[pick[r]].reshape(-1, nkv, hd)[:n] for t in (k10, v10))
        for h in range(nq):
            s = k[:, h // (nq // nkv)] @ q[r, h * hd:(h + 1) * hd].double() * hd ** -0.5
            want = torch.softmax(s, 0) @ v[:, h // (nq // nkv)]
            err = (out[r, h * hd:(h + 1) * hd].double() - want).norm() / want.norm()
            assert err < 2.0 ** -8, (r, h, float(err))      # half a step of bfloat16 at most a value, and much less in the mean
    ops.check_kernel_status()


@pytest.mark.parametrize("scale_v,scale_k", [(1e-6, 1.0), (1e5, 1.0), (1e-30, 1e-3), (1.0, 50.0), (1e30, 30.0), (3.0, 1e-20)])
def test_decode_attention_at_extreme_sizes(ops, scale_v, scale_k):
    """Values and keys far from 1: nothing in between may leave the range of a 16-bit number."""
    nq, nkv, hd, page, n = 8, 2, 128, 16, 200
    g = torch.Generator().manual_seed(8)
    k = torch.randn(n, nkv, hd, generator=g) * scale_k
    v = torch.randn(n, nkv, hd, generator=g) * scale_v * torch.logspace(-3, 0, n)[:, None, None]       # tokens of very different sizes
    rows = [plain.pack(w, *plain.quantise(x)) for w, x in (("k", k), ("v", v))]
    kv, vv = (plain.unpack(w, r, hd) for w, r in zip("kv", rows))
    pages = [torch.nn.functional.pad(r, (0, 0, 0, 0, 0, 8), value=255).view(13, page, nkv, -1).transpose(1, 2).contiguous().cuda() for r in rows]
    table = torch.arange(13, dtype=torch.int32, device="cuda")[None]
    q = torch.randn(1, nq * hd, generator=g).to(BF16)
    out = torch.empty(1, nq * hd, dtype=BF16, device="cuda")
    pos, seq = torch.tensor([n - 1], dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    run_decode(ops, q.cuda(), nq * hd, out, pages, table, seq.cuda(), pos.cuda(), nq, nkv, hd, page, 0, 0.0, None, None, n)
    want, largest, value = plain.attention(q.view(1, nq, hd), [kv], [vv], pos, seq, hd ** -0.5)
    # relative to the largest term that counts, not to the largest value: a weight times a scale keeps 2^-25 of the largest such product
    check_decode(out.view(1, nq, hd), want, hd, largest, n, value)
    assert float((out.view(1, nq, hd).double().cpu() - want).norm() / want.norm()) < 2.0 ** -7 + 4 * score_error(hd, largest)


def test_a_query_of_any_size(ops):
    nq, nkv, hd, page, n = 4, 1, 64, 16, 50
    pages, table, (k, v) = made_cache(3, [n], nkv, hd, page)
    pos, seq = torch.tensor([n - 1] * 4, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    q = torch.randn(4, nq * hd, generator=torch.Generator().manual_seed(8))
    q = (q * torch.tensor([1e-30, 0.0, 1e-3, 40.0])[:, None]).to(BF16)
    out = torch.empty(4, nq * hd, dtype=BF16, device="cuda")
    run_decode(ops, q.cuda(), nq * hd, out, pages, table, seq.cuda(), pos.cuda(), nq, nkv, hd, page, 0, 0.0, None, None, n)
    want, largest, value = plain.attention(q.view(4, nq, hd), k, v, pos, seq, hd ** -0.5)
    check_decode(out.view(4, nq, hd), want, hd, largest, n, value)


def test_tokens_that_are_no_numbers_reach_only_who_sees_them(ops):
    """A key full of NaN, in one key head of one request, and queries before and behind it: decode, portions and the exact kernel."""
    nq, nkv, hd, page, n = 8, 2, 64, 16, 150
    pages, table, _values = made_cache(5, [n, n], nkv, hd, page)
    pages[0][table[0, 70 // page], 1, 70 % page] = 255
    pages[1][table[0, 70 // page], 1, 70 % page] = 136
    pages[1][table[0, 70 // page], 1, 70 % page, 32:] = 0                   # as the write leaves the value of such a token: zeros
    seq = torch.tensor([0] * n + [1], dtype=torch.int32, device="cuda")
    pos = torch.cat([torch.arange(n), torch.tensor([n - 1])]).int().cuda()
    q = torch.randn(n + 1, nq * hd, generator=torch.Generator().manual_seed(1)).to(BF16).cuda()

    def verify(out, window):
        bad = out.view(-1, 2, 4 * hd).isnan()
        assert not bool(bad[:, 0].any()) and not bool(bad[:70].any()) and not bool(bad[n:].any())
        assert bool(bad[70:min(n, 70 + (window or n)), 1].all()) and not bool(bad[70 + (window or n):].any())
    for window in (0, 20):
        for call in ("exact", "decode", "portion"):
            out = torch.empty(n + 1, nq * hd, dtype=BF16, device="cuda")
            if call == "exact":
                ops.paged_attention_int4(q, nq * hd, out, *pages, table, seq, pos, nq, nkv, hd, page, 0.125, window)
            elif call == "decode":
                run_decode(ops, q, nq * hd, out, pages, table, seq, pos, nq, nkv, hd, page, window, 0.0, None, None, n)
            else:
                run_portion(ops, q, out, pages, table, [n, 1], [n, n], nq, nkv, hd, page, window)
            verify(out, window)
    ops.check_kernel_status()


def run_portion(ops, q, out, pages, table, lens, held, nq, nkv, hd, page, window=0, softcap=0.0, sinks=None, slopes=None, keys=None, scratch=None):
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    keys = sum(held) if keys is None else keys
    if scratch is None:
        scratch = torch.full((ops.prefill_int4_scratch_ints(len(lens), keys, nkv, hd),), -1, dtype=torch.int32, device="cuda")      # NaNs
    ops.paged_attention_prefill_int4(q, q.shape[1], out, *pages, table, ints([sum(lens[:i]) for i in range(len(lens))]), ints(lens), ints(held), scratch,
                                     len(lens), keys, nq, nkv, hd, page, hd ** -0.5, window, softcap, gpu(sinks), gpu(slopes))
    return scratch


@pytest.mark.parametrize("rules", RULES + [dict(window=1), dict(window=64)], ids=str)
@pytest.mark.parametrize("nq,nkv,hd,page", [(4, 1, 128, 16), (8, 2, 64, 16), (3, 1, 128, 5), (6, 6, 64, 64), (14, 2, 128, 8), (16, 1, 64, 1)])
def test_attention_of_portions(ops, nq, nkv, hd, page, rules):
    held, lens = [140, 1, 64, 201, 70], [140, 1, 5, 66, 3]
    pages, table, (k, v) = made_cache(19 + hd + nq, held, nkv, hd, page)
    if rules.get("window") == 1:                            # pages that no query of the portion sees are gone
        for r, (n, p) in enumerate(zip(held, lens)):
            table[r, :(n - p) // page] = -1
    seq = torch.tensor([r for r, p in enumerate(lens) for _ in range(p)], dtype=torch.int32)
    pos = torch.tensor([n - p + i for n, p in zip(held, lens) for i in range(p)], dtype=torch.int32)
    q = torch.randn(len(seq), nq * hd, generator=torch.Generator().manual_seed(9)).to(BF16)
    window, softcap, sinks, slopes = rule_args(rules, nq)
    pick = torch.randperm(len(seq), generator=torch.Generator().manual_seed(1))[:60]        # rows that are compared
    want, largest, value = plain.attention(q.view(-1, nq, hd)[pick], k, v, pos[pick], seq[pick], hd ** -0.5, window, softcap, sinks, slopes)
    out = torch.full((len(seq) + 2, nq * hd), 9.0, dtype=BF16, device="cuda")
    for keys in (sum(held), sum(held) + 5000):
        run_portion(ops, q.cuda(), out[:-2], pages, table, lens, held, nq, nkv, hd, page, window, softcap, sinks, slopes, keys)
        got = out[:-2].view(-1, nq, hd)[pick.cuda()]
        # keys rounded to bfloat16: each product of a score by 2^-8; the capped score's short tanh by 2^-10 of the cap; weights and values by 2^-8
        ds = score_error(hd, largest + 200) + 2.0 ** -8 * largest + 2.0 ** -10 * softcap
        check(got, want, ds, 201, value, BF16, weight_error=2.0 ** -7, value_error=2.0 ** -8)
        # and all of it in the mean: three independent roundings beside the result's own
        assert float((got.double().cpu() - want).norm() / want.norm()) < 2.0 ** -7 + 2.0 ** -10 * softcap
        assert bool((out[-2:] == 9.0).all())
    ops.check_kernel_status()


def test_portions_count_entries_beyond_the_16_bit_range_as_its_end(ops):
    nq, nkv, hd, page, n = 4, 1, 64, 16, 40
    pages, table, (k, v) = made_cache(5, [n], nkv, hd, page, spread=3e4)
    clipped = v[0].clamp(-65504, 65504)
    assert bool((clipped != v[0]).any())
    q = (torch.randn(n, nq * hd, generator=torch.Generator().manual_seed(9)) * 1e-5).to(BF16)
    pos, seq = torch.arange(n, dtype=torch.int32), torch.zeros(n, dtype=torch.int32)
    out = torch.empty(n, nq * hd, dtype=BF16, device="cuda")
    run_portion(ops, q.cuda(), out, pages, table, [n], [n], nq, nkv, hd, page)
    want, largest, value = plain.attention(q.view(n, nq, hd), [k[0].clamp(-65504, 65504)], [clipped], pos, seq, hd ** -0.5)
    # keys, values and weights to 11 bits; queries of 1e-5 are below the smallest normal 16-bit number, 2^-14, and keep multiples of 2^-24
    ds = score_error(hd, largest) + 2.0 ** -11 * largest + hd * 2.0 ** -25 * 65504 * hd ** -0.5
    check(out.view(n, nq, hd), want, ds, n, value, BF16, weight_error=2.0 ** -10, value_error=2.0 ** -11)


def test_too_many_keys_for_a_portions_scratch_are_reported(ops):
    nq, nkv, hd, page = 4, 1, 64, 16
    held, lens = [2300, 10], [1, 1]
    pages, table, _values = made_cache(2, held, nkv, hd, page)
    q = torch.randn(2, nq * hd).to(BF16).cuda()
    out = torch.empty_like(q)
    run_portion(ops, q, out, pages, table, lens, held, nq, nkv, hd, page, keys=100)
    with pytest.raises(ops.KernelError, match="more keys"):
        ops.check_kernel_status()


@pytest.mark.parametrize("call", ["exact", "decode", "portion"])
@pytest.mark.parametrize("entry", [-1, 99])
def test_a_key_without_a_page_is_reported(ops, call, entry):
    nq, nkv, hd, page = 4, 1, 64, 16
    pages, table, _values = made_cache(2, [60], nkv, hd, page)
    table[0, 1] = entry
    q = torch.randn(2, nq * hd).to(BF16).cuda()
    out = torch.full_like(q, math.nan)
    seq, pos = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.tensor([58, 59], dtype=torch.int32, device="cuda")
    if call == "exact":
        ops.paged_attention_int4(q, nq * hd, out, *pages, table, seq, pos, nq, nkv, hd, page, 0.125)
    elif call == "decode":
        run_decode(ops, q, nq * hd, out, pages, table, seq, pos, nq, nkv, hd, page, 0, 0.0, None, None, 60)
    else:
        run_portion(ops, q, out, pages, table, [2], [60], nq, nkv, hd, page)
    with pytest.raises(ops.KernelError, match="names no page"):
        ops.check_kernel_status()
    assert bool(out.isfinite().all())


@pytest.mark.parametrize("call", ["exact", "neighbours", "decode"])
@pytest.mark.parametrize("seq,pos", [(1, 5), (7, 5), (0, 64), (0, 2 ** 31 - 1), (0, -1)])
def test_a_row_whose_request_or_position_there_is_not_is_reported(ops, call, seq, pos):
    """Beside rows that are in order, which keep their results."""
    nq, nkv, hd, page = 4, 1, 64, 16
    pages, table, (k, v) = made_cache(2, [60], nkv, hd, page)
    q = torch.randn(3, nq * hd, generator=torch.Generator().manual_seed(3)).to(BF16)
    seqs, poss = torch.tensor([0, seq, 0], dtype=torch.int32), torch.tensor([40, pos, 59], dtype=torch.int32)
    out = torch.full((3, nq * hd), math.nan, dtype=BF16, device="cuda")
    if call == "decode":
        run_decode(ops, q.cuda(), nq * hd, out, pages, table, seqs.cuda(), poss.cuda(), nq, nkv, hd, page, 0, 0.0, None, None, 64)
    else:
        ops.paged_attention_int4(q.cuda(), nq * hd, out, *pages, table, seqs.cuda(), poss.cuda(), nq, nkv, hd, page, 0.125, neighbours=call == "neighbours")
    with pytest.raises(ops.KernelError, match="names no page|context bound"):
        ops.check_kernel_status()
    assert not bool(out[1].any())
    want, largest, value = plain.attention(q[::2].view(2, nq, hd), k, v, poss[::2], seqs[::2], hd ** -0.5)
    check_decode(out[::2].view(2, nq, hd), want, hd, largest, 60, value)


@pytest.mark.parametrize("start,length,held", [(9, 4, 30), (-1, 4, 30), (2 ** 31 - 2, 4, 30), (0, 31, 30)])
def test_portions_that_are_not_the_outputs_are_reported(ops, start, length, held):
    nq, nkv, hd, page = 4, 1, 64, 16
    pages, table, _values = made_cache(2, [30], nkv, hd, page)
    q = torch.randn(12, nq * hd).to(BF16).cuda()
    out = torch.full_like(q, 7.0)
    ints = lambda v: torch.tensor([v], dtype=torch.int32, device="cuda")  # noqa: E731
    scratch = torch.zeros(ops.prefill_int4_scratch_ints(1, 64, nkv, hd), dtype=torch.int32, device="cuda")
    ops.paged_attention_prefill_int4(q, nq * hd, out, *pages, table, ints(start), ints(length), ints(held), scratch, 1, 64, nq, nkv, hd, page, 0.125, 0)
    with pytest.raises(ops.KernelError, match="portions"):
        ops.check_kernel_status()
    assert bool((out == 7.0).all())


def test_empty_calls(ops):
    nq, nkv, hd, page = 4, 1, 64, 16
    pages, table, _values = made_cache(2, [10], nkv, hd, page)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    q = torch.empty(0, nq * hd, dtype=BF16, device="cuda")
    ops.paged_attention_int4(q, nq * hd, q, *pages, table, none, none, nq, nkv, hd, page, 0.125)
    run_decode(ops, q, nq * hd, q, pages, table, none, none, nq, nkv, hd, page, 0, 0.0, None, None, 10, torch.zeros(1, device="cuda"))
    run_portion(ops, q, q, pages, table, [], [], nq, nkv, hd, page)
    rows = torch.empty(0, 6 * hd, dtype=BF16, device="cuda")
    tables = torch.ones(4, hd // 2, device="cuda")
    ops.rope_kv_write_int4(rows, None, None, None, 0.0, none, none, tables, tables, *pages, nq, nkv, hd, page)
    ops.read_int4(*pages, none, torch.empty(0, nkv, hd, device="cuda"), torch.empty(0, nkv, hd, device="cuda"), nkv, hd, page)
    ops.copy_pages([pages[0][None]], [], [])
    ops.check_kernel_status()


# ---------------------------------------------------------------------------------------------------------- copies of pages
@pytest.mark.parametrize("dtype,shapes,copies", [
    (BF16, [(3, 9, 2, 16, 64), (3, 9, 2, 16, 64)], 4), (torch.uint8, [(2, 40, 8, 16, 80)] * 2, 17), (F32, [(1, 5, 1, 1, 3)], 2),
    (torch.uint8, [(2, 7, 3, 5, 7)], 3), (torch.uint8, [(1, 1100, 1, 4, 20)], 520), (BF16, [(i + 1, 6, 1, 8, 24) for i in range(11)], 2),
    (F32, [(2, 4, 8, 64, 128)], 1)])
def test_copies_of_pages(ops, dtype, shapes, copies):
    g = torch.Generator().manual_seed(copies)
    pools = [torch.randint(0, 250, s, generator=g).to(dtype) for s in shapes]
    order = torch.randperm(shapes[0][1], generator=g).tolist()
    src, dst = order[:copies], order[copies:2 * copies]
    if copies > 1:
        src[1] = src[0]                                     # one page may be copied to several places
    got = [p.cuda() for p in pools]
    ops.copy_pages(got, src, dst)
    for p, t in zip(pools, got):
        p[:, dst] = p[:, src].clone()
        assert torch.equal(t.cpu(), p)
    ops.copy_pages(got, torch.tensor(src), torch.tensor(dst))
    assert all(torch.equal(t.cpu(), p) for t, p in zip(got, pools))


def test_copies_far_into_a_large_pool(ops):
    """Offsets beyond 2^32 bytes."""
    pool = torch.zeros(2, 40, 1, 1 << 20, 64, dtype=torch.uint8, device="cuda")        # pages of 64 MB
    pool[:, 1] = 5
    pool[1, 2] = 7
    ops.copy_pages([pool], [1, 2], [39, 38])
    assert bool((pool[:, 39] == 5).all()) and bool((pool[1, 38] == 7).all()) and not bool(pool[0, 38].any()) and not bool(pool[:, 37].any())


# ------------------------------------------------------------------------------------------------------------------ together
def test_written_read_forked_and_replayed_from_a_graph(ops):
    """A prompt is written and attended to, its last page is copied to a second request, both go on token by token from a captured graph
    whose positions, slots and pages change between replays; eagerly the same, bit for bit, and near float64."""
    nq, nkv, hd, page, prompt, steps = 8, 2, 128, 16, 70, 4
    made = made_rows(3, prompt + 2 * steps, nq, nkv, hd, BF16, True, True, positions=256)
    made["positions"] = torch.cat([torch.arange(prompt), torch.arange(prompt, prompt + steps).repeat_interleave(2)]).int()
    d = on_gpu(made)
    pools = [torch.full((1, 12, nkv, page, 80), 255, dtype=torch.uint8, device="cuda") for _ in "kv"]
    pages = [p[0] for p in pools]
    table = torch.tensor([[3, 8, 1, 10, 5, -1], [3, 8, 1, 10, 6, -1]], dtype=torch.int32, device="cuda")
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731

    def slot(r, p):
        return int(table[r, p // page]) * page + p % page
    rows = d["rows"].clone()
    first = rows[:prompt]
    ops.rope_kv_write_int4(first, d["bias"], d["q_norm"], d["k_norm"], 1e-5, d["positions"][:prompt], ints([slot(0, p) for p in range(prompt)]), d["cos"],
                           d["sin"], *pages, nq, nkv, hd, page)
    out = torch.empty(prompt, nq * hd, dtype=BF16, device="cuda")
    scratch = torch.zeros(ops.prefill_int4_scratch_ints(1, prompt, nkv, hd), dtype=torch.int32, device="cuda")
    ops.paged_attention_prefill_int4(first, first.shape[1], out, *pages, table, ints([0]), ints([prompt]), ints([prompt]), scratch, 1, prompt, nq, nkv, hd, page,
                                     hd ** -0.5, 0)
    ops.copy_pages(pools, [5], [6])
    step_rows = torch.empty(2, rows.shape[1], dtype=BF16, device="cuda")
    position, slots, seq = ints([0, 0]), ints([-1, -1]), ints([0, 1])
    splits = torch.zeros(ops.decode_int4_scratch_floats(2, nq, nkv, hd, 96), device="cuda")
    step_out = torch.empty(2, nq * hd, dtype=BF16, device="cuda")

    def step():
        ops.rope_kv_write_int4(step_rows, d["bias"], d["q_norm"], d["k_norm"], 1e-5, position, slots, d["cos"], d["sin"], *pages, nq, nkv, hd, page)
        ops.paged_attention_decode_int4(step_rows, step_rows.shape[1], step_out, *pages, table, seq, position, splits, nq, nkv, hd, page, hd ** -0.5, 0, 96)

    def all_steps(call):
        results = []
        for i in range(steps):
            step_rows.copy_(rows[prompt + 2 * i:prompt + 2 * i + 2])
            position.fill_(prompt + i)
            slots.copy_(ints([slot(0, prompt + i), slot(1, prompt + i)]))
            call()
            results.append(step_out.clone())
        return torch.stack(results)
    eager = all_steps(step)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step_rows.copy_(rows[prompt:prompt + 2])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
        replayed = all_steps(graph.replay)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(eager, replayed)
    q, k, v = plain.prepare_heads(made["rows"], made["bias"], made["q_norm"], made["k_norm"], 1e-5, made["positions"], made["cos"], made["sin"], nq, nkv, hd)
    stored = [[plain.unpack(w, p.cpu()[table[r, :5].long().cpu()].transpose(1, 2).reshape(-1, nkv, 80)[:prompt + steps], hd) for r in (0, 1)]
              for w, p in zip("kv", pages)]
    for which, want in ((0, k), (1, v)):                    # both requests share the prompt; their own tokens differ
        assert torch.equal(stored[which][0][:prompt], stored[which][1][:prompt])
        for r in (0, 1):
            mine = torch.cat([want[:prompt], want[prompt + r::2]])
            step_size = (mine.amax(-1, keepdim=True) - mine.amin(-1, keepdim=True)) / 15
            assert bool(((stored[which][r] - mine).abs() <= 0.6 * step_size + 0.01 * mine.abs().amax()).all())
    q16 = q.to(BF16)
    seqs = torch.cat([torch.zeros(prompt), torch.tensor([0, 1]).repeat(steps)]).int()
    want, largest, value = plain.attention(q16, stored[0], stored[1], made["positions"], seqs, hd ** -0.5)
    got = torch.cat([out, eager.reshape(-1, nq * hd)]).view(-1, nq, hd).double().cpu()
    assert float((got - want).norm() / want.norm()) < 2.0 ** -7        # queries in bfloat16 may differ by their last bit
    ops.check_kernel_status()


def test_on_a_stream_of_its_own(ops):
    nq, nkv, hd, page = 8, 2, 128, 16
    pages, table, (k, v) = made_cache(2, [200], nkv, hd, page)
    q = torch.randn(1, nq * hd, generator=torch.Generator().manual_seed(1)).to(BF16)
    pos, seq = torch.tensor([199], dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = torch.empty(1, nq * hd, dtype=BF16, device="cuda")
        run_decode(ops, q.cuda(), nq * hd, out, pages, table, seq.cuda(), pos.cuda(), nq, nkv, hd, page, 0, 0.0, None, None, 200)
    side.synchronize()
    want, largest, value = plain.attention(q.view(1, nq, hd), k, v, pos, seq, hd ** -0.5)
    check_decode(out.view(1, nq, hd), want, hd, largest, 200, value)
