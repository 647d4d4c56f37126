"""Operators for rows that bring several sequences their next tokens: head norms with rotation, the append to a paged cache, and
attention over it - each against the definition in 64 bits where lengths, pages, masks, alignments and values can go wrong."""
import math

import pytest
import torch

from portion_helpers import Cache, attend_all, attend_tolerance, row_table, turn

pytestmark = pytest.mark.gpu
EPS = 1e-6


def rnd(shape, dtype, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (scale * torch.randn(shape, generator=g, device="cuda")).to(dtype)


def freqs(rot, theta=1e4):
    return theta ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot) if rot else None


def weights(d, dtype, norm):
    return (1 + rnd((d,), dtype, 7, 0.2), 1 - rnd((d,), dtype, 8, 0.2)) if norm else (None, None)


def check_turn(out, ref):
    """One rounding of the type, and fp32 arithmetic: a norm's sum and the two products of a pair, whose terms are as large as the
    head's largest element; 2^-20 covers both (the sum of 256 squares is off by 2^-21 at most in pairs of chains)."""
    err = (out.double() - ref).abs()
    half = torch.finfo(out.dtype).eps / 2
    small = torch.finfo(out.dtype).smallest_normal * torch.finfo(out.dtype).eps
    assert (err <= ref.abs() * half * (1 + 2.0 ** -10) + ref.abs().amax(-1, keepdim=True) * 2.0 ** -20 + small).all(), err.max()


# ---- norm and rotation ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d,rot", [(128, 128), (128, 64), (64, 64), (80, 40), (96, 96), (256, 256), (256, 32), (20, 6), (33, 32), (8, 8),
                                   (2, 2), (128, 0)])
def test_turn(dtype, d, rot):
    from axono_b200 import ops

    for rows, hq, hkv, interleaved, norm in ((1, 4, 2, False, True), (37, 5, 1, True, False), (70, 24, 3, False, True), (3, 1, 1, True, True)):
        qkv = rnd((rows, (hq + 2 * hkv) * d), dtype, rows)
        q, k = qkv[:, :hq * d].view(rows, hq, d), qkv[:, hq * d:(hq + hkv) * d].view(rows, hkv, d)
        pos = torch.randint(0, 200000, (rows,), generator=torch.Generator().manual_seed(rows)).cuda()
        wq, wk = weights(d, dtype, norm)
        before = qkv.clone()
        oq, ok = ops.qk_norm_rope(q, k, pos if rot else None, freqs(rot), wq, wk, EPS, interleaved=interleaved, factor=1.25)
        assert torch.equal(qkv, before) and oq.is_contiguous() and ok.is_contiguous()
        check_turn(oq, turn(q, wq, EPS, pos, freqs(rot), interleaved, 1.25))
        check_turn(ok, turn(k, wk, EPS, pos, freqs(rot), interleaved, 1.25))
    assert ops.last_error() == 0


def test_turn_on_three_axes_and_far_positions():
    from axono_b200 import ops

    rows, section = 40, (24, 20, 20)
    for rot, far in ((128, 1 << 20), (64, (1 << 31) - 1), (128, 1 << 40)):
        q, k = rnd((rows, 4, 128), torch.float32, 1), rnd((rows, 2, 128), torch.float32, 2)
        pos = torch.randint(0, far, (3, rows), generator=torch.Generator().manual_seed(3)).cuda()
        pos[:, 0] = 0
        if far >= 1 << 40:
            pos = pos[:, :1]  # an angle in double is off by 2^-13 of a radian at 2^40: only the origin is exact
            q, k = q[:1], k[:1]
        oq, ok = ops.qk_norm_rope(q, k, pos, freqs(rot), eps=EPS, mrope_section=section)
        slack = 2.0 ** -52 * far * 4  # of the angle, in double
        for out, x in ((oq, q), (ok, k)):
            ref = turn(x, None, EPS, pos, freqs(rot), section=section)
            err = (out.double() - ref).abs()
            assert (err <= ref.abs() * 2.0 ** -23 + ref.abs().amax(-1, keepdim=True) * (2.0 ** -20 + (slack if far < 1 << 40 else 0))).all()


def test_turn_takes_any_alignment_and_one_of_the_two():
    from axono_b200 import ops

    buf = rnd((9 * 6 * 64 + 1,), torch.float16)
    q = buf[1:].view(9, 6, 64)  # two bytes off
    pos = torch.arange(9, device="cuda")
    oq, none = ops.qk_norm_rope(q, None, pos, freqs(64), interleaved=True)
    assert none is None
    check_turn(oq, turn(q, None, EPS, pos, freqs(64), True))
    none, ok = ops.qk_norm_rope(None, q.transpose(0, 1).contiguous().transpose(0, 1), pos, freqs(64))  # heads outermost: copied
    assert none is None
    check_turn(ok, turn(q, None, EPS, pos, freqs(64)))
    wide = rnd((9, 400), torch.float32)
    view = wide[:, 3:3 + 5 * 64].view(9, 5, 64)  # rows of 400, 12 bytes off
    check_turn(ops.qk_norm_rope(view, None, pos, freqs(32))[0], turn(view, None, EPS, pos, freqs(32)))


def test_turn_keeps_infinities_and_nan_in_their_heads():
    from axono_b200 import ops

    q = rnd((5, 4, 128), torch.float16)
    q[1, 2, 5], q[3, 0, 0] = math.nan, math.inf
    w = torch.ones(128, dtype=torch.float16, device="cuda")
    out, _ = ops.qk_norm_rope(q, None, torch.arange(5, device="cuda"), freqs(128), w)
    bad = ~torch.isfinite(out).all(-1)
    expect = torch.zeros((5, 4), dtype=torch.bool, device="cuda")
    expect[1, 2] = expect[3, 0] = True
    assert torch.equal(bad, expect)


# ---- append -----------------------------------------------------------------------------------------------------------

PORTIONS = [((1,), (0,)), ((3, 0, 5, 1), (62, 10, 0, 127)), ((130, 64, 1), (1, 64, 500)), ((0, 0, 7, 0), (5, 0, 63, 9)),
            (tuple(i % 4 for i in range(300)), tuple(i % 7 for i in range(300)))]


@pytest.mark.parametrize("dtype,d,rot,hq,hkv,page", [(torch.float16, 128, 128, 16, 8, 64), (torch.float32, 64, 32, 3, 1, 128),
                                                     (torch.float16, 80, 80, 6, 2, 64), (torch.float32, 36, 6, 2, 2, 64),
                                                     (torch.float16, 256, 0, 2, 1, 192)])
@pytest.mark.parametrize("counts,cached", PORTIONS)
@pytest.mark.parametrize("advance", [True, False])
def test_append(dtype, d, rot, hq, hkv, page, counts, cached, advance):
    from axono_b200 import ops

    lens = [n + c for n, c in zip(counts, cached)]
    cache = Cache(lens, hkv, d, dtype, page)
    starts, rows = row_table(counts, first=2), sum(counts) + 5  # rows of no sequence before and behind
    qkv = rnd((rows, (hq + 2 * hkv) * d + 8), dtype, 11)[:, :(hq + 2 * hkv) * d]
    wq, wk = weights(d, dtype, rot != 6)
    axes = rot == 128
    pos = torch.randint(0, 40000, (3, rows), generator=torch.Generator().manual_seed(5)).cuda() if axes else None
    section = (24, 20, 20) if axes else None
    before = torch.tensor(cached if advance else lens, dtype=torch.int32, device="cuda")
    lengths, k0, v0 = before.clone(), cache.k_pages.clone(), cache.v_pages.clone()
    out = torch.full((rows, hq, d), 7.0, dtype=dtype, device="cuda")
    got = ops.qkv_norm_rope_append_portions(qkv, hq, wq, wk, EPS, cache.k_pages, cache.v_pages, cache.table, lengths, starts, pos=pos,
                                            inv_freq=freqs(rot), interleaved=rot == 32, factor=0.75, mrope_section=section,
                                            advance=advance, out=out)
    assert got is out and ops.last_error() == 0
    assert lengths.tolist() == lens
    assert (out[:2] == 7).all() and (out[rows - 3:] == 7).all()
    touched = torch.zeros(k0.shape[:3], dtype=torch.bool, device="cuda")
    at = 2
    for b, (n, c) in enumerate(zip(counts, cached)):
        if not n:
            continue
        r = slice(at, at + n)
        at += n
        where = torch.arange(c, c + n, device="cuda") if pos is None else pos[:, r]
        q, k, v = qkv[r].split([hq * d, hkv * d, hkv * d], 1)
        check_turn(out[r], turn(q.reshape(n, hq, d), wq, EPS, where, freqs(rot), rot == 32, 0.75, section))
        keys, values = cache.read(b, c, n)
        check_turn(keys, turn(k.reshape(n, hkv, d), wk, EPS, where, freqs(rot), rot == 32, 0.75, section))
        assert torch.equal(values, v.reshape(n, hkv, d))
        page_, place = cache.place(b, c, n)
        touched[page_, :, place] = True
    same = lambda a, b: torch.equal(a[~touched].view(torch.uint8), b[~touched].view(torch.uint8))  # noqa: E731  (NaN equals itself)
    assert same(cache.k_pages, k0) and same(cache.v_pages, v0)


def test_append_of_one_token_each_gives_the_keys_of_the_single_token_operator():
    """Near the beginning, where a product of position and frequency in fp32 is exact enough: norms and rotation agree to the
    roundings of the single-token form (which also rounds between norm and rotation)."""
    from axono_b200 import ops

    batch, hq, hkv, d = 5, 8, 4, 128
    qkv, (wq, wk) = rnd((batch, (hq + 2 * hkv) * d), torch.float16, 3), weights(d, torch.float16, True)
    caches = [Cache([40 + b for b in range(batch)], hkv, d, torch.float16, more=1) for _ in range(2)]
    q1 = ops.qkv_norm_rope_append(qkv, hq, wq, wk, EPS, caches[0].k_pages, caches[0].v_pages, caches[0].table, caches[0].lens, theta=1e4)
    q2 = ops.qkv_norm_rope_append_portions(qkv, hq, wq, wk, EPS, caches[1].k_pages, caches[1].v_pages, caches[1].table, caches[1].lens,
                                           row_table([1] * batch), inv_freq=freqs(128))
    assert torch.equal(caches[0].lens, caches[1].lens)
    for b in range(batch):
        (k1, v1), (k2, v2) = (c.read(b, 40 + b, 1) for c in caches)
        assert torch.equal(v1, v2)
        assert (k1.double() - k2.double()).abs().max() <= 2.0 ** -9 * k1.abs().max()
    assert (q1.double() - q2.double()).abs().max() <= 2.0 ** -9 * q1.abs().max()


def test_append_reports_what_does_not_fit_and_bad_tables():
    from axono_b200 import _capi, ops

    hq, hkv, d = 2, 1, 64
    cache = Cache([60, 60, 60], hkv, d, torch.float16, more=4)  # one page each: room for 4
    lens0, k0 = cache.lens.clone(), cache.k_pages.clone()
    qkv = rnd((12, (hq + 2 * hkv) * d), torch.float16)
    run = lambda starts, table=None: ops.qkv_norm_rope_append_portions(  # noqa: E731
        qkv, hq, None, None, EPS, cache.k_pages, cache.v_pages, cache.table if table is None else table, cache.lens, starts,
        inv_freq=freqs(64), out=torch.zeros((12, hq, d), dtype=torch.float16, device="cuda"))
    q = run(row_table([4, 5, 3]))  # the second does not fit
    assert ops.last_error() == 4
    assert cache.lens.tolist() == [64, 60, 63]
    assert torch.isnan(cache.read(1, 60, 4)[0]).all() and torch.isfinite(cache.read(0, 60, 4)[0]).all()
    check_turn(q[4:9], turn(qkv[4:9, :hq * d].reshape(5, hq, d), None, EPS, torch.arange(60, 65, device="cuda"), freqs(64)))
    cache.lens.copy_(lens0)
    cache.k_pages.copy_(k0)
    bad = cache.table.clone()
    bad[2, 0] = cache.k_pages.shape[0]
    bad[0, 0] = -1
    run(row_table([1, 1, 1]), bad)
    assert ops.last_error() == 2
    assert cache.lens.tolist() == [60, 61, 60]
    cache.lens.copy_(lens0)
    run(torch.tensor([0, 2, 1, 3], dtype=torch.int32, device="cuda"))  # falls
    assert ops.last_error() & 16
    cache.lens.copy_(lens0)
    run(torch.tensor([0, 2, 4, 13], dtype=torch.int32, device="cuda"))  # passes the rows
    assert ops.last_error() & 16
    assert cache.lens.tolist() == [62, 62, 60]
    cache.lens.copy_(torch.tensor([1, 60, 60]))
    cache.lens[0] = 1
    ops.qkv_norm_rope_append_portions(qkv, hq, None, None, EPS, cache.k_pages, cache.v_pages, cache.table, cache.lens, row_table([3, 0, 0]),
                                      advance=False)  # a length that cannot count three rows
    assert ops.last_error() == 4
    assert _capi.lib().axb200_last_error() == 0


# ---- attention --------------------------------------------------------------------------------------------------------

def run_attention(counts, cached, hq, hkv, d, dtype, page=64, window=0, seed=0, spread=1.0, first=0, behind=0, bound=None, cache=None):
    from axono_b200 import ops

    lens = [n + c for n, c in zip(counts, cached)]
    cache = cache or Cache(lens, hkv, d, dtype, page, seed)
    starts = row_table(counts, first)
    rows = sum(counts) + first + behind
    q = rnd((rows, hq, d), dtype, seed + 1, spread)
    out = torch.full_like(q, 7.0)
    got = ops.gqa_attention_portions_paged(q, cache.k_pages, cache.v_pages, cache.table, cache.lens, starts, bound or max(max(lens), 1),
                                           window=window, out=out)
    assert got is out
    assert (out[:first] == 7).all() and (out[rows - behind:] == 7).all()
    return q, cache, starts.tolist(), out


def check_attention(q, cache, counts, starts, out, window=0):
    for rows, ref, mag, top in attend_all(q, cache, counts, starts, window):
        err = (out[rows].double() - ref).abs()
        tol = attend_tolerance(q.dtype, ref, mag, top)
        assert (err <= tol).all(), (float(err.max()), float((err / tol.clamp_min(1e-30)).max()))


SHAPES = [(16, 8, 128), (4, 4, 64), (12, 4, 80), (8, 1, 96), (6, 2, 40), (7, 1, 128), (2, 2, 8), (3, 1, 72), (32, 1, 64)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
@pytest.mark.parametrize("counts,cached", [((1,), (0,)), ((1, 5, 0, 2), (63, 64, 3, 1)), ((130, 64, 1), (1, 0, 500)), ((257,), (0,)),
                                           ((40, 3), (1000, 127))])
def test_attention(dtype, hq, hkv, d, counts, cached):
    from axono_b200 import ops

    for window in (0, 1, 70):
        q, cache, starts, out = run_attention(counts, cached, hq, hkv, d, dtype, window=window, first=1, behind=3)
        check_attention(q, cache, counts, starts, out, window)
    assert ops.last_error() == 0


@pytest.mark.parametrize("hq,hkv,d,page", [(4, 2, 20, 64), (4, 4, 256, 128), (2, 1, 136, 64), (130, 1, 64, 64), (260, 2, 16, 64), (3, 1, 33, 192)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_attention_of_unusual_heads(dtype, hq, hkv, d, page):
    counts, cached = (5, 0, 70), (100, 3, 0)
    q, cache, starts, out = run_attention(counts, cached, hq, hkv, d, dtype, page, spread=3.0)
    check_attention(q, cache, counts, starts, out)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_attention_over_long_caches(dtype):
    """Few rows over many keys, divided among CTAs and joined, and a loose bound of the lengths."""
    counts, cached = (2, 1, 17), (9000, 5000, 70)
    for window, bound in ((0, None), (0, 20000), (4097, None), (130, None)):
        q, cache, starts, out = run_attention(counts, cached, 8, 2, 128, dtype, window=window, spread=2.0, bound=bound, first=2, behind=1)
        check_attention(q, cache, counts, starts, out, window)


def test_attention_of_a_long_prompt():
    counts, cached = (1111, 700), (0, 1500)
    for dtype in (torch.float16, torch.float32):
        q, cache, starts, out = run_attention(counts, cached, 4, 2, 128, dtype)
        check_attention(q, cache, counts, starts, out)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_ignores_values_that_a_row_cannot_see(dtype, d):
    """Infinities and NaN in keys and values of later tokens and before a window touch only the rows that see them; stale bytes
    behind a sequence's end are NaN in every test here."""
    from axono_b200 import ops

    counts, cached, window = (90, 4), (50, 300), 60
    lens = [n + c for n, c in zip(counts, cached)]
    for bad in (math.inf, math.nan):
        cache = Cache(lens, 2, d, dtype)
        for b, at in ((0, 100), (1, 301), (1, 200)):
            cache.v[b][at, 1, 3] = bad
            if bad != bad:
                cache.k[b][at, 0, 2] = bad
            cache.write(b, 0, cache.k[b], cache.v[b])
        q, cache, starts, out = run_attention(counts, cached, 4, 2, d, dtype, window=window, cache=cache)
        for b, (n, c) in enumerate(zip(counts, cached)):
            pos = torch.arange(c, c + n, device="cuda")
            hit = torch.zeros(n, dtype=torch.bool, device="cuda")
            for bb, at in ((0, 100), (1, 301), (1, 200)):
                if bb == b:
                    hit |= (pos >= at) & (pos < at + window)
            rows = out[starts[b]:starts[b] + n]
            assert torch.isfinite(rows[~hit]).all()
            v_bad = rows[:, 2:, 3]  # heads of KV head 1, the element
            assert (v_bad[hit] == bad).all() if bad == math.inf else torch.isnan(v_bad[hit]).all()
            others = torch.ones(d, dtype=torch.bool, device="cuda")
            others[3] = False
            assert torch.isfinite(rows[:, 2:][..., others]).all()
            assert torch.isfinite(rows[:, :2]).all() if bad == math.inf else torch.isnan(rows[:, :2][hit]).all()
        clean = [cache.v[b].clone() for b in range(2)]
        for b in range(2):
            clean[b][~torch.isfinite(clean[b])] = 0
            cache.k[b][~torch.isfinite(cache.k[b])] = 0
        cache.v = clean
        for rows, ref, mag, top in attend_all(q, cache, counts, starts, window):
            b = 0 if rows.start == starts[0] else 1
            pos = torch.arange(cached[b], cached[b] + counts[b], device="cuda")
            hit = torch.zeros(counts[b], dtype=torch.bool, device="cuda")
            for bb, at in ((0, 100), (1, 301), (1, 200)):
                if bb == b:
                    hit |= (pos >= at) & (pos < at + window)
            err = (out[rows].double() - ref).abs()[~hit]
            assert (err <= attend_tolerance(dtype, ref, mag, top)[~hit]).all()
    assert ops.last_error() == 0


def test_attention_with_sharp_and_extreme_scores():
    """Scores up to the largest that fp16 inputs reach, one key that carries all the weight, and equal scores."""
    from axono_b200 import ops

    for dtype in (torch.float16, torch.float32):
        for spread in (60.0, 2000.0, 0.0):
            counts, cached = (65, 2), (10, 700)
            q, cache, starts, out = run_attention(counts, cached, 4, 2, 64, dtype, spread=spread)
            check_attention(q, cache, counts, starts, out)
    assert ops.last_error() == 0


def test_attention_reports_lengths_and_tables_that_are_wrong():
    from axono_b200 import ops

    cache = Cache([200, 100], 2, 64, torch.float16, poison=0.0)
    q = rnd((8, 4, 64), torch.float16)
    run = lambda starts, lens=None, table=None, bound=200: ops.gqa_attention_portions_paged(  # noqa: E731
        q, cache.k_pages, cache.v_pages, cache.table if table is None else table, cache.lens if lens is None else lens, starts, bound,
        out=torch.full_like(q, 7.0))
    good = run(row_table([4, 4]))
    assert ops.last_error() == 0
    out = run(row_table([4, 4]), bound=128)  # the first sequence is longer than the bound: its first 128 keys
    # The bound sizes the launch and so decides how keys are divided; a row whose keys are added up in another order is rounded otherwise:
    # with S the sum over keys before the last rounding and |S - exact| <= e for either division (what attend_tolerance counts beside that
    # rounding), the two may differ by 2e and land in neighbouring halves, but each is as near to the definition as any result.
    rows, ref, mag, top = attend_all(q, cache, (4, 4), [0, 4, 8])[1]
    for o in (out, good):
        assert ((o[rows].double() - ref).abs() <= attend_tolerance(torch.float16, ref, mag, top)).all()
    assert ops.last_error() == 4 and torch.isfinite(out).all()
    table = cache.table.clone()
    table[0, 1] = -5
    out = run(row_table([4, 4]), table=table)
    assert ops.last_error() == 2 and torch.isfinite(out).all() and torch.equal(out[4:], good[4:])
    out = run(torch.tensor([0, 4, 9], dtype=torch.int32, device="cuda"))
    assert ops.last_error() == 16 and torch.equal(out[:4], good[:4]) and (out[4:] == 7).all()
    out = run(row_table([4, 4]), lens=torch.tensor([200, 2], dtype=torch.int32, device="cuda"))  # two of the rows stand before the sequence
    assert ops.last_error() == 0 and (out[4:6] == 0).all() and torch.isfinite(out).all() and not (out[6:] == 0).all()
    out = run(row_table([4, 4]), lens=torch.tensor([200, 0], dtype=torch.int32, device="cuda"))
    assert ops.last_error() == 0 and (out[4:] == 0).all()


def test_attention_beyond_32_bits_of_a_pool():
    """Pages at the end of pools of more than 2^31 elements."""
    from axono_b200 import ops

    hkv, d, page, lens = 8, 128, 64, [150, 90]
    pages = (1 << 31) // (hkv * d * page) + 40
    small = Cache(lens, hkv, d, torch.float16)
    big = [torch.empty((pages, hkv, page, d), dtype=torch.float16, device="cuda") for _ in range(2)]
    shift = pages - small.k_pages.shape[0]
    for pool, src in zip(big, (small.k_pages, small.v_pages)):
        pool[shift:] = src
    small.k_pages, small.v_pages, small.table = *big, torch.where(small.table < src.shape[0], small.table + shift, pages + 1).to(torch.int32)
    counts = (20, 90)
    q, cache, starts, out = run_attention(counts, (130, 0), 16, hkv, d, torch.float16, cache=small)
    check_attention(q, cache, counts, starts, out)
    # and appended there
    qkv, lengths = rnd((110, 32 * d), torch.float16, 5), small.lens.clone()
    ops.qkv_norm_rope_append_portions(qkv, 16, None, None, EPS, *big, small.table, lengths, row_table(counts), advance=False)
    for b, (r0, n, c) in enumerate(((0, 20, 130), (20, 90, 0))):
        k, v = small.read(b, c, n)
        assert torch.equal(k.reshape(n, -1), qkv[r0:r0 + n, 16 * d:24 * d]) and torch.equal(v.reshape(n, -1), qkv[r0:r0 + n, 24 * d:])
    assert ops.last_error() == 0


def test_other_streams_graphs_and_two_calls_at_once():
    """A captured pair of append and attention follows lengths and row tables that change between replays, and gives what eager
    calls on two streams at once give."""
    from axono_b200 import ops

    hq, hkv, d, rows = 8, 2, 128, 40
    cache = Cache([700, 300, 90], hkv, d, torch.float16, more=40, poison=0.0)
    lens0 = cache.lens.clone()
    qkv = rnd((rows, (hq + 2 * hkv) * d), torch.float16, 3)
    starts = row_table([10, 20, 10])
    out = torch.zeros((rows, hq, d), dtype=torch.float16, device="cuda")

    def step(lens, starts, out, k=None, v=None):
        k, v = (cache.k_pages, cache.v_pages) if k is None else (k, v)
        q = ops.qkv_norm_rope_append_portions(qkv, hq, None, None, EPS, k, v, cache.table, lens, starts, inv_freq=freqs(128))
        return ops.gqa_attention_portions_paged(q, k, v, cache.table, lens, starts, 800, out=out)

    def eager(counts):
        lens, k, v = lens0.clone(), cache.k_pages.clone(), cache.v_pages.clone()
        return step(lens, row_table(counts), torch.zeros_like(out), k, v).clone(), lens

    first, lens1 = eager([10, 20, 10])
    second, lens2 = eager([1, 0, 33])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    lens = lens0.clone()
    with torch.cuda.stream(side):
        step(lens, starts, out)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(lens, starts, out)
    for counts, expect, after in (([10, 20, 10], first, lens1), ([1, 0, 33], second, lens2), ([10, 20, 10], first, lens1)):
        lens.copy_(lens0)
        starts.copy_(row_table(counts))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, expect) and torch.equal(lens, after)
    # two streams at once, each with its own outputs
    streams, outs = [torch.cuda.Stream() for _ in range(2)], [torch.zeros_like(out) for _ in range(2)]
    caches = [(cache.k_pages.clone(), cache.v_pages.clone()) for _ in range(2)]
    tables = [row_table([10, 20, 10]), row_table([1, 0, 33])]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, o, t, (k, v) in zip(streams, outs, tables, caches):
            with torch.cuda.stream(s):
                step(lens0.clone(), t, o, k, v)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], first) and torch.equal(outs[1], second)
    assert ops.last_error() == 0


def test_turn_in_place():
    """Through the C ABI, whose outputs may be its inputs where rows are contiguous."""
    from axono_b200 import _capi, ops

    for dtype, d, rot, interleaved in ((torch.float16, 128, 128, False), (torch.float32, 80, 40, True), (torch.float16, 20, 20, False)):
        q, k, w = rnd((300, 6, d), dtype, 1), rnd((300, 2, d), dtype, 2), 1 + rnd((d,), dtype, 3, 0.1)
        pos, f = torch.arange(300, device="cuda") * 7, freqs(rot)
        oq, ok = ops.qk_norm_rope(q, k, pos, f, w, w, EPS, interleaved)
        code = _capi.FLOAT16 if dtype == torch.float16 else _capi.FLOAT32
        assert _capi.lib().axb200_qk_norm_rope(q.data_ptr(), 6 * d, k.data_ptr(), 2 * d, w.data_ptr(), w.data_ptr(), EPS, pos.data_ptr(),
                                               f.data_ptr(), rot, int(interleaved), 1.0, 0, 0, 0, q.data_ptr(), k.data_ptr(), 300, 6, 2, d,
                                               code, torch.cuda.current_stream().cuda_stream) == 0
        assert torch.equal(q, oq) and torch.equal(k, ok)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_attention_of_many_sequences(dtype):
    """More sequences than a CTA has threads, most of them with nothing new, some long."""
    from axono_b200 import ops

    g = torch.Generator().manual_seed(3)
    for batch, most in ((500, 2), (900, 1)):
        counts = [int(n) if i % 5 else 0 for i, n in enumerate(torch.randint(0, most + 1, (batch,), generator=g))]
        cached = [int(n) for n in torch.randint(0, 90, (batch,), generator=g)]
        cached[7], cached[batch - 2], counts[batch - 2] = 3000, 2000, 1
        q, cache, starts, out = run_attention(counts, cached, 4, 2, 64, dtype, first=2, behind=2)
        check_attention(q, cache, counts, starts, out)
    counts, cached = [0] * 400, [1] * 400
    counts[350], cached[350] = 3, 4000
    q, cache, starts, out = run_attention(counts, cached, 4, 2, 128, dtype)
    check_attention(q, cache, counts, starts, out)
    assert ops.last_error() == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_attention_takes_any_alignment(dtype):
    """Queries and outputs that start off 16 bytes go through the FMA kernel, long caches in parts."""
    from axono_b200 import ops

    counts, lens = (3, 40), (2500, 60)
    cache, starts = Cache(lens, 2, 64, dtype), row_table(counts)
    q = rnd((43, 4, 64), dtype, 5)
    buf, obuf = torch.empty(q.numel() + 1, dtype=dtype, device="cuda"), torch.empty(q.numel() + 1, dtype=dtype, device="cuda")
    shifted, out = buf[1:].view(q.shape), obuf[1:].view(q.shape)
    shifted.copy_(q)
    for a, b in ((shifted, None), (q, out), (shifted, out)):
        got = ops.gqa_attention_portions_paged(a, cache.k_pages, cache.v_pages, cache.table, cache.lens, starts, 2500, out=b)
        check_attention(q, cache, counts, starts.tolist(), got)
    assert ops.last_error() == 0
    with pytest.raises(RuntimeError):
        ops.gqa_attention_portions_paged(q, cache.k_pages, cache.v_pages, cache.table, cache.lens, starts, 2500, out=q)


@pytest.mark.parametrize("what,scale", [("v", 1e-36), ("k", 1e-36), ("q", 1e-34), ("v", 1e36), ("v", 0.0)])
def test_fp32_attention_of_values_without_exact_parts(what, scale):
    """Values below 2^-100, whose lower bf16 parts would be subnormal, and large ones; a single such value is enough."""
    from axono_b200 import ops

    counts, lens = (70, 2), (300, 2500)
    cache, starts = Cache(lens, 2, 64, torch.float32), row_table(counts)
    q = rnd((72, 4, 64), torch.float32, 5)
    for some in (True, False):
        for b, n in enumerate(lens):
            at = slice(n // 3, n // 3 + 1) if some else slice(0, n)
            x = {"k": cache.k, "v": cache.v, "q": cache.k}[what][b]
            if what != "q":
                x[at] *= scale
                cache.write(b, 0, cache.k[b], cache.v[b])
        if what == "q":
            q[1 if some else slice(None)] *= scale
        out = ops.gqa_attention_portions_paged(q, cache.k_pages, cache.v_pages, cache.table, cache.lens, starts, 2500)
        for rows, ref, mag, top in attend_all(q, cache, counts, starts.tolist()):
            err = (out[rows].double() - ref).abs()
            tol = attend_tolerance(torch.float32, ref, mag, top) + 2.0 ** -149  # a subnormal result's own step
            # (1e36 twice is infinite: that key's value, and every result it joins)
            assert ((err <= tol) | (out[rows].double() == ref)).all(), (some, float((err / tol).max()))
    assert ops.last_error() == 0


def test_a_replayed_step_follows_the_growing_cache():
    """Single tokens as portions, captured once: every replay appends behind what the last one left, over the edges of tiles and pages,
    with the bits of eager calls."""
    from axono_b200 import ops

    hq, hkv, d, steps = 4, 2, 64, 70
    for lens, bound in (((30, 100, 0), 256), ((60, 4000, 900), 4200)):  # clusters, and parts
        caches = [Cache(lens, hkv, d, torch.float16, more=steps, poison=0.0) for _ in range(2)]
        starts, f = row_table([1, 1, 1]), freqs(d)
        qkv = torch.empty((3, (hq + 2 * hkv) * d), dtype=torch.float16, device="cuda")
        out = torch.empty((3, hq, d), dtype=torch.float16, device="cuda")

        def step(c, out=None):
            q = ops.qkv_norm_rope_append_portions(qkv, hq, None, None, EPS, c.k_pages, c.v_pages, c.table, c.lens, starts, inv_freq=f)
            return ops.gqa_attention_portions_paged(q, c.k_pages, c.v_pages, c.table, c.lens, starts, bound, out=out)

        qkv.zero_()
        first = caches[0].lens.clone()
        step(caches[0], out)  # once before the capture, taken back
        caches[0].lens.copy_(first)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(caches[0], out)
        for i in range(steps):
            qkv.copy_(rnd(qkv.shape, torch.float16, i))
            graph.replay()
            assert torch.equal(out, step(caches[1])), i
        assert caches[0].lens.tolist() == [n + steps for n in lens] and torch.equal(caches[0].lens, caches[1].lens)
        assert torch.equal(caches[0].k_pages, caches[1].k_pages) and torch.equal(caches[0].v_pages, caches[1].v_pages)
        for b in range(3):
            caches[1].k[b], caches[1].v[b] = caches[1].read(b, 0, lens[b] + steps)
        q = ops.qk_norm_rope(qkv[:, :hq * d].view(3, hq, d), None, caches[1].lens.long() - 1, f)[0]
        check_attention(q, caches[1], (1, 1, 1), [0, 1, 2, 3], out)
    assert ops.last_error() == 0


# ---- in the tower ---------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("use_mrope,qk_norm,dtype", [(True, True, torch.float16), (False, False, torch.float16), (False, True, torch.float32)])
def test_tower_extends_in_any_portions_as_it_decodes(use_mrope, qk_norm, dtype):
    """Prompts at once, in portions (some sequences pausing), and token by token through `decode_step` leave the same cache and logits
    but for roundings, and decoding goes on from any of them."""
    from axono_b200 import ops
    from axono_b200.decode import TextTower, TextTowerConfig

    cfg = TextTowerConfig(hidden=256, intermediate=512, n_q_heads=8, n_kv_heads=4, head_dim=64, vocab=1000, n_layers=3, use_mrope=use_mrope,
                          mrope_section=(12, 10, 10), qk_norm=qk_norm)
    g = torch.Generator().manual_seed(4)
    prompts = [torch.randint(0, 1000, (n,), generator=g) for n in (70, 3, 129)]
    tower = lambda batch=3: TextTower(cfg, batch, 320, dtype=dtype, seed=3)  # noqa: E731

    whole = tower()
    whole.extend(torch.cat(prompts), [70, 3, 129])
    parts = tower()
    done = [0, 0, 0]
    for counts in ([64, 1, 0], [0, 2, 100], [5, 0, 28], [1, 0, 1]):
        ids = torch.cat([p[a:a + n] for p, a, n in zip(prompts, done, counts)])
        parts.extend(ids, counts)
        done = [a + n for a, n in zip(done, counts)]
    assert parts.cache.seq_lens.tolist() == whole.cache.seq_lens.tolist() == [70, 3, 129]
    assert torch.equal(parts.pos3, whole.pos3) and whole.pos3[0].tolist() == [70, 3, 129]
    tol = 3e-2 if dtype == torch.float16 else 1e-3
    close = lambda a, b: (a.double() - b.double()).abs().max() <= tol * b.abs().max()  # noqa: E731
    for layer in range(cfg.n_layers):
        for b in range(3):
            for a, c in zip(parts.cache.gather(layer, b), whole.cache.gather(layer, b)):
                assert close(a, c)
    logits = []
    for b, prompt in enumerate(prompts):  # the single-token path, one sequence at a time
        one = tower(1)
        one.set_state([int(prompt[0])], [0])
        for i in range(len(prompt)):
            one.token_ids.fill_(int(prompt[i]))
            one.decode_step()
        logits.append(one.last_logits[0])
        for layer in range(cfg.n_layers):
            for a, c in zip(one.cache.gather(layer, 0), whole.cache.gather(layer, b)):
                assert close(a, c)
        assert close(whole.last_logits[b], one.last_logits[0])
    for t in (whole, parts):
        t.token_ids.copy_(torch.tensor([5, 6, 7]))
        t.decode_step()
    assert close(parts.last_logits, whole.last_logits)
    with pytest.raises(RuntimeError):
        whole.extend(torch.zeros(3, dtype=torch.int64), [1, 1])
    with pytest.raises(RuntimeError):
        whole.extend(torch.zeros(3, dtype=torch.int64), [1, 1, 0])
    assert ops.last_error() == 0


def test_windowed_cache_takes_portions():
    """A cache with a window: portions attend the last tokens only, as its decoding does."""
    from axono_b200 import ops
    from axono_b200.kv_cache import PagedKVCache, SlidingWindowKVCache

    hq, hkv, d, window = 4, 2, 128, 40
    caches = [SlidingWindowKVCache(window, 1, 2, hkv, d, 256), PagedKVCache(1, 2, hkv, d, 256)]
    starts = row_table([90, 60])
    qkv = rnd((150, (hq + 2 * hkv) * d), torch.float16, 3)
    outs = []
    for cache in caches:
        q = cache.append_portions(0, qkv, hq, starts, 90, inv_freq=freqs(d))
        outs.append(cache.attend_portions(0, q, starts))
    assert not torch.equal(outs[0], outs[1]) and torch.equal(outs[0][:window], outs[1][:window])
    ref = Cache([90, 60], hkv, d, torch.float16)
    ref.k, ref.v = zip(*[caches[0].gather(0, b) for b in range(2)])
    check_attention(q, ref, (90, 60), starts.tolist(), outs[0], window)
    one = rnd((2, (hq + 2 * hkv) * d), torch.float16, 9)
    q1 = caches[0].append_portions(0, one, hq, row_table([1, 1]), 1, inv_freq=freqs(d))
    a, b = caches[0].attend_portions(0, q1, row_table([1, 1])), caches[0].attend(0, q1)
    assert (a.double() - b.double()).abs().max() <= 2.0 ** -9 * b.abs().max()
    assert ops.last_error() == 0


def test_frequencies_of_the_single_token_operators():
    from axono_b200 import ops

    x = rnd((4, 2, 128), torch.float32)
    pos = torch.arange(4, device="cuda")
    a = ops.rope(x, pos, 5e5)
    b, _ = ops.qk_norm_rope(x, None, pos, ops.reference_frequencies(128, 5e5))
    assert (a - b).abs().max() <= 2.0 ** -20 * x.abs().max()


@pytest.mark.parametrize("dtype,d,hq,hkv,rows", [(torch.float32, 256, 60, 8, 60), (torch.float32, 128, 120, 10, 73), (torch.bfloat16, 256, 124, 5, 66),
                                                 (torch.float32, 256, 193, 7, 33), (torch.float16, 128, 250, 7, 40)])
def test_turn_of_many_heads(dtype, d, hq, hkv, rows):
    """Heads of few rows are shared among warps, some of which take part of two rows."""
    from axono_b200 import ops

    q, k, (wq, wk) = rnd((rows, hq, d), dtype, 1), rnd((rows, hkv, d), dtype, 2), weights(d, dtype, True)
    pos = torch.arange(rows, device="cuda") * 11
    oq, ok = ops.qk_norm_rope(q, k, pos, freqs(d), wq, wk, EPS)
    check_turn(oq, turn(q, wq, EPS, pos, freqs(d)))
    check_turn(ok, turn(k, wk, EPS, pos, freqs(d)))
    assert ops.last_error() == 0


def test_append_of_many_heads():
    from axono_b200 import ops

    hq, hkv, d, counts, cached = 56, 6, 256, (35, 0, 25), (3, 5, 64)
    cache = Cache(list(cached), hkv, d, torch.float32, more=40)
    qkv, (wq, wk) = rnd((60, (hq + 2 * hkv) * d), torch.float32, 4), weights(d, torch.float32, True)
    oq = ops.qkv_norm_rope_append_portions(qkv, hq, wq, wk, EPS, cache.k_pages, cache.v_pages, cache.table, cache.lens, row_table(counts),
                                           inv_freq=freqs(d))
    at = 0
    for b, n in enumerate(counts):
        q, k, v = qkv[at:at + n].view(n, hq + 2 * hkv, d).split([hq, hkv, hkv], 1)
        pos = cached[b] + torch.arange(n, device="cuda")
        ck, cv = cache.read(b, cached[b], n)
        check_turn(oq[at:at + n], turn(q, wq, EPS, pos, freqs(d)))
        check_turn(ck, turn(k, wk, EPS, pos, freqs(d)))
        assert torch.equal(cv, v)
        at += n
    assert cache.lens.tolist() == [38, 5, 89] and ops.last_error() == 0


# counts, cached tokens, query and KV heads, where values that are not finite stand: (sequence, token)
HIDDEN = {
    "clusters of two": ((3,) * 16, (900,) * 16, 16, 8, [(0, 902), (5, 448), (5, 449), (9, 901), (15, 0)]),
    "clusters of four": ((4,), (296,), 4, 2, [(0, 298), (0, 127)]),
    "clusters of eight": ((90,), (620,), 4, 2, [(0, 660), (0, 709), (0, 200)]),
    "clusters of eight, some without a key": ((90, 2), (0, 700), 4, 2, [(0, 60), (1, 701)]),
    "parts": ((20, 1, 3), (7000, 30, 6500), 4, 2, [(0, 7010), (0, 3000), (1, 30), (2, 6502), (2, 64)]),
}


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("where", HIDDEN)
def test_hidden_infinities_where_keys_are_divided(where, d, dtype):
    """Values that are not finite in one part of a block's keys: a row that does not see them is as if they were not there, one that does
    has what the definition gives, whichever CTAs the keys were divided among."""
    from axono_b200 import ops

    counts, cached, hq, hkv, places = HIDDEN[where]
    lens = [n + c for n, c in zip(counts, cached)]
    for bad, in_key in ((math.inf, False), (-math.inf, False), (math.nan, False), (math.nan, True)):
        cache = Cache(lens, hkv, d, dtype, seed=2)
        for i, (b, at) in enumerate(places):
            (cache.k if in_key else cache.v)[b][at, i % hkv, (7 * i) % d] = bad
            cache.write(b, 0, cache.k[b], cache.v[b])
        q, cache, starts, out = run_attention(counts, cached, hq, hkv, d, dtype, cache=cache, first=1, behind=2)
        for rows, ref, mag, top in attend_all(q, cache, counts, starts):
            got, fine = out[rows].double(), torch.isfinite(ref)
            assert torch.equal(torch.isnan(got), torch.isnan(ref)) and torch.equal(got[torch.isinf(ref)], ref[torch.isinf(ref)])
            tol = attend_tolerance(dtype, ref, mag, top if math.isfinite(top) else 8.0)[fine]
            assert ((got - ref)[fine].abs() <= tol).all()
    assert ops.last_error() == 0


BAD_TABLES = {  # rows of the launch, table, the sequences that are left
    "passes the rows": (8, [0, 4, 9], [0]),
    "falls at the end": (8, [0, 8, 4], [0]),
    "falls and rises": (9, [0, 6, 2, 9], [0]),  # what begins at 2 would share rows with the first
    "rises behind a fall": (9, [0, 2, 1, 5, 9], [0, 3]),
    "falls at the beginning": (8, [5, 3, 8], []),
    "begins below zero": (8, [-2, 4, 8], [1]),
}


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("d", [64, 20])
@pytest.mark.parametrize("cached", [100, 7000])
@pytest.mark.parametrize("what", BAD_TABLES)
def test_tables_that_do_not_count_up(what, cached, d, dtype):
    """What an entry names that does not count up is left out - not read, not written, whether keys are divided or not - and the other
    sequences have what they have under a good table."""
    from axono_b200 import ops

    rows, table, left = BAD_TABLES[what]
    hq, hkv, batch = 4, 2, len(table) - 1
    cache = Cache([cached + 10 * b for b in range(batch)], hkv, d, dtype, more=16, poison=0.0)
    lens, starts = cache.lens.tolist(), torch.tensor(table, dtype=torch.int32, device="cuda")
    qkv = rnd((rows, (hq + 2 * hkv) * d), dtype, 3)
    counts = [table[b + 1] - table[b] if b in left else 0 for b in range(batch)]
    before = (cache.k_pages.clone(), cache.v_pages.clone())
    # a workspace that holds counts and sums of another call
    q0 = rnd((rows, hq, d), dtype, 9)
    for _ in range(2):
        ops.gqa_attention_portions_paged(q0, cache.k_pages, cache.v_pages, cache.table, cache.lens, row_table([rows] + [0] * (batch - 1)), 7100)
    assert ops.last_error() == 0
    q = torch.full((rows, hq, d), 7.0, dtype=dtype, device="cuda")
    ops.qkv_norm_rope_append_portions(qkv, hq, None, None, EPS, cache.k_pages, cache.v_pages, cache.table, cache.lens, starts, out=q)
    assert ops.last_error() == 16
    assert cache.lens.tolist() == [n + c for n, c in zip(lens, counts)]
    owned = torch.zeros(rows, dtype=torch.bool, device="cuda")
    for b, n in enumerate(counts):
        if not n:
            continue
        r = slice(table[b], table[b + 1])
        owned[r] = True
        want_q, want_k, want_v = qkv[r].view(n, hq + 2 * hkv, d).split([hq, hkv, hkv], 1)
        k, v = cache.read(b, lens[b], n)
        assert torch.equal(q[r], want_q) and torch.equal(k, want_k) and torch.equal(v, want_v)
        cache.k[b], cache.v[b] = cache.read(b, 0, lens[b] + n)
        cache.write(b, lens[b], *(torch.zeros_like(k) for _ in range(2)))
    assert (q[~owned] == 7).all()
    assert torch.equal(cache.k_pages, before[0]) and torch.equal(cache.v_pages, before[1])  # and nothing else was written
    for b, n in enumerate(counts):
        if n:
            cache.write(b, 0, cache.k[b], cache.v[b])
    for _ in range(2):
        ops.gqa_attention_portions_paged(q0, cache.k_pages, cache.v_pages, cache.table, cache.lens, row_table([rows] + [0] * (batch - 1)), 7100)
    out = torch.full((rows, hq, d), 7.0, dtype=dtype, device="cuda")
    ops.gqa_attention_portions_paged(q0, cache.k_pages, cache.v_pages, cache.table, cache.lens, starts, 7100, out=out)
    assert ops.last_error() == 16
    assert (out[~owned] == 7).all()
    good = list(zip(*[(table[b], n) for b, n in enumerate(counts)]))[0]
    check_attention(q0, cache, counts, list(good), out)


@pytest.mark.parametrize("what", ["capacity", "page", "both"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_a_refused_portion_leaves_every_layer_as_it_was(what, dtype):
    """A portion that does not fit, or whose page is outside the pool, in a tower of three layers: no cached key or value of its sequence
    changes in any of them, nor its length, position and next token; the other sequences go on as if it had brought nothing."""
    from axono_b200 import ops
    from axono_b200.decode import TextTower, TextTowerConfig

    cfg = TextTowerConfig(hidden=256, intermediate=512, n_q_heads=8, n_kv_heads=4, head_dim=64, vocab=1000, n_layers=3, use_mrope=False)
    ids = torch.randint(0, 1000, (400,), generator=torch.Generator().manual_seed(1))
    towers = [TextTower(cfg, 3, 320, dtype=dtype, seed=3) for _ in range(2)]
    for t in towers:
        t.extend(ids, [300, 20, 80])
        assert ops.last_error() == 0
    tower, other = towers
    if what != "capacity":
        tower.cache.block_table[2, 1] = tower.cache.num_pages + 3  # the page of slots 64 .. 127: the portion begins in the middle of it
    refused, error = {"capacity": ([0], 4), "page": ([2], 2), "both": ([0, 2], 6)}[what]
    counts = [50 if 0 in refused else 5, 7, 6]
    fitting = [0 if b in refused else n for b, n in enumerate(counts)]
    lens, pos, tokens = tower.cache.seq_lens.clone(), tower.pos3.clone(), tower.token_ids.clone()
    pages = [[pool.clone() for pool in pools] for pools in (tower.cache.k_pages, tower.cache.v_pages)]
    more = torch.randint(0, 1000, (sum(counts),), generator=torch.Generator().manual_seed(2))
    nxt = tower.extend(more, counts)
    assert ops.last_error() & error == error
    parts = torch.split(more, counts)
    expect = other.extend(torch.cat([p for p, n in zip(parts, fitting) if n]), fitting)
    assert tower.cache.seq_lens.tolist() == other.cache.seq_lens.tolist() == [int(n) + c for n, c in zip(lens, fitting)]
    assert torch.equal(tower.pos3, other.pos3) and torch.equal(tower.pos3[:, refused], pos[:, refused])
    assert torch.equal(tower.token_ids[refused], tokens[refused])
    assert nxt.tolist() == [-1 if b in refused else int(expect[[i for i, n in enumerate(fitting) if n].index(b)]) for b in range(3)]
    table = other.cache.block_table
    for pools, old, theirs in zip((tower.cache.k_pages, tower.cache.v_pages), pages, (other.cache.k_pages, other.cache.v_pages)):
        for layer in range(cfg.n_layers):
            for b in range(3):
                n = int(lens[b]) if b in refused else int(lens[b]) + counts[b]
                page, place = table[b, torch.arange(n, device="cuda") // 64].long(), torch.arange(n, device="cuda") % 64
                got, was, want = (x[page, :, place] for x in (pools[layer], old[layer], theirs[layer]))
                assert torch.equal(got[:int(lens[b])], was[:int(lens[b])]), (layer, b)
                # another number of rows may take another algorithm of the projections
                assert (got.double() - want.double()).abs().max() <= 2.0 ** -7 * want.abs().max(), (layer, b)
    if what == "capacity":  # what fits is taken afterwards
        tower.extend(more[:20], [20, 0, 0])
        assert ops.last_error() == 0 and tower.cache.seq_lens.tolist() == [320, 27, 86]
        with pytest.raises(RuntimeError):
            tower.extend(ids[:321], [321, 0, 0])


@pytest.mark.parametrize("rows", [2, 70])  # one launch that also advances, and two
def test_slots_carry_what_was_accepted_to_later_layers(rows):
    from axono_b200 import ops

    hq, hkv, d = 4, 2, 64
    cache = Cache([100, 60, 10], hkv, d, torch.float16, more=rows, poison=0.0)
    counts, lens = [rows, 0, 1], cache.lens.clone()
    cache.table[2, 0] = -1
    qkv, slots = rnd((rows + 1, (hq + 2 * hkv) * d), torch.float16, 3), torch.full((5,), 77, dtype=torch.int32, device="cuda")
    run = lambda advance, lens, slots=slots: ops.qkv_norm_rope_append_portions(  # noqa: E731
        qkv, hq, None, None, EPS, cache.k_pages, cache.v_pages, cache.table, lens, row_table(counts), advance=advance, slots=slots)
    run(True, lens)
    assert ops.last_error() == 2 and slots.tolist() == [100, -1, -1, 77, 77] and lens.tolist() == [100 + rows, 60, 10]
    k = cache.read(0, 100, rows)[0].clone()
    cache.write(0, 100, *(torch.zeros_like(k) for _ in range(2)))
    run(False, lens)
    assert ops.last_error() == 0 and torch.equal(cache.read(0, 100, rows)[0], k)  # and nothing is reported twice
    k0 = cache.k_pages.clone()
    run(False, cache.lens)  # lengths that are not those of the step
    assert ops.last_error() == 4 and torch.equal(cache.k_pages, k0)
    for bad in (slots[:2], slots.long(), slots[::2], slots.cpu()):
        with pytest.raises(RuntimeError):
            run(False, lens, bad)


def test_extending_by_new_numbers_of_rows_makes_no_trial_products():
    """The product whose algorithm is timed on the first use of a shape takes the batch's rows alone; every other number of rows is one
    product per projection."""
    from axono_b200 import ops
    from axono_b200.decode import TextTower, TextTowerConfig

    cfg = TextTowerConfig(hidden=256, intermediate=512, n_q_heads=4, n_kv_heads=2, head_dim=64, vocab=500, n_layers=2, use_mrope=False)
    tower, timed = TextTower(cfg, 3, 640, seed=3), []
    inner = ops.linear_nobias
    tower._linear = lambda x, w: timed.append(x.shape[0]) or inner(x, w)
    for counts in ([70, 0, 0], [1, 1, 0], [5, 100, 33], [0, 0, 1], [1, 1, 1], [0, 3, 0]):
        tower.extend(torch.arange(sum(counts)) % 500, counts)
    tower.decode_step()
    assert timed and set(timed) == {3}
    assert ops.last_error() == 0


def narrow_tolerance(ref, mag, top, keys, largest):
    """What `attend_tolerance` counts for scores, exponentials and the result's rounding; weights in two fp16 parts, off by 2^-22 of themselves
    and 2^-32 of the largest where a part is subnormal; and the tensor core's sums over 1024 keys at most, 8 products to 64 of them, each of
    which drops less than a unit of the last place, 2^-23 of what is added up: 128 * 2^-23."""
    half = torch.finfo(torch.float16).eps / 2
    return ref.abs() * half * (1 + 2.0 ** -10) + mag * (2.0 ** -21 * (2 + 2 * top) + 2.0 ** -22 + 2.0 ** -16) + 2.0 ** -32 * keys * largest + \
        torch.finfo(torch.float16).smallest_normal * half


@pytest.mark.parametrize("hq,hkv,d", [(4, 4, 64), (6, 2, 80), (3, 1, 96), (4, 2, 40), (2, 2, 8), (8, 1, 120)])
def test_weights_of_narrow_heads_keep_more_than_their_type(hq, hkv, d):
    """Few keys that carry the weight, where a rounded weight would show: whole blocks, clusters, parts."""
    from axono_b200 import ops

    for counts, cached in (((200, 3), (0, 60)), ((90,), (600,)), ((20, 2), (7000, 40))):
        for window in (0, 50):
            q, cache, starts, out = run_attention(counts, cached, hq, hkv, d, torch.float16, window=window, spread=3.0)
            for rows, ref, mag, top in attend_all(q, cache, counts, starts, window):
                tol = narrow_tolerance(ref, mag, top, max(cached) + max(counts), max(float(v.abs().max()) for v in cache.v))
                err = (out[rows].double() - ref).abs()
                assert (err <= tol).all(), float((err / tol).max())
    assert ops.last_error() == 0


def test_long_sums_of_narrow_heads_are_not_pulled_towards_zero():
    """16384 keys in a row, values with a common offset: each product of the tensor core drops a part of a last bit, always towards zero, so
    that one sum over all keys is too small by 2^-15.  Sums over 1024 keys stay within 2^-16 of the whole, 128 products of less than 2^-23
    each; rounding the result is not biased: its mean over n elements is within four times 2^-11 / sqrt(3 n) of zero."""
    from axono_b200 import ops
    from axono_b200._capi import FLOAT16

    hq = hkv = 64  # three blocks per head: more than half of what runs at once, so that keys are not divided
    counts, cached, d = (384,), (16000,), 64
    cache = Cache([16384], hkv, d, torch.float16)
    cache.v[0].mul_(0.25).add_(1.0)
    cache.write(0, 0, cache.k[0], cache.v[0])
    assert ops._portions_workspace_bytes(384, 1, hq, hkv, d, 64, cache.table.shape[1], 16384, 0, True, FLOAT16) == 0
    q, cache, starts, out = run_attention(counts, cached, hq, hkv, d, torch.float16, cache=cache, spread=0.5)
    [(rows, ref, mag, top)] = attend_all(q, cache, counts, starts)
    bias = float(((out[rows].double() - ref) / ref).mean())
    assert abs(bias) <= 2.0 ** -16 + 4 * 2.0 ** -11 / math.sqrt(3 * ref.numel()), bias
    assert ops.last_error() == 0


# ---- what the cases above do not reach ------------------------------------------------------------------------------

EDGES = {  # counts, cached, query and KV heads: how the keys are divided is a function of these
    "whole": ((300, 130), (0, 10), 4, 2), "clusters of two": ((3,) * 16, (900,) * 16, 16, 8), "clusters of four": ((4,), (296,), 4, 2),
    "clusters of eight": ((13,), (1500,), 4, 2), "a long cluster": ((20,), (5000,), 4, 2), "parts": ((20, 1, 3), (7000, 30, 6500), 4, 2),
    "parts of a long cache": ((2,), (70000,), 2, 1), "parts of full blocks": ((640,), (9000,), 2, 1)}


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("d", [64, 128, 20])
@pytest.mark.parametrize("what", EDGES)
def test_no_key_is_lost_or_doubled_where_tiles_meet(what, d, dtype):
    """All the weight on the first and last key of every tile of 64, in equal shares: a key that is missing or counts twice changes a row by
    a share of it, many times the tolerance."""
    from axono_b200 import ops

    counts, cached, hq, hkv = EDGES[what]
    lens = [n + c for n, c in zip(counts, cached)]
    cache = Cache(lens, hkv, d, dtype, seed=4)
    u = torch.ones(d, device="cuda", dtype=torch.float64) / math.sqrt(d)
    height = 4.0 * d ** 0.25  # scores of +-16
    # with fp16 weights the tolerance is 2^-11 of the mean |value|, so that no more than a few hundred keys may share the weight: every
    # `apart`-th tile at a time
    apart = -(-max(lens) // 16384)
    starts, rows = row_table(counts), sum(counts)
    q = (height * u).expand(rows, hq, d).to(dtype).contiguous()
    q += (2.0 ** -6 * torch.randn(q.shape, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")).to(dtype)
    for phase in range(apart):
        for b, n in enumerate(lens):
            at = torch.arange(n, device="cuda")
            edge = (((at % 64 == 0) | (at % 64 == 63)) & (at // 64 % apart == phase)).double() * 2 - 1
            cache.k[b] = (height * edge[:, None, None] * u).expand(n, hkv, d).to(dtype).contiguous()
            cache.write(b, 0, cache.k[b], cache.v[b])
        out = ops.gqa_attention_portions_paged(q, cache.k_pages, cache.v_pages, cache.table, cache.lens, starts, max(lens))
        for r, ref, mag, top in attend_all(q, cache, counts, starts.tolist()):
            tol = attend_tolerance(dtype, ref, mag, top)
            err = (out[r].double() - ref).abs()
            assert (err <= tol).all(), float((err / tol).max())
            if len(counts) == 1:  # that a key's share stands out from the tolerance
                assert 0.5 * float(cache.v[0].abs().mean()) / (2 * lens[0] / 64 / apart) > 2 * float(tol.median())
    assert ops.last_error() == 0


@pytest.mark.parametrize("lens,bound,parts", [((700, 650, 90), 800, False), ((6100, 9000, 130), 9100, True)])
def test_a_replayed_step_with_clusters_and_with_parts(lens, bound, parts):
    """Captured once, replayed over a cache that grows past the edges of tiles and pages and over rows that move from one sequence to another:
    the bits of eager calls, with the keys divided in clusters and in parts that a second kernel joins."""
    from axono_b200 import ops
    from axono_b200._capi import FLOAT16

    hq, hkv, d, rows, steps = 4, 2, 128, 6, 24
    caches = [Cache(lens, hkv, d, torch.float16, more=rows * steps, poison=0.0) for _ in range(2)]
    blocks = caches[0].table.shape[1]
    assert (ops._portions_workspace_bytes(rows, 3, hq, hkv, d, 64, blocks, bound, 0, True, FLOAT16) > 0) == parts
    starts, f = row_table([2, 2, 2]), freqs(d)
    qkv = torch.zeros((rows, (hq + 2 * hkv) * d), dtype=torch.float16, device="cuda")
    out = torch.empty((rows, hq, d), dtype=torch.float16, device="cuda")

    def step(c, out=None):
        q = ops.qkv_norm_rope_append_portions(qkv, hq, None, None, EPS, c.k_pages, c.v_pages, c.table, c.lens, starts, inv_freq=f)
        return ops.gqa_attention_portions_paged(q, c.k_pages, c.v_pages, c.table, c.lens, starts, bound, out=out)

    first = caches[0].lens.clone()
    step(caches[0], out)
    caches[0].lens.copy_(first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(caches[0], out)
    for i in range(steps):
        starts.copy_(row_table([(2, 2, 2), (6, 0, 0), (0, 1, 5), (1, 4, 1)][i % 4]))
        qkv.copy_(rnd(qkv.shape, torch.float16, i))
        graph.replay()
        assert torch.equal(out, step(caches[1])), i
    assert torch.equal(caches[0].lens, caches[1].lens) and int(caches[0].lens.sum()) == sum(lens) + rows * steps
    assert torch.equal(caches[0].k_pages, caches[1].k_pages) and torch.equal(caches[0].v_pages, caches[1].v_pages)
    counts = [1, 4, 1]
    for b in range(3):
        caches[1].k[b], caches[1].v[b] = caches[1].read(b, 0, int(caches[1].lens[b]))
    pos = torch.cat([torch.arange(int(n) - c, int(n)) for n, c in zip(caches[1].lens, counts)]).cuda()
    q = ops.qk_norm_rope(qkv[:, :hq * d].view(rows, hq, d), None, pos, f)[0]
    check_attention(q, caches[1], counts, starts.tolist(), out)
    assert ops.last_error() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
def test_positions_beyond_32_bits(interleaved, dtype):
    """Frequencies of 2 pi / (3 * 2^k), for which a position's turns are known exactly: their upper 32 bits matter (2^32 is no multiple of
    3 * 2^k).  The product in double is off by 2^-52 of the turns, thrice."""
    from axono_b200 import ops

    rows, d, n = 50, 64, 32
    k = torch.arange(n) % 12 + 4
    period = 3 * 2 ** k.long()
    f = (2 * math.pi / period.double()).cuda()
    for far in (1 << 33, 1 << 36):
        pos = far + torch.randint(0, far, (rows,), generator=torch.Generator().manual_seed(5))
        turns = (pos[:, None] % period).double() / period  # exact but for one rounding
        x = rnd((rows, 2, d), dtype, 1)
        out, _ = ops.qk_norm_rope(x, None, pos.cuda(), f, interleaved=interleaved)
        c, s = (2 * math.pi * turns).cos().cuda()[:, None], (2 * math.pi * turns).sin().cuda()[:, None]
        xd = x.double()
        a, b = (xd[..., ::2], xd[..., 1::2]) if interleaved else (xd[..., :n], xd[..., n:])
        pair = (a * c - b * s, b * c + a * s)
        ref = torch.stack(pair, -1).flatten(-2) if interleaved else torch.cat(pair, -1)
        slack = 2 * math.pi * 2 * far / 48 * 2.0 ** -52 * 3
        half = torch.finfo(dtype).eps / 2
        assert ((out.double() - ref).abs() <= ref.abs() * half * (1 + 2.0 ** -10) + ref.abs().amax(-1, keepdim=True) * (2.0 ** -20 + slack)).all()


def test_far_keys_of_portions_and_of_single_tokens():
    """Single tokens are turned by the product of position and frequency in fp32, off by half a step, 2^-24 of the angle; portions by the
    angle itself.  So a key of either stands within that of the other, at any position of a long context."""
    from axono_b200 import ops

    hq, hkv, d, theta = 2, 2, 128, 1e6
    f = ops.reference_frequencies(d, theta)
    for at in (129, 4000, 30000, 131071):
        qkv = rnd((1, (hq + 2 * hkv) * d), torch.float32, at)
        caches = [Cache([5], hkv, d, torch.float32, more=1) for _ in range(2)]
        pos = torch.tensor([at], device="cuda")
        q1 = ops.qkv_norm_rope_append(qkv, hq, None, None, EPS, caches[0].k_pages, caches[0].v_pages, caches[0].table, caches[0].lens, pos=pos,
                                      theta=theta)
        q2 = ops.qkv_norm_rope_append_portions(qkv, hq, None, None, EPS, caches[1].k_pages, caches[1].v_pages, caches[1].table, caches[1].lens,
                                               row_table([1]), pos=pos, inv_freq=f)
        angle = (at * f * 2.0 ** -24).repeat(2)
        for a, b in ((q1, q2), (caches[0].read(0, 5, 1)[0], caches[1].read(0, 5, 1)[0])):
            a, b = a.double().view(-1, d), b.double().view(-1, d)
            size = (b[:, :d // 2].square() + b[:, d // 2:].square()).sqrt().repeat(1, 2)
            assert ((a - b).abs() <= size * (angle * (1 + 2.0 ** -10) + 2.0 ** -20)).all()
    assert ops.last_error() == 0


def test_tower_whose_heads_are_shared_between_two_ranks_extends():
    """Two ranks as threads of this process, each with half of the heads; what they gather goes through the host's barrier.  (No kernel
    waits for another rank's.)"""
    import threading

    from axono_b200 import ops, sharding
    from axono_b200.decode import TextTower, TextTowerConfig

    cfg = TextTowerConfig(hidden=256, intermediate=512, n_q_heads=8, n_kv_heads=4, head_dim=64, vocab=500, n_layers=2, use_mrope=False)
    make = lambda world, rank: TextTower(cfg, 2, 320, dtype=torch.float32, seed=3, world=world, rank=rank, fused_gather=False)  # noqa: E731
    towers, one, barrier, shares, me = [make(2, r) for r in range(2)], make(1, 0), threading.Barrier(2, timeout=60), {}, threading.local()

    def gather(attn):
        shares[me.rank] = attn
        barrier.wait()
        whole = torch.cat([shares[r] for r in range(2)], 1)
        barrier.wait()
        return whole

    steps, results, errors = [([70, 3], 73), ([1, 0], 1), ([5, 130], 135)], {}, []

    def run(rank):
        try:
            me.rank = rank
            for i, (counts, n) in enumerate(steps):
                results[rank, i] = (towers[rank].extend(torch.arange(n) * 7 % 500, counts), towers[rank].last_logits)
        except BaseException as e:  # noqa: BLE001 - the other rank must not wait for good
            errors.append(e)
            barrier.abort()

    inner = sharding.all_gather_heads
    sharding.all_gather_heads = gather
    try:
        threads = [threading.Thread(target=run, args=(r,)) for r in range(2)]
        [t.start() for t in threads]
        [t.join() for t in threads]
    finally:
        sharding.all_gather_heads = inner
    assert not errors, errors
    for i, (counts, n) in enumerate(steps):
        nxt = one.extend(torch.arange(n) * 7 % 500, counts)
        for rank in range(2):
            assert torch.equal(results[rank, i][0], nxt)
            assert (results[rank, i][1] - one.last_logits).abs().max() <= 1e-4 * one.last_logits.abs().max()
    assert ops.last_error() == 0


@pytest.mark.parametrize("batch", [1, 5, 30, 31, 32, 33, 64, 100])
def test_rows_of_random_tables(batch):
    """Tables with and without entries that do not count up, about the 32 that a warp holds at once: which rows are appended and attended,
    and which lengths grow, by the rule for each entry by itself."""
    from axono_b200 import ops

    rows, hq, hkv, d = 90, 2, 1, 64
    g = torch.Generator().manual_seed(batch)
    for trial in range(12):
        table = torch.sort(torch.randint(0, rows + 1, (batch + 1,), generator=g)).values
        for _ in range(trial // 3):  # none in the first three
            table[int(torch.randint(0, batch + 1, (1,), generator=g))] = int(torch.randint(-3, rows + 4, (1,), generator=g))
        table = table.tolist()
        up = [0 <= e <= rows and e >= max(table[:i], default=e) for i, e in enumerate(table)]
        owner = [-1] * rows
        for b in range(batch):
            if up[b] and up[b + 1]:
                for r in range(table[b], table[b + 1]):
                    assert owner[r] == -1
                    owner[r] = b
        grown = [owner.count(b) for b in range(batch)]
        cache = Cache([3] * batch, hkv, d, torch.float16, more=rows, poison=0.0)
        qkv, starts = rnd((rows, (hq + 2 * hkv) * d), torch.float16, trial), torch.tensor(table, dtype=torch.int32, device="cuda")
        q = torch.full((rows, hq, d), 7.0, dtype=torch.float16, device="cuda")
        ops.qkv_norm_rope_append_portions(qkv, hq, None, None, EPS, cache.k_pages, cache.v_pages, cache.table, cache.lens, starts, out=q)
        assert bool(ops.last_error() & 16) == (not all(up))
        assert cache.lens.tolist() == [3 + n for n in grown]
        out = torch.full((rows, hq, d), 7.0, dtype=torch.float16, device="cuda")
        ops.gqa_attention_portions_paged(qkv[:, :hq * d].reshape(rows, hq, d), cache.k_pages, cache.v_pages, cache.table, cache.lens, starts,
                                         3 + rows, out=out)
        assert bool(ops.last_error() & 16) == (not all(up))
        owned = torch.tensor([o >= 0 for o in owner], device="cuda")
        assert (q[~owned] == 7).all() and (out[~owned] == 7).all()
        assert torch.equal(q[owned], qkv[owned, :hq * d].view(-1, hq, d)) and not (out[owned] == 7).all(-1).any()
        for b in range(batch):
            if grown[b]:
                k, v = cache.read(b, 3, grown[b])
                r0 = table[b]
                assert torch.equal(k[:, 0], qkv[r0:r0 + grown[b], hq * d:(hq + 1) * d])
                assert torch.equal(v[:, 0], qkv[r0:r0 + grown[b], (hq + 1) * d:])


def test_an_output_between_the_rows_of_a_strided_product():
    """It shares no memory with what is read, and is taken."""
    from axono_b200 import ops

    hq, hkv, d, rows = 2, 1, 64, 5
    columns = (hq + 2 * hkv) * d
    buf = rnd((rows, columns + rows * hq * d + 64), torch.float16, 1)
    qkv, out = buf[:, :columns], buf.view(-1)[buf.shape[1] + columns:][:rows * hq * d].view(rows, hq, d)
    cache = Cache([0], hkv, d, torch.float16, more=64)
    before = qkv.clone()
    got = ops.qkv_norm_rope_append_portions(qkv, hq, None, None, EPS, cache.k_pages, cache.v_pages, cache.table, cache.lens, row_table([rows]), out=out)
    assert got is out and torch.equal(out, before[:, :hq * d].view(rows, hq, d)) and torch.equal(qkv, before)
    for bad in (buf.view(-1)[columns // 2:][:rows * hq * d].view(rows, hq, d), buf.view(-1)[columns + 128:][:rows * hq * d].view(rows, hq, d)):
        with pytest.raises(RuntimeError):
            ops.qkv_norm_rope_append_portions(qkv, hq, None, None, EPS, cache.k_pages, cache.v_pages, cache.table, cache.lens, row_table([rows]), out=bad)
    q = rnd((2 * rows, hq, d), torch.float16, 2)
    with pytest.raises(RuntimeError):
        ops.gqa_attention_portions_paged(q[:rows], cache.k_pages, cache.v_pages, cache.table, cache.lens, row_table([rows]), 64, out=q[3:3 + rows])
    assert cache.lens.tolist() == [rows] and ops.last_error() == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("d", [64, 128, 20])
@pytest.mark.parametrize("counts,cached,hq,hkv", [((130, 4), (0, 90), 4, 2), ((3,) * 16, (900,) * 16, 16, 8), ((20,), (700,), 4, 2), ((5, 1), (7000, 64), 4, 2)])
def test_scores_as_large_as_fp16_inputs_give(counts, cached, hq, hkv, d, dtype):
    """Scores of 2^30 and more, positive or negative, where one key carries all the weight: the result is its value.  (Rows whose two largest
    scores are nearer than the rounding of a sum in fp32, 2^-20 of the largest, have no such key.)"""
    from axono_b200 import ops

    lens = [n + c for n, c in zip(counts, cached)]
    for sign in (1, -1, 0):
        cache = Cache(lens, hkv, d, dtype, seed=6)
        rows = sum(counts)
        q = rnd((rows, hq, d), dtype, 5, 15000.0).clamp(-60000, 60000)
        for b in range(len(lens)):
            cache.k[b] = (cache.k[b].float() * 15000.0).clamp(-60000, 60000).to(dtype)
            if sign:  # all scores of one sign
                cache.k[b] = cache.k[b].abs()
            cache.write(b, 0, cache.k[b], cache.v[b])
        if sign:
            q = q.abs() * sign
        starts = row_table(counts)
        out = ops.gqa_attention_portions_paged(q, cache.k_pages, cache.v_pages, cache.table, cache.lens, starts, max(lens))
        assert torch.isfinite(out).all()
        clear = 0
        for b, (n, c) in enumerate(zip(counts, cached)):
            r0 = int(starts[b])
            seen = torch.arange(lens[b], device="cuda")[None] <= c + torch.arange(n, device="cuda")[:, None]
            for h in range(hq):
                s = (q[r0:r0 + n, h].double() @ cache.k[b][:, h * hkv // hq].double().T).masked_fill(~seen, -math.inf)
                top = s.topk(min(2, lens[b]), -1)
                alone = seen.sum(1) == 1
                gap = alone if top.values.shape[1] < 2 else alone | (top.values[:, 0] - top.values[:, 1] > 2.0 ** -20 * top.values[:, 0].abs() + 1e4)
                want = cache.v[b][top.indices[:, 0], h * hkv // hq]
                assert torch.equal(out[r0:r0 + n, h][gap], want[gap])
                clear += int(gap.sum())
        assert clear > 0.9 * rows * hq
    assert ops.last_error() == 0


def test_portions_over_an_arena_of_pages():
    """The cache that an arena gives: portions into reserved pages, one refused for want of them, taken once they are reserved."""
    from axono_b200 import ops
    from axono_b200.kv_cache import KVArena

    hq, hkv, d, layers = 4, 2, 64, 2
    arena = KVArena(layers, 12, hkv, d, 3, 320)
    cache, ids = arena.cache(), [arena.alloc_seq(64), arena.alloc_seq(128)]
    arena.sync()
    assert ids == [0, 1]
    qkvs = [rnd((170, (hq + 2 * hkv) * d), torch.float16, i) for i in range(layers)]
    f = freqs(d)

    def bring(counts):
        starts = row_table(counts)
        return [cache.attend_portions(i, cache.append_portions(i, x[:sum(counts)], hq, starts, max(counts), inv_freq=f), starts)
                for i, x in enumerate(qkvs)]

    bring([60, 100, 0])
    assert ops.last_error() == 0 and cache.seq_lens.tolist() == [60, 100, 0]
    kept = [[t.clone() for t in cache.gather(i, 0)] for i in range(layers)]
    bring([70, 20, 0])  # the first has no page behind its 64th token
    assert ops.last_error() & 6 and cache.seq_lens.tolist() == [60, 120, 0] and cache.portion_slots.tolist() == [-1, 100, -1]
    for i in range(layers):
        assert all(torch.equal(a, b) for a, b in zip(cache.gather(i, 0), kept[i]))
    arena.reserve(0, 130)
    arena.sync()
    outs = bring([70, 0, 0])
    assert ops.last_error() == 0 and cache.seq_lens.tolist() == [130, 120, 0]
    ref = Cache([130], hkv, d, torch.float16)
    for i in range(layers):
        k, v = cache.gather(i, 0)
        assert torch.equal(k[:60], kept[i][0]) and torch.equal(v[:60], kept[i][1])
        ref.k, ref.v = [k], [v]
        q = ops.qk_norm_rope(qkvs[i][:70, :hq * d].view(70, hq, d), None, torch.arange(60, 130, device="cuda"), f)[0]
        check_attention(q, ref, [70], [0], outs[i])
    arena.close()


def test_calls_without_rows():
    from axono_b200 import ops

    cache = Cache([70, 5], 2, 64, torch.float16)
    before, starts = cache.k_pages.clone(), row_table([0, 0])
    empty = torch.empty((0, 4 * 64 + 4 * 64), dtype=torch.float16, device="cuda")
    q = ops.qkv_norm_rope_append_portions(empty, 4, None, None, EPS, cache.k_pages, cache.v_pages, cache.table, cache.lens, starts)
    assert q.shape == (0, 4, 64)
    assert ops.gqa_attention_portions_paged(q, cache.k_pages, cache.v_pages, cache.table, cache.lens, starts, 100).shape == (0, 4, 64)
    oq, ok = ops.qk_norm_rope(q, q[:, :2], torch.empty(0, dtype=torch.int64, device="cuda"), freqs(64))
    assert oq.shape == (0, 4, 64) and ok.shape == (0, 2, 64)
    assert cache.lens.tolist() == [70, 5] and torch.equal(cache.k_pages.view(torch.int16), before.view(torch.int16)) and ops.last_error() == 0


@pytest.mark.parametrize("counts,cached,parts", [((384,), (5500,), False), ((2,) * 8, (6000,) * 8, True), ((2368,), (1300,), False)])
def test_restarted_sums_of_narrow_heads_in_clusters_and_parts(counts, cached, parts):
    """More than 1024 keys to a CTA of a cluster of four, to a part, and to a CTA with a block of its own: sums that were put aside are joined
    with those that follow, and with what they still owe to a maximum that grows - later keys have the larger scores."""
    from axono_b200 import ops
    from axono_b200._capi import FLOAT16

    hq, hkv, d = 16, 8, 64
    lens = [n + c for n, c in zip(counts, cached)]
    cache = Cache(lens, hkv, d, torch.float16, seed=8)
    for b, n in enumerate(lens):
        cache.k[b] = (cache.k[b].float() * torch.linspace(0.2, 3.0, n, device="cuda")[:, None, None]).half()
        cache.write(b, 0, cache.k[b], cache.v[b])
    assert (ops._portions_workspace_bytes(sum(counts), len(counts), hq, hkv, d, 64, cache.table.shape[1], max(lens), 0, True, FLOAT16) > 0) == parts
    q, cache, starts, out = run_attention(counts, cached, hq, hkv, d, torch.float16, cache=cache, spread=2.0)
    for rows, ref, mag, top in attend_all(q, cache, counts, starts):
        tol = narrow_tolerance(ref, mag, top, max(lens), max(float(v.abs().max()) for v in cache.v))
        err = (out[rows].double() - ref).abs()
        assert (err <= tol).all(), float((err / tol).max())
    assert ops.last_error() == 0
