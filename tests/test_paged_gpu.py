"""Requests of unequal length over one cache of pages in 8 bits, through the operators, against 64 bits on the CPU."""
import math

import numpy as np
import pytest
import torch

import paged_oracle as po
from kmll_b200 import ops
from kmll_b200.lib import KmllError

pytestmark = pytest.mark.gpu
THETA = 1.0e6


def ints(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


def freqs_of(n, hd):
    return np.array([THETA ** (-2.0 * d / hd) for d in range(n)], np.float32)


# ---- pages of a step --------------------------------------------------------------------------------------------------------
def run_plan(lengths, new, block, table, free, count, capacity, in_place=False):
    requests = len(lengths)
    t, length, left = ints(table).reshape(np.asarray(table).shape), ints(lengths), ints([count])
    context = length if in_place else ints([-7] * requests)
    out = left if in_place else ints([-7])
    start, positions, slots, status = ints([-7] * (requests + 1)), ints([-7] * capacity), ints([-7] * capacity), ints([-7])
    ops.paged_plan(length, ints(new), block, t, ints(free), left, context, start, positions, slots, out, status)
    return context.tolist(), start.tolist(), t.cpu().numpy(), positions.tolist(), slots.tolist(), out.item(), status.item()


def make_plan(rng, requests, block, longest, most_new, spare=3):
    lengths = [int(x) for x in rng.integers(0, longest + 1, requests)]
    new = [int(x) for x in rng.integers(0, most_new + 1, requests)]
    width = max([-(-(c + n) // block) for c, n in zip(lengths, new)] + [1]) + 1
    pages = sum(-(-(c + n) // block) for c, n in zip(lengths, new)) + spare
    order = rng.permutation(pages)
    table, at = np.full((requests, width), -1), 0
    for r, c in enumerate(lengths):
        held = -(-c // block)
        table[r, :held] = order[at:at + held]
        at += held
    free = np.concatenate([order[at:], np.full(5, -9)])
    return lengths, new, table, free, pages - at


@pytest.mark.parametrize("requests, block, longest, most_new, room", [
    (1, 16, 0, 1, 0), (1, 128, 500, 1, 3), (7, 16, 40, 3, 5), (64, 32, 900, 1, 0), (65, 64, 300, 90, 17), (300, 16, 200, 40, 1), (513, 32, 64, 2, 0), (1024, 16, 33, 5, 100),
    (3000, 128, 300, 1, 9)])
def test_plan(cuda, requests, block, longest, most_new, room):
    rng = np.random.default_rng(requests + block)
    lengths, new, table, free, count = make_plan(rng, requests, block, longest, most_new)
    capacity = sum(new) + room
    want = po.plan(lengths, new, block, table, free, count, capacity)
    for in_place in (False, True):
        got = run_plan(lengths, new, block, table, free, count, capacity, in_place)
        for g, w in zip(got, want):
            np.testing.assert_array_equal(g, w)


@pytest.mark.parametrize("what, code", [("pages", 1), ("table", 2), ("negative length", 3), ("negative new", 3), ("rows", 3), ("count", 3), ("negative count", 3)])
def test_plan_that_cannot_be_met_changes_nothing(cuda, what, code):
    rng = np.random.default_rng(5)
    lengths, new, table, free, count = make_plan(rng, 9, 16, 60, 30)
    lengths[2], new[2] = 5, 30
    capacity = sum(new) + 2
    if what == "pages":
        count = sum(-(-(c + n) // 16) - -(-c // 16) for c, n in zip(lengths, new)) - 1
    elif what == "table":
        new[4] = table.shape[1] * 16 - lengths[4] + 1
        capacity = sum(new)
    elif what == "negative length":
        lengths[3] = -1
    elif what == "negative new":
        new[8] = -1
    elif what == "rows":
        capacity = sum(new) - 1
    elif what == "count":
        count = len(free) + 1
    else:
        count = -1
    want = po.plan(lengths, new, 16, table, free, count, capacity)
    assert want[-1] == code
    for g, w in zip(run_plan(lengths, new, 16, table, free, count, capacity), want):
        np.testing.assert_array_equal(g, w)


def test_plan_of_no_requests_and_of_many(cuda):
    context, start, _, positions, slots, left, status = run_plan([], [], 16, np.zeros((0, 4), np.int64), [3, 1], 2, 5)
    assert (context, start, positions, slots, left, status) == ([], [0], [0] * 5, [-1] * 5, 2, 0)
    rng = np.random.default_rng(1)
    lengths, new, table, free, count = make_plan(rng, 8192, 16, 20, 2)
    want = po.plan(lengths, new, 16, table, free, count, sum(new))
    for g, w in zip(run_plan(lengths, new, 16, table, free, count, sum(new)), want):
        np.testing.assert_array_equal(g, w)


def test_release_gives_back_what_the_plan_took(cuda):
    rng = np.random.default_rng(8)
    lengths, new, table, free, count = make_plan(rng, 40, 32, 300, 3)
    context = [c + n for c, n in zip(lengths, new)]
    table2 = po.plan(lengths, new, 32, table, free, count, sum(new))[2]
    ended = rng.integers(0, 2, 40)
    t, c, stack, left, status = ints(table2), ints(context), ints(np.concatenate([free, np.zeros(500, np.int64)])), ints([1]), ints([-7])
    ops.paged_release(c, ints(ended), 32, t, stack, left, c, left, status)
    back = [int(p) for r in range(40) if ended[r] for p in table2[r, :-(-context[r] // 32)]]
    assert status.item() == 0 and left.item() == 1 + len(back) and stack.tolist()[1:1 + len(back)] == back
    assert c.tolist() == [0 if e else x for x, e in zip(context, ended)]
    kept = np.where((ended[:, None] != 0) & (np.arange(table2.shape[1]) < np.array([-(-x // 32) for x in context])[:, None]), -1, table2)
    np.testing.assert_array_equal(t.cpu().numpy(), kept)
    # a stack that is too small, a context beyond its row: nothing changes
    for contexts, room, code in ((context, len(back) - 1, 1), ([table2.shape[1] * 32 + 1] + context[1:], 600, 3)):
        t, c, stack, left, out, status = ints(table2), ints(contexts), ints(np.arange(room)), ints([0]), ints([-7]), ints([-7])
        o = ints([-7] * 40)
        ops.paged_release(c, ints(ended), 32, t, stack, left, o, out, status)
        assert status.item() == code and out.item() == 0 and o.tolist() == contexts and stack.tolist() == list(range(room))
        np.testing.assert_array_equal(t.cpu().numpy(), table2)


# ---- rotation and storage ---------------------------------------------------------------------------------------------------
def f64(t):
    return t.double().cpu().numpy()


def same_cache(cache, ks, vs):
    np.testing.assert_array_equal(cache.k_scales.cpu().numpy(), ks.scales)
    np.testing.assert_array_equal(cache.v_scales.cpu().numpy(), vs.scales)
    np.testing.assert_array_equal(cache.k_codes.cpu().numpy(), po.key_layout(ks.codes))
    np.testing.assert_array_equal(cache.v_codes.cpu().numpy(), po.value_layout(vs.codes))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads, kv, hd, block, rot", [(4, 2, 64, 16, 32), (8, 1, 128, 32, 64), (6, 3, 80, 64, 24), (2, 2, 16, 128, 8), (3, 1, 256, 16, 0), (16, 16, 32, 32, 16)])
def test_prepare_stores_codes_as_defined(cuda, dtype, heads, kv, hd, block, rot):
    """Portions of several lengths one after another into pages in a mixed order: codes and scales are the oracle's to the bit; turned queries are within the
    rounding of 32 bits (or of bf16) of the 64-bit ones."""
    rng = np.random.default_rng(hd + block)
    pages, width = 13, 3
    order = rng.permutation(pages)
    table = order[:4 * width].reshape(4, width)
    cache = ops.DevicePagedI8Cache.create(pages, block, kv, hd)
    ks, vs = po.Store(pages, block, kv, hd), po.Store(pages, block, kv, hd)
    freqs = freqs_of(rot, hd)
    lengths = [0, 0, 0, 0]
    for step, new in enumerate([(block + 3, 1, 5, 0), (1, 1, 1, 1), (1, block, 1, 2), (2, 1, block - 7, 1), (1, 1, 1, 1)]):
        slots, positions = [], []
        for r, n in enumerate(new):
            for p in range(lengths[r], lengths[r] + n):
                slots.append(int(table[r, p // block]) * block + p % block)
                positions.append(p + 100000 * r)
            lengths[r] += n
        slots.append(-1)  # a padded row
        positions.append(0)
        tokens = len(slots)
        q, k, v = (torch.tensor(rng.normal(0, 1 + step, (tokens, h, hd)), device="cuda").to(dtype) for h in (heads, kv, kv))
        turned = torch.full_like(q, 7.0)
        ops.prepare_paged_attention(q, k, v, torch.tensor(freqs, device="cuda") if rot else None, ints(positions), ints(slots), cache, query_rot=turned)
        want = po.rotate(f64(q), positions, freqs) if rot else f64(q)
        ks.append(po.rotate(f64(k), positions, freqs) if rot else f64(k), slots)
        vs.append(f64(v), slots)
        got = f64(turned)
        assert (got[-1] == 7.0).all()
        step_of = 2.0 ** -23 if dtype == torch.float32 else 2.0 ** -8
        assert (np.abs(got - want)[:-1] <= step_of * np.abs(want)[:-1] + 1e-30).all()  # one rounding, of 64 bits (and one to 32 for bf16)
        same_cache(cache, ks, vs)
    shown = [int(table[r, p // block]) * block + p % block for r in range(4) for p in range(lengths[r])]
    k, v = ops.paged_cache_rows(cache, ints(shown))
    np.testing.assert_array_equal(k.cpu().numpy(), ks.rows(shown))
    np.testing.assert_array_equal(v.cpu().numpy(), vs.rows(shown))


@pytest.mark.parametrize("tokens, block", [(600, 16), (1025, 64), (2300, 128)])
def test_prepare_of_long_prompts(cuda, tokens, block):
    """Past the size from which a thread block takes a page of tokens; runs begin in the middle of pages."""
    rng = np.random.default_rng(tokens)
    kv, hd, heads = 2, 64, 4
    pages = tokens // block + 9
    order = rng.permutation(pages)
    at, slots, positions, used = 0, [], [], 0
    while at < tokens:
        n = min(int(rng.integers(1, 3 * block)), tokens - at)
        first = int(rng.integers(0, block)) if used + -(-(n + block) // block) <= pages else 0
        if used + -(-(n + first) // block) > pages:
            break
        for p in range(first, first + n):
            slots.append(int(order[used + p // block]) * block + p % block)
            positions.append(p)
        used += -(-(n + first) // block)
        at += n
    cache, ks, vs = ops.DevicePagedI8Cache.create(pages, block, kv, hd), po.Store(pages, block, kv, hd), po.Store(pages, block, kv, hd)
    for s in (ks, vs):
        s.codes = np.clip(np.rint(rng.normal(0, 36, s.codes.shape)), -127, 127)
        s.scales = rng.uniform(0.005, 0.03, s.scales.shape).astype(np.float32)
    cache = ops.DevicePagedI8Cache.from_parts(torch.from_numpy(po.key_layout(ks.codes)).cuda(), torch.from_numpy(po.value_layout(vs.codes)).cuda(),
                                              torch.from_numpy(ks.scales.copy()).cuda(), torch.from_numpy(vs.scales.copy()).cuda())
    n = len(slots)
    x = torch.tensor(rng.normal(0, 1, (n, heads + 2 * kv, hd)), device="cuda", dtype=torch.float32)  # rows of one projection: strided views
    q, k, v = x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:]
    freqs = freqs_of(hd // 2, hd)
    turned = ops.prepare_paged_attention(q, k, v, torch.tensor(freqs, device="cuda"), ints(positions), ints(slots), cache)
    ks.append(po.rotate(f64(k), positions, freqs), slots)
    vs.append(f64(v), slots)
    same_cache(cache, ks, vs)
    want = po.rotate(f64(q), positions, freqs)
    assert (np.abs(f64(turned) - want) <= 2.0 ** -23 * np.abs(want) + 1e-30).all()


@pytest.mark.parametrize("requests, most, kv, hd, rot, block", [(66, 1, 2, 64, 32, 16), (300, 4, 1, 80, 24, 32), (700, 6, 1, 32, 16, 128), (40, 5, 3, 256, 0, 64)])
def test_prepare_of_short_runs(cuda, requests, most, kv, hd, rot, block):
    """Steps of a few tokens each for many requests, among them the first and last places of a page and padded rows, over steps in which scales grow."""
    rng = np.random.default_rng(requests)
    heads, pages = 2 * kv, 2 * requests
    cache, ks, vs = ops.DevicePagedI8Cache.create(pages, block, kv, hd), po.Store(pages, block, kv, hd), po.Store(pages, block, kv, hd)
    table, lengths, freqs = rng.permutation(pages).reshape(requests, 2), rng.integers(0, 2, requests) * (block - most), freqs_of(rot, hd)
    for step in range(3):
        slots, positions = [], []
        for r in range(requests):
            for p in range(lengths[r], lengths[r] + int(rng.integers(1, most + 1))):
                slots.append(int(table[r, p // block]) * block + p % block)
                positions.append(p + 7 * r)
                lengths[r] += 1
            if r % 50 == 7:
                slots.append(-1)
                positions.append(0)
        n = len(slots)
        q, k, v = (torch.tensor(rng.normal(0, 1 + step, (n, h, hd)), device="cuda", dtype=torch.float32) for h in (heads, kv, kv))
        turned = ops.prepare_paged_attention(q, k, v, torch.tensor(freqs, device="cuda") if rot else None, ints(positions), ints(slots), cache)
        ks.append(po.rotate(f64(k), positions, freqs) if rot else f64(k), slots)
        vs.append(f64(v), slots)
        want = po.rotate(f64(q), positions, freqs) if rot else f64(q)
        live = np.array(slots) >= 0
        assert (np.abs(f64(turned) - want) <= 2.0 ** -23 * np.abs(want) + 1e-30)[live].all()
        same_cache(cache, ks, vs)


def test_values_that_are_not_finite_do_not_spoil_their_page(cuda):
    cache, ks, vs = ops.DevicePagedI8Cache.create(3, 16, 1, 32), po.Store(3, 16, 1, 32), po.Store(3, 16, 1, 32)
    x = torch.randn(6, 1, 32, generator=torch.Generator("cuda").manual_seed(1), device="cuda")
    x[1, 0, 3], x[2, 0, 4], x[3, 0, 5] = math.inf, -math.inf, math.nan
    x[5] = 0.0
    slots = [16, 17, 18, 19, 20, 33]
    ops.prepare_paged_attention(x, x, x, None, None, ints(slots), cache)
    ks.append(f64(x), slots)
    vs.append(f64(x), slots)
    same_cache(cache, ks, vs)
    k, _ = ops.paged_cache_rows(cache, ints(slots))
    assert torch.isfinite(k).all() and k[1, 0, 3] == -k[2, 0, 4] > 0 and k[3, 0, 5] == 0 and (k[5] == 0).all()


def test_ties_of_codes_go_to_even(cuda):
    cache = ops.DevicePagedI8Cache.create(1, 16, 1, 16)
    x = torch.tensor([127.0, 0.5, 1.5, 2.5, -0.5, -1.5, 63.5, 64.5, 126.5, 0.49999997, 0.50000006, 3.0, 0, 0, 0, 0], device="cuda").view(1, 1, 16)
    ops.prepare_paged_attention(x, x, x, None, None, ints([0]), cache)
    assert cache.k_codes[0, 0, 0, 0].tolist() == [127, 0, 2, 2, 0, -2, 64, 64, 126, 0, 1, 3, 0, 0, 0, 0]
    y = torch.full((1, 1, 16), 254.0, device="cuda")  # the scale doubles: codes are halved
    ops.prepare_paged_attention(y, y, y, None, None, ints([1]), cache)
    assert cache.k_codes[0, 0, 0, 0].tolist() == [64, 0, 1, 1, 0, -1, 32, 32, 63, 0, 0, 2, 0, 0, 0, 0] and cache.k_scales.item() == 2.0


def test_keys_and_values_without_queries(cuda):
    cache, ks = ops.DevicePagedI8Cache.create(2, 16, 2, 32), po.Store(2, 16, 2, 32)
    x = torch.randn(5, 4, 32, generator=torch.Generator("cuda").manual_seed(2), device="cuda")
    none = x[:, :0]
    ops.prepare_paged_attention(none, x[:, :2], x[:, 2:], torch.tensor(freqs_of(16, 32), device="cuda"), ints(range(5)), ints(range(16, 21)), cache, query_rot=none)
    ks.append(po.rotate(f64(x[:, :2]), range(5), freqs_of(16, 32)), list(range(16, 21)))
    np.testing.assert_array_equal(cache.k_codes.cpu().numpy(), po.key_layout(ks.codes))


def test_rows_outside_the_cache_are_left_as_they_were(cuda):
    cache = ops.DevicePagedI8Cache.create(2, 16, 1, 32)
    x = torch.ones(3, 1, 32, device="cuda")
    turned = torch.full_like(x, 7.0)
    ops.prepare_paged_attention(x, x, x, None, None, ints([-5, 32, 2 ** 31 - 1]), cache, query_rot=turned)
    assert (turned == 7.0).all() and not cache.k_codes.any() and not cache.k_scales.any() and not cache.v_codes.any()
    k, v = torch.full((2, 1, 32), 5.0, device="cuda"), torch.full((2, 1, 32), 6.0, device="cuda")
    ops.paged_cache_rows(cache, ints([-1, 32]), k, v)
    assert (k == 5.0).all() and (v == 6.0).all()


# ---- attention --------------------------------------------------------------------------------------------------------------
def make_attention(seed, heads, kv, hd, block, cached, new, dtype, spare_rows=0, spread=1.0):
    rng = np.random.default_rng(seed)
    blocks = [-(-(c + n) // block) for c, n in zip(cached, new)]
    pages, width = sum(blocks) + 4, max(blocks) + 2
    order, table, at = rng.permutation(pages), np.full((len(new), width), 2 ** 30), 0  # (entries behind a context lie outside the cache)
    for r, n in enumerate(blocks):
        table[r, :n] = order[at:at + n]
        at += n
    codes = [np.clip(np.rint(rng.normal(0, 36, (pages, block, kv, hd))), -127, 127) for _ in range(2)]
    scales = [(rng.uniform(0.5, 1.5, (pages, kv)) * spread ** rng.uniform(-1, 1, (pages, kv)) * 3.5 / 127).astype(np.float32) for _ in range(2)]
    cache = ops.DevicePagedI8Cache.from_parts(torch.from_numpy(po.key_layout(codes[0])).cuda(), torch.from_numpy(po.value_layout(codes[1])).cuda(),
                                              torch.from_numpy(scales[0]).cuda(), torch.from_numpy(scales[1]).cuda())
    tokens = sum(new) + spare_rows
    q = torch.tensor(rng.normal(0, 1, (tokens, heads, hd)), device="cuda").to(dtype)
    start = np.concatenate([[0], np.cumsum(new)])
    values = [c * s.astype(np.float64)[:, None, :, None] for c, s in zip(codes, scales)]
    return dict(q=q, start=start, context=[c + n for c, n in zip(cached, new)], table=table, cache=cache, values=values, most=max(new), block=block)


def attention_bound(s, want, scale, window):
    """How far a result may be off.  Scores: q is rounded to 24 bits below its row's largest entry (f32; bf16 rows to 15 or more), products are
    summed in f32, so a score is off by at most d = scale * ((hd + 16) 2^-24 sum|q k| + 2^-24 (2^-15) max|q| sum|k|), a weight by a factor of
    exp(2 d), the result by 2 d max|v|; weights to 2^-24 (bf16: 16 bits or a relative 2^-11) of the largest and their sums add
    (64 + length / 16) 2^-23 (bf16: 2^-10) of max|v|; the result is rounded once."""
    q, (k, v) = f64(s["q"]), s["values"]
    bf16 = s["q"].dtype == torch.bfloat16
    tol = np.zeros_like(want)
    group = q.shape[1] // k.shape[2]
    for r, c in enumerate(s["context"]):
        at = np.arange(max(c, 0))
        page = s["table"][r, at // s["block"]]
        page = np.where((page >= 0) & (page < k.shape[0]), page, 0)
        if not len(at):
            continue
        kk, vv = np.abs(k[page, at % s["block"]]), np.abs(v[page, at % s["block"]])
        for i in range(s["start"][r], s["start"][r + 1]):
            for h in range(q.shape[1]):
                a = np.abs(q[i, h])
                d = scale * ((q.shape[2] + 16) * 2.0 ** -24 * (kk[:, h // group] @ a).max() + 2.0 ** (-15 if bf16 else -24) * a.max() * kk[:, h // group].sum(1).max())
                tol[i, h] = vv[:, h // group].max() * (np.expm1(2 * d) + (64 + c / 16) * 2.0 ** -23 + (2.0 ** -10 if bf16 else 0.0))
    return tol + np.abs(want) * (2.0 ** -8 if bf16 else 2.0 ** -24)


def check_attention(s, window=0, scale=None, fill=9.0, **over):
    cache, q = s["cache"], s["q"]
    heads, hd = q.shape[1], q.shape[2]
    scale = 1 / math.sqrt(hd) if scale is None else scale
    out = torch.full((q.shape[0], heads * hd), fill, dtype=q.dtype, device="cuda")
    args = dict(max_query=s["most"], max_context=max(max(s["context"]), 0)) | over
    ops.paged_attention(q, ints(s["start"]), ints(s["context"]), ints(s["table"]), cache, scale=scale, window=window, out=out, **args)
    want = po.attention(f64(q), s["start"], s["context"], s["table"], s["block"], *s["values"], scale, window, np.full(q.shape, fill))
    got = f64(out).reshape(want.shape)
    off, tol = np.abs(got - want), attention_bound(s, want, scale, window)
    assert np.isfinite(got).all()
    bad = ~(off <= tol)
    assert not bad.any(), (int(bad.sum()), float((off / np.maximum(tol, 1e-300)).max()), np.argwhere(bad)[:4].tolist())
    return out


DTYPES = [torch.float32, torch.bfloat16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads, kv, hd", [(8, 2, 128), (14, 2, 64), (3, 3, 64), (16, 1, 128), (5, 1, 128), (6, 2, 80), (4, 2, 256), (2, 1, 16), (24, 1, 64)])
@pytest.mark.parametrize("block", [16, 32, 64, 128])
def test_attention_of_single_tokens(cuda, dtype, heads, kv, hd, block):
    s = make_attention(heads * hd + block, heads, kv, hd, block, [0, 1, 15, 31, 32, 33, 63, 127, 128, 500], [1] * 10, dtype)
    check_attention(s)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window", [1, 2, 16, 31, 33, 100, 5000])
@pytest.mark.parametrize("hd, block", [(128, 32), (64, 16)])
def test_attention_of_single_tokens_in_a_window(cuda, dtype, window, hd, block):
    check_attention(make_attention(window + hd, 8, 2, hd, block, [0, 1, 30, 99, 100, 101, 415], [1] * 7, dtype), window)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads, kv, hd, block, cached, new, window", [
    (8, 2, 128, 32, [0, 7, 200], [2, 3, 1], 0), (4, 4, 64, 16, [0, 60, 5], [8, 1, 5], 0), (8, 2, 128, 64, [0], [130], 0), (8, 2, 128, 64, [0, 33, 257, 3], [65, 1, 40, 0], 0),
    (7, 1, 64, 16, [100, 0], [19, 37], 50), (4, 1, 128, 128, [300], [33], 128), (4, 1, 64, 32, [129, 0, 1], [128, 129, 1], 0), (2, 2, 128, 16, [140], [257], 100),
    (6, 2, 80, 32, [20, 0], [9, 40], 0), (16, 2, 128, 32, [1000], [5], 0), (4, 2, 64, 64, [0, 0, 0], [1, 200, 64], 1)])
def test_attention_of_portions(cuda, dtype, heads, kv, hd, block, cached, new, window):
    check_attention(make_attention(sum(new) + hd, heads, kv, hd, block, cached, new, dtype, spare_rows=3), window)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [1, 40])
def test_attention_over_scales_far_apart(cuda, dtype, new):
    """Pages whose scales differ by factors of a thousand, of keys and of values."""
    check_attention(make_attention(9, 4, 2, 128, 16, [300, 77], [new, new], dtype, spread=1000.0), scale=0.02)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_over_long_contexts(cuda, dtype):
    """The context is split over thread blocks and joined; requests of very unequal length."""
    check_attention(make_attention(4, 4, 1, 128, 32, [9000, 40, 2500], [1, 1, 1], dtype))
    check_attention(make_attention(5, 4, 1, 64, 64, [5000], [24], dtype))


@pytest.mark.parametrize("new", [(1, 1, 1), (40, 1, 30)])
def test_rows_that_attend_nothing_are_zero(cuda, new):
    """A context shorter than its rows, a context of 0, pages outside the cache."""
    s = make_attention(3, 4, 2, 128, 16, [40, 20, 0], list(new), torch.float32)
    s["context"][2] = 0
    s["context"][0] = new[0] // 2
    s["table"][1, :] = -1
    out = check_attention(s)
    assert not out[s["start"][1]:].any()


@pytest.mark.parametrize("new", [1, 30])
def test_what_lies_behind_a_context_is_not_seen(cuda, new):
    """Scales and codes of pages that no request attends, NaN among them, and codes behind the last token change nothing."""
    s = make_attention(6, 8, 2, 128, 32, [50, 100], [new, new], torch.float32)
    args = (ints(s["start"]), ints(s["context"]), ints(s["table"]), s["cache"], s["most"], max(s["context"]), 0.09)
    before = ops.paged_attention(s["q"], *args).clone()
    used = {int(s["table"][r, p // 32]) for r in range(2) for p in range(s["context"][r])}
    for page in range(s["cache"].pages):
        if page not in used:
            s["cache"].k_scales[page], s["cache"].v_scales[page] = math.nan, math.inf
    for r in range(2):
        page, at = int(s["table"][r, s["context"][r] // 32]), s["context"][r] % 32
        if at:
            s["cache"].k_codes[page, :, :, at:] = 127
            for i in range(at, 32):
                s["cache"].v_codes[page, :, i // 16, :, i % 16] = -128
    assert torch.equal(ops.paged_attention(s["q"], *args), before)


def test_queries_that_are_not_finite_stay_in_their_rows(cuda):
    for new in (1, 40):
        s = make_attention(7, 8, 2, 128, 32, [70, 30], [new, new], torch.float32)
        args = (ints(s["start"]), ints(s["context"]), ints(s["table"]), s["cache"], s["most"], max(s["context"]), 0.09)
        before = ops.paged_attention(s["q"], *args).view(-1, 8, 128).clone()
        s["q"][0, 3, 5] = math.nan
        s["q"][0, 5, 7] = math.inf
        after = ops.paged_attention(s["q"], *args).view(-1, 8, 128)
        assert torch.isnan(after[0, 3]).all() and torch.isnan(after[0, 5]).all()
        keep = torch.ones(after.shape[:2], dtype=torch.bool, device="cuda")
        keep[0, 3] = keep[0, 5] = False
        assert torch.equal(after[keep], before[keep])


def test_the_bounds_choose_shares_not_results(cuda):
    for new in (1, 20):
        s = make_attention(8, 8, 2, 128, 32, [600, 30], [new, new], torch.float32)
        check_attention(s, max_context=5000)
        check_attention(s, max_context=1)
        check_attention(s, max_query=64)


def test_attention_captured_and_replayed_with_other_lengths(cuda):
    """One workspace, one graph: lengths, tables and rows change between replays; calls leave the counters as they found them."""
    a, b = (make_attention(seed, 8, 2, 128, 32, cached, [1, 1, 1], torch.float32) for seed, cached in ((1, [700, 3, 90]), (2, [5, 900, 0])))
    cache, width = a["cache"], 40
    ws = ops.paged_attention_workspace(cache, 8, 3, 3, 1, 1200)
    q, start, context, table = a["q"].clone(), ints(a["start"]), ints(a["context"]), torch.zeros(3, width, dtype=torch.int32, device="cuda")
    out = torch.zeros(3, 8 * 128, device="cuda")

    def call():
        ops.paged_attention(q, start, context, table, cache, 1, 1200, 0.09, workspace=ws, out=out)

    def set_to(s):
        q.copy_(s["q"])
        context.copy_(ints(s["context"]))
        t = np.where(s["table"] < cache.pages, s["table"], 0)
        table[:, :t.shape[1]] = ints(t)[:, :width]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        set_to(a)
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for s in (a, b, a):
        set_to(s)
        graph.replay()
        replayed = out.clone()
        call()
        assert torch.equal(out, replayed)
    if ws is not None:
        want = po.attention(f64(a["q"]), a["start"], a["context"], a["table"], 32, *a["values"], 0.09, 0, np.zeros(a["q"].shape))
        assert np.abs(f64(out).reshape(want.shape) - want).max() <= attention_bound(a, want, 0.09, 0).max()


def test_python_refuses_what_does_not_fit(cuda):
    s = make_attention(6, 8, 2, 128, 32, [50, 100], [1, 1], torch.float32)
    good = dict(query=s["q"], query_start=ints(s["start"]), context=ints(s["context"]), block_table=ints(s["table"]), cache=s["cache"], max_query=1, max_context=101, scale=0.09)
    ops.paged_attention(**good)
    for bad in (dict(query=s["q"].half()), dict(query=s["q"][:, :, :64]), dict(query_start=ints([0, 1])), dict(context=ints([1])), dict(context=ints([1, 2]).long()),
                dict(query=s["q"].transpose(0, 1)), dict(out=torch.zeros(2, 1024, device="cuda", dtype=torch.bfloat16)), dict(query=s["q"][:, :7]), dict(scale=0.0),
                dict(block_table=ints(s["table"]).t()), dict(query=s["q"].cpu())):
        with pytest.raises(KmllError):
            ops.paged_attention(**(good | bad))
    k = torch.zeros(2, 2, 128, device="cuda")
    with pytest.raises(KmllError):
        ops.prepare_paged_attention(s["q"], k, k[:1], None, None, ints([0, 1]), s["cache"])
    with pytest.raises(KmllError):
        ops.prepare_paged_attention(s["q"], k, k.transpose(1, 2).contiguous().transpose(1, 2), None, None, ints([0, 1]), s["cache"])
    with pytest.raises(KmllError):
        ops.prepare_paged_attention(s["q"], k, k, torch.ones(65, device="cuda"), ints([0, 1]), ints([0, 1]), s["cache"])
    with pytest.raises(KmllError):
        ops.paged_plan(ints([1]), ints([1]), 16, ints([[0]]), ints([0]), ints([1]), ints([0]), ints([0, 0]), ints([0]), ints([0, 0]), ints([0]), ints([0]))


# ---- all of it together -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
def test_steps_of_a_server(cuda, dtype):
    """Requests arrive, decode, end and make room; pages are used again.  Every step: plan, rotation and storage, attention over the pages, choice
    of the next tokens - against the same steps on the CPU."""
    rng = np.random.default_rng(12)
    heads, kv, hd, block, pages, width, requests, vocab = 4, 2, 64, 16, 40, 12, 5, 700
    cache = ops.DevicePagedI8Cache.create(pages, block, kv, hd)
    ks, vs = po.Store(pages, block, kv, hd), po.Store(pages, block, kv, hd)
    freqs = freqs_of(hd // 2, hd)
    freqs_dev = torch.tensor(freqs, device="cuda")
    capacity = 160
    length, table, free, count = ints([0] * requests), ints(np.full((requests, width), -1)), ints(rng.permutation(pages)), ints([pages])
    start, positions, slots, status = ints([0] * (requests + 1)), ints([0] * capacity), ints([0] * capacity), ints([0])
    cpu = dict(length=[0] * requests, table=np.full((requests, width), -1), free=free.tolist(), count=pages)
    head = torch.tensor(rng.normal(0, 0.3, (heads * hd, vocab)), device="cuda", dtype=torch.float32)
    for step in range(9):
        new = [int(rng.integers(20, 60)) if c == 0 else int(rng.integers(0, 2)) if step % 3 == 2 else 1 for c in cpu["length"]]
        new[step % requests] = 0 if step == 4 else new[step % requests]
        ops.paged_plan(length, ints(new), block, table, free, count, length, start, positions, slots, count, status)
        c = po.plan(cpu["length"], new, block, cpu["table"], cpu["free"], cpu["count"], capacity)
        assert status.item() == 0 and c[6] == 0
        for g, w in zip((length, start, table, positions, slots), c[:5]):
            np.testing.assert_array_equal(g.cpu().numpy(), w)
        cpu |= dict(length=c[0], table=c[2], count=c[5])
        q, k, v = (torch.tensor(rng.normal(0, 1, (capacity, h, hd)), device="cuda").to(dtype) for h in (heads, kv, kv))
        turned = ops.prepare_paged_attention(q, k, v, freqs_dev, positions, slots, cache, query_rot=torch.zeros_like(q))
        ks.append(po.rotate(f64(k), c[3], freqs), c[4])
        vs.append(f64(v), c[4])
        same_cache(cache, ks, vs)
        s = dict(q=turned, start=c[1], context=c[0], table=np.asarray(c[2]), cache=cache, most=max(max(new), 1), block=block,
                 values=[x.codes * x.scales.astype(np.float64)[:, None, :, None] for x in (ks, vs)])
        out = check_attention(s)
        last = [c[1][r + 1] - 1 for r in range(requests) if new[r]]
        logits = out[last].float() @ head
        u = torch.tensor(rng.random(len(last)), device="cuda")
        tokens, _ = ops.sample_rows(logits, u, torch.full((len(last),), 0.8, device="cuda"), top_p=torch.full((len(last),), 0.9, device="cuda"))
        for t, row, x in zip(tokens.tolist(), logits.double().cpu().numpy(), u.tolist()):
            want, _, gap = po.sample(row, x, float(np.float32(0.8)), 0, float(np.float32(0.9)))
            assert t == want or gap < 1e-10
        if step in (3, 6):
            ended = [1 if r % 2 == step % 2 else 0 for r in range(requests)]
            ops.paged_release(length, ints(ended), block, table, free, count, length, count, status)
            assert status.item() == 0
            cpu |= dict(length=length.tolist(), table=table.cpu().numpy(), free=free.tolist(), count=count.item())
            assert [x == 0 for x in cpu["length"]] == [bool(e) for e in ended]
    held = [p for r in range(requests) for p in cpu["table"][r, :-(-cpu["length"][r] // block)]]
    assert sorted(held + cpu["free"][:cpu["count"]]) == list(range(pages))  # no page is lost or held twice


# ---- calls that are easily forgotten ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads, kv, hd, block, cached, new, window", [
    (24, 2, 64, 32, [50, 7, 0], [1, 2, 30], 0), (12, 1, 128, 16, [400, 90], [1, 25], 64), (8, 1, 128, 64, [77, 500], [1, 2], 0), (8, 2, 64, 16, [30, 3, 260], [3, 70, 4], 0),
    (71, 1, 64, 64, [200], [1], 0), (8, 8, 128, 32, [10, 0], [16, 17], 0)])
def test_attention_of_few_rows_beside_many(cuda, dtype, heads, kv, hd, block, cached, new, window):
    """Requests on either side of the number of rows that parts the kernels."""
    check_attention(make_attention(sum(cached) + heads, heads, kv, hd, block, cached, new, dtype, spare_rows=1), window)


@pytest.mark.parametrize("dtype", DTYPES)
def test_portions_whose_keys_are_split(cuda, dtype):
    """Few units over long contexts: parts of a unit's keys in different blocks, more parts than rows' tiles, and a part without any."""
    check_attention(make_attention(31, 4, 1, 128, 64, [2600, 0], [20, 9], dtype))
    check_attention(make_attention(32, 4, 1, 64, 16, [1500], [80], dtype), window=700)
    check_attention(make_attention(33, 2, 2, 128, 128, [900, 1300], [150, 40], dtype))


def test_more_units_than_are_put_in_order(cuda):
    n = 2100
    check_attention(make_attention(34, 1, 1, 64, 16, [i % 5 for i in range(n)], [9] * n, torch.bfloat16))


def test_pages_behind_two_gigabytes(cuda):
    """Codes of a page lie more than 2^31 bytes into the cache."""
    pages, block, kv, hd = 140000, 16, 8, 128
    cache = ops.DevicePagedI8Cache.create(pages, block, kv, hd)
    assert cache.k_codes.numel() > 2 ** 31
    rng = np.random.default_rng(3)
    here = [pages - 1, 3, pages - 7]
    slots = np.concatenate([np.arange(p * block, (p + 1) * block) for p in here])[:40]
    ks, vs = po.Store(3, block, kv, hd), po.Store(3, block, kv, hd)
    small = np.concatenate([np.arange(i * block, (i + 1) * block) for i in range(3)])[:40]
    for rows, heads in ((1, 16), (40, 8)):
        k, v = (torch.tensor(rng.normal(0, 1, (40, kv, hd)), device="cuda", dtype=torch.float32) for _ in range(2))
        ops.prepare_paged_attention(k[:, :0], k, v, None, None, ints(slots), cache, query_rot=k[:, :0])
        ks.append(f64(k), small.tolist())
        vs.append(f64(v), small.tolist())
        got = ops.paged_cache_rows(cache, ints(slots))
        np.testing.assert_array_equal(got[0].cpu().numpy(), ks.rows(small))
        np.testing.assert_array_equal(got[1].cpu().numpy(), vs.rows(small))
        q = torch.tensor(rng.normal(0, 1, (rows, heads, hd)), device="cuda", dtype=torch.float32)
        out = ops.paged_attention(q, ints([0, rows]), ints([40]), ints([here]), cache, rows, 40, 0.09)
        s = dict(q=q, start=[0, rows], context=[40], table=np.array([[0, 1, 2]]), block=block, values=[x.codes * x.scales.astype(np.float64)[:, None, :, None] for x in (ks, vs)])
        want = po.attention(f64(q), s["start"], s["context"], s["table"], block, *s["values"], 0.09, 0, np.zeros(q.shape))
        assert (np.abs(f64(out).reshape(want.shape) - want) <= attention_bound(s, want, 0.09, 0)).all()


def test_requests_that_share_pages(cuda):
    """A common beginning: the same pages in two rows of the table."""
    for new in (1, 20):
        s = make_attention(41, 8, 2, 128, 16, [100, 100], [new, new], torch.float32)
        s["table"][1, :6] = s["table"][0, :6]
        check_attention(s)


def test_two_streams_at_once(cuda):
    """Calls that overlap, each with a workspace of its own; operands are waited for by the caller, as with every operator."""
    a, b = make_attention(51, 8, 2, 128, 32, [900, 30], [1, 1], torch.float32), make_attention(52, 8, 2, 128, 32, [300], [60], torch.float32)
    args = [(ints(s["start"]), ints(s["context"]), ints(s["table"]), s["cache"], s["most"], max(s["context"]), 0.09) for s in (a, b)]
    alone = [ops.paged_attention(s["q"], *x).clone() for s, x in zip((a, b), args)]
    works = [ops.paged_attention_workspace(s["cache"], 8, len(s["context"]), s["q"].shape[0], s["most"], max(s["context"])) for s in (a, b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(10):
        for i, s in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                outs[i].append(ops.paged_attention(s["q"], *args[i], workspace=works[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(o, alone[i]) for i in range(2) for o in outs[i])


def test_bf16_results_keep_nan(cuda):
    for new in (1, 40):
        s = make_attention(61, 8, 2, 128, 32, [70], [new], torch.bfloat16)
        s["q"][0, 2, 9] = math.nan
        out = ops.paged_attention(s["q"], ints(s["start"]), ints(s["context"]), ints(s["table"]), s["cache"], s["most"], max(s["context"]), 0.09).view(-1, 8, 128)
        assert torch.isnan(out[0, 2]).all() and not torch.isnan(out[0, 3]).any()
        x = s["q"][:1, :2].clone()
        x[0, 0, 0] = math.nan
        turned = ops.prepare_paged_attention(x, x, x, torch.tensor(freqs_of(64, 128), device="cuda"), ints([5]), ints([0]), ops.DevicePagedI8Cache.create(1, 16, 2, 128))
        assert torch.isnan(turned[0, 0, 0]) and torch.isnan(turned[0, 0, 64]) and not torch.isnan(turned[0, 1]).any()


def test_prompt_attention_captured_and_replayed(cuda):
    """A captured step serves other lengths, single tokens beside portions, and leaves its workspace as it found it."""
    sets = [make_attention(71 + i, 8, 2, 128, 32, cached, new, torch.float32) for i, (cached, new) in enumerate((([600, 3, 90], [1, 50, 13]), ([0, 900, 0], [62, 1, 1])))]
    width = 40
    caches = [s["cache"] for s in sets]
    cache = caches[0] if caches[0].pages >= caches[1].pages else caches[1]
    ws = ops.paged_attention_workspace(cache, 8, 3, 64, 64, 1000)
    q, start, context, table, out = torch.zeros(64, 8, 128, device="cuda"), ints([0] * 4), ints([0] * 3), ints(np.zeros((3, width))), torch.zeros(64, 1024, device="cuda")

    def call():
        ops.paged_attention(q, start, context, table, cache, 64, 1000, 0.09, workspace=ws, out=out)

    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for s in (sets[0], sets[1], sets[0]):
        q.copy_(s["q"])
        start.copy_(ints(s["start"]))
        context.copy_(ints(s["context"]))
        t = np.where(s["table"] < cache.pages, s["table"], 0)
        table.zero_()
        table[:, :t.shape[1]] = ints(t)[:, :width]
        graph.replay()
        replayed = out.clone()
        again = ops.paged_attention(q, start, context, table, cache, 64, 1000, 0.09)
        assert torch.equal(replayed, again)


def test_the_device_reports_no_time_out(cuda):
    import ctypes

    from kmll_b200 import lib
    status = ctypes.c_int(-1)
    assert lib.load().kmll_device_status(ctypes.byref(status)) == 0 and status.value == 0


def test_one_workspace_for_calls_of_any_size(cuda):
    """What has to be zero lies at the same place whatever the sizes: scratch of one call is no counter of the next."""
    small = make_attention(81, 8, 2, 128, 32, [700], [1], torch.float32)
    large = make_attention(82, 8, 2, 128, 32, [300 + 17 * i for i in range(40)], [1] * 40, torch.float32)
    mixed = make_attention(83, 8, 2, 128, 32, [900, 40, 0], [30, 1, 90], torch.float32)
    ws = ops.paged_attention_workspace(mixed["cache"], 8, 64, 200, 90, 2000)
    for s in (small, large, mixed, small, mixed, large, large, small):
        check_attention(s, workspace=ws)


@pytest.mark.parametrize("new", [1, 40])
def test_pages_of_zeros_and_tiny_values(cuda, new):
    s = make_attention(84, 4, 1, 128, 16, [200, 90], [new, new], torch.float32)
    k, v = s["values"]
    cache = s["cache"]
    cache.v_scales.mul_(1e-20)
    zero = [int(p) for p in s["table"][:, 1]] + [int(s["table"][0, 4])]
    cache.v_scales[zero] = 0.0
    cache.v_codes[zero] = 0
    cache.k_scales[int(s["table"][0, 2])] = 0.0
    vc = cache.v_codes.cpu().numpy().transpose(0, 2, 4, 1, 3).reshape(v.shape).astype(np.float64)
    kc = cache.k_codes.cpu().numpy().transpose(0, 3, 1, 2, 4).reshape(k.shape).astype(np.float64)
    s["values"] = [kc * cache.k_scales.cpu().numpy().astype(np.float64)[:, None, :, None], vc * cache.v_scales.cpu().numpy().astype(np.float64)[:, None, :, None]]
    check_attention(s)


def test_steps_without_rows(cuda):
    cache = ops.DevicePagedI8Cache.create(2, 16, 2, 64)
    none = torch.zeros(0, 4, 64, device="cuda")
    assert ops.paged_attention(none, ints([0]), ints([]), ints(np.zeros((0, 2))), cache, 0, 0, 0.1).shape == (0, 256)
    assert ops.prepare_paged_attention(none, none[:, :2], none[:, :2], None, None, ints([]), cache).shape == (0, 4, 64)
    k, v = ops.paged_cache_rows(cache, ints([]))
    assert k.shape == v.shape == (0, 2, 64)
    assert ops.sample_rows(torch.zeros(0, 32, device="cuda"), torch.zeros(0, dtype=torch.float64, device="cuda"))[0].shape == (0,)
    out = torch.full((3, 256), 7.0, device="cuda")  # rows of no request
    ops.paged_attention(torch.ones(3, 4, 64, device="cuda"), ints([0, 0, 0]), ints([5, 9]), ints(np.zeros((2, 2))), cache, 4, 16, 0.1, out=out)
    assert (out == 7.0).all()


@pytest.mark.parametrize("new", [1, 3, 40])
def test_pages_in_front_of_a_window_are_not_looked_at(cuda, new):
    """They may be another request's by now, or hold anything: scales that are not finite, and far larger ones."""
    for trouble in (math.nan, math.inf, 1e20):
        s = make_attention(85, 4, 1, 128, 16, [400, 130], [new, new], torch.float32)
        cache, table = s["cache"], s["table"]
        for r, cached in enumerate((400, 130)):
            for i in range((cached - 49) // 16):
                cache.k_scales[int(table[r, i])] = trouble
                cache.v_scales[int(table[r, i])] = trouble
        check_attention(s, window=50)


def test_value_scales_below_the_smallest_that_prompts_tell_apart(cuda):
    """Their weights still count: a row whose other keys are of ordinary size keeps its sum."""
    s = make_attention(86, 4, 1, 128, 16, [200], [40], torch.float32)
    tiny = [int(s["table"][0, i]) for i in (0, 3, 7)]
    s["cache"].v_scales[tiny] = 1e-38
    s["values"][1][tiny] *= 0.0  # (below the tolerance by 20 orders)
    check_attention(s)


def test_prompt_calls_leave_their_workspace_as_they_found_it(cuda):
    """More blocks than run at once, keys of more tiles than stay in tensor memory: the counters and flags in front are zero behind every call, and
    calls repeat themselves to the bit whichever places their blocks found."""
    for s in (make_attention(91, 8, 8, 64, 64, [1500], [1100], torch.float32), make_attention(92, 8, 2, 128, 32, [3000, 900], [40, 70], torch.float32)):
        args = (ints(s["start"]), ints(s["context"]), ints(s["table"]), s["cache"], s["most"], max(s["context"]), 0.09)
        ws = ops.paged_attention_workspace(s["cache"], 8, len(s["context"]), s["q"].shape[0], s["most"], max(s["context"]))
        front = ws[:4 * (65536 + 296 + 5)]
        first = ops.paged_attention(s["q"], *args, workspace=ws)
        assert not front.any()
        for _ in range(20):
            assert torch.equal(ops.paged_attention(s["q"], *args, workspace=ws), first)
        assert not front.any()
    check_attention(s, scale=0.09)


# ---- rows with a sink: one key far above all others, whose value is nothing ---------------------------------------------------------
def make_sink(seed, heads, kv, hd, block, context, new, dtype, nats, mean, spread=1.0):
    """Key 0 lies `nats` above the others, which score about alike; its value codes are 0, so that the row's result is what the others hold."""
    s = make_attention(seed, heads, kv, hd, block, [context - new], [new], dtype, spread=spread)
    rng, cache, table = np.random.default_rng(seed + 1), s["cache"], s["table"][0]
    pages = cache.pages
    k, v = np.rint(rng.normal(0, 36, (pages, block, kv, hd))).clip(-127, 127), np.rint(rng.normal(mean, 20, (pages, block, kv, hd))).clip(-127, 127)
    k[..., 0] = 0
    k[table[0], 0], v[table[0], 0] = 0, 0
    k[table[0], 0, :, 0] = 127
    cache.k_codes.copy_(torch.from_numpy(po.key_layout(k)))
    cache.v_codes.copy_(torch.from_numpy(po.value_layout(v)))
    cache.k_scales.fill_(1 / 127)
    s["q"][..., 0] = nats * math.sqrt(hd)
    s["v_codes"], s["v_scales"] = v, cache.v_scales.cpu().numpy().astype(np.float64)
    s["values"] = [k * float(np.float32(1 / 127)), v * s["v_scales"][:, None, :, None]]
    return s


def sink_bound(s, want, prompt):
    """Elementwise, against what the weights hold: A = sum p_j |v_j| (p of sum 1).  Scores: q is held to 2^-23 of its row's largest entry (prompts: two planes of
    binary16, 2^-22; one of bf16 rows 2^-22 as well, q being bf16), their sums and the exponent are f32: d, a factor of exp(2 d) of each weight.  Weights: single
    tokens 2^-25 (bf16: 2^-17) of the largest weight times the largest value scale in a tile of 32 keys, where none is below 2^-14 (2^-10) of that, else 2^-41 (2^-33);
    (twice that at the end of its 16 bits); prompts 2^-32 of the row's largest weight times value scale, and 2^-22
    (bf16: 2^-11) of themselves.  ex2 and the sums of a few hundred f32 terms: 2^-18 A
    (accumulators that cut: 2^-22 a tile of 128 keys)."""
    q, (k, v) = f64(s["q"]), s["values"]
    bf16, block, group = s["q"].dtype == torch.bfloat16, s["block"], q.shape[1] // k.shape[2]
    scale, c, rows, tol = 1 / math.sqrt(q.shape[2]), s["context"][0], s["start"][1], np.zeros_like(want)
    at = np.arange(c)
    page = s["table"][0, at // block]
    for i in range(rows):
        n = c - rows + i + 1
        for h in range(q.shape[1]):
            kk, vv, codes, vs = k[page[:n], at[:n] % block, h // group], v[page[:n], at[:n] % block, h // group], s["v_codes"][page[:n], at[:n] % block, h // group], s["v_scales"][page[:n], h // group]
            z = kk @ q[i, h] * scale
            p = np.exp(z - z.max())
            total, pa = p.sum(), p * vs
            d = scale * 2.0 ** (-22 if prompt else -23) * np.abs(q[i, h]).max() * np.abs(kk).sum(1).max() + 8 * 2.0 ** -24 * (np.abs(z).max() + 8)
            if prompt:
                own = 2.0 ** -32 * pa.max() * np.abs(codes).sum(0) + 2.0 ** (-11 if bf16 else -22) * (p @ np.abs(vv))
            else:
                tile = np.arange(0, n, 32)
                most = (np.maximum.reduceat(p, tile) * np.maximum.reduceat(vs, tile))[at[:n] // 32]
                own = 1.01 * (np.minimum(2.0 ** (-17 if bf16 else -25) * most, 2.0 ** (-7 if bf16 else -11) * pa) + 2.0 ** (-32 if bf16 else -40) * most) @ np.abs(codes)
            a = p @ np.abs(vv) / total
            tol[i, h] = own / total + (np.expm1(2 * d) + 2.0 ** -18 + (n / 128 * 2.0 ** -22 if prompt else 0.0)) * a
    return tol + np.abs(want) * (2.0 ** -8 if bf16 else 2.0 ** -24)


def check_sink(s, prompt):
    q = s["q"]
    out = ops.paged_attention(q, ints(s["start"]), ints(s["context"]), ints(s["table"]), s["cache"], s["most"], s["context"][0], 1 / math.sqrt(q.shape[2]))
    want = po.attention(f64(q), s["start"], s["context"], s["table"], s["block"], *s["values"], 1 / math.sqrt(q.shape[2]), 0, np.zeros(q.shape))
    off, tol = np.abs(f64(out).reshape(want.shape) - want), sink_bound(s, want, prompt)
    bad = ~(off <= tol)
    assert not bad.any(), (int(bad.sum()), float((off / tol).max()), float(np.linalg.norm(off) / np.linalg.norm(want)))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nats", [6, 12, 14, 18])
@pytest.mark.parametrize("heads, kv, hd, block, context, mean, spread", [
    (8, 2, 128, 32, 8000, 50, 1.0), (8, 2, 128, 64, 4000, 0, 1.0), (14, 2, 64, 16, 5000, 50, 1000.0), (16, 1, 128, 16, 700, 50, 1.0), (4, 4, 64, 128, 32, 50, 1.0)])
def test_single_tokens_over_a_sink(cuda, dtype, nats, heads, kv, hd, block, context, mean, spread):
    check_sink(make_sink(nats, heads, kv, hd, block, context, 1, dtype, nats, mean, spread), False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nats", [6, 12, 14, 18])
@pytest.mark.parametrize("heads, kv, hd, block, context, new, mean, spread", [(4, 1, 128, 32, 4000, 36, 50, 1.0), (4, 1, 64, 64, 6000, 10, 0, 1.0), (7, 1, 128, 16, 900, 20, 50, 1000.0)])
def test_portions_over_a_sink(cuda, dtype, nats, heads, kv, hd, block, context, new, mean, spread):
    check_sink(make_sink(nats + 100, heads, kv, hd, block, context, new, dtype, nats, mean, spread), True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads, kv, hd, new", [(4, 4, 128, 6), (8, 2, 64, 40), (2, 1, 80, 9)])
def test_windows_as_long_as_32_bits_hold(cuda, dtype, heads, kv, hd, new):
    """Rows in front of position 0 attend nothing; the distance from them to a window's first position is no 32-bit number."""
    s = make_attention(87, heads, kv, hd, 16, [30, 0, 7], [new] * 3, dtype)
    s["context"] = [new - 4, new, new + 7]  # of the first request, four rows are in front of position 0
    outs = [check_attention(s, window=w) for w in (0, 2 ** 31 - 1, 2 ** 31 - 5, 2 ** 30)]
    assert all(torch.equal(o, outs[0]) for o in outs)


@pytest.mark.parametrize("heads, kv, hd, new, most", [(4, 2, 128, [1, 3, 1], 1), (8, 2, 64, [3, 40, 20], 20), (8, 2, 128, [5, 200, 1], 100), (2, 1, 80, [1, 4, 3], 3)])
def test_requests_of_more_rows_than_announced_are_left_as_they_were(cuda, heads, kv, hd, new, most):
    s = make_attention(88, heads, kv, hd, 32, [50, 90, 400], new, torch.float32)
    out = check_attention(s, fill=9.0)
    short = torch.full_like(out, 9.0)
    ops.paged_attention(s["q"], ints(s["start"]), ints(s["context"]), ints(s["table"]), s["cache"], most, 500, 1 / math.sqrt(hd), out=short)
    a, b = s["start"][1], s["start"][2]
    assert (short[a:b] == 9.0).all()
    tol = torch.from_numpy(attention_bound(s, f64(out).reshape(s["q"].shape), 1 / math.sqrt(hd), 0)).cuda().view_as(out)
    assert ((short - out).abs() <= 2 * tol)[:a].all() and ((short - out).abs() <= 2 * tol)[b:].all()


def test_release_passes_over_entries_that_are_no_pages(cuda):
    """Two requests with a common beginning end one after the other: the shared entries of the first one to end are set to -1, and every page comes back
    once; long rows with holes anywhere come back without them."""
    table = np.full((2, 90), -1)
    table[0, :5], table[1, :6] = [10, 11, 12, 13, 14], [10, 11, 12, 15, 16, 17]
    t, c, stack, left, status = ints(table), ints([70, 96]), ints([-5] * 20), ints([0]), ints([-7])
    t[0, :3] = -1
    ops.paged_release(c, ints([1, 0]), 16, t, stack, left, c, left, status)
    assert status.item() == 0 and left.item() == 2 and stack.tolist()[:3] == [13, 14, -5] and c.tolist() == [0, 96] and t[1].tolist() == table[1].tolist()
    ops.paged_release(c, ints([1, 1]), 16, t, stack, left, c, left, status)
    assert status.item() == 0 and left.item() == 8 and sorted(stack.tolist()[:8]) == list(range(10, 18)) and (t == -1).all()
    rng = np.random.default_rng(0)
    table = rng.permutation(40 * 90).reshape(40, 90)
    table[rng.random(table.shape) < 0.3] = -1
    context, ended = rng.integers(0, 90 * 16 + 1, 40), rng.integers(0, 2, 40)
    t, c, out, left, status = ints(table), ints(context), ints([-7] * 40), ints([3]), ints([-7])
    stack = ints(np.full(4000, -9))
    ops.paged_release(c, ints(ended), 16, t, stack, left, out, left, status)
    back = [int(p) for r in range(40) if ended[r] for p in table[r, :-(-context[r] // 16)] if p >= 0]
    assert status.item() == 0 and left.item() == 3 + len(back) and stack.tolist()[:4 + len(back)] == [-9] * 3 + back + [-9]
    kept = np.where((ended[:, None] != 0) & (np.arange(90) < -(-context // 16)[:, None]), -1, table)
    np.testing.assert_array_equal(t.cpu().numpy(), kept)
    assert out.tolist() == [0 if e else x for e, x in zip(ended, context.tolist())]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads, kv, hd, new", [(8, 2, 128, 1), (14, 1, 64, 1), (8, 1, 128, 3), (4, 1, 128, 20)])
def test_queries_with_a_strong_channel(cuda, dtype, heads, kv, hd, new):
    """One entry of 5000 beside entries of about 1, over few keys that have nothing there: what is left of the others decides.  The bound is that of the rows with a
    sink, whose first term is the rounding of q below its largest entry."""
    s = make_sink(93, heads, kv, hd, 32, 11 + new, new, dtype, 0.0, 0)
    s["cache"].k_codes[:, :, 0, :, 0] = 0
    s["values"][0][..., 0] = 0.0
    s["q"][..., 0] = 5000.0
    check_sink(s, new > 3)


def test_two_long_prompts_at_once(cuda):
    """Two streams, each with a workspace of its own, whose blocks claim their places for sums side by side; a captured call among them."""
    sets = [make_attention(94 + i, 8, 4, 128, 64, [1200], [700 + 100 * i], torch.float32) for i in range(2)]
    args = [(ints(s["start"]), ints(s["context"]), ints(s["table"]), s["cache"], s["most"], max(s["context"]), 0.09) for s in sets]
    works = [ops.paged_attention_workspace(s["cache"], 8, 1, s["q"].shape[0], s["most"], max(s["context"])) for s in sets]
    alone = [ops.paged_attention(s["q"], *x).clone() for s, x in zip(sets, args)]
    outs = [[torch.zeros_like(alone[i]) for _ in range(6)] for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=streams[1]):
        for out in outs[1]:
            ops.paged_attention(sets[1]["q"], *args[1], workspace=works[1], out=out)
    torch.cuda.synchronize()
    with torch.cuda.stream(streams[1]):
        graph.replay()
    with torch.cuda.stream(streams[0]):
        for out in outs[0]:
            ops.paged_attention(sets[0]["q"], *args[0], workspace=works[0], out=out)
    torch.cuda.synchronize()
    assert all(torch.equal(o, alone[i]) for i in range(2) for o in outs[i])
    assert not any(w[:4 * (65536 + 296 + 5)].any() for w in works)


@pytest.mark.parametrize("dtype", DTYPES)
def test_sinks_of_many_requests_in_a_window(cuda, dtype):
    """Requests of unequal length whose first visible key lies far above the rest, under a window that begins at it or behind it."""
    s = make_attention(96, 8, 2, 128, 32, [300, 64, 999, 31], [1] * 4, dtype)
    k, v = s["values"]
    for r, c in enumerate(s["context"]):
        at = max(0, c - 200) if r != 1 else 0
        page, place = int(s["table"][r, at // 32]), at % 32
        s["cache"].k_codes[page, :, :, place] = 0
        s["cache"].k_codes[page, :, 0, place, 0] = 127
        s["cache"].v_codes[page, :, place // 16, :, place % 16] = 0
        k[page, place], v[page, place] = 0.0, 0.0
        k[page, place, :, 0] = 127.0 * s["cache"].k_scales[page].cpu().numpy()
    s["q"][..., 0] = 60.0
    s["q"][..., 1:] *= 0.25
    for window in (0, 200, 199, 50):
        check_attention(s, window)
