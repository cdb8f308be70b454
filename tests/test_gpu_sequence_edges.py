"""GPU tests of packed and paged attention at the edges of a warp, of a tile and of the mask. Compared
in 64 bits with the bound of seq_util.attention64, or with what the call gives without the odd rows."""
from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")

from fp_b200 import kernels as K  # noqa: E402
from seq_util import DT, Cache, HeadRows, attention64, starts, within  # noqa: E402
from test_gpu_sequences import copy_desc, flag, gen, packed_desc, paged_desc, reference, rotary_desc, run_packed, run_paged, same_bits, stream  # noqa: E402

pytestmark = pytest.mark.gpu
F16, BF16 = K.FPK_DTYPE_F16, K.FPK_DTYPE_BF16
DEV = "cuda"


@pytest.mark.parametrize("last", [1, 31, 33, 95])
@pytest.mark.parametrize("split", [False, True])
def test_warps_with_and_without_rows(fpk, last, split):
    """Tiles whose last warp has rows in some of its lanes: whole (many short sequences), and cut over
    CTAs (one sequence, many keys)."""
    hq, hk, d = 4, 4, 128
    nq, nk = ([128 + last], [6000]) if split else ([128 + last, last + 17, 256 + last] * 12, None)
    nk = list(nq) if nk is None else nk
    g = gen(last)
    q = HeadRows(sum(nq) + 3, hq, d, BF16).set(torch.randn(sum(nq) + 3, hq, d, device=DEV, generator=g))
    k, v = (HeadRows(sum(nk), hk, d, BF16).set(torch.randn(sum(nk), hk, d, device=DEV, generator=g)) for _ in range(2))
    out, err = run_packed(fpk, q, k, v, nq, nk, not split, BF16)
    ref, bound = reference(q, k.get().double(), v.get().double(), nq, nk, not split, d, BF16)
    assert err == 0 and within(out.get(), ref, bound) <= 1 and out.untouched_around()


@pytest.mark.parametrize("nq", [1, 5, 300])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("layout", ["planar", "rows"])
def test_calls_read_what_the_call_before_wrote(fpk, nq, e4m3, layout):
    """A step's calls one behind the other, where each begins while the one before still runs: what they
    read (rows, scales, and slots, lengths and page numbers too) is new each time, in memory that the
    step before read. Every step gives what it gives with a wait behind every call."""
    n, hq, hk, d, page = 500, 8, 2, 128, 32
    g = gen(nq)
    pages = -(-n // page)
    inv = torch.tensor(K.rotary_frequencies(d), device=DEV)
    w = [torch.rand(d, device=DEV, generator=g) + 0.5 for _ in range(2)]
    steps = []
    for _ in range(6):
        order = torch.randperm(pages, device=DEV, generator=g).to(torch.int32)
        at = torch.arange(n, device=DEV)
        steps.append(dict(q=torch.randn(nq, hq, d, device=DEV, generator=g), k=torch.randn(n, hk, d, device=DEV, generator=g),
                          v=torch.randn(n, hk, d, device=DEV, generator=g), table=order, length=int(torch.randint(nq, n + 1, (), device=DEV, generator=g)),
                          slots=(order.long()[at // page] * page + at % page).to(torch.int32),
                          pos=torch.randint(0, 9000, (n,), device=DEV, generator=g, dtype=torch.int32)))

    def run(wait):
        q, k, v = (HeadRows(r, h, d, BF16, layout) for r, h in ((nq, hq), (n, hk), (n, hk)))
        out = HeadRows(nq, hq, d, BF16, layout)
        cache = Cache(pages, page, hk, d, BF16, e4m3)
        table, slots, pos = torch.zeros(1, pages, dtype=torch.int32, device=DEV), *(torch.zeros(n, dtype=torch.int32, device=DEV) for _ in range(2))
        length, qs, err = torch.zeros(1, dtype=torch.int32, device=DEV), starts([nq]), flag()
        none = HeadRows(n, 0, d, BF16, "rows")
        turn_q = rotary_desc(q, none, q, none, BF16, d, False, w, pos, inv)
        turn_k = rotary_desc(none, k, none, k, BF16, d, False, w, pos, inv)
        turn_q.rows = nq
        write = copy_desc(cache, k, v, slots, BF16, err)
        attend, ws = paged_desc(fpk, q, out, cache, qs, length, table, True, BF16, err)
        results = []
        for s in steps:
            for x, name in ((q, "q"), (k, "k"), (v, "v")):
                x.set(s[name])
            table[0], slots[:], pos[:] = s["table"], s["slots"], s["pos"]
            length.fill_(s["length"])
            for call, desc in ((K.qk_norm_rotary, turn_q), (K.qk_norm_rotary, turn_k), (K.cache_write, write), (K.attention_paged, attend)):
                call(fpk, desc, stream())
                if wait:
                    torch.cuda.synchronize()
            results.append(out.get().clone())
        torch.cuda.synchronize()
        assert err.item() == 0
        return results

    want = run(True)
    for _ in range(5):
        for a, b in zip(run(False), want):
            assert same_bits(a, b)


def one_cached(keys, k, v, dtype, page, g, e4m3=True):
    """One sequence in a paged cache: (cache, table, length, slots)."""
    pages = -(-keys // page)
    cache = Cache(pages, page, k.shape[1], k.shape[2], dtype, e4m3)
    table = torch.randperm(pages, device=DEV, generator=g).to(torch.int32)[None]
    at = torch.arange(keys, device=DEV)
    slots = table[0].long()[at // page] * page + at % page
    cache.put(0, slots, k.to(DT[dtype]))
    cache.put(1, slots, v.to(DT[dtype]))
    return cache, table, torch.tensor([keys], dtype=torch.int32, device=DEV), slots


def value_step(cache, slots):
    """448 times the largest scale of a row of values that is not all zeros: what attention64's bound counts
    the rounding of probabilities in. A row of zeros brings nothing to a product, whatever its scale is."""
    values = cache.values(1, slots)
    p, r = slots.long() // cache.page_rows, slots.long() % cache.page_rows
    scale = cache.scale[1][p, :, r].double()
    return 448.0 * float((scale * (values.abs().amax(-1) > 0)).max())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("nq,n", [(1, 300), (4, 300), (20, 300), (1, 20011), (150, 9000)])
@pytest.mark.parametrize("size", [1e-2, 1e-3, 1e-5])
@pytest.mark.parametrize("top", [False, True])
@pytest.mark.parametrize("d", [64, 128])
def test_rows_of_zeros_beside_small_values(fpk, dtype, nq, n, size, top, d):
    """Values of `size` with some rows of zeros (their scale is 1, far above the others'), the first, the
    last and more, which may have the highest scores. Values are positive, so that the bound is relative
    to each output."""
    hq, hk, page = 4, 2, 64
    g = gen(nq + n)
    q = HeadRows(nq, hq, d, dtype).set(0.75 + 0.5 * torch.rand(nq, hq, d, device=DEV, generator=g))
    k = 0.3 * torch.randn(n, hk, d, device=DEV, generator=g)
    v = size * (0.5 + torch.rand(n, hk, d, device=DEV, generator=g))
    rows = torch.tensor([0, 1, 17, n // 2, n // 2 + 40, n - 1], device=DEV)
    v[rows] = 0
    v[3, 0], v[n // 3, 1] = 0, 0  # in one head only
    if top:
        k[rows] = 0.05 * 128 / d ** 0.5 + 0.1 * torch.rand(len(rows), hk, d, device=DEV, generator=g)
    cache, table, length, slots = one_cached(n, k, v, dtype, page, g)
    out, err = run_paged(fpk, q, cache, [nq], length, table, False, dtype)
    ref, bound = reference(q, cache.values(0, slots), cache.values(1, slots), [nq], [n], False, d, dtype, v_step=value_step(cache, slots))
    # fp16's own rounding of an output below its normal range.
    bound = bound - 2.0 ** -24 + (2.0 ** -25 if dtype == F16 else 0.0)
    assert err == 0 and within(out.get(), ref, bound) <= 1


@pytest.mark.parametrize("nq,n", [(1, 300), (1, 20011), (150, 9000)])
def test_only_rows_of_zeros(fpk, nq, n):
    g = gen(n)
    q = HeadRows(nq, 4, 128, BF16).set(torch.randn(nq, 4, 128, device=DEV, generator=g))
    k = torch.randn(n, 2, 128, device=DEV, generator=g)
    cache, table, length, _ = one_cached(n, k, torch.zeros_like(k), BF16, 64, g)
    out, err = run_paged(fpk, q, cache, [nq], length, table, True, BF16)
    assert err == 0 and torch.count_nonzero(out.get()) == 0


@pytest.mark.parametrize("nq,n", [(1, 300), (5, 900), (1, 20011), (150, 9000)])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("first", [False, True])
@pytest.mark.parametrize("cached", ["packed", "same", "e4m3"])
def test_small_weights_beside_a_large_one_fp16(fpk, nq, n, d, first, cached):
    """One key with a score 19 above the others (their weights are some 2^-27 of its) and small values: the
    output is the others'. Their probabilities count to 2^-32 of the largest one: attention64's bound
    with its 2^-25 taken by 2^-7."""
    hq, hk = 4, 2
    g = gen(n)
    q = HeadRows(nq, hq, d, F16).set(torch.ones(nq, hq, d, device=DEV) + 0.05 * torch.randn(nq, hq, d, device=DEV, generator=g))
    k = 0.05 * torch.randn(n, hk, d, device=DEV, generator=g)
    v = 0.5 + torch.rand(n, hk, d, device=DEV, generator=g)
    at = 0 if first else n - 1
    k[at] += 19.0 / d ** 0.5
    v[at] *= 2.0 ** -24
    if cached == "packed":
        kr, vr = HeadRows(n, hk, d, F16).set(k), HeadRows(n, hk, d, F16).set(v)
        out, err = run_packed(fpk, q, kr, vr, [nq], [n], False, F16)
        kk, vv, step = kr.get().double(), vr.get().double(), 1.5
    else:
        cache, table, length, slots = one_cached(n, k, v, F16, 64, g, cached == "e4m3")
        out, err = run_paged(fpk, q, cache, [nq], length, table, False, F16)
        kk, vv = cache.values(0, slots), cache.values(1, slots)
        step = 1.5
    if cached == "e4m3":  # units of a row's scale: the largest product of weight and scale is the bound's unit
        p = torch.softmax(torch.einsum("qhd,khd->hqk", q.get().double(), kk.repeat_interleave(hq // hk, 1)) * d ** -0.5, -1)
        pg, r = slots.long() // cache.page_rows, slots.long() % cache.page_rows
        scale = cache.scale[1][pg, :, r].double().repeat_interleave(hq // hk, 1).T[:, None]
        step = 448.0 * float((p * scale).max())
    ref, bound = reference(q, kk, vv, [nq], [n], False, d, F16, v_step=step * 2.0 ** -7)
    bound = bound - 2.0 ** -24 + 2.0 ** -25
    assert err == 0 and within(out.get(), ref, bound) <= 1


# (query rows, key rows) of a sequence whose first queries see nothing, and what it takes: the streaming
# kernel's clusters (one CTA, several) and shares with a join, the tile kernel whole and cut.
BLIND = [([7], [3]), ([16, 2], [10, 1]), ([900], [860]), ([30] * 140, [21] * 140), ([600] * 40, [560] * 40), ([250], [9000]), ([300] + [1] * 199, [292] + [1] * 199)]


def with_bad_rows(x, rows, kind):
    """NaN, infinities or both in `rows` of x [n, heads, d]: one channel, or all of them."""
    x = x.clone()
    d = x.shape[2]
    if kind == "nan":
        x[rows, :, 5] = math.nan
    elif kind == "inf":
        x[rows, 0, d - 1], x[rows, -1, 8] = math.inf, -math.inf
    else:
        x[rows] = math.nan
    return x


@pytest.mark.parametrize("case", range(len(BLIND)))
@pytest.mark.parametrize("kind", ["nan", "inf", "all"])
@pytest.mark.parametrize("paged", [False, True])
def test_rows_that_see_nothing_are_zero_beside_bad_values(fpk, case, kind, paged):
    nq, nk = BLIND[case]
    hq, hk, d = 4, 2, 64
    g = gen(case)
    q = HeadRows(sum(nq), hq, d, F16).set(torch.randn(sum(nq), hq, d, device=DEV, generator=g))
    k = torch.randn(sum(nk), hk, d, device=DEV, generator=g)
    last = torch.tensor(nk, device=DEV).cumsum(0) - 1
    v = with_bad_rows(torch.randn(sum(nk), hk, d, device=DEV, generator=g), last, kind)
    if paged:
        width = -(-max(nk) // 16)
        cache = Cache(width * len(nk), 16, hk, d, F16)
        table = torch.randperm(width * len(nk), device=DEV, generator=g).to(torch.int32).reshape(len(nk), width)
        seq = torch.repeat_interleave(torch.arange(len(nk), device=DEV), torch.tensor(nk, device=DEV))
        i = torch.arange(sum(nk), device=DEV) - starts(nk)[seq].long()
        slots = table.long()[seq, i // 16] * 16 + i % 16
        cache.put(0, slots, k.half())
        cache.put(1, slots, v.half())
        out, err = run_paged(fpk, q, cache, nq, torch.tensor(nk, dtype=torch.int32, device=DEV), table, True, F16)
    else:
        out, err = run_packed(fpk, q, HeadRows(sum(nk), hk, d, F16).set(k), HeadRows(sum(nk), hk, d, F16).set(v), nq, nk, True, F16)
    got, at = out.get(), 0
    for x, y in zip(nq, nk):
        assert torch.count_nonzero(got[at:at + max(x - y, 0)]) == 0
        at += x
    assert err == 0


# (query rows, key rows, query heads, key heads, kernel): bad values among the keys that the last queries
# alone see, for every way through the kernels.
HIDDEN = {
    "cluster": ([6], [300], 8, 2), "one-cta": ([5, 1, 9], [70, 3, 9], 4, 4), "cluster-16": ([16], [500], 4, 2),
    "shares": ([7], [9000], 4, 2), "shares-many": ([13] * 150, [40] * 150, 2, 1), "shares-edge": ([300] + [1] * 199, [420] + [1] * 199, 4, 2),
    "tiles": ([300, 70, 513] * 8, None, 4, 4), "tiles-grouped": ([90, 200, 333] * 8, [700, 200, 400] * 8, 16, 2), "tiles-cut": ([250], [9000], 4, 2),
    "tiles-long": ([3000], None, 2, 1),
}


def seen_bad(v, first, hq, d):
    """What queries add to their sums from bad values of v [n, hk, d]: query i sees keys below first[i]."""
    n, hk, _ = v.shape
    big = n + 1
    key = torch.arange(n, device=v.device)[:, None, None]
    plus = torch.where((v == math.inf) | v.isnan(), key, big).amin(0)
    minus = torch.where((v == -math.inf) | v.isnan(), key, big).amin(0)
    see = lambda t: (t[None] < first[:, None, None]).repeat_interleave(hq // hk, 1)  # noqa: E731
    add = torch.zeros(len(first), hq, d, device=v.device)
    add[see(plus)] = math.inf
    add[see(minus)] += -math.inf
    return add


@pytest.mark.parametrize("name", HIDDEN)
@pytest.mark.parametrize("kind", ["nan", "inf", "all"])
@pytest.mark.parametrize("dtype,cached,layout,d,page", [(F16, "packed", "rows", 64, 0), (BF16, "packed", "planar", 128, 0), (BF16, "same", "rows", 128, 16),
                                                       (F16, "same", "rows", 64, 64), (BF16, "e4m3", "planar", 128, 32), (F16, "e4m3", "rows", 64, 16)])
def test_bad_values_reach_only_the_queries_that_see_them(fpk, name, kind, dtype, cached, layout, d, page):
    """Against 64 bits with zeros in their place, and what an infinity or NaN makes of the channels of the
    queries that see it."""
    nq, nk, hq, hk = HIDDEN[name]
    nk = list(nq) if nk is None else nk
    g = gen(len(name) + d)
    q = HeadRows(sum(nq), hq, d, dtype, layout).set(torch.randn(sum(nq), hq, d, device=DEV, generator=g))
    k = torch.randn(sum(nk), hk, d, device=DEV, generator=g)
    clean = torch.randn(sum(nk), hk, d, device=DEV, generator=g)
    bad, rows, first, at = clean, [], [], 0
    for x, y in zip(nq, nk):
        # Keys that the last query, some of the last ones and half of them see first, and one that all do.
        rows += [at + y - 1, at + y - 1 - (min(x, y) - 1) // 3, at + y - 1 - (min(x, y) - 1) // 2] + ([at] if len(rows) % 2 else [])
        first.append(at + y - x + 1 + torch.arange(x, device=DEV))
        at += y
    rows = torch.tensor(sorted(set(rows)), device=DEV)
    bad = with_bad_rows(clean, rows[::2], kind)
    bad = with_bad_rows(bad, rows[1::2], "nan" if kind == "nan" else "inf")
    if cached == "e4m3":
        bad = torch.where(bad.isfinite(), bad, math.nan)  # as the cache holds them
    zeroed = torch.where(bad.isfinite(), bad, 0.0)
    if cached == "packed":
        kr, vr = HeadRows(sum(nk), hk, d, dtype, layout).set(k), HeadRows(sum(nk), hk, d, dtype, layout).set(bad)
        out, err = run_packed(fpk, q, kr, vr, nq, nk, True, dtype, layout)
        kk, vv, step = kr.get().double(), zeroed.to(DT[dtype]).double(), None
    else:
        width = -(-max(nk) // page)
        cache = Cache(width * len(nk), page, hk, d, dtype, cached == "e4m3")
        table = torch.arange(width * len(nk) - 1, -1, -1, dtype=torch.int32, device=DEV).reshape(len(nk), width).contiguous()
        seq = torch.repeat_interleave(torch.arange(len(nk), device=DEV), torch.tensor(nk, device=DEV))
        i = torch.arange(sum(nk), device=DEV) - starts(nk)[seq].long()
        slots = table.long()[seq, i // page] * page + i % page
        cache.put(0, slots, k.to(DT[dtype]))
        cache.put(1, slots, bad.to(DT[dtype]))
        kk, vv = cache.values(0, slots), cache.values(1, slots).nan_to_num(0, 0, 0)
        out, err = run_paged(fpk, q, cache, nq, torch.tensor(nk, dtype=torch.int32, device=DEV), table, True, dtype, layout)
        step = 448.0 * float(cache.scale[1].nan_to_num(0).max()) if cached == "e4m3" else None
    ref, bound = reference(q, kk, vv, nq, nk, True, d, dtype, v_step=step)
    add, at_q, at_k = torch.empty(sum(nq), hq, d, device=DEV), 0, 0
    for x, y, f in zip(nq, nk, first):
        add[at_q:at_q + x] = seen_bad(bad[at_k:at_k + y], f - at_k, hq, d)
        at_q, at_k = at_q + x, at_k + y
    got, fine = out.get(), add == 0
    assert err == 0 and fine.any() and not fine.all()
    assert within(got[fine], ref[fine], bound[fine]) <= 1
    assert torch.equal(got[~fine].float().nan_to_num(1.0, 2.0, 3.0), add[~fine].nan_to_num(1.0, 2.0, 3.0))


@pytest.mark.parametrize("name", HIDDEN)
@pytest.mark.parametrize("which", ["k", "v", "all"])
def test_nothing_but_nan_comes_to_an_end(fpk, name, which):
    nq, nk, hq, hk = HIDDEN[name]
    nk = list(nq) if nk is None else nk
    g = gen(1)
    q, k, v = (HeadRows(n, h, 64, BF16).set(torch.randn(n, h, 64, device=DEV, generator=g)) for n, h in ((sum(nq), hq), (sum(nk), hk), (sum(nk), hk)))
    for x, n in ((q, "q"), (k, "k"), (v, "v")):
        if which in (n, "all"):
            x.v.fill_(math.nan)
    out, err = run_packed(fpk, q, k, v, nq, nk, True, BF16)
    assert err == 0 and out.untouched_around()
    at = 0
    for x, y in zip(nq, nk):
        blind = max(x - y, 0)
        assert torch.count_nonzero(out.get()[at:at + blind]) == 0 and out.get()[at + blind:at + x].isnan().all()
        at += x


@pytest.mark.parametrize("paged", [False, True])
def test_a_cut_tile_of_a_failed_cta_is_not_stored(fpk, paged):
    """A CTA that counts as one whose wait ran out (nothing waits here): the tiles that it has a piece of
    keep what the output held, the others are as ever, and the next call is whole again."""
    nq, n, hq, hk, d = 200, 9000, 6, 3, 64
    g = gen(2)
    q = HeadRows(nq, hq, d, F16).set(torch.randn(nq, hq, d, device=DEV, generator=g))
    k, v = (torch.randn(n, hk, d, device=DEV, generator=g) for _ in range(2))
    if paged:
        cache, table, length, _ = one_cached(n, k, v, F16, 32, g, False)
        run = lambda: run_paged(fpk, q, cache, [nq], length, table, True, F16)  # noqa: E731
    else:
        kr, vr = HeadRows(n, hk, d, F16).set(k), HeadRows(n, hk, d, F16).set(v)
        run = lambda: run_packed(fpk, q, kr, vr, [nq], [n], True, F16)  # noqa: E731
    whole = run()[0].get().clone()
    missing = torch.zeros(nq, hq, dtype=torch.bool, device=DEV)
    try:
        for share in (0, 1, 5, 70, 147, 10 ** 6):
            assert fpk.lib.fpk_attention_test_fail_share(share) == -1
            out, err = run()
            assert fpk.lib.fpk_attention_test_fail_share(-1) == share and err == 0
            kept = (out.get() == 3.0).all(-1)  # what run_packed and run_paged fill in
            assert torch.equal(torch.where(kept[..., None], whole, out.get()), whole)
            # Tiles: 256 rows of (token, head of the group) of one key head; a share lies in one or two.
            tiles = kept.reshape(nq, hk, hq // hk).permute(1, 0, 2).reshape(hk, -1)
            count = sum(bool(tiles[h, a:a + 256].any()) for h in range(hk) for a in (0, 256))
            assert all(tiles[h, a:a + 256].any() == tiles[h, a:a + 256].all() for h in range(hk) for a in (0, 256))
            assert (1 <= count <= 2) if share < 148 else count == 0
            missing |= kept
    finally:
        fpk.lib.fpk_attention_test_fail_share(-1)
    assert missing.any() and not missing.all() and same_bits(run()[0].get(), whole)


def test_every_pointer_must_be_on_the_device(fpk):
    """A host array in the place of any pointer of a call is refused before a kernel could read it."""
    host = torch.zeros(1 << 16, dtype=torch.uint8)
    address = -(-host.data_ptr() // 16) * 16
    d, n = 64, 20
    q, k, v, out, ko = (HeadRows(n, h, d, F16).set(torch.zeros(n, h, d, device=DEV)) for h in (4, 2, 2, 4, 2))
    g = gen(1)
    ints = torch.zeros(n, dtype=torch.int32, device=DEV)
    floats = torch.ones(d, device=DEV)
    err, qs = flag(), starts([n])
    cache, table, length, slots = one_cached(n, k.get(), v.get(), F16, 16, g)
    rotary = lambda: rotary_desc(q, k, out, ko, F16, d, False, (floats, floats), ints, floats)  # noqa: E731
    copy = lambda: copy_desc(cache, k, v, slots.to(torch.int32), F16, err)  # noqa: E731
    packed = lambda: packed_desc(fpk, q, k, v, out, qs, qs, True, F16, err)[0]  # noqa: E731
    paged = lambda: paged_desc(fpk, q, out, cache, qs, length, table, True, F16, err)[0]  # noqa: E731
    scales = ["cache.k", "cache.v", "cache.k_scale", "cache.v_scale"]
    for call, make, names in ((K.qk_norm_rotary, rotary, ["q.data", "k.data", "q_out.data", "k_out.data", "q_weight", "k_weight", "positions", "inv_freq"]),
                              (K.cache_write, copy, scales + ["k.data", "v.data", "slots", "error_flag"]),
                              (K.cache_read, copy, scales + ["k.data", "v.data", "slots", "error_flag"]),
                              (K.attention_packed, packed, ["q.data", "k.data", "v.data", "out.data", "q_starts", "kv_starts", "error_flag", "workspace"]),
                              (K.attention_paged, paged, scales + ["q.data", "out.data", "q_starts", "kv_lengths", "page_table", "error_flag", "workspace"])):
        for name in names:
            desc = make()
            at = desc
            for part in name.split(".")[:-1]:
                at = getattr(at, part)
            setattr(at, name.split(".")[-1], address)
            with pytest.raises(K.FpkError, match="device memory"):
                call(fpk, desc, stream())
    torch.cuda.synchronize()


@pytest.mark.parametrize("tiles", [False, True])
def test_most_sequences_nearly_all_empty(fpk, tiles):
    """2^20 sequences of which the first and the last have rows: a walk over all the others ends in time."""
    n_seq, d, hk = 1 << 20, 64, 1
    hq = 128 if tiles else 2
    nq = [70000, 62000] if tiles else [300, 200]
    g = gen(1)
    q = HeadRows(sum(nq), hq, d, F16, around=0.0).set(torch.randn(sum(nq), hq, d, device=DEV, generator=g))
    # Many rows of keys, of which 400 are some sequence's: the choice of the kernel goes by the average.
    k, v = (HeadRows(300000, hk, d, F16).set(torch.randn(300000, hk, d, device=DEV, generator=g)) for _ in range(2))
    out = HeadRows(sum(nq), hq, d, F16, around=3.0)
    qs, ks = torch.full((n_seq + 1,), nq[0], dtype=torch.int32, device=DEV), torch.full((n_seq + 1,), 250, dtype=torch.int32, device=DEV)
    qs[0], qs[-1], ks[0], ks[-1] = 0, sum(nq), 0, 400
    err = flag()
    desc, ws = packed_desc(fpk, q, k, v, out, qs, ks, False, F16, err)
    K.attention_packed(fpk, desc, stream())
    torch.cuda.synchronize()
    assert err.item() == 0
    few = torch.randperm(sum(nq), device=DEV, generator=g)[:200].sort().values
    for rows, keys in ((few[few < nq[0]], slice(0, 250)), (few[few >= nq[0]], slice(250, 400))):
        kk, vv = (x.get()[keys].double() for x in (k, v))
        ref, bound = attention64(q.get()[rows].double(), kk, vv, False, d ** -0.5, F16)
        assert within(out.get()[rows], ref, bound) <= 1
