"""GPU tests of packed and paged attention where their splits, statistics and
checks are at their limits: maxima that grow inside a block of keys, batches of
more sequences than a CTA has threads, starts that overlap, caches with unusual
scales, two calls at once, replayed prompts. Compared in 64 bits with the bound of
seq_util.attention64."""
from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")

from fp_b200 import kernels as K  # noqa: E402
from seq_util import DT, Cache, HeadRows, attention64, starts, within  # noqa: E402
from test_gpu_sequences import flag, gen, packed_desc, paged_desc, reference, run_packed, run_paged, same_bits, stream  # noqa: E402

pytestmark = pytest.mark.gpu
F16, BF16 = K.FPK_DTYPE_F16, K.FPK_DTYPE_BF16
DEV = "cuda"


def scores_of(kind, n, g):
    """Scores (natural) along the keys: the running maximum moves inside blocks of 64 and of 128."""
    j = torch.arange(n, device=DEV).float()
    if kind == "ramp":
        return 0.15 * j
    if kind == "fall":
        return -0.15 * j
    if kind == "steps":  # up by 12 in the middle of each 128 keys
        return 12.0 * ((j + 64) // 128)
    spikes = torch.zeros(n, device=DEV)
    at = torch.randperm(n, device=DEV, generator=g)[:20].sort().values
    spikes[at] = torch.arange(1, 21, device=DEV).float() * 6.0
    return spikes


def one_table(n, page, g):
    pages = -(-n // page)
    table = torch.randperm(pages, device=DEV, generator=g).to(torch.int32)[None]
    i = torch.arange(n, device=DEV)
    return table, table[0].long()[i // page] * page + i % page


@pytest.mark.parametrize("kind", ["ramp", "fall", "steps", "spikes"])
@pytest.mark.parametrize("nq", [3, 130, 300])
@pytest.mark.parametrize("cached", ["packed", "same", "e4m3"])
def test_maximum_moves_inside_a_block(fpk, kind, nq, cached):
    n, hq, hk, d, page = 700, 4, 2, 128, 64
    g = gen(len(kind) + nq)
    q = HeadRows(nq, hq, d, BF16).set(0.75 + 0.5 * torch.rand(nq, hq, d, device=DEV, generator=g))
    k = scores_of(kind, n, g)[:, None, None] + 0.5 * torch.randn(n, hk, d, device=DEV, generator=g)
    v = torch.randn(n, hk, d, device=DEV, generator=g)
    if cached == "packed":
        kr, vr = HeadRows(n, hk, d, BF16).set(k), HeadRows(n, hk, d, BF16).set(v)
        out, err = run_packed(fpk, q, kr, vr, [nq], [n], True, BF16, scale=1.0 / d)
        kk, vv, v_step = kr.get().double(), vr.get().double(), None
    else:
        cache = Cache(-(-n // page), page, hk, d, BF16, cached == "e4m3")
        table, slots = one_table(n, page, g)
        cache.put(0, slots, k.to(DT[BF16]))
        cache.put(1, slots, v.to(DT[BF16]))
        out, err = run_paged(fpk, q, cache, [nq], torch.tensor([n], dtype=torch.int32, device=DEV), table, True, BF16, scale=1.0 / d)
        kk, vv = cache.values(0, slots), cache.values(1, slots)
        v_step = 448.0 * float(cache.scale[1].nan_to_num(0).max()) if cached == "e4m3" else None
    ref, bound = reference(q, kk, vv, [nq], [n], True, d, BF16, scale=1.0 / d, v_step=v_step)
    assert err == 0 and within(out.get(), ref, bound) <= 1


@pytest.mark.parametrize("most", [3, 150])
@pytest.mark.parametrize("paged", [False, True])
def test_more_sequences_than_threads(fpk, most, paged):
    """700 sequences of 0 to `most` rows: the search for a CTA's first sequence takes several passes."""
    n_seq, hq, hk, d, page = 700, 2, 1, 64, 16
    g = gen(most)
    nq = torch.randint(0, most + 1, (n_seq,), device=DEV, generator=g)
    nq[torch.randperm(n_seq, device=DEV, generator=g)[:60]] = 0
    nq = nq.tolist()
    rows = sum(nq)
    q, k, v = (HeadRows(rows + 5, h, d, F16).set(torch.randn(rows + 5, h, d, device=DEV, generator=g)) for h in (hq, hk, hk))
    if paged:
        width = -(-most // page)
        cache = Cache(n_seq * width, page, hk, d, F16)
        table = torch.randperm(n_seq * width, device=DEV, generator=g).to(torch.int32).reshape(n_seq, width)
        seq = torch.repeat_interleave(torch.arange(n_seq, device=DEV), torch.tensor(nq, device=DEV))
        i = torch.arange(rows, device=DEV) - starts(nq)[seq].long()
        slots = table.long()[seq, i // page] * page + i % page
        cache.put(0, slots, k.get()[:rows])
        cache.put(1, slots, v.get()[:rows])
        out, err = run_paged(fpk, q, cache, nq, torch.tensor(nq, dtype=torch.int32, device=DEV), table, True, F16)
    else:
        out, err = run_packed(fpk, q, k, v, nq, nq, True, F16)
    ref, bound = reference(q, k.get().double(), v.get().double(), nq, nq, True, d, F16)
    assert err == 0 and within(out.get(), ref, bound) <= 1 and out.untouched_around()


@pytest.mark.parametrize("rows,keys", [(20, 100), (20, 9000), (400, 500)])
def test_starts_that_overlap_are_reported(fpk, rows, keys):
    """Starts that go back: whatever the results are, the call ends, reports it and stays in its buffers."""
    hq, hk, d = 4, 2, 64
    g = gen(rows)
    q = HeadRows(rows, hq, d, F16).set(torch.randn(rows, hq, d, device=DEV, generator=g))
    k, v = (HeadRows(keys, hk, d, F16).set(torch.randn(keys, hk, d, device=DEV, generator=g)) for _ in range(2))
    for qs, ks in (([0, rows, rows // 3, rows], [0, 50, 80, keys]), ([0, 5, 9, rows], [keys, 0, keys, 7]), ([rows, 0, -4, rows + 9], [0, keys, 0, keys]),
                   ([0, 2 ** 31 - 1, -2 ** 31, rows], [-2 ** 31, 2 ** 31 - 1, 0, keys])):
        out = HeadRows(rows, hq, d, F16, around=3.0).remember()
        err = flag()
        qs, ks = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in (qs, ks))
        desc, ws = packed_desc(fpk, q, k, v, out, qs, ks, True, F16, err)
        K.attention_packed(fpk, desc, stream())
        torch.cuda.synchronize()
        assert err.item() == K.FPK_ERROR_STARTS and out.untouched_around()


@pytest.mark.parametrize("nq", [2, 100])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_e4m3_rows_of_unusual_scales(fpk, nq, dtype):
    """Keys and values from 2^-40 to 2^14 in one cache, rows of zeros, and a row with a NaN, which only
    the queries that see it get."""
    n, hq, hk, d, page = 300, 4, 2, 64, 32
    g = gen(nq)
    cache = Cache(-(-n // page), page, hk, d, dtype, True)
    table, slots = one_table(n, page, g)
    size = torch.exp2(torch.randint(-40, 1, (n, hk, 1), device=DEV, generator=g).float())
    k = (torch.randn(n, hk, d, device=DEV, generator=g) * size).to(DT[dtype])
    size = torch.exp2(torch.randint(-40 if dtype == BF16 else -14, 13, (n, hk, 1), device=DEV, generator=g).float())
    v = (torch.randn(n, hk, d, device=DEV, generator=g) * size).to(DT[dtype])
    k[5], v[6] = 0, 0
    k[n - 1, 1, 3] = math.nan
    cache.put(0, slots, k)
    cache.put(1, slots, v)
    q = HeadRows(nq, hq, d, dtype).set(torch.randn(nq, hq, d, device=DEV, generator=g))
    out, err = run_paged(fpk, q, cache, [nq], torch.tensor([n], dtype=torch.int32, device=DEV), table, True, dtype)
    v_step = 448.0 * float(cache.scale[1].nan_to_num(0).max())
    ref, bound = reference(q, cache.values(0, slots), cache.values(1, slots), [nq], [n], True, d, dtype, v_step=v_step)
    got = out.get()
    assert err == 0 and got[-1, hq // hk:].isnan().all()
    assert within(got[:-1], ref[:-1], bound[:-1]) <= 1 and within(got[-1:, :hq // hk], ref[-1:, :hq // hk], bound[-1:, :hq // hk]) <= 1


def test_prompts_and_tokens_at_once(fpk):
    """A prompt's attention and a token's, with a workspace each, on two streams, captured and replayed
    while the other runs: every time what each gives alone."""
    d, page = 128, 16
    g = gen(4)
    nq = [700, 33, 1, 900]
    q, k, v = (HeadRows(sum(nq), h, d, BF16).set(torch.randn(sum(nq), h, d, device=DEV, generator=g)) for h in (8, 2, 2))
    out = HeadRows(sum(nq), 8, d, BF16, around=0.0)
    n = 9000
    cache = Cache(-(-n // page), page, 2, d, BF16)
    table, slots = one_table(n, page, g)
    for side in range(2):
        cache.put(side, slots, torch.randn(n, 2, d, device=DEV, generator=g).to(DT[BF16]))
    q1 = HeadRows(1, 8, d, BF16).set(torch.randn(1, 8, d, device=DEV, generator=g))
    out1 = HeadRows(1, 8, d, BF16, around=0.0)
    err = flag()
    qs, qs1, lengths = starts(nq), starts([1]), torch.tensor([n], dtype=torch.int32, device=DEV)
    prompt, ws = packed_desc(fpk, q, k, v, out, qs, qs, True, BF16, err)
    token, ws1 = paged_desc(fpk, q1, out1, cache, qs1, lengths, table, True, BF16, err)
    K.attention_packed(fpk, prompt, stream())
    K.attention_paged(fpk, token, stream())
    torch.cuda.synchronize()
    alone, alone1 = out.get().clone(), out1.get().clone()
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    graphs = []
    for s, call, desc in ((side[0], K.attention_packed, prompt), (side[1], K.attention_paged, token)):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            call(fpk, desc, torch.cuda.current_stream().cuda_stream)
            call(fpk, desc, torch.cuda.current_stream().cuda_stream)  # again behind itself: one workspace in turn
        graphs.append(graph)
    for _ in range(5):
        out.v.fill_(0)
        out1.v.fill_(0)
        torch.cuda.synchronize()
        for graph, s in zip(graphs, side):
            with torch.cuda.stream(s):
                for _ in range(3):
                    graph.replay()
        torch.cuda.synchronize()
        assert same_bits(out.get(), alone) and same_bits(out1.get(), alone1)
    assert err.item() == 0


@pytest.mark.parametrize("nq,nk", [(1, 1), (1, 64), (1, 65), (16, 127), (17, 128), (64, 4097), (65, 4097), (128, 129), (129, 255), (256, 256), (257, 1),
                                   (1, 4096), (1, 4097), (33, 2047)])
@pytest.mark.parametrize("causal", [False, True])
def test_sizes_around_tiles_and_variants(fpk, nq, nk, causal):
    hq, hk, d = 6, 2, 64
    g = gen(nq * 7 + nk)
    q = HeadRows(nq, hq, d, F16).set(torch.randn(nq, hq, d, device=DEV, generator=g))
    k, v = (HeadRows(nk, hk, d, F16).set(torch.randn(nk, hk, d, device=DEV, generator=g)) for _ in range(2))
    out, err = run_packed(fpk, q, k, v, [nq], [nk], causal, F16)
    ref, bound = reference(q, k.get().double(), v.get().double(), [nq], [nk], causal, d, F16)
    assert err == 0 and within(out.get(), ref, bound) <= 1 and out.untouched_around()
