"""GPU tests of packed and paged attention at the edges of a warp, of a tile and of the mask. Compared
in 64 bits with the bound of seq_util.attention64, or with what the call gives without the odd rows."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from fp_b200 import kernels as K  # noqa: E402
from seq_util import Cache, HeadRows, starts, within  # noqa: E402
from test_gpu_sequences import copy_desc, flag, gen, paged_desc, reference, rotary_desc, run_packed, same_bits, stream  # noqa: E402

pytestmark = pytest.mark.gpu
BF16 = K.FPK_DTYPE_BF16
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
