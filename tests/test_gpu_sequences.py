"""GPU tests of the operators over heads, packed sequences and the paged cache
(fpk_qk_norm_rotary, fpk_cache_write / _read, fpk_attention_packed,
fpk_attention_paged) against plain implementations in 64 bits. Attention is compared
element by element with the bound of seq_util.attention64, which counts the kernels'
roundings; e4m3 codes, scales and 16-bit copies have to be equal."""
from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")

from fp_b200 import kernels as K  # noqa: E402
from seq_util import (DT, HALF_STEP, LAYOUTS, Cache, HeadRows, attention64, quantise, starts, within)  # noqa: E402

pytestmark = pytest.mark.gpu
F16, BF16 = K.FPK_DTYPE_F16, K.FPK_DTYPE_BF16
DEV = "cuda"


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def flag():
    return torch.zeros(1, dtype=torch.int32, device=DEV)


def stream():
    return torch.cuda.current_stream().cuda_stream


# ---------------------------------------------------------------------------
# norm and rotation

def rotate64(x, positions, inv_freq, r, interleaved, weight, eps, scale):
    y = x.double()
    if weight is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    out = y.clone()
    angle = (positions.double()[:, None] * inv_freq.double()[None])[:, None] if r else None
    if r:
        c, s = angle.cos() * scale, angle.sin() * scale
        a, b = (y[..., 0:r:2], y[..., 1:r:2]) if interleaved else (y[..., :r // 2], y[..., r // 2:r])
        u, v = (out[..., 0:r:2], out[..., 1:r:2]) if interleaved else (out[..., :r // 2], out[..., r // 2:r])
        u.copy_(a * c - b * s)
        v.copy_(b * c + a * s)
    # What a pair brings to a rounding: magnitudes of both members.
    mag = y.abs()
    if r:
        mag = mag.clone()
        lo, hi = (mag[..., 0:r:2], mag[..., 1:r:2]) if interleaved else (mag[..., :r // 2], mag[..., r // 2:r])
        both = (lo + hi) * abs(scale)
        lo.copy_(both)
        hi.copy_(both)
    return out, mag


def rotary_desc(q, k, q_out, k_out, dtype, r, interleaved, weights, positions, inv_freq, scale=1.0, eps=1e-6):
    rows, _, d = q.shape
    ptr = lambda t: t.data_ptr() if t is not None else None  # noqa: E731
    return K.QkRotaryDesc(q=q.heads, k=k.heads, q_out=q_out.heads, k_out=k_out.heads, rows=rows, q_heads=q.shape[1],
                          kv_heads=k.shape[1], head_dim=d, rotary_dim=r, interleaved=int(interleaved), q_weight=ptr(weights[0]),
                          k_weight=ptr(weights[1]), eps=eps, positions=ptr(positions), inv_freq=ptr(inv_freq),
                          rotary_scale=scale, dtype=dtype)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("rows,hq,hk,d,r,interleaved,norm,far", [
    (1, 4, 4, 128, 128, False, "both", 0), (37, 3, 1, 64, 64, True, "both", 5000), (33, 8, 2, 128, 64, False, "none", 1 << 20),
    (65, 5, 1, 96, 32, True, "q", 2 ** 31 - 70), (7, 1, 1, 256, 256, False, "k", 40000), (5, 2, 2, 8, 0, False, "both", 0),
    (130, 12, 4, 64, 16, False, "both", 777), (3, 40, 8, 128, 128, True, "none", 100)])
def test_rotary_matches_64_bits(fpk, dtype, layout, rows, hq, hk, d, r, interleaved, norm, far):
    g = gen(rows * 7 + hq)
    q, k = (HeadRows(rows, h, d, dtype, layout).set(torch.randn(rows, h, d, device=DEV, generator=g) * 2) for h in (hq, hk))
    qo, ko = (HeadRows(rows, h, d, dtype, layout).remember() for h in (hq, hk))
    w = [1 + 0.3 * torch.randn(d, device=DEV, generator=g) if norm in ("both", n) else None for n in ("q", "k")]
    pos = (far + torch.arange(rows, device=DEV)).to(torch.int32)
    inv = torch.tensor(K.rotary_frequencies(max(r, 2)), device=DEV)[:r // 2].contiguous()
    K.qk_norm_rotary(fpk, rotary_desc(q, k, qo, ko, dtype, r, interleaved, w, pos, inv, scale=0.9), stream())
    torch.cuda.synchronize()
    for x, y, weight in ((q, qo, w[0]), (k, ko, w[1])):
        ref, mag = rotate64(x.get(), pos, inv, r, interleaved, weight, 1e-6, 0.9)
        # Half a step of the type (2^-25 below fp16's normal range) and fp32 arithmetic: the norm's sum (d
        # terms), the turn (2^-23 of pi) and a handful of products.
        bound = HALF_STEP[dtype] * ref.abs() + (d / 2 + 24) * 2.0 ** -24 * mag * 1.01 + 2.0 ** -25
        assert within(y.get(), ref, bound) <= 1
        assert y.untouched_around()


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_in_place_equals_out_of_place(fpk, layout, interleaved):
    g = gen(3)
    rows, hq, hk, d, r = 45, 6, 2, 128, 64
    q, k = (HeadRows(rows, h, d, BF16, layout).set(torch.randn(rows, h, d, device=DEV, generator=g)) for h in (hq, hk))
    qo, ko = (HeadRows(rows, h, d, BF16, layout) for h in (hq, hk))
    w = [torch.rand(d, device=DEV, generator=g) + 0.5 for _ in range(2)]
    pos = torch.randint(0, 10 ** 6, (rows,), device=DEV, generator=g, dtype=torch.int32)
    inv = torch.tensor(K.rotary_frequencies(r, factor=8.0, trained_length=4096), device=DEV)
    K.qk_norm_rotary(fpk, rotary_desc(q, k, qo, ko, BF16, r, interleaved, w, pos, inv), stream())
    K.qk_norm_rotary(fpk, rotary_desc(q, k, q, k, BF16, r, interleaved, w, pos, inv), stream())
    torch.cuda.synchronize()
    assert torch.equal(q.get(), qo.get()) and torch.equal(k.get(), ko.get())


def test_rotary_between_layouts_and_one_side_only(fpk):
    """Planar projections into row-major heads, and no keys at all."""
    g = gen(4)
    q = HeadRows(50, 4, 64, F16, "planar").set(torch.randn(50, 4, 64, device=DEV, generator=g))
    a, b = HeadRows(50, 4, 64, F16, "rows").remember(), HeadRows(50, 4, 64, F16, "planar").remember()
    pos = torch.arange(50, device=DEV, dtype=torch.int32)
    inv = torch.tensor(K.rotary_frequencies(64), device=DEV)
    for out in (a, b):
        desc = rotary_desc(q, q, out, out, F16, 64, False, (None, None), pos, inv)
        desc.kv_heads = 0
        desc.k = desc.k_out = K.Heads()
        K.qk_norm_rotary(fpk, desc, stream())
    torch.cuda.synchronize()
    ref, mag = rotate64(q.get(), pos, inv, 64, False, None, 0, 1.0)
    for out in (a, b):
        assert within(out.get(), ref, HALF_STEP[F16] * ref.abs() + 60 * 2.0 ** -24 * mag + 2.0 ** -25) <= 1 and out.untouched_around()


def test_rotary_infinity_stays_in_its_pair(fpk):
    for layout in ("rows", "planar"):
        x = torch.ones(2, 1, 64)
        x[1, 0, 5] = math.inf
        x[1, 0, 60] = math.nan
        q = HeadRows(2, 1, 64, F16, layout).set(x.to(DEV))
        out = HeadRows(2, 1, 64, F16, layout)
        pos = torch.tensor([3, 4], dtype=torch.int32, device=DEV)
        inv = torch.tensor(K.rotary_frequencies(32), device=DEV)
        desc = rotary_desc(q, q, out, out, F16, 32, False, (None, None), pos, inv)
        desc.kv_heads = 0
        K.qk_norm_rotary(fpk, desc, stream())
        torch.cuda.synchronize()
        bad = ~out.get().isfinite()
        want = torch.zeros(2, 1, 64, dtype=torch.bool, device=DEV)
        want[1, 0, [5, 21, 60]] = True
        assert torch.equal(bad, want)


# ---------------------------------------------------------------------------
# cache

def copy_desc(cache, k, v, slots, dtype, err=None):
    return K.CacheCopyDesc(cache=cache.desc, k=k.heads, v=v.heads, rows=len(slots), slots=slots.data_ptr(), dtype=dtype,
                           error_flag=err.data_ptr() if err is not None else None)


def same_bits(a, b):
    if a is None:
        return b is None
    size = {1: torch.uint8, 2: torch.int16, 4: torch.int32}[a.element_size()]
    return torch.equal(a.contiguous().view(size), b.contiguous().view(size))


def rows_to_store(n, heads, d, dtype, seed):
    """Rows of very different sizes, zeros, ties of the rounding, infinities and NaN among them."""
    g = gen(seed)
    x = torch.randn(n, heads, d, device=DEV, generator=g)
    x *= torch.exp2(torch.randint(-9, 9, (n, heads, 1), device=DEV, generator=g).float())
    if n > 3:
        x[1] = 0
        x[2, 0, :5] = torch.tensor([448.0, -448.0, 17.0, 19.0, 449.0], device=DEV)
        x[3, 0, 1], x[3, 0, 2], x[3, -1, 3] = math.inf, -math.inf, math.nan
    return x.to(DT[dtype])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("n,heads,d,page", [(1, 1, 64, 16), (33, 3, 128, 16), (70, 8, 128, 64), (129, 2, 64, 256)])
def test_cache_write_and_read(fpk, dtype, e4m3, layout, n, heads, d, page):
    pages = n // page + 3
    cache, want = (Cache(pages, page, heads, d, dtype, e4m3) for _ in range(2))
    k, v = (HeadRows(n, heads, d, dtype, layout).set(rows_to_store(n, heads, d, dtype, s)).remember() for s in (1, 2))
    slots = torch.randperm(pages * page, device=DEV, generator=gen(5))[:n].to(torch.int32)
    if n > 8:
        slots[7] = -1  # a padded row
    err = flag()
    K.cache_write(fpk, copy_desc(cache, k, v, slots, dtype, err), stream())
    kept = slots >= 0
    for side, x in ((0, k), (1, v)):
        want.put(side, slots[kept], x.get()[kept])
        if e4m3:  # any NaN code will do
            a, b = cache.data[side], want.data[side]
            assert torch.equal(a.view(torch.float8_e4m3fn).float().nan_to_num(1e9), b.view(torch.float8_e4m3fn).float().nan_to_num(1e9))
        else:
            assert same_bits(cache.data[side], want.data[side])
        assert same_bits(cache.scale[side], want.scale[side])
    ko, vo = (HeadRows(n, heads, d, dtype, layout, around=7.0).remember() for _ in range(2))
    K.cache_read(fpk, copy_desc(cache, ko, vo, slots, dtype, err), stream())
    torch.cuda.synchronize()
    assert err.item() == 0
    for side, (x, src) in enumerate(((ko, k), (vo, v))):
        got = x.get()
        if e4m3:
            ref = want.values(side, slots[kept])
            top = torch.finfo(DT[dtype]).max
            ref = ref.clamp(-top, top).float().to(DT[dtype])
            assert torch.equal(got[kept].nan_to_num(1e4), ref.nan_to_num(1e4))
        else:
            assert same_bits(got[kept], src.get()[kept])
        assert (got[~kept] == 7.0).all() and x.untouched_around()


def test_cache_extremes_saturate_on_reading(fpk):
    """The largest values round up in e4m3 and come back as the type's largest; the smallest scale is 2^-100."""
    for dtype in (F16, BF16):
        top, tiny = torch.finfo(DT[dtype]).max, 2.0 ** (-24 if dtype == F16 else -120)
        x = torch.zeros(2, 1, 64, device=DEV)
        x[0, 0, 0], x[0, 0, 1], x[1, 0, 0] = top, -top, tiny
        k = HeadRows(2, 1, 64, dtype).set(x)
        cache = Cache(1, 16, 1, 64, dtype, True)
        slots = torch.tensor([3, 9], dtype=torch.int32, device=DEV)
        K.cache_write(fpk, copy_desc(cache, k, k, slots, dtype), stream())
        out = HeadRows(2, 1, 64, dtype)
        K.cache_read(fpk, copy_desc(cache, out, out, slots, dtype), stream())
        torch.cuda.synchronize()
        codes, scale = quantise(k.get())
        assert torch.equal(cache.scale[0][0, 0, [3, 9]], scale[:, 0])
        got = out.get()
        assert got[0, 0, 0].item() == top and got[0, 0, 1].item() == -top
        assert got[1, 0, 0].item() == (tiny if dtype == F16 else 0.0)


def test_cache_reports_slots_outside(fpk):
    cache, want = Cache(2, 16, 1, 64, F16), Cache(2, 16, 1, 64, F16)
    x = torch.randn(4, 1, 64, device=DEV, generator=gen(8))
    k = HeadRows(4, 1, 64, F16).set(x)
    slots = torch.tensor([5, 32, 2 ** 31 - 1, 31], dtype=torch.int32, device=DEV)
    err = flag()
    K.cache_write(fpk, copy_desc(cache, k, k, slots, F16, err), stream())
    torch.cuda.synchronize()
    want.put(0, slots[[0, 3]], k.get()[[0, 3]])
    assert err.item() == K.FPK_ERROR_SLOT and same_bits(cache.data[0], want.data[0])
    out = HeadRows(4, 1, 64, F16, around=2.0)
    err = flag()
    K.cache_read(fpk, copy_desc(cache, out, out, slots, F16, err), stream())
    torch.cuda.synchronize()
    assert err.item() == K.FPK_ERROR_SLOT and (out.get()[1:3] == 2.0).all() and same_bits(out.get()[[0, 3]], k.get()[[0, 3]])


def test_cache_offsets_past_32_bits(fpk):
    """Slots whose bytes lie beyond 4 GB of the cache, written, read and attended to."""
    heads, d, page = 8, 128, 128
    pages = (9 << 29) // (heads * d * 2 * page)  # 4.8 GB for keys, as much for values
    big = torch.empty(pages, heads, d // 8, page, 8, dtype=torch.bfloat16, device=DEV)
    big2 = torch.empty_like(big)
    cache = Cache(1, page, heads, d, BF16)
    cache.n_pages, cache.data = pages, [big, big2]
    n = 40
    k, v = (HeadRows(n, heads, d, BF16).set(torch.randn(n, heads, d, device=DEV, generator=gen(s))) for s in (1, 2))
    last = (pages - 1) * page
    slots = torch.arange(last, last + n, dtype=torch.int32, device=DEV)
    err = flag()
    K.cache_write(fpk, copy_desc(cache, k, v, slots, BF16, err), stream())
    out = HeadRows(n, heads, d, BF16), HeadRows(n, heads, d, BF16)
    K.cache_read(fpk, copy_desc(cache, *out, slots, BF16, err), stream())
    torch.cuda.synchronize()
    assert err.item() == 0 and same_bits(out[0].get(), k.get()) and same_bits(out[1].get(), v.get())
    table = torch.tensor([[pages - 1]], dtype=torch.int32, device=DEV)
    for nq in (1, 40):
        q = HeadRows(nq, heads, d, BF16).set(torch.randn(nq, heads, d, device=DEV, generator=gen(3)))
        o, err = run_paged(fpk, q, cache, [nq], torch.tensor([n], dtype=torch.int32, device=DEV), table, True, BF16)
        ref, bound = attention64(q.get().double(), k.get().double(), v.get().double(), True, d ** -0.5, BF16)
        assert err == 0 and within(o.get(), ref, bound) <= 1


# ---------------------------------------------------------------------------
# attention

def packed_desc(fpk, q, k, v, out, q_starts, kv_starts, causal, dtype, err, scale=0.0):
    desc = K.PackedAttentionDesc(q=q.heads, k=k.heads, v=v.heads, out=out.heads, q_heads=q.shape[1], kv_heads=k.shape[1],
                                 head_dim=q.shape[2], n_seq=len(q_starts) - 1, q_rows=q.shape[0], kv_rows=k.shape[0],
                                 q_starts=q_starts.data_ptr(), kv_starts=kv_starts.data_ptr(), causal=int(causal), scale=scale,
                                 dtype=dtype, error_flag=err.data_ptr())
    n = K.attention_packed_workspace_bytes(fpk, desc)
    ws = torch.full((max(n, 16),), 0xFF, dtype=torch.uint8, device=DEV)
    desc.workspace, desc.workspace_bytes = ws.data_ptr(), n
    return desc, ws


def run_packed(fpk, q, k, v, nq, nk, causal, dtype, layout="rows", scale=0.0):
    out = HeadRows(q.shape[0], q.shape[1], q.shape[2], dtype, layout, around=3.0).remember()
    err = flag()
    qs, ks = starts(nq), starts(nk)
    desc, ws = packed_desc(fpk, q, k, v, out, qs, ks, causal, dtype, err, scale)
    K.attention_packed(fpk, desc, stream())
    torch.cuda.synchronize()
    return out, err.item()


def run_paged(fpk, q, cache, nq, lengths, table, causal, dtype, layout="rows", q_starts=None, scale=0.0):
    out = HeadRows(q.shape[0], q.shape[1], q.shape[2], dtype, layout, around=3.0).remember()
    err = flag()
    qs = starts(nq) if q_starts is None else q_starts
    desc, ws = paged_desc(fpk, q, out, cache, qs, lengths, table, causal, dtype, err, scale)
    K.attention_paged(fpk, desc, stream())
    torch.cuda.synchronize()
    return out, err.item()


def paged_desc(fpk, q, out, cache, q_starts, lengths, table, causal, dtype, err, scale=0.0):
    desc = K.PagedAttentionDesc(q=q.heads, out=out.heads, cache=cache.desc, q_heads=q.shape[1], n_seq=len(q_starts) - 1,
                                q_rows=q.shape[0], q_starts=q_starts.data_ptr(), kv_lengths=lengths.data_ptr(),
                                page_table=table.data_ptr(), table_pages=table.shape[1], causal=int(causal), scale=scale,
                                dtype=dtype, error_flag=err.data_ptr())
    n = K.attention_paged_workspace_bytes(fpk, desc)
    ws = torch.full((max(n, 16),), 0xFF, dtype=torch.uint8, device=DEV)
    desc.workspace, desc.workspace_bytes = ws.data_ptr(), n
    return desc, ws


def reference(q, k, v, nq, nk, causal, d, dtype, scale=0.0, v_step=None):
    """All sequences; rows of none are left at 3 (what run_packed fills in)."""
    out = torch.full(q.shape, 3.0, dtype=torch.float64, device=DEV)
    bound = torch.zeros_like(out)
    a = b = 0
    for x, y in zip(nq, nk):
        o, e = attention64(q.get()[a:a + x].double(), k[b:b + y], v[b:b + y], causal, scale or d ** -0.5, dtype, v_step)
        out[a:a + x], bound[a:a + x] = o, e
        a, b = a + x, b + y
    return out, bound


SHAPES = [  # query rows, key rows (None: the same), query heads, key heads, d, causal, rows behind the last sequence
    ([1], None, 1, 1, 64, True, 0),
    ([5, 0, 1, 17, 3], None, 4, 4, 128, False, 6),
    ([64, 1, 127, 128, 129], None, 4, 2, 128, True, 3),
    ([7, 3, 20], [0, 3, 9], 8, 2, 64, True, 1),      # rows that see nothing
    ([1, 1, 1], [500, 64, 1], 32, 8, 128, False, 0),
    ([300], [1000], 8, 1, 128, True, 0),
    ([77, 200, 0], [13, 333, 50], 6, 2, 64, False, 5),
    ([16, 2], [2500, 700], 20, 4, 128, True, 0),
    ([513], None, 3, 3, 64, True, 2),
    ([2, 1], [40, 30], 96, 2, 64, True, 0),          # 48 query heads to a key head
    ([100], [0], 2, 1, 128, False, 0),
]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_packed_attention_matches_64_bits(fpk, dtype, layout, case):
    nq, nk, hq, hk, d, causal, spare = SHAPES[case]
    nk = list(nq) if nk is None else nk
    g = gen(case)
    q = HeadRows(sum(nq) + spare, hq, d, dtype, layout).set(torch.randn(sum(nq) + spare, hq, d, device=DEV, generator=g) * 2)
    k, v = (HeadRows(sum(nk) + spare, hk, d, dtype, layout).set(torch.randn(sum(nk) + spare, hk, d, device=DEV, generator=g)) for _ in range(2))
    # Rows of no sequence hold what must not reach a result.
    for x, n in ((q, sum(nq)), (k, sum(nk)), (v, sum(nk))):
        x.v[n:] = math.nan
    out, err = run_packed(fpk, q, k, v, nq, nk, causal, dtype, layout)
    ref, bound = reference(q, k.get().double(), v.get().double(), nq, nk, causal, d, dtype)
    assert err == 0
    assert within(out.get(), ref, bound) <= 1
    assert out.untouched_around()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("page", [16, 64, 1024])
@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_paged_attention_matches_64_bits(fpk, dtype, e4m3, page, case):
    nq, nk, hq, hk, d, causal, spare = SHAPES[case]
    nk = list(nq) if nk is None else nk
    g = gen(100 + case)
    need = [-(-n // page) for n in nk]
    width = max(max(need), 1) + 1
    pages = sum(need) + 2
    order = torch.randperm(pages, device=DEV, generator=g).to(torch.int32)
    table = torch.full((len(nk), width), 2 ** 30, dtype=torch.int32, device=DEV)  # unused entries are not read
    cache = Cache(pages, page, hk, d, dtype, e4m3)  # stale slots hold NaN
    ks, vs, at = [], [], 0
    for s, n in enumerate(nk):
        table[s, :need[s]] = order[at:at + need[s]]
        at += need[s]
        i = torch.arange(n, device=DEV)
        slots = table[s].long()[i // page] * page + i % page
        for side, keep, spread in ((0, ks, 0.0), (1, vs, 4.0)):
            x = torch.randn(n, hk, d, device=DEV, generator=g)
            x = (x * torch.exp2(spread * torch.randn(n, hk, 1, device=DEV, generator=g).clamp(-2, 2))).to(DT[dtype])
            cache.put(side, slots, x)
            keep.append(cache.values(side, slots))
    layout = LAYOUTS[case % 4]
    q = HeadRows(sum(nq) + spare, hq, d, dtype, layout).set(torch.randn(sum(nq) + spare, hq, d, device=DEV, generator=g) * 2)
    lengths = torch.tensor(nk, dtype=torch.int32, device=DEV)
    out, err = run_paged(fpk, q, cache, nq, lengths, table, causal, dtype, layout)
    v_step = 448.0 * float(cache.scale[1].nan_to_num(0).max()) if e4m3 else None
    ref, bound = reference(q, torch.cat(ks), torch.cat(vs), nq, nk, causal, d, dtype, v_step=v_step)
    assert err == 0
    assert within(out.get(), ref, bound) <= 1
    assert out.untouched_around()


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("nq", [1, 3, 150])
def test_long_cache_is_split_and_joined(fpk, nq, e4m3):
    """Few rows over many keys: every CTA works on a part of the axis, whose partials are joined."""
    hq, hk, d, page, n = 8, 2, 128, 64, 20011
    g = gen(nq)
    cache = Cache(n // page + 1, page, hk, d, BF16, e4m3)
    table = torch.randperm(n // page + 1, device=DEV, generator=g).to(torch.int32)[None]
    i = torch.arange(n, device=DEV)
    slots = table[0].long()[i // page] * page + i % page
    # Later keys weigh more, so that the running maximum moves from part to part.
    k = (torch.randn(n, hk, d, device=DEV, generator=g) * torch.linspace(0.1, 2.0, n, device=DEV)[:, None, None]).to(torch.bfloat16)
    v = torch.randn(n, hk, d, device=DEV, generator=g).to(torch.bfloat16)
    cache.put(0, slots, k)
    cache.put(1, slots, v)
    q = HeadRows(nq, hq, d, BF16).set(torch.randn(nq, hq, d, device=DEV, generator=g))
    lengths = torch.tensor([n], dtype=torch.int32, device=DEV)
    out, err = run_paged(fpk, q, cache, [nq], lengths, table, True, BF16)
    v_step = 448.0 * float(cache.scale[1].nan_to_num(0).max()) if e4m3 else None
    ref, bound = reference(q, cache.values(0, slots), cache.values(1, slots), [nq], [n], True, d, BF16, v_step=v_step)
    assert err == 0 and within(out.get(), ref, bound) <= 1
    again, _ = run_paged(fpk, q, cache, [nq], lengths, table, True, BF16)
    assert same_bits(out.get(), again.get())


@pytest.mark.parametrize("rows", [3, 200])
def test_masks_hide_infinities(fpk, rows):
    """A score of the type's lowest value, keys that are infinite where the causal mask hides them, and
    rows whose every score is -inf."""
    d = 64
    g = gen(rows)
    q = HeadRows(rows, 2, d, F16).set(torch.rand(rows, 2, d, device=DEV, generator=g) + 0.1)
    k = HeadRows(rows, 2, d, F16).set(torch.randn(rows, 2, d, device=DEV, generator=g))
    v = HeadRows(rows, 2, d, F16).set(torch.randn(rows, 2, d, device=DEV, generator=g))
    k.v[rows - 1] = math.inf       # seen by the last query only
    k.v[1] = -65504.0              # a very low score for everybody
    out, err = run_packed(fpk, q, k, v, [rows], [rows], True, F16)
    ref, bound = reference(q, k.get().double(), v.get().double(), [rows], [rows], True, d, F16)
    assert err == 0 and within(out.get()[:rows - 1], ref[:rows - 1], bound[:rows - 1]) <= 1
    assert out.get()[rows - 1].isnan().all()


def test_scale_is_used(fpk):
    g = gen(1)
    for rows in (4, 140):
        q, k, v = (HeadRows(rows, 2, 128, BF16).set(torch.randn(rows, 2, 128, device=DEV, generator=g)) for _ in range(3))
        out, _ = run_packed(fpk, q, k, v, [rows], [rows], False, BF16, scale=0.02)
        ref, bound = reference(q, k.get().double(), v.get().double(), [rows], [rows], False, 128, BF16, scale=0.02)
        assert within(out.get(), ref, bound) <= 1


@pytest.mark.parametrize("nq", [1, 90])
def test_bad_pages_and_lengths_are_reported(fpk, nq):
    """A page number outside the cache hides its keys; a length past the table is clamped; starts
    that pass the buffer are. Nothing outside the buffers is read."""
    hk, d, page = 2, 64, 16
    cache = Cache(4, page, hk, d, F16)
    g = gen(6)
    slots = torch.arange(64, device=DEV)
    x = torch.randn(64, hk, d, device=DEV, generator=g).to(torch.float16)
    cache.put(0, slots, x)
    cache.put(1, slots, x)
    q = HeadRows(nq, hk, d, F16).set(torch.randn(nq, hk, d, device=DEV, generator=g))
    lengths = torch.tensor([60], dtype=torch.int32, device=DEV)
    for bad in (4, -1, 2 ** 31 - 1):
        table = torch.tensor([[2, bad, 0, 3]], dtype=torch.int32, device=DEV)
        out, err = run_paged(fpk, q, cache, [nq], lengths, table, False, F16)
        keep = torch.cat([slots[32:48], slots[0:16], slots[48:60]])
        ref, bound = reference(q, x[keep].double(), x[keep].double(), [nq], [44], False, d, F16)
        assert err == K.FPK_ERROR_PAGE and within(out.get(), ref, bound) <= 1
    table = torch.tensor([[2, 1, 0, 3]], dtype=torch.int32, device=DEV)
    for length, keys in ((65, 64), (2 ** 31 - 1, 64), (-5, 0)):
        out, err = run_paged(fpk, q, cache, [nq], torch.tensor([length], dtype=torch.int32, device=DEV), table, False, F16)
        keep = torch.cat([slots[32:48], slots[16:32], slots[0:16], slots[48:64]])[:keys]
        ref, bound = reference(q, x[keep].double(), x[keep].double(), [nq], [keys], False, d, F16)
        assert err == K.FPK_ERROR_LENGTH and within(out.get(), ref, bound) <= 1
    bad_starts = torch.tensor([0, nq + 7], dtype=torch.int32, device=DEV)
    out, err = run_paged(fpk, q, cache, [nq], lengths, table, False, F16, q_starts=bad_starts)
    keep = torch.cat([slots[32:48], slots[16:32], slots[0:16], slots[48:64]])[:60]
    ref, bound = reference(q, x[keep].double(), x[keep].double(), [nq], [60], False, d, F16)
    assert err == K.FPK_ERROR_STARTS and within(out.get(), ref, bound) <= 1 and out.untouched_around()


# ---------------------------------------------------------------------------
# together, as they are used

def test_block_from_gemm_to_cached_tokens(fpk):
    """A transformer block's attention: QKV projection (fpk_gemm, planar), norm and rotation in place,
    the prompt by fpk_attention_packed, its rows into a cache, then two more tokens one by one by
    fpk_attention_paged. Every step is checked in 64 bits on what the step before left, and the
    cached prompt gives the packed result."""
    from kp8_util import Planar

    hq, hk, d, dt = 4, 2, 128, F16
    heads = hq + 2 * hk
    lengths = [50, 131]
    total = sum(lengths)
    extra = 2
    rows = total + extra * len(lengths)
    g = torch.Generator().manual_seed(0)
    x = Planar(rows, 512, torch.float16).set((torch.randn(rows, 512, generator=g)).to(DEV))
    w = (torch.randn(heads * d, 512, generator=g) / 512 ** 0.5).to(DEV).to(torch.float16)
    bias = torch.zeros(heads * d, device=DEV)
    qkv = Planar(rows, heads * d, torch.float16)
    err = flag()
    desc = K.GemmDesc(a=x.base, a_plane_stride=x.plane_stride, rows=rows, cin=512, taps=1, w=w.data_ptr(), cout=heads * d,
                      bias=bias.data_ptr(), dst=qkv.base, dst_plane_stride=qkv.plane_stride, dst_mode=K.FPK_DST_SAME, img_rows=rows,
                      grid_w=rows, valid_h=1, valid_w=rows, dtype=dt, error_flag=err.data_ptr())
    K.gemm(fpk, desc, stream())
    torch.cuda.synchronize()
    proj = qkv.get().reshape(rows, heads, d).clone()
    ref = (x.get().double() @ w.double().T).reshape(rows, heads, d)
    assert (proj.double() - ref).abs().max() <= 2.0 ** -11 * ref.abs().max() * 1.1
    view = lambda channel: K.Heads.planar(qkv.base, qkv.plane_stride, d, channel)  # noqa: E731
    pos = torch.cat([torch.arange(n) for n in lengths] + [torch.tensor([n + e]) for e in range(extra) for n in lengths]).to(torch.int32).to(DEV)
    inv = torch.tensor(K.rotary_frequencies(d), device=DEV)
    wq, wk = torch.rand(d, device=DEV) + 0.5, torch.rand(d, device=DEV) + 0.5
    K.qk_norm_rotary(fpk, K.QkRotaryDesc(q=view(0), k=view(hq * d), q_out=view(0), k_out=view(hq * d), rows=rows, q_heads=hq, kv_heads=hk,
                                         head_dim=d, rotary_dim=d, q_weight=wq.data_ptr(), k_weight=wk.data_ptr(), eps=1e-6,
                                         positions=pos.data_ptr(), inv_freq=inv.data_ptr(), rotary_scale=1.0, dtype=dt), stream())
    torch.cuda.synchronize()
    now = qkv.get().reshape(rows, heads, d)
    for part, weight in ((slice(0, hq), wq), (slice(hq, hq + hk), wk)):
        ref, mag = rotate64(proj[:, part], pos, inv, d, False, weight, 1e-6, 1.0)
        assert within(now[:, part], ref, HALF_STEP[dt] * ref.abs() + 90 * 2.0 ** -24 * mag + 2.0 ** -25) <= 1
    assert torch.equal(now[:, hq + hk:], proj[:, hq + hk:])
    q, k, v = (now[:, a:b].double() for a, b in ((0, hq), (hq, hq + hk), (hq + hk, heads)))

    out = Planar(rows, hq * d, torch.float16)
    out_heads = K.Heads.planar(out.base, out.plane_stride, d)
    st = starts(lengths)
    packed = K.PackedAttentionDesc(q=view(0), k=view(hq * d), v=view((hq + hk) * d), out=out_heads, q_heads=hq, kv_heads=hk, head_dim=d,
                                   n_seq=2, q_rows=total, kv_rows=total, q_starts=st.data_ptr(), kv_starts=st.data_ptr(), causal=1, dtype=dt,
                                   error_flag=err.data_ptr())
    ws = torch.empty(max(16, K.attention_packed_workspace_bytes(fpk, packed)), dtype=torch.uint8, device=DEV)
    packed.workspace, packed.workspace_bytes = ws.data_ptr(), ws.numel()
    K.attention_packed(fpk, packed, stream())
    torch.cuda.synchronize()
    got = out.get().reshape(rows, hq, d)
    at = 0
    for n in lengths:
        ref, bound = attention64(q[at:at + n], k[at:at + n], v[at:at + n], True, d ** -0.5, dt)
        assert within(got[at:at + n], ref, bound) <= 1
        at += n
    assert torch.count_nonzero(got[total:]) == 0

    page = 32
    cache = Cache(16, page, hk, d, dt)
    table = torch.randperm(16, generator=g).to(torch.int32).reshape(2, 8).to(DEV)
    slot = lambda s, i: table[s].long()[i // page] * page + i % page  # noqa: E731
    slots = torch.cat([slot(s, torch.arange(n, device=DEV)) for s, n in enumerate(lengths)]
                      + [slot(s, torch.tensor([n + e], device=DEV)) for e in range(extra) for s, n in enumerate(lengths)]).to(torch.int32)

    def write(first, n):
        K.cache_write(fpk, K.CacheCopyDesc(cache=cache.desc, k=K.Heads.planar(qkv.base + first * 16, qkv.plane_stride, d, hq * d),
                                           v=K.Heads.planar(qkv.base + first * 16, qkv.plane_stride, d, (hq + hk) * d), rows=n,
                                           slots=slots[first:].data_ptr(), dtype=dt, error_flag=err.data_ptr()), stream())

    def attend(first, n_rows, q_starts, kv_lengths):
        p = K.PagedAttentionDesc(q=K.Heads.planar(qkv.base + first * 16, qkv.plane_stride, d), out=K.Heads.planar(out.base + first * 16, out.plane_stride, d),
                                 cache=cache.desc, q_heads=hq, n_seq=2, q_rows=n_rows, q_starts=q_starts.data_ptr(),
                                 kv_lengths=kv_lengths.data_ptr(), page_table=table.data_ptr(), table_pages=8, causal=1, dtype=dt,
                                 error_flag=err.data_ptr())
        w2 = torch.empty(max(16, K.attention_paged_workspace_bytes(fpk, p)), dtype=torch.uint8, device=DEV)
        p.workspace, p.workspace_bytes = w2.data_ptr(), w2.numel()
        K.attention_paged(fpk, p, stream())
        torch.cuda.synchronize()

    write(0, total)
    before = got.clone()
    attend(0, total, st, torch.tensor(lengths, dtype=torch.int32, device=DEV))
    got = out.get().reshape(rows, hq, d)
    assert torch.equal(got[:total], before[:total])
    for e in range(extra):
        first = total + e * 2
        write(first, 2)
        attend(first, 2, torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV), torch.tensor([n + e + 1 for n in lengths], dtype=torch.int32, device=DEV))
        got = out.get().reshape(rows, hq, d)
        at = 0
        for s, n in enumerate(lengths):
            own = torch.cat([torch.arange(at, at + n)] + [torch.tensor([total + i * 2 + s]) for i in range(e + 1)]).to(DEV)
            ref, bound = attention64(q[first + s:first + s + 1], k[own], v[own], True, d ** -0.5, dt)
            assert within(got[first + s:first + s + 1], ref, bound) <= 1
            at += n
    assert err.item() == 0


def test_captured_calls_follow_the_device_values(fpk):
    """One captured token step (rotate, write, attend) replayed for growing sequences on a side stream,
    and two captured graphs with a workspace each replayed on two streams at once."""
    hq, hk, d, page, dt = 8, 2, 64, 16, BF16
    n_seq, width = 3, 40
    g = gen(9)
    cache = Cache(n_seq * width, page, hk, d, dt, True)
    table = torch.arange(n_seq * width, dtype=torch.int32, device=DEV).reshape(n_seq, width)
    q_in, k_in, v_in = (HeadRows(n_seq, h, d, dt) for h in (hq, hk, hk))
    q, k = HeadRows(n_seq, hq, d, dt), HeadRows(n_seq, hk, d, dt)
    pos = torch.zeros(n_seq, dtype=torch.int32, device=DEV)
    lengths = torch.zeros(n_seq, dtype=torch.int32, device=DEV)
    slots = torch.zeros(n_seq, dtype=torch.int32, device=DEV)
    inv = torch.tensor(K.rotary_frequencies(d), device=DEV)
    qs = starts([1] * n_seq)
    err = flag()
    outs, graphs, keep = [], [], []
    rot = rotary_desc(q_in, k_in, q, k, dt, d, False, (None, None), pos, inv)
    wr = copy_desc(cache, k, v_in, slots, dt, err)
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(2):
        out = HeadRows(n_seq, hq, d, dt, around=0.0)
        desc, ws = paged_desc(fpk, q, out, cache, qs, lengths, table, True, dt, err)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side[i]):
            s = torch.cuda.current_stream().cuda_stream
            if i == 0:
                K.qk_norm_rotary(fpk, rot, s)
                K.cache_write(fpk, wr, s)
            K.attention_paged(fpk, desc, s)
        outs.append(out)
        graphs.append(graph)
        keep.append((desc, ws))
    ks, vs = [[] for _ in range(n_seq)], [[] for _ in range(n_seq)]
    for step in range(40):
        for x in (q_in, k_in, v_in):
            x.set(torch.randn(x.shape, device=DEV, generator=g))
        pos.fill_(step)
        lengths.copy_(torch.tensor([step + 1, step // 2 + 1, 1]))  # sequence 1 grows every other step, 2 stays
        at = torch.tensor([step, step // 2, 0], device=DEV)
        slots.copy_(table[torch.arange(n_seq, device=DEV), at // page] * page + at % page)
        torch.cuda.synchronize()
        graphs[0].replay()
        torch.cuda.synchronize()
        first = outs[0].get().clone()
        for graph, s in zip(graphs, side):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        assert same_bits(first, outs[0].get()) and same_bits(first, outs[1].get())
        for s in range(n_seq):
            n = int(lengths[s])
            i = torch.arange(n, device=DEV)
            sl = table[s].long()[i // page] * page + i % page
            ref, bound = attention64(q.get()[s:s + 1].double(), cache.values(0, sl), cache.values(1, sl), True, d ** -0.5, dt,
                                     448.0 * float(cache.scale[1].nan_to_num(0).max()))
            assert within(first[s:s + 1], ref, bound) <= 1
    assert err.item() == 0


def test_refuses_memory_that_is_not_on_the_device(fpk):
    x = torch.zeros(4, 1, 64, dtype=torch.float16).pin_memory()
    q = HeadRows(4, 1, 64, F16)
    pos = torch.zeros(4, dtype=torch.int32, device=DEV)
    inv = torch.ones(32, device=DEV)
    desc = rotary_desc(q, q, q, q, F16, 64, False, (None, None), pos, inv)
    desc.q.data = x.data_ptr()
    with pytest.raises(K.FpkError, match="device memory"):
        K.qk_norm_rotary(fpk, desc, stream())
