"""CPU: what the calls over heads, packed sequences and the paged cache refuse before they reach
CUDA, empty calls, and the table of rotary frequencies."""
from __future__ import annotations

import math

import pytest

from fp_b200 import kernels as K

F16, BF16, E4M3 = K.FPK_DTYPE_F16, K.FPK_DTYPE_BF16, K.FPK_DTYPE_E4M3
A = 1 << 20  # an address that is never followed


@pytest.fixture(scope="module")
def fl():
    return K.FpkLibrary()


def heads(**kw):
    return K.Heads(**{**dict(data=A, head_stride=256, row_stride=2048, plane_stride=16), **kw})


def rotary(**kw):
    return K.QkRotaryDesc(**{**dict(q=heads(), k=heads(), q_out=heads(), k_out=heads(), rows=4, q_heads=8, kv_heads=2, head_dim=128,
                                    rotary_dim=128, q_weight=A, k_weight=A, eps=1e-6, positions=A, inv_freq=A, rotary_scale=1.0,
                                    dtype=BF16), **kw})


def cache(**kw):
    return K.KvCache(**{**dict(k=A, v=A, n_pages=8, page_rows=16, kv_heads=2, head_dim=64, dtype=F16), **kw})


def copy(**kw):
    return K.CacheCopyDesc(**{**dict(cache=cache(), k=heads(), v=heads(), rows=4, slots=A, dtype=F16), **kw})


def packed(**kw):
    return K.PackedAttentionDesc(**{**dict(q=heads(), k=heads(), v=heads(), out=heads(), q_heads=8, kv_heads=2, head_dim=64, n_seq=2,
                                           q_rows=10, kv_rows=10, q_starts=A, kv_starts=A, dtype=F16, workspace=A,
                                           workspace_bytes=1 << 40), **kw})


def paged(**kw):
    return K.PagedAttentionDesc(**{**dict(q=heads(), out=heads(), cache=cache(), q_heads=8, n_seq=2, q_rows=2, q_starts=A, kv_lengths=A,
                                          page_table=A, table_pages=4, dtype=F16, workspace=A, workspace_bytes=1 << 40), **kw})


REFUSED = [
    (K.qk_norm_rotary, rotary, [
        (dict(dtype=K.FPK_DTYPE_F32), "dtype"), (dict(head_dim=100), "sizes"), (dict(head_dim=264), "sizes"), (dict(rows=-1), "sizes"),
        (dict(q_heads=-1), "sizes"), (dict(q_heads=65535), "sizes"), (dict(rotary_dim=24), "rotary_dim"), (dict(rotary_dim=144), "rotary_dim"),
        (dict(q=heads(data=None)), "null"), (dict(k_out=heads(data=None)), "null"), (dict(q=heads(data=A + 8)), "16 bytes"),
        (dict(k=heads(row_stride=2056)), "16 bytes"), (dict(q_out=heads(plane_stride=8)), "16 bytes"), (dict(positions=None), "positions"),
        (dict(inv_freq=None), "positions"), (dict(eps=-1.0), "eps"), (dict(eps=math.nan), "eps")]),
    (K.cache_write, copy, [
        (dict(dtype=E4M3), "dtype"), (dict(dtype=BF16), "rows' type"), (dict(cache=cache(dtype=E4M3)), "k_scale"),
        (dict(cache=cache(dtype=K.FPK_DTYPE_F32)), "rows' type"), (dict(cache=cache(head_dim=96)), "head_dim"),
        (dict(cache=cache(page_rows=24)), "page_rows"), (dict(cache=cache(page_rows=8)), "page_rows"),
        (dict(cache=cache(page_rows=2048)), "page_rows"), (dict(cache=cache(n_pages=0)), "n_pages"),
        (dict(cache=cache(n_pages=1 << 27)), "2\\^31"), (dict(cache=cache(k=None)), "null"), (dict(cache=cache(v=A + 4)), "aligned"),
        (dict(slots=None), "slots"), (dict(rows=-1), "sizes"), (dict(v=heads(data=None)), "null"), (dict(k=heads(head_stride=8)), "16 bytes")]),
    (K.cache_read, copy, [(dict(dtype=BF16), "rows' type"), (dict(slots=None), "slots"), (dict(k=heads(data=None)), "null")]),
    (K.attention_packed, packed, [
        (dict(dtype=K.FPK_DTYPE_F32), "dtype"), (dict(head_dim=80), "head_dim"), (dict(q_heads=9), "multiple"), (dict(kv_heads=0), "multiple"),
        (dict(q_heads=258), "multiple"), (dict(n_seq=-1), "negative"), (dict(q_rows=-1), "negative"), (dict(kv_rows=-1), "negative"),
        (dict(q_rows=1 << 30), "too many"), (dict(scale=-1.0), "scale"), (dict(scale=math.inf), "scale"), (dict(scale=math.nan), "scale"),
        (dict(q=heads(data=None)), "null"), (dict(v=heads(data=None)), "null"), (dict(out=heads(data=A + 2)), "16 bytes"),
        (dict(q_starts=None), "q_starts"), (dict(kv_starts=None), "q_starts"), (dict(workspace=None), "workspace"),
        (dict(workspace_bytes=15), "workspace"), (dict(workspace=A + 8), "aligned")]),
    (K.attention_paged, paged, [
        (dict(dtype=E4M3), "dtype"), (dict(dtype=BF16), "rows' type"), (dict(cache=cache(page_rows=0)), "page_rows"),
        (dict(cache=cache(dtype=E4M3, k_scale=A)), "k_scale"), (dict(q_heads=7), "multiple"), (dict(table_pages=-1), "negative"),
        (dict(table_pages=1 << 28), "2\\^31"), (dict(page_table=None), "page_table"), (dict(kv_lengths=None), "kv_lengths"),
        (dict(q_starts=None), "q_starts"), (dict(out=heads(data=None)), "null"), (dict(workspace_bytes=0), "workspace")]),
]


@pytest.mark.parametrize("call,make,change,match", [(c, m, k, t) for c, m, rows in REFUSED for k, t in rows])
def test_refusals(fl, call, make, change, match):
    with pytest.raises(K.FpkError, match=match):
        call(fl, make(**change))


def test_null_descriptors_are_refused(fl):
    for name in ("fpk_qk_norm_rotary", "fpk_cache_write", "fpk_cache_read", "fpk_attention_packed", "fpk_attention_paged"):
        assert getattr(fl.lib, name)(None, None) != 0
        assert b"null descriptor" in fl.lib.fpk_last_error()
    assert fl.lib.fpk_attention_packed_workspace_bytes(None) == 0
    assert fl.lib.fpk_attention_paged_workspace_bytes(None) == 0


def test_empty_calls_do_nothing(fl):
    K.qk_norm_rotary(fl, rotary(rows=0))
    K.qk_norm_rotary(fl, rotary(q_heads=0, kv_heads=0))
    K.cache_write(fl, copy(rows=0, slots=None))
    K.cache_read(fl, copy(rows=0))
    K.attention_packed(fl, packed(n_seq=0))
    K.attention_packed(fl, packed(q_rows=0))
    K.attention_paged(fl, paged(n_seq=0))
    K.attention_paged(fl, paged(q_rows=0))


def test_heads_of_the_two_layouts():
    p = K.Heads.planar(A, 4096, 64, 128)
    assert (p.data, p.head_stride, p.row_stride, p.plane_stride) == (A + 16 * 4096, 8 * 4096, 16, 4096)
    r = K.Heads.rows(A, 640, 64, 128)
    assert (r.data, r.head_stride, r.row_stride, r.plane_stride) == (A + 256, 128, 1280, 16)


def test_rotary_frequencies():
    plain = K.rotary_frequencies(64, 10000.0)
    assert len(plain) == 32 and plain[0] == 1.0 and math.isclose(plain[16], 0.01)
    assert all(math.isclose(a / 4, b) for a, b in zip(plain, K.rotary_frequencies(64, factor=4.0)))
    parts = K.rotary_frequencies(64, factor=4.0, trained_length=4096)
    turns = [4096 * f / (2 * math.pi) for f in plain]
    for f, p, t in zip(plain, parts, turns):
        if t >= 32:
            assert math.isclose(f, p)
        elif t <= 1:
            assert math.isclose(f / 4, p)
        else:
            assert f / 4 < p < f
    for bad in (dict(rotary_dim=3), dict(rotary_dim=4, factor=0), dict(rotary_dim=4, slow_turns=5, fast_turns=2)):
        with pytest.raises(ValueError):
            K.rotary_frequencies(**bad)


def test_cache_copies_of_too_many_heads_are_refused(fl):
    for call in (K.cache_write, K.cache_read):
        with pytest.raises(K.FpkError, match="sizes"):
            call(fl, copy(cache=cache(kv_heads=4097)))


@pytest.mark.parametrize("call,make,change", [
    (K.qk_norm_rotary, rotary, dict(positions=A + 2)), (K.qk_norm_rotary, rotary, dict(inv_freq=A + 1)), (K.qk_norm_rotary, rotary, dict(q_weight=A + 3)),
    (K.cache_write, copy, dict(slots=A + 2)), (K.cache_read, copy, dict(error_flag=A + 1)),
    (K.attention_packed, packed, dict(q_starts=A + 2)), (K.attention_packed, packed, dict(kv_starts=A + 1)),
    (K.attention_packed, packed, dict(error_flag=A + 2)), (K.attention_paged, paged, dict(kv_lengths=A + 2)),
    (K.attention_paged, paged, dict(page_table=A + 3)),
    (K.attention_paged, paged, dict(cache=cache(dtype=E4M3, k_scale=A + 2, v_scale=A)))])
def test_misaligned_arrays_are_refused(fl, call, make, change):
    with pytest.raises(K.FpkError, match="4-byte aligned"):
        call(fl, make(**change))


def test_key_counts_that_would_overflow_are_refused(fl):
    with pytest.raises(K.FpkError, match="2\\^31 - 1024"):
        K.attention_packed(fl, packed(kv_rows=2 ** 31 - 1))
    with pytest.raises(K.FpkError, match="2\\^31 - 1024"):
        K.attention_paged(fl, paged(table_pages=(1 << 27) - 1))  # pages of 16 rows


@pytest.mark.parametrize("call,make,change,match", [
    (K.qk_norm_rotary, rotary, dict(rows=2 ** 31 - 1), "2\\^31 - 1024"), (K.qk_norm_rotary, rotary, dict(rows=2 ** 31 - 1023), "2\\^31 - 1024"),
    (K.cache_write, copy, dict(rows=2 ** 31 - 1), "2\\^31 - 1024"), (K.cache_read, copy, dict(rows=2 ** 31 - 1023), "2\\^31 - 1024"),
    # 4 query heads to a key head: 2^31 - 200 rows of tiles, which 255 more would take past 2^31.
    (K.attention_packed, packed, dict(q_rows=2 ** 29 - 50 - 64, n_seq=2), "too many"),
    (K.attention_packed, packed, dict(q_rows=2 ** 29 - 256, n_seq=0), None), (K.attention_packed, packed, dict(q_rows=2 ** 29 - 255, n_seq=0), "too many"),
    (K.attention_packed, packed, dict(n_seq=2 ** 20 + 1), "sequences"), (K.attention_paged, paged, dict(n_seq=2 ** 20 + 1), "sequences"),
    (K.attention_packed, packed, dict(scale=3e38), "scale"), (K.attention_paged, paged, dict(scale=2.5e38), "scale")])
def test_sizes_at_the_end_of_32_bits(fl, call, make, change, match):
    if match is None:
        call(fl, make(**change))
        return
    with pytest.raises(K.FpkError, match=match):
        call(fl, make(**change))
