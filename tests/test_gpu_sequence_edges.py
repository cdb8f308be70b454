"""GPU tests of packed and paged attention at the edges of a warp, of a tile and of the mask. Compared
in 64 bits with the bound of seq_util.attention64, or with what the call gives without the odd rows."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from fp_b200 import kernels as K  # noqa: E402
from seq_util import HeadRows, within  # noqa: E402
from test_gpu_sequences import gen, reference, run_packed  # noqa: E402

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
