"""Helpers of the tests of heads, packed sequences and the paged cache: tensors in
the layouts that fpk_heads_t names, descriptors, and plain attention in 64 bits
with the bound on what the kernels may be off by."""
from __future__ import annotations

import math

import torch

from fp_b200 import kernels as K

DT = {K.FPK_DTYPE_F16: torch.float16, K.FPK_DTYPE_BF16: torch.bfloat16}
# (dtype of the kernels, half a step of rounding relative to the value)
HALF_STEP = {d: torch.finfo(t).eps / 2 for d, t in DT.items()}
LAYOUTS = ("planar", "rows", "heads_first", "padded")


class HeadRows:
    """[rows, heads, d] values of a 16-bit type, held in one of LAYOUTS, with the bytes around them
    set to `around` so that stray reads and writes show."""

    def __init__(self, rows, heads, d, dtype, layout="rows", around=float("nan"), device="cuda"):
        self.shape, self.layout = (rows, heads, d), layout
        t = DT[dtype]
        full = lambda *s: torch.full(s, around, dtype=t, device=device)  # noqa: E731
        if layout == "planar":  # guard rows before and behind
            self.t = full(heads * d // 8, rows + 48, 8)
            self.v = self.t[:, 16:16 + rows].view(heads, d // 8, rows, 8).permute(2, 0, 1, 3)
        elif layout == "rows":
            self.t = full(rows + 4, heads, d)
            self.v = self.t[2:2 + rows].view(rows, heads, d // 8, 8)
        elif layout == "heads_first":
            self.t = full(heads, rows + 3, d)
            self.v = self.t[:, 1:1 + rows].unflatten(2, (d // 8, 8)).permute(1, 0, 2, 3)
        else:  # rows of a wider projection
            self.t = full(rows + 2, heads * d + 72)
            self.v = self.t[1:1 + rows, 40:40 + heads * d].unflatten(1, (heads, d // 8, 8))
        self.before = None

    @property
    def heads(self) -> K.Heads:
        r, h, g, _ = self.v.stride()
        return K.Heads(self.v.data_ptr(), h * 2, r * 2, g * 2)

    def set(self, x):
        self.v.copy_(x.reshape(self.v.shape))
        return self

    def get(self):
        return self.v.reshape(self.shape)

    def remember(self):
        self.before = self.t.clone()
        return self

    def untouched_around(self) -> bool:
        """Every byte outside the rows is what remember() saw."""
        a, b = self.before.clone(), self.t.clone()
        self._view_of(a).zero_()
        self._view_of(b).zero_()
        return torch.equal(a.view(torch.int16), b.view(torch.int16))

    def _view_of(self, t):
        rows, heads, d = self.shape
        if self.layout == "planar":
            return t[:, 16:16 + rows]
        if self.layout == "rows":
            return t[2:2 + rows]
        if self.layout == "heads_first":
            return t[:, 1:1 + rows]
        return t[1:1 + rows, 40:40 + heads * d]


def power_of_two(e):
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def quantise(x):
    """x [..., d] (16-bit) -> e4m3 codes (uint8) and scale [...]: the smallest power of two >= 2^-100
    with max|finite x| <= 448 scale, 1 for zeros; infinities and NaN become NaN."""
    f = x.float()
    finite = torch.where(f.isfinite(), f, torch.zeros_like(f)).abs().amax(-1)
    m, e = torch.frexp(finite)
    e = torch.where(m <= 0.875, e - 9, e - 8).clamp(min=-100)
    e = torch.where(finite == 0, torch.zeros_like(e), e)
    y = f * power_of_two(-e)[..., None]
    y = torch.where(y.isfinite(), y, torch.full_like(y, float("nan")))
    return y.to(torch.float8_e4m3fn).view(torch.uint8), power_of_two(e)


class Cache:
    """A paged cache; every slot begins as `stale`."""

    def __init__(self, n_pages, page_rows, heads, d, dtype, e4m3=False, device="cuda"):
        self.n_pages, self.page_rows, self.h, self.d, self.dtype, self.e4m3 = n_pages, page_rows, heads, d, dtype, e4m3
        if e4m3:
            make = lambda: torch.full((n_pages, heads, d // 16, page_rows, 16), 0x7F, dtype=torch.uint8, device=device)  # noqa: E731
            self.scale = [torch.full((n_pages, heads, page_rows), float("nan"), device=device) for _ in range(2)]
        else:
            make = lambda: torch.full((n_pages, heads, d // 8, page_rows, 8), float("nan"), dtype=DT[dtype], device=device)  # noqa: E731
            self.scale = [None, None]
        self.data = [make(), make()]

    @property
    def desc(self) -> K.KvCache:
        s = [x.data_ptr() if x is not None else None for x in self.scale]
        return K.KvCache(self.data[0].data_ptr(), self.data[1].data_ptr(), s[0], s[1], self.n_pages, self.page_rows, self.h,
                         self.d, K.FPK_DTYPE_E4M3 if self.e4m3 else self.dtype)

    def put(self, side, slots, x):
        """Row i of x [n, heads, d] into slot slots[i] (the definition of fpk_cache_write)."""
        p, r = slots.long() // self.page_rows, slots.long() % self.page_rows
        if self.e4m3:
            codes, scale = quantise(x)
            self.data[side][p, :, :, r] = codes.reshape(len(x), self.h, self.d // 16, 16)
            self.scale[side][p, :, r] = scale
        else:
            self.data[side][p, :, :, r] = x.reshape(len(x), self.h, self.d // 8, 8)

    def values(self, side, slots):
        """[n, heads, d] in 64 bits."""
        p, r = slots.long() // self.page_rows, slots.long() % self.page_rows
        x = self.data[side][p, :, :, r]
        if self.e4m3:
            return x.view(torch.float8_e4m3fn).double().reshape(len(slots), self.h, self.d) * self.scale[side][p, :, r].double()[..., None]
        return x.double().reshape(len(slots), self.h, self.d)


def starts(lengths, device="cuda"):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32, device=device)


def attention64(q, k, v, causal, scale, dtype, v_step=None):
    """One sequence: q [nq, hq, d], k, v [nk, hk, d] in 64 bits -> (out, bound) [nq, hq, d].

    The bound counts what the kernels round: probabilities to the type (half a step of each, and for
    fp16 2^-25 below its normal range, in units of the row's largest probability times v_step, the
    largest value or 448 times the largest e4m3 scale), scores in fp32 (d + 2 additions that may
    truncate, 2^-23 of the sum of magnitudes each; twice, as it moves the probability and the sum),
    exp2 (2^-21 with its argument's rounding, numerator and sum), and the output."""
    nq, hq, d = q.shape
    nk, hk = k.shape[:2]
    out = torch.zeros(nq, hq, d, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    if nk == 0 or nq == 0:
        return out, bound
    step = HALF_STEP[dtype]
    g = hq // hk
    for h in range(hq):
        kk, vv = k[:, h // g], v[:, h // g]
        s = q[:, h] @ kk.T * scale
        seen = torch.ones(nq, nk, dtype=torch.bool, device=q.device)
        if causal:
            i = torch.arange(nq, device=q.device)[:, None]
            seen = torch.arange(nk, device=q.device)[None] <= nk - nq + i
        # Where a key is hidden its values do not count, whatever they are.
        s = torch.where(seen, s, torch.full_like(s, -math.inf))
        any_seen = seen.any(1)
        top = torch.where(any_seen, s.amax(1), torch.zeros_like(s[:, 0]))
        p = torch.exp(s - top[:, None])
        total = torch.where(any_seen, p.sum(1), torch.ones_like(top))
        p = p / total[:, None]
        out[:, h] = p @ vv
        mean_abs = p @ vv.abs()
        mag = torch.where(seen, q[:, h].abs() @ kk.abs().T * scale, torch.zeros_like(s)).amax(1)
        # The argument of exp2 (log2 e times the score) is rounded at its own size, up to mag.
        rel = 2 * ((d + 2) * 2.0 ** -23 * mag * 1.5 + 2.0 ** -21 * (1 + mag))
        tiny = (nk * 2.0 ** -25 * (v_step if v_step is not None else vv.abs().max().item())) if dtype == K.FPK_DTYPE_F16 or v_step is not None else 0.0
        bound[:, h] = (step + rel)[:, None] * mean_abs + step * out[:, h].abs() + tiny * any_seen[:, None] + 2.0 ** -24
    return out, bound


def within(got, ref, bound):
    """Largest error in units of its bound (nan counts as infinite)."""
    e = (got.double() - ref).abs() / bound.clamp(min=1e-300)
    e = torch.where((got.double() == ref), torch.zeros_like(e), e)
    return float(torch.nan_to_num(e, nan=math.inf).max()) if e.numel() else 0.0
