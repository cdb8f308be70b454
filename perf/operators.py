"""Cases, plain forms and calls of the kernel-level attention operators over heads and cached rows.

Four operators that follow one another in a decoder-style transformer block, next to the library's
GEMM and fixed-length self-attention:

  rotate   RMS norm of every query and key head and the rotary position, in one pass
  packed   attention over packed sequences of different lengths, grouped heads, causal or full
  write /  rows of keys and values into a paged cache (16-bit, or e4m3 with one power-of-two
  read     scale per row and head), and back
  paged    attention of the newest tokens of each sequence (one, or a chunk) over the paged cache

`own` False computes them with elementary torch operations; True calls the library's kernels.
Activations come in the library's planar layout ("planar": [group of 8 channels][row][8]) or row by
row ("rows": [row][head][channel]); queries, keys and values are parts of one projection's output.
"""
from __future__ import annotations

import functools
import math
import random
import sys
from pathlib import Path

import torch

own = False

_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
_E4M3_MAX = 448.0
_SCALE_EXP_MIN = -100


# ---------------------------------------------------------------------------
# cases

def listed():
    return [
        # One new token of each of 8 sequences: what every decoded token pays before its attention.
        {"name": "rotate-tokens", "op": "rotate", "rows": 8, "q_heads": 32, "kv_heads": 8, "d": 128, "type": "bf16",
         "layout": "rows", "norm": True, "interleaved": False, "rotary": 128, "far": 5000},
        # The prompts of a batch, normalised and rotated whole.
        {"name": "rotate-prompts", "op": "rotate", "rows": 16384, "q_heads": 32, "kv_heads": 8, "d": 128,
         "type": "bf16", "layout": "rows", "norm": True, "interleaved": False, "rotary": 128, "far": 16384},
        # Planar activations as the library's GEMM leaves them: half of the head rotated, pairs of neighbours,
        # positions of a long recording, an odd number of rows.
        {"name": "rotate-far-planar", "op": "rotate", "rows": 5003, "q_heads": 4, "kv_heads": 4, "d": 128,
         "type": "f16", "layout": "planar", "norm": False, "interleaved": True, "rotary": 64, "far": 1000000},
        # Cross-hypothesis attention of a group of 8 objects, each with its own number of hypotheses.
        {"name": "packed-hypotheses", "op": "packed", "n_seq": 8, "max_q": 252, "min_q": 3, "max_kv": 0, "q_heads": 4,
         "kv_heads": 4, "d": 128, "type": "f16", "layout": "planar", "causal": False},
        # Self-attention over the 400 crop tokens of 252 hypotheses.
        {"name": "packed-crops", "op": "packed", "n_seq": 252, "max_q": 400, "min_q": 400, "max_kv": 0, "q_heads": 4,
         "kv_heads": 4, "d": 128, "type": "f16", "layout": "planar", "causal": False},
        # Prompts of different lengths, causal, eight query heads to a key head.
        {"name": "packed-prompts", "op": "packed", "n_seq": 4, "max_q": 8192, "min_q": 700, "max_kv": 0,
         "q_heads": 16, "kv_heads": 2, "d": 128, "type": "bf16", "layout": "rows", "causal": True},
        # The new rows of 64 decoded sequences into a 16-bit cache.
        {"name": "write-tokens", "op": "write", "rows": 64, "slots": 8192, "kv_heads": 8, "d": 128, "type": "bf16",
         "cache": "same", "page": 64, "layout": "rows"},
        # A prompt's rows into an e4m3 cache.
        {"name": "write-prompt-e4m3", "op": "write", "rows": 16384, "slots": 32768, "kv_heads": 8, "d": 128,
         "type": "bf16", "cache": "e4m3", "page": 64, "layout": "rows"},
        # The cached rows of a sequence read back, an odd number of them, for a pass that wants them dense.
        {"name": "read-e4m3", "op": "read", "rows": 20011, "slots": 32768, "kv_heads": 8, "d": 128, "type": "bf16",
         "cache": "e4m3", "page": 64, "layout": "rows"},
        # One token of each of 4 short sequences: latency alone.
        {"name": "paged-token-short", "op": "paged", "n_seq": 4, "max_q": 1, "min_q": 1, "max_kv": 1000, "min_kv": 40,
         "q_heads": 32, "kv_heads": 8, "d": 128, "type": "bf16", "cache": "same", "page": 64, "layout": "rows",
         "causal": True},
        # One token of each of 8 sequences of very different lengths, the longest long, over an e4m3 cache.
        {"name": "paged-token-long-e4m3", "op": "paged", "n_seq": 8, "max_q": 1, "min_q": 1, "max_kv": 131072,
         "min_kv": 8000, "q_heads": 32, "kv_heads": 8, "d": 128, "type": "bf16", "cache": "e4m3", "page": 64,
         "layout": "rows", "causal": True},
        # A chunk of a prompt over what is cached of it, small pages.
        {"name": "paged-chunk", "op": "paged", "n_seq": 4, "max_q": 512, "min_q": 100, "max_kv": 12000,
         "min_kv": 2000, "q_heads": 32, "kv_heads": 8, "d": 128, "type": "bf16", "cache": "same", "page": 16,
         "layout": "rows", "causal": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["rotate", "packed", "packed", "write", "read", "paged", "paged", "paged"])
    heads = rng.choice([(4, 4), (32, 8), (16, 2), (12, 4), (8, 1), (6, 2), (20, 4)])
    case = {"op": op, "q_heads": heads[0], "kv_heads": heads[1], "d": rng.choice([64, 128]),
            "type": rng.choice(["f16", "bf16"]), "layout": rng.choice(["planar", "rows"])}
    if op == "rotate":
        case["rows"] = _log_int(rng, 1, 16384)
        case["norm"] = rng.random() < 0.6
        case["interleaved"] = rng.random() < 0.5
        case["rotary"] = rng.choice([case["d"], case["d"], case["d"] // 2, 32])
        case["far"] = _log_int(rng, 100, 1000000)
        return case
    if op in ("write", "read"):
        del case["q_heads"]
        case["page"] = rng.choice([16, 32, 64, 128])
        case["rows"] = _log_int(rng, 1, 16384 if op == "write" else 20011)
        case["slots"] = -(-int(case["rows"] * rng.uniform(1.0, 1.6)) // case["page"]) * case["page"]
        case["cache"] = rng.choice(["same", "e4m3"])
        return case
    if op == "packed":
        while True:
            case["n_seq"] = _log_int(rng, 1, 252)
            case["max_q"] = _log_int(rng, 1, 8192)
            # 0: keys and queries are the same rows; otherwise keys of another sequence of rows.
            case["max_kv"] = rng.choice([0, 0, _log_int(rng, 1, 8192)])
            if case["n_seq"] * case["q_heads"] * case["max_q"] * max(case["max_q"], case["max_kv"]) <= 4 * 16 * 8192 ** 2:
                break
        case["min_q"] = rng.choice([1, max(1, case["max_q"] // 2), case["max_q"]])
        case["causal"] = rng.random() < 0.5
        return case
    while True:
        case["n_seq"] = _log_int(rng, 1, 64)
        case["max_q"] = rng.choice([1, 1, _log_int(rng, 2, 16), _log_int(rng, 17, 600)])
        case["max_kv"] = _log_int(rng, max(16, case["max_q"]), 131072)
        pairs = case["n_seq"] * case["q_heads"] * case["max_q"] * case["max_kv"]
        keys = case["n_seq"] * case["kv_heads"] * case["max_kv"]
        if pairs <= 4 * 32 * 512 * 12000 and keys <= 8 * 8 * 131072:
            break
    case["min_q"] = rng.choice([1, case["max_q"]])
    case["min_kv"] = rng.choice([case["max_q"], max(case["max_q"], case["max_kv"] // 2)])
    case["cache"] = rng.choice(["same", "e4m3"])
    case["page"] = rng.choice([16, 32, 64, 128])
    case["causal"] = rng.random() < 0.8
    return case


def _lengths(case):
    """(query rows, key rows) of every sequence: fixed by the case, the first sequence the longest."""
    rng = random.Random(case["n_seq"] * 7919 + case["max_q"] * 31 + case["max_kv"])
    n = case["n_seq"]
    q = [case["max_q"]] + [_log_int(rng, case["min_q"], case["max_q"]) for _ in range(n - 1)]
    if case["op"] == "paged":
        kv = [case["max_kv"]] + [_log_int(rng, case["min_kv"], case["max_kv"]) for _ in range(n - 1)]
        return q, kv
    if case["max_kv"] == 0:
        return q, list(q)
    return q, [case["max_kv"]] + [_log_int(rng, 1, case["max_kv"]) for _ in range(n - 1)]


def _pairs(case):
    """Allowed (query, key) pairs over all sequences."""
    total = 0
    for nq, nk in zip(*_lengths(case)):
        if not case["causal"]:
            total += nq * nk
            continue
        # Query i sees keys 0 .. nk - nq + i.
        first = nk - nq + 1
        skipped = max(0, -first + 1) if first < 1 else 0  # rows that see nothing
        rows = nq - min(nq, skipped)
        last = nk
        total += rows * (last - rows + 1 + last) // 2
    return total


def work(case):
    op, d = case["op"], case["d"]
    hk = case["kv_heads"]
    if op == "rotate":
        n = case["rows"] * (case["q_heads"] + hk)
        return {"bytes": 4 * n * d + 4 * case["rows"] + 2 * case["rotary"] + (8 * d if case["norm"] else 0),
                "flops": n * ((4 * d if case["norm"] else 0) + 3 * case["rotary"])}
    if op in ("write", "read"):
        row = 2 * hk * d
        held = row * (1 if case["cache"] == "e4m3" else 2) + (8 * hk if case["cache"] == "e4m3" else 0)
        return {"bytes": case["rows"] * (2 * row + held + 4), "flops": case["rows"] * row * (2 if case["cache"] == "e4m3" else 0)}
    q, kv = _lengths(case)
    rows = 4 * sum(q) * case["q_heads"] * d
    if op == "paged":
        key = 2 * hk * d * (1 if case["cache"] == "e4m3" else 2) + (8 * hk if case["cache"] == "e4m3" else 0)
        table = 4 * sum(-(-n // case["page"]) for n in kv)
        return {"bytes": rows + sum(kv) * key + table + 8 * case["n_seq"], "flops": 4 * d * case["q_heads"] * _pairs(case)}
    return {"bytes": rows + sum(kv) * 4 * hk * d + 8 * case["n_seq"], "flops": 4 * d * case["q_heads"] * _pairs(case)}


# ---------------------------------------------------------------------------
# inputs

def _activation(rows, heads, d, dtype, layout, gen, scale=1.0):
    shape = (heads * d // 8, rows, 8) if layout == "planar" else (rows, heads, d)
    x = torch.empty(shape, dtype=dtype, device="cuda")
    x.normal_(0.0, scale, generator=gen)
    return x


def _heads_of(x, layout, first, heads, d):
    """[rows, heads, d] of heads first .. first + heads of an activation tensor."""
    if layout == "rows":
        return x[:, first:first + heads]
    g = d // 8
    y = x[first * g:(first + heads) * g]
    return y.reshape(heads, g, -1, 8).permute(2, 0, 1, 3).reshape(-1, heads, d)


def _laid_out(y, layout):
    """[rows, heads, d] in an activation tensor's layout."""
    if layout == "rows":
        return y
    rows, heads, d = y.shape
    return y.reshape(rows, heads * d // 8, 8).permute(1, 0, 2)


def _zeros(rows, heads, d, dtype, layout):
    shape = (heads * d // 8, rows, 8) if layout == "planar" else (rows, heads, d)
    return torch.zeros(shape, dtype=dtype, device="cuda")


def _power_of_two(e):
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _quantised(x):
    """e4m3 values and their power-of-two scale over the last dimension of x (fp32)."""
    m, e = torch.frexp(x.abs().amax(-1, keepdim=True))
    e = torch.where(m <= 0.875, e - 9, e - 8).clamp(min=_SCALE_EXP_MIN)
    e = torch.where(m == 0, torch.zeros_like(e), e)
    return (x * _power_of_two(-e)).to(torch.float8_e4m3fn), _power_of_two(e)[..., 0]


def _cache_tensors(case, pages, gen, filled):
    """Pages [page][head][group of 16 bytes][row][16 bytes] and, for e4m3, scales [page][head][row]."""
    hk, d, page = case["kv_heads"], case["d"], case["page"]
    state = {}
    for name in ("k", "v"):
        if case["cache"] == "same":
            x = torch.zeros((pages, hk, d // 8, page, 8), dtype=_TYPES[case["type"]], device="cuda")
            if filled:
                x.normal_(0.0, 1.0, generator=gen)
            state[name + "_cache"] = x
            continue
        x = torch.zeros((pages, hk, d // 16, page, 16), dtype=torch.uint8, device="cuda")
        s = torch.ones((pages, hk, page), dtype=torch.float32, device="cuda")
        if filled:
            for at in range(0, pages, 2048):  # in pieces: the fp32 values of a long cache are large
                part = torch.empty((min(2048, pages - at), hk, page, d), device="cuda")
                part.normal_(0.0, 1.0, generator=gen)
                part *= torch.rand(part.shape[:-1] + (1,), device="cuda", generator=gen) * 1.5 + 0.2
                q, sc = _quantised(part)
                x[at:at + 2048] = q.view(torch.uint8).reshape(-1, hk, page, d // 16, 16).transpose(2, 3)
                s[at:at + 2048] = sc
        state[name + "_cache"], state[name + "_scale"] = x, s
    return state


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, d, hk, dtype, layout = case["op"], case["d"], case["kv_heads"], _TYPES[case["type"]], case["layout"]
    state = {"case": case}
    if op == "rotate":
        rows, hq = case["rows"], case["q_heads"]
        state["qkv"] = _activation(rows, hq + 2 * hk, d, dtype, layout, gen, 1.3)
        state["q_out"] = _zeros(rows, hq, d, dtype, layout)
        state["k_out"] = _zeros(rows, hk, d, dtype, layout)
        # A batch of consecutive runs that start anywhere.
        start = torch.randint(0, max(1, case["far"] - rows), (1,), device="cuda", generator=gen)
        state["positions"] = (start + torch.arange(rows, device="cuda")).to(torch.int32)
        half = case["rotary"] // 2
        state["inv_freq"] = (10000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)).to(torch.float32)
        state["q_weight"] = state["k_weight"] = None
        if case["norm"]:
            state["q_weight"] = 1.0 + 0.2 * torch.randn(d, device="cuda", generator=gen)
            state["k_weight"] = 1.0 + 0.2 * torch.randn(d, device="cuda", generator=gen)
        return state
    if op in ("write", "read"):
        rows, pages = case["rows"], case["slots"] // case["page"]
        state.update(_cache_tensors(case, pages, gen, filled=op == "read"))
        state["slots"] = torch.randperm(case["slots"], device="cuda", generator=gen)[:rows].to(torch.int32)
        if op == "write":
            state["kv"] = _activation(rows, 2 * hk, d, dtype, layout, gen)
        else:
            state["k_out"] = _zeros(rows, hk, d, dtype, layout)
            state["v_out"] = _zeros(rows, hk, d, dtype, layout)
        return state
    q, kv = _lengths(case)
    hq = case["q_heads"]
    starts = lambda n: torch.tensor([sum(n[:i]) for i in range(len(n) + 1)], dtype=torch.int32, device="cuda")  # noqa: E731
    state.update(max_q=max(q), max_kv=max(kv), q_rows=sum(q), kv_rows=sum(kv), q_starts=starts(q))
    if op == "packed":
        state["kv_starts"] = starts(kv)
        if case["max_kv"] == 0:  # one projection's output
            state["q_in"] = state["kv_in"] = _activation(sum(q), hq + 2 * hk, d, dtype, layout, gen)
            state["k_first"] = hq
        else:
            state["q_in"] = _activation(sum(q), hq, d, dtype, layout, gen)
            state["kv_in"] = _activation(sum(kv), 2 * hk, d, dtype, layout, gen)
            state["k_first"] = 0
    else:
        state["q_in"] = _activation(sum(q), hq, d, dtype, layout, gen)
        page = case["page"]
        need = [-(-n // page) for n in kv]
        state.update(_cache_tensors(case, sum(need) + 3, gen, filled=True))
        order = torch.randperm(sum(need) + 3, device="cuda", generator=gen).to(torch.int32)
        table = torch.zeros((len(kv), max(need)), dtype=torch.int32, device="cuda")
        at = 0
        for s, n in enumerate(need):
            table[s, :n] = order[at:at + n]
            at += n
        state["page_table"] = table
        state["kv_lengths"] = torch.tensor(kv, dtype=torch.int32, device="cuda")
    state["out"] = _zeros(sum(q), hq, d, dtype, layout)
    return state


# ---------------------------------------------------------------------------
# plain forms

def _plain_rotate(state):
    case = state["case"]
    hq, hk, d, r = case["q_heads"], case["kv_heads"], case["d"], case["rotary"]
    angle = state["positions"].double()[:, None] * state["inv_freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    for first, heads, weight, out in ((0, hq, state["q_weight"], state["q_out"]), (hq, hk, state["k_weight"], state["k_out"])):
        x = _heads_of(state["qkv"], case["layout"], first, heads, d).float()
        if weight is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight
        y = x.clone()
        a, b = (x[..., 0:r:2], x[..., 1:r:2]) if case["interleaved"] else (x[..., :r // 2], x[..., r // 2:r])
        c, e = (y[..., 0:r:2], y[..., 1:r:2]) if case["interleaved"] else (y[..., :r // 2], y[..., r // 2:r])
        c.copy_(a * cos - b * sin)
        e.copy_(b * cos + a * sin)
        out.copy_(_laid_out(y, case["layout"]))
    return {"q": state["q_out"], "k": state["k_out"]}


def _plain_write(state):
    case = state["case"]
    hk, d, page = case["kv_heads"], case["d"], case["page"]
    slots = state["slots"].long()
    p, r = slots // page, slots % page
    for name, first in (("k", 0), ("v", hk)):
        x = _heads_of(state["kv"], case["layout"], first, hk, d)
        cache = state[name + "_cache"]
        if case["cache"] == "e4m3":
            q, scale = _quantised(x.float())
            cache[p, :, :, r] = q.view(torch.uint8).reshape(-1, hk, d // 16, 16)
            state[name + "_scale"][p, :, r] = scale
        else:
            cache[p, :, :, r] = x.reshape(-1, hk, d // 8, 8)
    return _cache_values(state)


def _cache_values(state):
    out = {}
    for name in ("k", "v"):
        cache = state[name + "_cache"]
        if state["case"]["cache"] == "e4m3":
            out[name] = cache.view(torch.float8_e4m3fn)
            out[name + "_scale"] = state[name + "_scale"]
        else:
            out[name] = cache
    return out


def _saturated(x, dtype):
    top = torch.finfo(dtype).max
    return x.clamp(-top, top).to(dtype)


def _plain_read(state):
    case = state["case"]
    hk, d, page, dtype = case["kv_heads"], case["d"], case["page"], _TYPES[case["type"]]
    slots = state["slots"].long()
    p, r = slots // page, slots % page
    for name in ("k", "v"):
        x = state[name + "_cache"][p, :, :, r]
        if case["cache"] == "e4m3":
            x = x.view(torch.float8_e4m3fn).float() * state[name + "_scale"][p, :, r][..., None, None]
        x = _saturated(x.reshape(-1, hk, d).float(), dtype)
        state[name + "_out"].copy_(_laid_out(x, case["layout"]))
    return {"k": state["k_out"], "v": state["v_out"]}


def _plain_attention(state, k, v, kv_lengths):
    """k, v: [sequence, key, head, d], padded to the longest."""
    case = state["case"]
    hq, hk, d = case["q_heads"], case["kv_heads"], case["d"]
    group, mq, mk = hq // hk, state["max_q"], k.shape[1]
    starts = state["q_starts"].long()
    q_lengths = starts[1:] - starts[:-1]
    i, j = torch.arange(mq, device="cuda"), torch.arange(mk, device="cuda")
    at = (starts[:-1, None] + i).clamp(max=state["q_rows"] - 1)
    q = _heads_of(state["q_in"], case["layout"], 0, hq, d)[at].float()
    q = q.reshape(-1, mq, hk, group, d).permute(0, 2, 3, 1, 4).reshape(-1, hk, group * mq, d)
    s = q @ k.permute(0, 2, 3, 1).float()
    s *= 1.0 / math.sqrt(d)
    seen = kv_lengths[:, None].expand(-1, mq)
    if case["causal"]:
        seen = torch.minimum(seen, (kv_lengths - q_lengths)[:, None] + i + 1)
    hidden = (j >= seen[..., None])[:, None, None]
    s = s.view(-1, hk, group, mq, mk).masked_fill_(hidden, -math.inf)
    top = s.amax(-1, keepdim=True)
    s -= torch.where(top == -math.inf, torch.zeros_like(top), top)
    s.exp_()
    total = s.sum(-1, keepdim=True)
    o = (s.view(-1, hk, group * mq, mk) @ v.permute(0, 2, 1, 3).float()).view(-1, hk, group, mq, d)
    o /= torch.where(total == 0, torch.ones_like(total), total)
    o = o.permute(0, 3, 1, 2, 4).reshape(-1, mq, hq, d)
    row = torch.arange(state["q_rows"], device="cuda")
    seq = torch.searchsorted(starts[1:].contiguous(), row, right=True)
    state["out"].copy_(_laid_out(o[seq, row - starts[seq]], case["layout"]))
    return {"out": state["out"]}


def _plain_packed(state):
    case = state["case"]
    hk, d, first = case["kv_heads"], case["d"], state["k_first"]
    starts = state["kv_starts"].long()
    at = (starts[:-1, None] + torch.arange(state["max_kv"], device="cuda")).clamp(max=state["kv_rows"] - 1)
    k = _heads_of(state["kv_in"], case["layout"], first, hk, d)[at]
    v = _heads_of(state["kv_in"], case["layout"], first + hk, hk, d)[at]
    return _plain_attention(state, k, v, starts[1:] - starts[:-1])


def _plain_paged(state):
    case = state["case"]
    hk, d = case["kv_heads"], case["d"]
    table = state["page_table"].long()
    rows = []
    for name in ("k", "v"):
        x = state[name + "_cache"][table]  # [sequence, page, head, group, row, channels]
        if case["cache"] == "e4m3":
            x = x.view(torch.float8_e4m3fn).float() * state[name + "_scale"][table][:, :, :, None, :, None]
        rows.append(x.permute(0, 1, 4, 2, 3, 5).reshape(len(table), -1, hk, d))
    return _plain_attention(state, *rows, state["kv_lengths"].long())


# ---------------------------------------------------------------------------
# the library's calls

@functools.lru_cache(None)
def _library():
    sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "foundation-pose-inference-library_b200" / "python"))
    from fp_b200 import kernels

    return kernels, kernels.FpkLibrary()


def _view(x, layout, first, d):
    """The heads from `first` on of an activation tensor, as the library takes them."""
    kernels, _ = _library()
    if layout == "rows":
        return kernels.Heads(x.data_ptr() + first * d * 2, d * 2, x.stride(0) * 2, 16)
    plane = x.stride(0) * 2
    return kernels.Heads(x.data_ptr() + first * (d // 8) * plane, (d // 8) * plane, 16, plane)


def _cache_of(state):
    kernels, _ = _library()
    case = state["case"]
    scale = lambda n: state[n + "_scale"].data_ptr() if case["cache"] == "e4m3" else None  # noqa: E731
    kind = kernels.FPK_DTYPE_E4M3 if case["cache"] == "e4m3" else _dtype(case)
    return kernels.KvCache(k=state["k_cache"].data_ptr(), v=state["v_cache"].data_ptr(), k_scale=scale("k"), v_scale=scale("v"),
                           n_pages=len(state["k_cache"]), page_rows=case["page"], kv_heads=case["kv_heads"],
                           head_dim=case["d"], dtype=kind)


def _dtype(case):
    kernels, _ = _library()
    return kernels.FPK_DTYPE_BF16 if case["type"] == "bf16" else kernels.FPK_DTYPE_F16


def _describe(state):
    """The call's descriptor, error flag and workspace, which a program keeps from step to step."""
    kernels, lib = _library()
    case = state["case"]
    op, d, layout, hk = case["op"], case["d"], case["layout"], case["kv_heads"]
    state["error"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    ptr = lambda n: state[n].data_ptr() if state[n] is not None else None  # noqa: E731
    if op == "rotate":
        hq = case["q_heads"]
        state["desc"] = kernels.QkRotaryDesc(
            q=_view(state["qkv"], layout, 0, d), k=_view(state["qkv"], layout, hq, d), q_out=_view(state["q_out"], layout, 0, d),
            k_out=_view(state["k_out"], layout, 0, d), rows=case["rows"], q_heads=hq, kv_heads=hk, head_dim=d,
            rotary_dim=case["rotary"], interleaved=int(case["interleaved"]), q_weight=ptr("q_weight"), k_weight=ptr("k_weight"),
            eps=1e-6, positions=ptr("positions"), inv_freq=ptr("inv_freq"), rotary_scale=1.0, dtype=_dtype(case))
        state["call"] = kernels.qk_norm_rotary
    elif op in ("write", "read"):
        k, v = ((state["kv"], 0), (state["kv"], hk)) if op == "write" else ((state["k_out"], 0), (state["v_out"], 0))
        state["desc"] = kernels.CacheCopyDesc(cache=_cache_of(state), k=_view(k[0], layout, k[1], d), v=_view(v[0], layout, v[1], d),
                                              rows=case["rows"], slots=ptr("slots"), dtype=_dtype(case), error_flag=ptr("error"))
        state["call"] = kernels.cache_write if op == "write" else kernels.cache_read
    else:
        common = dict(q=_view(state["q_in"], layout, 0, d), out=_view(state["out"], layout, 0, d), q_heads=case["q_heads"],
                      n_seq=case["n_seq"], q_rows=state["q_rows"], q_starts=ptr("q_starts"), causal=int(case["causal"]),
                      dtype=_dtype(case), error_flag=ptr("error"))
        if op == "packed":
            state["desc"] = kernels.PackedAttentionDesc(
                k=_view(state["kv_in"], layout, state["k_first"], d), v=_view(state["kv_in"], layout, state["k_first"] + hk, d),
                kv_heads=hk, head_dim=d, kv_rows=state["kv_rows"], kv_starts=ptr("kv_starts"), **common)
            state["call"], size = kernels.attention_packed, kernels.attention_packed_workspace_bytes
        else:
            state["desc"] = kernels.PagedAttentionDesc(
                cache=_cache_of(state), kv_lengths=ptr("kv_lengths"), page_table=ptr("page_table"),
                table_pages=state["page_table"].shape[1], **common)
            state["call"], size = kernels.attention_paged, kernels.attention_paged_workspace_bytes
        n = size(lib, state["desc"])
        state["workspace"] = torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")
        state["desc"].workspace, state["desc"].workspace_bytes = state["workspace"].data_ptr(), n


_RESULTS = {"rotate": lambda s: {"q": s["q_out"], "k": s["k_out"]}, "write": _cache_values,
            "read": lambda s: {"k": s["k_out"], "v": s["v_out"]}, "packed": lambda s: {"out": s["out"]},
            "paged": lambda s: {"out": s["out"]}}
_PLAIN = {"rotate": _plain_rotate, "write": _plain_write, "read": _plain_read, "packed": _plain_packed, "paged": _plain_paged}


def run(state):
    op = state["case"]["op"]
    if not own:
        return _PLAIN[op](state)
    if "desc" not in state:
        _describe(state)
    state["call"](_library()[1], state["desc"], torch.cuda.current_stream().cuda_stream)
    return _RESULTS[op](state)


# ---------------------------------------------------------------------------
# from the definitions, in 64 bits

def _rows64(x, layout, d):
    """An activation tensor as [row, head, d] in 64 bits."""
    if layout == "planar":
        x = torch.movedim(x, 0, 1).flatten(1)
    else:
        x = x.flatten(1)
    return x.double().unflatten(1, (-1, d))


def _cached64(state, name, page, row):
    """Row `row` of page `page` of the cache (index tensors): [.., head, d] in 64 bits."""
    x = state[name + "_cache"]
    if state["case"]["cache"] == "e4m3":
        s = state[name + "_scale"][page, :, row].double()
        return x[page, :, :, row].view(torch.float8_e4m3fn).double().flatten(-2) * s[..., None]
    return x[page, :, :, row].double().flatten(-2)


def exact(case, seed):
    state = prepare(case, seed)
    op, d, layout, hk = case["op"], case["d"], case["layout"], case["kv_heads"]
    back = lambda y: y if layout == "rows" else torch.movedim(y.flatten(1).unflatten(1, (-1, 8)), 0, 1)  # noqa: E731
    if op == "rotate":
        x = _rows64(state["qkv"], layout, d)
        theta = torch.outer(state["positions"].double(), state["inv_freq"].double())
        turn = torch.polar(torch.ones_like(theta), theta)[:, None]
        results = []
        for part, w in ((x[:, :case["q_heads"]], state["q_weight"]), (x[:, case["q_heads"]:case["q_heads"] + hk], state["k_weight"])):
            if w is not None:
                part = part / (part.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
            r = case["rotary"]
            pairs = part[..., :r].unflatten(-1, (-1, 2)) if case["interleaved"] else part[..., :r].unflatten(-1, (2, -1)).transpose(-1, -2)
            z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
            z = z.flatten(-2) if case["interleaved"] else z.transpose(-1, -2).flatten(-2)
            results.append(back(torch.cat([z, part[..., r:]], -1)))
        return {"q": results[0], "k": results[1]}
    if op == "write":
        x = _rows64(state["kv"], layout, d)
        out = {}
        page, row = state["slots"].long() // case["page"], state["slots"].long() % case["page"]
        for name, part in (("k", x[:, :hk]), ("v", x[:, hk:])):
            if case["cache"] == "e4m3":
                top = part.abs().amax(-1, keepdim=True)
                e = torch.ceil(torch.log2(top / _E4M3_MAX) - 1e-12).clamp(min=_SCALE_EXP_MIN)
                scale = torch.where(top == 0, torch.ones_like(top), torch.exp2(e))
                # The grid of e4m3: three bits behind the leading one, steps of 2^-9 below 2^-6.
                y = part / scale
                step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
                full = torch.zeros((case["slots"] // case["page"], hk, d // 16, case["page"], 16), dtype=torch.float64, device="cuda")
                full[page, :, :, row] = (torch.round(y / step) * step).unflatten(-1, (-1, 16))
                scales = torch.ones(full.shape[:2] + (case["page"],), dtype=torch.float64, device="cuda")
                scales[page, :, row] = scale[..., 0]
                out[name], out[name + "_scale"] = full, scales
            else:
                full = torch.zeros((case["slots"] // case["page"], hk, d // 8, case["page"], 8), dtype=torch.float64, device="cuda")
                full[page, :, :, row] = part.unflatten(-1, (-1, 8))
                out[name] = full
        return out
    if op == "read":
        page, row = state["slots"].long() // case["page"], state["slots"].long() % case["page"]
        return {n: back(_cached64(state, n, page, row)) for n in ("k", "v")}
    q_len, kv_len = _lengths(case)
    group = case["q_heads"] // hk
    q_all = _rows64(state["q_in"], layout, d)
    if op == "packed":
        kv_all = _rows64(state["kv_in"], layout, d)
    result = torch.zeros((sum(q_len), case["q_heads"], d), dtype=torch.float64, device="cuda")
    q_at = kv_at = 0
    for s, (nq, nk) in enumerate(zip(q_len, kv_len)):
        if op == "packed":
            first = state["k_first"]
            k, v = kv_all[kv_at:kv_at + nk, first:first + hk], kv_all[kv_at:kv_at + nk, first + hk:first + 2 * hk]
        else:
            at = torch.arange(nk, device="cuda")
            page = state["page_table"][s].long()[at // case["page"]]
            k, v = (_cached64(state, n, page, at % case["page"]) for n in ("k", "v"))
        offset = nk - nq
        for h in range(case["q_heads"]):
            logits = q_all[q_at:q_at + nq, h] @ k[:, h // group].T / math.sqrt(d)
            if case["causal"]:
                logits = logits + torch.full_like(logits, -math.inf).triu(offset + 1)
            p = torch.softmax(logits, -1)
            result[q_at:q_at + nq, h] = torch.nan_to_num(p, nan=0.0) @ v[:, h // group]
        q_at, kv_at = q_at + nq, kv_at + nk
    return {"out": back(result)}
