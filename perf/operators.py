"""Operators of a serving step over an 8-bit paged KV cache, and the draw of its next tokens: their performance cases.

The cache holds K and V as bytes.  16 consecutive tokens of one KV head (a block) share one scale 2^e; a value is
(byte - 128) * 2^e.  A page holds ``page_tokens`` tokens of every KV head, K as [head][token][dim], V block by block as
[head][block][dim][16 tokens], and one exponent per head and block for each.  Sequence b's tokens lie in the pages of
row b of the page table; its new rows are rows row_start[b] .. of q, k and v, the first of them at position
kv_offset[b] (one row per sequence where there is no row_start).

Where ``own`` is false, ``run`` computes in elementary torch operations; where it is true it calls the framework.
Sizes are those of the repository's model configuration, benchmark and tests (12 query and 2 KV heads of 128,
vocabulary 151936, prompts in chunks of 512) and generic ones around them.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

BLOCK = 16         # tokens that share a scale
E_MIN = -126       # the smallest exponent of a block
THETA = 1e6        # base of the rotation's angles


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one decoded token of one sequence goes into its cache (and the cache's rows are handed back): latency
        {"name": "append_1", "kind": "append", "batch": 1, "low": 500, "high": 500, "new": 1, "n_q": 12, "n_kv": 2,
         "hd": 128, "page": 64, "dtype": "f16"},
        # one decoded token each of 64 sequences of 1 to 512 tokens
        {"name": "append_64", "kind": "append", "batch": 64, "low": 1, "high": 512, "new": 1, "n_q": 12, "n_kv": 2,
         "hd": 128, "page": 64, "dtype": "f16"},
        # the prompt chunks of four requests, up to 2048 tokens each
        {"name": "append_prompt", "kind": "append", "batch": 4, "low": 700, "high": 2048, "new": 2048, "n_q": 12,
         "n_kv": 2, "hd": 128, "page": 64, "dtype": "f16"},
        # the cache of a ragged batch of 16 back as contiguous fp16 rows (hand-over to the fp16 path)
        {"name": "read_16", "kind": "read", "batch": 16, "low": 128, "high": 8192, "n_q": 12, "n_kv": 2, "hd": 128,
         "page": 64, "dtype": "f16"},
        # decode attention of one sequence at the benchmark's 2048-token prefix: latency
        {"name": "attn_1", "kind": "attn", "batch": 1, "low": 2049, "high": 2049, "new": 1, "n_q": 12, "n_kv": 2,
         "hd": 128, "page": 64, "dtype": "f16"},
        # decode attention of 16 sequences of very different lengths
        {"name": "attn_ragged_16", "kind": "attn", "batch": 16, "low": 128, "high": 8192, "new": 1, "n_q": 12,
         "n_kv": 2, "hd": 128, "page": 64, "dtype": "f16"},
        # decode attention of eight long documents: the cache's bytes
        {"name": "attn_long_8", "kind": "attn", "batch": 8, "low": 16384, "high": 65536, "new": 1, "n_q": 12,
         "n_kv": 2, "hd": 128, "page": 256, "dtype": "f16"},
        # a 512-token prompt chunk that follows 1536 cached tokens
        {"name": "attn_prompt_512", "kind": "attn", "batch": 1, "low": 2048, "high": 2048, "new": 512, "n_q": 12,
         "n_kv": 2, "hd": 128, "page": 64, "dtype": "f16"},
        # ragged prompts of four requests in one call, fp32 queries and results, heads of 64, small pages
        {"name": "attn_prompt_ragged", "kind": "attn", "batch": 4, "low": 17, "high": 1501, "new": 700, "n_q": 28,
         "n_kv": 4, "hd": 64, "page": 16, "dtype": "f32"},
        # one sequence's next token with the engine's default settings: latency
        {"name": "sample_1", "kind": "sample", "rows": 1, "vocab": 151936, "mode": "engine", "spread": "peaked"},
        # a batch of 16 requests, each with its own settings, greedy ones among them
        {"name": "sample_16", "kind": "sample", "rows": 16, "vocab": 151936, "mode": "mixed", "spread": "peaked"},
        # 256 sequences, nucleus sampling alone, from broad distributions: thousands of tokens are kept
        {"name": "sample_256", "kind": "sample", "rows": 256, "vocab": 151936, "mode": "nucleus", "spread": "flat"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "append", "read", "attn", "attn", "attn", "sample", "sample"])
    if kind == "sample":
        rows = _log(rng, 1, 256)
        return {"kind": kind, "rows": rows, "vocab": _log(rng, 1000, 262144 if rows <= 128 else 151936),
                "mode": rng.choice(["engine", "mixed", "nucleus"]), "spread": rng.choice(["peaked", "flat"])}
    n_kv = rng.choice([1, 2, 2, 4, 8])
    heads = rng.choice([1, 2, 4, 6, 7, 8, 16]) if n_kv <= 2 else rng.choice([1, 3, 4, 7])
    case = {"kind": kind, "n_q": n_kv * heads, "n_kv": n_kv, "hd": rng.choice([64, 128, 128]),
            "page": rng.choice([16, 32, 64, 128, 256]), "dtype": rng.choice(["f16", "f16", "f32"])}
    if kind == "attn" and rng.random() < 0.5:  # prompt chunks
        batch = rng.choice([1, 1, 2, 5])
        high = _log(rng, 20, 3000 // batch)
        case |= {"batch": batch, "high": high, "new": _log(rng, 2, min(high, 700))}
    elif kind == "attn":
        high = _log(rng, 16, 32768)
        case |= {"batch": _log(rng, 1, max(1, min(64, 262144 // (high * n_kv)))), "high": high,
                 "new": rng.choice([1, 1, 1, 2, 3])}
    elif kind == "append":
        high = _log(rng, 4, 2048)
        case |= {"batch": _log(rng, 1, max(1, min(64, 32768 // (high * n_kv)))), "high": high,
                 "new": rng.choice([1, 1, _log(rng, 1, high)])}
    else:
        high = _log(rng, 16, 8192)
        case |= {"batch": _log(rng, 1, max(1, min(16, 131072 // (high * n_kv)))), "high": high}
    return case | {"low": max(1, case["high"] // rng.randint(1, 40))}


def _lengths(case):
    """Tokens of each sequence once its new rows are in: evenly spread from low to high."""
    B = case["batch"]
    return [case["high"] if B == 1 else case["low"] + (case["high"] - case["low"]) * b // (B - 1) for b in range(B)]


def _new(case):
    """New rows of each sequence."""
    return [min(case.get("new", 0), n) for n in _lengths(case)]


# ------------------------------------------------------------------------------------------------ inputs
def _normal(g, shape, scale=1.0):
    return scale * torch.randn(shape, device="cuda", generator=g)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _exponents(amax):
    """The smallest e >= E_MIN with amax <= 127 * 2^e."""
    m, x = torch.frexp(amax)
    return torch.where(amax > 0, torch.where(m <= 127 / 128, x - 7, x - 6), E_MIN).clamp_min(E_MIN).to(torch.int32)


def _blocks_of(x):
    """[B, L, heads, dims] as [B, blocks, 16, heads, dims]."""
    return x.unflatten(1, (-1, BLOCK))


def _encode(x):
    """Whole numbers of x [B, L, heads, dims] (multiples of 16 tokens) and the exponents [B, blocks, heads]."""
    e = _exponents(_blocks_of(x).abs().amax((2, 4)))
    return torch.round(torch.ldexp(_blocks_of(x), -e[:, :, None, :, None])).flatten(1, 2), e


def _to_pages(c, e, table, pages, page, is_v):
    """Whole numbers and exponents of whole sequences into a pool of pages; pages of nobody hold zeros."""
    n, hd = c.shape[2], c.shape[3]
    at = table[table >= 0].long()
    c = (c + 128).to(torch.uint8).unflatten(1, (-1, page))[table >= 0]        # [used, page, n, hd]
    c = c.unflatten(1, (-1, BLOCK)).permute(0, 3, 1, 4, 2) if is_v else c.permute(0, 2, 1, 3)
    pool = torch.full((pages, *c.shape[1:]), 128, dtype=torch.uint8, device="cuda")
    exps = torch.full((pages, n, page // BLOCK), E_MIN, dtype=torch.int8, device="cuda")
    pool[at] = c
    exps[at] = e.to(torch.int8).unflatten(1, (-1, page // BLOCK))[table >= 0].transpose(1, 2)
    return pool, exps


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    s = {"case": case}
    if case["kind"] == "sample":
        _prepare_sample(case, g, s)
    else:
        _prepare_cache(case, g, s)
    if own:
        _prepare_own(case, s)
    torch.cuda.synchronize()
    return s


def _prepare_sample(case, g, s):
    R, V = case["rows"], case["vocab"]
    s["logits"] = _normal(g, (R, V), 2.0)
    if case["spread"] == "peaked":  # a few tokens stand out, as after a clear context
        at = torch.randint(0, V, (R, 64), device="cuda", generator=g)
        s["logits"].scatter_add_(1, at, 4 + 12 * torch.rand(R, 64, device="cuda", generator=g))

    def of(values):
        pick = torch.randint(0, len(values), (R,), device="cuda", generator=g)
        return torch.tensor(values, device="cuda")[pick]

    mode = case["mode"]
    s["temperature"] = of({"engine": [0.7], "nucleus": [1.0]}.get(mode, [0.0, 0.3, 0.7, 1.0, 1.5]))
    s["top_k"] = of({"engine": [40], "nucleus": [0]}.get(mode, [0, 1, 20, 40, 500])).to(torch.int32)
    s["top_p"] = of({"engine": [0.9], "nucleus": [0.95]}.get(mode, [0.5, 0.8, 0.95, 1.0]))
    s["min_p"] = of({"mixed": [0.0, 0.02, 0.1]}.get(mode, [0.0]))
    s["u"] = torch.rand(R, dtype=torch.float64, device="cuda", generator=g)
    s["tokens"] = torch.zeros(R, dtype=torch.int32, device="cuda")


def _prepare_cache(case, g, s):
    B, n, hd, page = case["batch"], case["n_kv"], case["hd"], case["page"]
    lens, new = _lengths(case), _new(case)
    per = [-(-x // page) for x in lens]
    width = max(per)
    L, R, t = width * page, sum(new), torch.float16 if case["dtype"] == "f16" else torch.float32
    order = torch.randperm(sum(per) + 3, device="cuda", generator=g).to(torch.int32)  # pages in any order
    first = np.cumsum([0] + per)
    table = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    for b in range(B):
        table[b, :per[b]] = order[first[b]:first[b + 1]]
    kind = case["kind"]
    held = [x - (m if kind == "append" else 0) for x, m in zip(lens, new)]  # tokens that are in the cache
    live = (torch.arange(L, device="cuda") < _i32(held)[:, None])[:, :, None, None]
    # K: channels of different strength, a few of them strong, as trained models have them; V: even
    strength = torch.exp(0.5 * _normal(g, (n, hd))) * (1 + 5 * (torch.rand(n, hd, device="cuda", generator=g) < 0.03))
    for name, scale in (("k", strength), ("v", torch.ones_like(strength))):
        c, e = _encode((_normal(g, (B, L, n, hd), 0.5) * scale).half().float() * live)
        s[name + "_pages"], s[name + "_exp"] = _to_pages(c, e, table, len(order), page, name == "v")
        if kind == "append":
            s[name] = (_normal(g, (R, n, hd), 0.5) * scale).to(t)
    s["table"] = table
    s["offset"] = _i32([x - m for x, m in zip(lens, new)])
    s["row_start"] = None if max(new) <= 1 and min(new) == max(new) else _i32([0] + list(np.cumsum(new)))
    if kind != "read":
        s["q"] = _normal(g, (R, case["n_q"], hd)).to(t)
        s["out"] = torch.zeros_like(s["q"])
    if kind == "append":
        angle = torch.arange(L, device="cuda", dtype=torch.float64)[:, None] * \
            THETA ** (-torch.arange(hd // 2, device="cuda", dtype=torch.float64) * 2 / hd)
        s["cos"], s["sin"] = (f(angle).half().repeat(1, 2).contiguous() for f in (torch.cos, torch.sin))
    if kind != "attn":
        s["k_out"], s["v_out"] = (torch.zeros(B, L, n, hd, dtype=t, device="cuda") for _ in "kv")


def _prepare_own(case, s):
    """The handles that a program keeps: the library, the cache and batch descriptions, scratch memory."""
    from vte_amd.kernels import KVPages, KVRows, kernels
    K = s["K"] = kernels()
    if case["kind"] == "sample":
        s["scratch"] = torch.zeros(K.sample_scratch_bytes(case["rows"]), dtype=torch.uint8, device="cuda")
        return
    new = _new(case)
    s["pages"] = KVPages.of(s["k_pages"].data_ptr(), s["v_pages"].data_ptr(), s["k_exp"].data_ptr(),
                            s["v_exp"].data_ptr(), len(s["k_pages"]), case["page"], case["n_kv"], case["hd"])
    start = None if s["row_start"] is None else s["row_start"].data_ptr()
    s["rows"] = KVRows.of(case["batch"], sum(new), max(new), start, s["offset"].data_ptr(), s["table"].data_ptr(),
                          s["table"].shape[1])
    if case["kind"] == "attn":
        s["scratch"] = torch.zeros(K.attn_pages_scratch_bytes(s["pages"], s["rows"], case["n_q"]), dtype=torch.uint8,
                                   device="cuda")


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    return _run_own(s) if own else {"append": _append, "read": _read, "attn": _attn, "sample": _sample}[
        s["case"]["kind"]](s)


def _run_own(s):
    case, K = s["case"], s["K"]
    kind, st = case["kind"], torch.cuda.current_stream().cuda_stream
    if kind == "sample":
        K.sample(s["logits"].data_ptr(), case["rows"], case["vocab"], s["tokens"].data_ptr(), s["scratch"].data_ptr(),
                 temperature=s["temperature"].data_ptr(), top_k=s["top_k"].data_ptr(), top_p=s["top_p"].data_ptr(),
                 min_p=s["min_p"].data_ptr(), u=s["u"].data_ptr(), stream=st)
        return s["tokens"]
    pages, rows = s["pages"], s["rows"]
    if kind == "attn":
        K.attn_pages(pages, rows, s["q"].data_ptr(), s["out"].data_ptr(), case["n_q"], 1 / math.sqrt(case["hd"]),
                     s["scratch"].data_ptr(), s["scratch"].numel(), dtype=case["dtype"], stream=st)
        return s["out"]
    if kind == "append":
        K.kv_pages_append(pages, rows, s["k"].data_ptr(), s["v"].data_ptr(), q=s["q"].data_ptr(),
                          q_out=s["out"].data_ptr(), n_q=case["n_q"], rope_cos=s["cos"].data_ptr(),
                          rope_sin=s["sin"].data_ptr(), rope_rows=s["cos"].shape[0], dtype=case["dtype"], stream=st)
    K.kv_pages_read(pages, rows, s["k_out"].data_ptr(), s["v_out"].data_ptr(), s["k_out"].shape[1],
                    dtype=case["dtype"], stream=st)
    return [s["out"], s["k_out"], s["v_out"]] if kind == "append" else [s["k_out"], s["v_out"]]


def _rows(s):
    """(sequence, place in the sequence's new rows) of every row."""
    if s["row_start"] is None:
        seq = torch.arange(len(s["q"]), device="cuda")
        return seq, torch.zeros_like(seq)
    at = torch.arange(len(s["q"]), device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s["row_start"][1:], at, right=True)
    return seq, at - s["row_start"][seq]


def _ends(s):
    """Tokens of each sequence with its new rows."""
    if "q" not in s:
        return s["offset"]
    if s["row_start"] is None:
        return s["offset"] + 1
    return s["offset"] + s["row_start"].diff()


def _from_pages(s, name):
    """Whole numbers [B, L, heads, dims] in fp32 and exponents [B, blocks, heads] of the sequences' pages."""
    at = s["table"].clamp_min(0).long()
    c = s[name + "_pages"][at]                                   # [B, pages, heads, page, hd], V: [.., blocks, hd, 16]
    c = c.permute(0, 1, 3, 5, 2, 4).flatten(1, 3) if name == "v" else c.permute(0, 1, 3, 2, 4).flatten(1, 2)
    return c.float() - 128, s[name + "_exp"][at].transpose(2, 3).flatten(1, 2).int()


def _values(c, e):
    return torch.ldexp(_blocks_of(c), e[:, :, None, :, None]).flatten(1, 2)


def _rotate(x, cos, sin):
    """x [rows, heads, dims] in fp32: the halves (x0, x1) -> (x0 cos - x1 sin, x0 sin + x1 cos)."""
    a, b = x.chunk(2, 2)
    return torch.cat([a * cos - b * sin, a * sin + b * cos], 2)


def _append(s):
    seq, i = _rows(s)
    pos = (s["offset"][seq] + i).long()
    half = s["cos"].shape[1] // 2
    cos, sin = (s[n][pos, None, :half].float() for n in ("cos", "sin"))
    q = _rotate(s["q"].float(), cos, sin).to(s["q"].dtype)
    L = s["k_out"].shape[1]
    t = torch.arange(L, device="cuda")
    inside = (t < _ends(s)[:, None])[:, :, None, None]
    first = s["offset"][:, None]                                 # tokens before it are in the cache already
    old_block = (t[::BLOCK] < first)[:, :, None]                 # blocks that hold some of them
    out = []
    for name in ("k", "v"):
        x = s[name].float()
        x = _rotate(x, cos, sin) if name == "k" else x
        c, e_old = _from_pages(s, name)
        new = torch.zeros_like(c)
        new[seq, pos] = x
        e_new = _exponents(_blocks_of(new).abs().amax((2, 4)))
        e_old = torch.where(old_block, e_old, E_MIN)
        e = torch.maximum(e_old, e_new)                          # a block's scale only grows
        c = torch.round(torch.ldexp(_blocks_of(c), (e_old - e)[:, :, None, :, None]))
        x = torch.round(torch.ldexp(_blocks_of(new), -e[:, :, None, :, None]))
        c = torch.where(_blocks_of((t >= first)[:, :, None, None]), x, c).flatten(1, 2)
        out.append((_values(c, e) * inside).to(s["q"].dtype))
    return [q, *out]


def _read(s):
    inside = (torch.arange(s["k_out"].shape[1], device="cuda") < _ends(s)[:, None])[:, :, None, None]
    return [(_values(*_from_pages(s, n)) * inside).to(s["k_out"].dtype) for n in ("k", "v")]


def _attn(s):
    case, q = s["case"], s["q"].float()
    B, n, hd = case["batch"], case["n_kv"], case["hd"]
    heads = case["n_q"] // n
    seq, i = _rows(s)
    most = max(_new(case))
    k, v = (_values(*_from_pages(s, x)).transpose(1, 2) for x in ("k", "v"))           # [B, n, L, hd]
    rows = torch.zeros(B, most, case["n_q"], hd, device="cuda")
    rows[seq, i] = q
    rows = rows.reshape(B, most, n, heads, hd).transpose(1, 2).flatten(2, 3)           # [B, n, most * heads, hd]
    x = rows.matmul(k.transpose(2, 3).contiguous()) * (1 / math.sqrt(hd))
    pos = s["offset"][:, None] + torch.arange(most, device="cuda")                     # [B, most]
    seen = torch.arange(k.shape[2], device="cuda") <= pos[:, :, None]
    seen = seen & (s["table"] >= 0).repeat_interleave(case["page"], 1)[:, None]
    x.unflatten(2, (most, heads)).masked_fill_(~seen[:, None, :, None], -math.inf)
    x = torch.exp(x - x.amax(3, keepdim=True))
    x = x.matmul(v.contiguous()) / x.sum(3, keepdim=True)
    x = x.unflatten(2, (most, heads)).transpose(1, 2).reshape(B, most, case["n_q"], hd)
    return x[seq, i].to(s["q"].dtype)


def _sample(s):
    x, at = torch.sort(s["logits"], dim=1, descending=True, stable=True)
    V = x.shape[1]
    x, T = x.double(), s["temperature"].double()[:, None]
    w = torch.exp((x - x[:, :1]) / torch.where(T > 0, T, 1.0))
    k, p = s["top_k"][:, None], s["top_p"].double()[:, None]
    kept = torch.arange(V, device="cuda") < torch.where(k > 0, k, V)
    mass = torch.cumsum(w * kept, 1)
    before = torch.cat([torch.zeros_like(T), mass[:, :-1]], 1)
    kept = kept & ((before <= p * mass[:, -1:]) | (p <= 0) | (p >= 1)) & (w >= s["min_p"].double()[:, None])
    mass = torch.cumsum(w * kept, 1)
    place = (mass <= s["u"][:, None] * mass[:, -1:]).sum(1, keepdim=True)
    place = torch.minimum(place, kept.sum(1, keepdim=True) - 1)
    return at.gather(1, torch.where(T > 0, place, 0))[:, 0].int()


# ------------------------------------------------------------------------------------------------ what it costs
def work(case):
    if case["kind"] == "sample":
        return {"bytes": case["rows"] * (4 * case["vocab"] + 28), "flops": 2 * case["rows"] * case["vocab"]}
    lens, new, n, nq, hd = _lengths(case), _new(case), case["n_kv"], case["n_q"], case["hd"]
    size = 2 if case["dtype"] == "f16" else 4
    token = 2 * n * (hd + 1 / BLOCK)                             # a token's bytes and its share of the exponents
    rows = sum(new)
    if case["kind"] == "attn":
        seen = sum((2 * x - m + 1) * m // 2 for x, m in zip(lens, new))
        return {"bytes": int(sum(lens) * token + 2 * rows * nq * hd * size), "flops": 4 * nq * hd * seen}
    out = sum(lens) * (token + 2 * n * hd * size)                # the rows handed back
    if case["kind"] == "read":
        return {"bytes": int(out), "flops": 2 * sum(lens) * n * hd}
    move = rows * (2 * n * hd * size + token + 2 * nq * hd * size + 2 * hd)
    return {"bytes": int(out + move), "flops": rows * hd * (3 * nq + 7 * n) + 2 * sum(lens) * n * hd}


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "sample":
        return torch.tensor([_exact_token(s, r) for r in range(case["rows"])], dtype=torch.int32)
    lens, new = _lengths(case), _new(case)
    first = np.cumsum([0] + new)
    if case["kind"] == "attn":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        for b in range(case["batch"]):
            k, v = (_exact_rows(s, x, b, lens[b]) for x in ("k", "v"))
            place = torch.arange(lens[b], device="cuda")
            hidden = place[None] > torch.arange(lens[b] - new[b], lens[b], device="cuda")[:, None]
            for h in range(case["n_q"]):
                j = h // (case["n_q"] // case["n_kv"])
                x = s["q"][first[b]:first[b + 1], h].double() @ k[:, j].T / math.sqrt(case["hd"])
                out[first[b]:first[b + 1], h] = torch.softmax(x.masked_fill(hidden, -math.inf), 1) @ v[:, j]
        return out
    L = s["k_out"].shape[1]
    k_all, v_all = (torch.zeros(s["k_out"].shape, dtype=torch.float64, device="cuda") for _ in "kv")
    q = None
    if case["kind"] == "append":
        q = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b in range(case["batch"]):
        a, z = lens[b] - new[b], lens[b]
        for name, full in (("k", k_all), ("v", v_all)):
            if case["kind"] == "read":
                full[b, :z] = _exact_rows(s, name, b, z)
                continue
            x = s[name][first[b]:first[b + 1]].double()
            full[b, :z] = _exact_append(s, name, b, a, _exact_turn(s, x, a) if name == "k" else x)
        if q is not None:
            q[first[b]:first[b + 1]] = _exact_turn(s, s["q"][first[b]:first[b + 1]].double(), a)
    assert L >= max(lens)
    return [k_all, v_all] if q is None else [q, k_all, v_all]


def _exact_codes(s, name, b, count):
    """(bytes, exponents) of the first `count` tokens of sequence b, token by token: [count, heads, dims], [count, heads]."""
    page = s["case"]["page"]
    t = torch.arange(count, device="cuda")
    p, r = s["table"][b].long()[t // page], t % page
    if name == "k":
        c = s["k_pages"][p, :, r]
    else:
        c = s["v_pages"][p, :, r // BLOCK, :, r % BLOCK]
    return c.double() - 128, s[name + "_exp"][p, :, r // BLOCK].double()


def _exact_rows(s, name, b, count):
    c, e = _exact_codes(s, name, b, count)
    return c * torch.exp2(e)[:, :, None]


def _exact_turn(s, x, a):
    cos, sin = (s[n][a:a + len(x)].double()[:, None] for n in ("cos", "sin"))
    h = x.shape[2] // 2
    return torch.cat([x[..., :h] * cos[..., :h] - x[..., h:] * sin[..., :h],
                      x[..., h:] * cos[..., h:] + x[..., :h] * sin[..., h:]], 2)


def _exact_append(s, name, b, a, x):
    """Sequence b's values once rows x stand at positions a, a + 1, ..."""
    full = torch.cat([_exact_rows(s, name, b, a), x])
    _, e = _exact_codes(s, name, b, a)
    c = full.clone()
    start = a // BLOCK * BLOCK
    for lo in range(start, len(full), BLOCK):
        part = full[lo:lo + BLOCK]
        most = part[max(0, a - lo):].abs().amax((0, 2))          # of the new rows, each head
        step = torch.ceil(torch.log2((most / 127).clamp_min(2.0 ** E_MIN)))
        step = torch.where(most > 127 * torch.exp2(step), step + 1, step)
        step = torch.where(most <= 127 * torch.exp2(step - 1), step - 1, step).clamp_min(E_MIN)
        step = torch.maximum(step, e[lo]) if lo < a else step
        unit = torch.exp2(step)[None, :, None]
        c[lo:lo + BLOCK] = torch.round(part / unit) * unit
    return c


def _exact_token(s, r):
    x = s["logits"][r].double().cpu().numpy()
    T, k, p, floor, u = (float(s[n][r]) for n in ("temperature", "top_k", "top_p", "min_p", "u"))
    order = np.argsort(-x, kind="stable")
    if T <= 0:
        return int(order[0])
    order = order[:int(k)] if k > 0 else order
    w = np.exp((x[order] - x[order[0]]).astype(np.longdouble) / np.longdouble(T))
    total = np.cumsum(w)
    if 0 < p < 1:
        w = w[:1 + int(np.searchsorted(total[:-1], p * total[-1], side="right"))]
    w = w[w >= floor]
    total = np.cumsum(w)
    return int(order[min(int(np.searchsorted(total, u * total[-1], side="right")), len(w) - 1)])
