"""Operators of long conversations over the 8-bit paged KV cache: their performance cases.

* ``norm``: queries and keys normed head by head and rotated by their positions (the pairs' frequencies are given, so
  that scaled rotations for long contexts are, too), for a cache that is not paged;
* ``append``: the same on the way into the pages, and the cache's rows handed back;
* ``attn``: attention of decoded tokens or prompt chunks that see a sliding window and the first few tokens;
* ``fork``: sequences that ended give their pages back, others' prompts are shared with them, and they get room for
  their next tokens; ``compact``: the used pages of a scattered pool move to its beginning.

The cache holds K and V as bytes.  16 consecutive tokens of one KV head (a block) share one scale 2^e; a value is
(byte - 128) * 2^e.  A page holds ``page`` tokens of every KV head, K as [head][token][dim], V block by block as
[head][block][dim][16 tokens], and one exponent per head and block for each.  Sequence b's tokens lie in the pages of
row b of the page table; its new rows are rows row_start[b] .. of q, k and v, the first of them at position
kv_offset[b] (one row per sequence where there is no row_start).  Each page has a count of its users, 0: free; one
table serves every layer's pages.

Where ``own`` is false, ``run`` computes in elementary torch operations; where it is true it calls the framework.
Sizes are those of the repository's model configurations, benchmark and tests (12 query and 2 KV heads, 28 and 4, of
128, 28 layers, prompts in chunks of 512) and generic ones around them.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
BLOCK = 16         # tokens that share a scale
E_MIN = -126       # the smallest exponent of a block
EPS = 1e-6         # of the norms
THETA = 1e6        # base of the rotation's angles


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # q and k of one decoded token: latency
        {"name": "norm_1", "kind": "norm", "rows": 1, "n_q": 12, "n_kv": 2, "hd": 128, "rot": 128, "inter": False,
         "scaled": False, "far": 2048, "dtype": "f16"},
        # prompts of 4096 tokens at far positions, half of each head rotated in neighbouring pairs, fp32
        {"name": "norm_prompt", "kind": "norm", "rows": 4096, "n_q": 28, "n_kv": 4, "hd": 128, "rot": 64, "inter": True,
         "scaled": True, "far": 131072, "dtype": "f32"},
        # one decoded token each of 64 sequences of 1 to 512 tokens
        {"name": "append_64", "kind": "append", "batch": 64, "low": 1, "high": 512, "new": 1, "n_q": 12, "n_kv": 2,
         "hd": 128, "rot": 128, "inter": False, "scaled": False, "page": 64, "dtype": "f16"},
        # the prompt chunks of four requests, up to 2048 tokens each, a rotation scaled for long contexts
        {"name": "append_prompt", "kind": "append", "batch": 4, "low": 700, "high": 2048, "new": 2048, "n_q": 12,
         "n_kv": 2, "hd": 128, "rot": 128, "inter": False, "scaled": True, "page": 64, "dtype": "f16"},
        # the next token of one conversation of 32768 tokens: latency
        {"name": "window_1", "kind": "attn", "batch": 1, "low": 32768, "high": 32768, "new": 1, "n_q": 12, "n_kv": 2,
         "hd": 128, "page": 64, "window": 4096, "sinks": 4, "dtype": "f16"},
        # the next tokens of 64 conversations, some shorter than the window, most far beyond: the windows' bytes
        {"name": "window_64", "kind": "attn", "batch": 64, "low": 1000, "high": 65000, "new": 1, "n_q": 28, "n_kv": 4,
         "hd": 128, "page": 64, "window": 4096, "sinks": 16, "dtype": "f16"},
        # a 512-token prompt chunk at the end of 32768 tokens
        {"name": "window_prompt_512", "kind": "attn", "batch": 1, "low": 32768, "high": 32768, "new": 512, "n_q": 12,
         "n_kv": 2, "hd": 128, "page": 64, "window": 4096, "sinks": 4, "dtype": "f16"},
        # ragged prompts of four requests whose windows are shorter than they are: fp32, heads of 64, small pages
        {"name": "window_prompt_ragged", "kind": "attn", "batch": 4, "low": 17, "high": 2501, "new": 1500, "n_q": 28,
         "n_kv": 4, "hd": 64, "page": 16, "window": 300, "sinks": 1, "dtype": "f32"},
        # eight answers to one prompt of the benchmark's length, pages of 28 layers
        {"name": "fork_8", "kind": "fork", "parents": 1, "children": 8, "low": 2049, "high": 2049, "new": 1, "n_kv": 2,
         "hd": 128, "page": 64, "layers": 28, "spare": 64},
        # four answers to each of 16 prompts of very different lengths, with room for 100 tokens each
        {"name": "fork_64", "kind": "fork", "parents": 16, "children": 64, "low": 90, "high": 4000, "new": 100,
         "n_kv": 2, "hd": 128, "page": 64, "layers": 28, "spare": 300},
        # a small pool of small pages, a quarter of them free
        {"name": "compact_256", "kind": "compact", "pages": 256, "used": 192, "seqs": 8, "n_kv": 2, "hd": 64,
         "page": 16, "layers": 28},
        # a pool of 28 layers half full of scattered pages
        {"name": "compact_1024", "kind": "compact", "pages": 1024, "used": 512, "seqs": 32, "n_kv": 2, "hd": 128,
         "page": 64, "layers": 28},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "append", "append", "attn", "attn", "attn", "fork", "fork", "compact"])
    if kind == "fork":
        parents, page, layers = _log(rng, 1, 16), rng.choice([16, 32, 64, 128]), rng.choice([1, 7, 28])
        high = _log(rng, 4, 4000)
        return {"kind": kind, "parents": parents, "children": _log(rng, 1, 64), "low": max(1, high // rng.randint(1, 40)),
                "high": high, "new": _log(rng, 1, 300), "n_kv": rng.choice([1, 2, 4]) if page < 64 else 2,
                "hd": rng.choice([64, 128]), "page": page, "layers": layers, "spare": _log(rng, 30, 300)}
    if kind == "compact":
        pages, page = _log(rng, 10, 1024), rng.choice([16, 32, 64])
        return {"kind": kind, "pages": pages, "used": rng.randint(0, pages), "seqs": _log(rng, 1, 32),
                "n_kv": rng.choice([1, 2]), "hd": rng.choice([64, 128]), "page": page, "layers": rng.choice([1, 7, 28])}
    n_kv = rng.choice([1, 2, 2, 4, 8])
    heads = rng.choice([1, 2, 4, 6, 7, 8, 16]) if n_kv <= 2 else rng.choice([1, 3, 4, 7])
    hd = rng.choice([64, 128, 128])
    case = {"kind": kind, "n_q": n_kv * heads, "n_kv": n_kv, "hd": hd, "dtype": rng.choice(["f16", "f16", "f32"])}
    if kind != "attn":
        case |= {"rot": rng.choice([hd, hd, hd // 2, 2 * rng.randint(1, hd // 2)]), "inter": rng.random() < 0.4,
                 "scaled": rng.random() < 0.5}
    if kind == "norm":
        case["hd"] = rng.choice([64, 128, 256]) if case["rot"] <= 64 else rng.choice([128, 256])
        values = 4096 * 32 * 128 // (n_kv * (heads + 1) * case["hd"])
        return case | {"rows": _log(rng, 1, min(4096, values)), "far": _log(rng, 2, 1000000)}
    case["page"] = rng.choice([16, 32, 64, 128, 256])
    if kind == "append":
        high = _log(rng, 4, 2048)
        case |= {"batch": _log(rng, 1, max(1, min(64, 32768 // (high * n_kv)))), "high": high,
                 "new": rng.choice([1, 1, _log(rng, 1, high)])}
    else:
        case |= {"window": _log(rng, 1, 8192), "sinks": rng.choice([0, 1, 4, 16, rng.randint(0, 200)])}
        if rng.random() < 0.5:  # prompt chunks
            high = _log(rng, 20, 20000)
            case |= {"batch": rng.choice([1, 1, 2, 5]), "high": high}
            case["window"] = min(case["window"], 4096 // case["batch"])
            most = 12_000_000_000 // (4 * hd * case["n_q"] * min(high, case["window"] + case["sinks"]) * case["batch"])
            case["new"] = _log(rng, 2, max(2, min(high, most, 2000 // case["batch"])))
        else:
            high = _log(rng, 16, 65000)
            seen = min(high, case["window"] + case["sinks"] + 2)
            case |= {"batch": _log(rng, 1, max(1, min(64, 500000 // (seen * n_kv)))), "high": high,
                     "new": rng.choice([1, 1, 1, 2, 3])}
    return case | {"low": max(1, case["high"] // rng.randint(1, 40))}


def _lengths(case, n=None):
    """Tokens of each sequence once its new rows are in: evenly spread from low to high."""
    B = n or case["batch"]
    return [case["high"] if B == 1 else case["low"] + (case["high"] - case["low"]) * b // (B - 1) for b in range(B)]


def _new(case):
    """New rows of each sequence."""
    return [min(case["new"], n) for n in _lengths(case)]


# ------------------------------------------------------------------------------------------------ inputs
def _normal(g, shape, scale=1.0):
    return scale * torch.randn(shape, device=DEVICE, generator=g)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _type(case):
    return torch.float16 if case["dtype"] == "f16" else torch.float32


def _exponents(amax):
    """The smallest e >= E_MIN with amax <= 127 * 2^e."""
    m, x = torch.frexp(amax)
    return torch.where(amax > 0, torch.where(m <= 127 / 128, x - 7, x - 6), E_MIN).clamp_min(E_MIN).to(torch.int32)


def _blocks_of(x):
    """[B, L, heads, dims] as [B, blocks, 16, heads, dims]."""
    return x.unflatten(1, (-1, BLOCK))


def _pool(x, is_v):
    """Pages x [pages, token, heads, dims] as bytes and exponents."""
    e = _exponents(_blocks_of(x).abs().amax((2, 4)))                                 # [pages, blocks, heads]
    c = (torch.round(torch.ldexp(_blocks_of(x), -e[:, :, None, :, None])) + 128).to(torch.uint8)
    c = c.permute(0, 3, 1, 4, 2) if is_v else c.flatten(1, 2).permute(0, 2, 1, 3)
    return c.contiguous(), e.transpose(1, 2).to(torch.int8).contiguous()


def _frequencies(rot, scaled):
    """Radians per position of each pair, and what cos and sin are multiplied with.  Scaled: for eight times the context
    of 32768 tokens, pairs that turn less than once in it eight times slower, those of over 32 turns as they are."""
    f = THETA ** (-np.arange(0, rot, 2, dtype=np.float64) / rot)
    if not scaled:
        return f, 1.0
    turns = 32768 * f / (2 * math.pi)
    keep = np.clip((turns - 1) / (32 - 1), 0, 1)
    return f * (keep + (1 - keep) / 8), 0.1 * math.log(8) + 1


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(seed))
    s = {"case": case}
    {"norm": _prepare_norm, "append": _prepare_cache, "attn": _prepare_cache, "fork": _prepare_fork,
     "compact": _prepare_compact}[case["kind"]](case, g, s)
    if own:
        _prepare_own(case, s)
    if DEVICE == "cuda":
        torch.cuda.synchronize()
    return s


def _prepare_form(case, g, s):
    """Weights of the norms, around one and a few of them large, and the rotation."""
    f, s["amplitude"] = _frequencies(case["rot"], case["scaled"])
    s["freq"] = torch.from_numpy(f).to(DEVICE)
    for name in ("q_norm", "k_norm"):
        strong = 1 + 4 * (torch.rand(case["hd"], device=DEVICE, generator=g) < 0.05)
        s[name] = ((1 + _normal(g, (case["hd"],), 0.2)) * strong).half()


def _prepare_norm(case, g, s):
    t, R, hd = _type(case), case["rows"], case["hd"]
    _prepare_form(case, g, s)
    s["q"], s["k"] = (_normal(g, (R, case[n], hd), 2.0).to(t) for n in ("n_q", "n_kv"))
    s["q_out"], s["k_out"] = torch.zeros_like(s["q"]), torch.zeros_like(s["k"])
    first = torch.randint(0, max(1, case["far"] - R), (1,), device=DEVICE, generator=g)
    s["pos"] = (first + torch.arange(R, device=DEVICE)).to(torch.int32)


def _prepare_cache(case, g, s):
    B, n, hd, page = case["batch"], case["n_kv"], case["hd"], case["page"]
    lens, new, t = _lengths(case), _new(case), _type(case)
    width = -(-max(lens) // page)
    L, R = width * page, sum(new)
    s["offset"] = _i32([x - m for x, m in zip(lens, new)])
    s["row_start"] = None if max(new) <= 1 and min(new) == max(new) else _i32([0] + list(np.cumsum(new)))
    # pages in any order; those that no row sees any more are given back
    at = torch.arange(width, device=DEVICE) * page
    live = at < _i32(lens)[:, None]
    if case["kind"] == "attn":
        live &= (at < case["sinks"]) | (at + page > s["offset"][:, None] + 1 - case["window"])
    count = int(live.sum())
    order = torch.randperm(count + 3, device=DEVICE, generator=g).to(torch.int32)
    s["table"] = torch.full((B, width), -1, dtype=torch.int32, device=DEVICE)
    s["table"][live] = order[:count]
    # K: channels of different strength, a few of them strong, as trained models have them; V: even
    strength = torch.exp(0.5 * _normal(g, (n, hd))) * (1 + 5 * (torch.rand(n, hd, device=DEVICE, generator=g) < 0.03))
    for name, scale in (("k", strength), ("v", torch.ones_like(strength))):
        x = _normal(g, (count + 3, page, n, hd), 0.5) * scale
        s[name + "_pages"], s[name + "_exp"] = _pool(x, name == "v")
        if case["kind"] == "append":
            s[name] = (_normal(g, (R, n, hd), 0.5) * scale).to(t)
    s["q"] = _normal(g, (R, case["n_q"], hd)).to(t)
    s["out"] = torch.zeros_like(s["q"])
    if case["kind"] == "append":
        _prepare_form(case, g, s)
        s["k_out"], s["v_out"] = (torch.zeros(B, L, n, hd, dtype=torch.float16, device=DEVICE) for _ in "kv")


def _prepare_pools(case, pages, g, s):
    """Every layer's pages: any bytes."""
    n, hd, page, layers = case["n_kv"], case["hd"], case["page"], case["layers"]
    for name, shape in (("k_pages", (n, page, hd)), ("v_pages", (n, page // BLOCK, hd, BLOCK)),
                        ("k_exp", (n, page // BLOCK)), ("v_exp", (n, page // BLOCK))):
        low, high, t = (0, 256, torch.uint8) if "pages" in name else (-20, 20, torch.int8)
        s[name] = torch.randint(low, high, (layers, pages, *shape), dtype=t, device=DEVICE, generator=g)


def _prepare_fork(case, g, s):
    """Parents with their prompts, children with what is left of earlier answers."""
    P, C, page = case["parents"], case["children"], case["page"]
    lens = _lengths(case, P)
    rows = [-(-x // page) for x in lens] + [1 + (7 * i) % 5 for i in range(C)]
    width = max(max(rows), -(-(max(lens) + case["new"]) // page))
    held = torch.arange(width, device=DEVICE) < _i32(rows)[:, None]
    pages = sum(rows) + case["spare"]
    s["table"] = torch.full((P + C, width), -1, dtype=torch.int32, device=DEVICE)
    s["table"][held] = torch.randperm(pages, device=DEVICE, generator=g)[:sum(rows)].to(torch.int32)
    s["refs"] = torch.zeros(pages, dtype=torch.int32, device=DEVICE)
    s["refs"][s["table"][held].long()] = 1
    s["parent"] = _i32([i % P for i in range(C)])
    s["child"] = _i32([P + i for i in range(C)])
    s["length"] = _i32([lens[i % P] for i in range(C)])
    s["missing"] = torch.zeros(2, dtype=torch.int32, device=DEVICE)
    _prepare_pools(case, pages, g, s)


def _prepare_compact(case, g, s):
    """Tables whose entries are the used pages, some of them shared by two sequences."""
    pages, used, seqs = case["pages"], case["used"], case["seqs"]
    width = -(-(used + used // 4) // seqs) + 1
    entries = torch.full((seqs * width,), -1, dtype=torch.int32, device=DEVICE)
    mine = torch.randperm(pages, device=DEVICE, generator=g)[:used].to(torch.int32)
    entries[:used] = mine
    entries[used:used + used // 4] = mine[:used // 4]
    s["table0"] = entries.reshape(seqs, width)
    s["refs0"] = torch.zeros(pages, dtype=torch.int32, device=DEVICE)
    s["refs0"].index_add_(0, entries.clamp_min(0), (entries >= 0).int())
    s["table"], s["refs"] = s["table0"].clone(), s["refs0"].clone()
    s["where"] = torch.zeros(pages, dtype=torch.int32, device=DEVICE)
    s["used"] = torch.zeros(1, dtype=torch.int32, device=DEVICE)
    _prepare_pools(case, pages, g, s)


def _prepare_own(case, s):
    """The handles that a program keeps: the library, descriptions of the cache, the batch and the model, scratch memory."""
    from vte_amd.kernels import HeadForm, KVPages, KVRows, KVTables, kernels
    K = s["K"] = kernels()
    kind = case["kind"]
    if kind in ("norm", "append"):
        s["form"] = HeadForm.of(s["freq"].data_ptr(), case["rot"], case["inter"], s["amplitude"],
                                s["q_norm"].data_ptr(), s["k_norm"].data_ptr(), EPS)
    if kind in ("append", "attn"):
        new = _new(case)
        s["pages"] = KVPages.of(s["k_pages"].data_ptr(), s["v_pages"].data_ptr(), s["k_exp"].data_ptr(),
                                s["v_exp"].data_ptr(), len(s["k_pages"]), case["page"], case["n_kv"], case["hd"])
        start = None if s["row_start"] is None else s["row_start"].data_ptr()
        s["rows"] = KVRows.of(case["batch"], sum(new), max(new), start, s["offset"].data_ptr(), s["table"].data_ptr(),
                              s["table"].shape[1])
    if kind == "attn":
        n = K.attn_pages_window_scratch_bytes(s["pages"], s["rows"], case["n_q"], case["window"], case["sinks"])
        s["scratch"] = torch.zeros(n, dtype=torch.uint8, device=DEVICE)
    if kind in ("fork", "compact"):
        pages = s["refs"].numel()
        s["layers"] = (KVPages * case["layers"])(*[
            KVPages.of(s["k_pages"][i].data_ptr(), s["v_pages"][i].data_ptr(), s["k_exp"][i].data_ptr(),
                       s["v_exp"][i].data_ptr(), pages, case["page"], case["n_kv"], case["hd"])
            for i in range(case["layers"])])
        s["tables"] = KVTables.of(s["table"].data_ptr(), s["refs"].data_ptr(), s["table"].shape[0],
                                  s["table"].shape[1], pages, case["page"])
        n = K.kv_pages_fork_scratch_bytes(case["children"]) if kind == "fork" else \
            K.kv_pages_compact_scratch_bytes(s["tables"])
        s["scratch"] = torch.zeros(n, dtype=torch.uint8, device=DEVICE)


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    return _run_own(s) if own else {"norm": _norm, "append": _append, "attn": _attn, "fork": _fork,
                                    "compact": _compact}[s["case"]["kind"]](s)


def _run_own(s):
    case, K = s["case"], s["K"]
    kind, st = case["kind"], torch.cuda.current_stream().cuda_stream
    if kind == "norm":
        K.qk_norm_rope(s["form"], case["rows"], s["pos"].data_ptr(), q=s["q"].data_ptr(), q_out=s["q_out"].data_ptr(),
                       n_q=case["n_q"], k=s["k"].data_ptr(), k_out=s["k_out"].data_ptr(), n_kv=case["n_kv"],
                       head_dim=case["hd"], dtype=case["dtype"], stream=st)
        return [s["q_out"], s["k_out"]]
    if kind == "append":
        K.kv_pages_append_norm(s["pages"], s["rows"], s["form"], s["k"].data_ptr(), s["v"].data_ptr(),
                               q=s["q"].data_ptr(), q_out=s["out"].data_ptr(), n_q=case["n_q"], dtype=case["dtype"],
                               stream=st)
        K.kv_pages_read(s["pages"], s["rows"], s["k_out"].data_ptr(), s["v_out"].data_ptr(), s["k_out"].shape[1],
                        stream=st)
        return [s["out"], s["k_out"], s["v_out"]]
    if kind == "attn":
        K.attn_pages_window(s["pages"], s["rows"], s["q"].data_ptr(), s["out"].data_ptr(), case["n_q"],
                            1 / math.sqrt(case["hd"]), case["window"], case["sinks"], s["scratch"].data_ptr(),
                            s["scratch"].numel(), dtype=case["dtype"], stream=st)
        return s["out"]
    if kind == "fork":
        n, child, missing = case["children"], s["child"].data_ptr(), s["missing"].data_ptr()
        K.kv_pages_free(s["tables"], n, seqs=child, stream=st)
        K.kv_pages_fork(s["layers"], s["tables"], n, s["parent"].data_ptr(), child, s["length"].data_ptr(), missing,
                        s["scratch"].data_ptr(), s["scratch"].numel(), stream=st)
        K.kv_pages_reserve(s["tables"], n, s["length"].data_ptr(), case["new"], missing + 4, seqs=child, stream=st)
        return [s["table"], s["refs"], s["missing"], *_bytes(s)]
    s["table"].copy_(s["table0"])  # (scattered again; the pages moved from still hold their bytes)
    s["refs"].copy_(s["refs0"])
    K.kv_pages_compact(s["layers"], s["tables"], s["where"].data_ptr(), s["used"].data_ptr(), s["scratch"].data_ptr(),
                       s["scratch"].numel(), stream=st)
    return [s["table"], s["refs"], s["where"], s["used"], *_bytes(s)]


def _bytes(s):
    """The pages as they stand.  Copies know no values: whole numbers, equal byte for byte."""
    return [s["k_pages"].view(torch.int32), s["v_pages"].view(torch.int32), s["k_exp"], s["v_exp"]]


def _rows(s):
    """(sequence, place in the sequence's new rows) of every row."""
    if s["row_start"] is None:
        seq = torch.arange(len(s["q"]), device=DEVICE)
        return seq, torch.zeros_like(seq)
    at = torch.arange(len(s["q"]), device=DEVICE, dtype=torch.int32)
    seq = torch.searchsorted(s["row_start"][1:], at, right=True)
    return seq, at - s["row_start"][seq]


def _ends(s):
    """Tokens of each sequence with its new rows."""
    return s["offset"] + (1 if s["row_start"] is None else s["row_start"].diff())


def _turned(s, x, weight, pos):
    """x [rows, heads, dims] in fp32: normed, and its first dims rotated by the rows' positions."""
    rot, inter = s["case"]["rot"], s["case"]["inter"]
    x = x * torch.rsqrt(x.square().mean(2, keepdim=True) + EPS) * weight.float()
    angle = pos.double()[:, None, None] * s["freq"]
    cos, sin = (f(angle).float() * s["amplitude"] for f in (torch.cos, torch.sin))
    y, rest = x[..., :rot], x[..., rot:]
    a, b = (y[..., 0::2], y[..., 1::2]) if inter else y.chunk(2, 2)
    a, b = a * cos - b * sin, a * sin + b * cos
    return torch.cat([torch.stack([a, b], 3).flatten(2) if inter else torch.cat([a, b], 2), rest], 2)


def _norm(s):
    return [_turned(s, s[n].float(), s[n + "_norm"], s["pos"]).to(s[n].dtype) for n in ("q", "k")]


def _from_pages(s, name):
    """Whole numbers [B, L, heads, dims] in fp32 and exponents [B, blocks, heads] of the sequences' pages."""
    at = s["table"].clamp_min(0).long()
    c = s[name + "_pages"][at]                                   # [B, pages, heads, page, hd], V: [.., blocks, hd, 16]
    c = c.permute(0, 1, 3, 5, 2, 4).flatten(1, 3) if name == "v" else c.permute(0, 1, 3, 2, 4).flatten(1, 2)
    return c.float() - 128, s[name + "_exp"][at].transpose(2, 3).flatten(1, 2).int()


def _append(s):
    seq, i = _rows(s)
    pos = (s["offset"][seq] + i).long()
    q = _turned(s, s["q"].float(), s["q_norm"], pos).to(s["q"].dtype)
    t = torch.arange(s["k_out"].shape[1], device=DEVICE)
    inside = (t < _ends(s)[:, None])[:, :, None, None]
    first = s["offset"][:, None]                                 # tokens before it are in the cache already
    old_block = (t[::BLOCK] < first)[:, :, None]                 # blocks that hold some of them
    out = []
    for name in ("k", "v"):
        x = s[name].float()
        x = _turned(s, x, s["k_norm"], pos) if name == "k" else x
        c, e_old = _from_pages(s, name)
        new = torch.zeros_like(c)
        new[seq, pos] = x
        e_new = _exponents(_blocks_of(new).abs().amax((2, 4)))
        e_old = torch.where(old_block, e_old, E_MIN)
        e = torch.maximum(e_old, e_new)                          # a block's scale only grows
        c = torch.round(torch.ldexp(_blocks_of(c), (e_old - e)[:, :, None, :, None]))
        x = torch.round(torch.ldexp(_blocks_of(new), -e[:, :, None, :, None]))
        c = torch.where(_blocks_of((t >= first)[:, :, None, None]), x, c)
        out.append((torch.ldexp(c, e[:, :, None, :, None]).flatten(1, 2) * inside).half())
    return [q, *out]


def _attn(s):
    case, q = s["case"], s["q"].float()
    B, n, hd, page, sinks = case["batch"], case["n_kv"], case["hd"], case["page"], case["sinks"]
    heads, most, window = case["n_q"] // n, max(_new(case)), min(case["window"], case["high"])
    seq, i = _rows(s)
    off = s["offset"][:, None]
    low = (off + 1 - window).clamp_min(0)                        # the first token of the first row's window
    t = torch.cat([torch.arange(min(sinks, case["high"]), device=DEVICE).expand(B, -1),
                   low + torch.arange(window + most - 1, device=DEVICE)], 1)            # [B, U]
    there = t < _ends(s)[:, None]
    there[:, :min(sinks, case["high"])] &= t[:, :min(sinks, case["high"])] < low         # (each token once)
    t = t.clamp_max(s["table"].shape[1] * page - 1)
    at = torch.gather(s["table"], 1, t // page).long()
    there &= at >= 0
    at, r = at.clamp_min(0), t % page
    k = s["k_pages"][at, :, r]                                   # [B, U, n, hd]
    v = s["v_pages"][at, :, r // BLOCK, :, r % BLOCK]
    k, v = (torch.ldexp(c.float() - 128, s[e][at, :, r // BLOCK].int()[..., None]).transpose(1, 2)
            for c, e in ((k, "k_exp"), (v, "v_exp")))
    rows = torch.zeros(B, most, case["n_q"], hd, device=DEVICE)
    rows[seq, i] = q
    rows = rows.reshape(B, most, n, heads, hd).transpose(1, 2).flatten(2, 3)            # [B, n, most * heads, hd]
    x = rows.matmul(k.transpose(2, 3).contiguous()) * (1 / math.sqrt(hd))
    pos = off + torch.arange(most, device=DEVICE)                                       # [B, most]
    seen = (t[:, None] <= pos[:, :, None]) & ((t[:, None] > pos[:, :, None] - case["window"]) | (t[:, None] < sinks))
    seen = seen & there[:, None]
    x.unflatten(2, (most, heads)).masked_fill_(~seen[:, None, :, None], -math.inf)
    x = torch.exp(x - x.amax(3, keepdim=True))
    x = x.matmul(v.contiguous()) / x.sum(3, keepdim=True)
    x = x.unflatten(2, (most, heads)).transpose(1, 2).reshape(B, most, case["n_q"], hd)
    return x[seq, i].to(s["q"].dtype)


def _users(s, entries, by):
    s["refs"].index_add_(0, entries.clamp_min(0).flatten(), by * (entries >= 0).int().flatten())


def _lowest_free(s, wanted):
    """Free pages for the places where `wanted` (any shape) is true, in order, the lowest first; -1 where they end."""
    taken = (s["refs"] > 0).int()
    order = torch.argsort(taken, stable=True).int()
    rank = torch.cumsum(wanted.flatten(), 0).reshape(wanted.shape) - 1
    got = wanted & (rank < (1 - taken).sum())
    new = torch.where(got, order[rank.clamp(0, len(order) - 1)], -1)
    _users(s, new, 1)
    return new, (wanted & ~got).sum()


def _fork(s):
    page = s["case"]["page"]
    table, child, n = s["table"], s["child"].long(), s["length"][:, None]
    _users(s, table[child], -1)                                  # the ended ones' pages
    parent = table[s["parent"].long()]
    j = torch.arange(table.shape[1], device=DEVICE)
    shared = torch.where(j < n // page, parent, -1)
    _users(s, shared, 1)
    begun = (n // page).clamp_max(table.shape[1] - 1).long()     # the page that is not full
    source = parent.gather(1, begun)
    new, s["missing"][0] = _lowest_free(s, (n % page > 0) & (source >= 0))
    here = torch.where(new >= 0, new, source).clamp_min(0).flatten().long()  # (those without one: onto themselves)
    source = source.clamp_min(0).flatten().long()
    for name in ("k_pages", "v_pages", "k_exp", "v_exp"):
        s[name][:, here] = s[name][:, source]
    row = torch.where(j == n // page, new, shared)
    room = (j * page < n + s["case"]["new"]) & ((j + 1) * page > n)
    more, s["missing"][1] = _lowest_free(s, room & (row < 0))
    table[child] = torch.where(more >= 0, more, row)
    return [table, s["refs"], s["missing"], *_bytes(s)]


def _compact(s):
    s["table"].copy_(s["table0"])
    s["refs"].copy_(s["refs0"])
    taken = s["refs"] > 0
    p = torch.arange(len(taken), device=DEVICE)
    used = taken.sum()
    source, to = torch.nonzero(taken & (p >= used))[:, 0], torch.nonzero(~taken & (p < used))[:, 0]
    for name in ("k_pages", "v_pages", "k_exp", "v_exp"):
        s[name][:, to] = s[name][:, source]
    where = torch.where(taken, p, -1).int()
    where[source] = to.int()
    s["refs"][to] = s["refs"][source]
    s["refs"][source] = 0
    s["table"].copy_(torch.where(s["table"] >= 0, where[s["table"].clamp_min(0)], -1))
    return [s["table"], s["refs"], where, used.int().reshape(1), *_bytes(s)]


# ------------------------------------------------------------------------------------------------ what it costs
def work(case):
    kind, n, hd = case["kind"], case["n_kv"], case["hd"]
    if kind in ("fork", "compact"):
        page = 2 * n * case["page"] * (hd + 1 / BLOCK) * case["layers"]      # of all layers
        if kind == "compact":  # used pages that lie behind the first `used`: moved
            moved = case["used"] * (1 - case["used"] / case["pages"])
            entries = case["seqs"] * (-(-(case["used"] + case["used"] // 4) // case["seqs"]) + 1)
            return {"bytes": int(2 * moved * page + 12 * case["pages"] + 16 * entries), "flops": 0}
        lens = _lengths(case, case["parents"])
        lens = [lens[i % len(lens)] for i in range(case["children"])]
        copied = sum(x % case["page"] > 0 for x in lens)
        entries = sum(-(-(x + case["new"]) // case["page"]) for x in lens)
        return {"bytes": int(2 * copied * page + 16 * entries), "flops": 0}
    size, nq = 2 if case["dtype"] == "f16" else 4, case["n_q"]
    token = 2 * n * (hd + 1 / BLOCK)                             # a token's bytes and its share of the exponents
    turn = 5 * hd + 3 * case.get("rot", 0)                       # a head's norm and rotation
    if kind == "norm":
        return {"bytes": case["rows"] * (2 * (nq + n) * hd * size + 4), "flops": case["rows"] * (nq + n) * turn}
    lens, new = _lengths(case), _new(case)
    rows = sum(new)
    if kind == "attn":
        W, S = case["window"], case["sinks"]
        held = sum(x - max(0, x - m + 1 - W - S) for x, m in zip(lens, new))
        seen = sum(min(p + 1, W + min(S, max(0, p + 1 - W))) for x, m in zip(lens, new) for p in range(x - m, x))
        return {"bytes": int(held * token + 2 * rows * nq * hd * size), "flops": 4 * nq * hd * seen}
    out = sum(lens) * (token + 2 * n * hd * 2)                   # the rows handed back
    move = rows * (2 * n * hd * size + token + 2 * nq * hd * size)
    return {"bytes": int(out + move), "flops": rows * ((nq + n) * turn + 4 * n * hd) + 2 * sum(lens) * n * hd}


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    if case["kind"] in ("fork", "compact"):
        return None  # (whole numbers)
    s = prepare(case, seed)
    if case["kind"] == "norm":
        return [_exact_turn(s, s[n].double(), s[n + "_norm"], s["pos"].double()) for n in ("q", "k")]
    lens, new = _lengths(case), _new(case)
    first = np.cumsum([0] + new)
    if case["kind"] == "attn":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
        for b in range(case["batch"]):
            p = torch.arange(lens[b] - new[b], lens[b], device=DEVICE)[:, None]
            t = torch.arange(lens[b], device=DEVICE)
            t = t[(t < case["sinks"]) | (t > lens[b] - new[b] - case["window"])]
            hidden = (t > p) | ((t <= p - case["window"]) & (t >= case["sinks"]))
            k, v = (_exact_values(s, x, b, t) for x in ("k", "v"))
            for h in range(case["n_q"]):
                j = h // (case["n_q"] // case["n_kv"])
                x = s["q"][first[b]:first[b + 1], h].double() @ k[:, j].T / math.sqrt(case["hd"])
                out[first[b]:first[b + 1], h] = torch.softmax(x.masked_fill(hidden, -math.inf), 1) @ v[:, j]
        return out
    q = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
    full = {n: torch.zeros(s["k_out"].shape, dtype=torch.float64, device=DEVICE) for n in "kv"}
    for b in range(case["batch"]):
        a, z, mine = lens[b] - new[b], lens[b], slice(first[b], first[b + 1])
        pos = torch.arange(a, z, device=DEVICE).double()
        q[mine] = _exact_turn(s, s["q"][mine].double(), s["q_norm"], pos)
        full["k"][b, :z] = _exact_append(s, "k", b, a, _exact_turn(s, s["k"][mine].double(), s["k_norm"], pos))
        full["v"][b, :z] = _exact_append(s, "v", b, a, s["v"][mine].double())
    return [q, full["k"], full["v"]]


def _exact_turn(s, x, weight, pos):
    """Pair by pair, as complex numbers."""
    rot, inter = s["case"]["rot"], s["case"]["inter"]
    x = x / torch.sqrt((x * x).sum(2, keepdim=True) / x.shape[2] + EPS) * weight.double()
    i = torch.arange(rot // 2, device=DEVICE)
    i, j = (2 * i, 2 * i + 1) if inter else (i, i + rot // 2)
    z = torch.complex(x[..., i], x[..., j]) * torch.polar(torch.full((), s["amplitude"], dtype=torch.float64,
                                                                     device=DEVICE), (pos[:, None] * s["freq"]))[:, None]
    x[..., i], x[..., j] = z.real, z.imag
    return x


def _exact_codes(s, name, b, t):
    """(bytes - 128, exponents) of sequence b's tokens t: [tokens, heads, dims], [tokens, heads]."""
    page = s["case"]["page"]
    p, r = s["table"][b].long()[t // page], t % page
    c = s["k_pages"][p, :, r] if name == "k" else s["v_pages"][p, :, r // BLOCK, :, r % BLOCK]
    return c.double() - 128, s[name + "_exp"][p, :, r // BLOCK].double()


def _exact_values(s, name, b, t):
    c, e = _exact_codes(s, name, b, t)
    return c * torch.exp2(e)[:, :, None]


def _exact_append(s, name, b, a, x):
    """Sequence b's values once rows x stand at positions a, a + 1, ..."""
    old = torch.arange(a, device=DEVICE)
    full = torch.cat([_exact_values(s, name, b, old), x])
    _, e = _exact_codes(s, name, b, old)
    c = full.clone()
    for lo in range(a // BLOCK * BLOCK, len(full), BLOCK):
        part = full[lo:lo + BLOCK]
        most = part[max(0, a - lo):].abs().amax((0, 2))          # of the new rows, each head
        step = torch.ceil(torch.log2((most / 127).clamp_min(2.0 ** E_MIN)))
        step = torch.where(most > 127 * torch.exp2(step), step + 1, step)
        step = torch.where(most <= 127 * torch.exp2(step - 1), step - 1, step).clamp_min(E_MIN)
        step = torch.maximum(step, e[lo]) if lo < a else step
        unit = torch.exp2(step)[None, :, None]
        c[lo:lo + BLOCK] = torch.round(part / unit) * unit
    return c
