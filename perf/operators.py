"""The operators of the 8-bit key/value cache, for performance measurement and comparison.

A case is a dict of plain values; ``kind`` selects the operator:

  attend   cache_attention: the newest ``q`` tokens of every sequence against its cached keys and values (their own among
           them); ``weights`` also adds up the attention weight that every cached token receives
  append   cache_append of new keys and values, then cache_read of the blocks that they went to
  evict    cache_evict by accumulated weight into fresh pages, then cache_read of what was kept

The cache: pages of 64 tokens. ``k`` and ``v`` are float8_e4m3fn (pages, kv_heads, 64, head_dim), ``k_scale`` and ``v_scale``
float32 (pages, kv_heads), powers of two: one scale for each block of 64 tokens and head. ``desc`` (optional) holds one int32 for each
token: bit 0 prefix, 1 context, 2 in a span, 3 [MASKQ], 4 same-span rule armed, 5..7 the classes of keys (prefix, context, span) that
the token sees as a query wherever they are, 8.. the span id. ``table`` (batch, blocks) names the pages of a sequence in order, ``lens``
its number of tokens.

``run`` computes the plain form, or calls the framework where ``own`` is true.
"""
import math

import numpy as np
import torch

own = False

PAGE = 64
_DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}


def _attend(name, B, H, G, D, T, q, dtype, mask="causal", weights=False):
    return {"name": name, "kind": "attend", "B": B, "H": H, "G": G, "D": D, "T": T, "q": q, "dtype": dtype, "mask": mask, "weights": weights}


def _append(name, B, Hkv, D, T, n, dtype, layout="bthd"):
    return {"name": name, "kind": "append", "B": B, "Hkv": Hkv, "D": D, "T": T, "n": n, "dtype": dtype, "layout": layout}


def _evict(name, B, Hkv, D, T, keep, recent, first):
    return {"name": name, "kind": "evict", "B": B, "Hkv": Hkv, "D": D, "T": T, "keep": keep, "recent": recent, "first": first}


def listed():
    return [
        # a token of one request's short generation, a key head for each query head: latency is what it costs
        _attend("decode_b1_t173", 1, 16, 1, 64, 173, 1, "bfloat16"),
        # a few requests with the hierarchical mask, head dim 64, heads in groups of 4
        _attend("decode_b8_t2048_hier", 8, 16, 4, 64, 2048, 1, "bfloat16", mask="hier"),
        # a serving batch at an ordinary length
        _attend("decode_b32_t4096", 32, 32, 4, 128, 4096, 1, "bfloat16"),
        # one request with a very long context, fp16: few rows, one long axis
        _attend("decode_b1_t131072", 1, 32, 4, 128, 131071, 1, "float16"),
        # the largest batch of single tokens
        _attend("decode_b128_t8192", 128, 16, 2, 128, 8192, 1, "bfloat16"),
        # verification of drafted tokens: a handful of queries for each sequence, of which some have fewer; an odd head dim
        _attend("verify_q5_d80", 16, 12, 3, 80, 1357, 5, "float16", mask="hier"),
        # a chunk of a long prompt against all that is cached before it
        _attend("chunk_q512_t8192", 2, 32, 4, 128, 8192, 512, "bfloat16", mask="hier"),
        # single tokens whose attention weights are added up for a later eviction
        _attend("weigh_b8_t4096", 8, 32, 4, 128, 4096, 1, "bfloat16", weights=True),
        # one token of every sequence joins the cache
        _append("append_step_b64", 64, 8, 128, 2000, 1, "bfloat16"),
        # a batch of prompts joins it, lengths that end inside a block
        _append("append_prompt_t4093", 8, 8, 128, 37, 4093, "bfloat16"),
        # a short cache gives up half of its tokens
        _evict("evict_b2_t1000", 2, 16, 64, 1000, 500, 128, 4),
        # long caches give up three quarters
        _evict("evict_b4_t32768", 4, 8, 128, 32768, 8192, 1024, 16),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    tops = [work(c) for c in listed()]
    most = {m: 0.8 * max(w[m] for w in tops) for m in ("bytes", "flops")}
    while True:
        kind = rng.choices(("attend", "append", "evict"), (6, 2, 2))[0]
        D = rng.choice((64, 64, 128, 128, 128, 16, 32, 48, 80, 96, 112))
        Hkv = rng.choice((1, 2, 3, 4, 4, 5, 8, 8, 16))
        B = _log_uniform(rng, 1, 128)
        if kind == "attend":
            G = rng.choice((1, 1, 2, 3, 4, 4, 5, 8, 16))
            q = 1 if rng.random() < 0.6 else _log_uniform(rng, 2, 512)
            T = max(q, _log_uniform(rng, 24, 131072))
            c = _attend("", B, Hkv * G, G, D, T, q, rng.choice(("bfloat16", "float16")), rng.choice(("causal", "hier")), rng.random() < 0.3)
        elif kind == "append":
            n = 1 if rng.random() < 0.4 else _log_uniform(rng, 2, 8192)
            c = _append("", B, Hkv, D, rng.randint(0, 4000), n, rng.choice(("bfloat16", "float16", "float32")), rng.choice(("bthd", "bhtd")))
        else:
            T = _log_uniform(rng, 24, 65536)
            keep = max(8, int(T * rng.uniform(0.1, 0.9)))
            c = _evict("", B, Hkv, D, T, keep, int(keep * rng.uniform(0.0, 0.5)), rng.choice((0, 0, 4, min(16, keep // 4))))
        del c["name"]
        w = work(c)
        scores = c["B"] * c["H"] * c["q"] * c["T"] * 4 if kind == "attend" else 0   # the plain form holds them all
        if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"] and scores <= 1.1e9:
            return c


# ---- inputs -----------------------------------------------------------------------------------------------------

def _quantise(x):
    """e4m3 values and power-of-two scales of blocks: x (..., tokens, D) float32."""
    e = _exponent(x.abs().amax((-2, -1)))
    s = _factor(e)
    return (x / s[..., None, None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn), s


def _factor(e):
    """2**e in float32, to the bit."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _exponent(amax):
    """The smallest e with amax <= 448 * 2**e, from -32 to 31: 448 = 0.875 * 2**9."""
    m, e = torch.frexp(amax)
    e = e.float() - 9 + (m > 0.875).float()
    return torch.where(amax > 0, e, torch.full_like(e, -32.0)).clamp(-32.0, 31.0)


def _channels(g, Hkv, D, spread, device):
    """Keys have channels that are much larger than others, the same ones for all tokens."""
    return torch.exp(spread * torch.randn((1, Hkv, 1, D), generator=g, device=device))


def _pool(g, case, pages):
    """A pool of pages as earlier appends have left them."""
    Hkv, D, dev = case["Hkv"], case["D"], g.device
    k, v = (torch.randn((pages, Hkv, PAGE, D), generator=g, device=dev) for _ in range(2))
    k = k.mul_(_channels(g, Hkv, D, 0.5, dev))
    v = v.mul_(torch.exp(0.3 * torch.randn((pages, Hkv, 1, 1), generator=g, device=dev)))
    k, ks = _quantise(k)
    v, vs = _quantise(v)
    return k, v, ks, vs


def _table(g, B, blocks, pages):
    return torch.randperm(pages, generator=g, device=g.device)[: B * blocks].view(B, blocks).to(torch.int32)


def _blocks(tokens):
    return -(-tokens // PAGE)


def _lens(rng, B, lo, hi):
    """Ragged lengths, the longest of them `hi`."""
    n = rng.integers(max(lo, 0), hi + 1, size=B)
    n[rng.integers(0, B)] = hi
    return n.astype(np.int32)


def _descriptors(rng, B, T, lens):
    """Tokens of a sequence: a prefix, context, spans of tens of tokens, and at last the context that is being generated; the newest token of
    one sequence in eight is the [MASKQ]."""
    pos = np.arange(T)[None, :]
    n = lens.astype(np.int64)[:, None]
    prefix, spans, after = n // 16, n // 2, n - np.maximum(n // 8, 1)
    is_prefix = pos < prefix
    in_span = (pos >= spans) & (pos < after)
    width = rng.integers(8, 97, size=(B, 1))
    sid = np.where(in_span, (pos - spans) // width + 1, 0)
    maskq = (pos == n - 1) & (rng.random((B, 1)) < 0.125)
    context = ~is_prefix & ~in_span & ~maskq
    d = is_prefix * 1 + context * 2 + in_span * 4 + maskq * 8 + in_span * 16
    sees = (is_prefix | context | maskq) * 1 + in_span * 2 + maskq * 4
    sid = np.where(maskq, -1, sid) & 0xFFFFFF
    return (d + (sees << 5) + (sid << 8)).astype(np.uint32).view(np.int32)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    rng = np.random.default_rng(seed)
    c = dict(case)
    B, D, T = c["B"], c["D"], c["T"]
    cuda = lambda a: torch.from_numpy(a).to(dev)  # noqa: E731
    if c["kind"] == "attend":
        c["Hkv"] = c["H"] // c["G"]
        blocks = _blocks(T)
        pages = B * blocks + 3
        k, v, ks, vs = _pool(g, c, pages)
        lens = _lens(rng, B, max(c["q"], T // 2), T)
        q_lens = _lens(rng, B, max(1, c["q"] // 2), c["q"])
        s = {"k": k, "v": v, "k_scale": ks, "v_scale": vs, "desc": None, "table": _table(g, B, blocks, pages)}
        # queries in the model's (batch, time, heads, dim) memory, large enough for weights that are far from even
        q = torch.randn((B, c["q"], c["H"], D), generator=g, device=dev) * 1.5
        s |= {"q": q.to(_DTYPES[c["dtype"]]).transpose(1, 2), "lens": cuda(lens), "q_lens": cuda(q_lens) if c["q"] > 1 else None}
        if c["mask"] == "hier":
            d = cuda(_descriptors(rng, B, blocks * PAGE, lens)).view(B, blocks, 1, PAGE).expand(-1, -1, c["Hkv"], -1)
            s["desc"] = torch.zeros((pages, c["Hkv"], PAGE), dtype=torch.int32, device=dev)
            s["desc"][s["table"].long()] = d
    elif c["kind"] == "append":
        blocks = _blocks(T + c["n"]) + 1
        pages = B * blocks + 1   # the last page belongs to nobody
        k, v, ks, vs = _pool(g, c, pages)
        s = {"k": k, "v": v, "k_scale": ks, "v_scale": vs, "desc": None, "table": _table(g, B, blocks, pages - 1)}
        new = torch.randn((2, B, c["n"], c["Hkv"], D), generator=g, device=dev)
        new[0] *= _channels(g, c["Hkv"], D, 0.5, dev).transpose(1, 2)
        if c["layout"] == "bhtd":
            new = new.transpose(2, 3).contiguous().transpose(2, 3)
        new = new.to(_DTYPES[c["dtype"]]).transpose(2, 3)
        lens = cuda(_lens(rng, B, T // 2, T))
        n_new = cuda(_lens(rng, B, -(-c["n"] // 2), c["n"]))
        s |= {"new_k": new[0], "new_v": new[1], "lens": lens, "n_new": n_new, "total": lens + n_new, "first": lens // PAGE * PAGE}
    else:
        blocks, out = _blocks(T), _blocks(c["keep"])
        pages = B * (blocks + out) + 1   # the last page belongs to nobody
        k, v, ks, vs = _pool(g, c, pages)
        table = _table(g, B, blocks + out, pages - 1)
        s = {"k": k, "v": v, "k_scale": ks, "v_scale": vs, "desc": None, "table": table[:, :blocks].contiguous(), "out": table[:, blocks:].contiguous()}
        # few tokens receive most of the weight; many have received none, and some equal amounts
        w = torch.exp(2.0 * torch.randn((B, c["Hkv"], T), generator=g, device=dev))
        w = torch.where(w < 0.2, torch.zeros_like(w), torch.where(w < 0.5, (w * 64).round() / 64, w))
        s |= {"weights": w, "lens": cuda(_lens(rng, B, T // 2, T))}
    s["case"] = c
    return s


# ---- the framework's calls --------------------------------------------------------------------------------------

def _handle(s):
    """The cache object that a program keeps."""
    if "handle" not in s:
        from kerneldev_b200 import KVCache
        s["handle"] = KVCache(s["k"], s["v"], s["k_scale"], s["v_scale"], s["desc"])
    return s["handle"]


def _own_attend(s):
    from kerneldev_b200 import cache_attention
    c = s["case"]
    if c["weights"]:
        w = torch.zeros((c["B"], c["Hkv"], c["T"]), device=s["q"].device)
        return cache_attention(s["q"], _handle(s), s["table"], s["lens"], s["q_lens"], weights=w), w
    return cache_attention(s["q"], _handle(s), s["table"], s["lens"], s["q_lens"], return_lse=True)


def _own_append(s):
    from kerneldev_b200 import cache_append, cache_read
    cache_append(_handle(s), s["new_k"], s["new_v"], s["table"], s["lens"], s["n_new"])
    return cache_read(_handle(s), s["table"], s["total"], s["case"]["n"] + PAGE - 1, start=s["first"])


def _own_evict(s):
    from kerneldev_b200 import cache_evict, cache_read
    c = s["case"]
    index, lens, weights = cache_evict(_handle(s), s["table"], s["lens"], s["weights"], s["out"], c["keep"], recent=c["recent"], first=c["first"])
    k, v = cache_read(_handle(s), s["out"], lens, c["keep"])
    return index, lens, weights, k, v


# ---- the plain forms --------------------------------------------------------------------------------------------

def _values(pool, scale, table):
    """float32 values of the pages that `table` names, (B, Hkv, blocks, 64, D)."""
    t = table.long()
    x = pool.view(torch.uint8)[t].view(torch.float8_e4m3fn).float() * scale[t][..., None, None]
    return x.transpose(1, 2)


def _visible(s, T):
    """(B, 1 or Hkv, q, T) truth values: which cached tokens each query sees."""
    c, lens = s["case"], s["lens"].long()
    B, Q, dev = c["B"], c["q"], s["q"].device
    q_lens = s["q_lens"].long() if s["q_lens"] is not None else torch.full_like(lens, Q)
    i, j = torch.arange(Q, device=dev), torch.arange(T, device=dev)
    at = (lens - q_lens)[:, None] + i
    live = (i < q_lens[:, None])[:, None, :, None] & (j < lens[:, None])[:, None, None, :]
    causal = (at[:, :, None] >= j)[:, None]
    if s["desc"] is None:
        return live & causal
    d = s["desc"][s["table"].long()].transpose(1, 2).reshape(B, c["Hkv"], -1)[..., :T]
    dq = torch.gather(d, 2, at.clamp(0, T - 1)[:, None].expand(-1, c["Hkv"], -1))[..., None]
    dk = d[:, :, None, :]
    sees = ((dq >> 5) & dk & 7) != 0
    both = (dq & dk & 2) != 0
    span = ((dq & 16) != 0) & ((dk & 4) != 0) & ((dq >> 8) == (dk >> 8))
    return live & (sees | (both & causal) | span)


def _plain_attend(s):
    c = s["case"]
    B, H, Hkv, G, Q, D, T = c["B"], c["H"], c["Hkv"], c["G"], c["q"], c["D"], c["T"]
    k = _values(s["k"], s["k_scale"], s["table"]).reshape(B, Hkv, -1, D)[:, :, :T]
    x = (s["q"].reshape(B, Hkv, G * Q, D).float() @ k.transpose(2, 3)) * (D ** -0.5)
    del k
    see = _visible(s, T)[:, :, None]
    x = x.view(B, Hkv, G, Q, T).masked_fill_(~see, -math.inf)
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    x = x.sub_(m).exp_()
    l = x.sum(-1, keepdim=True)
    x = x.div_(torch.where(l > 0, l, torch.ones_like(l)))
    v = _values(s["v"], s["v_scale"], s["table"]).reshape(B, Hkv, -1, D)[:, :, :T]
    o = (x.view(B, Hkv, G * Q, T) @ v).view(B, H, Q, D).to(s["q"].dtype)
    if c["weights"]:
        return o, x.sum((2, 3))
    return o, ((m + l.log()) * math.log2(math.e)).view(B, H, Q)


def _store(s, table, values, keep):
    """Writes blocks of values (B, Hkv, blocks, 64, D) with scales into the pages of `table` where `keep` (B, blocks) says so."""
    t = torch.where(keep, table.long(), s["k"].shape[0] - 1)
    for_k, for_v = values
    for_k, for_v = (_rounded(x, e) for x, e in (for_k, for_v))
    s["k"].view(torch.uint8)[t], s["k_scale"][t] = for_k[0].transpose(1, 2).contiguous().view(torch.uint8), for_k[1].transpose(1, 2)
    s["v"].view(torch.uint8)[t], s["v_scale"][t] = for_v[0].transpose(1, 2).contiguous().view(torch.uint8), for_v[1].transpose(1, 2)


def _power(scale):
    """The exponents of powers of two, which a logarithm may miss by a hair."""
    return torch.frexp(scale)[1].float() - 1


def _rounded(x, e):
    s = _factor(e)
    return (x / s[..., None, None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn), s


def _read(s, table, lens, start, count):
    """bfloat16 (B, Hkv, count, D): the cached tokens start .. start + count - 1, zeros at and beyond lens."""
    at = start.long()[:, None] + torch.arange(count, device=table.device)
    inside = (at < lens[:, None])[:, None, :, None]
    at = at.clamp(max=table.shape[1] * PAGE - 1)[:, None, :, None]
    k, v = (_values(p, e, table).flatten(2, 3) for p, e in ((s["k"], s["k_scale"]), (s["v"], s["v_scale"])))
    at = at.expand(-1, k.shape[1], -1, k.shape[3])
    return (torch.where(inside, torch.gather(k, 2, at), 0.0).to(torch.bfloat16), torch.where(inside, torch.gather(v, 2, at), 0.0).to(torch.bfloat16))


def _plain_append(s):
    c = s["case"]
    B, Hkv, D, n = c["B"], c["Hkv"], c["D"], c["n"]
    dev = s["k"].device
    lens, n_new, total = s["lens"].long(), s["n_new"].long(), s["total"].long()
    W = _blocks(n) + 1
    block = (lens // PAGE)[:, None] + torch.arange(W, device=dev)
    touched = block * PAGE < total[:, None]
    block = block.clamp(max=s["table"].shape[1] - 1)
    table = torch.gather(s["table"], 1, block)
    at = (lens // PAGE * PAGE)[:, None] + torch.arange(W * PAGE, device=dev)
    there, fresh = (at < lens[:, None])[:, None, :, None], ((at >= lens[:, None]) & (at < total[:, None]))[:, None, :, None]
    source = (at - lens[:, None]).clamp(0, n - 1)[:, None, :, None].expand(-1, Hkv, -1, D)
    held = there.view(B, 1, W, PAGE).any(-1)
    out = _merged(s["k"], s["k_scale"], s["new_k"], table, source, there, fresh, held), _merged(s["v"], s["v_scale"], s["new_v"], table, source, there, fresh, held)
    _store(s, table, out, touched)
    return _read(s, s["table"], s["total"], s["first"], n + PAGE - 1)


def _merged(pool, scale, new, table, source, there, fresh, held):
    """The blocks with their new tokens, and the exponents of their scales: no smaller than that of what a block holds already."""
    old = _values(pool, scale, table)
    B, Hkv, W, _, D = old.shape
    new = torch.where(fresh, torch.gather(new.float(), 2, source), 0.0).view(B, Hkv, W, PAGE, D)
    e = _exponent(new.abs().amax((-2, -1)))
    e = torch.where(held, torch.maximum(e, _power(scale[table.long()]).transpose(1, 2)), e)
    return torch.where(there.view(B, 1, W, PAGE, 1), old, new), e


def _plain_evict(s):
    c = s["case"]
    B, Hkv, D, T, keep = c["B"], c["Hkv"], c["D"], c["T"], c["keep"]
    dev = s["k"].device
    lens = s["lens"].long()[:, None, None]
    j = torch.arange(T, device=dev)
    w = torch.where((j < c["first"]) | (j >= lens - c["recent"]), math.inf, s["weights"])
    w = torch.where(j < lens, w, -math.inf)
    index = torch.sort(w, dim=2, descending=True, stable=True)[1][:, :, :keep]
    index = torch.sort(torch.where(index < lens, index, T), dim=2)[0]
    kept = index < lens
    new_lens = s["lens"].clamp(max=keep)
    at = index.clamp(max=T - 1)
    weights = torch.where(kept, torch.gather(s["weights"], 2, at), 0.0)
    blocks = _blocks(keep)
    pad = blocks * PAGE - keep
    at = torch.nn.functional.pad(at, (0, pad))[..., None].expand(-1, -1, -1, D)
    inside = torch.nn.functional.pad(kept, (0, pad))[..., None]
    k, v = (torch.where(inside, torch.gather(_values(p, e, s["table"]).flatten(2, 3), 2, at), 0.0).view(B, Hkv, blocks, PAGE, D)
            for p, e in ((s["k"], s["k_scale"]), (s["v"], s["v_scale"])))
    out = (k, _exponent(k.abs().amax((-2, -1)))), (v, _exponent(v.abs().amax((-2, -1))))
    _store(s, s["out"], out, torch.arange(blocks, device=dev) * PAGE < new_lens[:, None])
    index = torch.where(kept, index, -1).to(torch.int32)
    return (index, new_lens, weights) + _read(s, s["out"], new_lens, torch.zeros_like(new_lens), keep)


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"attend": _own_attend, "append": _own_append, "evict": _own_evict}[kind](state)
    return {"attend": _plain_attend, "append": _plain_append, "evict": _plain_evict}[kind](state)


# ---- what a pass cannot do without ------------------------------------------------------------------------------

def work(case):
    c = case
    if c["kind"] == "attend":
        # lengths lie evenly between half of T and T, counts of queries between half of q and q
        Hkv, tokens = c["H"] // c["G"], c["B"] * max(c["q"], 0.75 * c["T"])
        rows = c["B"] * c["H"] * (c["q"] if c["q"] == 1 else 0.75 * c["q"])
        size = 2
        return {"bytes": tokens * Hkv * (2 * c["D"] + (4 if c["mask"] == "hier" else 0) + (4 if c["weights"] else 0)) + rows * c["D"] * 2 * size,
                "flops": 4 * rows * 0.75 * c["T"] * c["D"]}
    if c["kind"] == "append":
        size = {"float32": 4}.get(c["dtype"], 2)
        n = c["n"] if c["n"] == 1 else 0.75 * c["n"]
        values = c["B"] * c["Hkv"] * n * c["D"] * 2
        whole = c["B"] * c["Hkv"] * (c["n"] + PAGE - 1) * c["D"] * 2
        return {"bytes": values * (size + 1) + values * 1 + whole * 2, "flops": 4 * values}
    n, kept = 0.75 * c["T"], min(c["keep"], 0.75 * c["T"])
    values = c["B"] * c["Hkv"] * kept * c["D"] * 2
    return {"bytes": c["B"] * c["Hkv"] * (4 * n + 8 * c["keep"]) + values * 3 + c["B"] * c["Hkv"] * c["keep"] * c["D"] * 2 * 2, "flops": 4 * values}


# ---- the definition in 64 bits ----------------------------------------------------------------------------------

def _grid(x, e):
    """x rounded to the numbers that e4m3 has, times 2**e: four significant bits, none below 2**-9, ties to even."""
    y = x * torch.exp2(-e)
    step = torch.exp2((torch.frexp(y)[1].double() - 4).clamp(min=-9.0))
    return torch.clamp(torch.round(y / step) * step, -448.0, 448.0) * torch.exp2(e)


def _scale_of(amax):
    x = torch.ceil(torch.log2(torch.where(amax > 0, amax, 1e-30) / 448.0))
    x = torch.where(448.0 * torch.exp2(x - 1) >= amax, x - 1, x)   # log2 of an exact power may come out a hair above
    x = torch.where(448.0 * torch.exp2(x) < amax, x + 1, x)
    return x.clamp(-32.0, 31.0)


def _whole(pool, scale, pages):
    """All tokens of one sequence, (Hkv, tokens, D)."""
    x = torch.stack([pool[p].double() * scale[p].double()[:, None, None] for p in pages])
    return x.permute(1, 0, 2, 3).flatten(1, 2)


def exact(case, seed):
    s = prepare(case, seed)
    c, table, lens = s["case"], s["table"].tolist(), s["lens"].tolist()
    B, D, dev = c["B"], c["D"], s["k"].device
    Hkv = c["Hkv"]

    def attend():
        H, G, Q, T = c["H"], c["G"], c["q"], c["T"]
        if B * T > 1_200_000:
            return None
        o = torch.zeros((B, H, Q, D), dtype=torch.float64, device=dev)
        lse = torch.full((B, H, Q), -math.inf, dtype=torch.float64, device=dev)
        weights = torch.zeros((B, Hkv, T), dtype=torch.float64, device=dev)
        for b in range(B):
            n, q = lens[b], int(s["q_lens"][b]) if s["q_lens"] is not None else Q
            pages = table[b][:_blocks(n)]
            k, v = (_whole(p, e, pages)[:, :n] for p, e in ((s["k"], s["k_scale"]), (s["v"], s["v_scale"])))
            j = torch.arange(n, device=dev)
            at = j[n - q:, None]
            for h in range(Hkv):
                see = at >= j
                if s["desc"] is not None:
                    d = torch.cat([s["desc"][p, h] for p in pages])[:n].long() & 0xFFFFFFFF
                    dq = d[n - q:, None]
                    see = (((dq // 32) & d & 7) > 0) | (((dq & 2) > 0) & ((d & 2) > 0) & see) | (((dq & 16) > 0) & ((d & 4) > 0) & (dq // 256 == d // 256))
                for head in range(h * G, h * G + G):
                    x = s["q"][b, head, :q].double() @ k[h].T / math.sqrt(D)
                    x = torch.where(see, x, -math.inf)
                    top = torch.logsumexp(x, 1, keepdim=True)
                    p = torch.where(see, torch.exp(x - top), 0.0)
                    o[b, head, :q] = p @ v[h]
                    lse[b, head, :q] = top[:, 0] / math.log(2.0)
                    weights[b, h, :n] += p.sum(0)
        return (o, weights) if c["weights"] else (o, lse)

    def append():
        count = c["n"] + PAGE - 1
        if B * (count // PAGE + 1) > 4000:
            return None
        outs = torch.zeros((2, B, Hkv, count, D), dtype=torch.float64, device=s["k"].device)
        for b in range(B):
            n, start = int(s["n_new"][b]), lens[b] // PAGE * PAGE
            for which, (pool, scale, new) in enumerate(((s["k"], s["k_scale"], s["new_k"]), (s["v"], s["v_scale"], s["new_v"]))):
                for block in range(start // PAGE, _blocks(lens[b] + n)):
                    lo, page = block * PAGE, table[b][block]
                    old = max(0, lens[b] - lo)
                    x = new[b, :, max(lo - lens[b], 0):max(min(lo + PAGE - lens[b], n), 0)].double()
                    e = _scale_of(x.abs().amax((1, 2)))
                    if old:
                        e = torch.maximum(e, torch.frexp(scale[page].double())[1] - 1)
                    held = pool[page][:, :old].double() * scale[page].double()[:, None, None]
                    at = lo - start
                    outs[which, b, :, at:at + old + x.shape[1]] = _grid(torch.cat((held, x), 1), e[:, None, None])
        return outs[0], outs[1]

    def evict():
        keep = c["keep"]
        if B * Hkv * _blocks(keep) > 20000:
            return None
        index = torch.full((B, Hkv, keep), -1, dtype=torch.int32, device=dev)
        weights = torch.zeros((B, Hkv, keep), dtype=torch.float64, device=dev)
        outs = torch.zeros((2, B, Hkv, keep, D), dtype=torch.float64, device=dev)
        for b in range(B):
            n = lens[b]
            m = min(n, keep)
            held = [_whole(p, e, table[b][:_blocks(n)])[:, :n] for p, e in ((s["k"], s["k_scale"]), (s["v"], s["v_scale"]))]
            for h in range(Hkv):
                w = s["weights"][b, h, :n].double()
                free = np.arange(n)
                free = free[(free >= c["first"]) & (free < n - c["recent"])]
                forced = np.setdiff1d(np.arange(n), free)
                order = free[np.argsort(-w.cpu().numpy()[free], kind="stable")]
                chosen = np.sort(np.concatenate((forced, order[:m - len(forced)]))) if n > keep else np.arange(n)
                at = torch.from_numpy(chosen).to(dev)
                index[b, h, :m] = at.to(torch.int32)
                weights[b, h, :m] = w[at]
                for which in range(2):
                    x = torch.nn.functional.pad(held[which][h, at], (0, 0, 0, _blocks(m) * PAGE - m)).view(-1, PAGE, D)
                    e = _scale_of(x.abs().amax((1, 2)))
                    outs[which, b, h, :m] = _grid(x, e[:, None, None]).flatten(0, 1)[:m]
        return index, s["lens"].clamp(max=keep), weights, outs[0], outs[1]

    return {"attend": attend, "append": append, "evict": evict}[c["kind"]]()
