"""Operators of a step of generation and of training beside the attention, for performance measurement and comparison.

A case is a dict of plain values; ``kind`` selects the operator:

  rotate   rotate_heads: norms of the queries and keys of each head, and the rotation by their positions; ``train`` with its gradients
  append   cache_append of new keys and values to a cache in 4 bits, then cache_read of them
  attend   cache_attention over a cache in 4 bits: the newest ``q`` tokens of every sequence against its cached keys and values (their own among them)

Rotation. Pair p of ``R`` / 2 (elements p and p + R / 2 of a row, or 2 p and 2 p + 1 where ``interleaved``) turns by position * base ** (-2 p / R); with
``sections`` the pairs are divided among that many axes, each with positions of its own. Elements from R on stay. ``norm``: a row is divided
by the root of its mean square (plus ``EPS``) and multiplied with a weight for each element, before it is turned.

The cache: pages of 64 tokens. ``k`` and ``v`` are uint8 (pages, kv_heads, 64, head_dim / 2), two e2m1 numbers in a byte, the even element in the low half;
``k_scale`` and ``v_scale`` uint8 (pages, kv_heads, 64, head_dim / 16): the scale of 16 numbers, whose byte is bits 14 .. 7 of a float16 (5 bits of
exponent, 3 of mantissa, no sign), up to 10240; 255 stands for 16 NaN. A number is stored as the e2m1 number nearest to it divided by the scale, the scale is the one nearest to
a sixth of the largest magnitude, ties go to even. ``desc`` (optional) holds one int32 for each token: bit 0 prefix, 1 context, 2 in a span, 3 [MASKQ], 4
same-span rule armed, 5..7 the classes of keys (prefix, context, span) that the token sees as a query wherever they are, 8.. the span id. ``table`` (batch,
blocks) names the pages of a sequence in order, ``lens`` its number of tokens.

``run`` computes the plain form, or calls the framework where ``own`` is true.
"""
import math

import numpy as np
import torch

own = False

PAGE, GROUP, TOP = 64, 16, 226   # tokens of a page, numbers of a scale, the byte of the largest scale
EPS = 1e-6
_DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _rotate(name, B, H, Hk, T, D, R, dtype, norm, train, base=10000.0, sections=(), interleaved=False, far=0, layout="bthd", offsets=False):
    return {"name": name, "kind": "rotate", "B": B, "H": H, "Hk": Hk, "T": T, "D": D, "R": R, "dtype": dtype, "norm": norm, "train": train, "base": base,
            "sections": ",".join(map(str, sections)), "interleaved": interleaved, "far": far, "layout": layout, "offsets": offsets}


def _sections(case):
    return tuple(int(n) for n in case["sections"].split(",") if n)


def _append(name, B, Hkv, D, T, n, dtype, layout="bthd"):
    return {"name": name, "kind": "append", "B": B, "Hkv": Hkv, "D": D, "T": T, "n": n, "dtype": dtype, "layout": layout}


def _attend(name, B, H, G, D, T, q, dtype, mask="causal"):
    return {"name": name, "kind": "attend", "B": B, "H": H, "G": G, "D": D, "T": T, "q": q, "dtype": dtype, "mask": mask}


def listed():
    return [
        # the newest token of every sequence of a serving batch, behind what the cache holds of it: latency is what it costs
        _rotate("rotate_step_b64", 64, 32, 8, 1, 128, 128, "bfloat16", True, False, base=1e6, far=8192, offsets=True),
        # a long prompt far into a document, fp16, no norm; only half of a head turns, neighbours with neighbours
        _rotate("rotate_prefill_t16384", 1, 32, 8, 16384, 128, 64, "float16", False, False, interleaved=True, far=1000000),
        # the headline's training step: all heads have norms, heads outermost in memory
        _rotate("rotate_train_t4096", 16, 16, 16, 4096, 64, 64, "bfloat16", True, True, layout="bhtd"),
        # training on video in float32: patches with time, height and width, an odd head dim, an odd number of tokens
        _rotate("rotate_train_video_fp32", 2, 12, 4, 2945, 80, 80, "float32", True, True, sections=(8, 16, 16)),
        # one token of every sequence joins the cache
        _append("append4_step_b64", 64, 8, 128, 2000, 1, "bfloat16"),
        # a batch of prompts joins it, lengths that end inside a block
        _append("append4_prompt_t4093", 8, 8, 128, 37, 4093, "bfloat16"),
        # a token of one request's short generation, a key head for each query head
        _attend("decode4_b1_t173", 1, 16, 1, 64, 173, 1, "bfloat16"),
        # a serving batch at an ordinary length
        _attend("decode4_b32_t4096", 32, 32, 4, 128, 4096, 1, "bfloat16"),
        # one request with a very long context, fp16: few rows, one long axis
        _attend("decode4_b1_t131071", 1, 32, 4, 128, 131071, 1, "float16"),
        # the largest batch of single tokens
        _attend("decode4_b128_t8192", 128, 16, 2, 128, 8192, 1, "bfloat16"),
        # verification of drafted tokens: a handful of queries for each sequence, of which some have fewer; an odd head dim
        _attend("verify4_q5_d80", 16, 12, 3, 80, 1357, 5, "float16", mask="hier"),
        # a chunk of a long prompt against all that is cached before it
        _attend("chunk4_q512_t8192", 2, 32, 4, 128, 8192, 512, "bfloat16", mask="hier"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    tops = [work(c) for c in listed()]
    most = {m: 0.8 * max(w[m] for w in tops) for m in ("bytes", "flops")}
    while True:
        kind = rng.choices(("rotate", "append", "attend"), (4, 2, 5))[0]
        D = rng.choice((64, 64, 128, 128, 128, 16, 32, 48, 80, 96, 112))
        Hkv = rng.choice((1, 2, 3, 4, 4, 5, 8, 8, 16))
        G = rng.choice((1, 1, 2, 3, 4, 4, 5, 8, 16))
        B = _log_uniform(rng, 1, 128)
        dtype = rng.choice(("bfloat16", "float16", "float32"))
        if kind == "rotate":
            T = 1 if rng.random() < 0.3 else _log_uniform(rng, 2, 32768)
            R = D if rng.random() < 0.7 else 16 * rng.randint(1, D // 16)
            sections = ()
            if rng.random() < 0.3:
                cuts = sorted(rng.randint(0, R // 2) for _ in range(rng.choice((1, 2))))
                sections = tuple(b - a for a, b in zip([0] + cuts, cuts + [R // 2]))
            c = _rotate("", B, Hkv * G, Hkv, T, D, R, dtype, rng.random() < 0.7, rng.random() < 0.5, rng.choice((1e4, 5e5, 1e6)), sections, rng.random() < 0.3,
                        rng.choice((0, 0, 4096, 1000000)), rng.choice(("bthd", "bhtd")), not sections and rng.random() < 0.3)
        elif kind == "append":
            n = 1 if rng.random() < 0.4 else _log_uniform(rng, 2, 8192)
            c = _append("", B, Hkv, D, rng.randint(0, 4000), n, dtype, rng.choice(("bthd", "bhtd")))
        else:
            q = 1 if rng.random() < 0.6 else _log_uniform(rng, 2, 512)
            T = max(q, _log_uniform(rng, 24, 131072))
            c = _attend("", B, Hkv * G, G, D, T, q, rng.choice(("bfloat16", "float16")), rng.choice(("causal", "hier")))
        del c["name"]
        w = work(c)
        scores = c["B"] * c["H"] * c["q"] * c["T"] * 4 if kind == "attend" else 0   # the plain form holds them all
        if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"] and scores <= 1.1e9:
            return c


# ---- inputs -----------------------------------------------------------------------------------------------------

def _channels(g, Hkv, D, spread, device):
    """Keys have channels that are much larger than others, the same ones for all tokens."""
    return torch.exp(spread * torch.randn((1, Hkv, 1, D), generator=g, device=device))


def _pool(g, case, pages):
    """A pool of pages as earlier appends have left them."""
    Hkv, D, dev = case["Hkv"], case["D"], g.device
    channels = _channels(g, Hkv, D, 0.5, dev)
    out = [torch.empty((pages, Hkv, PAGE, n), dtype=torch.uint8, device=dev) for n in (D // 2, D // 2, D // GROUP, D // GROUP)]
    step = max(1, (1 << 27) // (Hkv * PAGE * D))   # some pages at a time: the numbers in 32 bits take eight times the room
    for lo in range(0, pages, step):
        n = min(step, pages - lo)
        k, v = (torch.randn((n, Hkv, PAGE, D), generator=g, device=dev) for _ in range(2))
        v = v * torch.exp(0.3 * torch.randn((n, Hkv, 1, 1), generator=g, device=dev))
        for x, codes, scale in ((k * channels, out[0], out[2]), (v, out[1], out[3])):
            codes[lo:lo + n], scale[lo:lo + n] = _quantise(x)
    return out


def _table(g, B, blocks, pages):
    return torch.randperm(pages, generator=g, device=g.device)[: B * blocks].view(B, blocks).to(torch.int32)


def _blocks(tokens):
    return -(-tokens // PAGE)


def _lens(rng, B, lo, hi):
    """Ragged lengths, the longest of them `hi`."""
    n = rng.integers(max(lo, 0), hi + 1, size=B)
    n[rng.integers(0, B)] = hi
    return n.astype(np.int32)


def _descriptors(rng, T, lens):
    """Tokens of a sequence: a prefix, context, spans of tens of tokens, and at last the context that is being generated; the newest token of
    one sequence in eight is the [MASKQ]."""
    B = len(lens)
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


def _heads(g, B, H, T, D, dtype, layout, spread=0.0):
    """(B, H, T, D) as a projection leaves them: heads inside of the tokens, or outside."""
    x = torch.randn((B, T, H, D) if layout == "bthd" else (B, H, T, D), generator=g, device=g.device)
    if spread:
        x *= torch.exp(spread * torch.randn(D, generator=g, device=g.device))
    x = x.to(_DTYPES[dtype])
    return x.transpose(1, 2) if layout == "bthd" else x


def _positions(rng, case):
    """int64 (B, T), or (axes, B, T): tokens of a sequence in order from somewhere in a document; frames of patches, of which rows and columns start anew."""
    B, T, far, axes = case["B"], case["T"], case["far"], len(_sections(case))
    at = rng.integers(far // 2, far + 1, size=(B, 1)) + np.arange(T)[None, :]
    if axes == 0:
        return at
    width = 1 + math.isqrt(max(T // 5, 1))
    height = max(1, width - 2)
    i = np.broadcast_to(np.arange(T)[None, :], (B, T))
    frame = at[:, :1] + i // (width * height)
    return np.stack((frame, i // width % height, i % width)[:axes] if axes > 1 else (at,))


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    rng = np.random.default_rng(seed)
    c = dict(case)
    B, D, T = c["B"], c["D"], c["T"]
    cuda = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
    if c["kind"] == "rotate":
        s = {"q": _heads(g, B, c["H"], T, D, c["dtype"], c["layout"], 0.5), "k": _heads(g, B, c["Hk"], T, D, c["dtype"], c["layout"], 0.5),
             "q_weight": None, "k_weight": None, "positions": None, "offsets": None}
        if c["norm"]:
            for name in ("q_weight", "k_weight"):
                s[name] = (1.0 + 0.2 * torch.randn(D, generator=g, device=dev)).to(_DTYPES[c["dtype"]])
        if c["offsets"]:
            s["offsets"] = cuda(_lens(rng, B, c["far"] // 2, c["far"]))
        else:
            s["positions"] = cuda(_positions(rng, c))
        if c["train"]:
            s["grads"] = tuple(torch.randn(s[x].shape, generator=g, device=dev).to(s[x].dtype) for x in ("q", "k"))
            for name in ("q", "k", "q_weight", "k_weight"):
                if s[name] is not None:
                    s[name].requires_grad_(True)
    elif c["kind"] == "attend":
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
            d = cuda(_descriptors(rng, blocks * PAGE, lens)).view(B, blocks, 1, PAGE).expand(-1, -1, c["Hkv"], -1)
            s["desc"] = torch.zeros((pages, c["Hkv"], PAGE), dtype=torch.int32, device=dev)
            s["desc"][s["table"].long()] = d
    else:
        blocks = _blocks(T + c["n"]) + 1
        pages = B * blocks + 1   # the last page belongs to nobody
        k, v, ks, vs = _pool(g, c, pages)
        s = {"k": k, "v": v, "k_scale": ks, "v_scale": vs, "desc": None, "table": _table(g, B, blocks, pages - 1)}
        new = [_heads(g, B, c["Hkv"], c["n"], D, c["dtype"], c["layout"], spread) for spread in (0.5, 0.0)]
        lens = cuda(_lens(rng, B, T // 2, T))
        n_new = cuda(_lens(rng, B, -(-c["n"] // 2), c["n"]))
        s |= {"new_k": new[0], "new_v": new[1], "lens": lens, "n_new": n_new, "total": lens + n_new}
    s["case"] = c
    return s


# ---- the framework's calls --------------------------------------------------------------------------------------

def _handle(s):
    """The cache object that a program keeps."""
    if "handle" not in s:
        from kerneldev_b200 import KVCache
        s["handle"] = KVCache(s["k"], s["v"], s["k_scale"], s["v_scale"], s["desc"])
    return s["handle"]


def _rotation(s):
    """The table of frequencies that a program keeps."""
    if "rotation" not in s:
        from kerneldev_b200 import Rotation
        c = s["case"]
        s["rotation"] = Rotation(c["D"], rotary_dim=c["R"], base=c["base"], sections=_sections(c) or None, interleaved=c["interleaved"], device=s["q"].device)
    return s["rotation"]


def _own_rotate(s):
    from kerneldev_b200 import rotate_heads
    return rotate_heads(s["q"], s["k"], _rotation(s), s["positions"], offsets=s["offsets"], q_weight=s["q_weight"], k_weight=s["k_weight"], eps=EPS, out_layout="input")


def _own_append(s):
    from kerneldev_b200 import cache_append, cache_read
    cache_append(_handle(s), s["new_k"], s["new_v"], s["table"], s["lens"], s["n_new"])
    return cache_read(_handle(s), s["table"], s["total"], s["case"]["n"], start=s["lens"])


def _own_attend(s):
    from kerneldev_b200 import cache_attention
    return cache_attention(s["q"], _handle(s), s["table"], s["lens"], s["q_lens"], return_lse=True)


# ---- the plain forms --------------------------------------------------------------------------------------------

def _angles(s):
    """float64 (B, 1, T, R / 2): far positions lose their angles in 32 bits."""
    c, dev = s["case"], s["q"].device
    pairs = c["R"] // 2
    f = c["base"] ** (-2.0 * torch.arange(pairs, dtype=torch.float64, device=dev) / c["R"])
    if s["offsets"] is not None:
        at = (s["offsets"].long()[:, None] + torch.arange(c["T"], device=dev))[..., None]
    elif c["sections"]:
        at = torch.cat([s["positions"][a][..., None].expand(-1, -1, n) for a, n in enumerate(_sections(c))], 2)
    else:
        at = s["positions"][..., None]
    return (at.double() * f)[:, None]


def _turned(x, w, cos, sin, c):
    x32 = x.float()
    if w is not None:
        x32 = x32 * torch.rsqrt(x32.square().mean(-1, keepdim=True) + EPS) * w.float()
    R = c["R"]
    a, b = (x32[..., 0:R:2], x32[..., 1:R:2]) if c["interleaved"] else (x32[..., :R // 2], x32[..., R // 2:R])
    y = (a * cos - b * sin, b * cos + a * sin)
    y = torch.stack(y, -1).flatten(-2) if c["interleaved"] else torch.cat(y, -1)
    return torch.cat((y, x32[..., R:]), -1).to(x.dtype)


def _plain_rotate(s):
    c = s["case"]
    angle = _angles(s)
    cos, sin = angle.cos().float(), angle.sin().float()
    return _turned(s["q"], s["q_weight"], cos, sin, c), _turned(s["k"], s["k_weight"], cos, sin, c)


def _with_gradients(s, forward):
    out = forward(s)
    if not s["case"]["train"]:
        return out
    leaves = [s[x] for x in ("q", "k", "q_weight", "k_weight") if s[x] is not None]
    grads = torch.autograd.grad(out, leaves, s["grads"])
    return tuple(x.detach() for x in out) + grads


def _quantise(x):
    """Bytes of e2m1 numbers and of scales: x (..., D) float32."""
    g = x.unflatten(-1, (-1, GROUP))
    top = g.abs().amax(-1)
    bad = ~torch.isfinite(top)
    byte = _scale_byte(top / torch.full_like(top, 6.0))
    s = _scale_of(byte)[..., None]
    y = torch.where(s > 0, g.abs() / torch.where(s > 0, s, 1.0), 0.0)
    # the steps of e2m1: halves up to 2, ones up to 4, twos
    y = torch.where(y < 2.0, torch.round(y * 2.0) / 2.0, torch.where(y < 4.0, torch.round(y), torch.round(y / 2.0) * 2.0)).clamp(max=6.0)
    code = torch.where(y < 2.0, y * 2.0, torch.where(y < 4.0, y + 2.0, y / 2.0 + 4.0))   # 0 .. 7
    code = torch.where(bad[..., None], 0.0, code).to(torch.uint8) + (torch.signbit(g) & ~bad[..., None]).to(torch.uint8) * 8
    code = code.flatten(-2)
    return code[..., 0::2] + code[..., 1::2] * 16, torch.where(bad, 255, byte).to(torch.uint8)


def _scale_byte(x):
    """The nearest number with 3 bits of mantissa and exponents from -14, ties to even; its place among them is its byte."""
    e = (torch.frexp(torch.where(torch.isfinite(x), x, 1.0))[1].to(torch.int32) - 1).clamp(min=-14)
    n = torch.round(torch.ldexp(torch.where(torch.isfinite(x), x, 1.0), 3 - e)).to(torch.int32)   # eighths of 2**e: up to 16
    return torch.where(e > 13, TOP, ((e + 14) * 8 + n).clamp(max=TOP))


def _scale_of(byte):
    """float32 values of scale bytes."""
    return (byte.to(torch.int16) << 7).view(torch.float16).float()


def _numbers(codes, scale):
    """float32 (..., D) of bytes (..., D / 2) and scale bytes (..., D / 16)."""
    levels = torch.tensor(_E2M1 + tuple(-x for x in _E2M1), device=codes.device)
    x = torch.stack((levels[(codes & 15).int()], levels[(codes >> 4).int()]), -1).flatten(-2)
    return (x.unflatten(-1, (-1, GROUP)) * _scale_of(scale)[..., None]).flatten(-2)


def _values(codes, scale, table):
    """float32 values of the pages that `table` names, (B, Hkv, blocks, 64, D)."""
    t = table.long()
    return _numbers(codes[t], scale[t]).transpose(1, 2)


def _plain_append(s):
    n, dev = s["case"]["n"], s["k"].device
    i = torch.arange(n, device=dev)
    live = i < s["n_new"][:, None]
    at = s["lens"].long()[:, None] + i
    page = torch.where(live, torch.gather(s["table"].long(), 1, (at // PAGE).clamp(max=s["table"].shape[1] - 1)), s["k"].shape[0] - 1)
    slot = at % PAGE
    for new, codes, scale in ((s["new_k"], s["k"], s["k_scale"]), (s["new_v"], s["v"], s["v_scale"])):
        b, e = _quantise(new.transpose(1, 2).float())
        codes[page, :, slot], scale[page, :, slot] = b, e
    read = []
    for codes, scale in ((s["k"], s["k_scale"]), (s["v"], s["v_scale"])):
        x = _numbers(codes[page, :, slot], scale[page, :, slot]).transpose(1, 2)
        read.append(torch.where(live[:, None, :, None], x, 0.0).to(torch.bfloat16))
    return tuple(read)


def _visible(s, T):
    """(B, 1 or Hkv, q, T) truth values: which cached tokens each query sees."""
    c, lens = s["case"], s["lens"].long()
    Q, dev = c["q"], s["q"].device
    q_lens = s["q_lens"].long() if s["q_lens"] is not None else torch.full_like(lens, Q)
    i, j = torch.arange(Q, device=dev), torch.arange(T, device=dev)
    at = (lens - q_lens)[:, None] + i
    live = (i < q_lens[:, None])[:, None, :, None] & (j < lens[:, None])[:, None, None, :]
    causal = (at[:, :, None] >= j)[:, None]
    if s["desc"] is None:
        return live & causal
    d = s["desc"][s["table"].long()].transpose(1, 2).reshape(c["B"], c["Hkv"], -1)[..., :T]
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
    return o, ((m + l.log()) * math.log2(math.e)).view(B, H, Q)


def run(state):
    kind = state["case"]["kind"]
    if kind == "rotate":
        return _with_gradients(state, _own_rotate if own else _plain_rotate)
    if own:
        return {"attend": _own_attend, "append": _own_append}[kind](state)
    return {"attend": _plain_attend, "append": _plain_append}[kind](state)


# ---- what a pass cannot do without ------------------------------------------------------------------------------

def work(case):
    c = case
    D, size = c["D"], 4 if c["dtype"] == "float32" else 2
    if c["kind"] == "rotate":
        values = c["B"] * c["T"] * (c["H"] + c["Hk"]) * D
        position = c["B"] * (4 if c["offsets"] else 8 * c["T"] * max(1, len(_sections(c))))
        # forward: read and write; backward: the inputs once more, the gradients in and out
        return {"bytes": values * size * (5 if c["train"] else 2) + position * (2 if c["train"] else 1), "flops": values * (24 if c["train"] else 8)}
    row = D / 2 + D / GROUP   # of one operand
    if c["kind"] == "attend":
        # lengths lie evenly between half of T and T, counts of queries between half of q and q
        Hkv, tokens = c["H"] // c["G"], c["B"] * max(c["q"], 0.75 * c["T"])
        rows = c["B"] * c["H"] * (c["q"] if c["q"] == 1 else 0.75 * c["q"])
        return {"bytes": tokens * Hkv * (2 * row + (4 if c["mask"] == "hier" else 0)) + rows * D * 2 * size, "flops": 4 * rows * 0.75 * c["T"] * D}
    n = c["n"] if c["n"] == 1 else 0.75 * c["n"]
    rows, whole = c["B"] * c["Hkv"] * n * 2, c["B"] * c["Hkv"] * c["n"] * 2
    # tokens in, bytes out, bytes in, bfloat16 out
    return {"bytes": rows * (D * size + 2 * row) + whole * D * 2, "flops": 4 * rows * D}


# ---- the definition in 64 bits ----------------------------------------------------------------------------------

def _exact_rotate(s):
    c = s["case"]
    B, T, D, R = c["B"], c["T"], c["D"], c["R"]
    dev = s["q"].device
    first = [2 * p if c["interleaved"] else p for p in range(R // 2)]
    second = [2 * p + 1 if c["interleaved"] else p + R // 2 for p in range(R // 2)]
    axis = [a for a, n in enumerate(_sections(c)) for _ in range(n)] if c["sections"] else [0] * (R // 2)
    freq = torch.tensor([c["base"] ** (-2.0 * p / R) for p in range(R // 2)], dtype=torch.float64, device=dev)
    outs, grads, weights = [], [], []
    for which, name in enumerate(("q", "k")):
        x_all, w = s[name].detach(), s[name + "_weight"]
        out = torch.empty(x_all.shape, dtype=torch.float64, device=dev)
        dx, dw = torch.empty_like(out) if c["train"] else None, torch.zeros(D, dtype=torch.float64, device=dev)
        for b in range(B):
            if s["offsets"] is not None:
                at = (int(s["offsets"][b]) + torch.arange(T, device=dev))[:, None].expand(T, R // 2)
            elif c["sections"]:
                at = s["positions"][axis, b].T
            else:
                at = s["positions"][b][:, None].expand(T, R // 2)
            z = torch.polar(torch.ones((T, R // 2), dtype=torch.float64, device=dev), at.double() * freq)   # e^(i angle)
            x = x_all[b].double()
            root = torch.sqrt((x * x).sum(-1, keepdim=True) / D + EPS)
            gain = w.detach().double() if w is not None else torch.ones(D, dtype=torch.float64, device=dev)
            unit = x / root if w is not None else x
            y = unit * gain
            turned = torch.complex(y[..., first], y[..., second]) * z
            out[b] = y
            out[b][..., first], out[b][..., second] = turned.real, turned.imag
            if c["train"]:
                g = s["grads"][which][b].double()
                back = torch.complex(g[..., first], g[..., second]) * z.conj()
                g[..., first], g[..., second] = back.real, back.imag
                if w is None:
                    dx[b] = g
                else:
                    dw += (g * unit).sum((0, 1))
                    h = g * gain
                    dx[b] = (h - unit * (h * unit).sum(-1, keepdim=True) / D) / root
        outs.append(out)
        if c["train"]:
            grads.append(dx)
            if w is not None:
                weights.append(dw)
    return tuple(outs) + tuple(grads) + tuple(weights)


def _exact_levels(dev):
    return torch.tensor([(-1.0 if i & 8 else 1.0) * _E2M1[i & 7] for i in range(16)], dtype=torch.float64, device=dev)


def _exact_scales(dev):
    """Values of all scale bytes that are written: eighths of powers of two."""
    return torch.tensor([(b % 8 + 8) * 2.0 ** (b // 8 - 18) if b >= 8 else b * 2.0 ** -17 for b in range(TOP + 1)], dtype=torch.float64, device=dev)


def _nearest(x, grid):
    """Index of the nearest of an ascending grid, of two equally near ones the even index; x beyond the last has the last."""
    middle = (grid[1:] + grid[:-1]) / 2
    lower, upper = torch.searchsorted(middle, x), torch.searchsorted(middle, x, right=True)
    return torch.where((lower != upper) & (lower % 2 == 1), upper, lower)


def _exact_append(s):
    c = s["case"]
    n, dev = c["n"], s["k"].device
    scales, levels = _exact_scales(dev), torch.tensor(_E2M1, dtype=torch.float64, device=dev)
    outs = []
    for name in ("new_k", "new_v"):
        out = torch.zeros((c["B"], c["Hkv"], n, c["D"]), dtype=torch.float64, device=dev)
        for b in range(c["B"]):
            m = int(s["n_new"][b])
            x = s[name][b, :, :m].double().unflatten(-1, (-1, GROUP)).contiguous()
            size = scales[_nearest(x.abs().amax(-1, keepdim=True) / 6.0, scales)]
            v = levels[_nearest(x.abs() / size.clamp(min=2.0 ** -17), levels)] * torch.sign(x) * size
            out[b, :, :m] = v.flatten(-2)
        outs.append(out)
    return tuple(outs)


def _exact_sequence(codes, scale, pages):
    """All tokens of one sequence, (Hkv, tokens, D) float64."""
    c = codes[pages].transpose(0, 1).flatten(1, 2).int()
    levels = _exact_levels(codes.device)
    x = torch.stack((levels[c % 16], levels[c // 16]), -1).flatten(-2)
    size = _exact_scales(codes.device)[scale[pages].transpose(0, 1).flatten(1, 2).int()]
    return x * size.repeat_interleave(GROUP, -1)


def _exact_attend(s):
    c = s["case"]
    B, H, G, Q, D = c["B"], c["H"], c["G"], c["q"], c["D"]
    if B * c["T"] > 1_200_000:
        return None
    dev = s["k"].device
    lens = s["lens"].tolist()
    o = torch.zeros((B, H, Q, D), dtype=torch.float64, device=dev)
    lse = torch.full((B, H, Q), -math.inf, dtype=torch.float64, device=dev)
    for b in range(B):
        n, q = lens[b], int(s["q_lens"][b]) if s["q_lens"] is not None else Q
        pages = s["table"][b, :_blocks(n)].long()
        k, v = (_exact_sequence(p, e, pages)[:, :n] for p, e in ((s["k"], s["k_scale"]), (s["v"], s["v_scale"])))
        j = torch.arange(n, device=dev)
        at = j[n - q:, None]
        for h in range(c["Hkv"]):
            see = at >= j
            if s["desc"] is not None:
                d = s["desc"][pages, h].flatten()[:n].long() & 0xFFFFFFFF
                dq = d[n - q:, None]
                see = (((dq // 32) & d & 7) > 0) | (((dq & 2) > 0) & ((d & 2) > 0) & see) | (((dq & 16) > 0) & ((d & 4) > 0) & (dq // 256 == d // 256))
            for head in range(h * G, h * G + G):
                x = s["q"][b, head, :q].double() @ k[h].T / math.sqrt(D)
                x = torch.where(see, x, -math.inf)
                top = torch.logsumexp(x, 1, keepdim=True)
                o[b, head, :q] = torch.where(see, torch.exp(x - top), 0.0) @ v[h]
                lse[b, head, :q] = top[:, 0] / math.log(2.0)
    return o, lse


def exact(case, seed):
    s = prepare(case, seed)
    return {"rotate": _exact_rotate, "append": _exact_append, "attend": _exact_attend}[case["kind"]](s)
