"""The operators around a paged int8 K/V cache, each in its plain form and as the package's own call.

Three kinds of call, told apart by a case's "op":
  rotary     q and k [B,H,N,D] (or packed [tokens, heads, D]) rotated by their positions; "inverse" is the gradient
  append     the new tokens' keys (rotated on the way) and values quantised into a paged int8 cache with one scale for each
             "block" of tokens and head; "H" > 0: the tokens' queries are rotated and quantised in the same call
  attention  packed int8 query rows against such a cache: one row a sequence (decode), a few, a chunk, whole prompts
"new" and "len" are the longest of a batch of "S" sequences: new tokens (query rows), and tokens in the cache with them.  The
others' lengths follow from the case alone.  Caches are [pages, heads, page, D], their scales [pages, heads, page // block].
"""
import importlib
import math
import random

import torch

own = False          # True: the package's calls; False: the plain form


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def _rotary(B, H, Hkv, N, D, *, rot=None, dtype="fp16", interleaved=False, inverse=False, far=0, packed=False):
    return {"op": "rotary", "B": B, "H": H, "Hkv": Hkv, "N": N, "D": D, "rot": rot or D, "dtype": dtype, "interleaved": interleaved,
            "inverse": inverse, "far": far, "packed": packed}


def _append(S, H, Hkv, new, length, D, *, page=64, block=1, rot=None, dtype="fp16", interleaved=False):
    return {"op": "append", "S": S, "H": H, "Hkv": Hkv, "new": new, "len": length, "D": D, "page": page, "block": block,
            "rot": rot or D, "dtype": dtype, "interleaved": interleaved}


def _attention(S, H, Hkv, new, length, D, *, page=64, block=1, causal=True, out="fp16"):
    return {"op": "attention", "S": S, "H": H, "Hkv": Hkv, "new": new, "len": length, "D": D, "page": page, "block": block,
            "causal": causal, "out": out}


def listed():
    cases = {
        # one decode step's q and k of a small batch, packed: a launch and little else
        "rotary_step": _rotary(1, 32, 8, 16, 128, packed=True, far=4000),
        # q and k of the headline attention workload's heads, a long prompt
        "rotary_prompt": _rotary(2, 32, 8, 8192, 128, dtype="bf16", interleaved=True),
        # the gradient of a partly rotated head at an odd length, in fp32
        "rotary_gradient": _rotary(3, 16, 16, 3001, 64, rot=32, dtype="fp32", inverse=True),
        # decode: one token of each sequence, q with it, positions anywhere in a long context
        "append_step": _append(64, 32, 8, 1, 8192, 128),
        # the prompts of a ragged batch, all of their tokens
        "append_prompt": _append(12, 32, 8, 2048, 2048, 128, dtype="bf16"),
        # chunks that begin and end inside a block of 16 tokens with one scale, no q, half of the head rotated
        "append_blocks": _append(40, 0, 8, 200, 5000, 64, page=16, block=16, rot=32, interleaved=True),
        # decode of one short sequence: latency
        "decode_short": _attention(1, 32, 8, 1, 513, 128, page=16),
        # decode of a ragged batch, the ordinary case
        "decode_batch": _attention(64, 32, 8, 1, 8192, 128),
        # one long context, one scale for 16 tokens
        "decode_long": _attention(1, 32, 8, 1, 131072, 128, page=16, block=16),
        # a few rows a sequence (a draft to be verified), bf16 output, head dim 64
        "verify": _attention(32, 32, 8, 4, 4097, 64, page=32, out="bf16"),
        # chunked prefill: up to 512 new rows against longer caches
        "chunk": _attention(4, 32, 8, 512, 8192, 128),
        # prompts of a ragged batch, nothing in the cache before them
        "prompt": _attention(6, 32, 8, 4096, 4096, 128, out="bf16"),
    }
    return [dict(c, name=n) for n, c in cases.items()]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread evenly over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("rotary", "append", "append", "decode", "decode", "few", "chunk"))
    hkv, ratio = rng.choice((1, 2, 4, 8, 8, 16)), rng.choice((1, 2, 4, 4, 7, 8))
    D = rng.choice((64, 128, 128, 128, 256))
    page = rng.choice((8, 16, 32, 64, 64, 128, 256))
    block = rng.choice((1, 1, 1, 4, 16, page))
    block = min(block, page)
    inter = rng.random() < 0.4
    if kind == "rotary":
        D = rng.choice((16, 32, 64, 128, 128, 256))
        c = _rotary(_log(rng, 1, 8), hkv * ratio, hkv, _log(rng, 1, 16384), D, rot=rng.choice((D, D, D // 2, 16)),
                    dtype=rng.choice(("fp16", "bf16", "fp32")), interleaved=inter, inverse=rng.random() < 0.4,
                    far=rng.choice((0, 0, 10000)), packed=rng.random() < 0.4)
        if c["packed"]:
            c["B"] = 1
    elif kind == "append":
        new = rng.choice((1, 1, _log(rng, 2, 4096)))
        c = _append(_log(rng, 1, 64 if new > 1 else 256), rng.choice((0, hkv * ratio)), hkv, new, new + _log(rng, 1, 16384), D, page=page, block=block,
                    rot=rng.choice((D, D, D // 2)), dtype=rng.choice(("fp16", "bf16")), interleaved=inter)
    elif kind == "decode":
        c = _attention(_log(rng, 1, 128), hkv * ratio, hkv, 1, _log(rng, 16, 131072), D, page=page, block=block, out=rng.choice(("fp16", "bf16")))
    elif kind == "few":
        new = _log(rng, 2, 16)
        c = _attention(_log(rng, 1, 64), hkv * ratio, hkv, new, new + _log(rng, 16, 32768), D, page=page, block=block,
                       causal=rng.random() < 0.8, out=rng.choice(("fp16", "bf16")))
    else:
        new = _log(rng, 17, 4096)
        c = _attention(_log(rng, 1, 8), hkv * ratio, hkv, new, new + rng.choice((0, _log(rng, 1, 16384))), D, page=page, block=block,
                       causal=rng.random() < 0.8, out=rng.choice(("fp16", "bf16")))
    tops = [_cost(x) for x in listed() if x["op"] == c["op"]]
    while any(x > max(t[i] for t in tops) for i, x in enumerate(_cost(c))):
        if c.get("S", c.get("B", 1)) > 1:
            key = "S" if "S" in c else "B"
            c[key] = (c[key] + 1) // 2
        elif c["op"] == "rotary":
            c["N"] = max(1, c["N"] * 2 // 3)
        elif c["new"] > 1 and c["new"] * 2 >= c["len"]:
            c["new"], c["len"] = c["new"] * 2 // 3, max(c["len"] * 2 // 3, c["new"] * 2 // 3)
        elif c["op"] == "attention":
            c["len"] = max(c["new"], c["len"] * 2 // 3)
        else:
            c["new"] = max(1, c["new"] * 2 // 3)
    return c


def _lengths(case):
    """(new tokens, tokens in the cache with them) of each sequence: the first has the most of both."""
    r = random.Random("%(S)d %(new)d %(len)d" % case)
    new = [case["new"]] + [r.randint(max(1, case["new"] // 4), case["new"]) for _ in range(case["S"] - 1)]
    old = case["len"] - case["new"]
    return new, [n + (old if i == 0 else r.randint(old // 4, old)) for i, n in enumerate(new)]


def work(case):
    D = case["D"]
    if case["op"] == "rotary":
        size = 4 if case["dtype"] == "fp32" else 2
        rows = case["B"] * case["N"] * (case["H"] + case["Hkv"])
        return {"bytes": 2 * rows * D * size + case["N"] * case["rot"] * 4, "flops": 3 * rows * case["rot"]}
    new, length = _lengths(case)
    if case["op"] == "append":
        T, H, Hkv = sum(new), case["H"], case["Hkv"]
        scales = T * H + 2 * sum((b - 1) // case["block"] - (b - n) // case["block"] + 1 for n, b in zip(new, length)) * Hkv
        return {"bytes": T * (3 * (2 * Hkv + H) * D + case["rot"] * 4) + 4 * scales, "flops": T * ((Hkv + H) * case["rot"] * 3 + (2 * Hkv + H) * D * 3)}
    pairs = sum(n * b - (n * (n - 1) // 2 if case["causal"] else 0) for n, b in zip(new, length))
    cache = 2 * case["Hkv"] * sum(b * D + 4 * -(-b // case["block"]) for b in length)
    return {"bytes": cache + sum(new) * case["H"] * (D * 3 + 4), "flops": 4 * pairs * case["H"] * D}


def _cost(c):
    """What the limits of draw() apply to: bytes, operations, and what the plain form holds at once (the padded scores)."""
    w = work(c)
    return w["bytes"], w["flops"], c["S"] * c["H"] * c["new"] * c["len"] if c["op"] == "attention" else 0


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
_TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _table(n, rot, dev):
    """(cos, sin) of every position and pair, from angles in 64 bits."""
    freq = 10000.0 ** (-torch.arange(0, rot, 2, device=dev, dtype=torch.float64) / rot)
    angle = torch.arange(n, device=dev, dtype=torch.float64)[:, None] * freq
    return torch.stack([angle.cos(), angle.sin()], -1).float().contiguous()


def _pages(case, length, g, dev, first=None):
    """(block table, number of pages): pages in no order.  `first`: only pages from those positions on are real, page 0 stands for the
    rest (an append does not look at them)."""
    page = case["page"]
    width = max(-(-b // page) for b in length)
    counts = torch.tensor([-(-b // page) for b in length], device=dev)
    skip = torch.tensor([0 if first is None else first[i] // page for i in range(len(length))], device=dev)
    col = torch.arange(width, device=dev)[None]
    real = (col < counts[:, None]) & (col >= skip[:, None])
    used = int(real.sum())
    pages = used + used // 4 + 8
    table = torch.zeros(len(length), width, dtype=torch.int32, device=dev)
    table[real] = (1 + torch.randperm(pages - 1, generator=g, device=dev)[:used]).int()
    return table, pages


def _quantised(shape, block, g, dev):
    """A cache of normal values quantised with one scale for each block of tokens."""
    P, H, page, D = shape
    x8 = torch.empty(shape, dtype=torch.int8, device=dev)
    scale = torch.empty(P, H, page // block, device=dev)
    wide = torch.where(torch.arange(D, device=dev) % 37 == 5, 4.0, 1.0)          # channels that stand out, as keys have them
    step = max(1, (1 << 27) // (H * page * D))
    for i in range(0, P, step):
        n = min(step, P - i)
        x = (torch.randn(n, H, page, D, generator=g, device=dev) * wide).view(n, H, page // block, block * D)
        s = x.abs().amax(-1) / 127
        x8[i:i + n] = (x / s[..., None]).round().to(torch.int8).view(n, H, page, D)
        scale[i:i + n] = s
    return x8, scale


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(seed)
    D, st = case["D"], {"case": case}
    if case["op"] == "rotary":
        B, N, t = case["B"], case["N"], _TYPES[case["dtype"]]
        shape = (lambda h: (N, h, D)) if case["packed"] else (lambda h: (B, h, N, D))
        q, k = (torch.randn(shape(h), generator=g, device=dev).to(t) for h in (case["H"], case["Hkv"]))
        positions = torch.arange(case["far"], case["far"] + N, device=dev, dtype=torch.int32)
        if case["packed"]:               # tokens of several sequences
            positions = positions[torch.randperm(N, generator=g, device=dev)]
        return dict(st, q=q, k=k, positions=positions, table=_table(case["far"] + N, case["rot"], dev))
    new, length = _lengths(case)
    T = sum(new)
    one = case["new"] == 1               # one token a sequence: no cu_seqlens
    ends = torch.tensor([0] + new, device=dev).cumsum(0).to(torch.int32)
    st.update(cu=None if one else ends, lens=torch.tensor(length, dtype=torch.int32, device=dev))
    first = [b - n for n, b in zip(new, length)]
    if case["op"] == "append":
        t = _TYPES[case["dtype"]]
        st["table"], pages = _pages(case, length, g, dev, first)
        for x in ("k", "v"):
            st[x] = torch.randn(T, case["Hkv"], D, generator=g, device=dev).to(t)
            st[x + "c"], st[x + "s"] = _quantised((pages, case["Hkv"], case["page"], D), case["block"], g, dev)
        st["q"] = torch.randn(T, case["H"], D, generator=g, device=dev).to(t) if case["H"] else None
        st["rot"] = _table(case["len"], case["rot"], dev)
        return st
    st["table"], pages = _pages(case, length, g, dev)
    for x in ("k", "v"):
        st[x + "c"], st[x + "s"] = _quantised((pages, case["Hkv"], case["page"], D), case["block"], g, dev)
    q = torch.randn(T, case["H"], D, generator=g, device=dev)
    st["qs"] = q.abs().amax(-1) / 127
    st["q"] = (q / st["qs"][..., None]).round().to(torch.int8)
    st["most"] = case["new"]
    return st


# ---------------------------------------------------------------------------------------------------------------------
# the plain form
# ---------------------------------------------------------------------------------------------------------------------
def _rotated(x, cs, interleaved, inverse=False):
    """x [..., D] in fp32, rotated by cs [..., rot/2, 2]: each product rounded by itself."""
    half = cs.shape[-2]
    c, s = cs[..., 0], -cs[..., 1] if inverse else cs[..., 1]
    y = x.clone()
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        y[..., 0:2 * half:2], y[..., 1:2 * half:2] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        y[..., :half], y[..., half:2 * half] = a * c - b * s, b * c + a * s
    return y


def _plain_rotary(st):
    case = st["case"]
    cs = st["table"][st["positions"].long()]
    cs = cs[:, None] if case["packed"] else cs[None, None]
    return [_rotated(x.float(), cs, case["interleaved"], case["inverse"]).to(x.dtype) for x in (st["q"], st["k"])]


def _places(st):
    """Of every new token: its sequence, position, page and slot."""
    case, lens = st["case"], st["lens"].long()
    T, dev = st["k"].shape[0], lens.device
    cu = torch.arange(case["S"] + 1, device=dev) if st["cu"] is None else st["cu"].long()
    t = torch.arange(T, device=dev)
    seq = torch.searchsorted(cu, t, right=True) - 1
    first = lens - (cu[1:] - cu[:-1])
    pos = first[seq] + t - cu[seq]
    return seq, first, pos, st["table"][seq, pos // case["page"]].long(), pos % case["page"]


def _rounded(x, s):
    return torch.where(s > 0, (x / s).round(), 0.0).to(torch.int8)


def _plain_append(st):
    case = st["case"]
    block, page_size = case["block"], case["page"]
    seq, first, pos, page, slot = _places(st)
    cs = st["rot"][pos][:, None]
    n127 = torch.full((), 127.0, device=pos.device)
    # tokens before the first new one, in its block
    back = torch.arange(1, block, device=pos.device)
    old = first[:, None] - back[None]
    s_old, i_old = torch.nonzero((old >= 0) & (old // block == first[:, None] // block), as_tuple=True)
    old = old[s_old, i_old]
    old_page, old_slot = st["table"][s_old, old // page_size].long(), old % page_size
    for x, cache, scale in ((_rotated(st["k"].float(), cs, case["interleaved"]), st["kc"], st["ks"]), (st["v"].float(), st["vc"], st["vs"])):
        s = x.abs().amax(-1) / n127
        if block > 1:
            before = scale[old_page, :, old_slot // block]
            began = (pos // block * block < first[seq])[:, None]
            scale[page, :, slot // block] = torch.where(began, scale[page, :, slot // block], 0.0)
            flat = (page[:, None] * case["Hkv"] + torch.arange(case["Hkv"], device=pos.device)) * (page_size // block) + (slot // block)[:, None]
            scale.view(-1).scatter_reduce_(0, flat.view(-1), s.view(-1), "amax")
            s = scale[page, :, slot // block]
            after = scale[old_page, :, old_slot // block]
            ratio = torch.where(after > 0, before / after, 0.0)[..., None]
            cache[old_page, :, old_slot] = (cache[old_page, :, old_slot].float() * ratio).round().to(torch.int8)
        else:
            scale[page, :, slot] = s
        cache[page, :, slot] = _rounded(x, s[..., None])
    # (codes are whole numbers that both sides come to by the same operations; they are compared as such, with their scales)
    outs = [st["kc"], st["ks"], st["vc"], st["vs"]]
    if st["q"] is not None:
        q = _rotated(st["q"].float(), cs, case["interleaved"])
        s = q.abs().amax(-1) / n127
        outs += [_rounded(q, s[..., None]), s]
    return outs


def _gathered(st, x, dtype):
    """A cache as [S, heads, keys, D] in `dtype`, every sequence as long as the longest."""
    case = st["case"]
    t = st["table"].long()
    codes = st[x + "c"][t].to(dtype)                                   # [S, pages, heads, page, D]
    scale = st[x + "s"][t].to(dtype).repeat_interleave(case["block"], -1)
    return (codes * scale[..., None]).transpose(1, 2).flatten(2, 3)


def _plain_attention(st):
    case = st["case"]
    H, Hkv, D, n, S = case["H"], case["Hkv"], case["D"], st["most"], case["S"]
    lens = st["lens"].long()
    dev, T = lens.device, st["q"].shape[0]
    cu = torch.arange(S + 1, device=dev) if st["cu"] is None else st["cu"].long()
    rows = cu[1:] - cu[:-1]
    i = torch.arange(n, device=dev)
    at = (cu[:-1, None] + i).clamp(max=T - 1)                          # [S, n]: rows past a sequence's own are not taken back
    q = (st["q"].float() * st["qs"][..., None])[at]                    # [S, n, H, D]
    q = q.view(S, n, Hkv, H // Hkv, D).permute(0, 2, 3, 1, 4).flatten(2, 3)
    k, v = _gathered(st, "k", torch.float32), _gathered(st, "v", torch.float32)
    x = torch.matmul(q, k.transpose(-1, -2)) * (D ** -0.5)
    last = (lens - rows)[:, None] + i if case["causal"] else (lens - 1)[:, None].expand(S, n)
    last = torch.minimum(last, lens[:, None] - 1)
    seen = torch.arange(k.shape[2], device=dev) <= last[..., None]     # [S, n, keys]
    x.view(S, Hkv, H // Hkv, n, -1).masked_fill_(~seen[:, None, None], -math.inf)
    p = torch.exp_(x.sub_(x.amax(-1, keepdim=True)))
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    o = o.view(S, H, n, D).transpose(1, 2)
    seq = torch.searchsorted(cu, torch.arange(T, device=dev), right=True) - 1
    return o[seq, torch.arange(T, device=dev) - cu[seq]].to(_TYPES[case["out"]])


def run(state):
    case = state["case"]
    if case["op"] == "rotary":
        if own:
            intfa = importlib.import_module("int-flashattention_b200")
            return list(intfa.rotary(state["q"], state["k"], state["table"], state["positions"], interleaved=case["interleaved"], inverse=case["inverse"]))
        return _plain_rotary(state)
    if case["op"] == "append":
        if own:
            intfa = importlib.import_module("int-flashattention_b200")
            q = intfa.append_int8_paged(state["k"], state["v"], state["kc"], state["vc"], state["ks"], state["vs"], state["table"], state["lens"],
                                        state["cu"], q=state["q"], table=state["rot"], interleaved=case["interleaved"])
            return [state["kc"], state["ks"], state["vc"], state["vs"], *(q or ())]
        return _plain_append(state)
    if own:
        intfa = importlib.import_module("int-flashattention_b200")
        return intfa.attention_int8_paged(state["q"], state["kc"], state["vc"], state["qs"], state["ks"], state["vs"], state["table"], state["lens"],
                                          state["cu"], case["causal"], case["D"] ** -0.5, out_dtype=_TYPES[case["out"]])
    return _plain_attention(state)


# ---------------------------------------------------------------------------------------------------------------------
# from the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def _turned(x, cs, interleaved, inverse=False):
    """As a product of complex numbers: pair j times cos + i sin."""
    half = cs.shape[-2]
    z = torch.complex(*((x[..., 0:2 * half:2], x[..., 1:2 * half:2]) if interleaved else (x[..., :half], x[..., half:2 * half])))
    w = torch.view_as_complex(cs.contiguous())
    z = z * (w.conj() if inverse else w)
    pair = torch.view_as_real(z).flatten(-2) if interleaved else torch.cat([z.real, z.imag], -1)
    return torch.cat([pair, x[..., 2 * half:]], -1)


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "rotary":
        cs = st["table"].double()[st["positions"].long()]
        cs = cs[:, None] if case["packed"] else cs[None, None]
        return [_turned(x.double(), cs.expand(*x.shape[:-1], -1, -1), case["interleaved"], case["inverse"]) for x in (st["q"], st["k"])]
    new, length = _lengths(case)
    if case["op"] == "append":
        cs, block, size = st["rot"].double(), case["block"], case["page"]
        ks, vs = st["ks"].double(), st["vs"].double()
        qs, at = [], 0
        for s, (n, b) in enumerate(zip(new, length)):
            pos = torch.arange(b - n, b, device=ks.device)
            turn = cs[pos][:, None]
            page, blk = st["table"][s, pos // size].long(), pos % size // block
            for x, scale in ((_turned(st["k"][at:at + n].double(), turn.expand(-1, case["Hkv"], -1, -1), case["interleaved"]), ks), (st["v"][at:at + n].double(), vs)):
                most = x.abs().amax(-1) / 127                          # [n, heads]
                run_of = pos // block - pos[0] // block                # the blocks that the chunk touches, in turn
                top = torch.zeros(int(run_of[-1]) + 1, case["Hkv"], dtype=torch.float64, device=ks.device)
                if (b - n) % block:
                    top[0] = scale[page[0], :, blk[0]]
                top = top.scatter_reduce(0, run_of[:, None].expand(-1, case["Hkv"]), most, "amax")
                scale[page, :, blk] = top[run_of]
            if st["q"] is not None:
                qs.append(_turned(st["q"][at:at + n].double(), turn.expand(-1, case["H"], -1, -1), case["interleaved"]).abs().amax(-1) / 127)
            at += n
        return [None, ks, None, vs] + ([None, torch.cat(qs)] if qs else [])
    out, at, ratio = [], 0, case["H"] // case["Hkv"]
    for s, (n, b) in enumerate(zip(new, length)):
        pages = st["table"][s, :-(-b // case["page"])].long()
        o = torch.empty(n, case["H"], case["D"], dtype=torch.float64, device=pages.device)
        for h in range(case["Hkv"]):
            k, v = ((st[x + "c"][pages, h].double() * st[x + "s"][pages, h].double().repeat_interleave(case["block"], -1)[..., None]).flatten(0, 1)[:b] for x in "kv")
            for r in range(h * ratio, (h + 1) * ratio):
                x = st["q"][at:at + n, r].double() * st["qs"][at:at + n, r].double()[:, None] @ k.T * case["D"] ** -0.5
                if case["causal"] and n > 1:
                    x += torch.full_like(x, -math.inf).triu(b - n + 1)
                o[:, r] = torch.softmax(x, -1) @ v
        out.append(o)
        at += n
    return torch.cat(out)
