"""The operators of a serving step over a paged, packed KV cache, as cases that can be timed.

A step of a serving program gives its new queries and keys their rotary positions (`rotary`), appends the new keys and
values to the pages of their sequences (`append`; read back here as the values that the pages then hold) and lets the new
queries attend to everything that the pages hold (`attend`: single tokens, a few tokens to verify, chunks of a prompt, whole
prompts, and queries over another sequence's states).

A page holds a 128-token block of every KV head: [pages, KV heads, block bytes], as the packed caches of this package lay a
block out.  Codes are those of normally distributed rotated values, which is what the rotation makes of any rows.
"""
from __future__ import annotations

import functools
import math

import torch

own = False

D, BLOCK = 128, 128
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
FORMATS = (("turbo3", "turbo3"), ("turbo4", "turbo4"), ("turbo2", "turbo2"), ("turbo4", "turbo3"), ("turbo4", "turbo2"),
           ("q8_0", "turbo3"), ("q8_0", "turbo2"), ("q8_0", "turbo4"), ("q8_0", "q8_0"), ("turbo3", "q8_0"))
HEADS = ((32, 8), (64, 8), (32, 4), (40, 8), (16, 16), (8, 1))     # query heads, KV heads
# codebooks for coordinates of unit vectors in 128 dims
CENTROIDS = {
    2: (-0.133462, -0.039994, 0.039994, 0.133462),
    3: (-0.190685, -0.117832, -0.065717, -0.021460, 0.021460, 0.065717, 0.117832, 0.190685),
    4: (-0.1739, -0.1172, -0.0895, -0.0688, -0.0513, -0.0356, -0.0210, -0.0069,
        0.0069, 0.0210, 0.0356, 0.0513, 0.0688, 0.0895, 0.1172, 0.1739),
}


def listed():
    return [
        # one step of 64 users: launch and host latency are all of it
        dict(name="rotary_step_64", path="rotary", tokens=64, hq=32, hkv=8, d=128, rot=128, layout="half", scaling="none",
             far=32768, inverse=False, dtype="fp16"),
        # a 32K prompt, the benchmark's heads
        dict(name="rotary_prompt_32k", path="rotary", tokens=32768, hq=32, hkv=8, d=128, rot=128, layout="half", scaling="none",
             far=32768, inverse=False, dtype="fp16"),
        # an odd number of tokens far out in a long context, half of each head rotated, neighbouring pairs
        dict(name="rotary_part_far_yarn", path="rotary", tokens=5003, hq=40, hkv=8, d=128, rot=64, layout="interleaved",
             scaling="yarn", far=1000000, inverse=False, dtype="bf16"),
        # one step of 64 users at as many places in their pages
        dict(name="append_step_64", path="append", k="turbo3", v="turbo3", batch=64, hkv=8, new=1, ragged=False, pos=8000, dtype="fp16"),
        # chunks of different lengths that begin inside a page, 8-bit K rows
        dict(name="append_chunk_ragged", path="append", k="q8_0", v="turbo2", batch=5, hkv=8, new=777, ragged=True, pos=1500, dtype="bf16"),
        # a 16K prompt into empty pages
        dict(name="append_prompt_16k", path="append", k="turbo4", v="turbo4", batch=1, hkv=8, new=16384, ragged=False, pos=0, dtype="fp16"),
        # one user's decode step at a short context: latency
        dict(name="attend_step_one_4k", path="attend", k="turbo3", v="turbo3", batch=1, hq=32, hkv=8, new=1, context=4000, ragged=False,
             causal=True, dtype="fp16"),
        # a batch of users whose contexts differ widely
        dict(name="attend_step_ragged_32k", path="attend", k="turbo4", v="turbo4", batch=32, hq=32, hkv=8, new=1, context=32768, ragged=True,
             causal=True, dtype="fp16"),
        # a few drafted tokens of every user to verify, eight query heads to a KV head
        dict(name="attend_verify_5", path="attend", k="turbo3", v="turbo3", batch=16, hq=64, hkv=8, new=5, context=8000, ragged=True,
             causal=True, dtype="bf16"),
        # the last chunk of a 32K prompt
        dict(name="attend_chunk_2048_at_32k", path="attend", k="turbo3", v="turbo3", batch=1, hq=32, hkv=8, new=2048, context=32768,
             ragged=False, causal=True, dtype="fp16"),
        # whole prompts of different odd lengths, 8-bit K rows
        dict(name="attend_prompts_ragged", path="attend", k="q8_0", v="turbo3", batch=6, hq=40, hkv=8, new=2501, context=2501, ragged=True,
             causal=True, dtype="bf16"),
        # decoder prompts over the packed states of an encoder
        dict(name="attend_cross_1500", path="attend", k="turbo4", v="turbo4", batch=4, hq=16, hkv=16, new=448, context=1500, ragged=False,
             causal=False, dtype="fp16"),
    ]


def _log(rng, lo, hi):
    """An integer from lo to hi, spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    path = rng.choice(("rotary", "append", "attend", "attend"))
    hq, hkv = rng.choice(HEADS)
    if path == "rotary":
        d = rng.choice((64, 128, 128, 256))
        return dict(path=path, tokens=_log(rng, 1, 32768 * 40 * 128 // ((hq + hkv) * d)), hq=hq, hkv=hkv, d=d,
                    rot=rng.choice((d, d, d // 2, d // 4)), layout=rng.choice(("half", "interleaved")),
                    scaling=rng.choice(("none", "linear", "ntk", "yarn")), far=rng.choice((4096, 131072, 1000000)),
                    inverse=rng.random() < 0.3, dtype=rng.choice(("fp16", "bf16")))
    k, v = rng.choice(FORMATS)
    if path == "append":
        batch = _log(rng, 1, 64)
        return dict(path=path, k=k, v=v, batch=batch, hkv=hkv, new=_log(rng, 1, 16384 * 8 // (hkv * batch)), ragged=rng.random() < 0.5,
                    pos=rng.choice((0, 1, 1)) * _log(rng, 1, 8000), dtype=rng.choice(("fp16", "bf16", "fp32")))
    batch, causal = _log(rng, 1, 32), rng.random() < 0.8
    new = rng.choice((1, _log(rng, 2, 16), _log(rng, 16, 2048)))
    # no more products and no more padded places than the largest listed cases have
    most = min(131072, 2048 * 32768 * 32 // (batch * new * hq), 32 * 32768 * 8 // (batch * hkv))
    context = _log(rng, min(64, most), most)
    if causal:
        new = min(new, context)
    return dict(path=path, k=k, v=v, batch=batch, hq=hq, hkv=hkv, new=new, context=context, ragged=rng.random() < 0.5, causal=causal,
                dtype=rng.choice(("fp16", "bf16")))


# ---- what a program keeps -------------------------------------------------------------------------------------------

def _bits(fmt):
    return 8 if fmt == "q8_0" else int(fmt[-1])


def _block_bytes(fmt):
    return BLOCK * 136 if fmt == "q8_0" else BLOCK * (16 * _bits(fmt) + 2)


@functools.lru_cache(maxsize=None)
def _signs(side):
    """The two sign diagonals of K's or V's rotation."""
    gen = torch.Generator().manual_seed(1000 + side)
    return [torch.randint(0, 2, (D,), generator=gen).double().mul_(2).sub_(1) for _ in range(2)]


@functools.lru_cache(maxsize=None)
def _bit_places(bits, kind):
    """[bits, 128 tokens * 128 dims] on the GPU: the byte of a block and the shift in it at which each bit of a code lies."""
    token, dim = torch.meshgrid(torch.arange(BLOCK), torch.arange(D), indexing="ij")
    if kind == "k":
        row, pair, half = token, dim >> 1, dim & 1
    else:   # rows are dims, two to a row, of 64 tokens
        row, pair, half = (token & 64) | (dim & 63), (token & 60) | ((dim >> 6) << 1) | ((token >> 1) & 1), token & 1
    group, p = pair >> 4, pair & 15
    at = (half * bits)[None] + torch.arange(bits)[:, None, None]          # bit of the pair's code
    if bits == 3:
        tail = 6 * (p - 12) + at
        dword = torch.where(p >= 12, tail >> 3, p >> 2)
        bit = torch.where(p >= 12, 24 + (tail & 7), 6 * (p & 3) + at)
    else:
        per = 32 // (2 * bits)
        dword = (p // per).expand(bits, -1, -1)
        bit = 2 * bits * (p % per) + at
    byte = dword * 2048 + row * 16 + group * 4 + (bit >> 3)
    return byte.reshape(bits, -1).cuda(), (bit & 7).reshape(bits, -1).to(torch.uint8).cuda()


@functools.lru_cache(maxsize=None)
def _byte_sources(bits, kind):
    """The inverse: for each bit of a block's code bytes the code (token * 128 + dim) and the bit of it that lie there."""
    byte, shift = _bit_places(bits, kind)
    code = torch.zeros(BLOCK * 16 * bits * 8, dtype=torch.int64, device="cuda")
    bit = torch.zeros(BLOCK * 16 * bits * 8, dtype=torch.uint8, device="cuda")
    place = (byte * 8 + shift).reshape(-1)
    code[place] = torch.arange(BLOCK * D, device="cuda").repeat(bits)
    bit[place] = torch.arange(bits, device="cuda", dtype=torch.uint8).repeat_interleave(BLOCK * D)
    return code, bit


@functools.lru_cache(maxsize=None)
def _q8_places(kind):
    """Bytes of a block at which the 8-bit values lie [128 * 128], and those of their scales' fp16 words (in words)."""
    token, dim = torch.meshgrid(torch.arange(BLOCK), torch.arange(D), indexing="ij")
    if kind == "k":
        byte = (dim >> 4) * 2048 + token * 16 + (dim & 15)
        scale = token * 4 + (dim >> 5)
    else:   # rows are dims of 64 tokens; a row's first 64 bytes are the lower dims' tokens
        row, col = (token & 64) | (dim & 63), (dim >> 6) * 64 + (token & 63)
        byte = (col >> 4) * 2048 + row * 16 + (col & 15)
        scale = ((token >> 6) * 4 + (dim >> 5)) * 64 + (token & 63)
    return byte.reshape(-1).cuda(), scale.reshape(-1).cuda()


def _pages(gen, fmt, kind, n, heads, spread):
    """n pages of random rows: uint8 [n, heads, block bytes]."""
    out = torch.empty((n * heads, _block_bytes(fmt)), dtype=torch.uint8, device="cuda")
    for lo in range(0, n * heads, 4096):
        m = min(4096, n * heads - lo)
        size = torch.exp(spread * torch.randn((m, BLOCK, 1), generator=gen, device="cuda"))
        x = torch.randn((m, BLOCK, D), generator=gen, device="cuda")
        if fmt == "q8_0":
            x *= size
            scale = (x.view(m, BLOCK, 4, 32).abs().amax(-1) / 127).half()
            q = torch.round(x.view(m, BLOCK, 4, 32) / scale.float()[..., None]).clamp_(-127, 127).to(torch.int8).view(m, -1)
            byte, word = _q8_places(kind)
            out[lo:lo + m, byte] = q.view(torch.uint8)
            halves = out[lo:lo + m, BLOCK * D:].contiguous().view(torch.float16)
            halves[:, word] = scale.repeat_interleave(32, dim=-1).view(m, -1)
            out[lo:lo + m, BLOCK * D:] = halves.view(torch.uint8)
            continue
        bits = _bits(fmt)
        c = torch.tensor(CENTROIDS[bits], device="cuda")
        code = torch.bucketize(x / math.sqrt(D), (c[1:] + c[:-1]) / 2).to(torch.uint8).view(m, -1)
        src, bit = _byte_sources(bits, kind)
        weight = torch.arange(8, device="cuda", dtype=torch.uint8)
        out[lo:lo + m, :BLOCK * 16 * bits] = (((code[:, src] >> bit) & 1).view(m, -1, 8) << weight).sum(-1, dtype=torch.uint8)
        out[lo:lo + m, BLOCK * 16 * bits:] = (math.sqrt(D) * size).half().view(m, BLOCK).view(torch.uint8)
    return out.view(n, heads, -1)


def _lengths(case, top, gen=None):
    """A length of every sequence: `top`, or, ragged, from an eighth of it to all of it, even over the logarithm (the first:
    all) and, given a generator, in another order each time."""
    b = case["batch"]
    if not case["ragged"]:
        return torch.full((b,), top)
    f = torch.exp(-torch.remainder(torch.arange(b) * 0.6180339887498949, 1.0) * math.log(8.0))
    return (f * top).long().clamp_(min=1)[torch.randperm(b, generator=gen) if gen is not None else slice(None)]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    rows = lambda *shape: torch.randn(shape, generator=gen, device="cuda").to(dtype)  # noqa: E731
    s = dict(case)
    if case["path"] == "rotary":
        s["q"], s["k"] = rows(case["tokens"], case["hq"], case["d"]), rows(case["tokens"], case["hkv"], case["d"])
        first = int(torch.randint(0, max(1, case["far"] - case["tokens"]) + 1, (1,), generator=host))
        s["positions"] = (torch.arange(case["tokens"]) + first).cuda()
        if case["tokens"] <= 512:       # a step: every row at a place of its own
            s["positions"] = torch.randint(0, case["far"], (case["tokens"],), generator=host).cuda()
        return s
    hkv = case["hkv"]
    new = _lengths(case, case["new"]) if case["path"] == "append" or case["new"] > 16 else torch.full((case["batch"],), case["new"])
    if case["path"] == "append":
        start = (torch.rand((case["batch"],), generator=host) * (case["pos"] + 1)).long()
        total = start + new
    elif case["causal"]:
        total = torch.maximum(_lengths(case, case["context"], host), new) if case["new"] < case["context"] else new
    else:
        total = _lengths(case, case["context"], host)
    blocks = (total + BLOCK - 1) // BLOCK
    widest, used = int(blocks.max()), int(blocks.sum())
    free = torch.randperm(used + 3, generator=host)[:used]      # a few pages of the pool belong to nobody
    table = torch.zeros((case["batch"], widest), dtype=torch.int32)
    table[torch.arange(widest)[None] < blocks[:, None]] = free.to(torch.int32)
    s["table"], s["max_context"] = table.cuda(), widest * BLOCK
    s["cu"] = torch.cat([torch.zeros(1, dtype=torch.long), new.cumsum(0)]).to(torch.int32).cuda()
    s["rows"], s["longest"] = int(new.sum()), int(new.max())
    if case["path"] == "append":
        s["start"] = start.to(torch.int32).cuda()
        s["key"], s["value"] = rows(s["rows"], hkv, D), rows(s["rows"], hkv, D)
        channels = torch.argsort(torch.rand((hkv, D), generator=gen, device="cuda"), dim=-1)[:, :4]
        s["key"] *= torch.ones((hkv, D), device="cuda").scatter_(1, channels, 15.0).to(dtype)
        s["k_pages"] = torch.zeros((used + 3, hkv, _block_bytes(case["k"])), dtype=torch.uint8, device="cuda")
        s["v_pages"] = torch.zeros((used + 3, hkv, _block_bytes(case["v"])), dtype=torch.uint8, device="cuda")
        return s
    s["lens"] = total.to(torch.int32).cuda()
    s["q"] = rows(s["rows"], case["hq"], D)
    s["k_pages"] = _pages(gen, case["k"], "k", used + 3, hkv, 0.3)
    s["v_pages"] = _pages(gen, case["v"], "v", used + 3, hkv, 0.3)
    return s


# ---- the plain forms: elementary torch operations in 32 bits ----------------------------------------------------------

def _frequencies(case):
    """Angle per position of each rotated pair (64 bits), and what the rotated values are multiplied by."""
    r, base, factor, trained = case["rot"], 10000.0, 8.0, 4096
    i = torch.arange(r // 2, dtype=torch.float64, device="cuda")
    if case["scaling"] == "ntk":
        base = base * factor ** (r / (r - 2))
    f = base ** (-2 * i / r)
    if case["scaling"] == "linear":
        f = f / factor
    if case["scaling"] != "yarn":
        return f, 1.0
    pair_of = lambda turns: r * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
    lo, hi = max(math.floor(pair_of(32.0)), 0), min(math.ceil(pair_of(1.0)), r - 1)
    ramp = ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
    return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1.0


def _rotate_plain(x, cos, sin, case):
    r = case["rot"]
    y = x.float()
    if case["layout"] == "half":
        u, w = y[..., :r // 2], y[..., r // 2:r]
        turned = torch.cat([u * cos - w * sin, w * cos + u * sin], -1)
    else:
        u, w = y[..., 0:r:2], y[..., 1:r:2]
        turned = torch.stack([u * cos - w * sin, w * cos + u * sin], -1).flatten(-2)
    return torch.cat([turned, y[..., r:]], -1).to(x.dtype)


def _hadamard(dtype):
    i = torch.arange(D, device="cuda")
    b = i[:, None] & i[None]
    b = b ^ (b >> 4)
    b = b ^ (b >> 2)
    b = (b ^ (b >> 1)) & 1
    return (1 - 2 * b).to(dtype) / math.sqrt(D)


def _rotation(side, dtype):
    """R with y = R x: sign diagonals around the Hadamard matrix."""
    s1, s2 = (t.to(device="cuda", dtype=dtype) for t in _signs(side))
    return s2[:, None] * _hadamard(dtype) * s1[None]


def _values(pages, fmt, kind):
    """[n, heads, block bytes] -> [n, heads, 128, 128] in 32 bits, turbo rows in the rotated domain."""
    n, heads, _ = pages.shape
    flat = pages.reshape(n * heads, -1)
    if fmt == "q8_0":
        byte, word = _q8_places(kind)
        q = flat[:, byte].view(torch.int8).float()
        return (q * flat[:, BLOCK * D:].contiguous().view(torch.float16)[:, word].float()).view(n, heads, BLOCK, D)
    bits = _bits(fmt)
    byte, shift = _bit_places(bits, kind)
    weight = torch.arange(bits, device="cuda", dtype=torch.uint8)[:, None]
    code = (((flat[:, byte.reshape(-1)].view(-1, bits, BLOCK * D) >> shift) & 1) << weight).sum(1, dtype=torch.uint8)
    c = torch.tensor(CENTROIDS[bits], device="cuda")
    norm = flat[:, BLOCK * 16 * bits:].contiguous().view(torch.float16).float()
    return c[code.int()].view(n, heads, BLOCK, D) * norm.view(n, heads, BLOCK, 1)


def _stored_plain(x, fmt, side):
    """What a cache holds of rows [.., 128], as fp16 values.  Codes are decided in 64 bits: a value next to a border."""
    y = x.double()
    if fmt == "q8_0":
        g = y.float().view(*y.shape[:-1], 4, 32)
        scale = g.abs().amax(-1, keepdim=True) / 127
        inverse = torch.where(scale > 0, 1 / scale, 0)
        t = g * inverse
        q = torch.trunc(t + torch.copysign(torch.full_like(t, 0.49999997), t))
        return (q * scale.half().float()).view(y.shape).half()
    c = torch.tensor(CENTROIDS[_bits(fmt)], device="cuda", dtype=torch.float64)
    R = _rotation(side, torch.float64)
    norm = y.square().sum(-1, keepdim=True).sqrt()
    code = torch.bucketize(y / torch.where(norm > 0, norm, 1) @ R.T, (c[1:] + c[:-1]) / 2)
    got = c[code]
    size = got.square().sum(-1, keepdim=True).sqrt()
    return ((got * (norm / size).half().double()) @ R).half()


def _attend_plain(s):
    batch, hq, hkv, n = s["batch"], s["hq"], s["hkv"], s["longest"]
    k, v = (_values(s[side + "_pages"][s["table"].reshape(-1).long()], s[side], side) for side in "kv")
    lay = lambda x: x.view(batch, -1, hkv, BLOCK, D).transpose(1, 2).reshape(batch, hkv, -1, D)  # noqa: E731
    k, v = lay(k), lay(v)
    cu, lens = s["cu"].long(), s["lens"].long()
    length = cu[1:] - cu[:-1]
    at = torch.arange(n, device="cuda")[None] - (n - length)[:, None]       # a sequence's row, padded in front
    there = at >= 0
    q = s["q"][(cu[:-1, None] + at.clamp(min=0)).reshape(-1)].view(batch, n, hq, D).float()
    if s["k"] != "q8_0":
        q = q @ _rotation(0, torch.float32).T
    g = hq // hkv
    q = q.view(batch, n, hkv, g, D).permute(0, 2, 3, 1, 4).reshape(batch, hkv, g * n, D)
    logits = (q @ k.transpose(-1, -2)).view(batch, hkv, g, n, -1)
    logits *= 1 / math.sqrt(D)
    seen = lens[:, None] - length[:, None] + at + 1 if s["causal"] else lens[:, None].expand(batch, n)
    place = torch.arange(k.shape[2], device="cuda")
    logits.masked_fill_((place >= seen[..., None])[:, None, None], -math.inf)
    top = logits.amax(-1, keepdim=True)
    logits -= torch.where(top == -math.inf, 0, top)
    w = logits.exp_()
    total = w.sum(-1, keepdim=True)
    o = (w.view(batch, hkv, g * n, -1) @ v).view(batch, hkv, g, n, D) / torch.where(total > 0, total, 1)
    if s["v"] != "q8_0":
        o = o @ _rotation(1, torch.float32)
    return o.permute(0, 3, 1, 2, 4).reshape(batch, n, hq, D)[there].to(s["q"].dtype)


# ---- the calls that a user makes ----------------------------------------------------------------------------------------

@functools.lru_cache(maxsize=None)
def _rotary(rot, layout, scaling):
    import turboquant_plus_amd as tqa
    how = {"none": None, "linear": tqa.RotaryScaling("linear", 8.0), "ntk": tqa.RotaryScaling("ntk", 8.0),
           "yarn": tqa.RotaryScaling("yarn", 8.0, trained_tokens=4096)}[scaling]
    return tqa.Rotary(rot, base=10000.0, interleaved=layout == "interleaved", scaling=how)


@functools.lru_cache(maxsize=None)
def _codec(fmt, side):
    import turboquant_plus_amd as tqa
    if fmt == "q8_0":
        return None
    s1, s2 = _signs(side)
    return tqa.TurboCodec(_bits(fmt), signs1=s1.numpy(), signs2=s2.numpy(), centroids=CENTROIDS[_bits(fmt)])


@functools.lru_cache(maxsize=None)
def _attention(k, v, hq, hkv, causal):
    import turboquant_plus_amd as tqa
    return tqa.PagedAttention(_codec(k, 0), _codec(v, 1), hq, hkv, causal=causal)


def _run_own(s):
    import turboquant_plus_amd as tqa
    if s["path"] == "rotary":
        return _rotary(s["rot"], s["layout"], s["scaling"])(s["q"], s["k"], s["positions"], inverse=s["inverse"])
    if s["path"] == "append":
        codecs = _codec(s["k"], 0), _codec(s["v"], 1)
        tqa.append_paged(*codecs, s["key"], s["value"], s["k_pages"], s["v_pages"], s["table"], s["start"], s["cu"])
        return tqa.load_paged(*codecs, s["k_pages"], s["v_pages"], s["table"], s["start"], s["cu"], s["rows"])
    return _attention(s["k"], s["v"], s["hq"], s["hkv"], s["causal"])(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"],
                                                                      s["cu"], max_context=s["max_context"], max_new=s["longest"])


def run(state):
    if own:
        return _run_own(state)
    if state["path"] == "rotary":
        f, size = _frequencies(state)
        a = state["positions"].double()[:, None, None] * f * (-1 if state["inverse"] else 1)
        cos, sin = (size * a.cos()).float(), (size * a.sin()).float()
        return _rotate_plain(state["q"], cos, sin, state), _rotate_plain(state["k"], cos, sin, state)
    if state["path"] == "append":
        return _stored_plain(state["key"], state["k"], 0), _stored_plain(state["value"], state["v"], 1)
    return _attend_plain(state)


# ---- in 64 bits, from the definitions -----------------------------------------------------------------------------------

def _transform(x, side, back):
    """The rotation of the last axis by butterflies, or its transpose."""
    s1, s2 = (t.cuda() for t in _signs(side))
    y = x * (s2 if back else s1)
    step = 1
    while step < D:
        y = y.reshape(*x.shape[:-1], D // (2 * step), 2, step)
        y = torch.stack([y[..., 0, :] + y[..., 1, :], y[..., 0, :] - y[..., 1, :]], -2)
        step *= 2
    return y.reshape(x.shape) * (s1 if back else s2) / D ** 0.5


def _nearest(y, levels):
    """Indices of the levels (ascending) that lie nearest; halfway: the lower one."""
    best, dist = torch.zeros_like(y, dtype=torch.long), (y - levels[0]).abs()
    for i in range(1, len(levels)):
        d = (y - levels[i]).abs()
        best, dist = torch.where(d < dist, i, best), torch.minimum(d, dist)
    return best


def _exact_stored(x, fmt, side):
    y = x.double()
    if fmt == "q8_0":
        g = y.view(*y.shape[:-1], 4, 32)
        d = g.abs().amax(-1, keepdim=True) / 127
        t = g / torch.where(d > 0, d, 1)
        return (t.sign() * (t.abs() + 0.5).floor() * d.half().double()).view(y.shape)
    levels = [float(c) for c in CENTROIDS[_bits(fmt)]]
    norm = torch.linalg.vector_norm(y, dim=-1, keepdim=True)
    z = _transform(y, side, False) / torch.where(norm > 0, norm, 1)
    got = torch.tensor(levels, device="cuda", dtype=torch.float64)[_nearest(z, levels)]
    norm = (norm / torch.linalg.vector_norm(got, dim=-1, keepdim=True)).half().double()
    return _transform(got * norm, side, True)


def _exact_rows(block, fmt, kind, side):
    """Packed blocks [n, bytes] of one head -> rows [n * 128, 128] of the original domain, by words."""
    n = block.shape[0]
    if fmt == "q8_0":
        q = block[:, :BLOCK * D].contiguous().view(torch.int8).view(n, 8, BLOCK, 16).double()
        scale = block[:, BLOCK * D:].contiguous().view(torch.float16).double()
        if kind == "k":
            return (q.permute(0, 2, 1, 3).reshape(n, BLOCK, 4, 32) * scale.view(n, BLOCK, 4, 1)).reshape(-1, D)
        # [chunk = half * 4 + token / 16][tile * 64 + dim % 64][token % 16]
        q = q.view(n, 2, 4, 2, 64, 16).permute(0, 3, 2, 5, 1, 4).reshape(n, 2, 64, 4, 32)
        return (q * scale.view(n, 2, 4, 64).transpose(2, 3).unsqueeze(-1)).reshape(-1, D)
    bits = _bits(fmt)
    words = block[:, :BLOCK * 16 * bits].contiguous().view(torch.int32).long() & 0xffffffff
    words = words.view(n, bits, BLOCK, 4).permute(0, 2, 3, 1)               # [block, row, group, word of the group]
    if bits == 3:
        tail = (words[..., 0] >> 24) | ((words[..., 1] >> 24) << 8) | ((words[..., 2] >> 24) << 16)
        words, per = torch.cat([words & 0xffffff, tail[..., None]], -1), 4
    else:
        per = 16 // bits
    pairs = torch.stack([(words >> (2 * bits * i)) & (4 ** bits - 1) for i in range(per)], -1).flatten(-2)     # [.., 16 pairs]
    codes = torch.stack([pairs & (2 ** bits - 1), pairs >> bits], -1)       # [block, row, group, pair, 2]
    if kind == "k":
        codes = codes.reshape(n, BLOCK, D)
    else:   # row = tile * 64 + dim % 64; group, pair -> four tokens, half of the dims, two tokens
        codes = codes.view(n, 2, 64, 4, 4, 2, 2, 2).permute(0, 1, 3, 4, 6, 7, 5, 2).reshape(n, BLOCK, D)
    value = torch.tensor(CENTROIDS[bits], device="cuda", dtype=torch.float64)[codes]
    norm = block[:, BLOCK * 16 * bits:].contiguous().view(torch.float16).double()
    return _transform((value * norm[..., None]).view(-1, D), side, True)


def _exact_frequencies(case):
    """Pair by pair: how far a pair turns per position; yarn: pairs that turn 32 times and more over the trained tokens keep their
    speed, those that turn once or less get an eighth of it, with a straight line over the (whole) pair numbers between."""
    r, how = case["rot"], case["scaling"]
    base = 10000.0 * (8.0 ** (r / (r - 2)) if how == "ntk" else 1.0)
    plain = [math.exp(-math.log(base) * 2 * i / r) for i in range(r // 2)]
    if how == "linear":
        plain = [f / 8.0 for f in plain]
    if how == "yarn":
        # plain[i] * 4096 = 2 pi turns  <=>  i = r log(4096 / (2 pi turns)) / (2 log base)
        first, last = (r * math.log(4096 / (2 * math.pi * turns)) / (2 * math.log(base)) for turns in (32.0, 1.0))
        first, last = max(math.floor(first), 0), min(math.ceil(last), r - 1)
        part = [min(max((i - first) / max(last - first, 1e-3), 0.0), 1.0) for i in range(r // 2)]
        plain = [f * (1 - w + w / 8.0) for f, w in zip(plain, part)]
    return torch.tensor(plain, dtype=torch.float64, device="cuda"), 1.0 + 0.1 * math.log(8.0) if how == "yarn" else 1.0


def exact(case, seed):
    s = prepare(case, seed)
    if case["path"] == "rotary":
        f, size = _exact_frequencies(case)
        turn = torch.polar(torch.full((1,), size, dtype=torch.float64, device="cuda"), torch.outer(s["positions"].double(), f))
        turn = (turn.conj() if case["inverse"] else turn)[:, None]
        out = []
        for x in (s["q"], s["k"]):
            y, r = x.double().clone(), case["rot"]
            lower, upper = (slice(0, r // 2), slice(r // 2, r)) if case["layout"] == "half" else (slice(0, r, 2), slice(1, r, 2))
            z = torch.complex(y[..., lower], y[..., upper]) * turn
            y[..., lower], y[..., upper] = z.real, z.imag
            out.append(y)
        return tuple(out)
    if case["path"] == "append":
        return _exact_stored(s["key"], case["k"], 0), _exact_stored(s["value"], case["v"], 1)
    cu, lens, table = s["cu"].tolist(), s["lens"].tolist(), s["table"].long()
    if sum((b - a) * c for a, b, c in zip(cu, cu[1:], lens)) * case["hq"] > 1 << 33:
        return None
    g, out = case["hq"] // case["hkv"], torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, c in enumerate(lens):
        n = cu[b + 1] - cu[b]
        pages = table[b, :-(-c // BLOCK)]
        place = torch.arange(c, device="cuda")
        row = torch.arange(n, device="cuda")
        for h in range(case["hkv"]):
            k = _exact_rows(s["k_pages"][pages, h], case["k"], "k", 0)[:c]
            v = _exact_rows(s["v_pages"][pages, h], case["v"], "v", 1)[:c]
            for j in range(h * g, (h + 1) * g):
                logits = s["q"][cu[b]:cu[b + 1], j].double() @ k.T / D ** 0.5
                if case["causal"]:
                    logits = torch.where(place[None] > c - n + row[:, None], -math.inf, logits)
                out[cu[b]:cu[b + 1], j] = torch.softmax(logits, -1) @ v
    return out


def work(case):
    """Inputs read once, outputs written once; of ragged batches the mean lengths."""
    each = 4 if case["dtype"] == "fp32" else 2
    if case["path"] == "rotary":
        return {"bytes": 2 * case["tokens"] * (case["hq"] + case["hkv"]) * case["d"] * each + 8 * case["tokens"],
                "flops": 3 * case["tokens"] * (case["hq"] + case["hkv"]) * case["rot"]}
    mean = (1 - 1 / 8) / math.log(8.0) if case["ragged"] else 1.0       # of _lengths
    size = (_block_bytes(case["k"]) + _block_bytes(case["v"])) / BLOCK
    if case["path"] == "append":
        rows = case["batch"] * case["new"] * mean * case["hkv"]
        return {"bytes": rows * (2 * D * each + 2 * size + 2 * D * 2), "flops": rows * 2 * (2 * D * 7 + 8 * D)}
    prompt = case["causal"] and case["new"] >= case["context"]
    new = case["new"] * (mean if case["new"] > 16 else 1.0)
    context = case["context"] * mean
    pairs = new * context
    if case["causal"]:
        pairs = new * (context - new / 2 + 0.5)
    if prompt and case["ragged"]:       # the same lengths: the mean of their squares
        pairs = case["new"] ** 2 / 2 * (1 - 1 / 64) / (2 * math.log(8.0))
    return {"bytes": case["batch"] * (context * case["hkv"] * size + 2 * new * case["hq"] * D * 2),
            "flops": 4 * D * case["batch"] * case["hq"] * pairs}
