"""What is measured of the operators around the paged cache: attention over a cache held in 8 bits, appending to a paged
cache, and the norm and rotation of queries and keys.  Each has a plain form in elementary torch operations (fp32, rounded
once at the end), the framework's own call, and its definition in 64 bits.

An 8-bit cache holds e4m3 codes, (blocks, kv heads, block size, D), and an fp32 scale for each block and kv head: a code c
stands for c * scale.  The scale that an append gives a block is the least power of two that keeps the block's largest
magnitude within 448, the largest e4m3 number; a block that already holds tokens keeps the larger of that and the scale it
has, and what it holds is rounded again where the scale has grown.
"""
import math

import torch

own = False

E4M3 = torch.float8_e4m3fn
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def attend(name, dtype, seqs, lo, hi, heads, kv_heads, D, block, empty=0):
    """`empty`: every so many-th sequence has no keys (0: none)."""
    return {"name": name, "op": "attend", "dtype": dtype, "seqs": seqs, "lo": lo, "hi": hi, "heads": heads,
            "kv_heads": kv_heads, "D": D, "block": block, "empty": empty}


def append(name, dtype, bits, seqs, new_lo, new_hi, old_lo, old_hi, kv_heads, D, block, rotary, interleaved=False, pad=0):
    """new_lo .. new_hi new tokens a sequence behind old_lo .. old_hi cached ones; pad: rows behind the last sequence."""
    return {"name": name, "op": "append", "dtype": dtype, "bits": bits, "seqs": seqs, "new_lo": new_lo, "new_hi": new_hi,
            "old_lo": old_lo, "old_hi": old_hi, "kv_heads": kv_heads, "D": D, "block": block, "rotary": rotary,
            "interleaved": interleaved, "pad": pad}


def rotary(name, dtype, batch, tokens, heads, kv_heads, D, size, weights, backward, interleaved=False, heads_first=False):
    """tokens 0: `batch` single tokens, (batch, heads, D), at positions of their own.  weights: "" for no norm."""
    return {"name": name, "op": "rotary", "dtype": dtype, "batch": batch, "tokens": tokens, "heads": heads,
            "kv_heads": kv_heads, "D": D, "rotary": size, "weights": weights, "backward": backward,
            "interleaved": interleaved, "heads_first": heads_first}


def listed():
    return [
        # one request that has just begun: nothing but latency
        attend("attend, one short sequence", "bf16", 1, 300, 300, 32, 8, 128, 16),
        # the decode batch of this repository's benchmark, over a cache of half the bytes
        attend("attend, 64 sequences", "fp16", 64, 512, 8192, 32, 8, 128, 16),
        # a large batch of short requests with slots that are free, every head with keys of its own
        attend("attend, 300 short, some empty", "bf16", 300, 1, 700, 16, 16, 64, 32, empty=11),
        # a few long documents, twelve query heads to a kv head
        attend("attend, long documents", "fp16", 3, 40001, 120001, 48, 4, 256, 64),
        # a single token of a single request into a 16-bit cache
        append("append, one token", "bf16", 16, 1, 1, 1, 700, 700, 8, 128, 16, 128),
        # the decode step of a batch: one token each
        append("append, 64 tokens to 8 bits", "bf16", 8, 64, 1, 1, 0, 480, 8, 128, 16, 128),
        # prompts of a batch, with the rows that pad it to a fixed size
        append("append, prompts to 8 bits", "bf16", 8, 16, 37, 2011, 0, 90, 8, 128, 16, 128, pad=100),
        # prompts of a model with many small heads that turns half of each, pairs side by side
        append("append, prompts to 16 bits", "fp16", 16, 5, 1, 3501, 0, 0, 32, 64, 32, 32, interleaved=True),
        # the decode step of a batch
        rotary("rotary, 64 tokens", "bf16", 64, 0, 32, 8, 128, 128, "bf16", False),
        # a long prompt, heads as the projection leaves them
        rotary("rotary, prompt", "bf16", 1, 8192, 32, 8, 128, 128, "bf16", False),
        # a training step
        rotary("rotary, training", "bf16", 2, 4096, 32, 8, 128, 128, "fp32", True),
        # a training step without norm, heads in front, an odd length
        rotary("rotary, training without norm", "fp16", 3, 1021, 16, 16, 64, 64, "", True, interleaved=True, heads_first=True),
    ]


def spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind, dtype = rng.choice(("attend", "append", "rotary")), rng.choice(("bf16", "fp16"))
    D = rng.choice((64, 128, 128, 128, 256, 16, 32, 512))
    block = rng.choice((16, 16, 32, 64, 128, 8, 24, 20))
    kv_heads = rng.choice((1, 2, 3, 4, 8, 8, 16))
    if kind == "attend":
        group = rng.choice((1, 2, 4, 4, 5, 8, 12, 16, 20))
        seqs = spread(rng, 1, 300)
        most = max(1, min(130000, 250_000_000 // (seqs * kv_heads * D)))   # keys a sequence: the plain form pads to the longest
        hi = spread(rng, 1, most)
        return attend("", dtype, seqs, rng.choice((hi, max(1, hi // 16))), hi, group * kv_heads, kv_heads, D, block,
                      rng.choice((0, 0, 5)) if seqs > 1 else 0)
    interleaved = rng.choice((False, False, True))
    size = D if D < 32 else rng.choice((D, D, D // 2))
    if kind == "append":
        seqs = spread(rng, 1, 256)
        new = 1 if rng.random() < 0.4 else spread(rng, 1, max(1, min(4000 * block, 30_000_000 // (kv_heads * D)) // seqs))
        old = spread(rng, 1, max(1, min(2000, 60_000_000 // (seqs * kv_heads * D))))
        return append("", dtype, rng.choice((8, 8, 16)), seqs, rng.choice((new, max(1, new // 9))), new, rng.choice((0, old)), old,
                      kv_heads, D, block, rng.choice((size, size, 0)), interleaved, rng.choice((0, 0, 13)) if new > 1 else 0)
    heads, backward = kv_heads * rng.choice((1, 2, 4, 7)), rng.choice((False, True))
    rows = spread(rng, 1, max(1, 45_000_000 // ((heads + kv_heads) * D)))
    batch = rng.choice((1, 1, 2, 3))
    one_each = rows < 1000 and not backward and rng.random() < 0.5
    return rotary("", dtype, rows if one_each else batch, 0 if one_each else max(1, rows // batch), heads, kv_heads, D, size,
                  rng.choice((dtype, "fp32", "")), backward, interleaved, rng.choice((False, True)) and not one_each)


def between(lo, hi, n):
    """n lengths spread evenly over lo .. hi."""
    return [lo + ((hi - lo) * (2 * i + 1)) // (2 * n) for i in range(n)] if n > 1 else [hi]


def lengths_of(c):
    lens = between(c["lo"], c["hi"], c["seqs"])
    return [0 if c["empty"] and i % c["empty"] == c["empty"] // 2 else n for i, n in enumerate(lens)]


def bytes_of(dtype):
    return 4 if dtype == "fp32" else 2


def work(case):
    c = case
    if c["op"] == "attend":
        keys = sum(lengths_of(c)) * c["kv_heads"]
        blocks = sum(-(-n // c["block"]) for n in lengths_of(c))
        return {"bytes": keys * 2 * c["D"] + blocks * (c["kv_heads"] * 8 + 4) + c["seqs"] * (c["heads"] * c["D"] * 2 * 2 + 4),
                "flops": keys * (c["heads"] // c["kv_heads"]) * c["D"] * 4}
    if c["op"] == "append":
        news = between(c["new_lo"], c["new_hi"], c["seqs"])
        values, blocks = sum(news) * c["kv_heads"] * c["D"] * 2, sum(-(-n // c["block"]) for n in news)
        scales = blocks * c["kv_heads"] * 2 * 4 if c["bits"] == 8 else 0
        return {"bytes": values * (2 + c["bits"] // 8) + scales + sum(news) * c["rotary"] * 4 + blocks * 4 + c["seqs"] * 8,
                "flops": values // 2 * 3 * (c["rotary"] > 0) + values * 2 * (c["bits"] == 8)}
    rows = c["batch"] * max(1, c["tokens"]) * (c["heads"] + c["kv_heads"])
    table = max(1, c["tokens"]) * (1 if c["tokens"] else c["batch"]) * c["rotary"] * 4
    weights = 2 * c["D"] * bytes_of(c["weights"]) if c["weights"] else 0
    passes = 2 + (3 if c["weights"] else 2) * c["backward"]   # read and write; gradient (and input) read, gradient written
    return {"bytes": rows * c["D"] * 2 * passes + table * (1 + c["backward"]) + weights * (1 + 2 * c["backward"]),
            "flops": rows * c["D"] * (3 + 4 * bool(c["weights"])) * (1 + 2 * c["backward"])}


# ------------------------------------------------------------------------------------------------ inputs ----
def scale_for(peak):
    """The least power of two that keeps `peak` within 448, between 2^-118 and 2^120."""
    mantissa, exponent = torch.frexp(peak)   # peak = mantissa * 2^exponent, mantissa in [0.5, 1); 448 = 0.875 * 2^9
    exponent = exponent - 9 + (mantissa > 0.875).to(exponent.dtype)
    exponent = torch.where(peak > 0, exponent, -118).clamp(-118, 120)
    return torch.ldexp(torch.ones_like(peak), exponent)


def tables(positions, size):
    angle = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * \
        10000.0 ** -(torch.arange(0, size, 2, device="cuda", dtype=torch.float64) / size)
    return angle.cos().float(), angle.sin().float()


def prepare(case, seed):
    c, g = case, torch.Generator(device="cuda").manual_seed(seed)
    dtype, D = TYPES[c["dtype"]], c["D"]

    def normal(*shape, dtype=dtype):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)

    def filled_cache(blocks):
        """Keys or values of a running request: magnitudes differ from head to head and drift from block to block."""
        x = torch.randn((blocks, c["kv_heads"], c["block"], D), generator=g, device="cuda")
        x *= torch.exp(0.7 * torch.randn((blocks, c["kv_heads"], 1, 1), generator=g, device="cuda"))
        if c.get("bits", 8) == 16:
            return x.to(dtype), None
        scale = scale_for(x.abs().amax((2, 3)))
        return (x / scale[:, :, None, None]).to(E4M3), scale

    def block_table(rows, longest):
        """Blocks in no order, as an allocator that has run for a while hands them out."""
        width = -(-longest // c["block"])
        order = torch.randperm(rows * width + 3, generator=g, device="cuda")
        return order[:rows * width].reshape(rows, width).to(torch.int32), rows * width + 3

    def shuffled(lens):
        return torch.tensor(lens, device="cuda", dtype=torch.int32)[torch.randperm(len(lens), generator=g, device="cuda")]

    if c["op"] == "attend":
        lens = shuffled(lengths_of(c))
        longest = max(1, max(lengths_of(c)))
        table, blocks = block_table(c["seqs"], longest)
        (kc, ks), (vc, vs) = filled_cache(blocks), filled_cache(blocks)
        return {"case": c, "q": normal(c["seqs"], c["heads"], D), "kc": kc, "ks": ks, "vc": vc, "vs": vs, "lens": lens,
                "table": table, "scale": D ** -0.5, "longest": longest}
    if c["op"] == "append":
        news, olds = shuffled(between(c["new_lo"], c["new_hi"], c["seqs"])), shuffled(between(c["old_lo"], c["old_hi"], c["seqs"]))
        total, longest = sum(between(c["new_lo"], c["new_hi"], c["seqs"])) + c["pad"], c["new_hi"] + c["old_hi"]
        table, blocks = block_table(c["seqs"], longest)
        (kc, ks), (vc, vs) = filled_cache(blocks), filled_cache(blocks)
        starts = None
        if c["new_hi"] > 1:
            starts = torch.zeros(c["seqs"] + 1, device="cuda", dtype=torch.int32)
            starts[1:] = news.cumsum(0)
        cos, sin = tables(longest, c["rotary"]) if c["rotary"] else (None, None)
        return {"case": c, "k": normal(total, c["kv_heads"], D), "v": normal(total, c["kv_heads"], D), "kc": kc, "ks": ks,
                "vc": vc, "vs": vs, "lens": news + olds, "table": table, "starts": starts, "cos": cos, "sin": sin}
    state = {"case": c, "positions": None, "wq": None, "wk": None}
    shapes = []
    for heads in (c["heads"], c["kv_heads"]):
        T = c["tokens"]
        shapes.append((c["batch"], heads, D) if not T else (c["batch"], heads, T, D) if c["heads_first"] else (c["batch"], T, heads, D))
    for name, shape in zip("qk", shapes):
        for x in (name, "g" + name) if c["backward"] else (name,):
            t = normal(*shape)
            state[x] = t.transpose(1, 2) if c["tokens"] and not c["heads_first"] else t
        state[name].requires_grad_(c["backward"])
    if c["weights"]:
        for name in ("wq", "wk"):
            state[name] = (1 + 0.2 * normal(D, dtype=torch.float32)).to(TYPES[c["weights"]]).requires_grad_(c["backward"])
    positions = c["tokens"]
    if not positions:
        positions = 4096
        state["positions"] = torch.randint(0, positions, (c["batch"],), generator=g, device="cuda", dtype=torch.int32)
    state["cos"], state["sin"] = tables(positions, c["rotary"])
    return state


# ------------------------------------------------------------------------------------------- plain forms ----
def plain_rotate(x, cos, sin, interleaved):
    """x (..., D) fp32 with cos, sin (..., size / 2): the first `size` values turned in pairs."""
    size = 2 * cos.shape[-1]
    turned, rest = x[..., :size], x[..., size:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = turned[..., :size // 2], turned[..., size // 2:]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, rest), -1)


def plain_attend(s):
    q, lens, table = s["q"], s["lens"], s["table"].long()
    seqs, heads, D = q.shape
    kv_heads, block = s["kc"].shape[1:3]
    keys = table.shape[1] * block

    def gathered(codes, scales):   # (seqs, kv heads, keys, D)
        x = codes[table].float() * scales[table][..., None, None]
        return x.permute(0, 2, 1, 3, 4).reshape(seqs, kv_heads, keys, D)

    grouped = q.float().view(seqs, kv_heads, heads // kv_heads, D)
    scores = torch.matmul(grouped, gathered(s["kc"], s["ks"]).transpose(2, 3)) * s["scale"]
    seen = torch.arange(keys, device=q.device) < lens[:, None, None, None]
    scores = scores.masked_fill(~seen, -math.inf)
    peak = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(peak == -math.inf, 0.0, peak))
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights, gathered(s["vc"], s["vs"])) / torch.where(total == 0, 1.0, total)
    return out.view(seqs, heads, D).to(q.dtype)


def plain_append(s):
    c, lens, table = s["case"], s["lens"].long(), s["table"].long()
    block, rows = c["block"], s["k"].shape[0]
    starts = s["starts"].long() if s["starts"] is not None else torch.arange(c["seqs"] + 1, device=lens.device)
    row = torch.arange(rows, device=lens.device)
    seq = torch.searchsorted(starts[1:].contiguous(), row, right=True)
    there = seq < c["seqs"]
    seq = seq.clamp(max=c["seqs"] - 1)
    place = lens[seq] - starts[seq + 1] + row
    there = there & (place >= 0)
    first = there.int().argmax()          # a row that is appended stands in for those that are not
    row, seq, place = (torch.where(there, x, x[first]) for x in (row, seq, place))
    k, v = s["k"].float()[row], s["v"].float()[row]
    if c["rotary"]:
        k = plain_rotate(k, s["cos"][place][:, None], s["sin"][place][:, None], c["interleaved"])
    into, slot = table[seq, place // block], place % block
    # the block each sequence begins in, which may hold earlier tokens; sequences without new tokens repeat another's
    begin = torch.maximum(lens - (starts[1:] - starts[:-1]), torch.zeros_like(lens))
    some = (starts[1:] > starts[:-1]) & (lens > 0)
    stand = some.int().argmax()
    begin = torch.where(some, begin, begin[stand])
    partial = table[torch.where(some, torch.arange(c["seqs"], device=lens.device), stand), begin // block]
    held = (begin % block)[:, None, None, None]
    for x, cache, scales in ((k, s["kc"], s["ks"]), (v, s["vc"], s["vs"])):
        if scales is None:
            cache.permute(0, 2, 1, 3)[into, slot] = x.to(cache.dtype)
            continue
        finite = torch.where(x.isfinite(), x.abs(), 0.0).amax(-1)
        peak = torch.zeros_like(scales).scatter_reduce_(0, into[:, None].expand_as(finite), finite, "amax")
        before = scales[partial]
        needed = scale_for(peak[into])
        scales[into] = needed
        after = torch.where(held[:, :, 0, 0] > 0, torch.maximum(before, scale_for(peak[partial])), scales[partial])
        scales[partial] = after
        old = cache[partial]
        again = (old.float() * (before / after)[..., None, None]).to(E4M3)
        cache[partial] = torch.where(torch.arange(block, device=lens.device)[:, None] < held, again.float(), old.float()).to(E4M3)
        cache.permute(0, 2, 1, 3)[into, slot] = (x * (1.0 / scales[into])[..., None]).to(E4M3)
    return [t for t in (s["kc"], s["vc"], s["ks"], s["vs"]) if t is not None]


def plain_rotary(s):
    c, outs = s["case"], []
    cos, sin = (s[x] if s["positions"] is None else s[x][s["positions"].long()][:, None] for x in ("cos", "sin"))
    for x, w in ((s["q"], s["wq"]), (s["k"], s["wk"])):
        y = x.float()
        if w is not None:
            y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-6) * w.float()
        outs.append(plain_rotate(y, cos, sin, c["interleaved"]).to(x.dtype))
    return outs


def run(state):
    s, c = state, state["case"]
    if c["op"] == "attend":
        if own:
            import flag_attn
            return flag_attn.paged_attention_fp8(s["q"], s["kc"], s["vc"], s["ks"], s["vs"], s["lens"], s["table"], s["scale"], s["longest"])
        return plain_attend(s)
    if c["op"] == "append":
        if own:
            import flag_attn
            flag_attn.paged_append(s["k"], s["v"], s["kc"], s["vc"], s["lens"], s["table"], query_starts=s["starts"],
                                   key_scales=s["ks"], value_scales=s["vs"], cos=s["cos"], sin=s["sin"], interleaved=c["interleaved"])
            return [t for t in (s["kc"], s["vc"], s["ks"], s["vs"]) if t is not None]
        return plain_append(s)
    if own:
        import flag_attn
        outs = flag_attn.norm_rotary(s["q"], s["k"], s["cos"], s["sin"], positions=s["positions"], q_weight=s["wq"],
                                     k_weight=s["wk"], eps=1e-6, interleaved=c["interleaved"])
    else:
        outs = plain_rotary(s)
    if not c["backward"]:
        return list(outs)
    leaves = [s[x] for x in ("q", "k", "wq", "wk") if s[x] is not None]
    return [o.detach() for o in outs] + list(torch.autograd.grad(outs, leaves, (s["gq"], s["gk"])))


# --------------------------------------------------------------------------------------- the definitions ----
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"attend": exact_attend, "append": exact_append, "rotary": exact_rotary}[case["op"]](case, s)


def exact_attend(c, s):
    group = c["heads"] // c["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for i, n in enumerate(s["lens"].tolist()):
        if n == 0:
            continue
        at = s["table"][i, :-(-n // c["block"])].long()
        for h in range(c["kv_heads"]):
            k, v = ((codes[at, h].double() * scales[at, h].double()[:, None, None]).reshape(-1, c["D"])[:n]
                    for codes, scales in ((s["kc"], s["ks"]), (s["vc"], s["vs"])))
            heads = slice(h * group, (h + 1) * group)
            out[i, heads] = torch.softmax(s["q"][i, heads].double() @ k.T * s["scale"], -1) @ v
    return out


def exact_turn(a, b, angle_cos, angle_sin):
    """The pair (a, b) as a complex number, times cos + i sin."""
    z = torch.complex(a, b) * torch.complex(angle_cos, angle_sin)
    return z.real, z.imag


def exact_rotate(x, cos, sin, interleaved, back=False):
    y, half = x.clone(), cos.shape[-1]
    first = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    second = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    cos, sin = torch.broadcast_tensors(cos.double(), (-sin if back else sin).double())
    shape = x[..., first].shape
    y[..., first], y[..., second] = exact_turn(x[..., first], x[..., second], cos.expand(shape), sin.expand(shape))
    return y


def exact_e4m3(x):
    """x rounded to the nearest e4m3 number, ties to the even one: steps of 1/8 of the power of two below, at least 2^-9."""
    step = torch.exp2((torch.frexp(x)[1] - 1).clamp(min=-6).double() - 3)
    return torch.round(x / step) * step


def exact_append(c, s):
    ends = s["starts"].tolist() if s["starts"] is not None else list(range(c["seqs"] + 1))
    block, result = c["block"], []
    caches = {"k": (s["kc"].double(), s["ks"].double() if s["ks"] is not None else None),
              "v": (s["vc"].double(), s["vs"].double() if s["vs"] is not None else None)}
    for i, n in enumerate(s["lens"].tolist()):
        news = min(ends[i + 1] - ends[i], n)
        for x, (codes, scales) in caches.items():
            new = s[x][ends[i + 1] - news:ends[i + 1]].double()
            if x == "k" and c["rotary"]:
                new = exact_rotate(new, s["cos"][n - news:n, None], s["sin"][n - news:n, None], c["interleaved"])
            place = n - news
            while place < n:
                b, slot = int(s["table"][i, place // block]), place % block
                take = min(block - slot, n - place)
                part = new[place - (n - news):][:take].transpose(0, 1)          # (kv heads, take, D)
                if scales is not None:
                    peak = part.abs().amax((1, 2))
                    fit = torch.exp2(torch.ceil(torch.log2(peak / 448)).clamp(-118, 120))
                    scale = torch.maximum(fit, scales[b]) if slot else fit
                    if slot:
                        codes[b, :, :slot] = exact_e4m3(codes[b, :, :slot] * (scales[b] / scale)[:, None, None])
                    scales[b] = scale
                    part = exact_e4m3(part / scale[:, None, None])
                codes[b, :, slot:slot + take] = part
                place += take
    result = [caches["k"][0], caches["v"][0]]
    return result + [caches["k"][1], caches["v"][1]] if s["ks"] is not None else result


def exact_rotary(c, s):
    outs, grads, weight_grads = [], [], []
    cos, sin = (s[x] if s["positions"] is None else s[x][s["positions"].long()][:, None] for x in ("cos", "sin"))
    for x in "qk":
        value, w = s[x].double(), s["w" + x]
        norm = 1 / torch.sqrt(value.square().mean(-1, keepdim=True) + 1e-6) if w is not None else 1.0
        scaled = value * norm
        outs.append(exact_rotate(scaled * w.double() if w is not None else scaled, cos, sin, c["interleaved"]))
        if c["backward"]:
            back = exact_rotate(s["g" + x].double(), cos, sin, c["interleaved"], back=True)
            if w is None:
                grads.append(back)
                continue
            weight_grads.append((back * scaled).sum((0, 1, 2)))
            back = back * w.double()
            grads.append(norm * (back - scaled * (back * scaled).mean(-1, keepdim=True)))
    return outs + grads + weight_grads
