"""Performance cases of what lies between a decoder's QKV and O projections: rotary positions, the quantized key/value cache, and the
attention that reads it, for one sequence each or behind a prefix that the whole batch shares.

Kinds of case:
  rotary     heads of a packed QKV buffer are turned by their positions (`Context.rotary`).
  cache      the new tokens' keys and values are normalised, turned, quantized and written (`Context.cache_write`, which turns the
             queries too), and a context that holds them is read back as 16-bit rows (`Context.cache_read`).
  attention  queries against the quantized, paged cache (`Context.cached_attention`): a token per sequence (decode), some (drafts
             to be checked), or a chunk of a prompt.
  prefix     the same behind a prefix that all sequences share, such as a voice prompt.

Heads and widths are those of the benchmark's synthetic decoder (16 query heads on 8 key/value heads of 128) and generic ones around
it. `own` selects the framework's calls; otherwise the same outputs come from elementary torch operations.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
RANGE = {"int8": 127.0, "fp8": 448.0}
#: (query heads, key/value heads, head size)
HEADS = ((16, 8, 128), (32, 8, 128), (16, 2, 128), (16, 8, 64), (8, 8, 64), (16, 2, 64))
BASE, ORIGINAL, FACTOR, EPSILON = 1.0e6, 8192, 8.0, 1e-6


def listed():
    return [
        # Three streams of a small decoder that turns part of each head: latency alone.
        {"name": "rotary_interleaved_m3", "kind": "rotary", "rows": 3, "heads": 16, "head_dim": 64, "dims": 32, "interleaved": True,
         "scaling": "linear", "first": 700, "dtype": "f16"},
        # A batch of long prompts, scaled for a long context, at far positions.
        {"name": "rotary_yarn_m8191", "kind": "rotary", "rows": 8191, "heads": 16, "head_dim": 128, "dims": 128, "interleaved": False,
         "scaling": "yarn", "first": 60000, "dtype": "bf16"},
        # One decode step of the benchmark's 64 streams.
        {"name": "cache_int8_m64", "kind": "cache", "rows": 64, "read": 64, "heads": 16, "kv_heads": 8, "head_dim": 128, "page": 64,
         "format": "int8", "interleaved": False, "scaling": "none", "norm": True, "dtype": "bf16"},
        # A ragged chunk of a prompt is written, and all of its context read back for a kernel that wants 16-bit rows.
        {"name": "cache_fp8_m1021_r8190", "kind": "cache", "rows": 1021, "read": 8190, "heads": 16, "kv_heads": 8, "head_dim": 128,
         "page": 16, "format": "fp8", "interleaved": False, "scaling": "yarn", "norm": False, "dtype": "f16"},
        # One stream, a short context: the smallest attention there is.
        {"name": "attention_int8_s1_l777", "kind": "attention", "sequences": 1, "tokens": 1, "length": 777, "ragged": False,
         "heads": 16, "kv_heads": 8, "head_dim": 128, "page": 64, "format": "int8", "prefix": 0, "dtype": "bf16"},
        # The benchmark's 64 streams, every one at a length of its own.
        {"name": "attention_int8_s64_l4096", "kind": "attention", "sequences": 64, "tokens": 1, "length": 4096, "ragged": True,
         "heads": 16, "kv_heads": 8, "head_dim": 128, "page": 64, "format": "int8", "prefix": 0, "dtype": "bf16"},
        # Some long contexts, four query heads to a cached one, small pages.
        {"name": "attention_fp8_s13_l16001", "kind": "attention", "sequences": 13, "tokens": 1, "length": 16001, "ragged": True,
         "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 16, "format": "fp8", "prefix": 0, "dtype": "bf16"},
        # Drafts of a few tokens that are checked at once.
        {"name": "attention_int8_s7_t5_l1500", "kind": "attention", "sequences": 7, "tokens": 5, "length": 1500, "ragged": True,
         "heads": 16, "kv_heads": 8, "head_dim": 128, "page": 32, "format": "int8", "prefix": 0, "dtype": "f16"},
        # Chunks of prompts against what is cached of them.
        {"name": "attention_fp8_s3_t700_l2500", "kind": "attention", "sequences": 3, "tokens": 700, "length": 2500, "ragged": True,
         "heads": 16, "kv_heads": 8, "head_dim": 128, "page": 64, "format": "fp8", "prefix": 0, "dtype": "bf16"},
        # A few streams of a narrow decoder behind a short prompt of odd length.
        {"name": "prefix_fp8_s24_p509_l64", "kind": "attention", "sequences": 24, "tokens": 1, "length": 64, "ragged": True,
         "heads": 16, "kv_heads": 2, "head_dim": 64, "page": 16, "format": "fp8", "prefix": 509, "dtype": "f16"},
        # The benchmark's streams behind one voice prompt.
        {"name": "prefix_int8_s64_p2048_l300", "kind": "attention", "sequences": 64, "tokens": 1, "length": 300, "ragged": True,
         "heads": 16, "kv_heads": 8, "head_dim": 128, "page": 64, "format": "int8", "prefix": 2048, "dtype": "bf16"},
        # Twice as many behind a long one.
        {"name": "prefix_int8_s128_p16384_l600", "kind": "attention", "sequences": 128, "tokens": 1, "length": 600, "ragged": True,
         "heads": 16, "kv_heads": 8, "head_dim": 128, "page": 128, "format": "int8", "prefix": 16384, "dtype": "bf16"},
    ]


def _spread(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(("rotary", "rotary", "cache", "cache", "attention", "attention", "attention", "prefix", "prefix"))
    heads, kv_heads, head_dim = rng.choice(HEADS)
    dtype, scaling = rng.choice(sorted(DTYPES)), rng.choice(("none", "linear", "ntk", "yarn", "wavelength"))
    if kind == "rotary":
        return {"kind": kind, "rows": _spread(rng, 1, 8191 * 16 * 128 // (heads * head_dim)), "heads": heads, "head_dim": head_dim,
                "dims": rng.choice((head_dim // 4, head_dim // 2, head_dim)), "interleaved": rng.random() < 0.5, "scaling": scaling,
                "first": rng.choice((0, _spread(rng, 1, 120000))), "dtype": dtype}
    page, form = rng.choice((16, 32, 64, 128, 256)), rng.choice(sorted(RANGE))
    common = {"heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "format": form, "dtype": dtype}
    if kind == "cache":
        rows = _spread(rng, 1, 1021)
        return {"kind": kind, "rows": rows, "read": _spread(rng, rows, 8190), "interleaved": rng.random() < 0.3, "scaling": scaling,
                "norm": rng.random() < 0.5, **common}
    width = kv_heads * head_dim
    if kind == "prefix":
        sequences, tokens = _spread(rng, 2, 128), rng.choice((1, 1, 1, 2, 3))
        return {"kind": "attention", "sequences": sequences, "tokens": tokens, "length": _spread(rng, 4, 600), "ragged": True,
                "prefix": _spread(rng, 64, 16384 // tokens if heads <= 16 else 8192 // tokens), **common}
    tokens = rng.choice((1, 1, 1, _spread(rng, 2, 16), _spread(rng, 17, 700)))
    sequences = _spread(rng, 1, 64 if tokens <= 16 else 3)
    most = 64 * 4096 * 8 * 128 // (sequences * width) if tokens <= 16 else 2500 * 16 // heads
    return {"kind": kind, "sequences": sequences, "tokens": tokens, "length": _spread(rng, min(32, most), min(most, 32000)),
            "ragged": rng.random() < 0.8, "prefix": 0, **common}


# ----------------------------------------------------------------------------------------------------------------- shapes
def _lengths(case):
    """(cached tokens, query tokens) of each sequence: spread over the range, and an idle slot in larger batches."""
    some = []
    for b in range(case["sequences"]):
        part = (0.618 * (b + 1)) % 1.0 if case["ragged"] else 1.0
        n = 1 + round((case["tokens"] - 1) * ((0.414 * (b + 1)) % 1.0 if case["ragged"] else 1.0))
        length = max(n, round(case["length"] * part))
        some.append((0, 1 if case["tokens"] == 1 else 0) if case["ragged"] and b == 5 and not case["prefix"] else (length, n))
    return some


def _turns(case):
    """Turns per position of each pair of columns, in 64 bits, and the factor on cosine and sine."""
    dims = case.get("dims", case["head_dim"])
    base = BASE * (FACTOR ** (dims / (dims - 2)) if case["scaling"] == "ntk" else 1.0)
    index = torch.arange(dims // 2, dtype=torch.float64)
    rate, scale = base ** (-2.0 * index / dims), 1.0
    if case["scaling"] == "linear":
        rate = rate / FACTOR
    elif case["scaling"] == "yarn":
        low, high = (dims * math.log(ORIGINAL / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (32.0, 1.0))
        low, high = max(math.floor(low), 0), min(math.ceil(high), dims - 1)
        ramp = ((index - low) / max(high - low, 1e-3)).clamp(0, 1)
        rate, scale = rate / FACTOR * ramp + rate * (1 - ramp), 0.1 * math.log(FACTOR) + 1.0
    elif case["scaling"] == "wavelength":
        share = ((ORIGINAL * rate / (2 * math.pi) - 1.0) / 3.0).clamp(0, 1)
        rate = rate / FACTOR * (1 - share) + rate * share
    return rate / (2 * math.pi), scale


# ---------------------------------------------------------------------------------------------------------------- prepare
class _State:
    pass


def _normal(generator, shape, dtype=torch.float32, std=1.0, mean=0.0):
    return (torch.randn(shape, generator=generator, device="cuda") * std + mean).to(dtype)


def _pages(generator, case, count):
    """Random bytes as keys or values take them when quantized by the largest of each row."""
    shape = (count, case["kv_heads"], case["page"], case["head_dim"])
    if case["format"] == "int8":
        values = (torch.randn(shape, generator=generator, device="cuda", dtype=torch.float16) * 42).clamp_(-127, 127).round_()
        values = values.to(torch.int8).view(torch.uint8)
    else:
        values = (torch.randn(shape, generator=generator, device="cuda", dtype=torch.float16) * 150).clamp_(-448, 448)
        values = values.to(torch.float8_e4m3fn).view(torch.uint8)
    scales = torch.rand(shape[:3], generator=generator, device="cuda") * 0.5 + 0.75
    return values, scales * (1.0 / (42 if case["format"] == "int8" else 150))


_contexts = {}


def _context(form):
    """One context for all states: a program has one per device and stream."""
    from breeze_tts_cpp_b200 import ops
    if form not in _contexts:
        _contexts[form] = ops.Context(form, workspace_bytes=64 << 20)
    return _contexts[form]


def prepare(case, seed):
    s, g = _State(), torch.Generator(device="cuda").manual_seed(seed)
    s.case, s.dtype, kind = case, DTYPES[case["dtype"]], case["kind"]
    heads, head_dim = case["heads"], case["head_dim"]
    if kind in ("rotary", "cache"):
        turns, s.scale = _turns(case)
        s.turns, rows = turns.cuda(), case["rows"]
        kv_heads = case.get("kv_heads", heads // 2)
        s.qkv = _normal(g, (rows, (heads + 2 * kv_heads) * head_dim), s.dtype)
        s.q, s.k, s.v = s.qkv.split((heads * head_dim, kv_heads * head_dim, kv_heads * head_dim), 1)
        s.q_out = torch.empty(rows, heads * head_dim, dtype=s.dtype, device="cuda")
    if kind == "rotary":
        start = int(torch.randint(0, 1000, (1,), generator=g, device="cuda"))
        s.positions = torch.arange(rows, dtype=torch.int32, device="cuda") + case["first"] + start
        if own:
            from breeze_tts_cpp_b200 import ops
            s.rotary, s.ctx = ops.Rotary(s.turns, case["interleaved"], s.scale), _context("int8")
        return s
    if kind == "cache":
        # The new tokens are the last of the context that is read; its pages lie anywhere.
        read, page = case["read"], case["page"]
        count = -(-read // page) + 3
        s.keys, s.key_scales = _pages(g, case, count)
        s.values, s.value_scales = _pages(g, case, count)
        order = torch.randperm(count, generator=g, device="cuda")[: -(-read // page)]
        slots = (order[:, None] * page + torch.arange(page, device="cuda")).reshape(-1)[:read].to(torch.int32)
        s.read_slots, s.slots = slots, slots[read - rows:].contiguous()
        s.positions = torch.arange(read - rows, read, dtype=torch.int32, device="cuda")
        s.q_norm, s.k_norm = (_normal(g, (head_dim,), s.dtype, 0.1, 1.0) if case["norm"] else None for _ in range(2))
        s.k_read, s.v_read = (torch.empty(read, kv_heads * head_dim, dtype=s.dtype, device="cuda") for _ in range(2))
    else:
        some, page = _lengths(case), case["page"]
        rows, most = sum(n for _, n in some), max(-(-max(length for length, _ in some) // page), 1)
        needed, shared = [-(-length // page) for length, _ in some], -(-case["prefix"] // page)
        count = sum(needed) + shared + 2
        s.keys, s.key_scales = _pages(g, case, count)
        s.values, s.value_scales = _pages(g, case, count)
        order = torch.randperm(count, generator=g, device="cuda").to(torch.int32)
        s.pages = torch.zeros(case["sequences"], most, dtype=torch.int32, device="cuda")
        used = (torch.arange(most)[None] < torch.tensor(needed)[:, None]).cuda()
        s.pages[used] = order[: sum(needed)]
        s.lengths = torch.tensor([length for length, _ in some], dtype=torch.int32, device="cuda")
        offsets = torch.tensor([0] + [n for _, n in some]).cumsum(0)
        s.offsets = offsets.to(torch.int32).cuda() if case["tokens"] > 1 else None
        s.prefix_pages = order[sum(needed): sum(needed) + shared].contiguous() if shared else None
        s.prefix_length = torch.tensor([case["prefix"]], dtype=torch.int32, device="cuda") if shared else None
        s.q = _normal(g, (rows, heads * head_dim), s.dtype, 1.5)
        s.out = torch.zeros(rows, heads * head_dim, dtype=s.dtype, device="cuda")
        s.tokens = max(n for _, n in some)
    if own:
        from breeze_tts_cpp_b200 import ops
        s.ctx = _context(case["format"])
        s.cache = ops.CacheView(s.keys, s.values, s.key_scales, s.value_scales, ops.FP8 if case["format"] == "fp8" else ops.I8)
        if kind == "cache":
            s.rotary = ops.Rotary(s.turns, case["interleaved"], s.scale)
    return s


# -------------------------------------------------------------------------------------------------------------------- run
def run(s):
    kind = s.case["kind"]
    if own:
        if kind == "rotary":
            return s.ctx.rotary(s.q, s.positions, s.rotary, s.case["head_dim"], out=s.q_out)
        if kind == "cache":
            s.ctx.cache_write(s.cache, s.k, s.v, s.slots, positions=s.positions, rotary=s.rotary, q=s.q, q_out=s.q_out,
                              q_norm=s.q_norm, k_norm=s.k_norm, epsilon=EPSILON)
            s.ctx.cache_read(s.cache, s.read_slots, s.k_read, s.v_read)
            return {"q": s.q_out, "k": s.k_read, "v": s.v_read}
        return s.ctx.cached_attention(s.q, s.cache, s.pages, s.lengths, s.out, query_offsets=s.offsets,
                                      prefix_pages=s.prefix_pages, prefix_length=s.prefix_length)
    if kind == "rotary":
        return _rotated(s, s.q.unflatten(1, (-1, s.case["head_dim"])).float()).flatten(1).to(s.dtype)
    if kind == "cache":
        return _written_and_read(s)
    return _attended(s)


def _rotated(s, x):
    """x [rows, heads, head_dim] in 32 bits, turned; angles in 64."""
    half = s.turns.numel()
    angle = s.positions.double()[:, None] * s.turns
    angle = (2 * math.pi) * (angle - angle.round())
    cos, sin = (s.scale * angle.cos()).float()[:, None], (s.scale * angle.sin()).float()[:, None]
    if s.case["interleaved"]:
        pairs = x[..., : 2 * half].unflatten(-1, (half, 2))
        a, b = pairs[..., 0], pairs[..., 1]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half: 2 * half]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, x[..., 2 * half:]), -1)


def _normed(x, weight):
    if weight is None:
        return x
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPSILON) * weight.float()


def _encoded(x, form):
    """x in 32 bits as bytes and one scale per row. The quotient is taken in 64 bits: values lie next to rounding borders."""
    most = x.abs().amax(-1)
    scale = torch.where(most == 0, torch.ones_like(most), most / RANGE[form])
    parts = x.double() / scale.double()[..., None]
    if form == "int8":
        return parts.round().clamp(-127, 127).to(torch.int8).view(torch.uint8), scale
    return parts.float().clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8), scale


def _decoded(values, scales, form):
    return values.view(torch.int8 if form == "int8" else torch.float8_e4m3fn).float() * scales[..., None]


def _written_and_read(s):
    form, page, shape = s.case["format"], s.case["page"], (s.case["kv_heads"], s.case["head_dim"])
    q = _rotated(s, _normed(s.q.unflatten(1, (-1, shape[1])).float(), s.q_norm))
    k = _rotated(s, _normed(s.k.unflatten(1, shape).float(), s.k_norm))
    at = (s.slots // page).long(), slice(None), (s.slots % page).long()
    s.keys[at], s.key_scales[at] = _encoded(k, form)
    s.values[at], s.value_scales[at] = _encoded(s.v.unflatten(1, shape).float(), form)
    at = (s.read_slots // page).long(), slice(None), (s.read_slots % page).long()
    return {"q": q.flatten(1).to(s.dtype), "k": _decoded(s.keys[at], s.key_scales[at], form).flatten(1).to(s.dtype),
            "v": _decoded(s.values[at], s.value_scales[at], form).flatten(1).to(s.dtype)}


def _attended(s):
    form, heads, kv_heads, head_dim = (s.case[x] for x in ("format", "heads", "kv_heads", "head_dim"))
    group, batch, rows = heads // kv_heads, s.pages.shape[0], s.q.shape[0]
    pages, device = s.pages.long(), s.q.device
    # [batch, kv_heads, positions, head_dim]
    keys = _decoded(s.keys[pages], s.key_scales[pages], form).transpose(1, 2).flatten(2, 3)
    values = _decoded(s.values[pages], s.value_scales[pages], form).transpose(1, 2).flatten(2, 3)
    offsets = s.offsets.long() if s.offsets is not None else torch.arange(batch + 1, device=device)
    first, count = offsets[:-1], offsets[1:] - offsets[:-1]
    token = torch.arange(s.tokens, device=device)
    q = s.q[(first[:, None] + token).clamp(max=rows - 1)].float()
    q = q.view(batch, s.tokens, kv_heads, group, head_dim).permute(0, 2, 3, 1, 4).flatten(2, 3)  # rows of a head: group, token
    scores = torch.matmul(q, keys.transpose(-1, -2)) * head_dim**-0.5
    last = s.lengths[:, None] - count[:, None] + token  # the last position that a query sees
    hidden = torch.arange(keys.shape[2], device=device) > last[..., None]
    scores.masked_fill_(hidden[:, None].repeat(1, 1, group, 1), -math.inf)
    most = scores.amax(-1, keepdim=True)
    if s.prefix_pages is not None:
        pages = s.prefix_pages.long()
        shared_keys = _decoded(s.keys[pages], s.key_scales[pages], form).transpose(0, 1).flatten(1, 2)
        shared_values = _decoded(s.values[pages], s.value_scales[pages], form).transpose(0, 1).flatten(1, 2)
        shared = torch.einsum("bhqd,hpd->bhqp", q, shared_keys) * head_dim**-0.5
        shared.masked_fill_(torch.arange(shared.shape[-1], device=device) >= s.prefix_length, -math.inf)
        most = torch.maximum(most, shared.amax(-1, keepdim=True))
    most = torch.where(most == -math.inf, torch.zeros_like(most), most)
    weights = torch.exp(scores - most)
    total, out = weights.sum(-1, keepdim=True), torch.matmul(weights, values)
    if s.prefix_pages is not None:
        weights = torch.exp(shared - most)
        total, out = total + weights.sum(-1, keepdim=True), out + torch.einsum("bhqp,hpd->bhqd", weights, shared_values)
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    out = out.unflatten(2, (group, s.tokens)).permute(0, 3, 1, 2, 4).flatten(2)  # [batch, tokens, heads * head_dim]
    row = torch.arange(rows, device=device)
    sequence = torch.searchsorted(offsets[1:], row, right=True)
    return out[sequence, row - first[sequence]].to(s.dtype)


# ------------------------------------------------------------------------------------------------------------------- work
def work(case):
    heads, head_dim = case["heads"], case["head_dim"]
    if case["kind"] == "rotary":
        elements = case["rows"] * heads * head_dim
        return {"bytes": 2 * 2 * elements + 4 * case["rows"] + 4 * case["dims"], "flops": 3 * case["rows"] * heads * case["dims"]}
    width, row = case["kv_heads"] * head_dim, case["kv_heads"] * (head_dim + 4)
    if case["kind"] == "cache":
        written = case["rows"] * (2 * 2 * heads * head_dim + 2 * 2 * width + 2 * row + 8)
        return {"bytes": written + case["read"] * (2 * row + 2 * 2 * width + 4),
                "flops": case["rows"] * (6 * heads * head_dim + 10 * width) + 2 * case["read"] * width}
    some = _lengths(case)
    seen = sum(max(0, length - n + i + 1) for length, n in some for i in range(n)) + sum(n for _, n in some) * case["prefix"]
    cached = sum(length for length, n in some if n) + case["prefix"]
    return {"bytes": cached * 2 * row + sum(n for _, n in some) * 2 * 2 * heads * head_dim, "flops": 4 * head_dim * heads * seen}


# ------------------------------------------------------------------------------------------------------------------ exact
def exact(case, seed):
    """From the definitions, in 64 bits, head by head and sequence by sequence."""
    s, kind = prepare(case, seed), case["kind"]
    if kind in ("rotary", "cache"):
        def turned(x, weight=None):
            x = x.double().reshape(x.shape[0], -1, case["head_dim"])
            if weight is not None:
                x = x / (x.pow(2).mean(2, True) + EPSILON).sqrt() * weight.double()
            y, half = x.clone(), s.turns.numel()
            angle = 2 * math.pi * torch.remainder(s.positions.double().outer(s.turns), 1.0)
            phase = torch.polar(torch.full_like(angle, s.scale), angle)
            for i in range(half):
                a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half)
                pair = torch.complex(x[:, :, a], x[:, :, b]) * phase[:, i, None]
                y[:, :, a], y[:, :, b] = pair.real, pair.imag
            return y

        if kind == "rotary":
            return turned(s.q).flatten(1)

        def stored(x):
            scale = x.abs().amax(2, True) / RANGE[case["format"]]
            scale = torch.where(scale == 0, 1.0, scale)
            if case["format"] == "int8":
                return (x / scale).round() * scale
            # e4m3: three bits behind the leading one down to 2^-6, steps of 2^-9 below
            step = torch.exp2(torch.floor(torch.log2((x / scale).abs().clamp(min=2.0**-6))) - 3)
            return (x / scale / step).round() * step * scale

        def held(values, scales):
            values = values.view(torch.int8 if case["format"] == "int8" else torch.float8_e4m3fn)
            rows = (values.double() * scales.double()[..., None]).transpose(1, 2).flatten(0, 1)
            return rows[s.read_slots.long()]

        keys, values, new = held(s.keys, s.key_scales), held(s.values, s.value_scales), case["read"] - case["rows"]
        keys[new:] = stored(turned(s.k, s.k_norm))
        values[new:] = stored(s.v.double().reshape(case["rows"], -1, case["head_dim"]))
        return {"q": turned(s.q, s.q_norm).flatten(1), "k": keys.flatten(1), "v": values.flatten(1)}

    kv_heads, group, page = case["kv_heads"], case["heads"] // case["kv_heads"], case["page"]
    kind_of = torch.int8 if case["format"] == "int8" else torch.float8_e4m3fn

    def rows_of(values, scales, pages, length):
        pages = pages[: -(-length // page)].long()
        x = values[pages].view(kind_of).double() * scales[pages].double()[..., None]
        return x.transpose(0, 1).reshape(kv_heads, -1, case["head_dim"])[:, :length]

    out, row = torch.zeros(s.q.shape, dtype=torch.float64, device="cuda"), 0
    shared = [rows_of(x, y, s.prefix_pages, case["prefix"]) for x, y in ((s.keys, s.key_scales), (s.values, s.value_scales))] \
        if case["prefix"] else None
    for b, (length, n) in enumerate(_lengths(case)):
        if not n:
            continue
        k = rows_of(s.keys, s.key_scales, s.pages[b], length)
        v = rows_of(s.values, s.value_scales, s.pages[b], length)
        seen = torch.arange(length, device="cuda")[None] <= torch.arange(length - n, length, device="cuda")[:, None]
        if shared:
            k, v = torch.cat((shared[0], k), 1), torch.cat((shared[1], v), 1)
            seen = torch.cat((seen.new_ones(n, case["prefix"]), seen), 1)
        if k.shape[1]:
            q = s.q[row: row + n].double().reshape(n, kv_heads, group, -1)
            for h in range(kv_heads):
                score = (q[:, h] @ k[h].T) / math.sqrt(case["head_dim"])  # [n, group, positions]
                score = score.masked_fill(~seen[:, None], -math.inf)
                got = torch.softmax(score, -1) @ v[h]
                got = torch.where(seen.any(1)[:, None, None], got, torch.zeros_like(got))
                out[row: row + n].view(n, kv_heads, group, -1)[:, h] = got
        row += n
    return out
