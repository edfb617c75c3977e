"""Operators for serving long contexts in few bytes, each in a plain form and through the library's entry points.

  decode   one generated token of a batch of sequences: the token's K and V rows go into the KV cache, then the query
           heads attend over what is visible.  The cache is BF16 or 8-bit (e4m3 codes, a power-of-two scale for every
           block of 16 tokens of a head), contiguous for each sequence or in pages of 256 tokens; visible is the whole
           context, or the last `window` tokens and the first `sinks`.
  prompt   a chunk of a prompt behind `past` tokens on the same caches.  The chunk's rows are stored first; attention reads
           what the cache holds.
  norm     the row step in front of a layer's projections: residual addition, root-mean-square norm, output in 8 bits with a
           power-of-two scale for each group of columns, or in the input's type.

Heads are the model's (16 query and 4 KV heads of 256 dims).  An 8-bit cache is [K, V][KV head][block of 16 tokens], a block
being 16 rows of 256 codes, the FP32 scale and 12 bytes of padding; a BF16 cache is [K, V][KV head][token][256].
"""
from __future__ import annotations

import math

import torch

own = False

HQ, HKV, D = 16, 4, 256
G = HQ // HKV
PAGE, BLOCK, BLOCK_BYTES = 256, 16, 4112
EPSILON = 1.0e-6
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
UNBOUNDED = 1 << 30


def listed():
    return [
        # one user early in a chat, FP32 activations as the reference's executor passes them: launches and latency
        {"name": "kv8_decode_777_paged_f32", "op": "decode", "batch": 1, "shortest": 777, "longest": 777, "paged": True,
         "cache": "e4m3", "window": 0, "sinks": 0, "dtype": "f32"},
        # one user behind the longest context of the benchmark
        {"name": "kv8_decode_128k", "op": "decode", "batch": 1, "shortest": 131000, "longest": 131000, "paged": False,
         "cache": "e4m3", "window": 0, "sinks": 0, "dtype": "bf16"},
        # a busy server, 64 sequences of 1 K to 32 K tokens, in half of the cache bytes
        {"name": "kv8_serving_64", "op": "decode", "batch": 64, "shortest": 1024, "longest": 32768, "paged": False,
         "cache": "e4m3", "window": 0, "sinks": 0, "dtype": "bf16"},
        # the same server with bounded attention: the last 4096 tokens and four sinks of each sequence
        {"name": "window_serving_64_paged", "op": "decode", "batch": 64, "shortest": 1024, "longest": 32768, "paged": True,
         "cache": "bf16", "window": 4096, "sinks": 4, "dtype": "bf16"},
        # a quiet server: nine sequences, some just begun, both savings at once
        {"name": "kv8_window_serving_9_paged_f32", "op": "decode", "batch": 9, "shortest": 100, "longest": 6000,
         "paged": True, "cache": "e4m3", "window": 1000, "sinks": 4, "dtype": "f32"},
        # a long prompt in one call, every token behind a window
        {"name": "window_prompt_4096", "op": "prompt", "tokens": 4096, "past": 0, "paged": False, "cache": "bf16",
         "window": 1024, "sinks": 4},
        # a chunk of a document that is fed in calls of 512 tokens
        {"name": "window_prompt_512_past_16384", "op": "prompt", "tokens": 512, "past": 16384, "paged": False,
         "cache": "bf16", "window": 4096, "sinks": 16},
        # a whole prompt of ragged length into the 8-bit cache
        {"name": "kv8_prompt_2709", "op": "prompt", "tokens": 2709, "past": 0, "paged": False, "cache": "e4m3",
         "window": 0, "sinks": 0},
        # the next turn of a chat on the page pool: a short question behind a longer past
        {"name": "kv8_prompt_201_past_1500_paged", "op": "prompt", "tokens": 201, "past": 1500, "paged": True,
         "cache": "e4m3", "window": 0, "sinks": 0},
        # the row of one generated token
        {"name": "norm_token", "op": "norm", "rows": 1, "columns": 4096, "dtype": "bf16", "output": "e4m3", "group": 0},
        # the rows of a long prompt, scales for blocks of 128 columns as 8-bit products take them
        {"name": "norm_4096", "op": "norm", "rows": 4096, "columns": 4096, "dtype": "bf16", "output": "e4m3",
         "group": 128},
        # a ragged chunk of FP32 rows that stay FP32
        {"name": "norm_2709_f32", "op": "norm", "rows": 2709, "columns": 4096, "dtype": "f32", "output": "f32", "group": 0},
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["decode", "decode", "decode", "prompt", "prompt", "norm"])
    cache = rng.choice(["bf16", "e4m3", "e4m3"])
    window = _log_uniform(rng, 1, 8000) if cache == "bf16" or rng.random() < 0.4 else 0
    sinks = rng.choice([0, rng.randint(1, 300)]) if window else 0
    if op == "decode":
        batch = _log_uniform(rng, 1, 64)
        longest = _log_uniform(rng, 16, min(32768, 900000 // batch))
        return {"op": op, "batch": batch, "shortest": _log_uniform(rng, 1, longest), "longest": longest,
                "paged": rng.random() < 0.5, "cache": cache, "window": window, "sinks": sinks,
                "dtype": rng.choice(["bf16", "f32"])}
    if op == "prompt":
        return {"op": op, "tokens": _log_uniform(rng, 1, 3000), "past": rng.choice([0, _log_uniform(rng, 1, 6000)]),
                "paged": rng.random() < 0.5, "cache": cache, "window": window, "sinks": sinks}
    dtype = rng.choice(["bf16", "f32", "f16"])
    columns = 128 * _log_uniform(rng, 2, 64)
    return {"op": op, "rows": _log_uniform(rng, 1, 4096 * 4096 // columns), "columns": columns, "dtype": dtype,
            "output": rng.choice(["e4m3", "e4m3", dtype]), "group": rng.choice([0, 32, 128])}


def lengths_of(case):
    """Contexts of a batch, the new token included: spread evenly over the range, in a shuffled order."""
    n, low, high = case["batch"], case["shortest"], case["longest"]
    values = [low + (high - low) * (2 * i + 1) // (2 * n) for i in range(n)] if n > 1 else [high]
    return [values[i] for i in sorted(range(n), key=lambda i: (i * 37) % 101)]


def work(case):
    if case["op"] == "norm":
        elements = case["rows"] * case["columns"]
        size = 4 if case["dtype"] == "f32" else 2
        scales = -(-case["columns"] // case["group"]) if case["group"] else 1
        out = elements + 4 * case["rows"] * scales if case["output"] == "e4m3" else elements * size
        return {"bytes": 3 * elements * size + out + case["columns"] * 4, "flops": 6 * elements}
    row = 2 * HKV * (BLOCK_BYTES / BLOCK if case["cache"] == "e4m3" else 2 * D)  # one token of the cache
    window, sinks = case["window"] or UNBOUNDED, case["sinks"]
    if case["op"] == "decode":
        seen = sum(min(n, window) + min(sinks, max(n - window, 0)) for n in lengths_of(case))
        size = 4 if case["dtype"] == "f32" else 2
        return {"bytes": seen * row + case["batch"] * (3 * HQ + 2 * HKV) * D * size, "flops": 4 * HQ * D * seen}
    tokens, past = case["tokens"], case["past"]
    pairs = sum(min(n, window) + min(sinks, max(n - window, 0)) for n in range(past + 1, past + tokens + 1))
    low = max(0, past + 1 - window)
    seen = past - low + min(sinks, low)
    return {"bytes": (seen + tokens) * row + tokens * (3 * HQ + 2 * HKV) * D * 2, "flops": 4 * HQ * D * pairs}


# ---- the scale rule --------------------------------------------------------------------------------------------------
def scale_of(amax):
    """The power of two 2^e, e in [-100, 119] and least with amax <= 448 * 2^e (448 = 1.75 * 2^8 is the largest code)."""
    mantissa, exponent = torch.frexp(amax)
    e = (exponent - 9 + (mantissa > 0.875).int()).clamp(-100, 119)
    e = torch.where(amax > 0, e, torch.full_like(e, -100))
    return ((e + 127) << 23).view(torch.float32)


def amax_of(x, dims):
    return torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax(dims)


def codes_of(x, scale):
    return (x / scale).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)


# ---- inputs ----------------------------------------------------------------------------------------------------------
def quantised_blocks(rows):
    """[..., blocks, 16, 256] FP32 -> [..., blocks, 4112] bytes."""
    scale = scale_of(amax_of(rows, (-1, -2)))
    out = torch.zeros(*rows.shape[:-2], BLOCK_BYTES, device=rows.device, dtype=torch.uint8)
    out[..., :BLOCK * D] = codes_of(rows, scale[..., None, None]).view(torch.uint8).flatten(-2)
    out[..., BLOCK * D:BLOCK * D + 4].view(torch.float32)[..., 0] = scale
    return out


def filled_cache(draw_rows, capacity, rows, cache):
    """One sequence's cache of `capacity` tokens (a multiple of 256) whose first `rows` are written."""
    x = draw_rows(2, HKV, capacity, D)
    x[:, :, rows:] = 0.0
    if cache == "bf16":
        return x.to(torch.bfloat16)
    return quantised_blocks(x.view(2, HKV, capacity // BLOCK, BLOCK, D))


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device).manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, device=device, generator=gen)
    if case["op"] == "norm":
        dtype = DTYPES[case["dtype"]]
        rows, columns = case["rows"], case["columns"]
        # hidden rows: a few columns are far larger than the rest, and rows differ in magnitude
        spread = torch.exp(0.5 * normal(columns)) * torch.where(normal(columns) > 3.0, 30.0, 1.0)
        magnitude = torch.exp(normal(rows, 1))
        s = {"case": case, "x": (normal(rows, columns) * spread).to(dtype),
             "residual": (normal(rows, columns) * spread * magnitude).to(dtype), "weight": 1.0 + 0.2 * normal(columns)}
        groups = -(-columns // case["group"]) if case["group"] else 1
        s["output"] = torch.empty(rows, columns, device=device,
                                  dtype=torch.float8_e4m3fn if case["output"] == "e4m3" else dtype)
        s["scales"] = torch.empty(rows, groups, device=device)
        s["residual_out"] = torch.empty(rows, columns, device=device, dtype=dtype)
        return s
    decode = case["op"] == "decode"
    lengths = lengths_of(case) if decode else [case["past"] + case["tokens"]]
    dtype = DTYPES[case["dtype"]] if decode else torch.bfloat16
    batch, tokens = (case["batch"], 1) if decode else (1, case["tokens"])
    blocks = -(-max(lengths) // PAGE)
    channel = torch.exp(0.4 * normal(D))  # keys differ in magnitude from dim to dim
    scaled = lambda *shape: normal(*shape) * torch.stack([channel, torch.ones_like(channel)]).view(2, 1, 1, D)
    written = [n - tokens for n in lengths]
    s = {"case": case, "batch": batch, "blocks": blocks,
         "query": normal(batch * tokens, HQ, D).to(dtype), "gate": normal(batch * tokens, HQ, D).to(dtype),
         "key": (normal(batch * tokens, HKV, D) * channel).to(dtype), "value": normal(batch * tokens, HKV, D).to(dtype),
         "positions": torch.tensor([n - 1 for n in lengths], device=device, dtype=torch.int32),
         "output": torch.empty(batch * tokens, HQ, D, device=device, dtype=dtype)}
    row_shape = (PAGE, D) if case["cache"] == "bf16" else (PAGE // BLOCK, BLOCK_BYTES)
    kind = torch.bfloat16 if case["cache"] == "bf16" else torch.uint8
    if case["paged"]:
        used = [-(-n // PAGE) for n in lengths]
        pages = sum(used) + 2
        order = torch.randperm(pages, device=device, generator=gen)
        s["cache"] = torch.zeros(pages, 2, HKV, *row_shape, device=device, dtype=kind)
        s["tables"] = torch.zeros(batch, blocks, device=device, dtype=torch.int32)
        at = 0
        for i, n in enumerate(used):
            one = filled_cache(scaled, n * PAGE, written[i], case["cache"])
            mine = order[at:at + n]
            s["cache"][mine] = one.view(2, HKV, n, *row_shape).permute(2, 0, 1, 3, 4)
            s["tables"][i, :n] = mine.int()
            at += n
        s["pages"] = pages
    else:
        s["cache"] = torch.zeros(batch, 2, HKV, blocks * row_shape[0], row_shape[1], device=device, dtype=kind)
        for i, n in enumerate(lengths):
            own_rows = -(-n // PAGE) * PAGE
            one = filled_cache(scaled, own_rows, written[i], case["cache"])
            s["cache"][i, :, :, :one.shape[2]] = one
        step = s["cache"][0].numel() * s["cache"].element_size()
        s["pointers"] = torch.tensor([s["cache"].data_ptr() + i * step for i in range(batch)], device=device)
        s["capacities"] = torch.full((batch,), blocks * PAGE, device=device, dtype=torch.int32)
    s["workspace"] = torch.empty(workspace_bytes(case, blocks), device=device, dtype=torch.uint8)
    return s


def workspace_bytes(case, blocks):
    """What a program sets aside: room for a prompt's context in BF16, or for the partial results of a decode step."""
    return blocks * PAGE * 2 * HKV * D * 2 + (1 << 16) if case["op"] == "prompt" else 8 << 20


# ---- the plain form --------------------------------------------------------------------------------------------------
def cache_rows(s, i, block):
    """Bytes or values of cache piece `block` (a token of a BF16 cache, a block of an 8-bit one) of sequence `i` (index
    tensors of one shape [...]): [..., 2, HKV, row]."""
    if s["case"]["paged"]:
        per_page = s["cache"].shape[3]
        page = s["tables"][i, block // per_page].long()
        return s["cache"][page, :, :, block % per_page]
    return s["cache"][i, :, :, block]


def set_cache_rows(s, i, block, rows):
    if s["case"]["paged"]:
        per_page = s["cache"].shape[3]
        s["cache"][s["tables"][i, block // per_page].long(), :, :, block % per_page] = rows
    else:
        s["cache"][i, :, :, block] = rows


def split_block(raw):
    """[..., 4112] bytes -> codes [..., 16, 256] in FP32, scale [...]."""
    codes = raw[..., :BLOCK * D].view(torch.float8_e4m3fn).float()
    return codes.unflatten(-1, (BLOCK, D)), raw[..., BLOCK * D:BLOCK * D + 4].view(torch.float32)[..., 0]


def store_rows(s, i, block, new, is_new, in_front):
    """Writes rows into 8-bit blocks.  new [..., 16, 2, HKV, 256] FP32, is_new and in_front [..., 16]: rows that are
    written, and rows that were there before and stay valid."""
    raw = cache_rows(s, i, block)
    codes, old = split_block(raw)
    new = new.movedim(-4, -2)  # [..., 2, HKV, 16, 256]
    fresh, kept = is_new[..., None, None, :, None], in_front[..., None, None, :, None]
    scale = scale_of(amax_of(torch.where(fresh, new, torch.zeros_like(new)), (-1, -2)))
    scale = torch.where(in_front.any(-1)[..., None, None], torch.maximum(scale, old), scale)
    wide = scale[..., None, None]
    moved = codes_of(codes * old[..., None, None], wide)
    written = torch.where(fresh, codes_of(new, wide).view(torch.uint8),
                          torch.where(kept, moved.view(torch.uint8), raw[..., :BLOCK * D].unflatten(-1, (BLOCK, D))))
    raw = raw.clone()
    raw[..., :BLOCK * D] = written.flatten(-2)
    raw[..., BLOCK * D:BLOCK * D + 4].view(torch.float32)[..., 0] = scale
    set_cache_rows(s, i, block, raw)


def read_rows(s, i, token):
    """K and V of tokens [...] of sequences [...] in FP32: [..., 2, HKV, 256]."""
    if s["case"]["cache"] == "bf16":
        return cache_rows(s, i, token).float()
    place, row = token // BLOCK, token % BLOCK
    if s["case"]["paged"]:
        page = s["tables"][i, token // PAGE].long()
        place = place % (PAGE // BLOCK)
        whole, first = s["cache"], page
    else:
        whole, first = s["cache"], i
    codes = whole[..., :BLOCK * D].unflatten(-1, (BLOCK, D))[first, :, :, place, row].view(torch.float8_e4m3fn).float()
    return codes * whole[..., BLOCK * D:BLOCK * D + 4].view(torch.float32)[first, :, :, place]


def returned_cache(s):
    if s["case"]["cache"] == "bf16":
        return (s["cache"],)
    return s["cache"][..., :BLOCK * D].view(torch.float8_e4m3fn), s["cache"][..., BLOCK * D:BLOCK * D + 4].view(torch.float32)


def plain_decode(s):
    case, batch, device = s["case"], s["batch"], s["cache"].device
    every = torch.arange(batch, device=device)
    position = s["positions"].long()
    new = torch.stack([s["key"], s["value"]], 1).float()  # [batch, 2, HKV, 256]
    if case["cache"] == "bf16":
        set_cache_rows(s, every, position, new.to(torch.bfloat16))
    else:
        row = torch.arange(BLOCK, device=device)
        store_rows(s, every, position // BLOCK, new[:, None].expand(-1, BLOCK, -1, -1, -1),
                   row == (position % BLOCK)[:, None], row < (position % BLOCK)[:, None])
    window, sinks = case["window"] or UNBOUNDED, case["sinks"]
    low = (position + 1 - window).clamp(min=0)[:, None]
    first = low.clamp(max=sinks)
    at = torch.arange(min(window + sinks, case["longest"]), device=device)
    token = torch.where(at < first, at, low + at - first)
    seen = token <= position[:, None]
    rows = read_rows(s, every[:, None], torch.where(seen, token, torch.zeros_like(token)))  # [batch, n, 2, HKV, 256]
    query = s["query"].float().view(batch, HKV, G, D)
    scores = torch.matmul(query, rows[:, :, 0].permute(0, 2, 3, 1)) / math.sqrt(D)
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    out = torch.matmul(weights, rows[:, :, 1].permute(0, 2, 1, 3)) / weights.sum(-1, keepdim=True)
    out = out.reshape(batch, HQ, D) / (1.0 + torch.exp(-s["gate"].float()))
    return (out.to(s["output"].dtype), *returned_cache(s))


def plain_prompt(s):
    case, device = s["case"], s["cache"].device
    tokens, past = case["tokens"], case["past"]
    context = past + tokens
    new = torch.stack([s["key"], s["value"]], 1).float()  # [tokens, 2, HKV, 256]
    if case["cache"] == "bf16":
        place = torch.arange(past, context, device=device)
        set_cache_rows(s, torch.zeros_like(place), place, new.to(torch.bfloat16))
    else:
        block = torch.arange(past // BLOCK, (context - 1) // BLOCK + 1, device=device)
        token = block[:, None] * BLOCK + torch.arange(BLOCK, device=device)
        is_new = (token >= past) & (token < context)
        store_rows(s, torch.zeros_like(block), block, new[(token - past).clamp(0, tokens - 1)], is_new, token < past)
    window, sinks = case["window"] or UNBOUNDED, case["sinks"]
    low = max(0, past + 1 - window)
    key = torch.cat([torch.arange(min(sinks, low), device=device), torch.arange(low, context, device=device)])
    rows = read_rows(s, torch.zeros_like(key), key)  # [n, 2, HKV, 256]
    position = torch.arange(past, context, device=device)[:, None]
    seen = (key <= position) & ((key > position - window) | (key < sinks))
    query = s["query"].float().view(tokens, HKV, G, D).permute(1, 2, 0, 3)
    scores = torch.matmul(query, rows[:, 0].permute(1, 2, 0)[:, None]) / math.sqrt(D)
    scores = scores.masked_fill(~seen, -math.inf)
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    out = torch.matmul(weights, rows[:, 1].permute(1, 0, 2)[:, None]) / weights.sum(-1, keepdim=True)
    out = out.permute(2, 0, 1, 3).reshape(tokens, HQ, D) / (1.0 + torch.exp(-s["gate"].float()))
    return (out.to(s["output"].dtype), *returned_cache(s))


def plain_norm(s):
    case = s["case"]
    h = s["x"].float() + s["residual"].float()
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPSILON) * s["weight"]
    if case["output"] != "e4m3":
        return y.to(s["x"].dtype), h.to(s["x"].dtype)
    grouped = y.unflatten(-1, (s["scales"].shape[1], -1))
    scale = scale_of(amax_of(grouped, -1))
    return codes_of(grouped, scale[..., None]).flatten(-2), scale, h.to(s["x"].dtype)


# ---- the library's entry points --------------------------------------------------------------------------------------
_stream = None


def stream():
    """The stream of this program; the library does not take the default one."""
    global _stream
    if _stream is None:
        _stream = torch.cuda.Stream()
    return _stream


def own_run(s):
    from raftinfer_b200 import kernels as K

    case = s["case"]
    dtypes = {"f32": K.DTYPE_F32, "bf16": K.DTYPE_BF16, "f16": K.DTYPE_F16, "e4m3": K.DTYPE_E4M3}
    if case["op"] == "norm":
        K.residual_rms_norm(s["x"], s["residual"], s["weight"], s["output"],
                            s["scales"] if case["output"] == "e4m3" else None, s["residual_out"], case["rows"],
                            case["columns"], case["group"] if case["output"] == "e4m3" else 0, EPSILON,
                            dtypes[case["dtype"]], K.DTYPE_F32, dtypes[case["output"]], stream())
        return (s["output"], s["scales"], s["residual_out"]) if case["output"] == "e4m3" else (s["output"], s["residual_out"])
    cache_dtype = K.KV_BF16 if case["cache"] == "bf16" else K.KV_E4M3
    size = s["workspace"].numel()
    if case["op"] == "decode":
        activations = dtypes[case["dtype"]]
        if case["paged"]:
            K.kv_paged_decode(s["query"], s["key"], s["value"], s["gate"], s["output"], s["cache"], s["pages"], s["tables"],
                              s["blocks"], s["positions"], s["batch"], HQ, HKV, case["window"], case["sinks"], activations,
                              cache_dtype, s["workspace"], size, stream())
        else:
            K.kv_batched_decode(s["query"], s["key"], s["value"], s["gate"], s["output"], s["pointers"], s["capacities"],
                                s["positions"], s["batch"], HQ, HKV, case["window"], case["sinks"], activations,
                                cache_dtype, s["workspace"], size, stream())
        return (s["output"], *returned_cache(s))
    shape = K.Qwen35AttentionShape(case["tokens"], HQ, HKV, D, s["blocks"] * PAGE, case["past"])
    if case["paged"]:
        K.kv_paged_prefill(s["query"], s["key"], s["value"], s["gate"], s["output"], s["cache"], s["pages"], s["tables"],
                           s["blocks"], s["workspace"], size, shape, case["window"], case["sinks"], K.DTYPE_BF16,
                           cache_dtype, stream())
    else:
        K.kv_attention_prefill(s["query"], s["key"], s["value"], s["gate"], s["output"], s["cache"],
                               s["cache"].numel() * s["cache"].element_size(), s["workspace"], size, shape, case["window"],
                               case["sinks"], K.DTYPE_BF16, cache_dtype, stream())
    return (s["output"], *returned_cache(s))


def run(state):
    if own:
        return own_run(state)
    return {"decode": plain_decode, "prompt": plain_prompt, "norm": plain_norm}[state["case"]["op"]](state)


# ---- from the definition, in 64 bits -----------------------------------------------------------------------------------
def exact_scale(largest):
    """Least power of two s with largest <= 448 s, between 2^-100 and 2^119, in 64 bits."""
    e = torch.ceil(torch.log2(largest.clamp(min=2.0 ** -149) / 448.0))
    power = lambda n: ((n.long() + 1023) << 52).view(torch.float64)
    e = torch.where(largest > 448.0 * power(e), e + 1, e)
    e = torch.where(largest <= 448.0 * power(e - 1), e - 1, e)
    return power(e.clamp(-100, 119))


def exact_code(v):
    """The e4m3 value nearest to v (|v| <= 448), ties to the even one: three bits behind the leading one, which is at 2^-6
    or higher."""
    leading = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6)))
    leading = torch.where(v.abs() < torch.exp2(leading.round()), leading - 1, leading).clamp(min=-6)
    unit = torch.exp2(leading - 3.0)
    return torch.round(v / unit) * unit


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        h = s["x"].double() + s["residual"].double()
        y = h / torch.sqrt(h.square().mean(-1, keepdim=True) + EPSILON) * s["weight"].double()
        if case["output"] != "e4m3":
            return y, h
        parts = y.reshape(case["rows"], s["scales"].shape[1], -1)
        scale = exact_scale(parts.abs().amax(-1))
        return exact_code(parts / scale[..., None]).reshape(y.shape), scale, h
    decode = case["op"] == "decode"
    lengths = lengths_of(case) if decode else [case["past"] + case["tokens"]]
    tokens = 1 if decode else case["tokens"]
    window, sinks = case["window"] or UNBOUNDED, case["sinks"]
    outs = []
    cache = s["cache"]
    for i, n in enumerate(lengths):
        past = n - tokens
        mine = slice(i * tokens, (i + 1) * tokens)
        pieces = cache.shape[3]
        pages = s["tables"][i, :-(-n // PAGE)].long() if case["paged"] else None
        held = cache[pages].permute(1, 2, 0, 3, 4).flatten(2, 3) if case["paged"] else cache[i]
        new = torch.stack([s["key"][mine], s["value"][mine]]).double().permute(0, 2, 1, 3)  # [2, HKV, tokens, 256]
        if case["cache"] == "bf16":
            held = held.clone()
            held[:, :, past:n] = new.to(torch.bfloat16)
            back, values = held, held
        else:
            whole = held.clone()
            first, last = past // BLOCK, (n - 1) // BLOCK + 1
            codes = whole[..., :BLOCK * D].view(torch.float8_e4m3fn).unflatten(-1, (BLOCK, D))
            scales = whole[..., BLOCK * D:BLOCK * D + 4].view(torch.float32)
            for b in range(first, last):
                lo, hi = max(past, b * BLOCK), min(n, (b + 1) * BLOCK)
                part = new[:, :, lo - past:hi - past]
                scale = exact_scale(part.abs().amax((-1, -2)))
                kept = lo - b * BLOCK
                if kept:
                    before = scales[:, :, b, 0].double()
                    scale = torch.maximum(scale, before)
                    moved = codes[:, :, b, :kept].double() * (before / scale)[..., None, None]
                    codes[:, :, b, :kept] = exact_code(moved).to(torch.float8_e4m3fn)
                codes[:, :, b, kept:hi - b * BLOCK] = exact_code(part / scale[..., None, None]).to(torch.float8_e4m3fn)
                scales[:, :, b, 0] = scale.float()
            back = whole
            values = None
        low = max(0, past + 1 - window)
        keys = list(range(min(sinks, low))) + list(range(low, n))
        keys = torch.tensor(keys, device=cache.device)
        if values is not None:
            rows = values[:, :, keys].double()
        else:
            rows = codes[:, :, keys // BLOCK, keys % BLOCK].double() * scales[:, :, keys // BLOCK].double()
        for first_row in range(0, tokens, 256):  # queries in pieces: scores are 64 bits wide
            at = torch.arange(past + first_row, min(past + first_row + 256, n), device=cache.device)[:, None]
            picked = slice(mine.start + first_row, mine.start + first_row + len(at))
            visible = (keys <= at) & ((at - keys < window) | (keys < sinks))
            query = s["query"][picked].double()
            for head in range(HQ):
                k, v = rows[0, head // G], rows[1, head // G]
                logits = (query[:, head] @ k.T) / 16.0
                weights = torch.softmax(logits.masked_fill(~visible, -math.inf), -1)
                outs.append(weights @ v * torch.sigmoid(s["gate"][picked, head].double()))
        if case["paged"]:
            cache[pages] = back.unflatten(2, (len(pages), pieces)).permute(2, 0, 1, 3, 4)
        else:
            cache[i] = back
    out = torch.cat([torch.stack(outs[i:i + HQ], 1) for i in range(0, len(outs), HQ)])
    return (out, *returned_cache(s))
