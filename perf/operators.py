"""The operators of a decoder layer around its one-bit projections, as timed cases.

A case is a plain dict. "kind" names the operator and its entry point in this package:

    attention  cache_attention: softmax(scale q k^T) v over a cache of 8-bit codes in pages of `block` tokens, with a scale
               for each page and key/value head; causal, the last `new` tokens of each sequence are the queries
    append     cache_append: the new tokens' keys rotated, keys and values quantised into the cache's pages, queries rotated
    rotary     rotary: rotary positions on (tokens, heads, head_dim), half and interleaved pairs, on a part of the head too
    norm       block_norm: h = residual_scale residual + block_scale gate post(x), y = norm(h) weight

Sizes: hidden sizes 512, 4096 and 8192, sixteen sequences, 500, 512 and 2048 tokens, heads of 64 and positions up to 1024
are this package's own; heads of 128, grouped by four, and caches of 4096 to 131072 tokens are generic.

Sequences of a batch have lengths between `shortest` and `longest` and between `new_least` and `new` new tokens each, by the
case's `mix` alone. Pages are handed out in a random order; page 0 belongs to no sequence.
"""
import math
import random

import torch

own = False

DEVICE = "cuda"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
MOST_CODE = {"e4m3": 448.0, "int8": 127.0}


def _attention(name, heads, kv_heads, dim, sequences, shortest, longest, new, dtype, code, block, new_least=None, mix=1):
    return dict(name=name, kind="attention", heads=heads, kv_heads=kv_heads, dim=dim, sequences=sequences, shortest=shortest,
                longest=longest, new=new, new_least=new if new_least is None else new_least, dtype=dtype, code=code, block=block, mix=mix)


def listed():
    return [
        # one sequence of a small model near the end of its positions, one token: latency and launches decide
        _attention("attend_1_token_small", 8, 4, 64, 1, 1000, 1000, 1, "fp16", "e4m3", 64),
        # sixteen sequences of different lengths decode together
        _attention("attend_16_sequences", 32, 8, 128, 16, 500, 4096, 1, "bf16", "e4m3", 64),
        # one token behind a very long document
        _attention("attend_long_int8", 32, 8, 128, 1, 131072, 131072, 1, "fp16", "int8", 128),
        # a batch of short prompts of no particular lengths, small pages
        _attention("attend_prompts_ragged", 8, 4, 64, 5, 37, 512, 512, "fp16", "e4m3", 16, new_least=37, mix=3),
        # one whole prompt
        _attention("attend_prompt_4096", 32, 8, 128, 1, 4096, 4096, 4096, "bf16", "e4m3", 64),
        # the next 500 tokens of a document that is taken in in pieces, a key/value head for each head
        _attention("attend_chunk_500", 32, 32, 128, 1, 8000, 8000, 500, "fp16", "int8", 32),
        # the write side of sixteen decoding sequences
        dict(name="append_16_sequences", kind="append", heads=32, kv_heads=8, dim=128, sequences=16, shortest=500, longest=4096,
             new=1, new_least=1, dtype="bf16", code="e4m3", block=64, mix=1, rotary_dim=128, interleaved=False),
        # a prompt goes into the cache
        dict(name="append_prompt_2048", kind="append", heads=32, kv_heads=8, dim=128, sequences=1, shortest=2048, longest=2048,
             new=2048, new_least=2048, dtype="fp16", code="e4m3", block=64, mix=1, rotary_dim=128, interleaved=False),
        # queries of sixteen decoding sequences
        dict(name="rotary_16_tokens", kind="rotary", tokens=16, heads=32, dim=128, rotary_dim=128, interleaved=False, dtype="bf16"),
        # a long prompt, interleaved pairs on half of each head
        dict(name="rotary_prompt_4001", kind="rotary", tokens=4001, heads=32, dim=128, rotary_dim=64, interleaved=True, dtype="fp16"),
        # between two blocks of a decoder layer, sixteen tokens
        dict(name="norm_16_tokens", kind="norm", tokens=16, hidden=4096, norm="rms", post=False, gate="none", dtype="fp16",
             residual="fp16", residual_scale=1.0, block_scale=1.0),
        # a prompt, norm on both sides of the block, a gate for each channel, residuals kept in 32 bits
        dict(name="norm_prompt_2048", kind="norm", tokens=2048, hidden=8192, norm="rms", post=True, gate="channel", dtype="bf16",
             residual="fp32", residual_scale=1.0, block_scale=0.5),
    ]


def _log_uniform(rng, low, high):
    return int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))


def _most(kind):
    """The most bytes and operations of the listed cases of an operator."""
    found = [work(c) for c in listed() if c["kind"] == kind]
    return max(w["bytes"] for w in found), max(w["flops"] for w in found)


def _draw_sequences(rng, kind):
    dim = rng.choice([64, 128, 128])
    kv_heads = rng.choice([1, 2, 4, 8, 8, 16, 32])
    heads = kv_heads * rng.choice([g for g in (1, 2, 4, 4, 8) if g * kv_heads <= 64])
    case = dict(kind=kind, heads=heads, kv_heads=kv_heads, dim=dim, dtype=rng.choice(["fp16", "bf16"]),
                code=rng.choice(["e4m3", "int8"]) if kind == "attention" else "e4m3", block=rng.choice([16, 32, 64, 64, 128]), mix=rng.randrange(1 << 20))
    form = rng.choice(["decode", "decode", "few", "prompt", "chunk"])
    case["sequences"] = _log_uniform(rng, 1, 64) if form in ("decode", "few") else _log_uniform(rng, 1, 8)
    case["new"] = 1 if form == "decode" else rng.randint(2, 8) if form == "few" else _log_uniform(rng, 16, 4096)
    case["new_least"] = case["new"] if rng.random() < 0.5 else rng.randint(1, case["new"])
    case["longest"] = case["new"] if form == "prompt" else min(131072, case["new"] + _log_uniform(rng, 1, 131072))
    case["shortest"] = case["longest"] if case["sequences"] == 1 else rng.randint(1, case["longest"])
    if kind == "append":
        case["rotary_dim"] = rng.choice([dim, dim, dim // 2])
        case["interleaved"] = rng.random() < 0.3
    return case


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "attention", "append", "append", "rotary", "norm"])
    most_bytes, most_flops = _most(kind)
    while True:
        if kind in ("attention", "append"):
            case = _draw_sequences(rng, kind)
        elif kind == "rotary":
            dim = rng.choice([64, 128, 128, 256])
            case = dict(kind=kind, tokens=_log_uniform(rng, 1, 8192), heads=rng.choice([1, 4, 8, 14, 32]), dim=dim,
                        rotary_dim=rng.choice([dim, dim, dim // 2, dim // 4]), interleaved=rng.random() < 0.5,
                        dtype=rng.choice(["fp16", "bf16", "fp32"]))
        else:
            dtype = rng.choice(["fp16", "bf16", "fp32"])
            case = dict(kind=kind, tokens=_log_uniform(rng, 1, 8192), hidden=rng.choice([512, 1408, 2048, 4096, 5000, 8192, 11008]),
                        norm=rng.choice(["rms", "rms", "layer"]), post=rng.random() < 0.4, gate=rng.choice(["none", "channel", "token"]),
                        dtype=dtype, residual=rng.choice([dtype, "fp32"]), residual_scale=rng.choice([1.0, 0.7]),
                        block_scale=rng.choice([1.0, 0.22]))
        w = work(case)
        # the cache that is there beside what an append touches is made and compared too: at most 256 MiB of it
        held = 2 * sum(_sequences(case)[0]) * case["kv_heads"] * case["dim"] if kind in ("attention", "append") else 0
        if w["bytes"] <= most_bytes and w["flops"] <= most_flops and held <= (270 << 20) and _scores(case) <= 1 << 30:
            return case


def _sequences(case):
    """(lengths with the new tokens, new tokens) of each sequence."""
    rng = random.Random(case["mix"])
    new = [rng.randint(case["new_least"], case["new"]) for _ in range(case["sequences"])]
    lengths = [max(n, rng.randint(case["shortest"], case["longest"])) for n in new]
    lengths[0] = max(lengths[0], case["longest"])
    new[0] = case["new"]
    return lengths, new


def _scores(case):
    """Scores that the plain form of a case holds."""
    if case["kind"] != "attention":
        return 0
    lengths, new = _sequences(case)
    return len(new) * case["heads"] * max(new) * max(lengths)


def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _normal(shape, g, dtype="fp32", std=1.0):
    return (torch.randn(shape, generator=g, device=DEVICE, dtype=torch.float32) * std).to(DTYPES[dtype])


def _rotary_table(positions, rotary_dim, base=10000.0):
    """fp32 (positions, rotary_dim): cos of each pair's angle, then sin."""
    rates = base ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=DEVICE) / rotary_dim)
    angles = torch.arange(positions, dtype=torch.float64, device=DEVICE)[:, None] * rates
    return torch.cat([angles.cos(), angles.sin()], dim=1).float()


def _codes(shape, code, g):
    """Codes of normal values whose largest, in blocks of some thousand, comes to about the largest code."""
    values = torch.randn(shape, generator=g, device=DEVICE, dtype=torch.float32) * (MOST_CODE[code] / 4)
    values = values.clamp_(-MOST_CODE[code], MOST_CODE[code])
    return values.round_().to(torch.int8) if code == "int8" else values.to(torch.float8_e4m3fn)


def _cache(case, g):
    lengths, new = _sequences(case)
    block = case["block"]
    width = -(-max(lengths) // block)
    need = [-(-n // block) for n in lengths]
    order = (torch.randperm(sum(need), generator=g, device=DEVICE) + 1).to(torch.int32)
    pages = torch.zeros((len(lengths), width), dtype=torch.int32, device=DEVICE)
    at = 0
    for s, n in enumerate(need):
        pages[s, :n] = order[at:at + n]
        at += n
    shape = (1 + sum(need), case["kv_heads"], block, case["dim"])
    # keys and values of about unit size, blocks and heads up to 1.5 times apart
    scale = 4 / MOST_CODE[case["code"]]
    return dict(k_cache=_codes(shape, case["code"], g), v_cache=_codes(shape, case["code"], g),
                k_scale=scale * (0.8 + 0.4 * torch.rand(shape[:2], generator=g, device=DEVICE)),
                v_scale=scale * (0.8 + 0.4 * torch.rand(shape[:2], generator=g, device=DEVICE)),
                pages=pages, lengths=torch.tensor(lengths, dtype=torch.int32, device=DEVICE),
                starts=torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device=DEVICE),
                max_new=max(new), max_length=max(lengths), tokens=sum(new))


def prepare(case, seed):
    """The cache with its tables, the rotary table and the norms' weights are what a program keeps; activations come in its
    own dtype. Queries of a decoder layer come as a view of its fused projection."""
    kind, g = case["kind"], _generator(16 * seed + 1)
    state = dict(kind=kind)
    if kind in ("attention", "append"):
        state.update(_cache(case, g), code=case["code"], block=case["block"])
        heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
        qkv = _normal((state["tokens"], heads + 2 * kv_heads, dim), g, case["dtype"], 1.5)
        state["q"] = qkv[:, :heads]
        if kind == "append":
            state.update(k=qkv[:, heads:heads + kv_heads], v=qkv[:, heads + kv_heads:], interleaved=case["interleaved"],
                         table=_rotary_table(state["max_length"], case["rotary_dim"]))
        else:
            state["scale"] = 1 / math.sqrt(dim)
    elif kind == "rotary":
        state.update(x=_normal((case["tokens"], case["heads"], case["dim"]), g, case["dtype"]), interleaved=case["interleaved"],
                     positions=torch.randint(0, 8192, (case["tokens"],), generator=g, device=DEVICE),
                     table=_rotary_table(8192, case["rotary_dim"]))
    else:
        tokens, hidden, dtype = case["tokens"], case["hidden"], case["dtype"]
        weight = lambda: (1 + 0.1 * _normal((hidden,), g)).to(DTYPES[dtype])  # noqa: E731
        state.update(x=_normal((tokens, hidden), g, dtype, 2.0), residual=_normal((tokens, hidden), g, case["residual"], 3.0), weight=weight(),
                     bias=_normal((hidden,), g, dtype, 0.1) if case["norm"] == "layer" else None,
                     post_weight=weight() if case["post"] else None, norm=case["norm"], residual_scale=case["residual_scale"],
                     block_scale=case["block_scale"], eps=1e-5,
                     gate=_normal((hidden,), g, dtype) if case["gate"] == "channel" else _normal((tokens, 1), g, dtype) if case["gate"] == "token" else None)
    return state


def run(state):
    kind = state["kind"]
    if own:
        import onebitsparsemul_amd as onebit
        if kind == "attention":
            return onebit.cache_attention(state["q"], state["k_cache"], state["v_cache"], state["k_scale"], state["v_scale"], state["pages"],
                                          state["lengths"], starts=state["starts"], scale=state["scale"], max_new=state["max_new"],
                                          max_length=state["max_length"])
        if kind == "append":
            q = onebit.cache_append(state["k"], state["v"], state["k_cache"], state["v_cache"], state["k_scale"], state["v_scale"],
                                    state["pages"], state["lengths"], starts=state["starts"], q=state["q"], rotary=state["table"],
                                    interleaved=state["interleaved"], max_new=state["max_new"])
            return dict(q=q, k_cache=state["k_cache"], v_cache=state["v_cache"], k_scale=state["k_scale"], v_scale=state["v_scale"])
        if kind == "rotary":
            return onebit.rotary(state["x"], state["positions"], state["table"], interleaved=state["interleaved"])
        return onebit.block_norm(state["x"], state["residual"], state["weight"], bias=state["bias"], post_weight=state["post_weight"],
                                 gate=state["gate"], residual_scale=state["residual_scale"], block_scale=state["block_scale"], eps=state["eps"],
                                 kind=state["norm"])
    if kind == "attention":
        return _plain_attention(state)
    if kind == "append":
        return _plain_append(state)
    if kind == "rotary":
        return _plain_rotary(state["x"].float(), state["table"][state["positions"]], state["interleaved"]).to(state["x"].dtype)
    return _plain_norm(state)


def _plain_rotary(x, rows, interleaved):
    """x (..., heads, dim) in fp32, rows (..., rotary_dim): cos and sin of each pair."""
    half = rows.shape[-1] // 2
    c, s = rows[..., None, :half], rows[..., None, half:]
    head, rest = x[..., :2 * half], x[..., 2 * half:]
    if interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
        turned = torch.stack([a * c - b * s, b * c + a * s], dim=-1).flatten(-2)
    else:
        a, b = head[..., :half], head[..., half:]
        turned = torch.cat([a * c - b * s, b * c + a * s], dim=-1)
    return torch.cat([turned, rest], dim=-1)


def _bits(codes):
    return codes.view(torch.uint8)  # what indexing takes of every code type


def _plain_attention(state):
    q, pages, lengths, starts, block = state["q"], state["pages"], state["lengths"], state["starts"], state["block"]
    tokens, heads, dim = q.shape
    sequences, width = pages.shape
    kv_heads = state["k_cache"].shape[1]
    most = state["max_new"]

    def dense(cache, scale):  # (sequences, kv_heads, width * block, dim)
        values = _bits(cache)[pages].view(cache.dtype).float() * scale[pages][..., None, None]
        return values.transpose(1, 2).reshape(sequences, kv_heads, width * block, dim)

    i = torch.arange(most, device=q.device)
    new = (starts[1:] - starts[:-1])[:, None]
    rows = (starts[:-1, None] + i).clamp(max=tokens - 1)                              # (sequences, most)
    padded = q[rows].float().reshape(sequences, most, kv_heads, heads // kv_heads, dim)
    padded = padded.permute(0, 2, 3, 1, 4).reshape(sequences, kv_heads, -1, dim)      # group, then token
    scores = torch.matmul(padded, dense(state["k_cache"], state["k_scale"]).transpose(-1, -2).contiguous())
    scores = (scores * state["scale"]).view(sequences, kv_heads, heads // kv_heads, most, width * block)
    seen = torch.arange(width * block, device=q.device) <= (lengths[:, None] - new + i)[:, None, None, :, None]
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = (p / torch.where(total == 0, 1.0, total)).view(sequences, kv_heads, -1, width * block)
    o = torch.matmul(p, dense(state["v_cache"], state["v_scale"]))
    o = o.view(sequences, kv_heads, heads // kv_heads, most, dim).permute(0, 3, 1, 2, 4).reshape(sequences * most, heads, dim)
    # back to the tokens' order: token t is number t - starts[s] of its sequence s
    token = torch.arange(tokens, device=q.device)
    s = (token[:, None] >= starts[1:]).sum(1)
    return o[s * most + token - starts[s]].to(q.dtype)


def _quantise(values, scale, code):
    """values / scale, rounded to a code; 0 where the scale is 0."""
    x = torch.where(scale == 0, 0.0, values / torch.where(scale == 0, 1.0, scale))
    return x.round().to(torch.int8) if code == "int8" else x.to(torch.float8_e4m3fn)


def _plain_append(state):
    pages, lengths, starts, block, code = state["pages"], state["lengths"].long(), state["starts"].long(), state["block"], state["code"]
    tokens = state["k"].shape[0]
    new = starts[1:] - starts[:-1]
    first = lengths - new
    touched = (state["max_new"] + block - 2) // block + 1
    j = first[:, None] // block + torch.arange(touched, device=pages.device)          # (sequences, touched)
    live = (j * block < lengths[:, None]) & (new[:, None] > 0)
    page = torch.where(live, pages.gather(1, j.clamp(max=pages.shape[1] - 1)).long(), 0)  # page 0 for what is not there
    at = j[..., None] * block + torch.arange(block, device=pages.device)              # positions (sequences, touched, block)
    old = (at < first[:, None, None]) & live[..., None]
    fresh = (at >= first[:, None, None]) & (at < lengths[:, None, None]) & live[..., None]
    rows = (starts[:-1, None, None] + at - first[:, None, None]).clamp(0, tokens - 1)
    angles = state["table"][at.clamp(max=state["table"].shape[0] - 1)]

    def put(x, cache, scales, turn):
        x = x[rows].float()                                                           # (sequences, touched, block, heads, dim)
        x = _plain_rotary(x, angles, state["interleaved"]) if turn else x
        x = torch.where(fresh[..., None, None], x, 0.0).transpose(2, 3)               # (sequences, touched, heads, block, dim)
        before = torch.where(old.any(-1, keepdim=True), scales[page], 0.0)
        scale = torch.maximum(before, x.abs().amax((-1, -2)) / MOST_CODE[code])
        codes = _bits(cache)[page].view(cache.dtype)
        again = _quantise(codes.float() * before[..., None, None], scale[..., None, None], code)
        put_codes = torch.where(fresh[:, :, None, :, None], _bits(_quantise(x, scale[..., None, None], code)),
                                torch.where(old[:, :, None, :, None], _bits(again), _bits(codes)))
        _bits(cache)[page] = put_codes
        scales[page] = torch.where(live[..., None], scale, scales[page])

    put(state["k"], state["k_cache"], state["k_scale"], True)
    put(state["v"], state["v_cache"], state["v_scale"], False)
    token = torch.arange(tokens, device=pages.device)
    s = (token[:, None] >= starts[1:]).sum(1)
    q = _plain_rotary(state["q"].float(), state["table"][first[s] + token - starts[s]], state["interleaved"]).to(state["q"].dtype)
    return dict(q=q, k_cache=state["k_cache"], v_cache=state["v_cache"], k_scale=state["k_scale"], v_scale=state["v_scale"])


def _plain_norm(state):
    def norm(x, weight, bias):
        if state["norm"] == "layer":
            x = x - x.mean(-1, keepdim=True)
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + state["eps"]) * weight.float()
        return x if bias is None else x + bias.float()

    x = state["x"].float()
    if state["post_weight"] is not None:
        x = norm(x, state["post_weight"], None)
    if state["gate"] is not None:
        x = x * state["gate"].float()
    h = state["residual_scale"] * state["residual"].float() + state["block_scale"] * x
    return h.to(state["residual"].dtype), norm(h, state["weight"], state["bias"]).to(state["x"].dtype)


def work(case):
    """Bytes: every input read once and every output written once: of a cache the codes and scales of the tokens that are in it,
    of an append those of the new tokens. flops: 4 dim for each query, head and key that it sees; 3 for each value that is
    turned, 2 for one that is quantised; about 8 for each value of a norm."""
    kind, size = case["kind"], BYTES[case["dtype"]]
    if kind in ("attention", "append"):
        lengths, new = _sequences(case)
        heads, kv_heads, dim, block = case["heads"], case["kv_heads"], case["dim"], case["block"]
        tokens = sum(new)
        tables = 4 * sum(-(-n // block) for n in lengths) + 8 * len(lengths)
    if kind == "attention":
        held = sum(2 * kv_heads * (n * dim + 4 * -(-n // block)) for n in lengths)
        keys = sum(n * (length - n) + n * (n + 1) // 2 for length, n in zip(lengths, new))
        return {"bytes": held + 2 * size * tokens * heads * dim + tables, "flops": 4.0 * keys * heads * dim}
    if kind == "append":
        touched = sum(-(-length // block) - (length - n) // block for length, n in zip(lengths, new))
        moved = tokens * dim * (2 * kv_heads * (size + 1) + 2 * heads * size)
        return {"bytes": moved + 4 * tokens * case["rotary_dim"] + 16 * touched * kv_heads + 12 * len(lengths) + 4 * touched,
                "flops": tokens * (3.0 * (heads + kv_heads) * case["rotary_dim"] + 4.0 * kv_heads * dim)}
    if kind == "rotary":
        tokens, heads = case["tokens"], case["heads"]
        return {"bytes": tokens * (2 * size * heads * case["dim"] + 4 * case["rotary_dim"] + 8), "flops": 3.0 * tokens * heads * case["rotary_dim"]}
    tokens, hidden, residual = case["tokens"], case["hidden"], BYTES[case["residual"]]
    vectors = 1 + (case["norm"] == "layer") + case["post"] + (case["gate"] == "channel")
    return {"bytes": tokens * hidden * (2 * size + 2 * residual) + size * (vectors * hidden + (tokens if case["gate"] == "token" else 0)),
            "flops": (8.0 + 5.0 * case["post"]) * tokens * hidden}


def _exact_turn(x, rows, interleaved):
    """The rotation as a product of complex numbers."""
    half = rows.shape[1] // 2
    turn = torch.complex(rows[:, :half], rows[:, half:])[:, None]
    out = x.clone()
    first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    z = torch.complex(x[..., first], x[..., second]) * turn
    out[..., first], out[..., second] = z.real, z.imag
    return out


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "rotary":
        return _exact_turn(state["x"].double(), state["table"].double()[state["positions"]], case["interleaved"])
    if kind == "norm":
        axis = dict(dim=1, keepdim=True)
        centre = (lambda t: t - t.sum(**axis) / t.shape[1]) if case["norm"] == "layer" else (lambda t: t)
        unit = lambda t: centre(t) * ((centre(t) ** 2).sum(**axis) / t.shape[1] + state["eps"]) ** -0.5  # noqa: E731
        block = state["x"].double()
        if case["post"]:
            block = unit(block) * state["post_weight"].double()
        if state["gate"] is not None:
            block = block * state["gate"].double().expand_as(block)
        h = case["residual_scale"] * state["residual"].double() + case["block_scale"] * block
        y = unit(h) * state["weight"].double()
        return h, y + state["bias"].double() if state["bias"] is not None else y
    lengths, new = _sequences(case)
    if kind == "attention":
        held = 8 * 2 * case["dim"] * max(lengths)
        if held * case["kv_heads"] > 16 << 30:
            return None
        group, outputs, at = case["heads"] // case["kv_heads"], [], 0
        for s, (length, n) in enumerate(zip(lengths, new)):
            use = state["pages"][s, :-(-length // case["block"])].long()
            o = torch.empty((n, case["heads"], case["dim"]), dtype=torch.float64, device=DEVICE)
            hidden = torch.arange(length, device=DEVICE) > torch.arange(length - n, length, device=DEVICE)[:, None]
            for h in range(case["kv_heads"]):
                k, v = ((_bits(cache)[use, h].view(cache.dtype).double() * scale[use, h].double()[:, None, None]).flatten(0, 1)[:length]
                        for cache, scale in ((state["k_cache"], state["k_scale"]), (state["v_cache"], state["v_scale"])))
                for one in range(h * group, (h + 1) * group):
                    scores = torch.mm(state["q"][at:at + n, one].double(), k.T.contiguous()) * state["scale"]
                    o[:, one] = torch.mm(torch.softmax(scores.masked_fill(hidden, -math.inf), dim=1), v)
            outputs.append(o)
            at += n
        return torch.cat(outputs)
    k, v, q = (state[name].double() for name in "kvq")
    table = state["table"].double()
    pools = {name: state[name].double() for name in ("k_scale", "v_scale")}
    pools.update({name: state[name].float().double() for name in ("k_cache", "v_cache")})
    at, turned = 0, []
    for s, (length, n) in enumerate(zip(lengths, new)):
        position = torch.arange(length - n, length, device=DEVICE)
        turned.append(_exact_turn(q[at:at + n], table[position], case["interleaved"]))
        fresh = dict(k=_exact_turn(k[at:at + n], table[position], case["interleaved"]), v=v[at:at + n])
        for j in range((length - n) // case["block"], -(-length // case["block"])):
            low, high = max(length - n, j * case["block"]), min(length, (j + 1) * case["block"])
            page = int(state["pages"][s, j])
            for name in "kv":
                codes, scale = pools[name + "_cache"][page], pools[name + "_scale"][page]
                x = fresh[name][low - (length - n):high - (length - n)].transpose(0, 1)
                held = scale.clone() if low > j * case["block"] else torch.zeros_like(scale)
                scale.copy_(torch.maximum(held, x.abs().amax((1, 2)) / MOST_CODE[case["code"]]))
                codes[:, :low - j * case["block"]] *= (held / scale)[:, None, None]
                codes[:, low - j * case["block"]:high - j * case["block"]] = x / scale[:, None, None]
        at += n
    return dict(pools, q=torch.cat(turned))
