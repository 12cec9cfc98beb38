"""From a decoder's last layer to its next tokens, as timed cases.

A case is a plain dict. "kind" names the operator and its entry point in this package:

    norm     block_norm_codes: h = residual + block_scale post(x), y = norm(h) weight, y as e4m3 codes with a scale for each 128 values of a row
    rows     quantize_rows: values as such codes and scales
    product  block_linear: y = x W^T (+ bias) of e4m3 codes, x with a scale for each 128 values of a row, W with one for each 128 x 128 values
    sample   sample: temperature, top-k, top-p and min-p, and the token at which the running mass passes a given random number

Sizes: hidden sizes 512, 4096 and 8192, 1408 and 11008 columns, a vocabulary of 4096, 16 sequences and 2048 tokens are this package's own; 5000 columns,
vocabularies of 32000 and 131072 and other counts of tokens are generic.

Rows of codes are padded with zeros to a multiple of 128.
"""
import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}
GROUP = 128
MOST_CODE = 448.0


def _product(name, tokens, columns, rows, out, bias=False):
    return dict(name=name, kind="product", tokens=tokens, columns=columns, rows=rows, out=out, bias=bias)


def _sample(name, rows, vocabulary, dtype, temperature, top_k, top_p, min_p, each, masked=0.0):
    """each: a parameter for each row (temperature and top_p up to the given one, top_k from 1 to it), else numbers for all; masked: share of tokens at -inf"""
    return dict(name=name, kind="sample", rows=rows, vocabulary=vocabulary, dtype=dtype, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p,
                each=each, masked=masked)


def listed():
    return [
        # the last norm of a step of sixteen sequences, in front of the logits
        dict(name="norm_codes_16", kind="norm", tokens=16, hidden=4096, dtype="fp16", residual="fp16", norm="rms", post=False, block_scale=1.0),
        # a prompt's, with a norm behind the block too and residuals kept in 32 bits
        dict(name="norm_codes_2048", kind="norm", tokens=2048, hidden=8192, dtype="bf16", residual="fp32", norm="rms", post=True, block_scale=0.5),
        # what an activation hands to the down projection, sixteen tokens
        dict(name="rows_16", kind="rows", tokens=16, columns=11008, dtype="fp16"),
        # a prompt's, columns that are no multiple of 128
        dict(name="rows_4001", kind="rows", tokens=4001, columns=5000, dtype="bf16"),
        # logits of one token of a small model: latency decides
        _product("logits_1_small", 1, 512, 4096, "fp32"),
        # logits of sixteen sequences over a large vocabulary: the weight's bytes decide
        _product("logits_16", 16, 4096, 131072, "bf16"),
        # a ragged batch through a projection with a bias, odd numbers of rows
        _product("project_333_ragged", 333, 1408, 4099, "fp16", bias=True),
        # a prompt through a projection: the matrix units decide
        _product("project_2048", 2048, 4096, 11008, "bf16"),
        # one sequence, top-p alone: all the vocabulary's mass counts
        _sample("sample_1_top_p", 1, 32000, "fp32", 0.8, 0, 0.95, 0.0, False),
        # sixteen sequences with parameters of their own
        _sample("sample_16_each", 16, 131072, "bf16", 1.2, 64, 0.95, 0.02, True),
        # many sequences, min-p, a grammar's mask on a third of the tokens
        _sample("sample_64_min_p", 64, 4096, "fp16", 1.0, 0, 1.0, 0.05, False, masked=0.35),
        # the largest batch, top-k and top-p
        _sample("sample_256", 256, 131072, "fp32", 1.0, 50, 0.9, 0.0, False),
    ]


def _log_uniform(rng, low, high):
    return int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))


def _most(kind):
    """The most bytes and operations of the listed cases of an operator."""
    found = [work(c) for c in listed() if c["kind"] == kind]
    return max(w["bytes"] for w in found), max(w["flops"] for w in found)


def draw(rng):
    kind = rng.choice(["product", "product", "product", "product", "sample", "sample", "sample", "norm", "rows"])
    most_bytes, most_flops = _most(kind)
    while True:
        if kind == "norm":
            dtype = rng.choice(["fp16", "bf16", "fp32"])
            case = dict(kind=kind, tokens=_log_uniform(rng, 1, 8192), hidden=rng.choice([512, 1408, 2048, 4096, 5000, 8192, 11008]), dtype=dtype,
                        residual=rng.choice([dtype, "fp32"]), norm=rng.choice(["rms", "rms", "layer"]), post=rng.random() < 0.4,
                        block_scale=rng.choice([1.0, 0.22]))
        elif kind == "rows":
            case = dict(kind=kind, tokens=_log_uniform(rng, 1, 8192), columns=rng.choice([512, 1408, 2048, 4096, 5000, 5001, 8192, 11008]),
                        dtype=rng.choice(["fp16", "bf16", "fp32"]))
        elif kind == "product":
            case = dict(kind=kind, tokens=_log_uniform(rng, 1, 64) if rng.random() < 0.5 else _log_uniform(rng, 17, 4096),
                        columns=rng.choice([512, 1408, 2048, 4096, 5000, 8192, 11008]), rows=_log_uniform(rng, 64, 131072),
                        out=rng.choice(["fp16", "bf16", "fp32"]), bias=rng.random() < 0.3)
        else:
            case = dict(kind=kind, rows=_log_uniform(rng, 1, 256), vocabulary=_log_uniform(rng, 1000, 131072), dtype=rng.choice(["fp16", "bf16", "fp32"]),
                        temperature=rng.choice([0.0, 0.5, 0.8, 1.0, 1.5]), top_k=rng.choice([0, 0, 1, 20, 50, 300, 1000]),
                        top_p=rng.choice([1.0, 1.0, 0.5, 0.9, 0.99]), min_p=rng.choice([0.0, 0.0, 0.01, 0.1]), each=rng.random() < 0.5,
                        masked=rng.choice([0.0, 0.0, 0.5, 0.999]))
        w = work(case)
        if w["bytes"] <= most_bytes and w["flops"] <= most_flops:
            return case


def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _normal(shape, g, dtype="fp32", std=1.0):
    return (torch.randn(shape, generator=g, device=DEVICE, dtype=torch.float32) * std).to(DTYPES[dtype])


def _padded(columns):
    return -(-columns // GROUP) * GROUP


def _row_codes(x):
    """(codes, scales) of rows in fp32"""
    tokens, columns = x.shape
    x = torch.nn.functional.pad(x, (0, _padded(columns) - columns)).view(tokens, -1, GROUP)
    scale = x.abs().amax(-1) / MOST_CODE
    codes = torch.where(scale[..., None] == 0, 0.0, x / torch.where(scale == 0, 1.0, scale)[..., None])
    return codes.view(tokens, -1).to(torch.float8_e4m3fn), scale


def _weight_codes(w):
    """(codes, scales) of a weight in fp32, a scale for each 128 x 128 values"""
    rows, columns = w.shape
    blocks = torch.nn.functional.pad(w, (0, _padded(columns) - columns, 0, _padded(rows) - rows)).view(-(-rows // GROUP), GROUP, -1, GROUP)
    scale = blocks.abs().amax((1, 3)) / MOST_CODE
    codes = blocks.div_(scale[:, None, :, None]).view(-1, _padded(columns))[:rows].to(torch.float8_e4m3fn)
    return codes, scale


def _logits(case, g):
    """Tokens' logits fall with the logarithm of their rank, in an order of their own for each row, some steeply, some slowly."""
    rows, vocabulary = case["rows"], case["vocabulary"]
    rank = torch.rand((rows, vocabulary), generator=g, device=DEVICE).argsort(-1).argsort(-1).float()
    slope = 1.0 + 1.5 * torch.rand((rows, 1), generator=g, device=DEVICE)
    logits = 12.0 - slope * torch.log(rank + 1.0) + 0.3 * torch.randn((rows, vocabulary), generator=g, device=DEVICE)
    if case["masked"]:
        hidden = torch.rand((rows, vocabulary), generator=g, device=DEVICE) < case["masked"]
        hidden[:, vocabulary // 2] = False  # a grammar allows something
        logits = logits.masked_fill(hidden, -math.inf)
    return logits.to(DTYPES[case["dtype"]])


def prepare(case, seed):
    """The weights, quantised once, are what a program keeps; activations and logits come from the layer in front."""
    kind, g = case["kind"], _generator(16 * seed + 3)
    if kind == "norm":
        tokens, hidden, dtype = case["tokens"], case["hidden"], case["dtype"]
        weight = lambda: (1 + 0.1 * _normal((hidden,), g)).to(DTYPES[dtype])  # noqa: E731
        return dict(kind=kind, x=_normal((tokens, hidden), g, dtype, 2.0), residual=_normal((tokens, hidden), g, case["residual"], 3.0), weight=weight(),
                    bias=_normal((hidden,), g, dtype, 0.1) if case["norm"] == "layer" else None, post_weight=weight() if case["post"] else None,
                    norm=case["norm"], block_scale=case["block_scale"], eps=1e-5)
    if kind == "rows":
        # some channels are many times the others, as activations have it
        channel = torch.exp(torch.randn(case["columns"], generator=g, device=DEVICE))
        return dict(kind=kind, x=(_normal((case["tokens"], case["columns"]), g) * channel).to(DTYPES[case["dtype"]]))
    if kind == "product":
        channel = torch.exp(0.5 * torch.randn(case["columns"], generator=g, device=DEVICE))
        codes, scales = _row_codes(_normal((case["tokens"], case["columns"]), g) * channel)
        weight_codes, weight_scales = _weight_codes(_normal((case["rows"], case["columns"]), g, std=case["columns"] ** -0.5))
        return dict(kind=kind, codes=codes, scales=scales, weight_codes=weight_codes, weight_scales=weight_scales,
                    bias=_normal((case["rows"],), g, case["out"]) if case["bias"] else None, out=DTYPES[case["out"]])
    rows = case["rows"]
    state = dict(kind=kind, logits=_logits(case, g), uniform=torch.rand(rows, generator=g, device=DEVICE), temperature=case["temperature"],
                 top_k=case["top_k"], top_p=case["top_p"], min_p=case["min_p"])
    if case["each"]:
        share = lambda: torch.rand(rows, generator=g, device=DEVICE)  # noqa: E731
        state.update(temperature=case["temperature"] * (0.5 + 0.5 * share()), top_p=case["top_p"] * (0.6 + 0.4 * share()), min_p=case["min_p"] * share(),
                     top_k=(case["top_k"] * share()).ceil().to(torch.int32))
    return state


def run(state):
    kind = state["kind"]
    if own:
        import onebitsparsemul_amd as onebit
        if kind == "norm":
            return onebit.block_norm_codes(state["x"], state["residual"], state["weight"], bias=state["bias"], post_weight=state["post_weight"],
                                           block_scale=state["block_scale"], eps=state["eps"], kind=state["norm"])
        if kind == "rows":
            return onebit.quantize_rows(state["x"])
        if kind == "product":
            return onebit.block_linear(state["codes"], state["scales"], state["weight_codes"], state["weight_scales"], bias=state["bias"],
                                       out_dtype=state["out"])
        return onebit.sample(state["logits"], state["uniform"], temperature=state["temperature"], top_k=state["top_k"], top_p=state["top_p"],
                             min_p=state["min_p"])
    if kind == "norm":
        return _plain_norm(state)
    if kind == "rows":
        return _row_codes(state["x"].float())
    if kind == "product":
        return _plain_product(state)
    return _plain_sample(state)


def _plain_norm(state):
    def norm(x, weight, bias):
        if state["norm"] == "layer":
            x = x - x.mean(-1, keepdim=True)
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + state["eps"]) * weight.float()
        return x if bias is None else x + bias.float()

    x = state["x"].float()
    if state["post_weight"] is not None:
        x = norm(x, state["post_weight"], None)
    h = state["residual"].float() + state["block_scale"] * x
    return h.to(state["residual"].dtype), *_row_codes(norm(h, state["weight"], state["bias"]))


def _plain_product(state):
    tokens, rows = state["codes"].shape[0], state["weight_codes"].shape[0]
    x = (state["codes"].float().view(tokens, -1, GROUP) * state["scales"][..., None]).view(tokens, -1)
    scales = state["weight_scales"].repeat_interleave(GROUP, 0)[:rows]
    w = state["weight_codes"].float().view(rows, -1, GROUP).mul_(scales[..., None]).view(rows, -1)
    y = torch.matmul(x, w.T)
    if state["bias"] is not None:
        y = y + state["bias"].float()
    return y.to(state["out"])


def _plain_sample(state):
    """In 64 bits: a token is whole, and which one it is turns on sums next to a border."""
    logits = state["logits"].double()
    rows, vocabulary = logits.shape

    def column(value):
        t = value if isinstance(value, torch.Tensor) else torch.full((rows,), value, dtype=torch.float32, device=logits.device)
        return t.double()[:, None]

    temperature, top_k, top_p, min_p = (column(state[name]) for name in ("temperature", "top_k", "top_p", "min_p"))
    top_k = torch.where(temperature <= 0, 1.0, torch.where(top_k <= 0, float(vocabulary), top_k))
    largest = logits.amax(-1, keepdim=True)
    w = torch.exp((logits - largest) / torch.where(temperature <= 0, 1.0, temperature))
    w = torch.where(logits == largest, 1.0, w)
    _, order = torch.sort(logits, dim=-1, descending=True, stable=True)
    place = torch.arange(vocabulary, device=logits.device)[None, :]
    sorted_w = w.gather(-1, order) * (place < top_k)
    running = sorted_w.cumsum(-1)
    keep = (place < top_k) & ((running - sorted_w < top_p * running[:, -1:]) | (top_p >= 1)) & (sorted_w >= min_p)
    w = w * torch.zeros_like(keep).scatter_(-1, order, keep | (place == 0))
    running = w.cumsum(-1)
    passed = (running <= column(state["uniform"]) * running[:, -1:]).sum(-1)
    last = torch.where(w > 0, place, 0).amax(-1)
    token = torch.minimum(passed, last)
    return torch.where(torch.isnan(logits).any(-1) | (largest[:, 0] == -math.inf), -1, token)


def work(case):
    """Bytes: every input read once and every output written once. flops: 2 for each code of the weight and token; about 8 for each value of a norm and 3 for one
    that is quantised; 1 for each logit, against the row's largest."""
    kind = case["kind"]
    if kind == "norm":
        tokens, hidden, size, residual = case["tokens"], case["hidden"], BYTES[case["dtype"]], BYTES[case["residual"]]
        vectors = 1 + (case["norm"] == "layer") + case["post"]
        return {"bytes": tokens * (hidden * (size + 2 * residual) + _padded(hidden) * (1 + 4 / GROUP)) + size * vectors * hidden,
                "flops": (11.0 + 5.0 * case["post"]) * tokens * hidden}
    if kind == "rows":
        tokens, columns = case["tokens"], case["columns"]
        return {"bytes": tokens * (columns * BYTES[case["dtype"]] + _padded(columns) * (1 + 4 / GROUP)), "flops": 3.0 * tokens * columns}
    if kind == "product":
        tokens, rows, columns = case["tokens"], case["rows"], _padded(case["columns"])
        size = BYTES[case["out"]]
        return {"bytes": tokens * columns * (1 + 4 / GROUP) + rows * columns + 4 * -(-rows // GROUP) * columns // GROUP + size * rows * (tokens + case["bias"]),
                "flops": 2.0 * tokens * rows * columns}
    rows = case["rows"]
    return {"bytes": rows * (case["vocabulary"] * BYTES[case["dtype"]] + 8 + 4 + (16 if case["each"] else 0)), "flops": 1.0 * rows * case["vocabulary"]}


def _exact_codes(y):
    """What codes and scales stand for without their rounding"""
    rows, columns = y.shape
    values = torch.zeros((rows, _padded(columns)), dtype=torch.float64, device=y.device)
    values[:, :columns] = y
    groups = values.unflatten(1, (-1, GROUP))
    scale = groups.abs().max(-1).values / MOST_CODE
    return (groups / scale.clamp(min=1e-300)[..., None]).flatten(1), scale


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "norm":
        axis = dict(dim=1, keepdim=True)
        centre = (lambda t: t - t.sum(**axis) / t.shape[1]) if case["norm"] == "layer" else (lambda t: t)
        unit = lambda t: centre(t) * ((centre(t) ** 2).sum(**axis) / t.shape[1] + state["eps"]) ** -0.5  # noqa: E731
        block = state["x"].double()
        if case["post"]:
            block = unit(block) * state["post_weight"].double()
        h = state["residual"].double() + case["block_scale"] * block
        y = unit(h) * state["weight"].double()
        return h, *_exact_codes(y + state["bias"].double() if state["bias"] is not None else y)
    if kind == "rows":
        return _exact_codes(state["x"].double())
    if kind == "product":
        total = torch.zeros((case["tokens"], case["rows"]), dtype=torch.float64, device=DEVICE)
        block_of = torch.arange(case["rows"], device=DEVICE) // GROUP
        for b in range(state["scales"].shape[1]):
            part = slice(b * GROUP, (b + 1) * GROUP)
            w = state["weight_codes"][:, part].double().T.contiguous()
            total += torch.mm(state["codes"][:, part].double(), w) * state["scales"][:, b, None].double() * state["weight_scales"][block_of, b].double()
        return total + state["bias"].double() if state["bias"] is not None else total
    logits, uniform = state["logits"].double().cpu(), state["uniform"].double().cpu()
    tokens = []
    for r in range(case["rows"]):
        of_row = lambda name: float(state[name][r] if isinstance(state[name], torch.Tensor) else torch.tensor(state[name], dtype=torch.float32))  # noqa: E731,B023
        temperature, top_k, top_p, min_p = (of_row(name) for name in ("temperature", "top_k", "top_p", "min_p"))
        order = torch.sort(-logits[r], stable=True).indices
        scores = logits[r][order]
        if temperature <= 0:
            order, scores = order[:1], scores[:1]
        elif top_k > 0:
            order, scores = order[:int(top_k)], scores[:int(top_k)]
        mass = torch.exp((scores - scores[0]) / (temperature if temperature > 0 else 1.0))
        if top_p < 1:
            in_front = torch.cat([mass.new_zeros(1), mass.cumsum(0)[:-1]])
            mass = mass[:max(1, int((in_front < top_p * mass.sum()).sum()))]
        mass = mass[:max(1, int((mass >= min_p).sum()))]
        kept, by_index = order[:len(mass)].sort()
        running = mass[by_index].cumsum(0)
        at = int(torch.searchsorted(running, uniform[r] * running[-1], right=True))
        tokens.append(int(kept[min(at, len(kept) - 1)]))
    return torch.tensor(tokens, device=DEVICE)
