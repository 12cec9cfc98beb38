"""What a decoder layer runs around its one-bit projections, on the HIP library (include/onebit_decoder.h): rotary positions, a
paged cache of 8-bit keys and values with the attention that reads it, and the norms around a block with its residual sum. For
inference, as BinaryLinear_2_4: the results have no gradient. No counterpart in the reference, whose layers stop at the
projection (onebit_sparse_mul/__init__.py:101-145).

onebitsparsemul_amd.decode runs them together.
"""
import math

import torch

__all__ = ["rotary", "rotary_table", "cache_append", "cache_attention", "block_norm", "QuantizedCache"]


_compiled = None


def _binding():
    global _compiled
    if _compiled is None:
        from . import onebit_sparse_cuda  # noqa: PLC0415  (compiled module, built in-tree)
        _compiled = onebit_sparse_cuda
    return _compiled


def rotary_table(positions, rotary_dim, base=10000.0, scaling=None, device="cuda"):
    """The table of `rotary` and `cache_append`: fp32 (positions, rotary_dim), the cosines of each pair's angle and then the
    sines. Pair i turns by position * base^(-2 i / rotary_dim), computed in 64 bits. `scaling` stretches it for contexts longer
    than the model was trained on:

        {"kind": "linear", "factor": f}   every rate divided by f
        {"kind": "base", "factor": f}     base multiplied by f^(rotary_dim / (rotary_dim - 2)): the slowest rate is divided by f
        {"kind": "bands", "factor": f, "original": n, "low": l, "high": h}
            rates that turn less than l times in n positions are divided by f, those that turn more than h times kept,
            between them both are mixed linearly in the number of turns
        {"kind": "ramp", "factor": f, "original": n, "fast": 32, "slow": 1}
            the same with the mix linear in the pair's index, and cosines and sines multiplied by 0.1 ln f + 1"""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and positive, got {rotary_dim}")
    index = torch.arange(0, rotary_dim, 2, dtype=torch.float64)
    kind = scaling["kind"] if scaling else None
    factor = float(scaling["factor"]) if scaling else 1.0
    if kind not in (None, "linear", "base", "bands", "ramp"):
        raise ValueError(f"scaling kind must be 'linear', 'base', 'bands' or 'ramp', got {kind!r}")
    if kind == "base":
        base = base * factor ** (rotary_dim / (rotary_dim - 2)) if rotary_dim > 2 else base
    rates = base ** (-index / rotary_dim)
    magnitude = 1.0
    if kind == "linear":
        rates = rates / factor
    elif kind == "bands":
        turns = scaling["original"] * rates / (2 * math.pi)
        keep = ((turns - scaling["low"]) / (scaling["high"] - scaling["low"])).clamp(0, 1)
        rates = rates * keep + rates / factor * (1 - keep)
    elif kind == "ramp":
        def pair_of(turns):  # the (fractional) index of the pair that turns so often in the original positions
            return rotary_dim * math.log(scaling["original"] / (turns * 2 * math.pi)) / (2 * math.log(base))
        first = max(math.floor(pair_of(scaling.get("fast", 32))), 0)
        last = min(math.ceil(pair_of(scaling.get("slow", 1))), rotary_dim - 1)  # (pairs end at rotary_dim / 2 - 1: the bound that models are trained with)
        stretched = ((index / 2 - first) / max(last - first, 1e-3)).clamp(0, 1)
        rates = rates * (1 - stretched) + rates / factor * stretched
        magnitude = 0.1 * math.log(factor) + 1 if factor > 1 else 1.0
    angles = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * rates.to(device)
    return (torch.cat([angles.cos(), angles.sin()], dim=1) * magnitude).float()


def rotary(x, positions, table, interleaved=False, out=None):
    """Rotary positions on x (tokens, heads, head_dim): the first table.shape[1] elements of each head are turned in pairs, half
    a part apart or interleaved, the others copied. positions (tokens,): int32 or int64; one outside of the table gives NaN. x may
    be strided; out may be x. Where it lies on the operands in another way, they are copied first."""
    return _binding().rotary(x, positions, table, interleaved, out)


def cache_append(k, v, k_cache, v_cache, k_scale, v_scale, pages, lengths, starts=None, q=None, rotary=None, interleaved=False, max_new=None):
    """Writes the new tokens' keys and values, (tokens, kv_heads, head_dim) each, into the 8-bit cache: codes (pages, kv_heads, block,
    head_dim) of type float8_e4m3fn or int8 and scales (pages, kv_heads), not negative, a value being its code times the scale of its page and head.
    pages (sequences, width) int32: the page of each `block` tokens of a sequence; lengths (sequences,) int32: tokens WITH the
    new ones; starts (sequences + 1,) int32: where a sequence's new tokens begin in k and v (None: equally many each); max_new: no
    sequence has more (host number; spares the launch a grid for all tokens in one sequence). With a rotary table keys are
    turned by their positions, and so are the queries q; returns them turned (None without q; rows of no sequence hold anything). A page's scale only grows while
    tokens are added to it; where it does, its older codes are rounded again. NaN and infinities make their page's scale such."""
    return _binding().cache_append(k, v, k_cache, v_cache, k_scale, v_scale, pages, lengths, starts, q, rotary, interleaved, max_new)


def cache_attention(q, k_cache, v_cache, k_scale, v_scale, pages, lengths, starts=None, scale=None, max_new=None, max_length=None, out=None):
    """softmax(scale q k^T) v of the new tokens' queries (tokens, heads, head_dim), float16 or bfloat16, over the cache, causal: the last of
    a sequence's new tokens sees all its `lengths` tokens. heads is a multiple of kv_heads. Other arguments as of cache_append; scale:
    1 / sqrt(head_dim) unless given; max_length: no sequence is longer (host number: what the launch is planned for). A row that
    sees nothing is 0. out may be q, as rotary's may be x."""
    return _binding().cache_attention(q, k_cache, v_cache, k_scale, v_scale, pages, lengths, starts, scale, max_new, max_length, out)


def block_norm(x, residual, weight, bias=None, post_weight=None, post_bias=None, gate=None, residual_scale=1.0, block_scale=1.0, eps=1e-5,
               kind="rms", out_dtype=None, residual_out=None):
    """(h, y): h = residual_scale residual + block_scale gate post(x), the residual behind a block with output x, and y = norm(h), the
    input of the next. post: a norm with post_weight (and post_bias), where given; gate: (hidden,), (..., 1), (..., hidden) or one value.
    kind "rms" or "layer". In fp32 throughout; h has the residual's type, y x's (or out_dtype). x None: y = norm(residual). residual_out
    may be the residual or x itself, as rotary's out may be x."""
    return _binding().block_norm(x, residual, weight, bias, post_weight, post_bias, gate, residual_scale, block_scale, eps, kind, out_dtype, residual_out)


class QuantizedCache:
    """Keys and values of one layer in 8 bits, in pages of `block` tokens with a scale for each page and head."""

    def __init__(self, pages, kv_heads, head_dim, block=64, dtype=torch.float8_e4m3fn, device="cuda"):
        if dtype not in (torch.float8_e4m3fn, torch.int8):
            raise TypeError(f"dtype must be torch.float8_e4m3fn or torch.int8, got {dtype}")
        if block not in (16, 32, 64, 128) or head_dim not in (64, 128):
            raise ValueError(f"block must be 16, 32, 64 or 128 and head_dim 64 or 128, got {block} and {head_dim}")
        self.block = block
        self.k = torch.zeros((pages, kv_heads, block, head_dim), dtype=dtype, device=device)
        self.v = torch.zeros_like(self.k)
        self.k_scale = torch.zeros((pages, kv_heads), dtype=torch.float32, device=device)
        self.v_scale = torch.zeros_like(self.k_scale)

    def append(self, k, v, pages, lengths, **options):
        """cache_append on this cache."""
        return cache_append(k, v, self.k, self.v, self.k_scale, self.v_scale, pages, lengths, **options)

    def attend(self, q, pages, lengths, **options):
        """cache_attention over this cache."""
        return cache_attention(q, self.k, self.v, self.k_scale, self.v_scale, pages, lengths, **options)
