"""From a decoder's last layer to its next tokens, on the HIP library (include/onebit_head.h): 8-bit codes with a scale for each 128 values, behind a norm or
by themselves, the matrix product of such codes, and tokens from logits. The projection onto a vocabulary stays in more than one bit, and is then the largest
thing that a step reads. For inference, as BinaryLinear_2_4: the results have no gradient. No counterpart in the
reference, whose layers stop at the projection (onebit_sparse_mul/__init__.py:101-145).

onebitsparsemul_amd.decode runs them together.
"""
import torch

from .decoder import _binding

__all__ = ["block_norm_codes", "quantize_rows", "quantize_weight", "block_linear", "BlockLinear", "sample"]

GROUP = 128  # values that share a scale
MOST = 448.0  # the largest e4m3


def block_norm_codes(x, residual, weight, bias=None, post_weight=None, post_bias=None, gate=None, residual_scale=1.0, block_scale=1.0, eps=1e-5,
                     kind="rms", residual_out=None):
    """(h, codes, scales): block_norm whose y leaves as codes and scales, quantised from the unrounded values as by quantize_rows."""
    return _binding().block_norm_codes(x, residual, weight, bias, post_weight, post_bias, gate, residual_scale, block_scale, eps, kind, residual_out)


def quantize_rows(x):
    """(codes, scales) of x (..., columns), float16, bfloat16 or float32: codes float8_e4m3fn (..., columns rounded up to a multiple of 128, 0 there), scales
    float32, one for each 128 columns. scale = largest magnitude / 448, code = value / scale, 0 where the scale is 0. NaN and infinities make their group's scale
    such and its codes 0, so that a product with them is NaN."""
    return _binding().quantize_rows(x)


@torch.no_grad()
def quantize_weight(weight):
    """(codes, scales) of a weight (rows, columns), once: codes float8_e4m3fn (rows, columns rounded up to a multiple of 128), scales float32 (rows / 128 rounded
    up, columns / 128 rounded up), one for each 128 x 128 values, as by quantize_rows."""
    if weight.dim() != 2 or not weight.is_floating_point():
        raise ValueError(f"weight must be a floating-point matrix, got {weight.dtype} of shape {tuple(weight.shape)}")
    rows, columns = weight.shape
    groups = -(-columns // GROUP)
    codes = torch.zeros((rows, groups * GROUP), dtype=torch.float8_e4m3fn, device=weight.device)
    scales = torch.empty((-(-rows // GROUP), groups), dtype=torch.float32, device=weight.device)
    step = 64 * GROUP  # what is held in 32 bits at a time
    most = scales.new_full((), MOST)  # (by a Python number the GPU multiplies with its reciprocal, which is another scale half of the time)
    for first in range(0, rows if columns else 0, step):
        part = weight[first:first + step].float()
        count = part.shape[0]
        blocks = torch.nn.functional.pad(part, (0, groups * GROUP - columns, 0, -count % GROUP)).view(-1, GROUP, groups, GROUP)
        scale = blocks.abs().amax((1, 3)) / most
        inside = ((scale > 0) & torch.isfinite(scale))[:, None, :, None]
        quotient = torch.where(inside, blocks / torch.where(inside, scale[:, None, :, None], 1.0), 0.0).clamp(-MOST, MOST)
        codes[first:first + count] = quotient.view(-1, groups * GROUP)[:count].to(torch.float8_e4m3fn)
        scales[first // GROUP:first // GROUP + blocks.shape[0]] = scale
    return codes, scales


def block_linear(codes, scales, weight_codes, weight_scales, bias=None, out_dtype=torch.float16, out=None):
    """y (..., rows) = x W^T (+ bias) of codes (..., columns) with their scales (quantize_rows, block_norm_codes) and a weight's (quantize_weight), sums in
    fp32, rounded once to out_dtype (float16, bfloat16 or float32, or out's). out: with whole rows, apart from the operands. For 16-bit results of more than 16 tokens the
    products of eight neighbouring columns are cut off at 2^-13 of the largest of them, which the matrix unit is twice as fast for: off by less than 7 2^-13 of the sum of
    those largest magnitudes. Where columns many times the others may cancel, ask for float32, which is never cut."""
    return _binding().block_linear(codes, scales, weight_codes, weight_scales, bias, out_dtype, out)


class BlockLinear(torch.nn.Module):
    """A linear layer on 8-bit codes with a scale for each 128 x 128 weights: y = x W^T (+ bias)."""

    def __init__(self, weight, bias=None, out_dtype=None):
        """weight (rows, columns), quantised here; out_dtype: of the result; None: x's, or float16 where x comes as codes."""
        super().__init__()
        codes, scales = quantize_weight(weight)
        self.columns = weight.shape[1]
        self.out_dtype = out_dtype
        self.register_buffer("codes", codes)
        self.register_buffer("scales", scales)
        self.register_buffer("bias", None if bias is None else bias.detach())

    def _apply(self, fn, recurse=True):
        # of a change of the module's type (half() and the like) codes and scales take the move alone
        before = {name: getattr(self, name) for name in ("codes", "scales")}
        super()._apply(fn, recurse)
        for name, t in before.items():
            now = getattr(self, name)
            if now.dtype != t.dtype:
                setattr(self, name, t.to(now.device))
        return self

    def forward(self, x):
        """x (..., columns), or its (codes, scales) of quantize_rows or block_norm_codes"""
        if isinstance(x, torch.Tensor):
            if x.shape[-1] != self.columns:
                raise ValueError(f"x must have {self.columns} columns, got shape {tuple(x.shape)}")
            return block_linear(*quantize_rows(x), self.codes, self.scales, self.bias, self.out_dtype or x.dtype)
        return block_linear(*x, self.codes, self.scales, self.bias, self.out_dtype or torch.float16)


def sample(logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """A token (int64) for each row of logits (..., vocabulary), float16, bfloat16 or float32, from a random number in [0, 1) for each, uniform (...) float32. In this
    order: logits divided by the temperature; of the tokens, larger logits first, equal ones by index, the first top_k stay; of these those in front of which less
    than top_p of their mass lies; of these those with at least min_p of the first one's probability; the first always stays. The token is the first of them by index at
    which the running mass exceeds uniform times its total. temperature 0: the largest logit. top_k 0, top_p 1, min_p 0: no such filter. Each is a number, or a
    tensor with one for each row (top_k int32, the others float32). -inf hides a token; a row with a NaN, and one that is hidden whole, gives -1. Weights are
    integers, multiples of 2^-42 of the largest: the same call gives the same token."""
    return _binding().sample(logits, uniform, temperature, top_k, top_p, min_p)
