"""A small decoder of one-bit projections with random weights: norms, rotation, 8-bit cache and attention as a serving program
calls them.

    python -m onebitsparsemul_amd.decode [--layers 2] [--hidden 512] [--sequences 16] [--prompt 512] [--tokens 64]

A prompt goes into the caches in one pass, tokens are decoded one by one behind it, and the logits are compared with those of one
pass over everything.
"""
import argparse
import time

import torch

from . import BinaryLinear_2_4, QuantizedCache, block_norm, forward_grouped, rotary_table


class DecoderLayer(torch.nn.Module):
    """One decoder layer on one-bit 2:4 projections: norm, q/k/v in one launch, rotation and cache write in one, attention, output
    projection; residual sum and norm in one; gate and up projection in one launch, down projection. The residual sum behind the down
    projection is the next layer's first norm's."""

    def __init__(self, hidden, intermediate, heads, kv_heads, head_dim, generator=None, device="cuda"):
        super().__init__()
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim

        def linear(k, m):  # random weights; a one-bit product of k / 2 terms is scaled by the norm or the residual behind it
            layer = BinaryLinear_2_4(k, m).to(device)
            layer.pack(torch.randn((m, k), generator=generator, device=device, dtype=torch.float32).half())
            return layer
        self.q, self.k, self.v = (linear(hidden, n * head_dim) for n in (heads, kv_heads, kv_heads))
        self.o = linear(heads * head_dim, hidden)
        self.gate, self.up, self.down = linear(hidden, intermediate), linear(hidden, intermediate), linear(intermediate, hidden)
        self.register_buffer("input_norm", torch.ones(hidden, dtype=torch.float16, device=device))
        self.register_buffer("post_norm", torch.ones(hidden, dtype=torch.float16, device=device))

    def forward(self, x, residual, cache, pages, lengths, starts, table, max_new, max_length):
        """x (tokens, hidden): the output of the block in front, already scaled, or None; returns (block output, residual)."""
        tokens = residual.shape[0]
        residual, h = block_norm(x, residual, self.input_norm)
        # a column of a one-bit weight has half its entries +-1: sums of `in_features / 2` terms
        q, k, v = (y.view(tokens, -1, self.head_dim) * self.q.infeatures**-0.5 for y in forward_grouped([self.q, self.k, self.v], h))
        q = cache.append(k, v, pages, lengths, starts=starts, q=q, rotary=table, max_new=max_new)
        o = cache.attend(q, pages, lengths, starts=starts, max_new=max_new, max_length=max_length)
        residual, h = block_norm(self.o(o.view(tokens, -1)), residual, self.post_norm, block_scale=self.o.infeatures**-0.5)
        gate, up = forward_grouped([self.gate, self.up], h)
        scale = self.gate.infeatures**-0.5
        return self.down(torch.nn.functional.silu(gate * scale) * (up * scale)) * self.down.infeatures**-0.5, residual


class Decoder:
    """A few layers with their caches, for the sequences of one batch: pages are handed out as the sequences grow."""

    def __init__(self, layers, sequences, length, hidden=512, intermediate=1408, heads=8, kv_heads=4, head_dim=64, vocabulary=4096, block=64,
                 dtype=torch.float8_e4m3fn, seed=0, device="cuda"):
        generator = torch.Generator(device=device)
        generator.manual_seed(seed)
        self.layers = [DecoderLayer(hidden, intermediate, heads, kv_heads, head_dim, generator, device) for _ in range(layers)]
        self.embedding = torch.randn((vocabulary, hidden), generator=generator, device=device).half()
        self.norm = torch.ones(hidden, dtype=torch.float16, device=device)
        width = -(-length // block)
        self.caches = [QuantizedCache(sequences * width, kv_heads, head_dim, block=block, dtype=dtype, device=device) for _ in range(layers)]
        # sequence s owns pages s, s + sequences, ...: nothing is to be gained from neighbouring pages
        self.pages = (torch.arange(width, device=device)[None, :] * sequences + torch.arange(sequences, device=device)[:, None]).to(torch.int32).contiguous()
        self.lengths = torch.zeros(sequences, dtype=torch.int32, device=device)
        self.table = rotary_table(length, head_dim, device=device)

    @torch.no_grad()
    def step(self, tokens, new, longest):
        """tokens: the ids of `new` tokens of each sequence, one sequence behind the other; longest: an upper bound of the lengths then.
        Returns the logits of each sequence's last token."""
        sequences = self.lengths.shape[0]
        self.lengths += new
        x, residual = None, self.embedding[tokens]
        for layer, cache in zip(self.layers, self.caches):
            x, residual = layer(x, residual, cache, self.pages, self.lengths, None, self.table, new, longest)
        _, h = block_norm(x, residual, self.norm)
        return h.view(sequences, new, -1)[:, -1].float() @ self.embedding.float().T


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--hidden", type=int, default=512)
    ap.add_argument("--intermediate", type=int, default=1408)
    ap.add_argument("--sequences", type=int, default=16)
    ap.add_argument("--prompt", type=int, default=512)
    ap.add_argument("--tokens", type=int, default=64, help="decoded behind the prompt")
    args = ap.parse_args(argv)
    heads = max(1, args.hidden // 64)
    sizes = dict(hidden=args.hidden, intermediate=args.intermediate, heads=heads, kv_heads=max(1, heads // 2))
    total = args.prompt + args.tokens
    stepwise, whole = (Decoder(args.layers, args.sequences, total, **sizes) for _ in range(2))
    ids = torch.randint(0, 4096, (args.sequences, total), device="cuda")
    for warm in (True, False):
        stepwise.lengths.zero_()
        stepwise.step(ids[:, :args.prompt].reshape(-1), args.prompt, args.prompt)
        torch.cuda.synchronize()
        begin = time.perf_counter()
        for t in range(args.prompt, total):
            logits = stepwise.step(ids[:, t], 1, t + 1)
        torch.cuda.synchronize()
        seconds = time.perf_counter() - begin
    begin = time.perf_counter()
    want = whole.step(ids.reshape(-1), total, total)
    torch.cuda.synchronize()
    prompt_seconds = time.perf_counter() - begin
    off = float((logits - want).norm() / want.norm())
    print(f"{args.layers} layers, {args.sequences} sequences: {args.tokens} tokens behind a prompt of {args.prompt}: {seconds / args.tokens * 1e6:.0f} us a step; "
          f"all {total} in one pass: {prompt_seconds * 1e3:.2f} ms")
    print(f"logits behind the last token, step by step against the one pass: {off:.4f} apart (the caches' pages are rounded again as they grow)")
    return off


if __name__ == "__main__":
    main()
