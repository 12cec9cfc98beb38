"""A small decoder of one-bit projections with random weights: norms, rotation, 8-bit cache and attention, and the way to the next
tokens, as a serving program calls them.

    python -m onebitsparsemul_amd.decode [--layers 2] [--hidden 512] [--sequences 16] [--prompt 512] [--tokens 64]
    python -m onebitsparsemul_amd.decode --head e4m3 [--temperature 0.8] [--top-k 50] [--top-p 0.95] [--min-p 0.0]

A prompt goes into the caches in one pass, tokens are decoded one by one behind it, and the logits are compared with those of one
pass over everything. With --head e4m3 the projection onto the vocabulary is in 8 bits, and each token is drawn from the logits in front of it.
"""
import argparse
import time

import torch

from . import BinaryLinear_2_4, BlockLinear, QuantizedCache, block_norm, block_norm_codes, forward_grouped, rotary_table, sample


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
                 dtype=torch.float8_e4m3fn, seed=0, device="cuda", head=None):
        """head: None, the logits from the embedding in 32 bits; "e4m3": from its 8-bit codes, with the last norm's output in such codes."""
        if head not in (None, "e4m3"):
            raise ValueError(f"head must be None or 'e4m3', got {head!r}")
        generator = torch.Generator(device=device)
        generator.manual_seed(seed)
        self.layers = [DecoderLayer(hidden, intermediate, heads, kv_heads, head_dim, generator, device) for _ in range(layers)]
        self.embedding = torch.randn((vocabulary, hidden), generator=generator, device=device).half()
        self.norm = torch.ones(hidden, dtype=torch.float16, device=device)
        self.head = BlockLinear(self.embedding, out_dtype=torch.float32) if head else None
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
        if self.head is not None:  # the last tokens' rows alone
            x, residual = (t if t is None else t.view(sequences, new, -1)[:, -1] for t in (x, residual))
            return self.head(block_norm_codes(x, residual, self.norm)[1:])
        _, h = block_norm(x, residual, self.norm)
        return h.view(sequences, new, -1)[:, -1].float() @ self.embedding.float().T

    @torch.no_grad()
    def generate(self, prompt, uniform, **options):
        """prompt (sequences, length): ids; uniform (tokens, sequences): a random number in [0, 1) for each token and sequence; options: sample's. Returns the ids of
        the tokens behind the prompt, (sequences, tokens); the caches hold the prompt and all but the last of them. A sequence whose logits give no token (a NaN among
        them) has -1 from there on, with id 0 in its caches."""
        count, new = uniform.shape[0], prompt.shape[1]
        ids, tokens = prompt.reshape(-1), []
        longest = int(self.lengths.max()) + new if count else 0
        if longest + count - 1 > self.table.shape[0]:
            raise ValueError(f"{count} tokens behind a length of {longest} need {longest + count - 1} places of a sequence, the decoder has {self.table.shape[0]}")
        for step in range(count):
            drawn = sample(self.step(ids, new, longest), uniform[step], **options)
            tokens.append(torch.where(tokens[-1] < 0, -1, drawn) if tokens else drawn)
            ids, new, longest = tokens[-1].clamp(min=0), 1, longest + 1
        return torch.stack(tokens, dim=1) if tokens else prompt.new_empty((prompt.shape[0], 0), dtype=torch.int64)


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--hidden", type=int, default=512)
    ap.add_argument("--intermediate", type=int, default=1408)
    ap.add_argument("--sequences", type=int, default=16)
    ap.add_argument("--prompt", type=int, default=512)
    ap.add_argument("--tokens", type=int, default=64, help="decoded behind the prompt")
    ap.add_argument("--head", choices=["e4m3"], default=None, help="logits from 8-bit codes, and tokens drawn from them")
    ap.add_argument("--temperature", type=float, default=0.8)
    ap.add_argument("--top-k", type=int, default=50)
    ap.add_argument("--top-p", type=float, default=0.95)
    ap.add_argument("--min-p", type=float, default=0.0)
    args = ap.parse_args(argv)
    heads = max(1, args.hidden // 64)
    sizes = dict(hidden=args.hidden, intermediate=args.intermediate, heads=heads, kv_heads=max(1, heads // 2))
    total = args.prompt + args.tokens
    stepwise, whole = (Decoder(args.layers, args.sequences, total, head=args.head, **sizes) for _ in range(2))
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
    if args.head:
        uniform = torch.rand((args.tokens, args.sequences), device="cuda")
        options = dict(temperature=args.temperature, top_k=args.top_k, top_p=args.top_p, min_p=args.min_p)
        for _ in range(2):
            stepwise.lengths.zero_()
            torch.cuda.synchronize()
            begin = time.perf_counter()
            drawn = stepwise.generate(ids[:, :args.prompt], uniform, **options)
            torch.cuda.synchronize()
            seconds = time.perf_counter() - begin
        print(f"{args.tokens} tokens drawn behind the prompt: {seconds * 1e3:.2f} ms with the prompt's pass; the first sequence's: {drawn[0, :12].tolist()}")
    return off


if __name__ == "__main__":
    main()
