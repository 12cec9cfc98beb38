"""The operators of a decoder layer around its one-bit projections against plain implementations in 64 bits.

Tolerances: u is the unit roundoff of a result's type (fp16 2^-11, bf16 2^-8, fp32 2^-24). Attention sums p_j v_j with p in at least
eleven bits (an error of 2^-11 of sum p |v| at most, whatever the signs) and rounds once; exponents are below 2^6 in magnitude here, so
that fp32 arguments add 2^-18 at most. Norms and rotations are a few fp32 operations and one rounding. Codes are those of the definition in fp32,
to the bit."""
import math

import pytest
import torch

import onebitsparsemul_amd as onebit

pytestmark = pytest.mark.gpu

U = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}
E4M3, INT8 = torch.float8_e4m3fn, torch.int8


def generator(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def bits(codes):
    return codes.view(torch.uint8)


def decoded(codes):
    return codes.float().double()


class Case:
    """A cache of random codes for sequences of the given lengths and new tokens, its pages in a random order."""

    def __init__(self, lengths, new, heads, kv_heads, dim, block, code, dtype, seed=0, spread=0.2, extra=3):
        g = generator(seed)
        need = [-(-n // block) for n in lengths]
        order = torch.randperm(sum(need) + extra, generator=g)
        self.pages = torch.full((len(lengths), max(max(need), 1)), -1, dtype=torch.int32)
        at = 0
        for s, n in enumerate(need):
            self.pages[s, :n] = order[at:at + n]
            at += n
        shape = (sum(need) + extra, kv_heads, block, dim)
        most = 448.0 if code == E4M3 else 127.0
        make = lambda: (torch.randn(shape, generator=g) * most / 4).clamp(-most, most)  # noqa: E731
        self.k, self.v = (make().to(E4M3) if code == E4M3 else make().round().to(INT8) for _ in range(2))
        self.k_scale, self.v_scale = (4 / most * torch.exp(spread * torch.randn(shape[:2], generator=g)) for _ in range(2))
        self.lengths, self.new, self.heads, self.kv_heads, self.dim, self.block = lengths, new, heads, kv_heads, dim, block
        self.q = torch.randn((sum(new), heads, dim), generator=g).to(dtype)
        self.starts = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32)

    def call(self, scale=None, q=None, starts=True, **options):
        d = lambda t: t.cuda()  # noqa: E731
        return onebit.cache_attention(d(self.q if q is None else q), d(self.k), d(self.v), d(self.k_scale), d(self.v_scale), d(self.pages),
                                      torch.tensor(self.lengths, dtype=torch.int32).cuda(), starts=d(self.starts) if starts else None,
                                      scale=scale, **options)

    def crowd(self, copies, **options):
        """The call with its sequences `copies` times over, which the launch is planned for; the first ones' rows"""
        rows = self.q.shape[0]
        starts = torch.cat([self.starts[:-1] + i * rows for i in range(copies)] + [torch.tensor([copies * rows])]).to(torch.int32)
        cuda = lambda t: t.cuda()  # noqa: E731
        out = onebit.cache_attention(cuda(self.q.repeat(copies, 1, 1)), cuda(self.k), cuda(self.v), cuda(self.k_scale), cuda(self.v_scale),
                                     cuda(self.pages.repeat(copies, 1)), torch.tensor(self.lengths * copies, dtype=torch.int32).cuda(), starts=cuda(starts), **options)
        assert torch.equal(out[:rows], out[-rows:])
        return out[:rows]

    def want(self, scale=None):
        """(outputs, sum p |v|) in 64 bits"""
        scale = 1 / math.sqrt(self.dim) if scale is None else scale
        group, outs, sizes, at = self.heads // self.kv_heads, [], [], 0
        for s, (length, n) in enumerate(zip(self.lengths, self.new)):
            length = min(length, self.pages.shape[1] * self.block)
            o = torch.zeros((n, self.heads, self.dim), dtype=torch.float64)
            size = torch.zeros_like(o)
            use = self.pages[s, :-(-length // self.block)].long()
            there = ((use >= 0) & (use < self.k.shape[0])).repeat_interleave(self.block)[:length]
            use = use.clamp(0, self.k.shape[0] - 1)
            seen = (torch.arange(length) <= torch.arange(length - n, length)[:, None]) & there
            for h in range(self.heads):
                kv = h // group
                k, v = ((decoded(bits(c)[use, kv].view(c.dtype)) * x[use, kv].double()[:, None, None]).flatten(0, 1)[:length]
                        for c, x in ((self.k, self.k_scale), (self.v, self.v_scale)))
                for i in range(n):
                    if not seen[i].any():
                        continue
                    p = torch.softmax((k[seen[i]] @ self.q[at + i, h].double()) * scale, 0)
                    o[i, h], size[i, h] = p @ v[seen[i]], p @ v[seen[i]].abs()
            outs.append(o)
            sizes.append(size)
            at += n
        return torch.cat(outs), torch.cat(sizes)

    def check(self, got, scale=None, rows=slice(None)):
        want, size = self.want(scale)
        u = U[self.q.dtype]
        error = (got.double().cpu() - want).abs()
        bound = u * (1 + 2.0**-11) * want.abs() + (2.0**-11 + 2.0**-18) * size + 1e-30
        if self.q.dtype == torch.float16:
            bound = bound + 2.0**-25  # half of the least subnormal
        assert got.dtype == self.q.dtype and bool(torch.isfinite(got).all())
        assert bool((error <= bound)[rows].all()), float((error / bound)[rows].max())


@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attention_of_single_tokens(code, dim, dtype):
    lengths = [1, 2, 15, 16, 17, 31, 32, 33, 64, 127, 128, 129, 300, 1000]
    case = Case(lengths, [1] * len(lengths), 8, 2, dim, 16, code, dtype, seed=dim)
    case.check(case.call(max_new=1, max_length=1000))
    case.check(case.call(starts=False))


@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 4), (6, 2), (10, 2), (16, 1), (40, 2)])
def test_attention_heads_and_blocks(block, heads, kv_heads):
    case = Case([200, 77, 130], [1, 1, 1], heads, kv_heads, 64, block, E4M3, torch.float16, seed=heads + block)
    case.check(case.call())


@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lengths,new", [([70], [70]), ([200], [33]), ([1, 40, 131, 90, 64], [1, 40, 3, 17, 64]), ([300, 5], [5, 5]),
                                         ([257], [129])])
def test_attention_of_several_tokens(code, dim, lengths, new):
    case = Case(lengths, new, 4, 2, dim, 32, code, torch.bfloat16 if code == INT8 else torch.float16, seed=sum(new))
    case.check(case.call(max_new=max(new)))
    case.check(case.call())


def test_attention_of_nothing():
    """No length, no new tokens, more new tokens than tokens: rows that see nothing are 0"""
    case = Case([0, 50, 3, 0, 64], [2, 0, 6, 0, 4], 4, 2, 64, 16, E4M3, torch.float16)
    got = case.call()
    assert bool((got[:2] == 0).all()) and bool((got[2:5] == 0).all())
    case.check(got)
    empty = case.call(q=case.q[:0], max_new=1)
    assert empty.shape == (0, 4, 64)


@pytest.mark.parametrize("hints", [dict(max_new=1, max_length=16), dict(max_new=1), dict(max_length=1), dict(max_length=1 << 30)])
def test_attention_with_wrong_lengths_in_the_plan(hints):
    """Longer sequences than the launch was planned for are right"""
    case = Case([900, 1500], [1, 1], 8, 2, 64, 32, E4M3, torch.float16)
    case.check(case.call(**hints))


def test_attention_leaves_out_missing_pages():
    case = Case([100, 70, 64], [3, 1, 64], 4, 2, 64, 16, E4M3, torch.float16)
    case.pages[0, 2], case.pages[1, 0], case.pages[2, 1] = -1, 1 << 20, -7
    case.check(case.call())
    case.lengths = [1000, 70, 64]  # more than its table holds
    case.check(case.call())


@pytest.mark.parametrize("new", [1, 40])
def test_attention_ignores_what_a_row_does_not_see(new):
    """NaN codes behind a sequence's end, NaN and infinite scales of pages that are not in use or that a row is too early for"""
    case = Case([75, 150], [new, new], 4, 2, 64, 32, E4M3, torch.float16)
    clean = case.call()
    poisoned = set(range(case.k.shape[0])) - set(case.pages.flatten().tolist())
    for page in poisoned:
        case.k_scale[page], case.v_scale[page] = math.nan, math.inf
        bits(case.k)[page], bits(case.v)[page] = 0x7f, 0x7f
    for s, length in enumerate(case.lengths):
        page, used = int(case.pages[s, length // 32]), length % 32
        bits(case.k)[page, :, used:], bits(case.v)[page, :, used:] = 0x7f, 0xff
    assert torch.equal(case.call(), clean)
    if new > 1:  # the last page of the second sequence holds its positions 128 ... 149; its first new token is at 110
        page = int(case.pages[1, 4])
        case.k_scale[page], case.v_scale[page] = math.nan, math.inf
        got = case.call()
        assert torch.equal(got[:new + 18], clean[:new + 18]) and not bool(torch.isfinite(got[new + 18:]).any())


@pytest.mark.parametrize("length,new,copies", [(400, 1, 1), (400, 48, 1), (400, 400, 1), (400, 130, 24), (400, 130, 36), (130, 130, 24)])
@pytest.mark.parametrize("block", [16, 32, 64])
@pytest.mark.parametrize("decades", [3, 13])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attention_with_scales_far_apart(length, new, copies, block, decades, dtype):
    """Scales of the pages over some decades, some 0: p takes them on without leaving fp16's range, and a row that sees small ones
    alone, beside large ones that it does not see, loses nothing"""
    case = Case([length], [new], 4, 2, 64, block, E4M3, dtype, seed=3)
    g = generator(9)
    case.v_scale = 10 ** (decades * torch.rand(case.v_scale.shape, generator=g) + 2 - decades)
    case.v_scale[case.pages[0, 1].long()] = 0
    case.k_scale[case.pages[0, -1].long()] = 0
    if dtype == torch.float16:
        case.v_scale *= 0.1
    case.check(case.crowd(copies, max_new=new))
    case.v_scale = torch.zeros_like(case.v_scale)
    assert bool((case.crowd(copies, max_new=new) == 0).all())


@pytest.mark.parametrize("dim,code", [(64, E4M3), (128, INT8)])
@pytest.mark.parametrize("lengths,new,copies,most", [([200, 77], [70, 33], 1, 1), ([200, 77], [70, 33], 1, 9), ([150], [150], 1, 20),
                                                     ([300], [300], 130, 20), ([300, 40], [300, 7], 130, 70), ([420], [410], 130, 129)])
def test_attention_of_more_rows_than_planned(dim, code, lengths, new, copies, most):
    """Sequences with more new tokens than the launch was planned for: its workgroups take their other rows one tile behind the other, few rows of them and many"""
    case = Case(lengths, new, 4, 2, dim, 16, code, torch.float16, seed=most)
    case.check(case.crowd(copies, max_new=most))


@pytest.mark.parametrize("dim,block,code", [(64, 16, E4M3), (128, 16, INT8), (64, 32, INT8)])
@pytest.mark.parametrize("lengths,new,heads,kv_heads,copies", [([5000, 4113, 2100], [1, 1, 1], 8, 4, 70), ([9000], [3], 4, 4, 200), ([5000], [2], 1, 1, 1),
                                                               ([2500, 1100], [130, 33], 4, 2, 90), ([2500], [130], 4, 2, 24), ([1025], [130], 4, 2, 90)])
def test_attention_over_more_pages_than_lanes(dim, block, code, lengths, new, heads, kv_heads, copies):
    """A wavefront knows 64 pages of its sequence at a time and reads on in the table where its keys go beyond; small pages, in one split and in several"""
    case = Case(lengths, new, heads, kv_heads, dim, block, code, torch.float16, seed=lengths[0])
    if len(lengths) > 1:
        case.pages[0, 66], case.pages[0, 64] = -1, 1 << 30  # two that are not there
    case.check(case.crowd(copies, max_new=max(new), max_length=max(lengths)))


# rows (tokens x heads of a key/value head) of one workgroup and more, enough of them that the kernel of prompts takes them
@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("dim,block", [(64, 16), (64, 32), (64, 128), (128, 16), (128, 64), (128, 32)])
@pytest.mark.parametrize("lengths,new,heads,kv_heads,copies", [([70, 33, 0, 200], [70, 33, 2, 40], 4, 2, 20), ([300], [129], 4, 2, 30), ([129], [1], 40, 1, 300),
                                                              ([64, 1, 65], [64, 1, 1], 12, 2, 30), ([300], [129], 4, 2, 40), ([129], [1], 40, 1, 400)])
def test_attention_of_many_prompts(code, dim, block, lengths, new, heads, kv_heads, copies):
    case = Case(lengths, new, heads, kv_heads, dim, block, code, torch.float16 if code == E4M3 else torch.bfloat16, seed=block)
    case.check(case.crowd(copies, max_new=max(new)))
    if len(lengths) > 1:  # a page that is missing in the middle, NaN where nothing is, and a scale that is not finite behind what most rows see
        case.pages[0, min(1, case.pages.shape[1] - 1)] = -1
        last = int(case.pages[3 if len(lengths) > 3 else 2, -(-lengths[-1] // block) - 1])
        bits(case.v)[last, :, lengths[-1] % block or block:] = 0x7f if code == E4M3 else 0x80
        case.check(case.crowd(copies, max_new=max(new)))
        if len(lengths) == 4 and block <= 32:  # the fourth sequence's new tokens are its positions 160 ... 199
            clean = case.crowd(copies, max_new=max(new))
            page, first = int(case.pages[3, 192 // block]), 192 - 160
            case.v_scale[page], case.k_scale[page, 1] = math.nan, math.inf
            spoilt = onebit.cache_attention(case.q.repeat(copies, 1, 1).cuda(), case.k.cuda(), case.v.cuda(), case.k_scale.cuda(), case.v_scale.cuda(),
                                            case.pages.repeat(copies, 1).cuda(), torch.tensor(lengths * copies, dtype=torch.int32).cuda(),
                                            starts=torch.cat([case.starts[:-1] + i * sum(new) for i in range(copies)] + [torch.tensor([copies * sum(new)])]).to(torch.int32).cuda(),
                                            max_new=max(new))[:sum(new)]
            seen = sum(new[:3]) + first
            assert torch.equal(spoilt[:seen], clean[:seen]) and not bool(spoilt[seen:].isfinite().any())


@pytest.mark.parametrize("new", [1, 64])
@pytest.mark.parametrize("size", [2.0**-40, 1.0, 2.0**60])
def test_attention_of_queries_of_any_size(new, size):
    case = Case([200], [new], 4, 2, 64, 32, INT8, torch.bfloat16)
    case.q = (case.q * size).to(torch.bfloat16)
    case.check(case.call(scale=0.125 / size), scale=0.125 / size)


@pytest.mark.parametrize("new", [1, 100])
def test_attention_with_large_scores(new):
    """A running maximum that keeps growing: keys in the order of their scores, up to 60 of them apart in the exponent"""
    case = Case([300], [new], 2, 1, 64, 16, E4M3, torch.float16, spread=0.0)
    ramp = torch.linspace(0, 30, 300)
    k = torch.zeros((case.pages.shape[1] * 16, 64))
    k[:300, 0] = ramp
    scale = 30 / 448
    use = case.pages[0].long()
    codes = (k / scale).to(E4M3)
    bits(case.k)[use, 0] = bits(codes).view(-1, 16, 64)
    case.k_scale[:] = scale
    case.q[:] = 0
    case.q[:, 0, 0], case.q[:, 1, 0] = 1.0, -1.0
    case.check(case.call(scale=2.0), scale=2.0)


# (copies of the sequence, new tokens): few rows, and enough of them that the kernel of prompts takes them
@pytest.mark.parametrize("new,copies", [(1, 1), (24, 1), (200, 24)])
@pytest.mark.parametrize("dim,block,code,dtype", [(64, 16, E4M3, torch.float16), (64, 128, INT8, torch.bfloat16), (128, 32, E4M3, torch.bfloat16),
                                                  (128, 64, INT8, torch.float16)])
@pytest.mark.parametrize("scale", [-0.5, -0.125, 0.0])
def test_attention_with_a_scale_that_is_not_positive(new, copies, dim, block, code, dtype, scale):
    """The largest exponent is then that of the least product; with a scale of 0 every key counts the same"""
    case = Case([500], [new], 4, 2, dim, block, code, dtype, seed=dim + new)
    case.check(case.crowd(copies, max_new=new, scale=scale), scale=scale)


@pytest.mark.parametrize("new", [16, 20, 40])
@pytest.mark.parametrize("dim,block,code", [(64, 16, E4M3), (64, 32, INT8), (64, 64, E4M3), (128, 16, INT8), (128, 32, E4M3), (128, 64, INT8)])
@pytest.mark.parametrize("apart", [30, 70, -30, -70])
def test_attention_is_blind_to_the_scales_of_later_pages(new, dim, block, code, apart):
    """Every other page has values 2^apart times as large, and the first new tokens see half of the first page alone, where others of the same tile of rows
    see the second: what a row does not see costs it no bits"""
    case = Case([block // 2 + new], [new], 2, 2, dim, block, code, torch.bfloat16, seed=block)
    case.v_scale[case.pages[0, 1::2].long()] *= 2.0**apart
    case.check(case.call())


@pytest.mark.parametrize("dim,block,code", [(64, 16, E4M3), (64, 32, INT8), (64, 64, E4M3), (128, 16, INT8), (128, 32, E4M3), (128, 64, INT8)])
@pytest.mark.parametrize("apart", [30, 70, -30, -70])
def test_attention_of_prompts_is_blind_to_the_scales_of_later_pages(dim, block, code, apart):
    """The same where many rows make a tile, and first pages whose codes count as 0"""
    case = Case([block // 2 + 64], [64], 2, 2, dim, block, code, torch.bfloat16, seed=block)
    case.v_scale[case.pages[0, 1::2].long()] *= 2.0**apart
    case.check(case.crowd(200, max_new=64))
    case.v_scale[case.pages[0, 0].long()] = 0
    got = case.crowd(200, max_new=64)
    case.check(got)
    assert bool((got[:block // 2] == 0).all())


def test_attention_beside_pages_beyond_the_range_of_a_sum():
    """Values 2^150 apart: the small ones of rows that see no others may count as 0, but as nothing else"""
    case = Case([24], [16], 2, 2, 64, 16, E4M3, torch.bfloat16)
    case.v_scale[case.pages[0, 0].long()] *= 2.0**-90
    case.v_scale[case.pages[0, 1].long()] *= 2.0**60
    got, want = case.call(), case.want()[0]
    case.check(got, rows=slice(8, None))
    assert bool(((got.double().cpu() - want).abs() <= want.abs() * (1 + 2.0**-7))[:8].all())


@pytest.mark.parametrize("new,copies", [(16, 1), (64, 200)])
@pytest.mark.parametrize("dim,block,code", [(64, 16, E4M3), (64, 64, INT8), (128, 32, E4M3), (128, 64, INT8)])
def test_attention_of_the_largest_values(new, copies, dim, block, code):
    """Values up to some 2^123, of which an append makes scales up to 2^121: their sums over the keys are within fp32 here"""
    case = Case([8 + new], [new], 2, 2, dim, block, code, torch.bfloat16, seed=block)
    case.v_scale *= 2.0**(119 if code == E4M3 else 117)
    case.check(case.crowd(copies, max_new=new))


def test_attention_views_streams_and_results_in_place():
    case = Case([130, 90], [20, 1], 8, 2, 128, 64, E4M3, torch.bfloat16)
    plain = case.call()
    fused = torch.randn((21, 12, 128)).to(torch.bfloat16).cuda()
    fused[:, :8] = case.q.cuda()
    assert torch.equal(case.call(q=fused[:, :8]), plain)
    apart = torch.zeros((21, 8, 129), dtype=torch.bfloat16)
    apart[..., 1:] = case.q
    assert torch.equal(case.call(q=apart[..., 1:]), plain)  # rows at odd addresses
    assert torch.equal(case.call(q=-(-case.q)), plain)
    out = torch.full((21, 12, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    assert case.call(out=out[:, 2:10]).data_ptr() == out[:, 2:10].data_ptr()
    assert torch.equal(out[:, 2:10], plain) and bool((out[:, :2] == 7).all()) and bool((out[:, 10:] == 7).all())
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        other = case.call()
    stream.synchronize()
    assert torch.equal(other, plain)


@pytest.mark.parametrize("lengths,new,heads", [([5000], [1], 8), ([5000, 4000], [200, 100], 8), ([40], [40], 64)])
def test_attention_gives_the_same_bits_every_time(lengths, new, heads):
    case = Case(lengths, new, heads, 2, 128, 64, E4M3, torch.float16)
    first = case.call(max_new=max(new), max_length=max(lengths))
    for _ in range(3):
        assert torch.equal(case.call(max_new=max(new), max_length=max(lengths)), first)


@pytest.mark.parametrize("new", [1, 130])
def test_attention_of_long_sequences(new):
    case = Case([3001, 2049, 4096], [new, new, new], 4, 1, 128, 64, INT8, torch.float16, seed=4)
    want = case.call(max_new=new, max_length=1 << 20)
    torch.testing.assert_close(case.call(max_new=new, max_length=4096).float(), want.float(), rtol=2.0**-9, atol=2.0**-9)
    if new == 1:
        case.check(want)
    else:  # the reference takes its time: the last tokens of each
        case.new, case.q = [2, 2, 2], torch.cat([case.q[new * s + new - 2:new * s + new] for s in range(3)])
        case.check(torch.cat([want[new * s + new - 2:new * s + new] for s in range(3)]))


def test_attention_and_append_beyond_32_bits():
    """Pages whose codes lie more than 4 GiB into the cache"""
    block, kv_heads, dim = 128, 8, 128
    pages = (5 << 30) // (block * kv_heads * dim)
    cache = onebit.QuantizedCache(pages, kv_heads, dim, block=block)
    g = generator(1)
    k, v = (torch.randn((300, kv_heads, dim), generator=g).half() for _ in range(2))
    table = torch.tensor([[pages - 1, pages - 3, 0]], dtype=torch.int32)
    lengths = torch.tensor([300], dtype=torch.int32).cuda()
    cache.append(k.cuda(), v.cuda(), table.cuda(), lengths)
    q = torch.randn((300, 8, dim), generator=g).half()
    got = cache.attend(q.cuda(), table.cuda(), lengths, max_new=300)
    case = Case([300], [300], 8, 8, dim, block, E4M3, torch.float16)
    use = table[0].long()
    case.k, case.v = (bits(c)[use.cuda()].view(E4M3).cpu() for c in (cache.k, cache.v))
    case.k_scale, case.v_scale = cache.k_scale[use.cuda()].cpu(), cache.v_scale[use.cuda()].cpu()
    case.pages, case.q = torch.tensor([[0, 1, 2]], dtype=torch.int32), q
    assert float(case.k_scale.min()) > 0
    case.check(got)
    last = cache.attend(q[299:].cuda(), table.cuda(), lengths)
    case.new, case.q = [1], q[299:]
    case.check(last)


# ---- rotary


def turned(x, rows, interleaved):
    """fp32 in the order of the definition"""
    half = rows.shape[-1] // 2
    c, s = rows[:, None, :half], rows[:, None, half:]
    y = x.clone()
    first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    a, b = x[..., first], x[..., second]
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    return y


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,dim,part", [(1, 1, 64, 64), (5, 3, 128, 128), (17, 7, 128, 64), (3, 2, 80, 20), (4, 5, 6, 2), (2, 3, 256, 32),
                                                   (300, 33, 128, 128), (700, 66, 128, 96), (9, 300, 64, 64)])
def test_rotary(dtype, interleaved, tokens, heads, dim, part):
    g = generator(tokens)
    x = torch.randn((tokens, heads, dim), generator=g).to(dtype)
    positions = torch.randint(0, 500, (tokens,), generator=g)
    table = onebit.rotary_table(500, part, device="cpu")
    want = turned(x.float(), table[positions], interleaved).to(dtype)
    for kind in (torch.int32, torch.int64):
        got = onebit.rotary(x.cuda(), positions.to(kind).cuda(), table.cuda(), interleaved=interleaved)
        assert torch.equal(got.cpu(), want)
    exact = turned(x.double(), table[positions].double(), interleaved)
    error = (got.cpu().double() - exact).abs()
    size = turned(x.double().abs(), torch.cat([table[positions][:, :part // 2].abs(), -table[positions][:, part // 2:].abs()], 1).double(), interleaved).abs()
    assert bool((error <= U[dtype] * exact.abs() + 2.0**-22 * (size + x.double().abs()) + 2.0**-25).all())
    # strided, and in place
    wide = torch.zeros((tokens, heads + 2, dim), dtype=dtype).cuda()
    wide[:, 1:-1] = x.cuda()
    view = wide[:, 1:-1]
    assert onebit.rotary(view, positions.cuda(), table.cuda(), interleaved=interleaved, out=view).data_ptr() == view.data_ptr()
    assert torch.equal(view.cpu(), want) and bool((wide[:, 0] == 0).all()) and bool((wide[:, -1] == 0).all())


def test_rotary_outside_of_the_table_and_of_nothing():
    table = onebit.rotary_table(10, 32)
    x = torch.ones((4, 2, 64), dtype=torch.float16, device="cuda")
    got = onebit.rotary(x, torch.tensor([-1, 0, 9, 10]).cuda(), table)
    assert bool(got[[0, 3], :, :32].isnan().all()) and bool((got[..., 32:] == 1).all()) and bool(torch.isfinite(got[1:3]).all())
    assert onebit.rotary(x[:0], torch.zeros(0, dtype=torch.int64, device="cuda"), table).shape == (0, 2, 64)
    strided = torch.randn((4, 2, 128), device="cuda")[..., ::2]
    assert torch.equal(onebit.rotary(strided, torch.arange(4).cuda(), table), onebit.rotary(strided.contiguous(), torch.arange(4).cuda(), table))


# ---- results on the memory of operands


def same_as_apart(call, memory, operands, result):
    """call(operands, out): the result on memory that operands lie on is that of copies of them; operands and result are taken from `memory`"""
    source = memory.clone()
    want = call([take(source).clone() for take in operands], None)
    out = result(memory)
    got = call([take(memory) for take in operands], out)
    assert got.data_ptr() == out.data_ptr() and torch.equal(got, want)


@pytest.mark.parametrize("part", [128, 64, 10])
def test_rotary_onto_its_operands_memory(part):
    tokens, heads, dim = 600, 8, 128
    g = generator(part)
    table, positions = onebit.rotary_table(700, part), torch.randint(0, 700, (600,), generator=g).cuda()
    memory = torch.randn((tokens + 1, heads + 1, dim), generator=g).half().cuda()
    turn = lambda x, out: onebit.rotary(x[0], positions, table, out=out)  # noqa: E731
    same_as_apart(turn, memory.clone(), [lambda m: m[1:, :heads]], lambda m: m[1:, 1:])     # a head further on
    same_as_apart(turn, memory.clone(), [lambda m: m[1:, 1:]], lambda m: m[1:, :heads])
    same_as_apart(turn, memory.clone(), [lambda m: m[:-1, :heads]], lambda m: m[1:, :heads])  # a token further on
    square = torch.randn((tokens, tokens // 40, dim), generator=g).half().cuda().view(-1)
    same_as_apart(turn, square, [lambda m: m.view(tokens // 40, tokens, dim).transpose(0, 1)], lambda m: m.view(tokens, tokens // 40, dim))  # other strides
    wide = memory.view(-1)[:tokens * heads * dim]
    same_as_apart(lambda x, out: onebit.rotary(x[0].expand(tokens, heads, dim), positions, table, out=out), wide.clone(),
                  [lambda m: m[dim * heads * 300:dim * heads * 300 + dim]], lambda m: m.view(tokens, heads, dim))  # one head for all
    # apart, though between one another: read in place, and left alone
    pair = torch.randn((tokens, 2 * heads, dim), generator=g).half().cuda()
    before = pair.clone()
    same_as_apart(turn, pair, [lambda m: m[:, :heads]], lambda m: m[:, heads:])
    assert torch.equal(pair[:, :heads], before[:, :heads])
    ids = torch.randn((tokens, heads, dim), generator=g).cuda()
    ids.view(torch.int32).view(-1)[:tokens] = positions.int()
    same_as_apart(lambda o, out: onebit.rotary(ids, o[0].view(torch.int32), table, out=out), ids.clone(), [lambda m: m.view(-1)[:tokens]], lambda m: m)


@pytest.mark.parametrize("new", [1, 150])
def test_attention_onto_its_queries_memory(new):
    case = Case([300] * 4, [new] * 4, 8, 2, 64, 32, E4M3, torch.float16)
    memory = torch.randn((4 * new + 1, 9, 64), generator=generator(new)).half().cuda()
    attend = lambda q, out: case.call(q=q[0], out=out, max_new=new)  # noqa: E731
    same_as_apart(attend, memory.clone(), [lambda m: m[1:, :8]], lambda m: m[1:, 1:])
    same_as_apart(attend, memory.clone(), [lambda m: m[:-1, 1:]], lambda m: m[1:, 1:])
    same_as_apart(attend, memory.clone(), [lambda m: m[1:, 1:]], lambda m: m[1:, 1:])  # the very same


@pytest.mark.parametrize("hidden", [512, 4096, 9000])
def test_block_norm_onto_its_operands_memory(hidden):
    rows = 300
    g = generator(hidden)
    memory = torch.randn((rows + 1, hidden), generator=g).half().cuda()
    other, weight = torch.randn((rows, hidden), generator=g).half().cuda(), torch.randn(hidden, generator=g).half().cuda()

    def check(operands, result, call):
        same_as_apart(lambda o, out: call(o, out)[0], memory.clone(), operands, result)
        now, source = memory.clone(), memory.clone()
        assert torch.equal(call([take(now) for take in operands], result(now))[1], call([take(source).clone() for take in operands], None)[1])

    first, second = (lambda m: m[:-1]), (lambda m: m[1:])
    norm = lambda x, residual, out, **options: onebit.block_norm(x, residual, options.pop("weight", weight), residual_out=out, **options)  # noqa: E731
    check([first], second, lambda o, out: norm(other, o[0], out))             # a residual a row further up
    check([first], second, lambda o, out: norm(o[0], other, out))             # a block's output
    check([first, second], second, lambda o, out: norm(o[0], o[1], out))
    check([second], second, lambda o, out: norm(o[0], other, out))            # the very same
    check([lambda m: m[1:, :1]], second, lambda o, out: norm(other, other, out, gate=o[0]))  # a column of it
    for row in (3, 200):
        take = [lambda m, row=row: m[row]]
        check(take, second, lambda o, out: norm(other, other, out, weight=o[0]))
        check(take, second, lambda o, out: norm(other, other, out, bias=o[0]))
        check(take, second, lambda o, out: norm(other, other, out, post_weight=o[0]))
        check(take, second, lambda o, out: norm(other, other, out, gate=o[0]))
    check([lambda m: m.view(-1)[:hidden * rows].view(hidden, rows).t()], first, lambda o, out: norm(other, o[0], out))  # other strides


def test_block_norm_of_a_residual_in_other_strides_than_its_result():
    """Without a block and with the scale 1 the residual is only to be moved: it is, also where both begin at one address"""
    memory = torch.randn((256, 256), generator=generator(1)).half().cuda()
    weight = torch.ones(256, dtype=torch.float16, device="cuda")
    for residual in (lambda m: m.t(), lambda m: m[:1].expand(256, 256), lambda m: m.view(128, 2, 256)[:, 0]):
        now, source = memory.clone(), memory.clone()
        x = residual(now)
        out = now[:x.shape[0]]
        h, y = onebit.block_norm(None, x, weight, residual_out=out)
        want = residual(source).contiguous()
        assert h.data_ptr() == now.data_ptr() and torch.equal(out, want) and torch.equal(y, onebit.block_norm(None, want, weight)[1])
    kept = memory.clone()
    assert onebit.block_norm(None, kept, weight, residual_out=kept)[0].data_ptr() == kept.data_ptr() and torch.equal(kept, memory)


# ---- the cache's write side


def quantised(values, scale, code):
    x = torch.where(scale > 0, values / torch.where(scale > 0, scale, torch.ones(())), torch.zeros(()))
    return bits(x.round().to(INT8) if code == INT8 else x.to(E4M3))


def appended(k_cache, v_cache, k_scale, v_scale, k, v, pages, lengths, new, code, table, interleaved):
    """The definition in fp32, token by token; the cache's tensors are changed"""
    block, at = k_cache.shape[2], 0
    most = torch.tensor(127.0 if code == INT8 else 448.0)
    for s, (length, n) in enumerate(zip(lengths, new)):
        position = torch.arange(length - n, length)
        fresh_k = k[at:at + n].float()
        if table is not None:
            fresh_k = turned(fresh_k, table[position.clamp(min=0)], interleaved)
        for j in range(max(length - n, 0) // block, -(-length // block)):
            low, high, page = max(length - n, j * block, 0), min(length, (j + 1) * block), int(pages[s, j])
            if low >= high or not 0 <= page < k_cache.shape[0]:
                continue
            for x, cache, scales in ((fresh_k, k_cache, k_scale), (v[at:at + n].float(), v_cache, v_scale)):
                x = x[low - (length - n):high - (length - n)].transpose(0, 1)
                held = scales[page].clone() if low > j * block else torch.zeros(cache.shape[1])
                scale = torch.maximum(held, x.abs().amax((1, 2)) / most)
                old = cache[page, :, :low - j * block]
                if low > j * block:
                    grown = scale != held
                    again = quantised(old.float() * held[:, None, None], scale[:, None, None], code)
                    bits(cache)[page, :, :low - j * block] = torch.where(grown[:, None, None], again, bits(old))
                bits(cache)[page, :, low - j * block:high - j * block] = quantised(x, scale[:, None, None], code)
                scales[page] = scale
        at += n


@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim,block,part,interleaved", [(64, 16, 64, False), (128, 64, 64, True), (128, 128, 128, False), (64, 32, 0, False),
                                                        (128, 32, 128, True)])
def test_append(code, dtype, dim, block, part, interleaved):
    """Several calls of different numbers of tokens, growing and shrinking magnitudes: the codes and scales of the definition to the bit"""
    kv_heads, heads, count = 3, 6, 4
    g = generator(dim + block)
    cache = onebit.QuantizedCache(40, kv_heads, dim, block=block, dtype=code)
    mirror = [t.cpu().clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    mirror[2][:], mirror[3][:] = 50.0, 60.0  # what a page that is handed out again still holds
    cache.k_scale[:], cache.v_scale[:] = 50.0, 60.0
    pages = torch.randperm(40, generator=g)[:count * 10].view(count, 10).to(torch.int32)
    table = onebit.rotary_table(10 * block, part, device="cpu") if part else None
    lengths = [0] * count
    for step, new in enumerate([[7, 1, 20, 0], [1, 1, 1, 1], [block, 2 * block + 3, 0, 5], [1, 0, 2, block - 1], [3, 3, 3, 3], [1, 1, 1, 1]]):
        lengths = [min(a + b, 10 * block) for a, b in zip(lengths, new)]
        tokens = sum(new)
        size = [1.0, 2.0, 0.5, 4.0, 1e-3, 30.0][step]
        q, k, v = (torch.randn((tokens, n, dim), generator=g).mul(size).to(dtype) for n in (heads, kv_heads, kv_heads))
        starts = torch.tensor([sum(new[:i]) for i in range(count + 1)], dtype=torch.int32).cuda()
        got = cache.append(k.cuda(), v.cuda(), pages.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(), starts=None if len(set(new)) == 1 else starts,
                           q=q.cuda() if part else None, rotary=table.cuda() if part else None, interleaved=interleaved,
                           max_new=max(new) if step % 2 else None)
        appended(*mirror, k, v, pages, lengths, new, code, table, interleaved)
        for mine, theirs in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), mirror):
            assert torch.equal(bits(mine.cpu()), bits(theirs)), step
        if part:
            positions = torch.cat([torch.arange(length - n, length) for length, n in zip(lengths, new)])
            assert torch.equal(got.cpu(), turned(q.float(), table[positions], interleaved).to(dtype))
        else:
            assert got is None


@pytest.mark.parametrize("most", [1, 3, 8, 9, 20, 64, 100, 1 << 31])
@pytest.mark.parametrize("dim,block,code", [(64, 64, E4M3), (128, 16, INT8), (64, 128, INT8)])
def test_append_leaves_out_tokens_beyond_max_new(most, dim, block, code):
    """Sequences with more new tokens than the call says: the first of them are written, to the bit, and nothing else; queries are turned all"""
    kv_heads, heads, new, first = 2, 4, [70, 1, 33, 150], [5, 90, 0, 61]
    g = generator(block)
    cache = onebit.QuantizedCache(60, kv_heads, dim, block=block, dtype=code)
    for codes in (cache.k, cache.v):
        bits(codes).copy_(torch.randint(0, 100, codes.shape, generator=g, dtype=torch.uint8))
    cache.k_scale.fill_(0.25)
    cache.v_scale.fill_(0.125)
    mirror = [t.cpu().clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    pages = torch.randperm(60, generator=g).view(4, 15).to(torch.int32)
    table = onebit.rotary_table(240, dim, device="cpu")
    q, k, v = (torch.randn((sum(new), n, dim), generator=g).half() for n in (heads, kv_heads, kv_heads))
    starts = torch.tensor([sum(new[:i]) for i in range(5)], dtype=torch.int32)
    lengths = [a + b for a, b in zip(first, new)]
    got = cache.append(k.cuda(), v.cuda(), pages.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(), starts=starts.cuda(), q=q.cuda(), rotary=table.cuda(),
                       max_new=most)
    left = [min(n, most) for n in new]
    rows = torch.cat([torch.arange(int(s), int(s) + n) for s, n in zip(starts, left)])
    appended(*mirror, k[rows], v[rows], pages, [a + b for a, b in zip(first, left)], left, code, table, False)
    for mine, theirs in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), mirror):
        assert torch.equal(bits(mine.cpu()), bits(theirs))
    positions = torch.cat([torch.arange(a, a + n) for a, n in zip(first, new)])
    assert torch.equal(got.cpu(), turned(q.float(), table[positions], False).to(q.dtype))


def test_append_refuses_keys_and_values_in_one_memory():
    """Attention takes them"""
    cache = onebit.QuantizedCache(4, 2, 64, block=16)
    x = torch.randn((5, 2, 64), generator=generator(1)).half().cuda()
    pages, lengths = torch.zeros((1, 1), dtype=torch.int32, device="cuda"), torch.tensor([5], dtype=torch.int32, device="cuda")
    for v, v_scale in ((cache.k, cache.v_scale), (cache.v, cache.k_scale)):
        with pytest.raises(ValueError, match="share memory"):
            onebit.cache_append(x, x, cache.k, v, cache.k_scale, v_scale, pages, lengths)
    both = torch.zeros((8, 2, 16, 64), dtype=E4M3, device="cuda")
    scales = torch.zeros((8, 2), device="cuda")
    onebit.cache_append(x, x, both[:4], both[4:], scales[:4], scales[4:], pages, lengths)
    cache.append(x, x, pages, lengths)
    assert torch.equal(bits(both)[:4], bits(cache.k)) and torch.equal(bits(both)[4:], bits(cache.v)) and torch.equal(scales[4:], cache.v_scale)
    want = cache.attend(x, pages, lengths)
    assert torch.equal(onebit.cache_attention(x, cache.k, cache.k, cache.k_scale, cache.k_scale, pages, lengths), want)


def test_append_is_as_near_as_its_codes():
    """Against 64 bits: within half a step of the code"""
    for code, relative, absolute in ((E4M3, 2.0**-4, 2.0**-10), (INT8, 0.0, 0.5)):
        cache = onebit.QuantizedCache(4, 2, 64, block=64, dtype=code)
        x = torch.randn((200, 2, 64), generator=generator(2)).half()
        pages = torch.tensor([[2, 0, 3, 1]], dtype=torch.int32)
        cache.append(x.cuda(), x.cuda(), pages.cuda(), torch.tensor([200], dtype=torch.int32).cuda())
        for codes, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
            scale = scale.cpu().double()[pages[0].long()].repeat_interleave(64, 0)[:200, :, None]
            got = decoded(bits(codes.cpu())[pages[0].long()].view(code)).transpose(1, 2).flatten(0, 1)[:200] * scale
            assert bool(((got - x.double()).abs() <= (relative * x.double().abs() + absolute * scale) * (1 + 2.0**-20)).all())


def test_append_of_what_is_not_finite():
    """It is seen by what attends to the page, and by nothing else"""
    for bad in (math.nan, math.inf, -math.inf):
        cache = onebit.QuantizedCache(4, 2, 64, block=16)
        x = torch.randn((40, 2, 64), generator=generator(3)).half()
        pages = torch.tensor([[0, 1, 2]], dtype=torch.int32).cuda()
        clean = onebit.QuantizedCache(4, 2, 64, block=16)
        clean.append(x.cuda(), x.cuda(), pages, torch.tensor([40], dtype=torch.int32).cuda())
        spoilt = x.clone()
        spoilt[20, 1, 5] = bad  # second page, second head
        cache.append(x.cuda(), spoilt.cuda(), pages, torch.tensor([40], dtype=torch.int32).cuda())
        scale = cache.v_scale.cpu()
        assert not math.isfinite(float(scale[1, 1])) and bool(torch.isfinite(scale[[0, 0, 1, 2, 2], [0, 1, 0, 0, 1]]).all())
        assert bool((bits(cache.v)[1, 1] == 0).all()) and torch.equal(bits(cache.v)[[0, 2]], bits(clean.v)[[0, 2]])
        q = torch.randn((40, 2, 64), generator=generator(4)).half().cuda()
        got, want = (c.attend(q, pages, torch.tensor([40], dtype=torch.int32).cuda()) for c in (cache, clean))
        assert torch.equal(got[:, 0], want[:, 0]) and torch.equal(got[:16, 1], want[:16, 1]) and bool(got[16:, 1].isnan().all())


def test_append_writes_only_where_it_may():
    """Missing pages, lengths beyond the table, more new tokens than tokens: nothing else is touched"""
    cache = onebit.QuantizedCache(6, 2, 64, block=16)
    before = [t.cpu().clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    x = torch.ones((30, 2, 64), dtype=torch.float16, device="cuda")
    pages = torch.tensor([[-1, 6], [3, 1 << 30], [5, -2]], dtype=torch.int32).cuda()
    cache.append(x, x, pages, torch.tensor([10, 20, 4], dtype=torch.int32).cuda(), starts=torch.tensor([0, 10, 22, 30], dtype=torch.int32).cuda())
    changed = {3, 5}
    for now, then in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), before):
        for page in range(6):
            assert torch.equal(bits(now.cpu())[page], bits(then)[page]) == (page not in changed)
    # sequence 1: positions 8 ... 19, of which 8 ... 15 have a page; sequence 2: eight rows for four positions
    assert bool((bits(cache.k)[3, :, :8] == 0).all()) and bool((cache.k.float()[3, :, 8:] == 448).all())
    assert bool((cache.k.float()[5, :, :4] == 448).all()) and bool((bits(cache.k)[5, :, 4:] == 0).all())


@pytest.mark.parametrize("code", [E4M3, INT8])
def test_every_code_is_read_and_written_as_torch_does(code):
    """All 256 codes through an append that keeps them (scale 1), and through attention with one key each"""
    every = torch.arange(256, dtype=torch.uint8).view(code).float()
    every = torch.where(every.isnan() | (every == -128), torch.zeros(()), every)
    x = every.view(4, 1, 64).repeat(1, 2, 1)
    x[:, 1] = x[:, 0].flip(0)
    most = 448.0 if code == E4M3 else 127.0
    x[0, :, 0] = most
    cache = onebit.QuantizedCache(4, 2, 64, block=16, dtype=code)
    for t in range(4):  # a page for each token
        x[t, :, 63] = most
    pages = torch.arange(4, dtype=torch.int32).view(4, 1).cuda()
    one = torch.ones(4, dtype=torch.int32, device="cuda")
    cache.append(x.cuda(), x.cuda(), pages, one)
    assert bool((cache.k_scale == 1).all()) and torch.equal(cache.k.float()[:, :, 0].cpu(), x)
    got = cache.attend(torch.ones((4, 2, 64), dtype=torch.float16, device="cuda"), pages, one)
    assert torch.equal(got.float().cpu(), x)


# ---- norms


def norm64(x, weight, bias, kind, eps):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()
    return x if bias is None else x + bias.double()


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("dtype,residual_dtype,weight_dtype", [(torch.float16, torch.float16, torch.float16), (torch.bfloat16, torch.float32, torch.float32),
                                                               (torch.float32, torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16, torch.bfloat16),
                                                               (torch.float16, torch.float32, torch.float16)])
@pytest.mark.parametrize("rows,hidden", [(1, 512), (3, 1), (5, 7), (2, 1000), (4, 4096), (300, 1408), (2, 8200), (2, 11008), (2, 20001), (1, 32768)])
def test_block_norm(kind, dtype, residual_dtype, weight_dtype, rows, hidden):
    g = generator(hidden)
    normal = lambda *shape: torch.randn(shape, generator=g)  # noqa: E731
    x, residual = normal(rows, hidden).mul(2).to(dtype), normal(rows, hidden).mul(3).to(residual_dtype)
    weight, bias, post_weight, post_bias = ((1 + 0.1 * normal(hidden)).to(weight_dtype) for _ in range(4))
    cuda = lambda t: None if t is None else t.cuda()  # noqa: E731
    for gate, use_post, use_bias in ((None, False, False), (normal(hidden).to(dtype), True, True), (normal(rows, 1).to(torch.float32), False, True),
                                     (normal(rows, hidden).to(dtype), True, False)):
        options = dict(kind=kind, eps=1e-5, residual_scale=0.75, block_scale=-1.5)
        h, y = onebit.block_norm(x.cuda(), residual.cuda(), weight.cuda(), bias=cuda(bias if use_bias else None),
                                 post_weight=cuda(post_weight if use_post else None), post_bias=cuda(post_bias if use_post and use_bias else None),
                                 gate=cuda(gate), **options)
        block = x.double()
        terms = block.abs()  # what fp32 rounds: the terms of the sum, where they cancel too
        if use_post:
            unbiased = norm64(block, post_weight, None, kind, 1e-5)
            block = unbiased + post_bias.double() if use_bias else unbiased
            terms = unbiased.abs() + (post_bias.double().abs() if use_bias else 0)
        if gate is not None:
            block, terms = block * gate.double(), terms * gate.double().abs()
        want = 0.75 * residual.double() - 1.5 * block
        assert h.dtype == residual_dtype and y.dtype == dtype
        # fp32 sums of up to 32768 squares, pairwise in part: 2^-18 of a norm's result is far above what they lose
        size = 0.75 * residual.double().abs() + 1.5 * terms
        spread = want.abs().amax(-1, keepdim=True)
        assert bool(((h.cpu().double() - want).abs() <= U[residual_dtype] * want.abs() + 2.0**-18 * size + 2.0**-25).all())
        normed = norm64(want, weight, bias if use_bias else None, kind, 1e-5)
        scale = (want - want.mean(-1, keepdim=True) if kind == "layer" else want).square().mean(-1, keepdim=True).add(1e-5).sqrt()
        slack = 2.0**-18 * (normed.abs() + 2 * (size + spread) / scale + 2)
        assert bool(((y.cpu().double() - normed).abs() <= U[dtype] * normed.abs() * (1 + 2.0**-8) + slack).all())


def test_block_norm_views_shapes_and_in_place():
    g = generator(0)
    x, residual, weight = (torch.randn(s, generator=g).half().cuda() for s in ((2, 5, 512), (2, 5, 512), (512,)))
    h, y = onebit.block_norm(x, residual, weight)
    assert h.shape == y.shape == (2, 5, 512)
    wide = torch.randn((10, 520), generator=g).half().cuda()
    for view in (wide[:, 8:], wide[:, 3:515]):  # aligned rows, rows at odd addresses
        view.copy_(x.view(10, 512))
        h2, y2 = onebit.block_norm(view, residual.view(10, 512), weight)
        assert torch.equal(h2, h.view(10, 512)) and torch.equal(y2, y.view(10, 512))
    assert torch.equal(onebit.block_norm(-(-x), residual, weight)[1], y)
    own = residual.clone()
    h3, y3 = onebit.block_norm(x, own, weight, residual_out=own)
    assert h3.data_ptr() == own.data_ptr() and torch.equal(own, h) and torch.equal(y3, y)
    same, only = onebit.block_norm(None, residual, weight)
    assert same.data_ptr() == residual.data_ptr()
    want = norm64(residual.cpu().double(), weight.cpu(), None, "rms", 1e-5)
    assert bool(((only.cpu().double() - want).abs() <= 2.0**-11 * want.abs() * 1.01 + 2.0**-18).all())
    scaled, _ = onebit.block_norm(None, residual, weight, residual_scale=0.5)
    assert torch.equal(scaled, residual * 0.5)
    assert onebit.block_norm(x, residual, weight, out_dtype=torch.float32)[1].dtype == torch.float32
    one = torch.tensor(0.25, device="cuda")
    assert torch.equal(onebit.block_norm(x, residual, weight, gate=one)[0], onebit.block_norm(x, residual, weight, block_scale=0.25)[0])
    assert torch.equal(onebit.block_norm(x, residual, weight, gate=one.expand(512))[0], onebit.block_norm(x, residual, weight, block_scale=0.25)[0])
    assert onebit.block_norm(x[:0], residual[:0], weight)[1].shape == (0, 5, 512)


@pytest.mark.parametrize("rows,hidden", [(32768, 512), (2048, 8192), (1000, 24000)])
def test_block_norm_of_many_rows_is_that_of_few(rows, hidden):
    """A residual of 64 MB and more is stored in another way: the same values, in place too"""
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    x = torch.randn((rows, hidden), generator=g, device="cuda").bfloat16()
    residual = torch.randn((rows, hidden), generator=g, device="cuda")
    weight = torch.randn(hidden, generator=g, device="cuda")
    h, y = onebit.block_norm(x, residual, weight, post_weight=weight)
    for first in range(0, rows - 512 + 1, rows // 2 - 256 if rows <= 2048 else 8192):
        part = slice(first, first + 512)
        few_h, few_y = onebit.block_norm(x[part], residual[part], weight, post_weight=weight)
        assert torch.equal(h[part], few_h) and torch.equal(y[part], few_y)
    _, again = onebit.block_norm(x, residual, weight, post_weight=weight, residual_out=residual)
    assert torch.equal(residual, h) and torch.equal(again, y)


# ---- together


def test_a_graph_of_a_decoding_step_replays():
    """Captured once, replayed with the eager work and synchronizations of a program in between; each replay is the eager result"""
    g = generator(5)
    count, heads, kv_heads, dim, hidden = 5, 8, 2, 64, 512
    cache, eager = (onebit.QuantizedCache(64, kv_heads, dim, block=16) for _ in range(2))
    pages = torch.arange(60, dtype=torch.int32).view(count, 12).cuda()
    lengths = torch.zeros(count, dtype=torch.int32, device="cuda")
    table = onebit.rotary_table(192, dim)
    qkv = torch.zeros((count, heads + 2 * kv_heads, dim), dtype=torch.float16, device="cuda")
    residual, weight = torch.randn((count, hidden), generator=g).half().cuda(), torch.ones(hidden, dtype=torch.float16, device="cuda")

    def step(c):
        q = c.append(qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:], pages, lengths, q=qkv[:, :heads], rotary=table)
        o = c.attend(q, pages, lengths, max_length=190)
        return onebit.block_norm(o.view(count, hidden), residual, weight) + (o,)

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        lengths.add_(1)
        step(cache)
        stream.synchronize()
        for t in (cache.k, cache.v, cache.k_scale, cache.v_scale):
            t.zero_()
        graph = torch.cuda.CUDAGraph()
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            outputs = step(cache)
    torch.cuda.synchronize()
    lengths.zero_()
    for _ in range(40):
        lengths.add_(1)
        qkv.copy_(torch.randn(qkv.shape, generator=g).half())
        graph.replay()
        torch.cuda.synchronize()
        for mine, theirs in zip(outputs, step(eager)):
            assert torch.equal(mine, theirs)
    assert torch.equal(bits(cache.k), bits(eager.k)) and torch.equal(cache.v_scale, eager.v_scale)


def test_a_decoder_in_pieces_is_the_decoder_in_one_pass():
    """Two layers with their one-bit projections. Pieces that end with pages leave the same cache as one pass, up to what the activations' fp16
    roundings (2^-11, of some ten operators in a row) turn in it: 1 % of the logits' norm at most. Single tokens round the pages that they grow into
    again, each by at most a code's half step (2^-4 of a value) once the page's largest has grown."""
    from onebitsparsemul_amd.decode import Decoder
    ids = torch.randint(0, 4096, (3, 192), generator=generator(7)).cuda()
    whole, pieces, single = (Decoder(2, 3, 192, block=32) for _ in range(3))
    want = whole.step(ids.reshape(-1), 192, 192)
    for begin, end in ((0, 64), (64, 96), (96, 192)):
        got = pieces.step(ids[:, begin:end].reshape(-1), end - begin, end)
    assert float((got - want).norm() / want.norm()) < 0.01
    single.step(ids[:, :160].reshape(-1), 160, 160)
    for t in range(160, 192):
        last = single.step(ids[:, t], 1, t + 1)
    assert float((last - want).norm() / want.norm()) < 2.0**-4
    assert bool((single.lengths == 192).all())
