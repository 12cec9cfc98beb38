"""From the last layer to the next tokens against plain implementations in 64 bits.

u is the unit roundoff of a result's type (fp16 2^-11, bf16 2^-8, fp32 2^-24). Codes are those of the definition in fp32, to the bit, where they come from given values. Products
of codes are exact in fp32; a sum over a group of 128, over the groups and with the scales takes at most 128 + 3 groups + 2 fp32 operations, each off by less than
2^-23 (a matrix unit that cuts off included) of the sum of all magnitudes. 16-bit results of more than 16 tokens come from the 8-bit matrix instruction, which
cuts the products of eight neighbouring columns off at 2^-13 of the largest of them: seven lose less than that each, so that all lose less than 7 2^-13 of the sum of all
magnitudes, and, their signs being mixed, 1.5e-5 of the result's norm over normal values. Tokens are whole: equal to those of sums in 64 bits."""
import math

import pytest
import torch

import onebitsparsemul_amd as onebit

pytestmark = pytest.mark.gpu

U = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}
E4M3 = torch.float8_e4m3fn
DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def generator(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def padded(columns):
    return -(-columns // 128) * 128


def want_codes(x):
    """The definition in fp32, on the host"""
    x = x.float().cpu()
    columns = x.shape[-1]
    x = torch.nn.functional.pad(x.reshape(-1, columns), (0, padded(columns) - columns)).view(-1, padded(columns) // 128, 128)
    largest = x.abs().amax(-1)
    scale = largest / 448
    fine = ((scale > 0) & torch.isfinite(scale))[..., None]
    codes = torch.where(fine, x / torch.where(fine, scale[..., None], 1.0), 0.0).clamp(-448, 448).to(E4M3)
    return codes.flatten(1), scale


def same(a, b):
    """Equal to the bit, NaN with NaN; codes 0 of either sign"""
    a, b = a.cpu().float(), b.cpu().float()
    return a.shape == b.shape and bool(((a == b) | (a.isnan() & b.isnan())).all())


# ---- codes


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,columns", [(1, 1), (1, 7), (3, 127), (2, 128), (5, 129), (17, 512), (33, 1000), (4, 1408), (7, 5001), (300, 8192)])
def test_rows_as_codes(dtype, rows, columns):
    g = generator(columns)
    x = (torch.randn((rows, columns), generator=g) * torch.exp(3 * torch.randn((rows, columns), generator=g))).to(dtype)
    codes, scales = onebit.quantize_rows(x.cuda())
    assert codes.dtype == E4M3 and codes.shape == (rows, padded(columns)) and scales.shape == (rows, padded(columns) // 128)
    want, scale = want_codes(x)
    assert same(codes, want) and same(scales, scale)


def test_rows_of_zeros_of_little_and_of_what_is_not_finite():
    x = torch.randn((8, 300), generator=generator(1))
    x[0] = 0
    x[1, 128:256] = 0
    x[2, 5], x[3, 200], x[4, 299], x[5, 1] = math.nan, math.inf, -math.inf, -math.nan
    x[6] *= 1e-42  # subnormal, and a scale that is 0 or a few of the least
    x[7] *= 1e37
    codes, scales = onebit.quantize_rows(x.cuda())
    want, scale = want_codes(x)
    assert same(codes, want) and same(scales, scale)
    assert bool(torch.isnan(scales[2, 0])) and bool(torch.isinf(scales[3, 1])) and float(scales[0].abs().sum()) == 0
    y = onebit.block_linear(codes, scales, *onebit.quantize_weight(torch.randn((40, 300)).cuda()), out_dtype=torch.float32)
    assert bool(torch.isnan(y[2:6]).all()) and bool(torch.isfinite(y[[0, 1, 6]]).all()) and bool((y[0] == 0).all())


def test_rows_that_are_strided_shaped_or_none():
    x = torch.randn((6, 5, 700), generator=generator(2)).half().cuda()
    base = onebit.quantize_rows(x)
    assert base[0].shape == (6, 5, 768) and base[1].shape == (6, 5, 6)
    for view in (x[:, 2], x[..., 3:131], x[..., ::2], x.transpose(0, 1), x[1:4, :, 1:], x.expand(6, 5, 700), x[:, :, :1], torch._neg_view(x)):
        codes, scales = onebit.quantize_rows(view)
        want, scale = want_codes(view)
        assert same(codes.flatten(0, -2), want) and same(scales.flatten(0, -2), scale)
    assert onebit.quantize_rows(x[0, 0])[0].shape == (768,) and onebit.quantize_rows(x[:0])[1].shape == (0, 5, 6)
    assert onebit.quantize_rows(x[..., :0])[0].shape == (6, 5, 0)


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("rows,hidden,dtype,residual", [(1, 512, torch.float16, torch.float16), (16, 4096, torch.bfloat16, torch.float32), (3, 1000, torch.float32, torch.float32),
                                                        (5, 77, torch.float16, torch.float32), (600, 8192, torch.bfloat16, torch.bfloat16), (2, 20000, torch.float16, torch.float16),
                                                        (2, 32768, torch.float32, torch.float32), (2, 16500, torch.float16, torch.float32), (700, 5000, torch.float16, torch.float16)])
def test_norms_as_codes(kind, post, rows, hidden, dtype, residual):
    """The codes of block_norm's fp32 result, to the bit, and its h"""
    g = generator(hidden + rows)
    make = lambda shape, t, std=1.0: (torch.randn(shape, generator=g) * std).to(t).cuda()  # noqa: E731
    x, r, weight = make((rows, hidden), dtype, 2), make((rows, hidden), residual, 3), make((hidden,), dtype)
    options = dict(bias=make((hidden,), dtype), post_weight=make((hidden,), dtype) if post else None, gate=make((rows, 1), dtype), residual_scale=0.7, block_scale=0.3, kind=kind)
    h, codes, scales = onebit.block_norm_codes(x, r, weight, **options)
    want_h, y = onebit.block_norm(x, r, weight, out_dtype=torch.float32, **options)
    assert torch.equal(h, want_h)
    want, scale = want_codes(y)
    assert same(codes, want) and same(scales, scale)


def test_norms_as_codes_in_place_without_a_block_and_of_what_is_not_finite():
    g = generator(4)
    x, r = (torch.randn((2, 9, 640), generator=g).half().cuda() for _ in range(2))
    weight = torch.randn(640, generator=g).half().cuda()
    h, codes, scales = onebit.block_norm_codes(None, r, weight)
    assert h is not x and torch.equal(h, r) and codes.shape == (2, 9, 640) and scales.shape == (2, 9, 5)
    want, scale = want_codes(onebit.block_norm(None, r, weight, out_dtype=torch.float32)[1])
    assert same(codes.flatten(0, 1), want) and same(scales.flatten(0, 1), scale)
    want = onebit.block_norm_codes(x, r, weight)
    in_place = r.clone()
    got = onebit.block_norm_codes(x, in_place, weight, residual_out=in_place)
    assert torch.equal(got[0], want[0]) and torch.equal(in_place, want[0]) and same(got[1], want[1]) and torch.equal(got[2], want[2])
    x[0, 3, 100] = math.nan
    _, codes, scales = onebit.block_norm_codes(x, r, weight)
    assert bool(torch.isnan(scales[0, 3]).all()) and bool((codes[0, 3].float() == 0).all()) and int(torch.isnan(scales).sum()) == 5
    # a row of the fused projection's output, as the last tokens of sequences are
    last = onebit.block_norm_codes(x[:, -1], r[:, -1], weight)
    assert same(last[1], want[1][:, -1]) and torch.equal(last[0], want[0][:, -1])
    assert onebit.block_norm_codes(x[:, :0], r[:, :0], weight)[1].shape == (2, 0, 640)


# ---- products


def random_codes(rows, columns, g, group_rows=1):
    codes = (torch.randn((rows, columns), generator=g) * 100).clamp(-448, 448).to(E4M3)
    scales = torch.exp(torch.randn((-(-rows // group_rows), columns // 128), generator=g)) * 0.01
    return codes, scales


def check_product(tokens, rows, columns, dtype=torch.float32, bias=False, seed=0, **options):
    g = generator(seed + tokens + rows + columns)
    (x, xs), (w, ws) = random_codes(tokens, columns, g), random_codes(rows, columns, g, 128)
    b = torch.randn(rows, generator=g).to(dtype) if bias else None
    cuda = lambda t: None if t is None else t.cuda()  # noqa: E731
    y = onebit.block_linear(x.cuda(), xs.cuda(), w.cuda(), ws.cuda(), bias=cuda(b), out_dtype=dtype, **options)
    xd = (x.float().double().view(tokens, -1, 128) * xs.double()[..., None]).view(tokens, -1).cuda()
    wd = (w.float().double().view(rows, -1, 128) * ws.double().repeat_interleave(128, 0)[:rows, :, None]).view(rows, -1).cuda()
    want, size = xd @ wd.T.contiguous(), xd.abs() @ wd.abs().T.contiguous()
    if bias:
        want, size = want + b.double().cuda(), size + b.double().abs().cuda()
    error = (y.double() - want).abs()
    bound = U[dtype] * (1 + 2.0**-10) * want.abs() + (130 + 3 * (columns // 128)) * 2.0**-23 * size
    cut = 7 * 2.0**-13 * size if dtype != torch.float32 and tokens > 16 else 0 * size
    if dtype == torch.float16:
        bound = bound + 2.0**-25
        # a value rounds to infinity from 65520 on, half a step above the largest: the sum before its rounding is off by the bound without that rounding, and all beyond 65504 + 32 + that are infinite
        before, infinite = (130 + 3 * (columns // 128)) * 2.0**-23 * size + cut, y.isinf()
        assert bool((want.abs() >= 65520 - before)[infinite].all()) and bool(infinite[want.abs() > 65520 + before].all()) and torch.equal(y[infinite].sign().double(), want[infinite].sign())
        y, want, error = torch.where(infinite, 0, y), torch.where(infinite, 0, want), torch.where(infinite, 0, error)
    if dtype != torch.float32 and tokens > 16:
        bound = bound + cut
        # (a rounding is off by u / sqrt(3) at most on average)
        assert float(error.norm()) <= (U[dtype] / math.sqrt(3) + 2.0**-13) * float(want.norm())
    assert y.dtype == dtype and y.shape == (tokens, rows) and bool(torch.isfinite(y).all())
    assert bool((error <= bound).all()), float((error / bound).max())
    return y


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens", [1, 2, 3, 5, 8, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 100, 127, 128, 129, 200, 256, 257, 500])
def test_products_by_tokens(tokens, dtype):
    check_product(tokens, 300, 640, dtype, bias=tokens % 2 == 0)


@pytest.mark.parametrize("tokens", [1, 4, 16, 20, 64, 90, 300])
@pytest.mark.parametrize("rows", [1, 3, 15, 16, 17, 64, 100, 127, 128, 129, 255, 257, 1000, 4099])
def test_products_by_rows(tokens, rows):
    check_product(tokens, rows, 256, torch.float16 if rows % 2 else torch.float32, bias=rows % 3 == 0)


@pytest.mark.parametrize("tokens", [1, 16, 37, 64, 150, 513])
@pytest.mark.parametrize("columns", [128, 256, 384, 1408, 4096, 5120, 11008, 28672])
def test_products_by_columns(tokens, columns):
    check_product(tokens, 200, columns, torch.bfloat16 if columns % 256 else torch.float32, bias=True)


@pytest.mark.parametrize("tokens,rows,columns", [(2048, 4096, 1024), (1000, 11008, 512), (16, 32000, 2048), (1, 131072, 256), (64, 50000, 512), (4096, 300, 2048), (700, 3000, 4096)])
def test_large_products(tokens, rows, columns):
    check_product(tokens, rows, columns, torch.float16)


@pytest.mark.parametrize("tokens,rows,columns", [(1, 64, 512), (16, 200, 1024), (40, 130, 2048), (64, 1000, 512), (129, 515, 640), (600, 700, 1152), (2000, 4000, 384)])
def test_products_of_whole_numbers_are_exact(tokens, rows, columns):
    """Codes -8 ... 8 with scales that are powers of two: sums are whole numbers below 2^24 of one unit: to the bit, whatever the order"""
    g = generator(tokens)
    x, w = (torch.randint(-8, 9, (n, columns), generator=g).float() for n in (tokens, rows))
    xs = 2.0 ** torch.randint(0, 2, (tokens, columns // 128), generator=g)
    ws = 2.0 ** torch.randint(0, 2, (-(-rows // 128), columns // 128), generator=g)
    y = onebit.block_linear(x.to(E4M3).cuda(), xs.cuda(), w.to(E4M3).cuda(), ws.cuda(), out_dtype=torch.float32)
    xd = x.double() * xs.double().repeat_interleave(128, 1)
    wd = w.double() * ws.double().repeat_interleave(128, 0)[:rows].repeat_interleave(128, 1)
    assert torch.equal(y.double().cpu(), xd @ wd.T)


# (each of the kernels and splits that the plan takes, among them whole rounds of tiles of 256 x 256 with what is left in halves)
KERNELS = [(1, 4099, 11008), (16, 900, 14336), (9, 11008, 2048), (20, 37000, 512), (17, 33000, 4096), (20, 37001, 1408), (33, 4099, 8192), (100, 2304, 4096), (128, 11008, 1408),
           (333, 4099, 1408), (1000, 8192, 640), (200, 37000, 512), (2048, 8192, 512), (512, 37000, 640), (2048, 11008, 512), (2049, 9001, 512), (4096, 4099, 1024), (3000, 7000, 640)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,rows,columns", KERNELS)
def test_products_of_every_kernel(tokens, rows, columns, dtype):
    check_product(tokens, rows, columns, dtype, bias=rows % 2 == 1)


@pytest.mark.parametrize("tokens,rows,columns", [shape for shape in KERNELS if shape[2] <= 1024] + [(1, 131072, 512), (70, 50257, 512)])
def test_small_whole_numbers_are_exact_in_any_type(tokens, rows, columns):
    """Codes -1 ... 1 and scales 1: sums of at most 1024, whole in fp16 and, below 256, in bf16, and no product below another's 2^-13"""
    g = generator(tokens)
    x, w = (torch.randint(-1, 2, (n, columns), generator=g).float().cuda() for n in (tokens, rows))
    xs, ws = torch.ones((tokens, columns // 128), device="cuda"), torch.ones((-(-rows // 128), columns // 128), device="cuda")
    want = x.double() @ w.double().T.contiguous()
    x, w = x.to(E4M3), w.to(E4M3)
    for dtype in DTYPES:
        assert torch.equal(onebit.block_linear(x, xs, w, ws, out_dtype=dtype), want.to(dtype))


def test_products_of_rows_far_apart():
    """Weights 2^24 codes apart, with an offset beyond 32 bits"""
    g = generator(5)
    (x, xs), (w, ws) = random_codes(40, 640, g), random_codes(300, 640, g, 128)
    x, xs, w, ws = x.cuda(), xs.cuda(), w.cuda(), ws.cuda()
    apart = torch.empty((300, 1 << 24), dtype=torch.uint8, device="cuda")
    apart[:, 64:704] = w.view(torch.uint8)
    want = onebit.block_linear(x, xs, w, ws, out_dtype=torch.float32)
    got = onebit.block_linear(x, xs, apart[:, 64:704].view(E4M3), ws, out_dtype=torch.float32)
    assert float((got - want).norm() / want.norm()) < 1e-5  # (fp32 sums in another order)


def test_products_of_views_into_given_results():
    g = generator(3)
    (x, xs), (w, ws) = random_codes(24, 1024, g), random_codes(333, 1024, g, 128)
    x, xs, w, ws = x.cuda(), xs.cuda(), w.cuda(), ws.cuda()
    want = onebit.block_linear(x, xs, w, ws)
    as_bytes = x.view(torch.uint8)
    wide = torch.full((24, 1040), 0x7f, dtype=torch.uint8, device="cuda")
    wide[:, 16:] = as_bytes
    odd = torch.full((24, 1031), 0x7f, dtype=torch.uint8, device="cuda")
    odd[:, 7:] = as_bytes
    for view in (wide[:, 16:], odd[:, 7:], as_bytes.T.contiguous().T, as_bytes.view(4, 6, 1024)):
        scales = xs.view(4, 6, 8) if view.dim() == 3 else xs.T.contiguous().T
        got = onebit.block_linear(view.view(E4M3) if view.is_contiguous() else view.view(E4M3), scales, w, ws)
        assert torch.equal(got.view(24, 333), want)
    for shape, stride, offset in (((24, 333), (333, 1), 0), ((24, 333), (340, 1), 3), ((24, 333), (336, 1), 8), ((24, 333), (1, 24), 0)):
        room = torch.full((24 * 400,), 9.0, dtype=torch.float16, device="cuda")
        out = room.as_strided(shape, stride, offset)
        if stride[1] != 1:
            with pytest.raises(ValueError, match="whole rows"):
                onebit.block_linear(x, xs, w, ws, out=out)
            continue
        assert onebit.block_linear(x, xs, w, ws, out=out) is not None and torch.equal(out, want)
        out.fill_(9.0)
        assert bool((room == 9).all())  # nothing beside
    # weights whose rows lie apart, a part of a weight's rows
    apart = torch.zeros((333, 1056), dtype=torch.uint8, device="cuda")
    apart[:, 32:] = w.view(torch.uint8)
    assert torch.equal(onebit.block_linear(x, xs, apart[:, 32:].view(E4M3), ws), want)
    assert torch.equal(onebit.block_linear(x, xs, w[128:300], ws[1:3]), want[:, 128:300])
    # none
    assert onebit.block_linear(x[:0], xs[:0], w, ws).shape == (0, 333) and onebit.block_linear(x, xs, w[:0], ws[:0]).shape == (24, 0)
    assert onebit.block_linear(x[0], xs[0], w, ws).shape == (333,) and torch.equal(onebit.block_linear(x[0], xs[0], w, ws), onebit.block_linear(x[:1], xs[:1], w, ws)[0])


@pytest.mark.parametrize("tokens", [1, 16, 30, 64, 65, 300])
def test_what_is_not_finite_stays_in_its_token(tokens):
    g = generator(8)
    (x, xs), (w, ws) = random_codes(tokens, 512, g), random_codes(200, 512, g, 128)
    clean = onebit.block_linear(x.cuda(), xs.cuda(), w.cuda(), ws.cuda())
    xs[tokens // 2, 1] = math.nan
    x.view(torch.uint8)[tokens // 2, 128:256] = 0
    got = onebit.block_linear(x.cuda(), xs.cuda(), w.cuda(), ws.cuda())
    others = [t for t in range(tokens) if t != tokens // 2]
    assert bool(torch.isnan(got[tokens // 2]).all()) and torch.equal(got[others], clean[others])
    # a code that is NaN, of a token and of a weight's row
    xs[tokens // 2, 1] = 1.0
    x.view(torch.uint8)[tokens // 2, 200] = 0x7f
    got = onebit.block_linear(x.cuda(), xs.cuda(), w.cuda(), ws.cuda())
    assert bool(torch.isnan(got[tokens // 2]).all()) and torch.equal(got[others], clean[others])
    x.view(torch.uint8)[tokens // 2, 200] = 0
    w.view(torch.uint8)[77, 500] = 0xff
    got = onebit.block_linear(x.cuda(), xs.cuda(), w.cuda(), ws.cuda())
    assert bool(torch.isnan(got[:, 77]).all()) and torch.equal(got[others][:, :77], clean[others][:, :77]) and torch.equal(got[others][:, 78:], clean[others][:, 78:])


@pytest.mark.parametrize("tokens", [1, 3, 16, 17, 64, 200])
def test_a_token_of_a_batch_is_that_token_alone_on_codes(tokens):
    """Up to the order of fp32 sums"""
    g = generator(tokens)
    (x, xs), (w, ws) = random_codes(tokens, 1024, g), random_codes(500, 1024, g, 128)
    x, xs, w, ws = x.cuda(), xs.cuda(), w.cuda(), ws.cuda()
    together = onebit.block_linear(x, xs, w, ws, out_dtype=torch.float32)
    alone = torch.cat([onebit.block_linear(x[t:t + 1], xs[t:t + 1], w, ws, out_dtype=torch.float32) for t in range(0, tokens, 7)])
    assert float((together[::7] - alone).norm() / alone.norm()) < 1e-5


def test_layers():
    g = generator(6)
    weight, bias = torch.randn((520, 700), generator=g), torch.randn(520, generator=g)
    layer = onebit.BlockLinear(weight.cuda(), bias=bias.cuda())
    x = torch.randn((3, 11, 700), generator=g).half().cuda()
    y = layer(x)
    codes, scales = onebit.quantize_rows(x)
    assert y.dtype == torch.float16 and y.shape == (3, 11, 520) and torch.equal(y, layer((codes, scales)))
    assert torch.equal(y, onebit.block_linear(codes, scales, layer.codes, layer.scales, bias=layer.bias))
    # codes of x and of the weight are off by half a step each, 2^-4: of all values at most that, and both of them
    size = x.double().abs() @ weight.double().abs().T.cuda()
    assert bool(((y.double() - (x.double() @ weight.double().T.cuda() + bias.double().cuda())).abs() <= 0.14 * size + 0.01).all())
    assert onebit.BlockLinear(weight.cuda(), out_dtype=torch.float32)(x).dtype == torch.float32 and layer(x.float()).dtype == torch.float32


# ---- tokens


def plain_tokens(logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """From the definition, row by row in 64 bits"""
    logits, uniform, out = logits.double().cpu(), uniform.double().cpu(), []
    for r in range(logits.shape[0]):
        t, k, p, m = (float(v[r]) if isinstance(v, torch.Tensor) else float(torch.tensor(float(v))) for v in (temperature, top_k, top_p, min_p))
        row = logits[r]
        if bool(row.isnan().any()) or float(row.max()) == -math.inf:
            out.append(-1)
            continue
        order = torch.sort(row, descending=True, stable=True).indices
        if not t > 0:
            out.append(int(order[0]))
            continue
        top = row[order[0]]
        w = torch.where(row == top, 1.0, torch.exp((row - top) / t))[order]
        if k > 0:
            w = w[:int(k)]
        if p < 1:
            in_front = torch.cat([w.new_zeros(1), w.cumsum(0)[:-1]])
            w = w[:max(1, int((in_front < p * w.sum()).sum()))]
        w = w[:max(1, int((w >= m).sum()))]
        kept, place = order[:len(w)].sort()
        w = w[place]
        running = w.cumsum(0)
        u = float(uniform[r]) if float(uniform[r]) > 0 else 0.0
        at = int((running <= u * running[-1]).sum())
        out.append(int(kept[min(at, int((w > 2.0**-43).nonzero()[-1]))]))  # (weights below half of 2^-42 are 0)
    return out


def check_tokens(logits, uniform, **options):
    cuda = lambda v: v.cuda() if isinstance(v, torch.Tensor) else v  # noqa: E731
    got = onebit.sample(logits.cuda(), uniform.cuda(), **{k: cuda(v) for k, v in options.items()})
    assert got.dtype == torch.int64 and got.shape == logits.shape[:-1]
    want = plain_tokens(logits, uniform, **options)
    assert got.tolist() == want, [(r, a, b) for r, (a, b) in enumerate(zip(got.tolist(), want)) if a != b][:5]
    return got


def random_logits(rows, vocabulary, g, dtype, spread=3.0):
    return (torch.randn((rows, vocabulary), generator=g) * spread).to(dtype)


FILTERS = [dict(), dict(temperature=0.7), dict(top_k=1), dict(top_k=5), dict(top_k=50, temperature=1.3), dict(top_p=0.9), dict(top_p=0.3, temperature=0.5), dict(min_p=0.05),
           dict(top_k=40, top_p=0.95, min_p=0.02, temperature=0.8), dict(temperature=0.0), dict(top_k=10**6), dict(top_p=0.0), dict(min_p=1.0), dict(min_p=2.0),
           dict(top_p=0.999, temperature=2.0), dict(top_k=1000, top_p=0.99), dict(temperature=100.0), dict(temperature=1e-6, top_p=0.9)]


@pytest.mark.parametrize("options", FILTERS, ids=str)
@pytest.mark.parametrize("vocabulary", [1, 2, 63, 64, 65, 1000, 4096, 32000])
@pytest.mark.parametrize("dtype", DTYPES)
def test_tokens(options, vocabulary, dtype):
    g = generator(vocabulary)
    check_tokens(random_logits(7, vocabulary, g, dtype), torch.rand(7, generator=g), **options)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocabulary", [(1, 131072), (40, 50257), (300, 1500), (3, 131071), (2, 1 << 20)])
def test_tokens_with_parameters_of_their_own(rows, vocabulary, dtype):
    g = generator(rows)
    logits = random_logits(rows, vocabulary, g, dtype)
    share = lambda: torch.rand(rows, generator=g)  # noqa: E731
    pick = lambda *values: torch.tensor(values)[torch.randint(0, len(values), (rows,), generator=g)]  # noqa: E731
    for _ in range(2):
        check_tokens(logits, share(), temperature=pick(0.0, 0.5, 1.0, 3.0), top_k=pick(0, 1, 30, 2000, 1 << 30).int(), top_p=pick(0.2, 0.9, 0.999, 1.0), min_p=pick(0.0, 0.01, 0.3))
        check_tokens(logits, share(), temperature=share() + 0.5, top_p=share())


@pytest.mark.parametrize("options", [dict(top_k=300), dict(top_k=700, top_p=0.9), dict(top_k=3000, top_p=0.5), dict(top_k=20000), dict(top_p=0.5), dict(top_p=0.95), dict(top_p=0.9995),
                                     dict(top_p=0.99, min_p=0.001), dict(min_p=0.01), dict(top_p=0.9, temperature=1.5)], ids=str)
@pytest.mark.parametrize("kind", ["spread", "flat", "two values", "steps", "ranks"])
@pytest.mark.parametrize("vocabulary", [3000, 8000, 40001, 131072])
def test_many_candidates(vocabulary, kind, options):
    """Lists of some hundred, of thousands, and rows that keep more than a list holds; bins full of equal logits"""
    g = generator(vocabulary)
    rows = 4
    ranks = torch.argsort(torch.rand((rows, vocabulary), generator=g), dim=1).float()
    logits = {"spread": lambda: torch.randn((rows, vocabulary), generator=g) * 2.5, "flat": lambda: torch.randn((rows, vocabulary), generator=g) * 0.3,
              "two values": lambda: (torch.rand((rows, vocabulary), generator=g) < 0.3).float() * 2, "steps": lambda: (torch.randn((rows, vocabulary), generator=g) * 8).round() / 4,
              "ranks": lambda: 12 - torch.tensor([1.0, 1.2, 1.5, 0.8])[:, None] * torch.log(ranks + 1)}[kind]()
    check_tokens(logits, torch.rand(rows, generator=g), **options)
    check_tokens(logits.bfloat16(), torch.rand(rows, generator=g), **options)


@pytest.mark.parametrize("dtype", DTYPES)
def test_equal_logits_go_by_index(dtype):
    """All equal, and few values: borders that fall on whole masses, ties that a filter takes in part"""
    g = generator(1)
    u = torch.tensor([0.0, 0.25, 0.5, 0.75, 0.999999])
    for value in (0.0, -0.0, 5.0, -60000.0):
        flat = torch.full((5, 1000), value).to(dtype)
        for options in (dict(), dict(top_k=7), dict(top_p=0.5), dict(top_k=64, top_p=0.25), dict(min_p=1.0), dict(temperature=0.0), dict(top_k=999)):
            check_tokens(flat, u, **options)
    signs = torch.where(torch.rand((5, 3000), generator=g) < 0.5, 0.0, -0.0).to(dtype)
    check_tokens(signs, u, top_k=1500)
    check_tokens(signs, u, temperature=0.0)
    few = torch.randint(0, 4, (5, 20000), generator=g).to(dtype)
    for options in (dict(), dict(top_k=100), dict(top_k=4990), dict(top_k=7000), dict(top_p=0.31), dict(top_k=9000, top_p=0.8), dict(min_p=0.2, top_p=0.9), dict(top_p=0.7, temperature=0.25)):
        check_tokens(few, u, **options)


@pytest.mark.parametrize("dtype", DTYPES)
def test_hidden_tokens(dtype):
    g = generator(2)
    logits = random_logits(9, 5000, g, dtype)
    logits[0, :] = -math.inf
    logits[1, :] = -math.inf
    logits[1, 4321] = -3.0
    logits[2, torch.rand(5000, generator=g) < 0.99] = -math.inf
    logits[3, 17] = math.nan
    logits[4, 4999] = -math.nan
    logits[5, [3, 400, 4000]] = math.inf
    logits[6, 0] = math.inf
    logits[7, :] = math.nan
    logits[8, 1:] = -math.inf
    least = torch.finfo(dtype).min
    for options in FILTERS:
        for u in (0.0, 0.4, 0.999):
            check_tokens(logits, torch.full((9,), u), **options)
    logits = torch.where(torch.rand((9, 5000), generator=g) < 0.9, least, random_logits(9, 5000, g, torch.float32)).to(dtype)  # a mask of the type's lowest value
    logits[0, :] = least
    for options in FILTERS:
        check_tokens(logits, torch.rand(9, generator=g), **options)


def test_random_numbers_at_and_beyond_their_ends():
    logits = random_logits(6, 700, generator(3), torch.float32)
    logits[:, -1] = -math.inf
    logits[:, -2] = -200.0  # a weight that rounds to 0
    u = torch.tensor([0.0, 1.0, 1.5, -1.0, math.inf, 1 - 2.0**-24])
    first, second = check_tokens(logits, u), check_tokens(logits, u, top_k=10)
    nan = onebit.sample(logits.cuda(), torch.full((6,), math.nan, device="cuda"))
    assert torch.equal(nan, onebit.sample(logits.cuda(), torch.zeros(6, device="cuda"))) and first.shape == second.shape


@pytest.mark.parametrize("place", ["front", "end", "sorted", "falling"])
def test_the_largest_logits_side_by_side(place):
    """What a filter keeps lies in one stretch of the row"""
    g = generator(4)
    logits = random_logits(4, 40000, g, torch.float32, 1.0)
    if place in ("sorted", "falling"):
        logits = logits.sort(-1, descending=place == "falling").values
    else:
        logits[:, slice(0, 3000) if place == "front" else slice(-3000, None)] += 12.0
    for options in (dict(top_k=50), dict(top_k=2500), dict(top_p=0.9), dict(min_p=0.01), dict(top_k=3500, top_p=0.999)):
        check_tokens(logits, torch.rand(4, generator=g), **options)


def test_logits_that_are_strided_shaped_or_none():
    g = generator(5)
    logits, u = random_logits(12, 1001, g, torch.float16).view(3, 4, 1001).cuda(), torch.rand((3, 4), generator=g).cuda()
    want = onebit.sample(logits, u, top_k=20)
    assert want.shape == (3, 4)
    room = torch.full((12, 1100), math.nan, dtype=torch.float16, device="cuda")
    for first in (0, 1, 3, 8):
        room[:, first:first + 1001] = logits.view(12, 1001)
        assert torch.equal(onebit.sample(room[:, first:first + 1001], u.view(12), top_k=20), want.view(12))
        room.fill_(math.nan)
    assert torch.equal(onebit.sample(logits.transpose(0, 1), u.T.contiguous(), top_k=20), want.T)
    assert torch.equal(onebit.sample(logits.flip(-1).flip(-1), u, top_k=20), want)
    spread = torch.empty((3, 4, 2002), dtype=torch.float16, device="cuda")
    spread[..., ::2] = logits
    assert torch.equal(onebit.sample(spread[..., ::2], u, top_k=20), want) and torch.equal(onebit.sample(torch._neg_view(-logits), u, top_k=20), want)
    one = onebit.sample(logits[0, 0], u[0, 0], top_k=20)
    assert one.shape == () and int(one) == int(want[0, 0])
    assert torch.equal(onebit.sample(logits[:1, :1].expand(3, 4, 1001), u, top_k=20), torch.stack([onebit.sample(logits[0, 0], v, top_k=20) for v in u.view(-1)]).view(3, 4))
    assert onebit.sample(logits[:0], u[:0]).shape == (0, 4)


def test_shares_of_many_draws():
    """65536 evenly spaced numbers: a token has its share of them, to one of them at each end"""
    logits = random_logits(1, 50, generator(6), torch.float32, 1.5)
    u = (torch.arange(65536) + 0.5) / 65536
    tokens = onebit.sample(logits.expand(65536, 50).cuda(), u.cuda(), temperature=0.9)
    share = torch.bincount(tokens.cpu(), minlength=50).double() / 65536
    assert float((share - torch.softmax(logits[0].double() / float(torch.tensor(0.9)), 0)).abs().max()) <= 2 / 65536


# ---- together


def head_step(x, residual, weight, layer, u, **options):
    h, codes, scales = onebit.block_norm_codes(x, residual, weight)
    logits = layer((codes, scales))
    return h, codes, scales, logits, onebit.sample(logits, u, **options)


@pytest.mark.parametrize("count", [1, 5, 16, 70])
def test_a_graph_of_the_last_steps_replays(count):
    """Captured once, replayed with a program's eager work and synchronizations in between; each replay is the eager result"""
    g = generator(count)
    layer = onebit.BlockLinear(torch.randn((3000, 512), generator=g).cuda())
    weight = torch.ones(512, dtype=torch.float16, device="cuda")
    x, residual = (torch.zeros((count, 512), dtype=torch.float16, device="cuda") for _ in range(2))
    u = torch.zeros(count, device="cuda")
    options = dict(temperature=torch.full((count,), 0.8, device="cuda"), top_k=40, top_p=0.95, min_p=0.01)
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        head_step(x, residual, weight, layer, u, **options)
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            outputs = head_step(x, residual, weight, layer, u, **options)
    torch.cuda.synchronize()
    for _ in range(12):
        x.copy_(torch.randn(x.shape, generator=g).half())
        residual.copy_(torch.randn(x.shape, generator=g).half())
        u.copy_(torch.rand(count, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        for mine, theirs in zip(outputs, head_step(x, residual, weight, layer, u, **options)):
            assert same(mine, theirs)
        torch.zeros(1000, device="cuda").sum().item()


def test_two_streams_at_once():
    g = generator(9)
    layer = onebit.BlockLinear(torch.randn((2000, 1024), generator=g).cuda())
    weight = torch.ones(1024, dtype=torch.float16, device="cuda")
    inputs = [(torch.randn((n, 1024), generator=g).half().cuda(), torch.randn((n, 1024), generator=g).half().cuda(), torch.rand(n, generator=g).cuda()) for n in (1, 16, 40, 300)]
    want = [head_step(x, r, weight, layer, u, top_p=0.9) for x, r, u in inputs]
    streams = [torch.cuda.Stream() for _ in inputs]
    torch.cuda.synchronize()
    got = [[] for _ in inputs]
    for _ in range(5):
        for i, (x, r, u) in enumerate(inputs):
            with torch.cuda.stream(streams[i]):
                got[i].append(head_step(x, r, weight, layer, u, top_p=0.9))
    torch.cuda.synchronize()
    for i, results in enumerate(got):
        for result in results:
            assert all(same(a, b) for a, b in zip(result, want[i]))


def test_a_decoder_answers_with_tokens():
    """Norm, codes, product and sampling behind two layers of one-bit projections, as decode.py runs them: the logits are those of the plain forms from the same rows, tokens those that
    their logits give, and a decoder that is given the drawn tokens in one pass comes to the same caches' lengths"""
    from onebitsparsemul_amd.decode import Decoder
    g = generator(3)
    prompt = torch.randint(0, 4096, (5, 48), generator=g).cuda()
    uniform = torch.rand((9, 5), generator=g).cuda()
    options = dict(temperature=0.9, top_k=40, top_p=0.9, min_p=0.01)
    decoder, again, plain = Decoder(2, 5, 64, block=16, head="e4m3"), Decoder(2, 5, 64, block=16, head="e4m3"), Decoder(2, 5, 64, block=16)
    tokens = decoder.generate(prompt, uniform, **options)
    assert tokens.shape == (5, 9) and bool((decoder.lengths == 48 + 8).all()) and bool(((tokens >= 0) & (tokens < 4096)).all())
    ids, new = prompt.reshape(-1), 48
    for step in range(9):
        logits = again.step(ids, new, 48 + step)
        assert logits.dtype == torch.float32 and tokens[:, step].tolist() == plain_tokens(logits, uniform[step], **options)
        ids, new = tokens[:, step], 1
    # codes of both sides are off by 2^-4 at most, their products' errors of mixed signs: far within 2^-4 of the logits' norm
    first, want = Decoder(2, 5, 64, block=16, head="e4m3").step(prompt.reshape(-1), 48, 48), plain.step(prompt.reshape(-1), 48, 48)
    assert float((first - want).norm() / want.norm()) < 2.0**-4
    assert Decoder(1, 2, 64, head="e4m3").generate(prompt[:2], uniform[:0]).shape == (2, 0)
    with pytest.raises(ValueError, match="head must be"):
        Decoder(1, 2, 64, head="int8")


def test_the_command_draws_tokens(capsys):
    from onebitsparsemul_amd import decode
    decode.main(["--layers", "1", "--sequences", "3", "--prompt", "33", "--tokens", "4", "--head", "e4m3"])
    assert "4 tokens drawn behind the prompt" in capsys.readouterr().out


@pytest.mark.parametrize("count", [1, 17])
def test_two_graphs_of_one_call_keep_apart(count):
    """Two captured calls with a workspace each, replayed in turn and together with an eager one"""
    g = generator(count)
    (x, xs), (w, ws) = random_codes(64, 8192, g), random_codes(100, 8192, g, 128)  # groups split over workgroups
    x, xs, w, ws = x.cuda(), xs.cuda(), w.cuda(), ws.cuda()
    logits, u = random_logits(count, 40000, g, torch.float16).cuda(), torch.rand(count, generator=g).cuda()
    inputs = [(x, logits), (x.flip(0).contiguous(), logits.flip(1).contiguous())]

    def call(codes, row):
        return onebit.block_linear(codes, xs, w, ws), onebit.sample(row, u, top_p=0.9)

    want = [call(*i) for i in inputs]
    stream = torch.cuda.Stream()
    graphs, results = [torch.cuda.CUDAGraph() for _ in inputs], []
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        for graph, i in zip(graphs, inputs):
            with torch.cuda.graph(graph, stream=stream):
                results.append(call(*i))
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    for _ in range(6):
        graphs[0].replay()
        with torch.cuda.stream(other):
            graphs[1].replay()
        eager = call(*inputs[0])
        torch.cuda.synchronize()
        for got, expected in zip([*results, eager], [*want, want[0]]):
            assert all(torch.equal(a, b) for a, b in zip(got, expected))


# ---- rows of several chunks of 4096 logits without a filter


@pytest.mark.parametrize("vocabulary", [700, 8193, 40000, 131072])
def test_a_random_number_that_is_none_counts_as_0(vocabulary):
    logits = random_logits(3, vocabulary, generator(vocabulary), torch.float32)
    u = torch.tensor([math.nan, -1.0, 0.0])
    for options in (dict(), dict(top_k=10), dict(top_p=0.9), dict(min_p=0.1)):
        assert plain_tokens(logits, u, **options) == plain_tokens(logits, torch.zeros(3), **options)
        check_tokens(logits, u, **options)


def test_a_number_between_two_chunks_sums():
    """Three chunks' masses a, b, c in 2^-42, a = b + c, whole numbers below 2^53. uniform 0.5 of a + b + c = 2 a is a, which the first chunk's sum does not exceed: the token is the second chunk's
    first. a + b is beyond 2^53 and lies between two doubles, of which the upper one is even: less b it is a + 1, which is where the second chunk seems to begin."""
    chunk, least = 4096, -42 * math.log(2)  # a weight of 1
    row = torch.full((1, 4 * chunk), -math.inf)
    row[0, chunk + 100:chunk + 1600] = 0.0  # a = 1500 2^42
    row[0, 2 * chunk + 100:2 * chunk + 1100], row[0, 2 * chunk + 1100:2 * chunk + 1103] = 0.0, least  # b = 1000 2^42 + 3
    row[0, 3 * chunk + 100:3 * chunk + 599], row[0, 3 * chunk + 599] = 0.0, -3 * 2.0**-42  # c = 499 2^42 + (2^42 - 3): of e^-x the rest, x^2 / 2 2^42, is 2^-39.8
    a, b = 1500 * 2**42, 1000 * 2**42 + 3
    assert int(float(a + b)) - b == a + 1 and float(2 * a) == 2 * a
    assert onebit.sample(row.cuda(), torch.tensor([0.5], device="cuda")).item() == 2 * chunk + 100
    below, above = 0.5 - 2.0**-25, 0.5 + 2.0**-24
    assert onebit.sample(row.cuda(), torch.tensor([below], device="cuda")).item() == chunk + 1599
    assert onebit.sample(row.cuda(), torch.tensor([above], device="cuda")).item() == 2 * chunk + 100


def test_chunks_whose_weights_are_all_0():
    """-40 below the largest is e^-40 = 2^-57.7 of it: less than half of 2^-42, a weight of 0, so that the last token with a weight is the largest logit, whatever stands behind it"""
    chunk = 4096
    row = torch.full((5, 3 * chunk), -40.0)
    row[:, 5] = 0.0
    u = torch.tensor([1.0, 1.5, math.inf, 1 - 2.0**-24, 0.0])
    assert onebit.sample(row.cuda(), u.cuda()).tolist() == [5] * 5
    # at an infinite temperature all finite logits weigh the same, beside an infinite one nothing
    row = torch.zeros((3, 3 * chunk))
    u = torch.tensor([0.2, 0.7, 1.0])
    assert onebit.sample(row.cuda(), u.cuda(), temperature=math.inf).tolist() == [math.floor(float(u[0]) * 3 * chunk), math.floor(float(u[1]) * 3 * chunk), 3 * chunk - 1]
    row[:, 5] = row[:, 9000] = math.inf
    for temperature in (1.0, math.inf):
        assert onebit.sample(row.cuda(), u.cuda(), temperature=temperature).tolist() == [5, 9000, 9000]
        # 0.6 of the mass takes both of the two, 0.4 the first
        assert onebit.sample(row.cuda(), u.cuda(), temperature=temperature, top_p=0.6).tolist() == [5, 9000, 9000]
        assert onebit.sample(row.cuda(), u.cuda(), temperature=temperature, top_p=0.4).tolist() == [5, 5, 5]


@pytest.mark.parametrize("rows,columns,dtype", [(1, 1, torch.float32), (130, 200, torch.float32), (1000, 1408, torch.bfloat16), (9000, 512, torch.float16)])
def test_weights_as_codes_are_those_of_the_host(rows, columns, dtype):
    """To the bit, and a weight of one row as quantize_rows has it"""
    w = torch.randn((rows, columns), generator=generator(rows)).to(dtype)
    for got, want in zip(onebit.quantize_weight(w.cuda()), onebit.quantize_weight(w)):
        assert got.is_cuda and same(got, want)
    for got, want in zip(onebit.quantize_weight(w[:1].cuda()), onebit.quantize_rows(w[:1].cuda())):
        assert same(got, want)


def test_a_sequence_behind_a_nan_draws_nothing_any_more():
    """A decoder without layers, whose logits come from the last id alone: an embedding with a NaN gives no token, and nothing is drawn from another id in its place"""
    from onebitsparsemul_amd.decode import Decoder
    decoder = Decoder(0, 3, 16, head="e4m3")
    decoder.embedding[7, 5] = math.nan
    prompt = torch.tensor([[7, 8], [8, 7], [9, 9]], device="cuda")
    tokens = decoder.generate(prompt, torch.rand((4, 3), generator=generator(1)).cuda(), top_k=3)
    assert bool((tokens[1] == -1).all()) and bool((tokens[[0, 2]] >= 0).all()) and bool((tokens[[0, 2]] != 7).all())


@pytest.mark.parametrize("kind", ["positive", "outliers", "outlier in a group", "cancelling"])
@pytest.mark.parametrize("tokens,rows,columns", [(300, 700, 4096), (64, 2304, 4096), (1000, 8192, 640), (600, 4099, 640)])
def test_products_that_the_8_bit_instruction_cuts(tokens, rows, columns, kind):
    """Seven products of eight neighbours lose less than 2^-13 of the largest of the eight each: the bound is 7 2^-13 of the sum of those largest ones, beside the roundings of the sums and the
    result's own. A result that outliers cancel in is off by as much, whatever is left of it, and the mean of all errors by that bound's mean, beside the mean of as many roundings (six times
    u / sqrt(3) of the results' root mean square, over the root of their number). fp32 results are cut nowhere."""
    g = generator(columns + tokens)
    x, w = (torch.randn((n, columns), generator=g, dtype=torch.float32).cuda() for n in (tokens, rows))
    at = torch.arange(columns, device="cuda")
    if kind == "positive":
        x, w = x.abs() * 100, w.abs() * 100
    elif kind == "cancelling":  # columns 3 and 11 of each group: 448 times the same weight, once less
        x, w = torch.where((at % 128 == 3) | (at % 128 == 11), 448.0, x), w * 100
        w[:, at % 128 == 11] = -w[:, at % 128 == 3]
    else:
        x, w = torch.where(at % (8 if kind == "outliers" else 128) == 3, x.sign() * 448, x), w * 100
    x, w = (t.clamp(-448, 448).to(E4M3) for t in (x, w))
    xs, ws = torch.full((tokens, columns // 128), 2.0**-8, device="cuda"), torch.full((-(-rows // 128), columns // 128), 2.0**-8, device="cuda")
    xd, wd = x.double() * 2.0**-8, w.double() * 2.0**-8
    want, size = xd @ wd.T.contiguous(), xd.abs() @ wd.abs().T.contiguous()
    largest = torch.zeros_like(want)  # (products of two codes are exact in fp32)
    for octet in range(0, columns, 8):
        a, b = xd[:, octet:octet + 8].float().abs(), wd[:, octet:octet + 8].float().abs()
        most = a[:, :1] * b[:, 0]
        for i in range(1, 8):
            most = torch.maximum(most, a[:, i:i + 1] * b[:, i])
        largest += most
    sums, cut = (130 + 3 * (columns // 128)) * 2.0**-23 * size, 7 * 2.0**-13 * largest
    for dtype in DTYPES:
        error = onebit.block_linear(x, xs, w, ws, out_dtype=dtype).double() - want
        of_sums = sums + cut if dtype != torch.float32 else sums
        bound = U[dtype] * (1 + 2.0**-10) * (want.abs() + of_sums) + of_sums + (2.0**-25 if dtype == torch.float16 else 0)
        assert bool((error.abs() <= bound).all()), (dtype, float((error.abs() / bound).max()))
        roundings = 6 * U[dtype] / math.sqrt(3) * float((want.norm() + of_sums.norm()) / want.numel())
        assert abs(float(error.mean())) <= float(of_sums.mean()) + roundings
