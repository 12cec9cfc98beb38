"""From the last layer to the next tokens, without a GPU: what the C ABI refuses, the header, weights as codes; and what the binding refuses on a GPU."""
import ctypes
import os
import re
import subprocess

import pytest
import torch

import onebitsparsemul_amd as onebit
from onebitsparsemul_amd import _native
from onebitsparsemul_amd import build as native_build

vp, i32, f32, i64 = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_longlong
HEADER = os.path.join(native_build.INCLUDE, "onebit_head.h")
A = 0x10000  # an address that nobody reads


class Codes(ctypes.Structure):
    _fields_ = [("codes", vp), ("scales", vp), ("row_stride", i64), ("scale_stride", i64)]


class Product(ctypes.Structure):
    _fields_ = [("x", Codes), ("weight", Codes), ("bias", vp), ("y", vp), ("y_stride", i64), ("tokens", i32), ("rows", i32), ("columns", i32),
                ("y_dtype", i32), ("bias_dtype", i32)]


class Sampling(ctypes.Structure):
    _fields_ = [("logits", vp), ("logits_stride", i64), ("logits_dtype", i32), ("rows", i32), ("vocabulary", i32), ("uniform", vp), ("temperatures", vp),
                ("top_ps", vp), ("min_ps", vp), ("top_ks", vp), ("temperature", f32), ("top_p", f32), ("min_p", f32), ("top_k", i32), ("tokens", vp)]


@pytest.fixture(scope="module")
def lib():
    lib = _native.lib()
    lib.onebit_block_linear_workspace.restype = lib.onebit_sample_workspace.restype = ctypes.c_size_t
    return lib


@pytest.mark.parametrize("change,message", [
    (dict(x=None), "x must not be null"), (dict(dtype=3), "dtype code"), (dict(rows=0), "rows must be positive"), (dict(columns=0), "columns 1 to"),
    (dict(codes=None), "null pointer"), (dict(codes=A + 8), "16-byte aligned"), (dict(row_stride=120), "multiple of 16")])
def test_rows_are_refused(lib, change, message):
    a = dict(dict(x=A, dtype=1, rows=2, columns=100, codes=A, row_stride=128), **change)
    out = Codes(a["codes"], A, a["row_stride"], 1)
    assert lib.onebit_quantize_rows(vp(a["x"]), a["dtype"], i64(100), a["rows"], a["columns"], ctypes.byref(out), None) == 1
    assert message in _native.last_error()


@pytest.mark.parametrize("change,message", [
    (dict(x=dict(codes=None)), "codes of x"), (dict(weight=dict(scales=None)), "codes of the weight"), (dict(weight=dict(codes=A + 4)), "the weight must be 16-byte"),
    (dict(x=dict(row_stride=8)), "multiple of 16"), (dict(y=None), "y must not be null"), (dict(tokens=0), "positive"), (dict(rows=-1), "positive"),
    (dict(columns=100), "multiple of 128"), (dict(columns=0), "multiple of 128"), (dict(y_dtype=5), "dtype codes"), (dict(bias=A, bias_dtype=3), "dtype codes")])
def test_products_are_refused(lib, change, message):
    good = dict(x=dict(codes=A, scales=A, row_stride=256, scale_stride=2), weight=dict(codes=A, scales=A, row_stride=256, scale_stride=2), y=A, y_stride=8, tokens=3,
                rows=8, columns=256, y_dtype=1)
    a = {**good, **{k: {**good[k], **v} if isinstance(v, dict) else v for k, v in change.items()}}
    p = Product(**{k: Codes(**v) if isinstance(v, dict) else v for k, v in a.items()})
    assert lib.onebit_block_linear(ctypes.byref(p), None, None) == 1
    assert message in _native.last_error()
    assert lib.onebit_block_linear_workspace(ctypes.byref(p)) == 0 and message in _native.last_error()
    assert lib.onebit_block_linear(None, None, None) == 1


@pytest.mark.parametrize("change,message", [
    (dict(logits=None), "must not be null"), (dict(uniform=None), "must not be null"), (dict(tokens=None), "must not be null"), (dict(logits_dtype=3), "dtype code"),
    (dict(rows=0), "rows must be positive"), (dict(vocabulary=0), "1 to 2^20"), (dict(vocabulary=(1 << 20) + 1), "1 to 2^20")])
def test_sampling_is_refused(lib, change, message):
    a = Sampling(**{**dict(logits=A, logits_stride=100, logits_dtype=0, rows=2, vocabulary=100, uniform=A, tokens=A, temperature=1, top_p=1), **change})
    assert lib.onebit_sample(ctypes.byref(a), None, None) == 1
    assert message in _native.last_error()
    assert lib.onebit_sample_workspace(ctypes.byref(a)) == 0 and message in _native.last_error()


def test_norms_with_codes_are_refused(lib):
    from test_decoder_host import Norm
    good = dict(residual=A, weight=A, rows=1, hidden=64, residual_scale=1, block_scale=1)
    out = Codes(A, A, 128, 1)
    for change, message in ((dict(residual=None), "must not be null"), (dict(rows=0), "rows must be positive"), (dict(hidden=32769), "hidden 1 to 32768"),
                            (dict(kind=2), "kind must be"), (dict(gate=A), "need the block's output")):
        assert lib.onebit_block_norm_codes(ctypes.byref(Norm(**{**good, **change})), ctypes.byref(out), None) == 1
        assert message in _native.last_error()
    for bad in (Codes(None, A, 128, 1), Codes(A + 1, A, 128, 1), Codes(A, A, 100, 1)):
        assert lib.onebit_block_norm_codes(ctypes.byref(Norm(**good)), ctypes.byref(bad), None) == 1 and "the result" in _native.last_error()


def test_header_is_plain_c_and_exported(lib, tmp_path):
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = re.findall(r"\b(onebit_\w+)\s*\(", text)
    assert len(names) == 6 and all(hasattr(lib, n) for n in names)
    source = tmp_path / "c.c"
    source.write_text('#include "onebit_head.h"\nint main(void){return sizeof(onebit_codes) == %d && sizeof(onebit_block_product) == %d && sizeof(onebit_sampling) == %d ? 0 : 1;}\n'
                      % (ctypes.sizeof(Codes), ctypes.sizeof(Product), ctypes.sizeof(Sampling)))
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", native_build.INCLUDE, str(source), "-o", str(tmp_path / "c")], check=True)
    subprocess.run([str(tmp_path / "c")], check=True)


@pytest.mark.parametrize("rows,columns", [(1, 1), (128, 128), (130, 200), (300, 1000), (8200, 129)])
def test_weights_as_codes(rows, columns):
    """A value is off by half a step of its code: 2^-4 of it, or half of the least subnormal, 2^-10 of the scale, and the scale's and the quotient's own roundings."""
    w = torch.randn((rows, columns), generator=torch.Generator().manual_seed(rows)).double()
    codes, scales = onebit.quantize_weight(w.float())
    padded = -(-columns // 128) * 128
    assert codes.dtype == torch.float8_e4m3fn and codes.shape == (rows, padded) and scales.shape == (-(-rows // 128), padded // 128)
    scale = scales.double().repeat_interleave(128, 0)[:rows].repeat_interleave(128, 1)
    values = codes.float().double() * scale
    assert bool((values[:, columns:] == 0).all())
    w = w.float().double()
    assert bool(((values[:, :columns] - w).abs() <= 2.0**-4 * (1 + 2.0**-20) * w.abs() + 2.0**-10 * scale[:, :columns]).all())
    blocks = torch.nn.functional.pad(w, (0, padded - columns, 0, -rows % 128)).view(-1, 128, padded // 128, 128).abs().amax((1, 3))
    assert torch.equal(scales, blocks.float() / 448)


def test_weights_that_are_not_finite():
    w = torch.ones((256, 256))
    w[3, 5], w[200, 7], w[200, 200] = float("nan"), float("inf"), 0.0
    w[:128, 128:] = 0
    codes, scales = onebit.quantize_weight(w)
    assert torch.isnan(scales[0, 0]) and scales[1, 0] == float("inf") and scales[0, 1] == 0 and scales[1, 1] == 1 / 448
    assert bool((codes[:, :128].float() == 0).all()) and bool((codes[:128, 128:].float() == 0).all()) and codes[255, 255].float() == 448
    with pytest.raises(ValueError):
        onebit.quantize_weight(torch.zeros(5))
    with pytest.raises(ValueError):
        onebit.quantize_weight(torch.zeros((5, 5), dtype=torch.int32))


def test_a_layer_keeps_its_codes_in_its_state(tmp_path):
    layer, other = onebit.BlockLinear(torch.randn(70, 130), bias=torch.randn(70)), onebit.BlockLinear(torch.zeros(70, 130), bias=torch.zeros(70))
    torch.save(layer.state_dict(), tmp_path / "layer.pt")
    other.load_state_dict(torch.load(tmp_path / "layer.pt", weights_only=True))
    for name in ("codes", "scales", "bias"):
        assert torch.equal(getattr(layer, name).float(), getattr(other, name).float())


def test_rows_that_would_overlap_and_sizes_beyond_int_are_refused(lib):
    for out in (Codes(A, A, 128, 2), Codes(A, A, 256, 1)):
        assert lib.onebit_quantize_rows(ctypes.c_void_p(A), 0, ctypes.c_longlong(200), 2, 200, ctypes.byref(out), None) == 1 and "must not overlap" in _native.last_error()
        from test_decoder_host import Norm
        assert lib.onebit_block_norm_codes(ctypes.byref(Norm(residual=A, weight=A, rows=2, hidden=200, residual_scale=1, block_scale=1, residual_stride=200)), ctypes.byref(out), None) == 1
        assert "must not overlap" in _native.last_error()
    good = dict(x=Codes(A, A, 256, 2), weight=Codes(A, A, 256, 2), y=A, y_stride=64, tokens=3, rows=64, columns=256, y_dtype=1)
    for change, message in ((dict(y_stride=63), "must not overlap"), (dict(tokens=(1 << 30) + 1), "at most 2^30"), (dict(rows=(1 << 30) + 1), "at most 2^30"),
                            (dict(columns=(1 << 30) + 128), "at most 2^30")):
        p = Product(**{**good, **change})
        assert lib.onebit_block_linear(ctypes.byref(p), None, None) == 1 and message in _native.last_error()


def test_a_layer_of_another_type_keeps_its_codes():
    layer = torch.nn.Sequential(onebit.BlockLinear(torch.randn(70, 130), bias=torch.randn(70)))
    codes, scales = layer[0].codes.clone(), layer[0].scales.clone()
    for change in (lambda m: m.half(), lambda m: m.to(torch.bfloat16), lambda m: m.double(), lambda m: m.to("cpu")):
        change(layer)
        assert layer[0].codes.dtype == torch.float8_e4m3fn and torch.equal(layer[0].codes.float(), codes.float()) and torch.equal(layer[0].scales, scales)
    assert layer[0].bias.dtype == torch.float64 and layer.to("meta")[0].codes.device.type == "meta"


def test_tensors_on_the_host_are_refused():
    x = torch.zeros((2, 256))
    codes, scales = onebit.quantize_weight(x)
    for call in (lambda: onebit.quantize_rows(x), lambda: onebit.block_norm_codes(x, x, x[0]), lambda: onebit.block_linear(codes, scales.expand(2, 2), codes, scales),
                 lambda: onebit.sample(x, x[:, 0])):
        with pytest.raises(ValueError, match="GPU"):
            call()


@pytest.mark.gpu
def test_the_binding_refuses():
    x = torch.zeros((3, 256), dtype=torch.float16, device="cuda")
    codes, scales = onebit.quantize_rows(x)
    w, ws = onebit.quantize_weight(torch.ones((200, 256), device="cuda"))
    u, logits = torch.zeros(3, device="cuda"), torch.zeros((3, 50), device="cuda")
    out = torch.empty((3, 200), dtype=torch.float16, device="cuda")
    whole = torch.zeros(4096, dtype=torch.uint8, device="cuda")
    inside = whole[:768].view(torch.float8_e4m3fn).view(3, 256)
    refused = [
        (TypeError, "x must be", lambda: onebit.quantize_rows(x.int())), (TypeError, "codes must be", lambda: onebit.block_linear(x, scales, w, ws)),
        (TypeError, "scales must be", lambda: onebit.block_linear(codes, scales.half(), w, ws)), (ValueError, "multiple of 128", lambda: onebit.block_linear(codes[:, :100], scales, w, ws)),
        (ValueError, "each 128 columns", lambda: onebit.block_linear(codes, scales[:2], w, ws)), (ValueError, "weight_codes must have", lambda: onebit.block_linear(codes, scales, w[:, :128], ws)),
        (ValueError, "each 128 x 128", lambda: onebit.block_linear(codes, scales, w, ws[:1])), (ValueError, "must live on", lambda: onebit.block_linear(codes, scales, w.cpu(), ws)),
        (TypeError, "float16, bfloat16 or float32", lambda: onebit.block_linear(codes, scales, w, ws, out_dtype=torch.int32)),
        (ValueError, "bias must be", lambda: onebit.block_linear(codes, scales, w, ws, bias=u)), (ValueError, "out must have", lambda: onebit.block_linear(codes, scales, w, ws, out=out[:2])),
        (ValueError, "out must have", lambda: onebit.block_linear(codes, scales, w[:100], ws[:1], out=out[:, ::2])),
        (RuntimeError, "single memory location", lambda: onebit.block_linear(codes, scales, w, ws, out=out[:1].expand(3, 200))),
        (ValueError, "must not overlap", lambda: onebit.block_linear(codes, scales, w, ws, out=out.as_strided((3, 200), (100, 1)))),
        (ValueError, "negated", lambda: onebit.block_linear(torch._neg_view(codes), scales, w, ws)),
        (ValueError, "apart from", lambda: onebit.block_linear(inside, scales, w, ws, out=whole.view(torch.float16)[100:700].view(3, 200))),
        (ValueError, "whole rows a multiple of 16", lambda: onebit.block_linear(codes, scales, w.as_strided((199, 256), (257, 1)), ws)),
        (TypeError, "uniform must be", lambda: onebit.sample(logits, u.half())), (ValueError, "one number for each row", lambda: onebit.sample(logits, u[:2])),
        (TypeError, "logits must be", lambda: onebit.sample(logits.int(), u)), (TypeError, "top_k must be", lambda: onebit.sample(logits, u, top_k=u)),
        (TypeError, "temperature must be", lambda: onebit.sample(logits, u, temperature=u.double())), (ValueError, "one entry for each row", lambda: onebit.sample(logits, u, top_p=u[:2])),
        (ValueError, "vocabulary", lambda: onebit.sample(logits[:, :0], u)), (ValueError, "must live on", lambda: onebit.sample(logits, u.cpu())),
        (ValueError, "must live on", lambda: onebit.sample(logits, u, min_p=u.cpu())), (RuntimeError, "2\\^20", lambda: onebit.sample(torch.zeros((1, (1 << 20) + 1), device="cuda"), u[:1])),
        (ValueError, "weight must be", lambda: onebit.block_norm_codes(x, x, u)), (ValueError, "columns", lambda: onebit.BlockLinear(torch.zeros((8, 100), device="cuda"))(x)),
    ]
    for kind, message, call in refused:
        with pytest.raises(kind, match=message):
            call()
    onebit.block_linear(codes, scales, w, ws, out=out)  # and goes on working
    torch.cuda.synchronize()
    assert bool((out == 0).all())


def test_a_weight_that_is_learned_leaves_no_graph():
    import copy
    linear = torch.nn.Linear(200, 130)
    layer, plain = onebit.BlockLinear(linear.weight, linear.bias), onebit.BlockLinear(linear.weight.detach().clone(), linear.bias.detach().clone())
    for t in (*onebit.quantize_weight(linear.weight), *layer.buffers()):
        assert not t.requires_grad and t.grad_fn is None
    assert not list(layer.parameters()) and set(dict(layer.named_buffers())) == {"codes", "scales", "bias"}
    for name, t in plain.named_buffers():
        assert torch.equal(getattr(layer, name).float(), t.float())
    other = copy.deepcopy(layer).half()
    assert other.codes.dtype == torch.float8_e4m3fn and torch.equal(other.scales, layer.scales) and other.bias.dtype == torch.float16
    assert linear.weight.requires_grad and linear.bias.requires_grad


@pytest.mark.parametrize("rows,columns", [(0, 0), (0, 200), (5, 0), (300, 0)])
def test_weights_without_values(rows, columns):
    codes, scales = onebit.quantize_weight(torch.zeros((rows, columns)))
    assert codes.shape == (rows, -(-columns // 128) * 128) and codes.dtype == torch.float8_e4m3fn
    assert scales.shape == (-(-rows // 128), -(-columns // 128)) and scales.dtype == torch.float32


def generating(monkeypatch, draws, length=64, caches=()):
    """A decoder without layers on the host, whose draws are given, and the ids and bounds that its steps are called with"""
    from onebitsparsemul_amd import decode
    decoder, draws, calls = decode.Decoder.__new__(decode.Decoder), iter(draws), []
    decoder.lengths, decoder.table, decoder.caches = torch.zeros(3, dtype=torch.int32), torch.zeros((length, 64)), list(caches)

    def step(tokens, new, longest):
        decoder.lengths += new
        calls.append((tokens.tolist(), new, longest))
    monkeypatch.setattr(decoder, "step", step)
    monkeypatch.setattr(decode, "sample", lambda logits, uniform: torch.tensor(next(draws)))
    return decoder, calls


def test_a_sequence_without_a_token_gets_none_any_more(monkeypatch):
    """-1 is no id: the rows that it stands for go on with id 0, and what they draw is not returned"""
    decoder, calls = generating(monkeypatch, [[4, -1, 6], [5, 3, -1], [1, 2, 2]])
    tokens = decoder.generate(torch.tensor([[1, 2], [3, 4], [5, 6]]), torch.zeros((3, 3)))
    assert tokens.tolist() == [[4, 5, 1], [-1, -1, -1], [6, -1, -1]]
    assert calls == [([1, 2, 3, 4, 5, 6], 2, 2), ([4, 0, 6], 1, 3), ([5, 0, 0], 1, 4)]


def test_more_tokens_than_the_caches_hold_are_refused(monkeypatch):
    """A prompt of two and four more, the last of which goes into no cache: five places"""
    decoder, calls = generating(monkeypatch, [[1, 1, 1]] * 4, length=5)
    assert decoder.generate(torch.zeros((3, 2), dtype=torch.int64), torch.zeros((4, 3))).shape == (3, 4) and len(calls) == 4
    for lengths, count in ((0, 5), (1, 4), (5, 1)):
        decoder, calls = generating(monkeypatch, [], length=5)
        decoder.lengths += lengths
        with pytest.raises(ValueError, match="places"):
            decoder.generate(torch.zeros((3, 2), dtype=torch.int64), torch.zeros((count, 3)))
        assert not calls and bool((decoder.lengths == lengths).all())


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_no_tokens_are_ids_too(monkeypatch, dtype):
    decoder, calls = generating(monkeypatch, [])
    tokens = decoder.generate(torch.zeros((3, 2), dtype=dtype), torch.zeros((0, 3)))
    assert tokens.shape == (3, 0) and tokens.dtype == torch.int64 and not calls
