"""The operators around the one-bit projections, without a GPU: what the C ABI refuses, the header, the rotary tables; and what the
binding refuses on a GPU."""
import ctypes
import math
import os
import re
import subprocess

import pytest
import torch

import onebitsparsemul_amd as onebit
from onebitsparsemul_amd import _native
from onebitsparsemul_amd import build as native_build

vp, i32, f32, i64 = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_longlong
HEADER = os.path.join(native_build.INCLUDE, "onebit_decoder.h")


class Heads(ctypes.Structure):
    _fields_ = [("data", vp), ("token_stride", i64), ("head_stride", i64)]


class Cache(ctypes.Structure):
    _fields_ = [("k", vp), ("v", vp), ("k_scale", vp), ("v_scale", vp), ("pages", i32), ("kv_heads", i32), ("block", i32), ("head_dim", i32), ("code", i32)]


class Sequences(ctypes.Structure):
    _fields_ = [("page_table", vp), ("lengths", vp), ("starts", vp), ("count", i32), ("width", i32), ("tokens", i32), ("max_new", i32), ("max_length", i32)]


class Norm(ctypes.Structure):
    _fields_ = [(n, vp) for n in ("x", "residual", "h_out", "y", "weight", "bias", "post_weight", "post_bias", "gate")] + \
               [(n, i64) for n in ("x_stride", "residual_stride", "h_stride", "y_stride", "gate_row_stride")] + \
               [(n, i32) for n in ("gate_column_stride", "x_dtype", "residual_dtype", "y_dtype", "weight_dtype", "gate_dtype", "rows", "hidden", "kind")] + \
               [(n, f32) for n in ("residual_scale", "block_scale", "eps")]


@pytest.fixture(scope="module")
def lib():
    lib = _native.lib()
    lib.onebit_cache_attention_workspace.restype = ctypes.c_size_t
    return lib


A = 0x10000  # an address that nobody reads
GOOD_CACHE = dict(k=A, v=A, k_scale=A, v_scale=A, pages=8, kv_heads=2, block=64, head_dim=128, code=0)
GOOD_SEQUENCES = dict(page_table=A, lengths=A, starts=None, count=4, width=2, tokens=4, max_new=1, max_length=0)


def attention(lib, cache=(), sequences=(), heads=8, dtype=1, q=A, stride=1024, workspace=None):
    c, s = Cache(**{**GOOD_CACHE, **dict(cache)}), Sequences(**{**GOOD_SEQUENCES, **dict(sequences)})
    rows = Heads(q, stride, 128)
    return lib.onebit_cache_attention(ctypes.byref(c), ctypes.byref(s), ctypes.byref(rows), ctypes.byref(rows), heads, dtype, f32(0.1), vp(workspace), None)


@pytest.mark.parametrize("change,message", [
    (dict(cache=dict(k=None)), "null pointer in the cache"), (dict(cache=dict(v_scale=None)), "null pointer in the cache"),
    (dict(cache=dict(v=A + 8)), "16-byte aligned"), (dict(cache=dict(block=48)), "block = 48"), (dict(cache=dict(head_dim=96)), "head_dim = 96"),
    (dict(cache=dict(pages=0)), "pages"), (dict(cache=dict(code=2)), "code must be"), (dict(sequences=dict(lengths=None)), "null pointer in the sequences"),
    (dict(sequences=dict(count=0)), "sequences"), (dict(sequences=dict(count=70000, tokens=70000)), "65535"), (dict(sequences=dict(tokens=0)), "positive"),
    (dict(sequences=dict(tokens=5)), "do not divide"), (dict(sequences=dict(width=1 << 25)), "int range"),
    (dict(sequences=dict(width=(1 << 24) + 1)), "2^30 tokens"), (dict(heads=7), "multiple of kv_heads"),
    (dict(heads=0), "multiple of kv_heads"), (dict(dtype=0), "dtype code"), (dict(dtype=3), "dtype code"), (dict(q=A + 2), "q must be 16-byte aligned"),
    (dict(q=None), "must not be null"), (dict(stride=1025), "multiples of eight"),
    (dict(sequences=dict(width=4096)), "needs a workspace of"), (dict(sequences=dict(width=4096), workspace=A + 4), "needs a workspace of"),
    (dict(heads=1 << 30), "int range")])
def test_attention_refuses(lib, change, message):
    assert attention(lib, **change) == 1
    assert message in _native.last_error()


def test_workspace_follows_the_split(lib):
    cache = Cache(**GOOD_CACHE)
    short, long = Sequences(**GOOD_SEQUENCES), Sequences(**{**GOOD_SEQUENCES, "width": 4096})
    assert lib.onebit_cache_attention_workspace(ctypes.byref(cache), ctypes.byref(short), 8) == 0
    bytes_ = lib.onebit_cache_attention_workspace(ctypes.byref(cache), ctypes.byref(long), 8)
    assert bytes_ > 0 and bytes_ % (4 * 8 * 130 * 4) == 0  # splits of 4 tokens x 8 heads x (128 sums, maximum, sum)
    # rows that would be more than a launch of the join has threads for go unsplit
    crowd = Sequences(**{**GOOD_SEQUENCES, "width": 4096, "tokens": 1 << 19, "max_new": 1, "starts": A})
    assert lib.onebit_cache_attention_workspace(ctypes.byref(cache), ctypes.byref(crowd), 8) == 0 and _native.last_error() == ""
    assert lib.onebit_cache_attention_workspace(None, ctypes.byref(long), 8) == 0 and "cache" in _native.last_error()


@pytest.mark.parametrize("change,message", [
    (dict(cache=dict(block=8)), "block = 8"), (dict(k=None), "k must not be null"), (dict(k=A + 8), "k must be 16-byte"), (dict(stride=100), "multiples of eight"),
    (dict(dtype=5), "dtype code"), (dict(rotary_dim=24), "multiples of 16"), (dict(rotary_dim=0), "rotary_dim = 0"), (dict(rotary_dim=144), "rotary_dim = 144"),
    (dict(rows=0), "must have rows"), (dict(table=A + 4), "16-byte aligned"), (dict(table=None), "needs a rotary table"), (dict(heads=0), "heads must be")])
def test_append_refuses(lib, change, message):
    a = dict(dict(cache={}, sequences={}, k=A, stride=1024, heads=4, dtype=1, table=A, rows=100, rotary_dim=128), **change)
    c, s = Cache(**{**GOOD_CACHE, **a["cache"]}), Sequences(**{**GOOD_SEQUENCES, **a["sequences"]})
    k, q = Heads(a["k"], a["stride"], 128), Heads(A, 1024, 128)
    assert lib.onebit_cache_append(ctypes.byref(c), ctypes.byref(s), ctypes.byref(k), ctypes.byref(q), ctypes.byref(q), ctypes.byref(q), a["heads"], a["dtype"],
                                   vp(a["table"]), a["rows"], a["rotary_dim"], 0, None) == 1
    assert message in _native.last_error()


@pytest.mark.parametrize("change,message", [
    (dict(x=None), "null operand"), (dict(positions=None), "null operand"), (dict(dtype=7), "dtype code"), (dict(tokens=0), "positive"), (dict(dim=65), "even"),
    (dict(heads=1 << 20), "2^24"), (dict(table=None), "must have rows"), (dict(part=66), "rotary_dim = 66"), (dict(part=7), "rotary_dim = 7")])
def test_rotary_refuses(lib, change, message):
    a = dict(dict(x=A, positions=A, dtype=1, tokens=3, heads=4, dim=64, table=A, rows=10, part=64), **change)
    x, out = Heads(a["x"], 256, 64), Heads(A, 256, 64)
    assert lib.onebit_rotary(ctypes.byref(x), ctypes.byref(out), a["dtype"], a["tokens"], a["heads"], a["dim"], vp(a["positions"]), 0, vp(a["table"]), a["rows"],
                             a["part"], 0, None) == 1
    assert message in _native.last_error()


@pytest.mark.parametrize("change,message", [
    (dict(residual=None), "must not be null"), (dict(weight=None), "must not be null"), (dict(rows=0), "rows must be positive"), (dict(hidden=32769), "hidden 1 to 32768"),
    (dict(kind=2), "kind must be"), (dict(x_dtype=4), "dtype codes"), (dict(y_dtype=-1), "dtype codes"), (dict(x=None, gate=A), "need the block's output"),
    (dict(x=None, post_weight=A), "need the block's output"), (dict(post_bias=A), "post_bias needs"), (dict(gate=A, gate_column_stride=2), "gate_column_stride")])
def test_norm_refuses(lib, change, message):
    n = Norm(**{**dict(x=A, residual=A, y=A, weight=A, rows=1, hidden=64, residual_scale=1, block_scale=1), **change})
    assert lib.onebit_block_norm(ctypes.byref(n), None) == 1
    assert message in _native.last_error()


def test_header_is_plain_c_and_exported(lib, tmp_path):
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = re.findall(r"\b(onebit_\w+)\s*\(", text)
    assert sorted(names) == ["onebit_block_norm", "onebit_cache_append", "onebit_cache_attention", "onebit_cache_attention_workspace", "onebit_rotary"]
    assert all(hasattr(lib, n) for n in names)
    source = tmp_path / "c.c"
    source.write_text('#include "onebit_decoder.h"\nint main(void){onebit_norm n = {0}; return sizeof n == %d && sizeof(onebit_cache) == %d && '
                      'sizeof(onebit_sequences) == %d ? 0 : 1;}\n' % (ctypes.sizeof(Norm), ctypes.sizeof(Cache), ctypes.sizeof(Sequences)))
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", native_build.INCLUDE, str(source), "-o", str(tmp_path / "c")], check=True)
    subprocess.run([str(tmp_path / "c")], check=True)


def test_rotary_tables():
    plain = onebit.rotary_table(50, 64, device="cpu")
    assert plain.dtype == torch.float32 and plain.shape == (50, 64)
    for p, i in ((0, 0), (49, 0), (49, 31), (7, 5)):
        angle = p * 10000.0 ** (-2 * i / 64)
        assert abs(float(plain[p, i]) - math.cos(angle)) < 1e-7 and abs(float(plain[p, 32 + i]) - math.sin(angle)) < 1e-7
    linear = onebit.rotary_table(200, 64, scaling=dict(kind="linear", factor=4.0), device="cpu")
    assert torch.allclose(linear[::4], plain, atol=2e-6)
    base = onebit.rotary_table(50, 64, scaling=dict(kind="base", factor=4.0), device="cpu")
    assert torch.equal(base[:, 0], plain[:, 0])  # the fastest pair is kept, the slowest four times slower
    assert abs(math.asin(float(base[40, 63])) * 4 - math.asin(float(plain[40, 63]))) < 1e-5
    for scaling in (dict(kind="bands", factor=8.0, original=1024, low=1.0, high=4.0), dict(kind="ramp", factor=8.0, original=1024)):
        table = onebit.rotary_table(50, 64, scaling=scaling, device="cpu")
        size = 0.1 * math.log(8) + 1 if scaling["kind"] == "ramp" else 1.0
        assert torch.allclose(table[:, 0], plain[:, 0] * size, atol=1e-6) and torch.allclose(table[:, :32] ** 2 + table[:, 32:] ** 2, torch.full((50, 32), size * size), atol=1e-5)
        rate = torch.atan2(table[1, 32:], table[1, :32]).double()
        kept = 10000.0 ** (-torch.arange(0, 64, 2).double() / 64)
        ratio = kept / rate
        assert bool((ratio[1:] >= ratio[:-1] - 1e-4).all()) and abs(float(ratio[-1]) - 8) < 1e-3
        turns = 1024 * kept / (2 * math.pi)
        if scaling["kind"] == "bands":
            assert bool(((ratio[turns > 4] - 1).abs() < 1e-5).all()) and bool(((ratio[turns < 1] - 8).abs() < 1e-2).all())
    for bad in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=64, scaling=dict(kind="other", factor=2))):
        with pytest.raises(ValueError):
            onebit.rotary_table(10, device="cpu", **bad)


def test_tensors_on_the_host_are_refused():
    x = torch.zeros((2, 2, 64), dtype=torch.float16)
    cache = onebit.QuantizedCache(2, 2, 64, device="cpu")
    pages, lengths = torch.zeros((2, 1), dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    for call in (lambda: onebit.rotary(x, torch.arange(2), onebit.rotary_table(4, 64, device="cpu")), lambda: cache.append(x, x, pages, lengths),
                 lambda: cache.attend(x, pages, lengths), lambda: onebit.block_norm(x, x, torch.ones(64, dtype=torch.float16))):
        with pytest.raises(ValueError, match="GPU"):
            call()
    with pytest.raises(TypeError):
        onebit.QuantizedCache(2, 2, 64, dtype=torch.float16, device="cpu")
    with pytest.raises(ValueError):
        onebit.QuantizedCache(2, 2, 64, block=24, device="cpu")


@pytest.mark.gpu
def test_the_binding_refuses():
    cache = onebit.QuantizedCache(4, 2, 64)
    x, q = (torch.zeros((3, n, 64), dtype=torch.float16, device="cuda") for n in (2, 4))
    pages, lengths = torch.zeros((3, 1), dtype=torch.int32, device="cuda"), torch.ones(3, dtype=torch.int32, device="cuda")
    table = onebit.rotary_table(8, 64)
    weight = torch.ones(64, dtype=torch.float16, device="cuda")
    rows = x[:, 0].contiguous()
    refused = [
        (ValueError, "shape", lambda: cache.attend(q[..., :32], pages, lengths)), (TypeError, "float16 or bfloat16", lambda: cache.attend(q.float(), pages, lengths)),
        (TypeError, "pages must be", lambda: cache.attend(q, pages.long(), lengths)), (ValueError, "one entry for each", lambda: cache.attend(q, pages, lengths[:2])),
        (ValueError, "starts must have", lambda: cache.attend(q, pages, lengths, starts=lengths)), (ValueError, "max_new", lambda: cache.attend(q, pages, lengths, max_new=0)),
        (RuntimeError, "multiple of kv_heads", lambda: cache.attend(q[:, :3], pages, lengths)), (ValueError, "out must have", lambda: cache.attend(q, pages, lengths, out=q[..., ::2])),
        (RuntimeError, "single memory location", lambda: cache.attend(q, pages, lengths, out=q[:1].expand(3, 4, 64))),
        (RuntimeError, "single memory location", lambda: onebit.rotary(x, lengths, table, out=x[:, :1].expand(3, 2, 64))),
        (RuntimeError, "do not divide", lambda: cache.attend(q[:2], pages, lengths)), (ValueError, "must live on", lambda: cache.attend(q, pages.cpu(), lengths)),
        (ValueError, "one shape and type", lambda: cache.append(x, x[:2], pages, lengths)), (ValueError, "for this cache", lambda: cache.append(q, q, pages, lengths)),
        (ValueError, "needs a rotary table", lambda: cache.append(x, x, pages, lengths, q=q)), (ValueError, "k's tokens", lambda: cache.append(x, x, pages, lengths, q=q.float(), rotary=table)),
        (RuntimeError, "multiples of 16", lambda: cache.append(x, x, pages, lengths, rotary=table[:, :20].contiguous())),
        (ValueError, "contiguous", lambda: cache.append(x, x, pages, lengths, rotary=table[:, ::2])),
        (TypeError, "positions", lambda: onebit.rotary(x, lengths.float(), table)), (ValueError, "one entry", lambda: onebit.rotary(x, lengths[:2], table)),
        (RuntimeError, "rotary_dim", lambda: onebit.rotary(x[..., :32].contiguous(), lengths, table)), (ValueError, "x's shape", lambda: onebit.rotary(x, lengths, table, out=q)),
        (TypeError, "float16, bfloat16 or float32", lambda: onebit.rotary(x.int(), lengths, table)),
        (ValueError, "weight must be", lambda: onebit.block_norm(rows, rows, weight[:32])), (ValueError, "residual's shape", lambda: onebit.block_norm(rows[:2], rows, weight)),
        (TypeError, "weight's type", lambda: onebit.block_norm(rows, rows, weight, bias=weight.float())), (ValueError, "gate must have", lambda: onebit.block_norm(rows, rows, weight, gate=weight[:8])),
        (ValueError, "'rms' or 'layer'", lambda: onebit.block_norm(rows, rows, weight, kind="batch")), (RuntimeError, "need the block's output", lambda: onebit.block_norm(None, rows, weight, post_weight=weight)),
        (ValueError, "residual_out", lambda: onebit.block_norm(rows, rows, weight, residual_out=rows.float())),
        (RuntimeError, "hidden 1 to 32768", lambda: onebit.block_norm(*(torch.zeros((1, 40000), dtype=torch.float16, device="cuda"),) * 2, torch.zeros(40000, dtype=torch.float16, device="cuda"))),
    ]
    for kind, message, call in refused:
        with pytest.raises(kind, match=message):
            call()
    cache.attend(q, pages, lengths)  # and goes on working
    torch.cuda.synchronize()
