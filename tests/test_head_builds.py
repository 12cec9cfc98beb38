"""Which kernels the calls of onebit_head.h launch, without a GPU: the library is linked against tests/host/launch_stub.cpp, which stands in for the HIP runtime (256 compute
units) and records the kernels' names. Each kernel is one that some call reaches."""
import ctypes
import os
import re
import subprocess

import pytest

from onebitsparsemul_amd import build as native_build
from test_head_host import A, Codes, Product, Sampling

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    folder = tmp_path_factory.mktemp("host")
    obj, out = str(folder / "launch_stub.o"), str(folder / "libhost.so")
    subprocess.run([os.path.join(os.path.dirname(native_build.HIPCC), "..", "llvm", "bin", "clang++"), "-O1", "-std=c++17", "-fPIC",
                    "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-c", os.path.join(HERE, "host", "launch_stub.cpp"), "-o", obj],
                   check=True)
    # -Bsymbolic: the stand-ins, not the HIP runtime that torch has loaded
    subprocess.run(["g++", "-shared", "-Wl,-Bsymbolic", "-o", out, obj, "-Wl,-u,onebit_block_linear", "-Wl,-u,onebit_sample", "-Wl,-u,onebit_quantize_rows",
                    native_build.STATIC_LIB, "-lpthread"], check=True)
    lib = ctypes.CDLL(out)
    lib.stub_launched.restype = lib.onebit_sparse_last_error.restype = ctypes.c_char_p
    lib.onebit_block_linear_workspace.restype = lib.onebit_sample_workspace.restype = ctypes.c_size_t
    return lib


def launched(lib, call, *args):
    lib.stub_reset()
    assert call(*args) == 0, lib.onebit_sparse_last_error()
    return [re.sub(r"^void onebit::|^onebit::|\(anonymous namespace\)::", "", name).split("(")[0] for name in lib.stub_launched().decode().splitlines()]


def product(lib, tokens, rows, columns, dtype, stride=None):
    p = Product(x=Codes(A, A, columns, columns // 128), weight=Codes(A, A, stride or columns, columns // 128), y=A, y_stride=rows, tokens=tokens, rows=rows, columns=columns,
                y_dtype=dtype)
    bytes_ = lib.onebit_block_linear_workspace(ctypes.byref(p))
    names = launched(lib, lib.onebit_block_linear, ctypes.byref(p), ctypes.c_void_p(A if bytes_ else None), None)
    assert (names[1:] == ["add_splits_kernel"]) == (bytes_ > 0)
    assert bytes_ % (4 * tokens * rows) == 0
    if bytes_:  # without one, and with one that is not aligned
        for workspace in (None, A + 4):
            assert lib.onebit_block_linear(ctypes.byref(p), ctypes.c_void_p(workspace), None) == 1 and b"needs a workspace of" in lib.onebit_sparse_last_error()
    return names[0]


def test_every_kernel_of_products_is_reached_and_no_other(host):
    shapes = [(t, r, c, d) for t in (1, 9, 16, 17, 33, 64, 128, 333, 1000, 2048, 4096) for r in (64, 1024, 4099, 11008, 37000, 131072) for c in (128, 512, 2048, 4096, 11008) for d in (0, 1, 2)]
    by_kernel = {}
    for shape in shapes:
        by_kernel.setdefault(product(host, *shape), []).append(shape)
    tiles = ["4, 1, 2, 2, 3", "2, 2, 2, 2, 4", "4, 2, 2, 2, 3", "4, 2, 4, 4, 3"]
    assert set(by_kernel) == {"few_kernel<1, 4, 2>", "few_kernel<1, 8, 2>", "few_kernel<4, 4, 1>", "mixed_kernel", "tile_kernel<2, 4, 8, 4, 2, true>",
                              *(f"tile_kernel<{t}, {narrow}>" for t in tiles for narrow in ("true", "false"))}
    # the 8-bit instruction: 16-bit results of more than 16 tokens alone
    for kernel, reached in by_kernel.items():
        if kernel == "mixed_kernel" or "true" in kernel:
            assert all(tokens > 16 and dtype != 0 for tokens, _, _, dtype in reached), kernel
        elif "false" in kernel:
            assert all(tokens <= 16 or dtype == 0 for tokens, _, _, dtype in reached), kernel


def test_rows_far_apart_take_no_tile(host):
    assert not product(host, 2048, 11008, 4096, 2).startswith("few_kernel")
    assert product(host, 2048, 11008, 4096, 2, stride=1 << 24).startswith("few_kernel")


@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_kernels_of_sampling(host, dtype):
    def names(rows, vocabulary):
        a = Sampling(logits=A, logits_stride=vocabulary, logits_dtype=dtype, rows=rows, vocabulary=vocabulary, uniform=A, tokens=A, temperature=1, top_p=1)
        bytes_ = host.onebit_sample_workspace(ctypes.byref(a))
        if bytes_:
            assert host.onebit_sample(ctypes.byref(a), None, None) == 1 and b"needs a workspace of" in host.onebit_sparse_last_error()
        return launched(host, host.onebit_sample, ctypes.byref(a), ctypes.c_void_p(A if bytes_ else None), None)
    assert names(5, 1000) == [f"sample_short_kernel<{dtype}, 256, 4096>"] and names(5, 8192) == [f"sample_short_kernel<{dtype}, 512, 8192>"]
    both = [f"chunk_kernel<{dtype}>", f"sample_long_kernel<{dtype}>"]
    assert names(5, 8193) == both and names(70000, 1 << 20) == 3 * both
