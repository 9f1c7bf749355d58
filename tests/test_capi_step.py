"""The C ABI of a decoding step without a GPU: argument checks that return before any device work, empty calls, and the
attention's workspace sizes; and the ops' refusal of CPU tensors."""
import ctypes

import pytest
import torch

BF16, F16, F32, E4M3 = 0, 1, 2, 3
ARG, SHAPE, ALIGN, DTYPE, LIMIT = 1, 2, 3, 4, 8


@pytest.fixture(scope="module")
def lib():
    from basal_b200 import _lib
    return _lib.lib()


def attention(lib, **kw):
    a = dict(q=None, q_dtype=BF16, q_row=512, q_head=128, k=None, v=None, kv_dtype=BF16, page=8192, head=2048, token=128,
             ks=None, vs=None, s_page=0, s_head=0, pages=4, page_size=16, table=None, table_row=2, width=2, lengths=None,
             rows=0, H=4, Hk=4, D=128, scale=1.0, window=0, out=None, work=None, work_bytes=0, stream=None)
    assert set(kw) <= set(a)
    return lib.basal200_paged_attention(*{**a, **kw}.values())


def test_attention_arguments(lib):
    assert attention(lib) == 0                       # no rows
    assert attention(lib, rows=-1) == ARG
    assert attention(lib, window=-1) == ARG
    assert attention(lib, H=6) == SHAPE              # 6 heads over 4
    assert attention(lib, D=96) == SHAPE
    assert attention(lib, q_dtype=F32) == DTYPE
    assert attention(lib, kv_dtype=F16) == DTYPE     # another 16-bit type than q's
    assert attention(lib, kv_dtype=E4M3) == ARG      # no scales
    assert attention(lib, token=132) == ALIGN
    assert attention(lib, page_size=0) == ARG
    assert attention(lib, width=1 << 28) == LIMIT    # positions past 32 bits
    assert attention(lib, rows=1) == ARG             # null pointers
    x = ctypes.c_void_p(4096)
    full = dict(q=x, k=x, v=x, table=x, lengths=x, out=x, rows=1)
    assert attention(lib, **{**full, "q": ctypes.c_void_p(4104)}) == ALIGN
    assert attention(lib, **full, q_head=130) == ALIGN
    assert attention(lib, **full, width=1024, table_row=1024) == ARG   # rows that need a workspace, and none
    assert attention(lib, **{**full, "rows": 70000}) == LIMIT


def test_attention_workspace(lib):
    ws = lib.basal200_paged_attention_workspace_bytes
    assert ws(4, 16, 4, 128, BF16, 16, 16, 0) == 0                      # rows of up to 256 positions: one part
    assert ws(4, 16, 4, 128, BF16, 17, 16, 0) == 4 * 16 * 2 * 130 * 4
    assert ws(4, 16, 4, 128, BF16, 1 << 16, 16, 0) == 4 * 16 * 111 * 130 * 4   # 444 CTAs over 4 key heads
    assert ws(4, 16, 4, 128, BF16, 1 << 16, 16, 200) == 0               # a window of 200 positions
    assert ws(4, 16, 4, 128, E4M3, 32, 16, 0) == 0                      # 8-bit: 512 positions a part
    assert ws(4, 16, 5, 128, BF16, 64, 16, 0) == 0 and ws(0, 16, 4, 128, BF16, 64, 16, 0) == 0
    assert ws(70000, 64, 1, 256, BF16, 1 << 20, 128, 0) > 1 << 32       # 64 bits


def test_append_arguments(lib):
    def call(dtype=BF16, kv=BF16, rows=0, T=1, Hk=2, D=64, page_size=16, strides=(8192, 1024, 64), ks=None, start=None):
        return lib.basal200_kv_append(None, None, dtype, 128, 128, 64, 128, 128, 64, None, None, kv, *strides, ks, ks, 0,
                                      0, 4, page_size, None, 2, 2, start, None, rows, T, Hk, D, None)
    assert call() == 0 and call(rows=3, T=0) == 0
    assert call(rows=-1) == ARG and call(T=-1) == ARG and call(rows=1) == ARG
    assert call(D=32) == SHAPE and call(dtype=F32, kv=F32) == DTYPE and call(kv=E4M3) == ARG
    assert call(strides=(8192, 1024, 68)) == ALIGN


def test_copy_arguments(lib):
    x = ctypes.c_void_p(4096)

    def call(src, dst, pages=8, bytes_=64, layers=2, base=x, npools=1, n=None):
        s, d = ((ctypes.c_int32 * max(1, len(v)))(*v) for v in (src, dst))
        return lib.basal200_kv_copy_pages((ctypes.c_void_p * 9)(*[base] * 9), (ctypes.c_int * 9)(*[layers] * 9),
                                          (ctypes.c_int64 * 9)(*[bytes_] * 9), npools, pages, s, d,
                                          len(src) if n is None else n, None)
    assert call([], []) == 0 and call([1], [2], npools=0) == 0
    assert call([1], [8]) == ARG and call([-1], [2]) == ARG
    assert call([1, 3], [2, 2]) == ARG              # written twice
    assert call([1, 2], [2, 4]) == ARG              # read and written
    assert call([3], [3]) == ARG
    many = list(range(100))
    assert call(many, [200 + i for i in many[:-1]] + [50], pages=400) == ARG     # the long list's bitmap
    assert call(many, [200] * 100, pages=400) == ARG
    assert call([1], [2], bytes_=6) == ALIGN and call([1], [2], base=ctypes.c_void_p(4098)) == ALIGN
    assert call([1], [2], npools=9) == LIMIT and call([1], [2], n=-1) == ARG


def test_gdn_step_arguments(lib):
    def call(dtype=BF16, ld=1024, b=768, a=770, rows=0, Hk=1, Hv=2, slots=4, x=None):
        return lib.basal200_gdn_step(x, dtype, ld, x, x, x, x, b, a, x, None, slots, rows, Hk, Hv, x, None)
    assert call() == 0
    assert call(rows=-1) == ARG and call(Hk=0) == ARG and call(Hk=3) == SHAPE and call(dtype=F32) == DTYPE
    assert call(rows=1) == ARG
    x = ctypes.c_void_p(4096)
    assert call(rows=1, x=x, ld=500) == SHAPE and call(rows=1, x=x, b=1023) == SHAPE
    assert call(rows=1, x=x, ld=1026) == ALIGN and call(rows=1, x=ctypes.c_void_p(4100)) == ALIGN
    assert call(rows=70000, x=x) == LIMIT


def test_constrain_arguments(lib):
    def call(dtype=F32, rows=0, V=100, T=0, N=0, x=None, past=None):
        return lib.basal200_constrain_logits(x, dtype, V, rows, V, None, 0, past, T, T, None, None, None, None, None, N, N,
                                             x, None)
    assert call() == 0 and call(rows=2, V=0) == 0
    assert call(rows=-1) == ARG and call(rows=1) == ARG and call(dtype=E4M3) == DTYPE
    x = ctypes.c_void_p(4096)
    assert call(rows=1, x=x, T=5) == ARG and call(rows=1, x=x, N=3) == ARG       # lengths without lists
    assert call(rows=1, x=x, T=70000, past=x) == LIMIT and call(rows=70000, x=x) == LIMIT


def test_ops_refuse_cpu_tensors():
    from basal_b200 import ops
    z = torch.zeros
    i = z(1, dtype=torch.int32)
    for f, a in ((ops.paged_attention, (z(1, 1, 64), z(1, 1, 16, 64), z(1, 1, 16, 64), i[None], i, 1.0)),
                 (ops.kv_append, (z(1, 1, 1, 64), z(1, 1, 1, 64), z(1, 1, 16, 64), z(1, 1, 16, 64), i[None], i)),
                 (ops.kv_copy_pages, ([z(1, 4, 4)], [0], [1])),
                 (ops.gdn_step, (z(1, 500), z(1, 3, 384), z(384, 4), z(1), z(1), z(1, 1, 128, 128), 1, 1, 384, 385)),
                 (ops.constrain_logits, (z(1, 10),))):
        with pytest.raises(ValueError, match="CUDA"):
            f(*a)


def test_the_torch_ops_are_those_of_the_installed_torch():
    """The library that build.py writes and the one that the package loads are the same file, named after this torch: one
    built against another torch is left alone."""
    import importlib.util
    import os

    from basal_b200 import _lib
    spec = importlib.util.spec_from_file_location("build_under_test", os.path.join(_lib.HERE, "build.py"))
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    assert build.torch_version() == torch.__version__
    assert build.TORCH_LIB == _lib.TORCH_LIB_PATH and torch.__version__ in os.path.basename(build.TORCH_LIB)


@pytest.mark.parametrize("there", [False, True])
def test_the_package_without_the_torch_ops(tmp_path, there):
    """Without the library of the C++ ops (or with one that does not load) the package is imported and its other ops are
    there; the five raise ImportError, with what to do, when they are called."""
    import os
    import shutil
    import subprocess
    import sys

    from basal_b200 import _lib
    copy = tmp_path / "basal_b200"
    shutil.copytree(_lib.HERE, copy, ignore=shutil.ignore_patterns("libbasal200_torch*", "__pycache__"))
    if there:
        (copy / os.path.basename(_lib.TORCH_LIB_PATH)).write_text("not a library")
    prog = ("import torch, basal_b200\nfrom basal_b200 import ops, hybrid\nassert basal_b200.__file__.startswith(%r)\n"
            "print(torch.ops.basal.fp8_act_quant.default)\n"
            "for f, n in ((ops.paged_attention, 6), (ops.kv_append, 6), (ops.gdn_step, 10), (ops.constrain_logits, 1)):\n"
            "    try:\n        f(*[None] * n)\n    except ImportError as e:\n        print('said', 'build.py' in str(e))\n"
            "try:\n    ops.kv_copy_pages([None], [0], [1])\nexcept ImportError as e:\n    print('said', 'build.py' in str(e))\n"
            % str(tmp_path))
    got = subprocess.run([sys.executable, "-c", prog], cwd=tmp_path, env={**os.environ, "PYTHONPATH": str(tmp_path)},
                         capture_output=True, text=True)
    assert got.returncode == 0, got.stderr
    assert got.stdout.split("\n")[:6] == ["basal.fp8_act_quant.default"] + ["said True"] * 5
