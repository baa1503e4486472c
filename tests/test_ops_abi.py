"""The operators' library on the CPU: what the header declares is exported, host
argument errors come back as codes before anything launches, and tensors that
are not on a GPU are refused.  No kernel is launched here."""

from __future__ import annotations

import ctypes
import os
import re
import shutil
import subprocess

import pytest
import torch

import minispeed_amd as ms
from minispeed_amd import build
from minispeed_amd.ops import _native

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "minispeed_ops.h")
P, I32, I64, F = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float


class Tokens(ctypes.Structure):
    _fields_ = [("data", P), ("n", I64), ("inner", I64), ("outer_stride", I64),
                ("inner_stride", I64), ("wide", I32), ("reserved", I32)]


class Rows(ctypes.Structure):
    _fields_ = [("data", P), ("n", I64), ("width", I64), ("inner", I64), ("outer_stride", I64),
                ("inner_stride", I64), ("dtype", I32), ("reserved", I32)]


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(build.OPS_OUTPUT)
    lib.ms_ops_error_string.restype = ctypes.c_char_p
    lib.ms_embedding_grad_workspace.restype = I64
    lib.ms_embedding_grad_workspace.argtypes = [I64, I64, I64]
    lib.ms_logprobs_workspace.restype = I64
    lib.ms_logprobs_workspace.argtypes = [I64, I64, I32, I32]
    return lib


def test_every_declared_function_is_exported(lib):
    text = re.sub(r"/\*.*?\*/", "", open(HEADER, encoding="utf-8").read(), flags=re.S)
    names = set(re.findall(r"\b(ms_[a-z0-9_]+)\s*\(", text))
    assert {"ms_embedding", "ms_logprobs", "ms_act8"} <= names
    for name in names:
        assert hasattr(lib, name), name
    assert lib.ms_ops_abi_version() == _native.ABI_VERSION == _native.load().abi_version()


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not available")
def test_struct_layout_is_plain_c(tmp_path):
    src = tmp_path / "probe.c"
    src.write_text('#include <stdio.h>\n#include "minispeed_ops.h"\nint main(void) {\n'
                   'printf("%zu %zu %d", sizeof(ms_tokens_t), sizeof(ms_rows_t), MS_OPS_BLOCK);\n'
                   'return 0; }\n')
    exe = tmp_path / "probe"
    subprocess.run(["gcc", "-Wall", "-Werror", "-I", os.path.dirname(HEADER), str(src), "-o", str(exe)],
                   check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()
    assert [int(x) for x in out] == [ctypes.sizeof(Tokens), ctypes.sizeof(Rows), 32]


def test_argument_errors_come_back_before_a_launch(lib):
    ids, bad_ids = Tokens(8, 4, 4, 0, 1, 1, 0), Tokens(None, 4, 4, 0, 1, 1, 0)
    table, none = Rows(8, 10, 16, 10, 0, 16, 1, 0), Rows(8, 0, 16, 1, 0, 16, 1, 0)
    odd = Rows(8, 10, 16, 10, 0, 16, 7, 0)
    ref = ctypes.byref
    e = lib.ms_embedding
    assert e(None, ref(table), F(1), P(8), None) == -1
    assert e(ref(bad_ids), ref(table), F(1), P(8), None) == -1
    assert e(ref(ids), ref(odd), F(1), P(8), None) == -1
    assert e(ref(ids), ref(none), F(1), P(8), None) == -1
    assert e(ref(ids), ref(table), F(1), None, None) == -1
    empty = Tokens(None, 0, 1, 0, 0, 1, 0)
    assert e(ref(empty), ref(table), F(1), None, None) == 0
    g = lib.ms_embedding_grad
    rows = Rows(8, 4, 16, 4, 0, 16, 1, 0)
    need = lib.ms_embedding_grad_workspace(4, 10, 16)
    assert need >= 0
    assert g(ref(ids), ref(table), I64(10), F(1), I64(-1), P(8), P(16), I64(need), None) == -1
    assert g(ref(ids), ref(rows), I64(-1), F(1), I64(-1), P(8), P(16), I64(need), None) == -1
    assert g(ref(ids), ref(rows), I64(10), F(1), I64(-1), None, P(16), I64(need), None) == -1
    long = Tokens(8, 2 ** 30 + 1, 2 ** 30 + 1, 0, 1, 1, 0)
    assert lib.ms_embedding_grad_workspace(2 ** 30 + 1, 10, 16) == -1
    assert g(ref(long), ref(Rows(8, 2 ** 30 + 1, 16, 2 ** 30 + 1, 0, 16, 1, 0)), I64(10), F(1),
             I64(-1), P(16), P(16), I64(1 << 40), None) == -1
    if need:
        assert g(ref(ids), ref(rows), I64(10), F(1), I64(-1), P(16), P(16), I64(need - 1), None) == -2
        assert g(ref(ids), ref(rows), I64(10), F(1), I64(-1), P(16), P(8), I64(need), None) == -2
    l = lib.ms_logprobs
    need = lib.ms_logprobs_workspace(4, 16, 1, 2)
    args = lambda x, t, top, lp=8, lse=8: (ref(x), ref(t), I64(-100), I32(top), P(lp), None, P(lse),  # noqa: E731
                                           P(8), P(8), P(16), I64(need), None)
    assert l(*args(rows, empty, 0)) == -1
    assert l(*args(rows, ids, 17)) == -1
    assert l(*args(rows, ids, -1)) == -1
    assert l(*args(rows, ids, 2, lp=None)) == -1
    assert l(*args(rows, ids, 2, lse=None)) == -1
    assert l(*args(Rows(8, 4, 0, 4, 0, 16, 1, 0), ids, 0)) == -1
    lg = lib.ms_logprobs_grad
    assert lg(ref(rows), ref(ids), I64(-100), None, None, None, None, P(8), None) == -1
    assert lg(ref(rows), ref(ids), I64(-100), P(8), None, None, P(8), P(8), None) == -1
    assert lib.ms_pack8(P(8), I32(3), I64(4), P(8), P(8), None) == -1
    assert lib.ms_pack8(None, I32(1), I64(4), P(8), P(8), None) == -1
    assert lib.ms_pack8(None, I32(1), I64(0), None, None, None) == 0
    assert lib.ms_unpack8(P(8), P(8), I64(-1), I32(1), P(8), None) == -1
    assert lib.ms_unpack8(P(8), None, I64(4), I32(1), P(8), None) == -1
    a = lib.ms_act8
    assert a(ref(rows), None, I32(4), P(8), P(8), P(8), None, None, None) == -1
    assert a(ref(rows), None, I32(3), P(8), P(8), P(8), P(8), P(8), None) == -1
    assert a(ref(rows), ref(rows), I32(0), P(8), P(8), P(8), P(8), P(8), None) == -1
    assert a(ref(rows), ref(table), I32(3), P(8), P(8), P(8), P(8), P(8), None) == -1
    assert a(ref(rows), None, I32(0), None, P(8), P(8), None, None, None) == -1
    ag = lib.ms_act8_grad
    assert ag(P(8), P(8), None, None, P(8), I32(1), I32(3), I64(4), P(8), P(8), None, None) == -1
    assert ag(P(8), P(8), None, None, P(8), I32(1), I32(0), I64(4), P(8), P(8), None, None) == -1
    assert ag(P(8), P(8), None, None, None, I32(1), I32(0), I64(4), P(8), None, None, None) == -1
    for code, word in ((0, b"ok"), (-1, b"invalid"), (-2, b"workspace"), (-77, b"unknown")):
        assert word in lib.ms_ops_error_string(code)


def test_cpu_tensors_are_refused():
    x, ids = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="cpu"):
        ms.ops.embedding(ids, x)
    with pytest.raises(RuntimeError, match="cpu"):
        ms.ops.embedding_grad(x, ids, 10)
    with pytest.raises(RuntimeError, match="cpu"):
        ms.ops.token_logprobs(x, ids)
    with pytest.raises(RuntimeError, match="cpu"):
        ms.ops.pack8(x)
    with pytest.raises(RuntimeError, match="cpu"):
        ms.ops.activation8(x, "gelu")


def test_a_missing_build_is_reported(monkeypatch):
    from minispeed_amd._native import NativeLibraryError

    def missing(name):
        raise ImportError("no file")

    monkeypatch.setattr(_native, "_module", None)
    monkeypatch.setattr(_native.importlib, "import_module", missing)
    with pytest.raises(NativeLibraryError, match="minispeed_amd.build"):
        _native.load()


def test_calls_beyond_one_launch_are_refused(lib):
    ref, n = ctypes.byref, 2 ** 36
    assert lib.ms_pack8(P(16), I32(1), I64(n * 2), P(16), P(16), None) == -1
    assert lib.ms_unpack8(P(16), P(16), I64(n), I32(1), P(16), None) == -1
    ids = Tokens(16, 2 ** 30, 2 ** 30, 0, 1, 1, 0)
    table, logits = Rows(16, 10, 4096, 10, 0, 4096, 1, 0), Rows(16, 2 ** 30, 40000, 2 ** 30, 0,
                                                                40000, 1, 0)
    assert lib.ms_embedding(ref(ids), ref(table), F(1), P(16), None) == -1
    assert lib.ms_logprobs(ref(logits), ref(ids), I64(-100), I32(0), P(16), None, P(16), None,
                           None, None, I64(0), None) == -1
    assert lib.ms_logprobs_grad(ref(logits), ref(ids), I64(-100), P(16), None, P(16), None, P(16),
                                None) == -1
    rows = Rows(16, 2 ** 30, 4096, 2 ** 30, 0, 4096, 1, 0)
    assert lib.ms_embedding_grad(ref(ids), ref(rows), I64(10), F(1), I64(-1), P(16), P(16),
                                 I64(2 ** 62), None) == -1


@pytest.mark.parametrize("dtype", ["float32", None, 5, torch.zeros(1)])
def test_a_checkpoint_of_no_dtype_is_refused(dtype):
    held = ms.ops.Checkpoint8(torch.zeros(32, dtype=torch.int8), torch.ones(1, dtype=torch.uint8),
                              (32,), dtype)
    with pytest.raises(TypeError, match="torch.dtype"):
        ms.ops.unpack8(held)


def test_two_checkpoints_of_different_tensors_are_refused():
    held = [ms.ops.Checkpoint8(torch.zeros(32, dtype=torch.int8), torch.ones(1, dtype=torch.uint8),
                               shape, dtype)
            for shape, dtype in (((4, 8), torch.float32), ((8, 4), torch.float32),
                                 ((4, 8), torch.float16))]
    grad = torch.zeros(4, 8)
    for up in held[1:]:
        with pytest.raises(ValueError, match="checkpoint"):
            ms.ops.activation8_grad((held[0], up), grad, "swiglu")


def test_sizes_whose_products_pass_64_bits_are_refused(lib):
    """Products that come out small or negative would make a small launch over rows of any length."""
    ref, most = ctypes.byref, 2 ** 63 - 1
    assert lib.ms_pack8(P(16), I32(1), I64(most), P(16), P(16), None) == -1
    assert lib.ms_unpack8(P(16), P(16), I64(most - 3), I32(1), P(16), None) == -1
    assert lib.ms_act8_grad(P(16), P(16), None, None, P(16), I32(1), I32(0), I64(most), P(16), None,
                            None, None) == -1
    for n, width in ((2 ** 31 - 1, 2 ** 33), (2 ** 31 - 1, 2 ** 34), (2 ** 30, 2 ** 34 + 2)):
        assert lib.ms_act8(ref(Rows(16, n, width, n, 0, width, 1, 0)), None, I32(0), P(16), P(16),
                           P(16), None, None, None) == -1
    ids = Tokens(16, 4, 4, 0, 1, 1, 0)
    for vocab, width in ((2 ** 31 - 1, 2 ** 32), (2 ** 31 - 1, 2 ** 33), (5, 2 ** 61), (5, 2 ** 62),
                         (1, most)):
        assert lib.ms_embedding_grad_workspace(4, vocab, width) == -1
        assert lib.ms_embedding_grad(ref(ids), ref(Rows(16, 4, width, 4, 0, width, 1, 0)), I64(vocab),
                                     F(1), I64(-1), P(16), P(16), I64(most), None) == -1
        assert lib.ms_embedding(ref(ids), ref(Rows(16, vocab, width, vocab, 0, width, 1, 0)), F(1),
                                P(16), None) == -1
    many = Tokens(16, 2 ** 31 - 1, 2 ** 31 - 1, 0, 1, 1, 0)
    assert lib.ms_embedding(ref(many), ref(Rows(16, 1, 2 ** 34, 1, 0, 0, 1, 0)), F(1), P(16),
                            None) == -1
