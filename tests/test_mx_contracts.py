"""What the MX FP4 operators promise beside their values: how their kernels read memory,
and what happens at the edges of the calls."""

import re
import sys
import sysconfig

import pytest
import torch

from conftest import REPO
from triton_chip_benchmarks_b200 import build as tcb_build
from triton_chip_benchmarks_b200 import mx

gpu = pytest.mark.gpu

CSRC = REPO / "triton_chip_benchmarks_b200" / "csrc"


def code(path) -> str:
    """A source without its comments."""
    return re.sub(r"//[^\n]*", "", re.sub(r"/\*.*?\*/", "", path.read_text(), flags=re.S))


def test_kernels_that_start_early_read_with_ordinary_loads():
    """A kernel launched beside the writers of its inputs must not use the read-only
    path, which is for memory that nobody writes while the kernel runs."""
    early = [p for p in sorted(CSRC.glob("*.cu")) if "wait_for_previous_kernels" in code(p)]
    assert {p.name for p in early} >= {"tcb_mx_convert.cu", "tcb_mx_rows.cu", "tcb_gemm_pair.cu"}
    for path in [*early, *sorted(CSRC.glob("tcb_mx*.cuh"))]:
        for word in ("__ldg", "__restrict__", "ld.global.nc", "__ldca", "__ldcg"):
            assert word not in code(path), (path.name, word)


@gpu
@pytest.mark.parametrize("shape", [(3, 64), (2, 3, 64)])
def test_a_layer_without_outputs_has_zero_gradients(cuda, shape):
    """dx sums over the outputs: over none it is zero, as dw is over no rows."""
    x, w = torch.ones(shape, device=cuda, dtype=torch.bfloat16), torch.ones(0, 64, device=cuda)
    y, saved = mx.linear_forward(x, w)
    assert y.shape == (*shape[:-1], 0)
    dx, dw = mx.linear_backward(torch.zeros(*shape[:-1], 0, device=cuda, dtype=torch.bfloat16), saved)
    assert dx.shape == x.shape and dx.dtype == x.dtype and (dx == 0).all()
    assert dw.shape == (0, 64) and dw.dtype == w.dtype


@gpu
def test_the_training_step_takes_status_words(cuda):
    x, w = torch.ones(40, 64, device=cuda), torch.ones(96, 64, device=cuda)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    y, saved = mx.linear_forward(x, w, status=status)
    mx.linear_backward(torch.ones_like(y), saved, status=status)
    assert status.item() == 0
    for wrong, error in ((torch.zeros(1, dtype=torch.int32), ValueError),
                         (torch.zeros(1, dtype=torch.int64, device=cuda), TypeError)):
        with pytest.raises(error, match="status"):
            mx.linear_forward(x, w, status=wrong)
        for needs in ({"need_dx": False}, {"need_dw": False}):
            with pytest.raises(error, match="status"):
                mx.linear_backward(torch.ones_like(y), saved, status=wrong, **needs)


def test_the_products_reach_the_library_with_their_status_word(monkeypatch):
    """linear_forward and linear_backward hand their word to each of their products."""
    words = []
    monkeypatch.setattr(mx, "matmul", lambda a, b, *, dtype, status=None: (
        words.append(status), torch.zeros(a.rows, b.rows, dtype=dtype))[1])
    monkeypatch.setattr(mx, "_quantizable", lambda x, rule: x)
    monkeypatch.setattr(mx, "_quantize", lambda *args: None)
    word = object()
    y, saved = mx.linear_forward(torch.zeros(4, 32), torch.zeros(8, 32), status=word)
    saved.x.index = -1  # host tensors
    mx.linear_backward(torch.zeros(4, 8), saved, status=word)
    assert words == [word] * 3


# ------------------------------------------------------- the module of entry points
def test_the_library_is_built_where_the_python_module_cannot_be(monkeypatch, tmp_path, capsys):
    monkeypatch.setattr(tcb_build, "CALLS", tmp_path / "_tcb_calls.so")
    monkeypatch.setattr(sysconfig, "get_paths", lambda: {"include": str(tmp_path)})  # no Python.h
    assert tcb_build.build() == tcb_build.LIBRARY and tcb_build.LIBRARY.exists()
    assert not tcb_build.CALLS.exists() and "tcb_pycalls.c" in capsys.readouterr().err


def test_the_python_module_is_named_for_its_python():
    assert tcb_build.CALLS.name.endswith(sysconfig.get_config_var("EXT_SUFFIX"))


def without_module(native, monkeypatch):
    """_native.calls() where _tcb_calls cannot be imported."""
    package = native.__package__
    monkeypatch.setitem(sys.modules, f"{package}._tcb_calls", None)
    monkeypatch.delattr(sys.modules[package], "_tcb_calls", raising=False)
    monkeypatch.setattr(native, "_bound_to", None)
    monkeypatch.setattr(native, "_calls", None)
    return native.calls()


def test_entry_points_without_the_python_module(native, monkeypatch):
    calls = without_module(native, monkeypatch)
    p = 0x1000  # never dereferenced
    assert not hasattr(calls, "bind")
    assert calls.tcb_mx_quantize(0, p, 4, 4, 3, 0, p, p, None, None, None) == native.ERR_INVALID_ARGUMENT
    assert calls.tcb_mx_gemm(p, p, p, p, None, 0, p, 8, 1 << 32, 8, 32, None, None) == \
        native.ERR_INVALID_ARGUMENT  # a size past int is not cut off
    assert calls.tcb_mx_gemm(None, None, None, None, None, 0, None, 8, 0, 8, 32, None, None) == native.OK
    with pytest.raises(TypeError):
        calls.tcb_mx_dequantize(0, p, p)
    with pytest.raises(TypeError):
        calls.tcb_mx_quantize(0, "x", 4, 4, 4, 0, p, p, None, None, None)
    with pytest.raises(OverflowError):
        calls.tcb_mx_quantize(0, 1 << 70, 4, 4, 4, 0, p, p, None, None, None)


@gpu
def test_operators_without_the_python_module(cuda, native, monkeypatch):
    x, w = torch.randn(3, 64, device=cuda).bfloat16(), torch.randn(40, 64, device=cuda)
    q = mx.quantize(w)
    expected = mx.linear(x, q), mx.matmul(q, q), mx.dequantize(q)
    without_module(native, monkeypatch)
    again = mx.quantize(w)
    for got, want in zip((mx.linear(x, again), mx.matmul(again, again), mx.dequantize(again)), expected):
        assert torch.equal(got, want)
