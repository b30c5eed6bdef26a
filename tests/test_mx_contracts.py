"""What the MX FP4 operators promise beside their values: how their kernels read memory,
and what happens at the edges of the calls."""

import re

import pytest
import torch

from conftest import REPO
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
