"""The low-bit path's edges without a GPU: which residuals its products take, with which row stride, and the order of loads from
tensor memory and of what uses them."""
import os
import re

import pytest
import torch

from dtas_b200 import _abi, ops
from dtas_b200.build import CSRC

F16 = torch.float16


def row_stride(rows, n, *residuals):
    """The row stride with which a product of `rows` rows of n reads these residuals."""
    out = torch.empty(rows, n, dtype=F16)
    return ops._tail_args("gemm_f8", out, n, rows, None, residuals[0], residuals[1] if len(residuals) > 1 else None, None)[2]


def z(*shape):
    return torch.zeros(*shape, dtype=F16)


@pytest.mark.parametrize("residual,stride", [
    (z(4, 8), 8), (z(1, 4, 8), 8), (z(2, 2, 8), 8), (z(4, 20)[:, 4:12], 20), (z(1, 4, 20)[:, :, 4:12], 20), (z(8, 8)[::2], 16)])
def test_residual_rows(residual, stride):
    assert row_stride(4, 8, residual) == stride
    assert row_stride(4, 8, residual, residual) == stride


@pytest.mark.parametrize("residual", [z(8), z(1, 8), z(1, 1, 8), z(8, 1)])
def test_residual_of_one_row(residual):
    assert row_stride(1, 8, residual) == 8


def test_residual_of_one_column():
    assert row_stride(4, 1, z(4, 1)) == 1 and row_stride(4, 1, z(4, 6)[:, 2:3]) == 6


@pytest.mark.parametrize("residual", [
    z(8).expand(4, 8), z(1, 8).expand(4, 8), z(1, 1, 8).expand(1, 4, 8),      # a row stride of 0
    z(8, 4), z(16, 2), z(32), z(1, 8, 4),                                    # as many elements in another shape
    z(8, 4).t(), z(4, 16)[:, ::2],                                           # an inner stride
    z(2, 4, 8)[:, ::2], z(2, 2, 20)[:, :, :8],                               # rows that no one stride describes
    z(100).as_strided((4, 8), (4, 1)),                                       # rows that overlap
    z(4, 8).float()])
def test_residuals_that_a_row_stride_does_not_describe_are_refused(residual):
    for args in ((residual,), (z(4, 8), residual)):
        with pytest.raises(_abi.DtasError) as e:
            row_stride(4, 8, *args)
        assert e.value.code == _abi.EINVAL


def test_two_residuals_share_a_row_stride():
    with pytest.raises(_abi.DtasError):
        row_stride(4, 8, z(4, 8), z(4, 20)[:, :8])


def test_every_wait_for_tensor_memory_names_its_registers():
    """A tcgen05.ld's destination registers are the compiler's as soon as the load is issued: a wait that does not name
    them does not order arithmetic on them."""
    src = "".join(open(os.path.join(CSRC, f)).read() for f in sorted(os.listdir(CSRC)))
    assert src.count("tcgen05.wait::ld") == 1 and "void tmem_ld_wait(uint32_t (&r)[N])" in src
    lines = src.split("\n")
    for i, line in enumerate(lines):
        for words in re.findall(r"tmem_ld(?:16|32)\(t_addr[^;]*, (\w+)\);", line):
            assert any(f"tmem_ld_wait({words})" in x for x in lines[i:i + 16]), line
    assert not re.search(r"tmem_ld_wait\(\s*\)", src)


def test_activations_do_not_take_the_read_only_path():
    """A kernel may begin while the one that writes its x still runs: loads that promise that x does not change while
    the kernel runs (ld.global.nc) are not for it."""
    src = open(os.path.join(CSRC, "gemv_w4.cu")).read()
    assert "__ldg" not in src and "ld.global.nc" not in src
