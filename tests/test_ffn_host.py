"""The dense FFN and int8 operators without a GPU: the C-ABI of include/wr_ffn.h
(exports, layouts, argument checks before any HIP call), the Python entry
points' refusals, and the oracle's gradients against differences."""
import ctypes
import os
import re

import pytest
import torch

from tests import _ffn_oracle as O
from warp_route import GatedFFN, capi
from warp_route import functional as F
from warp_route.stack import MoEStack

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = open(os.path.join(ROOT, "include", "wr_ffn.h")).read()
FAKE = 0x1000  # 16-byte aligned, never dereferenced: every case fails validation first


def test_exports_every_declared_entry_point():
    names = re.findall(r"WR_API\s+[\w\s\*]+?\b(wr_\w+)\s*\(", HEADER)
    assert sorted(names) == sorted([
        "wr_ffn_saved_row", "wr_ffn_workspace_bytes", "wr_ffn_forward", "wr_ffn_backward",
        "wr_quantize_int8", "wr_int8_workspace_bytes", "wr_int8_matmul",
        "wr_ffn_int8_workspace_bytes", "wr_ffn_int8"])
    for n in names:
        assert hasattr(capi.lib(), n), n
    assert int(re.search(r"WR_INT8_MAX_K (\d+)", HEADER).group(1)) == capi.WR_INT8_MAX_K
    assert "WR_FFN_MAX_DIM (1 << 20)" in HEADER and capi.WR_FFN_MAX_DIM == 1 << 20


def test_struct_layouts():
    # 13 pointers, 4 int32, 2 pointer-sized; 5, 4, 2; 8, 4, 2: no padding.
    assert ctypes.sizeof(capi.WrFfnArgs) == 13 * 8 + 16 + 16
    assert ctypes.sizeof(capi.WrInt8Args) == 5 * 8 + 16 + 16
    assert ctypes.sizeof(capi.WrFfnInt8Args) == 8 * 8 + 16 + 16


def test_sizes():
    lib = capi.lib()
    assert [lib.wr_ffn_saved_row(n) for n in (0, 1, 64, 65, 2816, (1 << 20) + 1)] == [
        0, 64, 64, 128, 2816, 0]
    for T in (0, 1, 17, 4096):
        for back in (0, 1):
            assert lib.wr_ffn_workspace_bytes(back, capi.WR_BF16, 2048, 1408, T) > 0
        assert lib.wr_int8_workspace_bytes(T, 1408, 2048) > 0
        assert lib.wr_ffn_int8_workspace_bytes(2048, 1408, T) > 0
    assert lib.wr_ffn_workspace_bytes(0, capi.WR_FP8_E4M3, 64, 64, 1) == 0
    assert lib.wr_ffn_workspace_bytes(0, capi.WR_F16, 0, 64, 1) == 0
    assert lib.wr_ffn_workspace_bytes(0, capi.WR_F16, 64, 64, -1) == 0
    assert lib.wr_int8_workspace_bytes(1, 64, capi.WR_INT8_MAX_K + 1) == 0
    assert lib.wr_ffn_int8_workspace_bytes(64, capi.WR_INT8_MAX_K + 1, 1) == 0


def ffn_args():
    a = capi.WrFfnArgs()
    for n in ("x", "w_gate", "w_up", "w_down", "out", "saved_gate", "saved_up", "saved_act", "dout",
              "dx", "dw_gate", "dw_up", "dw_down", "workspace"):
        setattr(a, n, FAKE)
    a.dtype, a.batch_size, a.hidden_dim, a.intermediate_dim = capi.WR_F16, 3, 64, 96
    a.workspace_bytes = 16  # too small: nothing gets past the checks
    return a


BAD_FFN = [("dtype", capi.WR_MXFP4, capi.WR_EINVAL_DTYPE), ("dtype", -1, capi.WR_EINVAL_DTYPE),
           ("hidden_dim", 0, capi.WR_EINVAL_SHAPE), ("intermediate_dim", -1, capi.WR_EINVAL_SHAPE),
           ("hidden_dim", (1 << 20) + 1, capi.WR_EINVAL_SHAPE),
           ("batch_size", -1, capi.WR_EINVAL_BATCH), ("x", FAKE + 8, capi.WR_EINVAL_ALIGN),
           ("w_down", FAKE + 2, capi.WR_EINVAL_ALIGN), ("workspace", None, capi.WR_EINVAL_WORKSPACE),
           ("workspace_bytes", 16, capi.WR_EINVAL_WORKSPACE)]


@pytest.mark.parametrize("entry", ["wr_ffn_forward", "wr_ffn_backward"])
@pytest.mark.parametrize("field,value,want", BAD_FFN + [
    ("w_down", None, capi.WR_EINVAL_NULL), ("saved_act", None, capi.WR_EINVAL_NULL)])
def test_ffn_validation(entry, field, value, want):
    a = ffn_args()
    setattr(a, field, value)
    assert getattr(capi.lib(), entry)(ctypes.byref(a), None) == want
    assert getattr(capi.lib(), entry)(None, None) == capi.WR_EINVAL_NULL


def test_ffn_validation_of_one_direction():
    lib = capi.lib()
    a = ffn_args()
    a.out = None
    assert lib.wr_ffn_forward(ctypes.byref(a), None) == capi.WR_EINVAL_NULL
    a = ffn_args()
    a.dx = FAKE + 4
    assert lib.wr_ffn_backward(ctypes.byref(a), None) == capi.WR_EINVAL_ALIGN
    a.dx, a.dout = FAKE, None
    assert lib.wr_ffn_backward(ctypes.byref(a), None) == capi.WR_EINVAL_NULL
    a = ffn_args()  # what no wanted gradient reads may be absent
    a.dx = a.dw_gate = a.dw_up = None
    a.x = a.w_gate = a.w_up = a.w_down = a.saved_gate = a.saved_up = None
    assert lib.wr_ffn_backward(ctypes.byref(a), None) == capi.WR_EINVAL_WORKSPACE
    a.batch_size = 0  # no tokens, no weight gradients: nothing to do
    a.dw_down = None
    assert lib.wr_ffn_backward(ctypes.byref(a), None) == capi.WR_OK
    assert lib.wr_ffn_forward(ctypes.byref(a), None) == capi.WR_OK


def test_int8_validation():
    lib = capi.lib()

    def matmul(**bad):
        a = capi.WrInt8Args()
        a.x = a.x_scale = a.w = a.w_scale = a.out = a.workspace = FAKE
        a.out_dtype, a.rows, a.out_features, a.in_features, a.workspace_bytes = 1, 3, 64, 96, 16
        for k, v in bad.items():
            setattr(a, k, v)
        return lib.wr_int8_matmul(ctypes.byref(a), None)

    assert matmul() == capi.WR_EINVAL_WORKSPACE
    assert matmul(out_dtype=capi.WR_FP8_E4M3) == capi.WR_EINVAL_DTYPE
    assert matmul(in_features=capi.WR_INT8_MAX_K + 1) == capi.WR_EINVAL_SHAPE
    assert matmul(out_features=0) == capi.WR_EINVAL_SHAPE
    assert matmul(rows=-1) == capi.WR_EINVAL_BATCH
    assert matmul(w_scale=None) == capi.WR_EINVAL_NULL
    assert matmul(w=FAKE + 1) == capi.WR_EINVAL_ALIGN
    assert matmul(rows=0) == capi.WR_OK

    def ffn(**bad):
        a = capi.WrFfnInt8Args()
        for n in ("x", "w_gate", "s_gate", "w_up", "s_up", "w_down", "s_down", "out", "workspace"):
            setattr(a, n, FAKE)
        a.dtype, a.batch_size, a.hidden_dim, a.intermediate_dim, a.workspace_bytes = 2, 3, 64, 96, 16
        for k, v in bad.items():
            setattr(a, k, v)
        return lib.wr_ffn_int8(ctypes.byref(a), None)

    assert ffn() == capi.WR_EINVAL_WORKSPACE
    assert ffn(dtype=9) == capi.WR_EINVAL_DTYPE
    assert ffn(intermediate_dim=capi.WR_INT8_MAX_K + 1) == capi.WR_EINVAL_SHAPE
    assert ffn(batch_size=-2) == capi.WR_EINVAL_BATCH
    assert ffn(s_up=None) == capi.WR_EINVAL_NULL
    assert ffn(x=FAKE + 8) == capi.WR_EINVAL_ALIGN
    assert ffn(batch_size=0) == capi.WR_OK

    q = lib.wr_quantize_int8
    assert q(FAKE, capi.WR_MXFP4, 1, 8, FAKE, FAKE, None) == capi.WR_EINVAL_DTYPE
    assert q(FAKE, capi.WR_F32, -1, 8, FAKE, FAKE, None) == capi.WR_EINVAL_BATCH
    assert q(FAKE, capi.WR_F32, 1, 0, FAKE, FAKE, None) == capi.WR_EINVAL_SHAPE
    assert q(FAKE, capi.WR_F32, 1, 8, None, FAKE, None) == capi.WR_EINVAL_NULL
    assert q(FAKE + 4, capi.WR_F32, 1, 8, FAKE, FAKE, None) == capi.WR_EINVAL_ALIGN
    assert q(FAKE, capi.WR_F32, 0, 8, FAKE, FAKE, None) == capi.WR_OK
    assert "16-byte" in capi.status_str(capi.WR_EINVAL_ALIGN)


@pytest.mark.parametrize("n", [(1 << 28) + 1, (1 << 31) - 1])
def test_more_rows_than_the_grid_is_planned_for_are_refused(n):
    """Rows are rounded up to tiles in 32 bits: 2**31 - 1 of them would wrap."""
    lib = capi.lib()
    assert n > capi.WR_FFN_MAX_ROWS
    a = capi.WrFfnArgs()
    for name, _ in capi.WrFfnArgs._fields_[:13]:
        setattr(a, name, FAKE)
    a.dtype, a.batch_size, a.hidden_dim, a.intermediate_dim = capi.WR_F16, n, 1, 1
    a.workspace, a.workspace_bytes = FAKE, 1 << 60
    assert lib.wr_ffn_forward(ctypes.byref(a), None) == capi.WR_EINVAL_BATCH
    assert lib.wr_ffn_backward(ctypes.byref(a), None) == capi.WR_EINVAL_BATCH
    assert lib.wr_ffn_workspace_bytes(0, capi.WR_F16, 1, 1, n) == 0
    assert lib.wr_int8_workspace_bytes(n, 1, 1) == 0
    assert lib.wr_ffn_int8_workspace_bytes(1, 1, n) == 0
    assert lib.wr_int8_workspace_bytes(capi.WR_FFN_MAX_ROWS, 1, 1) >= 16 * capi.WR_FFN_MAX_ROWS
    assert lib.wr_quantize_int8(FAKE, capi.WR_F16, n, 8, FAKE, FAKE, None) == capi.WR_EINVAL_BATCH


@pytest.mark.parametrize("cols", [(1 << 30) + 1, (1 << 31) - 1])
def test_columns_past_the_row_loop_are_refused(cols):
    """A step past the last column has to fit 32 bits, or the loop would not end."""
    assert cols > capi.WR_INT8_MAX_COLS
    st = capi.lib().wr_quantize_int8(FAKE, capi.WR_F16, 1, cols, FAKE, FAKE, None)
    assert st == capi.WR_EINVAL_SHAPE


def test_python_entry_points_refuse_host_tensors():
    x, w = torch.zeros(2, 8), torch.zeros(4, 8)
    for call in (lambda: F.gated_ffn(x, w, w, w.t().contiguous()), lambda: F.quantize_int8(x),
                 lambda: F.gated_ffn_int8(x, *[w.to(torch.int8), torch.ones(4)] * 3),
                 lambda: F.int8_matmul(x.to(torch.int8), torch.ones(2), w.to(torch.int8),
                                       torch.ones(4))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    with pytest.raises(RuntimeError, match="dimension"):
        F.gated_ffn(torch.tensor(1.0), w, w, w)
    with pytest.raises(ValueError, match="dimension"):
        F.quantize_int8(torch.tensor(1.0))
    with pytest.raises(ValueError, match="x_scale"):
        F.int8_matmul(x.to(torch.int8), torch.ones(3), w.to(torch.int8), torch.ones(4))


def test_modules_refuse():
    with pytest.raises(ValueError, match="dtype"):
        GatedFFN(8, 8, torch.float8_e4m3fn)
    assert [tuple(p.shape) for p in GatedFFN(8, 24).parameters()] == [(24, 8), (24, 8), (8, 24)]
    layers = [(torch.zeros(4, 8), torch.zeros(1))] * 2
    with pytest.raises(ValueError, match="one entry per layer"):
        MoEStack(layers, 4, 8, 8, 2, shared=[None])


def test_oracle_gradients_against_differences():
    """The formulas the kernels are tested against are the derivative of the
    forward formula: central differences in 64 bits, step 1e-6 (truncation of
    the order 1e-12, cancellation 1e-16 / 1e-6 of values of order 1)."""
    gen = torch.Generator().manual_seed(5)
    shapes = [(3, 6), (5, 6), (5, 6), (6, 5)]
    args = [torch.randn(s, generator=gen, dtype=torch.float64) for s in shapes]
    dy = torch.randn(3, 6, generator=gen, dtype=torch.float64)
    grads = [g for g, _ in O.ffn_grads(*args, dy)]
    for i, a in enumerate(args):
        for j in range(a.numel()):
            vals = []
            for sign in (1, -1):
                b = [t.clone() for t in args]
                b[i].view(-1)[j] += sign * 1e-6
                vals.append((O.ffn(*b)[0] * dy).sum())
            diff = ((vals[0] - vals[1]) / 2e-6).item()
            assert abs(diff - grads[i].view(-1)[j].item()) < 1e-7
