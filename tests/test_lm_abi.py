"""CPU-side checks of the language-model operators' C ABI: bad arguments are refused on the
host, before any CUDA call."""
import ctypes

from deltagrid_b200 import _lib

F = ctypes.c_float


def test_gated_scan_refusals():
    L = _lib.lib()
    tail = [None] * 8
    assert L.dg_gated_scan_forward(7, 1, 4, 8, None, 0, 0, None, 0, 0, None, 0, 0, *tail) == -1
    assert L.dg_gated_scan_forward(1, 1, 4, 8, None, 0, 0, None, 0, 0, None, 0, 0, *tail) == -2      # f64
    assert L.dg_gated_scan_forward(0, 1, 4, 8, None, 0, 0, None, 0, 0, None, 0, 0, *tail) == -1      # null x
    assert L.dg_gated_scan_forward(0, -1, 4, 8, None, 0, 0, None, 0, 0, None, 0, 0, *tail) == -1
    assert L.dg_gated_scan_forward(0, 0, 4, 8, None, 0, 0, None, 0, 0, None, 0, 0, *tail) == 0       # nothing to do
    one = ctypes.c_float(0)
    p = ctypes.addressof(one)
    args = [0, 1, 4, 8, p, 0, 0, p, 0, 0, p, 0, 0, None, None, p, p, 0, 0, None, p, 0, 0, p, 0, 0]
    assert L.dg_gated_scan_backward(*args, None, 0, 0, None, None, None) == -1        # out_gate without its gradient
    assert L.dg_gated_scan_step(0, 1, 8, None, 0, None, 0, None, 0, None, None, None) == -1
    assert L.dg_gated_scan_step(1, 1, 8, None, 0, None, 0, None, 0, None, None, None) == -2


def test_gated_ffn_refusals():
    L = _lib.lib()
    assert L.dg_gated_ffn_forward(3, 4, 8, 8, 0, None, 8, None, None, None, None, None) == -1
    assert L.dg_gated_ffn_forward(1, 4, 8, 8, 0, None, 8, None, None, None, None, None) == -2
    assert L.dg_gated_ffn_forward(3, 4, 8, 8, 9, None, 8, None, None, None, None, None) == -1        # activation
    assert L.dg_gated_ffn_forward(3, 4, 0, 8, 0, None, 8, None, None, None, None, None) == -1
    assert L.dg_gated_ffn_forward(3, 0, 8, 8, 0, None, 8, None, None, None, None, None) == 0
    one = ctypes.c_float(0)
    p = ctypes.addressof(one)
    assert L.dg_gated_ffn_forward(3, 4, 8, 8, 0, p, 7, p, None, p, None, None) == -1                 # ldx < D
    n = L.dg_gated_ffn_backward_workspace_size(3, 100, 64, 32)
    assert n >= 100 * 64 * 2
    assert L.dg_gated_ffn_backward_workspace_size(1, 100, 64, 32) == 0
    assert L.dg_gated_ffn_backward(3, 100, 64, 32, 0, p, 64, p, None, p, 32, p, p, p, None, 0, None, None) == -4


def test_sample_refusals():
    L = _lib.lib()
    tail = [None, F(1.0), None, 0, None, F(1.0), None, F(0.0), None, None, None]
    assert L.dg_sample(0, 1, 10, None, 10, None, *tail) == -1
    assert L.dg_sample(1, 1, 10, None, 10, None, *tail) == -2
    assert L.dg_sample(0, 1, 0, None, 10, None, *tail) == -1
    assert L.dg_sample(0, 0, 10, None, 10, None, *tail) == 0
