"""The low-bit operators' C ABI without a GPU: packed sizes, and refusals that happen before anything touches a device."""
import ctypes

import pytest
import torch

from cntk_amd import QuantizerLogicError, lowbit

INVALID, LOGIC = 1, 2


def up(a, b):
    return -(-a // b)


def test_packed_sizes():
    L = lowbit._bind()
    for rows in (0, 1, 16, 17, 64, 65, 2048, 9304):
        for cols in (0, 1, 31, 32, 33, 128, 129, 429, 2048, 100000):
            assert L.cntkq_mx4_bytes(rows, cols) == up(rows, 16) * 2 * up(cols, 256) * 1024 + up(rows, 64) * 2 * up(cols, 256) * 256
            assert L.cntkq_save8_bytes(rows, cols) == rows * up(cols, 32) * 33
    # few rows that are not kept need no workspace
    assert L.cntkq_mx4_linear_workspace_bytes(1, 9304, 2048, 2, 0) == 0
    assert L.cntkq_mx4_linear_workspace_bytes(1, 9304, 2048, 2, 1) == L.cntkq_mx4_bytes(1, 2048)
    assert L.cntkq_mx4_linear_workspace_bytes(4096, 9304, 2048, 2, 0) == L.cntkq_mx4_bytes(4096, 2048)
    assert L.cntkq_weight_gradient_workspace_bytes(5, 6, 7, 9) == 0


def test_sizes_of_what_is_empty():
    """Any side may be 0, alone or with others: no result is no workspace, whatever the number of rows."""
    L = lowbit._bind()
    sides = (0, 1, 16, 17, 1024, 1025, 2000, 1 << 22)
    for m in sides:
        for k in sides:
            for dtype in (0, 1, 2):
                assert L.cntkq_weight_gradient_workspace_bytes(m, 0, k, dtype) == 0
                L.cntkq_weight_gradient_workspace_bytes(m, k, 0, dtype)
                L.cntkq_weight_gradient_workspace_bytes(0, m, k, dtype)
                for save in (0, 1):
                    assert L.cntkq_mx4_linear_workspace_bytes(0, m, k, dtype, save) == 0
                    assert L.cntkq_mx4_linear_workspace_bytes(m, k, 0, dtype, save) == 0
                    L.cntkq_mx4_linear_workspace_bytes(m, 0, k, dtype, save)
            assert L.cntkq_mx4_bytes(m, 0) == L.cntkq_mx4_bytes(0, k) == L.cntkq_save8_bytes(m, 0) == L.cntkq_save8_bytes(0, k) == 0


def test_refusals_before_the_device():
    L = lowbit._bind()
    h = ctypes.create_string_buffer(4096)  # never read: the arguments are refused first
    p, odd = 4096, 4097
    q = L.cntkq_mx4_bytes(20, 40)
    s = L.cntkq_save8_bytes(20, 40)
    refused = [
        (INVALID, b"handle", L.cntkq_mx4_quantize_async, None, p, 0, 20, 40, 40, 1, p, q, None, 0),
        (LOGIC, b"element type", L.cntkq_mx4_quantize_async, h, p, 3, 20, 40, 40, 1, p, q, None, 0),
        (LOGIC, b"size", L.cntkq_mx4_quantize_async, h, p, 0, 20, 40, 40, 1, p, q - 1, None, 0),
        (INVALID, b"null", L.cntkq_mx4_quantize_async, h, p, 0, 20, 40, 40, 1, None, q, None, 0),
        (INVALID, b"null", L.cntkq_mx4_quantize_async, h, None, 0, 20, 40, 40, 1, p, q, None, 0),
        (INVALID, b"16 bytes", L.cntkq_mx4_quantize_async, h, p, 0, 20, 40, 40, 1, p + 8, q, None, 0),
        (INVALID, b"aligned", L.cntkq_mx4_quantize_async, h, odd, 2, 20, 40, 40, 1, p, q, None, 0),
        (LOGIC, b"size", L.cntkq_mx4_quantize_async, h, p, 0, 20, 40, 40, 1, p, q, p, s + 1),
        (INVALID, b"contiguous", L.cntkq_mx4_quantize_async, h, p, 0, 20, 40, 1, 20, p, q, p, s),
        (INVALID, b"2^31", L.cntkq_mx4_quantize_async, h, p, 0, 1 << 31, 40, 40, 1, p, q, None, 0),
        (INVALID, b"stride", L.cntkq_mx4_dequantize_async, h, p, q, 20, 40, p, 0, 39),
        (INVALID, b"stride", L.cntkq_mx4_matmul_async, h, p, q, 20, p, q, 20, 40, None, 0, p, 0, 19),
        (INVALID, b"2^25", L.cntkq_mx4_matmul_async, h, p, q, 20, p, q, 20, (1 << 25) + 1, None, 0, p, 0, 20),
        (LOGIC, b"size", L.cntkq_mx4_matmul_async, h, p, q, 20, p, q, 20, 257, None, 0, p, 0, 20),
        (LOGIC, b"element type", L.cntkq_mx4_matmul_async, h, p, q, 20, p, q, 20, 40, p, 7, p, 0, 20),
        (LOGIC, b"workspace", L.cntkq_mx4_linear_async, h, p, 0, 40, 20, p, q, 20, 40, None, 0, p, 0, 20, p, s, p, q - 1),
        (INVALID, b"workspace", L.cntkq_mx4_linear_async, h, p, 0, 40, 20, p, q, 20, 40, None, 0, p, 0, 20, p, s, None, q),
        (LOGIC, b"size", L.cntkq_save8_async, h, p, 0, 20, 40, 40, p, s - 33),
        (INVALID, b"stride", L.cntkq_load8_async, h, p, s, 20, 40, p, 0, 8),
        (LOGIC, b"activation", L.cntkq_activation_forward_async, h, 0, p, 40, None, 0, 0, 20, 40, p, 40, p, None, s),
        (INVALID, b"gate", L.cntkq_activation_forward_async, h, 1, p, 40, p, 40, 0, 20, 40, p, 40, p, None, s),
        (INVALID, b"gate", L.cntkq_activation_backward_async, h, 1, p, 40, 0, 20, 40, p, p, s, p, 40, None, 0),
        (LOGIC, b"workspace", L.cntkq_weight_gradient_async, h, p, 0, 30, 2000, 30, p, 100 * s, 40, p, 40, None, 0, p, 16),
        (INVALID, b"stride", L.cntkq_weight_gradient_async, h, p, 0, 30, 20, 30, p, s, 40, p, 39, None, 0, p, 1 << 30),
    ]
    for code, text, call, *args in refused:
        assert call(*args) == code, (call.__name__, args)
        assert text in L.cntkq_last_error(), (call.__name__, L.cntkq_last_error())
    # nothing to do: no device either
    assert L.cntkq_mx4_quantize_async(h, None, 0, 0, 40, 40, 1, None, 0, None, 0) == 0
    assert L.cntkq_save8_async(h, None, 0, 20, 0, 0, None, 0) == 0


def test_tensors_of_the_host_are_refused():
    for call in (lowbit.mx4_quantize, lowbit.save8, lambda t: lowbit.activation_forward("relu", t)):
        with pytest.raises(QuantizerLogicError):
            call(torch.zeros(4, 32))


def test_matrices_beyond_a_launch_are_refused():
    """A launch's threads are counted in 32 bits: what would need more is refused before the device is asked."""
    L = lowbit._bind()
    h = ctypes.create_string_buffer(4096)
    p, rows, cols = 4096, (1 << 31) - 64, 4096
    q, s, work = L.cntkq_mx4_bytes(rows, cols), L.cntkq_save8_bytes(rows, cols), 1 << 62
    few = 1 << 28
    refused = [
        (L.cntkq_mx4_quantize_async, h, p, 2, rows, cols, cols, 1, p, q, None, 0),
        (L.cntkq_mx4_dequantize_async, h, p, q, rows, cols, p, 2, cols),
        (L.cntkq_mx4_matmul_async, h, p, q, rows, p, q, rows, cols, None, 0, p, 2, rows),
        (L.cntkq_mx4_linear_async, h, p, 2, 40, 16, p, L.cntkq_mx4_bytes(few, 40), few, 40, None, 0, p, 2, few, None, 0, None, 0),
        (L.cntkq_save8_async, h, p, 2, rows, cols, cols, p, s),
        (L.cntkq_load8_async, h, p, s, rows, cols, p, 2, cols),
        (L.cntkq_activation_forward_async, h, 1, p, cols, None, 0, 2, rows, cols, p, cols, p, None, s),
        (L.cntkq_activation_backward_async, h, 1, p, cols, 2, rows, cols, p, None, s, p, cols, None, 0),
        (L.cntkq_weight_gradient_async, h, p, 2, rows, rows, rows, p, s, cols, p, cols, None, 0, p, work),
    ]
    for entry, *args in refused:
        assert entry(*args) == INVALID, entry.__name__
        assert b"too large for one launch" in L.cntkq_last_error()
