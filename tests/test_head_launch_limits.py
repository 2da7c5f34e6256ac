"""Calls of the head and e4m3 operators within the documented sizes whose launch would hold 2^32 work-items or more: refused as
unsupported on the host, before anything is launched (no GPU is needed)."""
import ctypes

import pytest

UNSUPPORTED = -7


@pytest.fixture(scope="module")
def lib():
    from prefilling_dllm_amd import _lib
    return _lib.lib


@pytest.fixture(scope="module")
def p():
    buf = (ctypes.c_char * 8192)()
    p.keep = buf
    return (ctypes.addressof(buf) + 255) & ~255


ROWS = 1 << 24


@pytest.mark.parametrize("v,d", [(33001, 64), (65537 + 256, 8)])
def test_head_tiles(lib, p, v, d):
    ws = lib.pdllm_head_workspace_bytes(ROWS, v)
    assert ws > 0
    assert lib.pdllm_head_selfinfo_logprob(p, d, p, d, p, ROWS, v, d, p, ws, p, None, None) == UNSUPPORTED
    assert lib.pdllm_head_conf_argmax(p, d, None, d, p, d, 1 << 19, 32, v, d, 1, p, ws, p, p, None) == UNSUPPORTED
    assert lib.pdllm_head_denoise_unmask(p, d, None, d, p, d, 1 << 19, 32, v, d, 1, p, 5, 0.9, p, ws, p, p, p, None,
                                         None) == UNSUPPORTED


def test_gradient_joins(lib, p):
    d = 1032
    ws = lib.pdllm_head_selfinfo_grad_workspace_bytes(ROWS, 300, d)
    assert ws > 0
    assert lib.pdllm_head_selfinfo_grad(p, d, p, d, p, p, p, p, ROWS, 300, d, p, ws, p, d, p, d, None) == UNSUPPORTED
    # no rows: grad_weight is cleared in tiles of 256 x 256
    assert lib.pdllm_head_selfinfo_grad(None, d, p, d, None, None, None, None, 0, 1 << 30, d, None, 0, None, d, p, d,
                                        None) == UNSUPPORTED


def test_e4m3(lib, p):
    n = 1 << 30
    for m in (1, 20):
        assert lib.pdllm_fp8_linear(p, 64, p, 1, m, p, 64, p, 1, 1, m, n, 64, p, n, None) == UNSUPPORTED
    assert lib.pdllm_fp8_linear_bf16(p, 64, p, 64, p, 1, 1, 16, n, 64, None, 0, p, n, None) == UNSUPPORTED
    assert lib.pdllm_fp8_linear(p, 64, p, 1, ROWS, p, 64, p, 1, 1, ROWS, 1 << 16, 64, p, 1 << 16, None) == UNSUPPORTED
    for q in (lib.pdllm_fp8_quantize_rows, lib.pdllm_fp8_quantize_blocks):
        k = 128 if q is lib.pdllm_fp8_quantize_rows else 1 << 19
        assert q(p, k, n, k, p, k, p, 1, 1, None) == UNSUPPORTED
