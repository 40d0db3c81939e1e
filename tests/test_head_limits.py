"""CPU: sizes that the head's operators cannot launch are refused by the C ABI before anything runs, forward and backward alike."""
import pytest

P = 1 << 20                       # an address that a refused call never touches


@pytest.fixture(scope="module")
def lib():
    from multiagentperception_amd import _build, _native
    _build.build()
    return _native.lib()


def test_norm_of_long_rows(lib):
    big = 1 << 60
    for rows, cols in ((1 << 22, 16385), ((1 << 31) - 1, 1 << 30)):
        assert lib.w2c_layer_norm_forward(P, 0, 1, rows, cols, P, P, 0, 1e-5, P, 0, P, P, 0) == -1
        assert lib.w2c_layer_norm_workspace_bytes(rows, cols, 1) == -1
        assert lib.w2c_layer_norm_backward(P, P, 0, 1, rows, cols, P, 0, P, P, P, 0, 0, P, big, 0) == -1
    assert lib.w2c_layer_norm_workspace_bytes((1 << 22) - 1, 16385, 1) > 0 and lib.w2c_layer_norm_workspace_bytes((1 << 31) - 1, 16384, 1) > 0


# one launch takes 2^32 - 1 work-items in blocks of 256: 16 columns to one of them, or a tile of at most 256 x 256
@pytest.mark.parametrize("M,N", [(1, 16 * 16777215 + 1), (24, 0x7FFFFFFF), (0x7FFFFFFF, 1), (25, 0x7FFFFFFF - 254), (513, 0x7FFFFFFF - 255), (1 << 21, 1 << 19)])
def test_product(lib, M, N):
    assert lib.w2c_matmul_fp8(P, P, 1, P, P, 1, M, N, 128, 0, P, 1, P, 1 << 60, 0) == -1
    assert lib.w2c_matmul_fp8_fast(P, P, 1, P, P, 1, M, N, 128, 0, P, 1, P, 1 << 60, 0) == -1


def test_quantiser(lib):
    cols = 128 * 16777215 + 1
    assert lib.w2c_quantize_fp8(P, 0, 1, cols, cols, 1, P, P, 0, 0, 0, 0, 0, 0) == -1


def test_optimizer_tensor(lib):
    import ctypes
    for n, ok in (((1 << 36) - 4096, True), ((1 << 36) - 4095, False)):
        row = (ctypes.c_longlong * 9)(P, P, P, P, P, P, P, n, 0)
        assert (lib.w2c_grad_squares_count(row, 1) > 0) == ok
        if not ok:
            assert lib.w2c_adamw_step(row, 1, 8, 1e-3, 0, 0.9, 0.999, 1e-8, 0.0, 0, 0, 0.0, 0, 0, P, 1 << 20, 0) == -1
