"""CPU tests of the microscaled 4-bit operators: what they refuse before any launch."""
import pytest
import torch


def _codes(M, K):
    c = -(-K // 256)
    return torch.zeros((8 * c, M, 16), dtype=torch.uint8), torch.zeros((2 * c, M, 4), dtype=torch.uint8)


def test_operand_class_checks():
    from samnerf_amd import ops
    q = ops.Mxfp4(*_codes(5, 300), 300)
    assert (q.M, q.K, q.shape) == (5, 300, (5, 300))
    codes, scales = _codes(6, 300)
    assert ops.Mxfp4(codes, scales, 300, (2, 3, 300)).shape == (2, 3, 300)
    for bad in (dict(K=0), dict(K=600), dict(K=256)):
        with pytest.raises((TypeError, ValueError)):
            ops.Mxfp4(codes, scales, **bad)
    with pytest.raises(TypeError):
        ops.Mxfp4(codes.float(), scales, 300)
    with pytest.raises(ValueError):
        ops.Mxfp4(codes, scales[:, :5], 300)
    with pytest.raises(ValueError):
        ops.Mxfp4(codes.transpose(0, 1).contiguous().transpose(0, 1), scales, 300)
    with pytest.raises(ValueError):
        ops.Mxfp4(codes, scales, 300, (7, 300))


def test_refusals_without_a_device():
    from samnerf_amd import ops
    w = ops.Mxfp4(*_codes(8, 64), 64)
    with pytest.raises(TypeError):
        ops.quantize_mxfp4(torch.zeros((2, 32), dtype=torch.float64))
    with pytest.raises(TypeError):
        ops.quantize_mxfp4([[1.0]])
    with pytest.raises(ValueError):
        ops.quantize_mxfp4(torch.zeros((2, 0)))
    with pytest.raises(ValueError):
        ops.quantize_mxfp4(torch.zeros(()))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.quantize_mxfp4(torch.zeros((2, 32)))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.dequantize_mxfp4(w)
    with pytest.raises(TypeError):
        ops.dequantize_mxfp4(w, torch.int8)
    with pytest.raises(TypeError):
        ops.dequantize_mxfp4(torch.zeros((2, 32)))
    with pytest.raises(TypeError):
        ops.linear_mxfp4(torch.zeros((2, 64)), torch.zeros((8, 64)))
    with pytest.raises(TypeError):
        ops.linear_mxfp4(torch.zeros((2, 64), dtype=torch.int32), w)
    with pytest.raises(ValueError):
        ops.linear_mxfp4(torch.zeros((2, 63)), w)
    with pytest.raises(ValueError):
        ops.linear_mxfp4(torch.zeros((2, 64)), w, act=7)
    with pytest.raises(TypeError):
        ops.linear_mxfp4(torch.zeros((2, 64)), w, out_dtype=torch.float64)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.linear_mxfp4(torch.zeros((2, 64)), w)


def test_the_library_refuses_before_any_launch():
    """Argument checks of the C entry points: host code, no device touched."""
    from samnerf_amd import _lib
    lib = _lib.load()
    p = 4096  # an aligned address that is never followed

    def refused(rc, word):
        assert rc == -1 and word in lib.snf_last_error(), (rc, lib.snf_last_error())

    refused(lib.snf_mxfp4_quantize(p, 7, 3, 64, 64, p, p, None), b"dtype")
    refused(lib.snf_mxfp4_quantize(p, 0, 3, 0, 64, p, p, None), b"sizes")
    refused(lib.snf_mxfp4_quantize(p, 0, -1, 64, 64, p, p, None), b"sizes")
    refused(lib.snf_mxfp4_quantize(p, 0, 3, 64, 63, p, p, None), b"overlap")
    refused(lib.snf_mxfp4_quantize(None, 0, 3, 64, 64, p, p, None), b"null")
    refused(lib.snf_mxfp4_quantize(p, 0, 3, 64, 64, p + 8, p, None), b"aligned")
    refused(lib.snf_mxfp4_quantize(p, 0, 2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31, p, p, None), b"too large")
    refused(lib.snf_mxfp4_quantize_planes(p, p, 3, 12, p, p, None), b"sizes")
    refused(lib.snf_mxfp4_quantize_planes(p, p + 2, 3, 16, p, p, None), b"aligned")
    refused(lib.snf_mxfp4_dequantize(p, p, 3, 64, p, 3, None), b"dtype")
    refused(lib.snf_mxfp4_dequantize(p, p, 3, 64, None, 0, None), b"null")
    refused(lib.snf_mxfp4_linear(p, p, p, p, None, 3, 64, 0, 0, p, 0, None), b"sizes")
    refused(lib.snf_mxfp4_linear(p, p, p, p, None, 3, 64, 8, 4, p, 0, None), b"activation")
    refused(lib.snf_mxfp4_linear(p, p, p, p, None, 3, 64, 8, 0, p, 5, None), b"dtype")
    refused(lib.snf_mxfp4_linear(p, p, p, p, None, 1 << 28, 64, 8, 0, p, 0, None), b"2^28")
    refused(lib.snf_mxfp4_linear(p + 4, p, p, p, None, 3, 64, 8, 0, p, 0, None), b"aligned")
    refused(lib.snf_mxfp4_linear_quantized(p, p, p, p, None, 3, 64, 40, 0, p, p, None), b"sizes")
    refused(lib.snf_mxfp4_linear_rows(p, 0, 64, p, p, None, 17, 64, 8, 0, p, 0, None), b"sizes")
    refused(lib.snf_mxfp4_linear_rows(p, 0, 63, p, p, None, 2, 64, 8, 0, p, 0, None), b"overlap")
    # calls without work need no memory
    assert lib.snf_mxfp4_quantize(None, 0, 0, 64, 64, None, None, None) == 0
    assert lib.snf_mxfp4_linear(None, None, None, None, None, 0, 64, 8, 0, None, 0, None) == 0


def test_linear_refuses_to_drop_a_gradient():
    """No gradient flows through the product: an x that asks for one is refused, unless nothing is recorded."""
    from samnerf_amd import ops
    w = ops.Mxfp4(*_codes(8, 64), 64)
    x = torch.zeros((2, 64), requires_grad=True)
    for kw in ({}, dict(quantized=True)):
        with pytest.raises(RuntimeError, match="requires a gradient"):
            ops.linear_mxfp4(x, w, **kw)
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            ops.linear_mxfp4(x.detach(), w, **kw)
        with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU fallback"):
            ops.linear_mxfp4(x, w, **kw)
