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
