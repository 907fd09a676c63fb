"""Launcher of the grouped products of 8-bit activations with 8-bit weights (quantize/fp8.py)."""
import torch

from .. import _lib
from ..quantize.fp8 import FP8, blocks, check_weight


def grouped_gemm_fp8(pairs, m_sizes: torch.Tensor, dtype: torch.dtype, transposed: bool = False) -> torch.Tensor:
    """sum over one or two (q, s, w, ws) of q w^T, or with `transposed` of q w, per expert: one fp32 accumulator, rounded once
    to `dtype`.  q (M, K) and s from `quantize_fp8_rows`, w (E, N, K) or, transposed, (E, K, N)."""
    assert 1 <= len(pairs) <= 2
    q0, _, w0, _ = pairs[0]
    M, K = q0.shape
    E, N = w0.shape[0], w0.shape[2 if transposed else 1]
    assert q0.is_cuda and m_sizes.device == q0.device and _lib.is_int_tensor(m_sizes)
    assert m_sizes.ndim == 1 and m_sizes.is_contiguous() and m_sizes.numel() == E
    args = []
    for q, s, w, ws in pairs:
        check_weight(w, ws)
        assert w.shape == ((E, K, N) if transposed else (E, N, K)) and w.device == q0.device
        assert q.shape == (M, K) and q.dtype == FP8 and q.is_contiguous() and q.device == q0.device
        assert s.shape == (blocks(K), M) and s.dtype == torch.float32 and s.device == q0.device
        assert (M <= 1 or s.stride(1) == 1) and (s.shape[0] == 1 or M == 0 or s.stride(0) == -(-M // 4) * 4)
        args += [_lib.ptr(q), _lib.ptr(s), _lib.ptr(w), _lib.ptr(ws)]
    args += [None] * (8 - len(args))
    m_sizes = _lib.as_index_tensor(m_sizes)
    y = torch.empty((M, N), device=q0.device, dtype=dtype)
    here, stream = _lib.launch_on(q0.device)
    with here:
        status = _lib.load().moe_grouped_gemm_fp8(
            int(transposed), *args, _lib.ptr(m_sizes), _lib.int_code(m_sizes.dtype), _lib.ptr(y), M, N, K, E,
            _lib.float_code(dtype), stream)
    _lib.check(status, "moe_grouped_gemm_fp8")
    return y
