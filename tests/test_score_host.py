"""Refusals of the 8-bit products and log-probability calls that need no GPU:
null contexts and handles, tensors on the CPU."""
import ctypes as C

import pytest
import torch

import har_cuda


def test_null_context_and_handles():
    lib = har_cuda.load_library()
    h = C.c_void_p()
    assert lib.har_cuda_i8_quantize(None, None, 0, 1, 1, 1, None, 1, None) == har_cuda.ERR_ARG
    assert lib.har_cuda_i8_weights_quantize(None, None, 0, 1, 1, 1, C.byref(h)) == har_cuda.ERR_ARG
    assert lib.har_cuda_i8_weights_wrap(None, None, 16, None, 1, 1, C.byref(h)) == har_cuda.ERR_ARG
    assert lib.har_cuda_i8_weights_free(None) == har_cuda.ERR_ARG
    assert lib.har_cuda_i8_matmul(None, None, None, 16, None, 1, None, 0, 1) == har_cuda.ERR_ARG
    assert lib.har_cuda_i8_linear(None, None, None, 0, 1, 1, None, 0, 1, None, 0) == har_cuda.ERR_ARG
    assert lib.har_cuda_i8_linear_workspace(None, 1) == -1
    assert lib.har_cuda_token_logprobs(None, None, 0, 1, 1, 1, None, 0, 0, None, None, None, None) == har_cuda.ERR_ARG
    assert lib.har_cuda_i8_head_workspace(None, 1, 1, 1) == -1
    assert lib.har_cuda_i8_head_logprobs(None, None, None, 0, 1, 1, None, 0, 0, None, None, None, None, None,
                                         0) == har_cuda.ERR_ARG


def _context():
    """A context without a device behind it: its calls get as far as the
    tensors' checks, and a null handle after them."""
    c = object.__new__(har_cuda.Context)
    c.lib, c.handle, c.device = har_cuda.load_library(), None, 0
    c.last_error = lambda: ""
    har_cuda._Types.load()
    return c


def test_tensors_on_the_cpu_are_refused():
    c = _context()
    x, q, s = torch.zeros(2, 16), torch.zeros(2, 16, dtype=torch.int8), torch.zeros(2)
    w = object.__new__(har_cuda.I8Weights)
    w.ctx, w.handle, w.N, w.K = c, None, 2, 16
    for f in (lambda: c.i8_quantize(x, q, s), lambda: c.wrap_i8(q, s), lambda: c.i8_weights(x),
              lambda: c.i8_matmul(w, q, s, x[:, :2]), lambda: c.i8_linear(w, x, x[:, :2]),
              lambda: c.token_logprobs(x), lambda: c.i8_head_logprobs(w, x)):
        with pytest.raises(har_cuda.HarCudaError) as e:
            f()
        assert e.value.status == har_cuda.ERR_ARG


def test_row_matrix_strides():
    q = har_cuda.i8_rows(3, 33, "cpu")
    assert tuple(q.shape) == (3, 33) and q.stride() == (48, 1)
