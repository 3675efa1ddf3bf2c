"""Refusals of the 8-bit products and log-probability calls that need no GPU:
null contexts and handles, tensors on the CPU."""
import ctypes as C
import os
import subprocess
import sys

import numpy as np
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


class _Fold(har_cuda.CudaMoeServingModel):
    """The scoring path with its device steps replaced by torch on the CPU: a
    layer step halves its row, the head's logits are the row itself."""

    def __init__(self, V):
        self.H = self.vocab = V
        self._torch, self._dev = torch, torch.device("cpu")
        self.embed = torch.eye(V)
        self.batches, self.ctx = [], type("C", (), {"synchronize": lambda s: None})()

    def _layers_device(self, x):
        self.batches.append(x.shape[0])
        return x * 0.5, []

    def _score_device(self, x, tokens, top):
        logp = torch.log_softmax(x.double(), 1)
        lp = torch.where(tokens < 0, 0.0, logp.gather(1, tokens.clamp(min=0).long().unsqueeze(1))[:, 0])
        best = logp.sort(dim=1, descending=True, stable=True)
        return lp, -(logp.exp() * logp).sum(1), best.indices[:, :top].int(), best.values[:, :top]


def test_score_folds_sequences_side_by_side():
    V = 7
    m = _Fold(V)
    rng = np.random.default_rng(1)
    h = rng.normal(size=(4, V)).astype(np.float32)
    seqs = [[3, 1, 1, 6], [2], [], [0, 5, 4]]
    outs = m.score(list(zip(h, seqs)), top=3)
    assert m.batches == [3, 2, 2, 1]           # sequences that still have a token
    for i, toks in enumerate(seqs):
        o, x = outs[i], h[i].astype(np.float64)
        assert o.logprobs.shape == (max(0, len(toks) - 1),) and o.entropy.shape == (len(toks),)
        assert o.top_ids.shape == (len(toks), 3) and o.top_logprobs.shape == (len(toks), 3)
        for j, t in enumerate(toks):
            x = (x + np.eye(V)[t]) * 0.5
            logp = x - np.log(np.exp(x).sum())
            assert np.allclose(o.entropy[j], -(np.exp(logp) * logp).sum(), atol=1e-6)
            assert o.top_ids[j].tolist() == np.argsort(-logp, kind="stable")[:3].tolist()
            if j + 1 < len(toks):
                assert np.allclose(o.logprobs[j], logp[toks[j + 1]], atol=1e-6)
    assert m.score([]) == []
    assert [o.entropy.size for o in m.score([(h[0], [])])] == [0]


def test_score_refuses():
    m = _Fold(5)
    for bad in ([5], [-1]):
        with pytest.raises(har_cuda.HarCudaError):
            m.score([(np.zeros(5, np.float32), bad)])
    with pytest.raises(har_cuda.HarCudaError):
        m.score([(np.zeros(5, np.float32), [1])], top=33)


def test_context_without_torch():
    """A program that works on numpy alone makes its context without torch."""
    code = """
import sys
sys.modules["torch"] = None                      # `import torch` raises ImportError
import har_cuda
class Library:
    def har_cuda_ctx_create(self, device, out): return 0
    def har_cuda_ctx_destroy(self, handle): return 0
har_cuda.load_library = Library
c = har_cuda.Context(0, use_torch_stream=False)
c.close()
"""
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "remora-lab_b200")
    r = subprocess.run([sys.executable, "-c", code], env={**os.environ, "PYTHONPATH": root}, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr


class _Routed(_Fold):
    """Two layers of routes: a row's experts follow from how often it was folded."""

    def __init__(self, V):
        super().__init__(V)
        self.telemetry = {"positions": 0, "expert_reads": 0, "shared_reads": 0}
        self.step = 0

    def _layers_device(self, x):
        y, _ = super()._layers_device(x)
        self.step += 1
        first = torch.arange(x.shape[0], dtype=torch.int32).unsqueeze(1) % 2  # experts 0, 1 or 1, 2
        ids = torch.cat([first, first + 1], 1)
        return y, [(ids, None), (ids * 0 + self.step, None)]                  # the second layer: one expert a step


def test_score_counts_what_it_folds():
    """Positions and weight reads of scored sequences, as batch_step counts its
    own: a step of the batch reads each expert that it uses once."""
    m = _Routed(7)
    h = np.zeros(7, np.float32)
    m.score([(h, [3, 1, 6]), (h, [2]), (h, []), (h, [0, 5])], top=1)
    assert m.batches == [3, 2, 1]
    # first layer: rows 0 1 2 use experts {0 1 2}, rows 0 1 the same three, row 0 two
    assert m.telemetry == {"positions": 6, "expert_reads": (3 + 1) + (3 + 1) + (2 + 1), "shared_reads": 3 * 2}
    m.score([], top=1)
    m.score([(h, [])])
    assert m.telemetry["positions"] == 6
