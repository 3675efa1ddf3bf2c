"""CudaMoeServingModel.score: a stack of MoE layers folded over sequences, the
LM head and the log-probability operators together, with a Q6_K, a Q4_K and an
8-bit head, against batch_step and the definitions in 64 bits."""
import numpy as np
import pytest
import torch

import har_cuda
import haro
from gpu_util import Layer, gen_tensor
from score_util import check_logprobs, logprobs64, product, quantize64

pytestmark = pytest.mark.gpu

E, H, I, V, K_USED = 8, 512, 256, 777, 3


@pytest.fixture(scope="module")
def setup():
    ctx = har_cuda.Context(0)
    layers = [Layer(ctx, E, H, I, 9000 + 10 * l) for l in range(2)]
    routers = [torch.from_numpy(haro.normal_f32(9100 + l, 0, E * H, 0.0, 0.05).reshape(E, H)).cuda() for l in range(2)]
    embed = haro.normal_f32(9200, 0, V * H, 0.0, 0.5).reshape(V, H)
    g = torch.Generator().manual_seed(9)
    heads = {"i8": ctx.i8_weights((torch.randn(V, H, generator=g) * 0.1).cuda()),
             "q6k": ctx.upload(har_cuda.GGML_Q6_K, haro.random_q6k(9300, V, H), 1, V, H)}
    q4, _ = gen_tensor(ctx, V, H, 9400)
    heads["q4k"] = ctx.wrap_q4k(q4, 1, V, H)
    yield ctx, layers, routers, embed, heads, (torch.randn(V, H, generator=torch.Generator().manual_seed(9)) * 0.1)
    ctx.synchronize()
    ctx.close()


def model_of(setup, head):
    ctx, layers, routers, embed, heads, _ = setup
    return har_cuda.CudaMoeServingModel(ctx, [l.layer for l in layers], embed, heads[head], K_USED, eos=V - 1,
                                        routers=routers)


def test_eight_bit_head_in_batch_step(setup):
    model = model_of(setup, "i8")
    wq, ws = quantize64(setup[5])
    for B in (1, 3, 7):
        inputs = [(haro.normal_f32(9500 + i, 0, H, 0.0, 0.3), (31 * i) % V) for i in range(B)]
        outs = model.batch_step(inputs)
        states = torch.from_numpy(np.stack([o.next for o in outs]))
        ref = product(*quantize64(states), wq, ws, torch.float32)
        assert np.array_equal(np.stack([o.logits for o in outs]), ref.numpy())
    assert model.weight_bytes_per_row() == V * (H + 4) + 2 * (K_USED + 1) * 3 * I * (H // 256) * 144


@pytest.mark.parametrize("head", ["i8", "q6k", "q4k"])
@pytest.mark.parametrize("lengths", [[1], [2, 5, 1, 0, 9], [4] * 40, [8, 3] * 12])
def test_score(setup, head, lengths):
    """Many short sequences rather than a long one: a stack without norms leaves
    the tensor-core path's f16 range after some tens of steps, and says so."""
    model = model_of(setup, head)
    rng = np.random.default_rng(len(lengths))
    inputs = [(haro.normal_f32(9600 + i, 0, H, 0.0, 0.3), rng.integers(0, V, n)) for i, n in enumerate(lengths)]
    outs = model.score(inputs, top=6)
    assert len(outs) == len(inputs)
    # the states by the fold, one sequence at a time (a step alone and in a
    # batch are equal on the default path), the logits by the head's own call on
    # the same rows: what is left is token_logprobs' definition
    states, nxt = [], []
    for h, toks in inputs:
        if len(toks):
            states += model.prefill_batch([(h, toks.tolist())])[0][0]
            nxt += toks[1:].tolist() + [-1]
    x = torch.from_numpy(np.stack(states)).cuda()
    logits = torch.cat([model._logits_device(x[p:p + model.SCORE_ROWS]) for p in range(0, len(x), model.SCORE_ROWS)])
    if head == "i8":
        assert torch.equal(logits.cpu(), product(*quantize64(x), *quantize64(setup[5]), torch.float32))
    got = {"logprobs": torch.from_numpy(np.concatenate([np.append(o.logprobs, 0.0) if o.entropy.size else o.logprobs
                                                        for o in outs])).unsqueeze(1),
           "entropy": torch.from_numpy(np.concatenate([o.entropy for o in outs])),
           "ids": torch.from_numpy(np.concatenate([o.top_ids for o in outs])),
           "top": torch.from_numpy(np.concatenate([o.top_logprobs for o in outs]))}
    check_logprobs(got, logprobs64(logits, np.array(nxt).reshape(-1, 1), 6), (head, lengths))


def test_score_refuses(setup):
    model = model_of(setup, "i8")
    with pytest.raises(har_cuda.HarCudaError):
        model.score([(np.zeros(H, np.float32), [V])])
    with pytest.raises(har_cuda.HarCudaError):
        model.score([(np.zeros(H, np.float32), [1])], top=33)


@pytest.mark.parametrize("head", ["i8", "q4k"])
def test_score_without_alternatives(setup, head):
    """top = 0: the same log probabilities and entropies, empty alternatives;
    and nothing to score at all."""
    model = model_of(setup, head)
    rng = np.random.default_rng(3)
    inputs = [(haro.normal_f32(9700 + i, 0, H, 0.0, 0.3), rng.integers(0, V, n)) for i, n in enumerate([4, 1, 0, 3])]
    with_top, without = model.score(inputs, top=5), model.score(inputs)
    for a, b in zip(with_top, without):
        assert np.array_equal(a.logprobs, b.logprobs) and np.array_equal(a.entropy, b.entropy)
        assert b.top_ids.shape == (len(b.entropy), 0) and b.top_logprobs.shape == (len(b.entropy), 0)
    assert model.score([]) == []
    (empty,) = model.score([(np.zeros(H, np.float32), [])], top=2)
    assert empty.logprobs.size == 0 and empty.top_ids.shape == (0, 2)
