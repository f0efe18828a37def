"""The decode step with its linears in 4 bits and its KV cache in 8 (neokernel_b200.qwen3):
linears, append and attention run together, eagerly and from a captured graph."""

import pytest
import torch

import neokernel_b200 as nk
from neokernel_b200 import qwen3, tp, w4

pytestmark = pytest.mark.gpu
DEV = "cuda"
DIMS = qwen3.Qwen3Dims(512, 1280, 8, 2, 128, 3, 1024)


def models(group=128, zeros=False):
    w = qwen3.Qwen3Weights(DIMS, seed=3)
    return w, qwen3.quantize_linears(w, group, zeros)


@pytest.mark.parametrize("B", (1, 5))
@pytest.mark.parametrize("zeros", (False, True))
def test_graph_and_eager_steps_agree_bit_for_bit(B, zeros):
    _, q = models(64, zeros)
    g = qwen3.GraphDecoder(q, B, 80, w4.linear, fused=True, cache="e4m3")
    st = qwen3.DecodeState(q, B, 80, cache="e4m3")
    tokens = torch.randint(0, DIMS.vocab, (B,), device=DEV)
    g.st.tokens.copy_(tokens)
    st.tokens.copy_(tokens)
    for _ in range(70):  # across the end of a block of 64
        g.step()
        qwen3.decode_step(st, q, w4.linear, fused=True)
        st.tokens.copy_(st.next_tokens)
        st.position.add_(1)
        assert torch.equal(g.st.tokens, st.tokens)
        assert torch.equal(g.st.logits, st.logits)
    for a, b in zip(g.st.q8, st.q8):
        assert torch.equal(a.k.view(torch.uint8), b.k.view(torch.uint8))
        assert torch.equal(a.v_scale, b.v_scale)
    assert nk.device_error() == 0


def test_one_layer_step_is_its_parts():
    """After one layer, each buffer is what the formula gives from the buffer before it."""
    d = qwen3.Qwen3Dims(512, 1280, 8, 2, 128, 1, 1024)
    q = qwen3.quantize_linears(qwen3.Qwen3Weights(d, seed=5), 32, True)
    B, cap = 3, 40
    st = qwen3.DecodeState(q, B, cap, cache="e4m3")
    lw, cache = q.layers[0], st.q8[0]
    for p in range(cap):
        st.tokens.copy_(torch.randint(0, d.vocab, (B,), device=DEV))
        qwen3.decode_step(st, q, w4.linear, fused=True)
        st.position.add_(1)
    x = q.embed[st.tokens]
    norm = qwen3.rms_norm(x, lw.input_norm, d.eps)
    K = d.hidden
    ref = norm.double() @ lw.qkv.dequantize().double().t()
    # the linear's tolerance (tests/test_w4_gpu.py), and one bf16 step (2^-7) of an activation whose
    # norm falls on the other side of a rounding border
    mag = norm.double().abs() @ lw.qkv.dequantize().double().abs().t()
    assert ((st.qkv.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -7 * mag / 8
            + (K + K / 32 + 64) * 2.0 ** -23 * mag).all()
    k, v = cache.dequantize()
    want_v = st.qkv.view(B, 12, 128)[:, 10:].double()
    got_v = v[:, :, cap - 1].double()
    step = cache.v_scale[:, :, -1, None].double()
    assert ((got_v - want_v).abs() <= 2.0 ** -4 * want_v.abs() + 2.0 ** -10 * step).all()
    qf = st.q.view(B, 2, 4, 128).double()
    w = torch.softmax(qf @ k.double().transpose(-1, -2) / 128 ** 0.5, dim=-1)
    out = (w @ v.double()).reshape(B, -1)
    slack = (w @ v.double().abs()).reshape(B, -1)
    # probabilities in f16 (2^-11), scores and exponentials as in tests/test_q8_cache_gpu.py
    assert ((st.attn.double() - out).abs() <= 2.0 ** -8 * out.abs() + 2.0 ** -10 * slack).all()


def test_quantised_step_keeps_decisive_tokens():
    """The decisive initialisation makes every greedy choice by tens of logits, far more than 4-bit
    weights and 8-bit keys and values move them: the tokens are those of the bf16 step."""
    w, q = models(64, True)
    prompt = torch.randint(0, DIMS.vocab, (2, 8), device=DEV)
    ref = qwen3.GraphDecoder(w, 2, 64, nk.mm, fused=True).greedy(prompt, 40)
    got = qwen3.GraphDecoder(q, 2, 64, w4.linear, fused=True, fused_head=True,
                             cache="e4m3").greedy(prompt, 40)
    assert torch.equal(ref, got)


@pytest.mark.parametrize("cache", ("bf16", "e4m3"))
def test_each_half_alone(cache):
    w, q = models()
    linear, model = (nk.mm, w) if cache == "e4m3" else (w4.linear, q)
    prompt = torch.randint(0, DIMS.vocab, (1, 4), device=DEV)
    ref = qwen3.GraphDecoder(w, 1, 64, nk.mm, fused=True).greedy(prompt, 20)
    got = qwen3.GraphDecoder(model, 1, 64, linear, fused=True, cache=cache).greedy(prompt, 20)
    assert torch.equal(ref, got)


def test_refusals():
    w, _ = models()
    with pytest.raises(ValueError):
        qwen3.DecodeState(w, 1, 16, cache="int8")
    st = qwen3.DecodeState(w, 1, 16, cache="e4m3")
    with pytest.raises(ValueError):
        qwen3.decode_step(st, w, nk.mm, fused=False)


def test_tensor_parallel_hooks_refuse_4_bit_weights():
    w = tp.TPWeights(DIMS, 3, 0, 1)
    _, q = models()
    st = qwen3.DecodeState(w, 2, 16)
    row_linear, _ = tp.make_hooks(w)(st)
    st.attn.zero_()
    row_linear(st.attn, w.layers[0].o, st.branch)
    with pytest.raises(ValueError, match="torch.Tensor"):
        row_linear(st.attn, q.layers[0].o, st.branch)


def test_tensor_parallel_hooks_over_an_8_bit_cache():
    """One rank: its shard is the whole model, so the tokens are those of the single-GPU step."""
    w, _ = models()
    t = tp.TPWeights(DIMS, 3, 0, 1)
    prompt = torch.randint(0, DIMS.vocab, (2, 6), device=DEV)
    ref = qwen3.GraphDecoder(w, 2, 64, nk.mm, fused=True, cache="e4m3").greedy(prompt, 30)
    got = qwen3.GraphDecoder(t, 2, 64, nk.mm, make_hooks=tp.make_hooks(t), fused=True,
                             cache="e4m3").greedy(prompt, 30)
    assert torch.equal(ref, got)
