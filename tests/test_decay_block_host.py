"""DecayAttentionLIF without a device: what its conversions and refusals leave."""
import pytest
import torch

from catfuse_b200.decay_block import DecayAttentionLIF

FP32 = ("inv_freq", "log_decay", "q_weight", "k_weight")


@pytest.mark.parametrize("convert", [lambda m: m.half(), lambda m: m.bfloat16(), lambda m: m.to(torch.float16),
                                     lambda m: torch.nn.Sequential(m).to(torch.bfloat16)[0],
                                     lambda m: m.half().bfloat16()])
def test_conversions_keep_the_fp32_parts(convert):
    m = DecayAttentionLIF(64, heads=4, kv_heads=2)
    with torch.no_grad():
        m.q_weight.uniform_(0.5, 1.5)
    before = {n: getattr(m, n).detach().clone() for n in FP32}
    convert(m)
    assert m.qkv.weight.dtype == m.proj.weight.dtype != torch.float32
    for n in FP32:
        t = getattr(m, n)
        assert t.dtype == torch.float32 and torch.equal(t, before[n])
    assert {"q_weight", "k_weight"} <= dict(m.named_parameters()).keys()


@pytest.mark.parametrize("tokens", [None, 5])
def test_another_batch_is_refused_and_the_states_stay(tokens):
    m = DecayAttentionLIF(64, heads=4, kv_heads=2)
    state, membrane = torch.randn(2, 2, 16, 16), torch.randn(2, 64)
    m.state.set(state.clone())
    m.membrane.set(membrane.clone())
    x = torch.randn(3, 64) if tokens is None else torch.randn(3, tokens, 64)
    pos = torch.zeros(x.shape[:-1], dtype=torch.int32)
    with pytest.raises(ValueError, match="reset"):
        (m.step if tokens is None else m)(x, pos)
    assert torch.equal(m.state.tensor, state) and torch.equal(m.membrane.tensor, membrane)


@pytest.mark.parametrize("carried", [False, True])
def test_a_prompt_without_tokens_changes_nothing(carried):
    m = DecayAttentionLIF(64, heads=4, kv_heads=2)
    state, membrane = torch.randn(2, 2, 16, 16), torch.randn(2, 64)
    if carried:
        m.state.set(state.clone())
        m.membrane.set(membrane.clone())
    out = m(torch.zeros(2, 0, 64), torch.zeros(2, 0, dtype=torch.int32))
    assert out.shape == (2, 0, 64) and out.dtype == torch.float32
    if carried:
        assert torch.equal(m.state.tensor, state) and torch.equal(m.membrane.tensor, membrane)
    else:
        assert m.state.tensor is None and m.membrane.tensor is None
