"""Types of LinearAttention's parameters: 16-bit layers keep the gate's bias in float32."""
import copy

import pytest
import torch

import dms_amd


def layer():
    torch.manual_seed(0)
    m = dms_amd.LinearAttention(8, 16, 2, sections=(2,))
    with torch.no_grad():
        m.gate_bias.copy_(torch.tensor([1.0 + 2.0 ** -20, -3.0 - 2.0 ** -19]))
    return m


@pytest.mark.parametrize("convert", [lambda m: m.bfloat16(), lambda m: m.half(), lambda m: m.to(torch.bfloat16),
                                     lambda m: m.to("cpu", torch.float16), lambda m: torch.nn.Sequential(m).bfloat16()[0],
                                     lambda m: copy.deepcopy(m).to(torch.bfloat16), lambda m: m.half().bfloat16()])
def test_conversions_leave_the_bias_of_the_gate(convert):
    m = layer()
    want = m.gate_bias.detach().clone()
    m = convert(m)
    assert m.gate_bias.dtype == torch.float32 and torch.equal(m.gate_bias, want) and m.gate_bias.requires_grad
    assert {p.dtype for n, p in m.named_parameters() if n != "gate_bias"} in ({torch.bfloat16}, {torch.float16})
    assert m.state_dict()["gate_bias"].dtype == torch.float32
    m.float()
    assert {p.dtype for p in m.parameters()} == {torch.float32} and torch.equal(m.gate_bias, want)


def test_other_conversions_and_gradients():
    m = layer()
    assert layer().double().gate_bias.dtype == torch.float64
    for p in m.parameters():
        p.grad = torch.full_like(p, 1.0 + 2.0 ** -20)
    bias = m.gate_bias
    m.bfloat16()
    assert m.gate_bias is bias and m.gate_bias.grad.dtype == torch.float32 and (m.gate_bias.grad == 1.0 + 2.0 ** -20).all()
    assert m.weight.grad.dtype == torch.bfloat16
    with torch.no_grad():
        m.gate_bias.add_(2.0 ** -20)
    assert m.gate_bias[0] == 1.0 + 2.0 ** -19
    other = layer().bfloat16()
    other.load_state_dict(m.state_dict())
    assert torch.equal(other.gate_bias, m.gate_bias)
    meta = dms_amd.LinearAttention(8, 16, 2).to("meta").to(torch.bfloat16)
    assert meta.gate_bias.dtype == torch.float32 and meta.gate_bias.is_meta
    old = torch.get_default_dtype()
    try:
        torch.set_default_dtype(torch.bfloat16)
        assert dms_amd.LinearAttention(8, 16, 2).gate_bias.dtype == torch.float32
    finally:
        torch.set_default_dtype(old)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_small_change_of_the_bias_reaches_the_state(dtype):
    """A step of 2^-12 in the bias of the gate: a 16-bit bias near 3 has no such step.  Over 4000 tokens that keep sigmoid(3)^(1/16) of the
    state, the change of the log decay, 2^-12 / 16 sigmoid(-3) a token, adds up to 2^-12 * 4000 * 0.0474 / 16 = 2.9e-3 of the state."""
    layer = dms_amd.LinearAttention(8, 16, 1).to(dtype).cuda()
    with torch.no_grad():
        for p in layer.parameters():
            p.zero_()
        states = []
        for step in (0.0, 2.0 ** -12):
            layer.gate_bias.fill_(3.0 + step)
            _, s = layer(torch.zeros(4000, 1, 8, dtype=dtype, device="cuda"), torch.ones(1, 1, 16, 16, device="cuda"))
            states.append(s.double())
    grown = float((states[1] / states[0] - 1).mean())
    want = float(torch.expm1(4000 / 16 * (torch.nn.functional.logsigmoid(torch.tensor(3.0 + 2.0 ** -12, dtype=torch.float64))
                                          - torch.nn.functional.logsigmoid(torch.tensor(3.0, dtype=torch.float64)))))
    # log sigmoid(3) = -0.0486 is right to 2 ulp, 2^-27, on either side: 4000 / 16 * 2^-26
    assert abs(grown - want) <= 4000 / 16 * 2.0 ** -26 + 2.0 ** -16
