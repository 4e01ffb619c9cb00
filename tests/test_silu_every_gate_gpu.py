"""SiLU(gate) * up of silu_mul_quant_mxfp4 over every finite bf16 gate, one at a time, by either of its two ways (approximation, table).

Four-bit codes show little of a bf16 value, so every gate meets two ups, chosen such that the correct product lies next to a border
between two codes and that of a SiLU one bf16 step larger (smaller) lies beyond it: a SiLU off by a step shows."""
import numpy as np
import pytest
import torch

from tests import mx_reference as ref

pytestmark = pytest.mark.gpu


def gates():
    bits = torch.arange(65536, dtype=torch.int32)
    return bits[(bits & 0x7FFF) < 0x7F80].to(torch.int16).view(torch.bfloat16)


def silu_fp32(g):
    """bf16(g / (1 + exp(-g))) with an exactly rounded exponential and fp32's add and divide."""
    v = g.double().numpy()
    with np.errstate(over="ignore"):
        e = np.exp(-v).astype(np.float32)
        return torch.from_numpy(g.float().numpy() / (np.float32(1.0) + e)).to(torch.bfloat16)


def codes(z):
    """Magnitude code of z >= 0, ties to even codes."""
    return (z > 0.25).int() + (z >= 0.75) + (z > 1.25) + (z >= 1.75) + (z > 2.5) + (z >= 3.5) + (z > 5)


def neighbour(s, step):
    """The bf16 value `step` (1, -1) away in magnitude."""
    return (s.view(torch.int16) + step).view(torch.bfloat16)


def telling_ups(s, power, step):
    """For every s != 0 an up whose product with s has another code, in units of 2^power, than its product with s's neighbour."""
    border = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64)
    scale = torch.exp2(power.double()).unsqueeze(1)
    near = (border * scale / s.double().abs().unsqueeze(1)).to(torch.bfloat16)
    ups = (near.view(torch.int16).unsqueeze(2) + torch.arange(-3, 4, dtype=torch.int16)).view(torch.bfloat16).flatten(1)

    def code(v):
        return codes(ref.bf16_round(v.double().abs().unsqueeze(1) * ups.double()) / scale)

    tells = code(s) != code(neighbour(s, step))
    assert tells.any(dim=1).all()
    return ups.gather(1, tells.int().argmax(dim=1, keepdim=True)).squeeze(1)


@pytest.mark.parametrize("by_table", [False, True])
def test_every_finite_gate(cuda_dev, by_table):
    from kb_nano_b200 import ops
    g = gates()
    s = silu_fp32(g)
    exact = ref.bf16_round(g.double() / (1 + torch.exp(-g.double())))
    assert torch.equal(s.double()[g >= -60], exact[g >= -60])                # what is compared with is the exactly rounded SiLU there
    _, ex = torch.frexp(s.double())
    power = (ex - 1).clamp(-110, 120)
    live = s != 0
    m = g.numel()
    x = torch.zeros(2, m, 64, dtype=torch.bfloat16)
    want = torch.zeros(2, m, 32, dtype=torch.float64)
    at = 1 + torch.arange(m) % 30                                             # the gate's place in its block of 32
    rows = torch.arange(m)
    for k, step in enumerate((1, -1)):
        up = torch.ones(m, dtype=torch.bfloat16)
        up[live] = telling_ups(s[live], power[live], step)
        up = torch.where(torch.arange(m) % 2 == 0, up, -up)
        x[k, :, 0], x[k, :, 32] = 64.0, (0.09375 * torch.exp2(power.double())).to(torch.bfloat16)      # SiLU(64) = 64: the product 6 * 2^power sets the scale
        x[k, rows, at], x[k, rows, 32 + at] = g, up
        want[k, :, 0] = 6.0 * torch.exp2(power.double())
        want[k, rows, at] = ref.bf16_round(s.double() * up.double())
        if by_table:                                                          # a gate below -60 sends its eight values to the table; its own product is -0
            other = at // 8 * 8 + torch.where(at % 8 == 7, 6, 7)
            x[k, rows, other] = -70.0
            want[k, rows, other] = -0.0
    x, want = x.view(2 * m, 64).to(cuda_dev), want.view(2 * m, 32).to(cuda_dev)
    q, sc = torch.empty(2 * m, 16, dtype=torch.uint8, device=cuda_dev), torch.empty(2 * m, 1, dtype=torch.uint8, device=cuda_dev)
    ops.silu_mul_quant_mxfp4(x, q, sc)
    for r in range(0, 2 * m, 32768):
        cw, sw = ref.quant(want[r:r + 32768])
        assert torch.equal(sc[r:r + 32768], sw) and torch.equal(q[r:r + 32768], cw)
