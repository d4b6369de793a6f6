"""How far products of floats as sums of three bfloat16 are off, of which the six largest of nine products are made (hetuctr_amd/csrc/matmul.h)."""
import pytest
import torch

from hetuctr_amd import nn
from tests import products_reference as ref

gpu = pytest.mark.gpu


def parts(a):
    """The three bfloat16 of floats, in 64 bits: the nearest, the nearest to what is left, and what is then left"""
    out, left = [], a.double()
    for _ in range(3):
        out.append(left.float().bfloat16().double())        # (what is left is a float)
        left = left - out[-1]
    assert (left == 0).all()
    return out


def worst():
    """Floats of 1 .. 2 whose second and third part no other exceeds both, and these, relative to the float"""
    a = (torch.arange(2 ** 23, dtype=torch.int32) + 0x3f800000).view(torch.float32)
    _, second, third = (p.abs() / a.double() for p in parts(a))
    order = torch.argsort(second, descending=True)
    most = torch.cummax(third[order], 0).values
    new = torch.cat((torch.tensor([True]), most[1:] > most[:-1]))
    return a[order][new], second[order][new], third[order][new]


def test_what_the_three_products_left_out_amount_to():
    # of any two floats: the largest of second times third, either way, and of third times third
    a, second, third = worst()
    out = second[:, None] * third + third[:, None] * second + third[:, None] * third
    assert 0.99 * 2 ** -24 < out.max().item() < 2 ** -24
    # and some pairs come near: 1 + 2^-8 - 2^-17 with itself
    one = torch.tensor([1 + 2.0 ** -8 - 2.0 ** -17])
    p = parts(one)
    made = sum(p[i] * p[j] for i in range(3) for j in range(3 - i))
    exact = one.double() ** 2
    assert 2 ** -25 < ((made - exact).abs() / exact).item() < 2 ** -24


@gpu
@pytest.mark.parametrize("rows, hidden", [(300, 130), (3000, 1000), (5003, 1001)])
def test_products_of_floats_one_by_one(rows, hidden):
    # sums of one product, at sizes that take tiles of 64, 128 and 256: what is left out, the matrix cores' sums (a unit of the sum and one of the small parts,
    # which are 2^-7 of it, two each since they may cut off), and nothing else before it is a float
    a, _, _ = worst()
    gen = torch.Generator().manual_seed(1)
    draw = lambda n: (torch.cat((a, torch.randn(n, generator=gen)))[torch.randint(0, len(a) + n, (n,), generator=gen)] * torch.tensor([1.0, -1.0, 3.0])[torch.randint(0, 3, (n,), generator=gen)]).cuda()
    x, w = draw(rows)[:, None], draw(hidden)[:, None]
    x[:len(a), 0], w[:len(a), 0] = a.cuda(), a.cuda()
    _, gate, up = nn.gated_linear(x, w, -w, activation="relu", saved=True)
    exact = x.double() @ w.double().T
    slack = (1 + 2 * (1 + 2.0 ** -6)) * ref.U * exact.abs()
    ref.check(gate, exact, slack, "gate")
    ref.check(up, -exact, slack, "up")
