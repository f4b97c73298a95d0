"""gelu's tail keeps its relative accuracy.  Phi(z) = t e^(P(t) - x^2) / 2 with x = |z| / sqrt 2 <= 8.5 in fp32, u = 2^-24: x is
off by 2 u (its constant, its product), so x^2 by 4 u x^2; the fused P - x^2 adds u x^2, its product with log2 e 2 u of
x^2 (constant and product): 7 u x^2 = 3.0e-5 at most, as a relative error of the exponential; P's own roundings (below 4
in size, 10 of them), t's and the products' add 50 u = 3e-6.  The rest is one rounding to bf16."""
import math

import pytest
import torch
from test_gpu_linear import BF16, close, ops

pytestmark = pytest.mark.gpu


def test_gelu_tail():
    z = -torch.linspace(4, 12, 4096, device='cuda').to(BF16)
    w = torch.eye(64, dtype=BF16, device='cuda')
    y = ops().linear(z.view(-1, 64), w, activation='gelu').view(-1)
    want = 0.5 * z.double() * torch.special.erfc(-z.double() / math.sqrt(2))
    close(y, want, (torch.finfo(BF16).eps / 2 * 1.0001 + 3.3e-5) * want.abs(), 'tail')
