"""The linear products' pipelines where tiles meet: contractions as long as a kernel's ring of stages, one stage less
and one more, with several tiles to a workgroup.  Formulas and bounds are test_gpu_linear's."""
import pytest
import torch
from test_gpu_linear import BF16, F16, close, expert_reference, groups_of, normal, ops

pytestmark = pytest.mark.gpu

# experts, rows of each, n, k: forward products in 256 x 128, 128 x 128, 64 x 128 and 64 x 64 tiles, whose rings hold 3, 4,
# 6 and 9 stages of 64 of k
FORWARD = [(128, 522, 32, 128), (32, 2067, 32, 192), (128, 528, 32, 256), (128, 258, 32, 192), (16, 2101, 32, 256),
           (64, 521, 32, 320), (32, 8, 1032, 320), (64, 8, 520, 384), (16, 8, 2128, 448), (64, 8, 264, 512),
           (64, 8, 272, 576), (3, 8, 5752, 640)]
# gradients of the weights in 128 x 128, 64 x 128 and 64 x 64 tiles, whose rings hold 4, 5 and 8 stages of 64 rows
WEIGHTS = [(128, 145, 408, 32), (128, 205, 392, 32), (128, 275, 408, 32), (32, 196, 1072, 32), (32, 261, 1072, 32),
           (16, 196, 32, 2120), (8, 260, 32, 4232), (64, 331, 32, 520), (16, 390, 1032, 32), (32, 467, 32, 520),
           (32, 530, 520, 32)]


def gathered(E, per, n, k, dtype):
    P = E * per
    g = torch.Generator(device='cuda').manual_seed(P)
    R = P // 2
    rows = torch.randint(0, R, (P,), generator=g, device='cuda')
    x, w = normal(R, k, dtype=dtype, seed=1), normal(E, n, k, dtype=dtype, seed=2, scale=k ** -0.5)
    return x, w, groups_of([per] * E), rows, normal(P, n, dtype=dtype, seed=3)


@pytest.mark.parametrize('case', FORWARD)
def test_rows_of_the_next_tile(case):
    x, w, starts, rows, _ = gathered(*case, BF16 if case[3] % 128 else F16)
    close(ops().expert_linear(x, w, starts, rows=rows), *expert_reference(x, w, starts, rows=rows)['y'], 'y')


@pytest.mark.parametrize('case', WEIGHTS)
def test_rows_of_the_next_weights(case):
    x, w, starts, rows, dy = gathered(*case, BF16 if case[1] % 2 else F16)
    close(ops().expert_linear_grad(dy, x, w, starts, rows, need_x=False, need_bias=False)[1],
          *expert_reference(x, w, starts, rows=rows, dy=dy)['dw'], 'dw')


@pytest.mark.parametrize('counts,n,k', [([2146, 2146], 160, 14464), ([888, 1, 1776, 887], 136, 12312), ([3900, 33], 152, 14400)])
def test_rows_of_parts(counts, n, k):
    """256 x 256 tiles of a contraction in 16 parts of which the last is short (64) or empty, with more of these
    than workgroups."""
    P = sum(counts)
    rows = torch.randint(0, P, (P,), generator=torch.Generator(device='cuda').manual_seed(k), device='cuda')
    x, w = normal(P, k, seed=1), normal(len(counts), n, k, seed=2, scale=k ** -0.5)
    starts = groups_of(counts)
    close(ops().expert_linear(x, w, starts, rows=rows), *expert_reference(x, w, starts, rows=rows)['y'], 'y')


@pytest.mark.parametrize('m,n,k', [(4097, 2120, 2048), (8193, 1344, 1032), (4097, 2048, 2104), (2049, 4104, 2056)])
def test_one_row_left_and_few_columns(m, n, k):
    """dW in 256 x 256 tiles whose contraction ends with one row and whose last tiles have fewer than 128 columns."""
    x, dy = normal(m, k, seed=1), normal(m, n, seed=2)
    _, dw, _ = ops().linear_grad(dy, x, normal(n, k, seed=3), need_x=False, need_bias=False)
    starts = groups_of([m])
    close(dw, *[t[0] for t in expert_reference(x, torch.zeros(1, n, k, dtype=BF16, device='cuda'), starts, dy=dy)['dw']], 'dw')


@pytest.mark.parametrize('gather', [False, True])
@pytest.mark.parametrize('counts,n,k', [([2049, 4097, 65], 2168, 2056), ([129] * 16, 1288, 2104), ([1, 0, 2113, 65], 4104, 2168)])
def test_one_row_left_of_groups(counts, n, k, gather):
    P = sum(counts)
    rows = torch.randint(0, 3, (P,), generator=torch.Generator(device='cuda').manual_seed(k), device='cuda') if gather else None
    x, dy = normal(3 if gather else P, k, seed=1), normal(P, n, seed=2)
    w, starts = torch.zeros(len(counts), n, k, dtype=BF16, device='cuda'), groups_of(counts)
    dw = ops().expert_linear_grad(dy, x, w, starts, rows, need_x=False, need_bias=False)[1]
    close(dw, *expert_reference(x, w, starts, rows=rows, dy=dy)['dw'], 'dw')
