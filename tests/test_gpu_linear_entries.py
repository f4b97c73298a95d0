"""ferry_expert_linear and the gradients' C entries in the forms that the Python functions do not use.  Formulas and bounds are
test_gpu_linear's."""
import pytest
import torch
from test_gpu_linear import BF16, F16, close, groups_of, layer, normal, product, rounding

from ferry_amd._lib import last_error, lib

pytestmark = pytest.mark.gpu
NUMBERS = {None: 0, 'relu': 1, 'silu': 2, 'gelu': 3, 'gelu_tanh': 4}


def at(t):
    return None if t is None else t.data_ptr()


def scratch(op, pairs, n, k, groups):
    size = lib().ferry_linear_workspace_bytes(op, pairs, n, k, groups)
    return torch.empty(max(size, 16), dtype=torch.uint8, device='cuda'), size


def forward(x, w, starts=None, rows=None, bias=None, act=None, residual=None, pre=None, out=None, strides=()):
    """ferry_expert_linear of x [rows, k] and w [groups, n, k]; strides: those of x, w, residual and out that are not
    their tensors'."""
    E, n, k = w.shape
    pairs = x.shape[0] if rows is None else rows.numel()
    s = dict(x=x.stride(0), w=w.stride(1), residual=n, out=out.stride(0), **{})
    s.update(strides)
    ws, size = scratch(0, pairs, n, k, E)
    status = lib().ferry_expert_linear(
        at(x), 0 if x.dtype is BF16 else 2, x.shape[0], k, s['x'], at(rows), pairs, at(starts), E, at(w), n, s['w'], n * k,
        at(bias), n, NUMBERS[act], at(residual), s['residual'], at(pre), at(out), s['out'], 0, at(ws), size,
        torch.cuda.current_stream().cuda_stream)
    assert status == 0, last_error()
    torch.cuda.synchronize()
    return out


SIZES = [([20], 264, 512), ([3, 0, 17], 256, 256), ([300, 200], 512, 320), ([2100, 1996], 2048, 2048), ([4096], 2048, 512),
         ([4000, 3000, 1192], 6144, 256), ([60, 77], 35, 131), ([2146, 2146], 160, 14464)]


@pytest.mark.parametrize('case', range(len(SIZES)))
def test_gathered_rows_with_an_epilogue(case):
    """Rows by their numbers together with an activation, its kept argument and a residual, at each kernel's sizes."""
    counts, n, k = SIZES[case]
    dtype, act = (F16 if case % 2 else BF16), ['silu', 'gelu', 'relu', 'gelu_tanh'][case % 4]
    P, E = sum(counts), len(counts)
    R = max(1, P // 2)
    rows = torch.randint(0, R, (P,), generator=torch.Generator(device='cuda').manual_seed(case), device='cuda')
    x, w = normal(R, k, dtype=dtype, seed=1), normal(E, n, k, dtype=dtype, seed=2, scale=k ** -0.5)
    bias, res, starts = normal(E, n, dtype=dtype, seed=3), normal(P, n, dtype=dtype, seed=4), groups_of(counts)
    new = lambda: torch.full((P, n), 7.5, dtype=dtype, device='cuda')
    all_three, pre = new(), new()
    forward(x, w, starts, rows, bias, act, res, pre, all_three)
    only_act, only_res, only_pre, kept = (new() for _ in range(4))
    forward(x, w, starts, rows, act=act, out=only_act)
    forward(x, w, starts, rows, residual=res, out=only_res)
    forward(x, w, starts, rows, pre=kept, out=only_pre)
    ends = starts.tolist()
    for e in range(E):
        g = slice(ends[e], ends[e + 1])
        xe = x[rows[g]]
        y, b, z, zb = layer(xe, w[e], bias[e], act, res[g])
        close(all_three[g], y, b, 'all')
        close(pre[g], z, zb + rounding(z, dtype), 'pre')
        close(only_act[g], *layer(xe, w[e], None, act)[:2], 'activation')
        close(only_res[g], *layer(xe, w[e], None, None, res[g])[:2], 'residual')
        z, zb = product(xe.double(), w[e].double().t())
        close(only_pre[g], z, zb + rounding(z, dtype), 'no activation')
        close(kept[g], z, zb + rounding(z, dtype), 'pre without an activation')


@pytest.mark.parametrize('groups', [1, 2])
@pytest.mark.parametrize('m,n,k', [(5, 264, 512), (300, 512, 320), (2100, 2048, 128), (4104, 4096, 512), (77, 35, 131)])
def test_pre_without_an_activation(m, n, k, groups):
    """pre is the rounded argument of any activation, none among them: the product and its bias."""
    x, w, bias, res = normal(m, k, seed=1), normal(groups, n, k, seed=2, scale=k ** -0.5), normal(groups, n, seed=3), normal(m, n, seed=4)
    starts = groups_of([m]) if groups == 1 else groups_of([m // 2, m - m // 2])
    out, pre = (torch.full((m, n), 7.5, dtype=BF16, device='cuda') for _ in range(2))
    forward(x, w, starts, None, bias, None, res, pre, out)
    ends = starts.tolist()
    for e in range(groups):
        g = slice(ends[e], ends[e + 1])
        y, b, z, zb = layer(x[g], w[e], bias[e], None, res[g])
        close(out[g], y, b, 'out')
        close(pre[g], z, zb + rounding(z, BF16), 'pre')


@pytest.mark.parametrize('stride', [0, 8, -8, 1 << 40])
@pytest.mark.parametrize('groups,n,k', [(1, 264, 512), (64, 27136, 8), (3, 35, 131), (1, 1528, 46616)])
def test_one_row_of_any_stride(groups, n, k, stride):
    """One row's strides are not used: x, residual, out and, in the gradients, dz and x."""
    x, w, res = normal(1, k, seed=1), normal(groups, n, k, seed=2, scale=k ** -0.5), normal(1, n, seed=3)
    g = groups // 2
    starts = torch.tensor([0] * (g + 1) + [1] * (groups - g), dtype=torch.int64, device='cuda')
    beyond = torch.full((n + 64,), 7.5, dtype=BF16, device='cuda')
    forward(x, w, starts, None, None, 'gelu', res, None, beyond.view(1, -1),
            dict(x=stride, out=stride, residual=max(stride, 0)))
    close(beyond[:n][None], *layer(x, w[g], None, 'gelu', res)[:2], 'out')
    assert bool((beyond[n:] == 7.5).all())
    if groups * n * k > 1 << 25:
        return
    dz = normal(1, n, seed=4)
    stream = torch.cuda.current_stream().cuda_stream
    ws, size = scratch(2, 1, n, k, groups)
    dw = torch.empty(groups, n, k, dtype=BF16, device='cuda')
    assert lib().ferry_expert_linear_grad_w(at(dz), 0, 1, n, stride, at(x), 1, k, stride, None, at(starts), groups, at(dw),
                                            at(ws), size, stream) == 0, last_error()
    want, bound = product(dz.double().t(), x.double())
    close(dw[g], want, bound + rounding(want, BF16), 'dw')
    assert not dw[:g].any() and not dw[g + 1:].any()
    ws, size = scratch(1, 1, n, k, groups)
    dx = torch.empty(1, k, dtype=BF16, device='cuda')
    assert lib().ferry_expert_linear_grad_x(at(dz), 0, 1, n, stride, at(starts), groups, at(w), k, k, n * k, at(dx), 0, at(ws),
                                            size, stream) == 0, last_error()
    want, bound = product(dz.double(), w[g].double())
    close(dx, want, bound + rounding(want, BF16), 'dx')
