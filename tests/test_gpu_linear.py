"""linear, expert_linear and their gradients against their formulas in 64 bits, at the sizes, strides and
groups where the kernels change their way of working.

Bounds.  With u = eps / 2 of the type and g = (c + 8) 2^-24 for a contraction of c (fp32 products of two
such values are exact, each addition is off by at most 2^-24 of a partial sum that the sum of magnitudes
bounds), a sum is off by g times the sum of magnitudes.  Activations have slopes of at most 1.13 and second
derivatives of at most 1.13 (silu: 1.1 and 0.5, gelu and its tanh form: 1.13 and 0.8 to 1.13), and are
evaluated to 4e-6 of their argument's size (three fp32 roundings, the hardware's exp2 and reciprocal, and
their constants).  An output is rounded once, by u of its size, or 2^-25 below fp16's normal numbers.
dz = dy f'(z) is off by u |dz| for its rounding, 1.13 |dy| times the error of z (that of the sum, and u |z|
for pre's rounding) and 1e-5 |dy|."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16
ACTS = [None, 'relu', 'silu', 'gelu', 'gelu_tanh']


def ops():
    from ferry_amd import expert_ops
    return expert_ops


def normal(*shape, dtype=BF16, seed=0, scale=1.0):
    g = torch.Generator(device='cuda').manual_seed(seed)
    return (torch.randn(shape, generator=g, device='cuda') * scale).to(dtype)


def strided(t, left, right):
    """The same matrix as part of a wider one, `left` columns into it; NaN all around."""
    wide = torch.full((t.shape[0], left + t.shape[1] + right), math.nan, dtype=t.dtype, device=t.device)
    view = wide[:, left:left + t.shape[1]]
    view.copy_(t)
    return view


def f64(act, z):
    """(f(z), f'(z)) in 64 bits."""
    if act is None:
        return z, torch.ones_like(z)
    if act == 'relu':
        return z.clamp(min=0), (z > 0).double()
    if act == 'silu':
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if act == 'gelu':
        p = 0.5 * torch.special.erfc(-z / math.sqrt(2))
        return z * p, p + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    c = 2 * math.sqrt(2 / math.pi)
    s = torch.sigmoid(c * (z + 0.044715 * z ** 3))
    return z * s, s + z * s * (1 - s) * c * (1 + 3 * 0.044715 * z * z)


def rounding(v, dtype):
    return torch.finfo(dtype).eps / 2 * v.abs() + 2.0 ** -25


def product(a, b):
    """(a b, the bound of an fp32 sum's error) of float64 matrices; exact enough in 64 bits."""
    return a @ b, (a.shape[1] + 8) * 2.0 ** -24 * (a.abs() @ b.abs())


def close(got, want, bound, what):
    got = got.double()
    bad = ~((got - want).abs() <= bound)
    if bool(bad.any()):
        at = tuple(int(i) for i in bad.nonzero()[0])
        raise AssertionError(f'{what}: {int(bad.sum())} of {bad.numel()} off, first at {at}: {got[at].item()} for '
                             f'{want[at].item()} +- {bound[at].item()}')


def layer(x, w, bias=None, act=None, residual=None):
    """Float64 (y, bound, z, bound of z)."""
    z, zb = product(x.double(), w.double().t())
    if bias is not None:
        z = z + bias.double()
        zb = zb + 2.0 ** -23 * z.abs()
    y, _ = f64(act, z)
    b = 1.13 * zb + 4e-6 * z.abs()
    if residual is not None:
        y = y + residual.double()
        b = b + 2.0 ** -23 * y.abs()
    return y, b + rounding(y, x.dtype), z, zb


def layer_grad(dy, x, w, z, zb, act):
    """{name: (gradient, bound)} in float64."""
    dt, dy, x, w = x.dtype, dy.double(), x.double(), w.double()
    slope = f64(act, z)[1]
    dz = dy * slope
    if act is None:
        db_err = err = torch.zeros_like(dz)
    else:
        db_err = dy.abs() * (1.13 * (zb + rounding(z, dt)) + 1e-5)
        if act == 'relu':   # where the sign of z is open, the slope is
            db_err = torch.where(z.abs() <= zb, dy.abs(), dy.abs() * 1e-5)
        err = db_err + rounding(dz, dt)
    out = {}
    dx, e = product(dz, w)
    out['dx'] = dx, e * 2 + err @ w.abs() * 1.01 + rounding(dx, dt) * 1.01
    dw, e = product(dz.t(), x)
    out['dw'] = dw, e * 2 + err.t() @ x.abs() * 1.01 + rounding(dw, dt) * 1.01
    db = dz.sum(0)
    out['db'] = db, db_err.sum(0) + (dz.shape[0] + 8) * 2.0 ** -24 * dz.abs().sum(0) * 2 + rounding(db, dt) * 1.01
    return out


SIZES = [(1, 1, 1), (1, 8, 8), (2, 16, 64), (3, 5, 7), (16, 64, 128), (17, 33, 65), (31, 40, 24), (64, 64, 64),
         (65, 72, 200), (127, 129, 130), (128, 128, 128), (129, 136, 320), (256, 256, 64), (257, 264, 1000),
         (300, 1001, 777), (1, 2048, 2048), (4, 520, 4104), (16, 200, 8200), (1030, 64, 64), (520, 1032, 96),
         (2100, 2048, 128), (640, 2304, 256)]


@pytest.mark.parametrize('dtype', [BF16, F16])
@pytest.mark.parametrize('m,n,k', SIZES)
def test_linear(m, n, k, dtype):
    x, w = normal(m, k, dtype=dtype, seed=1), normal(n, k, dtype=dtype, seed=2, scale=k ** -0.5)
    bias, res = normal(n, dtype=dtype, seed=3), normal(m, n, dtype=dtype, seed=4)
    y, b, _, _ = layer(x, w)
    close(ops().linear(x, w), y, b, 'plain')
    act = ACTS[1 + (m + n + k) % 4]
    y, b, z, zb = layer(x, w, bias, act, res)
    got, pre = ops().linear(x, w, bias, act, res, return_pre=True)
    close(got, y, b, act)
    close(pre, z, zb + rounding(z, dtype), 'pre')


@pytest.mark.parametrize('act', ACTS)
@pytest.mark.parametrize('dtype', [BF16, F16])
def test_activations(act, dtype):
    """Each activation over its whole range: arguments of every size, through an identity weight."""
    v = torch.cat([torch.linspace(-12, 12, 4096), torch.logspace(-8, 4, 512), -torch.logspace(-8, 4, 512)]).cuda().to(dtype)
    x = v.reshape(-1, 64)
    w = torch.eye(64, dtype=dtype, device='cuda')
    y, b, z, zb = layer(x, w, None, act)
    got, pre = ops().linear(x, w, activation=act, return_pre=True)
    close(got, y, b, act)
    dy = normal(x.shape[0], 64, dtype=dtype, seed=5)
    dx, dw, db = ops().linear_grad(dy, x, w, pre, act)
    for name, got in (('dx', dx), ('dw', dw), ('db', db)):
        close(got, *layer_grad(dy, x, w, z, zb, act)[name], f'{act} {name}')


@pytest.mark.parametrize('act', ACTS)
def test_special_values(act):
    """NaN, infinities and the largest values, as torch's own functions have them."""
    x = torch.tensor([math.nan, math.inf, 1e30, -1e30, 0.0, -0.0, 1.0, -200.0], device='cuda').to(BF16)[:, None]
    w = torch.ones((1, 1), dtype=BF16, device='cuda')
    got, pre = ops().linear(x, w, activation=act, return_pre=True)
    v = x.double()
    ref = {None: v, 'relu': torch.relu(v), 'silu': torch.nn.functional.silu(v),
           'gelu': torch.nn.functional.gelu(v), 'gelu_tanh': torch.nn.functional.gelu(v, approximate='tanh')}[act]
    assert torch.equal(torch.nan_to_num(got.double(), 7.5), torch.nan_to_num(ref.to(BF16).double(), 7.5))
    if act is not None:
        dx, _, _ = ops().linear_grad(torch.ones_like(x), x, w, pre, act, need_weight=False, need_bias=False)
        d = dx.double().flatten()
        assert math.isnan(d[0]) and d[2] == 1 and d[3] == 0


@pytest.mark.parametrize('left,right', [(0, 8), (8, 0), (16, 48), (1, 0), (3, 5)])
@pytest.mark.parametrize('m,n,k', [(5, 24, 40), (130, 136, 200), (33, 35, 37)])
def test_strides(m, n, k, left, right):
    """Parts of wider matrices, NaN in what surrounds them; an output whose surroundings stay as they were."""
    x, w = normal(m, k, seed=1), normal(n, k, seed=2, scale=k ** -0.5)
    bias, res, dy = normal(n, seed=3), normal(m, n, seed=4), normal(m, n, seed=5)
    y, b, z, zb = layer(x, w, bias, 'silu', res)
    xs, ws, rs, ds = (strided(t, left, right) for t in (x, w, res, dy))
    out = strided(torch.zeros_like(res), left, right)
    got, pre = ops().linear(xs, ws, bias, 'silu', rs, out=out, return_pre=True)
    assert got is out
    close(out, y, b, 'out')
    wide = out.as_strided((m, left + n + right), (left + n + right, 1), 0)
    assert bool(wide[:, :left].isnan().all()) and bool(wide[:, left + n:].isnan().all())
    dx, dw, db = ops().linear_grad(ds, xs, ws, pre, 'silu')
    want = layer_grad(dy, x, w, z, zb, 'silu')
    for name, got in (('dx', dx), ('dw', dw), ('db', db)):
        close(got, *want[name], name)
    _, _, z, zb = layer(x, w)
    want = layer_grad(dy, x, w, z, zb, None)   # without an activation grad itself enters the products
    for name, got in zip(('dx', 'dw', 'db'), ops().linear_grad(ds, xs, ws)):
        close(got, *want[name], name)


def test_out_is_the_residual():
    x, w, res = normal(70, 96, seed=1), normal(48, 96, seed=2, scale=0.1), normal(70, 48, seed=3)
    y, b, _, _ = layer(x, w, None, 'gelu', res)
    out = ops().linear(x, w, activation='gelu', residual=res, out=res)
    assert out is res
    close(res, y, b, 'in place')


def test_leading_dimensions_and_no_rows():
    x, w = normal(2, 3, 64, seed=1), normal(40, 64, seed=2)
    y = ops().linear(x, w)
    assert y.shape == (2, 3, 40) and torch.equal(y.view(6, 40), ops().linear(x.view(6, 64), w))
    assert torch.equal(ops().linear(x[0, 0], w), y[0, 0])
    none = ops().linear(x[:, :0], w, activation='relu', return_pre=True)
    assert none[0].shape == (2, 0, 40) and none[1].shape == (0, 40)
    dx, dw, db = ops().linear_grad(none[0], x[:, :0], w, none[1], 'relu')
    assert dx.shape == (2, 0, 64) and not dw.any() and not db.any()


def test_bad_rows_of_x_stay_in_their_own():
    x, w = normal(200, 256, seed=1), normal(264, 256, seed=2)
    clean = ops().linear(x, w)
    x[77] = math.nan
    x[130, 3] = math.inf
    y = ops().linear(x, w)
    keep = torch.ones(200, dtype=torch.bool, device='cuda')
    keep[[77, 130]] = False
    assert torch.equal(y[keep], clean[keep]) and bool(y[77].isnan().all())
    assert not bool(y[130].isfinite().any())


@pytest.mark.parametrize('act', ACTS)
@pytest.mark.parametrize('m,n,k', [(1, 8, 8), (3, 5, 7), (64, 64, 64), (65, 129, 72), (300, 200, 1001), (1030, 520, 264),
                                   (2048, 256, 128), (5000, 72, 40), (17, 2304, 2048)])
def test_linear_grad(m, n, k, act):
    dtype = F16 if (m + n) % 2 else BF16
    x, w = normal(m, k, dtype=dtype, seed=1), normal(n, k, dtype=dtype, seed=2, scale=k ** -0.5)
    bias, dy = normal(n, dtype=dtype, seed=3), normal(m, n, dtype=dtype, seed=4)
    _, pre = ops().linear(x, w, bias, act, return_pre=True)
    got = ops().linear_grad(dy, x, w, pre, act)
    _, _, z, zb = layer(x, w, bias)
    want = layer_grad(dy, x, w, z, zb, act)
    for name, v in zip(('dx', 'dw', 'db'), got):
        close(v, *want[name], name)
    for need in ((True, False, False), (False, True, False), (False, False, True)):
        some = ops().linear_grad(dy, x, w, pre, act, *need)
        for a, b, c in zip(some, got, need):
            assert (a is None) if not c else torch.equal(a, b)


def test_autograd_and_differences():
    """Gradients through autograd are linear_grad's, and those of the 64-bit loss by central differences."""
    x, w, b, r = (normal(6, 40, seed=1), normal(24, 40, seed=2, scale=0.3), normal(24, seed=3), normal(6, 24, seed=4))
    dy = normal(6, 24, seed=5)
    for act in ACTS:
        leaves = [t.clone().requires_grad_() for t in (x, w, b, r)]
        y = ops().linear(leaves[0], leaves[1], leaves[2], act, leaves[3])
        got = torch.autograd.grad(y, leaves, dy)
        _, pre = ops().linear(x, w, b, act, r, return_pre=True)
        for a, c in zip(got, (*ops().linear_grad(dy, x, w, pre, act), dy)):
            assert torch.equal(a, c)
        _, _, z, zb = layer(x, w, b)
        bounds = layer_grad(dy, x, w, z, zb, act)

        def loss(px, pw, pb):
            return float(((f64(act, px @ pw.t() + pb)[0]) * dy.double()).sum())
        at = [t.double() for t in (x, w, b)]
        for i, name in enumerate(('dx', 'dw', 'db')):
            v = normal(*at[i].shape, seed=9 + i).double()
            h = 1e-6
            hi, lo = list(at), list(at)
            hi[i], lo[i] = at[i] + h * v, at[i] - h * v
            diff = (loss(*hi) - loss(*lo)) / (2 * h)
            mine = float((got[i].double() * v).sum())
            assert abs(mine - diff) <= float((bounds[name][1] * v.abs()).sum()) + 1e-4 * abs(diff) + 1e-4, (act, name)


def test_autograd_gives_what_is_asked():
    x, w = normal(6, 40, seed=1), normal(24, 40, seed=2)
    y = ops().linear(x, w.clone().requires_grad_(), activation='gelu')
    y.sum().backward()   # a gradient of stride 0
    assert not ops().linear(x, w).requires_grad
    with torch.no_grad():
        assert not ops().linear(x, w.clone().requires_grad_()).requires_grad
    xr = x.clone().requires_grad_()
    z = ops().linear(ops().linear(xr, w, activation='silu'), normal(16, 24, seed=3))
    z.float().square().sum().backward()
    assert xr.grad.shape == x.shape and bool(xr.grad.isfinite().all())


FEW = [(m, n, k) for m in (1, 7, 16, 17, 32, 33, 50, 64) for n, k in ((8, 8), (37, 264), (1000, 1032), (2064, 520), (40, 4160))]


@pytest.mark.parametrize('m,n,k', FEW)
def test_few_rows(m, n, k):
    dtype = F16 if (m + n) % 3 else BF16
    x, w = normal(m, k, dtype=dtype, seed=1), normal(n, k, dtype=dtype, seed=2, scale=k ** -0.5)
    bias, res = normal(n, dtype=dtype, seed=3), normal(m, n, dtype=dtype, seed=4)
    act = ACTS[(m + n + k) % 5]
    y, b, z, zb = layer(x, w, bias, act, res)
    got, pre = ops().linear(x, w, bias, act, res, return_pre=True)
    close(got, y, b, act)
    if act:
        close(pre, z, zb + rounding(z, dtype), 'pre')


LARGE = [(2056, 2312, 264), (4104, 1032, 72), (1800, 4096, 8), (2304, 2048, 136), (257, 12296, 320), (2500, 2048, 1160)]


@pytest.mark.parametrize('dtype', [BF16, F16])
@pytest.mark.parametrize('m,n,k', LARGE)
def test_large_tiles(m, n, k, dtype):
    """Sizes of many tiles, most of them with partial tiles and a contraction that ends inside a stage."""
    x, w = normal(m, k, dtype=dtype, seed=1), normal(n, k, dtype=dtype, seed=2, scale=k ** -0.5)
    bias, res, dy = normal(n, dtype=dtype, seed=3), normal(m, n, dtype=dtype, seed=4), normal(m, n, dtype=dtype, seed=5)
    act = ACTS[(m + n + k) // 8 % 5]
    y, b, z, zb = layer(x, w, bias, act, res)
    got, pre = ops().linear(x, w, bias, act, res, return_pre=True)
    close(got, y, b, act)
    want = layer_grad(dy, x, w, z, zb, act)
    for name, v in zip(('dx', 'dw', 'db'), ops().linear_grad(dy, x, w, pre, act)):
        close(v, *want[name], name)
    close(ops().linear(x, w), *layer(x, w)[:2], 'plain')


# -- experts ------------------------------------------------------------------------------------------

def groups_of(counts, head=0):
    return torch.tensor([head + sum(counts[:i]) for i in range(len(counts) + 1)], dtype=torch.int64, device='cuda')


def expert_reference(x, w, starts, bias=None, rows=None, dy=None):
    """Float64 {name: (value, bound)}; rows of no expert are 0."""
    ends = starts.tolist()
    P = x.shape[0] if rows is None else rows.numel()
    dt = x.dtype
    E, n, k = w.shape
    token = torch.arange(P, device='cuda') if rows is None else rows
    zeros = lambda *s: torch.zeros(s, dtype=torch.float64, device='cuda')
    out = {name: (zeros(*s), zeros(*s)) for name, s in
           (('y', (P, n)), ('dxp', (P, k)), ('dw', (E, n, k)), ('db', (E, n)))}
    for e in range(E):
        at = slice(ends[e], ends[e + 1])
        xe = x[token[at]]
        y, b, z, zb = layer(xe, w[e], None if bias is None else bias[e])
        out['y'][0][at], out['y'][1][at] = y, b
        if dy is not None:
            g = layer_grad(dy[at], xe, w[e], z, zb, None)
            out['dxp'][0][at], out['dxp'][1][at] = g['dx']
            out['dw'][0][e], out['dw'][1][e] = g['dw']
            out['db'][0][e], out['db'][1][e] = g['db']
    return out


COUNTS = [([1] * 40 + [0] * 30 + [9] * 20 + [200], 520, 1032), ([20, 30, 0, 33, 16, 17] * 5, 2064, 264),
          ([64, 50, 0, 10] * 9, 1000, 520), ([1], 2000, 2048), ([2, 0, 1], 4104, 72),
          ([300, 0, 1, 700, 256, 255, 257, 0, 600, 31], 1032, 264), ([0, 900, 513, 0, 64, 2, 1100], 2048, 1032),
          ([1], 8, 8), ([0, 3, 0], 24, 40), ([0, 1, 63, 64, 65, 0, 200, 3], 72, 136), ([5] * 33, 64, 64),
          ([300, 0, 7], 35, 37), ([0] * 60 + [2] + [0] * 67, 256, 512), ([1, 0, 2] * 100, 40, 72),
          ([129, 127, 255, 257, 1, 16, 17, 33], 264, 200), ([1000, 30, 500, 2], 520, 96), ([0, 0], 16, 16),
          ([64] * 8, 1032, 1032), ([3] * 512, 16, 24)]


@pytest.mark.parametrize('gather', [False, True])
@pytest.mark.parametrize('case', range(len(COUNTS)))
def test_expert_linear(case, gather):
    counts, n, k = COUNTS[case]
    dtype = F16 if case % 2 else BF16
    E, P = len(counts), sum(counts)
    g = torch.Generator(device='cuda').manual_seed(case)
    R = max(1, P // 2) if gather else P
    x, w = normal(R, k, dtype=dtype, seed=1), normal(E, n, k, dtype=dtype, seed=2, scale=k ** -0.5)
    bias, dy = normal(E, n, dtype=dtype, seed=3), normal(P, n, dtype=dtype, seed=4)
    rows = torch.randint(0, R, (P,), generator=g, device='cuda') if gather else None
    starts = groups_of(counts)
    want = expert_reference(x, w, starts, bias, rows, dy)
    close(ops().expert_linear(x, w, starts, bias, rows), *want['y'], 'y')
    dx, dw, db = ops().expert_linear_grad(dy, x, w, starts, rows)
    for name, v in (('dxp', dx), ('dw', dw), ('db', db)):
        close(v, *want[name], name)


def test_rows_of_no_expert():
    """Rows before the first group and behind the last: zeros in a new output, untouched in a given one, and
    no part of any gradient, whatever they hold."""
    counts, head, P, n, k = [3, 0, 70, 9], 5, 120, 40, 72
    starts = groups_of(counts, head)
    x, w, dy = normal(P, k, seed=1), normal(4, n, k, seed=2, scale=0.1), normal(P, n, seed=3)
    x[:head], x[head + 82:] = math.nan, math.inf
    dy[:head], dy[head + 82:] = math.inf, math.nan
    want = expert_reference(x, w, starts, None, None, dy)
    close(ops().expert_linear(x, w, starts), *want['y'], 'y')
    out = torch.full((P, n), 3.0, dtype=BF16, device='cuda')
    ops().expert_linear(x, w, starts, out=out)
    assert bool((out[:head] == 3).all()) and bool((out[head + 82:] == 3).all())
    close(out[head:head + 82], want['y'][0][head:head + 82], want['y'][1][head:head + 82], 'out')
    dx, dw, db = ops().expert_linear_grad(dy, x, w, starts)
    for name, v in (('dxp', dx), ('dw', dw), ('db', db)):
        close(v, *want[name], name)


def test_neighbours_stay_out_of_sums():
    """NaN rows of one expert leave the others' outputs and gradients alone."""
    counts, n, k = [7, 65, 1, 130], 48, 56
    starts = groups_of(counts)
    x, w, dy = normal(203, k, seed=1), normal(4, n, k, seed=2, scale=0.1), normal(203, n, seed=3)
    y = ops().expert_linear(x, w, starts)
    got = ops().expert_linear_grad(dy, x, w, starts)
    bad, bdy = x.clone(), dy.clone()
    bad[7:72], bdy[7:72] = math.nan, math.inf
    y2 = ops().expert_linear(bad, w, starts)
    got2 = ops().expert_linear_grad(bdy, bad, w, starts)
    keep = torch.ones(203, dtype=torch.bool, device='cuda')
    keep[7:72] = False
    assert torch.equal(y[keep], y2[keep]) and torch.equal(got[0][keep], got2[0][keep])
    for e in (0, 2, 3):
        assert torch.equal(got[1][e], got2[1][e]) and torch.equal(got[2][e], got2[2][e])
    assert not bool(got2[1][1].isfinite().any())


def test_weights_in_cache_rows():
    """Gate|up and down matrices where the expert cache holds them: strides of experts larger than a matrix."""
    H, I, E = 64, 48, 5
    cache = normal(E, 3 * H * I, seed=1, scale=0.1)
    up = cache[:, :2 * H * I].unflatten(1, (2 * I, H))
    down = cache[:, 2 * H * I:].unflatten(1, (H, I))
    starts = groups_of([3, 0, 70, 1, 20])
    x, a = normal(94, H, seed=2), normal(94, I, seed=3)
    close(ops().expert_linear(x, up, starts), *expert_reference(x, up, starts)['y'], 'up')
    want = expert_reference(a, down, starts, dy=x)
    close(ops().expert_linear(a, down, starts), *want['y'], 'down')
    close(ops().expert_linear_grad(x, a, down, starts)[0], *want['dxp'], 'dx')
    one = normal(1, 32, H, seed=4).expand(E, 32, H)   # one matrix for every expert
    close(ops().expert_linear(x, one, starts), *expert_reference(x, one, starts)['y'], 'shared')


def test_starts_and_rows_out_of_range():
    """Starts outside the pairs are forced into them, a group that ends before it starts has no rows, and rows of x
    that are not there read as zeros."""
    x, w = normal(50, 64, seed=1), normal(4, 32, 64, seed=2)
    wild = torch.tensor([-5, 10, 10, 1 << 40, 1 << 33], dtype=torch.int64, device='cuda')
    tame = torch.tensor([0, 10, 10, 50, 50], dtype=torch.int64, device='cuda')
    assert torch.equal(ops().expert_linear(x, w, wild), ops().expert_linear(x, w, tame))
    dy = normal(50, 32, seed=3)
    for a, b in zip(ops().expert_linear_grad(dy, x, w, wild), ops().expert_linear_grad(dy, x, w, tame)):
        assert torch.equal(a, b)
    back = torch.tensor([0, 10, 3, 10, 50], dtype=torch.int64, device='cuda')   # group 1 ends before it starts
    assert bool(ops().expert_linear_grad(dy, x, w, back)[1][1].eq(0).all())
    rows = torch.arange(50, device='cuda')
    rows[[4, 30]] = torch.tensor([-1, 50], device='cuda')
    zeroed = x.clone()
    zeroed[[4, 30]] = 0
    assert torch.equal(ops().expert_linear(x, w, tame, rows=rows), ops().expert_linear(zeroed, w, tame))
    assert torch.equal(ops().expert_linear_grad(dy, x, w, tame, rows=rows)[1],
                       ops().expert_linear_grad(dy, zeroed, w, tame)[1])


@pytest.mark.parametrize('counts,n,k', [([40, 3], 512, 320), ([300, 0, 513, 40], 1032, 264), ([700, 400, 900], 2048, 200),
                                        ([2, 1, 0, 5], 72, 1000), ([600, 500], 35, 141)])
def test_bad_rows_in_every_kernel(counts, n, k):
    """Entries of rows that name no row of x, their high words set among them, read as zeros, at the sizes of each
    kernel; NaN in the row they would name otherwise."""
    P = sum(counts)
    starts = groups_of(counts)
    x, w, dy = normal(P, k, seed=1), normal(len(counts), n, k, seed=2, scale=k ** -0.5), normal(P, n, seed=3)
    rows = torch.randperm(P, device='cuda')
    bad = rows.clone()
    at = [0, P // 2, P - 1]
    bad[at] = torch.tensor([-1, P, (1 << 32) + 1], device='cuda')
    zeroed = x[rows]
    zeroed[at] = 0
    want = expert_reference(zeroed, w, starts, dy=dy)
    close(ops().expert_linear(x, w, starts, rows=bad), *want['y'], 'y')
    close(ops().expert_linear_grad(dy, x, w, starts, rows=bad)[1], *want['dw'], 'dw')


@pytest.mark.parametrize('n,k', [(512, 256), (40, 72), (33, 65)])
def test_experts_without_rows(n, k):
    """No expert has a row, or x has none: zeros, and nothing of what is there."""
    x, w = torch.full((300, k), math.nan, dtype=BF16, device='cuda'), normal(5, n, k, seed=1)
    starts = torch.zeros(6, dtype=torch.int64, device='cuda')
    assert not ops().expert_linear(x, w, starts).any()
    dy = torch.full((300, n), math.inf, dtype=BF16, device='cuda')
    for g in ops().expert_linear_grad(dy, x, w, starts):
        assert not g.any()
    y = ops().expert_linear(x[:0], w, starts)
    assert y.shape == (0, n)
    dx, dw, db = ops().expert_linear_grad(y, x[:0], w, starts)
    assert dx.shape == (0, k) and not dw.any() and not db.any()
    rows = torch.zeros(7, dtype=torch.int64, device='cuda')   # rows of an x without any
    spread = torch.tensor([0, 7, 7, 7, 7, 7], device='cuda')
    assert not ops().expert_linear(x[:0], w, spread, rows=rows).any()
    assert not ops().expert_linear_grad(normal(7, n, seed=2), x[:0], w, spread, rows=rows)[1].any()


@pytest.mark.parametrize('m', [3, 300, 2100])
def test_unaligned_bias_residual_and_pre(m):
    """A bias, a residual and an output that start at any element, on operands that do not."""
    n, k = 520, 264
    x, w = normal(m, k, seed=1), normal(n, k, seed=2, scale=k ** -0.5)
    bias, res = normal(n + 1, seed=3)[1:], normal(m * n + 3, seed=4)[3:].view(m, n)
    y, b, _, _ = layer(x, w, bias, 'gelu', res)
    close(ops().linear(x, w, bias, 'gelu', res), y, b, 'y')
    close(ops().linear(x, w, bias, 'gelu', res.clone(), out=res), y, b, 'out')


def test_one_row_of_any_stride_and_single_columns():
    x, w = normal(1, 64, seed=1), normal(48, 64, seed=2)
    assert torch.equal(ops().linear(x.as_strided((1, 64), (7, 1)), w), ops().linear(x, w))
    y, b, z, zb = layer(x[:, :1], w[:, :1])
    close(ops().linear(x[:, :1], w[:, :1]), y, b, 'k = 1')
    y, b, _, _ = layer(normal(50, 64, seed=3), w[:1])
    close(ops().linear(normal(50, 64, seed=3), w[:1]), y, b, 'n = 1')
    for bad in ((x[:, :0], w[:, :0]), (x, w[:0])):
        with pytest.raises(RuntimeError, match='at least 1'):
            ops().linear(*bad)
    with pytest.raises(RuntimeError, match='at least 1'):
        ops().expert_linear(x, w[None, :0], groups_of([1]))


def test_refusals_on_the_device():
    x, w = normal(6, 64, seed=1), normal(48, 64, seed=2)
    starts = groups_of([6])
    cases = [
        (lambda: ops().linear(x.float(), w.float()), 'bf16 or fp16'), (lambda: ops().linear(x, w.half()), 'weight must be'),
        (lambda: ops().linear(x, w[:, :32]), 'weight must be'), (lambda: ops().linear(x.t(), w[:, :6]), 'contiguous'),
        (lambda: ops().linear(x, w, bias=w[0]), 'bias must be'), (lambda: ops().linear(x, w, residual=x), 'residual must be'),
        (lambda: ops().linear(x, w, out=x), 'out must be'),
        (lambda: ops().linear(x, w, out=torch.empty(48, 6, dtype=BF16, device='cuda').t()), 'contiguous'),
        (lambda: ops().linear(x, w, bias=w[:, 0]), 'contiguous'), (lambda: ops().linear(x, w.cpu()), 'CUDA'),
        (lambda: ops().linear(x.clone().requires_grad_(), w, out=torch.empty(6, 48, dtype=BF16, device='cuda')), 'no gradients'),
        (lambda: ops().linear(x.clone().requires_grad_(), w, return_pre=True), 'no gradients'),
        (lambda: ops().linear_grad(x, x, w), 'grad must be'), (lambda: ops().linear_grad(x @ w.t(), x, w, None, 'silu'), 'pre must be'),
        (lambda: ops().expert_linear(x, w, starts), 'experts, n, k'), (lambda: ops().expert_linear(x, w[None], starts[:1]), 'starts must'),
        (lambda: ops().expert_linear(x, w[None], starts.int()), 'starts must'),
        (lambda: ops().expert_linear(x, w[None].transpose(1, 2).contiguous().transpose(1, 2), starts), 'rows of weight'),
        (lambda: ops().expert_linear(x, w[None], starts, bias=w[:1]), 'bias must be'),
        (lambda: ops().expert_linear(x, w[None], starts, rows=starts.int()), 'rows must'),
        (lambda: ops().expert_linear(x.clone().requires_grad_(), w[None], starts, rows=torch.arange(6, device='cuda')), 'pair_pos'),
        (lambda: ops().expert_linear(x, w[None].expand(513, 48, 64), torch.zeros(514, dtype=torch.int64, device='cuda')), 'groups must'),
        (lambda: ops().sum_pairs(x, torch.zeros(7, dtype=torch.int32, device='cuda'), 3), 'pair_pos must')]
    for call, word in cases:
        with pytest.raises(RuntimeError, match=word):
            call()


@pytest.mark.parametrize('dtype', [BF16, F16])
@pytest.mark.parametrize('tokens,topk,k', [(1, 1, 8), (5, 3, 7), (70, 6, 2048), (300, 8, 1001)])
def test_sum_pairs(tokens, topk, k, dtype):
    part = normal(tokens * topk, k, dtype=dtype, seed=1)
    g = torch.Generator(device='cuda').manual_seed(2)
    pos = torch.randperm(tokens * topk, generator=g, device='cuda').to(torch.int32)
    want = part.double()[pos.long()].view(tokens, topk, k)
    bound = (topk * 2.0 ** -24) * want.abs().sum(1) + rounding(want.sum(1), dtype)
    close(ops().sum_pairs(part, pos, tokens), want.sum(1), bound, 'sum')
    pos[0] = -1
    pos[-1] = tokens * topk
    want[0, 0] = 0
    want[-1, -1] = 0
    close(ops().sum_pairs(part, pos, tokens), want.sum(1), bound + 2.0 ** -8 * part.double().abs().max(), 'left out')
    assert ops().sum_pairs(part[:0], pos[:0], 0).shape == (0, k)


def moe_inputs(T=90, H=64, I=40, E=8, k=3, dtype=BF16):
    g = torch.Generator(device='cuda').manual_seed(7)
    x = normal(T, H, dtype=dtype, seed=1)
    logits = torch.randn((T, E), generator=g, device='cuda')
    weights, ids = ops().router_topk(logits, k)
    lay = ops().layout(ids, weights, E)
    up = normal(E, 2 * I, H, dtype=dtype, seed=2, scale=H ** -0.5)
    down = normal(E, H, I, dtype=dtype, seed=3, scale=I ** -0.5)
    return x, lay, up, down


def test_moe_layer_trains():
    """Router, layout, grouped gate|up, SwiGLU, grouped down, sum over the pairs, a dense layer with a residual:
    a training step's gradients against those of the same steps in 64 bits."""
    T, H, I, E, k = 90, 64, 40, 8, 3
    x, lay, up, down = moe_inputs(T, H, I, E, k)
    dense, bias = normal(H, H, seed=4, scale=H ** -0.5), normal(H, seed=5)
    gate = lay.w_sorted.view(-1)[(lay.rows * k + lay.cols)]
    dy = normal(T, H, seed=6)
    leaves = [t.clone().requires_grad_() for t in (x, up, down, dense, bias)]

    def step(px, pup, pdown, pdense, pbias, own):
        if own:
            h = ops().expert_linear(px, pup, lay.starts, rows=lay.rows, pair_pos=lay.pair_pos)
        else:
            h = torch.cat([px[lay.rows[s:e]] @ pup[i].t() for i, (s, e) in enumerate(zip(ends, ends[1:]))])
        a = torch.nn.functional.silu(h[:, :I]) * h[:, I:]
        if own:
            y = ops().expert_linear(a, pdown, lay.starts)
        else:
            y = torch.cat([a[s:e] @ pdown[i].t() for i, (s, e) in enumerate(zip(ends, ends[1:]))])
        y = (y * gate.to(y.dtype)[:, None])[lay.pair_pos.long()].view(T, k, H).sum(1)
        if own:
            return ops().linear(y, pdense, pbias, 'gelu', px)
        return torch.nn.functional.gelu(y @ pdense.t() + pbias) + px
    ends = lay.starts.tolist()
    out = step(*leaves, True)
    got = torch.autograd.grad(out, leaves, dy)
    ref = [t.double().requires_grad_() for t in (x, up, down, dense, bias)]
    out64 = step(*ref, False)
    want = torch.autograd.grad(out64, ref, dy.double())
    # seven roundings of u = 2^-8 in a chain (h, silu, the product, y, its sum, z, dz and their gradients) in
    # norm: at most 14 u with those of the way back
    for a, b in zip((out, *got), (out64, *want)):
        assert float((a.detach().double() - b).norm()) <= 14 * 2.0 ** -8 * float(b.detach().norm())
    # the gradient of the tokens is the sum of its pairs' rows
    h_dy = normal(T * k, 2 * I, seed=8)
    dxp = ops().expert_linear_grad(h_dy, x, up, lay.starts, lay.rows)[0]
    dx = ops().expert_linear_grad(h_dy, x, up, lay.starts, lay.rows, lay.pair_pos)[0]
    assert torch.equal(dx, ops().sum_pairs(dxp, lay.pair_pos, T))


# -- how calls are made ----------------------------------------------------------------------------------

def all_outputs(x, w, b, dy, experts):
    y, pre = ops().linear(x, w, b, 'silu', return_pre=True)
    ex, ew, starts, rows, edy, pos = experts
    ey = ops().expert_linear(ex, ew, starts, rows=rows)
    return [y, pre, *ops().linear_grad(dy, x, w, pre, 'silu'), ey,
            *ops().expert_linear_grad(edy, ex, ew, starts, rows, pos)]


@pytest.mark.parametrize('m,n,k', [(1, 256, 512), (300, 264, 1000), (700, 72, 40)])
def test_captured_and_replayed(m, n, k):
    """A captured step replays with new inputs, eager work in between, and gives the eager bits."""
    T, topk, E = m, 2, 6
    g = torch.Generator(device='cuda').manual_seed(1)
    ids = torch.rand((T, E), generator=g, device='cuda').argsort(1)[:, :topk].sort(1)[0].contiguous()
    lay = ops().layout(ids, None, E)

    def inputs(seed):
        return [normal(m, k, seed=seed), normal(n, k, seed=seed + 1, scale=k ** -0.5), normal(n, seed=seed + 2),
                normal(m, n, seed=seed + 3), normal(T, k, seed=seed + 4),
                normal(E, n, k, seed=seed + 5, scale=k ** -0.5), normal(T * topk, n, seed=seed + 6)]
    held = inputs(0)

    def step(v):
        return all_outputs(*v[:4], (v[4], v[5], lay.starts, lay.rows, v[6], lay.pair_pos))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(held)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(held)
    for seed in (10, 20, 30):
        new = inputs(seed)
        for h, v in zip(held, new):
            h.copy_(v)
        graph.replay()
        eager = step(new)
        torch.cuda.synchronize()
        for a, b in zip(outs, eager):
            assert torch.equal(a, b)


def test_same_bits_every_time_and_on_other_streams():
    x, w, b, dy = normal(333, 520, seed=1), normal(200, 520, seed=2), normal(200, seed=3), normal(333, 200, seed=4)
    starts = groups_of([100, 0, 200, 33])
    ew = normal(4, 200, 520, seed=5)
    args = (x, w, b, dy, (x, ew, starts, None, dy, None))
    first = all_outputs(*args)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for s in streams:
        with torch.cuda.stream(s):
            outs.append(all_outputs(*args))
    torch.cuda.synchronize()
    for other in outs:
        for a, c in zip(first, other):
            assert torch.equal(a, c)


def test_capture_with_autograd_is_refused():
    x, w = normal(4, 16, seed=1), normal(8, 16, seed=2).requires_grad_()
    starts = groups_of([4])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        keep = x + 1
        with pytest.raises(RuntimeError, match='linear_grad under torch.no_grad'):
            ops().linear(x, w)
        with pytest.raises(RuntimeError, match='expert_linear_grad under'):
            ops().expert_linear(x, w[None], starts)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(keep, x + 1)


@pytest.mark.parametrize('k', [64, 63])
def test_offsets_past_32_bits(k):
    """Rows more than 4 GiB apart."""
    stride = (1 << 31) + 64
    buf = torch.empty(2 * stride + 64, dtype=BF16, device='cuda')
    x = buf.as_strided((3, k), (stride, 1), 0)
    x.copy_(normal(3, k, seed=1))
    w = normal(16, k, seed=2)
    y, b, z, zb = layer(x.contiguous(), w)
    close(ops().linear(x, w), y, b, 'x')
    out = buf.as_strided((3, 16), (stride, 1), 0)
    xc = x.contiguous()
    ops().linear(xc, w, out=out)
    close(out, y, b, 'out')
    x.copy_(xc)
    dy = normal(3, 16, seed=3)
    want = layer_grad(dy, xc, w, z, zb, None)
    close(ops().linear_grad(dy, x, w)[1], *want['dw'], 'dw')
    rows = torch.tensor([2, 0, 1, 2], device='cuda')
    starts = groups_of([3, 1])
    ew = normal(2, 16, k, seed=4)
    edy = normal(4, 16, seed=5)
    ref = expert_reference(xc, ew, starts, rows=rows, dy=edy)
    close(ops().expert_linear(x, ew, starts, rows=rows), *ref['y'], 'gathered')
    close(ops().expert_linear_grad(edy, x, ew, starts, rows)[1], *ref['dw'], 'gathered dw')
    del x, out
    wide = buf.as_strided((2, 16, k), (stride, k, 1), 0)   # experts' weights far apart
    wide.copy_(ew)
    close(ops().expert_linear(xc, wide, starts, rows=rows), *expert_reference(xc, ew, starts, rows=rows)['y'], 'w')


@pytest.mark.parametrize('activation', ['relu', 'silu', 'gelu', 'gelu_tanh'])
def test_activation_argument_beyond_fp16(activation):
    """z = -+90,000 is finite in the sums and infinite where it is kept in fp16: f' there is still 0 or 1."""
    x = torch.tensor([[300.0], [-300.0]], dtype=torch.float16, device='cuda')
    w = torch.full((9, 1), 300.0, dtype=torch.float16, device='cuda')
    y, pre = ops().linear(x, w, None, activation, return_pre=True)
    assert bool(torch.isinf(pre).all()) and bool((y[1] == 0).all())
    dy = torch.ones(2, 9, dtype=torch.float16, device='cuda')
    dx, dw, db = ops().linear_grad(dy, x, w, pre, activation)
    assert dx.flatten().tolist() == [2700, 0]      # 9 * 1 * 300, exact in fp16 (a multiple of 2 below 4,096)
    assert bool((dw == 300).all()) and bool((db == 1).all())


def test_out_is_seen_by_autograd():
    x, w = normal(8, 16), normal(24, 16, seed=1)
    starts = torch.tensor([0, 8], device='cuda')
    out = torch.zeros(8, 24, dtype=BF16, device='cuda')
    for write in (lambda: ops().linear(x, w, out=out), lambda: ops().expert_linear(x, w[None], starts, out=out)):
        scale = torch.ones(8, 24, dtype=BF16, device='cuda', requires_grad=True)
        product = scale * out
        write()
        with pytest.raises(RuntimeError, match='modified by an inplace operation'):
            product.sum().backward()
    with torch.inference_mode():
        assert torch.equal(ops().linear(x, w, out=torch.empty(8, 24, dtype=BF16, device='cuda')), ops().linear(x, w))
