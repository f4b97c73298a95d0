"""mxfp4_expert_ffn in calls of few (token, expert) pairs, whose activations between up and down are kept finer than
bf16: eight columns share an exponent, and each has one of its own within it.  Columns of very different size, infinities,
NaNs."""
import pytest
import torch

from test_gpu_mxfp4_ffn import Case

pytestmark = pytest.mark.gpu


def down_codes(c, e):
    """The codes of an expert's down matrix, uint8 [H, I / 2], in place."""
    n = c.H * c.I
    return c.cache[int(c.slot_of[e])][n:n + n // 2].view(c.H, c.I // 2)


def scales(c, e, part):
    """The scale bytes of an expert's gate (0), up (1) or down (2) matrix, [rows, blocks], in place."""
    n = c.H * c.I // 32
    s = c.cache[int(c.slot_of[e])][48 * n:].view(3, n)[part]
    return s.view(c.H if part == 2 else c.I, -1)


def reference(c, x):
    """(values, bound, bound with activations in bf16) float64 [P, H]."""
    P = c.rows.numel()
    out = torch.zeros((P, c.H), dtype=torch.float64, device='cuda')
    bounds = [torch.zeros_like(out), torch.zeros_like(out)]
    eps = 2.0 ** -24
    for e in range(c.E):
        lo, hi = int(c.starts[e]), int(c.starts[e + 1])
        wg, wu, wd = c.weights(e)
        xe = x.double()[c.rows[lo:hi]]
        g, u = xe @ wg.t(), xe @ wu.t()
        a = g * torch.sigmoid(g) * u
        # fp32 sums of H products (H + 8 roundings of the sum of magnitudes), |d silu| <= 1.1 |dg|, about 10 roundings of
        # the SwiGLU
        dg = (c.H + 8) * eps * (xe.abs() @ wg.abs().t())
        du = (c.H + 8) * eps * (xe.abs() @ wu.abs().t())
        d0 = 1.1 * dg * u.abs() + (g * torch.sigmoid(g)).abs() * du + dg * du + 16 * eps * a.abs()
        # the largest of eight, rounded to 11 bits, lies in [2^j, 2^(j + 1)): down to 2^(j - 14) a column has 11 bits, half
        # a step of which is at most 2^-11 of it, and below that steps of 2^(j - 24), half of one at most 2^-25 of the largest
        most = (a.abs() + d0).reshape(-1, 8).amax(1, keepdim=True).expand(-1, 8).reshape(a.shape)
        fine = d0 + 2.0 ** -11 * (a.abs() + d0) + 2.0 ** -25 * (1 + 2.0 ** -10) * most
        y = a @ wd.t()
        wt = c.w[c.rows[lo:hi], c.cols[lo:hi]].double()[:, None]
        out[lo:hi] = y * wt
        for tol, da in zip(bounds, (fine, d0 + 2.0 ** -8 * (a.abs() + d0))):
            dy = da @ wd.abs().t() + (c.I + 8) * eps * ((a.abs() + da) @ wd.abs().t())
            tol[lo:hi] = dy * wt + 2.0 ** -8 * ((y * wt).abs() + dy * wt) + 4 * eps * (y * wt).abs()
    return out, *bounds


CASES = [(2048, 768, [1] * 8, 8), (512, 2816, [8, 5, 1, 0, 8], 4), (128, 128, [1], 1), (384, 640, [2, 3, 7, 8, 1], 8)]


@pytest.mark.parametrize('H,I,counts,k', CASES)
@pytest.mark.parametrize('more', [0, 10, 13])
def test_large_columns_over_zero_weights(device, H, I, counts, k, more):
    """Every fourth column 2^more times the others, with 0 as its down weight: the others alone make the outputs."""
    c = Case(counts, H, I, k=k, seed=H + I + more)
    assert c.R * c.k <= 64
    for e in range(c.E):
        if more:
            scales(c, e, 1)[1::4] += more
            down_codes(c, e)[:, 0::2] &= 0x0f
    got = c.run(False)[:c.rows.numel()].double()
    want, tol, bf16 = reference(c, c.x)
    if more <= 10:
        assert bool((tol <= bf16).all())   # nowhere less than bf16 gives
    assert bool(((got - want).abs() <= tol).all()), \
        f'off by up to {((got - want).abs() / tol).max().item():.3g} of the bound'
    assert torch.equal(c.run(False, counts=False, max_rows=16)[:c.rows.numel()].double(), got)


@pytest.mark.parametrize('huge', [90, 126])
def test_an_infinite_column_stays_one(device, huge):
    """A column that overflows is an infinity: its neighbours keep their values, and the outputs where its weight is not
    0 are infinities of the weight's sign, as in a call of many pairs."""
    H, I, j = 256, 128, 5
    c = Case([2, 3], H, I, k=2, seed=3)
    few = torch.rand((c.R, H), generator=torch.Generator(device='cuda').manual_seed(1), device='cuda').to(torch.bfloat16)
    for e in range(c.E):      # gate and up: all products of column j are positive
        row = c.cache[int(c.slot_of[e])]
        for part in (0, 1):
            codes = row[part * H * I // 2:(part + 1) * H * I // 2].view(I, H // 2)
            codes[j] = 0x22   # ones
            scales(c, e, part)[j] = 127 + (4 if part == 0 else huge)
        down = down_codes(c, e)[:, j // 2]
        down.copy_((down & 0x0f) | torch.tensor([0x00, 0x20, 0xa0, 0x50], dtype=torch.uint8, device='cuda').repeat(H // 4))
    got = c.run(False, x=few)[:c.rows.numel()].float()
    # column j is 16 * 2^huge * sum(x)^2, sum(x) about 128: an infinity with 126, finite with 90
    if huge == 126:
        inf = float('inf')
        want = torch.tensor([float('nan'), inf, -inf, inf], device='cuda').repeat(H // 4).expand(got.shape)
        assert torch.equal(torch.nan_to_num(got, nan=7.0, posinf=8.0, neginf=9.0),
                           torch.nan_to_num(want, nan=7.0, posinf=8.0, neginf=9.0))
        m = Case([40, 40], H, I, k=2, seed=4)   # rows of the same kind in a call of many: bf16 between up and down
        m.cache, m.slot_of = c.cache, c.slot_of
        many = m.run(False, x=few[torch.arange(m.R, device='cuda') % c.R])[:m.rows.numel()].float()
        assert torch.equal(torch.nan_to_num(many, nan=7.0, posinf=8.0, neginf=9.0),
                           torch.nan_to_num(want[:1].expand(many.shape), nan=7.0, posinf=8.0, neginf=9.0))
    else:
        y, tol, _ = reference(c, few)
        assert bool(((got.double() - y).abs() <= tol).all())


def test_a_nan_reaches_every_output_of_its_row(device):
    H, I = 256, 128
    c = Case([2, 3], H, I, k=2, seed=5)
    want = c.run(False)
    for place in range(4):
        s = scales(c, 0, 1)
        keep = s[8 + place].clone()
        s[8 + place] = 255        # one up row: one column
        got = c.run(False)
        s[8 + place] = keep
        n = int(c.starts[1])
        assert bool(torch.isnan(got[:n]).all()) and torch.equal(got[n:], want[n:])
    assert torch.equal(c.run(False), want)


@pytest.mark.parametrize('scale', [2.0 ** -50, 2.0 ** -30, 2.0 ** 40])
def test_sizes_of_the_activations(device, scale):
    """Activations of 2^-100 or so up to 2^80."""
    c = Case([3, 8, 1], 256, 256, k=3, seed=7)
    x = (c.x.float() * scale).to(torch.bfloat16)
    got = c.run(False, x=x)[:c.rows.numel()].double()
    want, tol, _ = reference(c, x)
    assert bool(((got - want).abs() <= tol).all())
