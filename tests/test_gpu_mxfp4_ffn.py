"""mxfp4_expert_ffn against its formulas in 64 bits, at the row counts, sizes and layouts where the kernels
change their way of working."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def mx_values(x):
    """float64 values of the MXFP4 form of float64 rows (length a multiple of 32)."""
    b = x.reshape(-1, 32)
    amax = b.abs().amax(1, keepdim=True)
    e = (torch.frexp(amax)[1] - 3).clamp(-127, 127)
    e = torch.where(amax == 0, torch.full_like(e, -127), e)
    a = torch.ldexp(b, -e)
    step = torch.where(a.abs() < 2, 0.5, torch.where(a.abs() < 4, 1.0, 2.0)).double()
    return torch.ldexp((torch.round(a / step) * step).clamp(-6, 6), e).reshape(x.shape)


class Case:
    """Rows of every expert as given by counts, on random tokens (distinct experts for a token)."""

    def __init__(self, counts, H, I, R=None, k=None, seed=0, scale=0.05):
        g = torch.Generator(device='cuda').manual_seed(seed)
        rng = np.random.default_rng(seed)
        E = len(counts)
        self.counts, self.H, self.I, self.E = np.asarray(counts), H, I, E
        P = int(sum(counts))
        self.k = k = k or 3
        self.R = R = R or max(max(counts), -(-P // k), 1)
        # every token has k places; an expert takes a free place of distinct tokens
        free = np.zeros(R, np.int64)
        rows, cols = [], []
        for e in np.argsort(-self.counts, kind='stable'):
            order = np.lexsort((rng.random(R), free))[:counts[e]]
            rows.append((e, np.sort(order)))
            free[order] += 1
        assert free.max(initial=0) <= k
        rows = [r for _, r in sorted(rows, key=lambda t: t[0])]
        used = np.zeros(R, np.int64)
        for r in rows:
            cols.append(used[r].copy())
            used[r] += 1
        self.starts = torch.from_numpy(np.concatenate([[0], np.cumsum(counts)]).astype(np.int64)).cuda()
        self.rows = torch.from_numpy(np.concatenate(rows + [np.zeros(0, np.int64)]).astype(np.int64)).cuda()
        self.cols = torch.from_numpy(np.concatenate(cols + [np.zeros(0, np.int64)]).astype(np.int64)).cuda()
        self.slots = E + 2
        self.slot_of = rng.permutation(self.slots)[:E].astype(np.int32)
        from ferry_amd import expert_ops as ops
        w = (torch.randn((self.slots, 3 * H * I), generator=g, device='cuda') * scale).to(torch.bfloat16)
        self.cache = ops.mxfp4_expert_rows(w)
        self.x = torch.randn((R, H), generator=g, device='cuda').to(torch.bfloat16)
        self.w = (torch.rand((R, k), generator=g, device='cuda') + 0.2).to(torch.bfloat16)

    def weights(self, e):
        """float64 gate, up, down of an expert, from the cache bytes."""
        row = self.cache[int(self.slot_of[e])]
        n = 3 * self.H * self.I
        c = row[:n // 2].long()
        c = torch.stack([c & 15, c >> 4], 1).reshape(-1)
        table = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device='cuda')
        v = table[c & 7] * torch.where(c >= 8, -1.0, 1.0).double()
        m = v * torch.exp2(row[n // 2:].double() - 127).repeat_interleave(32)
        n = self.H * self.I
        return m[:n].view(self.I, self.H), m[n:2 * n].view(self.I, self.H), m[2 * n:].view(self.H, self.I)

    def reference(self, quantised, experts, x=None, fine=False):
        """(values, error bound) float64 [P, H] of the grouped rows; NaN rows for experts not in the list.  fine: the
        activations keep 13 bits of the largest of four columns."""
        P = self.rows.numel()
        out = torch.full((P, self.H), float('nan'), dtype=torch.float64, device='cuda')
        tol = torch.zeros_like(out)
        x = (self.x if x is None else x).double()
        if quantised:
            x = mx_values(x)
        for e in experts:
            lo, hi = int(self.starts[e]), int(self.starts[e + 1])
            r, c = self.rows[lo:hi], self.cols[lo:hi]
            wg, wu, wd = self.weights(e)
            xe = x[r]
            g, u = xe @ wg.t(), xe @ wu.t()
            a = g * torch.sigmoid(g) * u
            # |error| of a: fp32 sums of K exact products (K + 8 roundings of 2^-24 of the sum of magnitudes),
            # |d silu| <= 1.1 |dg|, and about 10 fp32 roundings of the SwiGLU
            eps = 2.0 ** -24
            dg = (self.H + 8) * eps * (xe.abs() @ wg.abs().t())
            du = (self.H + 8) * eps * (xe.abs() @ wu.abs().t())
            silu = (g * torch.sigmoid(g)).abs()
            da = 1.1 * dg * u.abs() + silu * du + dg * du + 16 * eps * a.abs()
            if quantised:
                b, d = a.reshape(-1, 32), da.reshape(-1, 32)
                av = mx_values(a)
                # an error can move an element by at most one step past a border that it is near, and
                # the whole block by a factor of two of its scale where the largest magnitude is near a power
                # of two
                amax, worst = b.abs().amax(1, keepdim=True), d.amax(1, keepdim=True)
                top = torch.exp2(torch.frexp(amax)[1].double() - 1)
                flips = ((amax - top < worst) | (2 * top - amax < worst)).expand_as(b)
                step = top / 4
                y = (b / step).abs()
                near = torch.zeros_like(b, dtype=torch.bool)
                for m in (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0):
                    near |= (y - m).abs() <= d / step
                da = torch.where(near | flips, 2 * top, torch.zeros_like(b)).reshape(a.shape)
                a = av
            elif fine:   # steps of 2^-12 of the largest's power of two, at most 2^-12 of it; the largest can be 8191 of 8192
                most = (a.abs() + da).reshape(-1, 4).amax(1, keepdim=True).expand(-1, 4).reshape(a.shape)
                da = da + 2.0 ** -13 * most
            else:
                da = da + 2.0 ** -8 * (a.abs() + da)   # the operand's rounding to bf16
            y = a @ wd.t()
            wt = self.w[r, c].double()[:, None]
            dy = da @ wd.abs().t() + (self.I + 8) * eps * ((a.abs() + da) @ wd.abs().t())
            out[lo:hi] = y * wt
            tol[lo:hi] = dy * wt + 2.0 ** -8 * ((y * wt).abs() + dy * wt) + 4 * eps * (y * wt).abs() + 1e-30
        return out, tol

    def run(self, quantised, experts=None, out_mode=1, counts=True, phases=(3,), x=None, out=None, **kw):
        from ferry_amd import expert_ops as ops
        P = self.R * self.k
        act = (torch.full((P * (self.I // 32 * 17),), 0xEE, dtype=torch.uint8, device='cuda') if quantised else
               torch.full((P, self.I), 9.0, dtype=torch.bfloat16, device='cuda'))
        if out is None:
            out = torch.full((P, self.H), 7.0, dtype=torch.bfloat16, device='cuda')
        x = self.x if x is None else x
        if quantised:
            x = ops.mxfp4_quantize(x)
        experts = np.arange(self.E) if experts is None else experts
        for ph in phases:
            ops.mxfp4_expert_ffn(self.cache, x, self.w, self.starts, self.rows, self.cols, experts, self.slot_of,
                                 self.H, self.I, act, out, out_mode=out_mode, phases=ph,
                                 counts=self.counts if counts else None, **kw)
        return out

    def check(self, quantised, experts=None, out_mode=1, fine=False, **kw):
        out = self.run(quantised, experts, out_mode, **kw)
        experts = range(self.E) if experts is None else experts
        want, tol = self.reference(quantised, experts, kw.get('x'), fine)
        n = self.rows.numel()
        at = self.rows * self.k + self.cols if out_mode == 0 else torch.arange(n, device='cuda')
        live = ~torch.isnan(want[:, 0])
        got = out[at].double()
        assert bool((got[live] - want[live]).abs().le(tol[live]).all()), \
            f'off by up to {((got[live] - want[live]).abs() / tol[live]).max().item():.3g} of the bound'
        rest = torch.ones(out.shape[0], dtype=torch.bool, device='cuda')
        rest[at[live]] = False
        assert bool((out[rest] == 7).all())
        return out


QUANTISED = [False, True]


@pytest.mark.parametrize('quantised', QUANTISED)
@pytest.mark.parametrize('H,I,counts', [
    (128, 128, [1]), (256, 128, [16, 0, 1, 7]), (384, 640, [2, 3, 16]), (2048, 768, [1, 2, 1, 5]),
    (1024, 1408, [4, 9]), (128, 2816, [3, 15, 0])])
def test_few_rows(device, H, I, counts, quantised):
    c = Case(counts, H, I, seed=H + I)
    c.check(quantised)
    c.check(quantised, out_mode=0)


@pytest.mark.parametrize('quantised', QUANTISED)
@pytest.mark.parametrize('H,I,counts', [
    (256, 128, [17]), (256, 256, [64, 65, 0, 16, 33]), (512, 384, [255, 256, 257, 1]),
    (2048, 768, [300, 40, 3]), (768, 1408, [128, 129, 500]), (256, 128, [1023, 31, 18, 5, 0, 700])])
def test_many_rows(device, H, I, counts, quantised):
    c = Case(counts, H, I, seed=H + I)
    c.check(quantised)
    c.check(quantised, out_mode=0)


@pytest.mark.parametrize('H,I,counts,k', [(2048, 768, [1] * 8, 8), (512, 2816, [8, 5, 1, 0, 8], 4), (128, 128, [1], 1),
                                          (384, 640, [2, 3, 7, 8, 1], 8), (2048, 4352, [3, 1], 2)])
@pytest.mark.parametrize('scale', [1.0, 2.0 ** -40, 2.0 ** 25])
def test_few_pairs_keep_more_than_bf16(device, H, I, counts, k, scale):
    c = Case(counts, H, I, k=k, seed=H + I)
    assert c.R * c.k <= 64
    x = (c.x.float() * scale).to(torch.bfloat16)
    c.check(False, x=x, fine=True)
    c.check(False, x=x, fine=True, out_mode=0, counts=False, max_rows=16)


@pytest.mark.parametrize('quantised', QUANTISED)
@pytest.mark.parametrize('H,I,more', [(4224, 2944, []), (4352, 2816, [40, 130])])
def test_many_small_experts_with_long_rows(device, H, I, more, quantised):
    """Several groups of weight rows a workgroup, rows of more units than it holds; alone and behind tiles."""
    c = Case([int(v) for v in np.random.default_rng(1).integers(0, 17, 40)] + more, H, I, k=8, seed=11, scale=0.02)
    whole = c.check(quantised)
    out = torch.full_like(whole, 7.0)
    for e in range(0, c.E, 3):
        c.run(quantised, [e], out=out)
        at = slice(int(c.starts[e]), int(c.starts[e + 1]))
        assert torch.equal(out[at], whole[at])


@pytest.mark.parametrize('quantised', QUANTISED)
@pytest.mark.parametrize('counts', [[1380, 17, 720, 1224, 90, 1046, 562, 0, 276, 129, 3],
                                    [3380, 17, 1720, 2224, 90, 3046, 562, 0, 1276, 129, 3, 200]])
def test_more_tiles_than_workgroups(device, counts, quantised):
    """Tiles of every size, several to a workgroup, with every count of rows that they are cut to; an expert by itself
    runs in smaller ones and gives the same bits."""
    c = Case(counts, 2048, 1024, seed=5)
    whole = c.check(quantised)
    out = torch.full_like(whole, 7.0)
    for e in range(c.E):
        c.run(quantised, [e], out=out)
    assert torch.equal(out, whole)
    assert torch.equal(c.run(quantised, spare_cus=100), whole)
    assert torch.equal(c.run(quantised, counts=False), whole)


@pytest.mark.parametrize('quantised', QUANTISED)
def test_forms_of_a_call_give_the_same_bits(device, quantised):
    """Without row counts, phase by phase, on parts of the list, with spare CUs."""
    c = Case([3, 0, 70, 16, 17, 300, 1], 512, 256, seed=4)
    whole = c.check(quantised)
    assert torch.equal(c.run(quantised, counts=False), whole)
    assert torch.equal(c.run(quantised, phases=(1, 2)), whole)
    assert torch.equal(c.run(quantised, phases=(1, 2), counts=False), whole)
    assert torch.equal(c.run(quantised, spare_cus=100), whole)
    out = c.run(quantised, experts=[5, 0, 6])
    out = c.run(quantised, experts=[4, 3, 2, 1], out=out)
    assert torch.equal(out, whole)
    c.check(quantised, experts=[2, 6])
    c.check(quantised, experts=[])


@pytest.mark.parametrize('quantised', QUANTISED)
def test_many_experts(device, quantised):
    rng = np.random.default_rng(3)
    c = Case(list(rng.integers(0, 40, 300)), 256, 128, k=8, seed=5)
    whole = c.check(quantised)
    assert torch.equal(c.run(quantised, counts=False), whole)


@pytest.mark.parametrize('quantised', QUANTISED)
def test_no_rows(device, quantised):
    c = Case([0, 0], 256, 128, R=5)
    assert bool((c.run(quantised) == 7).all()) and bool((c.run(quantised, counts=False) == 7).all())


@pytest.mark.parametrize('quantised', QUANTISED)
def test_special_rows(device, quantised):
    """A token with an infinity or a NaN changes its own rows only; zero rows give zeros."""
    c = Case([40, 9], 256, 128, k=2, seed=6)
    want = c.run(quantised)
    x = c.x.clone()
    x[0, 3] = float('inf')
    x[1, 5] = float('nan')
    x[2] = 0
    got = c.run(quantised, x=x)
    tok = c.rows
    n = tok.numel()
    other = torch.ones(got.shape[0], dtype=torch.bool, device='cuda')
    other[:n] = tok >= 3
    assert torch.equal(got[other], want[other])
    assert bool(torch.isnan(got[:n][tok == 1]).all())
    assert not bool(torch.isfinite(got[:n][tok == 0]).any()) or not quantised
    assert bool((got[:n][tok == 2] == 0).all())


def test_special_rows_of_few_pairs(device):
    c = Case([4, 2], 256, 128, k=2, seed=6)
    x = c.x.clone()
    want = c.run(False)
    x[0, 3] = float('inf')
    x[1, 5] = float('nan')
    x[2] = 0
    got = c.run(False, x=x)
    n, tok = c.rows.numel(), c.rows
    assert torch.equal(got[:n][tok == 3], want[:n][tok == 3]) and bool((got[n:] == 7).all())
    assert bool(torch.isnan(got[:n][tok == 1]).all()) and not bool(torch.isfinite(got[:n][tok == 0]).any())
    assert bool((got[:n][tok == 2] == 0).all())


@pytest.mark.parametrize('quantised', QUANTISED)
def test_scale_bytes_at_the_ends(device, quantised):
    """Weight blocks with the smallest scale, and an expert row with a NaN scale."""
    c = Case([5, 20], 256, 128, k=2, seed=8)
    n = 3 * 256 * 128
    s0, s1 = int(c.slot_of[0]), int(c.slot_of[1])
    c.cache[s0, n // 2:n // 2 + 8] = 0           # the first gate row: 2^-127
    c.cache[s1, n // 2 + 3] = 0
    c.check(quantised)
    c.cache[s0, n // 2 + 256 * 128 // 32 * 2] = 255   # a NaN in the first down row
    got = c.run(quantised)
    assert bool(torch.isnan(got[:5, 0]).all()) and bool(torch.isfinite(got[:5, 1:]).all())
    assert bool(torch.isfinite(got[5:25]).all())


@pytest.mark.parametrize('quantised', QUANTISED)
def test_graph_replays(device, quantised):
    from ferry_amd import expert_ops as ops
    c = Case([3, 90, 1, 25], 512, 256, seed=9)
    act = (torch.zeros(c.R * c.k * (c.I // 32 * 17), dtype=torch.uint8, device='cuda') if quantised else
           torch.zeros((c.R * c.k, c.I), dtype=torch.bfloat16, device='cuda'))
    out = torch.zeros((c.R * c.k, c.H), dtype=torch.bfloat16, device='cuda')
    x = c.x.clone()

    def call():
        xin = ops.mxfp4_quantize(x) if quantised else x
        return ops.mxfp4_expert_ffn(c.cache, xin, c.w, c.starts, c.rows, c.cols, np.arange(c.E), c.slot_of, c.H,
                                    c.I, act, out, out_mode=1, counts=c.counts)
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for seed in range(4):
        x.copy_(torch.randn(x.shape, generator=torch.Generator(device='cuda').manual_seed(seed), device='cuda'))
        want = c.run(quantised, x=x)[:c.rows.numel()]
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[:c.rows.numel()], want)


def test_two_streams(device):
    c = Case([3, 90, 1, 25], 512, 256, seed=10)
    want = [c.run(q) for q in QUANTISED]
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for s, q in ((s1, False), (s2, True)):
        with torch.cuda.stream(s):
            for _ in range(3):
                got.append((q, c.run(q)))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[q]) for q, o in got)


def test_gate_to_combine(device):
    """The operators as a layer uses them: a sigmoid gate with groups, layout, MXFP4 experts, combine."""
    from ferry_amd import expert_ops as ops
    E, k, H, I, T = 32, 4, 512, 256, 100
    g = torch.Generator(device='cuda').manual_seed(1)
    x = torch.randn((T, H), generator=g, device='cuda').to(torch.bfloat16)
    gate = (torch.randn((E, H), generator=g, device='cuda') * 0.05).to(torch.bfloat16)
    pool = (torch.randn((E, 3 * H * I), generator=g, device='cuda') * 0.05).to(torch.bfloat16)
    bias = torch.randn(E, generator=g, device='cuda') * 0.1
    w, sel = ops.route_experts(ops.gate_logits(x, gate), k, scoring='sigmoid', bias=bias, groups=4, topk_groups=2,
                               group_score='top2', scale=2.5)
    lay = ops.layout(sel, w, E, check=True)
    cache = ops.mxfp4_expert_rows(pool)
    counts = np.diff(lay.starts.cpu().numpy())
    act = torch.empty((T * k, I), dtype=torch.bfloat16, device='cuda')
    part = torch.empty((T * k, H), dtype=torch.bfloat16, device='cuda')
    ops.mxfp4_expert_ffn(cache, x, lay.w_sorted, lay.starts, lay.rows, lay.cols, np.flatnonzero(counts),
                         np.arange(E), H, I, act, part, counts=counts)
    out = ops.combine(part, T, k, H)
    # the bf16 experts on the rows' values: the same layer, but for bf16 roundings of g, u and y
    deq = ops.mxfp4_dequantize(cache[:, :3 * H * I // 2], cache[:, 3 * H * I // 2:])
    ref = torch.zeros((T, H), dtype=torch.float64, device='cuda')
    for t in range(T):
        for j in range(k):
            e = int(sel[t, j])
            m = deq[e].double()
            wg, wu, wd = (m[i * H * I:(i + 1) * H * I] for i in range(3))
            xe = x[t].double()
            gt, u = wg.view(I, H) @ xe, wu.view(I, H) @ xe
            ref[t] += (wd.view(H, I) @ (gt * torch.sigmoid(gt) * u)) * w[t, j].double()
    # three bf16 roundings of half a step (operand, part, sum), as a share of the row's size
    err = (out.double() - ref).norm(dim=1) / ref.norm(dim=1)
    assert err.max().item() < 3 * 2.0 ** -8


@pytest.mark.parametrize('quantised', QUANTISED)
def test_an_expert_listed_twice(device, quantised):
    c = Case([5, 40, 0, 17], 256, 384, seed=9)
    assert torch.equal(c.run(quantised, [1, 0, 3, 1, 0]), c.run(quantised))


@pytest.mark.parametrize('quantised', QUANTISED)
def test_slots_past_4_gib(device, quantised):
    c = Case([4, 60, 130], 2048, 768, seed=10)
    want = c.run(quantised)
    cache = torch.zeros((2000, c.cache.shape[1]), dtype=torch.uint8, device='cuda')   # 5 GB
    slots = np.array([1997, 1999, 1800], np.int32)
    for e in range(c.E):
        cache[int(slots[e])] = c.cache[int(c.slot_of[e])]
    c.cache, c.slot_of = cache, slots
    assert torch.equal(c.run(quantised), want)


@pytest.mark.parametrize('quantised', QUANTISED)
def test_fetched_experts(device, quantised):
    """MXFP4 rows in a pinned pool, fetched into fewer cache slots than experts while the resident ones run."""
    from ferry_amd import expert_ops as ops
    c = Case([5, 40, 0, 16, 200, 3, 30, 9], 256, 384, seed=8)
    want = c.run(quantised, out_mode=0)
    pool = torch.empty((c.E, c.cache.shape[1]), dtype=torch.uint8, pin_memory=True)
    pool.copy_(c.cache[torch.from_numpy(c.slot_of.astype(np.int64)).cuda()])
    cache = torch.zeros((5, c.cache.shape[1]), dtype=torch.uint8, device='cuda')
    torch.cuda.synchronize()   # the engine's streams do not wait for this one's work on the cache
    x = ops.mxfp4_quantize(c.x) if quantised else c.x
    P = c.R * c.k
    act = (torch.empty(P * (c.I // 32 * 17), dtype=torch.uint8, device='cuda') if quantised else
           torch.empty((P, c.I), dtype=torch.bfloat16, device='cuda'))
    out = torch.full((P, c.H), 7.0, dtype=torch.bfloat16, device='cuda')
    eng = ops.H2DEngine(cache, pool)
    slot_of = np.full(c.E, -1, np.int32)

    def fetch(slots, experts):
        eng.fetch(slots, experts)
        slot_of[np.isin(slot_of, slots)] = -1
        slot_of[experts] = slots

    def run(experts):
        eng.wait_stream(slot_of[experts])
        ops.mxfp4_expert_ffn(cache, x, c.w, c.starts, c.rows, c.cols, experts, slot_of, c.H, c.I, act, out,
                             counts=c.counts)
        eng.mark_used(slot_of[experts])
    fetch([0, 1, 2], [0, 1, 3])
    fetch([3, 4], [4, 5])
    run([0, 1, 3])
    fetch([1, 2], [6, 7])
    run([4, 5])
    run([6, 7])
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    with pytest.raises(RuntimeError, match='not cached'):
        ops.mxfp4_expert_ffn(cache, x, c.w, c.starts, c.rows, c.cols, [1], slot_of, c.H, c.I, act, out, counts=c.counts)


def test_refusals(device):
    from ferry_amd import expert_ops as ops
    c = Case([3, 20], 256, 128, k=2)
    act = torch.zeros((c.R * c.k, c.I), dtype=torch.bfloat16, device='cuda')
    out = torch.zeros((c.R * c.k, c.H), dtype=torch.bfloat16, device='cuda')
    good = dict(cache=c.cache, x=c.x, w_sorted=c.w, starts=c.starts, rows=c.rows, cols=c.cols, expert_list=[0, 1],
                slot_of=c.slot_of, hidden=256, intermediate=128, act=act, out=out, counts=c.counts)
    ops.mxfp4_expert_ffn(**good)
    q = ops.mxfp4_quantize(c.x)
    for bad in (dict(cache=c.cache.to(torch.int8)), dict(cache=c.cache[:, :-1].contiguous()), dict(x=c.x.float()),
                dict(x=c.x[:-1]), dict(x=c.x.t().contiguous().t()), dict(x=q), dict(x=(q[0], q[1][:, :-1])),
                dict(x=(q[0].cpu(), q[1])), dict(hidden=128), dict(hidden=192, intermediate=128),
                dict(expert_list=[0, 2]), dict(expert_list=[-1]), dict(slot_of=np.array([0, 4], np.int32)),
                dict(slot_of=np.array([0], np.int32), experts=2), dict(act=act[:-1]), dict(out=out[:-1]),
                dict(act=act.float()), dict(out=out.cpu()), dict(starts=c.starts[:-1]), dict(rows=c.rows.int()),
                dict(w_sorted=c.w.float()), dict(out_mode=2), dict(phases=0), dict(spare_cus=-1),
                dict(spare_cus=129)):
        with pytest.raises(RuntimeError):
            ops.mxfp4_expert_ffn(**{**good, **bad})
    h = Case([3, 20], 384, 128, k=2)      # tiles cover the hidden dimension in 256 columns
    with pytest.raises(RuntimeError, match='256'):
        h.run(False)


@pytest.mark.parametrize('quantised', QUANTISED)
def test_index_lists_that_are_too_short(device, quantised):
    """Row and slot lists that end before the pairs of the call do are refused, and counts that name more pairs than there
    are output rows; longer lists are not."""
    from ferry_amd import expert_ops as ops
    c = Case([3, 20, 0], 256, 128, k=2)
    P = c.R * c.k
    x = ops.mxfp4_quantize(c.x) if quantised else c.x
    act = (torch.zeros(P * (c.I // 32 * 17), dtype=torch.uint8, device='cuda') if quantised else
           torch.zeros((P, c.I), dtype=torch.bfloat16, device='cuda'))

    def call(**other):
        out = torch.full((P, c.H), 7.0, dtype=torch.bfloat16, device='cuda')
        args = dict(cache=c.cache, x=x, w_sorted=c.w, starts=c.starts, rows=c.rows, cols=c.cols, expert_list=[0, 1],
                    slot_of=c.slot_of, hidden=256, intermediate=128, act=act, out=out, counts=c.counts, out_mode=1)
        return ops.mxfp4_expert_ffn(**{**args, **other})
    want = call()
    none = torch.zeros(0, dtype=torch.int64, device='cuda')
    for bad in (dict(cols=c.cols[:-1]), dict(rows=c.rows[:-1]), dict(rows=c.rows[:-1], cols=c.cols[:-1]),
                dict(rows=none, cols=none), dict(cols=none), dict(cols=c.cols[:-1], counts=None),
                dict(rows=none, counts=None), dict(rows=c.rows.data_ptr(), cols=c.cols[:-1]),
                dict(rows=c.rows[:-1], cols=c.cols.data_ptr()), dict(counts=[3, P - 2, 0]),
                dict(counts=[3, 20, 18], expert_list=[0])):
        with pytest.raises(RuntimeError, match='rows'):
            call(**bad)
    usual = [torch.cat([t, t[:P - t.numel()]]) for t in (c.rows, c.cols)]   # an entry for every output row
    with pytest.raises(RuntimeError, match='rows'):
        call(rows=usual[0], cols=usual[1], counts=[3, P - 2, 0])
    longer = torch.cat([c.rows, c.rows]), torch.cat([c.cols, c.cols])
    for good in (dict(counts=list(c.counts)), dict(rows=usual[0], cols=usual[1]), dict(rows=longer[0], cols=longer[1]), dict(counts=None),
                 dict(rows=c.rows.data_ptr(), cols=c.cols.data_ptr()), dict(counts=[3, 20, 0, 1000], experts=3),
                 dict(expert_list=[0, 1, 1, 0, 1])):   # 66 pairs if each time counted
        assert torch.equal(call(**good), want)
    out = call(rows=none, cols=none, counts=[0, 0, 0], expert_list=[0, 1])
    assert bool((out == 7).all())


@pytest.mark.parametrize('H,I', [(2048, 1408), (2048, 128), (2048, 256), (256, 2816)])
def test_largest_tiles(device, H, I):
    """4-bit activations with rows enough for tiles of 256 x 256: odd numbers of 128 along K (I = 1408, 128: the last step is
    half a one), one step in all (I = 128 and 256 down, H = 256 up), and small experts behind them."""
    counts = [4000, 17, 3300, 3, 12, 2900, 250, 0, 16, 129, 1800, 65, 1, 180]
    c = Case(counts, H, I, seed=H + I)
    tiles = sum(-(-n // 64) for n in counts if n > 16)
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    assert tiles * max(I // 128 if H == 256 else 0, H // 256) >= 6 * cus   # the rule for these tiles, of the product meant
    whole = c.check(True)
    out = torch.full_like(whole, 7.0)
    for e in range(c.E):      # each by itself: in the smaller tiles
        c.run(True, [e], out=out)
    assert torch.equal(out, whole)
    assert torch.equal(c.run(True, counts=False), whole)


@pytest.mark.parametrize('counts', [[40, 9], [300, 2], [40, 30, 70, 17]])
def test_infinite_rows_of_bf16_activations(device, counts):
    """An infinity in a token's row makes all of that token's outputs infinities or NaNs, in every kernel, and no others."""
    c = Case(counts, 256, 128, k=2, seed=6)
    want = c.run(False)
    for column in (0, 3, 255):
        x = c.x.clone()
        x[0, column] = float('inf')
        x[5, column] = -float('inf')
        got = c.run(False, x=x)
        n = c.rows.numel()
        hit = (c.rows == 0) | (c.rows == 5)
        assert bool(hit.any()) and not bool(torch.isfinite(got[:n][hit]).any())
        assert torch.equal(got[:n][~hit], want[:n][~hit]) and bool((got[n:] == 7).all())
