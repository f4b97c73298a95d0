"""The operators for MXFP4 experts and general expert gates: what is timed, and their plain forms.

Kinds (`case["kind"]`):
  route     route_experts: scores (softmax or sigmoid), balance bias, expert groups, top-k, weights
  quantize  mxfp4_quantize and mxfp4_dequantize: rows to 4-bit elements with a scale per 32, and back
  ffn       mxfp4_expert_ffn on bf16 activations: the grouped SwiGLU experts of one layer call
  ffnq      mxfp4_quantize of the hidden rows, then mxfp4_expert_ffn on them: 4-bit activations too

Shapes are the two models this package evaluates (Qwen3-30B-A3B: hidden 2048, 128 experts of
intermediate 768, top 8; DeepSeek-V2-Lite: hidden 2048, 64 experts of intermediate 1408, top 6) and
generic gates of up to 512 experts.  Expert popularity is Zipf over a seeded permutation: in a prefill
the largest expert gets thousands of rows and many get fewer than 64.
"""
import math

import numpy as np
import torch

own = False

# hidden, intermediate, experts, top-k, Zipf exponent of the experts' popularity
MODELS = {'qwen3': (2048, 768, 128, 8, 1.1), 'deepseek': (2048, 1408, 64, 6, 0.9)}
DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}


def _ffn_case(name, kind, model, tokens):
    h, i, e, k, z = MODELS[model]
    return dict(name=name, kind=kind, tokens=tokens, hidden=h, inter=i, experts=e, topk=k, zipf=z)


def listed():
    return [
        # one token through a sigmoid gate of 8 groups with a balance bias: pure latency
        dict(name='route_sigmoid_t1', kind='route', tokens=1, experts=256, topk=8, groups=8,
             topk_groups=4, group_score='top2', scoring='sigmoid', bias=True, renorm=True, scale=2.5,
             dtype='fp32'),
        # a ragged prompt through a softmax gate whose groups are scored by their best expert
        dict(name='route_softmax_t777', kind='route', tokens=777, experts=160, topk=6, groups=8,
             topk_groups=3, group_score='max', scoring='softmax', bias=False, renorm=False, scale=16.0,
             dtype='bf16'),
        # a large prefill batch through the sigmoid gate
        dict(name='route_sigmoid_t32768', kind='route', tokens=32768, experts=256, topk=8, groups=8,
             topk_groups=4, group_score='top2', scoring='sigmoid', bias=True, renorm=True, scale=2.5,
             dtype='fp32'),
        # the hidden rows of one decode step of 16 requests
        dict(name='quantize_t16', kind='quantize', rows=16, cols=2048, dtype='bf16'),
        # fp32 rows whose length is no multiple of a block: the last block of each is partial
        dict(name='quantize_ragged', kind='quantize', rows=7777, cols=1001, dtype='fp32'),
        # a layer's expert rows, as a program quantises a bf16 pool once
        dict(name='quantize_experts', kind='quantize', rows=128, cols=3 * 2048 * 768, dtype='bf16'),
        # one request's decode step: 8 experts of one row
        _ffn_case('ffn_qwen3_t1', 'ffn', 'qwen3', 1),
        # a decode step of 16 requests, the weights of some 40 experts
        _ffn_case('ffn_qwen3_t16', 'ffn', 'qwen3', 16),
        # one prompt of ordinary, ragged length
        _ffn_case('ffn_deepseek_t777', 'ffn', 'deepseek', 777),
        # the Qwen3 prefill batch
        _ffn_case('ffn_qwen3_t8192', 'ffn', 'qwen3', 8192),
        # a short prompt with 4-bit activations
        _ffn_case('ffnq_deepseek_t256', 'ffnq', 'deepseek', 256),
        # the Qwen3 prefill batch with 4-bit activations
        _ffn_case('ffnq_qwen3_t8192', 'ffnq', 'qwen3', 8192),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(['route', 'route', 'quantize', 'quantize', 'ffn', 'ffn', 'ffn', 'ffnq', 'ffnq'])
    if kind == 'route':
        groups = rng.choice([1, 1, 4, 8, rng.randint(2, 16)])
        size = rng.randint(2, 512 // groups)
        topk_groups = rng.randint(1, groups)
        scoring = rng.choice(['softmax', 'sigmoid'])
        experts = groups * size
        return dict(kind=kind, tokens=_log_uniform(rng, 1, 32768), experts=experts,
                    topk=rng.randint(1, min(16, topk_groups * size)), groups=groups,
                    topk_groups=topk_groups, group_score=rng.choice(['max', 'top2']), scoring=scoring,
                    bias=rng.random() < 0.5, renorm=rng.random() < 0.6,
                    scale=rng.choice([1.0, 2.5, 16.0]), dtype=rng.choice(['fp32', 'bf16', 'fp16']))
    if kind == 'quantize':
        cols = _log_uniform(rng, 1, 20000)
        rows = _log_uniform(rng, 1, 3e8 / cols)
        return dict(kind=kind, rows=rows, cols=cols, dtype=rng.choice(['bf16', 'fp16', 'fp32']))
    while True:
        hidden, inter = 256 * rng.randint(1, 16), 128 * rng.randint(1, 16)
        experts = _log_uniform(rng, 2, 128)
        topk = rng.randint(1, min(8, experts))
        if rng.random() < 0.4:   # one of the two models
            hidden, inter, experts, topk, _ = MODELS[rng.choice(sorted(MODELS))]
        tokens = _log_uniform(rng, 1, 8192)
        if (tokens * topk * hidden * inter <= 8192 * 8 * 2048 * 768
                and experts * hidden * inter <= 128 * 2048 * 768):
            return dict(kind=kind, tokens=tokens, hidden=hidden, inter=inter, experts=experts,
                        topk=topk, zipf=round(rng.uniform(0.0, 1.2), 2))


# -- inputs -------------------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device='cuda')
    g.manual_seed(seed)
    return g


def _routing(case, seed):
    """Distinct experts of every token, ascending, int64 [tokens, topk]: the top-k of N(0, 1) plus the
    experts' log popularity."""
    rng = np.random.default_rng(seed)
    T, E, k = case['tokens'], case['experts'], case['topk']
    pop = -case['zipf'] * np.log(1.0 + rng.permutation(E))
    z = rng.standard_normal((T, E), dtype=np.float32) + pop.astype(np.float32)
    return np.sort(np.argpartition(-z, k - 1, axis=1)[:, :k], axis=1).astype(np.int64)


# the values of the 16 codes of a 4-bit element: sign, two exponent bits, one mantissa bit
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def _quantize(x):
    """(codes [n, blocks, 16] uint8, scales [n, blocks] uint8) of fp32 or fp64 rows [n, cols]."""
    n, cols = x.shape
    blocks = -(-cols // 32)
    if cols % 32:
        x = torch.cat([x, x.new_zeros(n, blocks * 32 - cols)], 1)
    x = x.reshape(n, blocks, 32)
    amax = x.abs().amax(-1)
    # frexp: amax = m * 2^e with m in [0.5, 1), so floor(log2(amax)) = e - 1
    e = (torch.frexp(amax)[1] - 3).clamp(-127, 127)
    e = torch.where(amax == 0, torch.full_like(e, -127), e)
    y = torch.ldexp(x, -e[..., None])
    a = y.abs()
    # nearest value, ties to the even code; above 5 everything is 6
    code = (a > 0.25).to(torch.uint8)
    code += a >= 0.75
    code += a > 1.25
    code += a >= 1.75
    code += a > 2.5
    code += a >= 3.5
    code += a > 5.0
    code |= torch.signbit(y).to(torch.uint8) << 3
    scales = (e + 127).to(torch.uint8)
    scales = torch.where(torch.isfinite(amax), scales, torch.full_like(scales, 255))
    return code[..., 0::2] | (code[..., 1::2] << 4), scales


def _values(codes, scales, dtype=torch.float32):
    """The values of codes [n, blocks, 16] with scales [n, blocks], [n, blocks * 32]."""
    table = torch.tensor(E2M1, dtype=dtype, device=codes.device)
    nib = torch.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:2], 32)
    s = torch.ldexp(torch.ones((), dtype=dtype, device=codes.device), scales.to(torch.int32) - 127)
    s = torch.where(scales == 255, torch.full_like(s, math.nan), s)
    return (table[nib.long()] * s[..., None]).reshape(codes.shape[0], -1)


def _expert_rows(case, g):
    """MXFP4 cache rows uint8 [experts, 3 H I * 17 / 32]: each expert's codes of [gate | up | down], then
    its scales; from N(0, 0.02) weights, a few experts at a time to bound the memory."""
    n = 3 * case['hidden'] * case['inter']
    rows = torch.empty((case['experts'], n // 32 * 17), dtype=torch.uint8, device='cuda')
    step = max(1, (1 << 27) // n)
    for lo in range(0, case['experts'], step):
        hi = min(lo + step, case['experts'])
        w = torch.randn((hi - lo, n), generator=g, device='cuda') * 0.02
        codes, scales = _quantize(w.to(torch.bfloat16).float())
        rows[lo:hi, :n // 2] = codes.reshape(hi - lo, -1)
        rows[lo:hi, n // 2:] = scales
    return rows


def prepare(case, seed):
    g = _gen(seed)
    if case['kind'] == 'route':
        T, E = case['tokens'], case['experts']
        logits = torch.randn((T, E), generator=g, device='cuda') * 1.5
        bias = torch.randn(E, generator=g, device='cuda') * 0.1 if case['bias'] else None
        return dict(case=case, logits=logits.to(DTYPES[case['dtype']]), bias=bias)
    if case['kind'] == 'quantize':
        n, cols = case['rows'], case['cols']
        x = torch.empty((n, cols), dtype=DTYPES[case['dtype']], device='cuda')
        step = max(1, (1 << 28) // cols)
        for lo in range(0, n, step):   # rows of different sizes, from the first to the last 4 binades
            r = torch.randn((min(step, n - lo), cols), generator=g, device='cuda')
            x[lo:lo + step] = r * torch.exp2(4 * torch.rand((r.shape[0], 1), generator=g, device='cuda') - 7)
        return dict(case=case, x=x)
    T, E, k = case['tokens'], case['experts'], case['topk']
    H, I = case['hidden'], case['inter']
    ids = _routing(case, seed)
    order = np.argsort(ids.reshape(-1), kind='stable')
    counts = np.bincount(ids.reshape(-1), minlength=E)
    starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int64)
    x = torch.randn((T, H), generator=g, device='cuda')
    w = torch.rand((T, k), generator=g, device='cuda') + 0.1
    slot_of = np.random.default_rng(seed + 1).permutation(E).astype(np.int32)
    act = (torch.empty((T * k, I), dtype=torch.bfloat16, device='cuda') if case['kind'] == 'ffn' else
           torch.empty((T * k, I // 32 * 17), dtype=torch.uint8, device='cuda'))
    return dict(case=case, cache=_expert_rows(case, g), x=x.to(torch.bfloat16),
                w=(w / w.sum(1, keepdim=True)).to(torch.bfloat16),
                starts=torch.from_numpy(starts).cuda(), rows=torch.from_numpy(order // k).cuda(),
                cols=torch.from_numpy(order % k).cuda(), experts=np.flatnonzero(counts).astype(np.int32),
                slot_of=slot_of, counts=counts, act=act,
                out=torch.empty((T * k, H), dtype=torch.bfloat16, device='cuda'))


# -- one pass -----------------------------------------------------------------------------------

def _plain_route(s):
    c = s['case']
    T, E, G, k = c['tokens'], c['experts'], c['groups'], c['topk']
    # 64 bits: two experts' scores may lie next to each other
    x = s['logits'].double()
    if c['scoring'] == 'softmax':
        p = torch.exp(x - x.amax(1, keepdim=True))
        p = p / p.sum(1, keepdim=True)
    else:
        p = 1 / (1 + torch.exp(-x))
    choice = p + s['bias'].double() if c['bias'] else p
    if G > 1:
        per = choice.view(T, G, E // G)
        top = torch.sort(per, dim=2, descending=True)[0]
        score = top[..., 0] if c['group_score'] == 'max' else top[..., :2].sum(2)
        best = torch.sort(score, dim=1, descending=True, stable=True)[1][:, :c['topk_groups']]
        keep = torch.zeros((T, G), dtype=torch.bool, device=x.device).scatter_(1, best, True)
        choice = per.masked_fill(~keep[..., None], -math.inf).view(T, E)
    ids = torch.sort(choice, dim=1, descending=True, stable=True)[1][:, :k].contiguous()
    w = p.gather(1, ids)
    if c['renorm']:
        w = w / w.sum(1, keepdim=True)
    return (w * c['scale']).to(torch.bfloat16), ids


def _plain_ffn(s):
    c = s['case']
    H, I, k = c['hidden'], c['inter'], c['topk']
    n = 3 * H * I
    x, out = s['x'].float(), s['out']
    quantised = c['kind'] == 'ffnq'
    if quantised:
        x = _values(*_quantize(x))
    starts = np.concatenate([[0], np.cumsum(s['counts'])])
    at = s['rows'] * k + s['cols']
    # one product per expert: their row counts differ
    for e in s['experts']:
        lo, hi = int(starts[e]), int(starts[e + 1])
        row = s['cache'][int(s['slot_of'][e])]
        m = _values(row[:n // 2].view(1, -1, 16), row[n // 2:].view(1, -1)).view(-1)
        gate, up, down = m[:I * H].view(I, H), m[I * H:2 * I * H].view(I, H), m[2 * I * H:].view(H, I)
        xe = x[s['rows'][lo:hi]]
        g = xe @ gate.t()
        a = g / (1 + torch.exp(-g)) * (xe @ up.t())
        if quantised:
            a = _values(*_quantize(a))
        y = (a @ down.t()) * s['w'].view(-1)[at[lo:hi]].float()[:, None]
        out[at[lo:hi]] = y.to(torch.bfloat16)
    return out


def run(s):
    c = s['case']
    kind = c['kind']
    if own:
        from ferry_amd import expert_ops as ops
        if kind == 'route':
            return ops.route_experts(s['logits'], c['topk'], scoring=c['scoring'], bias=s['bias'],
                                     groups=c['groups'], topk_groups=c['topk_groups'],
                                     group_score=c['group_score'], renorm=c['renorm'], scale=c['scale'])
        if kind == 'quantize':
            codes, scales = ops.mxfp4_quantize(s['x'])
            return ops.mxfp4_dequantize(codes, scales, columns=c['cols'], dtype=s['x'].dtype)
        x = ops.mxfp4_quantize(s['x']) if kind == 'ffnq' else s['x']
        return ops.mxfp4_expert_ffn(s['cache'], x, s['w'], s['starts'], s['rows'], s['cols'],
                                    s['experts'], s['slot_of'], c['hidden'], c['inter'], s['act'],
                                    s['out'], counts=s['counts'])
    if kind == 'route':
        return _plain_route(s)
    if kind == 'quantize':
        x = s['x']
        return _values(*_quantize(x.float()))[:, :x.shape[1]].contiguous().to(x.dtype)
    return _plain_ffn(s)


# -- the definitions in 64 bits -------------------------------------------------------------------

def _exact_mx(x):
    """Values of the MXFP4 form of float64 rows whose length is a multiple of 32, by distance to the
    representable values."""
    b = x.reshape(-1, 32)
    amax = b.abs().amax(1, keepdim=True)
    e = torch.floor(torch.log2(amax))
    e = torch.where(torch.exp2(e) > amax, e - 1, e)          # log2 rounded up to a whole number
    e = torch.where(torch.exp2(e + 1) <= amax, e + 1, e)     # ... or down from one
    scale = torch.exp2((e - 2).clamp(-127, 127))
    scale = torch.where(amax == 0, torch.full_like(scale, 2.0 ** -127), scale)
    a = b.abs() / scale
    # steps of 1/2 below 2, of 1 below 4, of 2 above; round() takes ties to the even multiple
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).to(a.dtype)
    v = torch.clamp(torch.round(a / step) * step, max=6.0)
    return (torch.sign(b) * v * scale).reshape(x.shape)


def _exact_weights(row, n):
    """float64 values of one expert's MXFP4 row, from the bits: sign, exponent, mantissa."""
    c = row[:n // 2].long()
    c = torch.stack([c & 15, c >> 4], 1).reshape(-1)
    ex, man = (c >> 1) & 3, (c & 1).double()
    v = torch.where(ex == 0, man * 0.5, torch.exp2(ex.double() - 1) * (1 + man / 2))
    v = torch.where(c >= 8, -v, v)
    return v * torch.exp2(row[n // 2:].double() - 127).repeat_interleave(32)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case['kind']
    if kind == 'quantize':
        n, cols = s['x'].shape
        out = torch.empty((n, cols), dtype=torch.float64, device=s['x'].device)
        step = max(1, (1 << 26) // cols)
        for lo in range(0, n, step):   # a part of the rows at a time, to bound the memory
            x = s['x'][lo:lo + step].double()
            pad = torch.zeros((x.shape[0], -cols % 32), dtype=torch.float64, device=x.device)
            out[lo:lo + step] = _exact_mx(torch.cat([x, pad], 1).contiguous())[:, :cols]
        return out
    if kind == 'route':
        x = s['logits'].double().cpu().numpy()
        T, E = x.shape
        if case['scoring'] == 'softmax':
            p = np.exp(x - x.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
        else:
            p = np.where(x >= 0, 1 / (1 + np.exp(-np.abs(x))), 1 - 1 / (1 + np.exp(-np.abs(x))))
        choice = p + s['bias'].double().cpu().numpy() if case['bias'] else p
        size = E // case['groups']
        per = np.sort(choice.reshape(T, -1, size), axis=2)
        score = per[..., -1] + (per[..., -2] if case['group_score'] == 'top2' else 0)
        rank = np.argsort(np.argsort(-score, axis=1, kind='stable'), axis=1, kind='stable')
        open_ = np.repeat(rank < case['topk_groups'], size, axis=1)
        # by group (open ones first), then by score, then by index
        order = np.lexsort((np.broadcast_to(np.arange(E), (T, E)), -choice, ~open_), axis=1)
        ids = order[:, :case['topk']]
        w = np.take_along_axis(p, ids, 1)
        if case['renorm']:
            w = w / w.sum(1, keepdims=True)
        return w * case['scale'], ids
    H, I, k = case['hidden'], case['inter'], case['topk']
    n = 3 * H * I
    x = s['x'].double()
    if kind == 'ffnq':
        x = _exact_mx(x)
    w = s['w'].double()
    out = torch.zeros((case['tokens'] * k, H), dtype=torch.float64, device=x.device)
    lo = 0
    for e, cnt in enumerate(s['counts']):
        if cnt == 0:
            continue
        r, c = s['rows'][lo:lo + cnt], s['cols'][lo:lo + cnt]
        lo += int(cnt)
        m = _exact_weights(s['cache'][int(s['slot_of'][e])], n)
        g = x[r] @ m[:I * H].view(I, H).t()
        a = g * torch.sigmoid(g) * (x[r] @ m[I * H:2 * I * H].view(I, H).t())
        if kind == 'ffnq':
            a = _exact_mx(a)
        out[r * k + c] = (a @ m[2 * I * H:].view(H, I).t()) * w[r, c][:, None]
    return out


# -- work -----------------------------------------------------------------------------------------

def work(case):
    if case['kind'] == 'route':
        T, E, k = case['tokens'], case['experts'], case['topk']
        size = 4 if case['dtype'] == 'fp32' else 2
        return dict(bytes=T * E * size + (4 * E if case['bias'] else 0) + T * k * 10, flops=4 * T * E)
    if case['kind'] == 'quantize':
        n, blocks = case['rows'] * case['cols'], case['rows'] * -(-case['cols'] // 32)
        size = 4 if case['dtype'] == 'fp32' else 2
        return dict(bytes=2 * (n * size + blocks * 17), flops=4 * n)
    T, H, I, k = case['tokens'], case['hidden'], case['inter'], case['topk']
    active = len(np.unique(_routing(case, 0)))
    # the active experts' rows, the hidden rows, the weights and indices, and the output rows
    return dict(bytes=active * 3 * H * I // 32 * 17 + T * H * 2 + T * k * (2 + 16 + H * 2),
                flops=6 * T * k * H * I)
