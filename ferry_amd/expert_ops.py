"""Python face of the HIP kernels (libferry_amd.so) with the reference's native-op names.

Reference: ``expert_ops()`` of ferry/runtime.py:26-31, i.e. the pybind11 module of
ferry/csrc/expert_ops.cpp:144-157 (execute_experts, pack_dispatch, unpack_dispatch,
reduce_partials, scatter_returned, H2DEngine).  The same names and argument meanings are kept
so that call sites written against the reference work unchanged; the fused hot-path entry
points (router_topk, layout, expert_ffn, combine, history_update) are exposed next to them.
All tensors are CUDA (HIP) tensors; every op runs on the current stream.
"""
import functools
import math
from operator import add, attrgetter

import numpy as np
import torch
import torch.nn.functional as F
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from ._lib import check, lib
from ._lib import check as _check_status
from .h2d import H2DEngine

__all__ = ['execute_experts', 'pack_dispatch', 'unpack_dispatch', 'reduce_partials',
           'scatter_returned', 'H2DEngine', 'router_topk', 'layout', 'gate_logits', 'expert_ffn',
           'combine', 'SharedExpert', 'route_experts', 'mxfp4_quantize', 'mxfp4_dequantize',
           'mxfp4_expert_rows', 'mxfp4_expert_ffn', 'linear', 'linear_grad', 'expert_linear', 'expert_linear_grad',
           'sum_pairs', 'history_update', 'history_ready_words', 'current_stream', 'PHASE_UP',
           'PHASE_DOWN', 'PHASE_BOTH']

MAX_EXPERTS = 512


def timing_enable(on=True):
    """Per-launch kernel timing: every kernel launch of the library gets a start/stop HIP event
    pair bracketing exactly that dispatch (hipExtLaunchKernel).  Turning it on clears the log."""
    check(lib().ferry_timing_enable(int(bool(on))), 'timing_enable')


def timing_summary(kernel):
    """(launches, total ms) of the timed launches of ``kernel`` (e.g. 'ffn_up_skinny')."""
    import ctypes
    n = ctypes.c_int64()
    ms = ctypes.c_double()
    check(lib().ferry_timing_summary(kernel.encode(), ctypes.byref(n), ctypes.byref(ms)),
          'timing_summary')
    return int(n.value), float(ms.value)


def timing_mark():
    """Position in the per-launch timing log (the number of launches recorded so far)."""
    return int(lib().ferry_timing_mark())


def timing_range(begin, end):
    """Summed ms of the timed launches at log positions [begin, end)."""
    import ctypes
    ms = ctypes.c_double()
    check(lib().ferry_timing_range(int(begin), int(end), ctypes.byref(ms)), 'timing_range')
    return float(ms.value)


def timing_overlap(begin, end, t0, t1):
    """ms that the timed launches at log positions [begin, end) overlap the window between
    two timing-enabled torch.cuda.Events (e.g. the first and last copy of a fetch)."""
    import ctypes
    ms = ctypes.c_double()
    check(lib().ferry_timing_overlap(int(begin), int(end), t0.cuda_event, t1.cuda_event,
                                     ctypes.byref(ms)), 'timing_overlap')
    return float(ms.value)


def current_stream(device=None):
    return torch.cuda.current_stream(device).cuda_stream


# handle of the current stream of a device index, without a Stream object (1.3 us less a call)
_raw_stream = getattr(torch._C, '_cuda_getCurrentRawStream', None) or current_stream


def _stream_of(t):
    """The current stream's handle on the device of a CUDA tensor."""
    return _raw_stream(t.get_device())


def _dev(t, name, dtype=None, contiguous=True):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise RuntimeError(f'{name} must be a CUDA tensor')
    if dtype is not None and t.dtype != dtype:
        raise RuntimeError(f'{name} must be {dtype}, got {t.dtype}')
    if contiguous and not t.is_contiguous():
        raise RuntimeError(f'{name} must be contiguous')
    return t.data_ptr()


# ------------------------------------------------------------------------------------------
# Hot-path entry points
# ------------------------------------------------------------------------------------------

def router_topk(logits, topk, renorm=True, scale=1.0, sorted=True, return_probs=False,
                tie_counter=None):
    """Softmax (fp32) + top-k + optional renorm, * scale, cast to bf16.

    Reference: ferry/model.py:141-146 (Qwen3: ``softmax(logits, -1, fp32)``, ``topk(k)``,
    ``w / w.sum(-1)``, ``.to(bf16)``) and the greedy DeepSeek-V2 gate reaching
    ferry/model.py:151-157 (``topk(sorted=False)``, ``* routed_scaling_factor``).
    Returns (weights bf16 [T, k], selected int64 [T, k]) and the fp32 probabilities when
    ``return_probs``.  Index selection is exactly torch's CPU ``topk``, ties included.
    """
    if logits.dim() != 2:
        raise RuntimeError('logits must be [tokens, experts]')
    dt = {torch.bfloat16: 0, torch.float32: 1}.get(logits.dtype)
    if dt is None:
        raise RuntimeError('logits must be bf16 or fp32')
    T, E = logits.shape
    idx = torch.empty((T, topk), dtype=torch.int64, device=logits.device)
    w = torch.empty((T, topk), dtype=torch.bfloat16, device=logits.device)
    probs = torch.empty((T, E), dtype=torch.float32, device=logits.device) if return_probs else None
    check(lib().ferry_router_topk(
        _dev(logits, 'logits'), dt, T, E, topk, int(bool(renorm)), float(scale), int(bool(sorted)),
        idx.data_ptr(), w.data_ptr(), probs.data_ptr() if probs is not None else None,
        _dev(tie_counter, 'tie_counter', torch.int32) if tie_counter is not None else None,
        _stream_of(logits)), 'router_topk')
    return (w, idx, probs) if return_probs else (w, idx)


_DTYPES = {torch.bfloat16: 0, torch.float32: 1, torch.float16: 2}   # FERRY_BF16, FERRY_F32, FERRY_F16
_current_device = getattr(torch._C, '_cuda_getDevice', None) or torch.cuda.current_device


def _matrix(rows, cols, dtype, device):
    """A new [rows, cols] tensor (torch.empty takes 0.4 us longer)."""
    return torch.empty_strided((rows, cols), (max(cols, 1), 1), dtype=dtype, device=device)


def _at(t, name, dtype, device):
    """The address of a contiguous tensor of ``dtype`` on the CUDA device of number ``device``."""
    if isinstance(t, torch.Tensor) and t.get_device() == device and t.dtype == dtype and t.is_contiguous():
        return t.data_ptr()
    _dev(t, name, dtype)
    raise RuntimeError(f'{name} must be on cuda:{device}')


def route_experts(logits, topk, scoring='softmax', bias=None, groups=1, topk_groups=None,
                  group_score='max', renorm=True, scale=1.0):
    """Expert selection of a general gate: ``scoring`` 'softmax' or 'sigmoid', an additive balance
    ``bias`` on the scores that choose (not on the weights), ``groups`` of consecutive experts of which
    the best ``topk_groups`` stay, scored by their largest choice score ('max') or by the sum of their two
    largest ('top2'), then the ``topk`` experts with the largest choice scores.

    ``logits`` is bf16, fp32 or fp16 [T, E], ``bias`` fp32 [E].  Returns (weights bf16 [T, topk], selected
    int64 [T, topk], by descending choice score): the chosen experts' scores, divided by their sum with
    ``renorm``, times ``scale``.  Ties go to the lowest index (``router_topk`` keeps torch's CPU order);
    scores are compared in 64 bits.  A logit of -inf masks an expert (chosen last, weight 0); the IDs of a
    row are distinct whatever the logits hold, and a softmax row with a NaN or +inf has NaN weights.
    No counterpart in the reference; the results carry no gradient.
    """
    if logits.dim() != 2:
        raise RuntimeError('logits must be [tokens, experts]')
    dt = _DTYPES.get(logits.dtype)
    if dt is None:
        raise RuntimeError('logits must be bf16, fp32 or fp16')
    if scoring not in ('softmax', 'sigmoid'):
        raise ValueError("scoring must be 'softmax' or 'sigmoid'")
    if group_score not in ('max', 'top2'):
        raise ValueError("group_score must be 'max' or 'top2'")
    T, E = logits.shape
    at, bias_at, device = _dev(logits, 'logits'), None, logits.device
    if bias is not None:
        bias_at = _at(bias, 'bias', torch.float32, device.index)
        if bias.shape != (E,):
            raise RuntimeError('bias must be fp32 [experts]')
    idx = _matrix(T, topk, torch.int64, device)
    w = _matrix(T, topk, torch.bfloat16, device)
    _native(logits, 'route_experts', lib().ferry_route_experts,
            at, dt, T, E, topk, int(scoring == 'sigmoid'), bias_at, groups,
            groups if topk_groups is None else topk_groups, int(group_score == 'top2'),
            int(bool(renorm)), float(scale), idx.data_ptr(), w.data_ptr())
    return w, idx


def _native(t, what, fn, *args):
    """``fn(*args, stream)`` on the device of the CUDA tensor ``t`` and its current stream there."""
    if t.get_device() == _current_device():
        check(fn(*args, _stream_of(t)), what)
    else:
        with torch.cuda.device(t.device):
            check(fn(*args, _stream_of(t)), what)


def _on_device(t, name, like):
    if not isinstance(t, torch.Tensor) or t.get_device() != like.get_device():
        raise RuntimeError(f'{name} must be on {like.device}')


def _row_stride(t, name):
    """Elements from one row of [rows, cols] to the next; the elements of a row follow each other."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise RuntimeError(f'{name} must be a CUDA tensor')
    if not t.dim():
        raise RuntimeError(f'{name} must hold rows')
    if t.dim() == 2 and (t.shape[1] <= 1 or t.stride(1) == 1) and (
            t.shape[0] <= 1 or t.stride(0) >= t.shape[1]):
        return t.stride(0) if t.shape[0] > 1 else t.shape[1]
    if not t.is_contiguous():
        raise RuntimeError(f'{name} must be contiguous, or a matrix of contiguous rows')
    return t.shape[-1]


def _mxfp4_quantize(x, stride, codes, ldc, scales, lds):
    cols = x.shape[-1]
    _native(x, 'mxfp4_quantize', lib().ferry_mxfp4_quantize, x.data_ptr(), _DTYPES[x.dtype],
            x.numel() // cols if cols else 0, cols, stride, codes, ldc, scales, lds)


def mxfp4_quantize(x):
    """(codes, scales) of the rows of ``x`` (bf16, fp32 or fp16 [..., cols]; a matrix may have a row
    stride) in MXFP4: uint8 codes [..., 16 * blocks], two elements a byte, the first in the low half, and
    uint8 scales [..., blocks], 2^(byte - 127), for ``blocks`` = ceil(cols / 32) blocks of 32 elements.

    A block's scale is 2^(floor(log2(its largest magnitude)) - 2), elements round to the nearest of 0,
    0.5, 1, 1.5, 2, 3, 4, 6 (ties to the even code) and saturate at 6; a block with an infinity or a NaN
    reads back as NaN.  No counterpart in the reference, whose expert rows are bf16."""
    stride = _row_stride(x, 'x')
    if x.dtype not in _DTYPES:
        raise RuntimeError('x must be bf16, fp32 or fp16')
    *lead, cols = x.shape
    blocks, device = -(-cols // 32), x.device
    n = math.prod(lead)
    codes = _matrix(n, blocks * 16, torch.uint8, device)
    scales = _matrix(n, blocks, torch.uint8, device)
    _mxfp4_quantize(x, stride, codes.data_ptr(), blocks * 16, scales.data_ptr(), blocks)
    return (codes, scales) if len(lead) == 1 else (codes.view(*lead, blocks * 16), scales.view(*lead, blocks))


def mxfp4_dequantize(codes, scales, columns=None, dtype=torch.bfloat16):
    """The values of ``mxfp4_quantize``'s (codes, scales) rounded to ``dtype`` (bf16 holds them exactly),
    [..., columns]; all 32 * blocks columns without ``columns``.  Both may be matrices with a row stride
    (the two parts of ``mxfp4_expert_rows``)."""
    if dtype not in _DTYPES:
        raise RuntimeError('dtype must be bf16, fp32 or fp16')
    ldc, lds = _row_stride(codes, 'codes'), _row_stride(scales, 'scales')
    if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
        raise RuntimeError('codes and scales must be uint8')
    blocks = scales.shape[-1]
    if codes.shape != (*scales.shape[:-1], 16 * blocks):
        raise RuntimeError('codes must have 16 bytes for every scale')
    _on_device(scales, 'scales', codes)
    cols = 32 * blocks if columns is None else int(columns)
    if not 32 * blocks - 32 < cols <= 32 * blocks:
        raise RuntimeError(f'columns must end in the last of the {blocks} blocks')
    *lead, _ = scales.shape
    n = math.prod(lead)
    out = _matrix(n, cols, dtype, codes.device)
    _native(codes, 'mxfp4_dequantize', lib().ferry_mxfp4_dequantize, codes.data_ptr(), ldc,
            scales.data_ptr(), lds, n if cols else 0, cols, out.data_ptr(), _DTYPES[dtype], cols)
    return out if len(lead) == 1 else out.view(*lead, cols)


def mxfp4_expert_rows(rows, out=None):
    """Expert rows ``[gate | up | down]`` (bf16, fp32 or fp16 [n, elements], the cache and pool row format)
    as MXFP4 rows: uint8 [n, elements / 32 * 17], a row's codes and then its scales.  ``elements`` must be
    a multiple of 128, as 3 * hidden * intermediate is.  ``out`` (optional) receives the rows."""
    if not isinstance(rows, torch.Tensor) or rows.dim() != 2 or rows.dtype not in _DTYPES:
        raise RuntimeError('rows must be bf16, fp32 or fp16 [experts, elements]')
    n, elements = rows.shape
    if elements % 128:
        raise RuntimeError('a row must hold a multiple of 128 elements')
    stride = _row_stride(rows, 'rows')
    width = elements // 32 * 17
    if out is None:
        out = torch.empty((n, width), dtype=torch.uint8, device=rows.device)
    elif out.shape != (n, width):
        raise RuntimeError(f'out must be uint8 [{n}, {width}]')
    at = _dev(out, 'out', torch.uint8)
    _on_device(out, 'out', rows)
    _mxfp4_quantize(rows, stride, at, width, at + elements // 2, width)
    return out


def _gate_kernel_takes(x, weight):
    """bf16 CUDA matrices that the gate kernel can read as they are, in a call that torch does not
    watch (a trace, autocast, autograd, forward mode, a transform)."""
    if (torch.jit.is_tracing() or x.dtype is not torch.bfloat16 or weight.dtype is not torch.bfloat16
            or not x.is_cuda or x.dim() != 2 or weight.dim() != 2 or x.shape[1] != weight.shape[1]
            or x.shape[1] % 64 or x.shape[1] > 1 << 24 or not x.numel() or not weight.numel()
            or x.shape[0] >= 1 << 30 or weight.shape[0] > 65536
            or x.get_device() != weight.get_device() or not x.is_contiguous()
            or not weight.is_contiguous() or torch.is_autocast_enabled()
            or (torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad))):
        return False
    # outside every dual level no tensor has a tangent (asking each costs 1 us)
    if (getattr(forward_ad, '_current_level', 0) >= 0
            and any(forward_ad.unpack_dual(t).tangent is not None for t in (x, weight))):
        return False
    try:
        return (x.data_ptr() | weight.data_ptr()) % 16 == 0
    except RuntimeError:   # a transform's tensor: its address is not to be had
        return False


def gate_logits(x, weight):
    """fp32 router logits of a gate: ``F.linear(x.float(), weight.float())`` (the DeepSeek-V2 gate
    feeding ferry/model.py:151-158).

    Plain bf16 CUDA matrices go to a kernel that reads them as they are (another order of the fp32
    additions); everything else, and a call that autograd, autocast, a transform or a trace takes part
    in, is the torch expression."""
    if _gate_kernel_takes(x, weight):
        out = torch.empty((x.shape[0], weight.shape[0]), dtype=torch.float32, device=x.device)
        check(lib().ferry_gate_logits(x.data_ptr(), x.shape[0], x.shape[1], weight.data_ptr(),
                                      weight.shape[0], out.data_ptr(), _stream_of(x)), 'gate_logits')
        return out
    return F.linear(x.float(), weight.float())


class Layout:
    """Device layout of one layer call (ferry/layout.py:12-94 at world = 1)."""

    __slots__ = ('tokens', 'topk', 'experts', 'send_ids', 'w_sorted', 'starts', 'rows', 'cols',
                 'pair_pos', 'workspace')


def layout_workspace_bytes(tokens, topk, experts):
    return int(lib().ferry_layout_workspace_bytes(tokens, topk, experts))


def layout_errors(lay):
    """Number of tokens of the last ``layout`` call into ``lay`` that had an expert ID outside
    [0, experts) or a repeated ID (waits for that call)."""
    return int(lay.workspace[:4].view(torch.int32).item())


def layout(selected, weights, experts, out=None, check=False):
    """Sorted packet IDs/weights, per-expert starts and the stable (rows, cols) permutation.

    Every token's IDs must be distinct and in [0, experts).  The kernel counts the tokens that
    break this; ``check=True`` waits for the result and raises RuntimeError when any did.
    """
    T, k = selected.shape
    dev = selected.device
    lay = out if out is not None else Layout()
    if out is None:
        lay.send_ids = torch.empty((T, k), dtype=torch.int64, device=dev)
        lay.w_sorted = torch.empty((T, k), dtype=torch.bfloat16, device=dev)
        lay.starts = torch.empty(experts + 1, dtype=torch.int64, device=dev)
        lay.rows = torch.empty(T * k, dtype=torch.int64, device=dev)
        lay.cols = torch.empty(T * k, dtype=torch.int64, device=dev)
        lay.pair_pos = torch.empty(T * k, dtype=torch.int32, device=dev)
        lay.workspace = torch.empty(layout_workspace_bytes(T, k, experts), dtype=torch.uint8,
                                    device=dev)
    lay.tokens, lay.topk, lay.experts = T, k, experts
    _check_status(lib().ferry_layout(
        _dev(selected, 'selected', torch.int64),
        _dev(weights, 'weights', torch.bfloat16) if weights is not None else None,
        T, k, experts, lay.send_ids.data_ptr(), lay.w_sorted.data_ptr(), lay.starts.data_ptr(),
        lay.rows.data_ptr(), lay.cols.data_ptr(), lay.pair_pos.data_ptr(),
        lay.workspace.data_ptr(), lay.workspace.numel(), _stream_of(selected)), 'layout')
    if check:
        _raise_bad_tokens(layout_errors(lay), experts)
    return lay


def layout_on_host(selected, weights, experts):
    """``layout(..., check=True)`` and its ``starts`` on the host (int64 numpy [experts + 1]), read
    back in one copy with the count of invalid tokens."""
    T, k = selected.shape
    dev = selected.device
    head = -(-(experts + 1) * 8 // 256) * 256
    buf = torch.empty(head + layout_workspace_bytes(T, k, experts), dtype=torch.uint8, device=dev)
    lay = Layout()
    lay.send_ids = torch.empty((T, k), dtype=torch.int64, device=dev)
    lay.w_sorted = torch.empty((T, k), dtype=torch.bfloat16, device=dev)
    lay.starts = buf[:(experts + 1) * 8].view(torch.int64)
    lay.rows = torch.empty(T * k, dtype=torch.int64, device=dev)
    lay.cols = torch.empty(T * k, dtype=torch.int64, device=dev)
    lay.pair_pos = torch.empty(T * k, dtype=torch.int32, device=dev)
    lay.workspace = buf[head:]
    layout(selected, weights, experts, out=lay)
    host = buf[:head + 4].cpu().numpy()
    _raise_bad_tokens(int(host[head:].view(np.int32)[0]), experts)
    return lay, host[:(experts + 1) * 8].view(np.int64)


def _raise_bad_tokens(bad, experts):
    if bad:
        raise RuntimeError(f'layout: {bad} token(s) with an expert ID out of [0, {experts}) '
                           'or repeated')


PHASE_UP, PHASE_DOWN, PHASE_BOTH = 1, 2, 3
SKINNY_MAX_ROWS = 64   # experts with at most this many rows run the small-expert kernels


def expert_ffn(cache, x, w_sorted, starts, rows, cols, expert_list, slot_of, hidden,
               intermediate, act, out, out_mode=0, max_rows=None, experts=None, phases=PHASE_BOTH,
               counts=None, spare_cus=0):
    """Grouped SwiGLU over cache slots for the experts in ``expert_list`` (host ints).

    phases: PHASE_UP (gate/up + SwiGLU into ``act``), PHASE_DOWN (down + routing weight from
    ``act`` into ``out``) or PHASE_BOTH.  ``counts`` (optional, host, indexed by expert) holds
    the row count of every expert, ``starts[e+1] - starts[e]``: the library then issues the
    experts with at most 64 rows (small-expert kernels, 17-64 rows first) and the larger ones
    (tiled kernels) as separate launches with exact row bounds, and skips experts without rows.
    ``rows`` and ``cols`` are CUDA tensors or raw device addresses (ints).  ``spare_cus`` keeps the
    tiled kernels off that many CUs, for kernels on other streams.
    """
    R, k = w_sorted.shape
    el = np.ascontiguousarray(expert_list, dtype=np.int32)
    so = np.ascontiguousarray(slot_of, dtype=np.int32)
    E = int(experts if experts is not None else len(so))
    args = (_dev(cache, 'cache', torch.bfloat16), cache.shape[0], hidden, intermediate,
            _dev(x, 'x', torch.bfloat16), R, k, _dev(w_sorted, 'w_sorted', torch.bfloat16),
            _dev(starts, 'starts', torch.int64),
            rows if isinstance(rows, int) else _dev(rows, 'rows', torch.int64),
            cols if isinstance(cols, int) else _dev(cols, 'cols', torch.int64))
    tail = (_dev(act, 'act', torch.bfloat16), _dev(out, 'out', torch.bfloat16), int(out_mode),
            int(phases), int(spare_cus), _stream_of(x))

    # the host lists as bytes: an array's address costs 2 us more
    n, el_at, so_at = len(el), el.tobytes(), so.tobytes()
    if counts is None:
        check(lib().ferry_expert_ffn_spare(*args, el_at, n, so_at, E,
                                     int(max_rows if max_rows is not None else R), 0, None, *tail),
              'expert_ffn')
        return out
    c = np.ascontiguousarray(np.asarray(counts, dtype=np.int64)[el], dtype=np.int32)
    if n:
        rows_of = c.tolist()
        check(lib().ferry_expert_ffn_spare(*args, el_at, n, so_at, E, max(rows_of), min(rows_of),
                                     c.tobytes(), *tail), 'expert_ffn')
    return out


def mxfp4_expert_ffn(cache, x, w_sorted, starts, rows, cols, expert_list, slot_of, hidden,
                     intermediate, act, out, out_mode=0, max_rows=None, experts=None, phases=PHASE_BOTH,
                     counts=None, spare_cus=0):
    """``expert_ffn`` over cache slots of MXFP4 rows (``mxfp4_expert_rows``: uint8 [slots, 3 * hidden *
    intermediate / 32 * 17]), read as they are: 4.25 bits a weight.

    ``x`` is bf16 [R, hidden], with ``act`` bf16 scratch of R * topk * intermediate elements (silu(g) * u rounded to
    bf16; with R * topk <= 64 experts of at most 8 rows keep 11 bits of it, in a format of their own); or
    ``mxfp4_quantize``'s (codes, scales) of the rows, with ``act`` uint8 scratch of R * topk *
    intermediate / 32 * 17 bytes: both products then take 4-bit operands on either side, which is the
    faster form for prompts, and silu(g) * u is quantised on the way.  Sums and SwiGLU are fp32; an
    output row is rounded to bf16 once, after its routing weight.  The other arguments are
    ``expert_ffn``'s; ``rows`` and ``cols`` have an entry for every pair of ``starts`` (at least the sum of
    ``counts``, where those are given); ``spare_cus`` leaves the room of that many CUs beside the tiled kernels (half the
    room of twice as many, where two workgroups share a CU), and gives the small experts launches of their own; rows of ``out`` that belong to experts outside the list are left as they are.
    No counterpart in the reference.
    """
    R, k = w_sorted.shape
    H, I = int(hidden), int(intermediate)
    quantised = isinstance(x, (tuple, list))
    codes, scales = x if quantised else (x, None)
    _dev(cache, 'cache', torch.uint8)
    if cache.dim() != 2 or cache.shape[1] * 32 != 3 * H * I * 17:
        raise RuntimeError('cache must be uint8 [slots, 3 * hidden * intermediate / 32 * 17]')
    dev = cache.get_device()
    kind = torch.uint8 if quantised else torch.bfloat16
    x_at, scales_at = _at(codes, 'x', kind, dev), _at(scales, 'x scales', kind, dev) if quantised else None
    if quantised:
        if codes.shape != (R, H // 2) or scales.shape != (R, H // 32):
            raise RuntimeError('x must be the codes [rows, hidden / 2] and scales [rows, hidden / 32]')
    elif codes.shape != (R, H):
        raise RuntimeError('x must be bf16 [rows, hidden]')
    el = np.ascontiguousarray(expert_list, dtype=np.int32)
    so = np.ascontiguousarray(slot_of, dtype=np.int32)
    E = int(experts if experts is not None else len(so))
    if E > len(so) or (counts is not None and E > len(counts)):
        raise RuntimeError('slot_of and counts must have an entry for every expert')
    rows_at = rows if isinstance(rows, int) else _at(rows, 'rows', torch.int64, dev)
    cols_at = cols if isinstance(cols, int) else _at(cols, 'cols', torch.int64, dev)
    weights, first = _at(w_sorted, 'w_sorted', torch.bfloat16, dev), _at(starts, 'starts', torch.int64, dev)
    if starts.numel() < E + 1:
        raise RuntimeError('starts must have an entry for every expert, and the end')
    act_at, out_at = _at(act, 'act', kind, dev), _at(out, 'out', torch.bfloat16, dev)
    if act.numel() < R * k * (I // 32 * 17 if quantised else I) or out.numel() < R * k * H:
        raise RuntimeError('act and out must hold the rows of rows * topk (token, expert) pairs')
    list_rows, most = None, int(max_rows if max_rows is not None else R)
    # entries of rows and cols; of a list that is an address as many as there are output rows
    pairs = R * k
    held = rows.numel() if isinstance(rows, torch.Tensor) else pairs
    slots = cols.numel() if isinstance(cols, torch.Tensor) else pairs
    if held != slots and isinstance(rows, torch.Tensor) and isinstance(cols, torch.Tensor):
        raise RuntimeError('rows and cols must have the same length')
    if counts is not None:
        counts = np.asarray(counts)
        # with lists of the usual length only the listed experts' counts are checked, in the library
        if (held != pairs or slots != pairs) and np.add.reduce(counts[:E]) > min(held, slots, pairs):
            raise RuntimeError('counts must name at most rows * topk pairs, with an entry of rows and cols for each')
    if not held or not slots:
        return out   # no pairs
    if counts is not None and len(el):
        try:
            list_rows, most = counts[el].astype(np.int32).tobytes(), -1
        except IndexError:
            raise RuntimeError(f'expert_list must name experts in [0, {E})') from None
    _native(cache, 'mxfp4_expert_ffn', lib().ferry_mxfp4_expert_ffn, cache.data_ptr(), cache.shape[0], H, I,
            x_at, scales_at, R, k, weights, first, rows_at, cols_at, el.tobytes(), len(el), so.tobytes(), E, most, 0,
            list_rows, act_at, out_at, int(out_mode), int(phases), int(spare_cus))
    return out


_ACTIVATIONS = {None: 0, 'relu': 1, 'silu': 2, 'gelu': 3, 'gelu_tanh': 4}   # FERRY_ACT_*
_LINEAR, _GRAD_X, _GRAD_W, _GRAD_Z = 0, 1, 2, 3                                # FERRY_LINEAR*
_HALF = {torch.bfloat16: 0, torch.float16: 2}                                 # FERRY_BF16, FERRY_F16


def _half_rows(t, name, device=None, dtype=None):
    """(address, row stride) of the rows of a bf16 or fp16 tensor, on ``device`` and of ``dtype`` if given."""
    if (dtype is not None and isinstance(t, torch.Tensor) and t.dtype is dtype and t.get_device() == device
            and t.is_contiguous() and t.dim()):   # the usual case (the checks below take 1 us longer)
        return t.data_ptr(), t.shape[-1]
    stride = _row_stride(t, name)
    if dtype is None:
        if t.dtype not in _HALF:
            raise RuntimeError(f'{name} must be bf16 or fp16')
    elif t.dtype != dtype:
        raise RuntimeError(f'{name} must be {dtype}, got {t.dtype}')
    if device is not None and t.get_device() != device:
        raise RuntimeError(f'{name} must be on cuda:{device}')
    return t.data_ptr(), stride


def _weight_groups(w, name, device, dtype):
    """(address, row stride, group stride) of [groups, n, k] weights whose rows are contiguous."""
    if not isinstance(w, torch.Tensor) or w.get_device() != device:
        raise RuntimeError(f'{name} must be on cuda:{device}')
    if w.dtype != dtype:
        raise RuntimeError(f'{name} must be {dtype}, got {w.dtype}')
    _, n, k = w.shape
    group, row, one = w.stride()
    if (k > 1 and one != 1) or (n > 1 and row < k):
        raise RuntimeError(f'the rows of {name} must be contiguous')
    return w.data_ptr(), row if n > 1 else k, group


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(product, pairs, n, k, groups, device):
    with torch.cuda.device(device):
        return lib().ferry_linear_workspace_bytes(product, pairs, n, k, groups)


def _workspace(product, pairs, n, k, groups, device):
    """(tensor or None, address, bytes) of a linear product's scratch memory."""
    need = _workspace_bytes(product, pairs, n, k, groups, device)
    if need <= 0:
        return None, None, 0
    ws = torch.empty(need, dtype=torch.uint8, device=device)
    return ws, ws.data_ptr(), need


def _written(out):
    """Tells autograd that ``out`` gets other values: a backward pass that saved the old ones refuses them."""
    if not out.is_inference():
        torch.autograd.graph.increment_version(out)


_tracing = torch._C._is_tracing   # torch.jit.is_tracing without its wrappers (0.2 us)


def _no_trace(what):
    """Refuses a call that torch.jit.trace records: the trace would hold the result's allocation and no launch."""
    raise RuntimeError(f'{what} cannot be traced')


def _watched(what, *tensors):
    """Whether autograd takes part in a call on these tensors (None among them)."""
    if _tracing():
        _no_trace(what)
    if (getattr(forward_ad, '_current_level', 0) >= 0
            and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)):
        raise RuntimeError(f'{what} has no forward-mode derivative')
    if not torch.is_grad_enabled() or not any(t is not None and t.requires_grad for t in tensors):
        return False
    if torch.cuda.is_current_stream_capturing():
        # autograd ties a captured backward pass to the streams of every eager one that shares a leaf
        raise RuntimeError(f'{what}: capture it and {what}_grad under torch.no_grad(); a graph with autograd '
                           'in it is not supported')
    return True


def _product(x, xs, k, rows, pairs, starts, groups, w, ws, wg, n, bias, bias_stride, act, residual, rs, pre, out,
             out_stride, zero_rest):
    scratch, at, size = _workspace(_LINEAR, pairs, n, k, groups, x.device)
    _native(x, 'linear' if starts is None else 'expert_linear', lib().ferry_expert_linear,
            x.data_ptr(), _HALF[x.dtype], x.numel() // k, k, xs, rows, pairs, starts, groups, w, n, ws, wg, bias,
            bias_stride, act, residual, rs, pre, out, out_stride, zero_rest, at, size)


def _linear(x, weight, bias, activation, residual, out, keep):
    """(out, pre or None) of ``linear``."""
    act = _ACTIVATIONS.get(activation, -1)
    if act < 0:
        raise ValueError("activation must be None, 'relu', 'silu', 'gelu' or 'gelu_tanh'")
    _, xs = _half_rows(x, 'x')
    dtype, dev = x.dtype, x.get_device()
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2 or weight.shape[1] != x.shape[-1]:
        raise RuntimeError('weight must be [n, k] for x [..., k]')
    w, ws = _half_rows(weight, 'weight', dev, dtype)
    n, k = weight.shape
    if not n or not k:
        raise RuntimeError('n and k must be at least 1')
    *lead, _ = x.shape
    m = math.prod(lead)
    shape = (*lead, n)
    if bias is not None and bias.shape != (n,):
        raise RuntimeError('bias must be [n]')
    b = _at(bias, 'bias', dtype, dev) if bias is not None else None
    r, rs = None, 0
    if residual is not None:
        r, rs = _half_rows(residual, 'residual', dev, dtype)
        if residual.shape != shape:
            raise RuntimeError(f'residual must be {list(shape)}')
    if out is None:
        out = _matrix(m, n, dtype, x.device)
        if len(lead) != 1:
            out = out.view(shape)
        at, stride = out.data_ptr(), n
    else:
        at, stride = _half_rows(out, 'out', dev, dtype)
        if out.shape != shape:
            raise RuntimeError(f'out must be {list(shape)}')
        _written(out)
    pre = _matrix(m, n, dtype, x.device) if keep and act else None
    if m:
        _product(x, xs, k, None, m, None, 1, w, ws, 0, n, b, 0, act, r, rs,
                 pre.data_ptr() if pre is not None else None, at, stride, 0)
    return out, pre


def linear(x, weight, bias=None, activation=None, residual=None, out=None, return_pre=False):
    """``activation(x @ weight.T + bias) + residual``, rounded once.

    ``x`` [..., k], ``weight`` [n, k] (a matrix may have a row stride), ``bias`` [n] and ``residual``
    [..., n] are bf16 or fp16, all the same; sums are fp32.  ``activation`` is None, 'relu', 'silu', 'gelu'
    (the normal distribution's) or 'gelu_tanh'.  ``out`` (optional) receives the result and may be
    ``residual`` itself, but share no memory with the other arguments.  ``return_pre=True`` returns (result,
    the activation's rounded argument [rows, n], or None without an activation), what ``linear_grad`` needs.
    Rows that start at multiples of 16 bytes are fastest; any other alignment is taken.

    The result carries the gradients of x, weight, bias and residual, except with ``out`` or ``return_pre``
    and inside a captured graph (there ``linear`` and ``linear_grad`` are called under torch.no_grad()).
    A torch.jit.trace is refused.  No counterpart in the reference."""
    if _watched('linear', x, weight, bias, residual, out):
        if out is not None or return_pre:
            raise RuntimeError('linear: out and return_pre carry no gradients; call it under torch.no_grad()')
        return _Linear.apply(x, weight, bias, residual, activation)
    y, pre = _linear(x, weight, bias, activation, residual, out, return_pre)
    return (y, pre) if return_pre else y


def _column_sums(grad, gs, rows, n, starts, groups, pre, act, dz, db):
    scratch, at, size = _workspace(_GRAD_Z, rows, n, 1, groups, grad.device) if db is not None else (None, None, 0)
    _native(grad, 'linear_grad', lib().ferry_linear_grad_z, grad.data_ptr(), _HALF[grad.dtype], rows, n, gs,
            pre.data_ptr() if pre is not None else None, act, starts, groups,
            dz.data_ptr() if dz is not None else None, db.data_ptr() if db is not None else None, at, size)


def _grad_x(dz, zs, pairs, starts, groups, w, ws, wg, n, k, zero_rest):
    dx = _matrix(pairs, k, dz.dtype, dz.device)
    if pairs:
        scratch, at, size = _workspace(_GRAD_X, pairs, n, k, groups, dz.device)
        _native(dz, 'linear_grad', lib().ferry_expert_linear_grad_x, dz.data_ptr(), _HALF[dz.dtype], pairs, n, zs,
                starts, groups, w, k, ws, wg, dx.data_ptr(), zero_rest, at, size)
    return dx


def _grad_w(dz, zs, pairs, n, x, xs, k, rows, starts, groups):
    dw = torch.empty((groups, n, k), dtype=dz.dtype, device=dz.device)
    scratch, at, size = _workspace(_GRAD_W, pairs, n, k, groups, dz.device)
    _native(dz, 'linear_grad', lib().ferry_expert_linear_grad_w, dz.data_ptr(), _HALF[dz.dtype], pairs, n, zs,
            x.data_ptr(), x.numel() // k, k, xs, rows, starts, groups, dw.data_ptr(), at, size)
    return dw


def linear_grad(grad, x, weight, pre=None, activation=None, need_x=True, need_weight=True, need_bias=True):
    """Gradients (dx, dweight, dbias) of ``linear`` for the gradient ``grad`` [..., n] of its result, None for
    those that are not needed; ``pre`` is ``linear(..., return_pre=True)``'s.  The residual's is ``grad``.

    dz = grad * f'(pre) is rounded to the inputs' type before the products; the bias's gradient sums it
    unrounded.  Makes no use of autograd, so it can be captured into a graph."""
    if _tracing():
        _no_trace('linear_grad')
    act = _ACTIVATIONS.get(activation, -1)
    if act < 0:
        raise ValueError("activation must be None, 'relu', 'silu', 'gelu' or 'gelu_tanh'")
    _, xs = _half_rows(x, 'x')
    dtype, dev = x.dtype, x.get_device()
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2 or weight.shape[1] != x.shape[-1]:
        raise RuntimeError('weight must be [n, k] for x [..., k]')
    w, ws = _half_rows(weight, 'weight', dev, dtype)
    n, k = weight.shape
    if not n or not k:
        raise RuntimeError('n and k must be at least 1')
    *lead, _ = x.shape
    m = math.prod(lead)
    _, gs = _half_rows(grad, 'grad', dev, dtype)
    if grad.shape != (*lead, n):
        raise RuntimeError(f'grad must be {[*lead, n]}')
    dz, zs = grad, gs
    db = torch.empty(n, dtype=dtype, device=x.device) if need_bias else None
    if act:
        if not isinstance(pre, torch.Tensor) or pre.shape != (m, n):
            raise RuntimeError('pre must be [rows, n], as linear returns it')
        _at(pre, 'pre', dtype, dev)
        dz, zs = _matrix(m, n, dtype, x.device), n
        _column_sums(grad, gs, m, n, None, 1, pre, act, dz, db)
    elif need_bias:
        _column_sums(grad, gs, m, n, None, 1, None, 0, None, db)
    dx = _grad_x(dz, zs, m, None, 1, w, ws, 0, n, k, 0).view(x.shape) if need_x else None
    dw = _grad_w(dz, zs, m, n, x, xs, k, None, None, 1).view(n, k) if need_weight else None
    return dx, dw, db


def _rows_of(grad):
    """``grad`` as autograd hands it over, with contiguous rows."""
    try:
        _row_stride(grad, 'grad')
        return grad
    except RuntimeError:
        return grad.contiguous()


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation):
        y, pre = _linear(x, weight, bias, activation, residual, None, any(ctx.needs_input_grad[:3]))
        ctx.activation = activation
        ctx.save_for_backward(x, weight, pre)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, weight, pre = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx = dw = db = None
        if any(need[:3]):
            dx, dw, db = linear_grad(_rows_of(grad), x, weight, pre, ctx.activation, *need[:3])
        return dx, dw, db, grad if need[3] else None, None


def _expert_args(x, weight, starts, rows):
    """What ``expert_linear`` and its gradients share: x's row stride, the weights' place, the pairs."""
    _, xs = _half_rows(x, 'x')
    dtype, dev = x.dtype, x.get_device()
    if x.dim() != 2 or not isinstance(weight, torch.Tensor) or weight.dim() != 3 or weight.shape[2] != x.shape[1]:
        raise RuntimeError('x must be [rows, k] and weight [experts, n, k]')
    if not weight.shape[0] or not weight.shape[1] or not weight.shape[2]:
        raise RuntimeError('experts, n and k must be at least 1')
    w, ws, wg = _weight_groups(weight, 'weight', dev, dtype)
    first = _at(starts, 'starts', torch.int64, dev)
    if starts.shape != (weight.shape[0] + 1,):
        raise RuntimeError('starts must have an entry for every expert, and the end')
    rows_at, pairs = None, x.shape[0]
    if rows is not None:
        rows_at, pairs = _at(rows, 'rows', torch.int64, dev), rows.numel()
    return xs, w, ws, wg, first, rows_at, pairs


def _expert_linear(x, weight, starts, bias, rows, out):
    xs, w, ws, wg, first, rows_at, pairs = _expert_args(x, weight, starts, rows)
    E, n, k = weight.shape
    b, bs = None, 0
    if bias is not None:
        b, bs = _half_rows(bias, 'bias', x.get_device(), x.dtype)
        if bias.shape != (E, n):
            raise RuntimeError('bias must be [experts, n]')
    zero = out is None
    if zero:
        out = _matrix(pairs, n, x.dtype, x.device)
        at, stride = out.data_ptr(), n
    else:
        at, stride = _half_rows(out, 'out', x.get_device(), x.dtype)
        if out.shape != (pairs, n):
            raise RuntimeError(f'out must be [{pairs}, {n}]')
        _written(out)
    if pairs:
        _product(x, xs, k, rows_at, pairs, first, E, w, ws, wg, n, b, bs, 0, None, 0, None, at, stride, int(zero))
    return out


def expert_linear(x, weight, starts, bias=None, rows=None, pair_pos=None, out=None):
    """Products grouped by expert: ``out[p] = x[rows[p]] @ weight[e].T + bias[e]`` for ``starts[e] <= p <
    starts[e + 1]``, [pairs, n], for one matrix of an expert, of any number of rows each.

    ``x`` [rows, k], ``weight`` [experts, n, k] (strides of experts and rows may be larger, as those of a
    part of cache rows are) and ``bias`` [experts, n] are bf16 or fp16, all the same; sums are fp32, a result
    is rounded once.  ``starts``, ``rows`` and ``pair_pos`` are ``layout``'s, on the device; without ``rows``
    ``x`` is in grouped order already.  An entry of ``rows`` that names no row of x reads as zeros.  Rows
    before ``starts[0]`` and from ``starts[experts]`` on are 0; in an ``out`` that is passed, which shares no
    memory with the other arguments, they stay as they were.

    The result carries the gradients of x, weight and bias (x's, with ``rows``, needs ``pair_pos`` [tokens *
    topk], the places of each row of x), except with ``out`` and inside a captured graph (there
    ``expert_linear`` and ``expert_linear_grad`` are called under torch.no_grad()).  A torch.jit.trace is
    refused.  No counterpart in the reference."""
    if _watched('expert_linear', x, weight, bias, out):
        if out is not None:
            raise RuntimeError('expert_linear: out carries no gradients; call it under torch.no_grad()')
        if rows is not None and pair_pos is None and x.requires_grad:
            raise RuntimeError('expert_linear: the gradient of gathered rows needs pair_pos')
        return _ExpertLinear.apply(x, weight, starts, bias, rows, pair_pos)
    return _expert_linear(x, weight, starts, bias, rows, out)


def expert_linear_grad(grad, x, weight, starts, rows=None, pair_pos=None, need_x=True, need_weight=True,
                       need_bias=True):
    """Gradients (dx, dweight, dbias) of ``expert_linear`` for the gradient ``grad`` [pairs, n] of its result,
    None for those that are not needed.  With ``rows``, dx[t] is the sum, j ascending, of the (rounded)
    gradients of the grouped rows ``pair_pos[t, j]``; without ``pair_pos`` it is those, [pairs, k], in
    grouped order.  Experts without rows have zero gradients; rows of ``grad`` that belong to no expert are
    not read.  Makes no use of autograd, so it can be captured into a graph."""
    if _tracing():
        _no_trace('expert_linear_grad')
    xs, w, ws, wg, first, rows_at, pairs = _expert_args(x, weight, starts, rows)
    E, n, k = weight.shape
    _, gs = _half_rows(grad, 'grad', x.get_device(), x.dtype)
    if grad.shape != (pairs, n):
        raise RuntimeError(f'grad must be [{pairs}, {n}]')
    dx = dw = db = None
    if need_bias:
        db = torch.empty((E, n), dtype=x.dtype, device=x.device)
        _column_sums(grad, gs, pairs, n, first, E, None, 0, None, db)
    if need_x:
        dx = _grad_x(grad, gs, pairs, first, E, w, ws, wg, n, k, 1)
        if rows is not None and pair_pos is not None:
            dx = sum_pairs(dx, pair_pos, x.shape[0])
    if need_weight:
        dw = _grad_w(grad, gs, pairs, n, x, xs, k, rows_at, first, E)
    return dx, dw, db


class _ExpertLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, starts, bias, rows, pair_pos):
        ctx.save_for_backward(x, weight, starts, rows, pair_pos)
        return _expert_linear(x, weight, starts, bias, rows, None)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, weight, starts, rows, pair_pos = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, dw, db = expert_linear_grad(_rows_of(grad), x, weight, starts, rows, pair_pos, need[0], need[1], need[3])
        return dx, dw, None, db, None, None


def sum_pairs(part, pair_pos, tokens):
    """out[t] = the fp32 sum, j ascending, of ``part[pair_pos[t, j]]``, rounded once, [tokens, k]: the gradient of
    rows that were gathered from tokens.  ``part`` is contiguous bf16 or fp16 [pairs, k], ``pair_pos`` int32
    with as many entries for every token, ``layout``'s; entries outside [0, pairs) add nothing."""
    if _tracing():
        _no_trace('sum_pairs')
    if not isinstance(part, torch.Tensor) or part.dim() != 2 or part.dtype not in _HALF:
        raise RuntimeError('part must be bf16 or fp16 [pairs, k]')
    at, (pairs, k) = _dev(part, 'part'), part.shape
    pos = _at(pair_pos, 'pair_pos', torch.int32, part.get_device())
    if tokens and (pair_pos.numel() % tokens or not pair_pos.numel()):
        raise RuntimeError('pair_pos must hold as many entries for every token')
    out = _matrix(tokens, k, part.dtype, part.device)
    if tokens:
        _native(part, 'sum_pairs', lib().ferry_sum_pairs, at, _HALF[part.dtype], pairs, k, pos, tokens,
                pair_pos.numel() // tokens, out.data_ptr())
    return out


def ffn_sync_timeouts():
    """Waits of the one-launch decode FFN that gave up on the current device (expected 0)."""
    import ctypes
    n = ctypes.c_int64()
    check(lib().ferry_expert_ffn_sync_timeouts(ctypes.byref(n)), 'ffn_sync_timeouts')
    return int(n.value)


def ffn_set_sync_spin_limit(limit):
    """How often a one-launch decode FFN's down phase polls for its up phase before it gives up
    (launches after the call): None or < 0 restores the default; 0 makes every wait give up at
    once, to check how a timeout is reported (no reference counterpart)."""
    check(lib().ferry_expert_ffn_set_sync_spin_limit(-1 if limit is None else int(limit)),
          'ffn_set_sync_spin_limit')


def hbm_read(buf, sink=None):
    """Read every byte of ``buf`` (a contiguous CUDA tensor, nbytes a multiple of 16) once at the
    HBM read rate, on the current stream: the measured read ceiling for the memory-bound
    kernels (no reference counterpart).  Returns ``sink`` (uint8, created when not given): one
    16-byte record per wavefront, the XOR of the 16-byte words it read."""
    if not (isinstance(buf, torch.Tensor) and buf.is_cuda and buf.is_contiguous()):
        raise RuntimeError('hbm_read: buf must be a contiguous CUDA tensor')
    nbytes = buf.numel() * buf.element_size()
    need = int(lib().ferry_hbm_read_sink_bytes(nbytes))
    if sink is None:
        sink = torch.empty(max(need, 16), dtype=torch.uint8, device=buf.device)
    st = torch.cuda.current_stream(buf.device).cuda_stream
    check(lib().ferry_hbm_read(buf.data_ptr(), nbytes, sink.data_ptr(), sink.numel(), st), 'hbm_read')
    return sink


def combine(part, tokens, topk, hidden, pair_pos=None, out=None, addend=None):
    """out[t] = bf16(sum_j fp32(part[src(t, j)])), j ascending (expert_ops.cpp:75-92).

    With ``addend`` (bf16 [tokens, hidden]) the result is bf16(fp32(out[t]) + fp32(addend[t])),
    the bf16 addition of the DeepSeek-V2 shared-expert output.
    """
    if out is None:
        out = torch.empty((tokens, hidden), dtype=torch.bfloat16, device=part.device)
    pp = _dev(pair_pos, 'pair_pos', torch.int32) if pair_pos is not None else None
    stream = _stream_of(part)
    if addend is None:
        check(lib().ferry_combine(_dev(part, 'part', torch.bfloat16), pp, tokens, topk, hidden,
                                  _dev(out, 'out', torch.bfloat16), stream), 'combine')
    else:
        if addend.shape != (tokens, hidden):
            raise RuntimeError('addend must be bf16 [tokens, hidden]')
        check(lib().ferry_combine_add(_dev(part, 'part', torch.bfloat16), pp, tokens, topk, hidden,
                                      _dev(addend, 'addend', torch.bfloat16),
                                      _dev(out, 'out', torch.bfloat16), stream), 'combine_add')
    return out


class SharedExpert:
    """Always-on SwiGLU expert applied to every token (DeepSeek-V2 shared experts).

    Not in the reference runtime: HF's DeepseekV2MoE adds ``shared_experts(residuals)``
    (a DeepseekV2MLP of intermediate n_shared * moe_intermediate, bf16 nn.Linear layers) to
    the routed output (transformers 4.57 modeling_deepseek_v2; installed analogue
    modeling_deepseek_v2.py:126-151).  Here the MLP runs on the grouped SwiGLU kernels as one
    expert whose rows are all tokens with routing weight 1, from one weight row
    ``[gate I*H | up I*H | down H*I]`` (the cache row format) resident in HBM.  The SwiGLU
    rounding is the routed experts' (silu(g) * u in fp32, one bf16 rounding).
    """

    def __init__(self, row, hidden, intermediate):
        if row.dtype != torch.bfloat16 or row.numel() != 3 * hidden * intermediate:
            raise RuntimeError('shared expert row must be bf16 [3 * intermediate * hidden]')
        self.row = row.reshape(1, -1).contiguous()
        self.hidden, self.intermediate = hidden, intermediate
        self._bufs = {}

    def _buffers(self, T, device):
        b = self._bufs.get(T)
        if b is None:
            b = dict(starts=torch.tensor([0, T], dtype=torch.int64, device=device),
                     rows=torch.arange(T, dtype=torch.int64, device=device),
                     cols=torch.zeros(T, dtype=torch.int64, device=device),
                     w=torch.ones((T, 1), dtype=torch.bfloat16, device=device),
                     act=torch.empty((T, self.intermediate), dtype=torch.bfloat16, device=device))
            self._bufs[T] = b
        return b

    def __call__(self, x, out=None, spare_cus=0):
        """bf16 [T, H] -> bf16 [T, H] = down(silu(x Wg^T) * (x Wu^T))."""
        T = x.shape[0]
        if out is None:
            out = torch.empty((T, self.hidden), dtype=torch.bfloat16, device=x.device)
        if T == 0:
            return out
        b = self._buffers(T, x.device)
        return expert_ffn(self.row, x.contiguous(), b['w'], b['starts'], b['rows'], b['cols'], [0],
                          np.zeros(1, np.int32), self.hidden, self.intermediate, b['act'], out,
                          out_mode=1, experts=1, counts=[T], spare_cus=spare_cus)


def history_update(selected, experts, window, layer, ring, counts, meta, scores, ids_out=None,
                   timeouts_out=None, ready_out=None, ready_value=0, records_out=None):
    """Device GateHistory update of ``layer`` (ferry/metadata.py:15-38, frequency rows).

    ``scores`` (fp32 [E]), ``ids_out`` (uint8 [T*k]) and ``timeouts_out`` (int32 [1]: the
    device's count of one-launch decode FFN waits that gave up, as ``ffn_sync_timeouts``) are
    CUDA tensors or raw device addresses (ints), e.g. of a mapped host buffer that the kernel
    writes directly.  ``ready_out`` (device address of ``history_ready_words(T, k)`` int32
    words, with ``ids_out``) receives ``ready_value`` in every word once the launch's other
    writes are visible to the host.  ``records_out`` (device address of ``history_count_blocks(T)``
    records of ``history_count_words(E)`` int32, instead of ``ids_out``) receives each expert's
    demand per 512 tokens; ``ready_out`` then has 1 + ``history_count_blocks(T)`` words."""
    T, k = selected.shape
    sp = scores if isinstance(scores, int) else _dev(scores, 'scores', torch.float32)
    ip = (ids_out if isinstance(ids_out, int) or ids_out is None
          else _dev(ids_out, 'ids_out', torch.uint8))
    tp = (timeouts_out if isinstance(timeouts_out, int) or timeouts_out is None
          else _dev(timeouts_out, 'timeouts_out', torch.int32))
    rp = (ready_out if isinstance(ready_out, int) or ready_out is None
          else _dev(ready_out, 'ready_out', torch.int32))
    if records_out is not None:
        if ids_out is not None:
            raise RuntimeError('history_update writes either IDs or demand records')
        check(lib().ferry_history_count(
            _dev(selected, 'selected', torch.int64), T, k, experts, window, layer,
            _dev(ring, 'ring', torch.int32), _dev(counts, 'counts', torch.int32),
            _dev(meta, 'meta', torch.int32), sp, int(records_out), tp, rp, int(ready_value),
            _stream_of(selected)), 'history_count')
        return
    check(lib().ferry_history_update(
        _dev(selected, 'selected', torch.int64), T, k, experts, window, layer,
        _dev(ring, 'ring', torch.int32), _dev(counts, 'counts', torch.int32),
        _dev(meta, 'meta', torch.int32), sp, ip, tp, rp, int(ready_value),
        _stream_of(selected)), 'history_update')


def history_ready_words(tokens, topk):
    """Number of int32 ready words ``history_update`` writes for a call of ``tokens``."""
    return int(lib().ferry_history_ready_words(int(tokens), int(topk)))


def history_count_blocks(tokens):
    """Number of demand records (512 tokens each) of a call of ``tokens``."""
    return int(lib().ferry_history_count_blocks(int(tokens)))


def history_count_words(experts):
    """int32 words of one demand record."""
    return int(lib().ferry_history_count_words(int(experts)))


# ------------------------------------------------------------------------------------------
# The reference's pybind names (ferry/csrc/expert_ops.cpp:144-157)
# ------------------------------------------------------------------------------------------

_numel, _data_ptr = torch.Tensor.numel, torch.Tensor.data_ptr
_get_device, _is_contiguous = torch.Tensor.get_device, torch.Tensor.is_contiguous
_dtype = attrgetter('dtype')


def _joined(tensors, dtype, device, unit=1):
    """(address, elements, owner) of the tensors one after the other, as ``dtype``: in place where
    they already follow each other in memory (views that split one tensor), else concatenated.
    ``owner`` keeps the memory alive.  Each tensor must hold a multiple of ``unit`` elements."""
    # builtin calls over the whole list: a Python loop over 100 views takes twice the time
    sizes = list(map(_numel, tensors))
    if math.gcd(unit, *sizes) != unit:
        raise RuntimeError(f'every part must hold whole rows of {unit} elements')
    parts = tensors if all(sizes) else [t for t in tensors if t.numel()]
    if not parts:
        return 0, 0, None
    if parts is not tensors:
        sizes = list(map(_numel, parts))
    at = list(map(_data_ptr, parts))
    ends = list(map(add, at, map(dtype.itemsize.__mul__, sizes)))
    if (at[1:] != ends[:-1] or set(map(_dtype, parts)) != {dtype}
            or set(map(_get_device, parts)) != {device.index} or not all(map(_is_contiguous, parts))):
        cat = torch.cat([u.reshape(-1) for u in tensors]).to(dtype).contiguous()
        _dev(cat, 'tensors of a group list')
        return cat.data_ptr(), cat.numel(), cat
    return at[0], (ends[-1] - at[0]) // dtype.itemsize, tensors


def execute_experts(cache, input, routing_weights, slots, rows, cols, hidden, intermediate):
    """Routed-expert MLPs of every (slot, rows, cols) group (expert_ops.cpp:16-45).

    Output i is ``down(silu(x Wg^T) * (x Wu^T)) * routing_weights[rows[i], cols[i]]`` for
    ``x = input[rows[i]]``, one bf16 [len(rows[i]), hidden] tensor per group.
    """
    _dev(cache, 'cache', torch.bfloat16)
    if cache.dim() != 2 or cache.shape[1] != 3 * hidden * intermediate:
        raise RuntimeError('cache must be [cap, 3 * hidden * intermediate]')
    if input.dim() != 2 or input.shape[1] != hidden:
        raise RuntimeError('input must be [rows, hidden]')
    if routing_weights.dim() != 2 or routing_weights.shape[0] != input.shape[0]:
        raise RuntimeError('routing_weights must be [rows, topk]')
    if not (len(slots) == len(rows) == len(cols)):
        raise RuntimeError('slots, rows and cols must have the same length')
    G = len(slots)
    if G == 0:
        return []
    if G > MAX_EXPERTS:
        raise RuntimeError(f'at most {MAX_EXPERTS} groups per call')
    slots = np.asarray(slots, np.int64)
    if slots.min() < 0 or slots.max() >= cache.shape[0]:
        raise RuntimeError('slot out of range')
    # before anything is queued: the group starts are written to memory on the input's device
    _dev(input, 'input', torch.bfloat16, contiguous=False)
    _dev(routing_weights, 'routing_weights', torch.bfloat16, contiguous=False)
    sizes = [r.numel() for r in rows]
    dev = input.device
    rows_at, P, _rows = _joined(rows, torch.int64, dev)
    cols_at, n_cols, _cols = _joined(cols, torch.int64, dev)
    if n_cols < P:
        raise RuntimeError('cols must name a weight for every row')
    starts = torch.empty(G + 1, dtype=torch.int64, device=dev)
    counts = np.array(sizes, np.int32)
    check(lib().ferry_starts(counts.tobytes(), G, starts.data_ptr(), _stream_of(starts)), 'starts')
    act = torch.empty((max(P, 1), intermediate), dtype=torch.bfloat16, device=dev)
    out = torch.empty((max(P, 1), hidden), dtype=torch.bfloat16, device=dev)
    if P:
        expert_ffn(cache, input.contiguous(), routing_weights.contiguous(), starts, rows_at, cols_at,
                   np.arange(G), slots, hidden, intermediate, act, out, out_mode=1, experts=G,
                   counts=counts)
    return list(out[:P].split(sizes))


def pack_dispatch(hidden, selected, weights, send_idx, send_ids, experts):
    """Dispatch packet rows ``[x (2H B) | weights in send_ids order (2k B) | IDs (k B)]``.

    Reference: expert_ops.cpp:88-104, on the ``ferry_pack_dispatch`` kernel.  At world = 1 the
    packet never leaves the GPU (the fused path reads the routing weights in send_ids order
    straight from the layout kernel); this gives callers of the reference's Transport the same
    bytes.
    """
    n, k = send_ids.shape
    T, H = hidden.shape
    payload = torch.empty((n, 2 * H + 3 * k), dtype=torch.uint8, device=hidden.device)
    check(lib().ferry_pack_dispatch(
        _dev(hidden, 'hidden', torch.bfloat16), T, H, _dev(selected, 'selected', torch.int64),
        _dev(weights, 'weights', torch.bfloat16), selected.shape[1],
        _dev(send_idx, 'send_idx', torch.int64), _dev(send_ids, 'send_ids', torch.int64), n, k,
        experts, payload.data_ptr(), _stream_of(hidden)), 'pack_dispatch')
    return payload


def unpack_dispatch(raw, hidden, topk):
    """Split packet rows back into bf16 [m, H] hidden states and [m, k] weights
    (expert_ops.cpp:106-111), on the ``ferry_unpack_dispatch`` kernel."""
    m = raw.shape[0]
    if raw.dim() != 2 or raw.shape[1] != 2 * hidden + 3 * topk:
        raise RuntimeError('raw must be uint8 [m, 2 * hidden + 3 * topk]')
    x = torch.empty((m, hidden), dtype=torch.bfloat16, device=raw.device)
    w = torch.empty((m, topk), dtype=torch.bfloat16, device=raw.device)
    check(lib().ferry_unpack_dispatch(_dev(raw, 'raw', torch.uint8), m, hidden, topk,
                                      x.data_ptr(), w.data_ptr(), _stream_of(raw)), 'unpack_dispatch')
    return [x, w]


def reduce_partials(parts, rows, received, hidden, like):
    """fp32 sum of expert outputs per received row, ascending group order, then bf16 (:76-83)."""
    if len(parts) == 0:
        return torch.zeros((received, hidden), dtype=torch.bfloat16, device=like.device)
    _dev(parts[0], 'parts', contiguous=False)   # the sums are written to memory on this device
    dev = parts[0].device
    part_at, n, _parts = _joined(parts, torch.bfloat16, dev, unit=hidden)
    if part_at % 16:
        _parts = torch.cat([p.reshape(-1) for p in parts])
        part_at = _parts.data_ptr()
    rows_at, entries, _rows = _joined(rows, torch.int64, dev)
    if entries > n // hidden:
        raise RuntimeError('rows must not outnumber the rows of parts')
    out = torch.empty((received, hidden), dtype=torch.bfloat16, device=dev)
    ws = torch.empty(lib().ferry_reduce_rows_full_workspace_bytes(received, entries) // 4,
                     dtype=torch.int32, device=dev)
    check(lib().ferry_reduce_rows(part_at, entries, hidden, rows_at, received, out.data_ptr(),
                                  ws.data_ptr(), ws.numel() * 4, _stream_of(out)),
          'reduce_partials')
    bad = int(ws[received].item())
    if bad:
        raise RuntimeError(f'reduce_partials: {bad} row(s) outside [0, {received})')
    return out


def scatter_returned(returned, send_idx, tokens):
    """Add returned rows back to their tokens in fp32 (expert_ops.cpp:86-92)."""
    output = torch.zeros((tokens, returned.shape[1]), dtype=torch.float32, device=returned.device)
    if returned.shape[0]:
        output.index_add_(0, send_idx, returned.float())
    return output.to(returned.dtype)
