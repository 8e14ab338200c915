"""The network in front of the determinants: operators between a configuration and its orbital
(or pairing) matrix, for training and for sampling one token at a time. Each runs as hand-written
HIP kernels of ``libfermix_amd.so``; there is no CPU path.

* ``distance_buckets`` / ``relative_bias``: a learned bias (or a learned pairing function) of the
  distance of two positions, by buckets, with its gradient;
* ``attention``: softmax attention with that bias, over whole sequences, with its gradients;
* ``attention_step``: attention of one new token over a paged key-value cache;
* ``residual_norm``: the norms before and after a block, fused with its gate and residual scale,
  with their gradients.

Element types are float32, bfloat16 and float16 (``relative_bias`` also float64); scores,
statistics and sums are held in float32 and each result is rounded once. For the 16-bit types attention's
weights (and what its gradient makes of them) are rounded to the type a first time, as an operand of
the next product. Every result is deterministic: its sums are in an order that depends on sizes and
lengths, for the bias' gradient and the float32 norms also on the tensors' alignment to 16 bytes.
Gradients are reverse mode, once (``torch.autograd``); forward mode and ``torch.func`` transforms raise.
``torch.jit.trace`` records calls, but for ``attention_step``.
"""

import ctypes
import math

import torch
import torch.autograd.forward_ad as fwAD
from torch.autograd.function import once_differentiable

from . import _lib
from ._diff import _dual
from ._kernels import _ptr, _stream, _workspace
from ._lib import (
    FX_MAX_BIAS_HEADS, FX_MAX_COLUMNS, FX_MAX_POSITIONS, FX_MAX_RADIUS, FX_MAX_SCALE, FX_MAX_STEP_TOKENS, FX_MIN_SCALE,
    FX_NORM_LAYER, FX_NORM_POST, FX_NORM_PRE, check, lib,
)

_TYPES = {torch.float32: _lib.FX_F32, torch.bfloat16: _lib.FX_BF16, torch.float16: _lib.FX_F16}
_BIAS_TYPES = {**_TYPES, torch.float64: _lib.FX_F64}
MAX_BUCKETS = 256  # of relative_bias
MAX_ATTENTION_BUCKETS = 64
MAX_DIM = 128


# ------------------------------------------------------------------ checks


def _tensor(x, name, like=None, dtype=None, dim=None):
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name}: expected a torch.Tensor, got {type(x).__name__}")
    if dtype is not None and x.dtype not in dtype:
        raise TypeError(f"{name}: expected {' or '.join(str(d) for d in dtype)}, got {x.dtype}")
    if dim is not None and x.dim() != dim:
        raise ValueError(f"{name}: expected {dim} dimensions, got {tuple(x.shape)}")
    if like is not None and x.device != like.device:
        raise ValueError(f"{name} is on {x.device}, expected {like.device}")
    return x


def _on_device(x):
    if not x.is_cuda:
        from .api import FermixDeviceError

        raise FermixDeviceError("fermix_amd runs on a ROCm GPU only; move the inputs to a 'cuda' device")


_INT = (torch.int32, torch.int64)


def _int32(x):
    return x.to(torch.int32).contiguous()


def _once(backward):
    """A backward without a derivative of its own (asking for one raises); the check costs nothing where
    none can be asked for."""
    checked = once_differentiable(backward)

    def either(ctx, *grads):
        return checked(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)

    return either


def _wants_grad(*xs):
    return torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in xs)


def _through_autograd(*xs):
    """Whether a call goes through its autograd function: where a gradient is wanted, and under torch.jit.trace, which
    records that and would otherwise record the allocation of the results alone."""
    return _wants_grad(*xs) or torch.jit.is_tracing()


def _refuse_forward_mode(*xs):
    """A dual tensor that needs no gradient would go to the kernels as its primal and come back without a tangent. (There
    are none outside a level of forward mode: looking at each tensor then is 1 us of every call.)"""
    if fwAD._current_level >= 0 and any(x is not None and _dual(x) for x in xs):
        raise NotImplementedError("fermix_amd's network operators have no forward mode: differentiate them in reverse mode")


def _call(name, device_of, *args):
    """One C entry point on the input's device and its current stream."""
    if device_of.get_device() == torch._C._cuda_getDevice():
        check(getattr(lib(), name)(*args, _stream(device_of)), name)
    else:
        with torch.cuda.device(device_of.device):
            check(getattr(lib(), name)(*args, _stream(device_of)), name)


def _check_buckets(buckets, table, most):
    _tensor(buckets, "buckets", table, (torch.uint8,), 1)
    if buckets.numel() % 2 == 0 or buckets.numel() > 2 * FX_MAX_RADIUS + 1:
        raise ValueError(
            f"buckets: expected 2 R + 1 entries for the distances -R .. R, R <= {FX_MAX_RADIUS}, got {buckets.numel()}"
        )
    if not 1 <= table.shape[0] <= most:
        raise ValueError(f"table: expected 1 to {most} buckets, got {table.shape[0]}")
    return buckets.contiguous()


# ------------------------------------------------------------------ distance buckets


def distance_buckets(num_buckets=32, max_distance=128, *, bidirectional=True, device="cuda"):
    """Bucket of each distance key - query in -max_distance .. max_distance, as the uint8 tensor
    of 2 max_distance + 1 entries that the operators below take (distances past its ends are in
    its end buckets). Of the buckets of one sign, the first half hold one distance each, the
    others grow by a constant factor up to max_distance; with ``bidirectional`` half the buckets
    are for keys after the query, else those share the bucket of distance 0. The limits
    are found in whole numbers. Any other map (of a lattice's displacements, say) can be
    given in its place."""
    side = num_buckets // 2 if bidirectional else num_buckets
    single = side // 2
    if single < 1 or num_buckets > MAX_BUCKETS:
        raise ValueError(f"num_buckets: expected {4 if bidirectional else 2} to {MAX_BUCKETS}, got {num_buckets}")
    if not single < max_distance <= FX_MAX_RADIUS:
        raise ValueError(f"max_distance: expected {single + 1} to {FX_MAX_RADIUS}, got {max_distance}")
    grown = side - single
    row, b = [], 0
    for n in range(max_distance + 1):
        # bucket single + t begins at single (max_distance / single)^(t / grown)
        if n <= single:
            b = n
        while n > single and b + 1 < side and n**grown >= single ** (side - b - 1) * max_distance ** (b + 1 - single):
            b += 1
        row.append(b)
    after = [side + row[d] if bidirectional else row[0] for d in range(1, max_distance + 1)]
    return torch.tensor(row[:0:-1] + [row[0]] + after, dtype=torch.uint8, device=device)


# ------------------------------------------------------------------ relative bias


def _bias_forward(table, buckets, q, k):
    B, Q = q.shape
    K, H = k.shape[1], table.shape[1]
    out = torch.empty((B, H, Q, K), dtype=table.dtype, device=table.device)
    _call("fx_relative_bias", table, _ptr(table), _ptr(buckets), buckets.numel() // 2, table.shape[0], _ptr(q), _ptr(k),
          B, H, Q, K, _BIAS_TYPES[table.dtype], _ptr(out))
    return out


class _RelativeBias(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, buckets, q, k):
        ctx.save_for_backward(buckets, q, k)
        ctx.shape = table.shape
        return _bias_forward(table.contiguous(), buckets, q, k)

    @staticmethod
    @_once
    def backward(ctx, grad):
        buckets, q, k = ctx.saved_tensors
        nb, H = ctx.shape
        grad = grad.contiguous()
        B, Q, K = q.shape[0], q.shape[1], k.shape[1]
        out = torch.empty((nb, H), dtype=grad.dtype, device=grad.device)
        kind = _BIAS_TYPES[grad.dtype]
        ws, wsb = _workspace(lib().fx_relative_bias_grad_workspace(nb, B, H, Q, K, kind), grad.device)
        _call("fx_relative_bias_grad", grad, _ptr(grad), _ptr(buckets), buckets.numel() // 2, nb, _ptr(q), _ptr(k), B, H,
              Q, K, kind, _ptr(out), _ptr(ws), wsb)
        return out, None, None, None


def relative_bias(table, buckets, q_pos, k_pos):
    """Learned bias of the distance of two positions, by buckets: (..., H, Q, K) with

        out[..., h, i, j] = table[bucket(k_pos[..., j] - q_pos[..., i]), h]

    table (num_buckets, H) float32, float64, bfloat16 or float16, num_buckets <= 256, H <= 4096; buckets from
    ``distance_buckets`` (entries past the table count as its last); q_pos (..., Q) and k_pos
    (..., K) int32 (or int64 values of its range), leading dimensions broadcast. As a pairing
    function of the electrons' distance the result goes straight into ``slogpf``. Differentiable in
    table."""
    _tensor(table, "table", dtype=_BIAS_TYPES, dim=2)
    buckets = _check_buckets(buckets, table, MAX_BUCKETS)
    q, k = (_tensor(x, n, table, _INT) for x, n in ((q_pos, "q_pos"), (k_pos, "k_pos")))
    if not q.dim() or not k.dim():
        raise ValueError("q_pos and k_pos: expected (..., Q) and (..., K)")
    if not 1 <= table.shape[1] <= FX_MAX_BIAS_HEADS:
        raise ValueError(f"table: expected 1 to {FX_MAX_BIAS_HEADS} heads, got {table.shape[1]}")
    if max(q.shape[-1], k.shape[-1]) > FX_MAX_POSITIONS:
        raise ValueError(f"q_pos and k_pos: expected up to {FX_MAX_POSITIONS} positions, got {q.shape[-1]} and {k.shape[-1]}")
    _refuse_forward_mode(table)
    _on_device(table)
    lead = q.shape[:-1]
    if len(lead) != 1 or k.shape[:-1] != lead:  # broadcasting takes as long as a small launch
        lead = torch.broadcast_shapes(lead, k.shape[:-1])
        q, k = (x.expand(lead + x.shape[-1:]).reshape(math.prod(lead), x.shape[-1]) for x in (q, k))
    q, k = _int32(q), _int32(k)
    if _through_autograd(table):
        out = _RelativeBias.apply(table, buckets, q, k)
    else:
        out = _bias_forward(table.contiguous(), buckets, q, k)
    return out if len(lead) == 1 else out.reshape(lead + out.shape[1:])


# ------------------------------------------------------------------ attention


def _rows(x):
    """x with its last dimension contiguous."""
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()


def _attention_args(q, k, v, table, buckets, q_pos, k_pos, lengths, q_lengths, mask, causal, offset, scale, out, stats,
                    low=None):
    B, N, H, D = q.shape
    K, Hkv = k.shape[1], k.shape[2]
    qb, qn, qh, _ = q.stride()
    kb, kn, kh, _ = k.stride()
    vb, vn, vh, _ = v.stride()
    radius, count = (0, 0) if table is None else (buckets.shape[0] // 2, table.shape[0])
    return _lib.FxAttention(
        B, N, K, H, Hkv, D, _TYPES[q.dtype], causal, offset, radius, count, scale,
        q.data_ptr(), k.data_ptr(), v.data_ptr(), qb, qn, qh, kb, kn, kh, vb, vn, vh,
        _ptr(table), _ptr(buckets), _ptr(q_pos), _ptr(k_pos), _ptr(lengths), _ptr(q_lengths), _ptr(mask),
        out.data_ptr(), _ptr(low), _ptr(stats),
    )


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, table, *rest):
        B, N, H, D = q.shape
        out = torch.empty((B, N, H, D), dtype=q.dtype, device=q.device)
        stats = torch.empty((B, H, N, 2), dtype=torch.float32, device=q.device)
        a = _attention_args(q, k, v, table, *rest, out, stats)
        low = None
        if lib().fx_attention_keeps_low(ctypes.byref(a)):
            low = torch.empty((B, N, H, D), dtype=torch.float16, device=q.device)
            a.out_low = low.data_ptr()
        _call("fx_attention_forward", q, ctypes.byref(a))
        buckets, q_pos, k_pos, lengths, q_lengths, mask, *ctx.plain = rest
        ctx.save_for_backward(q, k, v, table, buckets, q_pos, k_pos, lengths, q_lengths, mask, out, stats, low)
        return out

    @staticmethod
    @_once
    def backward(ctx, grad):
        q, k, v, table, buckets, q_pos, k_pos, lengths, q_lengths, mask, out, stats, low = ctx.saved_tensors
        a = _attention_args(q, k, v, table, buckets, q_pos, k_pos, lengths, q_lengths, mask, *ctx.plain, out, stats, low)
        grad = grad.contiguous()
        dq, dk, dv = (torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in (q, k, v))
        dt = torch.empty_like(table) if ctx.needs_input_grad[3] else None
        a.grad_out = _ptr(grad)
        a.grad_q, a.grad_k, a.grad_v, a.grad_table = _ptr(dq), _ptr(dk), _ptr(dv), _ptr(dt)
        ws, wsb = _workspace(lib().fx_attention_grad_workspace(ctypes.byref(a)), q.device)
        _call("fx_attention_grad", q, ctypes.byref(a), _ptr(ws), wsb)
        return (dq, dk, dv, dt) + (None,) * 9


def _check_heads(q, k, v):
    if q.shape[-1] != k.shape[-1] or k.shape != v.shape:
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not fit")
    if not 1 <= q.shape[-1] <= MAX_DIM:
        raise ValueError(f"expected a head dimension of 1 to {MAX_DIM}, got {q.shape[-1]}")
    if k.shape[-2] < 1 or q.shape[-2] < 1 or q.shape[-2] % k.shape[-2]:
        raise ValueError(f"the {q.shape[-2]} heads of q are no multiple of the {k.shape[-2]} of k and v")


def _check_bias(table, buckets, heads, like):
    if (table is None) != (buckets is None):
        raise ValueError("table and buckets come together")
    if table is None:
        return None, None
    _tensor(table, "table", like, (torch.float32,), 2)
    if table.shape[1] != heads:
        raise ValueError(f"table: expected (num_buckets, {heads}), got {tuple(table.shape)}")
    return table.contiguous(), _check_buckets(buckets, table, MAX_ATTENTION_BUCKETS)


def _check_scale(scale, dim):
    scale = 1.0 / math.sqrt(dim) if scale is None else float(scale)
    if not FX_MIN_SCALE <= scale <= FX_MAX_SCALE:
        raise ValueError(f"scale: expected {FX_MIN_SCALE} to {FX_MAX_SCALE}, got {scale}")
    return scale


def attention(q, k, v, *, table=None, buckets=None, q_pos=None, k_pos=None, lengths=None, q_lengths=None, mask=None,
              causal=False, offset=0, scale=None):
    """Softmax attention with a learned relative position bias: out (B, N, H, D) of

        softmax over keys of (scale q k^T + table[bucket(k_pos - q_pos)]), times v.

    q (B, N, H, D), k and v (B, K, Hkv, D), float32, bfloat16 or float16, any strides (D is
    made contiguous if it is not), D <= 128, H a multiple of Hkv: heads h Hkv / H share a key head.
    table (num_buckets, H) float32 (up to 64 buckets) with buckets as for ``relative_bias``, or
    None for no bias. Positions: q_pos (B, N) and k_pos (B, K), or None: offset + i and j. Positions
    and lengths are int32, or int64 of its range.
    lengths (B,): keys at or past it are left out; mask (B, K) bool: keys that are False are; both may
    hide anything, NaN and infinities included. causal: query i sees keys j <= offset + i (what is
    hidden by it alone has to be finite). q_lengths (B,): queries at or past it give 0. A query with no key
    gives 0 and no gradient (its cotangent has to be finite). An entry -inf of table forbids its bucket. scale,
    1e-30 to 1e30, defaults to 1 / sqrt(D).

    For bfloat16 and float16 the softmax' weights are rounded to the type for their product with v, and dS in the
    gradient likewise: out has 1.2 times, dq, dk and dv 1.4 times the error of one rounding. (float16's are scaled by
    powers of two before, so that small weights and cotangents keep their digits.)

    Differentiable in q, k, v and table. The gradient keeps q, k, v, out and two float32 a query and
    head; for 16-bit types past 128 queries or keys also what out lost to rounding, as float16."""
    _tensor(q, "q", dtype=_TYPES, dim=4)
    _tensor(k, "k", q, (q.dtype,), 4)
    _tensor(v, "v", q, (q.dtype,), 4)
    _check_heads(q, k, v)
    B, N, H, D = q.shape
    K = k.shape[1]
    if k.shape[0] != B:
        raise ValueError(f"q has {B} samples, k and v {k.shape[0]}")
    if N > FX_MAX_POSITIONS or K > FX_MAX_POSITIONS:
        raise ValueError(f"expected up to {FX_MAX_POSITIONS} queries and keys, got {N} and {K}")
    table, buckets = _check_bias(table, buckets, H, q)
    if (q_pos is None) != (k_pos is None):
        raise ValueError("q_pos and k_pos come together")
    for x, name, shape in ((q_pos, "q_pos", (B, N)), (k_pos, "k_pos", (B, K)), (lengths, "lengths", (B,)),
                           (q_lengths, "q_lengths", (B,)), (mask, "mask", (B, K))):
        if x is None:
            continue
        _tensor(x, name, q, (torch.bool,) if name == "mask" else _INT)
        if x.shape != shape:
            raise ValueError(f"{name}: expected {shape}, got {tuple(x.shape)}")
    offset = int(offset)
    if not 0 <= offset <= 2**31 - 1 - max(N, K):
        raise ValueError(f"offset: expected 0 to {2**31 - 1 - max(N, K)}, got {offset}")
    scale = _check_scale(scale, D)
    _refuse_forward_mode(q, k, v, table)
    _on_device(q)
    q, k, v = _rows(q), _rows(k), _rows(v)
    q_pos, k_pos, lengths, q_lengths = (None if x is None else _int32(x) for x in (q_pos, k_pos, lengths, q_lengths))
    mask = None if mask is None else mask.contiguous()
    rest = (buckets, q_pos, k_pos, lengths, q_lengths, mask, bool(causal), offset, scale)
    if _through_autograd(q, k, v, table):
        return _Attention.apply(q, k, v, table, *rest)
    out = torch.empty((B, N, H, D), dtype=q.dtype, device=q.device)
    _call("fx_attention_forward", q, ctypes.byref(_attention_args(q, k, v, table, *rest, out, None)))
    return out


def attention_step(q, k_cache, v_cache, pages, lengths, *, k=None, v=None, table=None, buckets=None, scale=None):
    """Attention of one new token of each sample over a paged key-value cache: out (B, H, D).

    q (B, H, D); k_cache and v_cache (P, page, Hkv, D) contiguous; pages (B, M): token t of
    sample b is token t % page of cache page pages[b, t // page]; lengths (B,): the tokens
    that a sample has in the cache (both int32, or int64 of its range). With k and v (B, Hkv, D) the new token's are stored as token
    lengths[b] (in place; the caller counts lengths up) and its query, at that position, attends
    to tokens 0 .. lengths[b]; a sample of negative length is left out. Without them the query is that
    of the cache's last token. table, buckets and scale as for ``attention``; a key's distance
    is its token less the query's. Samples may share pages that they only read (walkers that branched).
    A sample with no token gives 0; one that its row of pages cannot hold, or that names a page outside
    the cache, gives NaN. For bfloat16 and float16 with shared key heads the weights are rounded to the type, as in
    ``attention``. No gradient."""
    _tensor(q, "q", dtype=_TYPES, dim=3)
    for x, name in ((k_cache, "k_cache"), (v_cache, "v_cache")):
        _tensor(x, name, q, (q.dtype,), 4)
        if not x.is_contiguous():
            raise ValueError(f"{name}: expected a contiguous tensor")
    _check_heads(q, k_cache, v_cache)
    B, H, D = q.shape
    P, page, Hkv, _ = k_cache.shape
    if page < 1:
        raise ValueError("k_cache: a page holds at least one token")
    if (k is None) != (v is None):
        raise ValueError("k and v come together")
    for x, name in ((k, "k"), (v, "v")):
        if x is not None:
            _tensor(x, name, q, (q.dtype,), 3)
            if x.shape != (B, Hkv, D):
                raise ValueError(f"{name}: expected {(B, Hkv, D)}, got {tuple(x.shape)}")
    _tensor(pages, "pages", q, _INT, 2)
    _tensor(lengths, "lengths", q, _INT, 1)
    if pages.shape[0] != B or lengths.shape[0] != B:
        raise ValueError(f"pages {tuple(pages.shape)} and lengths {tuple(lengths.shape)} do not fit {B} samples")
    if pages.shape[1] * page > FX_MAX_STEP_TOKENS or page * Hkv * D >= 2**32:
        raise ValueError(f"expected pages of up to {FX_MAX_STEP_TOKENS} tokens for a sample, of less than 2^32 elements each")
    table, buckets = _check_bias(table, buckets, H, q)
    scale = _check_scale(scale, D)
    _refuse_forward_mode(q, k_cache, v_cache, k, v, table)
    _on_device(q)
    if _wants_grad(q, k_cache, v_cache, k, v, table):
        raise NotImplementedError("attention_step has no gradient: call it under torch.no_grad(), or train with attention")
    if torch.jit.is_tracing():
        raise NotImplementedError("attention_step writes the caches in place, which torch.jit.trace does not record")
    q, pages, lengths = q.contiguous(), _int32(pages), _int32(lengths)
    k, v = (None if x is None else x.contiguous() for x in (k, v))
    out = torch.empty((B, H, D), dtype=q.dtype, device=q.device)
    radius, count = (0, 0) if table is None else (buckets.shape[0] // 2, table.shape[0])
    a = ctypes.byref(_lib.FxAttentionStep(
        B, H, Hkv, D, _TYPES[q.dtype], P, page, pages.shape[1], radius, count, scale, q.data_ptr(), _ptr(k), _ptr(v),
        k_cache.data_ptr(), v_cache.data_ptr(), pages.data_ptr(), lengths.data_ptr(), _ptr(table), _ptr(buckets), out.data_ptr(),
    ))
    ws, wsb = _workspace(lib().fx_attention_step_workspace(a), q.device)
    _call("fx_attention_step_run", q, a, _ptr(ws), wsb)
    if k is not None:
        torch.autograd.graph.increment_version((k_cache, v_cache))  # a graph that saved the caches must not use them
    return out


# ------------------------------------------------------------------ residual norm

_COLUMNS = ("post_weight", "post_bias", "scale", "pre_weight", "pre_bias")


def _gate_view(gate, x):
    """How x's rows are seen as samples x rows so that the gate is constant over rows, over
    samples and rows, or over neither: (samples, rows, swapped, gate strides). swapped: the samples
    are the last row dimension (a gate of the position alone)."""
    lead = x.shape[:-1]
    B, N = math.prod(lead[:-1]), lead[-1] if lead else 1
    if gate is None:
        return B, N, False, (0, 0, 0)
    shape = (1,) * (x.dim() - gate.dim()) + tuple(gate.shape)
    C = x.shape[-1]
    if gate.dim() > x.dim() or any(s not in (1, n) for s, n in zip(shape, x.shape)):
        raise ValueError(f"gate: {tuple(gate.shape)} does not broadcast to {tuple(x.shape)}")
    gc = int(shape[-1] != 1 or C == 1)
    outer, inner = shape[:-2], shape[-2] if len(shape) > 1 else 1
    full_n, none_n = inner == N, inner == 1
    full_b, none_b = tuple(outer) == tuple(lead[:-1]), all(s == 1 for s in outer)
    w = C if gc else 1
    if full_b and full_n:
        return B, N, False, (N * w, w, gc)
    if full_b and none_n:
        return B, N, False, (w, 0, gc)
    if none_b and none_n:
        return 1, B * N, False, (0, 0, gc)
    if none_b and full_n:
        return N, B, True, (w, 0, gc)
    raise ValueError(
        f"gate: {tuple(gate.shape)} is broadcast over some of the leading dimensions of {tuple(x.shape)}; expected all or none"
    )


def _norm_args(x, h, gate, columns, alpha, eps, flags, y=None, z=None, stats=None):
    """x, h contiguous."""
    C = x.shape[-1]
    S, R, swapped, (gs, gr, gc) = _gate_view(gate, x)
    # rows of x: sample s, row r is row s R + r, or r S + s where the samples are the inner dimension
    s, r = (C, S * C) if swapped else (R * C, C)
    wide = next((t.dtype for t in columns if t is not None), torch.float32)
    return _lib.FxResidualNorm(
        S, R, C, _TYPES[x.dtype], _TYPES[wide], flags, eps, alpha, x.data_ptr(), h.data_ptr(), _ptr(gate), s, r, s, r, gs, gr, gc,
        s, r, *(_ptr(t) for t in columns), _ptr(y), _ptr(z), _ptr(stats),
    )


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, h, gate, post_weight, post_bias, scale, pre_weight, pre_bias, alpha, eps, flags):
        columns = (post_weight, post_bias, scale, pre_weight, pre_bias)
        stats = torch.empty(x.shape[:-1] + (4,), dtype=torch.float32, device=x.device)
        y = torch.empty_like(x)
        z = torch.empty_like(x) if flags & FX_NORM_PRE else None
        a = _norm_args(x, h, gate, columns, alpha, eps, flags, y, z, stats)
        _call("fx_residual_norm_forward", x, ctypes.byref(a))
        ctx.save_for_backward(x, h, gate, stats, *columns)
        ctx.plain = alpha, eps, flags
        ctx.set_materialize_grads(False)
        return y if z is None else (y, z)

    @staticmethod
    @_once
    def backward(ctx, grad_y, grad_z=None):
        if grad_y is None and grad_z is None:
            return (None,) * 11
        x, h, gate, stats, *columns = ctx.saved_tensors
        a = _norm_args(x, h, gate, columns, *ctx.plain, stats=stats)
        grad_y, grad_z = (None if g is None else g.contiguous() for g in (grad_y, grad_z))
        dx, dh = torch.empty_like(x), torch.empty_like(h)
        dgate = None if gate is None else torch.empty_like(gate)
        dcolumns = [
            torch.empty_like(t) if t is not None and need else None for t, need in zip(columns, ctx.needs_input_grad[3:8])
        ]
        a.grad_y, a.grad_z = _ptr(grad_y), _ptr(grad_z)
        a.grad_x, a.grad_h, a.grad_gate = _ptr(dx), _ptr(dh), _ptr(dgate)
        for name, t in zip(_COLUMNS, dcolumns):
            setattr(a, "grad_" + name, _ptr(t))
        ws, wsb = _workspace(lib().fx_residual_norm_grad_workspace(ctypes.byref(a)), x.device)
        _call("fx_residual_norm_grad", x, ctypes.byref(a), _ptr(ws), wsb)
        return (dx, dh, dgate, *dcolumns, None, None, None)


def residual_norm(x, h, *, post_weight=None, post_bias=None, gate=None, scale=None, pre_weight=None, pre_bias=None,
                  norm="rms", eps=1e-6, post_norm=True, pre_norm=True):
    """The end of a residual block and the beginning of the next in one pass: (y, z) with

        y = x + scale * gate * (norm(h) * post_weight + post_bias)     the residual stream
        z = norm(y) * pre_weight + pre_bias                            the next block's input

    x and h (..., C) float32, bfloat16 or float16, C <= 8192. norm: "rms", t / sqrt(mean(t^2) + eps),
    or "layer", the same of t - mean(t). Weights, biases and scale (C,) of x's type or float32 (all
    alike), each optional; scale may be a number. gate: any shape that broadcasts to x's, over all
    of the dimensions before the last two or none (a gate per element, row, sample, channel, ..), of
    x's type. post_norm=False leaves h as it is; pre_norm=False returns y alone.

    z is formed from y before y is rounded. Differentiable in every tensor; the gradient keeps x, h and
    four float32 a row and forms the rest again."""
    _tensor(x, "x", dtype=_TYPES)
    _tensor(h, "h", x, (x.dtype,))
    if not x.dim() or x.shape != h.shape:
        raise ValueError(f"x {tuple(x.shape)} and h {tuple(h.shape)}: expected one shape (..., C)")
    C = x.shape[-1]
    if not 1 <= C <= FX_MAX_COLUMNS:
        raise ValueError(f"expected 1 to {FX_MAX_COLUMNS} columns, got {C}")
    if norm not in ("rms", "layer"):
        raise ValueError(f'norm: expected "rms" or "layer", got {norm!r}')
    if not (post_norm or (post_weight is None and post_bias is None)):
        raise ValueError("post_weight and post_bias belong to post_norm")
    if not (pre_norm or (pre_weight is None and pre_bias is None)):
        raise ValueError("pre_weight and pre_bias belong to pre_norm")
    if not eps >= 0.0:
        raise ValueError(f"eps: expected a number that is not negative, got {eps}")
    alpha = 1.0
    if scale is not None and not isinstance(scale, torch.Tensor):
        alpha, scale = float(scale), None
    columns = [post_weight, post_bias, scale, pre_weight, pre_bias]
    kinds = set()
    for i, (t, name) in enumerate(zip(columns, _COLUMNS)):
        if t is None:
            continue
        _tensor(t, name, x, (x.dtype, torch.float32))
        if t.shape != (C,):
            raise ValueError(f"{name}: expected ({C},), got {tuple(t.shape)}")
        kinds.add(t.dtype)
        columns[i] = t.contiguous()
    if len(kinds) > 1:
        raise TypeError("weights, biases and scale: expected one type")
    if gate is not None:
        _tensor(gate, "gate", x, (x.dtype,))
        _gate_view(gate, x)
        gate = gate.contiguous()
    _refuse_forward_mode(x, h, gate, *columns)
    _on_device(x)
    flags = (FX_NORM_LAYER if norm == "layer" else 0) | (FX_NORM_POST if post_norm else 0) | (FX_NORM_PRE if pre_norm else 0)
    x, h = x.contiguous(), h.contiguous()
    if _through_autograd(x, h, gate, *columns):
        return _ResidualNorm.apply(x, h, gate, *columns, alpha, float(eps), flags)
    y = torch.empty_like(x)
    z = torch.empty_like(x) if pre_norm else None
    _call("fx_residual_norm_forward", x, ctypes.byref(_norm_args(x, h, gate, columns, alpha, float(eps), flags, y, z)))
    return (y, z) if pre_norm else y


__all__ = ["distance_buckets", "relative_bias", "attention", "attention_step", "residual_norm"]
