"""MLP blocks with experts: router, products grouped by expert, and the sum
that brings the experts' rows back to their tokens.

One block for tokens ``x`` [T, D], expert weights ``w1`` [E, H, D], ``w2``
[E, D, H] and router logits [T, E]::

    plan = route(logits, k)
    h = grouped_gemm(x, w1, plan.offsets, b1, 'gelu', rows=plan.tokens)
    y = grouped_gemm(h, w2, plan.offsets, b2, 'bias')
    x = combine(y, plan.positions, plan.weights, residual=x)

The plan stays on the device: no call waits for it.  With MXFP4 weights,
``x`` and ``h`` pass through :func:`.mxfp4.quantize` first.

Each call runs hand-written HIP kernels on the operands' device, on the
caller's current stream there.  Memory beside the operands comes from torch's
allocator: the result and, for :func:`grouped_gemm` of many rows, a workspace;
a call that is given both (a capture that torch does not know of) allocates
nothing.  There is no backward pass and no forward-mode derivative.
"""
import collections
import functools

from . import checks, mxfp4, native

EPILOGUES = {'none': 0, 'gelu': 1, 'bias_gelu': 1, 'bias': 3}


class Plan(collections.namedtuple(
        'Plan', ('experts', 'weights', 'tokens', 'positions', 'offsets',
                 'counts'))):
    """What :func:`route` decides.

    ``experts`` int32 [T, k]: each token's experts, best first (-1: none).
    ``weights`` fp32 [T, k]: their weights (0: none).
    ``tokens`` int32 [T * k]: the token of each expert row (-1 behind the
    last one).  ``positions`` int32 [T, k]: the expert row of each slot (-1:
    none).  ``offsets`` int32 [E + 1]: expert e has the rows ``offsets[e] ..
    offsets[e + 1] - 1``, its tokens in rising order.  ``counts``: scratch of
    the call, kept for a further one (None: it needs none)."""

    __slots__ = ()


def empty_plan(tokens, experts, k, device='cuda'):
    """An unwritten :class:`Plan`: ``out`` of :func:`route`."""
    import torch
    return _new_plan(functools.partial(torch.empty, device=device), tokens,
                     experts, k)


def _new_plan(new, tokens, experts, k):
    import torch
    words = native.load().route_count_words(tokens, experts)
    i32 = torch.int32
    return Plan(new((tokens, k), dtype=i32),
                new((tokens, k), dtype=torch.float32),
                new((tokens * k,), dtype=i32), new((tokens, k), dtype=i32),
                new((experts + 1,), dtype=i32),
                new((words,), dtype=i32) if words else None)


def route(logits, k, renormalize=True, out=None):
    """Each token's ``k`` experts of the largest logits, and the plan that
    groups the tokens' rows by expert.

    ``logits`` [T, E] fp32 or bf16; E up to 1024, k up to 32.  Ties go to the
    lower expert.  ``-inf`` masks an expert: it is never chosen, and a token
    with fewer than k experts left has slots without one (expert and position
    -1, weight 0), which no group holds; a padded token has none at all.  A
    NaN ranks above every number, and the token's weights are NaN (as with
    ``+inf``).  Weights are the softmax of the chosen experts' logits
    (``renormalize``) or of all the token's logits, in fp32.  ``out``: a
    :class:`Plan` to write to."""
    import torch
    device = checks.tensor(logits, 'logits',
                           (torch.bfloat16, torch.float32), dims=2, align=2)
    mod = native.load()
    tokens, experts = logits.shape
    k = int(k)
    if not 1 <= experts <= mod.route_max_experts:
        raise ValueError('route takes 1 to %d experts, not %d' % (
            mod.route_max_experts, experts))
    if not 1 <= k <= min(experts, mod.route_max_k):
        raise ValueError('k must lie in 1 .. %d, not be %d' % (
            min(experts, mod.route_max_k), k))
    checks.int32(tokens * k, 'tokens * k')
    if out is None:
        out = _new_plan(logits.new_empty, tokens, experts, k)
    else:
        if not isinstance(out, Plan):
            raise ValueError('out must be a Plan (empty_plan makes one)')
        shapes = {'experts': (tokens, k), 'weights': (tokens, k),
                  'tokens': (tokens * k,), 'positions': (tokens, k),
                  'offsets': (experts + 1,)}
        words = mod.route_count_words(tokens, experts)
        if words and (out.counts is None or out.counts.numel() < words):
            raise ValueError('out.counts is too small')
        for name in Plan._fields:
            part = getattr(out, name)
            if part is None and name == 'counts':
                continue
            checks.tensor(part, 'out.' + name,
                          torch.float32 if name == 'weights' else torch.int32,
                          device, shapes.get(name), align=4)
        checks.all_apart('out', logits, *out)
    checks.run(device, mod.route, logits.data_ptr(), logits.dtype ==
               torch.bfloat16, tokens, experts, k, bool(renormalize),
               out.experts.data_ptr(), out.weights.data_ptr(),
               out.tokens.data_ptr(), out.positions.data_ptr(),
               out.offsets.data_ptr(), checks.pointer(out.counts))
    return out


def _parts(t):
    return tuple(t) if isinstance(t, mxfp4.Mxfp4) else (t, None)


def workspace_bytes(a, b, rows=None):
    """Size of the workspace that :func:`grouped_gemm` uses for these
    operands."""
    import torch
    mx = isinstance(b, mxfp4.Mxfp4)
    a_data, b_data = _parts(a)[0], _parts(b)[0]
    device = checks.tensor(a_data, 'a', torch.uint8 if mx else torch.bfloat16,
                           dims=2)
    checks.tensor(b_data, 'b', a_data.dtype, device, dims=3)
    return checks.product_workspace(
        native.load(), device, mx, True, rows is not None, a_data.shape[0],
        a_data.shape[0] if rows is None else rows.numel(), b_data.shape[1],
        a_data.shape[1] * a_data.element_size(), b_data.shape[0])


def grouped_gemm(a, b, offsets, bias=None, epilogue='none', rows=None,
                 out=None, workspace=None):
    """``out[i] = epi(a[rows[i]] @ b[e].T)`` for ``offsets[e] <= i <
    offsets[e + 1]``: one product per expert over its own rows.

    ``a`` [R, K] and ``b`` [E, N, K], both bf16 or both
    :class:`.mxfp4.Mxfp4`; ``offsets`` int32 [E + 1] on the device, rising;
    groups may be empty.  ``rows`` int32: row i of the product reads row
    ``rows[i]`` of ``a`` (default: row i).  ``epilogue``: ``'none'``,
    ``'bias'`` (+ ``bias[e]``, fp32 [E, N]) or ``'gelu'`` (``gelu_tanh`` of
    that).  K must be a multiple of 64 (MXFP4: 128), N of 16, E up to 65536.

    Rows that belong to no group are zero in a new result and left as they
    are in ``out``.  The offsets and ``rows`` are not read on the host: what
    points outside its tensor is brought inside it, so a wrong plan gives
    wrong rows but no access outside the operands.  ``workspace``: an fp32
    tensor of :func:`workspace_bytes` that no other call uses at the same
    time (default: a temporary one)."""
    import torch
    mx = isinstance(b, mxfp4.Mxfp4)
    if mx != isinstance(a, mxfp4.Mxfp4):
        raise ValueError('a and b must both be bf16 or both be Mxfp4')
    if mx:
        device, (rows_a, k) = mxfp4.check(a, 'a', dims=2)
        experts, n, k2 = mxfp4.check(b, 'b', device, dims=3)[1]
    else:
        device = checks.tensor(a, 'a', torch.bfloat16, dims=2)
        checks.tensor(b, 'b', torch.bfloat16, device, dims=3)
        rows_a, k = a.shape
        experts, n, k2 = b.shape
    if k != k2:
        raise ValueError('inner dimensions differ: %d vs %d' % (k, k2))
    deep = 128 if mx else 64
    if n < 16 or n % 16 or k < deep or k % deep or experts < 1:
        raise ValueError('unsupported shape E=%d N=%d K=%d (need N %% 16 == '
                         '0, K %% %d == 0)' % (experts, n, k, deep))
    checks.tensor(offsets, 'offsets', torch.int32, device, (experts + 1,),
                  align=4)
    if rows is not None:
        checks.tensor(rows, 'rows', torch.int32, device, dims=1, align=4)
    count = rows_a if rows is None else rows.numel()
    if count and not rows_a:
        raise ValueError('a has no rows')
    if epilogue not in EPILOGUES:
        raise ValueError('epilogue %r' % (epilogue,))
    epi = EPILOGUES[epilogue]
    if epi:
        if bias is None:
            raise ValueError('epilogue %r needs a bias' % epilogue)
        checks.tensor(bias, 'bias', torch.float32, device, (experts, n))
    elif bias is not None:
        raise ValueError("epilogue 'none' takes no bias")
    (a_data, a_scales), (b_data, b_scales) = _parts(a), _parts(b)
    fresh = out is None
    if fresh:
        out = a_data.new_empty((count, n), dtype=torch.bfloat16)
    else:
        checks.tensor(out, 'out', torch.bfloat16, device, (count, n))
        checks.apart(out, 'out', a_data, a_scales, b_data, b_scales, offsets,
                     rows, bias)
    mod = native.load()
    row_bytes = k // 2 if mx else k * 2
    if max(rows_a, count, n, row_bytes) > checks.LARGEST:
        for size, name in ((rows_a, 'rows of a'), (count, 'rows'), (n, 'N'),
                           (row_bytes, 'row bytes')):
            checks.int32(size, name)
    if experts > mod.product_max_experts:
        raise ValueError('E is %d: the limit is %d' % (
            experts, mod.product_max_experts))
    given = workspace
    workspace = checks.workspace(given, checks.product_workspace(
        mod, device, mx, True, rows is not None, rows_a, count, n, row_bytes,
        experts), device)
    if given is not None:
        checks.apart(given, 'workspace', a_data, a_scales, b_data,
                     b_scales, offsets, rows, bias, out)
    checks.run(device, mod.product, a_data.data_ptr(),
               checks.pointer(a_scales), b_data.data_ptr(),
               checks.pointer(b_scales), out.data_ptr(), checks.pointer(bias),
               0, offsets.data_ptr(), checks.pointer(rows), rows_a, count, n,
               row_bytes, experts, epi, fresh,
               checks.compute_units(mod, device), checks.pointer(workspace))
    return out


def combine(y, positions, weights, residual=None, out=None):
    """``out[t] = residual[t] + sum_j weights[t, j] * y[positions[t, j]]``:
    the experts' rows ``y`` [R, D] (bf16, D a multiple of 8) back at their
    tokens, summed in fp32 in the order of j and rounded once.  A position
    outside ``y`` (-1: a slot without an expert) adds nothing.  ``residual``
    [T, D] bf16 may be ``out``."""
    import torch
    device = checks.tensor(y, 'y', torch.bfloat16, dims=2)
    rows, width = y.shape
    checks.tensor(positions, 'positions', torch.int32, device, dims=2,
                  align=4)
    tokens, k = positions.shape
    checks.tensor(weights, 'weights', torch.float32, device, (tokens, k),
                  align=4)
    if width < 8 or width % 8:
        raise ValueError('rows of %d elements, not a multiple of 8' % width)
    if k < 1:
        raise ValueError('positions has no slots')
    if max(tokens, k, rows, width) > checks.LARGEST:
        for size, name in ((tokens, 'T'), (k, 'k'), (rows, 'R'),
                           (width, 'D')):
            checks.int32(size, name)
    if residual is not None:
        checks.tensor(residual, 'residual', torch.bfloat16, device,
                      (tokens, width))
    if out is None:
        out = y.new_empty((tokens, width))
    else:
        checks.tensor(out, 'out', torch.bfloat16, device, (tokens, width))
        checks.apart(out, 'out', y, positions, weights)
        checks.same_or_apart(out, 'out', residual)
    checks.run(device, native.load().combine, y.data_ptr(),
               positions.data_ptr(), weights.data_ptr(),
               checks.pointer(residual), out.data_ptr(), tokens, k, rows,
               width)
    return out
