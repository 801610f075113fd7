"""Argument checks of the expert-MLP and 4-bit operators.

Everything a kernel assumes of its operands is checked on the host before
the launch: a bad call raises ``ValueError`` and no kernel runs.
"""


def device_of(t, name):
    """The GPU that ``t`` lies on; a host tensor is refused."""
    if not getattr(t, 'is_cuda', False):
        raise ValueError('%s must be a CUDA tensor' % name)
    return t.device


class _Forward(object):
    """Stands for torch's forward_ad until the first call: inside a level."""
    _current_level = 0


_FORWARD = _Forward


def tangent(t):
    """Whether ``t`` is a dual tensor of forward-mode differentiation."""
    global _FORWARD  # pylint: disable=global-statement
    if _FORWARD is _Forward:
        from torch.autograd import forward_ad as _FORWARD
    return _FORWARD._current_level >= 0 and \
        _FORWARD.unpack_dual(t).tangent is not None


def tensor(t, name, dtypes, device=None, shape=None, dims=None, align=16):
    """Refuse a tensor that a kernel cannot take: another device, type or
    shape, holes between its elements, an address that is not a multiple of
    ``align`` bytes, or one whose gradient or tangent would be lost.
    ``dtypes``: a type or a tuple of them."""
    where = t.device if getattr(t, 'is_cuda', False) else device_of(t, name)
    dtype = t.dtype
    if dtype is not dtypes and not (isinstance(dtypes, tuple)
                                    and dtype in dtypes):
        if not isinstance(dtypes, tuple):
            dtypes = (dtypes,)
        raise ValueError('%s must be %s, not %s' % (
            name, ' or '.join(str(d)[6:] for d in dtypes), str(dtype)[6:]))
    if device is not None and where != device:
        raise ValueError('%s is on %s, not on %s' % (name, where, device))
    if dims is not None and t.dim() != dims:
        raise ValueError('%s must have %d dimensions, not %d' % (
            name, dims, t.dim()))
    if shape is not None and t.shape != shape:
        raise ValueError('%s must be %s, not %s' % (
            name, list(shape), list(t.shape)))
    if not t.is_contiguous():
        raise ValueError('%s must be contiguous' % name)
    # (an empty tensor has the address 0)
    if t.data_ptr() % align:
        raise ValueError('%s must start at a multiple of %d bytes' % (
            name, align))
    if t.requires_grad:
        import torch
        if torch.is_grad_enabled():
            raise ValueError('%s requires a gradient: these operators have '
                             'no backward pass (use torch.no_grad())' % name)
    # (outside every level one comparison, 0.03 us)
    if _FORWARD._current_level >= 0 and tangent(t):
        raise ValueError('%s has a tangent: these operators have no '
                         'derivative (forward_ad.unpack_dual gives the '
                         'tensor without it)' % name)
    return where


def span(t):
    """Byte range ``[begin, end)`` of a contiguous tensor."""
    return t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()


def apart(out, name, *others):
    """Refuse an output that shares memory with what the kernel reads."""
    lo, hi = span(out)
    for other in others:
        if other is None:
            continue
        begin, end = span(other)
        if lo < end and begin < hi:
            raise ValueError('%s overlaps an input' % name)


def all_apart(name, *parts):
    """Refuse parts of an output that share memory with one another or with
    an input among ``parts``."""
    end = 0
    for begin, after in sorted(span(t) for t in parts
                               if t is not None and t.numel()):
        if begin < end:
            raise ValueError('%s overlaps itself or an input' % name)
        end = after


def same_or_apart(out, name, other):
    """As :func:`apart`, but ``other`` itself may be the output (it is read
    and written element by element by the same thread)."""
    if other is not None and span(out) != span(other):
        apart(out, name, other)


# what a kernel's 32-bit arithmetic holds: up to 2^24 is added to a size (the
# end of a tile, of a workgroup's stretch)
LARGEST = 0x7f000000


def int32(value, name):
    """Refuse a size above :data:`LARGEST`."""
    if value > LARGEST:
        raise ValueError('%s = %d is above the limit of 2^31 - 2^24' % (
            name, value))
    return int(value)


def pointer(t):
    return 0 if t is None else t.data_ptr()


_CUS = {}


def compute_units(mod, device):
    """Compute units of a device (asked for once)."""
    index = device.index
    if index not in _CUS:
        _CUS[index] = mod.device_cus(index)
    return _CUS[index]


def product_workspace(mod, device, mx, grouped, gather, rows_a, rows, n,
                      row_bytes, experts):
    """Bytes of workspace that a product uses."""
    # (few rows: none, without asking)
    if rows <= 12 * experts:
        return 0
    return mod.product_workspace(mx, grouped, gather, rows_a, rows, n,
                                 row_bytes, experts,
                                 compute_units(mod, device))


def workspace(given, size, device):
    """The caller's workspace, or a new one of ``size`` bytes (None: 0)."""
    import torch
    if given is None:
        return torch.empty(size // 4, dtype=torch.float32,
                           device=device) if size else None
    tensor(given, 'workspace', torch.float32, device)
    if given.numel() * 4 < size:
        raise ValueError('workspace has %d bytes, not %d' % (
            given.numel() * 4, size))
    return given if size else None


def run(device, launch, *args):
    """``launch(*args, stream)`` on the caller's current stream of the
    operands' device, which need not be the current one.  (The raw stream
    handle: building a ``torch.cuda.Stream`` and entering a device context on
    every call cost 3 us, as much as the launch.)"""
    import torch
    index = device.index
    stream = torch._C._cuda_getCurrentRawStream(index)
    if index == torch._C._cuda_getDevice():
        launch(*args, stream)
    else:
        with torch.cuda.device(index):
            launch(*args, stream)
