"""The expert-MLP and MXFP4 operators: refusals (CPU) and numerics (MI355X)
against plain float64 implementations.

Tolerances: one rounding to bf16 is off by 2^-8 of the value; an fp32 sum of
K terms by at most K 2^-23 of the sum of their magnitudes (2^-23, not 2^-24:
the matrix unit may truncate); gelu passes an error on with at most 1.13 of
its size and adds |x| 2^-21 of its own (exp2 and reciprocal of 1 ulp, their
argument rounded twice); fp32 weights of k terms by (k + 8) 2^-24."""
import math
import os
import subprocess
import sys

import pytest

torch = pytest.importorskip('torch')

from kiosk_autoscaler_amd.ops import (checks, experts, mxfp4,  # noqa: E402
                                      native)

gpu = pytest.mark.gpu
BF16 = torch.bfloat16
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ---------------------------------------------------------------------------
# plain implementations

def ref_route(logits, k, renormalize=True):
    """Straight from the definition, a token at a time, on the host."""
    rows = logits.double().cpu().tolist()
    num, chosen, weights = len(rows[0]) if rows else logits.shape[1], [], []
    for row in rows:
        rank = sorted(range(num), key=lambda e: (
            -math.inf if math.isnan(row[e]) else -row[e], e))
        nans = [e for e in rank if math.isnan(row[e])]
        rank = nans + [e for e in rank if not math.isnan(row[e])
                       and row[e] > -math.inf]
        pick = rank[:k]
        nan = bool(nans) or (bool(rank) and row[rank[0]] == math.inf)
        live = [row[e] for e in (pick if renormalize else rank)]
        total = 0.0 if nan else sum(math.exp(v - live[0]) for v in live)
        chosen.append(pick + [-1] * (k - len(pick)))
        weights.append([math.nan if nan else math.exp(row[e] - live[0])
                        / total for e in pick] + [0.0] * (k - len(pick)))
    groups = [[] for _ in range(num)]
    for t, pick in enumerate(chosen):
        for j, e in enumerate(pick):
            if e >= 0:
                groups[e].append((t, j))
    offsets, tokens = [0], []
    positions = [[-1] * k for _ in rows]
    for group in groups:
        for t, j in group:
            positions[t][j] = len(tokens)
            tokens.append(t)
        offsets.append(len(tokens))
    tokens += [-1] * (len(rows) * k - len(tokens))
    return chosen, weights, tokens, positions, offsets


def power(e):
    """2 ** e in float64, exactly."""
    table = torch.tensor([2.0 ** i for i in range(-200, 201)],
                         dtype=torch.float64, device=e.device)
    return table[e.long() + 200]


def ref_quantize(x):
    """(values in float64, scale bytes) of the format's definition."""
    blocks = x.double().reshape(-1, 32)
    peak = blocks.abs().amax(1)
    bad = ~torch.isfinite(blocks).all(1)
    exponent = torch.frexp(torch.where(bad | (peak == 0), 1.0,
                                       peak)).exponent
    e = torch.where(peak == 0, -127, (exponent - 3).clamp(min=-127))
    grid = torch.tensor(E2M1, dtype=torch.float64, device=x.device)
    # ties to even: the even code of two equally near ones
    order = torch.tensor((0, 2, 4, 6, 1, 3, 5, 7), device=x.device)
    step = power(e)
    dist = (blocks.abs().unsqueeze(-1) / step[:, None, None]
            - grid[order]).abs()
    code = order[dist.argmin(-1)]
    values = torch.copysign(grid[code] * step[:, None], blocks)
    values[bad] = math.nan
    scales = torch.where(bad, 255, e + 127)
    return (values.reshape(x.shape),
            scales.reshape(x.shape[:-1] + (x.shape[-1] // 32,)))


def values_of(q):
    """What codes and scale bytes stand for, in float64."""
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1),
                         dtype=torch.float64, device=q.codes.device)
    code = torch.stack((q.codes & 15, q.codes >> 4), -1).flatten(-2).long()
    scale = torch.where(q.scales == 255, math.nan,
                        power(q.scales.int() - 127))
    return table[code] * scale.repeat_interleave(32, -1)


def gelu(x):
    u = math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)
    return 0.5 * x * (1 + torch.tanh(u))


def check_product(out, a, b, epilogue, bias=None, residual=None):
    """``out`` against float64 operands ``a`` [M, K], ``b`` [N, K]."""
    y = a @ b.t()
    slack = a.shape[1] * 2.0 ** -23 * (a.abs() @ b.abs().t())
    if epilogue != 'none':
        y = y + bias.double()
        slack = slack + 2.0 ** -23 * y.abs()
    if epilogue == 'gelu':
        slack = 1.13 * slack + 2.0 ** -21 * y.abs()
        y = gelu(y)
    if epilogue == 'residual':
        y = y + residual.double()
        slack = slack + 2.0 ** -23 * y.abs()
    tol = slack + 2.0 ** -8 * (y.abs() + slack)
    err = (out.double() - y).abs()
    bad = ~(err <= tol) & ~(out.isnan() & y.isnan())
    assert not bad.any(), (int(bad.sum()), float(err.max()),
                           bad.nonzero()[:4].tolist())


def rand(*shape, seed=0, scale=1.0, dtype=BF16):
    g = torch.Generator(device='cuda').manual_seed(seed)
    return (torch.randn(*shape, generator=g, device='cuda')
            * scale).to(dtype)


def cut(rows, groups, seed):
    """Ragged offsets: some groups empty, one large."""
    g = torch.Generator().manual_seed(seed)
    cuts = torch.randint(0, rows + 1, (groups - 1,), generator=g)
    cuts = torch.cat([torch.tensor([0, rows]), cuts]).sort().values
    return cuts.to(torch.int32).cuda()


def random_mx(*shape, seed=0):
    g = torch.Generator(device='cuda').manual_seed(seed)
    codes = torch.randint(0, 256, shape[:-1] + (shape[-1] // 2,),
                          generator=g, device='cuda', dtype=torch.uint8)
    scales = torch.randint(118, 132, shape[:-1] + (shape[-1] // 32,),
                           generator=g, device='cuda', dtype=torch.uint8)
    return mxfp4.Mxfp4(codes, scales)


# ---------------------------------------------------------------------------
# refusals: nothing reaches a launch

class NoLaunch(object):
    """Stands in for the native module: sizes yes, launches no."""

    route_max_experts, route_max_k = 1024, 32
    product_max_experts = 65536

    @staticmethod
    def route_count_words(tokens, experts):
        return 0 if tokens <= 100 else -(-tokens // 100) * (experts + 1)

    @staticmethod
    def device_cus(index):
        return 256

    @staticmethod
    def product_workspace(*sizes):
        return 4096

    def __getattr__(self, name):
        raise AssertionError('%s was launched' % name)


@pytest.fixture
def host(monkeypatch):
    """Host tensors pass as device tensors; a launch fails the test."""
    monkeypatch.setattr(checks, 'device_of', lambda t, name: t.device)
    monkeypatch.setattr(native, 'load', lambda *a, **k: NoLaunch())


def zeros(*shape, dtype=BF16):
    return torch.zeros(shape, dtype=dtype)


def mx_zeros(*shape):
    return mxfp4.Mxfp4(zeros(*shape[:-1], shape[-1] // 2, dtype=torch.uint8),
                       zeros(*shape[:-1], shape[-1] // 32,
                             dtype=torch.uint8))


def misaligned(*shape, dtype=BF16):
    count = math.prod(shape)
    return torch.zeros(count + 64, dtype=dtype)[1:1 + count].view(shape)


def test_host_tensors_are_refused():
    for call in (lambda: experts.route(zeros(2, 4), 1),
                 lambda: experts.grouped_gemm(zeros(2, 64), zeros(2, 16, 64),
                                              zeros(3, dtype=torch.int32)),
                 lambda: experts.combine(zeros(2, 8),
                                         zeros(1, 2, dtype=torch.int32),
                                         zeros(1, 2, dtype=torch.float32)),
                 lambda: mxfp4.quantize(zeros(2, 32)),
                 lambda: mxfp4.dequantize(mx_zeros(2, 32)),
                 lambda: mxfp4.gemm(mx_zeros(2, 128), mx_zeros(16, 128))):
        with pytest.raises(ValueError, match='CUDA tensor'):
            call()


@pytest.mark.parametrize('logits,k,match', [
    (zeros(2, 4, dtype=torch.float64), 1, 'bfloat16 or float32'),
    (zeros(4), 1, '2 dimensions'),
    (zeros(2, 4), 0, 'k must lie'),
    (zeros(2, 4), 5, 'k must lie'),
    (zeros(2, 64), 33, 'k must lie'),
    (zeros(2, 1025), 1, '1 to 1024'),
    (zeros(2, 0), 1, '1 to 1024'),
    (zeros(4, 2).t(), 1, 'contiguous'),
    (zeros(2, 4, dtype=torch.float32).requires_grad_(), 1, 'gradient'),
    (zeros(1, 4).expand(1 << 27, 4).as_strided((1 << 27, 4), (0, 1)), 4,
     'contiguous'),
])
def test_route_refuses(host, logits, k, match):
    with pytest.raises(ValueError, match=match):
        experts.route(logits, k)


def test_route_takes_any_row_of_logits(host):
    """Rows of an odd number of bf16 logits start at odd multiples of two
    bytes."""
    logits = zeros(4, 5)
    for first in range(4):
        with pytest.raises(AssertionError, match='launched'):
            experts.route(logits[first:], 2)


def test_route_refuses_a_wrong_plan(host):
    logits = zeros(200, 8)
    good = experts.empty_plan(200, 8, 2, 'cpu')
    for name, part in (
            ('experts', zeros(200, 3, dtype=torch.int32)),
            ('weights', zeros(200, 2)), ('tokens', good.tokens[:-1]),
            ('positions', good.positions.t()),
            ('offsets', zeros(8, dtype=torch.int32)),
            ('counts', good.counts[:-1]), ('counts', None)):
        with pytest.raises(ValueError, match=name):
            experts.route(logits, 2, out=good._replace(**{name: part}))
    with pytest.raises(ValueError, match='Plan'):
        experts.route(logits, 2, out=tuple(good))
    for shared in (dict(positions=good.experts),
                   dict(tokens=good.positions.view(-1)),
                   dict(weights=logits.view(torch.float32).view(-1)[:400]
                        .view(200, 2))):
        with pytest.raises(ValueError, match='out overlaps'):
            experts.route(logits, 2, out=good._replace(**shared))
    with pytest.raises(AssertionError, match='launched'):
        experts.route(logits, 2, out=good)


def test_sizes_leave_room_for_the_end_of_a_tile():
    assert checks.int32(0x7f000000, 'rows') == 0x7f000000
    for size in (0x7f000001, (1 << 31) - 1, 1 << 31):
        with pytest.raises(ValueError, match='rows = %d' % size):
            checks.int32(size, 'rows')


def test_grouped_gemm_refuses_too_many_experts(host):
    with pytest.raises(ValueError, match='E is 65537'):
        experts.grouped_gemm(zeros(1, 64), zeros(65537, 16, 64),
                             zeros(65538, dtype=torch.int32))


@pytest.mark.parametrize('change,match', [
    (dict(a=zeros(6, 64, dtype=torch.float16)), 'a must be bfloat16'),
    (dict(a=zeros(6, 128)), 'inner dimensions'),
    (dict(a=mx_zeros(6, 128)), 'both'),
    (dict(b=zeros(16, 64)), '3 dimensions'),
    (dict(b=zeros(3, 24, 64), bias=zeros(3, 24, dtype=torch.float32)),
     'unsupported shape'),
    (dict(b=zeros(3, 16, 32), a=zeros(6, 32)), 'unsupported shape'),
    (dict(b=zeros(0, 16, 64), offsets=zeros(1, dtype=torch.int32)),
     'unsupported shape'),
    (dict(b=zeros(3, 64, 16).transpose(1, 2)), 'contiguous'),
    (dict(a=misaligned(6, 64)), 'multiple of 16'),
    (dict(offsets=zeros(3, dtype=torch.int32)), 'offsets must be'),
    (dict(offsets=zeros(4, dtype=torch.int64)), 'offsets must be int32'),
    (dict(rows=zeros(4, dtype=torch.int64)), 'rows must be int32'),
    (dict(rows=zeros(2, 2, dtype=torch.int32)), '1 dimensions'),
    (dict(a=zeros(0, 64), rows=zeros(4, dtype=torch.int32)), 'no rows'),
    (dict(epilogue='residual'), 'epilogue'),
    (dict(epilogue='gelu', bias=None), 'needs a bias'),
    (dict(epilogue='none'), 'takes no bias'),
    (dict(bias=zeros(3, 16)), 'bias must be float32'),
    (dict(bias=zeros(16, dtype=torch.float32)), 'bias must be'),
    (dict(out=zeros(5, 16)), 'out must be'),
    (dict(out=zeros(6, 16, dtype=torch.float32)), 'out must be bfloat16'),
])
def test_grouped_gemm_refuses(host, change, match):
    call = dict(a=zeros(6, 64), b=zeros(3, 16, 64), epilogue='bias',
                offsets=zeros(4, dtype=torch.int32),
                bias=zeros(3, 16, dtype=torch.float32))
    call.update(change)
    with pytest.raises(ValueError, match=match):
        experts.grouped_gemm(**call)


def test_outputs_that_overlap_an_input_are_refused(host):
    buf = zeros(4096)
    a, b = buf[:6 * 64].view(6, 64), zeros(1, 64, 64)
    off = zeros(2, dtype=torch.int32)
    for at in (0, 8, 6 * 64 - 8):
        with pytest.raises(ValueError, match='overlaps'):
            experts.grouped_gemm(a, b, off,
                                 out=buf[at:at + 6 * 64].view(6, 64))
    with pytest.raises(AssertionError, match='launched'):
        experts.grouped_gemm(a, b, off, out=buf[384:768].view(6, 64))
    y = buf[:64].view(4, 16)
    where = dict(positions=zeros(4, 1, dtype=torch.int32),
                 weights=zeros(4, 1, dtype=torch.float32))
    with pytest.raises(ValueError, match='overlaps'):
        experts.combine(y, out=y, **where)
    res = buf[64:128].view(4, 16)
    with pytest.raises(ValueError, match='overlaps'):
        experts.combine(y, residual=res, out=buf[72:136].view(4, 16),
                        **where)
    with pytest.raises(AssertionError, match='launched'):
        experts.combine(y, residual=res, out=res, **where)


def test_workspaces_are_checked(host):
    rows = 300
    a, b = zeros(rows, 64), zeros(1, 16, 64)
    off = zeros(2, dtype=torch.int32)
    f32 = dict(dtype=torch.float32)
    assert experts.workspace_bytes(a, b) == 4096
    assert experts.workspace_bytes(a, b, zeros(3, dtype=torch.int32)) == 0
    for workspace, match in ((zeros(1023, **f32), 'workspace has 4092 bytes'),
                             (zeros(2048), 'workspace must be float32'),
                             (zeros(64, 64, **f32).t(), 'contiguous')):
        with pytest.raises(ValueError, match=match):
            experts.grouped_gemm(a, b, off, workspace=workspace)
    out = zeros(rows, 16)
    with pytest.raises(ValueError, match='workspace overlaps'):
        experts.grouped_gemm(a, b, off, out=out,
                             workspace=out.view(torch.float32).view(-1))
    with pytest.raises(AssertionError, match='launched'):
        experts.grouped_gemm(a, b, off, workspace=zeros(1024, **f32))
    a, b = mx_zeros(rows, 128), mx_zeros(16, 128)
    assert mxfp4.workspace_bytes(a, b) == 4096
    with pytest.raises(ValueError, match='workspace has 0 bytes'):
        mxfp4.gemm(a, b, workspace=zeros(0, **f32))


@pytest.mark.parametrize('change,match', [
    (dict(y=zeros(4, 12)), 'multiple of 8'),
    (dict(y=zeros(4, 0)), 'multiple of 8'),
    (dict(y=zeros(4, 16, dtype=torch.float32)), 'y must be bfloat16'),
    (dict(positions=zeros(3, 2, dtype=torch.int64)), 'positions'),
    (dict(positions=zeros(3, 0, dtype=torch.int32),
          weights=zeros(3, 0, dtype=torch.float32)), 'no slots'),
    (dict(weights=zeros(3, 1, dtype=torch.float32)), 'weights'),
    (dict(residual=zeros(4, 16)), 'residual'),
    (dict(out=zeros(3, 8)), 'out'),
])
def test_combine_refuses(host, change, match):
    call = dict(y=zeros(4, 16), positions=zeros(3, 2, dtype=torch.int32),
                weights=zeros(3, 2, dtype=torch.float32))
    call.update(change)
    with pytest.raises(ValueError, match=match):
        experts.combine(**call)


def test_mxfp4_refuses(host):
    for x, match in ((zeros(2, 48), 'multiple of 32'),
                     (zeros(2, 32, dtype=torch.float16), 'x must be'),
                     (torch.tensor(1.0), 'multiple of 32'),
                     (zeros(32, 2).t(), 'contiguous'),
                     (misaligned(2, 32), 'multiple of 16')):
        with pytest.raises(ValueError, match=match):
            mxfp4.quantize(x)
    q = mx_zeros(2, 64)
    with pytest.raises(ValueError, match='out must be'):
        mxfp4.quantize(zeros(2, 32), out=q)
    with pytest.raises(ValueError, match='Mxfp4'):
        mxfp4.quantize(zeros(2, 64), out=tuple(q))
    with pytest.raises(ValueError, match='scales'):
        mxfp4.dequantize(mxfp4.Mxfp4(q.codes, q.scales[:, :1].contiguous()))
    with pytest.raises(ValueError, match='dtype'):
        mxfp4.dequantize(q, dtype=torch.float16)
    with pytest.raises(ValueError, match='out'):
        mxfp4.dequantize(q, out=zeros(2, 32))
    a, b = mx_zeros(2, 128), mx_zeros(32, 128)
    f32 = zeros(32, dtype=torch.float32)
    for call, match in (
            (dict(a=zeros(2, 128)), 'Mxfp4'),
            (dict(b=mx_zeros(32, 256)), 'inner'),
            (dict(b=mx_zeros(24, 128)), 'unsupported'),
            (dict(a=mx_zeros(2, 64), b=mx_zeros(32, 64)), 'unsupported'),
            (dict(epilogue='gelu'), 'needs a bias'),
            (dict(epilogue='swish'), 'epilogue'),
            (dict(bias=f32), 'takes no bias'),
            (dict(epilogue='residual', bias=f32), 'needs a residual'),
            (dict(epilogue='bias', bias=f32, residual=zeros(2, 32)),
             'takes no residual'),
            (dict(out=zeros(2, 16)), 'out must be'),
            (dict(out=a.codes.view(BF16).view(2, 32)), 'overlaps')):
        with pytest.raises(ValueError, match=match):
            mxfp4.gemm(**dict(dict(a=a, b=b), **call))


def test_only_the_kernels_that_calls_reach_are_built():
    """No bf16 product takes a residual (gemm does): none is compiled."""
    paths = native.extension_candidates()
    if not paths:
        pytest.skip('the extension is not built')
    with open(paths[0], 'rb') as f:
        built = f.read()
    for name in (b'product_tile_kernel', b'product256_bf16_kernel',
                 b'product_rows_kernel'):
        assert name + b'ILi' in built
    # <mode 0 (bf16), epilogue 2 (residual), ...>
    for name in (b'product_tile_kernelILi0ELi2E',
                 b'product256_bf16_kernelILi2E',
                 b'product_rows_kernelILi0ELi2E'):
        assert name not in built
    assert b'product_tile_kernelILi1ELi2E' in built


@pytest.mark.parametrize('mx,rows,num,n,row_bytes', [
    # few rows, with one wave a workgroup and with more
    (True, 131072, 65536, 32768, 64), (False, 65536, 65536, 16384, 4096),
    (True, 786432, 65536, 65536, 2048),
    # 256x256 tiles, in one group and in many
    (False, 0x7f000000, 1, 1 << 20, 2048),
    (True, 0x7f000000, 65536, 1 << 20, 192),
    # 128x128 tiles (weights past 32-bit offsets)
    (False, 1 << 24, 1, 1 << 24, 1024)])
def test_more_tiles_than_a_launch_takes_are_refused(mx, rows, num, n,
                                                    row_bytes):
    """A grid has fewer than 2^32 threads: an error before anything runs."""
    if not native.extension_candidates():
        pytest.skip('the extension is not built')
    mod = native.load()
    with pytest.raises(ValueError, match='more tiles than one launch'):
        mod.product(0, 16 if mx else 0, 0, 16 if mx else 0, 0, 0, 0, 16, 0,
                    rows, rows, n, row_bytes, num, 0, True, 256, 0, 0)


def test_dual_tensors_are_refused(host):
    """A tangent would be lost without a word."""
    forward = torch.autograd.forward_ad
    f32, off = torch.float32, zeros(2, dtype=torch.int32)
    calls = {
        'logits': lambda t: experts.route(t, 1),
        'a': lambda t: experts.grouped_gemm(t, zeros(1, 16, 64), off),
        'b': lambda t: experts.grouped_gemm(zeros(2, 64),
                                            t.view(1, 16, 64), off),
        'bias': lambda t: mxfp4.gemm(mx_zeros(2, 128), mx_zeros(16, 128),
                                     bias=t, epilogue='bias'),
        'y': lambda t: experts.combine(t, zeros(2, 1, dtype=torch.int32),
                                       zeros(2, 1, dtype=f32)),
        'x': mxfp4.quantize}
    for name, call in calls.items():
        t = {'b': zeros(16, 64), 'bias': zeros(16, dtype=f32)}.get(
            name, zeros(2, 64))
        with forward.dual_level():
            with pytest.raises(ValueError, match=name + ' has a tangent'):
                call(forward.make_dual(t, torch.ones_like(t)))
            # a tensor without one passes within the level too
            with pytest.raises(AssertionError, match='launched'):
                call(t)
        with pytest.raises(AssertionError, match='launched'):
            call(t)


# ---------------------------------------------------------------------------
# numerics

@gpu
@pytest.mark.parametrize('dtype', [torch.float32, BF16])
@pytest.mark.parametrize('tokens,num,k', [
    (0, 8, 2), (1, 1, 1), (1, 16, 2), (3, 5, 5), (127, 64, 4), (128, 65, 8),
    (129, 128, 8), (300, 256, 3), (1000, 300, 32), (515, 1024, 7),
    (256, 128, 8), (257, 33, 32),
    (128, 1024, 32), (129, 1024, 32), (200, 300, 32), (40000, 12, 2)])
def test_route(tokens, num, k, dtype):
    logits = rand(tokens, num, seed=tokens + num, dtype=dtype)
    if dtype == BF16:
        logits = (logits * 4).round() / 4            # many ties
    if tokens > 100:
        logits[5] = -math.inf                        # a padded token
        logits[7, :num - 1] = -math.inf              # one expert left
        logits[20:, 0] = -math.inf                   # an expert nobody wants
    if tokens > 100 and num > 2:
        logits[9, 1] = math.nan
        logits[11, 2] = math.inf
        logits[13] = torch.finfo(dtype).min          # lowest, not masked
    for renormalize in (True, False):
        plan = experts.route(logits, k, renormalize)
        chosen, weights, rows, positions, offsets = ref_route(logits, k,
                                                              renormalize)
        shape = (tokens, k)
        assert plan.experts.tolist() == chosen
        assert plan.positions.tolist() == positions
        assert plan.offsets.tolist() == offsets
        assert plan.tokens.tolist() == rows
        want = torch.tensor(weights, dtype=torch.float64).view(shape)
        # exp of a difference rounded once: |l| 2^-24 more
        spread = float(logits.float().nan_to_num(0, 0, 0).abs().clamp(
            max=100).max()) if tokens else 0
        torch.testing.assert_close(
            plan.weights.double().cpu(), want, equal_nan=True, atol=1e-37,
            rtol=((num if not renormalize else k) + 8 + spread) * 2.0 ** -24)


@gpu
@pytest.mark.parametrize('tokens', [2, 300])
@pytest.mark.parametrize('renormalize', [True, False])
def test_route_of_infinite_and_nan_logits(tokens, renormalize):
    """+inf is the largest number, a NaN is above it; both make the token's
    weights NaN.  The other tokens do not notice."""
    logits = rand(tokens, 24, seed=5, dtype=torch.float32)
    want = experts.route(logits, 3, renormalize)
    bad = logits.clone()
    bad[0, 7] = math.inf
    bad[0, 9] = math.nan
    bad[1, 20] = math.inf
    got = experts.route(bad, 3, renormalize)
    assert got.experts[0, :2].tolist() == [9, 7]
    assert got.experts[1, 0].item() == 20
    assert bool(got.weights[:2].isnan().all())
    assert torch.equal(got.experts[2:], want.experts[2:])
    assert torch.equal(got.weights[2:], want.weights[2:])


@gpu
@pytest.mark.parametrize('num,k', [(5, 2), (27, 4), (301, 3)])
def test_route_of_rows_at_odd_addresses(num, k):
    logits = rand(700, num, seed=7)
    for first in (1, 2, 3):
        part = logits[first:]
        got, want = experts.route(part, k), experts.route(part.clone(), k)
        for a, b in zip(got[:5], want[:5]):
            assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize('kernel,m,n,k', [
    ('rows', 5, 272, 16768), ('rows', 30, 4096, 2176),
    ('tile128', 300, 528, 2176), ('tile256', 300, 528, 8576)])
def test_mxfp4_products_of_scales_at_any_word(kernel, m, n, k):
    """Scale rows of an odd number of words, from the second row on."""
    a, b = whole_mx(m + 1, k, seed=m), whole_mx(n + 1, k, seed=n)
    part_a, part_b = (mxfp4.Mxfp4(q.codes[1:], q.scales[1:])
                      for q in (a, b))
    assert part_b.scales.data_ptr() % 8
    assert kernel_of(part_a, part_b, grouped=False) == kernel
    assert torch.equal(mxfp4.gemm(part_a, part_b), exact_product(
        values_of(part_a), values_of(part_b)))


@gpu
def test_route_writes_into_a_plan_and_repeats():
    logits = rand(1500, 40, seed=3)
    first = experts.route(logits, 4)
    plan = experts.empty_plan(1500, 40, 4)
    for _ in range(3):
        assert experts.route(logits, 4, out=plan) is plan
        for a, b in zip(first[:5], plan[:5]):
            assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize('tokens,k,width', [
    (1, 1, 8), (1, 2, 4096), (33, 3, 72), (257, 8, 2056), (5, 32, 1024)])
@pytest.mark.parametrize('residual', [False, True])
def test_combine(tokens, k, width, residual):
    rows = tokens * k
    y = rand(rows + 3, width, seed=1)
    g = torch.Generator().manual_seed(2)
    positions = torch.randint(-1, rows + 3, (tokens, k), generator=g,
                              dtype=torch.int32)
    positions[0] = -1                                # nothing at all
    if tokens > 2:
        positions[1] = positions[1, 0]               # the same row k times
        positions[2, 0] = rows + 3                   # outside y: nothing
    positions = positions.cuda()
    y[rows + 2] = math.nan                           # one row is poison
    weights = rand(tokens, k, seed=4, dtype=torch.float32)
    res = rand(tokens, width, seed=5) if residual else None
    out = experts.combine(y, positions, weights, residual=res)
    live = (positions >= 0) & (positions < rows + 3)
    terms = y.double()[positions.clamp(0, rows + 2).long()] \
        * weights.double().unsqueeze(-1)
    terms = torch.where(live.unsqueeze(-1), terms, 0.0)
    want = terms.sum(1) + (res.double() if residual else 0)
    mag = terms.abs().sum(1) + (res.double().abs() if residual else 0)
    tol = 2.0 ** -8 * want.abs() + (k + 1) * 2.0 ** -23 * mag
    err = (out.double() - want).abs()
    assert torch.equal(out.isnan(), want.isnan())
    assert (err <= tol)[~want.isnan()].all()
    if residual:                                     # in place
        assert torch.equal(experts.combine(
            y, positions, weights, residual=res, out=res).view(torch.int16),
            out.view(torch.int16))


@gpu
@pytest.mark.parametrize('dtype', [torch.float32, BF16])
@pytest.mark.parametrize('shape', [(32,), (1, 64), (3, 5, 96), (7, 4096),
                                   (0, 64), (1000, 160)])
def test_quantize_and_dequantize(shape, dtype):
    x = rand(*shape, seed=6, dtype=dtype)
    if x.numel() > 1000:
        rows = x.view(-1, 32)
        rows[0] = 0
        rows[1] = -0.0
        rows[2, 3] = math.nan
        rows[3, 31] = math.inf
        rows[4, 0] = -math.inf
        rows[5] = torch.finfo(dtype).max
        rows[6] = torch.finfo(dtype).tiny            # least normal number
        rows[7] = torch.finfo(dtype).tiny / 8        # and below it
        rows[8] *= 1e-38
        # every border and its neighbours at scale 1
        edge = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0,
                             7.0, 7.96875, 4.0])
        rows[9, :11], rows[9, 11:22] = edge, -edge
        rows[10, :11] = edge * (1 + 2.0 ** -7)
        rows[10, 11:22] = edge * (1 - 2.0 ** -7)
        rows[10, 31] = 4.0
    q = mxfp4.quantize(x)
    want, scales = ref_quantize(x)
    assert q.shape == tuple(shape)
    assert torch.equal(q.scales.int(), scales.int())
    torch.testing.assert_close(values_of(q), want, rtol=0, atol=0,
                               equal_nan=True)
    for to in (BF16, torch.float32):
        got = mxfp4.dequantize(q, dtype=to)
        assert got.dtype == to
        torch.testing.assert_close(got, want.to(to), rtol=0, atol=0,
                                   equal_nan=True)


@gpu
def test_dequantize_every_code_and_scale():
    codes = torch.arange(256, dtype=torch.uint8, device='cuda')
    codes = codes.repeat(16).view(256, 16)
    scales = torch.arange(256, dtype=torch.uint8, device='cuda').view(256, 1)
    q = mxfp4.Mxfp4(codes.contiguous(), scales)
    want = values_of(q)
    for dtype in (BF16, torch.float32):
        got = mxfp4.dequantize(q, dtype=dtype)
        torch.testing.assert_close(got, want.to(dtype), rtol=0, atol=0,
                                   equal_nan=True)


@gpu
def test_mxfp4_product_reads_every_element_at_its_place():
    """One-hot rows against distinct values: a wrong lane, nibble or scale
    byte shows as a wrong number, exactly."""
    k, n = 512, 512
    eye = torch.eye(k, device='cuda', dtype=BF16)
    a = mxfp4.quantize(eye)
    b = random_mx(n, k, seed=8)
    out = mxfp4.gemm(a, b)
    assert torch.equal(out.double(), values_of(b).t())
    # and the activations' side
    out = mxfp4.gemm(b, a)
    assert torch.equal(out.double(), values_of(b))


@gpu
def test_mxfp4_product_of_nan_blocks_and_extreme_scales():
    a, b = random_mx(40, 256, seed=1), random_mx(48, 256, seed=2)
    a.scales[3, 5] = 255
    b.scales[7, 1] = 255
    a.codes[5, :16] = 0
    a.scales[5, 0] = 0                               # a block of zeros
    out = mxfp4.gemm(a, b)
    check_product(out, values_of(a), values_of(b), 'none')
    assert out[3].isnan().all() and out[:, 7].isnan().all()
    assert int(out.isnan().sum()) == 40 + 48 - 1
    # scales far from 1 that cancel
    a, b = random_mx(40, 256, seed=1), random_mx(48, 256, seed=2)
    big = mxfp4.Mxfp4(a.codes, a.scales + 100)
    small = mxfp4.Mxfp4(b.codes, b.scales - 100)
    assert torch.equal(mxfp4.gemm(big, small), mxfp4.gemm(a, b))


GEMM_SHAPES = [(1, 16, 128), (1, 4096, 4096), (2, 48, 384), (17, 512, 256),
               (64, 256, 640), (130, 272, 128), (200, 1040, 1152),
               (513, 528, 512), (1500, 2064, 896), (2048, 4096, 1024),
               (16, 16384, 512), (3, 128, 16384), (300, 528, 16640),
              (129, 272, 8192), (1000, 1040, 8192), (300, 272, 8320),
              (200, 1040, 8576), (40, 528, 128), (300, 528, 384)]


@gpu
@pytest.mark.parametrize('m,n,k', GEMM_SHAPES)
@pytest.mark.parametrize('epilogue', ['none', 'bias', 'gelu', 'residual'])
def test_mxfp4_gemm(m, n, k, epilogue):
    a = mxfp4.quantize(rand(m, k, seed=m))
    b = mxfp4.quantize(rand(n, k, seed=n, scale=k ** -0.5))
    bias = None if epilogue == 'none' else rand(n, seed=3,
                                                dtype=torch.float32)
    res = rand(m, n, seed=4) if epilogue == 'residual' else None
    out = mxfp4.gemm(a, b, bias, res, epilogue)
    check_product(out, values_of(a), values_of(b), epilogue, bias, res)
    again = mxfp4.gemm(a, b, bias, res, epilogue)
    assert torch.equal(out, again)
    if res is not None:                              # in place
        assert torch.equal(mxfp4.gemm(a, b, bias, res, epilogue, out=res),
                           out)


GROUPED = [  # rows, experts, n, k
    # long rows and few tiles: slices; full and half tiles in each
    (300, 1, 272, 4096), (900, 2, 528, 8192), (2000, 3, 1040, 8448),
    (1100, 8, 4096, 2048), (4500, 4, 4096, 8192),
    (1, 1, 16, 128), (2, 8, 4096, 4096), (5, 3, 48, 384), (64, 16, 272, 256),
    (100, 4, 1040, 640), (300, 70, 528, 128), (777, 7, 2064, 896),
    (2000, 5, 512, 1024), (4096, 64, 256, 256), (1300, 3, 1024, 2048),
    (31, 200, 64, 512),
    # small groups in many tiles, in one tile for each CU, in fewer
    (800, 64, 2048, 256), (600, 32, 2048, 384), (300, 32, 2048, 384),
    # 128 x 128 tiles: one for each CU and two, a row of a step and less
    (900, 5, 528, 1152), (1500, 1, 4096, 1088 * 2), (700, 3, 1040, 128),
    # few rows: tiles of 32 rows, wide and narrow; short rows of many columns
    (128, 16, 1024, 2176), (100, 8, 1024, 4352), (400, 16, 2560, 512)]


@gpu
@pytest.mark.parametrize('mx', [False, True])
@pytest.mark.parametrize('rows,num,n,k', GROUPED)
@pytest.mark.parametrize('epilogue', ['none', 'bias', 'gelu'])
def test_grouped_gemm(rows, num, n, k, epilogue, mx):
    offsets = cut(rows, num, rows)
    source = max(rows // 3, 1)
    a = rand(source, k, seed=1)
    b = rand(num, n, k, seed=2, scale=k ** -0.5)
    index = torch.randint(0, source, (rows,), device='cuda',
                          dtype=torch.int32,
                          generator=torch.Generator('cuda').manual_seed(3))
    bias = None if epilogue == 'none' else rand(num, n, seed=4,
                                                dtype=torch.float32)
    if mx:
        a, b = mxfp4.quantize(a), mxfp4.quantize(b)
    out = experts.grouped_gemm(a, b, offsets, bias, epilogue, rows=index)
    va, vb = (values_of(a), values_of(b)) if mx else (a.double(), b.double())
    bounds = offsets.tolist()
    for e in range(num):
        lo, hi = bounds[e], bounds[e + 1]
        if lo < hi:
            check_product(out[lo:hi], va[index[lo:hi].long()], vb[e],
                          epilogue, None if bias is None else bias[e])
    assert torch.equal(out, experts.grouped_gemm(a, b, offsets, bias,
                                                 epilogue, rows=index))
    # without a gather, on the gathered rows
    if mx:
        direct = mxfp4.Mxfp4(a.codes[index.long()], a.scales[index.long()])
    else:
        direct = a[index.long()]
    assert torch.equal(out, experts.grouped_gemm(direct, b, offsets, bias,
                                                 epilogue))


@gpu
@pytest.mark.parametrize('mx', [False, True])
@pytest.mark.parametrize('rows', [40, 700])
def test_rows_outside_the_groups(rows, mx):
    """Zero in a new result, as they were in ``out``; NaN there, or in
    another expert's weights, reaches no other row."""
    num, n, k = 4, 160, 256
    a, b = rand(rows, k, seed=1), rand(num, n, k, seed=2)
    a[:3] = math.nan
    a[rows - 5:] = math.nan
    b[3] = math.nan                                  # its group is empty
    offsets = torch.tensor([3, 9, 9, rows - 5, rows - 5], dtype=torch.int32,
                           device='cuda')
    if mx:
        a, b = mxfp4.quantize(a), mxfp4.quantize(b)
    out = experts.grouped_gemm(a, b, offsets)
    assert (out[:3] == 0).all() and (out[rows - 5:] == 0).all()
    assert out[3:rows - 5].isfinite().all()
    kept = torch.full((rows, n), 7.0, dtype=BF16, device='cuda')
    assert experts.grouped_gemm(a, b, offsets, out=kept) is kept
    assert (kept[:3] == 7).all() and (kept[rows - 5:] == 7).all()
    assert torch.equal(kept[3:rows - 5], out[3:rows - 5])
    none = torch.zeros(num + 1, dtype=torch.int32, device='cuda')
    assert (experts.grouped_gemm(a, b, none) == 0).all()
    assert (experts.grouped_gemm(a, b, none, out=kept)[0] == 7).all()
    empty = mxfp4.quantize(rand(0, k)) if mx else rand(0, k)
    assert experts.grouped_gemm(empty, b, none).shape == (0, n)


@gpu
@pytest.mark.parametrize('mx', [False, True])
@pytest.mark.parametrize('rows', [9, 600])
def test_a_wrong_plan_stays_inside_the_operands(rows, mx):
    """Indexes and offsets that point anywhere: no access outside, the rows
    of sound groups are right."""
    num, n, k = 5, 64, 128
    a, b = rand(rows, k, seed=1), rand(num, n, k, seed=2)
    if mx:
        a, b = mxfp4.quantize(a), mxfp4.quantize(b)
    index = torch.arange(rows, dtype=torch.int32, device='cuda')
    good = experts.grouped_gemm(a, b, torch.tensor(
        [0, 4, 4, 4, 4, rows], dtype=torch.int32, device='cuda'))
    index[1], index[2] = -1, 1 << 30
    offsets = torch.tensor([-7, 4, 4, 4, 4, 1 << 30], dtype=torch.int32,
                           device='cuda')
    out = experts.grouped_gemm(a, b, offsets, rows=index)
    assert torch.equal(out[3:], good[3:]) and torch.equal(out[0], good[0])
    falling = torch.tensor([rows, 4, 2, 1, 0, -3], dtype=torch.int32,
                           device='cuda')
    experts.grouped_gemm(a, b, falling, rows=index)
    torch.cuda.synchronize()


@gpu
@pytest.mark.parametrize('mx', [False, True])
@pytest.mark.parametrize('num,rows,n,k', [(9, 1024, 256, 2048),
                                          (70, 2560, 48, 4096),
                                          (9, 200, 64, 256)])
def test_groups_that_overlap_stay_inside_the_workspace(num, rows, n, k, mx):
    """Offsets that go up and down make more rows than there are: what is
    behind the workspace and the result stays as it was."""
    a, b = rand(rows, k, seed=1), rand(num, n, k, seed=2)
    if mx:
        a, b = mxfp4.quantize(a), mxfp4.quantize(b)
    offsets = torch.tensor([0, rows] * (num + 1), dtype=torch.int32,
                           device='cuda')[:num + 1]
    words = experts.workspace_bytes(a, b) // 4
    whole = torch.full((words + 65536 * 4,), 7.0, device='cuda')
    out = torch.full((rows + 256, n), 3.0, dtype=BF16, device='cuda')
    experts.grouped_gemm(a, b, offsets.contiguous(), out=out[:rows],
                         workspace=whole[:words])
    assert bool((whole[words:] == 7).all()) and bool((out[rows:] == 3).all())


@gpu
def test_combine_of_many_tokens():
    """More tokens than one grid takes."""
    tokens = (1 << 23) + 5
    y = rand(37, 8, seed=1)
    positions = torch.arange(tokens, dtype=torch.int32, device='cuda') % 40
    weights = torch.full((tokens, 1), 0.5, device='cuda')
    residual = torch.ones(tokens, 8, dtype=BF16, device='cuda')
    out = experts.combine(y, positions.view(-1, 1), weights, residual)
    table = torch.zeros(40, 8, device='cuda')
    table[:37] = y
    assert torch.equal(out, (1 + 0.5 * table).to(BF16)[positions.long()])


CAPTURE = """
import torch
from kiosk_autoscaler_amd.ops import experts, mxfp4
from kiosk_autoscaler_amd.ops import native
native.load()
g = torch.Generator().manual_seed(3)
x = torch.randn(300, 256, generator=g).to(torch.bfloat16).cuda()
w = torch.randn(4, 512, 256, generator=g).to(torch.bfloat16).cuda()
logits = torch.randn(300, 4, generator=g).cuda()
torch.cuda.synchronize()


def run():
    plan = experts.route(logits, 2)
    h = experts.grouped_gemm(x, w, plan.offsets, rows=plan.tokens)
    q = mxfp4.quantize(h)
    v = mxfp4.Mxfp4(q.codes[:64], q.scales[:64])
    return experts.combine(mxfp4.gemm(q, v), plan.positions, plan.weights)


graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = run()
for _ in range(3):
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, run())
print('same')
"""


@gpu
def test_the_first_calls_of_a_process_may_be_captured():
    done = subprocess.run([sys.executable, '-c', CAPTURE], timeout=100,
                          capture_output=True, text=True,
                          cwd=os.path.dirname(os.path.dirname(__file__)))
    assert done.returncode == 0 and 'same' in done.stdout, done.stderr


@gpu
@pytest.mark.parametrize('mx', [False, True])
def test_one_row_does_not_depend_on_its_neighbours(mx):
    """A row's result is the same wherever the batch puts it within one
    size, and a NaN row stays alone."""
    rows, n, k = 300, 256, 384
    a, b = rand(rows, k, seed=1), rand(1, n, k, seed=2)
    a[17] = math.nan
    offsets = torch.tensor([0, rows], dtype=torch.int32, device='cuda')
    order = torch.randperm(rows, generator=torch.Generator().manual_seed(1))
    order = order.to(torch.int32).cuda()
    if mx:
        a, b = mxfp4.quantize(a), mxfp4.quantize(b)
    out = experts.grouped_gemm(a, b, offsets)
    assert out[17].isnan().all() and int(out.isnan().sum()) == n
    moved = experts.grouped_gemm(a, b, offsets, rows=order)
    assert torch.equal(moved.view(torch.int16),
                       out[order.long()].view(torch.int16))


@gpu
def test_results_and_inputs_past_two_to_the_31():
    """More than 2^31 elements in the result, 4 GiB in a gathered input."""
    rows, n, k, num = 140000, 16384, 64, 2
    offsets = torch.tensor([0, 70001, rows], dtype=torch.int32,
                           device='cuda')
    a, b = rand(rows, k, seed=1), rand(num, n, k, seed=2)
    out = experts.grouped_gemm(a, b, offsets)
    for at, e in ((0, 0), (70000, 0), (70001, 1), (131072, 1), (rows - 1, 1)):
        check_product(out[at:at + 1], a[at:at + 1].double(), b[e].double(),
                      'none')
    del out
    rows, k = 600000, 4096
    a = torch.empty(rows, k, dtype=BF16, device='cuda')
    a[:] = rand(1, k, seed=3)
    a[-3:] = rand(3, k, seed=4)
    b = rand(1, 32, k, seed=5)
    index = torch.tensor([rows - 1, 0, rows - 3], dtype=torch.int32,
                         device='cuda')
    out = experts.grouped_gemm(a, b, torch.tensor(
        [0, 3], dtype=torch.int32, device='cuda'), rows=index)
    check_product(out, a[index.long()].double(), b[0].double(), 'none')
    wide = index.repeat(300)
    out = experts.grouped_gemm(a, b, torch.tensor(
        [0, 900], dtype=torch.int32, device='cuda'), rows=wide)
    check_product(out, a[wide.long()].double(), b[0].double(), 'none')
    x = a.view(-1)[:(1 << 31) + 64].view(-1, 32)
    x[-1] = rand(32, seed=6)
    q = mxfp4.quantize(x)
    want, scales = ref_quantize(x[-2:])
    assert torch.equal(q.scales[-2:].int(), scales.int())
    assert torch.equal(mxfp4.dequantize(q)[-2:].double(), want)


def expert_mlp(x, logits, w1, b1, w2, b2, k, mx):
    plan = experts.route(logits, k)
    h = experts.grouped_gemm(mxfp4.quantize(x) if mx else x, w1,
                             plan.offsets, b1, 'gelu', rows=plan.tokens)
    y = experts.grouped_gemm(mxfp4.quantize(h) if mx else h, w2,
                             plan.offsets, b2, 'bias')
    return experts.combine(y, plan.positions, plan.weights, residual=x)


@gpu
@pytest.mark.parametrize('mx', [False, True])
@pytest.mark.parametrize('tokens', [1, 3, 64, 300])
def test_expert_mlp_block(tokens, mx):
    """The operators as one block, against float64 with the same storage
    points."""
    num, k, dim, hidden = 8, 2, 256, 512
    x, logits = rand(tokens, dim, seed=1), rand(tokens, num, seed=2)
    if tokens > 3:
        logits[-2:] = -math.inf                      # padding: y = x
    w1 = rand(num, hidden, dim, seed=3, scale=dim ** -0.5)
    w2 = rand(num, dim, hidden, seed=4, scale=hidden ** -0.5)
    b1 = rand(num, hidden, seed=5, scale=0.1, dtype=torch.float32)
    b2 = rand(num, dim, seed=6, scale=0.1, dtype=torch.float32)
    if mx:
        w1, w2 = mxfp4.quantize(w1), mxfp4.quantize(w2)
    out = expert_mlp(x, logits, w1, b1, w2, b2, k, mx)
    chosen, weights, _, _, _ = ref_route(logits, k)
    v1, v2 = (values_of(w1), values_of(w2)) if mx else (w1.double(),
                                                        w2.double())
    want = x.double().clone()
    for t in range(tokens):
        xt = ref_quantize(x[t])[0] if mx else x[t].double()
        for e, w in zip(chosen[t], weights[t]):
            if e < 0:
                continue
            h = gelu(v1[e] @ xt + b1[e].double()).to(BF16)
            h = ref_quantize(h)[0] if mx else h.double()
            y = (v2[e] @ h + b2[e].double()).to(BF16)
            want[t] += w * y.double()
    # h and y are rounded to bf16 on both sides; where fp32 and float64 round
    # h apart (one step, 2^-7 of it) y moves by |w2| |h| 2^-7 at the worst of
    # a few elements, and with MXFP4 such an element may step by a quarter of
    # the block's largest: bounds on the whole vector, not an element
    err = (out.double() - want).norm(dim=1)
    size = want.norm(dim=1)
    assert (err <= (2.0 ** -4 if mx else 2.0 ** -7) * size).all(), \
        float((err / size).max())
    if tokens > 3:
        assert torch.equal(out[-2:], x[-2:])


@gpu
@pytest.mark.parametrize('mx', [False, True])
def test_block_in_a_captured_graph(mx):
    """Captured on a side stream and replayed with new inputs between eager
    calls; every replay equals the eager block bit for bit."""
    tokens, num, k, dim, hidden = 200, 8, 2, 256, 512
    w1 = rand(num, hidden, dim, seed=3, scale=dim ** -0.5)
    w2 = rand(num, dim, hidden, seed=4, scale=hidden ** -0.5)
    b1 = rand(num, hidden, seed=5, dtype=torch.float32)
    b2 = rand(num, dim, seed=6, dtype=torch.float32)
    if mx:
        w1, w2 = mxfp4.quantize(w1), mxfp4.quantize(w2)
    x, logits = rand(tokens, dim, seed=1), rand(tokens, num, seed=2)
    expert_mlp(x, logits, w1, b1, w2, b2, k, mx)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = expert_mlp(x, logits, w1, b1, w2, b2, k, mx)
    other = torch.cuda.CUDAGraph()
    with torch.cuda.graph(other):
        second = expert_mlp(x, logits, w1, b1, w2, b2, k, mx)
    for seed in range(4):
        x.copy_(rand(tokens, dim, seed=10 + seed))
        logits.copy_(rand(tokens, num, seed=20 + seed))
        eager = expert_mlp(x, logits, w1, b1, w2, b2, k, mx)
        graph.replay()
        other.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        assert torch.equal(second, eager)


@gpu
def test_block_in_the_native_stream_graph():
    """With ``out`` for every call the native graph holds no memory that the
    allocator hands to someone else."""
    mod = native.load()
    tokens, num, k, dim, n = 300, 8, 2, 256, 128
    logits, x = rand(tokens, num, seed=1), rand(tokens, dim, seed=2)
    w = rand(num, n, dim, seed=3)
    res = rand(tokens, n, seed=4)
    plan = experts.empty_plan(tokens, num, k)
    y = torch.empty(tokens * k, n, dtype=BF16, device='cuda')
    out = torch.empty(tokens, n, dtype=BF16, device='cuda')

    def block():
        experts.route(logits, k, out=plan)
        experts.grouped_gemm(x, w, plan.offsets, rows=plan.tokens, out=y)
        experts.combine(y, plan.positions, plan.weights, res, out=out)
    block()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        graph = mod.StreamGraph(side.cuda_stream)
        graph.begin()
        block()
        graph.end()
    for seed in range(3):
        x.copy_(rand(tokens, dim, seed=30 + seed))
        block()
        want = out.clone()
        out.zero_()
        junk = [torch.full((1 << 20,), math.nan, device='cuda')
                for _ in range(4)]
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.launch()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        del junk
    graph.reset()


@gpu
def test_calls_run_on_the_callers_stream():
    """Inputs written on a side stream just before the call on it."""
    side = torch.cuda.Stream()
    a, b = rand(512, 4096, seed=1), rand(1, 4096, 4096, seed=2)
    offsets = torch.tensor([0, 512], dtype=torch.int32, device='cuda')
    want = experts.grouped_gemm(a, b, offsets)
    staged = torch.zeros_like(a)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(20):
            staged.copy_(b[0, :512] * 0)
        staged.copy_(a)
        got = experts.grouped_gemm(staged, b, offsets)
        q = mxfp4.dequantize(mxfp4.quantize(staged))
    side.synchronize()
    assert torch.equal(got, want)
    assert torch.equal(q, mxfp4.dequantize(mxfp4.quantize(a)))


@gpu
@pytest.mark.parametrize('mx', [False, True])
def test_calls_on_two_streams_at_once(mx):
    """Products on streams of their own, sliced ones among them, each with
    its temporary workspace."""
    sizes = ((300, 512, 4096), (520, 384, 8192), (300, 512, 16384))
    jobs, sliced = [], 0
    for i, (m, n, k) in enumerate(sizes):
        a, b = rand(m, k, seed=i), rand(2, n, k, seed=7 + i)
        if mx:
            a, b = mxfp4.quantize(a), mxfp4.quantize(b)
        offsets = torch.tensor([0, m // 3, m], dtype=torch.int32,
                               device='cuda')
        sliced += experts.workspace_bytes(a, b) > 0
        jobs.append((a, b, offsets, experts.grouped_gemm(a, b, offsets),
                     torch.cuda.Stream()))
    assert sliced
    torch.cuda.synchronize()
    got = []
    for _ in range(30):
        for a, b, offsets, want, stream in jobs:
            with torch.cuda.stream(stream):
                got.append((experts.grouped_gemm(a, b, offsets), want))
    torch.cuda.synchronize()
    for out, want in got:
        assert torch.equal(out, want)


def kernel_of(a, b, rows=None, grouped=True):
    """The kernel that a product runs on."""
    mx = isinstance(a, mxfp4.Mxfp4)
    part_a, part_b = (a.codes, b.codes) if mx else (a, b)
    return native.load().product_kernel(
        mx, grouped, rows is not None, part_a.shape[0],
        part_a.shape[0] if rows is None else rows.numel(), part_b.shape[-2],
        part_a.shape[1] * part_a.element_size(),
        part_b.shape[0] if grouped else 1,
        native.load().device_cus(part_a.device.index))


def whole_mx(*shape, seed):
    """Multiples of a half up to 24, every code under three scales."""
    q = random_mx(*shape, seed=seed)
    g = torch.Generator(device='cuda').manual_seed(seed + 1)
    q.scales[:] = torch.randint(127, 130, q.scales.shape, generator=g,
                                device='cuda', dtype=torch.uint8)
    return q


def whole_bf16(*shape, seed):
    """Whole numbers up to 56, a power of two for every 32 of them."""
    g = torch.Generator(device='cuda').manual_seed(seed)
    x = torch.randint(-7, 8, shape[:-1] + (shape[-1] // 32, 32), generator=g,
                      device='cuda')
    e = torch.randint(0, 4, shape[:-1] + (shape[-1] // 32, 1), generator=g,
                      device='cuda')
    return (x << e).view(shape).to(BF16)


def exact_product(a, b, bias=None, residual=None):
    """The product of whole numbers, rounded once.  All terms are multiples
    of a quarter and their magnitudes add up to less than 2^22: every sum of
    some of them is an fp32 number, in whichever order they are added."""
    y = a @ b.t()
    size = a.abs() @ b.abs().t()
    for part in (bias, residual):
        if part is not None:
            y, size = y + part.double(), size + part.double().abs()
    assert float(size.max()) < 2.0 ** 22
    assert torch.equal(y.float().double(), y)
    return y.float().to(BF16)


# kernel, rows, experts, n, K of MXFP4, K of bf16.  Rows of MXFP4 end with
# half a step of 128 bytes wherever K is no multiple of 256; of the few-rows
# kernel with 64, 128 or 192 bytes behind the last 256
EXACT = [
    # few rows, a wave for every quarter of the row, many turns each
    ('rows', 3, 1, 128, 16384, 8192), ('rows', 17, 1, 96, 32768, 8256),
    ('rows', 50, 2, 272, 16768, 4160),
    # one to four rows a group, many columns: rows of 2 KiB and more
    ('rows', 8, 8, 2048, 3968, 960), ('rows', 4, 4, 4096, 8576, 2112),
    # five and more: four waves, one wave
    ('rows', 24, 4, 4096, 8448, 2112), ('rows', 128, 16, 4096, 3968, 960),
    ('rows', 100, 4, 4096, 8576, 2112), ('rows', 100, 4, 9632, 2176, 576),
    # 128 x 128 tiles: at most one for each CU, two
    ('tile128', 300, 1, 528, 2176, 576), ('tile128', 900, 5, 528, 1920, 512),
    ('tile128', 900, 5, 4096, 4096, 1024),
    # 256 x 256 tiles: slices of few tiles and of a last round, none
    ('tile256', 300, 2, 528, 16768, 4160), ('tile256', 300, 1, 272, 8576,
                                            2112),
    ('tile256', 2000, 3, 4624, 8448, 2112), ('tile256', 1100, 8, 8192, 1152,
                                             320),
    ('tile256', 5000, 7, 2064, 8320, 2240)]


@gpu
@pytest.mark.parametrize('mx', [False, True])
@pytest.mark.parametrize('kernel,rows,num,n,k_mx,k_bf16', EXACT)
def test_products_of_whole_numbers_are_exact(kernel, rows, num, n, k_mx,
                                             k_bf16, mx):
    """A block of the inner dimension that is lost, read twice or scaled by
    its neighbour's scale shows as a wrong number."""
    k, make = (k_mx, whole_mx) if mx else (k_bf16, whole_bf16)
    a, b = make(rows, k, seed=rows), make(num, n, k, seed=n)
    offsets = cut(rows, num, 1)
    assert kernel_of(a, b) == kernel
    bias = torch.randint(-99, 100, (num, n), device='cuda',
                         generator=torch.Generator('cuda').manual_seed(
                             5)).float()
    out = experts.grouped_gemm(a, b, offsets, bias, 'bias')
    va, vb = (values_of(a), values_of(b)) if mx else (a.double(), b.double())
    bounds = offsets.tolist()
    for e in range(num):
        lo, hi = bounds[e], bounds[e + 1]
        if lo < hi:
            assert torch.equal(out[lo:hi], exact_product(va[lo:hi], vb[e],
                                                         bias[e])), e
    order = torch.randperm(rows, generator=torch.Generator().manual_seed(2))
    order = order.to(torch.int32).cuda()
    assert kernel_of(a, b, order) == kernel
    out = experts.grouped_gemm(a, b, offsets, rows=order)
    for e in range(num):
        lo, hi = bounds[e], bounds[e + 1]
        if lo < hi:
            assert torch.equal(out[lo:hi], exact_product(
                va[order[lo:hi].long()], vb[e])), e


@gpu
@pytest.mark.parametrize('kernel,m,n,k', [
    ('rows', 3, 128, 16384), ('rows', 1, 4096, 16768),
    ('rows', 30, 4096, 8576), ('tile128', 300, 528, 2176),
    ('tile128', 900, 4096, 4096), ('tile256', 300, 528, 16768),
    ('tile256', 1000, 1040, 8320), ('tile256', 2600, 8208, 1152)])
def test_mxfp4_products_with_a_residual_are_exact(kernel, m, n, k):
    a, b = whole_mx(m, k, seed=m), whole_mx(n, k, seed=n)
    assert kernel_of(a, b, grouped=False) == kernel
    g = torch.Generator(device='cuda').manual_seed(3)
    bias = torch.randint(-99, 100, (n,), generator=g, device='cuda').float()
    res = torch.randint(-99, 100, (m, n), generator=g, device='cuda').to(BF16)
    want = exact_product(values_of(a), values_of(b), bias, res)
    assert torch.equal(mxfp4.gemm(a, b, bias, res, 'residual'), want)
    assert torch.equal(mxfp4.gemm(a, b, bias, res, 'residual', out=res), want)


@gpu
@pytest.mark.parametrize('n,k', [(32, 4096), (16400, 4096), (65552, 1024)])
def test_few_rows_out_of_a_large_input_are_exact(n, k):
    """Groups of up to 64 rows, gathered from more than 4 GiB."""
    rows = (1 << 32) // (2 * k) + 7
    a = torch.zeros(rows, k, dtype=BF16, device='cuda')
    at = torch.cat([torch.arange(30), torch.arange(rows - 30, rows)])
    a[at.cuda()] = whole_bf16(60, k, seed=1)
    b = whole_bf16(1, n, k, seed=2)
    index = at.to(torch.int32).cuda()
    assert kernel_of(a, b, index) == 'rows'
    out = experts.grouped_gemm(a, b, torch.tensor(
        [0, 60], dtype=torch.int32, device='cuda'), rows=index)
    assert torch.equal(out, exact_product(a[at.cuda()].double(),
                                          b[0].double()))


@gpu
@pytest.mark.parametrize('mx', [False, True])
@pytest.mark.parametrize('rows,n', [(700, 272), (700, 16400)])
def test_rows_outside_the_groups_of_large_tiles(rows, n, mx):
    """256 x 256 tiles, sliced and whole: zero in a new result, as they were
    in ``out``; NaN there, or in an empty group's weights, reaches no other
    row."""
    num, k = 4, (10240 if mx else 2560) if n < 1024 else (640 if mx else 320)
    a, b = rand(rows, k, seed=1), rand(num, n, k, seed=2)
    a[:3] = math.nan
    a[rows - 5:] = math.nan
    b[3] = math.nan                                  # its group is empty
    offsets = torch.tensor([3, 9, 9, rows - 5, rows - 5], dtype=torch.int32,
                           device='cuda')
    if mx:
        a, b = mxfp4.quantize(a), mxfp4.quantize(b)
    assert kernel_of(a, b) == 'tile256'
    assert (experts.workspace_bytes(a, b) > 0) is (n < 1024)
    out = experts.grouped_gemm(a, b, offsets)
    assert (out[:3] == 0).all() and (out[rows - 5:] == 0).all()
    assert out[3:rows - 5].isfinite().all()
    kept = torch.full((rows, n), 7.0, dtype=BF16, device='cuda')
    assert experts.grouped_gemm(a, b, offsets, out=kept) is kept
    assert (kept[:3] == 7).all() and (kept[rows - 5:] == 7).all()
    assert torch.equal(kept[3:rows - 5], out[3:rows - 5])
    none = torch.zeros(num + 1, dtype=torch.int32, device='cuda')
    assert (experts.grouped_gemm(a, b, none) == 0).all()
    kept.fill_(7)
    assert (experts.grouped_gemm(a, b, none, out=kept) == 7).all()


@gpu
@pytest.mark.parametrize('mx', [False, True])
@pytest.mark.parametrize('kernel,rows,n,k', [
    ('rows', 30, 256, 8576), ('tile256', 300, 256, 10240),
    ('tile256', 300, 65552, 640)])
def test_one_row_does_not_depend_on_its_neighbours_in_any_kernel(
        kernel, rows, n, k, mx):
    """A row's result is the same wherever the batch puts it within one size,
    and a NaN row stays alone: few rows, and 256 x 256 tiles in slices and
    whole ones (the 128 x 128 ones have a test of their own)."""
    a, b = rand(rows, k, seed=1), rand(1, n, k, seed=2)
    a[17] = math.nan
    offsets = torch.tensor([0, rows], dtype=torch.int32, device='cuda')
    order = torch.randperm(rows, generator=torch.Generator().manual_seed(1))
    order = order.to(torch.int32).cuda()
    if mx:
        a, b = mxfp4.quantize(a), mxfp4.quantize(b)
    assert kernel_of(a, b) == kernel_of(a, b, order) == kernel
    out = experts.grouped_gemm(a, b, offsets)
    assert out[17].isnan().all() and int(out.isnan().sum()) == n
    moved = experts.grouped_gemm(a, b, offsets, rows=order)
    assert torch.equal(moved.view(torch.int16),
                       out[order.long()].view(torch.int16))


@gpu
def test_combine_of_a_wide_row():
    """More stretches of columns than 16 bits count."""
    width = (1 << 27) + 2048 + 8
    y = torch.ones(1, width, dtype=BF16, device='cuda')
    y[0, 1 << 27:] = 3
    positions = torch.zeros(1, 1, dtype=torch.int32, device='cuda')
    out = experts.combine(y, positions, torch.full((1, 1), 0.5,
                                                   device='cuda'))
    assert torch.equal(out, y / 2)


@gpu
@pytest.mark.parametrize('m,n,k', [(4, 512, 512), (512, 512, 1024),
                                   (1500, 1024, 4096)])
def test_a_bf16_residual_is_refused_by_the_binding(m, n, k):
    """Whatever tile the size picks: an error, nothing launched."""
    mod = native.load()
    a, b, out = rand(m, k), rand(n, k), rand(m, n, seed=2)
    bias = rand(n, dtype=torch.float32)
    offsets = torch.tensor([0, m], dtype=torch.int32, device='cuda')
    want = out.clone()
    with pytest.raises(RuntimeError, match='invalid'):
        mod.product(a.data_ptr(), 0, b.data_ptr(), 0, out.data_ptr(),
                    bias.data_ptr(), out.data_ptr(), offsets.data_ptr(), 0,
                    m, m, n, 2 * k, 1, 2, False, 256, 0,
                    torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(out, want)


@gpu
def test_grad_is_refused_and_no_grad_is_not():
    a = rand(4, 64, seed=1).requires_grad_()
    b, off = rand(1, 16, 64), torch.tensor([0, 4], dtype=torch.int32,
                                           device='cuda')
    with pytest.raises(ValueError, match='gradient'):
        experts.grouped_gemm(a, b, off)
    with torch.no_grad():
        assert experts.grouped_gemm(a, b, off).shape == (4, 16)
