"""torch.ops.vectra.residual_norm on the CPU and the GPU against the definition in
64 bits, with bounds derived from the roundings (oracle/block.py)."""

import itertools

import pytest
import torch

from oracle import block as oracle
from vectra_amd.kernels import block

DEVICES = ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)]
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [(F32, F32), (F16, F16), (F16, F32), (BF16, BF16), (BF16, F32)]
NAMES = ('x', 'residual', 'weight', 'bias', 'gate', 'post_weight', 'post_bias')


def make(shape, dtype, stream, *, norm='rms', post='none', gate=None, affine=True, p=0.0, scale=1.0, vectors=None, device='cpu',
         seed=0, offset=0.0, spread=1.0):
    """Arguments by name, and the options."""
    gen = torch.Generator().manual_seed(seed)
    vectors = vectors or stream
    width = shape[-1]

    def normal(*sizes, to, factor=1.0, plus=0.0):
        return torch.randn(*sizes, generator=gen).mul_(factor).add_(plus).to(to).to(device)

    t = {'x': normal(*shape, to=dtype, plus=offset, factor=spread), 'residual': normal(*shape, to=stream, factor=2.0, plus=offset)}
    if affine:
        t['weight'] = normal(width, to=vectors, factor=0.3, plus=1.0)
        if norm == 'layer':
            t['bias'] = normal(width, to=vectors, factor=0.3)
        if post != 'none':
            t['post_weight'] = normal(width, to=vectors, factor=0.3, plus=0.5)
        if post == 'layer':
            t['post_bias'] = normal(width, to=vectors, factor=0.3)
    if gate is not None:
        t['gate'] = normal(*gate, to=vectors, factor=0.5, plus=0.2)
    options = {'norm': norm, 'post': post, 'eps': 1e-5, 'residual_scale': scale, 'p': p, 'stream': 3}
    if p:
        options['rng'] = torch.tensor([seed * 77 + 5, 2], device=device)
    return t, options


def check(t, options, device, grads=(True, True), seed=99):
    """Forward and backward of one call within the oracle's bounds; returns the outputs."""
    leaves = {k: v.clone().requires_grad_() for k, v in t.items()} if any(grads) else t
    h, n = torch.ops.vectra.residual_norm(**{k: leaves.get(k) for k in NAMES}, **options)
    assert h.dtype == t['residual'].dtype and n.dtype == t['x'].dtype and h.shape == n.shape == t['x'].shape
    assert h.is_contiguous() and n.is_contiguous()
    told = {**options, 'rng': tuple(options['rng'].tolist()) if 'rng' in options else (0, 0)}
    want = oracle.Stream(**t, **told)
    for name, (value, bound) in want.forward().items():
        oracle.assert_within({'h': h, 'n': n}[name], value, bound)
    if not any(grads):
        return h, n, {}
    gen = torch.Generator().manual_seed(seed)
    gh = torch.randn(h.shape, generator=gen).to(h.dtype).to(device) if grads[0] else None
    gn = torch.randn(n.shape, generator=gen).to(n.dtype).to(device) if grads[1] else None
    outs = [(o, g) for o, g in ((h, gh), (n, gn)) if g is not None]
    got = torch.autograd.grad([o for o, _ in outs], list(leaves.values()), [g for _, g in outs], allow_unused=True)
    expected = want.backward(gh, gn)
    for name, g in zip(leaves, got):
        value, bound = expected[name]
        if g is None:
            assert not bool(value.any()), name
            continue
        assert g.dtype == t[name].dtype and g.shape == t[name].shape
        oracle.assert_within(g, value, bound)
    return h, n, dict(zip(leaves, got))


# Widths at the edges of a lane, of 128 to 1024 lanes and of two chunks per lane.
WIDTHS = [1, 7, 8, 9, 127, 128, 129, 256, 257, 512, 520, 1000, 1024, 1032, 2048, 2056, 4096, 4104]


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('width', WIDTHS)
def test_widths(width, device):
    for norm, post in (('rms', 'none'), ('layer', 'layer'), ('rms', 'rms')):
        check(*make((5, width), BF16, F32, norm=norm, post=post, gate=(width,) if post != 'none' else None, device=device,
                    seed=width), device)


@pytest.mark.gpu
@pytest.mark.parametrize('width', [6000, 8192, 8200, 12288, 16384])
@pytest.mark.parametrize('dtype,stream', [(BF16, F32), (F32, F32)])
def test_the_widest_rows(width, dtype, stream):
    check(*make((6, width), dtype, stream, norm='layer', post='layer', gate=(width,), p=0.25, device='cuda', seed=width), 'cuda')
    check(*make((6, width), dtype, stream, norm='rms', device='cuda', seed=width), 'cuda')


@pytest.mark.gpu
@pytest.mark.parametrize('width', [4097, 8190, 8192, 9001, 16383, 16384])
@pytest.mark.parametrize('gate,post', [('none', 'none'), ('none', 'layer'), ('vector', 'none'), ('sequence', 'rms'), ('full', 'layer')])
def test_the_widest_rows_of_several_turns(width, gate, post):
    """Sums of several rows in a workgroup, with each set of vectors."""
    shape = (3, 230, width)
    gate = {'none': None, 'vector': (width,), 'sequence': (3, 1, width), 'full': shape}[gate]
    check(*make(shape, BF16, F32, norm='layer', post=post, gate=gate, p=0.25 if post == 'layer' else 0.0, device='cuda', seed=width), 'cuda')


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('dtype,stream', TYPES, ids=str)
@pytest.mark.parametrize('norm', block.NORMS)
@pytest.mark.parametrize('post', block.POST_NORMS)
def test_types_norms_gates(dtype, stream, norm, post, device):
    shape = (3, 7, 136)
    for i, (gate, p, scale) in enumerate(itertools.product((None, (136,), (3, 1, 136), (3, 7, 136)), (0.0, 0.3), (1.0, -0.75))):
        check(*make(shape, dtype, stream, norm=norm, post=post, gate=gate, p=p, scale=scale, device=device, seed=i,
                    vectors=dtype if i % 2 else F32, affine=i % 3 != 2), device)


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('rows', [1, 2, 15, 16, 17, 33, 100, 1000])
def test_rows(rows, device):
    check(*make((rows, 128), BF16, BF16, norm='layer', p=0.1, device=device, seed=rows), device)
    check(*make((rows, 96), F16, F32, post='rms', gate=(96,), device=device, seed=rows), device)
    check(*make((rows, 600), F32, F32, norm='layer', post='layer', gate=(1, 600), device=device, seed=rows), device)


@pytest.mark.gpu
def test_many_rows():
    """Rows enough for several turns of every workgroup, of each geometry."""
    for width, rows in ((128, 40000), (256, 9000), (512, 9001), (1024, 4001), (2048, 2100), (4096, 1100), (8192, 600)):
        check(*make((rows, width), BF16, F32, norm='layer', post='rms', gate=(width,), device='cuda', seed=width), 'cuda')
    check(*make((66560, 128), BF16, BF16, norm='layer', p=0.1, device='cuda'), 'cuda')


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('batch,tokens', [(1, 9), (9, 1), (40, 3), (3, 200), (2, 17)])
@pytest.mark.parametrize('width', [64, 300, 1032])
def test_gates_of_sequences(batch, tokens, width, device):
    """Gradients of shared and of broadcast gates, rows of a group in one part and in several."""
    for gate in ((batch, 1, width), (1, 1, width), (width,), (batch, tokens, width)):
        check(*make((batch, tokens, width), F32, F32, norm='layer', gate=gate, p=0.2, device=device, seed=tokens), device)


@pytest.mark.gpu
def test_gates_of_more_sequences_than_workgroups():
    check(*make((3000, 5, 128), BF16, BF16, norm='layer', gate=(3000, 1, 128), post='layer', device='cuda'), 'cuda')
    check(*make((700, 9, 1152), F16, F16, gate=(700, 1, 1152), device='cuda'), 'cuda')
    check(*make((2, 3, 500, 64), F32, F32, gate=(2, 3, 1, 64), device='cuda'), 'cuda')
    check(*make((2, 3, 500, 64), F32, F32, gate=(2, 1, 1, 64), device='cuda'), 'cuda')


@pytest.mark.parametrize('device', DEVICES)
def test_one_of_the_two_gradients(device):
    for grads in ((True, False), (False, True)):
        check(*make((6, 100), F32, F32, norm='layer', p=0.3, device=device), device, grads)
        check(*make((6, 100), BF16, F32, post='layer', gate=(100,), device=device), device, grads)


@pytest.mark.parametrize('device', DEVICES)
def test_only_the_wanted_gradients(device):
    t, options = make((5, 72), F32, F32, norm='layer', post='layer', gate=(72,), p=0.2, device=device)
    _, _, full = check(t, options, device)
    gen = torch.Generator().manual_seed(99)
    gh, gn = (torch.randn(5, 72, generator=gen).to(device) for _ in range(2))
    for name in t:
        leaves = {k: v.clone().requires_grad_(k == name) for k, v in t.items()}
        h, n = block.residual_norm(**leaves, **options)
        g, = torch.autograd.grad((h, n), leaves[name], (gh, gn))
        assert torch.equal(g, full[name]), name


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('kwargs', [dict(norm='layer', post='layer', gate=(3, 1, 5), p=0.25, scale=0.5), dict(norm='rms', p=0.4),
                                    dict(norm='rms', post='rms', gate=(5,))])
def test_gradients_against_differences(kwargs, device):
    """Central differences of the operator itself, in fp32: a step of 2^-8 leaves a relative error of its square
    (times a third derivative of order one) and of the sums' roundings over it."""
    t, options = make((3, 2, 5), F32, F32, device=device, **kwargs)
    leaves = {k: v.clone().requires_grad_() for k, v in t.items()}
    gen = torch.Generator().manual_seed(4)
    gh, gn = (torch.randn(3, 2, 5, generator=gen).to(device) for _ in range(2))

    def total(args):
        h, n = block.residual_norm(**args, **options)
        return float((h.double() * gh).sum() + (n.double() * gn).sum())

    h, n = block.residual_norm(**leaves, **options)
    got = dict(zip(leaves, torch.autograd.grad((h, n), list(leaves.values()), (gh, gn))))
    step = 2.0 ** -8
    for name, value in t.items():
        for at in range(0, value.numel(), 3):
            sides = []
            for sign in (1, -1):
                moved = {k: v.clone() for k, v in t.items()}
                moved[name].view(-1)[at] += sign * step
                sides.append(total(moved))
            slope = (sides[0] - sides[1]) / (2 * step)
            # 60 outputs of magnitude below 8, each off by at most 64 u; third derivatives of a norm of five
            # elements with deviations above 1/2 stay below 200.
            limit = 60 * 8 * 64 * oracle.U / step + 200 * step ** 2
            assert abs(float(got[name].view(-1)[at]) - slope) < limit, (name, at)


@pytest.mark.parametrize('device', DEVICES)
def test_strides(device):
    t, options = make((4, 9, 40), BF16, F32, norm='layer', gate=(4, 1, 40), p=0.2, device=device)
    h, n = block.residual_norm(**t, **options)
    wide = torch.zeros(4, 9, 100, dtype=BF16, device=device)
    wide[..., 3:43] = t['x']
    turned = t['residual'].transpose(0, 2).contiguous().transpose(0, 2)
    spread = torch.zeros(80, device=device)
    spread[::2] = t['weight']
    lines = torch.zeros(4, 3, 40, device=device)
    lines[:, :1] = t['gate']
    for other in ({'x': wide[..., 3:43]}, {'residual': turned}, {'weight': spread[::2]}, {'gate': lines[:, :1]}):
        h2, n2 = block.residual_norm(**{**t, **other}, **options)
        assert torch.equal(h, h2) and torch.equal(n, n2)
    # Broadcast inputs: their gradients are summed by autograd's expand.
    x = t['x'][:, :1].clone().requires_grad_()
    h, n = block.residual_norm(**{**t, 'x': x.expand(4, 9, 40)}, **options)
    g, = torch.autograd.grad(h.sum() + n.sum().float(), x)
    assert g.shape == x.shape
    # Gradients of any stride, expanded ones too.
    leaf = t['x'].clone().requires_grad_()
    h, n = block.residual_norm(**{**t, 'x': leaf}, **options)
    one = torch.ones((), device=device)
    a, = torch.autograd.grad((h, n), leaf, (one.expand(4, 9, 40), one.to(BF16).expand(4, 9, 40)), retain_graph=True)
    b, = torch.autograd.grad((h, n), leaf, (torch.ones_like(h), torch.ones_like(n)))
    assert torch.equal(a, b)


@pytest.mark.parametrize('device', DEVICES)
def test_hard_values(device):
    """A mean far above the deviation, tiny and large rows, constant rows, zeros."""
    for offset, spread in ((100.0, 1.0), (0.0, 1e-4), (0.0, 1e4)):
        check(*make((7, 264), F32, F32, norm='layer', post='layer', offset=offset, spread=spread, device=device), device)
    zero = torch.zeros(3, 50, device=device)
    h, n = block.residual_norm(zero, zero, norm='layer', post='layer')
    assert not bool(h.any()) and not bool(n.any())
    h, n = block.residual_norm(zero + 3, zero + 5, norm='layer', eps=1e-5)
    assert bool((h == 8).all()) and float(n.abs().max()) <= 8 * oracle.ROW_DEPTH * oracle.U * 1e-5 ** -0.5


@pytest.mark.parametrize('device', DEVICES)
def test_rows_with_nan_and_infinity_stay_alone(device):
    t, options = make((20, 130), F32, F32, norm='layer', post='layer', gate=(130,), device=device)
    h, n = block.residual_norm(**t, **options)
    t['x'][3, 129] = float('nan')
    t['residual'][7, 0] = float('inf')
    h2, n2 = block.residual_norm(**t, **options)
    assert bool(torch.isnan(n2[3]).all()) and bool(torch.isnan(n2[7]).any())
    others = [r for r in range(20) if r not in (3, 7)]
    assert torch.equal(h[others], h2[others]) and torch.equal(n[others], n2[others])


@pytest.mark.parametrize('device', DEVICES)
def test_empty(device):
    for shape in ((0, 8), (3, 0), (0, 0), (2, 0, 8), (0,)):
        t, options = make(shape, F32, F32, norm='layer', post='layer', gate=shape[-1:], device=device)
        leaves = {k: v.requires_grad_() for k, v in t.items()}
        h, n = block.residual_norm(**leaves, **options)
        assert h.shape == n.shape == torch.Size(shape)
        for leaf, g in zip(leaves.values(), torch.autograd.grad((h, n), list(leaves.values()), (h, n))):
            assert g.shape == leaf.shape and not bool(g.any())
    t, options = make((4, 0, 8), F32, F32, gate=(4, 1, 8), device=device)
    g, = torch.autograd.grad(block.residual_norm(**{**t, 'gate': t['gate'].requires_grad_()}, **options)[1].sum(), t['gate'])
    assert g.shape == (4, 1, 8) and not bool(g.any())


@pytest.mark.parametrize('device', DEVICES)
def test_dropout_is_the_operator_s_own(device):
    t, options = make((6, 90), F32, F32, p=0.35, device=device)
    h, _ = block.residual_norm(**t, **options)
    y = block.dropout(t['x'], 0.35, options['rng'], options['stream'])
    assert torch.equal(h, t['residual'] + y)


@pytest.mark.parametrize('device', DEVICES)
def test_eight_bit_rows_are_the_quantised_norm(device):
    for width in (1, 100, 128, 129, 512, 1000, 4096):
        t, options = make((9, width), F32, F32, norm='layer', post='rms', gate=(width,), device=device, seed=width)
        h, n = block.residual_norm(**t, **options)
        h8, codes, scales = block.residual_norm_8bit(**t, **options)
        assert torch.equal(h, h8)
        want = oracle.quantize(n, 1)
        assert codes.shape == want[0].shape and scales.shape == want[1].shape
        assert torch.equal(codes.view(torch.uint8).cpu(), want[0]) and torch.equal(scales.view(torch.uint8).cpu(), want[1])


@pytest.mark.parametrize('device', DEVICES)
def test_refusals(device):
    t, options = make((4, 9, 16), BF16, F32, norm='layer', post='layer', gate=(4, 1, 16), p=0.5, device=device)

    def refuse(match, error=RuntimeError, **other):
        with pytest.raises(error, match=match):
            block.residual_norm(**{**t, **options, **other})
        with pytest.raises(error, match=match):
            block.residual_norm_8bit(**{**t, **options, **other})

    refuse('of one shape', residual=t['residual'][:3])
    refuse('x must be float32', x=t['x'].double())
    refuse("residual must have x's dtype or float32", residual=t['residual'].half())
    for name in ('weight', 'bias', 'post_weight', 'post_bias'):
        refuse(f'{name} must be', **{name: torch.ones(15, device=device)})
        refuse(f"{name} must have x's dtype or float32", **{name: t[name].half()})
    refuse('gate must be', gate=torch.ones(1, 9, 16, device=device))
    refuse('gate must be', gate=torch.ones(4, 16, device=device))
    refuse('last dimension must be', gate=torch.ones(4, 1, 1, device=device))
    refuse("gate must have x's dtype", gate=t['gate'].half())
    refuse('need a post norm', post='none')
    refuse('norm must be', ValueError, norm='none')
    refuse('post must be', ValueError, post='batch')
    refuse('eps must be', ValueError, eps=-1e-6)
    refuse('eps must be', ValueError, eps=float('inf'))
    refuse('p must be', ValueError, p=1.0)
    refuse('needs rng', rng=None)
    refuse('rng must be', rng=options['rng'].int())
    refuse('stream must be', ValueError, stream=-1)
    with torch.autograd.forward_ad.dual_level():
        refuse('forward', (NotImplementedError, RuntimeError), x=torch.autograd.forward_ad.make_dual(t['x'], t['x']))
    leaf = t['x'].clone().requires_grad_()
    with pytest.raises(RuntimeError, match='gradients of gradients'):
        torch.autograd.grad(block.residual_norm(**{**t, 'x': leaf}, **options)[1].sum(), leaf, create_graph=True)
    codes = block.residual_norm_8bit(**{**t, 'x': leaf}, **options)
    with pytest.raises(RuntimeError, match='not implemented'):
        codes[0].sum().backward()


@pytest.mark.gpu
def test_rows_too_wide_are_refused():
    x = torch.zeros(2, 16385, device='cuda')
    with pytest.raises(RuntimeError, match="exceeds the kernels' range"):
        block.residual_norm(x, x)
    with pytest.raises(RuntimeError, match='residual must be on'):
        block.residual_norm(x, x.cpu())


def test_refusals_of_the_backward_operator():
    t, options = make((4, 16), F32, F32, norm='layer', gate=(16,))
    g = torch.ones(4, 16)

    def call(h=None, x=t['x'], residual=t['residual'], grad_h=g, grad_n=g, gate=t['gate'], post='none', dtype=F32,
             wanted=(True,) + (False,) * 6):
        return torch.ops.vectra.residual_norm_backward(grad_h, grad_n, h, x, residual, t['weight'], t['bias'], gate, None, None,
                                                       'layer', post, 1e-5, 1.0, 0.0, None, 0, dtype, wanted)

    assert call()[0].shape == (4, 16)
    for kwargs, match in ((dict(x=None), 'x and residual'), (dict(gate=None, x=None, residual=None), 'needs h'),
                          (dict(grad_h=g[:3]), 'grad_h must be'), (dict(grad_n=g.half()), 'grad_n must be'),
                          (dict(dtype=BF16), 'x must have dtype'), (dict(dtype=torch.float64), 'dtype'),
                          (dict(wanted=(False,) * 5 + (True, False)), 'not given'),
                          (dict(gate=None, h=t['x'], wanted=(False,) * 4 + (True, False, False)), 'not given')):
        with pytest.raises(RuntimeError, match=match):
            call(**kwargs)


def test_opcheck():
    utils = ('test_schema', 'test_faketensor', 'test_autograd_registration')
    for kwargs in (dict(norm='layer', post='layer', gate=(2, 1, 130), p=0.25), dict(norm='rms')):
        t, options = make((2, 3, 130), F16, F32, **kwargs)
        args = tuple(t[k].requires_grad_() if k in t else None for k in NAMES)
        torch.library.opcheck(torch.ops.vectra.residual_norm.default, args, options, test_utils=utils)
        with torch.no_grad():
            plain = tuple(None if a is None else a.detach() for a in args)
            torch.library.opcheck(torch.ops.vectra.residual_norm_8bit.default, plain, options,
                                  test_utils=('test_schema', 'test_faketensor'))
    t, _ = make((2, 3, 130), F16, F32, norm='layer', gate=(130,))
    g = torch.ones(2, 3, 130)
    torch.library.opcheck(torch.ops.vectra.residual_norm_backward.default,
                          (g, g.half(), None, t['x'], t['residual'], t['weight'], t['bias'], t['gate'], None, None, 'layer', 'none',
                           1e-5, 1.0, 0.0, None, 0, F16, [True] * 5 + [False] * 2), test_utils=('test_schema', 'test_faketensor'))


@pytest.mark.gpu
def test_results_do_not_depend_on_the_run_or_the_stream():
    t, options = make((500, 3, 640), BF16, F32, norm='layer', post='layer', gate=(500, 1, 640), p=0.2, device='cuda')
    leaves = {k: v.requires_grad_() for k, v in t.items()}

    def run():
        h, n = block.residual_norm(**leaves, **options)
        return [h, n, *torch.autograd.grad((h, n), list(leaves.values()), (h.detach(), n.detach()))]

    want = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = run()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, again))


@pytest.mark.gpu
def test_captured_graphs_and_eager_calls_between_replays():
    """Two captured backward passes with workspaces of their own; rng moves with the replays."""
    ops = torch.ops.vectra
    graphs = []
    for width, seed in ((384, 1), (1024, 2)):
        t, options = make((70, width), BF16, F32, norm='layer', post='rms', gate=(width,), p=0.3, device='cuda', seed=seed)
        gh, gn = torch.randn(70, width, device='cuda'), torch.randn(70, width, device='cuda').bfloat16()
        wanted = [True] * 6 + [False]

        def step(t=t, o=options, gh=gh, gn=gn, wanted=wanted):
            h, n = ops.residual_norm(*(t.get(k) for k in NAMES), **o)
            return [h, n, *ops.residual_norm_backward(gh, gn, None, *(t.get(k) for k in NAMES), o['norm'], o['post'], o['eps'],
                                                      o['residual_scale'], o['p'], o['rng'], o['stream'], BF16, wanted)]

        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
            options['rng'][1].add_(1)
        graphs.append((graph, out, step, t, options))
    for _ in range(3):
        wants = []
        for graph, out, step, t, options in graphs:
            t['x'].normal_()
            wants.append(step())
        for graph, *_ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for want, (_, out, *_) in zip(wants, graphs):
            assert all(torch.equal(a, b) for a, b in zip(want, out))


@pytest.mark.parametrize('device', DEVICES)
@pytest.mark.parametrize('width', [40, 1000])
@pytest.mark.parametrize('norm', block.NORMS)
def test_rows_whose_mean_square_is_subnormal(width, norm, device):
    """Without eps.  Elements of 1e-20 to 2e-20 in alternating signs: each square, their
    mean and its product with 1 / width are off by half of 2^-149 at most, 7e-6 of 1e-40
    or more, and the root halves relative errors: less than 2^-16 together."""
    x = torch.rand(3, width, dtype=torch.float64, generator=torch.Generator().manual_seed(width)).add(1).mul(1e-20).float()
    x[:, ::2].neg_()
    centred = x.double() - (x.double().mean(-1, keepdim=True) if norm == 'layer' else 0)
    want = centred / centred.square().mean(-1, keepdim=True).sqrt()
    _, n = torch.ops.vectra.residual_norm(x.to(device), torch.zeros(3, width, device=device), norm=norm, eps=0.0)
    assert (n.cpu().double() - want).abs().max() <= 2.0 ** -16 * want.abs().max()
