"""ops.row_norm / block_tail against their formulas in 64 bits.

Tolerance: with `mag` = the formula's value over the absolute values of its terms, fp32 arithmetic is off by at most n 2^-24 mag, n = the longest chain
of roundings into a value: 32 for the elementwise chain with both norms (each root, exponential and reciprocal within 2 ulp), and the additions of
a sum: a row's values per thread and the tree over threads (<= 64), for a column's sum the rows of a block (<= 64 here) -- n = 160.  Results in
bf16 are rounded once: 2^-8 of the value."""
import pytest
import torch

from ha2g_amd import ops

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
EPS = 1e-5


def stats(x, g, kind):
    x = x.unflatten(-1, (g, -1))
    mu = x.mean(-1, keepdim=True) if kind == 'layer' else torch.zeros_like(x[..., :1])
    r = ((x - mu).pow(2).mean(-1, keepdim=True) + EPS).rsqrt()
    m = (x.abs() + (x.abs().mean(-1, keepdim=True) if kind == 'layer' else 0)) * r
    return ((x - mu) * r).flatten(-2), r, m.flatten(-2)


def back(a, xhat, r, g, kind, ma, mx):
    """gradient of the norm's input, and its magnitude"""
    u = lambda t: t.unflatten(-1, (g, -1))      # noqa: E731
    a, x, ma, mx = u(a), u(xhat), u(ma), u(mx)
    d = a - x * (a * x).mean(-1, keepdim=True) - (a.mean(-1, keepdim=True) if kind == 'layer' else 0.0)
    m = ma + mx * (ma * mx).mean(-1, keepdim=True) + ma.mean(-1, keepdim=True)
    return (d * r).flatten(-2), (m * r).flatten(-2)


def ref(t, kind, G, act, alpha):
    """{name: (value, magnitude)}; t: tensors by name, absent ones None"""
    d = {n: x.double().cpu() for n, x in t.items() if x is not None}
    if d['y'].dim() == 1:
        d = {n: x[None] if n in ('y', 'res', 'dh', 'dz') else x for n, x in d.items()}
    one = torch.ones((), dtype=torch.float64)
    if 'w' in d:
        yh, r1, my = stats(d['y'], G, kind)
        n, mn = yh * d['w'], my * d['w'].abs()
        if 'b' in d:
            n, mn = n + d['b'], mn + d['b'].abs()
    else:
        n, mn = d['y'], d['y'].abs()
    a = da = one
    if 'gate' in d:
        s = torch.sigmoid(d['gate'])
        a, da = {ops.ACT_NONE: (d['gate'], torch.ones_like(s)), ops.ACT_SIGMOID: (s, s * (1 - s)), ops.ACT_SILU: (d['gate'] * s, s * (1 + d['gate'] * (1 - s)))}[act]
        ma, mda = a.abs(), {ops.ACT_NONE: torch.ones_like(s), ops.ACT_SIGMOID: s, ops.ACT_SILU: s * (1 + d['gate'].abs())}[act]
    else:
        ma = mda = one
    sc = d.get('scale', one)
    u, mu = n * a, mn * ma
    h, mh = sc * u, sc.abs() * mu
    if 'res' in d:
        h, mh = h + alpha * d['res'], mh + abs(alpha) * d['res'].abs()
    out = dict(h=(h, mh))
    if 'w2' in d:
        hh, r2, _ = stats(h, 1, kind)
        m2 = (mh + (mh.mean(-1, keepdim=True) if kind == 'layer' else 0)) * r2.flatten(-2)
        # the root's own sensitivity: d(1/std)/std <= mean(|h| mh) r^2
        m2 = m2 + hh.abs() * (h.abs() * mh).mean(-1, keepdim=True) * r2.flatten(-2) ** 2
        z, mz = hh * d['w2'], m2 * d['w2'].abs()
        if 'b2' in d:
            z, mz = z + d['b2'], mz + d['b2'].abs()
        out['z'] = z, mz
    if 'dh' not in d and 'dz' not in d:
        return out
    rows = tuple(range(h.dim() - 1))
    dh = d['dh'] if 'dh' in d else torch.zeros_like(h)
    mdh = dh.abs()
    if 'w2' in d:
        dz = d.get('dz', torch.zeros_like(h))
        x, m = back(dz * d['w2'], hh, r2, 1, kind, (dz * d['w2']).abs(), m2)
        dh, mdh = dh + x, mdh + m
        out.update(dw2=((dz * hh).sum(rows), (dz.abs() * m2).sum(rows)), db2=(dz.sum(rows), dz.abs().sum(rows)))
    out.update(dres=(alpha * dh, abs(alpha) * mdh), dscale=((dh * u).sum(rows), (mdh * mu).sum(rows)))
    du, mdu = dh * sc, mdh * sc.abs()
    if 'gate' in d:
        g, m = du * n * da, mdu * mn * mda
        if d['gate'].shape != h.shape:
            ax = tuple(range(1, h.dim() - 1))
            g, m = g.sum(ax, keepdim=True), m.sum(ax, keepdim=True)
        out['dgate'] = g, m
    dn, mdn = du * a, mdu * ma
    if 'w' in d:
        out.update(dw=((dn * yh).sum(rows), (mdn * my).sum(rows)), db=(dn.sum(rows), mdn.sum(rows)))
        out['dy'] = back(dn * d['w'], yh, r1, G, kind, mdn * d['w'].abs(), my)
    else:
        out['dy'] = dn.expand_as(h), mdn.expand_as(h)
    return out


def check_all(shape, dt, kind='rms', G=1, act=ops.ACT_SILU, alpha=1.0, parts=('w', 'b'), gate=None, seed=0, row_norm=False, odd=False, grads=('dh', 'dz'), fill=None):
    gen = torch.Generator().manual_seed(seed)
    C = shape[-1]

    def r(*s, dt=torch.float32, at=0.0):
        x = (torch.randn(*s, generator=gen) + at).to(dt)
        return (torch.cat([x.new_zeros(1), x.flatten()]).to(DEV)[1:].view(x.shape) if odd else x.to(DEV)).requires_grad_()
    t = dict(y=r(*shape, dt=dt, at=0.4))
    if fill is not None:
        with torch.no_grad():
            t['y'][fill[0]] = fill[1]
    for n in ('w', 'b', 'scale', 'w2', 'b2'):
        t[n] = r(C, at=1.0 if n in ('w', 'w2') else 0.2) if n in parts else None
    t['res'] = r(*shape, dt=dt) if 'res' in parts else None
    t['gate'] = None if gate is None else r(*(shape if gate == 'token' else (shape[0],) + (1,) * (len(shape) - 2) + (C,)), dt=dt)
    dh, dz = r(*shape, dt=dt).detach(), r(*shape, dt=dt).detach()
    if row_norm:
        outs = (ops.row_norm(t['y'], t['w'], t['b'], kind=kind, groups=G, eps=EPS),)
    else:
        outs = ops.block_tail(t['y'], t['res'], gate=t['gate'], weight=t['w'], bias=t['b'], scale=t['scale'], alpha=alpha, kind=kind, groups=G, gate_act=act,
                              next_weight=t['w2'], next_bias=t['b2'], eps=EPS)
        outs = outs if t['w2'] is not None else (outs,)
    names = [n for n, x in t.items() if x is not None]
    use = [(o, n, d) for o, n, d in zip(outs, ('dh', 'dz'), (dh, dz)) if n in grads]
    got = dict(zip(('h', 'z'), (o.detach() for o in outs)))
    got.update(zip(('d' + n for n in names), torch.autograd.grad([o for o, _, _ in use], [t[n] for n in names], [d for _, _, d in use])))
    want = ref({**{n: None if x is None else x.detach() for n, x in t.items()}, **{n: d for _, n, d in use}}, kind, G, act, alpha)
    for n, x in got.items():
        v, m = (a[0] if a.dim() > x.dim() else a for a in want[n])
        tol = 160 * 2.0 ** -24 * m
        if x.dtype == torch.bfloat16:
            tol = tol + 2.0 ** -8 * (v.abs() + tol)
        off = (x.double().cpu() - v).abs()
        assert x.shape == v.shape and (off <= tol + 1e-37).all(), (n, float((off / (tol + 1e-37)).max()))
    return t, got


DTS = pytest.mark.parametrize('dt', (torch.float32, torch.bfloat16), ids=('fp32', 'bf16'))


@DTS
@pytest.mark.parametrize('kind', ('rms', 'layer'))
@pytest.mark.parametrize('C,G', ((1, 1), (3, 1), (4, 1), (16, 4), (27, 3), (64, 1), (126, 2), (300, 1), (300, 5), (300, 100), (300, 300), (1024, 8), (1025, 1), (1028, 1),
                                 (2000, 8), (2048, 16), (4100, 1), (5000, 5), (8191, 1), (16384, 128), (284, 4), (5270, 2), (16383, 3), (16384, 8192),
                                 (1026, 513), (9, 3), (2815, 5), (12, 4), (6000, 1000)))
def test_row_norm_sizes_and_groups(C, G, kind, dt):
    check_all((13, C), dt, kind=kind, G=G, row_norm=True, seed=C)


@DTS
@pytest.mark.parametrize('shape', ((1, 1, 24), (0, 5, 24), (3, 0, 24), (70, 24), (24,), (3, 2, 5, 24), (130, 7, 60)))
def test_shapes(shape, dt):
    check_all(shape, dt, row_norm=True)
    if len(shape) > 1:
        check_all(shape, dt, parts=('w', 'res', 'scale', 'w2', 'b2'), gate='sequence')


@DTS
@pytest.mark.parametrize('gate', (None, 'token', 'sequence'))
@pytest.mark.parametrize('parts', ((), ('w',), ('res',), ('w', 'b', 'res', 'scale'), ('w', 'b', 'res', 'scale', 'w2', 'b2'), ('res', 'w2'), ('scale', 'w2', 'b2')))
def test_every_part_alone_and_together(parts, gate, dt):
    check_all((4, 21, 40), dt, parts=parts, gate=gate, G=2, alpha=0.75, seed=len(parts))


@DTS
@pytest.mark.parametrize('act', (ops.ACT_NONE, ops.ACT_SIGMOID, ops.ACT_SILU))
@pytest.mark.parametrize('C', (40, 300, 1500, 2048, 4100, 5001, 9999))
def test_gates_and_widths(C, act, dt):
    check_all((2, 9, C), dt, kind='layer', G=3 if C % 3 == 0 else 1, parts=('w', 'b', 'res', 'scale', 'w2', 'b2'), gate='token', act=act, seed=C)


@DTS
def test_unaligned_and_strided_operands(dt):
    check_all((3, 11, 64), dt, parts=('w', 'b', 'res', 'scale', 'w2', 'b2'), gate='sequence', odd=True)
    x = torch.randn(7, 64, 5, device=DEV).to(dt).transpose(1, 2)
    w = torch.randn(64, device=DEV)
    assert torch.equal(ops.row_norm(x, w), ops.row_norm(x.contiguous(), w))


@pytest.mark.parametrize('grads', (('dh',), ('dz',)))
def test_a_gradient_that_never_came(grads):
    check_all((2, 9, 40), torch.float32, parts=('w', 'b', 'res', 'scale', 'w2', 'b2'), gate='token', grads=grads)


def test_constant_rows_and_one_bad_row():
    """a row of one value (no variance) is exact zeros under `layer`; a row that is not finite keeps to itself"""
    y = torch.full((5, 60), 0.5, device=DEV)
    assert torch.equal(ops.row_norm(y, torch.ones(60, device=DEV), kind='layer'), torch.zeros_like(y))
    y = torch.randn(6, 60, device=DEV)
    clean = ops.row_norm(y, torch.ones(60, device=DEV), groups=3)
    y[2, 5] = float('nan')
    y[3, 59] = float('inf')
    out = ops.row_norm(y, torch.ones(60, device=DEV), groups=3)
    keep = torch.ones(6, 60, dtype=torch.bool, device=DEV)
    keep[2, :20] = False
    keep[3, 40:] = False
    assert torch.equal(out[keep], clean[keep]) and not torch.isfinite(out[2, :20]).any()


def test_many_rows_in_few_blocks():
    """more rows than one pass of the grid holds: 40 000 of 24 values, forward and gradients of y only row by row"""
    y = torch.randn(40000, 24, device=DEV).requires_grad_()
    w = torch.randn(24, device=DEV).requires_grad_()
    dh = torch.randn(40000, 24, device=DEV)
    h = ops.row_norm(y, w)
    dy, dw = torch.autograd.grad(h, [y, w], dh)
    part = [torch.autograd.grad(ops.row_norm(y[i:i + 8000], w), [y, w], dh[i:i + 8000]) for i in range(0, 40000, 8000)]
    assert torch.equal(dy, sum(p[0] for p in part))
    yd = y.detach().double()
    yh = yd / (yd.pow(2).mean(1, keepdim=True) + EPS).sqrt()
    want, mag = (dh.double() * yh).sum(0), (dh.double() * yh).abs().sum(0)
    assert ((dw.double() - want).abs() <= 160 * 2.0 ** -24 * mag).all()


def test_graph_replays_and_streams():
    def run(y, res, gate, w, w2, dh, dz):
        ls = [x.detach().requires_grad_() for x in (y, res, gate, w, w2)]
        h, z = ops.block_tail(ls[0], ls[1], gate=ls[2], weight=ls[3], next_weight=ls[4], groups=2)
        return [h.detach(), z.detach(), *torch.autograd.grad([h, z], ls, [dh, dz])]

    def make(seed):
        g = torch.Generator().manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=g).to(DEV)      # noqa: E731
        return [r(5, 60, 40), r(5, 60, 40), r(5, 1, 40), r(40), r(40), r(5, 60, 40), r(5, 60, 40)]
    a, b = make(1), make(2)
    want = [[x.clone() for x in run(*t)] for t in (a, b)]
    s = torch.cuda.Stream()
    held = [x.clone() for x in a]
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run(*held)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out = run(*held)
    for src, w in ((b, want[1]), (a, want[0]), (b, want[1])):
        for x, y in zip(held, src):
            x.copy_(y)
        graph.replay()
        eager = run(*a)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, w)) and all(torch.equal(p, q) for p, q in zip(eager, want[0]))


def test_rows_past_two_to_the_32_elements():
    """2^32 + elements of bf16, forward and backward: the rows at the end are those of a small call"""
    C, rows = 4100, 2 ** 20 + 5
    assert rows * C > 2 ** 32
    y = torch.empty(rows, C, dtype=torch.bfloat16, device=DEV)
    y[:8].normal_()
    y[8:-8] = 0.0
    y[-8:].normal_()
    w = torch.randn(C, device=DEV)
    h = ops.row_norm(y, w)
    assert torch.equal(h[-8:], ops.row_norm(y[-8:], w)) and torch.equal(h[:8], ops.row_norm(y[:8], w)) and not h[8:-8:4097].any()
    y.requires_grad_()
    h = ops.row_norm(y, w)
    dy, = torch.autograd.grad(h, y, h.detach())
    tail = y.detach()[-8:].clone().requires_grad_()
    ht = ops.row_norm(tail, w)
    assert torch.equal(dy[-8:], torch.autograd.grad(ht, tail, ht.detach())[0])


def test_the_residual_may_be_changed_in_place_unless_the_second_norm_reads_it():
    y, res, w, w2 = (torch.randn(*s, device=DEV).requires_grad_() for s in ((6, 40), (6, 40), (40,), (40,)))
    dh = torch.randn(6, 40, device=DEV)
    want = torch.autograd.grad(ops.block_tail(y, res * 1, weight=w, alpha=0.5), (y, res, w), dh)
    r = res * 1
    h = ops.block_tail(y, r, weight=w, alpha=0.5)
    r.add_(1.0)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(h, (y, res, w), dh), want)) and torch.equal(want[1], 0.5 * dh)
    r = res * 1
    h, z = ops.block_tail(y, r, weight=w, next_weight=w2)
    r.add_(1.0)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        torch.autograd.grad(z, y, dh)


def test_a_second_derivative_is_refused():
    y, w = torch.randn(3, 8, device=DEV).requires_grad_(), torch.ones(8, device=DEV)
    gy, = torch.autograd.grad(ops.row_norm(y, w).square().sum(), y, create_graph=True)
    with pytest.raises(RuntimeError, match='once_differentiable'):
        (gy.sum() + y.sum()).backward()


@DTS
@pytest.mark.parametrize('gate', ('token', 'sequence'))
@pytest.mark.parametrize('C,G,kind', ((300, 2, 'layer'), (480, 4, 'rms'), (512, 1, 'rms'), (1000, 2, 'layer'), (1500, 2, 'rms'), (2000, 5, 'layer'), (2702, 2, 'rms'),
                                      (4096, 1, 'layer'), (4097, 1, 'layer'), (4100, 2, 'rms'), (4104, 3, 'layer'), (8192, 64, 'rms'), (8196, 4, 'layer'),
                                      (12001, 11, 'layer'), (16384, 1, 'rms')))
def test_everything_behind_the_norm_at_each_width(C, G, kind, gate, dt):
    check_all((2, 7, C), dt, kind=kind, G=G, parts=('w', 'b', 'res', 'scale', 'w2', 'b2'), gate=gate, alpha=0.7)


@pytest.mark.parametrize('parts,gate,grads', ((('w',), None, ('dh',)), (('res',), None, ('dh',)), (('scale', 'res'), 'sequence', ('dh',)), (('w2', 'b2'), None, ('dz',)),
                                              (('w2',), 'token', ('dh', 'dz')), (('w', 'b', 'w2'), None, ('dz',)), ((), 'sequence', ('dh',))))
@pytest.mark.parametrize('C,G', ((4200, 2), (16383, 3)))
def test_parts_of_wide_rows(C, G, parts, gate, grads):
    check_all((3, 5, C), torch.float32, kind='layer', G=G, parts=parts, gate=gate, grads=grads)


def test_wide_rows_of_many_slices():
    """more rows than a turn of every block, in slices that end inside one: the sums over 2 x 333 rows, and a gate for each sequence"""
    check_all((2, 333, 4098), torch.bfloat16, G=3, parts=('w', 'b', 'res', 'scale', 'w2', 'b2'), gate='sequence', odd=True)
    check_all((1, 700, 8200), torch.float32, kind='layer', parts=('w', 'b', 'res', 'scale', 'w2', 'b2'), gate='token')


@DTS
@pytest.mark.parametrize('kind', ('rms', 'layer'))
@pytest.mark.parametrize('C,G', ((40, 2), (300, 5), (300, 2), (1000, 8), (1500, 2), (2000, 8), (2702, 2), (4200, 3), (9000, 4), (12, 6)))
def test_without_an_eps(C, G, kind, dt, monkeypatch):
    """eps = 0 on rows that have a scale of their own: places that a row does not fill reach neither the second norm nor a gradient"""
    monkeypatch.setitem(globals(), 'EPS', 0.0)
    check_all((2, 5, C), dt, kind=kind, G=G, parts=('w', 'b', 'res', 'scale', 'w2', 'b2'), gate='sequence', alpha=0.7, seed=C + G)


@pytest.mark.parametrize('act', (ops.ACT_SIGMOID, ops.ACT_SILU))
def test_gates_far_from_zero(act):
    """y = 1 and a gate from -80 to 80, forward and backward: the exponential is within 2 ulp of its value, the sum, the quotient and the products behind
    it within half each, 1 - sigmoid by its own distance from 1: 8 2^-24 of the value, for a derivative 8 2^-24 of its terms' magnitudes."""
    gate = torch.linspace(-80, 80, 4096, device=DEV).view(4, 1024).requires_grad_()
    y = torch.ones(4, 1024, device=DEV, requires_grad=True)
    h = ops.block_tail(y, gate=gate, gate_act=act)
    dy, dg = torch.autograd.grad(h, (y, gate), torch.ones_like(h))
    x = gate.detach().double()
    s, c = torch.sigmoid(x), torch.sigmoid(-x)
    want = s if act == ops.ACT_SIGMOID else x * s
    der, mag = (s * c, s) if act == ops.ACT_SIGMOID else (s * (1 + x * c), s * (1 + x.abs()))
    u = 8 * 2.0 ** -24
    for got, w, m in ((h.detach(), want, want.abs()), (dy, want, want.abs()), (dg, der, mag)):
        assert ((got.double() - w).abs() <= u * m + 1e-37).all(), float(((got.double() - w).abs() / (u * m)).max())
    gate = torch.tensor([float('inf'), float('-inf'), float('nan'), 3e38, -3e38, 200.0, -200.0], device=DEV)
    h = ops.block_tail(torch.ones_like(gate), gate=gate, gate_act=act).cpu()
    want = [1.0, 0.0, None, 1.0, 0.0, 1.0, 0.0] if act == ops.ACT_SIGMOID else [float('inf'), None, None, 3e38, 0.0, 200.0, 0.0]
    for x, w in zip(h.tolist(), want):
        assert x != x if w is None else abs(x - w) <= 1e-37 or x == torch.tensor(w).item(), (x, w)
