"""optim.adamw_step / FusedAdamW against the formula in 64 bits.

Tolerance (fp32 elements, u = 2^-24): m and v are three roundings of sums of two terms: 4 u (|b1 m| + |(1 - b1) g|).  The parameter: 2 u of itself, and
of the update's size 8 u of its own chain plus the errors of m (4 u) and of the root of v (2 u + its rounding): 16 u; where m's terms cancel the
update is measured by their absolute values.  8-bit states: the value to be held is known to `err` (4 u of m's terms, which may cancel; the root of v to 4 u of itself) and its place between two
codes is formed to 2^-19 of a step more (a sum below 17 in fp32), so a code is checked bit for bit wherever the dithered place is further than
err / step + 2^-15 from a border, and to a neighbour elsewhere."""
import pytest
import torch

from ha2g_amd import optim

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
U = 2.0 ** -24
HP = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
SIZES = (1, 3, 4, 127, 128, 129, 300, 1000, 2047, 2048, 2049, 4095, 4096, 4097, 10000, 70001)


def formula(p, g, m, v, t, hp=HP):
    (b1, b2), lr = hp['betas'], hp['lr']
    p, g, m, v = (x.double().cpu() for x in (p, g, m, v))
    am = b1 * m.abs() + (1 - b1) * g.abs()
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    den = (v / (1 - b2 ** t)).sqrt() + hp['eps']
    q = p * (1 - lr * hp['weight_decay']) - lr / (1 - b1 ** t) * m / den
    return q, m, v, 2 * U * p.abs() + 16 * U * lr / (1 - b1 ** t) * am / den + U * q.abs(), 4 * U * am, 4 * U * v


def tensors(sizes, dt, seed, scale=1.0, odd=False):
    gen = torch.Generator().manual_seed(seed)
    out = []
    for n in sizes:
        x = (torch.randn(n + odd, generator=gen) * scale).to(dt).to(DEV)
        out.append(x[1:] if odd else x)
    return out


@pytest.mark.parametrize('odd', (False, True), ids=('aligned', 'odd'))
@pytest.mark.parametrize('gt', (torch.float32, torch.bfloat16), ids=('g32', 'g16'))
@pytest.mark.parametrize('pt', (torch.float32, torch.bfloat16), ids=('p32', 'p16'))
def test_fp32_states(pt, gt, odd):
    sizes = SIZES + (0,) + SIZES * 4                 # more than one launch's table
    p, g = tensors(sizes, pt, 1, odd=odd), tensors(sizes, gt, 2, 1e-2, odd)
    m, v = tensors(sizes, torch.float32, 3, 1e-2, odd), [x.square() for x in tensors(sizes, torch.float32, 4, 1e-2, odd)]
    step = torch.full((1,), 6, dtype=torch.int32, device=DEV)
    before = [[x.clone() for x in ts] for ts in (p, g, m, v)]
    optim.adamw_step(p, g, m, v, step, **HP)
    assert int(step) == 7
    for i in range(len(sizes)):
        wp, wm, wv, tp, tm, tv = formula(*(b[i] for b in before), 7)
        if pt == torch.bfloat16:
            tp = tp + 2.0 ** -8 * (wp.abs() + tp)
        for x, w, tol in ((p[i], wp, tp), (m[i], wm, tm), (v[i], wv, tv)):
            assert ((x.double().cpu() - w).abs() <= tol + 1e-37).all(), (i, sizes[i])
        assert torch.equal(g[i], before[1][i])


def hash32(x):
    x = ((x ^ (x >> 16)) * 0x9e3779b9) & 0xffffffff
    x = ((x ^ (x >> 15)) * 0xc13fa9a9) & 0xffffffff
    return x ^ (x >> 16)


def dither(seed, t, tensor, n):
    h = lambda a, b: hash32(torch.tensor(a ^ b))      # noqa: E731
    key = int(h(int(h(int(hash32(torch.tensor(seed))), t)), tensor))
    d = hash32(torch.arange(n) ^ key)
    return d >> 16, d & 0xffff


VALUES = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()


def check_codes(x, err, codes, scales, d):
    """codes and scales hold x (64 bits, known to err), rounded with dither d"""
    n = x.numel()
    blocks = torch.nn.functional.pad(x, (0, -n % 128)).view(-1, 128)
    top = blocks.abs().amax(1)
    s = torch.where(top > 0, torch.exp2(torch.ceil(torch.log2(top / 448))), 0.0).clamp_min(2.0 ** -126)
    got = scales.double().cpu()
    edge = ((top / 448).log2() - (top / 448).log2().round()).abs() < 1e-5         # within rounding of the next power of two
    assert (torch.isclose(got, s, rtol=0) | (edge & ((got == 2 * s) | (got == s / 2)))).all()
    a = (blocks.abs() / got[:, None]).flatten()[:n]
    low = (torch.searchsorted(VALUES, a.clamp(max=447.999), right=True) - 1).clamp(0, 125)
    w = (a - VALUES[low]) / (VALUES[low + 1] - VALUES[low]) + d / 65536.0
    c = codes.cpu().view(torch.uint8).long()
    assert ((c >= 128) == (x < 0))[(c & 127) > 0].all()
    c = c & 127
    want = (low + w.floor().long()).clamp(max=126)
    per = got.repeat_interleave(128)[:n] * (VALUES[low + 1] - VALUES[low])
    border = (w - w.round()).abs() < 2.0 ** -15 + err / per
    assert ((c == want) | (border & ((c - want).abs() <= 1))).all(), int(((c != want) & ~border).sum())


def states8(sizes, seed):
    out = []
    gen = torch.Generator().manual_seed(seed)
    for n in sizes:
        c = torch.randint(0, 127, (n,), generator=gen, dtype=torch.uint8)
        s = torch.exp2(torch.randint(-24, -14, (-(-n // 128),), generator=gen).float())
        out.append((c, s))
    return out


def value(st):
    c, s = st
    return c.view(torch.float8_e4m3fn).double().cpu() * s.double().cpu().repeat_interleave(128)[:c.numel()]


@pytest.mark.parametrize('odd', (False, True), ids=('aligned', 'odd'))
@pytest.mark.parametrize('pt,gt', ((torch.float32, torch.float32), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32)))
def test_8_bit_states(pt, gt, odd):
    sizes = SIZES + (0, 200000) + (260,) * 50
    p, g = tensors(sizes, pt, 1, odd=odd), tensors(sizes, gt, 2, 1e-3, odd)
    m, v = states8(sizes, 3), states8(sizes, 4)
    place = lambda c: torch.cat([c.new_zeros(1), c]).to(DEV)[1:] if odd else c.to(DEV)      # noqa: E731
    m = [(place(torch.where(torch.arange(c.numel()) % 3 == 0, c | 128, c)).view(torch.float8_e4m3fn), s.to(DEV)) for c, s in m]
    v = [(place(c).view(torch.float8_e4m3fn), s.to(DEV)) for c, s in v]
    step = torch.full((1,), 41, dtype=torch.int32, device=DEV)
    before = [x.clone() for x in p], [value(x) for x in m], [value(x) for x in v]
    seed = 0xfedcba98
    optim.adamw_step(p, g, m, v, step, seed=seed, **HP)
    for i, n in enumerate(sizes):
        wp, wm, wv, tp, tm, _ = formula(before[0][i], g[i], before[1][i], before[2][i] ** 2, 42)
        if pt == torch.bfloat16:
            tp = tp + 2.0 ** -8 * (wp.abs() + tp)
        assert ((p[i].double().cpu() - wp).abs() <= tp).all(), i
        dm, dr = dither(seed, 42, i, n)
        check_codes(wm, tm, *m[i], dm)
        check_codes(wv.sqrt(), 4 * U * wv.sqrt(), *v[i], dr)


def test_the_dither_is_fair_and_slow_decay_is_not_lost():
    """200 steps of g = 0 with beta2 = 0.99: round to nearest would leave every code of r where it is; dithered, the mean of r decays by 0.99^(1/2) a step.
    A step's rounding moves an element by at most one of its codes (1/8 of its value); over 16384 independent elements and 200 steps the mean is
    off by less than 5 sigma = 5 sqrt(200) / 8 / 128 = 7 %; the mean measured against the exact decay has to be inside that."""
    n = 16384
    p = [torch.zeros(n, device=DEV)]
    g = [torch.zeros(n, device=DEV)]
    m, v = [optim.adamw_state8(p[0])], [optim.adamw_state8(p[0])]
    gen = torch.Generator().manual_seed(5)
    v[0][0].view(torch.uint8).copy_(torch.randint(60, 126, (n,), generator=gen, dtype=torch.uint8))
    v[0][1].fill_(2.0 ** -10)
    r0 = value(v[0])
    step = torch.zeros(1, dtype=torch.int32, device=DEV)
    for _ in range(200):
        optim.adamw_step(p, g, m, v, step, lr=1e-3, betas=(0.9, 0.99), weight_decay=0.0, seed=9)
    ratio = float((value(v[0]) / r0).mean()) / 0.99 ** 100
    assert abs(ratio - 1) < 0.07, ratio
    assert torch.equal(value(m[0]), torch.zeros(n, dtype=torch.float64))


def test_values_that_are_not_finite_keep_to_their_elements():
    n = 1000
    bad = {5: float('nan'), 200: float('inf'), 999: float('-inf')}
    for bits in (32, 8):
        p, g = tensors((n,), torch.float32, 1), tensors((n,), torch.float32, 2, 1e-3)
        mk = (lambda: [torch.zeros(n, device=DEV)]) if bits == 32 else (lambda: [optim.adamw_state8(p[0])])      # noqa: E731
        q = [p[0].clone()]
        (m, v), (m2, v2) = (mk(), mk()), (mk(), mk())
        steps = [torch.zeros(1, dtype=torch.int32, device=DEV) for _ in range(2)]
        g2 = [g[0].clone()]
        for i, x in bad.items():
            g2[0][i] = x
            g[0][i] = 0.0
        for _ in range(3):
            optim.adamw_step(p, g, m, v, steps[0], **HP)
            optim.adamw_step(q, g2, m2, v2, steps[1], **HP)
        ok = torch.ones(n, dtype=torch.bool)
        ok[list(bad)] = False
        assert torch.equal(p[0].cpu()[ok], q[0].cpu()[ok]) and not torch.isfinite(q[0].cpu()[~ok]).any()
        if bits == 8:
            assert torch.equal(value(m[0])[ok], value(m2[0])[ok]) and torch.isnan(value(m2[0])[~ok]).all()


def test_guard_and_channels_last_and_zero_step():
    p = [torch.randn(8, 4, 3, 3, device=DEV).contiguous(memory_format=torch.channels_last)]
    g = [torch.randn_like(p[0])]
    m, v = [torch.zeros_like(p[0])], [torch.zeros_like(p[0])]
    step, guard = torch.zeros(1, dtype=torch.int32, device=DEV), torch.ones(1, dtype=torch.int32, device=DEV)
    held = p[0].clone()
    optim.adamw_step(p, g, m, v, step, guard=guard, **HP)
    assert torch.equal(p[0], held) and int(step) == 0 and not m[0].any()
    guard.zero_()
    optim.adamw_step(p, g, m, v, step, guard=guard, **HP)
    wp, _, _, tp, _, _ = formula(held, g[0], torch.zeros_like(held), torch.zeros_like(held), 1)
    assert int(step) == 1 and ((p[0].double().cpu() - wp).abs() <= tp).all()
    optim.adamw_step([], [], [], [], step)
    with pytest.raises(ValueError):
        optim.adamw_step([p[0], p[0]], [g[0], g[0]], [m[0], m[0]], [v[0], v[0]], step)
    with pytest.raises(ValueError):
        optim.adamw_step(p, [g[0].contiguous()], m, v, step)


@pytest.mark.parametrize('bits', (32, 8))
def test_captured_steps_advance(bits):
    sizes = (300, 5000, 64)
    make = lambda: (tensors(sizes, torch.float32, 1), tensors(sizes, torch.float32, 2, 1e-2))      # noqa: E731

    def states(p):
        return ([torch.zeros_like(x) for x in p] if bits == 32 else [optim.adamw_state8(x) for x in p] for _ in range(2))
    (p, g), (q, h) = make(), make()
    (m, v), (m2, v2) = states(p), states(q)
    steps = [torch.zeros(1, dtype=torch.int32, device=DEV) for _ in range(2)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        optim.adamw_step(q, h, m2, v2, steps[1], **HP)
    for i in range(4):
        for x, y in zip(g, h):
            y.copy_(x.mul_(0.9 + 0.05 * i))
        graph.replay()
        optim.adamw_step(p, g, m, v, steps[0], **HP)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(p, q)) and int(steps[1]) == i + 1
    if bits == 8:
        assert all(torch.equal(value(a), value(b)) for a, b in zip(m + v, m2 + v2))


@pytest.mark.parametrize('bits', (32, 8))
def test_fused_adamw_on_a_module(bits):
    """FusedAdamW against torch.optim.AdamW (biases not decayed): fp32 states track it to rounding; 8-bit ones exactly on the first step (states are
    rounded only behind it), and stay close in direction afterwards"""
    torch.manual_seed(0)
    from ha2g_amd import hierarchy_net as hn
    net = [hn.Linear(300, 70).to(DEV), hn.Linear(70, 9).to(DEV)]
    ps = [p for l in net for p in l.parameters()]
    twin = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    opt = optim.FusedAdamW(ps, lr=1e-3, weight_decay=0.1, no_decay=[p for p in ps if p.dim() < 2], state_bits=bits, seed=4)
    ref = torch.optim.AdamW([dict(params=[p for p in twin if p.dim() > 1], weight_decay=0.1), dict(params=[p for p in twin if p.dim() < 2], weight_decay=0.0)], lr=1e-3)
    gen = torch.Generator().manual_seed(1)
    for i in range(5):
        opt.zero_grad()
        for p, q in zip(ps, twin):
            gr = torch.randn(p.shape, generator=gen).to(DEV) * 1e-2
            if i == 3:
                p.grad = gr.clone()                     # a foreign tensor: folded back
            else:
                p.grad.add_(gr)
            q.grad = gr
        opt.step()
        ref.step()
        if bits == 32 or i == 0:
            for p, q in zip(ps, twin):
                assert ((p - q).abs() <= 32 * U * (q.abs() + (i + 1) * 1e-3)).all()
    for p, q in zip(ps, twin):
        assert float((p - q).norm()) <= 0.2 * 5e-3 * p.numel() ** 0.5
    assert opt.param_groups[0]['weight_decay'] == 0.1


@pytest.mark.parametrize('kind', ('adamw', 'adamw8'))
def test_the_trainer_steps_with_it(kind):
    from bench import Vocab
    from ha2g_amd import procedural as proc
    from ha2g_amd.config import hierarchy_args
    from ha2g_amd.train import HierarchyTrainer
    torch.manual_seed(0)
    tr = HierarchyTrainer(hierarchy_args(hidden_size=32, n_layers=2, optimizer=kind, weight_decay=0.05), Vocab(50), Vocab(7), 27, torch.device(DEV))
    assert all(type(o) is optim.FusedAdamW for o in tr.gen_opts + [tr.audio_opt, tr.text_opt, tr.dis_opt])
    batch = [torch.from_numpy(x).to(DEV) for x in proc.make_batch(3, 27, 50, 7, 5)]
    before = [o.flat_p.clone() for o in tr.gen_opts]
    for _ in range(2):
        ret = tr.train_iter(11, *batch)
        assert all(x == x for x in ret.values())
    tr.sync()
    assert int(tr.gen_opts[0].step_t) == 2
    for o, b in zip(tr.gen_opts, before):
        d = (o.flat_p - b).abs()
        assert torch.isfinite(o.flat_p).all() and 0 < float(d.max()) <= 2 * float(tr.args.learning_rate) * 2.0 ** 0.5 * (1 + 0.05) * 4


def test_a_tensor_of_more_than_two_to_the_31_elements():
    n, m0 = 2 ** 31 + 300, 2 ** 31 - 128
    p, g = torch.zeros(n, dtype=torch.bfloat16, device=DEV), torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    m, v = optim.adamw_state8(p), optim.adamw_state8(p)
    (pt,), (gt,) = tensors((n - m0,), torch.bfloat16, 1), tensors((n - m0,), torch.bfloat16, 2, 1e-3)
    p[m0:], g[m0:] = pt, gt
    step = torch.full((1,), 9, dtype=torch.int32, device=DEV)
    optim.adamw_step([p], [g], [m], [v], step, seed=3, **HP)
    wp, wm, wv, tp, tm, _ = formula(pt, gt, torch.zeros(n - m0), torch.zeros(n - m0), 10)
    tp = tp + 2.0 ** -8 * (wp.abs() + tp)
    assert ((p[m0:].double().cpu() - wp).abs() <= tp).all() and not p[:m0:65537].any()
    key = hash32(torch.tensor(int(hash32(torch.tensor(int(hash32(torch.tensor(3))) ^ 10)))))
    d = hash32(torch.arange(m0, n) ^ int(key))
    check_codes(wm, tm, m[0][m0:], m[1][m0 // 128:], d >> 16)
    check_codes(wv.sqrt(), 4 * U * wv.sqrt(), v[0][m0:], v[1][m0 // 128:], d & 0xffff)


def test_lists_without_elements_and_tensors_listed_twice():
    none = lambda k: [torch.empty(0, device=DEV) for _ in range(k)]      # noqa: E731
    step = torch.zeros(1, dtype=torch.int32, device=DEV)
    optim.adamw_step(none(70), none(70), none(70), none(70), step)
    assert int(step) == 1
    # a whole launch's table of them in front of one that has elements
    p, g, m, v = ([*none(64), x] for x in (torch.ones(5, device=DEV), torch.ones(5, device=DEV), torch.zeros(5, device=DEV), torch.zeros(5, device=DEV)))
    optim.adamw_step(p, g, m, v, step, **HP)
    want, _, _, tol, _, _ = formula(torch.ones(5), torch.ones(5), torch.zeros(5), torch.zeros(5), 2)
    assert ((p[-1].double().cpu() - want).abs() <= tol).all()
    a, b, c, d = (torch.ones(8, device=DEV) for _ in range(4))
    e = torch.empty(0, device=DEV)
    for ps, gs, ms, vs in (([a], [b], [c], [c]), ([a], [b], [a], [c]), ([a, a, e], [b, b, e], [c, d, e], [b.clone(), b.clone(), e])):
        with pytest.raises(ValueError, match='twice'):
            optim.adamw_step(ps, gs, ms, vs, step)
    s8 = [optim.adamw_state8(a)]
    with pytest.raises(ValueError, match='twice'):
        optim.adamw_step([a], [b], s8, s8, step)
    assert int(step) == 2 and (a == 1).all()


def test_a_graph_that_saved_the_old_parameter_refuses_its_backward_pass():
    p = torch.ones(8, device=DEV).requires_grad_()
    y = (p * p).sum()
    step, z = torch.zeros(1, dtype=torch.int32, device=DEV), [torch.zeros(8, device=DEV) for _ in range(2)]
    optim.adamw_step([p], [torch.ones(8, device=DEV)], z[:1], z[1:], step)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.backward()
    with torch.inference_mode():
        q, z = torch.ones(8, device=DEV), [torch.zeros(8, device=DEV) for _ in range(2)]
        optim.adamw_step([q], [torch.ones(8, device=DEV)], z[:1], z[1:], step)
    assert (q < 1).all()


@pytest.mark.parametrize('bits', (32, 8))
def test_a_captured_optimizer_advances_on_each_replay(bits):
    """FusedAdamW.step in a graph, with eager steps of a twin in between: the same bits after every replay, two groups of decay included"""
    def make():
        torch.manual_seed(3)
        ps = [torch.nn.Parameter(torch.randn(*s, device=DEV)) for s in ((40, 30), (30,), (129, 7))]
        return ps, optim.FusedAdamW(ps, lr=3e-3, weight_decay=0.1, no_decay=ps[1:2], state_bits=bits, seed=5)
    (p, a), (q, b) = make(), make()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        b.step()
    for i in range(4):
        g = torch.randn_like(a.flat_g) * (0.5 + i)
        a.flat_g.copy_(g)
        b.flat_g.copy_(g)
        graph.replay()
        a.step()
        torch.cuda.synchronize()
        assert int(a.step_t) == int(b.step_t) == i + 1 and torch.equal(a.flat_p, b.flat_p)
    assert all(torch.equal(x, y) for x, y in zip(p, q))


def test_a_root_that_is_not_zero_is_not_stored_as_zero():
    """A root far below its block's largest is held as the smallest code: it divides the next update.  A root of zero stays zero."""
    n = 640
    p, g = [torch.zeros(n, device=DEV)], [torch.full((n,), 1e-9, device=DEV)]
    g[0][::128] = 1.0
    g[0][1::128] = 0.0
    m, v = [optim.adamw_state8(p[0])], [optim.adamw_state8(p[0])]
    step = torch.zeros(1, dtype=torch.int32, device=DEV)
    for _ in range(3):
        optim.adamw_step(p, g, m, v, step, seed=11, **HP)
        codes = v[0][0].view(torch.uint8).cpu().view(5, 128)
        assert (codes[:, 1] == 0).all() and (codes[:, 0] > 100).all() and (codes[:, 2:] == 1).all()


def test_small_gradients_beside_a_large_one_move_a_parameter_by_no_more_than_a_few_steps():
    """One gradient of 1 and 127 of 1e-8 in each block, which vanish after 20 of 40 steps.  With b1 = 1/2: a code of m is off by at most an eighth of
    its value and the smallest code step s, so a small m is held as at most (9/16 g + s) / (1 - 9/16) = 9/7 g + 16/7 s, s <= 2^-9 (2 / 448) (1 - b1^t)
    (the scale is within a factor of 2 of the largest m / 448).  A root is at least sqrt(b2) times the smallest code, 2^-9 / 448 sqrt(1 - b2^t).  So
    an update is at most lr (16/7 + 1.15 g / (1 - b1) / (2^-9 / 448)) / sqrt(b2) = 2.30 lr where the large element's m and root are exact; they are off
    by their own codes, an eighth a step at most and without bias: 8 lr leaves a factor of three for them.  After the gradients have vanished m
    falls faster than its root, and the bound stays."""
    n, lr = 128 * 40, 1e-3
    p = [torch.zeros(n, device=DEV)]
    g = [torch.full((n,), 1e-8, device=DEV)]
    g[0][::128] = 1.0
    m, v = [optim.adamw_state8(p[0])], [optim.adamw_state8(p[0])]
    step = torch.zeros(1, dtype=torch.int32, device=DEV)
    small = torch.arange(n, device=DEV) % 128 != 0
    for t in range(40):
        if t == 20:
            g[0].zero_()
        old = p[0].clone()
        optim.adamw_step(p, g, m, v, step, lr=lr, betas=(0.5, 0.999), weight_decay=0.0, seed=2)
        assert float((p[0] - old)[small].abs().max()) <= 8 * lr, t


def test_scales_listed_twice_are_refused():
    p, g = [torch.zeros(200, device=DEV)], [torch.zeros(200, device=DEV)]
    (mc, s), (vc, r) = optim.adamw_state8(p[0]), optim.adamw_state8(p[0])
    step = torch.zeros(1, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match='twice'):
        optim.adamw_step(p, g, [(mc, s)], [(vc, s)], step)
    assert int(step) == 0
    optim.adamw_step(p, g, [(mc, s)], [(vc, r)], step)


@pytest.mark.parametrize('kind', ('adamw', 'adamw8'))
def test_what_the_trainer_decays(kind):
    """a step with gradients of zero multiplies what is decayed by fp32(1 - lr wd) and leaves the rest: biases, norm weights, the gains of weight norms"""
    from bench import Vocab
    from ha2g_amd.config import hierarchy_args
    from ha2g_amd.train import HierarchyTrainer
    torch.manual_seed(0)
    tr = HierarchyTrainer(hierarchy_args(hidden_size=32, n_layers=2, optimizer=kind, weight_decay=0.05), Vocab(50), Vocab(7), 27, torch.device(DEV))
    gains = 0
    for m, o in zip([*tr.gens, tr.audio_encoder, tr.text_encoder, tr.discriminator], [*tr.gen_opts, tr.audio_opt, tr.text_opt, tr.dis_opt]):
        before = {n: p.detach().clone() for n, p in m.named_parameters() if p.requires_grad}
        o.zero_grad()
        o.step()
        keep = torch.tensor(1.0 - o.param_groups[0]['lr'] * 0.05, dtype=torch.float32, device=DEV)
        for n, p in m.named_parameters():
            if p.requires_grad:
                still = p.dim() < 2 or n.split('.')[-1] == 'weight_g'
                gains += p.dim() > 1 and still
                assert torch.equal(p.detach(), before[n] if still else before[n] * keep), n
    assert gains > 0
