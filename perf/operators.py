"""The cases on which the sequence-block operators are measured: linear attention with a decay per head (chunked, backward, single token), the
per-row norms and the fused block tail, and the AdamW step over many tensors.  `run` computes them in elementary torch operations, or -- with
`own` -- through ha2g_amd; `exact` computes them in 64 bits from their definitions."""
import math

import torch

own = False
DEV = 'cuda'
DT = {'fp32': torch.float32, 'bf16': torch.bfloat16}
Q8_BLOCK = 128            # elements of a tensor that share one scale of an 8-bit AdamW state


def listed():
    return [
        # streaming one clip: the next pose frame of a batch of one (300 channels as 5 heads of 60); a launch's latency is all there is
        dict(name='la_step_stream', op='la_step', dtype='fp32', B=1, H=5, Hqk=5, Dk=60, Dv=60),
        # serving many streams at once: the states are most of what moves
        dict(name='la_step_serving', op='la_step', dtype='bf16', B=256, H=16, Hqk=4, Dk=128, Dv=128),
        # prompts of ragged length in one padded batch, no gradient, states kept for the tokens that follow
        dict(name='la_prompt_ragged', op='la', dtype='bf16', B=3, T=5003, H=12, Hqk=12, Dk=64, Dv=128, ragged=True, train=False),
        # one long prompt: few heads, so the time axis has to be split
        dict(name='la_prompt_long', op='la', dtype='fp32', B=1, T=32768, H=8, Hqk=8, Dk=64, Dv=64, ragged=False, train=False),
        # a train step at the pose decoder's own sizes: 128 windows of 34 frames
        dict(name='la_train_window', op='la', dtype='fp32', B=128, T=34, H=5, Hqk=5, Dk=60, Dv=60, ragged=False, train=True),
        # a train step on long sequences, queries and keys shared by four heads each
        dict(name='la_train_long', op='la', dtype='bf16', B=2, T=8192, H=16, Hqk=4, Dk=128, Dv=128, ragged=False, train=True),
        # the norm in front of a block: one streamed window
        dict(name='norm_window', op='row_norm', dtype='fp32', B=1, T=34, C=300, G=1, kind='layer', train=False),
        # the same in training, normalised per head
        dict(name='norm_train', op='row_norm', dtype='bf16', B=4, T=2048, C=4096, G=32, kind='rms', train=True),
        # the tail of a block at the pose decoder's sizes: per-head norm, one gate per window and channel (as squeeze-and-excitation gates)
        dict(name='tail_window', op='block_tail', dtype='fp32', B=128, T=34, C=300, G=5, kind='layer', gate='sequence', next=False, train=True),
        # the tail of a wide block and the norm before the next one, gated per token
        dict(name='tail_train', op='block_tail', dtype='bf16', B=8, T=2048, C=2048, G=16, kind='rms', gate='token', next=True, train=True),
        # the optimizer step of one pose generator (hidden size 300, 4 layers, 20 000 words), everything in 32 bits
        dict(name='adamw_generator', op='adamw', bits=32, hidden=300, layers=4, words=20000, pdtype='fp32', gdtype='fp32'),
        # a wide one whose states are held in 8 bits and whose gradients arrive in bf16
        dict(name='adamw8_wide', op='adamw', bits=8, hidden=1200, layers=4, words=20000, pdtype='fp32', gdtype='bf16'),
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    op = rng.choice(['la_step', 'la', 'la', 'row_norm', 'block_tail', 'adamw'])
    dtype = rng.choice(['fp32', 'bf16'])
    if op in ('la_step', 'la'):
        H = rng.choice([1, 2, 4, 5, 6, 8, 12, 16])
        Hqk = rng.choice([h for h in (1, 2, 4, H) if H % h == 0])
        Dk, Dv = (rng.choice([8, 16, 25, 32, 50, 60, 64, 75, 96, 100, 128]) for _ in range(2))
        if op == 'la_step':
            return dict(op=op, dtype=dtype, B=log_int(1, max(1, min(512, (1 << 26) // (H * Dk * Dv)))), H=H, Hqk=Hqk, Dk=Dk, Dv=Dv)
        T = log_int(1, 20000)
        B = log_int(1, max(1, min(256, (1 << 24) // (T * H * max(Dk, Dv)))))
        return dict(op=op, dtype=dtype, B=B, T=T, H=H, Hqk=Hqk, Dk=Dk, Dv=Dv, ragged=rng.random() < 0.5, train=rng.random() < 0.5)
    if op in ('row_norm', 'block_tail'):
        G = rng.choice([1, 1, 2, 4, 5, 8, 16])
        C = G * log_int(8, 6000 // G)
        T = log_int(1, 4096)
        c = dict(op=op, dtype=dtype, B=log_int(1, max(1, min(128, (1 << 24) // (T * C)))), T=T, C=C, G=G, kind=rng.choice(['rms', 'layer']),
                 train=rng.random() < 0.6)
        if op == 'block_tail':
            c.update(gate=rng.choice(['none', 'sequence', 'token']), next=rng.random() < 0.5)
        return c
    return dict(op='adamw', bits=rng.choice([8, 32]), hidden=log_int(32, 1000), layers=rng.randint(1, 4), words=log_int(50, 20000),
                pdtype=rng.choice(['fp32', 'fp32', 'bf16']), gdtype=rng.choice(['fp32', 'bf16']))


# ---- inputs ----------------------------------------------------------------------------------------------------------------------------------

def _shapes(case):
    """parameter shapes of a pose generator: word table, temporal convolutions, bidirectional recurrent layers, head"""
    h, out = case['hidden'], [(case['words'], 300)]
    for l in range(case['layers']):
        out += [(h, 300 if l == 0 else h, 2), (h, h, 2), (h,), (h,)]
        out += [s for _ in range(2) for s in ((3 * h, 108 if l == 0 else 2 * h), (3 * h, h), (3 * h,), (3 * h,))]
    return out + [(max(1, h // 2), h), (max(1, h // 2),), (27, max(1, h // 2)), (27,)]


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)

    def randn(*s, dt=torch.float32, scale=1.0, grad=False):
        return (torch.randn(*s, device=DEV, generator=gen) * scale).to(dt).requires_grad_(grad)
    st = dict(case=case)
    if case['op'] in ('la', 'la_step'):
        B, H, Hqk, Dk, Dv, dt = (case[k] for k in ('B', 'H', 'Hqk', 'Dk', 'Dv', 'dtype'))
        dt = DT[dt]
        lead, train = ((B,) if case['op'] == 'la_step' else (B, case['T'])), bool(case.get('train'))
        st.update(q=randn(*lead, Hqk, Dk, dt=dt, grad=train), k=randn(*lead, Hqk, Dk, dt=dt, grad=train), v=randn(*lead, H, Dv, dt=dt, grad=train),
                  # decays as multi-scale retention sets them: 1 - 2^-5 for the first head, towards 1 - 2^-12 for the last
                  g=torch.log1p(-torch.exp2(-torch.linspace(5, 12, H, dtype=torch.float64))).float().to(DEV),
                  state=randn(B, H, Dk, Dv, scale=2.0, grad=train))
        if case['op'] == 'la':
            st['lengths'] = None
            if case['ragged']:
                n = case['T'] - (torch.rand(B, device=DEV, generator=gen) * 0.5 * case['T']).int()
                st['lengths'] = n.int()
            if train:
                st.update(do=randn(B, case['T'], H, Dv, dt=dt), ds=randn(B, H, Dk, Dv))
    elif case['op'] in ('row_norm', 'block_tail'):
        B, T, C, dt = case['B'], case['T'], case['C'], DT[case['dtype']]
        train = case['train']
        vec = lambda at: (randn(C, scale=0.2) + at).requires_grad_(train)      # noqa: E731
        st.update(y=(randn(B, T, C) + 0.3).to(dt).requires_grad_(train), w=vec(1.0), b=vec(0.0))
        if train:
            st['dh'] = randn(B, T, C, dt=dt)
        if case['op'] == 'block_tail':
            st.update(res=randn(B, T, C, dt=dt, grad=train), scale=vec(0.5), gate=None)
            if case['gate'] != 'none':
                st['gate'] = randn(B, 1 if case['gate'] == 'sequence' else T, C, dt=dt, grad=train)
            if case['next']:
                st.update(w2=vec(1.0), b2=vec(0.0))
                if train:
                    st['dz'] = randn(B, T, C, dt=dt)
    else:
        shapes = _shapes(case)
        n = [math.prod(s) for s in shapes]
        nb = [-(-x // Q8_BLOCK) for x in n]
        at = [0]
        for x in nb:
            at.append(at[-1] + x)
        total = at[-1] * Q8_BLOCK
        # one arena per role; every tensor starts on a block of its own, the elements behind its end are no tensor's
        live = torch.zeros(total, dtype=torch.bool, device=DEV)
        for a, x in zip(at, n):
            live[a * Q8_BLOCK:a * Q8_BLOCK + x] = True

        def arena(dt, scale):
            return randn(total, scale=scale).mul_(live).to(dt)
        p, g = arena(DT[case['pdtype']], 0.05), arena(DT[case['gdtype']], 1e-3)
        cut = lambda t: [t[a * Q8_BLOCK:a * Q8_BLOCK + x].view(s) for a, x, s in zip(at, n, shapes)]      # noqa: E731
        flat = lambda t: [t[a * Q8_BLOCK:a * Q8_BLOCK + x] for a, x in zip(at, n)]                         # noqa: E731
        st.update(p=p, g=g, params=cut(p), grads=cut(g), step=torch.full((1,), 1000, dtype=torch.int32, device=DEV), seed=seed % 65536,
                  first=torch.tensor(at[:-1], device=DEV))
        if case['bits'] == 32:
            m, v = arena(torch.float32, 3e-4), arena(torch.float32, 1e-3).square_()
            st.update(m=m, v=v, ms=cut(m), vs=cut(v))
        else:
            # states as earlier steps left them: any code, a scale for every block (m up to 1e-3, the root of v up to 4e-3)
            mc = torch.randint(0, 256, (total,), device=DEV, generator=gen, dtype=torch.uint8)
            rc = torch.randint(40, 127, (total,), device=DEV, generator=gen, dtype=torch.uint8)
            mc = torch.where((mc & 127) == 127, mc - 1, mc) * live
            rc = rc * live
            e = torch.randint(0, 3, (2, at[-1]), device=DEV, generator=gen)
            sm, sr = torch.exp2(e[0] - 21.0), torch.exp2(e[1] - 19.0)
            mc, rc = mc.view(torch.float8_e4m3fn), rc.view(torch.float8_e4m3fn)
            per = lambda t: [t[a:b] for a, b in zip(at[:-1], at[1:])]      # noqa: E731
            st.update(m=mc, v=rc, sm=sm, sr=sr, ms=list(zip(flat(mc), per(sm))), vs=list(zip(flat(rc), per(sr))))
    return st


# ---- one pass --------------------------------------------------------------------------------------------------------------------------------

LR, BETAS, EPS, WD = 5e-4, (0.5, 0.999), 1e-8, 0.01


def run(st):
    case = st['case']
    return {'la': _run_la, 'la_step': _run_la_step, 'row_norm': _run_row_norm, 'block_tail': _run_block_tail, 'adamw': _run_adamw}[case['op']](st, case)


def _run_la(st, case):
    args = st['q'], st['k'], st['v'], st['g']
    if own:
        from ha2g_amd import ops
        o, s = ops.linear_attention(*args, state=st['state'], lengths=st['lengths'], return_state=True)
    else:
        o, s = _plain_la(*args, st['state'], st['lengths'])
    if not case['train']:
        return dict(o=o, state=s)
    leaves = [st[n] for n in ('q', 'k', 'v', 'state')]
    grads = torch.autograd.grad([o, s], leaves, [st['do'], st['ds']])
    return dict(zip(('o', 'state', 'dq', 'dk', 'dv', 'dstate'), (o.detach(), s.detach(), *grads)))


def _run_la_step(st, case):
    if own:
        from ha2g_amd import ops
        return dict(o=ops.linear_attention_step(st['q'], st['k'], st['v'], st['g'], st['state']), state=st['state'])
    H = case['H']
    q, k, v = (st[n].float().repeat_interleave(H // st[n].shape[1], 1) for n in 'qkv')
    s = st['state']
    s.mul_(torch.exp(st['g'])[:, None, None]).add_(k.unsqueeze(3) * v.unsqueeze(2))
    o = (q * case['Dk'] ** -0.5).unsqueeze(2) @ s
    return dict(o=o.squeeze(2).to(st['v'].dtype), state=s)


def _run_row_norm(st, case):
    if own:
        from ha2g_amd import ops
        h = ops.row_norm(st['y'], st['w'], st['b'], kind=case['kind'], groups=case['G'])
    else:
        h = (_plain_norm(st['y'].float(), case['kind'], case['G']) * st['w'] + st['b']).to(st['y'].dtype)
    if not case['train']:
        return h
    grads = torch.autograd.grad(h, [st['y'], st['w'], st['b']], st['dh'])
    return dict(zip(('h', 'dy', 'dw', 'db'), (h.detach(), *grads)))


def _run_block_tail(st, case):
    nxt = case['next']
    if own:
        from ha2g_amd import ops
        out = ops.block_tail(st['y'], st['res'], gate=st['gate'], weight=st['w'], bias=st['b'], scale=st['scale'], kind=case['kind'],
                             groups=case['G'], gate_act=ops.ACT_SILU, next_weight=st.get('w2'), next_bias=st.get('b2'))
    else:
        u = _plain_norm(st['y'].float(), case['kind'], case['G']) * st['w'] + st['b']
        if st['gate'] is not None:
            gate = st['gate'].float()
            u = u * (gate / (1.0 + torch.exp(-gate)))
        h = st['res'].float() + st['scale'] * u
        out = h.to(st['y'].dtype)
        if nxt:
            out = out, (_plain_norm(h, case['kind'], 1) * st['w2'] + st['b2']).to(st['y'].dtype)
    out = out if nxt else (out,)
    names = [n for n in ('y', 'res', 'gate', 'w', 'b', 'scale', 'w2', 'b2') if st.get(n) is not None]
    res = dict(zip(('h', 'z'), (o.detach() for o in out)))
    if case['train']:
        grads = torch.autograd.grad(out, [st[n] for n in names], [st['dh'], st['dz']] if nxt else [st['dh']])
        res.update(zip(('d' + n for n in names), grads))
    return res


def _run_adamw(st, case):
    if own:
        from ha2g_amd import optim
        optim.adamw_step(st['params'], st['grads'], st['ms'], st['vs'], st['step'], lr=LR, betas=BETAS, eps=EPS, weight_decay=WD, seed=st['seed'])
    else:
        _plain_adamw(st, case['bits'])
    return {n: st[n] for n in ('p', 'm', 'v', 'sm', 'sr') if n in st}


# ---- plain forms -----------------------------------------------------------------------------------------------------------------------------

def _plain_la(q, k, v, g, state, lengths, C=64):
    B, T, _, Dk = q.shape
    H, Dv, dt = g.shape[0], v.shape[3], v.dtype
    q, k, v = (x.float().repeat_interleave(H // x.shape[2], 2).transpose(1, 2) for x in (q, k, v))
    t = torch.arange(T, device=q.device)
    n = torch.full((B,), T, device=q.device) if lengths is None else lengths.long()
    there = (t < n[:, None])[:, None, :, None]
    k, v = torch.where(there, k, 0.0), torch.where(there, v, 0.0)
    g = g.double()

    def power(e):                  # exp(g * e) for a table of whole exponents; those below zero count as no contribution
        return torch.where(e >= 0, torch.exp(g[:, None, None] * e.clamp_min(0)), 0.0).float()
    # the state behind the last token
    w = power((n[:, None] - 1 - t).unsqueeze(1).transpose(0, 1).reshape(1, B, T)).transpose(0, 1)                        # [B, H, T]
    last = torch.exp(g * n[:, None]).float()[:, :, None, None] * state + (k * w.unsqueeze(3)).transpose(2, 3) @ v
    # chunks of C tokens: products inside a chunk, and the state that enters it
    nc = -(-T // C)
    q, k, v = (torch.nn.functional.pad(x, (0, 0, 0, nc * C - T)).reshape(B, H, nc, C, x.shape[3]) for x in (q, k, v))
    i = torch.arange(C, device=q.device)
    c = torch.arange(nc, device=q.device)
    inside = ((q @ k.transpose(3, 4)) * power((i[:, None] - i)[None])[:, None]) @ v
    kv = (k * power((C - 1 - i)[None, None])[:, :, :, None].expand(H, 1, C, 1)).transpose(3, 4) @ v
    enter = power((C * (c[:, None] - 1 - c))[None]) @ kv.reshape(B, H, nc, Dk * Dv) + power((C * c)[None, None]).transpose(1, 2) * state.reshape(B, H, 1, Dk * Dv)
    before = (q * power((i + 1)[None, None])[:, :, :, None]) @ enter.reshape(B, H, nc, Dk, Dv)
    o = ((inside + before) * Dk ** -0.5).reshape(B, H, nc * C, Dv)[:, :, :T]
    return torch.where(there, o, 0.0).transpose(1, 2).to(dt), last


def _plain_norm(x, kind, groups, eps=1e-5):
    x = x.reshape(*x.shape[:-1], groups, -1)
    if kind == 'layer':
        x = x - x.mean(-1, keepdim=True)
    return (x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)).flatten(-2)


def _hash32(x):
    """multiply / xor-shift mixing of 32-bit words held in int64; the factors are 2^32 over the golden ratio and over the plastic number"""
    x = ((x ^ (x >> 16)) * 0x9e3779b9) & 0xffffffff
    x = ((x ^ (x >> 15)) * 0xc13fa9a9) & 0xffffffff
    return x ^ (x >> 16)


def _dither(st, t):
    """one word per element from (seed, step, tensor, place in the tensor); its halves are the two dithers in [0, 1)"""
    nblk = st['sm'].numel()
    b = torch.arange(nblk, device=DEV)
    tensor = torch.searchsorted(st['first'], b, right=True) - 1
    key = _hash32(_hash32(_hash32(torch.full_like(tensor, st['seed'])) ^ t) ^ tensor)
    local = (b - st['first'][tensor])[:, None] * Q8_BLOCK + torch.arange(Q8_BLOCK, device=DEV)
    h = _hash32(local ^ key[:, None])
    return (h >> 16), (h & 0xffff)


def _encode(x, d):
    """[blocks, Q8_BLOCK] values -> e4m3 codes and power-of-two scales: the largest of a block lands in (224, 448]; the part below a code is rounded up
    where the dither exceeds what is left to one"""
    f, e = torch.frexp(x.abs().amax(1))
    se = torch.where(f > 0, (e - 9 + (f > 0.875)).clamp_min(-126), -126)
    power = lambda n: ((n + 127) << 23).view(torch.float32)      # noqa: E731
    a = x.abs() * power(-se)[:, None]
    ue = torch.where(a > 0, torch.frexp(a)[1] - 1, -6).clamp_min(-6)
    k = torch.floor(a * power(3 - ue) + d.float() / 65536)
    code = ((ue.long() + 7) * 8 + k.long() - 8).clamp_max(126)
    return (code + 128 * (x < 0)).to(torch.uint8).view(torch.float8_e4m3fn), power(se)


def _plain_adamw(st, bits):
    """in place on the arenas; the step's scalars in 64 bits, the elements in 32"""
    b1, b2 = BETAS
    t = st['step'].add_(1).double()
    step = (LR / (1 - b1 ** t)).float()
    root = (1 / torch.sqrt(1 - b2 ** t)).float()
    g = st['g'].float()
    if bits == 32:
        m, v = st['m'], st['v']
    else:
        m = (st['m'].float().view(-1, Q8_BLOCK) * st['sm'][:, None]).view(-1)
        v = (st['v'].float().view(-1, Q8_BLOCK) * st['sr'][:, None]).view(-1).square()
    m = b1 * m + (1 - b1) * g
    v = b2 * v + ((1 - b2) * g) * g
    p = st['p'].float() * (1 - LR * WD)
    st['p'].copy_(p - step * m / (torch.sqrt(v) * root + EPS))
    if bits == 32:
        st['m'].copy_(m)
        st['v'].copy_(v)
    else:
        dm, dr = _dither(st, st['step'].long())
        for x, d, codes, scales in ((m, dm, st['m'], st['sm']), (v.sqrt(), dr, st['v'], st['sr'])):
            c, s = _encode(x.view(-1, Q8_BLOCK), d)
            codes.copy_(c.view(-1))
            scales.copy_(s)


# ---- 64 bits ---------------------------------------------------------------------------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        return {'la': _exact_la, 'la_step': _exact_la_step, 'row_norm': _exact_norms, 'block_tail': _exact_norms, 'adamw': _exact_adamw}[case['op']](st, case)


def _heads(x, H, dim):
    return x.double().repeat_interleave(H // x.shape[dim], dim)


def _exact_la_step(st, case):
    q, k, v = (_heads(st[n], case['H'], 1) for n in 'qkv')
    s = torch.exp(st['g'].double())[:, None, None] * st['state'].double() + torch.einsum('bhd,bhe->bhde', k, v)
    return dict(o=torch.einsum('bhd,bhde->bhe', q, s) / math.sqrt(case['Dk']), state=s)


def _exact_la(st, case):
    """the recurrence, a token at a time, and its transpose from the end"""
    B, T, H = case['B'], case['T'], case['H']
    q, k, v = (_heads(st[n], H, 2) for n in 'qkv')
    lam, scale = torch.exp(st['g'].double())[:, None, None], case['Dk'] ** -0.5
    n = st['lengths'] if st['lengths'] is not None else torch.full((B,), T, device=DEV)
    S = st['state'].double()
    o = torch.zeros_like(v)
    do = st['do'].double() if case['train'] else None
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    full = st['lengths'] is None
    for t in range(T):
        N = lam * S + k[:, t].unsqueeze(3) * v[:, t].unsqueeze(2)
        S = N if full else torch.where((t < n)[:, None, None, None], N, S)
        o[:, t] = (q[:, t].unsqueeze(2) @ S).squeeze(2)
        if case['train']:
            dq[:, t] = (S @ do[:, t].unsqueeze(3)).squeeze(3)
    there = (torch.arange(T, device=DEV) < n[:, None])[:, :, None, None]
    out = dict(o=torch.where(there, o * scale, 0.0), state=S)
    if not case['train']:
        return out
    R = st['ds'].double() / scale
    for t in reversed(range(T)):
        here = (t < n)[:, None, None, None]
        R2 = R + q[:, t].unsqueeze(3) * do[:, t].unsqueeze(2)
        dk[:, t] = (R2 @ v[:, t].unsqueeze(3)).squeeze(3)
        dv[:, t] = (k[:, t].unsqueeze(2) @ R2).squeeze(2)
        R = lam * R2 if full else torch.where(here, lam * R2, R)
    share = lambda d, x: (torch.where(there, d * scale, 0.0)).unflatten(2, (x.shape[2], -1)).sum(3)      # noqa: E731
    out.update(dq=share(dq, st['q']), dk=share(dk, st['k']), dv=share(dv, st['v']), dstate=R * scale)
    return out


def _exact_norms(st, case):
    G, kind, eps = case['G'], case['kind'], 1e-5
    d = {n: (x.double() if torch.is_tensor(x) else x) for n, x in st.items()}

    def stats(x, g):
        x = x.unflatten(-1, (g, -1))
        mu = x.mean(-1, keepdim=True) if kind == 'layer' else torch.zeros_like(x[..., :1])
        r = ((x - mu).pow(2).mean(-1, keepdim=True) + eps).rsqrt()
        return ((x - mu) * r).flatten(-2), r

    def back(dxhat, xhat, r, g):
        a, x = dxhat.unflatten(-1, (g, -1)), xhat.unflatten(-1, (g, -1))
        a = a - x * (a * x).mean(-1, keepdim=True) - (a.mean(-1, keepdim=True) if kind == 'layer' else 0.0)
        return (a * r).flatten(-2)
    rows = (0, 1)
    yh, r1 = stats(d['y'], G)
    nrm = yh * d['w'] + d['b']
    if case['op'] == 'row_norm':
        if not case['train']:
            return nrm
        dh = d['dh']
        return dict(h=nrm, dy=back(dh * d['w'], yh, r1, G), dw=(dh * yh).sum(rows), db=dh.sum(rows))
    sig = torch.sigmoid(d['gate']) if d['gate'] is not None else None
    act = d['gate'] * sig if sig is not None else 1.0
    u = nrm * act
    h = d['res'] + d['scale'] * u
    out = dict(h=h)
    if case['next']:
        hh, r2 = stats(h, 1)
        out['z'] = hh * d['w2'] + d['b2']
    if not case['train']:
        return out
    dh = d['dh']
    if case['next']:
        dh = dh + back(d['dz'] * d['w2'], hh, r2, 1)
        out.update(dw2=(d['dz'] * hh).sum(rows), db2=d['dz'].sum(rows))
    du = dh * d['scale']
    dn = du * act
    out.update(dres=dh, dscale=(dh * u).sum(rows), dw=(dn * yh).sum(rows), db=dn.sum(rows), dy=back(dn * d['w'], yh, r1, G))
    if sig is not None:
        dg = du * nrm * sig * (1 + d['gate'] * (1 - sig))
        out['dgate'] = dg.sum(1, keepdim=True) if case['gate'] == 'sequence' else dg
    return out


def _exact_adamw(st, case):
    b1, b2 = BETAS
    t = int(st['step']) + 1
    p, g, m, v = (st[n].double() for n in 'pgmv')
    if case['bits'] == 8:
        m = m * st['sm'].double().repeat_interleave(Q8_BLOCK)
        v = (v * st['sr'].double().repeat_interleave(Q8_BLOCK)) ** 2
    m.lerp_(g, 1 - b1)
    v.lerp_(g * g, 1 - b2)
    p = p * (1 - LR * WD) - LR * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + EPS)
    if case['bits'] == 32:
        return dict(p=p, m=m, v=v)
    values = torch.arange(127, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn).double()      # what the codes stand for, ascending
    out = dict(p=p)
    for x, d, code, scale in zip((m, v.sqrt()), _dither(st, torch.tensor(t, device=DEV)), ('m', 'v'), ('sm', 'sr')):
        x = x.view(-1, Q8_BLOCK)
        top = x.abs().amax(1)
        s = torch.where(top > 0, torch.exp2(torch.ceil(torch.log2(top / 448))), 0.0).clamp_min(2.0 ** -126)
        a = x.abs() / s[:, None]
        low = (torch.searchsorted(values, a, right=True) - 1).clamp(0, 125)
        up = torch.floor((a - values[low]) / (values[low + 1] - values[low]) + d / 65536.0).long()
        out[code], out[scale] = (values[(low + up).clamp_max(126)] * x.sign()).view(-1), s
    return out


def work(case):
    e = {'fp32': 4, 'bf16': 2}
    if case['op'] == 'la_step':
        n, s = case['B'], case['B'] * case['H'] * case['Dk'] * case['Dv']
        return dict(bytes=8 * s + n * (2 * case['Hqk'] * case['Dk'] + 2 * case['H'] * case['Dv']) * e[case['dtype']], flops=4 * s)
    if case['op'] == 'la':
        n = case['B'] * case['T'] * (0.75 if case['ragged'] else 1.0)
        qk, v = 2 * case['Hqk'] * case['Dk'], case['H'] * case['Dv']
        s = 8 * case['B'] * case['H'] * case['Dk'] * case['Dv']
        by = n * (qk + 2 * v) * e[case['dtype']] + s
        fl = 4 * n * case['H'] * case['Dk'] * case['Dv']
        if case['train']:
            by += n * (2 * qk + 3 * v) * e[case['dtype']] + 2 * s      # q k v do in, dq dk dv out, three states
            fl += 10 * n * case['H'] * case['Dk'] * case['Dv']
        return dict(bytes=int(by), flops=int(fl))
    if case['op'] in ('row_norm', 'block_tail'):
        n, b = case['B'] * case['T'] * case['C'], e[case['dtype']]
        fwd, bwd = 2, 3
        if case['op'] == 'block_tail':
            tok = case['gate'] == 'token'
            fwd, bwd = 3 + tok + case['next'], 5 + 2 * tok + case['next']
        return dict(bytes=n * b * (fwd + (bwd if case['train'] else 0)) + 16 * case['C'], flops=n * (40 if case['train'] else 12))
    n = sum(math.prod(s) for s in _shapes(case))
    return dict(bytes=n * (2 * e[case['pdtype']] + e[case['gdtype']] + (16 if case['bits'] == 32 else 4)), flops=16 * n)
