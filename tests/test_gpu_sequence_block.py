"""The sequence-block operators together: norm -> projections -> linear attention -> tail -> head, trained for a step with FusedAdamW, then streamed a
token at a time from the same weights."""
import pytest
import torch

from ha2g_amd import hierarchy_net as hn, ops, optim

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
C, H, D, B, T = 60, 5, 12, 3, 34


class Block(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.qkv, self.gate, self.out = hn.Linear(C, 3 * C), hn.Linear(C, C), hn.Linear(C, 7)
        for n in ('pre', 'post', 'nxt'):
            setattr(self, n, torch.nn.Parameter(torch.ones(C)))
        self.scale = torch.nn.Parameter(torch.full((C,), 0.5))
        self.register_buffer('g', torch.log1p(-torch.exp2(-torch.linspace(2, 6, H))))

    def mix(self, x):
        n = ops.row_norm(x, self.pre)
        return self.qkv(n).unflatten(-1, (3, H, D)).unbind(-3), self.gate(n)

    def tail(self, o, x, gate):
        h, z = ops.block_tail(o.flatten(-2), x, gate=gate, weight=self.post, scale=self.scale, groups=H, next_weight=self.nxt)
        return h, self.out(z)

    def forward(self, x, lengths=None, state=None):
        (q, k, v), gate = self.mix(x)
        o, s = ops.linear_attention(q, k, v, self.g, state=state, lengths=lengths, return_state=True)
        return self.tail(o, x, gate)[1], s

    def step(self, x, state):
        (q, k, v), gate = self.mix(x)
        return self.tail(ops.linear_attention_step(q, k, v, self.g, state), x, gate)[1]


def plain(block, x):
    """the block in 64 bits"""
    w = {n: p.detach().double() for n, p in block.state_dict().items()}
    w = {n: p.requires_grad_() for n, p in w.items()}
    rms = lambda t, g: (t.unflatten(-1, (g, -1)) / (t.unflatten(-1, (g, -1)).pow(2).mean(-1, keepdim=True) + 1e-5).sqrt()).flatten(-2)      # noqa: E731
    n = rms(x, 1) * w['pre']
    q, k, v = (n @ w['qkv.weight'].t() + w['qkv.bias']).unflatten(-1, (3, H, D)).unbind(-3)
    t = torch.arange(x.shape[1], device=x.device)
    decay = torch.where(t[:, None] >= t, torch.exp(w['g'][:, None, None] * (t[:, None] - t).clamp_min(0)), 0.0)
    o = torch.einsum('bhts,bshd->bthd', torch.einsum('bthd,bshd->bhts', q, k) * D ** -0.5 * decay, v)
    gate = n @ w['gate.weight'].t() + w['gate.bias']
    h = x + w['scale'] * (rms(o.flatten(-2), H) * w['post']) * gate * torch.sigmoid(gate)
    return (rms(h, 1) * w['nxt']) @ w['out.weight'].t() + w['out.bias'], w


def test_a_block_is_trained_and_streamed():
    torch.manual_seed(1)
    block = Block().to(DEV)
    ps = list(block.parameters())
    opt = optim.FusedAdamW(ps, lr=1e-3, weight_decay=0.01, no_decay=[p for p in ps if p.dim() < 2], state_bits=8)
    x, dy = torch.randn(B, T, C, device=DEV), torch.randn(B, T, 7, device=DEV)
    opt.zero_grad()
    y, _ = block(x)
    y.backward(dy)
    want, w = plain(block, x.double().cpu().to(DEV))
    want.backward(dy.double())
    # a chain of eight fp32 operators: 2^-24 times the square root of the longest sums (180 terms) for each, one order of magnitude for their spread
    tol = 8 * 180 ** 0.5 * 2.0 ** -24 * 10
    assert float((y.double() - want).norm() / want.norm()) <= tol
    for n, p in block.named_parameters():
        d = w[n].grad
        assert float((p.grad.double() - d).norm() / d.norm()) <= tol, n
    before = [p.detach().clone() for p in ps]
    opt.step()
    for p, b, n in zip(ps, before, (n for n, _ in block.named_parameters())):
        moved = (p - b).abs().max()
        assert 0 < float(moved) <= 1.1e-3 + 1e-5 * float(b.abs().max()), n
    with torch.no_grad():
        whole, last = block(x)
        state = torch.zeros(B, H, D, D, device=DEV)
        steps = torch.stack([block.step(x[:, t], state) for t in range(T)], 1)
        assert float((steps - whole).norm() / whole.norm()) <= tol and float((state - last).norm() / last.norm()) <= tol
        # a prompt of ragged rows, then tokens: the state of a shorter row is that of its own end
        lengths = torch.tensor([T, 5, 0], dtype=torch.int32, device=DEV)
        _, s = block(x, lengths=lengths)
        tok = torch.randn(B, C, device=DEV)
        got = block.step(tok, s)
        for b, n in enumerate(lengths.tolist()):
            row, _ = block(torch.cat([x[b:b + 1, :n], tok[b:b + 1, None]], 1))
            assert float((row[0, -1] - got[b]).norm() / got[b].norm()) <= tol


def test_training_mode_bf16_runs_end_to_end():
    torch.manual_seed(2)
    q, k, v = (torch.randn(2, 50, 4, 16, device=DEV, dtype=torch.bfloat16, requires_grad=True) for _ in range(3))
    g = torch.full((4,), -0.05, device=DEV)
    w = torch.ones(64, device=DEV, requires_grad=True)
    x = torch.randn(2, 50, 64, device=DEV, dtype=torch.bfloat16)
    h, z = ops.block_tail(ops.linear_attention(q, k, v, g).flatten(2), x, weight=w, groups=4, next_weight=w)
    (h.float().square().sum() + z.float().sum()).backward()
    for t in (q, k, v, w):
        assert torch.isfinite(t.grad).all() and t.grad.abs().max() > 0
