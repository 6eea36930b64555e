"""Fused Adam over flat parameter/gradient buffers (HIP kernel ha2g_adam_f32) with torch.optim.Adam semantics as the
reference sets it up (scripts/train.py:155-170: one optimizer per module, lr 5e-4 (D: x0.2), betas (0.5, 0.999)).

Construction re-points every parameter's storage into one flat fp32 buffer (layout-preserving, so channels_last conv
weights stay OHWI) and installs `.grad` views into a matching flat gradient buffer: the optimizer step is then ONE
HBM-streaming kernel, and data-parallel gradient exchange is ONE RCCL all-reduce per module (ha2g_amd/ddp.py).
"""
import array
import operator

import torch

from ._lib import check, lib
from .ops import _FLOATS, _need, _on, _stream, gru_cluster_error_tensor


def _storage_span(p):
    """Number of elements of the dense memory block a (possibly permuted-contiguous) parameter occupies."""
    return p.numel()


class FusedAdam(torch.optim.Optimizer):
    TABLE_STEPS = 1 << 20         # per-step Adam scalars kept for the lazy row updates of sparse tables (8 MB)

    def __init__(self, params, lr=5e-4, betas=(0.5, 0.999), eps=1e-8, sparse=()):
        """sparse: embedding tables (subset of params) updated ROW-WISE from compact gradients (ha2g_amd.ops.SparseTable, csrc/sparse.hip):
        they stay out of the flat buffers; results are bit-identical to the dense update (tests/test_gpu_sparse.py)."""
        params = [p for p in params]
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps))
        sparse_ids = {id(p) for p in sparse if p.requires_grad}
        ps = [p for p in self.param_groups[0]['params'] if p.requires_grad and id(p) not in sparse_ids]
        assert ps, 'no trainable parameters'
        dev = ps[0].device
        assert all(p.dtype == torch.float32 and p.device == dev for p in ps)
        offs, total = [], 0
        for p in ps:
            offs.append(total)
            total += (p.numel() + 3) // 4 * 4                     # keep every tensor 16-byte aligned
        self.flat_p = torch.zeros(total, dtype=torch.float32, device=dev)
        self.flat_g = torch.zeros(total, dtype=torch.float32, device=dev)
        self._make_states(ps, offs, total, dev)
        self.step_t = torch.zeros(1, dtype=torch.int32, device=dev)
        self._views = []
        with torch.no_grad():
            for p, o in zip(ps, offs):
                dense = p.is_contiguous() or (p.dim() == 4 and p.is_contiguous(memory_format=torch.channels_last))
                src = p.data if dense else p.data.contiguous()
                pv = torch.as_strided(self.flat_p, src.shape, src.stride(), o)
                pv.copy_(src)
                p.data = pv
                gv = torch.as_strided(self.flat_g, src.shape, src.stride(), o)
                p.grad = gv
                self._views.append((p, gv))
        self.total = total
        self.sparse_tables = []
        if sparse_ids:
            from .ops import SparseTable
            self.table = torch.zeros(self.TABLE_STEPS, 2, dtype=torch.float32, device=dev)
            self._host_step = 0
            for p in self.param_groups[0]['params']:
                if id(p) in sparse_ids:
                    st = SparseTable(p, self)
                    p._ha2g_sparse = st
                    self.sparse_tables.append(st)

    def _make_states(self, ps, offs, total, dev):
        self.flat_m = torch.zeros(total, dtype=torch.float32, device=dev)
        self.flat_v = torch.zeros(total, dtype=torch.float32, device=dev)

    def zero_grad(self, set_to_none=False):
        """Gradients live in the flat buffer: zero it in place and keep the views installed."""
        self.flat_g.zero_()
        for p, gv in self._views:
            if p.grad is not gv:
                p.grad = gv
        for st in self.sparse_tables:
            st.pending = []

    def _fold_grads(self):
        for p, gv in self._views:                                 # a foreign tensor installed as .grad: fold it back
            if p.grad is not gv:
                if p.grad is not None:
                    gv.copy_(p.grad)
                p.grad = gv

    @torch.no_grad()
    def step(self, closure=None):
        g = self.param_groups[0]
        self._fold_grads()
        st = _stream()
        # guard = the cluster-GRU error word of this device (None before the first cluster launch): while it is set the kernels below leave the
        # step counter, parameters and moments untouched -- a step whose recurrences timed out never reaches the optimizer state
        guard = gru_cluster_error_tensor(self.flat_p.device)
        gp = guard.data_ptr() if guard is not None else None
        check(lib.ha2g_adam_step_inc_guarded(self.step_t.data_ptr(), gp, st))
        check(lib.ha2g_adam_guarded_f32(self.flat_p.data_ptr(), self.flat_g.data_ptr(), self.flat_m.data_ptr(), self.flat_v.data_ptr(),
                                        self.total, float(g['lr']), float(g['betas'][0]), float(g['betas'][1]), float(g['eps']),
                                        self.step_t.data_ptr(), gp, st))
        if self.sparse_tables:
            self._host_step += 1        # informational; past TABLE_STEPS the row kernel recomputes the scalars itself (sparse.hip)
            check(lib.ha2g_adam_scalars(self.step_t.data_ptr(), float(g['lr']), float(g['betas'][0]), float(g['betas'][1]),
                                        self.table.data_ptr(), self.TABLE_STEPS, st))
            for tb in self.sparse_tables:
                tb.step()

    def sync_sparse(self):
        """Replay the pending zero-gradient updates of every row of the sparse tables (call before saving / exporting their weights)."""
        for tb in self.sparse_tables:
            tb.sync()

    def allreduce_grads(self, group=None, async_op=False):
        """Data-parallel: average the flat gradient buffer over ranks (one RCCL all-reduce over xGMI)."""
        from . import ddp
        for tb in self.sparse_tables:
            ddp.exchange_sparse_(tb, group)
        return ddp.average_(self.flat_g, group, async_op)


# a tensor's properties as functions: passes over the lists of a model's tensors run in map()
_numel, _address, _contiguous, _device = torch.Tensor.numel, torch.Tensor.data_ptr, torch.Tensor.is_contiguous, torch.Tensor.get_device
_dtype = operator.attrgetter('dtype')
Q8_BLOCK = 128            # consecutive elements of a tensor that share a scale of an 8-bit state


def adamw_state8(p):
    """A zero 8-bit state of parameter `p`: (e4m3 codes [numel], fp32 scales [ceil(numel / 128)]); it stands for codes * scale."""
    n = p.numel()
    return (torch.zeros(n, dtype=torch.uint8, device=p.device).view(torch.float8_e4m3fn),
            torch.full((-(-n // Q8_BLOCK),), 2.0 ** -126, dtype=torch.float32, device=p.device))


def _alike(p, t):
    """t's memory holds the same elements in the same order as p's"""
    return t.shape == p.shape and (t.stride() == p.stride() or (p.is_contiguous() and t.is_contiguous()))


def _dense(t):
    """one dense block of memory, in whatever order of dimensions"""
    return t.is_contiguous() or (t.dim() == 4 and t.is_contiguous(memory_format=torch.channels_last))


def _ptrs(ts):
    return array.array('l', map(_address, ts))


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, seed=0, guard=None):
    """One AdamW step over lists of tensors, in place (kernel ha2g_adamw_multi: 64 tensors per launch).  `step` (int32 [1] on the device) is advanced first.
    params, grads: fp32 or bf16, one type each, dense and laid out alike (contiguous tensors: of as many elements).  States in 32 bits: fp32 tensors
    laid out like the parameters.  In 8 bits:
    pairs (codes, scales) as adamw_state8 makes them, exp_avg_sqs holding the ROOT of the second moment; `seed` (32 bits) varies the rounding's dither.
    A root above zero is held as at least the smallest code of its block (some 2^-18 of the largest root): it divides the next update.
    No two of the written tensors share memory (one listed twice is refused).  guard: optional int32 device word; while it is not zero the step changes
    nothing.  Everything lies on one device."""
    n = len(params)
    _need(n == len(grads) == len(exp_avgs) == len(exp_avg_sqs), 'adamw_step: %d parameters, %d gradients, %d and %d states', n, len(grads), len(exp_avgs),
          len(exp_avg_sqs))
    _need(step.dtype == torch.int32 and step.numel() == 1, 'adamw_step: step is an int32 tensor of one element')
    _need(guard is None or (guard.dtype == torch.int32 and guard.device == step.device), 'adamw_step: guard is an int32 word on the device of step')
    q8 = n > 0 and isinstance(exp_avgs[0], (tuple, list))
    if q8:
        _need(all(len(s) == 2 for st in (exp_avgs, exp_avg_sqs) for s in st), 'adamw_step: an 8-bit state is a pair (codes, scales)')
        ms, vs, sm, sr = ([s[i] for s in st] for st, i in ((exp_avgs, 0), (exp_avg_sqs, 0), (exp_avgs, 1), (exp_avg_sqs, 1)))
    else:
        ms, vs, sm, sr = exp_avgs, exp_avg_sqs, (), ()
    dev, f32 = step.device, torch.float32
    pt, gt = (params[0].dtype, grads[0].dtype) if n else (f32, f32)
    num = list(map(_numel, params))
    # the usual case in passes over the lists, a few of a tensor's properties each (a step of a model has the time of ~50 tensors in the kernel)
    good = step.is_cuda and pt in _FLOATS and gt in _FLOATS
    if good:
        at, mt = step.get_device(), torch.float8_e4m3fn if q8 else f32
        lists = [(params, pt, num), (grads, gt, num), (ms, mt, num), (vs, mt, num)]
        if q8:
            blocks = [(k + Q8_BLOCK - 1) // Q8_BLOCK for k in num]
            lists += [(sm, f32, blocks), (sr, f32, blocks)]
        for ts, dt, want in lists:
            good = good and list(map(_numel, ts)) == want and set(map(_dtype, ts)) <= {dt} and all(map(_contiguous, ts)) and set(map(_device, ts)) <= {at}
    if not good:
        _adamw_check(params, grads, ms, vs, sm, sr, q8, dev, pt, gt, num)
    if n == 0:
        return
    pp, pm, pv, psm, psr = (_ptrs(ts) for ts in (params, ms, vs, sm, sr))
    written = (pp, pm, pv, psm, psr) if q8 else (pp, pm, pv)
    own = [x for t in written for x in t] if 0 not in num else [x for t in written for x, k in zip(t, num) if k]
    _need(len(set(own)) == len(own), 'adamw_step: a parameter or a state is listed twice')
    with _on(step):
        st, gp = _stream(), None if guard is None else guard.data_ptr()
        sc = torch.empty(4, dtype=f32, device=dev)
        sp = sc.data_ptr()
        b1, b2, lr = float(betas[0]), float(betas[1]), float(lr)
        check(lib.ha2g_adamw_scalars(step.data_ptr(), gp, lr, b1, b2, sp, st))
        check(lib.ha2g_adamw_multi(n, pp, _ptrs(grads), pm, pv, psm if q8 else None, psr if q8 else None, array.array('l', num),
                                   pt is torch.bfloat16, gt is torch.bfloat16, 8 if q8 else 32, lr, b1, b2, float(eps), float(weight_decay),
                                   int(seed) & 0xffffffff, 0, sp, gp, st))
    # a graph that saved a parameter's old value refuses its backward pass from here on
    try:
        torch.autograd.graph.increment_version(params)
    except RuntimeError:                                  # inference tensors have no versions
        torch.autograd.graph.increment_version([p for p in params if not p.is_inference()])


def _adamw_check(params, grads, ms, vs, sm, sr, q8, dev, pt, gt, num):
    """what adamw_step's quick pass did not cover: tensors that are dense in another order of dimensions, and everything that is refused"""
    every = [*params, *grads, *ms, *vs, *sm, *sr]
    _need(all(isinstance(t, torch.Tensor) for t in every), 'adamw_step: lists of tensors (8-bit states: of pairs)')
    _need({t.device for t in every} <= {dev}, 'adamw_step: everything lies on the device of step')
    _need({pt, gt} <= set(_FLOATS) and all(t.dtype == pt for t in params) and all(t.dtype == gt for t in grads),
          'adamw_step: parameters %s, gradients %s (one of fp32, bf16 each)', pt, gt)
    for p, g in zip(params, grads):
        _need(_dense(p) and _alike(p, g), 'adamw_step: a gradient %s %s for a parameter %s %s', tuple(g.shape), g.stride(), tuple(p.shape), p.stride())
    if q8:
        _need(all(t.dtype == torch.float8_e4m3fn for t in (*ms, *vs)) and all(t.dtype == torch.float32 for t in (*sm, *sr)),
              'adamw_step: 8-bit states are float8_e4m3fn codes and fp32 scales')
        blocks = [-(-k // Q8_BLOCK) for k in num]
        _need(all(t.is_contiguous() for st in (ms, vs, sm, sr) for t in st) and [t.numel() for t in ms] == num == [t.numel() for t in vs] and
              [t.numel() for t in sm] == blocks == [t.numel() for t in sr], 'adamw_step: 8-bit states of other sizes than their parameters')
    else:
        _need(all(t.dtype == torch.float32 for t in (*ms, *vs)), 'adamw_step: states are fp32 tensors, or pairs for 8 bits')
        for p, m, v in zip(params, ms, vs):
            _need(_alike(p, m) and _alike(p, v), 'adamw_step: a state %s %s for a parameter %s %s', tuple(m.shape), m.stride(), tuple(p.shape), p.stride())
    _need(dev.type == 'cuda', 'adamw_step: GPU tensors (there is no CPU path)')


class FusedAdamW(FusedAdam):
    """torch.optim.AdamW semantics on FusedAdam's flat parameter and gradient buffers (same data-parallel exchange, same guard against flagged steps),
    with decoupled weight decay and moments in 32 or 8 bits (state_bits; 8: adamw_state8, 2.06 instead of 8 bytes per parameter).  no_decay: parameters
    that are not decayed (biases, norm weights).  Row-wise embedding tables (sparse=) are FusedAdam's alone: a decayed row moves on every step."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, no_decay=(), state_bits=32, seed=0):
        _need(state_bits in (8, 32), 'FusedAdamW: states of %r bits (8 or 32)', state_bits)
        self.state_bits, self.seed = state_bits, int(seed)
        self._no_decay = {id(p) for p in no_decay}
        super().__init__(params, lr=lr, betas=betas, eps=eps)
        self.param_groups[0]['weight_decay'] = weight_decay

    def _make_states(self, ps, offs, total, dev):
        cut = lambda t: [t[o:o + p.numel()] for p, o in zip(ps, offs)]      # noqa: E731
        self._scalars = torch.zeros(4, dtype=torch.float32, device=dev)
        if self.state_bits == 32:
            super()._make_states(ps, offs, total, dev)
            ms, vs, sm, sr = cut(self.flat_m), cut(self.flat_v), None, None
        else:
            self.states8 = [(adamw_state8(p), adamw_state8(p)) for p in ps]
            ms, vs = [m[0] for m, _ in self.states8], [v[0] for _, v in self.states8]
            sm, sr = [m[1] for m, _ in self.states8], [v[1] for _, v in self.states8]
        # the buffers are this optimizer's own and stay where they are: their tables are built once, decayed tensors first
        order = sorted(range(len(ps)), key=lambda i: id(ps[i]) in self._no_decay)
        n_decay = sum(id(p) not in self._no_decay for p in ps)
        self._tables = []
        for idx in (order[:n_decay], order[n_decay:]):
            pick = lambda ts: None if ts is None else _ptrs([ts[i] for i in idx])      # noqa: E731
            self._tables.append((len(idx), pick(cut(self.flat_p)), pick(cut(self.flat_g)), pick(ms), pick(vs), pick(sm), pick(sr),
                                 array.array('l', [ps[i].numel() for i in idx])))

    @torch.no_grad()
    def step(self, closure=None):
        g = self.param_groups[0]
        self._fold_grads()
        with _on(self.flat_p):
            st, guard = _stream(), gru_cluster_error_tensor(self.flat_p.device)
            gp = guard.data_ptr() if guard is not None else None
            b1, b2, sp = float(g['betas'][0]), float(g['betas'][1]), self._scalars.data_ptr()
            check(lib.ha2g_adamw_scalars(self.step_t.data_ptr(), gp, float(g['lr']), b1, b2, sp, st))
            first = 0
            for (n, p, gr, m, v, sm, sr, num), wd in zip(self._tables, (float(g['weight_decay']), 0.0)):
                check(lib.ha2g_adamw_multi(n, p, gr, m, v, sm, sr, num, 0, 0, self.state_bits, float(g['lr']), b1, b2, float(g['eps']), wd,
                                           self.seed & 0xffffffff, first, sp, gp, st))
                first += n
