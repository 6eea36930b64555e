"""What the sequence-block operators refuse, before anything reaches the device: types, shapes, heads, groups, states, and CPU tensors."""
import pytest
import torch

from ha2g_amd import ops, optim


def _la(B=2, T=3, H=4, Dk=8, Dv=6, dt=torch.float32, step=False):
    lead = (B,) if step else (B, T)
    return dict(q=torch.zeros(*lead, H, Dk, dtype=dt), k=torch.zeros(*lead, H, Dk, dtype=dt), v=torch.zeros(*lead, H, Dv, dtype=dt),
                log_decay=torch.full((H,), -0.1), state=torch.zeros(B, H, Dk, Dv))


LA_BAD = dict(
    other_type=lambda a: a.update(k=a['k'].bfloat16()), half=lambda a: a.update(q=a['q'].half(), k=a['k'].half(), v=a['v'].half()),
    dims=lambda a: a.update(v=a['v'][0]), head_size=lambda a: a.update(k=a['k'][..., :5]), batch=lambda a: a.update(k=a['k'][:1]),
    too_wide=lambda a: a.update(v=torch.zeros(*a['v'].shape[:-1], 129), state=None), heads=lambda a: a.update(q=a['q'][..., :3, :]),
    decay_type=lambda a: a.update(log_decay=a['log_decay'].double()), decay_shape=lambda a: a.update(log_decay=a['log_decay'][:, None]),
    decay_grad=lambda a: a.update(log_decay=a['log_decay'].requires_grad_()), state_shape=lambda a: a.update(state=a['state'][:, :2]),
    state_type=lambda a: a.update(state=a['state'].bfloat16()), cpu=lambda a: None)


@pytest.mark.parametrize('bad', sorted(LA_BAD))
@pytest.mark.parametrize('step', (False, True))
def test_linear_attention_refuses(bad, step):
    a = _la(step=step)
    LA_BAD[bad](a)
    with pytest.raises(ValueError, match='linear_attention'):
        (ops.linear_attention_step if step else ops.linear_attention)(**a)


@pytest.mark.parametrize('lengths', (torch.zeros(2), torch.zeros(2, dtype=torch.int64), torch.zeros(3, dtype=torch.int32)))
def test_linear_attention_refuses_lengths(lengths):
    with pytest.raises(ValueError):
        ops.linear_attention(**_la(), lengths=lengths)


NORM_BAD = dict(half=dict(x=torch.zeros(2, 8).half()), weight_type=dict(weight=torch.ones(8).bfloat16()), weight_shape=dict(weight=torch.ones(4)),
                no_weight=dict(weight=None), groups=dict(groups=3), kind=dict(kind='batch'), wide=dict(x=torch.zeros(1, 16385), weight=torch.ones(16385)),
                empty=dict(x=torch.zeros(2, 0), weight=torch.ones(0)), cpu=dict())


@pytest.mark.parametrize('bad', sorted(NORM_BAD))
def test_row_norm_refuses(bad):
    with pytest.raises(ValueError):
        ops.row_norm(**{**dict(x=torch.zeros(2, 8), weight=torch.ones(8)), **NORM_BAD[bad]})


TAIL_BAD = dict(residual=dict(residual=torch.zeros(2, 4, 8)), residual_type=dict(residual=torch.zeros(2, 3, 8).bfloat16()), act=dict(gate_act=1),
                gate_shape=dict(gate=torch.zeros(1, 3, 8)), gate_type=dict(gate=torch.zeros(2, 3, 8).bfloat16()), bias=dict(weight=None, bias=torch.zeros(8)),
                next_bias=dict(next_bias=torch.zeros(8)), scale=dict(scale=torch.ones(1)), cpu=dict())


@pytest.mark.parametrize('bad', sorted(TAIL_BAD))
def test_block_tail_refuses(bad):
    with pytest.raises(ValueError):
        ops.block_tail(**{**dict(y=torch.zeros(2, 3, 8), weight=torch.ones(8)), **TAIL_BAD[bad]})


def _adamw(bits=32):
    p = [torch.zeros(3, 5), torch.zeros(200)]
    st = [torch.zeros_like(x) for x in p] if bits == 32 else [optim.adamw_state8(x) for x in p]
    st2 = [torch.zeros_like(x) for x in p] if bits == 32 else [optim.adamw_state8(x) for x in p]
    return dict(params=p, grads=[torch.zeros_like(x) for x in p], exp_avgs=st, exp_avg_sqs=st2, step=torch.zeros(1, dtype=torch.int32))


ADAMW_BAD = dict(
    count=lambda a: a['grads'].pop(), mixed=lambda a: a['params'].__setitem__(0, torch.zeros(3, 5).bfloat16()), step=lambda a: a.update(step=torch.zeros(1)),
    shape=lambda a: a['grads'].__setitem__(0, torch.zeros(5, 3)[:, :2]), layout=lambda a: a['grads'].__setitem__(0, torch.zeros(5, 3).t()),
    gap=lambda a: (a['params'].__setitem__(0, torch.zeros(3, 6)[:, :5]), a['grads'].__setitem__(0, torch.zeros(3, 6)[:, :5])),
    half=lambda a: a.update(params=[x.half() for x in a['params']]), guard=lambda a: a.update(guard=torch.zeros(1)), cpu=lambda a: None)


@pytest.mark.parametrize('bits', (32, 8))
@pytest.mark.parametrize('bad', sorted(ADAMW_BAD))
def test_adamw_step_refuses(bad, bits):
    a = _adamw(bits)
    ADAMW_BAD[bad](a)
    with pytest.raises(ValueError):
        optim.adamw_step(**a)


@pytest.mark.parametrize('state', (lambda s: (s[0].float(), s[1]), lambda s: (s[0], s[1][:-1]), lambda s: (s[0][:-1], s[1]), lambda s: s[:1],
                                   lambda s: (s[0], s[1].double()), lambda s: s[0]))
def test_adamw_step_refuses_8_bit_states(state):
    a = _adamw(8)
    a['exp_avgs'][1] = state(a['exp_avgs'][1])
    with pytest.raises((ValueError, TypeError)):
        optim.adamw_step(**a)


def test_adamw_step_refuses_fp32_states_of_another_type_or_size():
    for bad in (torch.zeros(3, 5).bfloat16(), torch.zeros(5, 3), torch.zeros(3, 4)):
        a = _adamw()
        a['exp_avg_sqs'][0] = bad
        with pytest.raises(ValueError):
            optim.adamw_step(**a)


def test_fused_adamw_refuses_state_bits_and_the_trainer_an_unknown_optimizer():
    with pytest.raises(ValueError):
        optim.FusedAdamW([torch.nn.Parameter(torch.zeros(4))], state_bits=16)
    from ha2g_amd.config import hierarchy_args
    from ha2g_amd.train import HierarchyTrainer
    tr = HierarchyTrainer.__new__(HierarchyTrainer)
    tr.sparse_embeddings, tr.args = False, hierarchy_args(optimizer='sgd')
    with pytest.raises(ValueError, match='optimizer'):
        tr.make_optimizers()
    tr.sparse_embeddings, tr.args = True, hierarchy_args(optimizer='adamw8')
    with pytest.raises(ValueError, match='row-wise'):
        tr.make_optimizers()


def test_c_entries_return_errors_instead_of_launching():
    import array
    from ha2g_amd._lib import lib
    st = array.array('l', [0] * 12)
    la = lambda B, H, rq, Dk, Dv: lib.ha2g_linattn_fwd(None, None, None, None, None, None, None, None, st, B, 1, H, rq, 1, 1, Dk, Dv, 1.0, 0, None, None)      # noqa: E731
    assert la(0, 1, 1, 8, 8) == 0
    for bad in ((1, 1, 1, 8, 8), (0, 3, 2, 8, 8), (0, 1, 1, 129, 8), (0, 1, 1, 8, 0), (0, 0, 1, 8, 8)):
        assert la(*bad) != 0 and lib.ha2g_last_error()
    one = array.array('l', [0])
    assert lib.ha2g_adamw_multi(1, one, one, one, one, None, None, array.array('l', [5]), 0, 0, 32, 0.1, 0.9, 0.9, 1e-8, 0.0, 0, 0, None, None, None) != 0
    assert lib.ha2g_adamw_multi(0, None, None, None, None, None, None, None, 0, 0, 16, 0.1, 0.9, 0.9, 1e-8, 0.0, 0, 0, None, None, None) != 0
    assert lib.ha2g_head_sum(None, None, 1, 0, 1, 4, 0, None) != 0
    tail = lambda outer, C, G, act: lib.ha2g_block_tail_fwd(*[None] * 14, outer, 4, 0, C, G, 0, act, 1.0, 1e-5, 0, None)      # noqa: E731
    assert tail(0, 8, 2, 4) == 0
    for bad in ((1, 8, 2, 4), (0, 8, 3, 4), (0, 8, 2, 1), (0, 20000, 1, 4), (70000, 8, 2, 4)):
        assert tail(*bad) != 0 and lib.ha2g_last_error()


class _Cube(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y):
        ctx.save_for_backward(x)
        return x ** 3 + y

    @staticmethod
    @ops._once
    def backward(ctx, d):
        x, = ctx.saved_tensors
        return 3 * x * x * d, d if ctx.needs_input_grad[1] else None


def test_gradients_of_a_pass_without_a_backward_of_its_own_refuse_a_second_derivative():
    """a gradient penalty whose incoming gradient is a constant would lose its term in silence (12 instead of 300 at x = 2)"""
    x = torch.tensor(2.0, requires_grad=True)
    for loss in (lambda o: o, lambda o: o * x, lambda o: o.square()):
        o = _Cube.apply(x, torch.tensor(1.0))
        g, = torch.autograd.grad(loss(o), x, create_graph=True)
        assert g.requires_grad
        with pytest.raises(RuntimeError, match='once_differentiable'):
            (o + g.square()).backward()
        with pytest.raises(RuntimeError, match='once_differentiable'):
            torch.autograd.grad(g, x)
    # first derivatives are what they were, with and without a graph of them, and a gradient that depends on nothing is a constant
    assert torch.autograd.grad(_Cube.apply(x, torch.tensor(1.0)), x)[0] == 12
    assert torch.autograd.grad(_Cube.apply(x, torch.tensor(1.0)), x, create_graph=True)[0] == 12
    y = torch.tensor(1.0, requires_grad=True)
    g, = torch.autograd.grad(_Cube.apply(x.detach(), y), y, create_graph=True)
    assert g == 1 and not g.requires_grad


def test_c_entries_refuse_null_strides_and_operands():
    """in words of their own, before anything is launched (any address that is not null stands for an operand: none is read)"""
    from ha2g_amd._lib import lib
    at = 4096

    def refused(rc):
        assert rc != 0
        e = lib.ha2g_last_error()
        return b'null' in e if isinstance(e, bytes) else 'null' in str(e)
    assert refused(lib.ha2g_linattn_fwd(at, at, at, at, at, None, None, None, None, 1, 1, 1, 1, 1, 1, 8, 8, 1.0, 0, None, None))
    assert refused(lib.ha2g_linattn_bwd(at, at, at, at, at, at, at, at, None, None, None, None, None, 1, 1, 1, 1, 1, 1, 8, 8, 1.0, 0, 0, 0, 0, None, None, None))
    assert refused(lib.ha2g_linattn_step(at, at, at, at, at, at, None, 1, 1, 1, 1, 1, 8, 8, 1.0, 0, None))
    assert refused(lib.ha2g_head_sum(None, at, 1, 1, 2, 4, 0, None)) and refused(lib.ha2g_head_sum(at, None, 1, 1, 2, 4, 0, None))
