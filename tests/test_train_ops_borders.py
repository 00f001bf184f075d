"""The training operators at the borders of what a caller may do: saved tensors that come back in another layout, other kinds of derivatives, many steps,
optimiser groups and checkpoints.  References in 64 bits; the bounds are those of test_train_ops.py unless a test derives its own."""
import contextlib
import os
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, 'tests'))

from unopticalflow_amd import ops, optim  # noqa: E402
from test_train_ops import DTYPES, _check_orthogonal, _inputs, _matrix, _muon, device  # noqa: E402,F401


# ------------------------------------------------------------------------------------------ linear_cross_entropy under saved-tensor hooks
def _cut(x, before, behind):
    """x as columns of a wider matrix, NaN around it."""
    wide = torch.full((len(x), before + x.shape[1] + behind), float('nan'), dtype=x.dtype, device=x.device)
    wide[:, before:before + x.shape[1]] = x
    return wide[:, before:before + x.shape[1]]


def _shifted(t):
    """A copy that starts one element behind an aligned address."""
    room = torch.zeros(t.numel() + 1, dtype=t.dtype, device=t.device)
    return room[1:].view(t.shape).copy_(t)


RETURNS = {
    'dense': lambda t: t.contiguous().clone(),
    'shifted': _shifted,
    'columns': lambda t: _cut(t, 3, 5) if t.is_floating_point() and t.dim() == 2 else _shifted(t),
    'transposed': lambda t: t.mT.clone().mT if t.dim() == 2 else t.clone(),
}


@pytest.mark.parametrize('back', list(RETURNS))
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('rows,dim', [(9, 40), (20, 40), (70, 40), (70, 37)])
def test_saved_tensors_in_another_layout(device, dtype, rows, dim, back):
    """Offloading hands back what was saved in a layout of its own.  Every layout of the forward pass (aligned, wider rows, rows that start
    anywhere, one of the two operands only) with every layout of the backward pass gives the bits of the call without hooks."""
    h, w, t = _inputs(rows, 50, dim, dtype, device)
    layouts = (lambda x: x, lambda x: _cut(x, 0, 24), lambda x: _cut(x, 1, 0), _shifted)
    for lay_h, lay_w in [(a, a) for a in layouts] + [(layouts[0], layouts[2]), (layouts[2], layouts[0])]:
        a, b = lay_h(h).requires_grad_(), lay_w(w).requires_grad_()
        want = torch.autograd.grad(ops.linear_cross_entropy(a, b, t), (a, b))
        with torch.autograd.graph.saved_tensors_hooks(lambda x: x, RETURNS[back]):
            got = torch.autograd.grad(ops.linear_cross_entropy(a, b, t), (a, b))
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_offloading_to_the_host(device):
    h, w, t = _inputs(70, 50, 40, torch.float32, device)
    a, b = _cut(h, 0, 24).requires_grad_(), _cut(w, 3, 5).requires_grad_()
    want = torch.autograd.grad(ops.linear_cross_entropy(a, b, t), (a, b))
    with torch.autograd.graph.save_on_cpu():
        got = torch.autograd.grad(ops.linear_cross_entropy(a, b, t), (a, b))
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_saved_tensors_of_another_kind_are_refused():
    """What a hook hands back has to be what was saved: another type, shape or size is an error before anything is launched."""
    import train_on_host
    with train_on_host.patched():
        h, w, t = _inputs(70, 50, 40, torch.float32, 'cpu')
        h.requires_grad_()
        for wrong in (lambda x: x.to(torch.bfloat16) if x.is_floating_point() else x, lambda x: x[:-1] if x.dim() == 2 else x,
                      lambda x: x[:, :-1] if x.dim() == 2 else x, lambda x: x[:-1] if x.dtype == torch.int64 else x,
                      lambda x: x[:-256] if x.dtype == torch.uint8 else x, lambda x: x.int() if x.dtype == torch.int64 else x):
            with torch.autograd.graph.saved_tensors_hooks(lambda x: x, wrong):
                loss = ops.linear_cross_entropy(h, w, t)
                with pytest.raises(RuntimeError):
                    torch.autograd.grad(loss, h)


def test_entry_points_check_what_was_kept():
    """The C entries take the size of what the forward pass kept, whose last bits say which inputs it holds packed."""
    import ctypes
    import __graft_entry__ as ge
    ge.build()
    from unopticalflow_amd import _lib
    lib = _lib.load()
    k, a, b = ctypes.c_longlong(), ctypes.c_longlong(), ctypes.c_longlong()

    def kept(hidden, weight, n=100, dtype=1):
        assert lib.unflow_linear_ce_workspace(hidden, 40, weight, 40, n, 50, 40, dtype, 1, 1, ctypes.byref(k), ctypes.byref(a), ctypes.byref(b)) == 0
        return k.value
    base, off = 4096, 4098
    sizes = [kept(base, base), kept(off, base), kept(base, off), kept(off, off)]
    assert [s % 256 for s in sizes] == [0, 1, 2, 3] and kept(base, base, dtype=0) % 256 == 3
    assert kept(off, off, 16) % 256 == 0 and kept(base, off, 20) % 256 == 0          # few rows: nothing but statistics
    fwd = lambda size: lib.unflow_linear_ce_fwd_ex(off, 40, off, 40, base, 100, 50, 40, 1, 1.0, -100, 1, base, base, size, base, 16, None)  # noqa: E731
    assert all(fwd(s) == -22 for s in sizes + [0, -1])                               # (a workspace of 16 bytes, or a wrong size)
    need = lambda size, dtype=1, n=100: lib.unflow_linear_ce_bwd_workspace(off, 40, off, 40, n, 50, 40, dtype, 1, 1, size, ctypes.byref(b))  # noqa: E731
    assert all(need(s) == 0 and b.value > 0 for s in sizes)
    assert all(need(s) == -22 for s in [x + 256 for x in sizes] + [sizes[0] + 1, sizes[3] - 1, 0, -1]) and need(sizes[3], n=130) == -22
    # (100 rows and 101 need as many lines of 256 bytes, 1604 or 1620 bytes of statistics and 8000 or 8080 of packed rows, so one's buffer is large enough for the other)
    assert need(sizes[3], n=101) == 0
    whole = kept(base, base, dtype=0)
    assert need(whole, 0) == 0 and need(whole - 1, 0) == -22 and need(whole - 2, 0) == -22
    bwd = lambda size, at=base: lib.unflow_linear_ce_bwd_ex(off, 40, off, 40, base, base, 100, 50, 40, 1, 1.0, -100, 1, base, None, at, size, base, 1 << 40, None)  # noqa: E731
    assert bwd(sizes[3] + 256) == -22 and bwd(0) == -22 and bwd(sizes[3], None) == -22 and bwd(sizes[3], base + 2) == -22


# ------------------------------------------------------------------------------------------ orthogonalize: many steps
def _deficient(kind, shape):
    """Matrices of low rank, of numbers of 24 bits: products of thin factors, equal rows, one column alone."""
    g = torch.Generator().manual_seed(0)
    m, n = min(shape), max(shape)
    if kind == 'equal rows':
        x = torch.randn(1, n, generator=g).expand(m, n).clone()
    elif kind == 'one column':
        x = torch.zeros(m, n)
        x[:, n // 2] = torch.randn(m, generator=g)
    else:
        x = torch.randn(m, kind, generator=g) @ torch.randn(kind, n, generator=g)
    return x if shape[0] < shape[1] else x.T.contiguous()


@pytest.mark.parametrize('coefficients,top', [((3.4445, -4.7750, 2.0315), 1.2025), ((2.0, -1.5, 0.5), 1.0018), ((1.5, -0.5, 0.0), 1.0)])
@pytest.mark.parametrize('kind,shape', [(3, (20, 60)), (1, (8, 500)), ('equal rows', (16, 40)), (5, (300, 32)), ('one column', (32, 33))])
@pytest.mark.parametrize('steps', [9, 12, 20, 40, 64])
def test_few_rows_of_low_rank_stay_bounded(device, steps, kind, shape, coefficients, top):
    """No singular value leaves what the polynomial reaches from [0, 1] (`top`), whatever rounding puts into the directions that the matrix does not
    have: 22 bits of each of the step's three matrices, 2^-10 of them together, on top of it."""
    x = _deficient(kind, shape).to(device)
    got = ops.orthogonalize(x, steps=steps, coefficients=coefficients).double()
    assert bool(torch.isfinite(got).all())
    size = torch.linalg.svdvals(got.cpu())
    assert float(size[0]) <= top * (1 + 2**-10), float(size[0])
    assert float(size[kind - 1 if isinstance(kind, int) else 0]) >= 0.5


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_many_muon_steps_of_few_rows(device, dtype):
    """A weight of few rows whose gradient has rank 1 moves by at most lr sqrt(max(1, rows / cols)) 1.2025 and the rounding of its type."""
    p = torch.zeros(40, 24, dtype=dtype, device=device)
    g = _deficient(1, (40, 24)).to(dtype).to(device)
    optim.muon_step_([p], [g], [torch.zeros(40, 24, device=device)], lr=0.5, steps=30)
    size = torch.linalg.svdvals(p.double().cpu())
    assert bool(torch.isfinite(size).all())
    assert float(size[0]) <= 0.5 * (40 / 24) ** 0.5 * 1.2025 * (1 + 2**-10) + torch.finfo(dtype).eps / 2 * float(p.double().norm())


@pytest.mark.parametrize('steps', [1, 5, 7, 8, 9, 10, 11])
def test_steps_on_both_sides_of_the_kernels_for_few_rows(device, steps):
    x = _matrix(24, 90, dtype=torch.float32, device=device)
    _check_orthogonal(ops.orthogonalize(x, steps=steps), x, steps=steps)


def test_the_workspace_depends_on_the_steps():
    """The size for given steps and coefficients is what a call checks; the one without them is enough for any."""
    import ctypes
    import __graft_entry__ as ge
    ge.build()
    from unopticalflow_amd import _lib
    lib = _lib.load()
    need, any_steps = ctypes.c_longlong(), ctypes.c_longlong()
    for rows, cols in ((20, 60), (300, 7), (70, 90)):
        m = (ops._Matrix * 1)((4096, 4096, None, rows, cols))
        assert lib.unflow_orthogonalize_workspace(m, 1, 0, ctypes.byref(any_steps)) == 0
        for steps in (1, 5, 12, 64):
            assert lib.unflow_orthogonalize_workspace_ex(m, 1, 0, steps, 3.4445, -4.7750, 2.0315, ctypes.byref(need)) == 0
            assert 0 < need.value <= any_steps.value
            assert lib.unflow_orthogonalize(m, 1, 0, steps, 3.4445, -4.7750, 2.0315, 1e-7, 4096, need.value - 1, None) == -22
    for bad in ((0, 3.4445, -4.7750, 2.0315), (65, 3.4445, -4.7750, 2.0315), (5, 9.0, 9.0, 9.0)):
        assert lib.unflow_orthogonalize_workspace_ex(m, 1, 0, *bad, ctypes.byref(need)) == -22


# ------------------------------------------------------------------------------------------ linear_cross_entropy: derivatives and tracers of other kinds
@pytest.mark.parametrize('which', ['hidden', 'weight'])
@pytest.mark.parametrize('no_grad', [False, True])
def test_no_forward_mode_derivative(device, which, no_grad):
    """A tangent is refused, as it is where an input asks for a gradient; it does not disappear."""
    from torch.autograd import forward_ad
    h, w, t = _inputs(5, 7, 8, torch.float32, device)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(h if which == 'hidden' else w, torch.ones_like(h if which == 'hidden' else w))
        with torch.set_grad_enabled(not no_grad), pytest.raises(NotImplementedError):
            ops.linear_cross_entropy(*((dual, w) if which == 'hidden' else (h, dual)), t)
        assert torch.isfinite(ops.linear_cross_entropy(h, w, t))             # (without tangents it is an ordinary call)


@pytest.mark.parametrize('gradient', [False, True])
def test_a_trace_calls_the_operator(device, gradient):
    """torch.jit.trace records the call, not the values of the traced one."""
    h, w, t = _inputs(5, 7, 8, torch.float32, device)
    h.requires_grad_(gradient)
    with pytest.warns(torch.jit.TracerWarning):
        traced = torch.jit.trace(lambda a, b: ops.linear_cross_entropy(a, b, t), (h, w), check_trace=False)
    other = _inputs(5, 7, 8, torch.float32, device, seed=1)[0]
    assert torch.equal(traced(other, w), ops.linear_cross_entropy(other, w, t))


def test_tracers_that_would_record_constants_are_refused(device):
    """make_fx sees the allocations around a kernel only, and jit.trace those of an operator that is no autograd function."""
    from torch.fx.experimental.proxy_tensor import make_fx
    h, w, t = _inputs(5, 7, 8, torch.float32, device)
    for x in (h, h.clone().requires_grad_()):
        with pytest.raises(RuntimeError, match='trace'):
            make_fx(lambda a: ops.linear_cross_entropy(a, w, t))(x)
    with pytest.raises(RuntimeError, match='trace'):
        make_fx(lambda a: ops.orthogonalize(a))(h)
    with pytest.raises(RuntimeError, match='trace'):
        torch.jit.trace(lambda a: ops.orthogonalize(a), (h,), check_trace=False)
    m = torch.zeros_like(h)

    def step(p, g):
        optim.muon_step_([p], [g], [m], lr=0.1)
        return p
    for tracer in (lambda: make_fx(step)(h.clone(), h), lambda: torch.jit.trace(step, (h.clone(), h), check_trace=False)):
        with pytest.raises(RuntimeError, match='trace'):
            tracer()
    assert not m.any()


# ------------------------------------------------------------------------------------------ linear_cross_entropy: gradients far from 1
@pytest.mark.parametrize('reduction', ['mean', 'sum', 'none'])
@pytest.mark.parametrize('dtype,sizes', [
    (torch.float32, (2.0**-40, 2.0**-66, 1.0)), (torch.float32, (2.0**-46, 2.0**-66, 1.0)), (torch.float32, (2.0**-53, 2.0**-66, 1.0)),
    (torch.float32, (2.0**-60, 2.0**60, 2.0**-66)), (torch.float32, (2.0**60, 2.0**-100, 1.0)), (torch.float32, (2.0**-60, 2.0**-10, 2.0**-20)),
    (torch.float32, (2.0**40, 2.0**-90, 2.0**-60)), (torch.bfloat16, (2.0**-53, 2.0**-66, 1.0)), (torch.bfloat16, (2.0**60, 2.0**-100, 1.0)),
    (torch.bfloat16, (2.0**40, 2.0**-90, 2.0**-60))], ids=str)
def test_gradients_of_any_magnitude(device, dtype, sizes, reduction):
    """Hidden rows, the upstream gradient and the scale times powers of two (the weights take the inverse, so that the logits stay): the gradients are
    those of the plain call times powers of two, bit for bit, as long as all of them are ordinary numbers of the type."""
    size, up, scale = sizes
    h, w, t = _inputs(40, 33, 24, dtype, device)
    base = torch.rand(40, generator=torch.Generator().manual_seed(3)).to(device) if reduction == 'none' else torch.tensor(0.75, device=device)

    def grads(h, w, upstream, scale):
        h, w = h.detach().requires_grad_(), w.detach().requires_grad_()
        return torch.autograd.grad(ops.linear_cross_entropy(h, w, t, scale=scale, reduction=reduction), (h, w), upstream)
    want = grads(h, w, base, 1.0)
    got = grads(h * size, w / (size * scale), base * up, scale)
    for x, y, factor in zip(got, want, (up / size, up * scale * size)):
        exact = y.double() * factor
        ordinary = (exact.abs() >= torch.finfo(dtype).smallest_normal) | (exact == 0)
        assert bool(ordinary.any()) and float(exact.abs().max()) <= torch.finfo(dtype).max
        assert torch.equal(x.double()[ordinary], exact[ordinary])
        assert bool(((x.double() - exact).abs() <= torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps).all())


# ------------------------------------------------------------------------------------------ FlowMuon
def _parameter(*shape, seed=0, dtype=torch.float32, device='cpu'):
    p = torch.nn.Parameter(torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(device))
    p.grad = torch.ones_like(p) * 0.5
    return p


def test_a_group_given_as_a_generator(device):
    """module.parameters() is a generator: its weights are in the group, and they train."""
    first, second = _parameter(3, 4, device=device), _parameter(5, 4, seed=1, device=device)
    opt = optim.FlowMuon([first], lr=0.1)
    group = {'params': (p for p in [second]), 'lr': 0.2}
    opt.add_param_group(group)
    assert [len(g['params']) for g in opt.param_groups] == [1, 1] and 'kind' not in group
    alone = _parameter(6, 4, seed=2, device=device)
    opt.add_param_group({'params': alone})
    before = [p.detach().clone() for p in (first, second, alone)]
    opt.step()
    assert not any(torch.equal(p, old) for p, old in zip((first, second, alone), before))
    with pytest.raises(ValueError):
        opt.add_param_group({'params': (p for p in [_parameter(4, device=device)])})


def test_sets_have_no_order():
    with pytest.raises(TypeError):
        optim.FlowMuon([_parameter(3, 4)]).add_param_group({'params': {_parameter(3, 4, seed=1)}})


@pytest.mark.parametrize('kind', ['others', 'anything'])
def test_a_further_group_holds_matrices(kind):
    """Adam's parameters are those of the constructor: a group that no step would reach is refused, and nothing is added."""
    opt = optim.FlowMuon([_parameter(3, 4), _parameter(4, seed=1)])
    for p in (_parameter(4, seed=2), _parameter(4, 4, seed=2)):
        with pytest.raises(ValueError, match='kind'):
            opt.add_param_group({'params': [p], 'kind': kind})
    assert [len(g['params']) for g in opt.param_groups] == [1, 1]


def test_checkpoints_of_another_optimiser_are_refused_whole(device):
    """An Adam state of the same groups, a momentum of another shape, moments that are missing: an error, and the optimiser is as it was."""
    def fresh(seed=0):
        ps = [_parameter(3, 4, seed=seed, device=device), _parameter(5, 2, seed=seed + 1, device=device), _parameter(4, seed=seed + 2, device=device)]
        return ps, optim.FlowMuon(ps, lr=0.1)
    only, narrow = [_parameter(3, 4, device=device), _parameter(5, 2, seed=1, device=device)], None
    narrow = optim.FlowMuon(only, lr=0.1)
    adam = torch.optim.Adam([p for p in only], lr=0.1)
    adam.step()
    narrow.step()
    kept = {k: v.clone() for p in only for k, v in ((p, narrow.state[p]['momentum_buffer']),)}
    with pytest.raises(ValueError):
        narrow.load_state_dict(adam.state_dict())
    assert narrow.param_groups[0]['kind'] == 'matrices' and all(torch.equal(narrow.state[p]['momentum_buffer'], m) for p, m in kept.items())
    narrow.step()
    if device == 'cuda':                                 # (the biases' Adam runs on the device only)
        params, opt = fresh()
        opt.step()
        good = opt.state_dict()
        for where, key, value in ((0, 'momentum_buffer', torch.zeros(4, 3, device=device)), (0, 'momentum_buffer', None), (1, 'momentum_buffer', torch.zeros(1, 1, device=device)),
                                  (2, 'exp_avg', None), (2, 'exp_avg_sq', None), (2, 'step', None), (2, 'exp_avg', torch.zeros(3, device=device))):
            state = {i: dict(s) for i, s in good['state'].items()}
            state[where].pop(key)
            if value is not None:
                state[where][key] = value
            else:                                        # (nothing at all is the state of a weight that has not stepped)
                state[where]['other'] = 1.0
            with pytest.raises(ValueError):
                opt.load_state_dict({'state': state, 'param_groups': good['param_groups']})
        opt.step()
        opt.load_state_dict(good)
        opt.step()
    state = narrow.state_dict()
    for wrong in (torch.zeros(4, 3), torch.zeros(1, 4), None, 3.0):
        with pytest.raises(ValueError):
            narrow.load_state_dict({'state': {0: {'momentum_buffer': wrong}, 1: state['state'][1]}, 'param_groups': state['param_groups']})
    narrow.load_state_dict({'state': {}, 'param_groups': state['param_groups']})         # (a run that has not stepped)
    narrow.step()
    assert all(bool(torch.isfinite(p).all()) for p in only)


def test_matrices_of_several_types_in_one_group(device):
    """Every type has a call of its own; the weights move as they do alone."""
    shapes, dtypes = [(12, 20), (40, 8), (9, 70), (33, 34)], [torch.float32, torch.bfloat16, torch.float16, torch.bfloat16]
    params = [_parameter(*s, seed=i, dtype=t, device=device) for i, (s, t) in enumerate(zip(shapes, dtypes))]
    for i, p in enumerate(params):
        p.grad = _matrix(*p.shape, dtype=p.dtype, device=device, seed=10 + i)
    before = [p.detach().clone() for p in params]
    optim.FlowMuon(params, lr=0.1).step()
    for t in set(dtypes):
        chosen = [i for i, d in enumerate(dtypes) if d == t]
        want = [before[i].clone() for i in chosen]
        optim.muon_step_(want, [params[i].grad for i in chosen], [torch.zeros_like(w, dtype=torch.float32) for w in want], lr=0.1)
        assert all(torch.equal(params[i], w) for i, w in zip(chosen, want))


def test_weights_that_no_step_takes_are_refused_at_once():
    """Types and sides that muon_step_ refuses: the optimiser is not made, and no group is added."""
    good = _parameter(3, 4)
    opt = optim.FlowMuon([good])
    for bad in (_parameter(3, 4, dtype=torch.float64), torch.nn.Parameter(torch.zeros(1, (1 << 18) + 1)), torch.nn.Parameter(torch.zeros(3, 4, dtype=torch.complex64))):
        with pytest.raises((TypeError, ValueError)):
            optim.FlowMuon([good, bad])
        with pytest.raises((TypeError, ValueError)):
            opt.add_param_group({'params': [bad]})
    assert len(opt.param_groups) == 1


# ------------------------------------------------------------------------------------------ muon_step_: what it writes
def _views(device, offsets, shape=(5, 8), size=200):
    buffer = torch.randn(size, generator=torch.Generator().manual_seed(4)).to(device)
    return buffer, [buffer[o:o + shape[0] * shape[1]].view(shape) for o in offsets]


def test_weights_that_share_memory_are_refused():
    """Overlapping views of one buffer as momenta, as parameters, as a parameter and a momentum, and a gradient within what another weight writes."""
    import train_on_host
    with train_on_host.patched():
        new = lambda: torch.ones(5, 8)  # noqa: E731
        for offsets in ((0, 20), (20, 0), (0, 39), (0, 0)):
            buffer, (a, b) = _views('cpu', offsets)
            kept = buffer.clone()
            ps, gs, ms = [new(), new()], [new(), new()], [new(), new()]
            for params, grads, momenta in ((ps, gs, [a, b]), ([a, b], gs, ms), ([a, ps[0]], gs, [ms[0], b]), (ps, [a, gs[0]], [ms[0], b]), ([ps[0], b], [a, gs[0]], ms)):
                with pytest.raises(ValueError):
                    optim.muon_step_(params, grads, momenta, lr=0.1)
            assert torch.equal(buffer, kept) and all(torch.equal(x, new()) for x in ps + gs + ms)
        buffer, (a, b) = _views('cpu', (0, 20))          # (a weight's own gradient is its momentum, and another's lies across it)
        with pytest.raises(ValueError):
            optim.muon_step_([new(), new()], [b, a], [b, new()], lr=0.1)
        half = torch.ones(200, dtype=torch.bfloat16)
        with pytest.raises(ValueError):                  # (weights of 2 bytes a number: 0 .. 79 and 78 .. 157)
            optim.muon_step_([half[:40].view(5, 8), half[39:79].view(5, 8)], [new().bfloat16()] * 2, [new(), new()], lr=0.1)


def test_neighbours_in_one_buffer_are_fine(device):
    """Views that touch but do not overlap, one gradient for two weights, a weight's own gradient in its momentum."""
    buffer, (a, b) = _views(device, (0, 40))
    other, (ma, mb) = _views(device, (40, 0))
    g = _matrix(5, 8, dtype=torch.float32, device=device)
    want = [a.clone(), b.clone()], [ma.clone(), mb.clone()]
    optim.muon_step_(want[0], [g, g.clone()], want[1], lr=0.1)
    optim.muon_step_([a, b], [g, g], [ma, mb], lr=0.1)
    assert all(torch.equal(x, y) for x, y in zip([a, b, ma, mb], want[0] + want[1]))
    m = g.clone()
    p, q = torch.ones(5, 8, device=device), torch.ones(5, 8, device=device)
    optim.muon_step_([p], [m], [m], lr=0.1)
    optim.muon_step_([q], [g], [g.clone()], lr=0.1)
    assert torch.equal(p, q) and torch.equal(m, g)


def test_the_entry_point_refuses_shared_memory():
    """The C entry over the host-executed kernels, and the library itself, which returns before any launch."""
    import __graft_entry__ as ge
    ge.build()
    from unopticalflow_amd import _lib
    import train_on_host
    with train_on_host.patched() as lib:
        x = torch.zeros(1000)
        base, ws = x.data_ptr(), torch.zeros(1 << 20, dtype=torch.uint8)
        call = lambda *m: lib.unflow_muon_step((ops._Matrix * len(m))(*m), len(m), 0, 0.1, 0.9, 0.0, 1, 5, 3.4445, -4.7750, 2.0315, 1e-7, ws.data_ptr(), ws.numel(), None)  # noqa: E731
        at = lambda *k: tuple(base + 4 * 40 * i for i in k) + (5, 8)  # noqa: E731
        assert call(at(0, 1, 2), at(3, 4, 5)) == 0 and call(at(0, 1, 2), at(0, 4, 5)) == 0 and call(at(2, 1, 2)) == 0 and call(at(1, 1, 2)) == 0
        for bad in ((at(0, 1, 2), at(3, 1, 5)), (at(0, 1, 2), at(3, 2, 5)), (at(0, 1, 1),), (at(0, 1, 2), at(1, 4, 5)), (at(0, 1, 2), at(2, 4, 5)),
                    (at(0, 1, 2), at(2.5, 4, 5)), (at(2, 1, 2), at(1.5, 4, 5))):
            assert call(*[tuple(int(v) for v in m) for m in bad]) == -22
    assert _lib.load().unflow_muon_step((ops._Matrix * 1)((4096, 8192, 8192, 5, 7)), 1, 0, 0.1, 0.9, 0.0, 1, 5, 3.4445, -4.7750, 2.0315, 1e-7, 4096, 1 << 30, None) == -22


def test_autograd_sees_what_a_step_writes(device):
    """A graph from before the step needs the old weight: its backward pass is an error, as behind torch's own optimisers."""
    w, x = _parameter(12, 20, device=device), torch.ones(3, 20, device=device)
    m = torch.zeros(12, 20, device=device)
    x.requires_grad_()
    loss = (x @ w.T).sum()
    versions = w._version, m._version
    optim.muon_step_([w], [w.grad], [m], lr=0.1)
    assert w._version > versions[0] and m._version > versions[1]
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        loss.backward()
    opt = optim.FlowMuon([w], lr=0.1)
    opt.step()
    loss = (x @ w.T).sum()
    opt.step()
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        loss.backward()
    (x @ w.T).sum().backward()                           # (a graph from behind the step is fine)


@contextlib.contextmanager
def _adam_on(where):
    """FlowAdam's kernel: on the device, or host-executed."""
    if where == 'cuda':
        yield
        return
    import hostexec
    with hostexec.patched(ops):
        yield


@pytest.mark.parametrize('where', ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)])
def test_autograd_sees_what_adam_writes(where):
    """FlowAdam's one launch counts as a write of the weights and moments, as torch.optim.Adam's does."""
    with _adam_on(where):
        w, x = _parameter(12, 20, device=where), torch.ones(3, 20, device=where, requires_grad=True)
        opt = optim.FlowAdam([w], lr=0.1)
        opt.step()
        versions = w._version, opt.state[w]['exp_avg']._version, opt.state[w]['exp_avg_sq']._version
        loss = (x @ w.T).sum()
        opt.step()
        assert opt.native_steps == 2
        assert all(a < b for a, b in zip(versions, (w._version, opt.state[w]['exp_avg']._version, opt.state[w]['exp_avg_sq']._version)))
        with pytest.raises(RuntimeError, match='modified by an inplace operation'):
            loss.backward()
        (x @ w.T).sum().backward()


# ------------------------------------------------------------------------------------------ lists, ranks and commands
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_lists_of_more_than_a_wave_of_matrices(device, dtype):
    """140 matrices of sides 3 to 130 (host-executed 70 of up to 60, in fp32), of more than 32 rows among them: past 64 a launch searches its table
    in several goes."""
    count, longest = (140, 130) if device == 'cuda' else (70, 60)
    if device != 'cuda' and dtype != torch.float32:
        pytest.skip('host-executed in fp32 only')
    g = torch.Generator().manual_seed(0)
    sides = torch.randint(3, longest + 1, (count, 2), generator=g).tolist()
    assert max(min(s) for s in sides) > 32
    xs = [_matrix(*s, dtype=dtype, device=device, seed=i) for i, s in enumerate(sides)]
    for x, y in zip(xs, ops.orthogonalize(xs)):
        _check_orthogonal(y, x)


class _Net(torch.nn.Module):
    """What FlowTrainer takes for a model, with a convolution, a projection and biases."""

    def __init__(self):
        super().__init__()
        self.conv = torch.nn.Conv2d(3, 36, 3)
        self.proj = torch.nn.Linear(36, 5)

    def forward(self, x):
        y = self.proj(torch.tanh(self.conv(x)).mean((2, 3)))
        return {'loss_pixel': y[:, 0].square(), 'loss_ssim': y[:, 1].square() + y[:, 4].exp(), 'loss_flow_smooth': y[:, 2].square(), 'loss_flow_consis': y[:, 3].square()}


class _Either:
    """Two libraries that each hold a part of the entry points."""

    def __init__(self, *libs):
        self.libs = libs

    def __getattr__(self, name):
        return getattr(next(lib for lib in self.libs if hasattr(lib, name)), name)


def _muon_rank(rank, world, port, flat, out_path):
    """One of two ranks of FlowTrainer(optimizer='muon') over gloo and the host-executed kernels: the eager step with its pieces sent from hooks, or
    (flat) the exchange of the replayed step without its graphs."""
    import hostexec
    import train_on_host
    import torch.distributed as dist
    from oracle import ref_cpu as R
    from unopticalflow_amd import _lib
    from unopticalflow_amd.parallel import init_distributed, shard_batch
    from unopticalflow_amd.trainer import FlowTrainer
    os.environ.update(RANK=str(rank), LOCAL_RANK=str(rank), WORLD_SIZE=str(world), MASTER_ADDR='127.0.0.1', MASTER_PORT=str(port))
    torch.set_num_threads(2)
    init_distributed('gloo')
    with hostexec.patched(ops) as lib, train_on_host.patched() as train:
        _lib._lib = _Either(lib, train)
        torch.manual_seed(rank)                          # (rank 0's weights win)
        model = _Net()
        trainer = FlowTrainer(R.default_cfg(), model, distributed=True, use_graph=flat, optimizer='muon', muon_lr=0.05, defer_bias_grads=False)
        assert type(trainer.optimizer) is optim.FlowMuon and trainer.optimizer.prepare()
        x = torch.randn(2 * world, 3, 8, 8, generator=torch.Generator().manual_seed(7))
        steps = []
        for _ in range(2):
            before = [p.detach().clone() for p in model.parameters()]
            momenta = [trainer.optimizer.state[p]['momentum_buffer'].clone() if p.dim() > 1 else None for p in model.parameters()]
            if flat:
                trainer.grads.zero()
                trainer._backward(trainer.total_loss(trainer.model(shard_batch(x, rank, world))))
                trainer.grads.pack_all()
                trainer.grads.all_reduce_flat()
                trainer.optimizer.step()
            else:
                trainer.step(shard_batch(x, rank, world))
            steps.append((before, [p.grad.clone() for p in model.parameters()], momenta, [p.detach().clone() for p in model.parameters()]))
        torch.save(steps, '%s.%d' % (out_path, rank))
    dist.barrier()
    dist.destroy_process_group()


@pytest.mark.parametrize('flat', [False, True])
def test_two_ranks_step_alike(tmp_path, flat):
    """Both ranks hold the same weights after every step, the gradients are those of the whole batch, and the weights move as the formula has it."""
    import socket
    import torch.multiprocessing as mp
    import hostexec
    import train_on_host
    from oracle import ref_cpu as R
    from unopticalflow_amd.core.config import generate_loss_weights_dict
    if hostexec.library() is None or train_on_host.library() is None:
        pytest.skip('needs the ROCm clang++')
    with socket.socket() as so:
        so.bind(('127.0.0.1', 0))
        port = so.getsockname()[1]
    out = str(tmp_path / 'rank')
    mp.spawn(_muon_rank, args=(2, port, flat, out), nprocs=2, join=True)
    ranks = [torch.load('%s.%d' % (out, r)) for r in range(2)]
    weights = generate_loss_weights_dict(R.default_cfg())
    x = torch.randn(4, 3, 8, 8, generator=torch.Generator().manual_seed(7))
    torch.manual_seed(0)
    model = _Net().double()
    for a, b in zip(*ranks):
        assert all(torch.equal(p, q) for p, q in zip(a[0] + a[1] + a[3], b[0] + b[1] + b[3]))
        before, grads, momenta, after = a
        with torch.no_grad():
            for p, v in zip(model.parameters(), before):
                p.copy_(v)
        loss = sum(weights[k] * v.mean() for k, v in model(x.double()).items())
        for p, old, g, exact, m, new in zip(model.parameters(), before, grads, torch.autograd.grad(loss, list(model.parameters())), momenta, after):
            # (fp32 sums of at most 4 x 36 x 27 terms of a gradient, and the network around them)
            assert float((g.double() - exact).norm()) <= 2**-24 * 200 * float(exact.norm())
            if p.dim() < 2:
                assert not torch.equal(old, new)
                continue
            want, _ = _muon(old, g, m, 0.05, 0.95, 0.0, True)
            plain, _ = _muon(old, g, m, 0.05, 0.95, 0.0, True, torch.float32)
            step = 0.05 * max(1.0, len(p) / (p.numel() / len(p))) ** 0.5 * p.numel() ** 0.5 * 1.3
            assert float((new.double() - want).norm()) <= 4 * float((plain.double() - want).norm()) + 16 * 2**-22 * step + 5 * 2**-24 * float(want.norm())


YAML = """cfg_name: 'default'
dataset: 'kitti_depth'
img_hw: [64, 128]
num_scales: 3
num_iterations: 4
w_ssim: 0.85
w_flow_smooth: 10.0
w_flow_consis: 0.01
h_flow_consist_alpha: 3.0
h_flow_consist_beta: 0.05
prepared_base_dir: './none'
gt_2012_dir: './none'
gt_2015_dir: './none'
"""


@pytest.mark.parametrize('given,want', [([], ('adam', 0.002, 1e-4)), (['--optimizer', 'muon'], ('muon', 0.002, 1e-4)),
                                        (['--optimizer', 'muon', '--muon_lr', '0.01', '--lr', '0.5'], ('muon', 0.01, 0.5))])
def test_the_train_command_passes_its_optimiser_on(tmp_path, monkeypatch, given, want):
    """What reaches FlowTrainer from the command line."""
    from unopticalflow_amd import train as cli, tuning
    seen = {}

    class Reached(Exception):
        pass

    def trainer(cfg, model, **kw):
        seen.update(kw, lr=cfg.lr)
        raise Reached
    for name, value in (('is_available', lambda: True), ('device_count', lambda: 1), ('set_device', lambda d: None)):
        monkeypatch.setattr(torch.cuda, name, value)
    monkeypatch.setattr(tuning, 'default_channels_last', lambda: 0)
    monkeypatch.setattr(cli, 'init_distributed', lambda *a, **k: (0, 0, 1))
    monkeypatch.setattr(cli, 'get_model', lambda mode: lambda cfg: type('Model', (), {'to': lambda self, dev: self})())
    monkeypatch.setattr(cli, 'FlowTrainer', trainer)
    monkeypatch.chdir(tmp_path)
    (tmp_path / 'cfg.yaml').write_text(YAML)
    with pytest.raises(Reached):
        cli.main(['-c', 'cfg.yaml', '--synthetic', '--no_test', '--miopen_find', '0'] + given)
    assert (seen['optimizer'], seen['muon_lr'], seen['lr']) == want
    with pytest.raises(SystemExit):
        cli.main(['-c', 'cfg.yaml', '--optimizer', 'sgd'])


@pytest.mark.gpu
@pytest.mark.parametrize('graph', ['0', '1'])
def test_the_train_command_with_muon(tmp_path, monkeypatch, graph):
    """Four iterations on synthetic triplets, checkpoints, and the last two again from the one in the middle; an Adam checkpoint is refused."""
    from unopticalflow_amd import train as cli
    monkeypatch.chdir(tmp_path)
    (tmp_path / 'cfg.yaml').write_text(YAML)
    common = ['-c', 'cfg.yaml', '--synthetic', '--no_test', '--miopen_find', '0', '--batch_size', '2', '--log_interval', '1', '--save_interval', '2', '--graph', graph]
    muon = common + ['--optimizer', 'muon', '--model_dir', 'muon']
    trainer = cli.main(muon)
    assert type(trainer.optimizer) is optim.FlowMuon and trainer.iteration == 3
    again = cli.main(muon + ['--resume', '--iter_start', '1'])
    assert all(bool(torch.isfinite(p).all()) for p in again.model.parameters())
    momenta = [again.optimizer.state[p]['momentum_buffer'] for p in again.model.parameters() if p.dim() > 1]
    assert len(momenta) == 49 and all(m.dtype == torch.float32 and bool(m.any()) for m in momenta)
    cli.main(common + ['--model_dir', 'adam', '--num_iterations', '2'])
    with pytest.raises(ValueError):
        cli.main(common + ['--optimizer', 'muon', '--model_dir', 'adam', '--resume', '--iter_start', '1'])


@pytest.mark.parametrize('rows,dim', [(20, 24), (64, 24), (65, 24), (100, 200), (20, 3)])
@pytest.mark.parametrize('outlier', [2.0**10, 2.0**23, 2.0**30])
def test_columns_far_larger_than_the_rest(device, rows, dim, outlier):
    """fp32 rows with one number `outlier` times the others, whose weight is as much smaller.  Up to 64 rows (of 4 numbers and more) fp32 products;
    beyond, a number x of a row whose largest is M is held to 2^-22 |x| + 2^-39 M, so that a logit is off by what test_train_ops.py derives and
    2^-39 (M_h sum |w| + M_w sum |h|) on top."""
    h, w, t = _inputs(rows, 50, dim, torch.float32, device, ignored=0.0)
    h[:, 1] *= outlier
    w[:, 1] /= outlier
    losses = ops.linear_cross_entropy(h, w, t, reduction='none').double()
    hd, wd = h.double(), w.double()
    z = hd @ wd.T
    exact = z.logsumexp(1) - z.gather(1, t[:, None])[:, 0]
    dz = (dim * 2**-24 + 2**-20) * float((hd.abs() @ wd.abs().T).max())
    if rows > 64 or dim < 4:
        dz += 2**-39 * float((hd.abs().amax(1)[:, None] * wd.abs().sum(1)[None] + hd.abs().sum(1)[:, None] * wd.abs().amax(1)[None]).max())
    assert bool(((losses - exact).abs() <= 2 * dz + (2 * float(z.abs().max()) + 128) * 2**-23).all())
