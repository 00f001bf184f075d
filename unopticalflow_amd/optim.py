"""Adam for the flow step: ``torch.optim.Adam`` (the reference's optimizer, train.py:39: default betas / eps, lr from the
command line) whose ``step`` is ONE HIP launch over all parameter tensors (csrc/optim.hip, ``unflow_adam_multi``).

Same class hierarchy, same ``state`` layout and ``state_dict`` as torch's capturable Adam (``step`` a float32 device scalar,
``exp_avg``, ``exp_avg_sq`` per parameter), so checkpoints interchange with ``torch.optim.Adam`` and with the reference's
``optimizer_state_dict`` (train.py:23-31).  The step counters are views of one device vector that the kernel advances, so the
optimizer can sit inside a captured hipGraph.  Anything the kernel does not take -- a CPU parameter, a parameter without a gradient,
a gradient whose layout differs from its parameter's, amsgrad / weight decay / maximize -- goes through ``torch.optim.Adam.step``.
"""
import ctypes

import torch

from . import _lib, ops


class _Slot(ctypes.Structure):
    _fields_ = [('p', ctypes.c_void_p), ('m', ctypes.c_void_p), ('v', ctypes.c_void_p), ('numel', ctypes.c_longlong)]


def _dense_like(a, b):
    return a.shape == b.shape and a.stride() == b.stride() and a.dtype == b.dtype and a.device == b.device


def _dense(t):
    """Every element of the storage span exactly once (row-major, channels_last or any permutation of them): the kernel walks
    numel() consecutive floats from data_ptr()."""
    n = 1
    for size, stride in sorted(zip(t.shape, t.stride()), key=lambda ss: ss[1]):
        if size == 1:
            continue
        if stride != n:
            return False
        n *= size
    return True


class FlowAdam(torch.optim.Adam):
    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8):
        super().__init__(params, lr=lr, betas=betas, eps=eps, capturable=True)
        self._tables = None                # (device slots, device chunk map, nchunks, key) of the current state tensors
        self._steps = None                 # one float per parameter; state[p]['step'] are its 0-dim views
        self.native_steps = 0              # steps taken by the HIP kernel (tests / diagnostics)

    # ---- state
    def _params(self):
        return [p for g in self.param_groups for p in g['params']]

    def _init_state(self, params):
        dev = params[0].device
        if self._steps is None or self._steps.numel() != len(params) or self._steps.device != dev:
            self._steps = torch.zeros(len(params), dtype=torch.float32, device=dev)
        for i, p in enumerate(params):
            st = self.state[p]
            if len(st) == 0:
                st['step'] = self._steps[i]
                st['exp_avg'] = torch.zeros_like(p, memory_format=torch.preserve_format)
                st['exp_avg_sq'] = torch.zeros_like(p, memory_format=torch.preserve_format)
            elif not torch.is_tensor(st['step']) or st['step'].data_ptr() != self._steps[i].data_ptr():
                # counters that came from a checkpoint (fresh tensors; plain ints in a torch-1.2 file of the reference) or from
                # torch's own step: tie them to the vector the kernel advances
                self._steps[i].copy_(torch.as_tensor(st['step'], dtype=torch.float32))
                st['step'] = self._steps[i]

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)
        self._tables = None                # new moment tensors: rebuild the device table at the next step

    def _build_tables(self, params):
        key = tuple((p.data_ptr(), self.state[p]['exp_avg'].data_ptr(), self.state[p]['exp_avg_sq'].data_ptr()) for p in params)
        if self._tables is not None and self._tables[3] == key:
            return self._tables
        chunk = _lib.load().unflow_adam_chunk()
        slots = (_Slot * len(params))()
        cmap = []
        for i, p in enumerate(params):
            st = self.state[p]
            slots[i] = _Slot(p.data_ptr(), st['exp_avg'].data_ptr(), st['exp_avg_sq'].data_ptr(), p.numel())
            cmap += [(i, c) for c in range((p.numel() + chunk - 1) // chunk)]
        dev = params[0].device
        raw = torch.frombuffer(bytearray(bytes(slots)), dtype=torch.uint8).to(dev)
        cm = torch.tensor(cmap, dtype=torch.int32).reshape(-1).to(dev)
        self._tables = (raw, cm, len(cmap), key)
        return self._tables

    def prepare(self):
        """Create everything a native step needs -- moments, the step vector, the device tables -- for ALL parameters now, whether
        or not they have a gradient yet.  A trainer calls it before it captures ``step()`` into a hipGraph: allocations, zero-fills
        and host-to-device copies made DURING a capture would become graph nodes (every replay would reset the moments and the
        step counters) or fail the capture outright."""
        params = self._params()
        if not params or not all(ops.on_device(p) and p.dtype == torch.float32 for p in params) or len(params) > 128:
            return False
        self._init_state(params)
        self._build_tables(params)
        return True

    def _capture_ready(self, params):
        if self._steps is None or self._steps.numel() != len(params) or self._tables is None:
            return False
        for i, p in enumerate(params):
            st = self.state.get(p)
            if not st or not torch.is_tensor(st.get('step')) or st['step'].data_ptr() != self._steps[i].data_ptr():
                return False
        return self._tables[3] == tuple((p.data_ptr(), self.state[p]['exp_avg'].data_ptr(), self.state[p]['exp_avg_sq'].data_ptr()) for p in params)

    def _native_ok(self, params):
        if not params or len(params) > 128:
            return False
        g = self.param_groups
        if len(g) != 1 or g[0].get('amsgrad') or g[0].get('weight_decay') or g[0].get('maximize') or g[0].get('differentiable'):
            return False
        if torch.is_tensor(g[0]['lr']):
            return False
        dev = params[0].device
        for p in params:
            if not ops.on_device(p) or p.device != dev or p.dtype != torch.float32 or p.grad is None or p.grad.is_sparse:
                return False
            if not _dense_like(p.grad, p) or not _dense(p):
                return False
        return True

    @torch.no_grad()
    def step(self, closure=None):
        params = self._params()
        capturing = bool(params) and params[0].is_cuda and torch.cuda.is_current_stream_capturing()
        if closure is not None or not self._native_ok(params):
            if capturing and self.native_steps > 0:
                # torch's Adam under capture next to native steps outside it would walk two sets of step counters (a model with a
                # parameter the loss never reaches takes torch's Adam in the warm-up AND in the capture: consistent, allowed)
                raise RuntimeError('FlowAdam.step() inside a hipGraph capture would fall back to torch.optim.Adam (a parameter without a '
                                   'gradient, or a layout the kernel does not take) after native steps: give the warm-up steps the '
                                   'gradient view of the capture')
            if self._steps is not None:
                self._tables = None
            return super().step(closure)
        if capturing and not self._capture_ready(params):
            raise RuntimeError('FlowAdam.step() inside a hipGraph capture would have to allocate its state (moments, step vector, device '
                               'tables): call FlowAdam.prepare() -- or take one step with the same gradients -- before the capture')
        self._init_state(params)
        for p in params:                   # the moments walk the parameter's memory: same dense layout (trainer.relayout_optimizer_state)
            st = self.state[p]
            if not (_dense_like(st['exp_avg'], p) and _dense_like(st['exp_avg_sq'], p)):
                return super().step(closure)
        slots, cmap, nchunks, _ = self._build_tables(params)
        grads = (ctypes.c_void_p * len(params))(*[p.grad.data_ptr() for p in params])
        g = self.param_groups[0]
        lib = _lib.load()
        with ops._on(params[0].device):
            rc = lib.unflow_adam_multi(ctypes.c_void_p(slots.data_ptr()), ctypes.c_void_p(cmap.data_ptr()), nchunks, grads, len(params),
                                       ctypes.c_void_p(self._steps.data_ptr()),
                                       ctypes.c_float(g['lr']), ctypes.c_float(g['betas'][0]), ctypes.c_float(g['betas'][1]),
                                       ctypes.c_float(g['eps']), ops._stream())
        _lib.check(rc, 'unflow_adam_multi')
        # (written through their addresses, which autograd does not see)
        torch.autograd.graph.increment_version(params + [self.state[p][k] for p in params for k in ('exp_avg', 'exp_avg_sq')])
        self.native_steps += 1
        return None


# ---- Muon: orthogonalised momentum for matrices
def _walks_as_matrix(t):
    """A dense tensor whose first dimension is the outermost one: [shape[0], the rest] in memory order (row-major, channels_last)."""
    return _dense(t) and (t.shape[0] == 1 or t.stride(0) == t.numel() // t.shape[0])


def _other_strides(a, b):
    return any(x != y and n > 1 for x, y, n in zip(a.stride(), b.stride(), b.shape))


def _check_apart(items, size):
    """Refuses weights whose parameters or momenta share memory with one another, or with another weight's gradient: the kernels work on all of them
    at once.  (A weight's own gradient may be its momentum or its parameter: whoever writes a number has read it.)  The library refuses the
    same, without a reason."""
    spans = []                                           # (first byte, byte behind the last, is written)
    for g, p, m, rows, cols in items:
        n = rows * cols
        spans += [(p, p + n * size, True), (m, m + 4 * n, True)]
        if g != p and (g != m or size != 4):
            spans.append((g, g + n * size, False))
    spans.sort()
    written = read = 0                                   # bytes behind what lies before
    for start, end, writes in spans:
        if start < written:
            raise ValueError('muon_step_: a parameter or momentum appears twice, or shares memory with another tensor of the step')
        if not writes:
            read = max(read, end)
        elif start < read:
            raise ValueError('muon_step_: a gradient shares memory with a parameter or momentum')
        else:
            written = end


@torch.no_grad()
def muon_step_(params, grads, momenta, lr, momentum=0.95, weight_decay=0.0, nesterov=True, steps=5, coefficients=(3.4445, -4.7750, 2.0315), eps=1e-7):
    """One Muon step over a list of weights, in place: every weight is a matrix [shape[0], the rest] (csrc/train/muon.hip, one launch per phase
    over all of them).

        m += (1 - momentum) (g - m);   u = g + momentum (m - g)   (nesterov; else m)
        p  = p (1 - lr weight_decay) - lr sqrt(max(1, rows / cols)) orthogonalize(u)

    ``params`` and ``grads`` are fp32, bf16 or fp16 (one type), ``momenta`` fp32 in their parameters' layout (row-major or channels_last;
    a gradient in another layout is copied).  No weight may appear twice, nor share memory with another."""
    ops._refuse_tracers('muon_step_')
    params, grads, momenta = list(params), list(grads), list(momenta)
    if not len(params) == len(grads) == len(momenta):
        raise ValueError('muon_step_: %d parameters, %d gradients, %d momenta' % (len(params), len(grads), len(momenta)))
    steps, coefficients = ops._check_newton_schulz('muon_step_', steps, coefficients, eps)
    keep = [i for i, p in enumerate(params) if p.numel()]
    if len(keep) < len(params):
        params, grads, momenta = ([v[i] for i in keep] for v in (params, grads, momenta))
    if not params:
        return
    copied = []                                    # (alive until the work on them is enqueued)
    dev, dtype = ops._dev_typed('muon_step_', *params, *grads)
    if {m.dtype for m in momenta} != {torch.float32} or {m.device for m in momenta} != {dev}:
        raise TypeError('muon_step_: momenta are fp32 on the parameters\' device')
    items = []
    for p, g, m in zip(params, grads, momenta):
        shape, stride = p.shape, p.stride()
        if len(shape) < 2 or g.shape != shape or m.shape != shape:
            raise ValueError('muon_step_: parameter, gradient and momentum must have one shape of two or more dimensions: {}, {}, {}'.format(
                tuple(shape), tuple(g.shape), tuple(m.shape)))
        rows, cols = shape[0], p.numel() // shape[0]
        if not (p.is_contiguous() or _walks_as_matrix(p)) or (m.stride() != stride and _other_strides(m, p)) or rows > ops._MATRIX_MAX_SIDE or cols > ops._MATRIX_MAX_SIDE:
            raise ValueError('muon_step_: a parameter must be dense with its first dimension outermost, its momentum of the same layout, sides up to {}; got shape {}, strides {} and {}'.format(
                ops._MATRIX_MAX_SIDE, tuple(shape), stride, m.stride()))
        if g.stride() != stride and _other_strides(g, p):
            g = torch.empty_like(p).copy_(g)
            copied.append(g)
        items.append((g.data_ptr(), p.data_ptr(), m.data_ptr(), rows, cols))
    try:
        ops._newton_schulz('unflow_muon_step', dev, dtype, (ops._Matrix * len(items))(*items), len(items),
                           (float(lr), float(momentum), float(weight_decay), int(bool(nesterov))), steps, coefficients, eps)
    except RuntimeError:
        _check_apart(items, params[0].element_size())
        raise
    torch.autograd.graph.increment_version(params + momenta)             # (written through their addresses, which autograd does not see)


class FlowMuon(torch.optim.Optimizer):
    """Muon for the weights of two or more dimensions (``muon_step_``), Adam (``FlowAdam``) for everything else.

    ``params`` is a list of parameters; it becomes two groups: 'matrices' (``lr``, ``momentum``, ``nesterov``, ``weight_decay``) and 'others'
    (``adam_lr`` as their ``lr``; betas and eps are FlowAdam's own).  Further groups (``add_param_group``) hold matrices.  Weights may be of
    different types (fp32, bf16, fp16): each type is a call of its own.  Momentum is kept in fp32 whatever the parameters' type.  Like FlowAdam it can be captured into a hipGraph once ``prepare()`` has created its state."""

    def __init__(self, params, lr=0.02, adam_lr=1e-4, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5, coefficients=(3.4445, -4.7750, 2.0315), eps=1e-7):
        params = [p for p in params]
        if not params or not all(torch.is_tensor(p) for p in params):
            raise ValueError('FlowMuon takes a non-empty list of parameters')
        ops._check_newton_schulz('FlowMuon', steps, coefficients, eps)
        matrices, others = [p for p in params if p.dim() >= 2], [p for p in params if p.dim() < 2]
        groups = [{'params': matrices, 'kind': 'matrices', 'lr': lr}] if matrices else []
        groups += [{'params': others, 'kind': 'others', 'lr': adam_lr}] if others else []
        super().__init__(groups, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, steps=steps, coefficients=tuple(coefficients), eps=eps))
        self._adam = FlowAdam(others, lr=adam_lr) if others else None
        self._share()

    def add_param_group(self, group):
        """Further groups hold matrices."""
        group = dict(group)
        params = group['params']
        if not isinstance(params, set):                                  # (which torch refuses: it has no order)
            group['params'] = [params] if torch.is_tensor(params) else list(params)                          # (it may be a generator)
        group.setdefault('kind', 'matrices')
        if group['kind'] != 'matrices' and hasattr(self, '_adam'):       # (the constructor's own group of others comes before)
            raise ValueError("FlowMuon: a further parameter group is of kind 'matrices', got %r" % (group['kind'],))
        if group['kind'] == 'matrices' and any(p.dim() < 2 for p in group['params'] if torch.is_tensor(p)):
            raise ValueError('FlowMuon: a further parameter group holds weights of two or more dimensions')
        for p in [p for p in group['params'] if torch.is_tensor(p) and p.requires_grad and group['kind'] == 'matrices']:
            if p.dtype not in ops._DTYPES:
                raise TypeError('FlowMuon takes fp32, bf16 or fp16 weights; got %s' % p.dtype)
            if p.numel() and max(p.shape[0], p.numel() // p.shape[0]) > ops._MATRIX_MAX_SIDE:
                raise ValueError('FlowMuon: weights are matrices [shape[0], the rest] of sides up to {}; got shape {}'.format(ops._MATRIX_MAX_SIDE, tuple(p.shape)))
        super().add_param_group(group)

    def _matrices(self):
        return [p for g in self.param_groups if g['kind'] == 'matrices' for p in g['params']]

    def _share(self):
        """One state for both: the inner Adam keeps its moments in this optimizer's ``state``."""
        if self._adam is not None:
            self._adam.state = self.state

    def _check_state(self, state_dict):
        """Refuses, before anything is replaced, a state that is not one of these parameters' and groups'."""
        groups = state_dict['param_groups']
        if [len(g['params']) for g in groups] != [len(g['params']) for g in self.param_groups]:
            return                                       # (Optimizer.load_state_dict says so)
        for given, own in zip(groups, self.param_groups):
            if given.get('kind') != own['kind']:
                raise ValueError("FlowMuon: a state whose parameter group is of kind %r, not %r" % (given.get('kind'), own['kind']))
            for i, p in zip(given['params'], own['params']):
                st = state_dict['state'].get(i)
                for key in () if not st else ('momentum_buffer',) if own['kind'] == 'matrices' else ('exp_avg', 'exp_avg_sq', 'step'):
                    v = st.get(key)
                    if v is None or (key != 'step' and (not torch.is_tensor(v) or v.shape != p.shape)):
                        raise ValueError('FlowMuon: a state without a %s for a parameter of shape %s' % (key, tuple(p.shape)))

    def load_state_dict(self, state_dict):
        self._check_state(state_dict)
        super().load_state_dict(state_dict)
        # (Optimizer.load_state_dict has cast the momentum to the parameter's type: taken again from what was given)
        for given, own in zip(state_dict['param_groups'], self.param_groups):
            for i, p in zip(given['params'], own['params']):
                if own['kind'] == 'matrices' and state_dict['state'].get(i):
                    self.state[p]['momentum_buffer'] = torch.empty_like(p, dtype=torch.float32).copy_(state_dict['state'][i]['momentum_buffer'])
        self._share()
        if self._adam is not None:
            self._adam._tables = None

    def _momentum(self, p):
        st = self.state[p]
        if 'momentum_buffer' not in st:
            if p.is_cuda and torch.cuda.is_current_stream_capturing():
                raise RuntimeError('FlowMuon.step() inside a hipGraph capture would have to create its state: call FlowMuon.prepare() before the capture')
            st['momentum_buffer'] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.preserve_format)
        return st['momentum_buffer']

    def prepare(self):
        """Create the state of all parameters now (before a capture)."""
        for p in self._matrices():
            self._momentum(p)
        return self._adam.prepare() if self._adam is not None else True

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for g in self.param_groups:
            if g['kind'] != 'matrices':
                continue
            alike = {}                                   # (a call takes weights of one type, on one device)
            for p in g['params']:
                if p.grad is not None:
                    alike.setdefault((p.dtype, p.device), []).append(p)
            for params in alike.values():
                muon_step_(params, [p.grad for p in params], [self._momentum(p) for p in params], lr=g['lr'], momentum=g['momentum'], weight_decay=g['weight_decay'],
                           nesterov=g['nesterov'], steps=g['steps'], coefficients=g['coefficients'], eps=g['eps'])
        if self._adam is not None:
            self._adam.param_groups[0]['lr'] = next(g['lr'] for g in self.param_groups if g['kind'] == 'others')
            self._adam.step()
        return loss
