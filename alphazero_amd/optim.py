"""Optimisers whose whole update is one launch: FlatSGD, and FlatAdamW further down.

FlatSGD: torch.optim.SGD as the reference configures it (alphazero/training.py:27-29: momentum, weight
decay) with the whole update in ONE launch of az_sgd_momentum (csrc/az_train.hip).

All parameters are moved into one flat fp32 buffer (each parameter becomes a view of it, channels last where it was,
so the module, its state_dict and everything that reads the weights keep working), gradients accumulate into a second flat buffer
through persistent `.grad` views, and the momentum is a third.  A step is then a single kernel over n elements
instead of three small launches per tensor.  It is a torch Optimizer, so MultiStepLR drives its learning rate
exactly as it drives SGD's (training.py:30-31)."""
import ctypes as C

import torch

from . import _lib


def _strided_like(flat, p):
    """`flat` (p.numel() elements) in the shape of p, in p's order of memory where that is dense."""
    if p.dim() == 4 and not p.is_contiguous() and p.is_contiguous(memory_format=torch.channels_last):
        return flat.as_strided(p.shape, p.stride(), flat.storage_offset())
    return flat.view(p.shape)


class FlatSGD(torch.optim.Optimizer):
    def __init__(self, params, lr, momentum=0.0, weight_decay=0.0):
        params = [p for p in params]
        seen, uniq = set(), []
        for p in params:                                   # the tower repeats one block: each tensor once
            if id(p) not in seen:
                seen.add(id(p))
                uniq.append(p)
        super().__init__(uniq, dict(lr=lr, momentum=momentum, weight_decay=weight_decay))
        dev = uniq[0].device
        if dev.type != 'cuda':
            raise _lib.AzError('FlatSGD runs on the GPU (az_sgd_momentum); use torch.optim.SGD for CPU tensors')
        assert all(p.device == dev and p.dtype == torch.float32 for p in uniq)
        self.lib = _lib.load()
        self.device = dev
        n = sum(p.numel() for p in uniq)
        self.flat_p = torch.empty(n, dtype=torch.float32, device=dev)
        self.flat_g = torch.zeros(n, dtype=torch.float32, device=dev)
        self.flat_m = torch.zeros(n, dtype=torch.float32, device=dev)
        off = 0
        with torch.no_grad():
            for p in uniq:
                k = p.numel()
                at_p = _strided_like(self.flat_p[off:off + k], p)
                at_p.copy_(p)
                p.grad = _strided_like(self.flat_g[off:off + k], p)
                p.data = at_p
                off += k
        self._steps = 0
        self.withheld = torch.zeros(1, dtype=torch.int32, device=dev)   # recorded steps whose update the guard refused
        self._lr_dev = None                                # learning rate in device memory, for recorded steps

    def zero_grad(self, set_to_none=False):
        self.flat_g.zero_()                                # the .grad views stay in place

    @torch.no_grad()
    def step(self, closure=None):
        g = self.param_groups[0]
        with torch.cuda.device(self.device):
            st = C.c_void_p(torch.cuda.current_stream(self.device).cuda_stream)
            _lib.check(self.lib.az_sgd_momentum(_lib.ptr(self.flat_p), _lib.ptr(self.flat_g), _lib.ptr(self.flat_m),
                                                self.flat_p.numel(), float(g['lr']), float(g['momentum']),
                                                float(g['weight_decay']), int(self._steps == 0), st))
        self._steps += 1

    def set_recorded_lr(self):
        """Puts the current learning rate where step_recorded's kernel reads it (a copy only when it changed)."""
        lr = float(self.param_groups[0]['lr'])
        if self._lr_dev is None:
            self._lr_dev = torch.empty(1, dtype=torch.float32, device=self.device)
            self._lr_host = None
        if self._lr_host != lr:
            self._lr_dev.fill_(lr)
            self._lr_host = lr

    @torch.no_grad()
    def step_recorded(self, guard=None, guard_limit=1e-6):
        """The same update with the learning rate read from device memory at run time (az_sgd_momentum_lr_dev):
        the launch can be captured in a HIP graph and replayed while a scheduler changes the rate.  Call
        set_recorded_lr() (outside the capture) before every run.
        guard: a one-element float32 device tensor written earlier in the same recorded sequence; the update is
        applied only while guard < guard_limit (az_sgd_momentum_guarded), otherwise nothing changes and
        self.withheld (device int32[1]) counts the step."""
        g = self.param_groups[0]
        assert self._lr_dev is not None, 'set_recorded_lr() first'
        with torch.cuda.device(self.device):
            st = C.c_void_p(torch.cuda.current_stream(self.device).cuda_stream)
            if guard is None:
                _lib.check(self.lib.az_sgd_momentum_lr_dev(_lib.ptr(self.flat_p), _lib.ptr(self.flat_g), _lib.ptr(self.flat_m),
                                                           self.flat_p.numel(), _lib.ptr(self._lr_dev), float(g['momentum']),
                                                           float(g['weight_decay']), st))
            else:
                assert guard.dtype == torch.float32 and guard.numel() == 1 and guard.device == self.device
                _lib.check(self.lib.az_sgd_momentum_guarded(_lib.ptr(self.flat_p), _lib.ptr(self.flat_g), _lib.ptr(self.flat_m),
                                                            self.flat_p.numel(), _lib.ptr(self._lr_dev), float(g['momentum']),
                                                            float(g['weight_decay']), _lib.ptr(guard), float(guard_limit),
                                                            _lib.ptr(self.withheld), st))
        self._steps += 1


class FlatAdamW(torch.optim.Optimizer):
    """torch.optim.AdamW (decoupled weight decay, bias correction; no amsgrad) with the whole update of all parameter
    groups in ONE launch of az_adamw_step (csrc/az_adamw.hip), beside FlatSGD.  With eps=0 an element that has had no
    gradient but zero has no update (torch's is 0 / 0).

    All parameters that require gradients at construction move into one flat buffer (each becomes a view of it, padded to 256
    elements), gradients accumulate into a second through persistent `.grad` views (use this class's zero_grad; a
    gradient that was replaced by another tensor is copied back into its view).  Parameters are float32, or bfloat16
    with a float32 master copy that the update works on (weights written between two steps, as by
    load_state_dict of the module, replace their masters).

    state_bits=8 keeps the two moments in one byte per element each: a float with 3 bits of mantissa relative to the
    largest of its block of 256, rounded at random by a function of (seed, step, element), so that the moments' small
    steps are kept in expectation; 12 bytes less traffic and 6 bytes less memory per parameter.  Ranks that hold the
    same weights give the same seed and stay bit-identical.

    Beside the step's own traffic a training loop pays for the views: zero_grad fills the gradients and autograd adds into
    them, some 16 bytes an element.  In a network of both types every flat buffer spans all parameters: 4 bytes of
    `flat_g` for each bfloat16 one, 4 of `flat_p16` and `flat_g16` for each float32 one, are never used.

    step() may be captured; in a launch that is replayed while a scheduler changes the rate use step_recorded(), as
    with FlatSGD.  The step count lives in device memory (`steps` reads it).  state_dict() is torch.optim.AdamW's
    (exp_avg and exp_avg_sq as the float32 values that the codes stand for, `master` for bfloat16 parameters) and
    load_state_dict() takes either's, whatever state_bits it was written with.  Parameter groups are fixed at
    construction."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, seed=0):
        if state_bits not in (8, 32):
            raise ValueError(f'state_bits is 8 or 32, got {state_bits!r}')
        self._bound = False
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))
        self.state_bits, self.seed = state_bits, int(seed) & (2 ** 64 - 1)
        for g in self.param_groups:
            self._check_group(g)
        order = []                                         # (group index, bfloat16?, parameter), run by run
        for k, g in enumerate(self.param_groups):
            for half in (False, True):
                order += [(k, half, p) for p in g['params'] if p.requires_grad and (p.dtype == torch.bfloat16) == half]
        if not order:
            raise ValueError('no parameter requires a gradient')
        if len({id(p) for _, _, p in order}) < len(order):
            raise ValueError('a parameter is given twice')
        dev = order[0][2].device
        if dev.type != 'cuda':
            raise _lib.AzError('FlatAdamW runs on the GPU (az_adamw_step); use torch.optim.AdamW for CPU tensors')
        for _, _, p in order:
            if p.device != dev or p.dtype not in (torch.float32, torch.bfloat16) or p.layout != torch.strided:
                raise ValueError(f'FlatAdamW takes dense float32 or bfloat16 parameters on one device, got {p.dtype} on {p.device}')
        self.lib, self.device = _lib.load(), dev           # (a parameter's device has its index)
        self._runs, self._places, block = [], [], 0
        for k, half, p in order:
            if not self._runs or (self._runs[-1][0], self._runs[-1][1]) != (k, half):
                self._runs.append((k, half, block))
            self._places.append((p, block * _lib.ADAMW_BLOCK))
            block += -(-p.numel() // _lib.ADAMW_BLOCK)
        if len(self._runs) > _lib.ADAMW_MAX_RUNS:
            raise ValueError(f'at most {_lib.ADAMW_MAX_RUNS} parameter groups (one of mixed types counts twice), got {len(self._runs)}')
        if block == 0:
            raise ValueError('the parameters have no elements')
        self._blocks, n = block, block * _lib.ADAMW_BLOCK
        wide, half = (any(r[1] == h for r in self._runs) for h in (False, True))
        zeros = lambda dtype, size=n: torch.zeros(size, dtype=dtype, device=dev)
        self.flat_p = zeros(torch.float32)
        self.flat_g = zeros(torch.float32) if wide else None
        self.flat_p16 = zeros(torch.bfloat16) if half else None
        self.flat_g16 = zeros(torch.bfloat16) if half else None
        self.flat_m = self.flat_v = self.codes_m = self.codes_v = self.tops = None
        if state_bits == 32:
            self.flat_m, self.flat_v = zeros(torch.float32), zeros(torch.float32)
        else:
            self.codes_m, self.codes_v = zeros(torch.uint8), zeros(torch.uint8)
            self.tops = zeros(torch.int16, 2 * block)
        self._step_dev = zeros(torch.int64, _lib.ADAMW_STEPS)   # a counter for each workgroup, all equal
        self.withheld = zeros(torch.int32, 1)              # recorded steps whose update the guard refused
        self._lr_dev, self._lr_host = None, None
        self._grads = []
        with torch.no_grad():
            for p, at in self._places:
                is16 = p.dtype == torch.bfloat16
                at_p = self._cut(self.flat_p, p, at)
                at_p.copy_(p)
                if is16:
                    at_p = self._cut(self.flat_p16, p, at)
                    at_p.copy_(p)
                grad = self._cut(self.flat_g16 if is16 else self.flat_g, p, at)
                if p.grad is not None:
                    grad.copy_(p.grad)
                p.data = at_p
                p.grad = grad
                self._grads.append(grad)
        self._addresses = [p.data_ptr() for p, _ in self._places]
        self._still = _lib.autograd().Places([p for p, _ in self._places], self._grads)
        b = _lib.AdamWBuffers()
        for name, t in (('p', self.flat_p), ('g', self.flat_g), ('p16', self.flat_p16), ('g16', self.flat_g16), ('m', self.flat_m),
                        ('v', self.flat_v), ('m8', self.codes_m), ('v8', self.codes_v), ('top', self.tops),
                        ('step', self._step_dev)):
            setattr(b, name, None if t is None else t.data_ptr())
        self._buffers = b
        self._args, self._settings = (_lib.AdamWRun * len(self._runs))(), None
        for a, (k, is16, first) in zip(self._args, self._runs):
            a.first_block, a.half, a.lr_index = first, int(is16), k
        self._bound = True

    @staticmethod
    def _check_group(g):
        b1, b2 = g['betas']
        if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
            raise ValueError(f'betas lie in [0, 1), got {g["betas"]}')
        if not (g['lr'] >= 0.0 and g['eps'] >= 0.0 and g['weight_decay'] >= 0.0):
            raise ValueError('lr, eps and weight_decay are not negative')
        if g.get('amsgrad') or g.get('maximize'):
            raise ValueError('FlatAdamW has no amsgrad and no maximize')

    @staticmethod
    def _cut(flat, p, at):
        return _strided_like(flat[at:at + p.numel()], p)

    def add_param_group(self, param_group):
        if self._bound:
            raise ValueError('the parameter groups of FlatAdamW are fixed at construction')
        super().add_param_group(param_group)

    @property
    def steps(self):
        """Updates applied so far (waits for the device)."""
        return int(self._step_dev[0].item())

    def zero_grad(self, set_to_none=False):
        for flat in (self.flat_g, self.flat_g16):          # the .grad views stay in place
            if flat is not None:
                flat.zero_()
        for (p, _), grad in zip(self._places, self._grads):
            if p.grad is not grad:
                p.grad = grad

    def _rebind(self):
        if self._still.in_place():
            return
        if [p.data_ptr() for p, _ in self._places] != self._addresses:
            raise _lib.AzError('a parameter of FlatAdamW was moved out of the flat buffer (module.to(), p.data = ...): move the '
                               'module first, then construct the optimizer')
        for (p, _), grad in zip(self._places, self._grads):
            if p.grad is not grad:
                if p.grad is None:
                    raise _lib.AzError('a parameter of FlatAdamW has no gradient: use its own zero_grad(), which keeps the '
                                       'gradients in place')
                with torch.no_grad():
                    grad.copy_(p.grad)
                p.grad = grad

    def _launch(self, lr_dev, guard, guard_limit):
        # (as numbers: a rate in a tensor, betas in a list may be changed in place)
        settings = [(float(g['lr']), *map(float, g['betas']), float(g['eps']), float(g['weight_decay'])) for g in self.param_groups]
        for a, (k, _, _) in zip(self._args, self._runs) if settings != self._settings else ():
            a.lr, a.beta1, a.beta2, a.eps, a.weight_decay = settings[k]
        self._settings = settings
        _lib.launch(self.device, self.lib.az_adamw_step, self._buffers, self._blocks, self._args, len(self._runs), self.state_bits,
                    _lib.ptr(lr_dev), self.seed, _lib.ptr(guard), guard_limit, self.withheld.data_ptr())

    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        self._rebind()
        self._launch(None, None, 0.0)
        return loss

    def set_recorded_lr(self):
        """Puts the current learning rates where step_recorded's kernel reads them (a write only where one changed)."""
        rates = [float(g['lr']) for g in self.param_groups]
        if self._lr_dev is None:
            self._lr_dev = torch.empty(_lib.ADAMW_MAX_RUNS, dtype=torch.float64, device=self.device)
            self._lr_host = [None] * len(rates)
        for k, lr in enumerate(rates):
            if self._lr_host[k] != lr:
                self._lr_dev[k].fill_(lr)
        self._lr_host = rates

    def step_recorded(self, guard=None, guard_limit=1e-6):
        """The same update with the learning rates read from device memory at run time, for launches captured in a HIP
        graph; the other settings are those of the capture.  Call set_recorded_lr() (outside the capture) before every
        run.  guard, guard_limit: as FlatSGD.step_recorded; a withheld step does not count."""
        assert self._lr_dev is not None, 'set_recorded_lr() first'
        if guard is not None:
            assert guard.dtype == torch.float32 and guard.numel() == 1 and guard.device == self.device
        self._rebind()
        self._launch(self._lr_dev, guard, guard_limit)

    @torch.no_grad()
    def state_values(self):
        """(exp_avg, exp_avg_sq) of all parameters as float32 in the layout of `flat_p`; with state_bits=8 the values
        that the codes stand for, in new tensors."""
        if self.state_bits == 32:
            return self.flat_m, self.flat_v
        m, v = torch.empty_like(self.flat_p), torch.empty_like(self.flat_p)
        _lib.launch(self.device, self.lib.az_adamw_decode8, self.codes_m.data_ptr(), self.codes_v.data_ptr(), self.tops.data_ptr(),
                    self._blocks, m.data_ptr(), v.data_ptr())
        return m, v

    def state_dict(self):
        packed = super().state_dict()
        number = {id(p): i for i, p in enumerate(p for g in self.param_groups for p in g['params'])}
        m, v = self.state_values()
        steps = float(self.steps)
        packed['state'] = {}
        for p, at in self._places:
            s = dict(step=torch.tensor(steps, dtype=torch.float64), exp_avg=self._cut(m, p, at).clone(), exp_avg_sq=self._cut(v, p, at).clone())
            if p.dtype == torch.bfloat16:
                s['master'] = self._cut(self.flat_p, p, at).clone()
            packed['state'][number[id(p)]] = s
        return packed

    @torch.no_grad()
    def load_state_dict(self, state_dict):
        state = state_dict['state']
        number = {id(p): i for i, p in enumerate(p for g in self.param_groups for p in g['params'])}
        entries = [state.get(number[id(p)]) for p, _ in self._places]
        if any(e is None for e in entries) and any(e is not None for e in entries):
            raise ValueError('the state holds moments for some of the parameters only')
        steps = {int(e['step']) for e in entries if e is not None} or {0}
        if len(steps) > 1:
            raise ValueError(f'the parameters have taken different numbers of steps: {sorted(steps)}')
        for (p, _), e in zip(self._places, entries):
            if e is not None and (e['exp_avg'].shape != p.shape or e['exp_avg_sq'].shape != p.shape):
                raise ValueError(f'moments of shape {tuple(e["exp_avg"].shape)} for a parameter of shape {tuple(p.shape)}')
        for g in state_dict['param_groups']:
            self._check_group(g)
        super().load_state_dict(dict(state_dict, state={}))
        m, v = (self.flat_m, self.flat_v) if self.state_bits == 32 else (torch.zeros_like(self.flat_p), torch.zeros_like(self.flat_p))
        m.zero_()
        v.zero_()
        for (p, at), e in zip(self._places, entries):
            if e is not None:
                self._cut(m, p, at).copy_(e['exp_avg'])
                self._cut(v, p, at).copy_(e['exp_avg_sq'])
            if p.dtype == torch.bfloat16:
                self._cut(self.flat_p, p, at).copy_(p if e is None or 'master' not in e else e['master'])
        if self.state_bits == 8:
            _lib.launch(self.device, self.lib.az_adamw_encode8, m.data_ptr(), v.data_ptr(), self._blocks, self.codes_m.data_ptr(),
                        self.codes_v.data_ptr(), self.tops.data_ptr())
        self._step_dev.fill_(steps.pop())
