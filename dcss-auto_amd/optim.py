"""AdamW over many tensors in a few launches, with moments in 32 or 8 bits (csrc/d1_optim.hip), and steps along
orthogonalised momenta for matrices (csrc/d1_muon.hip).

`Muon` is the torch optimizer of the latter, `muon_step` its step on lists of tensors, `orthogonalize` the
Newton-Schulz products alone. `AdamW` is the torch optimizer, `adamw_step` the step itself on lists of tensors, `read_moment` what
an 8-bit moment stands for. The step count, the global norm of a clip and the skip of a step whose
norm is not finite stay on the device, so a step can be captured in a HIP graph.
"""
import math

import torch

from .ops import call

BLOCK = 256                         # elements of an 8-bit moment that share an exponent


# options of the whole optimizer, which a group of parameters cannot have of its own
WHOLE = frozenset(('betas', 'eps', 'max_grad_norm', 'state_bits', 'seed', 'copies', 'amsgrad', 'maximize'))


def _check_group(group):
    if not WHOLE.isdisjoint(group):
        names = sorted(k for k in WHOLE.intersection(group) if group[k] or k not in ('amsgrad', 'maximize'))
        if names:
            raise ValueError(f'a group has lr and weight_decay of its own, not {", ".join(names)}')


def moment_blocks(numel):
    """Exponent bytes of an 8-bit moment of `numel` elements."""
    return -(-numel // BLOCK)


def _each(value, count):
    return [value] * count if isinstance(value, (int, float)) else value


def adamw_step(params, grads, exp_avg, exp_avg_sq, step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01,
               max_grad_norm=0.0, copies=None, exps=None, counters=None, seed=0, lags=None, other=None):
    """One AdamW step in place over lists of tensors.

    params: fp32 or bf16, contiguous. grads: fp32 or bf16 of the same sizes. exp_avg, exp_avg_sq:
    fp32 (32-bit moments), or uint8 codes with exps = (list of exp_avg's, list of exp_avg_sq's)
    exponents, uint8 of moment_blocks(numel) each, and counters: the first counter of each tensor's
    rounding draws, one an element (tensors whose ranges overlap round alike there). Zero codes
    and exponents are zero moments. step: int32 [8] on the device, zeros before the first step; [0]
    counts the steps made, [1] those skipped. copies: bf16 tensors that get the new fp32 parameters
    (None in the list: no copy). What the call changes gets a new version, as from torch's operations in
    place; the replay of a captured call cannot give it one. lr and weight_decay: one value or one for each tensor. lags: steps
    that each tensor has missed. other: the `step` of another step that has decided whether it is made and
    waits for this one (Muon.begin): both are made, or neither.

    With max_grad_norm > 0 the gradients are scaled by min(1, max_grad_norm / (norm + 1e-6)) with
    the norm over all of them, and a step whose norm is not finite changes nothing and is counted.
    Without, an element whose gradient (or its square) is not finite is lost alone; its 8-bit moments
    start anew, 32-bit ones stay not finite."""
    count = len(params)
    m_exps, v_exps = exps if exps is not None else (None, None)
    call('adamw_step', step, params, grads, exp_avg, exp_avg_sq, step, _each(lr, count), _each(weight_decay, count), betas[0],
         betas[1], eps, max_grad_norm, copies, m_exps, v_exps, counters, lags, seed & 0xFFFFFFFFFFFFFFFF, other)


def read_moment(code, exp, signed, out=None):
    """fp32 values of an 8-bit moment: uint8 codes and their exponents (signed: exp_avg's)."""
    return call('adamw_read', code, code, exp, bool(signed), out)


class AdamW(torch.optim.Optimizer):
    """AdamW on the device in a few launches for all tensors of all groups.

    lr and weight_decay may differ between groups; betas, eps, state_bits (32 or 8) and
    max_grad_norm (the clip by the global norm of all groups' gradients, 0 for none) are the
    optimizer's, and a group that names them is refused. copies: {parameter: bf16 tensor} that a step
    writes beside fp32 parameters. A parameter without a gradient is left as it is and keeps its own
    step count; the step in which it first takes part after others have, or does so again, waits for
    the device's count. A step can be captured in a graph after one with the same parameters taking
    part; replays use the lr, weight_decay, clip and seed of the capture, so a change of lr needs a
    new one. With max_grad_norm a step whose norm is not finite changes nothing; skipped_steps()
    counts those. The state dict holds moments and counts; betas, eps and the clip are those of the
    new optimizer."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, state_bits=32,
                 max_grad_norm=0.0, copies=None, seed=0):
        if state_bits not in (8, 32):
            raise ValueError('state_bits is 8 or 32')
        if not (lr >= 0 and weight_decay >= 0):
            raise ValueError('lr and weight_decay must not be negative')
        if not (0 <= betas[0] < 1 and 0 <= betas[1] < 1 and eps >= 0 and max_grad_norm >= 0):
            raise ValueError('betas must be in [0, 1), eps and max_grad_norm not negative')
        super().__init__(params, dict(lr=lr, weight_decay=weight_decay))
        self.betas, self.eps, self.state_bits, self.max_grad_norm, self.seed = betas, eps, state_bits, max_grad_norm, seed
        self.copies = copies or {}
        self.ctl = None                 # the device's step count, skips and norm (adamw_step's `step`)
        self._counter = 0

    def add_param_group(self, param_group):
        _check_group(param_group)
        super().add_param_group(param_group)

    def __getstate__(self):             # copies and pickles: the base class's holds no more than its own
        return {**super().__getstate__(), **{k: getattr(self, k) for k in (
            'betas', 'eps', 'state_bits', 'max_grad_norm', 'seed', 'copies', 'ctl', '_counter')}}

    @staticmethod
    def _not_captured():                # what a replay would do again, or not at all
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError('before a step is captured, make one with the same parameters taking part')

    def _state(self, p):
        s = self.state[p]
        if s:
            if s['left'] is not None:   # steps made since it last took part
                self._not_captured()
                s['lag'] += int(self.ctl[0]) - int(s['left'])
                s['left'] = None
        else:
            self._not_captured()
            s['lag'], s['left'], s['counter'] = 0 if self.ctl is None else int(self.ctl[0]), None, self._counter
            self._counter += moment_blocks(p.numel()) * BLOCK
            dtype = torch.uint8 if self.state_bits == 8 else torch.float32
            for name in ('exp_avg', 'exp_avg_sq'):
                s[name] = torch.zeros(p.shape, dtype=dtype, device=p.device)
                if self.state_bits == 8:
                    s[name + '_exp'] = torch.zeros(moment_blocks(p.numel()), dtype=torch.uint8, device=p.device)
        return s

    @torch.no_grad()
    def step(self, closure=None):
        for group in self.param_groups:
            _check_group(group)
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        self._step(None)
        return loss

    def _step(self, other):
        params, states, lr, decay = [], [], [], []
        for group in self.param_groups:
            for p in group['params']:
                if p.grad is not None:
                    params.append(p)
                    states.append(self._state(p))
                    lr.append(group['lr'])
                    decay.append(group['weight_decay'])
                elif self.state.get(p) and self.state[p]['left'] is None:
                    self._not_captured()
                    self.state[p]['left'] = self.ctl[:1].clone()
        if not params:
            return
        if self.ctl is None:
            self.ctl = torch.zeros(8, dtype=torch.int32, device=params[0].device)
        eight = self.state_bits == 8
        column = lambda name: [s[name] for s in states]  # noqa: E731
        adamw_step(params, [p.grad for p in params], column('exp_avg'), column('exp_avg_sq'), self.ctl, lr=lr,
                   betas=self.betas, eps=self.eps, weight_decay=decay, max_grad_norm=self.max_grad_norm,
                   copies=[self.copies.get(p) for p in params] if self.copies else None,
                   exps=(column('exp_avg_exp'), column('exp_avg_sq_exp')) if eight else None,
                   counters=column('counter') if eight else None, seed=self.seed,
                   lags=column('lag'), other=other)

    def skipped_steps(self):
        """Steps left out because the gradients' norm was not finite (waits for the device)."""
        return 0 if self.ctl is None else int(self.ctl[1].item())

    def grad_norm(self):
        """The last step's global gradient norm before the clip, fp32 on the device (max_grad_norm > 0)."""
        if self.ctl is None:
            raise RuntimeError('no step was made')
        return self.ctl[5:6].view(torch.float32)[0]

    def moments(self, p):
        """fp32 (exp_avg, exp_avg_sq) of a parameter."""
        s = self.state.get(p)
        if not s:
            raise ValueError('no step was made with this parameter')
        if self.state_bits == 32:
            return s['exp_avg'], s['exp_avg_sq']
        return (read_moment(s['exp_avg'], s['exp_avg_exp'], signed=True),
                read_moment(s['exp_avg_sq'], s['exp_avg_sq_exp'], signed=False))

    def state_dict(self):
        d = super().state_dict()
        d['d1'] = dict(state_bits=self.state_bits, ctl=None if self.ctl is None else self.ctl.clone(),
                       counter=self._counter, seed=self.seed)
        return d

    def load_state_dict(self, state_dict):
        own = state_dict.get('d1')
        if own is None:
            raise ValueError("not a state of this AdamW: another optimizer's moments and counts are kept otherwise")
        if own['state_bits'] != self.state_bits:
            raise ValueError(f"the state was saved with {own['state_bits']}-bit moments, this optimizer has {self.state_bits}")
        super().load_state_dict({k: v for k, v in state_dict.items() if k != 'd1'})
        # the base class casts tensors to the parameters' type: take the moments as they were saved
        saved = state_dict['state']
        ids = [i for group in state_dict['param_groups'] for i in group['params']]
        for i, p in zip(ids, (p for group in self.param_groups for p in group['params'])):
            for name, value in saved.get(i, {}).items():
                if torch.is_tensor(value):
                    self.state[p][name] = value.to(p.device, copy=True).contiguous()
        device = self.param_groups[0]['params'][0].device
        self.ctl = None if own['ctl'] is None else own['ctl'].to(device, copy=True)
        self._counter, self.seed = own['counter'], own['seed']


# the quintic a s + b s^3 + c s^5 that pulls singular values from (0, 1] to about 0.7 to 1.2 in five steps
NEWTON_SCHULZ = (3.4445, -4.7750, 2.0315)
_TERMS = {None: 0, 16: 1, 32: 3}


def _terms(product_bits):
    if product_bits not in _TERMS:
        raise ValueError('product_bits is None, 16 or 32')
    return _TERMS[product_bits]


def orthogonalize(updates, steps=5, coefficients=NEWTON_SCHULZ, eps=1e-7, product_bits=None):
    """The matrices with their singular values moved towards 1 by `steps` Newton-Schulz steps:

        X = U / (|U|_F + eps); then X = a X + (b A + c A A) X with A = X X^T (on the smaller side)

    updates: a tensor [..., rows, cols] or a list of such (they share launches), fp32, bf16 or fp16; the results are of the
    same types, contiguous. product_bits: operands of the products, 16 (fp16) or 32 (two fp16 halves, 22 bits, two to three times
    the time of large products); None: 32 for fp32 matrices and those with a side under 16, 16 for others (X, A and B are rounded to 11 bits in
    each step, which puts results 1e-3 to 3e-3 off as a whole, some of 20 x 20 by 5e-3; bf16's own last rounding is 1.6e-3). Accumulation is fp32. A matrix that is not finite gives NaN or what the formula
    gives. coefficients: singular values from [0, 1] have to stay under 3.8 through all steps."""
    a, b, c = coefficients
    alone = torch.is_tensor(updates)
    updates = [updates] if alone else list(updates)
    if not updates:
        return []
    out = call('orthogonalize', updates[0], updates, a, b, c, eps, steps, _terms(product_bits))
    return out[0] if alone else out


def muon_scale(shape, rms=False):
    """The factor of a matrix's step: sqrt(max(1, rows / cols)), or with `rms` 0.2 sqrt(max(rows, cols)), which
    gives an update the size of AdamW's."""
    rows, cols = shape[0], math.prod(shape[1:])
    return 0.2 * math.sqrt(max(rows, cols)) if rms else math.sqrt(max(1.0, rows / cols)) if cols else 1.0


def muon_step(params, grads, momenta, step, lr=0.02, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5,
              coefficients=NEWTON_SCHULZ, eps=1e-7, scales=None, copies=None, product_bits=None):
    """One step in place along the orthogonalised momenta of lists of matrices:

        m = momentum * m + g;  u = g + momentum * m (nesterov) or m;  p = p (1 - lr wd) - lr scale orthogonalize(u)

    params: fp32 or bf16, contiguous, of two dimensions or more (those behind the first count as one). grads: fp32 or bf16 of
    the same shapes. momenta: fp32. step: int32 [8] on the device, zeros before the first step; [0] counts the steps made,
    [1] those skipped: a step with a matrix whose u has no finite norm changes nothing else. scales: one for each matrix
    (None: muon_scale of its shape). copies: bf16 tensors that get the new fp32 parameters (None in the list: no copy).
    lr and weight_decay: one value or one for each matrix. product_bits: as in orthogonalize, None by the parameters' types and sides."""
    _muon(params, grads, momenta, step, lr, momentum, nesterov, weight_decay, steps, coefficients, eps, scales, copies, product_bits)


def _muon(params, grads, momenta, step, lr, momentum, nesterov, weight_decay, steps, coefficients, eps, scales, copies, product_bits,
          part=0, work=None):
    """part 0: muon_step; 1: its norms and whether it is made -> the `work` of part 2, which is the rest."""
    count = len(params)
    a, b, c = coefficients
    scales = [muon_scale(p.shape) for p in params] if scales is None else scales
    return call('muon_step', step, params, grads, momenta, step, _each(lr, count), scales, _each(weight_decay, count), copies,
                momentum, nesterov, a, b, c, eps, steps, _terms(product_bits), part, work)


class Muon(torch.optim.Optimizer):
    """Steps along orthogonalised momenta for matrices, in a few launches for all of them.

    params: of two dimensions or more (those behind the first count as one), fp32 or bf16. lr and weight_decay may differ
    between groups; the rest is the optimizer's, as in muon_step. rms: scale steps to the size of AdamW's (lr is then
    one for AdamW). copies: {parameter: bf16 tensor} that a step writes beside fp32 parameters. A parameter without a
    gradient is left as it is. A step with a matrix whose update has no finite norm changes nothing;
    skipped_steps() counts those. A step can be captured in a graph after one with the same parameters taking part."""

    def __init__(self, params, lr=0.02, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5, coefficients=NEWTON_SCHULZ,
                 eps=1e-7, rms=False, product_bits=None, copies=None):
        if not (lr >= 0 and weight_decay >= 0):
            raise ValueError('lr and weight_decay must not be negative')
        if not 0 <= momentum < 1:
            raise ValueError('momentum must be in [0, 1)')
        _terms(product_bits)
        super().__init__(params, dict(lr=lr, weight_decay=weight_decay))
        self.settings = dict(momentum=momentum, nesterov=nesterov, steps=steps, coefficients=tuple(coefficients), eps=eps,
                             product_bits=product_bits)
        self.rms, self.copies = rms, copies or {}
        self.ctl = None                 # the device's counts (muon_step's `step`)

    def add_param_group(self, param_group):
        names = set(param_group) - {'params', 'lr', 'weight_decay', 'param_names'}
        if names:
            raise ValueError(f'a group has lr and weight_decay of its own, not {", ".join(sorted(names))}')
        super().add_param_group(param_group)
        for p in self.param_groups[-1]['params']:
            if p.dim() < 2:
                del self.param_groups[-1]            # the optimizer stays as it was
                raise ValueError(f'a parameter must have two dimensions or more, not {list(p.shape)}')

    def __getstate__(self):
        return {**super().__getstate__(), **{k: getattr(self, k) for k in ('settings', 'rms', 'copies', 'ctl')}}

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        given = self._given()
        if given is not None:
            _muon(**given)
        return loss

    def begin(self):
        """The first part of a step that another one takes part in: the norms, and whether it is made, on the device (ctl). -> what
        `finish` takes after the other (adamw_step's `other`) has had its say; None where no parameter has a gradient."""
        with torch.no_grad():
            given = self._given()
            return None if given is None else (given, _muon(**given, part=1))

    @staticmethod
    def finish(begun):
        with torch.no_grad():
            _muon(**begun[0], part=2, work=begun[1])

    def _given(self):
        params, lr, decay = [], [], []
        for group in self.param_groups:
            for p in group['params']:
                if p.grad is None:
                    continue
                if not self.state[p]:
                    AdamW._not_captured()
                    self.state[p]['momentum'] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
                params.append(p)
                lr.append(group['lr'])
                decay.append(group['weight_decay'])
        if not params:
            return None
        if self.ctl is None:
            self.ctl = torch.zeros(8, dtype=torch.int32, device=params[0].device)
        return dict(params=params, grads=[p.grad for p in params], momenta=[self.state[p]['momentum'] for p in params], step=self.ctl,
                    lr=lr, weight_decay=decay, scales=[muon_scale(p.shape, self.rms) for p in params],
                    copies=[self.copies.get(p) for p in params] if self.copies else None, **self.settings)

    def skipped_steps(self):
        """Steps left out because an update's norm was not finite (waits for the device)."""
        return 0 if self.ctl is None else int(self.ctl[1].item())

    def state_dict(self):
        d = super().state_dict()
        d['d1'] = dict(muon=True, ctl=None if self.ctl is None else self.ctl.clone())
        return d

    def load_state_dict(self, state_dict):
        own = state_dict.get('d1')
        if own is None or not own.get('muon'):
            raise ValueError("not a state of Muon: another optimizer's is kept otherwise")
        super().load_state_dict({k: v for k, v in state_dict.items() if k != 'd1'})
        # the base class casts tensors to the parameters' type: momenta stay as they were saved
        ids = [i for group in state_dict['param_groups'] for i in group['params']]
        for i, p in zip(ids, (p for group in self.param_groups for p in group['params'])):
            if i in state_dict['state']:
                self.state[p]['momentum'] = state_dict['state'][i]['momentum'].to(p.device, copy=True).contiguous()
        device = self.param_groups[0]['params'][0].device
        self.ctl = None if own['ctl'] is None else own['ctl'].to(device, copy=True)


class MuonAdamW(torch.optim.Optimizer):
    """Muon for the matrices of a model's trunk and AdamW for the rest, stepped together. `named`: the model's
    named_parameters(); those of two dimensions or more are Muon's, but for heads and embeddings (a name with 'head' or
    'embed'). muon, adamw: further arguments of each. A step with a trunk's matrix whose update has no finite norm, or (with
    adamw's max_grad_norm, which clips by the norm of its own gradients alone: a trunk's step has its size whatever the gradient's) with
    other gradients without one, changes nothing at all. Its groups and states are those of the two, to which (`muon`, `adamw`)
    further groups are added."""

    def __init__(self, named, muon=None, adamw=None):
        named = list(named)
        trunk = [p for n, p in named if p.dim() >= 2 and 'head' not in n and 'embed' not in n]
        ids = {id(p) for p in trunk}
        rest = [p for _, p in named if id(p) not in ids]
        self.muon = Muon(trunk, **(muon or {})) if trunk else None
        self.adamw = AdamW(rest, **(adamw or {})) if rest else None
        self.both = [o for o in (self.muon, self.adamw) if o is not None]
        super().__init__(self.param_groups, {})

    # the base class's own lists stay unused
    @property
    def param_groups(self):
        return [g for o in self.both for g in o.param_groups]

    @param_groups.setter
    def param_groups(self, groups):
        pass

    @property
    def state(self):
        return {p: s for o in self.both for p, s in o.state.items()}

    @state.setter
    def state(self, state):
        pass

    def add_param_group(self, param_group):
        if not any(param_group is g for g in self.param_groups):
            raise ValueError('a group is added to .muon or to .adamw')

    def __getstate__(self):
        return dict(muon=self.muon, adamw=self.adamw, both=self.both, defaults=self.defaults)

    def zero_grad(self, set_to_none=True):
        for o in self.both:
            o.zero_grad(set_to_none=set_to_none)

    @torch.no_grad()
    def step(self, closure=None):
        for group in self.adamw.param_groups if self.adamw is not None else ():
            _check_group(group)
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        begun = None if self.muon is None else self.muon.begin()
        if self.adamw is not None:
            self.adamw._step(None if begun is None else self.muon.ctl)
        if begun is not None:
            self.muon.finish(begun)
        return loss

    def skipped_steps(self):
        """Steps left out because a norm was not finite (waits for the device)."""
        return max(o.skipped_steps() for o in self.both)

    def state_dict(self):
        return dict(muon=self.muon and self.muon.state_dict(), adamw=self.adamw and self.adamw.state_dict())

    def load_state_dict(self, state_dict):
        for o, d in ((self.muon, state_dict['muon']), (self.adamw, state_dict['adamw'])):
            if (o is None) != (d is None):
                raise ValueError('the state is of another split of parameters')
            if o is not None:
                o.load_state_dict(d)
