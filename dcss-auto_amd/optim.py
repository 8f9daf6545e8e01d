"""AdamW over many tensors in a few launches, with moments in 32 or 8 bits (csrc/d1_optim.hip).

`AdamW` is the torch optimizer, `adamw_step` the step itself on lists of tensors, `read_moment` what
an 8-bit moment stands for. The step count, the global norm of a clip and the skip of a step whose
norm is not finite stay on the device, so a step can be captured in a HIP graph.
"""
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
               max_grad_norm=0.0, copies=None, exps=None, counters=None, seed=0, lags=None):
    """One AdamW step in place over lists of tensors.

    params: fp32 or bf16, contiguous. grads: fp32 or bf16 of the same sizes. exp_avg, exp_avg_sq:
    fp32 (32-bit moments), or uint8 codes with exps = (list of exp_avg's, list of exp_avg_sq's)
    exponents, uint8 of moment_blocks(numel) each, and counters: the first counter of each tensor's
    rounding draws, one an element (tensors whose ranges overlap round alike there). Zero codes
    and exponents are zero moments. step: int32 [8] on the device, zeros before the first step; [0]
    counts the steps made, [1] those skipped. copies: bf16 tensors that get the new fp32 parameters
    (None in the list: no copy). What the call changes gets a new version, as from torch's operations in
    place; the replay of a captured call cannot give it one. lr and weight_decay: one value or one for each tensor. lags: steps
    that each tensor has missed.

    With max_grad_norm > 0 the gradients are scaled by min(1, max_grad_norm / (norm + 1e-6)) with
    the norm over all of them, and a step whose norm is not finite changes nothing and is counted.
    Without, an element whose gradient (or its square) is not finite is lost alone; its 8-bit moments
    start anew, 32-bit ones stay not finite."""
    count = len(params)
    m_exps, v_exps = exps if exps is not None else (None, None)
    call('adamw_step', step, params, grads, exp_avg, exp_avg_sq, step, _each(lr, count), _each(weight_decay, count), betas[0],
         betas[1], eps, max_grad_norm, copies, m_exps, v_exps, counters, lags, seed & 0xFFFFFFFFFFFFFFFF)


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
            return loss
        if self.ctl is None:
            self.ctl = torch.zeros(8, dtype=torch.int32, device=params[0].device)
        eight = self.state_bits == 8
        column = lambda name: [s[name] for s in states]  # noqa: E731
        adamw_step(params, [p.grad for p in params], column('exp_avg'), column('exp_avg_sq'), self.ctl, lr=lr,
                   betas=self.betas, eps=self.eps, weight_decay=decay, max_grad_norm=self.max_grad_norm,
                   copies=[self.copies.get(p) for p in params] if self.copies else None,
                   exps=(column('exp_avg_exp'), column('exp_avg_sq_exp')) if eight else None,
                   counters=column('counter') if eight else None, seed=self.seed,
                   lags=column('lag'))
        return loss

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
