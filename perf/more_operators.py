"""Operators of updates over sequences, as measurable cases.

Three groups: the clipped policy loss with its value, entropy and reference-KL terms and their gradients;
a gated linear recurrence over long sequences with its backward pass and its form for single steps; updates
orthogonalised by Newton-Schulz products and the momentum step made of them. `run` computes a case in plain
torch operations in 32 bits, or with `own` through the package's operators; `exact` computes it in 64 bits.
"""
import importlib
import math

import torch

own = False

DEV = 'cuda:0'
DTYPES = {'fp32': torch.float32, 'bf16': torch.bfloat16, 'fp16': torch.float16}
BYTES = {'fp32': 4, 'bf16': 2, 'fp16': 2}
CLIP = (0.2, 0.28)
VALUE_CLIP = 0.3
KL, VALUE, ENTROPY = 0.05, 0.5, 0.01
NS = (3.4445, -4.7750, 2.0315)
NS_STEPS, NS_EPS = 5, 1e-7
LR, DECAY, MOMENTUM = 0.02, 0.01, 0.95
POLICY = [(256, 1800), (256, 256), (17, 256)]       # the matrices of this repository's policy


def listed():
    return [
        # a PPO minibatch of single decisions: value and entropy terms, the smallest training call
        dict(name='loss_ppo', op='loss', rows=1, length=8192, dtype='fp32', level='token', mask=False, per_row=False,
             ref=False, value=True, entropy=True),
        # padded answers scored as a whole: an advantage a sequence, KL to a reference, a few sequences without a token
        dict(name='loss_answers', op='loss', rows=512, length=4097, dtype='bf16', level='sequence', mask=True, per_row=True,
             ref=True, value=False, entropy=False),
        # a whole rollout of 128 steps over 65,536 worlds with every term, worlds that were frozen left out
        dict(name='loss_rollout', op='loss', rows=128, length=65536, dtype='fp32', level='token', mask=True, per_row=False,
             ref=True, value=True, entropy=True),
        # a large batch of long sequences
        dict(name='loss_long', op='loss', rows=2048, length=16411, dtype='fp32', level='sequence', mask=True, per_row=False,
             ref=True, value=False, entropy=True),
        # acting: one step of a memory layer for 65,536 worlds, some of which began an episode
        dict(name='scan_step', op='scan', length=1, rows=65536, width=256, dtype='bf16', state=True, reset=True, grad=False),
        # a small ragged batch in fp32 with several sequences packed into a row
        dict(name='scan_packed', op='scan', length=1000, rows=37, width=1001, dtype='fp32', state=False, reset=True, grad=True),
        # the update's pass over a rollout: 128 steps of 8,192 worlds, forward and backward
        dict(name='scan_rollout', op='scan', length=128, rows=8192, width=256, dtype='bf16', state=True, reset=True, grad=True),
        # one long sequence
        dict(name='scan_long', op='scan', length=65537, rows=1, width=1024, dtype='bf16', state=True, reset=False, grad=True),
        # the policy's own matrices, fp32: latency
        dict(name='ortho_policy', op='muon', model='policy', layers=0, rows=0, cols=0, params='fp32', grads='fp32', step=False),
        # one matrix of odd sizes, taller than wide
        dict(name='ortho_ragged', op='muon', model='one', layers=1, rows=4001, cols=1000, params='bf16', grads='bf16', step=False),
        # two layers of a trunk with fp32 masters and bf16 gradients: the whole step
        dict(name='muon_trunk', op='muon', model='stack', layers=2, rows=1024, cols=0, params='fp32', grads='bf16', step=True),
        # a wide layer held in bf16
        dict(name='muon_wide', op='muon', model='stack', layers=1, rows=4096, cols=0, params='bf16', grads='bf16', step=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(['loss', 'loss', 'scan', 'scan', 'scan', 'muon', 'muon'])
    if op == 'loss':
        length = _log_int(rng, 1, 65536)
        rows = _log_int(rng, 1, max(1, min(16384, 30_000_000 // length)))
        return dict(op='loss', rows=rows, length=length, dtype=rng.choice(['fp32', 'fp32', 'bf16', 'fp16']),
                    level=rng.choice(['token', 'sequence']), mask=rng.random() < 0.7, per_row=rng.random() < 0.4,
                    ref=rng.random() < 0.6, value=rng.random() < 0.5, entropy=rng.random() < 0.5)
    if op == 'scan':
        length, width = _log_int(rng, 1, 65536), _log_int(rng, 16, 4096)
        rows = _log_int(rng, 1, max(1, min(16384, 60_000_000 // (length * width))))
        return dict(op='scan', length=length, rows=rows, width=width, dtype=rng.choice(['fp32', 'bf16', 'bf16', 'fp16']),
                    state=rng.random() < 0.6, reset=rng.random() < 0.6, grad=rng.random() < 0.7)
    params = rng.choice(['fp32', 'bf16'])
    if rng.random() < 0.3:
        width = _log_int(rng, 32, 2048)
        return dict(op='muon', model='stack', layers=rng.randint(1, 2), rows=width, cols=0, params=params,
                    grads=rng.choice([params, 'bf16']), step=rng.random() < 0.7)
    return dict(op='muon', model='one', layers=1, rows=_log_int(rng, 1, 6000), cols=_log_int(rng, 1, 6000), params=params,
                grads=rng.choice([params, 'bf16']), step=rng.random() < 0.4)


def _shapes(case):
    if case['model'] == 'policy':
        return POLICY
    if case['model'] == 'one':
        return [(case['rows'], case['cols'])]
    w = case['rows']
    return [(w, w), (w, w), (w, w), (w, w), (4 * w, w), (w, 4 * w)] * case['layers']


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=g, device=DEV)  # noqa: E731
    uniform = lambda *shape: torch.rand(*shape, generator=g, device=DEV)  # noqa: E731
    if case['op'] == 'loss':
        n, t, dt = case['rows'], case['length'], DTYPES[case['dtype']]
        old = uniform(n, t).clamp_(min=1e-6).log_().mul_(1.5)
        s = dict(op='loss', level=case['level'], old_logp=old.to(dt), logp=(old + 0.2 * normal(n, t)).clamp_(max=0).to(dt),
                 advantages=normal(n) if case['per_row'] else normal(n, t), ref_logp=None, entropy=None, values=None,
                 returns=None, old_values=None, mask=None)
        if case['ref']:
            s['ref_logp'] = (old + 0.3 * normal(n, t)).clamp_(max=0).to(dt)
        if case['entropy']:
            s['entropy'] = (2.5 * uniform(n, t)).to(dt)
        if case['value']:
            v = normal(n, t)
            s['old_values'] = v
            s['returns'] = v + 0.5 * normal(n, t)
            s['values'] = (v + 0.3 * normal(n, t)).to(dt)
        if case['mask']:             # a prefix of each row, some rows without any, some places inside left out
            lengths = (uniform(n, 1) * 1.3 - 0.05) * t
            s['mask'] = (torch.arange(t, device=DEV) < lengths) & (uniform(n, t) < 0.98)
        return s
    if case['op'] == 'scan':
        t, n, d, dt = case['length'], case['rows'], case['width'], DTYPES[case['dtype']]
        # channels that remember from a step or two to thousands
        s = dict(op='scan', x=normal(t, n, d).to(dt), gate=(normal(t, n, d) - 6.0 * uniform(d)).to(dt), state=None, reset=None,
                 grad=case['grad'])
        if case['state']:
            s['state'] = normal(n, d)
        if case['reset']:
            s['reset'] = uniform(t, n) < 0.01
        if case['grad']:
            s['dh'] = normal(t, n, d).mul_(0.1).to(dt)
            s['dlast'] = normal(n, d).mul_(0.1) if case['state'] else None
        return s
    shapes = _shapes(case)
    s = dict(op='muon', step_made=case['step'], grads=[])
    for r, c in shapes:              # gradients: a few strong directions over noise
        k = min(4, r, c)
        s['grads'].append((normal(r, c) + 0.5 * normal(r, k) @ normal(k, c)).mul_(1e-3).to(DTYPES[case['grads']]))
    if case['step']:
        s['params'] = [normal(r, c).mul_(0.02).to(DTYPES[case['params']]) for r, c in shapes]
        s['momenta'] = [normal(r, c).mul_(5e-3) for r, c in shapes]
        s['step'] = torch.zeros(8, dtype=torch.int32, device=DEV)
    else:
        s['grads'] = [x.to(DTYPES[case['params']]) for x in s['grads']]
    return s


def run(state):
    return (_own if own else _plain)[state['op']](state)


# ---- the plain forms

def _plain_loss(s):
    logp, old = s['logp'].double(), s['old_logp'].double()      # which side of the clip: differences in 64 bits
    n, t = logp.shape
    zero = torch.zeros((), device=DEV)
    mask = s['mask']
    mean = mask if mask is not None else torch.ones(n, t, dtype=torch.bool, device=DEV)
    if s['level'] == 'sequence':
        each = mean.sum(1, keepdim=True)
        rows = (each > 0).sum()
        w = mean / (each.clamp(min=1) * rows.clamp(min=1)).float()
    else:
        w = mean / mean.sum().clamp(min=1).float()
    adv = s['advantages'].float()
    adv = adv[:, None].expand(n, t) if adv.dim() == 1 else adv
    pick = lambda x: x if mask is None else torch.where(mask, x, zero)  # noqa: E731
    total = lambda x: (pick(x) * w).sum(dtype=torch.float64)  # noqa: E731
    d = logp - old
    clipped = torch.where(adv > 0, d > math.log1p(CLIP[1]), (adv < 0) & (d < math.log1p(-CLIP[0])))
    bound = torch.where(adv > 0, 1 + CLIP[1], 1 - CLIP[0])
    d = d.float()
    ratio = torch.exp(d)
    policy = -total(torch.where(clipped, bound, ratio) * adv)
    dlogp = torch.where(clipped, zero, -adv * ratio)
    out = dict(policy=policy, clipped=total(clipped.float()), drift=total(torch.expm1(d) - d))
    loss = policy
    if s['ref_logp'] is not None:
        x = (s['ref_logp'].double() - logp).float()
        e = torch.expm1(x)
        out['kl'] = total(e - x)
        loss = loss + KL * out['kl']
        dlogp = dlogp - KL * e
    out['dlogp'] = (pick(dlogp) * w).to(s['logp'].dtype)
    if s['entropy'] is not None:
        out['entropy'] = total(s['entropy'].float())
        loss = loss - ENTROPY * out['entropy']
        out['dentropy'] = (-ENTROPY * w).to(s['entropy'].dtype)
    if s['values'] is not None:
        v, old_v, ret = (s[name].double() for name in ('values', 'old_values', 'returns'))
        free = v - ret
        held = old_v + (v - old_v).clamp(-VALUE_CLIP, VALUE_CLIP) - ret
        use = free.square() >= held.square()
        out['value'] = total(0.5 * torch.where(use, free, held).float().square())
        loss = loss + VALUE * out['value']
        out['dvalues'] = (pick(torch.where(use, free.float(), zero)) * w * VALUE).to(s['values'].dtype)
    out['loss'] = loss                  # terms of either sign nearly cancel: rounded last
    return {name: x.float() if x.dim() == 0 else x for name, x in out.items()}


def _spread(a, b, back=False):
    """h[t] = a[t] h[t-1] + b[t] along the first dimension (from the end with `back`) by doubling spans."""
    step, n = 1, a.shape[0]
    while step < n:
        lo, hi = (slice(0, n - step), slice(step, n)) if not back else (slice(step, n), slice(0, n - step))
        more = a[hi] * b[lo]
        span = a[hi] * a[lo]
        b = b.clone()
        b[hi] += more
        a = a.clone()
        a[hi] = span
        step *= 2
    return b


def _plain_scan(s):
    x, gate = s['x'].float(), s['gate'].float()
    z, a = torch.sigmoid(gate), torch.sigmoid(-gate)
    keep = a if s['reset'] is None else torch.where(s['reset'][:, :, None], 0.0, a)
    b = z * x
    if s['state'] is not None:
        b[0] += keep[0] * s['state']
    h = _spread(keep, b)
    out = dict(h=h.to(s['x'].dtype), last=h[-1].clone())
    if s['grad']:
        carry = s['dh'].float()
        if s['dlast'] is not None:
            carry = carry.clone()
            carry[-1] += s['dlast']
        after = torch.cat([keep[1:], torch.zeros_like(keep[:1])])
        g = _spread(after, carry, back=True)
        before = torch.cat([torch.zeros_like(h[:1]) if s['state'] is None else s['state'][None], h[:-1]])
        if s['reset'] is not None:
            before = torch.where(s['reset'][:, :, None], 0.0, before)
        out['dx'] = (g * z).to(s['x'].dtype)
        out['dgate'] = (g * (x - before) * (z * a)).to(s['x'].dtype)
        if s['state'] is not None:
            out['dstate'] = keep[0] * g[0]
    return out


def _plain_ortho(u):
    x = u / (u.double().square().sum().sqrt().float() + NS_EPS)
    flip = x.shape[0] > x.shape[1]
    x = x.t().contiguous() if flip else x
    for _ in range(NS_STEPS):
        a = x @ x.t()
        x = NS[0] * x + (NS[1] * a + NS[2] * (a @ a)) @ x
    return x.t() if flip else x


def _plain_muon(s):
    if not s['step_made']:
        return [_plain_ortho(g.float()).to(g.dtype) for g in s['grads']]
    for p, g, m in zip(s['params'], s['grads'], s['momenta']):
        g = g.float()
        m.mul_(MOMENTUM).add_(g)
        o = _plain_ortho(g + MOMENTUM * m)
        scale = math.sqrt(max(1.0, p.shape[0] / p.shape[1]))
        p.copy_(p.float() * (1 - LR * DECAY) - (LR * scale) * o)
    return dict(params=s['params'], momenta=s['momenta'])


_plain = dict(loss=_plain_loss, scan=_plain_scan, muon=_plain_muon)


# ---- the package's operators

def _own_loss(s):
    L = importlib.import_module('dcss-auto_amd.losses')
    names = ('ref_logp', 'entropy', 'values', 'returns', 'old_values', 'mask')
    more = dict({name: s[name] for name in names}, clip=CLIP, value_clip=VALUE_CLIP, kl_coef=KL, value_coef=VALUE,
                entropy_coef=ENTROPY, level=s['level'])
    r, dlogp, dentropy, dvalues = L.policy_loss_grads(s['logp'], s['old_logp'], s['advantages'], **more)
    out = dict(policy=r.policy, clipped=r.clipped, drift=r.drift)
    if s['ref_logp'] is not None:
        out['kl'] = r.kl
    out['dlogp'] = dlogp
    if s['entropy'] is not None:
        out.update(entropy=r.entropy, dentropy=dentropy)
    if s['values'] is not None:
        out.update(value=r.value, dvalues=dvalues)
    out['loss'] = r.loss
    return out


def _own_scan(s):
    R = importlib.import_module('dcss-auto_amd.recurrence')
    if not s['grad']:
        h, last = R.gated_scan(s['x'], s['gate'], s['state'], s['reset'])
        return dict(h=h, last=last)
    h, last, marks = R.gated_scan_fwd(s['x'], s['gate'], s['state'], s['reset'])
    dx, dgate, dstate = R.gated_scan_bwd(s['dh'], s['dlast'], s['x'], s['gate'], s['state'], s['reset'], marks)
    out = dict(h=h, last=last, dx=dx, dgate=dgate)
    if s['state'] is not None:
        out['dstate'] = dstate
    return out


def _own_muon(s):
    O = importlib.import_module('dcss-auto_amd.optim')
    if not s['step_made']:
        return O.orthogonalize(s['grads'], steps=NS_STEPS, coefficients=NS, eps=NS_EPS)
    O.muon_step(s['params'], s['grads'], s['momenta'], s['step'], lr=LR, momentum=MOMENTUM, nesterov=True, weight_decay=DECAY,
                steps=NS_STEPS, coefficients=NS, eps=NS_EPS)
    return dict(params=s['params'], momenta=s['momenta'])


_own = dict(loss=_own_loss, scan=_own_scan, muon=_own_muon)


# ---- what a pass cannot do without

def work(case):
    if case['op'] == 'loss':
        n, b = case['rows'] * case['length'], BYTES[case['dtype']]
        each = 3 * b + (1 if case['mask'] else 0) + (0 if case['per_row'] else 4) + (b if case['ref'] else 0) + \
            (2 * b if case['entropy'] else 0) + (2 * b + 8 if case['value'] else 0)
        ops = 14 + (6 if case['ref'] else 0) + (2 if case['entropy'] else 0) + (12 if case['value'] else 0)
        return dict(bytes=n * each + (4 * case['rows'] if case['per_row'] else 0), flops=n * ops)
    if case['op'] == 'scan':
        cells = case['rows'] * case['width']
        n, b = case['length'] * cells, BYTES[case['dtype']]
        ends = 4 + (4 if case['state'] else 0) + (8 if case['grad'] and case['state'] else 0)
        return dict(bytes=n * b * (6 if case['grad'] else 3) + ends * cells +
                    (case['length'] * case['rows'] if case['reset'] else 0), flops=n * (8 + (10 if case['grad'] else 0)))
    move = math_ops = 0
    for r, c in _shapes(case):
        m, n = min(r, c), max(r, c)
        g, p = BYTES[case['grads']], BYTES[case['params']]
        move += r * c * (g + 2 * p + 8 if case['step'] else 2 * p)
        # two symmetric products (half of one each) and one whole product a step
        math_ops += NS_STEPS * (m * (m + 1) * n + m * (m + 1) * m + 2 * m * m * n)
    return dict(bytes=move, flops=math_ops)


# ---- the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return dict(loss=_exact_loss, scan=_exact_scan, muon=_exact_muon)[case['op']](s)


def _exact_loss(s):
    """Through the elementwise losses and autograd."""
    leaf = lambda x: x.to(torch.float64).requires_grad_()  # noqa: E731
    logp = leaf(s['logp'])
    rows, length = logp.shape
    keep = torch.ones(rows, length, dtype=torch.float64, device=DEV) if s['mask'] is None else s['mask'].to(torch.float64)
    if s['level'] == 'token':
        weight = keep / max(1.0, float(keep.sum()))
    else:
        count = keep.sum(1)
        some = max(1, int((count > 0).sum()))
        weight = keep / torch.clamp(count, min=1.0)[:, None] / some
    adv = s['advantages'].to(torch.float64).reshape(rows, -1)
    log_ratio = logp - s['old_logp'].to(torch.float64)
    ratio = log_ratio.exp()
    inside = torch.clamp(ratio, 1 - CLIP[0], 1 + CLIP[1])
    gain = torch.minimum(ratio * adv, inside * adv)
    terms = dict(policy=-(gain * weight).sum(), clipped=((inside * adv < ratio * adv) * weight).sum(),
                 drift=((ratio - 1 - log_ratio) * weight).sum())
    loss = terms['policy']
    if s['ref_logp'] is not None:
        gap = s['ref_logp'].to(torch.float64) - logp
        terms['kl'] = ((gap.exp() - gap - 1) * weight).sum()
        loss = loss + KL * terms['kl']
    if s['entropy'] is not None:
        entropy = leaf(s['entropy'])
        terms['entropy'] = (entropy * weight).sum()
        loss = loss - ENTROPY * terms['entropy']
    if s['values'] is not None:
        values, old = leaf(s['values']), s['old_values'].to(torch.float64)
        ret = s['returns'].to(torch.float64)
        near = torch.minimum(torch.maximum(values, old - VALUE_CLIP), old + VALUE_CLIP)
        terms['value'] = (torch.maximum((values - ret) ** 2, (near - ret) ** 2) * weight).sum() / 2
        loss = loss + VALUE * terms['value']
    loss.backward()
    out = {name: terms[name].detach() for name in ('policy', 'clipped', 'drift')}
    if s['ref_logp'] is not None:
        out['kl'] = terms['kl'].detach()
    out['dlogp'] = logp.grad
    if s['entropy'] is not None:
        out.update(entropy=terms['entropy'].detach(), dentropy=entropy.grad)
    if s['values'] is not None:
        out.update(value=terms['value'].detach(), dvalues=values.grad)
    out['loss'] = loss.detach()
    return out


def _exact_scan(s):
    """Step by step."""
    x, gate = s['x'], s['gate']
    steps, rows, width = x.shape
    open_ = None if s['reset'] is None else ~s['reset']
    h = torch.zeros(rows, width, dtype=torch.float64, device=DEV) if s['state'] is None else s['state'].to(torch.float64)
    hs = torch.empty(steps + 1, rows, width, dtype=torch.float64, device=DEV)
    hs[0] = h
    remember = torch.special.expit(-gate.to(torch.float64))
    if open_ is not None:
        remember *= open_[:, :, None]
    take = torch.special.expit(gate.to(torch.float64))
    torch.mul(take, x, out=hs[1:])
    for k in range(steps):
        hs[k + 1].addcmul_(remember[k], hs[k])
    out = dict(h=hs[1:], last=hs[-1])
    if not s['grad']:
        return out
    grad = s['dh'].to(torch.float64)
    if s['dlast'] is not None:
        grad[-1] += s['dlast']
    for k in range(steps - 1, 0, -1):
        grad[k - 1].addcmul_(remember[k], grad[k])
    if s['state'] is not None:
        dstate = remember[0] * grad[0]
    out['dx'] = grad * take
    before = hs[:-1]
    if open_ is not None:
        before = before * open_[:, :, None]
    slope = take * torch.special.expit(-gate.to(torch.float64))
    out['dgate'] = torch.sub(x, before).mul_(slope).mul_(grad)
    if s['state'] is not None:
        out['dstate'] = dstate
    return out


def _exact_ortho(u):
    rows, cols = u.shape
    y = u / (torch.linalg.matrix_norm(u) + NS_EPS)
    if rows > cols:                  # (a + b G + c G^2) on the smaller side
        for _ in range(NS_STEPS):
            gram = torch.mm(y.mT, y)
            y = torch.mm(y, NS[1] * gram + NS[2] * torch.mm(gram, gram)).add_(y, alpha=NS[0])
    else:
        for _ in range(NS_STEPS):
            gram = torch.mm(y, y.mT)
            y = torch.mm(NS[1] * gram + NS[2] * torch.mm(gram, gram), y).add_(y, alpha=NS[0])
    return y


def _exact_muon(s):
    grads = [g.to(torch.float64) for g in s['grads']]
    if not s['step_made']:
        return [_exact_ortho(g) for g in grads]
    params, momenta = [], []
    for p, g, m in zip(s['params'], grads, s['momenta']):
        m = MOMENTUM * m.to(torch.float64) + g
        w = p.to(torch.float64)
        tall = max(1.0, w.shape[0] / w.shape[1]) ** 0.5
        params.append(w - LR * DECAY * w - LR * tall * _exact_ortho(torch.add(g, m, alpha=MOMENTUM)))
        momenta.append(m)
    return dict(params=params, momenta=momenta)
