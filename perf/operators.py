"""The operators of a policy update outside the fused MLP step, as measurable cases.

Three groups: log probabilities of given tokens (actions) with entropy, top alternatives and the
gradient of the logits; layer norm with its backward pass; the AdamW step over many tensors with
states in 32 or 8 bits and the global-norm clip. `run` computes a case in plain torch operations in
32 bits, or with `own` through the package's operators; `exact` computes it in 64 bits.
"""
import importlib
import math

import torch

own = False

DEV = 'cuda:0'
DTYPES = {'fp32': torch.float32, 'bf16': torch.bfloat16, 'fp16': torch.float16}
BYTES = {'fp32': 4, 'bf16': 2, 'fp16': 2}
BETA1, BETA2, ADAM_EPS = 0.9, 0.999, 1e-5
LR, DECAY = 3e-4, 0.01
BLOCK = 256                # state elements that share a scale
LN_EPS = 1e-5
# parameter shapes of this repository's two policies
POLICY = [(256, 1800), (256,), (256, 256), (256,), (17, 256), (17,)]
AR_POLICY = [(256, 1800), (256,), (256, 256), (256,), (8, 256), (8,), (1, 256), (1,), (8, 16), (64, 272), (64,),
             (25, 64), (25,)]


def listed():
    return [
        # the policy's 16 logits beside its value (rows of 17) in a PPO minibatch: the smallest training call
        dict(name='tokens_ppo', op='tokens', rows=8192, vocab=16, pad=1, dtype='fp32', top=0, mask=False, grad=True),
        # the 25 targets of every verb of a large minibatch, with a mask of legal targets; a few rows allow none
        dict(name='tokens_targets', op='tokens', rows=65536, vocab=25, pad=0, dtype='fp32', top=3, mask=True, grad=True),
        # serving: the next token's log probability with 20 alternatives, one row of a long vocabulary
        dict(name='tokens_next', op='tokens', rows=1, vocab=131072, pad=0, dtype='bf16', top=20, mask=False, grad=False),
        # scoring a prompt: an odd vocabulary (rows unaligned), five alternatives a position
        dict(name='tokens_score', op='tokens', rows=512, vocab=50001, pad=0, dtype='fp16', top=5, mask=False, grad=False),
        # a training step's loss over a long vocabulary, forward and gradient
        dict(name='tokens_train', op='tokens', rows=4096, vocab=131072, pad=0, dtype='bf16', top=0, mask=False, grad=True),
        # a trunk layer of width 256 in a PPO minibatch, forward and backward
        dict(name='norm_ppo', op='norm', rows=8192, width=256, dtype='bf16', weights='fp32', grad=True),
        # the same layer in a rollout over 65,536 worlds, forward alone
        dict(name='norm_rollout', op='norm', rows=65536, width=256, dtype='bf16', weights='fp32', grad=False),
        # a ragged batch of fp32 observation rows
        dict(name='norm_obs', op='norm', rows=4133, width=1800, dtype='fp32', weights='fp32', grad=True),
        # a wide model's layer over a long batch of tokens
        dict(name='norm_wide', op='norm', rows=16384, width=8192, dtype='bf16', weights='bf16', grad=True),
        # the policy's six tensors as its trainer holds them: fp32 masters, bf16 gradients and copies, clip 0.5
        dict(name='adamw_policy', op='adamw', model='policy', layers=0, width=0, vocab=0, bits=32, grads='bf16',
             copy=True, clip=0.5),
        # a model of ragged sizes (49 tensors, 98 M parameters) with fp32 gradients from autograd, no clip
        dict(name='adamw_ragged', op='adamw', model='stack', layers=4, width=1000, vocab=50001, bits=32, grads='fp32',
             copy=False, clip=0.0),
        # a stack of wide layers (73 tensors, 369 M parameters), states in 8 bits
        dict(name='adamw_stack8', op='adamw', model='stack', layers=6, width=2048, vocab=32768, bits=8, grads='bf16',
             copy=True, clip=1.0),
    ]


def _log_int(rng, lo, hi):
    v = max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))
    return v + 1 if v == 3072 else v


def draw(rng):
    op = rng.choice(['tokens', 'tokens', 'tokens', 'norm', 'norm', 'adamw', 'adamw'])
    dtype = rng.choice(['fp32', 'bf16', 'bf16', 'fp16'])
    if op == 'tokens':
        if rng.random() < 0.4:      # action heads
            vocab, rows = _log_int(rng, 2, 1000), _log_int(rng, 16, 131072)
        else:                       # vocabularies
            vocab = _log_int(rng, 1001, 131071)
            rows = _log_int(rng, 1, max(1, min(16384, 400_000_000 // vocab)))
        grad = rng.random() < 0.5
        return dict(op='tokens', rows=rows, vocab=vocab, pad=rng.choice([0, 0, 1, 8]), dtype=dtype,
                    top=rng.choice([0, rng.randint(1, min(32, vocab))]), mask=rng.random() < 0.3, grad=grad)
    if op == 'norm':
        width = _log_int(rng, 8, 16384)
        rows = _log_int(rng, 1, max(1, min(262144, 120_000_000 // width)))
        return dict(op='norm', rows=rows, width=width, dtype=dtype, weights=rng.choice(['fp32', dtype]),
                    grad=rng.random() < 0.6)
    if rng.random() < 0.15:
        return dict(op='adamw', model='ar', layers=0, width=0, vocab=0, bits=rng.choice([8, 32]),
                    grads=rng.choice(['fp32', 'bf16']), copy=rng.random() < 0.5, clip=rng.choice([0.0, 0.5, 1.0]))
    width = _log_int(rng, 32, 1600)
    return dict(op='adamw', model='stack', layers=rng.randint(1, 8), width=width + (width == 768),
                vocab=_log_int(rng, 100, 32768), bits=rng.choice([8, 32]), grads=rng.choice(['fp32', 'bf16']),
                copy=rng.random() < 0.5, clip=rng.choice([0.0, 0.5, 1.0]))


def _shapes(case):
    if case['model'] == 'policy':
        return POLICY
    if case['model'] == 'ar':
        return AR_POLICY
    w = case['width']
    layer = [(w,), (w,), (w, w), (w, w), (w, w), (w, w), (w,), (w,), (4 * w, w), (4 * w,), (w, 4 * w), (w,)]
    return [(case['vocab'], w)] + layer * case['layers']


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def prepare(case, seed):
    g = _gen(seed)
    rand = lambda *shape, dtype=torch.float32: torch.randn(*shape, generator=g, device=DEV, dtype=dtype)  # noqa: E731
    if case['op'] == 'tokens':
        n, k, dt = case['rows'], case['vocab'], DTYPES[case['dtype']]
        logits = rand(n, k + case['pad'], dtype=dt).mul_(2.0)
        rows = torch.arange(n, device=DEV)
        # a trained head is sure of most rows: one entry stands out
        hot = torch.randint(0, k, (n,), generator=g, device=DEV)
        logits[rows, hot] += (6.0 + 2.0 * rand(n)).to(dt)
        tokens = torch.randint(0, k, (n,), generator=g, device=DEV)
        pick = torch.rand(n, generator=g, device=DEV)
        tokens = torch.where(pick < 0.6, hot, tokens)
        s = dict(op='tokens', logits=logits[:, :k], top=case['top'], mask=None, grad=case['grad'])
        if case['mask']:
            s['mask'] = torch.rand(n, k, generator=g, device=DEV) < 0.7
            s['mask'][::509] = False
        elif k > 1000:               # padded positions of a batch of sequences
            tokens = torch.where(pick > 0.97, -1, tokens)
        s['tokens'] = tokens
        if case['grad']:
            s['dlogp'] = rand(n) / n
            s['dentropy'] = torch.full((n,), -0.01 / n, device=DEV)
        return s
    if case['op'] == 'norm':
        n, d, dt, wt = case['rows'], case['width'], DTYPES[case['dtype']], DTYPES[case['weights']]
        shift = rand(d)
        s = dict(op='norm', x=(rand(n, d) * 1.5 + shift).to(dt), weight=(1 + 0.1 * rand(d)).to(wt),
                 bias=(0.1 * rand(d)).to(wt), grad=case['grad'])
        if case['grad']:
            s['dy'] = rand(n, d, dtype=dt).mul_(0.1)
        return s
    shapes = _shapes(case)
    sizes = [math.prod(x) for x in shapes]
    room = [-(-n // BLOCK) * BLOCK for n in sizes]
    at = [sum(room[:i]) for i in range(len(room))]
    total = sum(room)
    gd = DTYPES[case['grads']]
    views = lambda flat: [flat[o:o + n] for o, n in zip(at, sizes)]  # noqa: E731
    s = dict(op='adamw', bits=case['bits'], clip=case['clip'], seed=seed, at=at,
             p=torch.zeros(total, device=DEV), step=torch.zeros(8, dtype=torch.int32, device=DEV))
    s['step'][0] = 100               # steps made so far
    m, v = torch.zeros(total, device=DEV), torch.zeros(total, device=DEV)
    for o, n, shape in zip(at, sizes, shapes):
        s['p'][o:o + n].normal_(0, 0.02, generator=g)
        m[o:o + n].normal_(0, 2e-4, generator=g)
        v[o:o + n].normal_(0, 1e-3, generator=g)
    v.square_()
    s['grads'] = [rand(*shape, dtype=gd).mul_(1e-3) for shape in shapes]
    s['fill'] = [torch.zeros(r - n, device=DEV) for r, n in zip(room, sizes)]
    s['params'] = [x.view(shape) for x, shape in zip(views(s['p']), shapes)]
    if case['bits'] == 8:
        draw_ = _draws(seed, torch.zeros(1, dtype=torch.int64, device=DEV), total)
        s['m'], s['m_exp'] = _encode(m, 15, draw_ >> 16)
        s['v'], s['v_exp'] = _encode(v, 31, draw_ & 0xFFFF)
        exps = lambda flat: [flat[o // BLOCK:(o + r) // BLOCK] for o, r in zip(at, room)]  # noqa: E731
        s['m_exps'], s['v_exps'] = exps(s['m_exp']), exps(s['v_exp'])
    else:
        s['m'], s['v'] = m, v
    s['ms'], s['vs'] = views(s['m']), views(s['v'])
    s['copy'] = s['p'].to(torch.bfloat16) if case['copy'] else None
    s['copies'] = views(s['copy']) if case['copy'] else None
    return s


def run(state):
    return (_own if own else _plain)[state['op']](state)


# ---- the plain forms

def _plain_tokens(s):
    x, tokens, mask = s['logits'].float(), s['tokens'], s['mask']
    if mask is not None:
        x = torch.where(mask, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    lse = torch.where(total > 0, top + torch.log(total), 0.0)
    lp = x - lse
    p = e / torch.where(total > 0, total, 1.0)
    entropy = -(p * torch.where(p > 0, lp, 0.0)).sum(-1)
    at = tokens.clamp(min=0)[:, None]
    logp = torch.where(tokens < 0, 0.0, lp.gather(1, at).squeeze(1))
    out = dict(logp=logp, entropy=entropy)
    if s['top']:
        order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :s['top']]
        out['top_logp'] = lp.gather(1, order)
        out['top_ids'] = torch.where(out['top_logp'] > -math.inf, order, -1)
    if s['grad']:
        g = torch.where(tokens < 0, 0.0, s['dlogp'])[:, None]
        d = -p * (g + s['dentropy'][:, None] * (torch.where(p > 0, lp, 0.0) + entropy[:, None]))
        d.scatter_add_(1, at, g)
        if mask is not None:
            d = torch.where(mask, d, 0.0)
        out['dlogits'] = d.to(s['logits'].dtype)
    return out


def _plain_norm(s):
    x, w, b = s['x'].float(), s['weight'].float(), s['bias'].float()
    d = x - x.mean(-1, keepdim=True)
    r = 1.0 / torch.sqrt((d * d).mean(-1, keepdim=True) + LN_EPS)
    xh = d * r
    out = dict(y=(xh * w + b).to(s['x'].dtype))
    if s['grad']:
        dy = s['dy'].float()
        u = dy * w
        dx = r * (u - u.mean(-1, keepdim=True) - xh * (u * xh).mean(-1, keepdim=True))
        out.update(dx=dx.to(s['x'].dtype), dweight=(dy * xh).sum(0).to(s['weight'].dtype),
                   dbias=dy.sum(0).to(s['bias'].dtype))
    return out


def _mix(x):
    """A 32-bit word through two multiplications and three shifts (words held in int64)."""
    x = x ^ (x >> 16)
    x = (x * 0x9E3779B1) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0xB7E15163) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _draws(seed, step, total):
    """One 32-bit word for each state element from (seed, step, the element's counter)."""
    key = _mix(_mix(_mix(torch.full_like(step, seed & 0xFFFFFFFF)) ^ (seed >> 32)) ^ step)
    return _mix(torch.arange(total, device=step.device) ^ _mix(key))


def _power(e):
    """2^e as fp64, from its bits."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _encode(x, top, draw):
    """fp32 -> 8 bits against the block's power of two: 4 exponent bits and a sign (top 15) or 5
    exponent bits (top 31), 3 bits of mantissa, rounded up with the dropped part's probability."""
    a = x.abs().view(-1, BLOCK)
    e = (a.amax(1).view(torch.int32) + 0xFFFFF) >> 23
    y = (a.double() * _power(top - e)[:, None]).float().view(-1)
    code = ((y.view(torch.int32) + (draw << 4)) >> 20).clamp(max=(top + 1) * 8 - 1)
    code = torch.where(x < 0, code + 128, code) if top == 15 else torch.where(x > 0, code.clamp(min=1), code)
    return code.to(torch.uint8), e.to(torch.uint8)


def _decode(code, e, top):
    c = code.to(torch.int32)
    a = ((c & ((top + 1) * 8 - 1)) << 20).view(torch.float32).double().view(-1, BLOCK)
    x = (a * _power(e.to(torch.int64) - top)[:, None]).float().view(-1)
    return torch.where(c >= 128, -x, x) if top == 15 else x


def _plain_adamw(s):
    g = torch.cat([x for pair in zip((t.reshape(-1).float() for t in s['grads']), s['fill']) for x in pair])
    if s['clip'] > 0:
        norm = torch.sqrt(g.double().square().sum())
        g = g * (s['clip'] / (norm + 1e-6)).clamp(max=1.0).float()
    s['step'][0] += 1
    t = s['step'][:1].double()
    bc1, bc2 = 1.0 - BETA1 ** t, 1.0 - BETA2 ** t
    m, v = s['m'], s['v']
    if s['bits'] == 8:
        m, v = _decode(m, s['m_exp'], 15), _decode(v, s['v_exp'], 31)
    m = m * BETA1 + g * (1.0 - BETA1)
    v = v * BETA2 + (g * g) * (1.0 - BETA2)
    den = torch.sqrt(v) * (1.0 / torch.sqrt(bc2)).float() + ADAM_EPS
    s['p'].copy_(s['p'] * (1.0 - LR * DECAY) - (LR / bc1).float() * (m / den))
    if s['bits'] == 8:
        draw_ = _draws(s['seed'], s['step'][:1].to(torch.int64), m.numel())
        for name, x, top, d in (('m', m, 15, draw_ >> 16), ('v', v, 31, draw_ & 0xFFFF)):
            code, e = _encode(x, top, d)
            s[name].copy_(code)
            s[name + '_exp'].copy_(e)
        m, v = _decode(s['m'], s['m_exp'], 15), _decode(s['v'], s['v_exp'], 31)
    else:
        s['m'].copy_(m)
        s['v'].copy_(v)
    out = dict(p=s['p'], m=m, v=v)
    if s['copy'] is not None:
        s['copy'].copy_(s['p'])
        out['copy'] = s['copy']
    return out


_plain = dict(tokens=_plain_tokens, norm=_plain_norm, adamw=_plain_adamw)


# ---- the package's operators

def _own_tokens(s):
    T = importlib.import_module('dcss-auto_amd.tokens')
    r = T.token_logprobs(s['logits'], s['tokens'], mask=s['mask'], top=s['top'])
    out = dict(logp=r.logp, entropy=r.entropy)
    if s['top']:
        out.update(top_logp=r.top_logp, top_ids=r.top_ids)
    if s['grad']:
        out['dlogits'] = T.token_logprobs_bwd(s['logits'], s['tokens'], r, s['dlogp'], s['dentropy'], mask=s['mask'])
    return out


def _own_norm(s):
    N = importlib.import_module('dcss-auto_amd.norm')
    y, mean, rstd = N.layer_norm_fwd(s['x'], s['weight'], s['bias'], LN_EPS)
    out = dict(y=y)
    if s['grad']:
        out['dx'], out['dweight'], out['dbias'] = N.layer_norm_bwd(s['dy'], s['x'], s['weight'], s['bias'], mean, rstd)
    return out


def _own_adamw(s):
    A = importlib.import_module('dcss-auto_amd.optim')
    eight = s['bits'] == 8
    A.adamw_step(s['params'], s['grads'], s['ms'], s['vs'], s['step'], lr=LR, betas=(BETA1, BETA2), eps=ADAM_EPS,
                 weight_decay=DECAY, max_grad_norm=s['clip'], copies=s['copies'],
                 exps=(s['m_exps'], s['v_exps']) if eight else None, counters=s['at'] if eight else None,
                 seed=s['seed'])
    m, v = s['m'], s['v']
    if eight:
        m, v = A.read_moment(m, s['m_exp'], signed=True), A.read_moment(v, s['v_exp'], signed=False)
    out = dict(p=s['p'], m=m, v=v)
    if s['copy'] is not None:
        out['copy'] = s['copy']
    return out


_own = dict(tokens=_own_tokens, norm=_own_norm, adamw=_own_adamw)


# ---- what a pass cannot do without

def work(case):
    if case['op'] == 'tokens':
        n, k, b = case['rows'], case['vocab'], BYTES[case['dtype']]
        each = b * (2 if case['grad'] else 1) + (1 if case['mask'] else 0)
        # forward: difference, exponential, two sums; gradient: exponential and four products and sums
        return dict(bytes=n * (k * each + 16 + 12 * case['top'] + (8 if case['grad'] else 0)),
                    flops=n * k * (6 + (7 if case['grad'] else 0)))
    if case['op'] == 'norm':
        n, d, b = case['rows'], case['width'], BYTES[case['dtype']]
        return dict(bytes=n * d * b * (4 if case['grad'] else 2) + d * BYTES[case['weights']] * (4 if case['grad'] else 2),
                    flops=n * d * (8 + (12 if case['grad'] else 0)))
    n = sum(math.prod(x) for x in _shapes(case))
    each = 8 + BYTES[case['grads']] + (16 if case['bits'] == 32 else 4 + 4 / BLOCK + 8) + (2 if case['copy'] else 0)
    return dict(bytes=n * each, flops=n * (16 + (2 if case['clip'] else 0)))


# ---- the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case['op'] == 'tokens':
        return _exact_tokens(s)
    return _exact_norm(s) if case['op'] == 'norm' else _exact_adamw(s, case)


def _exact_tokens(s):
    z = s['logits'].to(torch.float64)
    n, k = z.shape
    if s['mask'] is not None:
        z = z.masked_fill(~s['mask'], -math.inf)
    some = z.amax(1) > -math.inf
    z[~some] = 0.0                                  # any finite row: replaced below
    ls = torch.log_softmax(z, 1)
    entropy = torch.special.entr(ls.exp()).sum(1).masked_fill(~some, 0.0)
    pad = s['tokens'] < 0
    index = s['tokens'].masked_fill(pad, 0)
    logp = ls[torch.arange(n, device=DEV), index].masked_fill(~some, -math.inf).masked_fill(pad, 0.0)
    out = dict(logp=logp, entropy=entropy)
    if s['top']:
        out['top_logp'] = ls.topk(s['top'], 1).values.masked_fill(~some[:, None], -math.inf)
        out['top_ids'] = None
    if s['grad']:
        g = s['dlogp'].double().masked_fill(pad, 0.0)
        h = s['dentropy'].double()
        prob = ls.exp()
        d = -torch.nan_to_num(ls, neginf=0.0).add_(entropy[:, None]).mul_(h[:, None]).add_(g[:, None]).mul_(prob)
        d[torch.arange(n, device=DEV), index] += g
        d[~some] = 0.0
        if s['mask'] is not None:
            d.masked_fill_(~s['mask'], 0.0)
        out['dlogits'] = d
    return out


def _exact_norm(s):
    x, w, b = (s[name].to(torch.float64) for name in ('x', 'weight', 'bias'))
    var, mu = torch.var_mean(x, -1, correction=0, keepdim=True)
    inv = torch.rsqrt(var + LN_EPS)
    out = dict(y=torch.addcmul(b, (x - mu) * inv, w))
    if s['grad']:
        n, d = x.shape
        dy, hat = s['dy'].to(torch.float64), (x - mu).mul_(inv)
        u = dy * w
        c1, c2 = u.sum(-1, keepdim=True) / d, (u * hat).sum(-1, keepdim=True) / d
        out.update(dx=(u - c1 - hat * c2) * inv, dweight=(dy * hat).sum(0), dbias=dy.sum(0))
    return out


def _exact_word(values):
    for shift, factor in ((16, 0x9E3779B1), (15, 0xB7E15163), (16, 1)):
        values = torch.bitwise_xor(values, values.div(1 << shift, rounding_mode='floor'))
        values = torch.remainder(values * factor, 1 << 32)
    return values


def _exact_round(x, top, chance):
    """The 8-bit value that stands for x: on a grid of eighths of its binade (of the lowest binade's
    below that), the next step up where the position between two steps and `chance` pass one."""
    rows = x.abs().reshape(-1, BLOCK)
    frac, e = torch.frexp(rows.amax(1, keepdim=True))           # amax = frac * 2^e, frac in [1/2, 1)
    e = torch.where(frac > 15 / 16, e + 1, e)                    # so that rounding up stays inside
    mine = torch.maximum(torch.frexp(rows).exponent, e - top + 1)   # the lowest full binade is top - 1 below
    step = torch.exp2((mine - 4).double())
    q = torch.floor(rows / step + chance.reshape(-1, BLOCK))
    if top == 31:
        q = torch.where((rows > 0) & (q < 1), 1.0, q)
    return (q * step).reshape(-1) * torch.sign(x)


def _exact_adamw(s, case):
    total = s['p'].numel()
    g = torch.zeros(total, dtype=torch.float64, device=DEV)
    for o, t in zip(s['at'], s['grads']):
        g[o:o + t.numel()] = t.reshape(-1).to(torch.float64)
    if case['clip'] > 0:
        norm = float(torch.linalg.vector_norm(g))
        g *= min(1.0, case['clip'] / (norm + 1e-6))
    t = int(s['step'][0]) + 1
    if case['bits'] == 8:
        m, v = (_decode(s[name], s[name + '_exp'], top).double() for name, top in (('m', 15), ('v', 31)))
    else:
        m, v = s['m'].double(), s['v'].double()
    m.lerp_(g, 1 - BETA1)
    v.mul_(BETA2).addcmul_(g, g, value=1 - BETA2)
    p = s['p'].double()
    p = p - LR * DECAY * p - LR * (m / (1 - BETA1 ** t)) / (torch.sqrt(v / (1 - BETA2 ** t)) + ADAM_EPS)
    if case['bits'] == 8:
        one = lambda x: torch.tensor([x], dtype=torch.int64, device=DEV)  # noqa: E731
        key = _exact_word(one(s['seed'] % (1 << 32)))
        key = _exact_word(torch.bitwise_xor(key, one(s['seed'] // (1 << 32))))
        key = _exact_word(_exact_word(torch.bitwise_xor(key, one(t))))
        word = _exact_word(torch.bitwise_xor(torch.arange(total, device=DEV), key))
        m = _exact_round(m, 15, word.div(65536, rounding_mode='floor').double() / 65536)
        v = _exact_round(v, 31, torch.remainder(word, 65536).double() / 65536)
    out = dict(p=p, m=m, v=v)
    if case['copy']:
        out['copy'] = p
    return out
