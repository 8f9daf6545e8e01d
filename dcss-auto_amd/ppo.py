"""PPO update over a resident rollout buffer.

Follows the reference's update (gpu-d1/scripts/run_ring_ablations.py:354-372;
gpu-d1/scripts/train_clear.py:149-172): reverse-time GAE, advantages normalised over
the whole buffer (unbiased std + 1e-8), then `epochs` passes of shuffled minibatches
with the clipped surrogate, a value loss and an entropy bonus, gradient-norm clipping
at 0.5 and Adam (lr 3e-4, eps 1e-5). C4's coefficients are clip 0.2, value 0.5 x
(0.5 * MSE) — the reference's 0.25 * MSE — and entropy 0.01. The trunk runs under bf16
autocast while the optimizer keeps fp32 master weights; GAE is the HIP kernel.
"""
import torch

from . import policy as P
from .losses import PolicyLoss, clip_pair, policy_loss
from .optim import AdamW, MuonAdamW

OBS = P.OBS
KERNEL_TYPES = (torch.float32, torch.bfloat16, torch.float16)        # of losses.policy_loss


class RolloutBuffer:
    """[T, N] rollout storage; observations stay uint8 (15.1 GB at T=128, N=65,536)."""

    def __init__(self, T, N, device='cuda', obs_bytes=OBS):
        self.T, self.N = T, N
        self.obs = torch.empty((T, N, obs_bytes), dtype=torch.uint8, device=device)
        self.actions = torch.zeros((T, N), dtype=torch.int64, device=device)
        self.logp = torch.zeros((T, N), dtype=torch.float32, device=device)
        self.values = torch.zeros((T, N), dtype=torch.float32, device=device)
        self.rewards = torch.zeros((T, N), dtype=torch.float32, device=device)
        self.dones = torch.zeros((T, N), dtype=torch.uint8, device=device)
        self.bootstrap = torch.zeros(N, dtype=torch.float32, device=device)


def ppo_loss(logits, values, actions, old_logp, adv, returns, clip=0.2, vcoef=0.5, ecoef=0.01):
    """Clipped surrogate + vcoef * 0.5*MSE - ecoef * entropy, in fp32 (logits upcast)."""
    logp_all = torch.log_softmax(logits.float(), -1)
    logp = logp_all.gather(1, actions[:, None]).squeeze(1)
    ratio = torch.exp(logp - old_logp)
    pg = -torch.minimum(ratio * adv, ratio.clamp(1 - clip, 1 + clip) * adv).mean()
    vloss = 0.5 * (values.float() - returns).square().mean()
    entropy = -(logp_all.exp() * logp_all).sum(-1).mean()
    return pg + vcoef * vloss - ecoef * entropy, pg.detach(), vloss.detach(), entropy.detach()


def broadcast_loss(logp, old_logp, adv, ref_logp, entropy, values, returns, old_values, clip, kl_coef, value_coef, value_clip,
                   entropy_coef):
    """losses.policy_loss in elementary operations, for results that are not all of logp's shape and of a type the kernel takes:
    each term is the mean over what broadcasting makes of it. clip: (low, high)."""
    gap = logp - old_logp
    ratio = torch.exp(gap)
    free, held = ratio * adv, ratio.clamp(1 - clip[0], 1 + clip[1]) * adv
    policy = -torch.minimum(free, held).mean()
    far = (values.float() - returns).square()
    if value_clip:
        near = old_values + (values.float() - old_values).clamp(-value_clip, value_clip)
        far = torch.maximum(far, (near - returns).square())
    value, entropy = 0.5 * far.mean(), entropy.mean()
    loss, kl = policy + value_coef * value - entropy_coef * entropy, policy.new_zeros(())
    if ref_logp is not None:
        x = ref_logp - logp
        kl = (x.exp() - 1 - x).mean()
        loss = loss + kl_coef * kl
    parts = loss, policy, value, entropy, kl, (held < free).float().mean(), (ratio - 1 - gap).mean(), torch.full_like(loss, gap.numel())
    terms = torch.stack([t.detach().float() for t in parts])
    return PolicyLoss(loss, *terms.unbind()[1:], terms)


class PPO:
    def __init__(self, model, lr=3e-4, eps=1e-5, clip=0.2, vcoef=0.5, ecoef=0.01, max_grad_norm=0.5,
                 epochs=4, minibatch=8192, gamma=0.99, lam=0.95, autocast=True):
        self.model = model
        self.opt = self._optimizer(lr, eps)
        self.clip, self.vcoef, self.ecoef, self.max_grad_norm = clip, vcoef, ecoef, max_grad_norm
        self.epochs, self.minibatch, self.gamma, self.lam, self.autocast = epochs, minibatch, gamma, lam, autocast

    def _optimizer(self, lr, eps):
        return torch.optim.Adam(self.model.parameters(), lr=lr, eps=eps, fused=True)

    def advantages(self, buf):
        adv, ret = P.gae(buf.rewards, buf.dones, buf.values, buf.bootstrap, self.gamma, self.lam)
        flat = adv.flatten()
        return (flat - flat.mean()) / (flat.std() + 1e-8), ret.flatten()

    def minibatch_step(self, obs, actions, old_logp, adv, ret):
        with torch.autocast('cuda', dtype=torch.bfloat16, enabled=self.autocast):
            logits, value = self.model(obs)
        loss, pg, vl, ent = ppo_loss(logits, value, actions, old_logp, adv, ret, self.clip, self.vcoef, self.ecoef)
        if not torch.isfinite(loss).item():   # as the reference's update loop (run_ring_ablations.py:369-370)
            raise RuntimeError('Non-finite PPO loss')
        self.opt.zero_grad(set_to_none=True)
        loss.backward()
        torch.nn.utils.clip_grad_norm_(self.model.parameters(), self.max_grad_norm)
        self.opt.step()
        return loss.detach()

    def update(self, buf, generator=None):
        adv, ret = self.advantages(buf)
        n = buf.T * buf.N
        obs = buf.obs.view(n, -1)
        actions, logp = buf.actions.flatten(), buf.logp.flatten()
        last = None
        for _ in range(self.epochs):
            perm = torch.randperm(n, device=obs.device, generator=generator)
            for inds in perm.split(self.minibatch):
                last = self.minibatch_step(obs.index_select(0, inds), actions[inds], logp[inds], adv[inds],
                                           ret[inds])
        return last


class ModulePPO(PPO):
    """PPO for any policy module with evaluate(obs, actions) -> (log probability, entropy, value), such as
    NormPolicy and ARPolicy: the module's layers by autograd, its log probabilities, layer norms, the loss and the
    update itself by this package's kernels. Interface and loss are PPO's; the optimizer is AdamW over all
    tensors at once (state_bits: 32 or 8) with the gradient clip in the same call, or with optimizer='muon' Muon (lr muon_lr) for
    the trunk's matrices and AdamW for the rest (MuonAdamW; the clip is then by the norm of the rest's gradients). What `evaluate` gives need
    not have the same shapes and types: with others than the loss's kernel takes (an entropy that is one number, a value that broadcasts, 64
    bits) the loss is elementary operations. clip may be a pair (low, high), value_clip holds the new value
    within that much of the old one; with `reference`, a policy that is left as it is, kl_coef times the KL to
    it is added to the loss. `terms`: the last minibatch's loss in its parts (losses.PolicyLoss). Nothing waits
    for the device between minibatches: a minibatch whose gradient norm is not finite changes nothing,
    and `update` raises at its end."""

    def __init__(self, model, lr=3e-4, eps=1e-5, clip=0.2, vcoef=0.5, ecoef=0.01, max_grad_norm=0.5, epochs=4,
                 minibatch=8192, gamma=0.99, lam=0.95, autocast=True, weight_decay=0.0, state_bits=32, seed=0, value_clip=None,
                 kl_coef=0.0, reference=None, optimizer='adamw', muon_lr=0.02):
        if not max_grad_norm > 0:
            raise ValueError('ModulePPO needs a gradient clip: its norm is what tells a non-finite loss')
        if optimizer not in ('adamw', 'muon'):
            raise ValueError(f"optimizer is 'adamw' or 'muon', not {optimizer!r}")
        if kl_coef and reference is None:
            raise ValueError('kl_coef needs a reference')
        self._adamw = dict(weight_decay=weight_decay, state_bits=state_bits, max_grad_norm=max_grad_norm, seed=seed)
        self._muon = dict(lr=muon_lr, weight_decay=weight_decay) if optimizer == 'muon' else None
        self.value_clip, self.kl_coef, self.reference, self.terms = value_clip, kl_coef, reference, None
        super().__init__(model, lr=lr, eps=eps, clip=clip, vcoef=vcoef, ecoef=ecoef, max_grad_norm=max_grad_norm,
                         epochs=epochs, minibatch=minibatch, gamma=gamma, lam=lam, autocast=autocast)

    def _optimizer(self, lr, eps):
        adamw = dict(lr=lr, eps=eps, **self._adamw)
        if self._muon is None:
            return AdamW(self.model.parameters(), **adamw)
        return MuonAdamW(self.model.named_parameters(), muon=self._muon, adamw=adamw)

    def _evaluate(self, evaluate, *args):
        with torch.autocast('cuda', dtype=torch.bfloat16, enabled=self.autocast):
            return evaluate(*args)

    def _learn(self, evaluated, ref_logp, old_logp, adv, ret, old_values):
        logp, entropy, value = evaluated
        low, high = clip_pair(self.clip)
        settings = dict(clip=(min(low, 1.0), high), kl_coef=self.kl_coef, value_coef=self.vcoef, value_clip=self.value_clip,
                        entropy_coef=self.ecoef)                      # a ratio is never under 0
        alike = [t for t in (logp, entropy, value, ref_logp) if t is not None]
        loss = policy_loss if all(t.shape == old_logp.shape and t.dtype in KERNEL_TYPES for t in alike) else broadcast_loss
        r = loss(logp, old_logp, adv, ref_logp=ref_logp, entropy=entropy, values=value, returns=ret, old_values=old_values, **settings)
        self.opt.zero_grad(set_to_none=True)
        r.loss.backward()
        self.opt.step()
        self.terms = r._replace(loss=r.loss.detach())
        return self.terms.loss

    def minibatch_step(self, obs, actions, old_logp, adv, ret, old_values=None):
        evaluated = self._evaluate(self.model.evaluate, obs, actions)
        ref_logp = None
        if self.kl_coef:
            with torch.no_grad():
                ref_logp = self._evaluate(self.reference.evaluate, obs, actions)[0]
        return self._learn(evaluated, ref_logp, old_logp, adv, ret, old_values)

    def _epochs(self, buf, generator):
        if self.value_clip is None:
            return super().update(buf, generator)
        adv, ret = self.advantages(buf)
        n = buf.T * buf.N
        obs, last = buf.obs.view(n, -1), None
        flat = buf.actions.flatten(), buf.logp.flatten(), adv, ret, buf.values.flatten()
        for _ in range(self.epochs):
            perm = torch.randperm(n, device=obs.device, generator=generator)
            for inds in perm.split(self.minibatch):
                last = self.minibatch_step(obs.index_select(0, inds), *(t[inds] for t in flat))
        return last

    def update(self, buf, generator=None):
        before = self.opt.skipped_steps()
        last = self._epochs(buf, generator)
        if self.opt.skipped_steps() > before:
            raise RuntimeError('Non-finite PPO loss')
        return last


class SequenceBuffer(RolloutBuffer):
    """A rollout of a policy with memory: also its state before the first step and where episodes began."""

    def __init__(self, T, N, width, device='cuda', obs_bytes=OBS):
        super().__init__(T, N, device, obs_bytes)
        self.state = torch.zeros((N, width), dtype=torch.float32, device=device)
        self.resets = torch.zeros((T, N), dtype=torch.uint8, device=device)


class SequencePPO(ModulePPO):
    """ModulePPO for a policy with memory (MemoryPolicy), over a SequenceBuffer: a minibatch is the whole rollout of some worlds,
    minibatch // T of them (one at least), whose states are made again from the one before the rollout through
    evaluate_sequence(obs, actions, state, resets). A reference's memory begins empty with each rollout."""

    def sequence_step(self, obs, actions, old_logp, adv, ret, state, resets, old_values=None):
        """One minibatch of sequences: obs [T, n, ...], the others [T, n], state [n, width]."""
        evaluated = self._evaluate(self.model.evaluate_sequence, obs, actions, state, resets)
        ref_logp = None
        if self.kl_coef:
            with torch.no_grad():
                ref_logp = self._evaluate(self.reference.evaluate_sequence, obs, actions, torch.zeros_like(state), resets)[0]
        return self._learn(evaluated, ref_logp, old_logp, adv, ret, old_values)

    def _epochs(self, buf, generator):
        adv, ret = (x.view(buf.T, buf.N) for x in self.advantages(buf))
        per, last = max(1, self.minibatch // buf.T), None
        for _ in range(self.epochs):
            perm = torch.randperm(buf.N, device=buf.obs.device, generator=generator)
            for w in perm.split(per):
                pick = lambda x: x.index_select(1, w)  # noqa: E731
                last = self.sequence_step(pick(buf.obs), pick(buf.actions), pick(buf.logp), pick(adv), pick(ret), buf.state[w],
                                          pick(buf.resets), pick(buf.values) if self.value_clip is not None else None)
        return last


# ----------------------------------------------------------------------------------------
# Graph-safe PPO: one libd1hip call (d1_ppo_step) per minibatch over flat parameter buffers.
# The step picks its minibatch from a device-side cursor, so a HIP graph holding several
# calls walks consecutive minibatches of the epoch's sample order.

_PARAMS = (('l1.weight', (256, 1800)), ('l1.bias', (256,)), ('l2.weight', (256, 256)), ('l2.bias', (256,)),
           ('head.weight', (17, 256)), ('head.bias', (17,)))


class FlatParams:
    """fp32 master weights, their bf16 copy, bf16 gradients and Adam moments, each one
    flat buffer; segments start on 64-element boundaries."""

    def __init__(self, policy, device):
        self.offsets, off = {}, 0
        for name, shape in _PARAMS:
            numel = 1
            for d in shape:
                numel *= d
            self.offsets[name] = (off, shape, numel)
            off += (numel + 63) // 64 * 64
        self.n = off
        self.p = torch.zeros(off, dtype=torch.float32, device=device)
        state = policy.state_dict()
        for name, (o, shape, numel) in self.offsets.items():
            self.p[o:o + numel].copy_(state[name].reshape(-1).float())
        self.pb = self.p.to(torch.bfloat16)
        self.g = torch.zeros(off, dtype=torch.bfloat16, device=device)
        self.m = torch.zeros(off, dtype=torch.float32, device=device)
        self.v = torch.zeros(off, dtype=torch.float32, device=device)

    def view(self, buf, name):
        o, shape, numel = self.offsets[name]
        return buf[o:o + numel].view(shape)

    def load_into(self, policy):
        with torch.no_grad():
            for name, (o, shape, numel) in self.offsets.items():
                dict(policy.named_parameters())[name].copy_(self.p[o:o + numel].view(shape))


class FastPPO:
    """PPO update with the minibatch step in libd1hip (four kernels: fused per-sample
    forward/loss/backward, grouped split-K weight gradients, fixed-order reduction, clip +
    Adam). Same interface and semantics as PPO with bf16 autocast; `minibatch` must be a
    multiple of 1024. With graph=True, `graph_steps` consecutive minibatch steps are
    captured in one HIP graph per buffer and replayed.

    A minibatch whose loss or gradient norm is not finite changes nothing, and neither does
    any later one until `clear_nonfinite()`; `update` then raises RuntimeError, as the
    reference's loop does at the first non-finite loss (run_ring_ablations.py:369-370),
    leaving the weights and Adam state of the last finite step."""

    def __init__(self, policy, lr=3e-4, eps=1e-5, clip=0.2, vcoef=0.5, ecoef=0.01, max_grad_norm=0.5,
                 epochs=4, minibatch=8192, gamma=0.99, lam=0.95, graph=True, graph_steps=16):
        from . import _lib
        if minibatch <= 0 or minibatch % 1024:
            raise ValueError('FastPPO needs a minibatch that is a multiple of 1024')
        dev = next(policy.parameters()).device
        self.flat = F = FlatParams(policy, dev)
        self.lr, self.eps, self.clip, self.vcoef, self.ecoef = lr, eps, clip, vcoef, ecoef
        self.max_grad_norm, self.epochs, self.minibatch, self.gamma, self.lam = max_grad_norm, epochs, minibatch, gamma, lam
        self.graph, self.graph_steps, self.dev = graph, graph_steps, dev
        self.step_t = torch.zeros(3, dtype=torch.float32, device=dev)   # Adam step, scratch, skipped steps
        self.cursor = torch.zeros(2, dtype=torch.int32, device=dev)
        self.loss_parts = torch.zeros(minibatch // 32 * 4, dtype=torch.float32, device=dev)
        nbytes = _lib.load().d1_ppo_work_bytes(minibatch)
        _lib.check(0 if nbytes > 0 else nbytes, 'd1_ppo_work_bytes')
        self.work = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        self.perm = None
        self.head_out = None   # [minibatch, 17] fp32: when set, each step writes its head outputs here
        self._packed = False
        self._g = self._g_buf = self._g_key = self._adv = self._ret = None
        self._args = self._args_key = None

    def _key(self, obs, actions, logp, adv, ret):
        """What a step's launches hold: the addresses they read and write, and the sample count."""
        return (obs.data_ptr(), actions.data_ptr(), logp.data_ptr(), adv.data_ptr(), ret.data_ptr(),
                self.perm.data_ptr(), obs.shape[0], 0 if self.head_out is None else self.head_out.data_ptr())

    def _struct(self, obs, actions, logp, adv, ret):
        from . import _lib
        key = self._key(obs, actions, logp, adv, ret)
        if self._args_key != key:
            F = self.flat
            if obs.shape[1] != OBS or not obs.is_contiguous() or obs.dtype != torch.uint8:
                raise ValueError('observations must be contiguous uint8 [n, 1800]')
            off = {name: o for name, (o, _, _) in F.offsets.items()}
            self._args = _lib.D1PPOStep(
                obs=obs.data_ptr(), perm=self.perm.data_ptr(), cursor=self.cursor.data_ptr(),
                actions=actions.data_ptr(), logp_old=logp.data_ptr(), adv=adv.data_ptr(), ret=ret.data_ptr(),
                n=obs.shape[0], mb=self.minibatch, p=F.p.data_ptr(), pb=F.pb.data_ptr(), g=F.g.data_ptr(),
                m=F.m.data_ptr(), v=F.v.data_ptr(), nparams=F.n, off_w1=off['l1.weight'], off_b1=off['l1.bias'],
                off_w2=off['l2.weight'], off_b2=off['l2.bias'], off_w3=off['head.weight'],
                off_b3=off['head.bias'], step=self.step_t.data_ptr(), loss_parts=self.loss_parts.data_ptr(), work=self.work.data_ptr(),
                work_bytes=self.work.numel(), clip=self.clip, vcoef=self.vcoef, ecoef=self.ecoef,
                max_grad_norm=self.max_grad_norm, lr=self.lr, beta1=0.9, beta2=0.999, eps=self.eps,
                z_out=None if self.head_out is None else self.head_out.data_ptr())
            self._args_key = key
        if not self._packed:   # kernel-ordered weight copies in the work buffer, from pb
            _lib.check(_lib.load().d1_ppo_prepare(self._args, torch.cuda.current_stream(self.dev).cuda_stream),
                       'd1_ppo_prepare')
            self._packed = True
        return self._args

    def record_head(self, on=True):
        """Have every following minibatch step write the head outputs its loss was computed
        from (16 logits + value, bf16-rounded, as fp32) into self.head_out [minibatch, 17]
        (NaN until a step writes it). A captured graph holds the buffer it was captured
        with, so this drops it and the next update captures again."""
        self._g = self._g_buf = None
        self.head_out = torch.full((self.minibatch, 17), float('nan'), device=self.dev) if on else None

    def set_order(self, perm):
        """Sample order of the next minibatches (int64 [n] on the device); resets the cursor
        so the next step takes perm[0:minibatch]."""
        if self.perm is None or self.perm.shape != perm.shape:
            self.perm = torch.empty_like(perm, dtype=torch.int64)
        if perm is not self.perm:
            self.perm.copy_(perm)
        self.cursor.zero_()

    def _step(self, obs, actions, logp, adv, ret):
        """One minibatch: samples perm[cursor*mb : (cursor+1)*mb]; advances the cursor."""
        from . import _lib
        args = self._struct(obs, actions, logp, adv, ret)
        _lib.check(_lib.load().d1_ppo_step(args, torch.cuda.current_stream(self.dev).cuda_stream), 'd1_ppo_step')

    def nonfinite_steps(self):
        """Minibatch steps skipped since the first non-finite loss or gradient norm."""
        return int(self.step_t[2].item())

    def clear_nonfinite(self):
        self.step_t[2].zero_()

    def loss_terms(self):
        """(pg, value, entropy) means of the last minibatch (reads device partials)."""
        return self.loss_parts.view(-1, 4)[:, :3].sum(0) / self.minibatch

    def _views(self, buf):
        n = buf.T * buf.N
        return buf.obs.view(n, -1), buf.actions.view(n), buf.logp.view(n)

    def _graph_len(self, n):
        steps = n // self.minibatch
        k = max(1, min(self.graph_steps, steps))
        while steps % k:
            k -= 1
        return k

    def _capture(self, buf):
        n = buf.T * buf.N
        if n < self.minibatch:
            raise ValueError('the buffer holds fewer samples than one minibatch')
        if self._adv is None or self._adv.numel() != n:
            self._adv = torch.zeros(n, device=self.dev)
            self._ret = torch.zeros(n, device=self.dev)
        if self.perm is None or self.perm.shape != (n,):
            self.perm = torch.zeros(n, dtype=torch.int64, device=self.dev)
        obs, actions, logp = self._views(buf)
        args = self._struct(obs, actions, logp, self._adv, self._ret)
        torch.cuda.synchronize(self.dev)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            for _ in range(self._graph_len(n)):
                self._step(obs, actions, logp, self._adv, self._ret)
        self._g, self._g_buf, self._g_args = g, buf, args
        self._g_key = self._key(obs, actions, logp, self._adv, self._ret)

    def advantages(self, buf, adv=None, ret=None):
        """The buffer's normalised advantages and its returns, flat (written to `adv` and `ret`
        when given: contiguous fp32 of the rewards' size)."""
        n, device = buf.rewards.numel(), buf.rewards.device   # what the GAE kernel writes, whatever T and N say
        adv, ret = (torch.empty(n, dtype=torch.float32, device=device) if t is None else t for t in (adv, ret))
        for t in (adv, ret):
            if not (t.dtype == torch.float32 and t.is_contiguous() and t.numel() == n and t.device == device):
                raise ValueError('adv and ret must be contiguous fp32 of the size of the rewards, on their device')
        return self._advantages(buf, adv, ret)

    def _advantages(self, buf, adv, ret):
        P.gae(buf.rewards, buf.dones, buf.values, buf.bootstrap, self.gamma, self.lam, adv=adv, returns=ret)
        return P.normalize_(adv), ret

    def update(self, buf, generator=None):
        n = buf.T * buf.N
        obs, actions, logp = self._views(buf)
        if self.graph:
            if self._g is None or self._g_buf is not buf:
                self._capture(buf)
            if _is(self.advantages, _ADVANTAGES):
                if buf.rewards.numel() != n or buf.rewards.device != self._adv.device:
                    raise ValueError('the buffer holds another number of rewards than T x N, or on another device')
                adv, ret = self._advantages(buf, self._adv, self._ret)
            else:   # replaced by the program, as advantages(buf)
                for mine, given in zip((self._adv, self._ret), self.advantages(buf)):
                    mine.copy_(given)
                adv, ret = self._adv, self._ret
            # the graph holds addresses: another order buffer (set_order with another size) or a
            # tensor of the buffer that was replaced needs a new one (looked at once GAE is queued)
            if self.perm.shape != (n,) or self._g_key != self._key(obs, actions, logp, adv, ret):
                self._capture(buf)
            if not self._packed:   # weights replaced outside the step (a checkpoint load): the graph
                self._struct(obs, actions, logp, adv, ret)   # only replays, so rebuild its weight copies here
        else:
            adv, ret = self.advantages(buf)
            if self.perm is None or self.perm.shape != (n,):
                self.perm = torch.empty(n, dtype=torch.int64, device=self.dev)
        steps = n // self.minibatch            # a ragged tail is dropped (T*N is a multiple in C4)
        for _ in range(self.epochs):
            if _is(self.set_order, _SET_ORDER):   # straight into the order buffer
                self.set_order(torch.randperm(n, out=self.perm, generator=generator))
            else:   # replaced by the program: an order of its own, which it may keep
                self.set_order(torch.randperm(n, device=self.dev, generator=generator))
            if self.graph:
                for _ in range(steps // self._graph_len(n)):
                    self._g.replay()
            else:
                for _ in range(steps):
                    self._step(obs, actions, logp, adv, ret)
        terms = self.loss_terms()   # queued before the wait for the step counter
        if self.nonfinite_steps():
            raise RuntimeError('Non-finite PPO loss')
        return terms


def _is(method, function):
    """Whether a bound method is `function` itself, not one that a subclass, an instance or a patched
    class puts in its place."""
    return getattr(method, '__func__', None) is function


_ADVANTAGES, _SET_ORDER = FastPPO.advantages, FastPPO.set_order
