"""Loads libd1hip.so (built in-tree by build.py) and declares its C ABI (include/d1hip.h) and the
entry points only this package calls (csrc/d1_internal.h); likewise libd1ops.so (include/d1ops.h)
and the learning task's libraries.

There is no fallback: without the built library every entry point raises."""
import ctypes as C
import importlib
import pathlib

HERE = pathlib.Path(__file__).resolve().parent
LIB_PATH = HERE / 'libd1hip.so'
_LIB = None

SYMBOLS = ('d1_state_bytes', 'd1_obs_bytes', 'd1_action_size', 'd1_out_size', 'd1_config_bytes',
           'd1_init', 'd1_step', 'd1_heuristic', 'd1_sample', 'd1_sample_dev', 'd1_gae', 'd1_obs_to_bf16', 'd1_obs_d4',
           'd1_ppo_work_bytes', 'd1_ppo_prepare', 'd1_ppo_step', 'd1_ppo_step_static', 'd1_wait_bytes', 'd1_wait_init', 'd1_wait_run',
           'd1_sample_ar', 'd1_los_table', 'd1_distance_rows', 'd1_policy_packed_elems', 'd1_policy_pack',
           'd1_policy_fwd', 'd1_policy_fwd_sample', 'd1_policy_ar_packed_elems', 'd1_policy_ar_pack',
           'd1_policy_fwd_sample_ar')
LEARN_SYMBOLS = ('learn_turn_cost', 'learn_return_gamma', 'learn_state_bytes', 'learn_obs_size',
                 'learn_action_size', 'learn_out_size', 'learn_config_bytes', 'learn_init', 'learn_step',
                 'learn_step_active', 'learn_heuristic')
OPS_SYMBOLS = ('d1_tokens_work_bytes', 'd1_tokens_fwd', 'd1_tokens_bwd', 'd1_norm_fwd', 'd1_norm_work_bytes',
               'd1_norm_bwd', 'd1_adamw_work_bytes', 'd1_adamw_step', 'd1_adamw_step_with', 'd1_adamw_read', 'd1_policy_loss_work_bytes',
               'd1_policy_loss', 'd1_scale', 'd1_scale_to', 'd1_scan_marks', 'd1_scan_work_bytes', 'd1_scan_fwd', 'd1_scan_bwd',
               'd1_muon_check', 'd1_muon_work_bytes', 'd1_muon_step')
_LEARN = {}
_OPS = _OPS_TORCH = None


class D1PPOStep(C.Structure):
    """The D1PPOStep struct of include/d1hip.h (one PPO minibatch update)."""
    _fields_ = [('obs', C.c_void_p), ('perm', C.c_void_p), ('cursor', C.c_void_p), ('actions', C.c_void_p),
                ('logp_old', C.c_void_p), ('adv', C.c_void_p), ('ret', C.c_void_p), ('n', C.c_int64),
                ('mb', C.c_int32), ('pad0', C.c_int32), ('p', C.c_void_p), ('pb', C.c_void_p),
                ('g', C.c_void_p), ('m', C.c_void_p), ('v', C.c_void_p), ('nparams', C.c_int64),
                ('off_w1', C.c_int64), ('off_b1', C.c_int64), ('off_w2', C.c_int64), ('off_b2', C.c_int64),
                ('off_w3', C.c_int64), ('off_b3', C.c_int64), ('step', C.c_void_p), ('loss_parts', C.c_void_p), ('work', C.c_void_p),
                ('work_bytes', C.c_int64), ('clip', C.c_float), ('vcoef', C.c_float), ('ecoef', C.c_float),
                ('max_grad_norm', C.c_float), ('lr', C.c_float), ('beta1', C.c_float), ('beta2', C.c_float),
                ('eps', C.c_float), ('z_out', C.c_void_p)]


def load():
    global _LIB
    if _LIB is None:
        if not LIB_PATH.exists():
            raise RuntimeError(f'{LIB_PATH} is missing: build it with __graft_entry__.build() '
                               '(the D:1 environment has no CPU fallback)')
        L = C.CDLL(str(LIB_PATH))
        p, i = C.c_void_p, C.c_int
        L.d1_state_bytes.argtypes = [i]
        for name in ('d1_obs_bytes', 'd1_action_size', 'd1_out_size', 'd1_config_bytes'):
            getattr(L, name).argtypes = []
        L.d1_init.argtypes = [p, i, i, p, p, C.c_uint64, p, p, p]
        L.d1_step.argtypes = [p, i, i, p, p, p, p, p, p, p, p]
        L.d1_step_into.argtypes = [p, i, i, p, p, p, p, p, p, p, p, p]
        L.d1_heuristic.argtypes = [p, i, i, p, i, p, p]
        L.d1_sample.argtypes = [p, i, i, i, C.c_uint64, C.c_uint32, p, p, p]
        L.d1_sample_dev.argtypes = [p, i, i, i, C.c_uint64, p, C.c_uint32, p, p, p]
        L.d1_obs_to_bf16.argtypes = [p, p, C.c_int64, p]
        L.d1_obs_d4.argtypes = [p, p, i, p, p]
        L.d1_ppo_work_bytes.argtypes = [i]
        L.d1_ppo_work_bytes.restype = C.c_int64
        L.d1_ppo_step.argtypes = [C.POINTER(D1PPOStep), p]
        L.d1_ppo_prepare.argtypes = [C.POINTER(D1PPOStep), p]
        L.d1_ppo_step_static.argtypes = [C.POINTER(D1PPOStep), p]
        L.d1_sample_ar.argtypes = [p, i, i, p, i, i, i, C.c_uint64, C.c_uint32, p, p, p, p, p]
        L.d1_wait_bytes.argtypes = []
        L.d1_wait_init.argtypes = [p, i, i, p, p, C.c_uint64, i, p]
        L.d1_wait_run.argtypes = [p, i, i, p, p, i, p, p]
        L.d1_gae.argtypes = [p, p, p, p, i, i, C.c_float, C.c_float, p, p, p]
        L.d1_adv_norm.argtypes = [p, C.c_int64, p, p, C.c_float, p]
        L.d1_los_table.argtypes = [p, i, p, p, p]
        L.d1_distance_rows.argtypes = [p, p, i, p, p]
        L.d1_policy_packed_elems.argtypes = []
        L.d1_policy_packed_elems.restype = C.c_int64
        L.d1_policy_pack.argtypes = [p, p, p, p, p]
        L.d1_policy_fwd.argtypes = [p, i, p, p, p, p, p, p, p]
        L.d1_policy_fwd_sample.argtypes = [p, i, p, p, p, p, C.c_uint64, p, C.c_uint32, p, p, p, p, p]
        L.d1_policy_ar_packed_elems.argtypes = []
        L.d1_policy_ar_packed_elems.restype = C.c_int64
        L.d1_policy_ar_pack.argtypes = [p, p, p, p, p, p, p, p]
        L.d1_policy_fwd_sample_ar.argtypes = [p, i, p, p, p, p, p, C.c_uint64, p, C.c_uint32, p, p, p, p, p, p, p, p]
        _LIB = L
    return _LIB


class D1AdamWTensor(C.Structure):
    """The D1AdamWTensor struct of include/d1ops.h (one tensor of an AdamW step)."""
    _fields_ = [('p', C.c_void_p), ('g', C.c_void_p), ('m', C.c_void_p), ('v', C.c_void_p), ('m_exp', C.c_void_p),
                ('v_exp', C.c_void_p), ('copy', C.c_void_p), ('n', C.c_int64), ('counter', C.c_int64),
                ('lr', C.c_double), ('weight_decay', C.c_double), ('lag', C.c_int32), ('ptype', C.c_uint8),
                ('gtype', C.c_uint8), ('pad', C.c_uint8 * 2)]


class D1AdamW(C.Structure):
    """The D1AdamW struct of include/d1ops.h."""
    _fields_ = [('beta1', C.c_double), ('beta2', C.c_double), ('eps', C.c_double), ('max_norm', C.c_double),
                ('seed', C.c_uint64), ('bits', C.c_int32), ('pad', C.c_int32)]


class D1LossInput(C.Structure):
    """The D1LossInput struct of include/d1ops.h."""
    _fields_ = [('data', C.c_void_p), ('row', C.c_int64), ('step', C.c_int64), ('type', C.c_int32), ('pad', C.c_int32)]


class D1PolicyLoss(C.Structure):
    """The D1PolicyLoss struct of include/d1ops.h."""
    _fields_ = [*((name, D1LossInput) for name in ('logp', 'old_logp', 'advantages', 'ref_logp', 'entropy', 'values', 'returns',
                                                   'old_values', 'mask')),
                ('rows', C.c_int64), ('length', C.c_int64), ('clip_low', C.c_double), ('clip_high', C.c_double),
                ('value_clip', C.c_double), ('kl_coef', C.c_double), ('value_coef', C.c_double), ('entropy_coef', C.c_double),
                ('sequence', C.c_int32), ('fp32_grads', C.c_int32)]


class D1Scan(C.Structure):
    """The D1Scan struct of include/d1ops.h."""
    _fields_ = [('x', C.c_void_p), ('gate', C.c_void_p), ('reset', C.c_void_p), ('state', C.c_void_p), ('marks', C.c_void_p),
                *((name, C.c_int64) for name in ('x_t', 'x_n', 'gate_t', 'gate_n', 'reset_t', 'reset_n', 'steps', 'rows')),
                ('width', C.c_int32), ('type', C.c_int32)]


class D1MuonTensor(C.Structure):
    """The D1MuonTensor struct of include/d1ops.h."""
    _fields_ = [('g', C.c_void_p), ('momentum', C.c_void_p), ('out', C.c_void_p), ('copy', C.c_void_p), ('rows', C.c_int64),
                ('cols', C.c_int64), ('lr', C.c_double), ('scale', C.c_double), ('weight_decay', C.c_double), ('type', C.c_int32),
                ('gtype', C.c_int32)]


class D1Muon(C.Structure):
    """The D1Muon struct of include/d1ops.h."""
    _fields_ = [*((name, C.c_double) for name in ('a', 'b', 'c', 'eps', 'momentum')),
                *((name, C.c_int32) for name in ('steps', 'nesterov', 'terms', 'part'))]


def load_ops():
    """libd1ops.so: the operators of a policy update beside the fused step (include/d1ops.h)."""
    global _OPS
    if _OPS is None:
        path = HERE / 'libd1ops.so'
        if not path.exists():
            raise RuntimeError(f'{path} is missing: build it with __graft_entry__.build() '
                               '(the operators have no CPU fallback)')
        L = C.CDLL(str(path))
        p, i, n, f = C.c_void_p, C.c_int, C.c_int64, C.c_float
        L.d1_tokens_work_bytes.argtypes = [n, i, i]
        L.d1_tokens_fwd.argtypes = [p, i, n, i, n, p, p, n, i, p, p, p, p, p, p, n, p]
        L.d1_tokens_bwd.argtypes = [p, i, n, i, n, p, p, n, p, p, p, p, p, p]
        L.d1_norm_fwd.argtypes = [p, i, n, i, n, p, p, i, f, p, p, p, p]
        L.d1_norm_work_bytes.argtypes = [n, i, i]
        L.d1_norm_bwd.argtypes = [p, n, p, i, n, i, n, p, i, p, p, p, p, p, p, n, p]
        L.d1_adamw_work_bytes.argtypes = [p, i, p]
        L.d1_adamw_step.argtypes = [p, i, p, p, p, n, p]
        L.d1_adamw_step_with.argtypes = [p, i, p, p, p, p, n, p]
        L.d1_adamw_read.argtypes = [p, p, n, i, p, p]
        L.d1_policy_loss_work_bytes.argtypes = [p]
        L.d1_policy_loss.argtypes = [p, p, p, p, p, p, n, p]
        L.d1_scale.argtypes = L.d1_scale_to.argtypes = [p, p, i, n, p, p]
        L.d1_scan_marks.argtypes = [p]
        L.d1_scan_work_bytes.argtypes = [p]
        L.d1_scan_fwd.argtypes = [p, p, n, n, p, p, n, p]
        L.d1_scan_bwd.argtypes = [p, p, n, n, p, p, n, n, p, n, n, p, p, n, p]
        L.d1_muon_check.argtypes = [p]
        L.d1_muon_work_bytes.argtypes = [p, i, p]
        L.d1_muon_step.argtypes = [p, i, p, p, p, n, p]
        for name in ('d1_tokens_work_bytes', 'd1_norm_work_bytes', 'd1_adamw_work_bytes', 'd1_policy_loss_work_bytes',
                     'd1_scan_marks', 'd1_scan_work_bytes', 'd1_muon_work_bytes'):
            getattr(L, name).restype = C.c_int64
        _OPS = L
    return _OPS


def load_ops_torch():
    """_d1ops.so: libd1ops.so's calls on torch tensors (csrc/d1_ops_torch.cpp)."""
    global _OPS_TORCH
    if _OPS_TORCH is None:
        path = HERE / '_d1ops.so'
        if not path.exists():
            raise RuntimeError(f'{path} is missing: build it with __graft_entry__.build() '
                               '(the operators have no CPU fallback)')
        _OPS_TORCH = importlib.import_module('._d1ops', __package__)
    return _OPS_TORCH


def load_learn(clump=0):
    """libd1learn_clump{0,1}.so: the learning task's learn_* ABI (include/d1learn.h)."""
    if clump not in (0, 1):
        raise ValueError('clump mode is 0 or 1')
    if clump not in _LEARN:
        path = HERE / f'libd1learn_clump{clump}.so'
        if not path.exists():
            raise RuntimeError(f'{path} is missing: build it with __graft_entry__.build() '
                               '(the learning task has no CPU fallback)')
        L = C.CDLL(str(path))
        p, i = C.c_void_p, C.c_int
        for name in ('learn_turn_cost', 'learn_return_gamma'):
            getattr(L, name).restype = C.c_float
            getattr(L, name).argtypes = []
        for name in ('learn_state_bytes', 'learn_obs_size', 'learn_action_size', 'learn_out_size',
                     'learn_config_bytes'):
            getattr(L, name).argtypes = []
        L.learn_init.argtypes = [p, i, p, p, C.c_uint64, p, p, p, i]
        L.learn_step.argtypes = [p, i, p, p, p, i, p, p, p, p, i]
        L.learn_step_active.argtypes = [p, i, p, p, p, i, p, p, p, p, p, i]
        L.learn_heuristic.argtypes = [p, i, p, p, p, p, i]
        _LEARN[clump] = L
    return _LEARN[clump]


def check(code, what):
    if code:
        raise RuntimeError(f'{what} failed with code {code}')
