"""In-tree build of the gfx950 libraries (hipcc, no CUDA, no JIT cache).

libd1hip.so          environment, wait workload, LOS compiler, MFMA trunk layer, sampling, GAE, PPO step
libd1ops.so          token log probabilities, layer norm, the AdamW step over many tensors (include/d1ops.h)
_d1ops.so            the Python module that calls it on torch tensors
libd1learn_clump0.so the d1-stairs-v2 learning task (learn_* ABI), CLUMP_MODE 0
libd1learn_clump1.so the same task with clumped placement in a third of resets
"""
import pathlib
import subprocess
import sysconfig

HERE = pathlib.Path(__file__).resolve().parent
CSRC = HERE / 'csrc'
FLAGS = ['--offload-arch=gfx950', '-O3', '-std=c++17', '-fPIC', '-shared', '-ffp-contract=off',
         '-Xclang', '-target-feature', '-Xclang', '-packed-fp32-ops']
TARGETS = {
    'libd1hip.so': ([CSRC / 'd1_env.hip', CSRC / 'd1_policy.hip', CSRC / 'd1_forward.hip', CSRC / 'd1_ppo.hip',
                     CSRC / 'd1_maps.hip'], []),
    'libd1ops.so': ([CSRC / 'd1_tokens.hip', CSRC / 'd1_norm.hip', CSRC / 'd1_optim.hip'], []),
    'libd1learn_clump0.so': ([CSRC / 'd1_learn.hip'], ['-DD1_CLUMP_MODE=0']),
    'libd1learn_clump1.so': ([CSRC / 'd1_learn.hip'], ['-DD1_CLUMP_MODE=1']),
}


# the torch binding: compiled beside the libraries, linked once libd1ops.so is there
BINDING, BINDING_SOURCE = '_d1ops.so', CSRC / 'd1_ops_torch.cpp'


def _binding_commands(obj, out):
    import torch
    from torch.utils import cpp_extension
    abi = int(torch._C._GLIBCXX_USE_CXX11_ABI)
    includes = [sysconfig.get_paths()['include'], *cpp_extension.include_paths()]
    libs = cpp_extension.library_paths()
    compile_ = ['g++', '-O2', '-std=c++17', '-fPIC', '-w', '-c', f'-D_GLIBCXX_USE_CXX11_ABI={abi}',
                '-DTORCH_EXTENSION_NAME=_d1ops', '-DTORCH_API_INCLUDE_EXTENSION_H',
                *(x for path in includes for x in ('-isystem', path)), str(BINDING_SOURCE), '-o', str(obj)]
    link = ['g++', '-shared', str(obj), '-o', str(out), *(f'-L{path}' for path in libs), '-lc10', '-ltorch_cpu', '-ltorch',
            '-ltorch_python', f'-L{HERE}', '-ld1ops', '-Wl,-rpath,$ORIGIN']
    return compile_, link


def build(verbose=False):
    start = lambda cmd: subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True)  # noqa: E731
    jobs, built, errors = [], [], []
    obj, bound, bound_tmp = HERE / '_d1ops.o', HERE / BINDING, HERE / (BINDING + '.tmp')
    compile_, link = _binding_commands(obj, bound_tmp)
    for name, (sources, defs) in TARGETS.items():
        out = HERE / name
        tmp = out.with_suffix('.so.tmp')
        cmd = ['hipcc', *FLAGS, *defs, '-I', str(HERE.parent / 'include'), '-o', str(tmp), *map(str, sources)]
        jobs.append((out, tmp, cmd, start(cmd)))
    jobs.append((obj, None, compile_, start(compile_)))
    for out, tmp, cmd, proc in jobs:
        _, err = proc.communicate()
        if proc.returncode:
            errors.append(f'{out.name}: {cmd[0]} failed:\n{err}')
            continue
        if tmp is not None:
            tmp.replace(out)
            built.append(out)
        if verbose:
            print(' '.join(cmd))
    if not errors:
        proc = start(link)
        _, err = proc.communicate()
        if proc.returncode:
            errors.append(f'{BINDING}: g++ failed:\n{err}')
        else:
            bound_tmp.replace(bound)
            obj.unlink()
            built.append(bound)
            if verbose:
                print(' '.join(link))
    if errors:
        raise RuntimeError('\n'.join(errors))
    return built


if __name__ == '__main__':
    print(build(verbose=True))
