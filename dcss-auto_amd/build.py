"""In-tree build of the gfx950 libraries (hipcc, no CUDA, no JIT cache).

libd1hip.so          environment, wait workload, LOS compiler, MFMA trunk layer, sampling, GAE, PPO step
libd1ops.so          token log probabilities, layer norm, the AdamW step over many tensors, the policy
                     loss, the gated recurrence, orthogonalised updates (include/d1ops.h)
_d1ops.so            the Python module that calls it on torch tensors
libd1learn_clump0.so the d1-stairs-v2 learning task (learn_* ABI), CLUMP_MODE 0
libd1learn_clump1.so the same task with clumped placement in a third of resets
"""
import pathlib
import subprocess
import sysconfig

HERE = pathlib.Path(__file__).resolve().parent
CSRC = HERE / 'csrc'
FLAGS = ['--offload-arch=gfx950', '-O3', '-std=c++17', '-fPIC', '-ffp-contract=off',
         '-Xclang', '-target-feature', '-Xclang', '-packed-fp32-ops']
TARGETS = {
    'libd1hip.so': ([CSRC / 'd1_env.hip', CSRC / 'd1_policy.hip', CSRC / 'd1_forward.hip', CSRC / 'd1_ppo.hip',
                     CSRC / 'd1_maps.hip'], []),
    'libd1ops.so': ([CSRC / 'd1_tokens.hip', CSRC / 'd1_norm.hip', CSRC / 'd1_optim.hip', CSRC / 'd1_loss.hip',
                    CSRC / 'd1_scan.hip', CSRC / 'd1_muon.hip'], []),
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
    """Every source file is an object of its own (compiled side by side, the longest first to start), then the links."""
    start = lambda cmd: subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True)  # noqa: E731
    built, errors = [], []

    def finish(what, cmd, proc):
        _, err = proc.communicate()
        if proc.returncode:
            errors.append(f'{what}: {cmd[0]} failed:\n{err}')
        elif verbose:
            print(' '.join(cmd))

    include = ['-I', str(HERE.parent / 'include')]
    binding_obj, bound, bound_tmp = HERE / '_d1ops.o', HERE / BINDING, HERE / (BINDING + '.tmp')
    compile_, link_binding = _binding_commands(binding_obj, bound_tmp)
    objects, jobs = {}, [(BINDING, compile_, start(compile_))]
    for name, (sources, defs) in TARGETS.items():
        objects[name] = [HERE / f'{pathlib.Path(name).stem}.{src.stem}.o' for src in sources]
        for src, obj in zip(sources, objects[name]):
            cmd = ['hipcc', *FLAGS, *defs, *include, '-c', str(src), '-o', str(obj)]
            jobs.append((name, cmd, start(cmd)))
    for job in jobs:
        finish(*job)
    if not errors:
        jobs = []
        for name, objs in objects.items():
            out, tmp = HERE / name, (HERE / name).with_suffix('.so.tmp')
            cmd = ['hipcc', '--offload-arch=gfx950', '-fPIC', '-shared', '-o', str(tmp), *map(str, objs)]
            jobs.append((out, tmp, cmd, start(cmd)))
        for out, tmp, cmd, proc in jobs:
            finish(out.name, cmd, proc)
            if tmp.exists() and not proc.returncode:
                tmp.replace(out)
                built.append(out)
    if not errors:
        proc = start(link_binding)
        finish(BINDING, link_binding, proc)
        if not proc.returncode:
            bound_tmp.replace(bound)
            built.append(bound)
    for obj in [binding_obj, *(o for objs in objects.values() for o in objs)]:
        obj.unlink(missing_ok=True)
    if errors:
        raise RuntimeError('\n'.join(errors))
    return built


if __name__ == '__main__':
    print(build(verbose=True))
