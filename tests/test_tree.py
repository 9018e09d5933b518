"""CPU tests of the tree itself: what its tools may do on a GPU, and what the build entry point does."""
import os, re
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SKIP_DIRS = {'.git', '.pytest_cache', '__pycache__', '_work', 'gpurun_out', 'profiles', 'build', 'build_tmp', '_ref', 'golden'}
SOURCE = ('.hip', '.hpp', '.h', '.c', '.cc', '.cpp', '.s', '.py', '.sh', '.mk', '.txt')

def sources(sub='.'):
    """(path from the root, text) of the sources, scripts and build files below sub"""
    for base, dirs, files in os.walk(os.path.join(ROOT, sub)):
        dirs[:] = [d for d in dirs if d not in SKIP_DIRS]
        for f in sorted(files):
            p = os.path.join(base, f)
            if (f.endswith(SOURCE) or f == 'Makefile') and not os.path.samefile(p, __file__):
                yield os.path.relpath(p, ROOT), open(p, encoding='utf-8', errors='replace').read()

def test_no_tool_brings_a_hang_about():
    """a launch that does not end is looked for by reading the code and on the CPU: no tool repeats a workload until one stops or holds the device's queues beside it"""
    bad = [p for p, t in sources('tools') if re.search(r'hang\d*\b|repro loop|holds? .{0,12}hardware queues', p + '\n' + t, re.I)]
    assert not bad, bad

def test_the_number_of_hardware_queues_is_a_fixed_small_one():
    for p, t in sources():
        for m in re.finditer(r"GPU_MAX_HW_QUEUES['\"]?\]?\s*[,=]\s*([^,);\s]+)", t):
            v = m.group(1).strip('\'"')
            assert v.isdigit() and int(v) <= 16, (p, m.group(0))

def test_no_gpu_code_writes_through_the_scalar_cache():
    """scalar stores and atomics, and that cache's write-back and discard, are named in no source, comments included: what a kernel writes goes through vector stores"""
    op = re.compile(r'(?<![A-Za-z0-9])s_(?:(?:buffer|scratch)_)?(?:store|atomic)_|(?<![A-Za-z0-9])s_dcache_(?:wb|discard)')
    bad = ['%s:%d' % (p, t.count('\n', 0, m.start()) + 1) for p, t in sources() for m in op.finditer(t)]
    assert not bad, bad

@pytest.fixture
def build_commands(monkeypatch):
    """build() with its commands recorded instead of run, on a machine where the reference's directory holds the given files (None: no such directory)"""
    import __graft_entry__ as entry
    real = {n: getattr(os.path, n) for n in ('exists', 'isfile', 'isdir')}
    def run(reference):
        top = '/root/reference'; cmds = []
        def faked(name):
            def f(p):
                s = os.fspath(p).rstrip('/')
                if s == top: return reference is not None and name != 'isfile'
                if s.startswith(top + '/'): return name != 'isdir' and s[len(top) + 1:] in (reference or ())
                return real[name](p)
            return f
        for n in real: monkeypatch.setattr(os.path, n, faked(n))
        monkeypatch.setattr(entry, '_run', lambda cmd, cwd=ROOT: cmds.append(list(cmd)))
        entry.build()
        return cmds
    return run

@pytest.mark.parametrize('reference,built', [(None, False), ((), False), (('README.md',), False), (('minialign.c', 'gaba.c', 'gaba_wrap.h'), True)],
                         ids=['no-directory', 'empty-directory', 'no-sources', 'sources'])
def test_the_reference_is_compiled_only_where_its_sources_are(build_commands, reference, built):
    assert any(c[0] == 'make' and 'ref' in c for c in build_commands(reference)) is built

def test_build_compiles_every_time_it_is_called(build_commands):
    """build() is the check that the tree builds: a library that is there already does not stand in for its sources"""
    made = [os.path.relpath(c[c.index('-o') + 1], ROOT) for c in build_commands(None) if '-o' in c]
    assert {'minialign_amd/libminialign_amd.so', 'minialign_amd/libminialign_amd_prof.so', 'minialign_amd/minialign', 'tools/gensim', 'tools/samcheck'} <= set(made), made
    assert any(c[0] == 'make' and 'oracle' in c and ('-B' in c or '--always-make' in c) for c in build_commands(None))

NO_PACKED_FP32 = '-Xclang -target-feature -Xclang -packed-fp32-ops'

def test_hip_code_is_compiled_without_packed_fp32():
    """some forms of the packed FP32 instructions have given wrong results now and then; the compiler makes them of ordinary float code unless it is told not to"""
    import __graft_entry__ as entry
    assert NO_PACKED_FP32 in ' '.join(entry.HIP_FLAGS)
    bad = ['%s: %s' % (p, l.strip()) for p, t in sources('tools') for l in t.splitlines() if 'hipcc -' in l and NO_PACKED_FP32 not in l]
    assert not bad, bad
    pk = [p for p, t in sources() if re.search(r'\bv_pk_(?:add|mul|fma)_f32\b', t)]
    assert not pk, pk

def test_the_library_holds_no_packed_fp32(tmp_path):
    """the same, in the code object of the library that is built"""
    import shutil, subprocess
    rocm = os.environ.get('ROCM_PATH', '/opt/rocm'); objdump = os.path.join(rocm, 'llvm', 'bin', 'llvm-objdump')
    lib = os.path.join(ROOT, 'minialign_amd', 'libminialign_amd.so')
    if not os.path.exists(objdump): pytest.skip('no llvm-objdump')
    shutil.copy(lib, tmp_path / 'lib.so')
    subprocess.run([objdump, '--offloading', 'lib.so'], cwd=tmp_path, check=True, stdout=subprocess.DEVNULL)
    objs = [f for f in os.listdir(tmp_path) if 'gfx950' in f]
    assert objs, os.listdir(tmp_path)
    for f in objs:
        asm = subprocess.run([objdump, '-d', f], cwd=tmp_path, check=True, stdout=subprocess.PIPE).stdout.decode()
        assert asm.count('\n') > 1000
        assert not re.search(r'\bv_pk_(?:add|mul|fma)_f32\b', asm), f

def test_pinned_memory_is_allocated_pinned():
    """memory that exists already is not registered with the driver: what has to be pinned is allocated that way (hipHostMalloc)"""
    bad = [p for p, t in sources() if re.search(r'\b(?:hip|cuda)Host(?:Unr|R)egister\w*\s*\(', t)]
    assert not bad, bad

def test_the_tools_name_only_tests_that_are_there():
    have = {m for p, t in sources('tests') for m in re.findall(r'def (test_\w+)', t)} | {os.path.basename(p)[:-3] for p, t in sources('tests') if p.endswith('.py')}
    gone = ['%s: %s' % (p, m) for p, t in sources('tools') for m in re.findall(r'\btest_\w+', t) if m not in have]
    assert not gone, gone
