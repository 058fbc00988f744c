"""Rules for the device code, read from the sources (no GPU needed): nothing writes through the scalar data cache; the entry points record
no memset (a caller may capture them in a HIP graph); every build line switches the packed float instructions off."""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
# scalar stores, scalar atomics, write-back and discard of the scalar cache
SCALAR_WRITE = re.compile(r'\bs_(?:store_|buffer_store_|scratch_store_|atomic_|buffer_atomic_|dcache_wb|dcache_discard)')


def device_sources():
    """Every file of the tree a GPU program is built or started from, and the tools that read their listings."""
    out = []
    for top in ('gendr_amd', 'include', 'oracle', 'tools', 'profiles'):
        for d, _, files in os.walk(os.path.join(ROOT, top)):
            out += [os.path.join(d, f) for f in files if f.endswith(('.h', '.hip', '.cpp', '.c', '.inc', '.py', '.sh', '.s'))]
    return sorted(out)


def test_no_write_through_the_scalar_cache():
    found = ['%s:%d' % (os.path.relpath(p, ROOT), i) for p in device_sources()
             for i, line in enumerate(open(p, encoding='utf-8'), 1) if SCALAR_WRITE.search(line)]
    assert not found, found


def test_entry_points_record_no_memset():
    csrc = os.path.join(ROOT, 'gendr_amd', 'csrc')
    found = ['%s:%d' % (f, i) for f in sorted(os.listdir(csrc)) if f.endswith(('.h', '.hip', '.cpp'))
             for i, line in enumerate(open(os.path.join(csrc, f), encoding='utf-8'), 1) if re.search(r'\b(?:hip|cuda)Memset', line)]
    assert not found, found


def test_no_build_makes_packed_float_instructions():
    from gendr_amd import build
    off = ['-Xclang', '-target-feature', '-Xclang', '-packed-fp32-ops']
    flags = build.HIPCC_FLAGS
    assert any(flags[i:i + 4] == off for i in range(len(flags))), flags
    assert not any('packed-fp32' in f for v in build.VARIANTS.values() for f in v)
    bare = ['%s:%d' % (os.path.relpath(p, ROOT), i) for p in device_sources()
            for i, line in enumerate(open(p, encoding='utf-8'), 1) if re.search(r'hipcc .*--offload-arch.*-O3', line) and ' '.join(off) not in line]
    assert not bare, bare
    written = ['%s:%d' % (os.path.relpath(p, ROOT), i) for p in device_sources() if p.endswith(('.h', '.hip'))
               for i, line in enumerate(open(p, encoding='utf-8'), 1) if re.search(r'v_pk_\w+_f32', line)]
    assert not written, written
