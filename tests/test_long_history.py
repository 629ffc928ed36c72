"""Long-history operators and sampling on the CPU: the host's bookkeeping, the struct layouts of include/dkv.h, and
arguments that the C entry points refuse before any device work."""
import ctypes
import os
import subprocess

import pytest
import torch

from conftest import REPO
from dkv import _lib
from dkv.gpu_cache import GPUCache, slab_bytes
from dkv.gpu_ops import sample
from test_abi import attn

HEADER = os.path.join(REPO, 'include')


def test_runs_of_one_row_tiles():
    """tile_singles counts the one-row 16-bit tiles up to each tile, however the segments were opened, and
    _single_rows() those after the index."""
    lengths, bits = [64, 1, 1, 65, 1, 1, 1, 1], [16, 16, 16, 16, 16, 8, 16, 16]
    want = [0, 1, 2, 0, 1, 2, 0, 1, 2]
    one, many = (GPUCache(None, layers=1, heads=1, max_tokens=256, device='cpu') for _ in range(2))
    at = 0
    for n, b in zip(lengths, bits):
        one._open_segment(at, n, b)
        at += n
    many._open_segments(0, lengths, bits)
    assert one.tile_singles == many.tile_singles == want
    assert [one._single_rows(n) for n in range(10)] == [0] + want
    one.n_indexed = 5
    assert [one._single_rows(n) for n in (4, 5, 6, 7, 9)] == [0, 0, 1, 0, 2]
    # the tiles of a run lie a one-row slab apart
    t = many.tiles_host
    assert all(t['offset'][i + 1] - t['offset'][i] == slab_bytes(1, 16, 1, 1) for i in (1, 4, 7))
    one.reset()
    assert one.tile_singles == [] and one._single_rows(0) == 0


@pytest.mark.parametrize('cls,cname', [(_lib.Sparse, 'dkv_sparse'), (_lib.EvictArgs, 'dkv_evict_args'),
                                       (_lib.Sampling, 'dkv_sampling')])
def test_struct_layout_matches_header(tmp_path, cls, cname):
    fields = ''.join(f'printf("{f} %zu\\n", offsetof({cname}, {f}));' for f, _ in cls._fields_)
    src, exe = tmp_path / 'probe.c', tmp_path / 'probe'
    src.write_text(f'#include <stdio.h>\n#include <stddef.h>\n#include "dkv.h"\n'
                   f'int main(void) {{ printf("size %zu\\n", sizeof({cname})); {fields} return 0; }}')
    subprocess.run(['gcc', '-std=c11', '-I', HEADER, str(src), '-o', str(exe)], check=True)
    found = dict(line.split() for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    assert int(found.pop('size')) == ctypes.sizeof(cls)
    assert {f: getattr(cls, f).offset for f, _ in cls._fields_} == {f: int(v) for f, v in found.items()}


def refused(rc, msg):
    assert rc == _lib.DKV_EINVAL
    assert msg in _lib.load().dkv_last_error().decode()


def test_index_refuses_bad_arguments():
    lib = _lib.load()
    for args, msg in [((4096, 4096, -1, 3, 1, 1, 4096), 'range'), ((4096, 4096, 4, 3, 1, 1, 4096), 'range'),
                      ((4096, 4096, 0, 3, 0, 1, 4096), 'range'), ((0, 4096, 0, 3, 1, 1, 4096), 'null'),
                      ((4096, 4096, 0, 3, 1, 1, 4100), 'misaligned')]:
        refused(lib.dkv_index(*args, None), msg)
    assert lib.dkv_index(0, 0, 3, 3, 1, 1, 0, None) == 0  # nothing to index
    assert lib.dkv_index_bytes(1, 2, 3) == lib.dkv_index_bytes(64, 2, 3) == 64 * 2 * 3 * 256
    assert lib.dkv_index_bytes(65, 2, 3) == 2 * 64 * 2 * 3 * 256


@pytest.mark.parametrize('kw,sparse,msg', [
    (dict(q=0), (0, 0, 1, 0), 'null'), (dict(q_heads=14), (0, 0, 1, 0), 'shape'), (dict(n_segs=17), (0, 0, 1, 0), 'n_segs'),
    (dict(v_new=0), (0, 0, 1, 0), 'aligned'), (dict(out=4104), (0, 0, 1, 0), 'aligned'), (dict(out_dtype=2), (0, 0, 1, 0), 'out bf16'),
    (dict(), (0, 3, 1, 0), 'bounds'), (dict(), (4100, 3, 1, 0), 'bounds'), (dict(), (0, 0, -1, 0), 'negative'),
    (dict(), (0, 0, 1, -1), 'negative'), (dict(precision=2), (0, 0, 1, 0), 'precision'), (dict(nq=70000), (0, 0, 1, 0), '65535'),
    (dict(q_tok_stride=60), (0, 0, 1, 0), 'aligned'), (dict(), (0, 0, 1, 0), 'workspace')])
def test_attend_sparse_refuses_bad_arguments(kw, sparse, msg):
    a, s = attn(**kw), _lib.Sparse(*sparse)
    a.nq = kw.get('nq', 1)
    if msg == 'workspace':
        a.tiles = a.arena = 4096
        a.n_tiles, a.past = 64, 4096
    refused(_lib.load().dkv_attend_sparse(ctypes.byref(a), ctypes.byref(s), None), msg)


@pytest.mark.parametrize('kw,stride,msg', [
    (dict(k_new=0), 64, 'null'), (dict(heads=0), 64, 'shape'), (dict(past=8, n_tiles=1, tiles=4096, arena=4096), 64, 'masses'),
    (dict(kn_head_stride=3), 64, 'aligned'), (dict(), 64, 'workspace'), (dict(layer=1), 64, 'shape')])
def test_attention_mass_refuses_bad_arguments(kw, stride, msg):
    a = attn(**kw)
    refused(_lib.load().dkv_attention_mass(ctypes.byref(a), 4096, stride, 0, None), msg)
    refused(_lib.load().dkv_attention_mass(ctypes.byref(a), None, stride, 0, None), 'null')


def evict_args(**kw):
    e = _lib.EvictArgs()
    e.arena, e.out_arena, e.tiles, e.out_tiles, e.mass, e.out_mass, e.kept = 1 << 20, 2 << 20, 4096, 8192, 12288, 16384, 20480
    e.arena_bytes = e.out_arena_bytes = 1 << 20
    e.layers = e.heads = 1
    e.n_tiles = e.end_tile = 2
    e.tokens = e.end_token = 128
    e.tail_offset = 2 * slab_bytes(64, 4, 1, 1)
    e.n_classes, e.class_bits[0], e.class_keep[0], e.class_held[0] = 1, 4, 100, 128
    e.mass_stride = e.out_mass_stride = 128
    e.workspace, e.workspace_bytes = 24576, 8 * 128
    for k, v in kw.items():
        if isinstance(v, tuple):
            getattr(e, k)[:] = v
        else:
            setattr(e, k, v)
    return e


@pytest.mark.parametrize('kw,msg', [
    (dict(layers=0), 'bad ranges'), (dict(end_tile=3), 'bad ranges'), (dict(end_token=129), 'bad ranges'),
    (dict(class_bits=(5, 0, 0)), 'bad ranges'), (dict(class_keep=(0, 0, 0)), 'bad ranges'), (dict(class_held=(99, 0, 0)), 'bad ranges'),
    (dict(class_held=(129, 0, 0)), 'bad ranges'), (dict(n_classes=2, class_bits=(4, 4, 0), class_keep=(5, 5, 0), class_held=(64, 64, 0)), 'bad ranges'),
    (dict(n_classes=4), 'bad ranges'), (dict(mass_stride=127), 'bad ranges'), (dict(out_mass_stride=99), 'bad ranges'),
    (dict(out_arena_bytes=2 * slab_bytes(64, 4, 1, 1) - 16 - 28 * 80), 'bad ranges'), (dict(tail_bytes=1 << 20), 'bad ranges'),
    (dict(tail_offset=8), 'bad ranges'), (dict(kept=0), 'null'), (dict(out_arena=(1 << 20) + 512), 'old ones'),
    (dict(out_tiles=4096), 'old ones'), (dict(out_mass=12288), 'old ones'), (dict(workspace_bytes=8 * 128 - 1), 'workspace'),
    (dict(workspace=0), 'workspace')])
def test_evict_refuses_bad_arguments(kw, msg):
    refused(_lib.load().dkv_evict(ctypes.byref(evict_args(**kw)), None), msg)


def test_evict_of_nothing_runs_nothing():
    e = _lib.EvictArgs()
    e.layers = e.heads = 1
    assert _lib.load().dkv_evict(ctypes.byref(e), None) == 0


@pytest.mark.parametrize('kw,msg', [
    (dict(vocab=0), 'vocab'), (dict(dtype=2), 'bf16'), (dict(u_dtype=2), 'fp64'), (dict(vocab=(1 << 22) + 1), 'at most'),
    (dict(t=-1.), 'temperature'), (dict(t=float('nan')), 'temperature'), (dict(p=0.), 'top_p'), (dict(p=1.1), 'top_p'),
    (dict(m=-.1), 'min_p'), (dict(m=1.1), 'min_p'), (dict(k=-1), 'top_k'), (dict(logits=0), 'null'), (dict(out=0), 'null'),
    (dict(ws=0), 'workspace'), (dict(ws_bytes=16), 'workspace'), (dict(ws=4100), 'workspace')])
def test_sample_refuses_bad_arguments(kw, msg):
    lib = _lib.load()
    p = _lib.Sampling(kw.get('t', 1.), kw.get('p', 1.), kw.get('m', 0.), kw.get('k', 0), None, None, None, None)
    vocab = kw.get('vocab', 100)
    refused(lib.dkv_sample(kw.get('logits', 4096), kw.get('dtype', 0), vocab, 1, vocab, 4096, kw.get('u_dtype', 0), ctypes.byref(p),
                           kw.get('out', 4096), kw.get('ws', 4096), kw.get('ws_bytes', 1 << 30), None), msg)


def test_sample_refuses_what_is_not_on_a_gpu():
    with pytest.raises(ValueError, match='CUDA'):
        sample(torch.zeros(2, 10), torch.zeros(2))


def test_shares_of_an_eviction():
    """Protected segments are whole ones; what is left goes to the widths in proportion, remainders to the largest
    (the wider one of two)."""
    c = GPUCache(None, layers=1, heads=1, max_tokens=4096, device='cpu')
    c._open_segments(0, [40, 64, 64, 64, 64, 64, 10], [16, 4, 8, 4, 16, 4, 16])
    c.seen = [370]
    every, middle = {16: 114, 4: 192, 8: 64}, {4: 192, 8: 64, 16: 64}
    assert c._eviction(200, 0, 0) == (0, 7, {16: 62, 4: 104, 8: 34}, every)
    assert c._eviction(200, 1, 1) == (1, 6, {4: 90, 8: 30, 16: 30}, middle)
    assert c._eviction(201, 40, 10) == (1, 6, {4: 91, 8: 30, 16: 30}, middle)
    assert c._eviction(202, 40, 10) == (1, 6, {4: 91, 8: 30, 16: 31}, middle)
    assert c._eviction(200, 41, 11) == (2, 5, {8: 7, 4: 7, 16: 8}, {8: 64, 4: 64, 16: 64})
    assert c._eviction(50, 40, 10) == (1, 6, {}, middle)
    assert c._eviction(370, 0, 0) == c._eviction(999, 5, 5) == (7, 7, {}, {})
    with pytest.raises(ValueError, match='protected'):
        c._eviction(49, 40, 10)


def test_graph_steps_refuse_other_masses_or_another_index():
    c = GPUCache(None, layers=1, heads=1, max_tokens=256, device='cpu')
    steps = c.begin_graph_steps(1)
    steps.mass, steps.bounds = c._own_mass(), None
    c.end_graph_steps()
    c.begin_graph_steps(1, steps=steps)
    steps._check_storage()
    branch = c.fork()
    assert branch._mass is c._mass and branch.mass().shape == (1, 1, 0) and branch._mass is not c._mass
    c._mass = c._mass.clone()
    with pytest.raises(ValueError, match='masses'):
        steps._check_storage()
    steps.mass = False
    c._bounds = torch.zeros(16, dtype=torch.uint8)
    with pytest.raises(ValueError, match='index'):
        steps._check_storage()
