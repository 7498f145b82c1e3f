"""
The index arithmetic of the trainable node layers on the CPU, over sizes and contents that no GPU test can hold or should be
given: the kernels' own functions out of the device headers, compiled by g++ with the lanes of a wave as one (MH_WAVE 1), and
the choices of tiles.
"""
import ctypes
import itertools
import os
import random
import re
import shutil
import subprocess
import sys
import types

import numpy as np
import pytest
import torch

import mace_hip_kernels
from mace_hip_kernels import _native, halves, matmul

CSRC = os.path.dirname(_native.DEVICE_HEADER)
SHIM = """
#include <algorithm>
#include <cstdint>
#include <cstring>
#include <cstdlib>
#define __device__
#define __forceinline__ inline
#define __restrict__
#define MH_WAVE 1
using std::max; using std::min;
struct dim { unsigned x, y, z; };
static dim threadIdx, blockIdx, blockDim, gridDim;
static int __shfl_up(int v, int, int) { return v; }
static int mh_bcast(int v, int) { return v; }
static unsigned long long __ballot(bool b) { return b; }
static unsigned __float_as_uint(float v) { unsigned u; memcpy(&u, &v, 4); return u; }
static float __uint_as_float(unsigned u) { float v; memcpy(&v, &u, 4); return v; }
static int __ffsll(unsigned long long v) { return v ? 1 + __builtin_ctzll(v) : 0; }
"""


def function(header, name):
    """The text of a function or struct of a device header, its template line and qualifiers included."""
    with open(os.path.join(CSRC, header)) as f:
        text = f.read()
    m = re.search(r'^(template <[^\n]*>\n)?(struct ' + name + r' \{|[^\n;]*\b' + name + r'\([^;{]*\{)', text, re.M)
    depth, end = 1, m.end()
    while depth:
        depth += {'{': 1, '}': -1}.get(text[end], 0)
        end += 1
    return text[m.start():end] + ';\n'


def host_library(src, tmp_path):
    c, so = tmp_path / 'part.cpp', tmp_path / 'part.so'
    c.write_text(SHIM + src)
    subprocess.run(['g++', '-O1', '-std=c++17', '-shared', '-fPIC', '-w', str(c), '-o', str(so)], check=True)
    return ctypes.CDLL(str(so))


needs_gxx = pytest.mark.skipif(shutil.which('g++') is None, reason='needs g++')


@needs_gxx
def test_slots_cover_every_row_once(tmp_path):
    """Whatever the offsets hold, the pieces that a launch has room for cover every row once: a group's by its own, the rows
    before and behind the groups by pieces of no group; and whole groups are the rows that their pieces are."""
    lib = host_library(function('mh_matmul.h', 'mm_groups') + function('mh_matmul.h', 'mm_slot') +
                       function('mh_matmul.h', 'mm_by_length') + function('mace_hip.cpp', 'pieces') + """
extern "C" long long count(const int* off, long long R, long long E, long long L) { return pieces(off, R, E, L); }
extern "C" int slot(const int* off, int E, int R, int L, int s, int* out) { return mm_slot(off, E, R, L, s, out[0], out[1], out[2]); }
extern "C" void group(const int* off, int E, int R, int k, int* out) { mm_by_length(off, E, R, k, out[0], out[1], out[2]); }
""", tmp_path)
    lib.count.restype, lib.count.argtypes = ctypes.c_longlong, [ctypes.c_void_p] + [ctypes.c_longlong] * 3
    lib.slot.argtypes = [ctypes.c_void_p] + [ctypes.c_int] * 4 + [ctypes.c_void_p]
    lib.group.argtypes = [ctypes.c_void_p] + [ctypes.c_int] * 3 + [ctypes.c_void_p]
    rng = random.Random(3)
    for n in range(600):
        R, E, L = rng.choice([1, 12, 100, 700]), rng.choice([1, 2, 3, 9, 130]), rng.choice([1, 16, 64, 256])
        if n % 4 == 0:                                   # any contents
            off = [rng.randint(-5, R + 5) for _ in range(E + 1)]
        else:
            off = sorted(rng.randint(0, R) for _ in range(E + 1))
            off[0] = min(off[0], rng.choice([0, R]))
        top, of = min(max(off[0], 0), R), np.full(R, -1)
        for e in range(E):
            hi = max(top, min(off[e + 1], R))
            of[top:hi], top = e, hi
        o, out = np.array(off, dtype=np.int32), np.zeros(3, dtype=np.int32)
        got, live = np.full(R, -2), True
        for s in range(lib.count(o.ctypes.data, R, E, L)):
            is_live = bool(lib.slot(o.ctypes.data, E, R, L, s, out.ctypes.data))
            assert live or not is_live
            live = is_live
            e, r0, r1 = (int(v) for v in out)
            assert 0 <= r0 <= R and r1 <= R and r1 - r0 <= L and (e >= 0) == live
            if r0 < R:
                assert (got[r0:r1] == -2).all()
                got[r0:r1] = e
        assert (got == of).all(), (off, R, L)
        # whole groups are the same rows
        got[:] = -1
        for k in range(E):
            lib.group(o.ctypes.data, E, R, k, out.ctypes.data)
            assert 0 <= out[1] <= out[2] <= R
            got[out[1]:out[2]] = out[0]
        assert (got == of).all(), (off, R)


@needs_gxx
def test_rows_behind_the_last_group_are_zeroed_near_the_largest_counts(tmp_path):
    """The rows past the last kept assignment are each zeroed once, and no other place is written, where their number and that
    of the workgroups' rows together pass 2^31."""
    lib = host_library("""
typedef long long ll;
static ll seen[1 << 16], n;                               // the places written
template <int TY> struct mm_type { typedef char t; };
template <int TY> struct mm_vec {
    static constexpr int V = 8;
    void zero() {}
    void put(char* p, int) { if (n < (1 << 16)) seen[n] = (ll)(uintptr_t)p; ++n; }
};
""" + function('mh_experts.h', 'ex_zero_tail') + """
// rows written by thread `t` of block `b` of a launch of T rows by 2^lg lanes each; the first at most 65,536 in `out`
extern "C" ll tail(int last, int A, int T, int lg, unsigned b, unsigned t, ll* out) {
    blockDim.x = 256, blockIdx.x = b, threadIdx.x = t, gridDim.x = (T + (256ll >> lg) - 1) / (256 >> lg), n = 0;
    ex_zero_tail<0>((char*)0, &last, 0, A, 1, lg);
    memcpy(out, seen, 8 * std::min(n, (ll)1 << 16));
    return n;
}
""", tmp_path)
    lib.tail.restype = ctypes.c_longlong
    lib.tail.argtypes = [ctypes.c_int] * 4 + [ctypes.c_uint] * 2 + [ctypes.c_void_p]
    out = np.zeros(1 << 16, dtype=np.int64)
    # one value a row: a lane each; T rows of k assignments, of which the first `last` are kept
    for T, k in ((1_080_000_000, 1), (2 ** 31 - 2 ** 21 - 1, 1), (700_000_000, 3), (500_000_000, 4), (1000, 2)):
        A, blocks = T * k, -(-T // 256)
        for last in (0, A // 2, A - 1000, A - 1, A):
            for b in sorted({0, 1, blocks // 2, blocks - 2, blocks - 1} & set(range(blocks))):
                for t in (0, 255):
                    got = lib.tail(last, A, T, 0, b, t, out.ctypes.data)
                    want = np.arange(last + b * 256 + t, A, blocks * 256)
                    assert got == len(want) and (out[:got] == want).all(), (T, k, last, b, t)


def test_wide_rows_take_tiles_with_64_bit_offsets(monkeypatch):
    """Rows that are as far apart as a tile straight to LDS cannot address, after copies to whole steps, as the product g act'(a)
    or as halves, go through registers instead; just below the limit they need not."""
    # a row's byte offset in the largest of those tiles, its steps included
    assert max(max(matmul.tile_shape(t, torch.bfloat16)) for t in matmul.FAST) * 2 * matmul.LD_MAX <= 2 ** 30
    chosen = []
    monkeypatch.setattr(matmul, 'module', lambda device, dtype, mode, tile=None, act=0: chosen.append((mode, tile)))
    monkeypatch.setattr(halves, 'module', lambda device, mode, act=0: chosen.append((mode, 'halves')))
    near = set(matmul.FAST) | {'halves'}

    def tiles(fn, dtype, *args):
        chosen.clear()
        numbers = fn(0, matmul.TYPES[dtype], *args)
        return {t for _, t in chosen if t} & near, numbers

    f32, b16 = torch.float32, torch.bfloat16
    wide = matmul.LD_MAX
    for K in (wide - 7, wide, wide + 1, 2 * wide + 1, 8 * wide + 3):
        for R, n in ((128, 128), (4096, 4096)):
            for ok in (0, 1):
                got, numbers = tiles(matmul._fwd_plan, b16, R, n, K, 1, 0, ok and K % 8 == 0 and K < wide, 0)
                assert not got and not any(numbers[4:]), (R, n, K)
    for N, K in ((2 * wide + 8, 4096), (wide + 8, 512), (512, wide + 8), (wide - 7, 64)):
        for made in (0, 1):
            got, numbers = tiles(matmul._bwd_plan, b16, 4096, N, K, 1, 0, made, made, 0, 0, 7)
            assert not got and not any(numbers[-3:]), (N, K, made)
    for mode, N, K in itertools.product(('fwd', 'dx', 'dw'), (2048, wide // 2, 2 * wide + 64), (2048, wide // 2, 2 * wide + 64)):
        assert max(N, K) == 2048 or not matmul._by_halves(2048, N, K, 1, False, mode)
    # more rows of weights than a launch counts
    assert not tiles(matmul._fwd_plan, b16, 10 ** 6, 2 ** 15, 9, 2 ** 16, 0, 0, 0)[0]
    # below the limits
    assert tiles(matmul._fwd_plan, b16, 4096, 4096, wide - 8, 1, 0, 1, 1)[0]
    assert tiles(matmul._bwd_plan, b16, 4096, 4096, 4096, 1, 0, 1, 1, 1, 1, 7)[0]
    assert all(matmul._by_halves(20000, 1024, 1024, 1, False, mode) for mode in ('fwd', 'dx', 'dw'))


def test_the_library_refuses_halves_that_a_tile_cannot_address():
    lib = _native.load()
    p = np.zeros(64, dtype=np.float32).ctypes.data
    wide = matmul.LD_MAX
    for call in (lambda: lib.mh_hv_mm(None, p, p, p, None, None, 0, None, None, p, p, None, 4, 4, wide // 2, 1, None),
                 lambda: lib.mh_hv_mm(None, p, p, p, None, None, 0, None, None, p, p, p, 4, wide, 4, 1, None),
                 lambda: lib.mh_hv_outer(None, p, p, p, None, None, p, p, p, p, 4, wide, 4, 1, 0, 1, None),
                 lambda: lib.mh_hv_outer(None, p, p, p, None, None, p, p, p, p, 4, 4, wide, 1, 0, 1, None)):
        assert call() != 0 and 'bad sizes' in lib.mh_last_error().decode()


@needs_gxx
@pytest.mark.parametrize('bits,rel,least', [(8, 2.0 ** -9, 2.0 ** -54), (9, 2.0 ** -10, 2.0 ** -29)], ids=['bf16', 'f16'])
def test_codes_of_slopes_are_near_at_every_size(bits, rel, least, tmp_path):
    """A slope and its code differ by at most 2^-16, and by at most half a step of its own magnitude down to ``least``; 0, 1 and
    NaN come back as they are, and every code stands for one slope."""
    lib = host_library('#define MM_F16 2\n' + function('mh_matmul.h', 'mm_slope_code') + f"""
typedef mm_slope_code<{2 if bits == 9 else 1}> code;
extern "C" void there(const float* v, unsigned short* c, int n) {{ for (int i = 0; i < n; ++i) c[i] = code::of(v[i]); }}
extern "C" void back(const unsigned short* c, float* v, int n) {{ for (int i = 0; i < n; ++i) v[i] = code::value(c[i]); }}
""", tmp_path)

    def there(v):
        c = np.empty(len(v), dtype=np.uint16)
        lib.there(v.ctypes.data_as(ctypes.c_void_p), c.ctypes.data_as(ctypes.c_void_p), len(v))
        return c

    def back(c):
        v = np.empty(len(c), dtype=np.float32)
        lib.back(c.ctypes.data_as(ctypes.c_void_p), v.ctypes.data_as(ctypes.c_void_p), len(c))
        return v

    rng = np.random.default_rng(1)
    v = np.concatenate([rng.uniform(-0.1290, 1.1290, 400_000), -2.0 ** rng.uniform(-90, -3, 200_000),
                        2.0 ** rng.uniform(-90, 0, 200_000), -2.0 ** np.arange(-40.0, -3), 2.0 ** np.arange(-60.0, 1)])
    v = v[(v > -0.129) & (v < 1.129)].astype(np.float32)
    w = back(there(v))
    off = np.abs(w.astype(np.float64) - v)
    assert (off <= 2.0 ** -16).all()
    inside = np.abs(v) >= least
    assert (off[inside] <= rel * np.abs(v[inside])).all()
    # below that half a step of the last binade, and what the scaled magnitude, no normal float32 any more, has lost before
    assert (off[~inside] <= rel * least + 2.0 ** -150 * least * 2.0 ** 126).all() and (np.signbit(w) == np.signbit(v))[w != 0].all()
    assert back(there(np.array([0, -0.0, 1, 0.5], dtype=np.float32))).tolist() == [0, 0, 1, 0.5]
    for nan in (0x7FC00000, 0xFFC00000, 0x7FC12345, 0x7FC02000):     # quiet, as arithmetic leaves them
        assert np.isnan(back(there(np.array([nan], dtype=np.uint32).view(np.float32))))[0]
    # the codes in use are each other's inverse
    used = np.concatenate([np.arange(1, 48771), np.arange(49536, 65535)]).astype(np.uint16)
    assert (there(back(used)) == used).all() and np.isnan(back(np.array([0xC000], dtype=np.uint16)))[0]


def test_the_library_refuses_bad_arguments_for_what_is_computed_again():
    lib = _native.load()
    p = np.zeros(64, dtype=np.float32).ctypes.data
    for call, text in (
            (lambda: lib.mh_hv_again_mm(None, p, 4, p, 4, p, None, None, 0, None, None, p, p, None, 2, 4, 0, 1, 8, None), 'bad sizes'),
            (lambda: lib.mh_hv_again_mm(None, p, 4, p, 4, p, None, None, 0, None, None, p, p, None, 2, 4, 4, 2, 8, None), 'bad sizes'),
            (lambda: lib.mh_hv_again_mm(None, p, 4, p, 4, p, None, None, 0, None, None, p, p, None, 2, 4, 4, 1, 0, None), 'bad sizes'),
            (lambda: lib.mh_hv_again_mm(None, p, 4, p, 4, p, None, None, 0, None, None, None, p, None, 2, 4, 4, 1, 8, None), 'NULL'),
            (lambda: lib.mh_hv_again_mm(None, p, 3, p, 4, p, None, None, 0, None, None, p, p, None, 2, 4, 4, 1, 8, None), 'overlap'),
            (lambda: lib.mh_hv_again_mm(None, p, 4, p, 4, p, None, None, 0, None, None, p, p, p, 2, 5, 4, 1, 8, None), 'overlap'),
            (lambda: lib.mh_hv_again_mm(None, p, 4, p, 4, p, None, None, 0, None, None, p, p, None, 2, 4, 4, 1, 8, None), 'not bound'),
            (lambda: lib.mh_hv_again_outer(None, p, 4, p, 4, p, None, None, p, p, p, p, 2, 4, 4, 1, 4, 0, 8, None), 'bad sizes'),
            (lambda: lib.mh_hv_again_outer(None, p, 4, p, 4, p, None, None, p, p, p, p, 2, 4, 4, 1, 4, 1, 8, None), 'NULL'),
            (lambda: lib.mh_hv_again_outer(None, p, 3, p, 4, p, None, None, p, p, p, p, 2, 4, 4, 1, 0, 1, 8, None), 'overlap'),
            (lambda: lib.mh_hv_again_outer(None, p, 4, p, 4, p, None, None, p, p, p, p, 2, 4, 4, 1, 0, 1, 8, None), 'not bound')):
        assert call() != 0 and text in lib.mh_last_error().decode(), (text, lib.mh_last_error())


def test_a_host_side_built_for_another_library_is_refused(monkeypatch):
    """_layers.so allocates what libmace_hip.so's kernels write: built from another header it is not used."""
    assert _native.layers().abi == _native.ABI_VERSION == _native.load().mh_version()
    for fake in (types.SimpleNamespace(abi=_native.ABI_VERSION - 1), types.SimpleNamespace()):
        monkeypatch.setattr(_native, '_layers', None)
        monkeypatch.setitem(sys.modules, 'mace_hip_kernels._layers', fake)
        monkeypatch.setattr(mace_hip_kernels, '_layers', fake)
        with pytest.raises(RuntimeError, match='another libmace_hip.so'):
            _native.layers()
