"""
Large float32 products of ``dense`` and ``expert_dense`` as three float16 products (``csrc/mh_halves.h``): the operands are
first written as two float16 halves each, scaled by a power of two per row or column, and the matrix cores then do three
products where the direct kernels' bf16 parts take six.  Worth its extra passes where the products are long enough;
``matmul`` decides by sizes.
"""
import functools

import torch

from . import _native

# waves (rows x columns), 16 x 16 fragments per wave (rows x columns): 128 x 128 a workgroup, two of them on a compute unit
# (with four waves 171 us where these take 166, at 20,000 x 1,024 x 1,024 with the halves' making; 256 x 256 about 220)
TILE = 2, 4, 4, 2
SIDE = 128
# the direct tile of what is computed again (matmul.SLOW's of 64 x 64)
AGAIN, AGAIN_SIDE = (4, 2, 1, 2, 64), 64


def pays(rows, n, K, groups, mode, product, direct):
    """Whether a product of [rows, K] and [groups, n, K] that takes ``direct`` seconds is faster by halves: by the seconds of
    the ``product`` of halves itself, the bytes of the halves (read and written once by rows, read twice by columns), the
    launches, and a margin of a tenth for what these leave out.  Measured (us, direct / halves): 20,000 x 1,024 x 1,024 forward
    247 / 165, dx 298 / 174, dw 287 / 259; 4,096 x 1,024 x 1,024 54 / 49, 63 / 54, 68 / 96; 8,192 x 512 x 2,048 106 / 70, 117 /
    95, 123 / 133; 5,000 x 512 x 512 28 / 36, 35 / 52, 38 / 61; 20,000 x 128 x 512 forward 26 / 41."""
    moved = {'fwd': 8 * (rows * K + groups * n * K), 'dx': 8 * rows * n + 12 * groups * n * K,
             'dw': 12 * rows * (n + K)}[mode]
    return 1.1 * (product + moved / 4.5e12 + (18e-6 if mode == 'dw' else 11e-6)) < direct


def source(mode, act=0):
    """HIP source of one module: 'split' (the halves of rows and columns), or 'fwd', 'dx', 'dw'."""
    L = [_native.layer_header('matmul', 'halves')]
    if mode == 'split':
        return L[0]
    b = lambda v: 'true' if v else 'false'  # noqa: E731
    L += [f'typedef mm_fast_tile<MM_F16, {b(mode == "dw")}, {b(mode != "fwd")}, {", ".join(map(str, TILE))}, 64, true> '
          'tile_t;',
          f'extern "C" __global__ __launch_bounds__(tile_t::THREADS) void hv_{mode}(const unsigned short* A, '
          'const unsigned short* B, float* C, ']
    again = [f'typedef mm_tile<MM_F32, {b(mode == "dw")}, {b(mode != "fwd")}, {", ".join(map(str, AGAIN))}> again_t;',
             f'extern "C" __global__ __launch_bounds__(again_t::THREADS) void hv_again_{mode}(const float* A, const float* B, '
             'float* C, ']
    if mode == 'dw':
        L += ['float* part, const int* off, const unsigned* pa, unsigned* ma, const unsigned* pb, const unsigned* mb, '
              'int R, int M, int N, int E, int L) {',
              '  hv_outer_body<tile_t>(A, B, C, part, off, pa, ma, pb, mb, R, M, N, E, L);', '}', *again,
              'float* part, const int* off, const unsigned* pa, const unsigned* ma, const unsigned* pb, const unsigned* mb, '
              'long long lda, long long ldb, int R, int M, int N, int E, int L, int blocks) {',
              '  hv_again_outer_body<again_t>(A, B, C, part, off, pa, ma, pb, mb, lda, ldb, R, M, N, E, L, blocks);', '}']
    else:
        L += ['const float* bias, const float* res, float* slope, const int* off, unsigned* pa, const unsigned* pb, '
              'const unsigned* mb, long long ldr, int R, int N, int K, int E) {',
              f'  hv_rows_body<{b(mode == "dx")}, {act}, tile_t>(A, B, C, bias, res, slope, off, pa, pb, mb, ldr, R, N, K, E);',
              '}', *again,
              'const float* bias, const float* res, float* slope, const int* off, const unsigned* pa, const unsigned* pb, '
              'const unsigned* mb, long long lda, long long ldb, long long ldr, int R, int N, int K, int E, int tiles) {',
              f'  hv_again_rows_body<{b(mode == "dx")}, {act}, again_t>(A, B, C, bias, res, slope, off, pa, pb, mb, lda, ldb, ldr, '
              'R, N, K, E, tiles);', '}']
    return '\n'.join(L) + '\n'


@functools.lru_cache(maxsize=None)
def module(device, mode, act=0):
    """The loaded module (compiled on first use, kept per device)."""
    code = _native.compile_source(source(mode, act))
    with torch.cuda.device(device):
        if mode == 'split':
            return _native.Module(code, {_native.MH_HV_ROWS: ('hv_rows', 256, 1), _native.MH_HV_PEAKS: ('hv_peaks', 256, 1),
                                         _native.MH_HV_COLUMNS: ('hv_columns', 256, 1)})
        kind = _native.MH_HV_OUTER if mode == 'dw' else _native.MH_HV_MM
        return _native.Module(code, {kind: (f'hv_{mode}', 64 * TILE[0] * TILE[1], SIDE, SIDE), _native.MH_HV_AGAIN: (
            f'hv_again_{mode}', 64 * AGAIN[0] * AGAIN[1], AGAIN_SIDE, AGAIN_SIDE)})
