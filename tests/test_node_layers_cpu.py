"""
The trainable node layers without a GPU: refusals that come before any launch (Python and C ABI), their choices of tiles and
pieces over the whole range, and code generation of every module for gfx950.
"""
import itertools
import random

import pytest
import torch

import mace_hip_kernels as mhk
from mace_hip_kernels import _native, experts, halves, matmul, norms


def test_host_tensors_and_other_types_are_refused():
    x, w = torch.zeros(4, 8), torch.zeros(6, 8)
    for call, text in [(lambda: mhk.dense(x, w), 'GPU tensor'), (lambda: mhk.dense(x.double(), w), 'float32, bfloat16'),
                       (lambda: mhk.dense([1.0], w), 'list'), (lambda: mhk.block_norm(x), 'GPU tensor'),
                       (lambda: mhk.block_norm(x.int()), 'float32, bfloat16'),
                       (lambda: mhk.expert_dense(x, w[None], torch.zeros(2, dtype=torch.int32)), 'GPU tensor'),
                       (lambda: mhk.expert_order(torch.zeros(4, 1, dtype=torch.int32), 3), 'GPU tensor'),
                       (lambda: mhk.expert_order(torch.zeros(4, 1), 3), 'int32 or int64'),
                       (lambda: mhk.dispatch(x, None), 'GPU tensor'), (lambda: mhk.combine(x, None, None), 'GPU tensor')]:
        with pytest.raises(TypeError, match=text):
            call()


def test_c_entry_points_refuse_bad_arguments():
    lib = _native.load()
    one = torch.zeros(64)
    p = one.data_ptr()
    cases = [
        (lambda: lib.mh_mm_rows(None, p, 8, p, 8, p, None, None, 0, None, None, -1, 4, 8, 1, None), 'bad sizes'),
        (lambda: lib.mh_mm_rows(None, p, 8, p, 8, p, None, None, 0, None, None, 2, 4, 8, 2, None), 'bad sizes'),
        (lambda: lib.mh_mm_rows(None, None, 8, p, 8, p, None, None, 0, None, None, 2, 4, 8, 1, None), 'NULL'),
        (lambda: lib.mh_mm_rows(None, p, 7, p, 8, p, None, None, 0, None, None, 2, 4, 8, 1, None), 'overlap'),
        (lambda: lib.mh_mm_rows(None, p, 8, p, 8, p, None, p, 3, None, None, 2, 4, 8, 1, None), 'overlap'),
        (lambda: lib.mh_mm_rows(None, p, 8, p, 8, p, None, None, 0, None, None, 2, 4, 8, 1, None), 'not bound'),
        (lambda: lib.mh_mm_outer(None, p, 4, p, 4, None, None, None, 2, 4, 4, 1, 0, 1, None), 'NULL'),
        (lambda: lib.mh_mm_outer(None, p, 4, p, 4, p, None, None, 2, 4, 4, 1, 16, 1, None), 'NULL'),
        (lambda: lib.mh_mm_outer(None, p, 4, p, 4, p, p, None, 2, 4, 4, 1, 16, 0, None), 'pieces'),
        (lambda: lib.mh_mm_outer(None, p, 3, p, 4, p, p, None, 2, 4, 4, 1, 0, 1, None), 'overlap'),
        (lambda: lib.mh_mm_sum(None, p, p, None, 4, 1, 0, 8, None), 'bad sizes'),
        (lambda: lib.mh_mm_sum(None, None, p, None, 4, 1, 4, 8, None), 'NULL'),
        (lambda: lib.mh_mm_slope(None, p, 4, None, None, 0, None, None, None, 2, 4, 1, 4, 1, None), 'NULL'),
        (lambda: lib.mh_mm_slope(None, p, 4, None, None, 0, None, p, None, 2, 4, 1, 1, 2, None), 'one slot'),
        (lambda: lib.mh_mm_bwd(None, None, None, p, 4, p, p, 4, p, 4, None, None, 0, p, p, p, p, 2, 4, 4, 1, 4, 1, 0, 1, None),
         'goes with slope'),
        (lambda: lib.mh_mm_slope(None, p, 4, None, p, 3, None, None, None, 2, 4, 1, 4, 1, None), 'padded'),
        (lambda: lib.mh_mm_pad(None, p, 4, p, 2, 4, 12, None), 'bad sizes'),
        (lambda: lib.mh_hv_rows(None, p, 3, p, p, 2, 4, None), 'overlap'),
        (lambda: lib.mh_hv_columns(None, p, 4, p, p, None, 6, 4, 4, 2, 4, 4, None), 'bad sizes'),
        (lambda: lib.mh_hv_mm(None, p, p, p, None, None, 0, None, None, p, None, None, 2, 4, 4, 1, None), 'NULL'),
        (lambda: lib.mh_hv_outer(None, p, p, p, None, None, p, p, p, p, 2, 4, 4, 1, 4, 1, None), 'NULL'),
        (lambda: lib.mh_expert_order(None, p, 0, 4, 1025, None, 1, p, p, p, None), 'bad sizes'),
        (lambda: lib.mh_expert_order(None, p, 0, 4, 3, None, 2, p, p, p, None), 'NULL'),
        (lambda: lib.mh_dispatch(None, p, 8, p, p, p, 2, 1, 8, 1, 7, None), 'bad sizes'),
        (lambda: lib.mh_dispatch(None, p, 7, p, p, p, 2, 1, 8, 1, 1, None), 'overlap'),
        (lambda: lib.mh_combine(None, p, None, None, None, 0, p, 2, 1, 8, 1, None), 'NULL'),
        (lambda: lib.mh_combine(None, p, None, p, None, 0, p, 1 << 30, 2, 8, 1, None), 'bad sizes'),
        (lambda: lib.mh_combine_bwd(None, p, 8, None, p, p, p, p, p, 2, 1, 8, 1, 1, None), 'NULL'),
        (lambda: lib.mh_norm_fwd(None, p, p, None, None, None, None, None, p, None, 2, 8, 1e-6, None), 'NULL'),
        (lambda: lib.mh_norm_fwd(None, p, None, None, None, None, None, None, p, None, 2, 8, 1e-6, None), 'null module'),
        (lambda: lib.mh_norm_bwd(None, None, p, p, p, None, None, None, None, None, None, p, None, None, p, p, 2, 8, 1, None),
         'NULL'),
    ]
    for i, (call, text) in enumerate(cases):
        assert call() != 0, i
        assert text in lib.mh_last_error().decode(), (i, text, lib.mh_last_error())


def test_pieces_cover_all_rows_with_enough_slots():
    """Every sum over rows that is split has slots for all its pieces, however the rows fall into groups."""
    rng = random.Random(0)
    for _ in range(400):
        groups, M, N = rng.choice([1, 2, 7, 64, 300]), rng.choice([1, 40, 512, 4096]), rng.choice([8, 100, 1024, 2048])
        R = rng.choice([0, 1, 255, 257, 3000, 20000, 10 ** 6])
        cuts = sorted(rng.randint(0, R) for _ in range(groups - 1))
        sizes = [b - a for a, b in zip([0] + cuts, cuts + [R])]
        dt, fast = rng.choice([(torch.float32, False), (torch.bfloat16, True), (torch.float16, False)])
        tile, *plan = matmul._outer_plan(R, M, N, groups, groups > 1, dt, fast)
        assert (tile in matmul.FAST) == fast and tile in matmul.tiles(dt)
        for L, slots in (plan, matmul._halves_pieces(R, groups, groups > 1, -(-M // 128) * -(-N // 128))):
            if L == 0:
                assert slots == groups
            else:
                assert L % 64 == 0 and sum(-(-s // L) for s in sizes) <= slots <= 65535


def test_norm_shapes_hold_a_row():
    for dt, C in itertools.product(matmul.TYPES, list(range(1, 600)) + [1023, 1024, 1025, 4096, 4097, 8191, 8192]):
        tpr, nv = norms.shape(C, dt)
        assert tpr * nv * 16 // dt.itemsize >= C and 1 <= nv <= 2 and tpr <= 1024


@pytest.mark.parametrize('dt', list(matmul.TYPES), ids=str)
def test_every_module_compiles_for_gfx950(dt):
    sources = [matmul.source(dt, 'sum'), experts.source(dt), experts.order_source()]
    sources += [matmul.source(dt, mode, tile) for mode in ('fwd', 'dx', 'dw') for tile in matmul.tiles(dt)]
    sources += [norms.source(dt, 64, 1, True, True, 0), norms.source(dt, 512, 2, False, True, 2)]
    if dt == torch.float32:
        sources += [halves.source(mode) for mode in ('split', 'fwd', 'dx', 'dw')]
    for src in sources:
        assert _native.compile_source(src)[:4] == b'\x7fELF'
