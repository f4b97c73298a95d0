"""CPU tier: how the MXFP4 expert FFN cuts its launches (mxfp4_plan.h, host arithmetic, built here by itself): what
spare CUs leave free, and that every tile and every small expert has a workgroup."""
import ctypes
import itertools
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / 'ferry_amd' / 'csrc'
SOURCE = '''
#include "mxfp4_plan.h"
extern "C" void plan(int quantised, long col_tiles, const long* rows, int small, int small_cols, long cus, long spare, int* out) {
  const int64_t tiles[3] = {rows[0], rows[1], rows[2]};
  const ferry::MxPlan p = ferry::plan_tiles(quantised, col_tiles, tiles, small, small_cols, cus, spare);
  out[0] = p.large, out[1] = p.tile_rows, out[2] = p.tile_wgs, out[3] = p.items, out[4] = p.small_wgs;
}
'''


@pytest.fixture(scope='module')
def plan(tmp_path_factory):
    where = tmp_path_factory.mktemp('plan')
    (where / 'plan.cpp').write_text(SOURCE)
    subprocess.run(['g++', '-std=c++17', '-O1', '-shared', '-fPIC', f'-I{CSRC}', '-o', str(where / 'plan.so'),
                    str(where / 'plan.cpp')], check=True)
    fn = ctypes.CDLL(str(where / 'plan.so')).plan

    def call(quantised, col_tiles, rows, small, small_cols, cus=256, spare=0):
        """rows: of each larger expert"""
        tiles = [sum(-(-n // r) for n in rows) for r in (256, 128, 64)]
        out = (ctypes.c_int * 5)()
        fn(int(quantised), ctypes.c_long(col_tiles), (ctypes.c_long * 3)(*tiles), small, small_cols, ctypes.c_long(cus),
           ctypes.c_long(spare), out)
        return dict(zip(('large', 'tile_rows', 'tile_wgs', 'items', 'small_wgs'), out))
    return call


ROWS = [[17], [40] * 30, [300, 65, 17], [5000, 900] + [100] * 40, [65536], [600] * 128]
CALLS = list(itertools.product([False, True], [1, 6, 8, 11, 22], ROWS, [0, 1, 47, 256]))


@pytest.mark.parametrize('spare', [1, 5, 16, 100, 127, 128])
def test_spare_cus_stay_free(plan, spare):
    for quantised, cols, rows, small in CALLS:
        p = plan(quantised, cols, rows, small, 32, spare=spare)
        per_cu = 1 if p['large'] else 2
        assert p['tile_wgs'] + p['small_wgs'] <= per_cu * (256 - spare)
        assert p['small_wgs'] == 0 and p['tile_wgs'] >= 8 and p['tile_wgs'] % 8 == 0


def test_few_cus(plan):
    for cus, spare in ((32, 16), (32, 128), (64, 60), (8, 128)):
        for quantised, cols, rows, small in CALLS:
            p = plan(quantised, cols, rows, small, 32, cus=cus, spare=spare)
            assert 8 <= p['tile_wgs'] <= (1 if p['large'] else 2) * max(cus - spare, 8)


def test_everything_has_a_workgroup(plan):
    for quantised, cols, rows, small in CALLS:
        p = plan(quantised, cols, rows, small, 32)
        work = 2 if p['large'] else 1      # workgroups of small experts that one of the launch does
        assert p['small_wgs'] * work * p['items'] == small * 32
        assert p['tile_wgs'] % 8 == 0 and 8 <= p['tile_wgs'] <= (256 if p['large'] else 512)
        assert p['tile_rows'] == 256 if p['large'] else p['tile_rows'] in (64, 128)
        assert quantised or not p['large']
        tiles = sum(-(-n // p['tile_rows']) for n in rows) * (2 * cols if quantised and not p['large'] else cols)
        assert p['tile_wgs'] <= -(-tiles // 8) * 8
