"""CPU tier: the arithmetic that the linear products' pipelines rest on (linear_plan.h, built here by itself).

Loads and stores of a wavefront complete in the order in which they were issued, and a wait says how many may be
outstanding after it.  The kernels' order of loads, stores and waits is written down here once more, and what is
read has to have landed by the waits alone, not by the time that passes."""
import ctypes
import itertools
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / 'ferry_amd' / 'csrc'
SOURCE = '''
#include "linear_plan.h"
using namespace ferry::lin;
extern "C" int stages(int tm, int tn, int gathered_dw) { return ring_stages(tm, tn, gathered_dw); }
extern "C" int rows_wait(int kt, int ring, int filling) { return ring_rows_wait(kt, ring, filling); }
'''


@pytest.fixture(scope='module')
def plan(tmp_path_factory):
    where = tmp_path_factory.mktemp('plan')
    (where / 'plan.cpp').write_text(SOURCE)
    subprocess.run(['g++', '-std=c++17', '-O1', '-shared', '-fPIC', f'-I{CSRC}', '-o', str(where / 'plan.so'),
                    str(where / 'plan.cpp')], check=True)
    return ctypes.CDLL(str(where / 'plan.so'))


class Memory:
    """The loads and stores of one wavefront, in order."""

    def __init__(self):
        self.last, self.issued, self.landed = {}, 0, 0

    def issue(self, name, count):
        self.issued += count
        self.last[name] = self.issued

    def wait(self, outstanding):
        self.landed = max(self.landed, self.issued - outstanding)

    def read(self, name):
        assert self.last[name] <= self.landed, f'{name} is read before its loads have landed'


def ring(plan, kts, tm, tn, waves, stores, gathered_dw):
    """ring_kernel with gathered rows on tiles of kts stages, as its first wavefront runs it."""
    m, S = Memory(), plan.stages(tm, tn, gathered_dw)
    la, lb = tm // (8 * waves), tn // (8 * waves)
    per_stage, batch = la + lb, 64 // (lb * 512 // tn)   # batch: stages whose row numbers are loaded at once
    at = dict(tile=0, stage=0)

    def rows(tile):
        m.issue(('rows', tile, 0), 2)

    def begin_tile(tile):
        at.update(tile=tile, stage=0)
        if not gathered_dw:
            m.read(('rows', tile, 0))
        rows(tile + 1)

    def load_stage(filling):
        tile, k = at['tile'], at['stage']
        if tile < len(kts):
            if gathered_dw:
                if k % batch == 0:
                    if batch < S and k:
                        m.wait(batch * per_stage)
                    if kts[tile] - k > batch:
                        m.issue(('rows', tile, k // batch + 1), 2)
                m.read(('rows', tile, k // batch))
        m.issue(('stage', tile, k), per_stage)
        at['stage'] += 1
        if tile < len(kts) and at['stage'] == kts[tile]:
            if tile + 1 < len(kts):
                if plan.rows_wait(kts[tile], S, filling):
                    m.wait(0)
                begin_tile(tile + 1)
            else:
                at.update(tile=len(kts), stage=0)   # stages of zeros

    rows(0)
    m.wait(0)
    begin_tile(0)
    for _ in range(S):
        load_stage(True)
    m.wait((S - 1) * per_stage)
    m.read(('stage', 0, 0))
    order = [(t, k) for t, kt in enumerate(kts) for k in range(kt)] + [(len(kts), 0)]
    early = done = 0
    for t, kt in enumerate(kts):
        if not gathered_dw:
            m.issue(('bias', t), 1)
        for _ in range(kt):
            m.wait((S - 2) * per_stage + (stores if early else 0))
            early = max(early - 1, 0)
            done += 1
            m.read(('stage', *order[done]))
            load_stage(False)
        if not gathered_dw:
            if kt < S:
                m.wait(0)
            m.read(('bias', t))
        early = S - 1
        m.issue(('stores', t), stores)


RINGS = [(256, 128, 8, 8), (128, 128, 8, 4), (64, 128, 8, 2), (64, 64, 4, 2)]   # tile, wavefronts, stores of one


@pytest.mark.parametrize('gathered_dw', [False, True])
@pytest.mark.parametrize('shape', RINGS)
def test_row_numbers_have_landed(plan, shape, gathered_dw):
    """Tiles as long as the ring, shorter and longer ones, in every order of three."""
    if gathered_dw and shape[0] == 256:
        return   # that kernel has no such form
    S = plan.stages(*shape[:2], gathered_dw)
    lengths = sorted({1, 2, S - 2, S - 1, S, S + 1, S + 2, 2 * S, 2 * S + 3} - {0})
    for kts in itertools.product(lengths, repeat=3):
        ring(plan, kts, *shape, gathered_dw)
    for kt in range(1, 30):
        ring(plan, [kt] * 6, *shape, gathered_dw)
