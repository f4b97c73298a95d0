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
extern "C" int early() { return kTile256Early; }
extern "C" unsigned half(int across, long there, unsigned ld2) { return half_offset(across, there, ld2); }
extern "C" int gathers(long c, long parts) { return tile256_gathers(c, parts); }
extern "C" long part(long c, long parts) { return part_length(c, parts); }
'''


@pytest.fixture(scope='module')
def plan(tmp_path_factory):
    where = tmp_path_factory.mktemp('plan')
    (where / 'plan.cpp').write_text(SOURCE)
    subprocess.run(['g++', '-std=c++17', '-O1', '-shared', '-fPIC', f'-I{CSRC}', '-o', str(where / 'plan.so'),
                    str(where / 'plan.cpp')], check=True)
    so = ctypes.CDLL(str(where / 'plan.so'))
    so.part.restype = ctypes.c_long
    so.half.argtypes = [ctypes.c_int, ctypes.c_long, ctypes.c_uint]
    so.gathers.argtypes = so.part.argtypes = [ctypes.c_long, ctypes.c_long]
    return so


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


def ring(plan, kts, tm, tn, waves, stores, gathered):
    """ring_kernel on tiles of kts stages, rows gathered for 'x' (forward), 'dw' or not at all, as its first wavefront runs
    it."""
    m, S = Memory(), plan.stages(tm, tn, gathered == 'dw')
    la, lb = tm // (8 * waves), tn // (8 * waves)
    per_stage, batch = la + lb, 64 // (lb * 512 // tn)   # batch: stages whose row numbers are loaded at once
    at = dict(tile=0, stage=0)

    def rows(tile):
        if gathered:
            m.issue(('rows', tile, 0), 2)

    def begin_tile(tile):
        at.update(tile=tile, stage=0)
        if gathered == 'x':
            m.read(('rows', tile, 0))
        rows(tile + 1)

    def load_stage(filling):
        tile, k = at['tile'], at['stage']
        if tile < len(kts):
            if gathered == 'dw':
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
                if gathered and plan.rows_wait(kts[tile], S, filling):
                    m.wait(0)
                begin_tile(tile + 1)
            else:
                at.update(tile=len(kts), stage=0)   # stages of zeros

    rows(0)
    if gathered:
        m.wait(0)
    begin_tile(0)
    for _ in range(S):
        load_stage(True)
    m.wait((S - 1) * per_stage)
    m.read(('stage', 0, 0))
    order = [(t, k) for t, kt in enumerate(kts) for k in range(kt)] + [(len(kts), 0)]
    early = done = 0
    for t, kt in enumerate(kts):
        if gathered != 'dw':
            m.issue(('bias', t), 1)
        for _ in range(kt):
            m.wait((S - 2) * per_stage + (stores if early else 0))
            early = max(early - 1, 0)
            done += 1
            m.read(('stage', *order[done]))
            load_stage(False)
        if gathered != 'dw':
            if kt < S:
                m.wait(0)
            m.read(('bias', t))
        early = S - 1
        m.issue(('stores', t), stores)


RINGS = [(256, 128, 8, 8), (128, 128, 8, 4), (64, 128, 8, 2), (64, 64, 4, 2)]   # tile, wavefronts, stores of one


@pytest.mark.parametrize('gathered', [None, 'x', 'dw'])
@pytest.mark.parametrize('shape', RINGS)
def test_stages_have_landed(plan, shape, gathered):
    """Tiles as long as the ring, shorter and longer ones, in every order of three."""
    if gathered == 'dw' and shape[0] == 256:
        return   # that kernel has no such form
    S = plan.stages(*shape[:2], gathered == 'dw')
    lengths = sorted({1, 2, S - 2, S - 1, S, S + 1, S + 2, 2 * S, 2 * S + 3} - {0})
    for kts in itertools.product(lengths, repeat=3):
        ring(plan, kts, *shape, gathered)
    for kt in range(1, 30):
        ring(plan, [kt] * 6, *shape, gathered)


def few(steps, mt, nb, ring, gathered):
    """A wavefront of few_kernel over its chunks of the contraction, of which the ring holds `ring`."""
    m, lw, lx = Memory(), 2 * nb, 2 * mt
    if gathered:
        m.issue('rows', 2)
    for i in range(ring):
        m.issue(('w', i), lw)
    if gathered:
        m.wait(ring * lw)
        m.read('rows')
    for i in range(ring):
        m.issue(('x', i), lx)
    more = max(steps - ring, 0)
    for i in range(steps):
        if i >= ring:
            m.wait(min(steps - 1 - i, ring - 1) * (lw + lx))
        else:
            m.wait((ring - 1 - i) * lx + (i * (lw + lx) if i <= more else 0))
        m.read(('w', i))
        m.read(('x', i))
        if i < more:
            m.issue(('w', i + ring), lw)
            m.issue(('x', i + ring), lx)


def test_chunks_have_landed():
    for mt, nb, ring_depth in ((1, 1, 4), (1, 2, 3), (2, 2, 2), (4, 2, 2), (4, 4, 2)):
        for steps in range(1, 20):
            few(steps, mt, nb, ring_depth, False)
            few(steps, mt, nb, ring_depth, True)


def tile256(plan, lengths, gathered):
    """tile256 on tiles whose contractions have these lengths, rows gathered for 'x' (forward), 'dw' or not at all, as its
    first wavefront runs it: four phases a stage, each of which reads one half of an operand and loads another."""
    m = Memory()
    kts = [-(-n // 64) for n in lengths]
    stream = dict(tile=0, stage=0)

    def begin_tile(tile):
        stream.update(tile=tile, stage=0)
        if gathered == 'x' and tile < len(kts):
            m.read(('rows', tile, 0))

    def begin_stage():
        tile, k = stream['tile'], stream['stage']
        if gathered == 'dw' and tile < len(kts):
            if k % 8 == 0 and kts[tile] - k > 8:
                m.issue(('rows', tile, k // 8 + 1), 2)
            if k < kts[tile]:
                m.read(('rows', tile, k // 8))

    def load(half):
        m.issue((half, stream['tile'], stream['stage']), 2)

    if gathered:
        m.issue(('rows', 0, 0), 2)
        m.wait(0)
    begin_tile(0)
    for _ in range(2):
        begin_stage()
        for half in ('B0', 'A0', 'B1', 'A1'):
            load(half)
        stream['stage'] += 1
    m.wait(12)
    m.read(('B0', 0, 0))
    m.wait(12)
    stores = False
    for t, n in enumerate(lengths):
        pairs = (n + 127) // 128
        early = plan.early() if stores else 0
        if gathered == 'x':
            m.issue(('bias', t), 1)
        if gathered:
            m.issue(('rows', t + 1, 0), 2)
        if gathered == 'dw' and pairs <= 1:
            m.wait(0)
        stages = max(2 * pairs, 2)
        for k in range(stages):
            if k == stages - 2:
                begin_tile(t + 1)   # the last two stages load the next tile's first two
            after = (t, k + 1) if k + 1 < stages else (t + 1, 0)
            begin_stage()
            for reads, loads in ((('A0', t, k), 'B0'), (('B1', t, k), 'A0'), (('A1', t, k), 'B1'), (('B0', *after), 'A1')):
                m.read(reads)
                load(loads)
                m.wait(28 if early > 0 else 12)
                early -= 1
            stream['stage'] += 1
        if gathered == 'x':
            m.read(('bias', t))
        m.issue(('stores', t), 16)
        stores = True


LENGTHS = [1, 64, 65, 128, 129, 192, 256, 500, 512, 513, 640, 1030, 1600]


@pytest.mark.parametrize('gathered', [None, 'x', 'dw'])
def test_halves_have_landed(plan, gathered):
    """Tiles of any contractions follow each other (gathered forward ones of more than 128)."""
    for lengths in itertools.product([n for n in LENGTHS if gathered != 'x' or n > 128], repeat=3):
        tile256(plan, lengths, gathered)
    if gathered != 'x':
        tile256(plan, [0, 0, 300, 0], gathered)


@pytest.mark.parametrize('parts', [1, 2, 4, 8, 16])
def test_row_numbers_of_parts_have_landed(plan, parts):
    """A gathered forward product in parts, the last of which may be short or empty: tile256's tiles of one workgroup are
    of any parts, so each is followed by each."""
    taken = 0
    for k in [*range(128 * parts, 1100 * parts, 8 * parts + 8), 14464, 14400, 20000, 65544]:
        if plan.gathers(k, parts):
            per = plan.part(k, parts)
            lengths = [max(0, min(per, k - s * per)) for s in range(parts)]
            assert sum(lengths) == k
            for pair in itertools.product(sorted(set(lengths)), repeat=2):
                tile256(plan, [*pair, per], 'x')
            taken += 1
    assert taken > 10


@pytest.mark.parametrize('across', [False, True])
def test_offsets_lie_in_their_buffers(plan, across):
    """An operand's buffer ends with the last element of the tile's last row.  The offset of every stage and half that
    tile256 loads has to lie in it: lanes are compared with what is left behind the offset, unsigned."""
    for there, c, spare in itertools.product((1, 8, 64, 120, 127, 128, 129, 136, 248, 256, 300), (1, 7, 8, 64, 65, 128, 129, 193, 8193),
                                             (0, 8, 1000)):
        inside = min(there, 256)
        # across: c rows of the indices; direct: a row of the contraction for every index
        rows, last = (c, inside) if across else (inside, c)
        ld = last + spare
        size = ((rows - 1) * ld + last) * 2
        half = plan.half(across, there, 2 * ld)
        for stage in range((c + 63) // 64):
            at = stage * 64 * (ld if across else 1) * 2
            assert at < size and at + half < size
            if there > 128:   # the half that is there: its first element
                assert half == 128 * 2 * (1 if across else ld)


def test_offsets_of_gathered_rows(plan):
    """Rows of x by their numbers, of which there may be one alone."""
    for there, x_rows in itertools.product((1, 8, 128, 129, 256), (1, 2, 100)):
        size = ((x_rows - 1) * there + min(there, 256)) * 2
        assert plan.half(True, there, 2 * there) < size
