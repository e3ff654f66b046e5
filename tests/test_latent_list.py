"""The list of work of attention over a cache of latent rows (fa_latent_list.h), compiled for the host: a sequence's units are those of its blocks,
every unit belongs to the block that a walk over them finds, and a block's tiles hold all that its rows see, up to the largest calls."""
import ctypes
import os
import random
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'aotriton_amd', 'csrc')
SOURCE = '''
#include "fa_latent_list.h"
struct Args { int32_t hq, block_rows, block_shift, group_shift, step_shift, margin; };
struct Call { Args a; int32_t start, tokens, length; int64_t room; };
static fa::LatentSeq seq(const Call& c) { return fa::latent_seq_of(c.a, c.start, c.tokens, c.length, c.room); }
extern "C" int64_t units(const Call* c) { return seq(*c).units(c->a); }
extern "C" int block_of(const Call* c, int64_t rel, int* unit) { return seq(*c).block_of(c->a, rel, *unit); }
extern "C" int tiles_of(const Call* c, int block) { return seq(*c).tiles_of(c->a, block); }
extern "C" int blocks(const Call* c) { return seq(*c).blocks; }
extern "C" int last_slot(const Call* c, int t) { return seq(*c).last_slot(t); }
'''


class Call(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int32) for n in ('hq', 'block_rows', 'block_shift', 'group_shift', 'step_shift', 'margin', 'start', 'tokens', 'length')] + [('room', ctypes.c_int64)]


@pytest.fixture(scope='module')
def lib(tmp_path_factory):
    if shutil.which('g++') is None:
        pytest.skip('no host compiler')
    d = tmp_path_factory.mktemp('latent_list')
    (d / 'x.cpp').write_text(SOURCE)
    subprocess.run(['g++', '-O2', '-std=c++17', '-shared', '-fPIC', '-fwrapv', '-I', CSRC, str(d / 'x.cpp'), '-o', str(d / 'x.so')], check=True)
    x = ctypes.CDLL(str(d / 'x.so'))
    x.units.restype = ctypes.c_int64
    x.block_of.argtypes = [ctypes.c_void_p, ctypes.c_int64, ctypes.c_void_p]
    return x


def _call(hq, block_rows, margin, tokens, length, room=1 << 29):
    """as the entry point forms them"""
    c = Call(hq, block_rows, block_rows.bit_length() - 1, 0, 0, margin, 0, tokens, length, room)
    while (2 << c.group_shift) * block_rows <= 32 * hq:
        c.group_shift += 1
    while (32 * hq << c.step_shift) < block_rows:
        c.step_shift += 1
    return c


def _block(lib, c, rel):
    unit = ctypes.c_int32(-1)
    return lib.block_of(ctypes.byref(c), rel, ctypes.byref(unit)), unit.value


CALLS = [(hq, rows, margin, tokens, length) for hq in (1, 3, 16, 40, 128) for rows in (32, 64, 128) for margin in (5, -1) for tokens, length in
         ((1, 0), (1, 4095), (33, 31), (70, 300), (300, 0), (129, 1000))]


@pytest.mark.parametrize('hq', [1, 3, 16, 40, 128])
def test_every_unit(lib, hq):
    for c in (_call(*x) for x in CALLS if x[0] == hq):
        p = ctypes.byref(c)
        at = 0
        for b in range(lib.blocks(p)):
            n = 1 if c.margin < 0 else lib.tiles_of(p, b) + 2 * c.margin
            for unit in {0, n // 2, n - 1}:
                assert _block(lib, c, at + unit) == (b, unit)
            at += n
            last = min((b + 1) * c.block_rows, c.tokens * hq) - 1
            assert lib.tiles_of(p, b) * 32 > c.length + last // hq
        assert at == lib.units(p)


@pytest.mark.parametrize('hq,rows,tokens,length', [
    (1024, 32, 200, 1 << 28), (1024, 32, 3000, (1 << 29) - 5000), (1024, 128, 3000, 1 << 28), (65536, 32, 100, 1 << 22), (65536, 128, 5000, 1 << 23), (65536, 32, 16383, 5),
    (300, 64, 3 << 20, 0), (1, 128, (1 << 30) - 1, 1 << 28)])
def test_the_largest_sequences(lib, hq, rows, tokens, length):
    """groups whose blocks' tiles together pass 32 bits"""
    c = _call(hq, rows, 5, tokens, length)
    p = ctypes.byref(c)
    blocks, group = lib.blocks(p), 1 << c.group_shift
    rng = random.Random(hq + tokens)
    wanted = sorted({0, 1, blocks - 1, blocks // 2} | {rng.randrange(blocks) for _ in range(40)})
    at = g = 0
    for b in wanted:
        while (g + 1) * group <= b:          # (whole groups in front; past the last short one all blocks have the same tiles)
            at += group * (lib.tiles_of(p, g * group) + 10)
            g += 1
        t = lib.tiles_of(p, b) + 10
        first = at + (b - g * group) * t
        for unit in (0, 1, t // 2, t - 1):
            assert _block(lib, c, first + unit) == (b, unit)
    assert first + t == lib.units(p)


@pytest.mark.parametrize('room', [0, 16, 1 << 29])
@pytest.mark.parametrize('length', [-2 ** 31, -2 ** 31 + 3, -1, 0, 1, 15, 16, 100, (1 << 29) - 2, 1 << 29, 2 ** 31 - 1000, 2 ** 31 - 2, 2 ** 31 - 1])
def test_the_last_slot_that_a_token_sees(lib, length, room):
    """no further than the table goes, wherever the length stands; none of a sequence that is not there"""
    tokens = 1 << 20
    c = _call(16, 32, 5, tokens, length, room)
    for t in (0, 1, 2, 3, 14, 15, 16, 999, 1000, tokens - 1):
        assert lib.last_slot(ctypes.byref(c), t) == (min(length + t, room - 1) if length >= 0 else -1)
