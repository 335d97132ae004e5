"""How the Newton-Schulz products divide their work, and what the C entries refuse, checked without a GPU."""
import ctypes as C
import pathlib
import subprocess

import pytest
import torch

BAD, LARGE = 9002, 9003
P = 1 << 20  # an aligned address that is never read
CSRC = pathlib.Path(__file__).resolve().parents[1] / 'dcss-auto_b200' / 'csrc'

LAYOUT = r'''
#include <cstdio>
#include <set>
#include <utility>
#include "d1_muon.h"
using namespace d1::muon;
int main() {
    for (int64_t rows : {1, 28, 64, 65, 512, 1000, 8192})
        for (int64_t cols : {1, 63, 64, 90, 3136, 8192}) {
            Matrix m;
            int64_t block = 7, part = 3;
            place(m, rows, cols, block, part);
            const int64_t n = (int64_t)m.rb * m.cb, s = m.sb == 1 ? 2 : (int64_t)m.sb * m.sb;
            if (block - 7 != blocks_needed(rows, cols) || part - 3 != m.parts || m.parts < 1 || m.parts > 256) return 1;
            if (m.hi[0] != 7 || m.hi[1] != m.hi[0] + n || m.lo != m.hi[1] + n || m.gram != m.lo + n || m.quad != m.gram + s || block != m.quad + s || m.fine != (m.sb == 1)) return 2;
            if (m.sb != (m.tall ? m.cb : m.rb) || m.tall != (rows > cols) || (int64_t)m.rb * 64 < rows || (int64_t)(m.rb - 1) * 64 >= rows) return 3;
            for (int side : {2, 4}) {
                std::set<std::pair<int, int>> seen;
                const int t = tiles_of(m.sb, side);
                for (int k = 0; k < symmetric_tiles(m, side); k++) {
                    int i, j;
                    symmetric_tile(k, i, j);
                    if (j > i || i >= t || j < 0 || !seen.insert({i, j}).second) return 4;
                }
                if ((int64_t)seen.size() != (int64_t)t * (t + 1) / 2) return 5;
                seen.clear();
                const int tm = tiles_of(m.rb, side), tn = tiles_of(m.cb, side);
                for (int k = 0; k < full_tiles(m, side); k++) {
                    int i, j;
                    grouped_tile(k, tm, tn, i, j);
                    if (i < 0 || i >= tm || j < 0 || j >= tn || !seen.insert({i, j}).second) return 6;
                }
                if ((int64_t)seen.size() != (int64_t)tm * tn) return 7;
            }
        }
    int i, j;
    for (int r : {0, 1, 4095, 4096, 5000, 20000, 40000, 65534}) {
        symmetric_tile((int)((int64_t)r * (r + 1) / 2), i, j);
        if (i != r || j != 0) return 8;
        symmetric_tile((int)((int64_t)r * (r + 1) / 2 + r), i, j);
        if (i != r || j != r) return 8;
    }
    for (int64_t tiles : {1, 10, 14, 15, 32, 33, 74, 75, 148, 1000})
        for (int depth : {1, 8, 16, 49, 1000}) {
            const int n = parts_for(tiles, depth);
            if (n != 1 && n != 2 && n != 4 && n != 8) return 10;
            if (n > 1 && (tiles * n > 148 || depth < 10)) return 11;
        }
    if (parts_for(10, 49) != 8 || parts_for(24, 49) != 4 || parts_for(74, 49) != 2 || parts_for(75, 1000) != 1 || parts_for(1, 8) != 1) return 12;
    for (int64_t rows : {1, 64, 128, 129, 700})
        for (int64_t cols : {1, 128, 600, 2000, 5000})
            for (int64_t count : {1, 14, 15, 33, 148, 149}) {
                Load load = load_of(2);
                Matrix m;
                int64_t block = 0, part = 0;
                place(m, rows, cols, block, part);
                load.add(m, count);
                const int n = load.small_together();
                if (n && (symmetric_tiles(m, 2) != 1 || full_tiles(m, 2) > 2 * n || count * n > 148 || (n & (n - 1)) || n > 8)) return 16;
                if (!n && symmetric_tiles(m, 2) == 1 && full_tiles(m, 2) <= 2 && count <= 148) return 17;
                if (n && count == 1 && m.cb <= 10 && m.rb <= 2 && n < 8 && n < full_tiles(m, 2)) return 18;
            }
    for (int64_t rows : {1, 8, 9, 64})
        for (int64_t cols : {1, 64, 500, 513, 1024, 1025, 20000})
            for (int64_t count : {1, 14, 15, 33, 149, 100000}) {
                Load load = load_of(2);
                Matrix m;
                int64_t block = 0, part = 0;
                place(m, cols, rows, block, part);
                load.add(m, count);
                if (!load.narrow() || load.most_parts != m.parts || load.most_eights != (int)((rows < cols ? rows : cols) + 7) / 8) return 19;
                const int n = load.whole_together(), c = load.clusters(8);
                if (n && ((n & (n - 1)) || n > 8 || m.parts > 2 * n || (n > 1 && count * n > room(n)))) return 20;
                if (!n && (m.parts <= 2 || (count == 1 && cols <= (rows <= 32 ? 1024 : 512)))) return 21;
                if (c < 1 || c > 8 || (c > 1 && count * c > room(c))) return 22;
                Matrix wide;
                place(wide, 65, 65, block, part);
                load.add(wide, 1);
                if (load.narrow()) return 23;
            }
    for (int64_t n : {64, 1000, 8192}) {
        Load small = load_of(2), large = load_of(4);
        Matrix m;
        int64_t block = 0, part = 0;
        place(m, n, n, block, part);
        small.add(m, 3), large.add(m, 3);
        if (small.symmetric != 3 * symmetric_tiles(m, 2) || large.full != 3 * full_tiles(m, 4) || small.depth[0] != (int)(n + 63) / 64 * (m.fine ? 3 : 1)) return 13;
        if (n == 64 && !(small.microseconds() < large.microseconds())) return 14;
        if (n == 8192 && !(large.microseconds() < small.microseconds())) return 15;
    }
    if (blocks_needed(0, 4) != -1 || blocks_needed(4, (1 << 21) + 1) != -1 || blocks_needed(1 << 21, 1) != 3 * 32768 + 4) return 9;
    std::puts("ok");
}
'''


def test_layout(tmp_path):
    source = tmp_path / 'layout.cpp'
    source.write_text(LAYOUT)
    subprocess.run(['g++', '-std=c++17', '-O1', '-I', str(CSRC), str(source), '-o', str(tmp_path / 'layout')], check=True)
    assert subprocess.run([str(tmp_path / 'layout')], capture_output=True, text=True).stdout == 'ok\n'


@pytest.fixture(scope='module')
def lib():
    from d1 import _lib
    return _lib.library()


def table(*shapes, **change):
    from d1.muon import _Tensor
    t = (_Tensor * len(shapes))()
    for i, (count, rows, cols) in enumerate(shapes):
        t[i] = _Tensor(*dict(dict(param=P, grad=2 * P, copy=None, count=count, rows=rows, cols=cols, decay=0.1, grad_type=0, reserved=0), **change).values())
    return t


def test_plans(lib):
    from d1.muon import _Tensor
    assert C.sizeof(_Tensor) == 64  # D1MuonTensor
    shapes = [(1, 32, 90), (3, 512, 100), (1, 1, 1), (2, 64, 64), (0, 5, 5)]
    t = table(*shapes)
    size, work = lib.d1_muon_plan_bytes(t, 5), lib.d1_muon_work_bytes(t, 5)
    blocks = sum(c * (3 * -(-r // 64) * -(-k // 64) + 2 * max(2 * (min(r, k) <= 64), min(-(-r // 64), -(-k // 64)) ** 2)) for c, r, k in shapes)
    assert work >= 8192 * blocks and size > 7 * 100
    host = (C.c_uint64 * ((size + 7) // 8))()
    assert lib.d1_muon_plan(t, 5, P, host, C.sizeof(host)) == 0
    head = list((C.c_int64 * 8).from_buffer(host))
    assert head[0] == size and head[1] == 7 and head[7] == blocks
    assert head[2] == sum(c * min(256, -(-r // 64) * -(-k // 64)) for c, r, k in shapes)
    assert lib.d1_muon_plan(t, 5, P, host, size - 1) == BAD
    assert lib.d1_muon_plan(t, 5, None, host, size) == BAD and lib.d1_muon_plan(t, 5, P + 4, host, size) == BAD
    for change in (dict(param=None), dict(grad=None), dict(grad_type=2), dict(grad_type=-1), dict(decay=float('nan')), dict(param=P + 2), dict(copy=P + 1)):
        assert lib.d1_muon_plan(table((1, 4, 4), **change), 1, P, host, size) == BAD, change
    for shape in ((1, 0, 4), (1, 4, 0), (-1, 4, 4), (1, 1 << 22, 4), (1, 4, 1 << 22), (1 << 25, 1, 1), (1 << 23, 64, 64), (0, 4, 4)):
        assert lib.d1_muon_plan_bytes(table(shape), 1) == -1 and lib.d1_muon_work_bytes(table(shape), 1) == -1, shape
    assert lib.d1_muon_plan_bytes(None, 1) == lib.d1_muon_plan_bytes(t, 0) == -1


def test_entries(lib):
    good = dict(host=P, plan=P, lr=1e-3, mu=0.9, nesterov=1, steps=5, work=P, s=None)
    for k, v in dict(host=None, plan=None, work=None, lr=float('nan'), mu=1.0, steps=0).items():
        assert lib.d1_muon(*dict(good, **{k: v}).values()) == BAD, k
    for k, v in dict(mu=-0.1, steps=65, work=P + 64, plan=P + 4).items():
        assert lib.d1_muon(*dict(good, **{k: v}).values()) == BAD, k
    good = dict(x=P, ldx=8, step=64, type=0, count=2, rows=8, cols=8, y=2 * P, y_type=1, steps=5, work=P, s=None)
    for k, v in dict(x=None, ldx=-1, step=-1, type=3, count=-1, rows=0, cols=0, y=None, y_type=0, steps=0, work=None).items():
        assert lib.d1_orthogonalize(*dict(good, **{k: v}).values()) == BAD, k
    for k, v in dict(x=P + 2, y=P + 508, type=-1, count=1 << 25, rows=1 << 22, steps=65, work=P + 8, y_type=3).items():
        assert lib.d1_orthogonalize(*dict(good, **{k: v}).values()) == BAD, k
    assert lib.d1_orthogonalize(*dict(good, count=0).values()) == 0
    size = lib.d1_orthogonalize_work_bytes
    assert size(1, 64, 64) == 7 * 8192 + 8 and size(0, 4, 4) == 0 and size(3, 65, 1) == 3 * (10 * 8192 + 16) and size(1, 65, 65) == 20 * 8192 + 32
    assert size(-1, 4, 4) == size(1, 0, 4) == size(1 << 25, 1, 1) == -1


def test_host_tensors_are_refused():
    from d1.muon import Muon, orthogonalize
    x = torch.zeros(4, 8)
    for bad in (lambda: Muon([x], [x]), lambda: orthogonalize(x)):
        with pytest.raises(ValueError):
            bad()
