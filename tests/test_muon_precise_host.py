"""Layout and work buffers of the products of pairs, checked without a GPU."""
import pathlib
import subprocess

import pytest

CSRC = pathlib.Path(__file__).resolve().parents[1] / 'dcss-auto_b200' / 'csrc'

LAYOUT = r'''
#include <algorithm>
#include <cstdio>
#include <vector>
#include "d1_muon.h"
using namespace d1::muon;
int main() {
    for (int64_t rows : {1, 64, 65, 128, 512, 1000})
        for (int64_t cols : {1, 63, 64, 90, 3136})
            for (bool precise : {false, true}) {
                Matrix m;
                int64_t block = 7, part = 0;
                place(m, rows, cols, block, part, precise);
                const int64_t n = (int64_t)m.rb * m.cb, s = (int64_t)m.sb * m.sb;
                if (block - 7 != blocks_needed(rows, cols, precise)) return 1;
                if (m.fine != (precise || m.sb == 1)) return 2;
                // X, what it is written to, A and F apart from one another and inside
                std::vector<std::pair<int64_t, int64_t>> spans{{m.hi[0], n}, {m.hi[1], n}, {m.lo, n}, {m.gram, m.fine ? 2 * s : s}, {m.quad, m.fine ? 2 * s : s}};
                // a tile that reads lo of other tiles' X writes elsewhere
                if (precise && m.sb > 1) {
                    if (m.lo2 == m.lo) return 3;
                    spans.push_back({m.lo2, n});
                } else if (m.lo2 != m.lo)
                    return 4;
                std::sort(spans.begin(), spans.end());
                int64_t at = 7;
                for (const auto &p : spans) {
                    if (p.first < at) return 5;
                    at = p.first + p.second;
                }
                if (at > block) return 6;
                Load load = load_of(2);
                load.add(m, 3);
                if (load.narrow() != (m.sb == 1)) return 7;
                if (load.depth[1] != m.sb * (m.fine ? 3 : 1)) return 8;
            }
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


def test_work_bytes_and_refusals(lib):
    size, single = lib.d1_orthogonalize_precise_work_bytes, lib.d1_orthogonalize_work_bytes
    assert size(1, 64, 300) == single(1, 64, 300) and size(2, 65, 65) == 2 * (32 * 8192 + 32) and size(0, 4, 4) == 0
    assert size(-1, 4, 4) == size(1, 0, 4) == size(1 << 25, 1, 1) == -1
    P = 1 << 20
    good = dict(x=P, ldx=8, step=64, type=0, count=2, rows=8, cols=8, y=2 * P, y_type=2, steps=5, work=P, s=None)
    for k, v in dict(x=None, ldx=-1, type=3, count=-1, rows=0, y=None, y_type=0, steps=0, work=None).items():
        assert lib.d1_orthogonalize_precise(*dict(good, **{k: v}).values()) == 9002, k
    assert lib.d1_orthogonalize_precise(*dict(good, count=0).values()) == 0


def test_plans(lib):
    from test_muon_host import table
    wide, narrow = ((1, 500, 300), (2, 64, 90))
    for shapes, more in (((wide,), 8 * 5 + 2 * 25), ((narrow,), 0), ((wide, narrow), 8 * 5 + 2 * 25)):
        t, p = table(*shapes), table(*shapes)
        for d in p:
            d.precise = 1
        n = len(shapes)
        assert lib.d1_muon_work_bytes(p, n) - lib.d1_muon_work_bytes(t, n) == 8192 * more
        assert lib.d1_muon_plan_bytes(p, n) > 0


DIVIDED = r"""
#include <cstdio>
#include "d1_muon.h"
using namespace d1::muon;
int main() {
    for (int rb = 1; rb <= 200; rb++)
        for (int cb = rb; cb <= 600; cb++) {
            Matrix m;
            int64_t block = 0, part = 0;
            place(m, rb * 64, cb * 64, block, part);
            Load load = load_of(2);
            load.add(m, 1);
            if (parts_for(load.full, load.depth[1]) > 1) return 1;
        }
    std::puts("ok");
}
"""


def test_single_products_apply_is_never_divided(tmp_path):
    """There is no kernel for it: no shape has few enough tiles of X' and long enough sums."""
    source = tmp_path / 'divided.cpp'
    source.write_text(DIVIDED)
    subprocess.run(['g++', '-std=c++17', '-O1', '-I', str(CSRC), str(source), '-o', str(tmp_path / 'divided')], check=True)
    assert subprocess.run([str(tmp_path / 'divided')], capture_output=True, text=True).stdout == 'ok\n'
