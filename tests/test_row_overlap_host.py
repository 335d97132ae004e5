"""rows_overlap (csrc/d1_rows.h) against the bytes themselves, and the entries
that refuse outputs by it. Built with the host compiler; no GPU."""
import ctypes as C
import pathlib
import random
import subprocess

import pytest

CSRC = pathlib.Path(__file__).resolve().parents[1] / 'dcss-auto_b200' / 'csrc'
BAD = 9002


@pytest.fixture(scope='module')
def overlap(tmp_path_factory):
    at = tmp_path_factory.mktemp('rows')
    (at / 'rows.cpp').write_text(f'''#include "{CSRC / 'd1_rows.h'}"
extern "C" int overlap(uint64_t p, int64_t rp, int64_t wp, int64_t lp, uint64_t q, int64_t rq, int64_t wq, int64_t lq) {{
    return d1::rows_overlap({{(uintptr_t)p, rp, wp, lp}}, {{(uintptr_t)q, rq, wq, lq}});
}}
''')
    subprocess.run(['g++', '-O1', '-std=c++17', '-shared', '-fPIC', '-o', str(at / 'rows.so'), str(at / 'rows.cpp')], check=True)
    f = C.CDLL(str(at / 'rows.so')).overlap
    f.argtypes = [C.c_uint64, C.c_int64, C.c_int64, C.c_int64] * 2
    return f


def test_against_the_bytes(overlap):
    rng = random.Random(4)
    seen = [0, 0]
    for _ in range(40000):
        same = rng.random() < 0.6
        a = [rng.randrange(1000, 1100), rng.randrange(0, 6), rng.randrange(1, 9), rng.randrange(0, 30)]
        b = [rng.randrange(1000, 1100), rng.randrange(0, 6), rng.randrange(1, 9), a[3] if same else rng.randrange(0, 30)]
        cells = [{p + i * ld + k for i in range(rows) for k in range(w)} for p, rows, w, ld in (a, b)]
        want = bool(cells[0] & cells[1])
        assert bool(overlap(*a, *b)) == want == bool(overlap(*b, *a)), (a, b)
        seen[want] += 1
    assert min(seen) > 5000


def test_large_ones(overlap):
    n = 1 << 33
    assert not overlap(1 << 40, 1 << 20, n // 2, n, (1 << 40) + n // 2, 1 << 20, n // 2, n)
    assert overlap(1 << 40, 1 << 20, n // 2 + 1, n, (1 << 40) + n // 2, 1 << 20, n // 2, n)
    assert not overlap(1 << 20, 1 << 20, 2, 4, (1 << 20) + (1 << 22), 1 << 20, 2, 4)


def test_the_gradient_of_log_probabilities_is_the_logits_or_apart():
    from d1 import _lib
    lib, P = _lib.library(), 1 << 20
    good = dict(x=P, ld=40, type=1, rows=4, vocab=40, tokens=P << 4, legal=None, ldl=0, t=1.0, stats=P << 5, ent=P << 6, dl=P << 7,
                dh=P << 8, d=P, ldd=40, s=None)
    for bad in (dict(d=P + 2), dict(d=P + 80), dict(d=P + 3 * 80 + 78), dict(d=P - 2), dict(ldd=48), dict(ld=60, ldd=60, d=P + 42),
                dict(ld=80, ldd=100, d=P + 80)):
        assert lib.d1_token_logprob_backward(*dict(good, **bad).values()) == BAD, bad


def test_layer_norm_in_place_or_apart():
    from d1 import _lib
    lib, P = _lib.library(), 1 << 20
    good = dict(x=P, ldx=8, type=1, rows=4, n=8, w=P << 4, b=P << 5, eps=1e-5, y=P, ldy=8, mean=P << 6, rstd=P << 7, s=None)
    for bad in (dict(y=P + 16), dict(y=P - 16), dict(y=P + 2), dict(ldy=16), dict(ldx=20, ldy=20, y=P + 14), dict(ldx=0), dict(ldx=4, ldy=8, y=P + 8)):
        assert lib.d1_layer_norm(*dict(good, **bad).values()) == BAD, bad
    good = dict(dy=P, lddy=8, x=P << 1, ldx=8, type=0, rows=4, n=8, w=None, mean=P << 4, rstd=P << 5, dx=P << 2, lddx=8, dw=P << 6,
                db=P << 7, work=P << 8, s=None)
    for bad in (dict(dx=P), dict(dx=P << 1), dict(dx=P + 32), dict(dx=(P << 1) - 4), dict(dx=(P << 1) + 100)):
        assert lib.d1_layer_norm_backward(*dict(good, **bad).values()) == BAD, bad
