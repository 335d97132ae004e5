"""row_piece (csrc/d1_rows.h): the 16-byte pieces by which layer norm copies rows
that start anywhere. Every source is aligned, also that of a piece that reads
nothing; together the pieces read the row, and before it only back to its
boundary. Built with the host compiler; no GPU."""
import ctypes as C
import pathlib
import subprocess

CSRC = pathlib.Path(__file__).resolve().parents[1] / 'dcss-auto_b200' / 'csrc'


def test_pieces(tmp_path):
    (tmp_path / 'piece.cpp').write_text(f'''#include "{CSRC / 'd1_rows.h'}"
extern "C" int piece(uint64_t row, int size, int p, uint64_t *from) {{
    const d1::RowPiece r = d1::row_piece((uintptr_t)row, size, p);
    *from = r.from;
    return r.bytes;
}}
''')
    subprocess.run(['g++', '-O1', '-std=c++17', '-shared', '-fPIC', '-o', str(tmp_path / 'piece.so'), str(tmp_path / 'piece.cpp')], check=True)
    f = C.CDLL(str(tmp_path / 'piece.so')).piece
    f.argtypes = [C.c_uint64, C.c_int, C.c_int, C.POINTER(C.c_uint64)]
    at = C.c_uint64()
    for offset in range(16):
        row = (1 << 44) + 4096 + offset
        for size in list(range(1, 70)) + [2222, 4444]:
            covered = 0
            for p in range(0, size + 15, 16):     # as far as a row at any offset goes
                n = f(row, size, p, C.byref(at))
                assert at.value % 16 == 0 and 0 <= n <= 16
                if n:
                    assert at.value == row - offset + p
                    covered += n
                else:
                    assert at.value == row - offset and row - offset + p >= row + size
            assert covered == offset + size
