"""How many CTAs join the records of attention behind a shared prefix: csrc/route.hpp, compiled with g++ and called here."""
import ctypes as C
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "tile-rs_b200" / "csrc"
SMS = 148


@pytest.fixture(scope="module")
def ctas(tmp_path_factory):
    out = tmp_path_factory.mktemp("join") / "libjoin.so"
    src = out.with_suffix(".cpp")
    src.write_text('#include "route.hpp"\nextern "C" long long ctas(long long rows, long long at_once, long long batch, int per_sm, int sms) {\n'
                   "  return tsm100::route::join_ctas(rows, at_once, batch, per_sm, sms);\n}\n")
    subprocess.run(["/usr/bin/g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{CSRC}", str(src), "-o", str(out)], check=True)
    f = C.CDLL(str(out)).ctas
    f.restype = C.c_longlong
    return lambda rows, at_once, batch, per_sm: f(C.c_longlong(rows), C.c_longlong(at_once), C.c_longlong(batch), per_sm, SMS)


@pytest.mark.parametrize("rows,at_once,batch,per_sm,want", [
    (32, 2, 8, 4, 16), (1, 2, 1, 4, 1), (2048 * 32, 2, 1, 4, 592), (2048 * 32, 1, 1, 2, 296), (4096 * 32, 2, 2, 4, 296), (1000, 2, 1, 4, 500), (64 * 32, 2, 64, 4, 64), (2048 * 32, 2, 1000, 4, 64)])
def test_ctas_of_a_sequence(ctas, rows, at_once, batch, per_sm, want):
    assert ctas(rows, at_once, batch, per_sm) == want


def test_few_sequences_of_many_rows_fill_the_sms(ctas):
    for batch in range(1, 40):
        for at_once, per_sm in ((2, 4), (1, 2), (4, 4)):
            got = ctas(1 << 20, at_once, batch, per_sm)
            assert batch * got >= per_sm * SMS and got >= 64
