"""How many parts decode's join reads of a head that reaches over an SM (r-mda_b200/csrc/moe_attn_args.h, plain C), whatever a
piece that gave up has left for it: checked without a GPU, by the arithmetic that the kernels use."""
import ctypes as C
import os
import random
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "r-mda_b200", "csrc")


@pytest.fixture(scope="module")
def parts(tmp_path_factory):
    d = tmp_path_factory.mktemp("join")
    (d / "join.c").write_text('#include "%s/moe_attn_args.h"\n' % CSRC + "unsigned parts(unsigned first, unsigned n, unsigned sms) { return moe_join_parts(first, n, sms); }\n")
    r = subprocess.run(["gcc", "-std=gnu17", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC", "-o", str(d / "join.so"), str(d / "join.c")],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    f = C.CDLL(str(d / "join.so")).parts
    f.restype, f.argtypes = C.c_uint32, [C.c_uint32] * 3
    return f


def test_parts_stay_in_the_work_area(parts):
    """Any count, also one made of an unwritten number of stages, below zero or past the last SM, reads nothing."""
    rng = random.Random(1)
    for sms in (1, 2, 132, 148):
        for first in range(sms):
            for n in range(sms + 2):
                assert parts(first, n, sms) == (n if first + n <= sms else 0)
            for n in [2 ** 32 - 1, 2 ** 32 - first, 2 ** 31] + [rng.randrange(2 ** 32) for _ in range(20)]:
                assert first + parts(first, n, sms) <= sms
        assert parts(sms, 1, sms) == 0 and parts(2 ** 32 - 1, 1, sms) == 0


def test_parts_of_garbage(parts):
    """The count as the decode kernel makes it, of a number of stages behind the piece that was never written."""
    rng = random.Random(2)
    for _ in range(2000):
        sms, total = 148, rng.randrange(148, 1 << 30)
        sm = rng.randrange(sms)
        behind = rng.randrange(2 ** 32)
        x = (total * (sm + 1) // sms + behind - 1) % 2 ** 64
        count = ((((x + 1) * sms - 1) % 2 ** 64) // total - sm + 1) % 2 ** 32
        assert sm + parts(sm, count, sms) <= sms


def test_the_join_asks(parts):
    """The join kernel takes its count from this function and nowhere else, and a piece that gave up tells of no head."""
    text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, "moe_decode.cu")).read())
    join = text[text.index("moe_attn_join_kernel(DecArgs a)"):text.index("void decode_launch")]
    assert "n = moe_join_parts(first, split.w, gridDim.x / a.group)" in join and join.count("split.w") == 1
    assert re.search(r"if \(left != 0\) \{\s*gave_up = true;", text) and text.count("over = make_uint4(key.x") == 1
    assert "if (here && !ends && !gave_up && threadIdx.x == 0) over = make_uint4(key.x" in text


@pytest.mark.parametrize("out,first,rows,row,ok", [(16, 4, 5, 32, True), (16, 4, 5, 24, False), (8, 4, 5, 32, False), (None, 4, 5, 32, False), (16, None, 5, 32, False),
                                                    (16, 2, 5, 32, False), (None, None, 0, 32, True), (None, None, 5, 0, True)])
def test_clear_refusals(tmp_path, out, first, rows, row, ok):
    (tmp_path / "c.c").write_text('#include "%s/moe_attn_args.h"\n' % CSRC
                                  + "const char *f(const void *o, const void *a, unsigned r, unsigned b) { return moe_clear_refusal(o, a, r, b); }\n")
    so = tmp_path / "c.so"
    r = subprocess.run(["gcc", "-std=gnu17", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC", "-o", str(so), str(tmp_path / "c.c")], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    f = C.CDLL(str(so)).f
    f.restype, f.argtypes = C.c_char_p, [C.c_void_p, C.c_void_p, C.c_uint32, C.c_uint32]
    assert (f(out, first, rows, row) is None) == ok
