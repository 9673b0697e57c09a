"""The rows of a sequence from the device's offsets (eddl_amd/csrc/sequence_rows.h), compiled for the host."""
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "eddl_amd", "csrc")
LOW, HIGH = -2 ** 31, 2 ** 31 - 1


@pytest.fixture(scope="module")
def rows_of(tmp_path_factory):
    folder = tmp_path_factory.mktemp("rows")
    source, program = str(folder / "rows.cpp"), str(folder / "rows")
    with open(source, "w") as fh:
        fh.write('#include <cstdio>\n#include "sequence_rows.h"\nint main() { int b, e, r; while (std::scanf("%d %d %d", &b, &e, &r) == 3) {\n'
                 'const eddlhip::SequenceRows s = eddlhip::sequence_rows(b, e, r); std::printf("%d %d\\n", s.row0, s.fresh); } }\n')
    subprocess.run(["g++", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-I", CSRC, source, "-o", program], check=True)

    def run(cases):
        text = subprocess.run([program], input="\n".join("%d %d %d" % c for c in cases), capture_output=True, text=True, check=True).stdout
        return [tuple(map(int, line.split())) for line in text.splitlines()]
    return run


def test_rows_stay_within_the_buffers_whatever_the_offsets_hold(rows_of):
    ends = [LOW, LOW + 1, LOW + 4, -7, -1, 0, 1, 4, 5, 6, 9, 10, 11, 1 << 20, HIGH - 5, HIGH]
    cases = [(b, e, r) for b in ends for e in ends for r in (0, 1, 9, 10, 1 << 30, HIGH)]
    for (b, e, r), (row0, fresh) in zip(cases, rows_of(cases)):
        assert 0 <= row0 and 0 <= fresh and row0 + fresh <= r, (b, e, r, row0, fresh)
        wanted = [i for i in range(max(b, 0), min(e, r, 12))]  # (those below 12, one by one)
        assert [i for i in range(row0, min(row0 + fresh, 12))] == wanted, (b, e, r, row0, fresh)
        assert fresh == max(0, min(e, r) - max(b, 0)), (b, e, r, row0, fresh)


def test_kernels_take_their_rows_from_there():
    """No kernel bounds and subtracts two offsets by itself."""
    for name in ("attention.hip", "rotary.hip"):
        with open(os.path.join(CSRC, name)) as fh:
            text = fh.read()
        assert "sequence_rows(" in text and "min(p.offsets" not in text
