"""How the adapters' kernel cuts a row into parts (adapter_parts.hh), compiled for the host: 32 parts at most, whole segments of 128 entries
but for the last, one behind the other up to the row's end, for rows of up to 2^31 - 1 entries."""
import os
import shutil
import subprocess

import pytest

from conftest import ROOT

PROGRAM = r"""
#include "adapter_parts.hh"
#include <cstdio>
#include <cstdlib>
using namespace cb200;
int main(int, char **of) {
    const unsigned len = (unsigned)std::strtoul(of[1], nullptr, 10);
    const auto share = part_entries(len);
    const auto parts = parts_of(len, share);
    unsigned long long at = 0; // no overflow here
    bool right = share >= 128u && share % 128u == 0u && parts <= 32u && (len == 0u) == (parts == 0u);
    for (unsigned part = 0; part < parts; ++part) {
        const auto begin = (decltype(share))part * share, end = part_end(begin, len, share);
        right = right && begin == at && end > begin && end <= len && (end - begin == share || part + 1 == parts);
        // the walk along a part, a segment at a time
        auto place = begin;
        place += (end - begin - 1u) / 128u * 128u;
        right = right && place < end && end - place <= 128u && place + 128u >= end;
        at = end;
    }
    return right && at == len ? 0 : 1;
}
"""

LENGTHS = [0, 1, 127, 128, 129, 4095, 4096, 4097, 33_538, 2 ** 20 + 3, 2 ** 30, 2_080_374_783, 2_080_374_784, 2_080_374_785, 2 ** 31 - 2 ** 26, 2 ** 31 - 129,
           2 ** 31 - 128, 2 ** 31 - 127, 2 ** 31 - 33, 2 ** 31 - 32, 2 ** 31 - 31, 2 ** 31 - 1]


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no host compiler")
    at = tmp_path_factory.mktemp("parts")
    (at / "parts.cc").write_text(PROGRAM)
    subprocess.run([cxx, "-O1", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-I", os.path.join(ROOT, "cellerator_b200", "csrc"),
                    "-o", str(at / "parts"), str(at / "parts.cc")], check=True)
    return str(at / "parts")


@pytest.mark.parametrize("length", LENGTHS)
def test_parts_cover_a_row(program, length):
    done = subprocess.run([program, str(length)], capture_output=True, text=True, timeout=60)
    assert done.returncode == 0, done.stderr
