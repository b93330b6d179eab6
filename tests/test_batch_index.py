"""The arithmetic by which a served batch's entries choose and place their work (phonon-2-c_amd/csrc/p2hip_index.h), compiled for
the host."""
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "phonon-2-c_amd", "csrc")


def run(tmp_path, program):
    src, exe = tmp_path / "index.cpp", tmp_path / "index"
    src.write_text(program)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
                    "-I", CSRC, "-o", str(exe), str(src)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr


FAR_ROWS = r"""
#include <climits>
#include <cstdio>
#include <initializer_list>
#include "p2hip_index.h"
#define CHECK(c) do { if (!(c)) { printf("line %d: %s\n", __LINE__, #c); return 1; } } while (0)

int main()
{
    for (int es : {2, 4})
        for (int pitch : {64, 4096, (1 << 26) - 8, 1 << 26, (1 << 26) + 8, 72000000, (1 << 27) - 8, 1 << 27, 1 << 28, 300000000,
                          1 << 29, 1 << 30, INT_MAX - 7, INT_MAX}) {
            const bool in = p2k::sixteen_rows_in_32_bits(pitch, es);
            const unsigned __int128 end = (unsigned __int128)16 * pitch * es;   /* behind the last element of the widest row */
            CHECK(in == (end <= ((unsigned __int128)1 << 32) - 16));
            if (in) CHECK((uint32_t)(15 * pitch + pitch - 1) * (uint32_t)es < 0xfffffff0u);   /* as the stores have it, an int first */
        }
    puts("ok");
    return 0;
}
"""


def test_rows_far_apart(tmp_path):
    """Pitches at which sixteen rows pass 32-bit offsets, and those at which their size passes 32 bits as a number."""
    run(tmp_path, FAR_ROWS)
