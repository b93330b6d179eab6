"""The index arithmetic of the attention kernels (phonon-2-c_amd/csrc/p2hip_index.h), compiled for the host and gone over by
brute force: which key blocks are taken, how they are split, and that no page table is read outside its row."""
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "phonon-2-c_amd", "csrc")

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <vector>
#include <climits>
#include "p2hip_index.h"
using namespace p2k;
#define CHECK(c) do { if (!(c)) { printf("line %d: %s\n", __LINE__, #c); return 1; } } while (0)

int main()
{
    /* every block with a visible key comes once, no other does, and the splits hand each out once */
    const int sinks[] = {0, 1, 3, 16, 17, 40, 200, 1 << 30}, bss[] = {16, 32, 64};
    for (int bs : bss)
        for (int hi = 0; hi <= 150; hi++)
            for (int lo = -3; lo <= hi; lo++)
                for (int sk : sinks) {
                    const KeyBlocks k = key_blocks(lo, hi, sk, bs);
                    std::vector<int> want, got;
                    for (int b = 0; b * bs < hi; b++) {
                        bool any = false;
                        for (int j = b * bs; j < (b + 1) * bs && j < hi; j++) any |= j >= lo || j < sk;
                        if (any) want.push_back(b);
                    }
                    for (int i = 0; i < k.total; i++) got.push_back(k.at(i));
                    CHECK(got == want);
                    for (int splits : {1, 2, 3, 7, 256}) {
                        int next = 0;
                        for (int s = 0; s < splits; s++) {
                            int a, b;
                            split_range(k.total, splits, s, &a, &b);
                            CHECK(a == next || (a == k.total && b == a));
                            CHECK(a <= b && b <= k.total);
                            if (b > a) next = b;
                        }
                        CHECK(next == k.total);
                    }
                }
    /* the largest places and windows do not overflow */
    const int big = (1 << 30) - 1;
    CHECK(key_blocks(big - (1 << 30) + 1, big, 0, 64).total == (big - 1) / 64 + 1);
    CHECK(key_blocks(-(1 << 30) - (1 << 30) + 1, 5, 1 << 30, 32).total == 1);
    CHECK(key_visible(0, big - 1, 1 << 30, 0, 0) && !key_visible(big - 1, -big, 1 << 30, 1 << 30, 1 << 30));
    CHECK(!key_visible(5, 4, 3, 0, 100) && key_visible(5, 4, 3, 1, 0) && !key_visible(1, 4, 3, 0, 0) && key_visible(1, 4, 3, 0, 2));

    /* pages: the row lies between guards that must not be read (they would give a page inside the cache) */
    const int ld = 5, pages = 9;
    int32_t mem[ld + 2] = {3, 0, 8, -1, 9, INT_MIN, 3};
    const int32_t *row = mem + 1;
    const int want[ld] = {0, 8, -1, -1, -1};
    for (int shift = 4; shift <= 10; shift++)
        for (long long t = -20; t < (8ll << shift); t++) {
            const int p = page_in(page_entry(row, ld, (int)t, shift), pages);
            CHECK(p == (t >= 0 && (t >> shift) < ld ? want[t >> shift] : -1));
        }
    CHECK(page_entry(row, 0, 0, 4) == -1 && page_entry(row, ld, INT_MAX, 4) == -1 && page_in(0, 0) == -1 && page_in(-1, 0) == -1);
    CHECK(kept_length(-1, 5, 16) == 0 && kept_length(81, 5, 16) == 80 && kept_length(80, 5, 16) == 80);
    CHECK(kept_length(INT_MAX, 1 << 20, 1024) == 1 << 30 && kept_length(7, 0, 16) == 0);

    /* rows of a sequence stay inside the rows, whatever the starts */
    const int32_t st[] = {-4, 3, 2, INT_MAX, INT_MIN, 50, 12};
    for (int s = 0; s < 6; s++)
        for (int rows : {0, 1, 10, 40}) {
            int a, b;
            seq_rows(st, s, rows, &a, &b);
            CHECK(a >= 0 && a <= b && b <= rows);
        }
    /* every tile of every sequence has one number below rows / bs + n, whatever sequences are empty */
    srand(3);
    for (int it = 0; it < 3000; it++) {
        const int n = 1 + rand() % 9, bs = 16 << (rand() % 4);
        std::vector<int32_t> st(n + 1);
        st[0] = rand() % 40;
        for (int s = 0; s < n; s++) st[s + 1] = st[s] + (rand() % 3 ? rand() % (3 * bs) : 0);
        const int rows = st[n] + rand() % 40;
        for (int s = 0; s < n; s++) {
            const int first = tile_start(st.data(), s, rows, bs), next = tile_start(st.data(), s + 1, rows, bs);
            CHECK(first >= 0 && first < next);
            CHECK(first + (st[s + 1] - st[s] + bs - 1) / bs <= next);
            CHECK(first + (st[s + 1] - st[s] + bs - 1) / bs <= rows / bs + n);
        }
    }
    int a, b;
    seq_rows(nullptr, 0, 12, &a, &b);
    CHECK(a == 0 && b == 12);
    puts("ok");
    return 0;
}
"""


def test_index_arithmetic(tmp_path):
    src, exe = tmp_path / "index.cpp", tmp_path / "index"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
                    "-I", CSRC, "-o", str(exe), str(src)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr


RULE = r"""
#include <cstdio>
#include <climits>
#include "p2hip_index.h"
using namespace p2k;
#define CHECK(c) do { if (!(c)) { printf("line %d: %s\n", __LINE__, #c); return 1; } } while (0)

int main()
{
    const int all = 1 << 30;
    auto f16 = [&](int dh, int q, int k, int n, int heads) { return few_queries(false, dh, q, k, n, heads, all, 0, 256); };
    auto f32 = [&](int q, int k, int n, int heads, int w) { return few_queries(true, 128, q, k, n, heads, w, 0, 256); };
    /* one sequence */
    CHECK(f16(128, 375, 375, 1, 8) && f16(128, 750, 750, 1, 8) && !f16(128, 1500, 1500, 1, 8) && !f16(128, 6000, 6000, 1, 32));
    CHECK(f16(64, 2000, 2000, 1, 8) && !f16(64, 4000, 4000, 1, 8) && !f16(64, 1100, 900, 1, 8));
    CHECK(f16(128, 16, 8000, 1, 64) && f16(128, 1, 8000, 1, 256));
    CHECK(f32(438, 438, 1, 8, 128) && f32(4000, 4000, 1, 8, all) && !f32(2000, 2000, 1, 32, all) && !f32(3000, 3000, 1, 8, 256));
    /* many sequences of few queries are many workgroups whatever their rows come to */
    CHECK(!f16(128, 64, 64000, 64, 32) && !f16(64, 256, 256000, 256, 32) && !f16(64, 64 * 8, 64 * 4000, 64, 32));
    CHECK(f16(128, 16, 16000, 16, 8) && f16(64, 16 * 8, 16 * 1000, 16, 32) && !f16(64, 16 * 8, 16 * 100, 16, 32));
    /* a tile of fp32 rows multiplies 128 of them whatever it holds */
    CHECK(f32(256 * 8, 256 * 100, 256, 32, all) && f32(256 * 16, 256 * 100, 256, 32, all) && !f32(256 * 17, 256 * 100, 256, 32, all));
    /* rows of a linear: a single one has no pitch */
    CHECK(rows_by_16(32, 1019, 2, 1) && rows_by_16(32, INT_MAX, 4, 1) && !rows_by_16(34, 1024, 2, 1) && !rows_by_16(40, 8, 2, 1));
    CHECK(rows_by_16(32, 1024, 2, 2) && !rows_by_16(32, 1020, 2, 2) && rows_by_16(32, 1020, 4, 13) && !rows_by_16(32, 1 << 25, 2, 2));
    /* empty sequences, no keys and the largest numbers */
    CHECK(f16(128, 1, 0, 100000, 8) && few_queries(true, 64, 1, 1, INT_MAX, 1, all, all, 256));
    CHECK(!few_queries(false, 64, all - 1, all - 1, 1, 65536, all, all, 256) && !few_queries(true, 128, all - 1, all - 1, 7, 65536, 1, 0, 256));
    puts("ok");
    return 0;
}
"""


def test_rule_for_few_queries(tmp_path):
    src, exe = tmp_path / "rule.cpp", tmp_path / "rule"
    src.write_text(RULE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
                    "-I", CSRC, "-o", str(exe), str(src)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr


SPANS = r"""
#include <cstdio>
#include <initializer_list>
#include "p2hip_index.h"
using namespace p2k;
#define CHECK(c) do { if (!(c)) { printf("line %d: %s\n", __LINE__, #c); return 1; } } while (0)

int main()
{
    const int all = 1 << 30, big = all - 1;
    /* places from the first query of 2^30 - 1 without a key to the last key of 2^30 - 1, at every end of the limits */
    const int ps[] = {-big, -big + 1, -130, -1, 0, 1, 77, big - 130, big - 2, big - 1}, ks[] = {0, 28, 64, 4096, big - 130, big - 63, big + 3};
    for (int Lk : {1, 200, big})
        for (int window : {1, 64, big, all})
            for (int ahead : {0, 5, big, all})
                for (int sinks : {0, 7, all})
                    for (int p : ps) {
                        if (p >= Lk) continue;
                        for (int k0 : ks) {
                            if (k0 > (long long)p + 127 + ahead) continue;   /* no query of the tile sees the block */
                            const KeySpan s = key_span(k0, p, Lk, window, ahead, sinks);
                            for (int e = 0; e < 64 && k0 + e < Lk; e++)
                                CHECK(key_visible(k0 + e, p, window, ahead, sinks) == (e <= s.last && (e >= s.first || e < s.sink)));
                            CHECK(k0 < Lk || s.last < 0);
                        }
                        for (int more : {0, 32, 96}) {
                            const int to = last_seen_by_all(p + more, Lk, ahead);
                            CHECK(to < Lk);
                            if (p + more < Lk && to >= 0) CHECK((long long)to - (p + more) <= ahead && (to == Lk - 1 || (long long)to + 1 - (p + more) > ahead));
                        }
                    }
    puts("ok");
    return 0;
}
"""


def test_key_spans(tmp_path):
    src, exe = tmp_path / "spans.cpp", tmp_path / "spans"
    src.write_text(SPANS)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
                    "-I", CSRC, "-o", str(exe), str(src)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr
