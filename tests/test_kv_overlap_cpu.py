"""Which outputs lie on what a call reads: the rows' arithmetic against sets of bytes, and what the library refuses by it."""
import ctypes
import os
import random
import shutil
import subprocess

import pytest

import b4gemv
from b4gemv import _lib
from test_kv_lists_cpu import byref, cache, refused

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PROGRAM = r"""
#include <cstdio>
#include "b4_kv_overlap.h"
int main() {
    long long v[2][7];                     // address, item, token stride, head stride, tokens, heads, columns
    while (true) {
        for (auto& r : v)
            for (long long& x : r)
                if (std::scanf("%lld", &x) != 1) return 0;
        b4::RowSet s[2];
        for (int i = 0; i < 2; ++i) s[i] = b4::row_set(reinterpret_cast<const void*>(v[i][0]), v[i][1], v[i][2], v[i][3], v[i][4], v[i][5], v[i][6]);
        std::printf("%d %d %d\n", b4::rows_meet(s[0], s[1]), b4::rows_meet(s[1], s[0]), b4::rows_overlap(s[0]));
    }
}
"""


def rows(at, item, tok, head, n, heads, columns):
    """Each row's bytes."""
    return [range(a, a + columns * item) for t in range(n) for h in range(heads) for a in [at + (t * tok + h * head) * item]]


def draw(rng):
    def one(item, tok):
        n, heads, columns = rng.choice((1, 1, 2, 3, 5)), rng.choice((1, 2, 3, 4)), rng.choice((1, 2, 4))
        return [1000 + rng.randrange(-60, 60), item, tok, rng.choice((0, 1, columns, columns, 3 * columns, -columns, 5, 17, 40)), n, heads, columns]

    tok = rng.choice((0, 1, 4, 8, 16, 24, 30, -16, 12))
    a = one(2, tok)
    b = one(rng.choice((2, 2, 4, 1)), tok)
    if rng.random() < 0.8 and tok * a[1] % b[1] == 0:
        b[2] = tok * a[1] // b[1]                                  # one stride in bytes
    return a, b


@pytest.mark.skipif(shutil.which("g++") is None, reason="no g++")
def test_rows_against_sets_of_bytes(tmp_path):
    (tmp_path / "rows.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", f"-I{ROOT}/int4-gemv_b200/csrc", str(tmp_path / "rows.cpp"), "-o", str(tmp_path / "rows")], check=True)
    rng = random.Random(5)
    cases = [draw(rng) for _ in range(20000)]
    # as they are used: columns of fused rows, a head's three together, heads first, far apart, sizes past 32 bits
    d = 128
    cases += [([0x1000, 2, 36 * d, d, 3000, 28, d], [0x1000 + 2 * 28 * d, 2, 36 * d, d, 3000, 4, d]), ([0, 2, 24 * d, 3 * d, 9, 8, d], [2 * d, 2, 24 * d, 3 * d, 9, 8, d]),
              ([0, 2, d, 9 * d, 9, 8, d], [2 * 8 * 9 * d, 2, d, 9 * d, 9, 2, d])]
    known = [0, 0, 0]
    cases += [([0, 2, 1 << 36, d, 1 << 20, 4, d], [4 * d * 2, 2, 1 << 36, d, 1 << 20, 1, d]), ([0, 2, 1 << 36, d, 1 << 20, 4, d], [(1 << 37) + 2 * d, 2, 1 << 36, d, 1 << 20, 1, d])]
    known += [0, 1]
    text = "\n".join(" ".join(map(str, a + b)) for a, b in cases)
    got = [list(map(int, x.split())) for x in subprocess.run([str(tmp_path / "rows")], input=text, capture_output=True, text=True, check=True).stdout.splitlines()]
    assert len(got) == len(cases)
    told = met = 0
    for (a, b), (ab, ba, own) in zip(cases[:20000], got):
        x, y = rows(*a), rows(*b)
        mine = [i for r in x for i in r]
        meet = bool(set(mine) & {i for r in y for i in r})
        alike = a[4] == 1 or b[4] == 1 or a[1] * a[2] == b[1] * b[2]
        assert ab == ba and own == (len(set(mine)) < len(mine)), (a, b)
        if alike:
            assert ab == meet, (a, b)
            told += not meet
            met += meet
        else:
            assert ab or not meet, (a, b)                          # never let through
    assert told > 2000 and met > 2000
    assert [g[0] for g in got[20000:]] == known and not any(g[2] for g in got[20000:])


ROTARY = dict(turns=1 << 40, axes=None, dim=64, n_axes=1, flags=0, scale=1.0)
ROWS = dict(q=1 << 30, k=1 << 31, v=1 << 32, q_out=1 << 33, positions=1 << 34, slots=1 << 35, position_stride=8, q_stride_token=256, q_stride_head=64,
            k_stride_token=128, k_stride_head=64, v_stride_token=128, v_stride_head=64, out_stride_token=256, out_stride_head=64, n_tokens=8, heads=4, dtype=0,
            out_dtype=0)


@pytest.mark.parametrize("bad", [
    dict(q_out=1 << 31), dict(q_out=(1 << 31) + 8 * 256 - 16), dict(q_out=(1 << 32) - 8 * 512 + 16), dict(q_out=1 << 34), dict(q_out=(1 << 35) - 8 * 512 + 16),
    dict(q_out=1 << 40), dict(q_out=4096), dict(q_out=(1 << 30) + 128), dict(q_out=1 << 30, out_stride_head=128, out_stride_token=512), dict(out_stride_token=0),
    dict(out_stride_token=192), dict(out_stride_head=0), dict(out_stride_head=56), dict(q_out=1 << 30, dtype=2, out_dtype=0),
    dict(k=(1 << 30) + 3 * 128, k_stride_token=256, q_out=1 << 30), dict(v=(1 << 30) + 256, v_stride_token=264, q_out=1 << 30)])
def test_outputs_on_inputs_are_refused(bad):
    """Rotated queries on keys, values, other queries, positions, slots, angles, the cache, or on one another."""
    assert refused("b4_kv_append_rotary", byref(cache()), byref(_lib.RotaryTable(**ROTARY)), byref(_lib.KvRows(**{**ROWS, **bad})), None)


CHOICE = dict(q=1 << 30, boxes=1 << 31, tables=1 << 32, ctx_len=1 << 33, q_starts=1 << 34, lists=1 << 35, seen=1 << 36, table_stride=5, q_stride_token=512,
              q_stride_head=64, table_width=5, n_req=3, total_q=8, max_q=4, heads=4, dtype=0, keep=4, first=1, last=1)


@pytest.mark.parametrize("bad", [
    dict(lists=1 << 30), dict(lists=(1 << 30) + 7 * 1024 + 508), dict(lists=(1 << 30) - 252), dict(lists=1 << 31), dict(lists=(1 << 31) + 4 * 2 * 144 - 4),
    dict(seen=1 << 30), dict(seen=(1 << 30) + 1024), dict(seen=(1 << 30) + 512 - 4), dict(seen=(1 << 31) - 28), dict(seen=(1 << 31) + 4 * 2 * 144 - 4),
    dict(seen=1 << 35), dict(seen=(1 << 32) + 14 * 4), dict(lists=(1 << 34) + 12)])
def test_choices_on_what_is_read_are_refused(bad):
    """Lists and seen on queries or boxes too, which other CTAs read while they are written."""
    assert refused("b4_kv_select", byref(cache()), byref(_lib.KvChoice(**{**CHOICE, **bad})), None)


LISTS = dict(q=1 << 30, out=1 << 31, lse=1 << 32, tables=1 << 33, ctx_len=1 << 34, q_starts=None, table_stride=8, q_stride_token=256, q_stride_head=64,
             out_stride_token=256, out_stride_head=64, table_width=4, n_req=0, total_q=8, max_q=0, heads=4, dtype=0, window=0, flags=0, scale=0.125)


@pytest.mark.parametrize("bad", [
    dict(out=1 << 33), dict(out=(1 << 33) + 7 * 32 + 16), dict(out=(1 << 33) - 8 * 512 + 16), dict(out=1 << 34), dict(out=(1 << 34) - 8 * 512 + 16), dict(out=4096),
    dict(out=(1 << 30) + 128), dict(out=1 << 30, out_stride_token=512), dict(out=(1 << 32) - 16), dict(lse=(1 << 31) + 512), dict(lse=1 << 33), dict(lse=(1 << 34) - 124),
    dict(lse=1 << 30), dict(lse=(1 << 30) + 8 * 512 - 4), dict(lse=4096), dict(out_stride_token=0), dict(out_stride_head=0), dict(out_stride_head=56)])
def test_attention_on_what_is_read_is_refused(bad):
    """Outputs on lists, seen, the cache, queries that are not the row's own, or on one another."""
    assert refused("b4_kv_attention_lists", byref(cache()), byref(_lib.KvAttn(**{**LISTS, **bad})), 4, 1 << 44, 1 << 40, None)
