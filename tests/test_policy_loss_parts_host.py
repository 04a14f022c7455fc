"""How the CTAs of a cluster share a long row of policy_loss, and what each
copies of its next row, replayed on the CPU from the kernel's own header: for
any number of clusters that a device may hold at once."""

import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest

HEADER = (Path(__file__).resolve().parent.parent / "alpha-yoo-for-great-kingdom_b200" / "csrc" / "gk_row_part.cuh")

REPLAY = r"""
#include "%s"
#include <algorithm>
#include <vector>

// What one CTA reads of its rows r, r + clusters, ... : -1 if a part does not fit `slots`, else how often it
// reads a slot that does not hold the row's own group. `past` 1: a rule that copies one slot past the part.
template <int V>
static long walk(long rows, long stride, int cols, int rank, int log_ranks, int clusters, long first, int slots, int past) {
    constexpr int kThreads = 256;
    std::vector<long> holds(slots, -1);  // row whose group lies in the slot
    long wrong = 0;
    gk::RowPart<V> part(first, stride, cols, rank, log_ranks);
    for (int k = 0; k < part.full_end - part.full; ++k) holds.at(k) = first;
    for (long r = first; r < rows; r += clusters) {
        const int count = part.full_end - part.full;
        if (count > slots) return -1;
        for (int k = 0; k < count; ++k) wrong += holds[k] != r;
        const long next_r = r + clusters;
        if (next_r >= rows) break;
        const gk::RowPart<V> next(next_r, stride, cols, rank, log_ranks);
        const int next_count = next.full_end - next.full;
        if (next_count > slots) return -1;
        for (int k = 0; k < std::min(count, next_count); ++k) holds[k] = next_r;
        if (past) {
            if (count < next_count && count >= 0) holds[count] = next_r;
        } else {
            std::vector<int> owner(slots, -1);
            bool one_each = true;
            for (int tid = 0; tid < kThreads; ++tid)
                gk::fill_past<kThreads>(tid, count, next_count, [&](int k) {
                    one_each = one_each && k >= count && k %% kThreads == tid && owner.at(k) < 0;
                    owner[k] = tid;
                    holds[k] = next_r;
                });
            wrong += !one_each;
        }
        part = next;
    }
    return wrong;
}

// The groups of all parts are the row's, each once and in order.
template <int V>
static bool covers(long r, long stride, int cols, int log_ranks) {
    int at = 0;
    gk::RowPart<V> last(r, stride, cols, 0, log_ranks);
    for (int rank = 0; rank < 1 << log_ranks; ++rank) {
        const gk::RowPart<V> p(r, stride, cols, rank, log_ranks);
        if (p.begin != at || p.end < p.begin || p.shift != last.shift) return false;
        // Whole groups lie in the row, and what is left is at most one group at the row's start and one at its end.
        if (p.full < p.begin || p.full_end > p.end || p.full - p.begin > (rank == 0)) return false;
        if (p.full < p.full_end && ((long)p.full * V - p.shift < 0 || (long)p.full_end * V - p.shift > cols)) return false;
        if (p.full <= p.full_end && p.end - p.full_end > 1) return false;
        at = p.end;
    }
    return (long)at * V - last.shift >= cols && ((long)at - 1) * V - last.shift < cols;
}

extern "C" long replay(long rows, long stride, int cols, int v, int log_ranks, int clusters, int slots, int past) {
    long wrong = 0;
    for (long first = 0; first < std::min<long>(clusters, rows); ++first)
        for (int rank = 0; rank < 1 << log_ranks; ++rank) {
            const long w = v == 8 ? walk<8>(rows, stride, cols, rank, log_ranks, clusters, first, slots, past)
                                  : walk<4>(rows, stride, cols, rank, log_ranks, clusters, first, slots, past);
            if (w < 0) return -1;
            wrong += w;
        }
    return wrong;
}
extern "C" int whole(long stride, int cols, int v, int log_ranks) {
    for (long r = 0; r < 8; ++r)
        if (!(v == 8 ? covers<8>(r, stride, cols, log_ranks) : covers<4>(r, stride, cols, log_ranks))) return 0;
    return 1;
}
"""


@pytest.fixture(scope="module")
def parts(tmp_path_factory):
    compiler = shutil.which("g++")
    if compiler is None:
        pytest.skip("no C++ compiler")
    folder = tmp_path_factory.mktemp("parts")
    source, library = folder / "replay.cpp", folder / "replay.so"
    source.write_text(REPLAY % HEADER)
    subprocess.run([compiler, "-std=c++17", "-O1", "-shared", "-fPIC", str(source), "-o", str(library)], check=True)
    lib = ctypes.CDLL(str(library))
    lib.replay.restype = ctypes.c_long
    lib.replay.argtypes = [ctypes.c_long, ctypes.c_long] + [ctypes.c_int] * 6
    lib.whole.restype = ctypes.c_int
    lib.whole.argtypes = [ctypes.c_long] + [ctypes.c_int] * 3
    return lib


def slots(cols, v, log_ranks):
    """What the launch makes room for: a share of the row with the largest shift."""
    groups = (cols + 2 * (v - 1)) // v
    return -(-groups // (1 << log_ranks))


@pytest.mark.parametrize("v", [4, 8])
@pytest.mark.parametrize("log_ranks", [0, 1, 2, 3])
def test_every_group_is_copied_before_it_is_read(parts, v, log_ranks):
    # 64 lengths in a row hold every remainder by the entries of a group and the CTAs of a cluster.
    for cols in (*range(2049, 2049 + 64), 6007, 9999):
        assert parts.whole(cols, cols, v, log_ranks), cols
        for clusters in (1, 2, 3, 4, 5, 7, 8):
            for stride in (cols, cols + 3):
                assert parts.replay(3 * clusters + 9, stride, cols, v, log_ranks, clusters, slots(cols, v, log_ranks),
                                    0) == 0, (cols, clusters, stride)


@pytest.mark.parametrize("rows,cols,v,log_ranks", [(512, 131071, 8, 2), (300, 131071, 8, 2), (1024, 128255, 8, 2),
                                                   (512, 65535, 4, 2), (600, 50255, 4, 2)])
def test_a_rule_of_one_slot_past_the_part_is_noticed(parts, rows, cols, v, log_ranks):
    room = slots(cols, v, log_ranks)
    assert parts.replay(rows, cols, cols, v, log_ranks, 111, room, 1) > 0
    assert parts.replay(rows, cols, cols, v, log_ranks, 111, room, 0) == 0


def test_short_rows_and_empty_parts(parts):
    for v in (4, 8):
        for cols in range(257, 257 + 40):
            for log_ranks in range(4):
                assert parts.whole(cols, cols, v, log_ranks)
                assert parts.replay(40, cols, cols, v, log_ranks, 3, slots(cols, v, log_ranks), 0) == 0
