// gk_row_part.cuh - how a cluster of CTAs shares a row, and how a CTA's part of
// one row gives way to its part of the next. Plain C++ too, so that the
// bookkeeping can be replayed without a GPU.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define GK_ROW_INLINE __host__ __device__ __forceinline__
#else
#define GK_ROW_INLINE inline
#endif

namespace gk {

// Groups of V entries that start on 16-byte boundaries of the rows' storage.
// Groups [full, full_end) lie in the row; a group before or after them is the
// row's ragged edge. A part without whole groups may have full_end < full.
template <int V>
struct RowPart {
    int shift, begin, end, full, full_end;
    GK_ROW_INLINE RowPart(int64_t r, int64_t stride, int cols, int rank, int log_ranks) {
        shift = (int)((uint32_t)r * (uint32_t)stride % V);
        const int groups = (cols + shift + V - 1) / V, each = (groups + (1 << log_ranks) - 1) >> log_ranks;
        begin = least(groups, rank * each);
        end = least(groups, begin + each);
        full = begin > 0 || shift == 0 ? begin : 1;
        full_end = least(end, (cols + shift) / V);
    }

private:
    GK_ROW_INLINE static int least(int a, int b) { return a < b ? a : b; }
};

// Group k of a part has slot k of shared memory, thread k % THREADS reads it,
// and the same thread copies the next row's group there after this row's last
// read: for k < min(count, next_count) as it goes, and past this row's part
// here. There may be several such slots: where the next row's shift saves it a
// group, every part but the last can be one group shorter, so that the last
// begins earlier and is up to a group a CTA longer.
template <int THREADS, typename F>
GK_ROW_INLINE void fill_past(int tid, int count, int next_count, F&& copy) {
    int k = tid;
    if (count > tid) k += (count - tid + THREADS - 1) / THREADS * THREADS;
    for (; k < next_count; k += THREADS) copy(k);
}

}  // namespace gk
