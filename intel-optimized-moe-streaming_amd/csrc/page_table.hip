// page_table.hip -- page tables and slots of a batch, on the device: new tokens of
// every sequence are given rows, positions and slots, pages come from a stack of
// free ones and go back to it.
//
// With n_b new tokens of sequence b, L_b held before and pages of S tokens:
//   starts_b = sum of n before b;  row t of b: position L_b + t - starts_b
//   slot     = page(position / S) * S + position % S
// and the pages b lacks, ceil((L_b + n_b) / S) - ceil(L_b / S), are popped from the
// stack in the order of sequences and columns: page j of the call is
// free[count - 1 - j].  So a row's page needs no table: it is an old column's, or
// follows from the prefix sum of the pages before.  Taking tokens back pushes the
// pages in the opposite order: what the last call took lies where it was.
//
// One launch.  What bounds it is latency: every workgroup sums all sequences anew
// (in LDS; a few thousand words from the last-level cache) and then works on rows
// and pages of its own, none waits for another.  Only lengths and the stack's count
// change in place: the workgroup that counts last, when all others have read them,
// writes them.
//
// 64 sequences that get one token each: 4.4 us, and 3.3 to take them back (an empty kernel
// is 2); 24 prompts of 65,000 tokens in all in pages of 16: 7.1 and 6.2.
//
// A call whose arguments are out of range, or for which the pages do not suffice,
// changes nothing and gives no rows.  The numbers of the pages themselves are met only
// where they are handed on: one that is none is reported there, and its rows get the slot
// past a cache of p.pages.

#include "mixers.h"

namespace mqh {

constexpr int PAGE_THREADS = 256, PAGE_ROWS = 4;   // rows of a thread

struct PageScan {
    int* start;        // [seqs + 1] extend: rows before the sequence
    int* first;        // [seqs + 1] pages before the sequence (that are taken or given back)
    int* held;         // [seqs] tokens it holds
    int64_t rows;      // sums
    int64_t moved;
    int count;         // free pages before the call
    bool ok;
};

__device__ __forceinline__ int pages_of(int tokens, int shift) { return (tokens + (1 << shift) - 1) >> shift; }

// the sequence whose share of `before` holds `at` (before[0] = 0 <= at < before[seqs])
__device__ __forceinline__ int owner(const int* before, int seqs, int at) {
    int lo = 0, hi = seqs;   // before[lo] <= at < before[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (before[mid] <= at) lo = mid;
        else hi = mid;
    }
    return lo;
}

template <bool EXTEND>
__device__ PageScan page_scan(const PageParams& p, int* lds) {
    __shared__ int64_t s_rows[PAGE_THREADS / 64], s_moved[PAGE_THREADS / 64];
    __shared__ int s_bad, s_count;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    PageScan s;
    s.start = lds;
    s.first = lds + p.seqs + 1;
    s.held = s.first + p.seqs + 1;
    s.rows = s.moved = 0;
    if (tid == 0) {   // (by one thread, that has it before the workgroup counts itself)
        s_count = *p.count;
        s_bad = s_count < 0 || s_count > p.pages;
    }
    __syncthreads();
    s.count = s_count;
    const int most = p.cols << p.page_shift;
    bool bad = false;
    for (int i = tid; i < p.seqs; i += PAGE_THREADS) {
        int n = p.change[i], held = p.lengths[i];
        bad |= n < 0 || held < 0 || held > most || (EXTEND && n > most - held);
        s.start[i] = n;
        s.held[i] = held;
    }
    if (bad) s_bad = 1;
    __syncthreads();
    s.ok = !s_bad;
    if (!s.ok) return s;
    // each thread a run of sequences
    const int per = (p.seqs + PAGE_THREADS - 1) / PAGE_THREADS, i0 = min(tid * per, p.seqs), i1 = min(i0 + per, p.seqs);
    int64_t rows = 0, moved = 0;
    for (int i = i0; i < i1; ++i) {
        const int n = s.start[i], held = s.held[i];
        const int pages = EXTEND ? pages_of(held + n, p.page_shift) - pages_of(held, p.page_shift)
                                 : pages_of(held, p.page_shift) - pages_of(min(held, n), p.page_shift);
        s.first[i] = pages;
        rows += n;
        moved += pages;
    }
    int64_t r = rows, m = moved;   // inclusive sums over the wave
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int64_t a = __shfl_up(r, d), b = __shfl_up(m, d);
        if (lane >= d) {
            r += a;
            m += b;
        }
    }
    if (lane == 63) {
        s_rows[wave] = r;
        s_moved[wave] = m;
    }
    __syncthreads();
    r -= rows;
    m -= moved;
#pragma unroll
    for (int w = 0; w < PAGE_THREADS / 64; ++w) {
        if (w < wave) {
            r += s_rows[w];
            m += s_moved[w];
        }
        s.rows += s_rows[w];
        s.moved += s_moved[w];
    }
    // (sums past 32 bits are refused by the caller before these are used)
    for (int i = i0; i < i1; ++i) {
        const int n = s.start[i], pages = s.first[i];
        s.start[i] = (int)r;
        s.first[i] = (int)m;
        r += n;
        m += pages;
    }
    if (tid == 0) {
        s.start[p.seqs] = (int)s.rows;
        s.first[p.seqs] = (int)s.moved;
    }
    __syncthreads();
    return s;
}

// whether this workgroup counts last (all others have read what the scan reads)
__device__ bool counts_last(const PageParams& p) {
    __shared__ int s_last;
    if (gridDim.x == 1) return true;
    if (threadIdx.x == 0) s_last = atomicAdd(&p.flags[FLAG_TICKET], 1) == (int)gridDim.x - 1;
    __syncthreads();
    if (s_last && threadIdx.x == 0) atomicExch(&p.flags[FLAG_TICKET], 0);
    return s_last;
}

__global__ __launch_bounds__(PAGE_THREADS) void k_pages_extend(PageParams p) {
    extern __shared__ int lds[];
    PageScan s = page_scan<true>(p, lds);
    const int tid = threadIdx.x, size = 1 << p.page_shift;
    const bool last = counts_last(p);
    const bool rows_ok = s.ok && s.rows <= p.rows, pages_ok = s.ok && s.moved <= s.count, ok = rows_ok && pages_ok;
    if (blockIdx.x == 0 && tid == 0 && !ok) atomicOr(&p.flags[rows_ok ? FLAG_NO_PAGES : FLAG_BAD_ID], 1);
    if (blockIdx.x == 0)
        for (int i = tid; i <= p.seqs; i += PAGE_THREADS) p.starts[i] = ok ? s.start[i] : 0;
    if (last && ok) {
        for (int i = tid; i < p.seqs; i += PAGE_THREADS) p.lengths[i] = s.held[i] + s.start[i + 1] - s.start[i];
        if (tid == 0) *p.count = s.count - (int)s.moved;
    }
    // ---- the table's new columns
    bool bad = false;
    if (ok) {
        for (int j = blockIdx.x * PAGE_THREADS + tid; j < (int)s.moved; j += gridDim.x * PAGE_THREADS) {
            const int b = owner(s.first, p.seqs, j);
            const int page = p.free_pages[s.count - 1 - j];
            bad |= (unsigned)page >= (unsigned)p.pages;
            p.table[(int64_t)b * p.cols + pages_of(s.held[b], p.page_shift) + j - s.first[b]] = page;
        }
    }
    // ---- the rows
    const int total = ok ? (int)s.rows : 0;
    const int row0 = (blockIdx.x * PAGE_THREADS + tid) * PAGE_ROWS;
    int b = row0 < total ? owner(s.start, p.seqs, row0) : p.seqs;
    for (int i = 0; i < PAGE_ROWS; ++i) {
        const int row = row0 + i;
        if (row >= p.rows) break;
        int position = -1;
        int64_t slot = -1;
        if (row < total) {
            while (s.start[b + 1] <= row) ++b;
            position = s.held[b] + row - s.start[b];
            const int col = position >> p.page_shift, had = pages_of(s.held[b], p.page_shift);
            const int page = col < had ? p.table[(int64_t)b * p.cols + col]
                                       : p.free_pages[s.count - 1 - (s.first[b] + col - had)];
            // (a page that is none gives a slot past the cache, which its calls report)
            const bool there = (unsigned)page < (unsigned)p.pages;
            bad |= !there;
            slot = there ? ((int64_t)page << p.page_shift) + (position & (size - 1)) : (int64_t)p.pages << p.page_shift;
        }
        p.slots[row] = slot;
        p.positions[row] = position;
    }
    if (bad) atomicOr(&p.flags[FLAG_BAD_ID], 1);
}

__global__ __launch_bounds__(PAGE_THREADS) void k_pages_trim(PageParams p) {
    extern __shared__ int lds[];
    PageScan s = page_scan<false>(p, lds);
    const int tid = threadIdx.x;
    const bool last = counts_last(p);
    const bool ok = s.ok && s.count + s.moved <= p.pages;
    if (!ok) {
        if (blockIdx.x == 0 && tid == 0) atomicOr(&p.flags[FLAG_BAD_ID], 1);
        return;
    }
    if (last) {
        for (int i = tid; i < p.seqs; i += PAGE_THREADS) p.lengths[i] = min(s.held[i], p.change[i]);
        if (tid == 0) *p.count = s.count + (int)s.moved;
    }
    bool bad = false;
    for (int j = blockIdx.x * PAGE_THREADS + tid; j < (int)s.moved; j += gridDim.x * PAGE_THREADS) {
        const int b = owner(s.first, p.seqs, j);
        const int left = pages_of(s.held[b], p.page_shift) - (s.first[b + 1] - s.first[b]);
        const int page = p.table[(int64_t)b * p.cols + left + j - s.first[b]];
        bad |= (unsigned)page >= (unsigned)p.pages;
        p.free_pages[s.count + s.moved - 1 - j] = page;
    }
    if (bad) atomicOr(&p.flags[FLAG_BAD_ID], 1);
}

static size_t page_lds(const PageParams& p) { return (size_t)(3 * p.seqs + 2) * sizeof(int); }

// 1024 rows a workgroup; pages that go back, 1024 a workgroup of what there can be
hipError_t launch_pages_extend(const PageParams& p, hipStream_t s) {
    const unsigned grid = (unsigned)std::max((p.rows + PAGE_THREADS * PAGE_ROWS - 1) / (PAGE_THREADS * PAGE_ROWS), 1);
    hipLaunchKernelGGL(k_pages_extend, dim3(grid), dim3(PAGE_THREADS), page_lds(p), s, p);
    return hipGetLastError();
}

hipError_t launch_pages_trim(const PageParams& p, hipStream_t s) {
    const int64_t most = std::min<int64_t>(p.pages, (int64_t)p.seqs * p.cols);
    const unsigned grid = (unsigned)std::min<int64_t>((most + 1023) / 1024, 32);
    hipLaunchKernelGGL(k_pages_trim, dim3(grid), dim3(PAGE_THREADS), page_lds(p), s, p);
    return hipGetLastError();
}

}  // namespace mqh
