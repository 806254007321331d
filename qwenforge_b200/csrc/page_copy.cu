// Rows of pages copied inside one storage, for every schedule entry (layer) at once: what a forked sequence needs of its parent's last page, what
// a rewound one needs of a page that others read too, and what moves pages to the front of the storage.
//   storage  [entries][pages][segments][rows][row bytes], a page dense, entries and pages at any distance
//   move     (from, to, rows): the first `rows` rows of every segment of page `from` become those of page `to`, in every entry
// No page is both a source and a target, and none is a target twice (the caller has checked), so the moves have no order.
// The moves travel as kernel arguments: the call costs one launch, with no copy of a table to the device before it.
// A block takes PC_THREADS x 4 vectors of one (entry, move). What bounds it: memory. Every thread has its four loads in flight before it stores.
// Measured (read and written bytes): 120 whole pages of 36 entries of 64 KB 85 us, 6.6 TB/s; 64 part pages of those 27 us; seven part pages of 24 entries of
// 32 KB 2.6 us, where it is latency.
#include <algorithm>
#include <new>
#include <vector>

#include "common.cuh"

#define PC_THREADS 256
#define PC_EACH 4

struct PageMove {
    int from, to, rows;
};
template <int N> struct PageMoves {
    PageMove move[N];
};

template <typename V, int N>
__global__ void __launch_bounds__(PC_THREADS)
page_copy_kernel(const __grid_constant__ PageMoves<N> moves, unsigned char* base, long long entry_bytes, long long page_bytes, int segments,
                 int segment_vecs, int row_vecs) {
    grid_chain_entry();
    const PageMove m = moves.move[blockIdx.y];
    const int run = m.rows * row_vecs;   // vectors of a segment that are copied
    const long long total = (long long)run * segments;
    const V* from = reinterpret_cast<const V*>(base + blockIdx.z * entry_bytes + m.from * page_bytes);
    V* to = reinterpret_cast<V*>(base + blockIdx.z * entry_bytes + m.to * page_bytes);
    const bool whole = run == segment_vecs;   // what is copied has no gaps
    for (long long i0 = (long long)blockIdx.x * (PC_THREADS * PC_EACH) + threadIdx.x; i0 < total; i0 += (long long)gridDim.x * (PC_THREADS * PC_EACH)) {
        V v[PC_EACH];
        long long at[PC_EACH];
#pragma unroll
        for (int u = 0; u < PC_EACH; ++u) {
            const long long i = i0 + u * PC_THREADS;
            at[u] = i;
            if (!whole && i < total) at[u] = i / run * segment_vecs + i % run;
            if (i < total) v[u] = from[at[u]];
        }
#pragma unroll
        for (int u = 0; u < PC_EACH; ++u)
            if (i0 + u * PC_THREADS < total) to[at[u]] = v[u];
    }
}

template <typename V, int N>
static cudaError_t launch_moves(const PageMove* moves, int n, unsigned char* base, int entries, long long entry_bytes, long long page_bytes,
                                int segments, long long segment_bytes, long long row_bytes, cudaStream_t stream) {
    PageMoves<N> some;
    int most = 0;
    for (int i = 0; i < n; ++i) {
        some.move[i] = moves[i];
        most = moves[i].rows > most ? moves[i].rows : most;
    }
    for (int i = n; i < N; ++i) some.move[i] = PageMove{0, 0, 0};
    const long long vecs = (long long)most * (row_bytes / (long long)sizeof(V)) * segments;
    long long across = (vecs + PC_THREADS * PC_EACH - 1) / (PC_THREADS * PC_EACH);
    if (across <= 0) return cudaSuccess;
    if (across > 1 << 20) across = 1 << 20;
    return launch_pdl(page_copy_kernel<V, N>, dim3((unsigned)across, (unsigned)n, (unsigned)entries), dim3(PC_THREADS), 0, stream, some, base, entry_bytes,
                      page_bytes, segments, (int)(segment_bytes / (long long)sizeof(V)), (int)(row_bytes / (long long)sizeof(V)));
}

// What is wrong with n moves of pages 0 .. n_pages - 1 of n_rows rows: 0 nothing, -1 a page outside, -2 rows outside, -3 a page that is the target of two
// moves, -4 one that is both a source and a target, -5 no memory for the check.
QF_EXPORT int qf_page_moves_check(const int* moves, int n, int n_pages, int n_rows) {
    const PageMove* m = reinterpret_cast<const PageMove*>(moves);
    for (int i = 0; i < n; ++i)
        if (m[i].from < 0 || m[i].from >= n_pages || m[i].to < 0 || m[i].to >= n_pages) return -1;
    for (int i = 0; i < n; ++i)
        if (m[i].rows < 0 || m[i].rows > n_rows) return -2;
    try {
        std::vector<int> targets(n > 0 ? n : 0);
        for (int i = 0; i < n; ++i) targets[i] = m[i].to;
        if (!std::is_sorted(targets.begin(), targets.end())) std::sort(targets.begin(), targets.end());
        for (int i = 1; i < n; ++i)
            if (targets[i] == targets[i - 1]) return -3;
        for (int i = 0; i < n; ++i)
            if ((i == 0 || m[i].from != m[i - 1].from) && std::binary_search(targets.begin(), targets.end(), m[i].from)) return -4;
    } catch (const std::bad_alloc&) {
        return -5;
    }
    return 0;
}

// moves: [n][3] int32 on the HOST. `unit`: 16, 4, 2 or 1 bytes, which divides the base address and every distance. Returns a CUDA error code, or what
// qf_page_moves_check says.
QF_EXPORT int qf_copy_pages(void* base, int entries, int pages, int rows, long long entry_bytes, long long page_bytes, int segments,
                            long long segment_bytes, long long row_bytes, int unit, const int* moves, int n, cudaStream_t stream) {
    const int wrong = qf_page_moves_check(moves, n, pages, rows);
    if (wrong) return wrong;
    if (entries <= 0 || n <= 0 || segments <= 0 || segment_bytes <= 0) return 0;
    if (entries > 65535 || segment_bytes / unit > 0x7fffffffll) return (int)cudaErrorInvalidValue;
    const PageMove* m = reinterpret_cast<const PageMove*>(moves);
    unsigned char* b = reinterpret_cast<unsigned char*>(base);
    constexpr int FEW = 64, MANY = 1024;   // (arguments of 768 bytes and of 12 KB: a launch of few moves 3.7 microseconds of host time against 6.6)
    for (int i = 0; i < n;) {
        const int here = n - i < MANY ? n - i : MANY;
        cudaError_t e = cudaErrorInvalidValue;
#define QF_PC(V) \
    e = here <= FEW ? launch_moves<V, FEW>(m + i, here, b, entries, entry_bytes, page_bytes, segments, segment_bytes, row_bytes, stream) \
                    : launch_moves<V, MANY>(m + i, here, b, entries, entry_bytes, page_bytes, segments, segment_bytes, row_bytes, stream)
        if (unit == 16) QF_PC(uint4);
        else if (unit == 4) QF_PC(uint32_t);
        else if (unit == 2) QF_PC(uint16_t);
        else if (unit == 1) QF_PC(unsigned char);
#undef QF_PC
        if (e != cudaSuccess) return (int)e;
        i += here;
    }
    return 0;
}
