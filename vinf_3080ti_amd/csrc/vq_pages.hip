// vq_pages.hip -- page copies and page-table entries of the paged caches (the device's side of pages_reserve, pages_fork,
// pages_copy and pages_compact).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <new>

#include "../../include/vq.h"
#include "vq_seq.h"

namespace {

// One launch's share of a call, in the kernel arguments (under the 4 KB that they may have).
constexpr int kPools = 32, kPairs = 192;
struct Pair {
    int32_t a, b;  // copies: page a to page b; entries: index a gets value b
};
struct Moves {
    uint8_t *pool[kPools];
    uint64_t bytes[kPools];  // of a page
    Pair copy[kPairs], entry[kPairs];
    int32_t *table;
    int copies, entries;
    uint32_t chunks;  // of the largest page
};
static_assert(sizeof(Moves) <= 4000, "kernel arguments");

// A workgroup copies one chunk of one page of one pool: 256 threads, four 16-byte pieces each, all loads before the first store
// (pools or pages that are not 16-byte aligned: two bytes, or one, at a time). The last workgroup writes the table's entries.
// Copies of a call neither read nor write a page that another one writes, so their order does not matter. Bound by bytes.
constexpr uint32_t kChunk = 256 * 64;
template <typename V>
__device__ __forceinline__ void copy_chunk(const uint8_t *from, uint8_t *to, uint64_t n) {
    const V *s = reinterpret_cast<const V *>(from);
    V *d = reinterpret_cast<V *>(to);
    const uint32_t count = static_cast<uint32_t>(n / sizeof(V));
    for (uint32_t i = threadIdx.x; i < count; i += 4 * 256) {
        V v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = s[min(i + 256 * j, count - 1)];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i + 256 * j < count) d[i + 256 * j] = v[j];
    }
}
__global__ __launch_bounds__(256) void move_pages_kernel(Moves m) {
    uint32_t b = blockIdx.x;
    const uint32_t work = m.copies * m.chunks;
    if (b >= work) {
        if (blockIdx.y == 0 && static_cast<int>(threadIdx.x) < m.entries) m.table[m.entry[threadIdx.x].a] = m.entry[threadIdx.x].b;
        return;
    }
    const uint32_t c = b / m.chunks, chunk = b - c * m.chunks;
    const uint64_t size = m.bytes[blockIdx.y], at = static_cast<uint64_t>(chunk) * kChunk;
    if (at >= size) return;
    const uint64_t n = size - at < kChunk ? size - at : kChunk;
    uint8_t *pool = m.pool[blockIdx.y];
    const uint8_t *from = pool + static_cast<uint64_t>(m.copy[c].a) * size + at;
    uint8_t *to = pool + static_cast<uint64_t>(m.copy[c].b) * size + at;
    const uint64_t low = reinterpret_cast<uintptr_t>(pool) | size;
    if (low % 16 == 0) copy_chunk<uint4>(from, to, n);
    else if (low % 2 == 0) copy_chunk<uint16_t>(from, to, n);
    else copy_chunk<uint8_t>(from, to, n);
}
static_assert(kPairs <= 256, "one workgroup writes the entries");

// Every page in range, no page written twice or both read and written.
int check_copies(const int32_t *copies, int n, int pages) {
    if (n == 0) return VQ_OK;
    uint8_t *seen = new (std::nothrow) uint8_t[pages]();
    if (!seen) return static_cast<int>(hipErrorOutOfMemory);
    int st = VQ_OK;
    for (int i = 0; i < n && st == VQ_OK; ++i) {
        const int a = copies[2 * i], b = copies[2 * i + 1];
        if (a < 0 || a >= pages || b < 0 || b >= pages) st = VQ_ERR_SHAPE;
        else if (seen[b] || (seen[a] & 2) || a == b) st = VQ_ERR_ARG;
        else seen[a] |= 1, seen[b] |= 2;
    }
    delete[] seen;
    return st;
}

}  // namespace

extern "C" int vq_move_pages(void *const *pools, const size_t *page_bytes, int npools, int pages, const int32_t *copies, int ncopies,
                             int32_t *page_table, int table_entries, const int32_t *entries, int nentries, void *stream) {
    if (ncopies < 0 || nentries < 0 || npools < 0) return VQ_ERR_SHAPE;
    if ((ncopies > 0 && (!copies || !pools || !page_bytes)) || (nentries > 0 && (!entries || !page_table))) return VQ_ERR_ARG;
    if (ncopies > 0 && pages < 1) return VQ_ERR_SHAPE;
    uint64_t largest = 0;
    if (ncopies > 0) {
        for (int i = 0; i < npools; ++i) {
            if (!pools[i]) return VQ_ERR_ARG;
            if (page_bytes[i] < 1 || page_bytes[i] > (1ull << 40)) return VQ_ERR_SHAPE;
            largest = page_bytes[i] > largest ? page_bytes[i] : largest;
        }
    }
    for (int i = 0; i < nentries; ++i)
        if (entries[2 * i] < 0 || entries[2 * i] >= table_entries) return VQ_ERR_SHAPE;
    if (const int st = check_copies(copies, ncopies, pages); st != VQ_OK) return st;
    const uint64_t chunks = (largest + kChunk - 1) / kChunk;
    if (chunks * kPairs >= (1ull << 31)) return VQ_ERR_SHAPE;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (npools == 0) ncopies = 0;
    int done = 0, written = 0;
    while (done < ncopies || written < nentries) {
        Moves m;
        m.chunks = static_cast<uint32_t>(chunks);
        m.table = page_table;
        m.copies = ncopies - done < kPairs ? ncopies - done : kPairs;
        m.entries = nentries - written < kPairs ? nentries - written : kPairs;
        for (int i = 0; i < m.copies; ++i) m.copy[i] = Pair{copies[2 * (done + i)], copies[2 * (done + i) + 1]};
        for (int i = 0; i < m.entries; ++i) m.entry[i] = Pair{entries[2 * (written + i)], entries[2 * (written + i) + 1]};
        for (int p = 0; p == 0 || (p < npools && m.copies > 0); p += kPools) {
            const int n = m.copies == 0 ? 1 : npools - p < kPools ? npools - p : kPools;
            for (int i = 0; i < n && m.copies > 0; ++i) {
                m.pool[i] = static_cast<uint8_t *>(pools[p + i]);
                m.bytes[i] = page_bytes[p + i];
            }
            const uint32_t blocks = m.copies * m.chunks + (m.entries > 0 ? 1 : 0);
            move_pages_kernel<<<dim3(blocks, n), 256, 0, s>>>(m);
            m.entries = 0;
        }
        done += m.copies;
        written += nentries - written < kPairs ? nentries - written : kPairs;
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return static_cast<int>(e);
    }
    return VQ_OK;
}
