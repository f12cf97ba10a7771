// vq_pages.hip -- the pages of the paged caches: the book of who holds which, on the host, and the launch that carries out what it
// decides, page copies and page-table entries.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <new>
#include <vector>

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
};
static_assert(sizeof(Moves) <= 4000, "kernel arguments");

// A workgroup copies one chunk of one page of one pool: 256 threads, four 16-byte pieces each, all loads before the first store
// (pools or pages that are not 16-byte aligned: two bytes, or one, at a time). The first workgroup writes the table's entries.
// Copies of a call neither read nor write a page that another one writes, so their order does not matter.
// Bound by bytes: 192 pages of 128 KB in four pools, 201 MB, in 36 us, 5.6 TB/s; small calls by latency, 4 pages in 8 pools 3.1 us.
// Chunks of 4 to 32 KB take the same within 2 %.
constexpr uint32_t kChunk = 256 * 64;
typedef uint32_t Piece __attribute__((ext_vector_type(4)));  // an array of uint4 goes through LDS: 40 us and 16
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
    // (Everything from the arguments, which lie in host memory, at once: none of these loads waits for another.)
    const Pair pages = m.copy[blockIdx.y];
    const uint64_t size = m.bytes[blockIdx.z], at = static_cast<uint64_t>(blockIdx.x) * kChunk;
    uint8_t *pool = m.pool[blockIdx.z];
    if ((blockIdx.x | blockIdx.y | blockIdx.z) == 0 && static_cast<int>(threadIdx.x) < m.entries)
        m.table[m.entry[threadIdx.x].a] = m.entry[threadIdx.x].b;
    if (m.copies == 0 || at >= size) return;
    const uint64_t n = size - at < kChunk ? size - at : kChunk;
    const uint8_t *from = pool + static_cast<uint64_t>(pages.a) * size + at;
    uint8_t *to = pool + static_cast<uint64_t>(pages.b) * size + at;
    const uint64_t low = reinterpret_cast<uintptr_t>(pool) | size;
    if (low % 16 == 0) copy_chunk<Piece>(from, to, n);
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

// What the lists say, in as few launches as the arguments hold. Every page and index is in range.
int launch_moves(void *const *pools, const size_t *page_bytes, int npools, const Pair *copies, int ncopies, int32_t *page_table,
                 const Pair *entries, int nentries, hipStream_t s) {
    uint64_t largest = 0;
    for (int i = 0; i < npools && ncopies > 0; ++i) largest = std::max<uint64_t>(largest, page_bytes[i]);
    const uint64_t chunks = (largest + kChunk - 1) / kChunk;
    if (chunks >= (1ull << 31)) return VQ_ERR_SHAPE;
    if (npools == 0) ncopies = 0;
    int done = 0, written = 0;
    while (done < ncopies || written < nentries) {
        Moves m;
        m.table = page_table;
        m.copies = std::min(ncopies - done, kPairs);
        m.entries = std::min(nentries - written, kPairs);
        std::copy(copies + done, copies + done + m.copies, m.copy);
        std::copy(entries + written, entries + written + m.entries, m.entry);
        done += m.copies;
        written += m.entries;
        for (int p = 0; p == 0 || (p < npools && m.copies > 0); p += kPools) {
            const int n = m.copies == 0 ? 1 : std::min(npools - p, kPools);
            for (int i = 0; i < n && m.copies > 0; ++i) {
                m.pool[i] = static_cast<uint8_t *>(pools[p + i]);
                m.bytes[i] = page_bytes[p + i];
            }
            move_pages_kernel<<<m.copies > 0 ? dim3(static_cast<unsigned>(chunks), m.copies, n) : dim3(1), 256, 0, s>>>(m);
            m.entries = 0;
        }
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return static_cast<int>(e);
    }
    return VQ_OK;
}

int check_pools(void *const *pools, const size_t *page_bytes, int npools) {
    for (int i = 0; i < npools; ++i) {
        if (!pools[i]) return VQ_ERR_ARG;
        if (page_bytes[i] < 1 || page_bytes[i] > (1ull << 40)) return VQ_ERR_SHAPE;
    }
    return VQ_OK;
}

// ---- the book of pages ----------------------------------------------------------------------------------------

}  // namespace

// Who holds which page, on the host. Free pages are a bit set searched from the lowest word that may have one, so a call costs what
// it changes (compact: the pages and the table once). Every vector but the plan's and the undo list's has its size from the start.
struct vq_book {
    int pages, page, per_slot, slots, free_pages;
    std::vector<int32_t> rows, count;  // [slot][per_slot], pages of each slot
    std::vector<int32_t> holders;
    std::vector<uint64_t> free_bits;
    size_t lowest = 0;  // no free page in the words before it
    std::vector<Pair> copies, entries;  // the last call's plan
    struct Undo {
        int32_t slot, index, before, taken;
    };
    std::vector<Undo> undo;
    std::vector<int32_t> root, filled;  // of a call's new slots: the slot that their pages come from (else -1), and how many
    char error[160] = "";

    int fail(int status, const char *format, ...) {
        va_list a;
        va_start(a, format);
        vsnprintf(error, sizeof(error), format, a);
        va_end(a);
        return status;
    }
    bool slot_ok(int s) const { return s >= 0 && s < slots; }
    // Pages that hold `length` positions, -1 where a slot cannot.
    int covering(long long length) const {
        const long long n = (length + page - 1) / page;
        return length < 0 || n > per_slot ? -1 : static_cast<int>(n);
    }
    int32_t *row(int s) { return rows.data() + static_cast<size_t>(s) * per_slot; }
    int take() {  // the lowest free page; free_pages > 0
        while (free_bits[lowest] == 0) ++lowest;
        const int p = static_cast<int>(lowest * 64) + __builtin_ctzll(free_bits[lowest]);
        free_bits[lowest] &= free_bits[lowest] - 1;
        --free_pages;
        holders[p] = 1;
        return p;
    }
    void give(int p) {
        holders[p] = 0;
        free_bits[p / 64] |= 1ull << (p % 64);
        lowest = std::min(lowest, static_cast<size_t>(p / 64));
        ++free_pages;
    }
    void drop(int p) {
        if (holders[p] == 1) give(p);
        else --holders[p];
    }
    void begin() {
        copies.clear();
        entries.clear();
        error[0] = 0;
    }
    void entry(int slot, int index, int p) { entries.push_back(Pair{slot * per_slot + index, p}); }

    int reserve(const int32_t *segs, int n);
    int fork(int src, const int32_t *dst, int n, int length);
    int copy(const int32_t *pairs, int n);
    int free(const int32_t *which, int n, int length);
    int compact();
};

int vq_book::reserve(const int32_t *segs, int n) {
    long long most = 0;  // pages that the segments touch: room in the lists for all of them before anything changes
    for (int i = 0; i < n; ++i) {
        const int slot = segs[4 * i], pos0 = segs[4 * i + 1], len = segs[4 * i + 2];
        const int end = pos0 < 0 || len < 1 ? -1 : covering(static_cast<long long>(pos0) + len);
        if (!slot_ok(slot) || end < 0) return fail(VQ_ERR_SHAPE, "segment (%d, %d, %d) outside the paged context", slot, pos0, len);
        most += end - pos0 / page;
    }
    undo.clear();
    undo.reserve(most);
    copies.reserve(most);
    entries.reserve(most);
    auto back = [&](int status) {
        for (size_t i = undo.size(); i-- > 0;) {
            const Undo &u = undo[i];
            if (u.before < 0) --count[u.slot];
            else row(u.slot)[u.index] = u.before, ++holders[u.before];
            give(u.taken);
        }
        copies.clear();
        entries.clear();
        return status;
    };
    for (int i = 0; i < n; ++i) {
        const int slot = segs[4 * i], pos0 = segs[4 * i + 1], len = segs[4 * i + 2], end = covering(static_cast<long long>(pos0) + len);
        int32_t *r = row(slot);
        if (pos0 / page > count[slot])
            return back(fail(VQ_ERR_SHAPE, "segment (%d, %d, %d): the slot holds %d pages, not all before its position", slot, pos0, len,
                             count[slot]));
        for (int k = pos0 / page; k < end; ++k) {
            const int old = k < count[slot] ? r[k] : -1;
            if (old >= 0 && holders[old] == 1) continue;
            if (free_pages == 0) return back(fail(VQ_ERR_NO_PAGES, "page pool exhausted"));
            const int fresh = take();
            undo.push_back(Undo{slot, k, old, fresh});
            if (old < 0) {
                r[count[slot]++] = fresh;
            } else {
                --holders[old];  // others hold it still
                r[k] = fresh;
                const long long a = static_cast<long long>(k) * page;
                if (pos0 > a || static_cast<long long>(pos0) + len < a + page) copies.push_back(Pair{old, fresh});
            }
            entry(slot, k, fresh);
        }
    }
    return VQ_OK;
}

int vq_book::fork(int src, const int32_t *dst, int n, int length) {
    const int k = covering(length);
    if (!slot_ok(src) || k < 0) return fail(VQ_ERR_SHAPE, "slot %d, %d positions: outside the paged context", src, length);
    if (k > count[src]) return fail(VQ_ERR_SHAPE, "slot %d holds %d pages, %d positions need %d", src, count[src], length, k);
    std::fill(root.begin(), root.end(), -1);
    for (int i = 0; i < n; ++i) {
        if (!slot_ok(dst[i])) return fail(VQ_ERR_SHAPE, "slot %d outside [0, %d)", dst[i], slots);
        if (count[dst[i]]) return fail(VQ_ERR_ARG, "slot %d holds %d pages (free them first)", dst[i], count[dst[i]]);
        if (root[dst[i]] >= 0) return fail(VQ_ERR_ARG, "slot %d is given twice", dst[i]);
        root[dst[i]] = src;
    }
    entries.reserve(static_cast<size_t>(n) * k);
    for (int i = 0; i < n; ++i) {
        std::copy(row(src), row(src) + k, row(dst[i]));
        count[dst[i]] = k;
        for (int j = 0; j < k; ++j) {
            ++holders[row(src)[j]];
            entry(dst[i], j, row(src)[j]);
        }
    }
    return VQ_OK;
}

int vq_book::copy(const int32_t *pairs, int n) {
    std::fill(root.begin(), root.end(), -1);
    long long need = 0;
    for (int i = 0; i < n; ++i) {
        const int src = pairs[3 * i], dst = pairs[3 * i + 1], length = pairs[3 * i + 2], k = covering(length);
        if (!slot_ok(src) || !slot_ok(dst) || k < 0)
            return fail(VQ_ERR_SHAPE, "slots %d, %d, %d positions: outside the paged context", src, dst, length);
        if (count[dst]) return fail(VQ_ERR_ARG, "slot %d holds %d pages (free them first)", dst, count[dst]);
        if (root[dst] >= 0) return fail(VQ_ERR_ARG, "slot %d is given twice", dst);
        // A slot that this call fills is read through the one that it is filled from.
        const int from = root[src] >= 0 ? root[src] : src, held = root[src] >= 0 ? filled[src] : count[src];
        if (k > held) return fail(VQ_ERR_SHAPE, "slot %d holds %d pages, %d positions need %d", src, held, length, k);
        root[dst] = from;
        filled[dst] = k;
        need += k;
    }
    if (need > free_pages) return fail(VQ_ERR_NO_PAGES, "page pool exhausted");
    copies.reserve(need);
    entries.reserve(need);
    for (int i = 0; i < n; ++i) {
        const int dst = pairs[3 * i + 1], k = covering(pairs[3 * i + 2]);
        for (int j = 0; j < k; ++j) {
            const int from = row(root[dst])[j], fresh = take();
            row(dst)[j] = fresh;
            copies.push_back(Pair{from, fresh});
            entry(dst, j, fresh);
        }
        count[dst] = k;
    }
    return VQ_OK;
}

int vq_book::free(const int32_t *which, int n, int length) {
    const int k = covering(length);
    if (k < 0) return fail(VQ_ERR_SHAPE, "%d positions outside the paged context", length);
    for (int i = 0; i < n; ++i)
        if (!slot_ok(which[i])) return fail(VQ_ERR_SHAPE, "slot %d outside [0, %d)", which[i], slots);
    for (int i = 0; i < n; ++i)
        while (count[which[i]] > k) drop(row(which[i])[--count[which[i]]]);
    return VQ_OK;
}

int vq_book::compact() {
    // The k-th page in use at n or above goes to the k-th free one below: nothing is both read and written.
    const int n = pages - free_pages;
    int hole = 0, moves = 0;
    long long touched = 0;
    for (int p = n; p < pages; ++p)
        if (holders[p]) ++moves, touched += holders[p];
    copies.reserve(moves);
    entries.reserve(touched);
    if (!moves) return VQ_OK;
    std::vector<int32_t> to(pages - n, -1);
    for (int p = n; p < pages; ++p) {
        if (!holders[p]) continue;
        while (holders[hole]) ++hole;
        copies.push_back(Pair{p, hole});
        to[p - n] = hole;
        holders[hole] = holders[p];
        holders[p] = 0;
    }
    for (int s = 0; s < slots; ++s)
        for (int j = 0; j < count[s]; ++j)
            if (int32_t &p = row(s)[j]; p >= n) {
                p = to[p - n];
                entry(s, j, p);
            }
    std::fill(free_bits.begin(), free_bits.end(), 0ull);
    for (int p = n; p < pages; ++p) free_bits[p / 64] |= 1ull << (p % 64);
    lowest = n / 64;
    return VQ_OK;
}

namespace {

// A book's call: no exception leaves it, and what could throw does so before anything has changed.
template <typename F>
int book_call(vq_book *b, F &&f) {
    if (!b) return VQ_ERR_ARG;
    b->begin();
    try {
        return f();
    } catch (const std::bad_alloc &) {
        return static_cast<int>(hipErrorOutOfMemory);
    } catch (...) {
        return VQ_ERR_ARG;
    }
}

}  // namespace

extern "C" {

int vq_move_pages(void *const *pools, const size_t *page_bytes, int npools, int pages, const int32_t *copies, int ncopies,
                  int32_t *page_table, int table_entries, const int32_t *entries, int nentries, void *stream) {
    if (ncopies < 0 || nentries < 0 || npools < 0) return VQ_ERR_SHAPE;
    if ((ncopies > 0 && (!copies || !pools || !page_bytes)) || (nentries > 0 && (!entries || !page_table))) return VQ_ERR_ARG;
    if (ncopies > 0) {
        if (pages < 1) return VQ_ERR_SHAPE;
        if (const int st = check_pools(pools, page_bytes, npools); st != VQ_OK) return st;
    }
    for (int i = 0; i < nentries; ++i)
        if (entries[2 * i] < 0 || entries[2 * i] >= table_entries) return VQ_ERR_SHAPE;
    if (const int st = check_copies(copies, ncopies, pages); st != VQ_OK) return st;
    return launch_moves(pools, page_bytes, npools, reinterpret_cast<const Pair *>(copies), ncopies, page_table,
                        reinterpret_cast<const Pair *>(entries), nentries, static_cast<hipStream_t>(stream));
}

vq_book *vq_book_create(int pages, int page_size, int pages_per_seq, int slots) {
    if (pages < 1 || page_size < 1 || pages_per_seq < 1 || slots < 1 || static_cast<long long>(slots) * pages_per_seq > INT32_MAX)
        return nullptr;
    try {
        auto *b = new vq_book{pages, page_size, pages_per_seq, slots, pages};
        try {
            b->rows.resize(static_cast<size_t>(slots) * pages_per_seq);
            b->count.resize(slots);
            b->root.resize(slots);
            b->filled.resize(slots);
            b->holders.resize(pages);
            b->free_bits.assign((static_cast<size_t>(pages) + 63) / 64, ~0ull);
            if (pages % 64) b->free_bits.back() = (1ull << (pages % 64)) - 1;
            return b;
        } catch (...) {
            delete b;
        }
    } catch (...) {
    }
    return nullptr;
}

void vq_book_destroy(vq_book *b) { delete b; }

int vq_book_reserve(vq_book *b, const int32_t *segs, int nseg) {
    if (nseg < 0 || (nseg > 0 && !segs)) return VQ_ERR_ARG;
    return book_call(b, [&] { return b->reserve(segs, nseg); });
}
int vq_book_fork(vq_book *b, int src, const int32_t *dst, int ndst, int length) {
    if (ndst < 0 || (ndst > 0 && !dst)) return VQ_ERR_ARG;
    return book_call(b, [&] { return b->fork(src, dst, ndst, length); });
}
int vq_book_copy(vq_book *b, const int32_t *pairs, int n) {
    if (n < 0 || (n > 0 && !pairs)) return VQ_ERR_ARG;
    return book_call(b, [&] { return b->copy(pairs, n); });
}
int vq_book_free(vq_book *b, const int32_t *slots, int n, int length) {
    if (n < 0 || (n > 0 && !slots)) return VQ_ERR_ARG;
    return book_call(b, [&] { return b->free(slots, n, length); });
}
int vq_book_compact(vq_book *b) {
    return book_call(b, [&] { return b->compact(); });
}

int vq_book_plan(const vq_book *b, const int32_t **copies, int *ncopies, const int32_t **entries, int *nentries) {
    if (!b || !copies || !ncopies || !entries || !nentries) return VQ_ERR_ARG;
    *copies = reinterpret_cast<const int32_t *>(b->copies.data());
    *ncopies = static_cast<int>(b->copies.size());
    *entries = reinterpret_cast<const int32_t *>(b->entries.data());
    *nentries = static_cast<int>(b->entries.size());
    return VQ_OK;
}
int vq_book_row(const vq_book *b, int slot, const int32_t **pages) {
    if (!b || !pages) return VQ_ERR_ARG;
    if (!b->slot_ok(slot)) return VQ_ERR_SHAPE;
    *pages = b->rows.data() + static_cast<size_t>(slot) * b->per_slot;
    return b->count[slot];
}
int vq_book_available(const vq_book *b) { return b ? b->free_pages : VQ_ERR_ARG; }
int vq_book_holders(const vq_book *b, int page) { return !b ? VQ_ERR_ARG : page < 0 || page >= b->pages ? VQ_ERR_SHAPE : b->holders[page]; }
const char *vq_book_error(const vq_book *b) { return b ? b->error : "no book"; }

int vq_book_apply(vq_book *b, void *const *pools, const size_t *page_bytes, int npools, int32_t *page_table, void *stream) {
    if (!b || !page_table || npools < 0 || (npools > 0 && (!pools || !page_bytes))) return VQ_ERR_ARG;
    if (const int st = check_pools(pools, page_bytes, npools); st != VQ_OK) return st;
    const int st = launch_moves(pools, page_bytes, npools, b->copies.data(), static_cast<int>(b->copies.size()), page_table,
                                b->entries.data(), static_cast<int>(b->entries.size()), static_cast<hipStream_t>(stream));
    b->begin();
    return st;
}

}  // extern "C"
