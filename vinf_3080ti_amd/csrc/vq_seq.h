// vq_seq.h -- what the sequence ops' translation units share: segment tables, cache addressing, cross-lane exchanges, operand
// types of the f16 products.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/vq.h"

namespace {

inline int status_of(hipError_t e) { return e == hipSuccess ? VQ_OK : static_cast<int>(e); }

// ---- segments and cache addressing ---------------------------------------------------------------------

// A pass's segment table, passed by value in the kernel arguments (1 KB at the maximum).
struct Seg {
    int slot, pos0, rows, row0;
};
struct SegTable {
    int n;
    int total;  // sum of rows (the blocks of a per-row grid)
    Seg s[VQ_MAX_SEGMENTS];
};

// Cross-row lane exchanges of gfx950 without LDS: v_permlane16_swap (rows 0<->1, 2<->3) and v_permlane32_swap (lane
// halves). Called with the same value twice, the pair holds each lane's value and its partner's (lane ^ 16 or
// lane ^ 32) in an order that depends on the lane, so max and (commutative) sums come out bit-identical on both
// partners, as with __shfl_xor.
__device__ __forceinline__ float xor16_max(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float xor32_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float xor16_add(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float xor32_add(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Global row index g (segments in table order) -> (segment, row within it).
__device__ __forceinline__ const Seg &seg_of_row(const SegTable &T, int g, int &local) {
    int i = 0;
    while (i + 1 < T.n && g >= T.s[i].rows) {
        g -= T.s[i].rows;
        ++i;
    }
    local = g;
    return T.s[i];
}

// KV cache rows: contiguous [kv_head][max_seq][hd] when pt is null, else a page pool
// [page][kv_head][page_size][hd] with the sequence slot's page ids at pt[slot * pps + pos / page_size].
struct KvMap {
    const int32_t *pt;
    int max_seq;  // contiguous caches
    int page, pps, kv_heads;
    __device__ __forceinline__ size_t row(int slot, int kvh, int pos) const {
        if (pt == nullptr) return static_cast<size_t>(kvh) * max_seq + pos;
        const int pg = pt[slot * pps + pos / page];
        return (static_cast<size_t>(pg) * kv_heads + kvh) * page + pos % page;
    }
    // The same with the layout fixed at compile time: no branch around the page-table load, so the compiler can
    // keep the loads that follow in flight (a load under a branch makes it wait for every outstanding load).
    template <bool PAGED>
    __device__ __forceinline__ size_t row_t(int slot, int kvh, int pos) const {
        return row_in<PAGED>(PAGED ? page_of(slot, pos) : 0, kvh, pos);
    }
    // The lookup in two parts, for a caller with other work between the page's load and its use.
    __device__ __forceinline__ int page_of(int slot, int pos) const { return pt[slot * pps + pos / page]; }
    template <bool PAGED>
    __device__ __forceinline__ size_t row_in(int pg, int kvh, int pos) const {
        if constexpr (!PAGED) return static_cast<size_t>(kvh) * max_seq + pos;
        return (static_cast<size_t>(pg) * kv_heads + kvh) * page + pos % page;
    }
};

inline KvMap paged(const int32_t *pt, int page_size, int pps, int kv_heads) { return KvMap{pt, 0, page_size, pps, kv_heads}; }
inline KvMap contiguous(int max_seq, int kv_heads) { return KvMap{nullptr, max_seq, 1, 1, kv_heads}; }

// Host side: validate a segment table ([n][4] int32: slot, pos0, rows, row0) into a SegTable.
inline int make_table(const int32_t *segs, int nseg, SegTable &T, int *rows_spanned) {
    if (segs == nullptr || nseg < 1 || nseg > VQ_MAX_SEGMENTS) return VQ_ERR_ARG;
    T.n = nseg;
    T.total = 0;
    int span = 0;
    for (int i = 0; i < nseg; ++i) {
        const Seg s{segs[4 * i], segs[4 * i + 1], segs[4 * i + 2], segs[4 * i + 3]};
        if (s.slot < 0 || s.pos0 < 0 || s.rows < 1 || s.row0 < 0) return VQ_ERR_SHAPE;
        T.s[i] = s;
        T.total += s.rows;
        span = s.row0 + s.rows > span ? s.row0 + s.rows : span;
    }
    if (rows_spanned) *rows_spanned = span;
    return VQ_OK;
}

inline SegTable one_segment(int pos0, int rows) {
    SegTable T{};
    T.n = 1;
    T.total = rows;
    T.s[0] = Seg{0, pos0, rows, 0};
    return T;
}

// ---- operands of the f16 products -----------------------------------------------------------------------

typedef float fa4 __attribute__((ext_vector_type(4)));
typedef _Float16 fh8 __attribute__((ext_vector_type(8)));
typedef _Float16 fh4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ fh8 ld_h8(const _Float16 *p) {
    const uint4 v = *reinterpret_cast<const uint4 *>(p);
    return __builtin_bit_cast(fh8, v);
}
__device__ __forceinline__ void split_h(float x, _Float16 &hi, _Float16 &lo) {
    hi = static_cast<_Float16>(x);
    lo = static_cast<_Float16>(x - static_cast<float>(hi));
}
inline int max_seg_rows(const SegTable &T) {
    int r = 0;
    for (int i = 0; i < T.n; ++i) r = T.s[i].rows > r ? T.s[i].rows : r;
    return r;
}

inline int check_paging(const int32_t *pt, int page_size, int pps, const SegTable &T) {
    if (pt == nullptr) return VQ_ERR_ARG;
    if (page_size < 1 || pps < 1) return VQ_ERR_SHAPE;
    for (int i = 0; i < T.n; ++i)
        if (static_cast<long>(T.s[i].pos0) + T.s[i].rows > static_cast<long>(page_size) * pps) return VQ_ERR_SHAPE;
    return VQ_OK;
}

}  // namespace
