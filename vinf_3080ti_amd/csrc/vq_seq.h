// vq_seq.h -- what the sequence ops' translation units share: segment tables, cache addressing, cross-lane exchanges, the
// query operand of the f16 attention products and the merge of a split context's chunks.
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

// ---- attention: the query operand and the merge of chunks ---------------------------------------------------

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
// The query vector of lane column c (dims 32 u + 8 g .. + 7), loaded raw; fa16_q_split turns it into the B
// operands, times 1/sqrt(hd) * 2^s, and returns 2^-s log2(e): scores leave the S product in base-2 units, so
// the softmax weights are exp2 (v_exp_f32) of their differences, and maxima are converted back (times ln 2) only
// where they leave the kernel. Split in two so that a block's K/V loads can be issued
// between them.
template <int HD>
__device__ __forceinline__ void fa16_q_load(const float *qrow, float4 (&qr)[HD / 16]) {
    const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int u = 0; u < HD / 32; ++u) {
        qr[2 * u] = *reinterpret_cast<const float4 *>(qrow + 32 * u + 8 * g);
        qr[2 * u + 1] = *reinterpret_cast<const float4 *>(qrow + 32 * u + 8 * g + 4);
    }
}
template <int HD>
__device__ __forceinline__ float fa16_q_split(const float4 (&qr)[HD / 16], float scale, fh8 (&qh)[HD / 32],
                                              fh8 (&ql)[HD / 32]) {
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < HD / 16; ++i)
        amax = fmaxf(fmaxf(amax, fmaxf(fabsf(qr[i].x), fabsf(qr[i].y))), fmaxf(fabsf(qr[i].z), fabsf(qr[i].w)));
    amax *= scale;
    amax = xor16_max(amax);
    amax = xor32_max(amax);
    int ex = 0;
    if (amax > 0.0f && amax <= 3.0e38f) frexpf(amax, &ex);  // amax = f 2^ex, f in [0.5, 1)
    // Capped at 2^126 so that the scale and its inverse stay finite for queries below ~1e-34 (their scores are
    // then tiny, as they should be, instead of NaN).
    const int e2 = 14 - ex < 126 ? 14 - ex : 126;
    const float up = ldexpf(1.0f, e2);
#pragma unroll
    for (int u = 0; u < HD / 32; ++u) {
        const float v[8] = {qr[2 * u].x, qr[2 * u].y, qr[2 * u].z, qr[2 * u].w,
                            qr[2 * u + 1].x, qr[2 * u + 1].y, qr[2 * u + 1].z, qr[2 * u + 1].w};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            _Float16 h, l;
            split_h(v[j] * scale * up, h, l);
            qh[u][j] = h;
            ql[u][j] = l;
        }
    }
    return ldexpf(1.0f, -e2) * 1.44269504088896341f;  // S in base-2 units: the softmax uses exp2
}

// out = sum_c e^(m_c - M) o_c / sum_c e^(m_c - M) l_c, M = max_c m_c; one workgroup of four waves per (row of the
// pass, head): the chunks' maxima through LDS, then wave w adds chunks w, w + 4, ... (lane = four head dims, one
// 16-byte load per chunk) and the four waves' sums are added in wave order (deterministic).
template <int HD>
__global__ __launch_bounds__(256) void attention_merge_kernel(const float *__restrict__ part, const float *__restrict__ pml,
                                                              float *__restrict__ out, SegTable T, int heads, int hd,
                                                              int nch) {
    __shared__ float smx[4];
    __shared__ float4 sacc[4][HD / 4];
    __shared__ float sl[4];
    int t;
    const Seg &s = seg_of_row(T, blockIdx.x / heads, t);
    const int h = blockIdx.x % heads;
    const size_t qv = static_cast<size_t>(s.row0 + t) * heads + h;
    const float *ml = pml + qv * nch * 2;
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    float mx = -INFINITY;
    for (int c = tid; c < nch; c += 256) mx = fmaxf(mx, ml[2 * c]);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off, 64));
    if (lane == 0) smx[wv] = mx;
    __syncthreads();
    const float M = fmaxf(fmaxf(smx[0], smx[1]), fmaxf(smx[2], smx[3]));
    float4 acc{0.f, 0.f, 0.f, 0.f};
    float L = 0.0f;
    if (4 * lane < HD) {
        // Chunks wv, wv + 4, ... in order, four at a time with all their loads in flight.
        for (int c0 = wv; c0 < nch; c0 += 16) {
            float4 p4[4];
            float mc[4], lc[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int c = c0 + 4 * k < nch ? c0 + 4 * k : c0;
                p4[k] = *reinterpret_cast<const float4 *>(part + (qv * nch + c) * HD + 4 * lane);
                mc[k] = ml[2 * c];
                lc[k] = ml[2 * c + 1];
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (c0 + 4 * k >= nch) break;
                const float f = mc[k] == -INFINITY ? 0.0f : expf(mc[k] - M);
                L = fmaf(lc[k], f, L);
                acc.x = fmaf(p4[k].x, f, acc.x);
                acc.y = fmaf(p4[k].y, f, acc.y);
                acc.z = fmaf(p4[k].z, f, acc.z);
                acc.w = fmaf(p4[k].w, f, acc.w);
            }
        }
        sacc[wv][lane] = acc;
    }
    if (lane == 0) sl[wv] = L;
    __syncthreads();
    if (wv == 0 && 4 * lane < HD) {
        const float Lt = ((sl[0] + sl[1]) + sl[2]) + sl[3];
        const float inv = Lt > 0.0f ? 1.0f / Lt : 0.0f;
        const float4 a = sacc[0][lane], b = sacc[1][lane], c = sacc[2][lane], d = sacc[3][lane];
        const float r[4] = {((a.x + b.x) + c.x) + d.x, ((a.y + b.y) + c.y) + d.y, ((a.z + b.z) + c.z) + d.z,
                            ((a.w + b.w) + c.w) + d.w};
        float *o = out + qv * hd;
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (4 * lane + k < hd) o[4 * lane + k] = r[k] * inv;
    }
}

inline int fa_hd(int hd) { return hd <= 64 ? 64 : hd <= 128 ? 128 : 256; }
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
