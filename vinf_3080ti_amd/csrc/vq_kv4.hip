// vq_kv4.hip -- the KV cache in 4 bits: append, read-back and attention (layout and rounding rule: include/vq.h).
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <type_traits>

#include "../../include/vq.h"
#include "vq_lds.h"
#include "vq_seq.h"

namespace {

constexpr int kSlab = 8;             // positions of a V word; pages are whole numbers of slabs
constexpr int kMaxHd = 256;
constexpr float kMaxScale = 4352.f;  // the largest scale whose 15-fold is still an f16
constexpr uint32_t kNanHeader = 0x7E00;

// ---- addressing ------------------------------------------------------------------------------------------

// Cache blocks of a pass: contiguous [kv_head] (pt null: one page of every position), else pools [page][kv_head].
struct Map4 {
    const int32_t *pt;
    int pps, pages, kv_heads;
    uint32_t spp, mul, shift;  // slabs per page; slab / spp = slab * mul >> shift for slab < 2^28
    size_t bytes;              // of a block
};

struct Place {
    size_t at;     // first byte of the block
    uint32_t slab;  // within it
    bool bad;      // the page table's entry is not a page
};

template <bool PAGED>
__device__ __forceinline__ Place place(const Map4 &M, int slot, int kvh, uint32_t slab) {
    if constexpr (!PAGED) return Place{static_cast<size_t>(kvh) * M.bytes, slab, false};
    const uint32_t p = static_cast<uint32_t>((static_cast<uint64_t>(slab) * M.mul) >> M.shift);
    const int pg = M.pt[static_cast<size_t>(slot) * M.pps + p];
    const bool bad = static_cast<uint32_t>(pg) >= static_cast<uint32_t>(M.pages);
    return Place{(static_cast<size_t>(bad ? 0 : pg) * M.kv_heads + kvh) * M.bytes, slab - p * M.spp, bad};
}

// ---- segments ----------------------------------------------------------------------------------------------

// Where each segment's rows (or other units of a grid) begin, and how many there are in all.
struct Starts {
    int total;
    int first[VQ_MAX_SEGMENTS];
};

// A segment as a workgroup finds it: the last one whose beginning is <= x. Lane i loads segment i and what goes with it, all at
// once, and the found one's values come from its lane. Kernel arguments lie in host memory, 2 us away at the first touch, and one
// load after the other (a walk over the segments, then their rows, then their bases) made up a third of a decode step's time.
struct Found {
    Seg s;
    int index, first, next;  // beginning of the segment, and of the next one
};
__device__ __forceinline__ int from_lane(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
__device__ __forceinline__ Found find_segment(const SegTable &T, const int *first, int total, int x) {
    const int lane = threadIdx.x & 63;
    const Seg mine = T.s[lane];
    const int f = first[lane], n = T.n;
    const int i = __builtin_popcountll(__ballot(lane < n && f <= x)) - 1;
    return Found{Seg{from_lane(mine.slot, i), from_lane(mine.pos0, i), from_lane(mine.rows, i), from_lane(mine.row0, i)}, i,
                 from_lane(f, i), i + 1 < n ? from_lane(f, i + 1 < 64 ? i + 1 : 63) : total};
}
// ---- values --------------------------------------------------------------------------------------------------

// Word of dim d among a V slab's hd words.
__device__ __forceinline__ int v_word(int d, int hd) {
    const int w = hd % 64 == 0 ? 4 : 2;
    return ((d / (16 * w)) * 16 + (d & 15)) * w + (d >> 4) % w;
}
// Bit position of element e in a word.
__device__ __forceinline__ int nib(int e) { return 4 * (e >> 1) + 16 * (e & 1); }

__device__ __forceinline__ float scale_of(uint32_t header) {
    return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(header & 0xFFF0u)));
}
__device__ __forceinline__ float value_of(uint32_t header, uint32_t code) {
    return scale_of(header) * static_cast<float>(static_cast<int>(code) - static_cast<int>(header & 15u));
}

// ---- append ------------------------------------------------------------------------------------------------

// x / d to the nearest whole number, ties to even, for |x / d| of up to 2^22: the rounded product with the reciprocal is at most
// one off, and the remainder x - n d is exact where it decides (n d has at most 12 significant bits). Off it is only near a tie,
// so the correction is behind a branch that few waves take.
template <int N>
__device__ __forceinline__ void nearest(const float (&x)[N], float d, float inv, float (&n)[N]) {
    const float half = 0.5f * d;
    bool near_tie = false;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        n[i] = rintf(x[i] * inv);
        near_tie = near_tie || fabsf(fmaf(-n[i], d, x[i])) >= half;
    }
    if (!__any(near_tie)) return;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float e = fmaf(-n[i], d, x[i]);
        const bool odd = n[i] - 2.0f * floorf(0.5f * n[i]) != 0.0f;
        if (e > half || (e == half && odd)) n[i] += 1.0f;
        else if (e < -half || (e == -half && odd)) n[i] -= 1.0f;
    }
}

// Scale of a group whose values, with zero, span [lo, hi]: the smallest k 2^e, k < 128, e >= -20, with 15 k 2^e >= hi - lo. The
// first guess from a rounded quotient is at most one k off; 15 k 2^e and the span are compared in 64 bits.
__device__ __forceinline__ float scale_for(float lo, float hi) {
    const double span = static_cast<double>(hi) - static_cast<double>(lo);
    const float t = static_cast<float>(span * (1.0 / 15.0));
    if (!(t < kMaxScale)) return kMaxScale;
    // t = f 2^ex, f in [0.5, 1); a span too small for t takes the smallest step.
    const int ex = t > 0.0f ? __builtin_amdgcn_frexp_expf(t) : -99, by = ex - 7 > -20 ? ex - 7 : -20;
    const float step = __uint_as_float(static_cast<uint32_t>(127 + by) << 23);
    float k = ceilf(t * __uint_as_float(static_cast<uint32_t>(127 - by) << 23));  // t / step, exact
    if (15.0 * static_cast<double>((k - 1.0f) * step) >= span && k > 0.0f) k -= 1.0f;
    if (15.0 * static_cast<double>(k * step) < span) k += 1.0f;
    return fminf(k * step, kMaxScale);
}

struct Group4 {
    uint32_t word;    // codes of the lane's eight dims
    uint32_t header;  // of the group of 32
};

// Four neighbouring lanes hold a group of 32 values, eight each.
__device__ __forceinline__ Group4 quantize_group4(const float (&x)[8]) {
    float lo = 0.0f, hi = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) lo = fminf(lo, x[e]), hi = fmaxf(hi, x[e]);
#pragma unroll
    for (int o = 1; o <= 2; o <<= 1) lo = fminf(lo, __shfl_xor(lo, o, 64)), hi = fmaxf(hi, __shfl_xor(hi, o, 64));
    float d = scale_for(lo, hi);
    const bool some = d > 0.0f;
    d = some ? d : 1.0f;
    // Values past 16 steps, which only the largest scale leaves, are cut: their code is at an end of the range anyway.
    float v[9], n[9];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = fminf(fmaxf(x[e], -16.0f * d), 16.0f * d);
    v[8] = fminf(-lo, 16.0f * d);
    nearest(v, d, 1.0f / d, n);
    const float z = fminf(n[8], 15.0f);
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) w |= static_cast<uint32_t>(fminf(fmaxf(n[e] + z, 0.0f), 15.0f)) << nib(e);
    if (!some) return Group4{0u, 0u};
    return Group4{w, static_cast<uint32_t>(__builtin_bit_cast(uint16_t, static_cast<_Float16>(d))) | static_cast<uint32_t>(z)};
}

// One workgroup of hd threads (64 at least) per (segment, slab of 8 positions, kv head): hd / 8 threads take a row, eight dims each,
// of k and then of v. K words and all headers are the row's own. V words hold eight positions of a dim: the codes meet in LDS and
// thread d puts dim d's word together; where the segment has only some of its positions the others' bits stay as they are, by an
// atomic exclusive-or of what changes (another segment of the launch may write the rest of the word). Bound by bytes: 8 read, 9/8
// written for a (k, v) pair.
template <bool PAGED>
__global__ __launch_bounds__(kMaxHd) void kv4_append_kernel(const float *__restrict__ k, const float *__restrict__ v, uint8_t *kc,
                                                            uint8_t *vc, SegTable T, Starts R, Map4 M, int hd) {
    __shared__ uint32_t vw[kSlab][kMaxHd / 8];
    __shared__ int broken[kSlab];
    const int kvh = blockIdx.y, tid = threadIdx.x;
    const Found found = find_segment(T, R.first, R.total, blockIdx.x);
    const Seg s = found.s;
    const int slab = s.pos0 / kSlab + (blockIdx.x - found.first);
    const int r0 = max(s.pos0 - slab * kSlab, 0), r1 = min(s.pos0 + s.rows - slab * kSlab, kSlab);
    const Place at = place<PAGED>(M, s.slot, kvh, slab);
    if (at.bad) return;
    const int per = hd / 8, row = tid / per, i = tid - row * per;
    const bool on = row >= r0 && row < r1;
    const size_t head = static_cast<size_t>(M.spp) * kSlab * (hd / 2);
    float x[2][8];
    if (tid < kSlab) broken[tid] = 0;
    __syncthreads();
    // Threads without a row read the segment's first one of the slab, and count as zeros.
    const size_t src = (static_cast<size_t>(s.row0 + slab * kSlab + (on ? row : r0) - s.pos0) * M.kv_heads + kvh) * hd + 8 * i;
    __builtin_memcpy(x[0], k + src, 32);
    __builtin_memcpy(x[1], v + src, 32);
    bool ok = true;
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[a][e] = on ? x[a][e] : 0.0f;
            ok = ok && fabsf(x[a][e]) < INFINITY;
        }
    if (!ok) broken[row] = 1;
    __syncthreads();
    const bool nan = on && broken[row] != 0;
#pragma unroll
    for (int a = 0; a < 2; ++a) {
        Group4 q = quantize_group4(x[a]);
        if (nan) q = Group4{0u, a == 0 ? kNanHeader : 0u};
        uint8_t *blk = (a == 0 ? kc : vc) + at.at;
        uint16_t *h = reinterpret_cast<uint16_t *>(blk + head);
        if (a == 0 && on) {
            const size_t pos = static_cast<size_t>(at.slab) * kSlab + row;
            reinterpret_cast<uint32_t *>(blk)[pos * per + (i & 3) * (hd / 32) + (i >> 2)] = q.word;
            if ((i & 3) == 0) h[pos * (hd / 32) + (i >> 2)] = static_cast<uint16_t>(q.header);
        }
        if (a == 1 && row < kSlab) {
            vw[row][i] = on ? q.word : 0u;
            if (on && (i & 3) == 0) h[(static_cast<size_t>(at.slab) * (hd / 32) + (i >> 2)) * 8 + row] = static_cast<uint16_t>(q.header);
        }
    }
    __syncthreads();
    if (tid >= hd) return;
    uint32_t w = 0, mine = 0;
#pragma unroll
    for (int r = 0; r < kSlab; ++r) {
        w |= ((vw[r][tid >> 3] >> nib(tid & 7)) & 15u) << nib(r);
        mine |= r >= r0 && r < r1 ? 15u << nib(r) : 0u;
    }
    uint32_t *to = reinterpret_cast<uint32_t *>(vc + at.at) + static_cast<size_t>(at.slab) * hd + v_word(tid, hd);
    if (mine == ~0u) *to = w;
    else atomicXor(to, (*to ^ w) & mine);
}

// The values held at the rows' positions, by the append kernel's workgroups: hd / 8 threads take a K row, a word each, and thread d
// the V word of dim d, whose positions are as many rows of the output. Bound by bytes: 9/8 read, 8 written for a (k, v) pair.
template <bool PAGED>
__global__ __launch_bounds__(kMaxHd) void kv4_read_kernel(const uint8_t *__restrict__ kc, const uint8_t *__restrict__ vc,
                                                          float *__restrict__ k, float *__restrict__ v, SegTable T, Starts R, Map4 M,
                                                          int hd) {
    const int kvh = blockIdx.y, tid = threadIdx.x;
    const Found found = find_segment(T, R.first, R.total, blockIdx.x);
    const Seg s = found.s;
    const int slab = s.pos0 / kSlab + (blockIdx.x - found.first);
    const int r0 = max(s.pos0 - slab * kSlab, 0), r1 = min(s.pos0 + s.rows - slab * kSlab, kSlab);
    const Place at = place<PAGED>(M, s.slot, kvh, slab);
    const int per = hd / 8, row = tid / per, i = tid - row * per;
    const size_t head = static_cast<size_t>(M.spp) * kSlab * (hd / 2);
    const size_t stride = static_cast<size_t>(M.kv_heads) * hd;  // of a row of k and v
    const size_t dst = (static_cast<size_t>(s.row0) * M.kv_heads + kvh) * hd;
    auto row_at = [&](int r) { return dst + static_cast<size_t>(slab * kSlab + r - s.pos0) * stride; };
    if (row >= r0 && row < r1) {
        const size_t pos = static_cast<size_t>(at.slab) * kSlab + row;
        const uint8_t *b = kc + at.at;
        const uint32_t w = reinterpret_cast<const uint32_t *>(b)[pos * per + (i & 3) * (hd / 32) + (i >> 2)];
        const uint32_t h = at.bad ? kNanHeader : reinterpret_cast<const uint16_t *>(b + head)[pos * (hd / 32) + (i >> 2)];
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = value_of(h, (w >> nib(e)) & 15u);
        __builtin_memcpy(k + row_at(row) + 8 * i, x, 32);
    }
    if (tid >= hd) return;
    const uint8_t *b = vc + at.at;
    const uint32_t w = reinterpret_cast<const uint32_t *>(b)[static_cast<size_t>(at.slab) * hd + v_word(tid, hd)];
    uint4 hv = *reinterpret_cast<const uint4 *>(b + head + (static_cast<size_t>(at.slab) * (hd / 32) + (tid >> 5)) * 16);
    if (at.bad) hv = uint4{kNanHeader * 0x10001u, kNanHeader * 0x10001u, kNanHeader * 0x10001u, kNanHeader * 0x10001u};
    const uint32_t h[4] = {hv.x, hv.y, hv.z, hv.w};
#pragma unroll
    for (int r = 0; r < kSlab; ++r)
        if (r >= r0 && r < r1) v[row_at(r) + tid] = value_of(h[r / 2] >> (16 * (r & 1)) & 0xFFFFu, (w >> nib(r)) & 15u);
}

// ---- attention -----------------------------------------------------------------------------------------------

typedef _Float16 fh2 __attribute__((ext_vector_type(2)));

// A 32-bit constant in a VGPR: a VOP3 instruction takes no literal and one SGPR at most, so (a & m) | b with two constants is one
// instruction only where they are in VGPRs.
__device__ __forceinline__ uint32_t in_vgpr(uint32_t c) {
    uint32_t r;
    asm("v_mov_b32 %0, %1" : "=v"(r) : "i"(c));
    return r;
}
// A code c in the low bits of the f16 1024 is 1024 + c, one in bits 4 .. 7 of the f16 64 is 64 + c: the first and second nibble of a
// register's halves become such pairs in one instruction. Less 1024 + z or 64 + z, and times the scale, both are exact.
__device__ __forceinline__ fh2 plus_1024(uint32_t w) { return __builtin_bit_cast(fh2, (w & in_vgpr(0x000F000Fu)) | in_vgpr(0x64006400u)); }
__device__ __forceinline__ fh2 plus_64(uint32_t w) { return __builtin_bit_cast(fh2, (w & in_vgpr(0x00F000F0u)) | in_vgpr(0x54005400u)); }

// A pair of headers' scales and zero points, in both forms.
__device__ __forceinline__ fh2 scales2(uint32_t h) { return __builtin_bit_cast(fh2, h & 0xFFF0FFF0u); }
__device__ __forceinline__ fh2 zeros2(uint32_t h, bool second) { return second ? plus_64(h << 4) : plus_1024(h); }

// The eight values of a word: elements 2 i, 2 i + 1 with scales d[i] and zero points z[i], of the second form for odd i.
__device__ __forceinline__ fh8 decode8(uint32_t w, const fh2 (&d)[4], const fh2 (&z)[4]) {
    fh8 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t x = i < 2 ? w : w >> 8;
        const fh2 v = ((i % 2 == 0 ? plus_1024(x) : plus_64(x)) - z[i]) * d[i];
        r[2 * i] = v[0];
        r[2 * i + 1] = v[1];
    }
    return r;
}
// All of them with the low (or high) header of a pair.
template <bool HIGH>
__device__ __forceinline__ fh8 decode8_one(uint32_t w, uint32_t h) {
    const fh2 d = scales2(h), z0 = zeros2(h, false), z1 = zeros2(h, true);
    const fh2 dd{d[HIGH], d[HIGH]}, a{z0[HIGH], z0[HIGH]}, b{z1[HIGH], z1[HIGH]};
    const fh2 ds[4] = {dd, dd, dd, dd}, zs[4] = {a, b, a, b};
    return decode8(w, ds, zs);
}

// N words (16 B aligned where N allows it) as N registers.
template <int N>
__device__ __forceinline__ void ld_words(const uint8_t *p, uint32_t (&w)[N]) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            const uint4 v = reinterpret_cast<const uint4 *>(p)[i];
            w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
        }
    } else if constexpr (N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            const uint2 v = reinterpret_cast<const uint2 *>(p)[i];
            w[2 * i] = v.x, w[2 * i + 1] = v.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = reinterpret_cast<const uint32_t *>(p)[i];
    }
}
// U headers (two bytes each) as pairs.
template <int U>
__device__ __forceinline__ void ld_heads(const uint8_t *p, uint32_t (&h)[(U + 1) / 2]) {
    if constexpr (U % 2 == 0) {
        ld_words<U / 2>(p, h);
    } else {
#pragma unroll
        for (int i = 0; i < (U + 1) / 2; ++i)
            h[i] = reinterpret_cast<const uint16_t *>(p)[2 * i] |
                   (2 * i + 1 < U ? static_cast<uint32_t>(reinterpret_cast<const uint16_t *>(p)[2 * i + 1]) << 16 : 0u);
    }
}

// Where the words and the headers of a slab begin: the same for K and V, whose slabs have the same sizes.
struct SlabAt {
    size_t words, heads;
    bool bad;
};
template <int U, bool PAGED>
__device__ __forceinline__ SlabAt slab_at(const Map4 &M, int slot, int kvh, int slab) {
    const Place p = place<PAGED>(M, slot, kvh, slab);
    return SlabAt{p.at + static_cast<size_t>(p.slab) * (128 * U), p.at + static_cast<size_t>(M.spp) * (128 * U) + static_cast<size_t>(p.slab) * (16 * U),
                  p.bad};
}

// Operand layout of v_mfma_f32_16x16x32_f16: lane l = (c = l & 15, g = l >> 4) gives row c of A and column c of B at the same eight
// k slots (g, j); the result has rows 4 g + r, column c. Over a block of 32 keys:
//  - S^T of key half h: A row c is key 8 (c >> 2) + 4 h + (c & 3), dims 32 u + 8 g + j (one K word); lane (c, g) ends with the
//    scores of keys 8 g + 4 h + r of query vector c.
//  - O^T += V^T P^T: k slot (g, j) is key 8 g + j, so B is the lane's own eight weights in order and A, dims 16 b + c of V^T at
//    positions 8 g .. 8 g + 7, is one V word of slab g.

// The lane's query vector (column c, dims 32 u + 8 g + j) as B operands: times a power of two that brings its largest element near
// 2^14, as f16 pairs hi + lo (22 significant bits). Returns the factor that takes a product back and into base-2 units of the
// softmax, log2(e) / sqrt(hd) over that power. 230 instructions: a short context's workgroup runs this once for a block or two.
__device__ __forceinline__ float max3_abs(float m, float a, float b) {
    asm("v_max3_f32 %0, %1, |%2|, |%3|" : "=v"(m) : "v"(m), "v"(a), "v"(b));
    return m;
}
template <int U>
__device__ __forceinline__ float load_query(const float *qrow, fh8 (&qh)[U], fh8 (&ql)[U]) {
    const int g = (threadIdx.x & 63) >> 4;
    float x[U][8], amax = 0.0f;
#pragma unroll
    for (int u = 0; u < U; ++u) __builtin_memcpy(x[u], qrow + 32 * u + 8 * g, 32);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < 8; j += 2) amax = max3_abs(amax, x[u][j], x[u][j + 1]);
    amax = xor32_max(xor16_max(amax));
    // amax = f 2^ex, f in [0.5, 1). Capped at 2^126, so that the power and its inverse are finite for the smallest queries.
    const int ex = amax > 0.0f && amax <= 3.0e38f ? __builtin_amdgcn_frexp_expf(amax) : 0, e2 = 14 - ex < 126 ? 14 - ex : 126;
    const float up = ldexpf(1.0f, e2);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            _Float16 hi, lo;
            split_h(x[u][j] * up, hi, lo);
            qh[u][j] = hi;
            ql[u][j] = lo;
        }
    return ldexpf(1.44269504088896341f / sqrtf(32.0f * U), -e2);
}

// Softmax step over a block's products s[h][r] (key kb + 8 g + 4 h + r; keys outside [qs, qe) are masked), which times `unit` are
// scores in base-2 units: new running maximum and sum, O rescaled where the maximum moved, the weights as an f16 pair (the first
// half rounded towards zero, the second the rest: 22 significant bits). The sum is of the weights before they are split.
template <int U>
__device__ __forceinline__ void softmax_step(const fa4 (&s)[2], float unit, int kb, int qs, int qe, float &m, float &l, fa4 (&o)[2 * U],
                                             fh8 &ph, fh8 &pl) {
    const int g = (threadIdx.x & 63) >> 4;
    float v[8], bm = -INFINITY;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = s[j >> 2][j & 3];
    if (__any(kb < qs || kb + 32 > qe)) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int p = kb + 8 * g + j;
            v[j] = p >= qs && p < qe ? v[j] : -INFINITY;
        }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) bm = fmaxf(bm, v[j]);
    bm = xor32_max(xor16_max(bm)) * unit;
    const float mn = fmaxf(m, bm), ms = mn == -INFINITY ? 0.0f : mn;  // ms: exp2(-inf - ms) is 0 also before any key
    const float alpha = __builtin_amdgcn_exp2f(m - ms);
    float ps = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        const float a = __builtin_amdgcn_exp2f(fmaf(v[j], unit, -ms)), b = __builtin_amdgcn_exp2f(fmaf(v[j + 1], unit, -ms));
        ps += a;
        ps += b;
        const fh2 hi = __builtin_bit_cast(fh2, __builtin_amdgcn_cvt_pkrtz(a, b));
        const fh2 lo = __builtin_bit_cast(fh2, __builtin_amdgcn_cvt_pkrtz(a - static_cast<float>(hi[0]), b - static_cast<float>(hi[1])));
        ph[j] = hi[0], ph[j + 1] = hi[1];
        pl[j] = lo[0], pl[j + 1] = lo[1];
    }
    ps = xor32_add(xor16_add(ps));
    l = l * alpha + ps;
    m = mn;
    if (__any(alpha != 1.0f)) {
#pragma unroll
        for (int b = 0; b < 2 * U; ++b) o[b] *= alpha;
    }
}

// How a pass's contexts are cut: chunks of `len` keys (a multiple of 128) from each segment's first key rounded down to 32, all
// segments' chunks in one list; segment i's begin at first[i], its partial results at base[i].
struct Cuts {
    int len, total, most;  // most: chunks of a segment
    int first[VQ_MAX_SEGMENTS], base[VQ_MAX_SEGMENTS];
};
// First key that any row of a segment sees, rounded down to a block.
__host__ __device__ __forceinline__ int first_key(const Seg &s, int window) {
    return window > 0 && s.pos0 + 1 > window ? (s.pos0 + 1 - window) & ~31 : 0;
}

// The keys that query row t of a segment sees.
struct Sees {
    int from, to;
};
__device__ __forceinline__ Sees sees(const Seg &s, int t, int bidirectional, int window) {
    const int end = s.pos0 + 1 + t;
    return Sees{window > 0 && end > window ? end - window : 0, bidirectional ? s.pos0 + s.rows : end};
}

// A workgroup's results for up to 16 query vectors: W waves' sums (each wave's [16][HD] in `sums`, maxima and totals in sm, sl) meet
// in wave order; written out, or as the chunk's unnormalised part where the context is cut.
template <int HD, int W>
__device__ __forceinline__ void meet(const float *sums, const float (&sm)[W][16], const float (&sl)[W][16], int threads, int tid, int j0,
                                     int nvec, int G, int kvh, int heads, int row0, float *out, float *part, float *pml, int n, int ci) {
    for (int e = tid; e < 16 * (HD / 4); e += threads) {
        const int c = e / (HD / 4), d4 = 4 * (e - c * (HD / 4)), j = j0 + c;
        if (j >= nvec) continue;
        const int t = j / G, h = kvh * G + j - t * G;
        float mx = sm[0][c];
#pragma unroll
        for (int w = 1; w < W; ++w) mx = fmaxf(mx, sm[w][c]);
        float L = 0.0f;
        float4 acc{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float f = sm[w][c] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(sm[w][c] - mx);
            L = fmaf(sl[w][c], f, L);
            const float4 p = *reinterpret_cast<const float4 *>(sums + (w * 16 + c) * HD + d4);
            acc.x = fmaf(p.x, f, acc.x);
            acc.y = fmaf(p.y, f, acc.y);
            acc.z = fmaf(p.z, f, acc.z);
            acc.w = fmaf(p.w, f, acc.w);
        }
        if (n == 1) {
            const float inv = L > 0.0f ? 1.0f / L : 0.0f;
            const float4 r{acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
            __builtin_memcpy(out + (static_cast<size_t>(row0 + t) * heads + h) * HD + d4, &r, 16);
        } else {
            const size_t at = (static_cast<size_t>(t) * heads + h) * n + ci;
            *reinterpret_cast<float4 *>(part + at * HD + d4) = acc;
            if (d4 == 0) pml[2 * at] = mx, pml[2 * at + 1] = L;
        }
    }
}

// A block's codes and headers in registers. Lane (c, g) has K rows 8 (c >> 2) + 4 h + (c & 3) at its dims, the V words of its dims in
// slab g, and of slab g the headers of group c.
template <int U>
struct Raw4 {
    uint32_t k[2][U], kh[2][(U + 1) / 2], v[2 * U];
    uint4 vh;
};
template <int U>
__device__ __forceinline__ void issue_k(const uint8_t *__restrict__ kc, const SlabAt &at, Raw4<U> &r) {
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int row = 4 * h + (c & 3);
        ld_words<U>(kc + at.words + row * (16 * U) + g * (4 * U), r.k[h]);
        ld_heads<U>(kc + at.heads + row * (2 * U), r.kh[h]);
    }
    if (at.bad) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < (U + 1) / 2; ++i) r.kh[h][i] = kNanHeader | kNanHeader << 16;
    }
}
template <int U>
__device__ __forceinline__ void issue_v(const uint8_t *__restrict__ vc, const SlabAt &at, Raw4<U> &r) {
    const int c = threadIdx.x & 15;
    constexpr int W = U % 2 == 0 ? 4 : 2;
#pragma unroll
    for (int i = 0; i < 2 * U / W; ++i) {
        uint32_t w[W];
        ld_words<W>(vc + at.words + (16 * i + c) * (4 * W), w);
#pragma unroll
        for (int k = 0; k < W; ++k) r.v[W * i + k] = w[k];
    }
    r.vh = *reinterpret_cast<const uint4 *>(vc + at.heads + 16 * min(c, U - 1));
}

template <int U>
__device__ __forceinline__ void scores(const Raw4<U> &r, const fh8 (&qh)[U], const fh8 (&ql)[U], fa4 (&s)[2]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        fa4 a0{0.f, 0.f, 0.f, 0.f}, a1{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const fh8 a = u % 2 == 0 ? decode8_one<false>(r.k[h][u], r.kh[h][u / 2]) : decode8_one<true>(r.k[h][u], r.kh[h][u / 2]);
            a0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qh[u], a0, 0, 0, 0);
            a1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ql[u], a1, 0, 0, 0);
        }
        s[h] = a0 + a1;
    }
}
// O^T += V^T P^T. Every lane of a row of 16 needs the headers of all groups of its slab: lane c takes group c's apart and the others
// read them from LDS (`hl`, the wave's own: [slab][group] scales, zero points; moving them by DPP costs 64 instructions a block of
// the kind that bounds this kernel).
template <int U>
constexpr int head_words = 4 * (8 * U + 8);
template <int U>
__device__ __forceinline__ void add_values(const Raw4<U> &r, const fh8 &ph, const fh8 &pl, uint32_t *hl, fa4 (&o)[2 * U]) {
    const int lane = threadIdx.x & 63, c = lane & 15;
    uint32_t *mine = hl + (lane >> 4) * (8 * U + 8);
    if (c < U) {
        const uint32_t raw[4] = {r.vh.x, r.vh.y, r.vh.z, r.vh.w};
        uint32_t d[4], z[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) d[i] = raw[i] & 0xFFF0FFF0u, z[i] = __builtin_bit_cast(uint32_t, zeros2(raw[i], i % 2 != 0));
        *reinterpret_cast<uint4 *>(mine + 8 * c) = uint4{d[0], d[1], d[2], d[3]};
        *reinterpret_cast<uint4 *>(mine + 8 * c + 4) = uint4{z[0], z[1], z[2], z[3]};
    }
    // A wave's LDS operations complete in order; the fence keeps the compiler from moving the reads above the writes.
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint4 dw = *reinterpret_cast<const uint4 *>(mine + 8 * u), zw = *reinterpret_cast<const uint4 *>(mine + 8 * u + 4);
        const fh2 d[4] = {__builtin_bit_cast(fh2, dw.x), __builtin_bit_cast(fh2, dw.y), __builtin_bit_cast(fh2, dw.z), __builtin_bit_cast(fh2, dw.w)};
        const fh2 z[4] = {__builtin_bit_cast(fh2, zw.x), __builtin_bit_cast(fh2, zw.y), __builtin_bit_cast(fh2, zw.z), __builtin_bit_cast(fh2, zw.w)};
#pragma unroll
        for (int b = 2 * u; b < 2 * u + 2; ++b) {
            const fh8 a = decode8(r.v[b], d, z);
            o[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ph, o[b], 0, 0, 0);
            o[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, pl, o[b], 0, 0, 0);
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");  // every lane has read before the next block's writes
    __builtin_amdgcn_wave_barrier();
}

// Decode and verify passes: one workgroup per (chunk, kv head, 16 query vectors); vector j of a segment is (row j / G, head j % G of
// the kv head's group). Its four waves take the chunk's 32-key blocks in turn, straight from the cache into registers, decoded
// there into MFMA operands, with an online softmax each; they meet in wave order.
template <int U, bool PAGED>
__global__ __launch_bounds__(256, 2) void attention4_split_kernel(const float *__restrict__ q, const uint8_t *__restrict__ kc,
                                                                  const uint8_t *__restrict__ vc, float *__restrict__ part,
                                                                  float *__restrict__ pml, float *__restrict__ out, SegTable T, Map4 M,
                                                                  Cuts C, int heads, int bidirectional, int window) {
    constexpr int HD = 32 * U;
    __shared__ __align__(16) float sums[4 * 16 * HD];
    __shared__ float sm[4][16], sl[4][16];
    __shared__ __align__(16) uint32_t vheads[4][head_words<U>];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
    const int kvh = blockIdx.x % M.kv_heads, list = blockIdx.x / M.kv_heads;
    const int bases = C.base[lane];
    const Found found = find_segment(T, C.first, C.total, list);
    const Seg s = found.s;
    const int ci = list - found.first, n = found.next - found.first;
    const int G = heads / M.kv_heads, nvec = s.rows * G, j0 = blockIdx.y * 16;
    if (j0 >= nvec) return;
    const int j = min(j0 + c, nvec - 1), t = j / G, h = kvh * G + j - t * G;  // vectors past the last repeat it; not written
    const Sees see = sees(s, t, bidirectional, window);
    const int k_lo = first_key(s, window) + ci * C.len, k_hi = min(k_lo + C.len, s.pos0 + s.rows);
    const int qe = min(see.to, k_hi), last = (k_hi - 1) / kSlab;
    float m = -INFINITY, l = 0.0f;
    fa4 o[2 * U];
#pragma unroll
    for (int b = 0; b < 2 * U; ++b) o[b] = fa4{0.f, 0.f, 0.f, 0.f};
    // Lane (c, g) takes K rows of slab c >> 2 and V words of slab g of a block; slabs past the last key's read that one's (masked).
    auto places = [&](int kb, SlabAt &ks, SlabAt &vs) {
        ks = slab_at<U, PAGED>(M, s.slot, kvh, min(kb / kSlab + (c >> 2), last));
        vs = slab_at<U, PAGED>(M, s.slot, kvh, min(kb / kSlab + g, last));
    };
    int kb = k_lo + 32 * wv;
    Raw4<U> r;
    SlabAt ks, vs;
    if (kb < k_hi) {
        places(kb, ks, vs);
        issue_k<U>(kc, ks, r);
        issue_v<U>(vc, vs, r);
    }
    fh8 qh[U], ql[U];
    const float unit = load_query<U>(q + (static_cast<size_t>(s.row0 + t) * heads + h) * HD, qh, ql);
    for (; kb < k_hi; kb += 128) {
        // The next block's K and V come into the registers that this block's have left.
        const bool more = kb + 128 < k_hi;
        if (more) places(kb + 128, ks, vs);
        fa4 sc[2];
        scores<U>(r, qh, ql, sc);
        if (more) issue_k<U>(kc, ks, r);
        fh8 ph, pl;
        softmax_step<U>(sc, unit, kb, see.from, qe, m, l, o, ph, pl);
        add_values<U>(r, ph, pl, vheads[wv], o);
        if (more) issue_v<U>(vc, vs, r);
    }
    float *ow = sums + wv * 16 * HD;
    if (j0 + c < nvec) {
#pragma unroll
        for (int b = 0; b < 2 * U; ++b) *reinterpret_cast<fa4 *>(ow + c * HD + 16 * b + 4 * g) = o[b];
        if (g == 0) sm[wv][c] = m, sl[wv][c] = l;
    }
    __syncthreads();
    const size_t base = from_lane(bases, found.index);
    meet<HD, 4>(sums, sm, sl, 256, threadIdx.x, j0, nvec, G, kvh, heads, s.row0, out, part + base * HD, pml + 2 * base, n, ci);
}

// The same for hd 128 and 256, whose waves are few (hd 256: 2 per SIMD, for the registers of O and q): the blocks come to LDS by DMA,
// kSlots of them for each wave, so that the loads of a whole block are in flight while another one is computed with, and no
// registers are spent on them. A slot: K pieces of 16 bytes in the order that lanes read them, V pieces, headers (lanes 0 .. 31 bring
// K's, row after row, the others V's). Page ids and addresses are wave-uniform and come by scalar loads: the only vector memory
// operations of the loop are the DMA's, which the waits count.
template <int U>
struct Ring {
    static constexpr int kSlots = U == 8 ? 2 : 3, kLoads = U + 1, kBytes = 1024 * kLoads;
};
// Where a block's slabs are. MODE: how many of the four slabs one look at the page table gives (4: pages of whole blocks, 2: of
// pairs of slabs), 0: a contiguous cache.
template <int MODE>
struct Slab4 {
    static constexpr int N = MODE == 0 ? 1 : 4 / MODE;
    size_t block[N];  // first byte of the cache block
    uint32_t slab[N];
    uint32_t bad;  // a bit for each slab whose page is none
};
template <int MODE>
__device__ __forceinline__ Slab4<MODE> look_up(const Map4 &M, int slot, int kvh, int kb, int last) {
    Slab4<MODE> r;
    r.bad = 0;
    if constexpr (MODE == 0) {
        r.block[0] = static_cast<size_t>(kvh) * M.bytes;
        r.slab[0] = kb / kSlab;
    } else {
        const auto *pt = (const __attribute__((address_space(4))) int32_t *)(M.pt) + static_cast<size_t>(slot) * M.pps;
#pragma unroll
        for (int i = 0; i < Slab4<MODE>::N; ++i) {
            // Slabs past the last key's: that one's page is read instead (their keys are masked).
            const uint32_t slab = min(kb / kSlab + MODE * i, last & ~(MODE - 1));
            const uint32_t p = static_cast<uint32_t>((static_cast<uint64_t>(slab) * M.mul) >> M.shift);
            const int pg = pt[p];
            const bool none = static_cast<uint32_t>(pg) >= static_cast<uint32_t>(M.pages);
            r.bad |= none ? ((1u << MODE) - 1) << (MODE * i) : 0u;
            r.block[i] = (static_cast<size_t>(none ? 0 : pg) * M.kv_heads + kvh) * M.bytes;
            r.slab[i] = slab - p * M.spp;
            // Opaque from here, or a lane's choice between two of them becomes one between addresses, in memory.
            asm("" : "+s"(r.block[i]), "+s"(r.slab[i]));
        }
    }
    return r;
}
// Slab i of the block, as a lane's own choice: (first byte of its block, slab in it).
template <int MODE>
__device__ __forceinline__ void choose(const Slab4<MODE> &s, int i, int last, size_t &block, uint32_t &slab) {
    if constexpr (MODE == 0) {
        block = s.block[0], slab = min(s.slab[0] + i, static_cast<uint32_t>(last));
    } else if constexpr (MODE == 4) {
        block = s.block[0], slab = s.slab[0] + i;
    } else {
        block = i & 2 ? s.block[1] : s.block[0], slab = (i & 2 ? s.slab[1] : s.slab[0]) + (i & 1);
    }
}
// 64 lanes x 16 bytes from each lane's own address to LDS at (wave-uniform) dst, in lane order.
__device__ __forceinline__ void dma16(const uint8_t *from, uint8_t *dst) {
    const uint32_t at = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(vq::lds_addr(dst))));
    asm volatile("s_mov_b32 m0, %1\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "s"(at), "v"(dst) : "memory", "m0");
}
// Operand row c's pieces (eight of 16 bytes, two rows to the 64 banks) change places by this.
__device__ __forceinline__ int k_swizzle(int c) { return c >> 1 & 7; }
template <int U, int MODE>
__device__ __forceinline__ void issue_dma(const uint8_t *kc, const uint8_t *vc, const Map4 &M, const Slab4<MODE> &at, int last, uint8_t *slot) {
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4, piece = min(lane & 31, 4 * U - 1);
    size_t block;
    uint32_t slab;
    // K, hd 256: a load brings eight rows of 128 bytes whole, operand rows 8 x + r (x: the load's half of them), pieces swizzled so that
    // the operand's reads spread over the banks. hd 128: a load brings the half's 16 rows of 64 bytes in operand order.
    const int r = U == 8 ? lane >> 3 : c, s = U == 8 ? lane & 7 : g;
    const uint8_t *k[2];
#pragma unroll
    for (int x = 0; x < U / 4; ++x) {
        choose<MODE>(at, U == 8 ? 2 * x + (r >> 2) : r >> 2, last, block, slab);
        k[x] = kc + block + static_cast<size_t>(slab) * (128 * U) + ((r & 3) * (16 * U) + (U == 8 ? s ^ k_swizzle(8 * x + r) : s) * 16);
    }
    choose<MODE>(at, g, last, block, slab);
    const uint8_t *v = vc + block + static_cast<size_t>(slab) * (128 * U) + c * 16;
    choose<MODE>(at, piece / U, last, block, slab);
    const uint8_t *h = (lane < 32 ? kc : vc) + block + static_cast<size_t>(M.spp) * (128 * U) + static_cast<size_t>(slab) * (16 * U) + piece % U * 16;
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int x = 0; x < U / 4; ++x) dma16(k[x] + half * (64 * U), slot + 1024 * (half * (U / 4) + x));
#pragma unroll
    for (int i = 0; i < U / 2; ++i) dma16(v + 256 * i, slot + 1024 * (U / 2 + i));
    dma16(h, slot + 1024 * U);
}
template <int U>
__device__ __forceinline__ void read_k(const uint8_t *slot, Raw4<U> &r) {
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int i = 0; i < U / 4; ++i) {
            const int at = U == 8 ? 128 * c + 16 * ((2 * g + i) ^ k_swizzle(c)) : 16 * lane;
            const uint4 w = *reinterpret_cast<const uint4 *>(slot + 256 * U * half + at);
            r.k[half][4 * i] = w.x, r.k[half][4 * i + 1] = w.y, r.k[half][4 * i + 2] = w.z, r.k[half][4 * i + 3] = w.w;
        }
        ld_words<U / 2>(slot + 1024 * U + (8 * (c >> 2) + 4 * half + (c & 3)) * (2 * U), r.kh[half]);
    }
}
template <int U>
__device__ __forceinline__ void read_v(const uint8_t *slot, Raw4<U> &r) {
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
#pragma unroll
    for (int i = 0; i < U / 2; ++i) {
        const uint4 w = *reinterpret_cast<const uint4 *>(slot + 1024 * (U / 2 + i) + 16 * lane);
        r.v[4 * i] = w.x, r.v[4 * i + 1] = w.y, r.v[4 * i + 2] = w.z, r.v[4 * i + 3] = w.w;
    }
    r.vh = *reinterpret_cast<const uint4 *>(slot + 1024 * U + 512 + 16 * (g * U + min(c, U - 1)));
}

template <int U, int MODE>
__global__ __launch_bounds__(256, 2) void attention4_stream_kernel(const float *__restrict__ q, const uint8_t *__restrict__ kc,
                                                                   const uint8_t *__restrict__ vc, float *__restrict__ part,
                                                                   float *__restrict__ pml, float *__restrict__ out, SegTable T, Map4 M,
                                                                   Cuts C, int heads, int bidirectional, int window) {
    constexpr int HD = 32 * U, SLOTS = Ring<U>::kSlots, BYTES = Ring<U>::kBytes, LOADS = Ring<U>::kLoads;
    static_assert(SLOTS * BYTES >= 16 * HD * 4, "the waves' sums go where their slots were");
    __shared__ __align__(16) uint8_t ring[4][SLOTS * BYTES];
    __shared__ float sm[4][16], sl[4][16];
    __shared__ __align__(16) uint32_t vheads[4][head_words<U>];
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
    const int kvh = blockIdx.x % M.kv_heads, list = blockIdx.x / M.kv_heads;
    const int bases = C.base[lane];
    const Found found = find_segment(T, C.first, C.total, list);
    const Seg s = found.s;
    const int ci = list - found.first, n = found.next - found.first;
    const int G = heads / M.kv_heads, nvec = s.rows * G, j0 = blockIdx.y * 16;
    if (j0 >= nvec) return;
    const int k_lo = first_key(s, window) + ci * C.len, k_hi = min(k_lo + C.len, s.pos0 + s.rows), last = (k_hi - 1) / kSlab;
    int kb = k_lo + 32 * wv;
    uint8_t *const mine = ring[wv];
    auto fetch = [&](int block, int slot) {
        const Slab4<MODE> at = look_up<MODE>(M, s.slot, kvh, block, last);
        issue_dma<U, MODE>(kc, vc, M, at, last, mine + slot * BYTES);
        return at.bad;
    };
    uint32_t bad[SLOTS] = {};
    if (kb < k_hi) bad[0] = fetch(kb, 0);
    const int j = min(j0 + c, nvec - 1), t = j / G, h = kvh * G + j - t * G;  // vectors past the last repeat it; not written
    const Sees see = sees(s, t, bidirectional, window);
    const int qe = min(see.to, k_hi);
    fh8 qh[U], ql[U];
    const float unit = load_query<U>(q + (static_cast<size_t>(s.row0 + t) * heads + h) * HD, qh, ql);
    float m = -INFINITY, l = 0.0f;
    fa4 o[2 * U];
#pragma unroll
    for (int b = 0; b < 2 * U; ++b) o[b] = fa4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 1; i < SLOTS; ++i)
        if (kb + 128 * i < k_hi) bad[i] = fetch(kb + 128 * i, i);
    while (kb < k_hi) {
#pragma unroll
        for (int slot = 0; slot < SLOTS; ++slot) {
            if (kb >= k_hi) break;
            // A SIMD serves its older wave first, which left the younger one to finish alone, 11 of 40 us (131071 keys). A wave
            // that nears its end steps back, so that they finish together.
            const int left = (k_hi - 1 - kb) / 128;
            if (left >= 3) __builtin_amdgcn_s_setprio(3);
            else if (left == 2) __builtin_amdgcn_s_setprio(2);
            else if (left == 1) __builtin_amdgcn_s_setprio(1);
            else __builtin_amdgcn_s_setprio(0);
            // Landed: all but the loads of the blocks behind this one.
            const int behind = min(left, SLOTS - 1);
            if (behind == 0) vq::wait_vm<0>();
            else if (behind == 1) vq::wait_vm<LOADS>();
            else vq::wait_vm<2 * LOADS>();
            Raw4<U> r;
            uint8_t *const from = mine + slot * BYTES;
            read_k<U>(from, r);
            if (MODE != 0 && bad[slot] != 0 && (bad[slot] >> (c >> 2) & 1)) {
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int x = 0; x < U / 2; ++x) r.kh[half][x] = kNanHeader | kNanHeader << 16;
            }
            fa4 sc[2];
            scores<U>(r, qh, ql, sc);
            fh8 ph, pl;
            softmax_step<U>(sc, unit, kb, see.from, qe, m, l, o, ph, pl);
            read_v<U>(from, r);
            add_values<U>(r, ph, pl, vheads[wv], o);
            vq::wait_lgkm0();  // the slot has been read
            if (kb + 128 * SLOTS < k_hi) bad[slot] = fetch(kb + 128 * SLOTS, slot);
            kb += 128;
        }
    }
    __syncthreads();  // every slot of every wave has been read
    float *sums = reinterpret_cast<float *>(&ring[0][0]), *ow = sums + wv * 16 * HD;
    if (j0 + c < nvec) {
#pragma unroll
        for (int b = 0; b < 2 * U; ++b) *reinterpret_cast<fa4 *>(ow + c * HD + 16 * b + 4 * g) = o[b];
        if (g == 0) sm[wv][c] = m, sl[wv][c] = l;
    }
    __syncthreads();
    const size_t base = from_lane(bases, found.index);
    meet<HD, 4>(sums, sm, sl, 256, threadIdx.x, j0, nvec, G, kvh, heads, s.row0, out, part + base * HD, pml + 2 * base, n, ci);
}

// out = sum_c 2^(m_c - M) o_c / sum_c 2^(m_c - M) l_c over a row's chunks, for segments of more than one. It is latency that this
// kernel spends, so a workgroup takes 64 dims of a (row, head) (32 where hd is no multiple of 64), a thread four dims of every 16th
// (32nd) chunk, four of them in flight, under a running maximum; the 16 (32) sums meet in order. 24 rows of 128 chunks, hd 256: 4 us;
// one workgroup of four waves for a row took 11.
template <int HD>
__global__ __launch_bounds__(256) void attention4_merge_kernel(const float *__restrict__ part, const float *__restrict__ pml,
                                                               float *__restrict__ out, SegTable T, Cuts C, Starts R, int heads) {
    constexpr int Q = HD % 64 == 0 ? 16 : 8, GROUPS = 256 / Q;
    __shared__ float sm[GROUPS], sl[GROUPS];
    __shared__ float4 sacc[GROUPS][Q];
    const int tid = threadIdx.x, lane = tid & 63, grp = tid / Q, quad = tid - grp * Q;
    const int row = blockIdx.x / heads, h = blockIdx.x - row * heads, d = 4 * (Q * blockIdx.y + quad);
    const int chunks = C.first[lane], bases = C.base[lane];
    const Found found = find_segment(T, R.first, R.total, row);
    const Seg s = found.s;
    const int t = row - found.first, i = found.index;
    const int n = (i + 1 < T.n ? from_lane(chunks, i + 1 < 64 ? i + 1 : 63) : C.total) - from_lane(chunks, i);
    if (n == 1) return;
    const size_t at = static_cast<size_t>(from_lane(bases, i)) + (static_cast<size_t>(t) * heads + h) * n;
    const float *ml = pml + 2 * at;
    float m = -INFINITY, L = 0.0f;
    float4 acc{0.f, 0.f, 0.f, 0.f};
    auto scale = [](float x, float to) { return x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(x - to); };
    for (int c0 = grp; c0 < n; c0 += 4 * GROUPS) {
        float4 p[4];
        float mc[4], lc[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int c = c0 + GROUPS * k < n ? c0 + GROUPS * k : c0;
            p[k] = *reinterpret_cast<const float4 *>(part + (at + c) * HD + d);
            mc[k] = c0 + GROUPS * k < n ? ml[2 * c] : -INFINITY;
            lc[k] = ml[2 * c + 1];
        }
        const float mn = fmaxf(fmaxf(m, fmaxf(mc[0], mc[1])), fmaxf(mc[2], mc[3])), f0 = scale(m, mn);
        m = mn;
        L *= f0;
        acc = float4{acc.x * f0, acc.y * f0, acc.z * f0, acc.w * f0};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (c0 + GROUPS * k >= n) break;
            const float f = scale(mc[k], mn);
            L = fmaf(lc[k], f, L);
            acc.x = fmaf(p[k].x, f, acc.x);
            acc.y = fmaf(p[k].y, f, acc.y);
            acc.z = fmaf(p[k].z, f, acc.z);
            acc.w = fmaf(p[k].w, f, acc.w);
        }
    }
    sacc[grp][quad] = acc;
    if (quad == 0) sm[grp] = m, sl[grp] = L;
    __syncthreads();
    if (tid >= Q) return;
    m = sm[0];
#pragma unroll
    for (int w = 1; w < GROUPS; ++w) m = fmaxf(m, sm[w]);
    L = 0.0f;
    acc = float4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < GROUPS; ++w) {
        const float4 a = sacc[w][quad];
        const float f = scale(sm[w], m);
        L = fmaf(sl[w], f, L);
        acc.x = fmaf(a.x, f, acc.x);
        acc.y = fmaf(a.y, f, acc.y);
        acc.z = fmaf(a.z, f, acc.z);
        acc.w = fmaf(a.w, f, acc.w);
    }
    const float inv = L > 0.0f ? 1.0f / L : 0.0f;
    const float4 r{acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
    __builtin_memcpy(out + (static_cast<size_t>(s.row0 + t) * heads + h) * HD + d, &r, 16);
}

// Prompt passes, and any pass without a workspace: a workgroup of NW waves takes NW / 2 tiles of 16 query vectors of a kv head, two
// waves each, one for the 32-key blocks of each parity (blocks at multiples of 32 keys whatever the rows, so a row's sums do not
// depend on the others); their sums meet at the end. Per step of 64 keys the threads load the next step's words, the waves consume
// the present one from LDS, decoded once for all tiles: K rows of HD + 16 f16, V^T [dim][32 positions] with 16-byte pieces swizzled
// by (dim >> 2) & 3; the loaded words are decoded into the other LDS buffer: one barrier per step.
__device__ __forceinline__ int vt_at(int d, int octet) { return d * 32 + ((octet ^ ((d >> 2) & 3)) << 3); }

template <int U, bool PAGED, int NW>
__global__ __launch_bounds__(64 * NW, 2) void attention4_tiled_kernel(const float *__restrict__ q, const uint8_t *__restrict__ kc,
                                                                      const uint8_t *__restrict__ vc, float *__restrict__ out,
                                                                      SegTable T, Starts R, Map4 M, int heads, int bidirectional, int window) {
    constexpr int HD = 32 * U, LDK = HD + 16, TH = 64 * NW, TILES = NW / 2;
    constexpr int KW = U % 4 == 0 ? 4 : U % 2 == 0 ? 2 : 1, W = U % 2 == 0 ? 4 : 2;  // words of a K unit, of a V unit
    constexpr int KUN = 64 * 4 * (U / KW), VUN = 8 * 16 * (2 * U / W);               // units of a step
    constexpr int KN = (KUN + TH - 1) / TH, VN = (VUN + TH - 1) / TH;                // of a thread
    constexpr int KB = 32 * LDK, VB = HD * 32;                                       // f16 elements of a block
    constexpr int BUF = 2 * (KB + VB), MEET = TILES * 2 * 16 * HD * 2;               // f16 elements: a buffer, the sums at the end
    __shared__ __align__(16) _Float16 kv[2 * BUF > MEET ? 2 * BUF : MEET];
    __shared__ SlabAt slabs[2][8];
    __shared__ float sm[TILES][2][16], sl[TILES][2][16];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, c = lane & 15, g = lane >> 4, tile = wv >> 1, par = wv & 1;
    const int kvh = blockIdx.x % M.kv_heads, G = heads / M.kv_heads;
    // Workgroups take the kv heads in turn, the last rows, which see the most keys, first.
    const int group = R.total - 1 - blockIdx.x / M.kv_heads;
    const Found found = find_segment(T, R.first, R.total, group);
    const Seg s = found.s;
    const int tb = group - found.first;
    const int nvec = s.rows * G, first = tb * 16 * TILES, j0 = first + 16 * tile;
    const bool on = j0 < nvec;
    const int j = min(j0 + c, nvec - 1), t = j / G, h = kvh * G + j - t * G;
    const Sees see = sees(s, t, bidirectional, window), a = sees(s, first / G, bidirectional, window),
               z = sees(s, min(first + 16 * TILES - 1, nvec - 1) / G, bidirectional, window);
    const int k0 = a.from & ~63, k_hi = z.to, steps = (k_hi - k0 + 63) / 64, s0 = a.from / kSlab, s1 = (k_hi - 1) / kSlab;
    auto look = [&](int step) { return slab_at<U, PAGED>(M, s.slot, kvh, min(max((k0 + 64 * step) / kSlab + (tid & 7), s0), s1)); };
    if (tid < 16) slabs[tid >> 3][tid & 7] = look(tid >> 3);
    fh8 qh[U], ql[U];
    const float unit = load_query<U>(q + (static_cast<size_t>(s.row0 + t) * heads + h) * HD, qh, ql);
    __syncthreads();
    uint32_t rk[KN][KW], rkh[KN][KW == 4 ? 2 : 1], rv[VN][W];
    uint4 rvh[VN][W / 2];
    auto issue = [&](int step) {
        const SlabAt *sa = slabs[step & 1];
#pragma unroll
        for (int i = 0; i < KN; ++i) {  // unit: (key, word group of dims, run of KW words)
            const int unit = (tid + TH * i) % KUN, key = unit / (4 * (U / KW)), rest = unit % (4 * (U / KW)), g4 = rest / (U / KW), u0 = rest % (U / KW) * KW;
            const SlabAt &at = sa[key >> 3];
            ld_words<KW>(kc + at.words + (key & 7) * (16 * U) + g4 * (4 * U) + 4 * u0, rk[i]);
            const uint8_t *hp = kc + at.heads + (key & 7) * (2 * U) + 2 * u0;
            if constexpr (KW == 4) ld_words<2>(hp, rkh[i]);
            else if constexpr (KW == 2) ld_words<1>(hp, rkh[i]);
            else rkh[i][0] = *reinterpret_cast<const uint16_t *>(hp);
            if (at.bad)
#pragma unroll
                for (auto &x : rkh[i]) x = kNanHeader | kNanHeader << 16;
        }
#pragma unroll
        for (int i = 0; i < VN; ++i) {  // unit: (slab, run of W dim tiles, dim of a tile)
            const int unit = (tid + TH * i) % VUN, slab = unit / (16 * (2 * U / W)), rest = unit % (16 * (2 * U / W));
            const SlabAt &at = sa[slab];
            ld_words<W>(vc + at.words + rest * (4 * W), rv[i]);
#pragma unroll
            for (int k = 0; k < W / 2; ++k) rvh[i][k] = *reinterpret_cast<const uint4 *>(vc + at.heads + 16 * ((rest >> 4) * (W / 2) + k));
        }
    };
    auto stage = [&](int step) {
        _Float16 *buf = kv + (step & 1) * BUF;
#pragma unroll
        for (int i = 0; i < KN; ++i) {
            const int unit = tid + TH * i, key = unit / (4 * (U / KW)), rest = unit % (4 * (U / KW)), g4 = rest / (U / KW), u0 = rest % (U / KW) * KW;
            if (KUN % TH && unit >= KUN) break;
            const int row = 16 * ((key >> 2) & 1) + 4 * ((key >> 3) & 3) + (key & 3);  // of the block's S^T operand
            _Float16 *kd = buf + (key >> 5) * (KB + VB) + row * LDK + 32 * u0 + 8 * g4;
#pragma unroll
            for (int k = 0; k < KW; ++k) {
                const uint32_t h2 = rkh[i][k / 2];
                *reinterpret_cast<fh8 *>(kd + 32 * k) = k % 2 == 0 ? decode8_one<false>(rk[i][k], h2) : decode8_one<true>(rk[i][k], h2);
            }
        }
#pragma unroll
        for (int i = 0; i < VN; ++i) {
            const int unit = tid + TH * i, slab = unit / (16 * (2 * U / W)), rest = unit % (16 * (2 * U / W));
            if (VUN % TH && unit >= VUN) break;
            _Float16 *vd = buf + (slab >> 2) * (KB + VB) + KB;
#pragma unroll
            for (int k = 0; k < W; ++k) {
                const uint4 x = rvh[i][k / 2];
                const fh2 ds[4] = {scales2(x.x), scales2(x.y), scales2(x.z), scales2(x.w)};
                const fh2 zs[4] = {zeros2(x.x, false), zeros2(x.y, true), zeros2(x.z, false), zeros2(x.w, true)};
                *reinterpret_cast<fh8 *>(vd + vt_at(16 * ((rest >> 4) * W + k) + (rest & 15), slab & 3)) = decode8(rv[i][k], ds, zs);
            }
        }
    };
    issue(0);
    float m = -INFINITY, l = 0.0f;
    fa4 o[2 * U];
#pragma unroll
    for (int b = 0; b < 2 * U; ++b) o[b] = fa4{0.f, 0.f, 0.f, 0.f};
    stage(0);
    __syncthreads();
    for (int step = 0; step < steps; ++step) {
        const bool more = step + 1 < steps;
        SlabAt next{};
        if (tid < 8) next = look(step + 2);
        if (more) issue(step + 1);
        const int kb = k0 + 64 * step + 32 * par;
        if (on && kb < k_hi) {
            const _Float16 *ks = kv + (step & 1) * BUF + par * (KB + VB), *vt = ks + KB;
            fa4 sc[2];
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
                fa4 a0{0.f, 0.f, 0.f, 0.f}, a1{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const fh8 k8 = *reinterpret_cast<const fh8 *>(ks + (16 * hh + c) * LDK + 8 * g + 32 * u);
                    a0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(k8, qh[u], a0, 0, 0, 0);
                    a1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(k8, ql[u], a1, 0, 0, 0);
                }
                sc[hh] = a0 + a1;
            }
            fh8 ph, pl;
            softmax_step<U>(sc, unit, kb, see.from, see.to, m, l, o, ph, pl);
#pragma unroll
            for (int b = 0; b < 2 * U; ++b) {
                const fh8 v8 = *reinterpret_cast<const fh8 *>(vt + vt_at(16 * b + c, g));
                o[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v8, ph, o[b], 0, 0, 0);
                o[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v8, pl, o[b], 0, 0, 0);
            }
        }
        if (more) stage(step + 1);
        if (tid < 8) slabs[step & 1][tid] = next;
        __syncthreads();
    }
    float *sums = reinterpret_cast<float *>(kv);
#pragma unroll
    for (int b = 0; b < 2 * U; ++b) *reinterpret_cast<fa4 *>(sums + (wv * 16 + c) * HD + 16 * b + 4 * g) = o[b];
    if (g == 0) sm[tile][par][c] = m, sl[tile][par][c] = l;
    __syncthreads();
    for (int i = 0; i < TILES; ++i)
        meet<HD, 2>(sums + i * 32 * HD, sm[i], sl[i], TH, tid, first + 16 * i, nvec, G, kvh, heads, s.row0, out, nullptr, nullptr, 1, 0);
}

// ---- host side -----------------------------------------------------------------------------------------------

size_t block_bytes(int positions, int hd) {
    const size_t p = (static_cast<size_t>(positions) + kSlab - 1) / kSlab * kSlab;
    return p * hd / 2 + p * hd / 16;
}

bool hd_ok(int hd) { return hd >= 32 && hd <= kMaxHd && hd % 32 == 0; }

// page > 0: a pool's map; else a contiguous cache of max_seq positions.
Map4 make_map(const int32_t *pt, int page, int pps, int pages, int kv_heads, int max_seq, int hd) {
    Map4 M{pt, pps, pages, kv_heads, 0, 0, 0, 0};
    const int positions = pt != nullptr ? page : max_seq;
    M.spp = (static_cast<uint32_t>(positions) + kSlab - 1) / kSlab;
    uint32_t log = 0;
    while ((1u << log) < M.spp) ++log;
    M.shift = 28 + log;
    M.mul = static_cast<uint32_t>((1ull << M.shift) / M.spp + 1);
    M.bytes = block_bytes(positions, hd);
    return M;
}

bool aligned16(const void *a, const void *b) { return ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15) == 0; }

// What every entry point over 4-bit caches checks; M is set on success.
int check_cache(const void *kc, const void *vc, int kv_heads, int hd, const SegTable &T, bool in_pages, const int32_t *pt, int page,
                int pps, int pages, int max_seq, Map4 &M) {
    if (!kc || !vc || !aligned16(kc, vc)) return VQ_ERR_ARG;
    if (kv_heads < 1 || kv_heads > 65535 || !hd_ok(hd)) return VQ_ERR_SHAPE;
    if (in_pages) {
        if (const int st = check_paging(pt, page, pps, T); st != VQ_OK) return st;
        if (page % kSlab || pages < 1) return VQ_ERR_SHAPE;
    }
    for (int i = 0; i < T.n; ++i)
        if (T.s[i].pos0 > INT32_MAX - kSlab - T.s[i].rows) return VQ_ERR_SHAPE;
    M = make_map(in_pages ? pt : nullptr, page, pps, pages, kv_heads, max_seq, hd);
    return VQ_OK;
}

Starts starts_of(const SegTable &T, int (*units)(const Seg &, int), int arg) {
    Starts R;
    R.total = 0;
    for (int i = 0; i < VQ_MAX_SEGMENTS; ++i) {
        R.first[i] = R.total;
        if (i < T.n) R.total += units(T.s[i], arg);
    }
    return R;
}
int slabs_of(const Seg &s, int) { return (s.pos0 + s.rows - 1) / kSlab - s.pos0 / kSlab + 1; }
int rows_of(const Seg &s, int) { return s.rows; }

int launch_append4(const float *k, const float *v, void *kc, void *vc, const SegTable &T, const Map4 &M, int hd, hipStream_t s) {
    if (!k || !v) return VQ_ERR_ARG;
    const Starts R = starts_of(T, slabs_of, 0);
    const dim3 grid(R.total, M.kv_heads);
    const int threads = (hd + 63) / 64 * 64;
    auto *kb = static_cast<uint8_t *>(kc), *vb = static_cast<uint8_t *>(vc);
    if (M.pt) kv4_append_kernel<true><<<grid, threads, 0, s>>>(k, v, kb, vb, T, R, M, hd);
    else kv4_append_kernel<false><<<grid, threads, 0, s>>>(k, v, kb, vb, T, R, M, hd);
    return status_of(hipGetLastError());
}

int launch_read4(const void *kc, const void *vc, float *k, float *v, const SegTable &T, const Map4 &M, int hd, hipStream_t s) {
    if (!k || !v) return VQ_ERR_ARG;
    const Starts R = starts_of(T, slabs_of, 0);
    const dim3 grid(R.total, M.kv_heads);
    const int threads = (hd + 63) / 64 * 64;
    auto *kb = static_cast<const uint8_t *>(kc), *vb = static_cast<const uint8_t *>(vc);
    if (M.pt) kv4_read_kernel<true><<<grid, threads, 0, s>>>(kb, vb, k, v, T, R, M, hd);
    else kv4_read_kernel<false><<<grid, threads, 0, s>>>(kb, vb, k, v, T, R, M, hd);
    return status_of(hipGetLastError());
}

// Chunks for about a round or a few of the 512 workgroups that run at once (two per CU). `rounds` full rounds need chunks of at
// least some length; among 1 to 4 rounds the least of rounds x (length + what a chunk costs besides its keys, in keys).
int chunks_of(const SegTable &T, int i, long long len, int window) {
    return static_cast<int>((T.s[i].pos0 + T.s[i].rows - first_key(T.s[i], window) + len - 1) / len);
}
Cuts make_cuts(const SegTable &T, int heads, int kv_heads, int window) {
    #ifndef KFIX
#define KFIX 160
#endif
    constexpr int kSlots = 512, kFixed = KFIX;
    int groups = 1;
    long long keys = 0;
    for (int i = 0; i < T.n; ++i) {
        groups = max(groups, (T.s[i].rows * (heads / kv_heads) + 15) / 16);
        keys += T.s[i].pos0 + T.s[i].rows - first_key(T.s[i], window);
    }
    auto count = [&](long long len) {
        long long n = 0;
        for (int i = 0; i < T.n; ++i) n += chunks_of(T, i, len, window);
        return n * kv_heads * groups;
    };
    long long best = 0, cost = 0;
    for (int rounds = 1; rounds <= 4; ++rounds) {
        long long len = (keys * kv_heads * groups / (kSlots * rounds) + 127) / 128 * 128;
        len = len < 128 ? 128 : len;
        for (int i = 0; i < 64 && count(len) > static_cast<long long>(kSlots) * rounds; ++i) len += 128;
        const long long c = rounds * (len + kFixed);
        if (best == 0 || c < cost) best = len, cost = c;
    }
    Cuts C;
    C.len = static_cast<int>(best);
    C.total = C.most = 0;
    int base = 0;
    for (int i = 0; i < VQ_MAX_SEGMENTS; ++i) {
        C.first[i] = C.total;
        C.base[i] = base;
        if (i >= T.n) continue;
        const int n = chunks_of(T, i, C.len, window);
        if (n > 1) base += n * T.s[i].rows * heads;
        C.total += n;
        C.most = max(C.most, n);
    }
    return C;
}
// Partial results of the pass: vectors x chunks where a segment has more than one.
size_t parts_of(const SegTable &T, const Cuts &C, int heads, int window) {
    size_t n = 0;
    for (int i = 0; i < T.n; ++i) {
        const size_t k = chunks_of(T, i, C.len, window);
        if (k > 1) n += k * T.s[i].rows * heads;
    }
    return n;
}
size_t attention4_ws_bytes(const SegTable &T, int heads, int kv_heads, int hd, int window) {
    if (max_seg_rows(T) > VQ_ATTN_ROW_MAX) return 0;
    const size_t n = parts_of(T, make_cuts(T, heads, kv_heads, window), heads, window);
    return n * (hd + 2) * 4 + 16;
}

template <typename F>
void for_hd(int hd, F &&f) {
    switch (hd / 32) {
        case 1: f(std::integral_constant<int, 1>{}); break;
        case 2: f(std::integral_constant<int, 2>{}); break;
        case 3: f(std::integral_constant<int, 3>{}); break;
        case 4: f(std::integral_constant<int, 4>{}); break;
        case 5: f(std::integral_constant<int, 5>{}); break;
        case 6: f(std::integral_constant<int, 6>{}); break;
        case 7: f(std::integral_constant<int, 7>{}); break;
        default: f(std::integral_constant<int, 8>{}); break;
    }
}

int launch_attention4(const float *q, const void *kc, const void *vc, float *out, const SegTable &T, const Map4 &M, int heads, int hd,
                      int bidirectional, int window, void *ws, size_t ws_bytes, hipStream_t s) {
    if (!q || !out) return VQ_ERR_ARG;
    if (heads < M.kv_heads || heads % M.kv_heads || window < 0) return VQ_ERR_SHAPE;
    const int G = heads / M.kv_heads;
    auto *kb = static_cast<const uint8_t *>(kc), *vb = static_cast<const uint8_t *>(vc);
    if (ws != nullptr && max_seg_rows(T) <= VQ_ATTN_ROW_MAX) {
        if ((reinterpret_cast<uintptr_t>(ws) & 15) || ws_bytes < attention4_ws_bytes(T, heads, M.kv_heads, hd, window))
            return VQ_ERR_WORKSPACE;
        const Cuts C = make_cuts(T, heads, M.kv_heads, window);
        const Starts R = starts_of(T, rows_of, 0);
        const size_t parts = parts_of(T, C, heads, window);
        float *part = static_cast<float *>(ws), *pml = part + parts * hd;
        const dim3 grid(C.total * M.kv_heads, (max_seg_rows(T) * G + 15) / 16);
        for_hd(hd, [&](auto u) {
            constexpr int U = decltype(u)::value;
            auto go = [&](auto kernel) { kernel<<<grid, 256, 0, s>>>(q, kb, vb, part, pml, out, T, M, C, heads, bidirectional, window); };
            if constexpr (U % 4 == 0) {
                if (!M.pt) return go(attention4_stream_kernel<U, 0>);
                if (M.spp % 4 == 0) return go(attention4_stream_kernel<U, 4>);
                if (M.spp % 2 == 0) return go(attention4_stream_kernel<U, 2>);
            }
            if (M.pt) go(attention4_split_kernel<U, true>);
            else if constexpr (U % 4 != 0) go(attention4_split_kernel<U, false>);
        });
        for_hd(hd, [&](auto u) {
            constexpr int U = decltype(u)::value;
            if (parts) attention4_merge_kernel<32 * U><<<dim3(T.total * heads, U % 2 == 0 ? U / 2 : U), 256, 0, s>>>(part, pml, out, T, C, R, heads);
        });
        return status_of(hipGetLastError());
    }
    constexpr int NW = 8, PER = 16 * (NW / 2);
    long long vectors = 0;
    for (int i = 0; i < T.n; ++i) vectors += static_cast<long long>(T.s[i].rows) * G + PER;
    if (vectors / PER * M.kv_heads > INT32_MAX) return VQ_ERR_SHAPE;
    const Starts R = starts_of(T, [](const Seg &x, int g) { return static_cast<int>((static_cast<long long>(x.rows) * g + PER - 1) / PER); }, G);
    const dim3 grid(static_cast<unsigned>(R.total) * M.kv_heads);
    for_hd(hd, [&](auto u) {
        constexpr int U = decltype(u)::value;
        if (M.pt) attention4_tiled_kernel<U, true, NW><<<grid, 64 * NW, 0, s>>>(q, kb, vb, out, T, R, M, heads, bidirectional, window);
        else attention4_tiled_kernel<U, false, NW><<<grid, 64 * NW, 0, s>>>(q, kb, vb, out, T, R, M, heads, bidirectional, window);
    });
    return status_of(hipGetLastError());
}

}  // namespace

extern "C" {

size_t vq_kv4_bytes(long long blocks, int positions, int hd) {
    if (blocks < 1 || positions < 1 || positions > INT32_MAX - kSlab || !hd_ok(hd)) return 0;
    const size_t b = block_bytes(positions, hd);
    return static_cast<unsigned long long>(blocks) > (SIZE_MAX >> 1) / b ? 0 : static_cast<size_t>(blocks) * b;
}

int vq_kv4_append(const float *k, const float *v, void *kc, void *vc, int ntok, int kv_heads, int max_seq, int hd, int pos0,
                  void *stream) {
    if (ntok < 1 || pos0 < 0 || max_seq < 1 || ntok > max_seq || pos0 > max_seq - ntok) return VQ_ERR_SHAPE;
    const SegTable T = one_segment(pos0, ntok);
    Map4 M;
    const int st = check_cache(kc, vc, kv_heads, hd, T, false, nullptr, 0, 0, 0, max_seq, M);
    return st != VQ_OK ? st : launch_append4(k, v, kc, vc, T, M, hd, static_cast<hipStream_t>(stream));
}

int vq_kv4_append_seg(const float *k, const float *v, void *kc, void *vc, const int32_t *segs, int nseg, int kv_heads, int hd,
                      const int32_t *page_table, int page_size, int pages_per_seq, int pages, void *stream) {
    SegTable T;
    Map4 M;
    int st = make_table(segs, nseg, T, nullptr);
    if (st == VQ_OK) st = check_cache(kc, vc, kv_heads, hd, T, true, page_table, page_size, pages_per_seq, pages, 0, M);
    return st != VQ_OK ? st : launch_append4(k, v, kc, vc, T, M, hd, static_cast<hipStream_t>(stream));
}

int vq_kv4_read(const void *kc, const void *vc, float *k, float *v, int ntok, int kv_heads, int max_seq, int hd, int pos0,
                void *stream) {
    if (ntok < 1 || pos0 < 0 || max_seq < 1 || ntok > max_seq || pos0 > max_seq - ntok) return VQ_ERR_SHAPE;
    const SegTable T = one_segment(pos0, ntok);
    Map4 M;
    const int st = check_cache(kc, vc, kv_heads, hd, T, false, nullptr, 0, 0, 0, max_seq, M);
    return st != VQ_OK ? st : launch_read4(kc, vc, k, v, T, M, hd, static_cast<hipStream_t>(stream));
}

int vq_kv4_read_seg(const void *kc, const void *vc, float *k, float *v, const int32_t *segs, int nseg, int kv_heads, int hd,
                    const int32_t *page_table, int page_size, int pages_per_seq, int pages, void *stream) {
    SegTable T;
    Map4 M;
    int st = make_table(segs, nseg, T, nullptr);
    if (st == VQ_OK) st = check_cache(kc, vc, kv_heads, hd, T, true, page_table, page_size, pages_per_seq, pages, 0, M);
    return st != VQ_OK ? st : launch_read4(kc, vc, k, v, T, M, hd, static_cast<hipStream_t>(stream));
}

size_t vq_attention4_workspace_bytes(int heads, int kv_heads, int hd, int seq_len, int ntok, int window) {
    if (kv_heads < 1 || heads < kv_heads || heads % kv_heads || !hd_ok(hd) || ntok < 1 || seq_len < 1 || window < 0 ||
        seq_len > INT32_MAX - kSlab - ntok)
        return 0;
    return attention4_ws_bytes(one_segment(seq_len - 1, ntok), heads, kv_heads, hd, window);
}

size_t vq_attention4_seg_workspace_bytes(const int32_t *segs, int nseg, int heads, int kv_heads, int hd) {
    SegTable T;
    if (make_table(segs, nseg, T, nullptr) != VQ_OK) return 0;
    if (kv_heads < 1 || heads < kv_heads || heads % kv_heads || !hd_ok(hd)) return 0;
    for (int i = 0; i < T.n; ++i)
        if (T.s[i].pos0 > INT32_MAX - kSlab - T.s[i].rows) return 0;
    return attention4_ws_bytes(T, heads, kv_heads, hd, 0);
}

int vq_attention4_ws(const float *q, const void *kc, const void *vc, float *out, int heads, int kv_heads, int hd, int max_seq,
                     int seq_len, int ntok, int bidirectional, int window, void *workspace, size_t workspace_bytes,
                     void *stream) {
    if (ntok < 1 || seq_len < 1 || ntok > max_seq || seq_len > max_seq - ntok + 1) return VQ_ERR_SHAPE;
    const SegTable T = one_segment(seq_len - 1, ntok);
    Map4 M;
    const int st = check_cache(kc, vc, kv_heads, hd, T, false, nullptr, 0, 0, 0, max_seq, M);
    return st != VQ_OK ? st : launch_attention4(q, kc, vc, out, T, M, heads, hd, bidirectional, window, workspace, workspace_bytes,
                                                static_cast<hipStream_t>(stream));
}

int vq_attention4_seg_ws(const float *q, const void *kc, const void *vc, float *out, const int32_t *segs, int nseg, int heads,
                         int kv_heads, int hd, const int32_t *page_table, int page_size, int pages_per_seq, int pages,
                         void *workspace, size_t workspace_bytes, void *stream) {
    SegTable T;
    Map4 M;
    int st = make_table(segs, nseg, T, nullptr);
    if (st == VQ_OK) st = check_cache(kc, vc, kv_heads, hd, T, true, page_table, page_size, pages_per_seq, pages, 0, M);
    return st != VQ_OK ? st : launch_attention4(q, kc, vc, out, T, M, heads, hd, 0, 0, workspace, workspace_bytes,
                                                static_cast<hipStream_t>(stream));
}

}  // extern "C"
