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

// How a pass is cut: each segment's query vectors in groups of 16 NT, its keys in chunks of `len` (a multiple of 128) from its first
// key rounded down to 32; segment i's groups x chunks begin at first[i] of one list, its partial results at base[i] (where it has
// more than one chunk).
struct Cuts {
    int len, total, most;  // most: of a segment's chunks
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

// Where a group's results go: the output where the segment has one chunk, else the chunk's unnormalised part.
struct Dest {
    float *out, *part, *pml;
    size_t base;
    int heads, G, kvh, row0, nvec, n, ci;
    template <int HD>
    __device__ __forceinline__ void put(int j, int d, const float4 &acc, float m, float l) const {
        const int t = j / G, h = kvh * G + j - t * G;
        if (n == 1) {
            const float inv = l > 0.0f ? 1.0f / l : 0.0f;
            const float4 r{acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
            __builtin_memcpy(out + (static_cast<size_t>(row0 + t) * heads + h) * HD + d, &r, 16);
        } else {
            const size_t at = base + (static_cast<size_t>(t) * heads + h) * n + ci;
            *reinterpret_cast<float4 *>(part + at * HD + d) = acc;
            if (d == 0) pml[2 * at] = m, pml[2 * at + 1] = l;
        }
    }
};
// A sum's share against maximum m where it was kept against `own`.
__device__ __forceinline__ float share(float own, float m) { return own == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(own - m); }

// Four waves' sums of 16 vectors (each wave's [16][HD], maxima and totals) meet in wave order.
template <int HD>
__device__ __forceinline__ void meet4(const float *sums, const float (&sm)[4][2][16], const float (&sl)[4][2][16], int j0, const Dest &to) {
    for (int e = threadIdx.x; e < 16 * (HD / 4); e += 256) {
        const int c = e / (HD / 4), d4 = 4 * (e - c * (HD / 4));
        if (j0 + c >= to.nvec) continue;
        const float mx = fmaxf(fmaxf(sm[0][0][c], sm[1][0][c]), fmaxf(sm[2][0][c], sm[3][0][c]));
        float L = 0.0f;
        float4 acc{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = share(sm[w][0][c], mx);
            L = fmaf(sl[w][0][c], f, L);
            const float4 p = *reinterpret_cast<const float4 *>(sums + (w * 16 + c) * HD + d4);
            acc.x = fmaf(p.x, f, acc.x);
            acc.y = fmaf(p.y, f, acc.y);
            acc.z = fmaf(p.z, f, acc.z);
            acc.w = fmaf(p.w, f, acc.w);
        }
        to.put<HD>(j0 + c, d4, acc, mx, L);
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
__device__ __forceinline__ void no_page(Raw4<U> &r) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < (U + 1) / 2; ++i) r.kh[h][i] = kNanHeader | kNanHeader << 16;
}
template <int U>
__device__ __forceinline__ void issue_k(const uint8_t *__restrict__ kc, const SlabAt &at, Raw4<U> &r) {
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int row = 4 * h + (c & 3);
        ld_words<U>(kc + at.words + row * (16 * U) + g * (4 * U), r.k[h]);
        ld_heads<U>(kc + at.heads + row * (2 * U), r.kh[h]);
    }
    if (at.bad) no_page<U>(r);
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

// ---- blocks by DMA ----

// For hd 128 and 256, whose waves are few (hd 256: 2 per SIMD, for the registers of O and q): the blocks come to LDS by DMA, kSlots of
// them for each wave, so that the loads of one are in flight while another is computed with, and no registers are spent on them. A
// slot is K's words, slab after slab, V's words, and 512 bytes each of K's and of V's headers, slab after slab. Page ids and
// addresses are wave-uniform and come by scalar loads: the only vector memory operations of the loop are the DMA's, which the waits
// count.
template <int U, int NT>
struct Ring {
    static constexpr int kSlots = U == 8 ? (NT == 1 ? 2 : 1) : (NT == 1 ? 3 : 2);
    static constexpr int kWords = 512 * U, kBytes = 2 * kWords + 1024;
    static constexpr int kLoads = kSlots == 1 ? U / 2 + 1 : U + 1;  // of half a slot that is filled by halves, or of a slot
};
// Where a block's four slabs are. MODE: how many of them one look at the page table gives (4: pages of whole blocks, 2: of pairs of
// slabs), 0: a contiguous cache.
struct Slab4 {
    size_t words0, words1, heads0, heads1;  // in the cache: of the first slab and (MODE 2) of the third
    int rest;                               // MODE 0: slabs behind the first
    uint32_t bad;                           // a bit for each slab whose page is none
};
// Slabs past the last key's: that one's page (a contiguous cache: that one) is read instead; their keys are masked.
template <int U, int MODE>
__device__ __forceinline__ uint32_t look_up_page(const Map4 &M, int slot, int kvh, int slab, int last, size_t &words, size_t &heads) {
    const auto *pt = (const __attribute__((address_space(4))) int32_t *)(M.pt) + static_cast<size_t>(slot) * M.pps;
    const uint32_t want = min(slab, last & ~(MODE - 1)), p = static_cast<uint32_t>((static_cast<uint64_t>(want) * M.mul) >> M.shift);
    const int pg = pt[p];
    const bool none = static_cast<uint32_t>(pg) >= static_cast<uint32_t>(M.pages);
    const size_t block = (static_cast<size_t>(none ? 0 : pg) * M.kv_heads + kvh) * M.bytes;
    const uint32_t at = want - p * M.spp;
    words = block + static_cast<size_t>(at) * (128 * U), heads = block + static_cast<size_t>(M.spp) * (128 * U) + static_cast<size_t>(at) * (16 * U);
    return none ? (1u << MODE) - 1 : 0u;
}
template <int U, int MODE>
__device__ __forceinline__ Slab4 look_up(const Map4 &M, int slot, int kvh, int kb, int last) {
    Slab4 r{};
    const int slab = kb / kSlab;
    if constexpr (MODE == 0) {
        const size_t block = static_cast<size_t>(kvh) * M.bytes;
        r.words0 = block + static_cast<size_t>(slab) * (128 * U);
        r.heads0 = block + static_cast<size_t>(M.spp) * (128 * U) + static_cast<size_t>(slab) * (16 * U);
        r.rest = last - slab;
    } else {
        r.bad = look_up_page<U, MODE>(M, slot, kvh, slab, last, r.words0, r.heads0);
        if constexpr (MODE == 2) r.bad |= look_up_page<U, MODE>(M, slot, kvh, slab + 2, last, r.words1, r.heads1) << 2;
    }
    return r;
}
// The active lanes x 16 bytes from each lane's own address to LDS at (wave-uniform) dst + 16 lane. The second form: from a uniform
// base and the lane's offset, which costs no vector instruction.
__device__ __forceinline__ uint32_t lds_at(uint8_t *dst) {
    return static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(vq::lds_addr(dst))));
}
__device__ __forceinline__ void dma16(const uint8_t *from, uint8_t *dst) {
    asm volatile("s_mov_b32 m0, %1\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "s"(lds_at(dst)), "s"(dst) : "memory", "m0");
}
__device__ __forceinline__ void dma16(const uint8_t *base, uint32_t off, uint8_t *dst) {
    asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds_at(dst)), "s"(dst) : "memory", "m0");
}
// Slab n's words begin at `key` 8 n. Its eight rows of 16 U bytes keep their order, but a row's pieces of 16 bytes (U / 2 for each of
// a word's four g) change places by this, so that rows 8 a + 4 h + r (a, r < 4) and rows 16 a + r (r < 16) spread over the banks.
template <int U>
__device__ __forceinline__ int swizzle(int key) {
    const int a = key >> 3 & 1, b = (key >> 2 ^ key >> 4) & 1;
    return U == 8 ? (key >> 1 & 1) | a << 1 | b << 2 : a | b << 1;
}
// A DMA load brings 1024 bytes: a slab of hd 256, two of hd 128.
template <int U, int MODE, bool K>
__device__ __forceinline__ void dma_words(const uint8_t *cache, const Slab4 &at, uint8_t *words) {
    const int lane = threadIdx.x & 63, slabs = 8 / U, sub = lane / (8 * U), piece = lane & (8 * U - 1);
#pragma unroll
    for (int x = 0; x < U / 2; ++x) {
        const int n = x * slabs;
        const int first = MODE == 0 ? min(n, at.rest) : n, step = MODE == 0 ? min(n + 1, at.rest) - first : 1;
        const uint8_t *base = cache + (MODE == 2 && n >= 2 ? at.words1 + (n - 2) * (128 * U) : at.words0 + static_cast<size_t>(first) * (128 * U));
        uint32_t off = 16 * piece;
        if (K) {
            const int row = piece / U, s = piece % U;
            off = row * (16 * U) + 16 * (s ^ swizzle<U>(8 * (n + sub) + row));
        }
        dma16(base, off + sub * step * (128 * U), words + 1024 * x);
    }
}
// The headers by lanes 0 to 31 (K's) and 32 to 63 (V's), or one of the two.
template <int U, int MODE>
__device__ __forceinline__ void dma_heads(const uint8_t *kc, const uint8_t *vc, const Slab4 &at, uint8_t *to, bool k, bool v) {
    const int lane = threadIdx.x & 63, piece = min(lane & 31, 4 * U - 1), n = piece / U;
    const uint8_t *from = (lane < 32 ? kc : vc) + piece % U * 16;
    // (Both are read, or the choice becomes one between their addresses, which puts them in memory.)
    const size_t h0 = at.heads0, h1 = at.heads1;
    if (MODE == 0) from += h0 + static_cast<size_t>(min(n, at.rest) * (16 * U));
    if (MODE == 4) from += h0 + n * (16 * U);
    if (MODE == 2) from += (n & 2 ? h1 : h0) + (n & 1) * (16 * U);
    if ((k && v) || (lane < 32) == k) dma16(from, to);
}
template <int U>
__device__ __forceinline__ void read_k(const uint8_t *words, const uint8_t *heads, Raw4<U> &r) {
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int i = 0; i < U / 4; ++i) {
            const int key = 8 * (c >> 2) + 4 * half + (c & 3);
            const uint4 w = *reinterpret_cast<const uint4 *>(words + (16 * U) * key + 16 * ((U / 4 * g + i) ^ swizzle<U>(key)));
            r.k[half][4 * i] = w.x, r.k[half][4 * i + 1] = w.y, r.k[half][4 * i + 2] = w.z, r.k[half][4 * i + 3] = w.w;
        }
        ld_words<U / 2>(heads + (8 * (c >> 2) + 4 * half + (c & 3)) * (2 * U), r.kh[half]);
    }
}
template <int U>
__device__ __forceinline__ void read_v(const uint8_t *words, const uint8_t *heads, Raw4<U> &r) {
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
#pragma unroll
    for (int i = 0; i < U / 2; ++i) {
        const uint4 w = *reinterpret_cast<const uint4 *>(words + (128 * U) * g + 256 * i + 16 * c);
        r.v[4 * i] = w.x, r.v[4 * i + 1] = w.y, r.v[4 * i + 2] = w.z, r.v[4 * i + 3] = w.w;
    }
    r.vh = *reinterpret_cast<const uint4 *>(heads + 16 * (g * U + min(c, U - 1)));
}
// At most N loads outstanding, for the few N that occur.
__device__ __forceinline__ void wait_loads(int n) {
    switch (n) {
        case 0: vq::wait_vm<0>(); break;
        case 5: vq::wait_vm<5>(); break;
        case 9: vq::wait_vm<9>(); break;
        default: vq::wait_vm<10>(); break;
    }
}

// ---- the products ----

// Query operands of NT tiles: in registers, or (more than 8 operand steps) in LDS, [u][tile][hi, lo][lane].
template <int U, int NT>
struct Query {
    static constexpr bool kLds = NT * U > 8;
    fh8 h[kLds ? 1 : NT][kLds ? 1 : U], l[kLds ? 1 : NT][kLds ? 1 : U];
};

// The NT tiles' products of a block: K decoded once for all of them. In steps of one word, each of which decodes the next one's while
// the matrix unit works, and reads its queries ahead; left to itself the compiler waits for each.
template <int U, int NT>
__device__ __forceinline__ void scores(const Raw4<U> &r, const Query<U, NT> &q, const uint8_t *qlds, fa4 (&s)[NT][2]) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = fa4{0.f, 0.f, 0.f, 0.f};
    fh8 qb[2][NT][2], kb[2];
    auto query = [&](int u) {
        if constexpr (Query<U, NT>::kLds) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int x = 0; x < 2; ++x) qb[u & 1][n][x] = *reinterpret_cast<const fh8 *>(qlds + ((u * NT + n) * 2 + x) * 1024 + 16 * lane);
        } else {
#pragma unroll
            for (int n = 0; n < NT; ++n) qb[u & 1][n][0] = q.h[n][u], qb[u & 1][n][1] = q.l[n][u];
        }
    };
    auto key = [&](int i) {
        const int u = i >> 1, h = i & 1;
        kb[i & 1] = u % 2 == 0 ? decode8_one<false>(r.k[h][u], r.kh[h][u / 2]) : decode8_one<true>(r.k[h][u], r.kh[h][u / 2]);
    };
    query(0);
    key(0);
#pragma unroll
    for (int i = 0; i < 2 * U; ++i) {
        const int u = i >> 1, h = i & 1;
        if constexpr (NT > 1) __builtin_amdgcn_sched_barrier(0);
        if (h == 0 && u + 1 < U) query(u + 1);
        if (i + 1 < 2 * U) key(i + 1);
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int n = 0; n < NT; ++n) s[n][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kb[i & 1], qb[u & 1][n][x], s[n][h], 0, 0, 0);
    }
    if constexpr (NT > 1) __builtin_amdgcn_sched_barrier(0);
}
// O^T += V^T P^T. Every lane of a row of 16 needs the headers of all groups of its slab: lane c takes group c's apart and the others
// read them from LDS (`hl`, the wave's own: [slab][group] scales, zero points; moving them by DPP costs 64 instructions a block of
// the kind that bounds this kernel).
template <int U>
constexpr int head_words = 4 * (8 * U + 8);
template <int U, int NT>
__device__ __forceinline__ void add_values(const Raw4<U> &r, const fh8 (&ph)[NT], const fh8 (&pl)[NT], uint32_t *hl, fa4 (&o)[NT][2 * U]) {
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
    uint4 dw[2], zw[2];
    fh8 vb[2];
    auto heads = [&](int u) {
        dw[u & 1] = *reinterpret_cast<const uint4 *>(mine + 8 * u), zw[u & 1] = *reinterpret_cast<const uint4 *>(mine + 8 * u + 4);
    };
    auto value = [&](int b) {
        const uint4 &x = dw[b >> 1 & 1], &y = zw[b >> 1 & 1];
        const fh2 d[4] = {__builtin_bit_cast(fh2, x.x), __builtin_bit_cast(fh2, x.y), __builtin_bit_cast(fh2, x.z), __builtin_bit_cast(fh2, x.w)};
        const fh2 z[4] = {__builtin_bit_cast(fh2, y.x), __builtin_bit_cast(fh2, y.y), __builtin_bit_cast(fh2, y.z), __builtin_bit_cast(fh2, y.w)};
        vb[b & 1] = decode8(r.v[b], d, z);
    };
    heads(0);
    value(0);
#pragma unroll
    for (int b = 0; b < 2 * U; ++b) {
        if constexpr (NT > 1) __builtin_amdgcn_sched_barrier(0);
        if (b % 2 == 0 && b + 2 < 2 * U) heads(b / 2 + 1);
        if (b + 1 < 2 * U) value(b + 1);
#pragma unroll
        for (int n = 0; n < NT; ++n) o[n][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vb[b & 1], ph[n], o[n][b], 0, 0, 0);
#pragma unroll
        for (int n = 0; n < NT; ++n) o[n][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vb[b & 1], pl[n], o[n][b], 0, 0, 0);
    }
    if constexpr (NT > 1) __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");  // every lane has read before the next block's writes
    __builtin_amdgcn_wave_barrier();
}

// One workgroup of four waves per (chunk of keys, kv head, group of 16 NT query vectors); vector j of a segment is (row j / G, head
// j % G of the kv head's group). The waves take the 32-key blocks in turn (wave w those whose index is w modulo 4, whatever the
// chunk: with one chunk a row's sums do not depend on the other rows of its pass), decode them once into MFMA operands for all of
// the group's tiles, with an online softmax each, and meet at the end.
//
// Bound by vector instructions: 640 a block and wave at hd 256 for one tile, 500 of them for the 16384 values decoded, 64 MFMAs
// beside them; a second tile adds 140 and 64. So groups of more than 16 vectors take two tiles (q in LDS then, for hd 256: O alone
// is half of the registers of two waves per SIMD). Keys by LDS tiles decoded once for 64 vectors (8 waves, a barrier per 64 keys)
// took 94 us for 512 rows over 2048 keys, its two waves per SIMD in step; this takes 74.
// MODE: see Slab4; -1 and -2: blocks by vector loads, in pages and contiguous.
template <int U, int NT, int MODE>
__global__ __launch_bounds__(256, 2) void attention4_kernel(const float *__restrict__ q, const uint8_t *__restrict__ kc,
                                                            const uint8_t *__restrict__ vc, float *__restrict__ part,
                                                            float *__restrict__ pml, float *__restrict__ out, SegTable T, Map4 M, Cuts C,
                                                            int heads, int bidirectional, int window) {
    constexpr bool DMA = MODE >= 0, QLDS = Query<U, NT>::kLds;
    constexpr int HD = 32 * U, S = DMA ? Ring<U, NT>::kSlots : 1, LD = Ring<U, NT>::kLoads, WORDS = Ring<U, NT>::kWords;
    // One slot only: its K part and its V part are filled again each as soon as it has been read.
    constexpr bool SPLIT = DMA && S == 1;
    constexpr int BYTES = Ring<U, NT>::kBytes, RING = DMA ? S * BYTES : 0, QB = QLDS ? U * NT * 2048 : 0, SUMS = 256 * HD;
    __shared__ __align__(16) uint8_t lds[4 * RING + QB > SUMS ? 4 * RING + QB : SUMS];
    __shared__ float sm[4][2][16], sl[4][2][16];
    __shared__ __align__(16) uint32_t vheads[4][head_words<U>];
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
    const int bases = C.base[lane];
    const Found found = find_segment(T, C.first, C.total, blockIdx.x / M.kv_heads);
    const Seg s = found.s;
    const int G = heads / M.kv_heads, nvec = s.rows * G, units = found.next - found.first;
    // A segment's kv heads x chunks x groups. One tile holds its vectors whole; of several groups (the last rows, which see the most
    // keys, first) those of a head and chunk go to one XCD, for its L2: eight heads and chunks at a time, then the rest.
    const int at = blockIdx.x - found.first * M.kv_heads;
    const int groups = NT == 1 ? 1 : (nvec + 16 * NT - 1) / (16 * NT), n = NT == 1 ? units : units / groups;
    int stream = at, group = 0;
    if (NT != 1) {
        const int streams = n * M.kv_heads, rest = streams & 7, eights = (streams - rest) * groups;
        if (at < eights) {
            const int block = at / (8 * groups), x = at - block * 8 * groups;
            group = x >> 3, stream = 8 * block + (x & 7);
        } else {
            group = (at - eights) / rest, stream = streams - rest + (at - eights) - group * rest;
        }
        group = groups - 1 - group;
    }
    const int ci = stream / M.kv_heads, kvh = stream - ci * M.kv_heads, j0 = group * 16 * NT;
    const Sees lo = sees(s, NT == 1 ? 0 : j0 / G, bidirectional, window);
    const Sees hi = sees(s, NT == 1 ? s.rows - 1 : min(j0 + 16 * NT - 1, nvec - 1) / G, bidirectional, window);
    const int c_lo = first_key(s, window) + ci * C.len;
    const int k_lo = max(c_lo, lo.from & ~31), k_hi = n == 1 ? hi.to : min(c_lo + C.len, hi.to), last = (k_hi - 1) / kSlab;
    if (k_lo >= k_hi) return;
    int kb = k_lo + 32 * ((wv - (k_lo >> 5)) & 3);
    uint8_t *const ring = lds + wv * RING, *const qlds = lds + 4 * RING;
    Raw4<U> r;
    SlabAt ks, vs;
    uint32_t bad = 0;  // four bits a slot
    // Lane (c, g) takes K rows of slab c >> 2 and V words of slab g of a block; slabs past the last key's read that one's (masked).
    auto places = [&](int block) {
        ks = slab_at<U, MODE == -1>(M, s.slot, kvh, min(block / kSlab + (c >> 2), last));
        vs = slab_at<U, MODE == -1>(M, s.slot, kvh, min(block / kSlab + g, last));
    };
    auto fetch = [&](int block, int slot) {
        if constexpr (DMA) {
            const Slab4 where = look_up<U, MODE>(M, s.slot, kvh, block, last);
            uint8_t *const to = ring + slot * BYTES;
            dma_words<U, MODE, true>(kc, where, to);
            if constexpr (SPLIT) dma_heads<U, MODE>(kc, vc, where, to + 2 * WORDS, true, false);
            dma_words<U, MODE, false>(vc, where, to + WORDS);
            dma_heads<U, MODE>(kc, vc, where, to + 2 * WORDS, !SPLIT, true);
            bad = (bad & ~(15u << 4 * slot)) | where.bad << 4 * slot;
        } else {
            places(block);
            issue_k<U>(kc, ks, r);
            issue_v<U>(vc, vs, r);
        }
    };
    if (kb < k_hi) fetch(kb, 0);
    // Vectors past the last one repeat it; they are not written.
    auto vector = [&](int tile) { return min(j0 + 16 * tile + c, nvec - 1); };
    auto qrow = [&](int j) {
        const int t = j / G;
        return q + (static_cast<size_t>(s.row0 + t) * heads + kvh * G + j - t * G) * HD;
    };
    Query<U, NT> qr;
    float unit[NT];
    Sees see[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        see[i] = sees(s, vector(i) / G, bidirectional, window);
        see[i].to = min(see[i].to, k_hi);
    }
    if constexpr (QLDS) {  // a wave makes every second step's operands of a tile
        __shared__ float units[NT][16];
        const int tile = wv % NT;
        fh8 h[U], l[U];
        const float x = load_query<U>(qrow(vector(tile)), h, l);
        if (wv < NT && g == 0) units[tile][c] = x;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (u % (4 / NT) != wv / NT) continue;
            *reinterpret_cast<fh8 *>(qlds + ((u * NT + tile) * 2) * 1024 + 16 * lane) = h[u];
            *reinterpret_cast<fh8 *>(qlds + ((u * NT + tile) * 2 + 1) * 1024 + 16 * lane) = l[u];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NT; ++i) unit[i] = units[i][c];
    } else {
#pragma unroll
        for (int i = 0; i < NT; ++i) unit[i] = load_query<U>(qrow(vector(i)), qr.h[i], qr.l[i]);
    }
    float m[NT], l[NT];
    fa4 o[NT][2 * U];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        m[i] = -INFINITY, l[i] = 0.0f;
#pragma unroll
        for (int b = 0; b < 2 * U; ++b) o[i][b] = fa4{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int i = 1; i < S; ++i)
        if (kb + 128 * i < k_hi) fetch(kb + 128 * i, i);
    while (kb < k_hi) {
#pragma unroll
        for (int slot = 0; slot < S; ++slot) {
            if (kb >= k_hi) break;
            // A SIMD serves its older wave first, which left the younger one to finish alone, 11 of 40 us (131071 keys). A wave
            // that nears its end steps back, so that they finish together.
            const int left = (k_hi - 1 - kb) / 128;
            if (left >= 3) __builtin_amdgcn_s_setprio(3);
            else if (left == 2) __builtin_amdgcn_s_setprio(2);
            else if (left == 1) __builtin_amdgcn_s_setprio(1);
            else __builtin_amdgcn_s_setprio(0);
            const bool more = left >= S;
            uint8_t *const from = ring + slot * BYTES;
            Slab4 where;
            if constexpr (DMA) {
                // Landed: all but this block's V and the blocks behind it. The page of the block that comes into the slot meanwhile.
                wait_loads(SPLIT ? LD : LD * min(left, S - 1));
                if (SPLIT && more) where = look_up<U, MODE>(M, s.slot, kvh, kb + 128 * S, last);
                read_k<U>(from, from + 2 * WORDS, r);
                if (MODE != 0 && bad != 0 && (bad >> (4 * slot + (c >> 2)) & 1)) no_page<U>(r);
            } else {
                if (more) places(kb + 128);
            }
            fa4 sc[NT][2];
            scores<U, NT>(r, qr, qlds, sc);
            if (more) {
                if constexpr (SPLIT) {
                    vq::wait_lgkm0();  // the part has been read
                    dma_words<U, MODE, true>(kc, where, from);
                    dma_heads<U, MODE>(kc, vc, where, from + 2 * WORDS, true, false);
                    bad = (bad & ~(15u << 4 * slot)) | where.bad << 4 * slot;
                } else if constexpr (!DMA) {
                    issue_k<U>(kc, ks, r);
                }
            }
            fh8 ph[NT], pl[NT];
#pragma unroll
            for (int i = 0; i < NT; ++i) softmax_step<U>(sc[i], unit[i], kb, see[i].from, see[i].to, m[i], l[i], o[i], ph[i], pl[i]);
            if constexpr (DMA) {
                if (SPLIT) wait_loads(more ? LD : 0);
                read_v<U>(from + WORDS, from + 2 * WORDS + 512, r);
            }
            add_values<U, NT>(r, ph, pl, vheads[wv], o);
            if (more) {
                if constexpr (DMA) {
                    vq::wait_lgkm0();
                    if constexpr (SPLIT) {
                        dma_words<U, MODE, false>(vc, where, from + WORDS);
                        dma_heads<U, MODE>(kc, vc, where, from + 2 * WORDS, false, true);
                    } else {
                        fetch(kb + 128 * S, slot);
                    }
                } else {
                    issue_v<U>(vc, vs, r);
                }
            }
            kb += 128;
        }
    }
    __builtin_amdgcn_s_setprio(0);
    __syncthreads();  // every slot of every wave, and the queries, have been read
    float *sums = reinterpret_cast<float *>(lds);
    const Dest to{out, part, pml, static_cast<size_t>(from_lane(bases, found.index)), heads, G, kvh, s.row0, nvec, n, ci};
    if constexpr (NT == 1) {
        if (j0 + c < nvec) {
#pragma unroll
            for (int b = 0; b < 2 * U; ++b) *reinterpret_cast<fa4 *>(sums + (wv * 16 + c) * HD + 16 * b + 4 * g) = o[0][b];
            if (g == 0) sm[wv][0][c] = m[0], sl[wv][0][c] = l[0];
        }
        __syncthreads();
        meet4<HD>(sums, sm, sl, j0, to);
    } else {
        // Waves 2 and 3 hand their sums to waves 0 and 1, then those two exchange a tile each. [wave or its partner][tile][lane's
        // values]: a lane reads what the same lane of the other wave wrote.
        auto give = [&](int box, int i) {
            float *to_box = sums + (box * 2 + i) * 16 * HD;
#pragma unroll
            for (int b = 0; b < 2 * U; ++b) *reinterpret_cast<fa4 *>(to_box + 256 * b + 4 * lane) = o[i][b];
            if (g == 0) sm[wv][i][c] = m[i], sl[wv][i][c] = l[i];
        };
        auto take = [&](int box, int i, int from, bool first) {  // `first`: the other wave's sums count as the left operand
            const float *box_at = sums + (box * 2 + i) * 16 * HD;
            const float om = sm[from][i][c], ol = sl[from][i][c], mx = fmaxf(m[i], om);
            const float own = share(m[i], mx), other = share(om, mx), fl = first ? other : own, fr = first ? own : other;
            l[i] = fmaf(first ? l[i] : ol, fr, (first ? ol : l[i]) * fl);
#pragma unroll
            for (int b = 0; b < 2 * U; ++b) {
                const fa4 x = *reinterpret_cast<const fa4 *>(box_at + 256 * b + 4 * lane);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[i][b][e] = first ? fmaf(o[i][b][e], fr, x[e] * fl) : fmaf(x[e], fr, o[i][b][e] * fl);
            }
            m[i] = mx;
        };
        if (wv >= 2) give(wv - 2, 0), give(wv - 2, 1);
        __syncthreads();
        if (wv < 2) take(wv, 0, wv + 2, false), take(wv, 1, wv + 2, false);
        __syncthreads();
        if (wv == 0) give(0, 1);
        if (wv == 1) give(1, 0);
        __syncthreads();
        if (wv >= 2) return;
        if (wv == 0) take(1, 0, 1, false);
        else take(0, 1, 0, true);
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const int j = j0 + 16 * i + c;
            if (wv != i || j >= nvec) continue;
#pragma unroll
            for (int b = 0; b < 2 * U; ++b) to.put<HD>(j, 16 * b + 4 * g, float4{o[i][b][0], o[i][b][1], o[i][b][2], o[i][b][3]}, m[i], l[i]);
        }
    }
}

// A row's chunks: [lo, hi) of n hold its keys; the part of (row, head, chunk) is at `at` + head n + chunk.
struct RowChunks {
    int t, n, lo, hi;
    size_t at;
};
template <int NT>
__device__ __forceinline__ RowChunks row_chunks(const Found &found, const SegTable &T, const Cuts &C, int chunks, int bases, int row, int heads, int G,
                                                int bidirectional, int window) {
    const Seg s = found.s;
    const int i = found.index, t = row - found.first;
    const int units = (i + 1 < T.n ? from_lane(chunks, i + 1 < 64 ? i + 1 : 63) : C.total) - from_lane(chunks, i);
    RowChunks r{t, NT == 1 ? units : units / ((s.rows * G + 16 * NT - 1) / (16 * NT)), 0, 0, 0};
    r.hi = r.n;
    if (NT != 1) {  // (one tile: every chunk has been written)
        const Sees see = sees(s, t, bidirectional, window);
        const int k0 = first_key(s, window);
        r.lo = (see.from - k0) / C.len, r.hi = min((see.to - 1 - k0) / C.len + 1, r.n);
    }
    r.at = static_cast<size_t>(from_lane(bases, i)) + static_cast<size_t>(t) * heads * r.n;
    return r;
}
// sum_c 2^(m_c - m) o_c and sum_c 2^(m_c - m) l_c over chunks lo, lo + step, ..: four of them in flight, under a running maximum.
// `o`: these dims of chunk 0's part, `ml`: its maximum and sum.
template <int HD>
__device__ __forceinline__ float4 merge_parts(const float *o, const float *ml, int lo, int hi, int step, float &m, float &L) {
    m = -INFINITY, L = 0.0f;
    float4 acc{0.f, 0.f, 0.f, 0.f};
    for (int c0 = lo; c0 < hi; c0 += 4 * step) {
        float4 p[4];
        float mc[4], lc[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int c = c0 + step * k < hi ? c0 + step * k : c0;
            p[k] = *reinterpret_cast<const float4 *>(o + static_cast<size_t>(c) * HD);
            mc[k] = c0 + step * k < hi ? ml[2 * c] : -INFINITY;
            lc[k] = ml[2 * c + 1];
        }
        const float mn = fmaxf(fmaxf(m, fmaxf(mc[0], mc[1])), fmaxf(mc[2], mc[3])), f0 = share(m, mn);
        m = mn;
        L *= f0;
        acc = float4{acc.x * f0, acc.y * f0, acc.z * f0, acc.w * f0};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (c0 + step * k >= hi) break;
            const float f = share(mc[k], mn);
            L = fmaf(lc[k], f, L);
            acc.x = fmaf(p[k].x, f, acc.x);
            acc.y = fmaf(p[k].y, f, acc.y);
            acc.z = fmaf(p[k].z, f, acc.z);
            acc.w = fmaf(p[k].w, f, acc.w);
        }
    }
    return acc;
}
__device__ __forceinline__ void put_merged(float *to, const float4 &acc, float L) {
    const float inv = L > 0.0f ? 1.0f / L : 0.0f;
    const float4 r{acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
    __builtin_memcpy(to, &r, 16);
}

// out = sum_c 2^(m_c - M) o_c / sum_c 2^(m_c - M) l_c over a row's chunks, for segments of more than one. It is latency that this
// kernel spends, so a workgroup takes 64 dims of a (row, head) (32 where hd is no multiple of 64), a thread four dims of every 16th
// (32nd) chunk; the 16 (32) sums meet in order. 24 rows of 128 chunks, hd 256: 4 us; one workgroup of four waves for a row took 11.
template <int HD, int NT>
__global__ __launch_bounds__(256) void attention4_merge_kernel(const float *__restrict__ part, const float *__restrict__ pml,
                                                               float *__restrict__ out, SegTable T, Cuts C, Starts R, int heads,
                                                               int G, int bidirectional, int window) {
    constexpr int Q = HD % 64 == 0 ? 16 : 8, GROUPS = 256 / Q;
    __shared__ float sm[GROUPS], sl[GROUPS];
    __shared__ float4 sacc[GROUPS][Q];
    const int tid = threadIdx.x, lane = tid & 63, grp = tid / Q, quad = tid - grp * Q;
    const int row = blockIdx.x / heads, h = blockIdx.x - row * heads, d = 4 * (Q * blockIdx.y + quad);
    const int chunks = C.first[lane], bases = C.base[lane];
    const Found found = find_segment(T, R.first, R.total, row);
    const RowChunks r = row_chunks<NT>(found, T, C, chunks, bases, row, heads, G, bidirectional, window);
    if (r.n == 1) return;
    const size_t at = r.at + static_cast<size_t>(h) * r.n;
    float m, L;
    float4 acc = merge_parts<HD>(part + at * HD + d, pml + 2 * at, r.lo + grp, r.hi, GROUPS, m, L);
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
        const float f = share(sm[w], m);
        L = fmaf(sl[w], f, L);
        acc.x = fmaf(a.x, f, acc.x);
        acc.y = fmaf(a.y, f, acc.y);
        acc.z = fmaf(a.z, f, acc.z);
        acc.w = fmaf(a.w, f, acc.w);
    }
    put_merged(out + (static_cast<size_t>(found.s.row0 + r.t) * heads + h) * HD + d, acc, L);
}
// The same for up to kFewChunks chunks: a thread takes four dims of a head, workgroups (row, 1024 values of it).
constexpr int kFewChunks = 8;
template <int HD, int NT>
__global__ __launch_bounds__(256) void attention4_merge_few_kernel(const float *__restrict__ part, const float *__restrict__ pml,
                                                                   float *__restrict__ out, SegTable T, Cuts C, Starts R, int heads,
                                                                   int G, int bidirectional, int window) {
    const int lane = threadIdx.x & 63, row = blockIdx.x;
    const int chunks = C.first[lane], bases = C.base[lane];
    const Found found = find_segment(T, R.first, R.total, row);
    const RowChunks r = row_chunks<NT>(found, T, C, chunks, bases, row, heads, G, bidirectional, window);
    const int e = blockIdx.y * 256 + threadIdx.x, h = e / (HD / 4), d = 4 * (e - h * (HD / 4));
    if (r.n == 1 || h >= heads) return;
    const size_t at = r.at + static_cast<size_t>(h) * r.n;
    float m, L;
    const float4 acc = merge_parts<HD>(part + at * HD + d, pml + 2 * at, r.lo, r.hi, 1, m, L);
    put_merged(out + (static_cast<size_t>(found.s.row0 + r.t) * heads + h) * HD + d, acc, L);
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

// Chunks for the 512 workgroups that run at once (two per CU): of the lengths that make one to four full rounds, and of whole
// contexts, the one with the least rounds x (keys of a chunk + what a chunk costs besides, in keys: its start and end, 160 keys' time,
// and with more than one chunk the partial results of a group, 100 for each tile).
struct Shape {
    int heads, kv_heads, tiles;
    int groups(const Seg &s) const { return (s.rows * (heads / kv_heads) + 16 * tiles - 1) / (16 * tiles); }
};
int keys_of(const Seg &s, int window) { return s.pos0 + s.rows - first_key(s, window); }
int chunks_of(const Seg &s, long long len, int window) { return static_cast<int>((keys_of(s, window) + len - 1) / len); }
Cuts make_cuts(const SegTable &T, const Shape &P, int window, bool whole) {
    constexpr long long kSlots = 512, kFixed = 160, kPart = 100;
    long long most = 0, work = 0;
    for (int i = 0; i < T.n; ++i) {
        most = max(most, static_cast<long long>(keys_of(T.s[i], window)));
        work += static_cast<long long>(keys_of(T.s[i], window)) * P.groups(T.s[i]) * P.kv_heads;
    }
    most = (most + 127) / 128 * 128;
    auto count = [&](long long len) {
        long long n = 0;
        for (int i = 0; i < T.n; ++i) n += static_cast<long long>(chunks_of(T.s[i], len, window)) * P.groups(T.s[i]);
        return n * P.kv_heads;
    };
    auto cost = [&](long long len) { return (count(len) + kSlots - 1) / kSlots * (len + kFixed + (len < most ? kPart * P.tiles : 0)); };
    long long best = most;
    for (int rounds = 1; rounds <= 4 && !whole; ++rounds) {
        long long lo = max(work / (kSlots * rounds) / 128, 1LL), hi = most / 128;  // the least length of at most that many rounds
        while (lo < hi) {
            const long long mid = (lo + hi) / 2;
            if (count(128 * mid) > kSlots * rounds) lo = mid + 1;
            else hi = mid;
        }
        if (128 * lo < most && cost(128 * lo) < cost(best)) best = 128 * lo;
    }
    Cuts C;
    C.len = static_cast<int>(best);
    C.total = C.most = 0;
    int base = 0;
    for (int i = 0; i < VQ_MAX_SEGMENTS; ++i) {
        C.first[i] = C.total;
        C.base[i] = base;
        if (i >= T.n) continue;
        const int n = chunks_of(T.s[i], C.len, window);
        if (n > 1) base += n * T.s[i].rows * P.heads;
        C.total += n * P.groups(T.s[i]);
        C.most = max(C.most, n);
    }
    return C;
}
// Partial results of the pass: vectors x chunks where a segment has more than one.
size_t parts_of(const SegTable &T, const Cuts &C, int heads, int window) {
    size_t n = 0;
    for (int i = 0; i < T.n; ++i) {
        const size_t k = chunks_of(T.s[i], C.len, window);
        if (k > 1) n += k * T.s[i].rows * heads;
    }
    return n;
}
// Two tiles to a group where a kv head has more than 16 query vectors in a segment; always without a workspace, so that a row's sums
// are the same in every pass.
Shape shape_of(const SegTable &T, int heads, int kv_heads, bool whole) {
    return Shape{heads, kv_heads, whole || max_seg_rows(T) * (heads / kv_heads) > 16 ? 2 : 1};
}
size_t attention4_ws_bytes(const SegTable &T, int heads, int kv_heads, int hd, int window) {
    const Cuts C = make_cuts(T, shape_of(T, heads, kv_heads, false), window, false);
    return parts_of(T, C, heads, window) * (hd + 2) * 4 + 16;
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
    if (static_cast<long long>(T.total) * heads > INT32_MAX / 2) return VQ_ERR_SHAPE;
    const bool whole = ws == nullptr;
    const Shape P = shape_of(T, heads, M.kv_heads, whole);
    const Cuts C = make_cuts(T, P, window, whole);
    const size_t parts = parts_of(T, C, heads, window);
    if (!whole && ((reinterpret_cast<uintptr_t>(ws) & 15) || ws_bytes < parts * (hd + 2) * 4 + 16)) return VQ_ERR_WORKSPACE;
    const Starts R = starts_of(T, rows_of, 0);
    auto *kb = static_cast<const uint8_t *>(kc), *vb = static_cast<const uint8_t *>(vc);
    float *part = static_cast<float *>(ws), *pml = part + parts * hd;
    const dim3 grid(static_cast<unsigned>(C.total) * M.kv_heads);
    auto pass = [&](auto u, auto tiles) {
        constexpr int U = decltype(u)::value, NT = decltype(tiles)::value;
        auto go = [&](auto kernel) { kernel<<<grid, 256, 0, s>>>(q, kb, vb, part, pml, out, T, M, C, heads, bidirectional, window); };
        // hd 128 and 256 by DMA but for pages of odd numbers of slabs.
        bool done = false;
        if constexpr (U % 4 == 0) {
            done = true;
            if (!M.pt) go(attention4_kernel<U, NT, 0>);
            else if (M.spp % 4 == 0) go(attention4_kernel<U, NT, 4>);
            else if (M.spp % 2 == 0) go(attention4_kernel<U, NT, 2>);
            else done = false;
        }
        if (!done && M.pt) go(attention4_kernel<U, NT, -1>);
        if constexpr (U % 4 != 0)
            if (!M.pt) go(attention4_kernel<U, NT, -2>);
        auto merge = [&](auto kernel, const dim3 &rows) {
            kernel<<<rows, 256, 0, s>>>(part, pml, out, T, C, R, heads, heads / M.kv_heads, bidirectional, window);
        };
        if (parts && C.most > kFewChunks) merge(attention4_merge_kernel<32 * U, NT>, dim3(T.total * heads, U % 2 == 0 ? U / 2 : U));
        else if (parts) merge(attention4_merge_few_kernel<32 * U, NT>, dim3(T.total, (heads * 8 * U + 255) / 256));
    };
    for_hd(hd, [&](auto u) {
        if (P.tiles == 1) pass(u, std::integral_constant<int, 1>{});
        else pass(u, std::integral_constant<int, 2>{});
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
