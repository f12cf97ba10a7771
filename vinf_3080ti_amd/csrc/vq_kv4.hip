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
// once, and the found one's values come from its lane: kernel arguments lie in host memory, and loads that wait for each other (a walk
// over the segments, then their rows, then their bases) would each pay that way.
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
// written for a (k, v) pair; 4001 tokens of 4 heads of 256, 42 MB, in 11.8 us.
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
typedef float ff2 __attribute__((ext_vector_type(2)));

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

__device__ __forceinline__ float max3_abs(float m, float a, float b) {
    asm("v_max3_f32 %0, %1, |%2|, |%3|" : "=v"(m) : "v"(m), "v"(a), "v"(b));
    return m;
}
// A query vector goes in as f16 pairs hi + lo (22 significant bits) of its elements times a power of two that brings the largest,
// `amax`, near 2^14. Returns that power; `unit` takes a product back and into base-2 units of the softmax, log2(e) / sqrt(hd) over it.
template <int U>
__device__ __forceinline__ float query_scale(float amax, float &unit) {
    // amax = f 2^ex, f in [0.5, 1). Capped at 2^126, so that the power and its inverse are finite for the smallest queries.
    const int ex = amax > 0.0f && amax <= 3.0e38f ? __builtin_amdgcn_frexp_expf(amax) : 0, e2 = 14 - ex < 126 ? 14 - ex : 126;
    unit = ldexpf(1.44269504088896341f / sqrtf(32.0f * U), -e2);
    return ldexpf(1.0f, e2);
}
__device__ __forceinline__ void split_query(const float (&x)[8], float up, fh8 &h, fh8 &l) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        _Float16 hi, lo;
        split_h(x[j] * up, hi, lo);
        h[j] = hi;
        l[j] = lo;
    }
}

// Softmax step over a lane's N products s of a block (masked ones are -inf), which times `unit` are scores in base-2 units: new
// reference m and sum, the factor for what was summed before, the weights 2^(score - m) as f16 pairs. m is the running maximum
// less kLift and follows only when the maximum is past m + kMost, since the sums' rescaling costs as much as the step: a row's
// largest weight lies between 2^kLift and 2^kMost, near the top of f16's range. So a weight is off by 2^-23 of itself or, where
// its second half is an f16 below the normal ones, by 2^-25, at most 2^-(25 + kLift) of the largest. Both halves are rounded to
// nearest: sums over thousands of keys would add up what rounding towards zero takes from each. 2048 keys, all but one of them
// 14 nats below that one, whose value is zero: 2e-7 to 5e-7 of the result, with kLift 7 up to 4e-5, with weights up to 1 rounded
// towards zero 1e-2. What kLift costs: 512 rows over 2048 keys take 62.8, 63.6, 65.5 us with 7, 11, 13. The sum is of the weights
// before they are split. `across`: over the lanes of a vector.
constexpr float kLift = 11.0f, kMost = 15.0f;
template <int N, typename Max, typename Add>
__device__ __forceinline__ float softmax_step(const float (&v)[N], float unit, float &m, float &l, fh8 (&ph)[N / 8], fh8 (&pl)[N / 8], Max max_across,
                                              Add add_across) {
    float bm = -INFINITY;
#pragma unroll
    for (int j = 0; j < N; ++j) bm = fmaxf(bm, v[j]);
    bm = max_across(bm) * unit;
    const float mn = bm > m + kMost ? bm - kLift : m, ms = mn == -INFINITY ? 0.0f : mn;  // ms: exp2(-inf - ms) is 0 also before any key
    const float alpha = __builtin_amdgcn_exp2f(m - ms);
    float x[N], ps = 0.0f;
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = fmaf(v[j], unit, -ms);
    // Past 2^21 the roundings of bm and m would show: an exponent could come to 16, an infinite f16, or the largest key's weight to
    // nothing. There products are rounded as bm was, which leaves the largest one an exponent of 0 or more, and exponents end at 15.
    const bool far = fabsf(mn) > 0x1p21f;
    if (__any(far)) {
#pragma clang fp contract(off)
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const float y = v[j] * unit - ms;
            x[j] = far ? (y > kMost ? kMost : y) : x[j];  // (NaN stays)
        }
    }
#pragma unroll
    for (int j = 0; j < N; j += 2) {
        const ff2 w{__builtin_amdgcn_exp2f(x[j]), __builtin_amdgcn_exp2f(x[j + 1])};
        ps += w[0];
        ps += w[1];
        const fh2 hi = __builtin_convertvector(w, fh2);
        const fh2 lo = __builtin_convertvector((ff2{w[0] - static_cast<float>(hi[0]), w[1] - static_cast<float>(hi[1])}), fh2);
        ph[j / 8][j % 8] = hi[0], ph[j / 8][j % 8 + 1] = hi[1];
        pl[j / 8][j % 8] = lo[0], pl[j / 8][j % 8 + 1] = lo[1];
    }
    l = l * alpha + add_across(ps);
    m = mn;
    return alpha;
}

// How a pass is cut: each segment's query vectors in groups of 16 or 32, its keys in chunks of `len` (a multiple of 128) from its first
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

// ---- blocks by DMA ----

// For hd 128 and 256, whose waves are few (hd 256: 2 per SIMD, for the registers of O and q): the blocks come to LDS by DMA, kSlots of
// them for each wave, so that the loads of one are in flight while another is computed with, and no registers are spent on them. A
// slot is K's words, slab after slab, V's words, and 512 bytes each of K's and of V's headers, slab after slab. Page ids and
// addresses are wave-uniform and come by scalar loads: the only vector memory operations of the loop are the DMA's, which the waits
// count.
template <int U, int VECS>
struct Ring {
    static constexpr int kSlots = (U == 8 ? 2 : 3) - (VECS == 32);
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
// At most N loads outstanding, for the few N that occur.
__device__ __forceinline__ void wait_loads(int n) {
    switch (n) {
        case 0: vq::wait_vm<0>(); break;
        case 5: vq::wait_vm<5>(); break;
        case 9: vq::wait_vm<9>(); break;
        default: vq::wait_vm<10>(); break;
    }
}

// ---- a wave's tile of query vectors: 16 or 32 ----

// Every lane needs the headers of all groups of its V slabs: 4 U lanes take a slab's group apart each and the others read them from
// LDS ([slab][group] scales, zero points, the wave's own; moving them by DPP costs 64 instructions a block of the kind that bounds
// this kernel).
template <int U>
constexpr int head_words = 4 * (8 * U + 8);
struct Heads2 {
    fh2 d[4], z[4];
};
__device__ __forceinline__ void put_heads(const uint4 &raw, uint32_t *to) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    uint32_t d[4], z[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) d[i] = w[i] & 0xFFF0FFF0u, z[i] = __builtin_bit_cast(uint32_t, zeros2(w[i], i % 2 != 0));
    *reinterpret_cast<uint4 *>(to) = uint4{d[0], d[1], d[2], d[3]};
    *reinterpret_cast<uint4 *>(to + 4) = uint4{z[0], z[1], z[2], z[3]};
}
__device__ __forceinline__ Heads2 get_heads(const uint32_t *from) {
    const uint4 x = *reinterpret_cast<const uint4 *>(from), y = *reinterpret_cast<const uint4 *>(from + 4);
    return Heads2{{__builtin_bit_cast(fh2, x.x), __builtin_bit_cast(fh2, x.y), __builtin_bit_cast(fh2, x.z), __builtin_bit_cast(fh2, x.w)},
                  {__builtin_bit_cast(fh2, y.x), __builtin_bit_cast(fh2, y.y), __builtin_bit_cast(fh2, y.z), __builtin_bit_cast(fh2, y.w)}};
}
// Of a slab's V headers those of positions below `to`: what lies behind the last key may never have been written, and a weight of zero
// does not take away a scale that is no number.
__device__ __forceinline__ uint4 heads_below(const uint4 &raw, int pos, int to) {
    uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] &= (pos + 2 * i < to ? 0xFFFFu : 0u) | (pos + 2 * i + 1 < to ? 0xFFFF0000u : 0u);
    return uint4{w[0], w[1], w[2], w[3]};
}
// A wave's LDS operations complete in order; the fence keeps the compiler from moving them over each other.
__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// 16 vectors by v_mfma_f32_16x16x32_f16: lane l = (c = l & 15, g = l >> 4) gives row c of A and column c of B at the same eight k
// slots (g, j); the result has rows 4 g + r, column c. Over a block of 32 keys:
//  - S^T of key half h: A row c is key 8 (c >> 2) + 4 h + (c & 3), dims 32 u + 8 g + j (one K word); lane (c, g) ends with the
//    scores of keys 8 g + 4 h + r of query vector c.
//  - O^T += V^T P^T: k slot (g, j) is key 8 g + j, so B is the lane's own eight weights in order and A, dims 16 b + c of V^T at
//    positions 8 g .. 8 g + 7, is one V word of slab g.
template <int U>
struct Tile16 {
    static constexpr int kVecs = 16, kQueryLds = 0;
    uint32_t k[2][U], kh[2][(U + 1) / 2], v[2 * U];
    uint4 vh;
    fh8 qh[U], ql[U];
    float unit, m, l;
    fa4 o[2 * U];

    static __device__ __forceinline__ int lane() { return threadIdx.x & 63; }
    static __device__ __forceinline__ int vec() { return lane() & 15; }
    static __device__ __forceinline__ int key(int h) { return 8 * (vec() >> 2) + 4 * h + (vec() & 3); }
    static __device__ __forceinline__ int kslab() { return vec() >> 2; }
    __device__ __forceinline__ void clear() {
        m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int b = 0; b < 2 * U; ++b) o[b] = fa4{0.f, 0.f, 0.f, 0.f};
    }
    __device__ __forceinline__ void no_page() {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < (U + 1) / 2; ++i) kh[h][i] = kNanHeader | kNanHeader << 16;
    }
    // 230 instructions at hd 256: a short context's workgroup runs this once for a block or two.
    __device__ __forceinline__ void load_query(const float *qrow, uint8_t *) {
        const int g = lane() >> 4;
        float x[U][8], amax = 0.0f;
#pragma unroll
        for (int u = 0; u < U; ++u) __builtin_memcpy(x[u], qrow + 32 * u + 8 * g, 32);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < 8; j += 2) amax = max3_abs(amax, x[u][j], x[u][j + 1]);
        const float up = query_scale<U>(xor32_max(xor16_max(amax)), unit);
#pragma unroll
        for (int u = 0; u < U; ++u) split_query(x[u], up, qh[u], ql[u]);
    }
    // From the cache: `at(slab)` is the place of a slab of the block.
    template <typename At>
    __device__ __forceinline__ void issue_k(const uint8_t *__restrict__ kc, At at) {
        const SlabAt p = at(kslab());
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int row = key(h) & 7;
            ld_words<U>(kc + p.words + row * (16 * U) + (lane() >> 4) * (4 * U), k[h]);
            ld_heads<U>(kc + p.heads + row * (2 * U), kh[h]);
        }
        if (p.bad) no_page();
    }
    template <typename At>
    __device__ __forceinline__ void issue_v(const uint8_t *__restrict__ vc, At at) {
        constexpr int W = U % 2 == 0 ? 4 : 2;
        const SlabAt p = at(lane() >> 4);
#pragma unroll
        for (int i = 0; i < 2 * U / W; ++i) {
            uint32_t w[W];
            ld_words<W>(vc + p.words + (16 * i + vec()) * (4 * W), w);
#pragma unroll
            for (int x = 0; x < W; ++x) v[W * i + x] = w[x];
        }
        vh = *reinterpret_cast<const uint4 *>(vc + p.heads + 16 * min(vec(), U - 1));
    }
    // From a slot.
    __device__ __forceinline__ void read_k(const uint8_t *words, const uint8_t *heads) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < U / 4; ++i) {
                const uint4 w = *reinterpret_cast<const uint4 *>(words + (16 * U) * key(h) + 16 * ((U / 4 * (lane() >> 4) + i) ^ swizzle<U>(key(h))));
                k[h][4 * i] = w.x, k[h][4 * i + 1] = w.y, k[h][4 * i + 2] = w.z, k[h][4 * i + 3] = w.w;
            }
            ld_words<U / 2>(heads + key(h) * (2 * U), kh[h]);
        }
    }
    __device__ __forceinline__ void read_v(const uint8_t *words, const uint8_t *heads) {
        const int g = lane() >> 4;
#pragma unroll
        for (int i = 0; i < U / 2; ++i) {
            const uint4 w = *reinterpret_cast<const uint4 *>(words + (128 * U) * g + 256 * i + 16 * vec());
            v[4 * i] = w.x, v[4 * i + 1] = w.y, v[4 * i + 2] = w.z, v[4 * i + 3] = w.w;
        }
        vh = *reinterpret_cast<const uint4 *>(heads + 16 * (g * U + min(vec(), U - 1)));
    }
    // A block's scores and its share of the sums; `between`: what is done when K's registers are free, `values`: V's come, under the
    // softmax.
    template <typename Between, typename Values>
    __device__ __forceinline__ void block(int kb, int k_hi, const Sees &see, const uint8_t *, uint32_t *heads, Between between, Values values) {
        const int g = lane() >> 4;
        fa4 s[2] = {fa4{0.f, 0.f, 0.f, 0.f}, fa4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const fh8 a = u % 2 == 0 ? decode8_one<false>(k[h][u], kh[h][u / 2]) : decode8_one<true>(k[h][u], kh[h][u / 2]);
                s[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qh[u], s[h], 0, 0, 0);
                s[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ql[u], s[h], 0, 0, 0);
            }
        between();
        values();
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = s[j >> 2][j & 3];
        if (__any(kb < see.from || kb + 32 > see.to)) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int p = kb + 8 * g + j;
                x[j] = p >= see.from && p < see.to ? x[j] : -INFINITY;
            }
        }
        fh8 ph[1], pl[1];
        const float alpha = softmax_step<8>(x, unit, m, l, ph, pl, [](float y) { return xor32_max(xor16_max(y)); },
                                            [](float y) { return xor32_add(xor16_add(y)); });
        if (__any(alpha != 1.0f)) {
#pragma unroll
            for (int b = 0; b < 2 * U; ++b) o[b] *= alpha;
        }
        uint32_t *mine = heads + g * (8 * U + 8);
        if (kb + 32 > k_hi) vh = heads_below(vh, kb + 8 * g, k_hi);
        if (vec() < U) put_heads(vh, mine + 8 * vec());
        wave_lds_fence();
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const Heads2 z = get_heads(mine + 8 * u);
#pragma unroll
            for (int b = 2 * u; b < 2 * u + 2; ++b) {
                const fh8 a = decode8(v[b], z.d, z.z);
                o[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ph[0], o[b], 0, 0, 0);
                o[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, pl[0], o[b], 0, 0, 0);
            }
        }
        wave_lds_fence();  // every lane has read before the next block's writes
    }
    // The waves' sums ([wave][16][HD] in `sums`) meet in wave order.
    __device__ __forceinline__ void finish(float *sums, float (*sm)[32], float (*sl)[32], int j0, const Dest &to) {
        constexpr int HD = 32 * U;
        const int wv = threadIdx.x >> 6, c = vec(), g = lane() >> 4;
        if (j0 + c < to.nvec) {
#pragma unroll
            for (int b = 0; b < 2 * U; ++b) *reinterpret_cast<fa4 *>(sums + (wv * 16 + c) * HD + 16 * b + 4 * g) = o[b];
            if (g == 0) sm[wv][c] = m, sl[wv][c] = l;
        }
        __syncthreads();
        for (int e = threadIdx.x; e < 16 * (HD / 4); e += 256) {
            const int x = e / (HD / 4), d4 = 4 * (e - x * (HD / 4));
            if (j0 + x >= to.nvec) continue;
            const float mx = fmaxf(fmaxf(sm[0][x], sm[1][x]), fmaxf(sm[2][x], sm[3][x]));
            float L = 0.0f;
            float4 acc{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float f = share(sm[w][x], mx);
                L = fmaf(sl[w][x], f, L);
                const float4 p = *reinterpret_cast<const float4 *>(sums + (w * 16 + x) * HD + d4);
                acc.x = fmaf(p.x, f, acc.x);
                acc.y = fmaf(p.y, f, acc.y);
                acc.z = fmaf(p.z, f, acc.z);
                acc.w = fmaf(p.w, f, acc.w);
            }
            to.template put<HD>(j0 + x, d4, acc, mx, L);
        }
    }
};

// 32 vectors by v_mfma_f32_32x32x16_f16: lane l = (c = l & 31, g = l >> 5) gives row c of A and column c of B at the eight k slots
// (g, j); the result has rows 8 (e >> 2) + 4 g + (e & 3), e < 16, column c. Over a block of 32 keys:
//  - S^T: A row c = 8 a + 4 h + r is key 16 (a >> 1) + 8 h + 4 (a & 1) + r, dims 32 u + 16 w + 8 g + j (the K word of 2 w + g); lane
//    (c, g) ends with the scores of keys 16 x + 8 g + j at e = 8 x + j.
//  - O^T += V^T P^T of keys 16 x + 8 g + j: B is the lane's own eight weights in order, A a V word of slab 2 x + g; row c of row
//    block b is dim 16 (U (c >> 4) + b) + (c & 15), so that a lane's words are whole pieces.
// A step decodes the next one's operand while the matrix unit works (and reads its queries ahead, for hd above 128 from LDS: O is
// half of the registers of two waves per SIMD); left to itself the compiler waits for each.
typedef float fa16 __attribute__((ext_vector_type(16)));
template <int U>
struct Tile32 {
    static constexpr int kVecs = 32;
    static constexpr bool kLds = U > 4;
    static constexpr int kQueryLds = kLds ? 4096 * U : 0;  // [step][hi, lo][lane]
    uint32_t k[2][U], kh[(U + 1) / 2], v[2][U];
    uint4 vh;
    fh8 qh[kLds ? 1 : 2 * U], ql[kLds ? 1 : 2 * U];
    float unit, m, l;
    fa16 o[U];

    static __device__ __forceinline__ int lane() { return threadIdx.x & 63; }
    static __device__ __forceinline__ int vec() { return lane() & 31; }
    static __device__ __forceinline__ int half() { return lane() >> 5; }
    static __device__ __forceinline__ int key() {
        const int c = vec(), a = c >> 3;
        return 16 * (a >> 1) + 8 * (c >> 2 & 1) + 4 * (a & 1) + (c & 3);
    }
    static __device__ __forceinline__ int kslab() { return key() >> 3; }
    static __device__ __forceinline__ int hslab() { return 2 * (lane() >> 4 & 1) + half(); }  // whose headers the lane takes apart
    __device__ __forceinline__ void clear() {
        m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int b = 0; b < U; ++b)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[b][e] = 0.0f;
    }
    __device__ __forceinline__ void no_page() {
#pragma unroll
        for (int i = 0; i < (U + 1) / 2; ++i) kh[i] = kNanHeader | kNanHeader << 16;
    }
    static __device__ __forceinline__ int dim(int step) { return 16 * step + 8 * half(); }
    // In LDS a wave makes every fourth step's operands; the maxima meet there first.
    __device__ __forceinline__ void load_query(const float *qrow, uint8_t *qlds) {
        if constexpr (kLds) {
            constexpr int N = (2 * U + 3) / 4;
            __shared__ float part[4][32];
            const int wv = threadIdx.x >> 6;
            float x[N][8], amax = 0.0f;
#pragma unroll
            for (int i = 0; i < N; ++i) __builtin_memcpy(x[i], qrow + dim(min(4 * i + wv, 2 * U - 1)), 32);
#pragma unroll
            for (int i = 0; i < N; ++i)
#pragma unroll
                for (int j = 0; j < 8; j += 2) amax = max3_abs(amax, x[i][j], x[i][j + 1]);
            amax = xor32_max(amax);
            if (half() == 0) part[wv][vec()] = amax;
            __syncthreads();
            amax = fmaxf(fmaxf(part[0][vec()], part[1][vec()]), fmaxf(part[2][vec()], part[3][vec()]));
            const float up = query_scale<U>(amax, unit);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int step = 4 * i + wv;
                if (step >= 2 * U) continue;
                fh8 h, lo;
                split_query(x[i], up, h, lo);
                *reinterpret_cast<fh8 *>(qlds + 2048 * step + 16 * lane()) = h;
                *reinterpret_cast<fh8 *>(qlds + 2048 * step + 1024 + 16 * lane()) = lo;
            }
            __syncthreads();
        } else {
            float x[2 * U][8], amax = 0.0f;
#pragma unroll
            for (int i = 0; i < 2 * U; ++i) __builtin_memcpy(x[i], qrow + dim(i), 32);
#pragma unroll
            for (int i = 0; i < 2 * U; ++i)
#pragma unroll
                for (int j = 0; j < 8; j += 2) amax = max3_abs(amax, x[i][j], x[i][j + 1]);
            const float up = query_scale<U>(xor32_max(amax), unit);
#pragma unroll
            for (int i = 0; i < 2 * U; ++i) split_query(x[i], up, qh[i], ql[i]);
        }
    }
    template <typename At>
    __device__ __forceinline__ void issue_k(const uint8_t *__restrict__ kc, At at) {
        const SlabAt p = at(kslab());
        const int row = key() & 7;
#pragma unroll
        for (int w = 0; w < 2; ++w) ld_words<U>(kc + p.words + row * (16 * U) + (2 * w + half()) * (4 * U), k[w]);
        ld_heads<U>(kc + p.heads + row * (2 * U), kh);
        if (p.bad) no_page();
    }
    template <typename At>
    __device__ __forceinline__ void issue_v(const uint8_t *__restrict__ vc, At at) {
        constexpr int W = U % 2 == 0 ? 4 : 2, L = U % 4 == 0 ? 4 : U % 2 == 0 ? 2 : 1;  // words of a piece, of a load
        const int c = vec();
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const SlabAt p = at(2 * x + half());
#pragma unroll
            for (int i = 0; i < U / L; ++i) {
                const int f = U * (c >> 4) + L * i;
                uint32_t w[L];
                ld_words<L>(vc + p.words + (16 * (f / W) + (c & 15)) * (4 * W) + f % W * 4, w);
#pragma unroll
                for (int y = 0; y < L; ++y) v[x][L * i + y] = w[y];
            }
        }
        vh = *reinterpret_cast<const uint4 *>(vc + at(hslab()).heads + 16 * min(c & 15, U - 1));
    }
    __device__ __forceinline__ void read_k(const uint8_t *words, const uint8_t *heads) {
#pragma unroll
        for (int w = 0; w < 2; ++w)
#pragma unroll
            for (int i = 0; i < U / 4; ++i) {
                const uint4 x = *reinterpret_cast<const uint4 *>(words + (16 * U) * key() + 16 * ((U / 4 * (2 * w + half()) + i) ^ swizzle<U>(key())));
                k[w][4 * i] = x.x, k[w][4 * i + 1] = x.y, k[w][4 * i + 2] = x.z, k[w][4 * i + 3] = x.w;
            }
        ld_words<U / 2>(heads + key() * (2 * U), kh);
    }
    __device__ __forceinline__ void read_v(const uint8_t *words, const uint8_t *heads) {
        const int c = vec();
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int i = 0; i < U / 4; ++i) {
                const uint4 w = *reinterpret_cast<const uint4 *>(words + (128 * U) * (2 * x + half()) + 256 * (U / 4 * (c >> 4) + i) + 16 * (c & 15));
                v[x][4 * i] = w.x, v[x][4 * i + 1] = w.y, v[x][4 * i + 2] = w.z, v[x][4 * i + 3] = w.w;
            }
        vh = *reinterpret_cast<const uint4 *>(heads + 16 * (hslab() * U + min(c & 15, U - 1)));
    }
    template <typename Between, typename Values>
    __device__ __forceinline__ void block(int kb, int k_hi, const Sees &see, const uint8_t *qlds, uint32_t *heads, Between between, Values values) {
        fa16 s;
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = 0.0f;
        fh8 q[2][2], a[2];
        auto query = [&](int i) {
            if constexpr (kLds) {
#pragma unroll
                for (int x = 0; x < 2; ++x) q[i & 1][x] = *reinterpret_cast<const fh8 *>(qlds + 2048 * i + 1024 * x + 16 * lane());
            } else {
                q[i & 1][0] = qh[i], q[i & 1][1] = ql[i];
            }
        };
        auto keys = [&](int i) {
            const int u = i >> 1, w = i & 1;
            a[i & 1] = u % 2 == 0 ? decode8_one<false>(k[w][u], kh[u / 2]) : decode8_one<true>(k[w][u], kh[u / 2]);
        };
        query(0);
        keys(0);
#pragma unroll
        for (int i = 0; i < 2 * U; ++i) {
            __builtin_amdgcn_sched_barrier(0);
            if (i + 1 < 2 * U) query(i + 1), keys(i + 1);
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[i & 1], q[i & 1][0], s, 0, 0, 0);
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[i & 1], q[i & 1][1], s, 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        between();
        values();
        float x[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = s[e];
        if (__any(kb < see.from || kb + 32 > see.to)) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int p = kb + 16 * (e >> 3) + 8 * half() + (e & 7);
                x[e] = p >= see.from && p < see.to ? x[e] : -INFINITY;
            }
        }
        fh8 ph[2], pl[2];
        const float alpha = softmax_step<16>(x, unit, m, l, ph, pl, [](float y) { return xor32_max(y); }, [](float y) { return xor32_add(y); });
        if (__any(alpha != 1.0f)) {
#pragma unroll
            for (int b = 0; b < U; ++b) o[b] *= alpha;
        }
        if (kb + 32 > k_hi) vh = heads_below(vh, kb + 8 * hslab(), k_hi);
        if ((lane() & 15) < U) put_heads(vh, heads + hslab() * (8 * U + 8) + 8 * (lane() & 15));
        wave_lds_fence();
        // Step i: row block i % U of keys 16 (i / U). Headers are read two steps ahead.
        Heads2 z[2];
        auto header = [&](int i) {
            const int xx = i / U, b = i % U;
            if (U % 2 != 0 || b % 2 == 0)
                z[U % 2 != 0 ? i & 1 : i >> 1 & 1] = get_heads(heads + (2 * xx + half()) * (8 * U + 8) + 8 * ((U * (vec() >> 4) + b) >> 1));
        };
        auto value = [&](int i) {
            const Heads2 &y = z[U % 2 != 0 ? i & 1 : i >> 1 & 1];
            a[i & 1] = decode8(v[i / U][i % U], y.d, y.z);
        };
        header(0);
        if (U % 2 != 0) header(1);
        value(0);
#pragma unroll
        for (int i = 0; i < 2 * U; ++i) {
            const int xx = i / U, b = i % U;
            __builtin_amdgcn_sched_barrier(0);
            if (i + 2 < 2 * U) header(i + 2);
            if (i + 1 < 2 * U) value(i + 1);
            o[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[i & 1], ph[xx], o[b], 0, 0, 0);
            o[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[i & 1], pl[xx], o[b], 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        wave_lds_fence();
    }
    // Waves 2 and 3 hand their sums to waves 0 and 1, then those two exchange half of the dims each: result rows 16 i .. of every row
    // block, e = 8 i .. 8 i + 7. A lane reads what the same lane of the other wave wrote.
    __device__ __forceinline__ void finish(float *sums, float (*sm)[32], float (*sl)[32], int j0, const Dest &to) {
        constexpr int HD = 32 * U;
        const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = vec();
        auto give = [&](float *box, int i) {
#pragma unroll
            for (int b = 0; b < U; ++b)
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const int e = 8 * i + 4 * y;
                    *reinterpret_cast<fa4 *>(box + 512 * b + 256 * y + 4 * lane()) = fa4{o[b][e], o[b][e + 1], o[b][e + 2], o[b][e + 3]};
                }
        };
        // o and the other wave's sums under their shares; `first`: the other's count as the left operand.
        auto take = [&](const float *box, int i, float own, float other, bool first) {
#pragma unroll
            for (int b = 0; b < U; ++b)
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const fa4 x = *reinterpret_cast<const fa4 *>(box + 512 * b + 256 * y + 4 * lane());
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float mine = o[b][8 * i + 4 * y + e];
                        o[b][8 * i + 4 * y + e] = first ? fmaf(mine, own, x[e] * other) : fmaf(x[e], other, mine * own);
                    }
                }
        };
        auto stats = [&](int from, bool first, float &own, float &other) {
            const float om = sm[from][c], ol = sl[from][c], mx = fmaxf(m, om);
            own = share(m, mx), other = share(om, mx);
            l = first ? fmaf(l, own, ol * other) : fmaf(ol, other, l * own);
            m = mx;
        };
        float *const box = sums + (wv & 1) * 32 * HD;  // of waves wv and wv ^ 2
        float own, other;
        if (wv >= 2) {
            give(box, 0), give(box + 16 * HD, 1);
            if (half() == 0) sm[wv][c] = m, sl[wv][c] = l;
        }
        __syncthreads();
        if (wv < 2) {
            stats(wv + 2, false, own, other);
            take(box, 0, own, other, false), take(box + 16 * HD, 1, own, other, false);
            give(box, 1 - wv);
            if (half() == 0) sm[wv][c] = m, sl[wv][c] = l;
        }
        __syncthreads();
        if (wv >= 2) return;
        const float *theirs = sums + (1 - wv) * 32 * HD;
        stats(1 - wv, wv == 1, own, other);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (wv != i) continue;
            take(theirs, i, own, other, i == 1);
            if (j0 + c >= to.nvec) continue;
#pragma unroll
            for (int b = 0; b < U; ++b)
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const int e = 8 * i + 4 * y;
                    to.template put<HD>(j0 + c, 16 * (U * i + b) + 8 * y + 4 * half(), float4{o[b][e], o[b][e + 1], o[b][e + 2], o[b][e + 3]}, m, l);
                }
        }
    }
};
template <int U, int VECS>
using Tile = std::conditional_t<VECS == 16, Tile16<U>, Tile32<U>>;

// One workgroup of four waves per (chunk of keys, kv head, group of VECS query vectors); vector j of a segment is (row j / G, head
// j % G of the kv head's group). The waves take the 32-key blocks in turn (wave w those whose index is w modulo 4, whatever the
// chunk: with one chunk a row's sums do not depend on the other rows of its pass), decode them once into MFMA operands for all of
// the group's vectors, with an online softmax, and meet at the end.
//
// Bound by vector instructions: at hd 256 500 a block and wave for the 16384 values decoded, 140 more for 16 vectors, beside 64 MFMAs
// of 16 cycles. So groups of more than 16 vectors take 32, by the larger MFMA, which halves the issue slots of the products and the
// keys' header work. Keys by LDS tiles decoded once for 64 vectors (8 waves, a barrier per 64 keys) took 94 us for 512 rows over
// 2048 keys, its two waves per SIMD in step; 32 vectors as two tiles of 16 70, this 61.
// MODE: see Slab4; -1 and -2: blocks by vector loads, in pages and contiguous.
template <int U, int VECS, int MODE>
__global__ __launch_bounds__(256, 2) void attention4_kernel(const float *__restrict__ q, const uint8_t *__restrict__ kc,
                                                            const uint8_t *__restrict__ vc, float *__restrict__ part,
                                                            float *__restrict__ pml, float *__restrict__ out, SegTable T, Map4 M, Cuts C,
                                                            int heads, int bidirectional, int window) {
    using Tile = Tile<U, VECS>;
    using Ring = Ring<U, VECS>;
    constexpr bool DMA = MODE >= 0;
    constexpr int HD = 32 * U, S = DMA ? Ring::kSlots : 1, LD = Ring::kLoads, WORDS = Ring::kWords;
    // One slot only: its K part and its V part are filled again each as soon as it has been read.
    constexpr bool SPLIT = DMA && S == 1;
    constexpr int BYTES = Ring::kBytes, RING = DMA ? S * BYTES : 0, QB = Tile::kQueryLds, SUMS = 256 * HD;
    __shared__ __align__(16) uint8_t lds[4 * RING + QB > SUMS ? 4 * RING + QB : SUMS];
    __shared__ float sm[4][32], sl[4][32];
    __shared__ __align__(16) uint32_t vheads[4][head_words<U>];
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int bases = C.base[lane];
    // The first workgroups, one to a CU, are joined by those past 256. Where that leaves some CUs with one, it is a prompt's longest
    // groups that are alone: the first and the last of the launch take the end of the list, which holds the shorter ones. 512 rows
    // over 2048 keys: 70.4 instead of 72.1 us, 480 over 480: 21.4 and 23.4. With several prompts the end of the list holds shorter and
    // longer ones: 256 and 256 rows over 2048 keys take 69 us either way, 300 and 300 over 800 34.0 and 34.3 with it.
    int unit = blockIdx.x;
    if (VECS != 16 && T.n == 1 && gridDim.x > 256 && gridDim.x < 512) {
        const int twice = gridDim.x - 256;
        unit = unit < twice ? gridDim.x - 1 - unit : unit - twice;
    }
    const Found found = find_segment(T, C.first, C.total, unit / M.kv_heads);
    const Seg s = found.s;
    const int G = heads / M.kv_heads, nvec = s.rows * G, units = found.next - found.first;
    // A segment's kv heads x chunks x groups. One tile of 16 holds its vectors whole; of several groups (the last rows, which see the
    // most keys, first) those of a head and chunk go to one XCD, for its L2: eight heads and chunks at a time, then the rest.
    const int at = unit - found.first * M.kv_heads;
    const int groups = VECS == 16 ? 1 : (nvec + VECS - 1) / VECS, n = VECS == 16 ? units : units / groups;
    int stream = at, group = 0;
    if (VECS != 16) {
        const int streams = n * M.kv_heads, rest = streams & 7, eights = (streams - rest) * groups;
        if (at < eights) {
            const int block = at / (8 * groups), x = at - block * 8 * groups;
            group = x >> 3, stream = 8 * block + (x & 7);
        } else {
            group = (at - eights) / rest, stream = streams - rest + (at - eights) - group * rest;
        }
        group = groups - 1 - group;
    }
    const int ci = stream / M.kv_heads, kvh = stream - ci * M.kv_heads, j0 = group * VECS;
    const Sees lo = sees(s, VECS == 16 ? 0 : j0 / G, bidirectional, window);
    const Sees hi = sees(s, VECS == 16 ? s.rows - 1 : min(j0 + VECS - 1, nvec - 1) / G, bidirectional, window);
    const int c_lo = first_key(s, window) + ci * C.len;
    const int k_lo = max(c_lo, lo.from & ~31), k_hi = n == 1 ? hi.to : min(c_lo + C.len, hi.to), last = (k_hi - 1) / kSlab;
    if (k_lo >= k_hi) return;
    int kb = k_lo + 32 * ((wv - (k_lo >> 5)) & 3);
    uint8_t *const ring = lds + wv * RING, *const qlds = lds + 4 * RING;
    Tile tile;
    uint32_t bad = 0;  // four bits a slot
    // Slabs past the last key's: that one is read (their keys are masked).
    auto place_in = [&](int block) { return [&, block](int slab) { return slab_at<U, MODE == -1>(M, s.slot, kvh, min(block / kSlab + slab, last)); }; };
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
            tile.issue_k(kc, place_in(block));
            tile.issue_v(vc, place_in(block));
        }
    };
    if (kb < k_hi) fetch(kb, 0);
    // Vectors past the last one repeat it; they are not written.
    const int j = min(j0 + Tile::vec(), nvec - 1), t = j / G;
    Sees see = sees(s, t, bidirectional, window);
    see.to = min(see.to, k_hi);
    tile.load_query(q + (static_cast<size_t>(s.row0 + t) * heads + kvh * G + j - t * G) * HD, qlds);
    tile.clear();
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
            Slab4 where{};
            if constexpr (DMA) {
                // Landed: all but the blocks behind this one (one slot: this one's V). One slot: the page of the block that comes into
                // it meanwhile.
                if (SPLIT && more) where = look_up<U, MODE>(M, s.slot, kvh, kb + 128 * S, last);
                if (SPLIT) asm volatile("" : "+s"(where.words0), "+s"(where.heads0));  // (before K's reads, which would wait for it)
                wait_loads(SPLIT ? LD : LD * min(left, S - 1));
                tile.read_k(from, from + 2 * WORDS);
                if (MODE != 0 && bad != 0 && (bad >> (4 * slot + Tile::kslab()) & 1)) tile.no_page();
            }
            tile.block(
                kb, k_hi, see, qlds, vheads[wv],
                [&] {
                    if (!more) return;
                    if constexpr (SPLIT) {
                        vq::wait_lgkm0();  // the part has been read
                        dma_words<U, MODE, true>(kc, where, from);
                        dma_heads<U, MODE>(kc, vc, where, from + 2 * WORDS, true, false);
                        bad = (bad & ~(15u << 4 * slot)) | where.bad << 4 * slot;
                    } else if constexpr (!DMA) {
                        tile.issue_k(kc, place_in(kb + 128));
                    }
                },
                [&] {
                    if constexpr (SPLIT) wait_loads(more ? LD : 0);
                    if constexpr (DMA) tile.read_v(from + WORDS, from + 2 * WORDS + 512);
                });
            if (more) {
                if constexpr (SPLIT) {
                    vq::wait_lgkm0();
                    dma_words<U, MODE, false>(vc, where, from + WORDS);
                    dma_heads<U, MODE>(kc, vc, where, from + 2 * WORDS, false, true);
                } else if constexpr (DMA) {
                    vq::wait_lgkm0();
                    fetch(kb + 128 * S, slot);
                } else {
                    tile.issue_v(vc, place_in(kb + 128));
                }
            }
            kb += 128;
        }
    }
    __builtin_amdgcn_s_setprio(0);
    __syncthreads();  // every slot of every wave, and the queries, have been read
    tile.finish(reinterpret_cast<float *>(lds), sm, sl, j0,
                Dest{out, part, pml, static_cast<size_t>(from_lane(bases, found.index)), heads, G, kvh, s.row0, nvec, n, ci});
}

// A row's chunks: [lo, hi) of n hold its keys; the part of (row, head, chunk) is at `at` + head n + chunk.
struct RowChunks {
    int t, n, lo, hi;
    size_t at;
};
template <int VECS>
__device__ __forceinline__ RowChunks row_chunks(const Found &found, const SegTable &T, const Cuts &C, int chunks, int bases, int row, int heads, int G,
                                                int bidirectional, int window) {
    const Seg s = found.s;
    const int i = found.index, t = row - found.first;
    const int units = (i + 1 < T.n ? from_lane(chunks, i + 1 < 64 ? i + 1 : 63) : C.total) - from_lane(chunks, i);
    RowChunks r{t, VECS == 16 ? units : units / ((s.rows * G + VECS - 1) / VECS), 0, 0, 0};
    r.hi = r.n;
    if (VECS != 16) {  // (one tile of 16: every chunk has been written)
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
template <int HD, int VECS>
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
    const RowChunks r = row_chunks<VECS>(found, T, C, chunks, bases, row, heads, G, bidirectional, window);
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
// The same where chunks are few or rows many: a thread takes four dims of a head over all chunks, a workgroup 1024 values of a row.
// 64 rows of 9 chunks, 24 heads, hd 256: 5.1 us, the kernel above 10.7; 8 rows of 128 chunks: 14.3, and 4.9.
template <int HD, int VECS>
__global__ __launch_bounds__(256) void attention4_merge_few_kernel(const float *__restrict__ part, const float *__restrict__ pml,
                                                                   float *__restrict__ out, SegTable T, Cuts C, Starts R, int heads,
                                                                   int G, int bidirectional, int window) {
    const int lane = threadIdx.x & 63, row = blockIdx.x;
    const int chunks = C.first[lane], bases = C.base[lane];
    const Found found = find_segment(T, R.first, R.total, row);
    const RowChunks r = row_chunks<VECS>(found, T, C, chunks, bases, row, heads, G, bidirectional, window);
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

// Passes whose numbers stay inside 32 bits: query vectors, and the positions that a wave may step to or chunks be rounded up to.
bool fits(const SegTable &T, int heads) {
    long long rows = 0;
    for (int i = 0; i < T.n; ++i) {
        if (T.s[i].pos0 > INT32_MAX - 1024 - T.s[i].rows) return false;
        rows += T.s[i].rows;
    }
    return rows <= INT32_MAX / 2 / heads;
}
// Chunks for the 512 workgroups that run at once (two per CU): of the lengths that make one to four full rounds, and of whole
// contexts, the one with the least rounds x (keys of a chunk + what a chunk costs besides, in keys: its start and end, 160 keys' time,
// and with more than one chunk the partial results of a group, 100 for each tile). Both were found at hd 256; half and twice as much
// change decode, verification and 16 rows of a prompt at hd 64, 96, 128 and 256 by 3 % at most, mostly by less than 1.
struct Shape {
    int heads, kv_heads, vecs;
    int groups(const Seg &s) const { return (s.rows * (heads / kv_heads) + vecs - 1) / vecs; }
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
    auto cost = [&](long long len) { return (count(len) + kSlots - 1) / kSlots * (len + kFixed + (len < most ? kPart * P.vecs / 16 : 0)); };
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
// 32 vectors to a group where a kv head has more than 16 in a segment; always without a workspace, so that a row's sums
// are the same in every pass.
Shape shape_of(const SegTable &T, int heads, int kv_heads, bool whole) {
    return Shape{heads, kv_heads, whole || max_seg_rows(T) * (heads / kv_heads) > 16 ? 32 : 16};
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
    if (!fits(T, heads)) return VQ_ERR_SHAPE;
    const bool whole = ws == nullptr;
    const Shape P = shape_of(T, heads, M.kv_heads, whole);
    const Cuts C = make_cuts(T, P, window, whole);
    const size_t parts = parts_of(T, C, heads, window);
    if (!whole && ((reinterpret_cast<uintptr_t>(ws) & 15) || ws_bytes < parts * (hd + 2) * 4 + 16)) return VQ_ERR_WORKSPACE;
    const Starts R = starts_of(T, rows_of, 0);
    auto *kb = static_cast<const uint8_t *>(kc), *vb = static_cast<const uint8_t *>(vc);
    float *part = static_cast<float *>(ws), *pml = part + parts * hd;
    const dim3 grid(static_cast<unsigned>(C.total) * M.kv_heads);
    // Which merge: by rows where no thread has more than two batches of chunks, or 256 workgroups' worth of rows with up to 32 chunks.
    const bool few = C.most <= 8 || (C.most <= 32 && static_cast<long long>(T.total) * heads * hd >= 1 << 18);
    auto pass = [&](auto u, auto vecs) {
        constexpr int U = decltype(u)::value, VECS = decltype(vecs)::value;
        auto go = [&](auto kernel) { kernel<<<grid, 256, 0, s>>>(q, kb, vb, part, pml, out, T, M, C, heads, bidirectional, window); };
        // hd 128 and 256 by DMA but for pages of odd numbers of slabs.
        bool done = false;
        if constexpr (U % 4 == 0) {
            done = true;
            if (!M.pt) go(attention4_kernel<U, VECS, 0>);
            else if (M.spp % 4 == 0) go(attention4_kernel<U, VECS, 4>);
            else if (M.spp % 2 == 0) go(attention4_kernel<U, VECS, 2>);
            else done = false;
        }
        if (!done && M.pt) go(attention4_kernel<U, VECS, -1>);
        if constexpr (U % 4 != 0)
            if (!M.pt) go(attention4_kernel<U, VECS, -2>);
        auto merge = [&](auto kernel, const dim3 &rows) {
            kernel<<<rows, 256, 0, s>>>(part, pml, out, T, C, R, heads, heads / M.kv_heads, bidirectional, window);
        };
        if (parts && !few) merge(attention4_merge_kernel<32 * U, VECS>, dim3(T.total * heads, U % 2 == 0 ? U / 2 : U));
        else if (parts) merge(attention4_merge_few_kernel<32 * U, VECS>, dim3(T.total, (heads * 8 * U + 255) / 256));
    };
    for_hd(hd, [&](auto u) {
        if (P.vecs == 16) pass(u, std::integral_constant<int, 16>{});
        else pass(u, std::integral_constant<int, 32>{});
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
    if (kv_heads < 1 || heads < kv_heads || heads % kv_heads || !hd_ok(hd) || ntok < 1 || seq_len < 1 || window < 0) return 0;
    const SegTable T = one_segment(seq_len - 1, ntok);
    return fits(T, heads) ? attention4_ws_bytes(T, heads, kv_heads, hd, window) : 0;
}

size_t vq_attention4_seg_workspace_bytes(const int32_t *segs, int nseg, int heads, int kv_heads, int hd) {
    SegTable T;
    if (make_table(segs, nseg, T, nullptr) != VQ_OK) return 0;
    if (kv_heads < 1 || heads < kv_heads || heads % kv_heads || !hd_ok(hd)) return 0;
    return fits(T, heads) ? attention4_ws_bytes(T, heads, kv_heads, hd, 0) : 0;
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
