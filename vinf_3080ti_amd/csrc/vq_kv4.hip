// vq_kv4.hip -- the KV cache in 4 bits: append, read-back and attention (layout and rounding rule: include/vq.h).
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <type_traits>

#include "../../include/vq.h"
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

// Value of dim d at a slab's position r (place from place<>(); spp and bytes of the block from M).
__device__ __forceinline__ float k_value(const uint8_t *kc, const Map4 &M, const Place &at, int r, int hd, int d) {
    const uint8_t *b = kc + at.at;
    const size_t pos = static_cast<size_t>(at.slab) * kSlab + r;
    const uint32_t w = reinterpret_cast<const uint32_t *>(b)[pos * (hd / 8) + ((d >> 3) & 3) * (hd / 32) + (d >> 5)];
    const uint16_t *h = reinterpret_cast<const uint16_t *>(b + static_cast<size_t>(M.spp) * kSlab * (hd / 2));
    return value_of(at.bad ? kNanHeader : h[pos * (hd / 32) + (d >> 5)], (w >> nib(d & 7)) & 15u);
}
__device__ __forceinline__ float v_value(const uint8_t *vc, const Map4 &M, const Place &at, int r, int hd, int d) {
    const uint8_t *b = vc + at.at;
    const uint32_t w = reinterpret_cast<const uint32_t *>(b)[static_cast<size_t>(at.slab) * hd + v_word(d, hd)];
    const uint16_t *h = reinterpret_cast<const uint16_t *>(b + static_cast<size_t>(M.spp) * kSlab * (hd / 2));
    return value_of(at.bad ? kNanHeader : h[(static_cast<size_t>(at.slab) * (hd / 32) + (d >> 5)) * 8 + r], (w >> nib(r)) & 15u);
}

// ---- append ------------------------------------------------------------------------------------------------

// x / d to the nearest whole number, ties to even, for |x / d| of up to 2^22: the rounded product with the reciprocal is at most
// one off, and the remainder x - n d is exact where it decides (n d has at most 12 significant bits).
__device__ __forceinline__ float nearest(float x, float d, float inv) {
    float n = rintf(x * inv);
    const float e = fmaf(-n, d, x), half = 0.5f * d;
    const bool odd = n - 2.0f * floorf(0.5f * n) != 0.0f;
    if (e > half || (e == half && odd)) n += 1.0f;
    else if (e < -half || (e == -half && odd)) n -= 1.0f;
    return n;
}

// Scale of a group whose values, with zero, span [lo, hi]: the smallest k 2^e, k < 128, e >= -20, with 15 k 2^e >= hi - lo. The
// first guess from a rounded quotient is at most one k off; 15 k 2^e and the span are compared in 64 bits.
__device__ __forceinline__ float scale_for(float lo, float hi) {
    const double span = static_cast<double>(hi) - static_cast<double>(lo);
    const float t = static_cast<float>(span / 15.0);
    if (!(t < kMaxScale)) return kMaxScale;
    int ex = -99;
    if (t > 0.0f) frexpf(t, &ex);  // t = f 2^ex, f in [0.5, 1); a span too small for t takes the smallest step
    const float step = ldexpf(1.0f, ex - 7 > -20 ? ex - 7 : -20);
    float k = ceilf(t / step);  // exact: step is a power of two
    while (k > 0.0f && 15.0 * static_cast<double>((k - 1.0f) * step) >= span) k -= 1.0f;
    while (15.0 * static_cast<double>(k * step) < span) k += 1.0f;
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
    const float d = scale_for(lo, hi);
    if (!(d > 0.0f)) return Group4{0u, 0u};
    const float inv = 1.0f / d, z = fminf(nearest(-lo, d, inv), 15.0f);
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        // Past the saturated range (d = 4352) only the sign of the quotient matters.
        const float c = fminf(fmaxf(nearest(fminf(fmaxf(x[e], -16.0f * d), 16.0f * d), d, inv) + z, 0.0f), 15.0f);
        w |= static_cast<uint32_t>(c) << nib(e);
    }
    return Group4{w, static_cast<uint32_t>(__builtin_bit_cast(uint16_t, static_cast<_Float16>(d))) | static_cast<uint32_t>(z)};
}

// One workgroup of hd threads (64 at least) per (segment, slab of 8 positions, kv head): hd / 8 threads take a row, eight dims each,
// of k and then of v. K words and all headers are the row's own. V words hold eight positions of a dim: the codes meet in LDS and
// thread d puts dim d's word together; where the segment has only some of its positions the others' bits stay as they are, by an
// atomic exclusive-or of what changes (another segment of the launch may write the rest of the word). Bound by bytes: 8 read, 9/8
// written for a (k, v) pair.
template <bool PAGED>
__global__ __launch_bounds__(kMaxHd) void kv4_append_kernel(const float *__restrict__ k, const float *__restrict__ v, uint8_t *kc,
                                                            uint8_t *vc, SegTable T, Map4 M, int hd) {
    __shared__ uint32_t vw[kSlab][kMaxHd / 8];
    __shared__ int broken[kSlab];
    const int kvh = blockIdx.y, tid = threadIdx.x;
    int b = blockIdx.x, si = 0;  // (segment, slab of it)
    while (si + 1 < T.n) {
        const int n = (T.s[si].pos0 + T.s[si].rows - 1) / kSlab - T.s[si].pos0 / kSlab + 1;
        if (b < n) break;
        b -= n;
        ++si;
    }
    const Seg &s = T.s[si];
    const int slab = s.pos0 / kSlab + b, r0 = max(s.pos0 - slab * kSlab, 0), r1 = min(s.pos0 + s.rows - slab * kSlab, kSlab);
    const Place at = place<PAGED>(M, s.slot, kvh, slab);
    if (at.bad) return;
    const int per = hd / 8, row = tid / per, i = tid - row * per;
    const bool on = row >= r0 && row < r1;
    const size_t head = static_cast<size_t>(M.spp) * kSlab * (hd / 2);
    float x[2][8];
    if (tid < kSlab) broken[tid] = 0;
    __syncthreads();
#pragma unroll
    for (int a = 0; a < 2; ++a) {
        const size_t src = on ? (static_cast<size_t>(s.row0 + slab * kSlab + row - s.pos0) * M.kv_heads + kvh) * hd + 8 * i : 0;
        bool ok = true;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[a][e] = on ? (a == 0 ? k : v)[src + e] : 0.0f;
            ok = ok && fabsf(x[a][e]) < INFINITY;
        }
        if (!ok) broken[row] = 1;
    }
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

// The values held at the rows' positions: one workgroup per (row, kv head), thread d dim d.
template <bool PAGED>
__global__ __launch_bounds__(kMaxHd) void kv4_read_kernel(const uint8_t *__restrict__ kc, const uint8_t *__restrict__ vc,
                                                          float *__restrict__ k, float *__restrict__ v, SegTable T, Map4 M, int hd) {
    int t;
    const Seg &s = seg_of_row(T, blockIdx.x, t);
    const int pos = s.pos0 + t, d = threadIdx.x;
    if (d >= hd) return;
    const Place at = place<PAGED>(M, s.slot, blockIdx.y, pos / kSlab);
    const size_t dst = (static_cast<size_t>(s.row0 + t) * M.kv_heads + blockIdx.y) * hd + d;
    k[dst] = k_value(kc, M, at, pos % kSlab, hd, d);
    v[dst] = v_value(vc, M, at, pos % kSlab, hd, d);
}

// ---- attention -----------------------------------------------------------------------------------------------

// One workgroup of four waves per (head, row): wave w takes the 64-key chunks w, w + 4, ...; lane = key for q . k, lane = dims for
// the sum over V; the waves' sums meet in wave order.
constexpr int kWaves = 4;
template <bool PAGED>
__global__ __launch_bounds__(64 * kWaves) void attention4_kernel(const float *__restrict__ q, const uint8_t *__restrict__ kc,
                                                                 const uint8_t *__restrict__ vc, float *__restrict__ out, SegTable T,
                                                                 Map4 M, int heads, int hd, int bidirectional, int window) {
    __shared__ float sq[kMaxHd], sp[kWaves][64], sm[kWaves], sl[kWaves], sacc[kWaves][kMaxHd];
    int t;
    const Seg &s = seg_of_row(T, blockIdx.y, t);
    const int h = blockIdx.x, lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const int qend = s.pos0 + 1 + t, end = bidirectional ? s.pos0 + s.rows : qend;
    const int start = window > 0 && qend > window ? qend - window : 0;
    const int kvh = h / (heads / M.kv_heads);
    const size_t qrow = (static_cast<size_t>(s.row0 + t) * heads + h) * hd;
    for (int d = threadIdx.x; d < hd; d += 64 * kWaves) sq[d] = q[qrow + d] * (1.0f / sqrtf(static_cast<float>(hd)));
    __syncthreads();
    float m = -INFINITY, l = 0.0f, acc[kMaxHd / 64] = {0.f, 0.f, 0.f, 0.f};
    for (int p0 = start + 64 * wv; p0 < end; p0 += 64 * kWaves) {
        const int p = p0 + lane;
        float sc = -INFINITY;
        if (p < end) {
            const Place at = place<PAGED>(M, s.slot, kvh, p / kSlab);
            sc = 0.0f;
            for (int d = 0; d < hd; ++d) sc = fmaf(sq[d], k_value(kc, M, at, p % kSlab, hd, d), sc);
        }
        float mn = sc;
        for (int o = 32; o > 0; o >>= 1) mn = fmaxf(mn, __shfl_xor(mn, o, 64));
        mn = fmaxf(m, mn);
        const float ms = mn == -INFINITY ? 0.0f : mn;
        const float pr = p < end ? expf(sc - ms) : 0.0f, rs = expf(m - ms);
        float ps = pr;
        for (int o = 32; o > 0; o >>= 1) ps += __shfl_xor(ps, o, 64);
        l = l * rs + ps;
        m = mn;
        sp[wv][lane] = pr;
        __builtin_amdgcn_wave_barrier();
        for (int r = 0; r < kMaxHd / 64; ++r) {
            const int d = lane + 64 * r;
            if (d >= hd) break;
            acc[r] *= rs;
            for (int j = 0; j < min(end - p0, 64); ++j)
                acc[r] = fmaf(sp[wv][j], v_value(vc, M, place<PAGED>(M, s.slot, kvh, (p0 + j) / kSlab), (p0 + j) % kSlab, hd, d), acc[r]);
        }
        __builtin_amdgcn_wave_barrier();
    }
    if (lane == 0) sm[wv] = m, sl[wv] = l;
    for (int r = 0; r < kMaxHd / 64; ++r)
        if (lane + 64 * r < hd) sacc[wv][lane + 64 * r] = acc[r];
    __syncthreads();
    if (wv != 0) return;
    float mx = -INFINITY, L = 0.0f, f[kWaves];
    for (int w = 0; w < kWaves; ++w) mx = fmaxf(mx, sm[w]);
    for (int w = 0; w < kWaves; ++w) {
        f[w] = sm[w] == -INFINITY ? 0.0f : expf(sm[w] - mx);
        L += sl[w] * f[w];
    }
    for (int d = lane; d < hd; d += 64) {
        float a = 0.0f;
        for (int w = 0; w < kWaves; ++w) a += sacc[w][d] * f[w];
        out[qrow + d] = a / L;
    }
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

int launch_append4(const float *k, const float *v, void *kc, void *vc, const SegTable &T, const Map4 &M, int hd, hipStream_t s) {
    if (!k || !v) return VQ_ERR_ARG;
    unsigned slabs = 0;
    for (int i = 0; i < T.n; ++i) slabs += (T.s[i].pos0 + T.s[i].rows - 1) / kSlab - T.s[i].pos0 / kSlab + 1;
    const dim3 grid(slabs, M.kv_heads);
    const int threads = (hd + 63) / 64 * 64;
    auto *kb = static_cast<uint8_t *>(kc), *vb = static_cast<uint8_t *>(vc);
    if (M.pt) kv4_append_kernel<true><<<grid, threads, 0, s>>>(k, v, kb, vb, T, M, hd);
    else kv4_append_kernel<false><<<grid, threads, 0, s>>>(k, v, kb, vb, T, M, hd);
    return status_of(hipGetLastError());
}

int launch_read4(const void *kc, const void *vc, float *k, float *v, const SegTable &T, const Map4 &M, int hd, hipStream_t s) {
    if (!k || !v) return VQ_ERR_ARG;
    const dim3 grid(T.total, M.kv_heads);
    const int threads = (hd + 63) / 64 * 64;
    auto *kb = static_cast<const uint8_t *>(kc), *vb = static_cast<const uint8_t *>(vc);
    if (M.pt) kv4_read_kernel<true><<<grid, threads, 0, s>>>(kb, vb, k, v, T, M, hd);
    else kv4_read_kernel<false><<<grid, threads, 0, s>>>(kb, vb, k, v, T, M, hd);
    return status_of(hipGetLastError());
}

int launch_attention4(const float *q, const void *kc, const void *vc, float *out, const SegTable &T, const Map4 &M, int heads, int hd,
                      int bidirectional, int window, hipStream_t s) {
    if (!q || !out) return VQ_ERR_ARG;
    if (heads < M.kv_heads || heads % M.kv_heads || window < 0) return VQ_ERR_SHAPE;
    const dim3 grid(heads, T.total);
    auto *kb = static_cast<const uint8_t *>(kc), *vb = static_cast<const uint8_t *>(vc);
    if (M.pt) attention4_kernel<true><<<grid, 64 * kWaves, 0, s>>>(q, kb, vb, out, T, M, heads, hd, bidirectional, window);
    else attention4_kernel<false><<<grid, 64 * kWaves, 0, s>>>(q, kb, vb, out, T, M, heads, hd, bidirectional, window);
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
    (void)heads, (void)kv_heads, (void)hd, (void)seq_len, (void)ntok, (void)window;
    return 0;
}

size_t vq_attention4_seg_workspace_bytes(const int32_t *segs, int nseg, int heads, int kv_heads, int hd) {
    (void)segs, (void)nseg, (void)heads, (void)kv_heads, (void)hd;
    return 0;
}

int vq_attention4_ws(const float *q, const void *kc, const void *vc, float *out, int heads, int kv_heads, int hd, int max_seq,
                     int seq_len, int ntok, int bidirectional, int window, void *workspace, size_t workspace_bytes,
                     void *stream) {
    (void)workspace, (void)workspace_bytes;
    if (ntok < 1 || seq_len < 1 || ntok > max_seq || seq_len > max_seq - ntok + 1) return VQ_ERR_SHAPE;
    const SegTable T = one_segment(seq_len - 1, ntok);
    Map4 M;
    const int st = check_cache(kc, vc, kv_heads, hd, T, false, nullptr, 0, 0, 0, max_seq, M);
    return st != VQ_OK ? st : launch_attention4(q, kc, vc, out, T, M, heads, hd, bidirectional, window, static_cast<hipStream_t>(stream));
}

int vq_attention4_seg_ws(const float *q, const void *kc, const void *vc, float *out, const int32_t *segs, int nseg, int heads,
                         int kv_heads, int hd, const int32_t *page_table, int page_size, int pages_per_seq, int pages,
                         void *workspace, size_t workspace_bytes, void *stream) {
    (void)workspace, (void)workspace_bytes;
    SegTable T;
    Map4 M;
    int st = make_table(segs, nseg, T, nullptr);
    if (st == VQ_OK) st = check_cache(kc, vc, kv_heads, hd, T, true, page_table, page_size, pages_per_seq, pages, 0, M);
    return st != VQ_OK ? st : launch_attention4(q, kc, vc, out, T, M, heads, hd, 0, 0, static_cast<hipStream_t>(stream));
}

}  // extern "C"
