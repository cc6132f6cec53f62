// keep_rows.hip — eviction of a model's rows to a budget: which rows stay (the
// `budget` largest accumulated weights), and the rows of any number of tensors, the
// optimiser's states among them, gathered in one launch.
//
// Selection.  The scores' bits are made an ordered 32-bit key (+0 and -0 alike, NaN
// lowest, protected rows highest).  Three histograms over 11 + 11 + 10 bits of the key,
// each restricted to the keys that share the digits found so far, give the budget-th
// largest key T and how many of the keys equal to T stay; those of the lowest index do.
// The kept rows are then counted per tile, the counts scanned, and the indices written in
// order.  All counts are integers: the result does not depend on the order of the atomics.
// Six launches, 37 us for 1M scores and 53 us for 5M (the scores are read five times, from
// the caches): each waits for the one before it, 2-8 us at any size up to 1M.  Up to 16384
// scores one workgroup does it all (10k: 14 us, the six 23 us and the gaps between them).
#include "gsr_blockscale.hpp"
#include "gsr_kernels.hpp"
#include "gsr_wave.hpp"

#pragma clang fp contract(off)

namespace gsr {

constexpr int SR_THREADS = 256, SR_BINS = 2048;
constexpr int SR_TILE = 4096;  // scores per workgroup of the counting and writing kernels
constexpr int SR_HIST_THREADS = 1024, SR_HIST_BLOCKS = 256, SR_COPIES = 8;
constexpr int SR_SCAN_TILES = 4096;  // up to here the writing workgroups add the counts before their tile themselves

struct SelectArgs {
    const float *score;
    const uint8_t *protect;  // NULL: none
    int64_t *rows;
    uint32_t *hist;  // [3][SR_BINS]
    uint32_t *ctrl;  // [3][2]: the digits found before each further pass, and how many of them to keep
    uint32_t *gt, *eq;  // per tile: keys above T, equal to T; then the counts before the tile
    int P, tiles;
    uint32_t budget;
};

__device__ __forceinline__ uint32_t score_key(float x, uint32_t protect) {
    const uint32_t b = as_u32(x + 0.0f);  // -0 + 0 = +0
    const uint32_t k = x != x ? 0u : (b >> 31 ? ~b : b | 0x80000000u);
    return protect ? 0xFFFFFFFFu : k;
}
// keys of the scores [i, i + 4); `live` of them exist
__device__ __forceinline__ int score_keys(const SelectArgs &a, int64_t i, uint32_t key[4]) {
    const int64_t left = a.P - i;
    const int live = left >= 4 ? 4 : (left > 0 ? (int)left : 0);
    if (live == 4) {
        const f32x4_u v = *reinterpret_cast<const f32x4_u *>(a.score + i);
        const uint32_t p = a.protect ? *reinterpret_cast<const u32_u *>(a.protect + i) : 0u;
        key[0] = score_key(v.x, p & 0xFFu), key[1] = score_key(v.y, p & 0xFF00u);
        key[2] = score_key(v.z, p & 0xFF0000u), key[3] = score_key(v.w, p & 0xFF000000u);
    } else {
        for (int j = 0; j < live; j++) key[j] = score_key(a.score[i + j], a.protect ? a.protect[i + j] : 0u);
    }
    return live;
}

// From the histogram of pass D (its bins' counts of keys with the digits `prefix`): the
// bin that holds the `keep`-th largest, and how many of its keys stay.  All threads.
template <int THREADS>
__device__ __forceinline__ void resolve_digit(const uint32_t *hist, uint32_t keep, uint32_t *sh, uint32_t *bin,
                                              uint32_t *rest) {
    constexpr int PER = SR_BINS / THREADS;
    uint32_t c[PER], sum = 0, tot;
    const int top = SR_BINS - 1 - (int)threadIdx.x * PER;
#pragma unroll
    for (int j = 0; j < PER; j++) sum += c[j] = hist[top - j];
    uint32_t before = block_inclusive_scan<THREADS>(sum, sh, &tot) - sum;
    if (before < keep && keep <= before + sum) {
#pragma unroll
        for (int j = 0; j < PER; j++) {
            if (before < keep && keep <= before + c[j]) sh[16] = (uint32_t)(top - j), sh[17] = keep - before;
            before += c[j];
        }
    }
    __syncthreads();
    *bin = sh[16];
    *rest = sh[17];
    __syncthreads();
}

__global__ void __launch_bounds__(SR_THREADS) select_clear_kernel(SelectArgs a) {
    const int i = blockIdx.x * SR_THREADS + threadIdx.x;
    if (i < 3 * SR_BINS) a.hist[i] = 0;
    if (i == 0) a.ctrl[0] = 0, a.ctrl[1] = a.budget;
}

// digits of pass D: bits [SHIFT, SHIFT + BITS); the keys counted share the bits above
template <int D, int THREADS = SR_THREADS>
__device__ __forceinline__ void pass_state(const SelectArgs &a, uint32_t *sh, uint32_t *prefix, uint32_t *keep) {
    *prefix = a.ctrl[2 * (D ? D - 1 : 0)], *keep = a.ctrl[2 * (D ? D - 1 : 0) + 1];
    if (D > 0) {
        uint32_t bin, rest;
        resolve_digit<THREADS>(a.hist + (D - 1) * SR_BINS, *keep, sh, &bin, &rest);
        *prefix = *prefix << (D == 3 ? 10 : 11) | bin;
        *keep = rest;
        if (D < 3 && blockIdx.x == 0 && threadIdx.x == 0) a.ctrl[2 * D] = *prefix, a.ctrl[2 * D + 1] = *keep;
    }
}

// Few workgroups of 16 waves: each ends in one atomic per bin that it met, and with 1024
// workgroups of four waves those are most of the pass (5M scores: 24 us the first pass
// instead of 10).  Where scores share a bin (equal ones), a wave's additions to one counter
// follow each other: every bin has SR_COPIES counters, one for every eighth lane (5M equal
// scores: 8 us a pass, 22 with one counter; scores that spread: the same).
template <int D>
__global__ void __launch_bounds__(SR_HIST_THREADS) select_hist_kernel(SelectArgs a) {
    __shared__ uint32_t h[SR_BINS * SR_COPIES], sh[32];
    constexpr int SHIFT = D == 0 ? 21 : (D == 1 ? 10 : 0), BITS = D == 2 ? 10 : 11;
    for (int i = threadIdx.x; i < SR_BINS * SR_COPIES; i += SR_HIST_THREADS) h[i] = 0;
    uint32_t prefix, keep;
    pass_state<D, SR_HIST_THREADS>(a, sh, &prefix, &keep);
    __syncthreads();
    const uint32_t copy = threadIdx.x % SR_COPIES;
    const int64_t stride = (int64_t)gridDim.x * SR_HIST_THREADS * 4;
    for (int64_t i = ((int64_t)blockIdx.x * SR_HIST_THREADS + threadIdx.x) * 4; i < a.P; i += stride) {
        uint32_t key[4];
        const int live = score_keys(a, i, key);
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (j < live && (D == 0 || key[j] >> (SHIFT + BITS) == prefix))
                atomicAdd(&h[(key[j] >> SHIFT & ((1u << BITS) - 1)) * SR_COPIES + copy], 1u);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < SR_BINS; i += SR_HIST_THREADS) {
        uint32_t n = 0;
#pragma unroll
        for (int c = 0; c < SR_COPIES; c++) n += h[i * SR_COPIES + c];
        if (n) atomicAdd(&a.hist[D * SR_BINS + i], n);
    }
}

__global__ void __launch_bounds__(SR_THREADS) select_count_kernel(SelectArgs a) {
    __shared__ uint32_t sh[32];
    uint32_t T, need;
    pass_state<3>(a, sh, &T, &need);
    uint32_t gt = 0, eq = 0;
#pragma unroll
    for (int u = 0; u < SR_TILE / (SR_THREADS * 4); u++) {
        uint32_t key[4];
        const int live = score_keys(a, (int64_t)blockIdx.x * SR_TILE + (u * SR_THREADS + threadIdx.x) * 4, key);
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (j < live) gt += key[j] > T, eq += key[j] == T;
    }
    gt = block_sum<SR_THREADS>(gt, sh);
    eq = block_sum<SR_THREADS>(eq, sh);
    if (threadIdx.x == 0) a.gt[blockIdx.x] = gt, a.eq[blockIdx.x] = eq;
}

__global__ void __launch_bounds__(1024) select_scan_kernel(SelectArgs a) {
    __shared__ uint32_t sh[16];
    block_exclusive_scan_inplace<1024, 4>(blockIdx.x ? a.eq : a.gt, a.tiles, sh);
}

template <bool SCANNED>
__global__ void __launch_bounds__(SR_THREADS) select_write_kernel(SelectArgs a) {
    __shared__ uint32_t sh[32];
    uint32_t T, need;
    pass_state<3>(a, sh, &T, &need);
    uint32_t gt0 = 0, eq0 = 0;
    if (SCANNED) {
        gt0 = a.gt[blockIdx.x], eq0 = a.eq[blockIdx.x];
    } else {
        for (int i = threadIdx.x; i < (int)blockIdx.x; i += SR_THREADS) gt0 += a.gt[i], eq0 += a.eq[i];
        gt0 = block_sum<SR_THREADS>(gt0, sh);
        eq0 = block_sum<SR_THREADS>(eq0, sh);
    }
    // keys above T in the low half, equal to T in the high half (4096 each at most); the kept
    // places are lined up in LDS and leave in one run (13 us for 5M scores)
    __shared__ uint16_t kept[SR_TILE];
    const int64_t tile0 = (int64_t)blockIdx.x * SR_TILE;
    uint32_t gt = 0, eq = eq0;
#pragma unroll
    for (int u = 0; u < SR_TILE / (SR_THREADS * 4); u++) {
        const uint32_t o = (u * SR_THREADS + threadIdx.x) * 4;
        uint32_t key[4], own = 0, tot;
        const int live = score_keys(a, tile0 + o, key);
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (j < live) own += key[j] > T ? 1u : (key[j] == T ? 0x10000u : 0u);
        const uint32_t before = block_inclusive_scan<SR_THREADS>(own, sh, &tot) - own;
        uint32_t g = gt + (before & 0xFFFFu), e = eq + (before >> 16);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (j >= live) continue;
            if (key[j] > T || (key[j] == T && e < need)) kept[g + min(e, need) - min(eq0, need)] = (uint16_t)(o + j);
            g += key[j] > T, e += key[j] == T;
        }
        gt += tot & 0xFFFFu, eq += tot >> 16;
    }
    __syncthreads();
    const uint32_t n = gt + min(eq, need) - min(eq0, need);
    int64_t *rows = a.rows + gt0 + min(eq0, need);
    for (uint32_t i = threadIdx.x; i < n; i += SR_THREADS) rows[i] = tile0 + kept[i];
}

// Up to SR_SMALL scores: one workgroup, the keys in registers (SR_PER consecutive ones a
// thread), the histograms in LDS: one launch instead of six.
constexpr int SR_PER = 16, SR_SMALL = SR_HIST_THREADS * SR_PER;
__global__ void __launch_bounds__(SR_HIST_THREADS) select_small_kernel(SelectArgs a) {
    __shared__ uint32_t h[SR_BINS * SR_COPIES], total[SR_BINS], sh[32];
    const int64_t i0 = (int64_t)threadIdx.x * SR_PER;
    const uint32_t copy = threadIdx.x % SR_COPIES;
    uint32_t key[SR_PER], prefix = 0, keep = a.budget;
    int live = 0;
#pragma unroll
    for (int j = 0; j < SR_PER; j += 4) live += score_keys(a, i0 + j, key + j);
#pragma unroll
    for (int d = 0; d < 3; d++) {
        const int shift = d == 0 ? 21 : (d == 1 ? 10 : 0), bits = d == 2 ? 10 : 11;
        for (int i = threadIdx.x; i < SR_BINS * SR_COPIES; i += SR_HIST_THREADS) h[i] = 0;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < SR_PER; j++)
            if (j < live && (d == 0 || key[j] >> (shift + bits) == prefix))
                atomicAdd(&h[(key[j] >> shift & ((1u << bits) - 1)) * SR_COPIES + copy], 1u);
        __syncthreads();
        for (int i = threadIdx.x; i < SR_BINS; i += SR_HIST_THREADS) {
            uint32_t n = 0;
#pragma unroll
            for (int c = 0; c < SR_COPIES; c++) n += h[i * SR_COPIES + c];
            total[i] = n;
        }
        __syncthreads();
        uint32_t bin, rest;
        resolve_digit<SR_HIST_THREADS>(total, keep, sh, &bin, &rest);
        prefix = prefix << bits | bin;
        keep = rest;
    }
    uint32_t own = 0, tot;
#pragma unroll
    for (int j = 0; j < SR_PER; j++)
        if (j < live) own += key[j] > prefix ? 1u : (key[j] == prefix ? 0x10000u : 0u);  // <= 16384 each
    const uint32_t before = block_inclusive_scan<SR_HIST_THREADS>(own, sh, &tot) - own;
    uint32_t g = before & 0xFFFFu, e = before >> 16;
#pragma unroll
    for (int j = 0; j < SR_PER; j++) {
        if (j >= live) continue;
        if (key[j] > prefix) a.rows[g++ + min(e, keep)] = i0 + j;
        else if (key[j] == prefix) {
            if (e < keep) a.rows[g + e] = i0 + j;
            e++;
        }
    }
}

size_t select_rows_scratch_bytes(int P) {
    return (3 * SR_BINS + 16 + 2 * (((size_t)P + SR_TILE - 1) / SR_TILE)) * 4;
}

hipError_t launch_select_rows(const float *score, const uint8_t *protect, int P, int budget, int64_t *rows,
                              void *scratch, hipStream_t st) {
    SelectArgs a;
    a.score = score, a.protect = protect, a.rows = rows;
    a.P = P, a.budget = (uint32_t)budget;
    if (P <= SR_SMALL) {
        hipLaunchKernelGGL(select_small_kernel, dim3(1), dim3(SR_HIST_THREADS), 0, st, a);
        return hipGetLastError();
    }
    a.tiles = (int)(((int64_t)P + SR_TILE - 1) / SR_TILE);
    a.hist = (uint32_t *)scratch;
    a.ctrl = a.hist + 3 * SR_BINS;
    a.gt = a.ctrl + 16;
    a.eq = a.gt + a.tiles;
    const int hb = (int)(((int64_t)P + SR_HIST_THREADS * 4 - 1) / (SR_HIST_THREADS * 4));
    const dim3 t(SR_THREADS), ht(SR_HIST_THREADS), hg(hb < SR_HIST_BLOCKS ? hb : SR_HIST_BLOCKS);
    hipLaunchKernelGGL(select_clear_kernel, dim3(3 * SR_BINS / SR_THREADS), t, 0, st, a);
    hipLaunchKernelGGL(select_hist_kernel<0>, hg, ht, 0, st, a);
    hipLaunchKernelGGL(select_hist_kernel<1>, hg, ht, 0, st, a);
    hipLaunchKernelGGL(select_hist_kernel<2>, hg, ht, 0, st, a);
    hipLaunchKernelGGL(select_count_kernel, dim3(a.tiles), t, 0, st, a);
    if (a.tiles > SR_SCAN_TILES) {
        hipLaunchKernelGGL(select_scan_kernel, dim3(2), dim3(1024), 0, st, a);
        hipLaunchKernelGGL(select_write_kernel<true>, dim3(a.tiles), t, 0, st, a);
    } else {
        hipLaunchKernelGGL(select_write_kernel<false>, dim3(a.tiles), t, 0, st, a);
    }
    return hipGetLastError();
}

// ------------------------------------------------------------ rows of many tensors
//
// dst[j] = src[rows[j]] for every segment, zeros where rows[j] is outside [0, P) (a
// fresh row; nothing is read).  The output is contiguous and is written in spans of L
// consecutive bytes a lane (16, the widest access), whatever the rows' length: a span's bytes
// come from two rows at most if row + gcd(row, L) >= L, since it starts at a multiple of
// gcd(row, L) in its row.  Both parts are one L-byte load at the alignment that the source
// happens to have, the second one from as many bytes before its row as the first part is
// long, so that its bytes arrive in their place and a mask joins the two.  Where a load would
// leave the source (its first and last rows) the lane reads its bytes one by one.  Rows that
// are too short for it (4-byte rows: opacities) move one unit a lane.
// Memory bounds it, counted in whole lines, those of dropped rows among them: 1M -> 500k
// Gaussians with fp32 states 152 us, 5M -> 3M with 8-bit states 600 us (3.1 GB moved, 5.1
// TB/s).  Stored non-temporally (161 -> 152 us), loaded through the caches, which hold the
// neighbouring rows' part of a line.
//
// 8-bit states (gsr_blockscale.hpp): the rows' values land in other blocks of 64, whose
// scale is formed anew from what they hold; powers of two, so only values below 2^-13 of
// their new block's largest lose bits.
constexpr int TR_THREADS = 256, TR_SEGS = 40, TR_ITEMS = 8, TR_SPANS = 2;
constexpr int TR_TILE = TR_THREADS * TR_ITEMS;        // units per workgroup, unit by unit
constexpr int TR_BYTES = TR_THREADS * TR_SPANS * 16;  // bytes or codes per workgroup in spans (four spans a lane: 677
                                                      // instead of 606 us at 5M -> 3M with 8-bit states)

struct TakeSeg {
    const void *src;
    void *dst;
    const uint8_t *src_scale;
    uint8_t *dst_scale;
    int64_t units;             // of dst: bytes in spans, codes, or units
    double inv_row;            // 1 / row
    uint32_t row, mul, shift;  // units per row; x / row = x * mul >> (31 + shift) for x < 2^31
    int32_t kind;
    __device__ __forceinline__ uint32_t divide(uint32_t x) const { return (uint32_t)((uint64_t)x * mul >> (31 + shift)); }
    // row and column of unit u < 2^34: the quotient from the reciprocal is off by one at most
    __device__ __forceinline__ int64_t place(int64_t u, uint32_t *col) const {
        int64_t q = (int64_t)((double)u * inv_row), c = u - q * row;
        if (c < 0) q--, c += row;
        if (c >= row) q++, c -= row;
        *col = (uint32_t)c;
        return q;
    }
};
struct TakeArgs {
    const int64_t *rows;
    int64_t P;
    int nseg;
    int block0[TR_SEGS + 1];
    TakeSeg seg[TR_SEGS];
};

template <typename U>
__device__ __forceinline__ void take_units(const TakeArgs &a, const TakeSeg &s, int64_t tile) {
    const int64_t u0 = tile * TR_TILE;
    uint32_t col0;
    const int64_t row0 = s.place(u0, &col0);
    const U *src = (const U *)s.src;
    U *dst = (U *)s.dst + u0;
    const uint32_t left = (uint32_t)(s.units - u0 < TR_TILE ? s.units - u0 : TR_TILE);
    int64_t from[TR_ITEMS];
    U v[TR_ITEMS];
#pragma unroll
    for (int j = 0; j < TR_ITEMS; j++) {
        const uint32_t o = j * TR_THREADS + threadIdx.x, x = col0 + o, q = s.divide(x);
        from[j] = -1;
        if (o < left) {
            const int64_t r = a.rows[row0 + q];
            if ((uint64_t)r < (uint64_t)a.P) from[j] = r * s.row + (x - q * s.row);
        }
    }
#pragma unroll
    for (int j = 0; j < TR_ITEMS; j++) {
        v[j] = U(0);
        if (from[j] >= 0) v[j] = src[from[j]];
    }
#pragma unroll
    for (int j = 0; j < TR_ITEMS; j++) {
        const uint32_t o = j * TR_THREADS + threadIdx.x;
        if (o < left) dst[o] = v[j];
    }
}

// L bytes in L / 4 words
template <int L>
struct Span;
template <>
struct Span<16> {
    typedef uint32_t V __attribute__((ext_vector_type(4)));
    typedef uint32_t V_u __attribute__((ext_vector_type(4), aligned(1)));
};
template <>
struct Span<4> {
    typedef uint32_t V __attribute__((ext_vector_type(1)));
    typedef uint32_t V_u __attribute__((ext_vector_type(1), aligned(1)));
};

// bytes of word i of a span from byte n of the span on, as 0x01 each / all their bits
__device__ __forceinline__ uint32_t ones_from(int n, int i) {
    return (uint32_t)(0x01010101ull << 8 * min(max(n - 4 * i, 0), 4));
}
__device__ __forceinline__ uint32_t bytes_from(int n, int i) {
    return (uint32_t)(0xFFFFFFFFull << 8 * min(max(n - 4 * i, 0), 4));
}

// bytes [lo, hi) of a span that lies at src + f (f < 0 or f + L > n where only these exist)
template <int L>
__device__ __forceinline__ typename Span<L>::V load_span(const uint8_t *src, int64_t f, int64_t n, int lo, int hi) {
    typename Span<L>::V v;
    if (f >= 0 && f + L <= n) {
        v = *reinterpret_cast<const typename Span<L>::V_u *>(src + f);
    } else {
#pragma unroll
        for (int i = 0; i < L / 4; i++) v[i] = 0;
        for (int j = lo; j < hi; j++) {
            const uint32_t b = (uint32_t)src[f + j] << 8 * (j & 3);
#pragma unroll
            for (int i = 0; i < L / 4; i++) v[i] |= j >> 2 == i ? b : 0u;
        }
    }
    return v;
}

struct SpanPlace {
    int live, k;       // bytes of the span that exist; of the first part
    int64_t fa, fb;    // where its bytes would lie in the source by the first and by the second part
    bool a, b;         // parts to load
};
template <int L>
__device__ __forceinline__ SpanPlace span_place(const TakeArgs &a, const TakeSeg &s, uint32_t o, int left, int64_t row0,
                                                uint32_t col0) {
    SpanPlace p;
    const uint32_t c = col0 + o, q = s.divide(c), col = c - q * s.row;
    p.live = min(max(left - (int)o, 0), L);
    p.k = (int)min((uint32_t)L, s.row - col);
    p.a = p.b = false;
    p.fa = p.fb = 0;
    if (p.live) {
        const int64_t r = a.rows[row0 + q];
        p.a = (uint64_t)r < (uint64_t)a.P;
        if (p.a) p.fa = r * s.row + col;
    }
    if (p.k < p.live) {
        const int64_t r = a.rows[row0 + q + 1];
        p.b = (uint64_t)r < (uint64_t)a.P;
        if (p.b) p.fb = r * s.row - p.k;
    }
    return p;
}
template <int L>
__device__ __forceinline__ typename Span<L>::V join(const SpanPlace &p, const typename Span<L>::V &A,
                                                    const typename Span<L>::V &B) {
    typename Span<L>::V w;
#pragma unroll
    for (int i = 0; i < L / 4; i++) {
        const uint32_t m = bytes_from(p.k, i);
        w[i] = (A[i] & ~m) | (B[i] & m);
    }
    return w;
}
template <int L>
__device__ __forceinline__ void store_span(uint8_t *dst, int live, const typename Span<L>::V &w) {
    if (live == L) {
        __builtin_nontemporal_store((typename Span<L>::V_u)w, reinterpret_cast<typename Span<L>::V_u *>(dst));
    } else {
#pragma unroll
        for (int j = 0; j < L; j++)
            if (j < live) dst[j] = (uint8_t)(w[j >> 2] >> 8 * (j & 3));
    }
}

__device__ __forceinline__ void take_spans(const TakeArgs &a, const TakeSeg &s, int64_t tile) {
    typedef Span<16>::V V;
    const int64_t u0 = tile * TR_BYTES, n = a.P * s.row;
    uint32_t col0;
    const int64_t row0 = s.place(u0, &col0);
    const int left = (int)(s.units - u0 < TR_BYTES ? s.units - u0 : TR_BYTES);
    const uint8_t *src = (const uint8_t *)s.src;
    SpanPlace p[TR_SPANS];
    V A[TR_SPANS], B[TR_SPANS];
#pragma unroll
    for (int t = 0; t < TR_SPANS; t++) p[t] = span_place<16>(a, s, (t * TR_THREADS + threadIdx.x) * 16, left, row0, col0);
#pragma unroll
    for (int t = 0; t < TR_SPANS; t++) {
        A[t] = B[t] = V(0);
        if (p[t].a) A[t] = load_span<16>(src, p[t].fa, n, 0, min(p[t].k, p[t].live));
        if (p[t].b) B[t] = load_span<16>(src, p[t].fb, n, p[t].k, p[t].live);
    }
#pragma unroll
    for (int t = 0; t < TR_SPANS; t++)
        store_span<16>((uint8_t *)s.dst + u0 + (t * TR_THREADS + threadIdx.x) * 16, p[t].live, join<16>(p[t], A[t], B[t]));
}

// L codes (in words, the lowest byte first) in units of the scale bytes `sc`, as codes of
// their new block, which 64 / L lanes of a DPP row hold (every lane of the wave calls): the
// new scale byte from the largest value, and the values in its units to nearest even by the
// hardware's conversion.  A quarter of each value keeps the largest code, 256, in fp32 under the
// largest scale; a code's four bits are exact down to 2^-138.
template <int L, bool SIGNED>
__device__ __forceinline__ typename Span<L>::V recode(const typename Span<L>::V &w, const typename Span<L>::V &sc,
                                                      uint32_t *byte) {
    float x[L], top = 0.f;
#pragma unroll
    for (int i = 0; i < L / 4; i++) {
        e4m3_decode4(w[i], x + 4 * i);
#pragma unroll
        for (int j = 4 * i; j < 4 * i + 4; j++) {
            x[j] = __builtin_ldexpf(x[j], (int)(sc[i] >> 8 * (j & 3) & 0xFFu) - 129);
            top = fmaxf(top, fabsf(x[j]));  // a NaN does not count
        }
    }
    uint32_t m = as_u32(top);
    if (L == 4) m = row_max(m);
    else {
        m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, DPP_QUAD_XOR1, 0xf, 0xf, true));
        m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, DPP_QUAD_XOR2, 0xf, 0xf, true));
    }
    *byte = scale_byte(m + (2u << 23));
    typename Span<L>::V c;
#pragma unroll
    for (int i = 0; i < L / 4; i++) {
        const int e = 129 - (int)*byte;
        int v = 0;
        v = __builtin_amdgcn_cvt_pk_fp8_f32(__builtin_ldexpf(x[4 * i], e), __builtin_ldexpf(x[4 * i + 1], e), v, false);
        v = __builtin_amdgcn_cvt_pk_fp8_f32(__builtin_ldexpf(x[4 * i + 2], e), __builtin_ldexpf(x[4 * i + 3], e), v, true);
        c[i] = (uint32_t)v;
        if (!SIGNED)  // nothing but zero becomes zero: 0x01 in the bytes that did
            c[i] |= ((w[i] + 0x7F7F7F7Fu) & ~(c[i] + 0x7F7F7F7Fu)) >> 7 & 0x01010101u;
    }
    return c;
}

template <int L, bool SIGNED>
__device__ __forceinline__ void take_code_spans(const TakeArgs &a, const TakeSeg &s, int64_t tile) {
    typedef typename Span<L>::V V;
    constexpr int TILE = TR_THREADS * TR_SPANS * L;
    const int64_t u0 = tile * TILE, n = a.P * s.row, last = (n - 1) / SCALE_BLOCK - 1;
    uint32_t col0;
    const int64_t row0 = s.place(u0, &col0);
    const int left = (int)(s.units - u0 < TILE ? s.units - u0 : TILE);
    SpanPlace p[TR_SPANS];
    V A[TR_SPANS], B[TR_SPANS];
    uint32_t sc[TR_SPANS];  // scale bytes: the first part's block, the next one, the second part's, the next one
#pragma unroll
    for (int t = 0; t < TR_SPANS; t++) p[t] = span_place<L>(a, s, (t * TR_THREADS + threadIdx.x) * L, left, row0, col0);
#pragma unroll
    for (int t = 0; t < TR_SPANS; t++) {
        A[t] = B[t] = V(0);
        sc[t] = 0;
        if (p[t].a) {
            A[t] = load_span<L>((const uint8_t *)s.src, p[t].fa, n, 0, min(p[t].k, p[t].live));
            const int64_t b = p[t].fa / SCALE_BLOCK, bl = b < last ? b : last;
            sc[t] = (uint32_t) * reinterpret_cast<const u16_u *>(s.src_scale + bl) >> (uint32_t)(b - bl) * 8;
        }
        if (p[t].b) {
            B[t] = load_span<L>((const uint8_t *)s.src, p[t].fb, n, p[t].k, p[t].live);
            const int64_t b = (p[t].fb + p[t].k) / SCALE_BLOCK, bl = b < last ? b : last;
            sc[t] |= (uint32_t) * reinterpret_cast<const u16_u *>(s.src_scale + bl) >> (uint32_t)(b - bl) * 8 << 16;
        }
    }
#pragma unroll
    for (int t = 0; t < TR_SPANS; t++) {
        V w = join<L>(p[t], A[t], B[t]), pick;
        const int cross_a = min(p[t].k, SCALE_BLOCK - (int)(p[t].fa & (SCALE_BLOCK - 1)));
        const int cross_b = p[t].k + SCALE_BLOCK - (int)((p[t].fb + p[t].k) & (SCALE_BLOCK - 1));
#pragma unroll
        for (int i = 0; i < L / 4; i++) {
            w[i] &= ~bytes_from(p[t].live, i);
            pick[i] = __builtin_amdgcn_perm(0, sc[t], ones_from(cross_a, i) + ones_from(p[t].k, i) + ones_from(cross_b, i));
        }
        uint32_t byte;
        const V c = recode<L, SIGNED>(w, pick, &byte);
        const uint32_t o = (t * TR_THREADS + threadIdx.x) * L;
        store_span<L>((uint8_t *)s.dst + u0 + o, p[t].live, c);
        if (p[t].live && o % SCALE_BLOCK == 0) s.dst_scale[(u0 + o) / SCALE_BLOCK] = (uint8_t)byte;
    }
}

// Element by element: rows of one code, and sources of at most one block
template <bool SIGNED>
__device__ __forceinline__ void take_codes(const TakeArgs &a, const TakeSeg &s, int64_t tile) {
    constexpr int TILE = TR_THREADS * TR_SPANS * 4;
    const int64_t u0 = tile * TILE;
    uint32_t col0;
    const int64_t row0 = s.place(u0, &col0);
    const int left = (int)(s.units - u0 < TILE ? s.units - u0 : TILE);
    const uint8_t *src = (const uint8_t *)s.src;
    for (int t = 0; t < TILE; t += TR_THREADS * 4) {
        const int o = t + (int)threadIdx.x * 4, live = min(max(left - o, 0), 4);
        Span<4>::V w(0), sc(0);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint32_t c = col0 + o + j, q = s.divide(c);
            if (j < live) {
                const int64_t r = a.rows[row0 + q];
                if ((uint64_t)r < (uint64_t)a.P) {
                    const int64_t f = r * s.row + (c - q * s.row);
                    w[0] |= (uint32_t)src[f] << 8 * j;
                    sc[0] |= (uint32_t)s.src_scale[f / SCALE_BLOCK] << 8 * j;
                }
            }
        }
        uint32_t byte;
        const Span<4>::V c = recode<4, SIGNED>(w, sc, &byte);
        store_span<4>((uint8_t *)s.dst + u0 + o, live, c);
        if (live && o % SCALE_BLOCK == 0) s.dst_scale[(u0 + o) / SCALE_BLOCK] = (uint8_t)byte;
    }
}

// a segment's kind: log2 of the unit's bytes, TAKE_SPANS, or TAKE_CODES and its flags
constexpr int TAKE_SPANS = 4, TAKE_CODES = 8, TAKE_SIGNED = 1, TAKE_BY_4 = 2, TAKE_BY_16 = 4;
__global__ void __launch_bounds__(TR_THREADS) take_rows_kernel(TakeArgs a) {
    int k = 0, hi = a.nseg;
    while (hi - k > 1) {
        const int mid = (k + hi) >> 1;
        if (a.block0[mid] <= (int)blockIdx.x) k = mid;
        else hi = mid;
    }
    const TakeSeg &s = a.seg[k];
    const int64_t tile = (int)blockIdx.x - a.block0[k];
    switch (s.kind) {
        case 0: take_units<uint8_t>(a, s, tile); break;
        case 1: take_units<uint16_t>(a, s, tile); break;
        case 2: take_units<uint32_t>(a, s, tile); break;
        case TAKE_SPANS: take_spans(a, s, tile); break;
        case TAKE_CODES: take_codes<false>(a, s, tile); break;
        case TAKE_CODES + TAKE_SIGNED: take_codes<true>(a, s, tile); break;
        case TAKE_CODES + TAKE_BY_4: take_code_spans<4, false>(a, s, tile); break;
        case TAKE_CODES + TAKE_BY_4 + TAKE_SIGNED: take_code_spans<4, true>(a, s, tile); break;
        case TAKE_CODES + TAKE_BY_16: take_code_spans<16, false>(a, s, tile); break;
        default: take_code_spans<16, true>(a, s, tile); break;
    }
}

// x / d = x * mul >> (31 + shift) for x < 2^31
static void divide_by(uint32_t d, uint32_t *mul, uint32_t *shift) {
    *shift = 0;
    while ((1ull << *shift) < d) ++*shift;
    *mul = (uint32_t)(((1ull << (31 + *shift)) + d - 1) / d);
}

// whether a span of L bytes never touches three rows
static bool spans_fit(int64_t row, int L) {
    int64_t g = L;
    while (row % g) g >>= 1;
    return row + g >= L;
}

// the segment's table entry; returns its workgroups
static int64_t take_entry(const gsr_rows_segment &q, int64_t P, int64_t K, TakeSeg *s) {
    s->src = q.src, s->dst = q.dst, s->src_scale = q.src_scale, s->dst_scale = q.dst_scale;
    int unit = 0;  // log2 of the bytes
    int64_t per = TR_BYTES;
    if (q.kind != GSR_ROWS_PLAIN) {
        s->kind = TAKE_CODES + (q.kind == GSR_ROWS_E4M3_SIGNED ? TAKE_SIGNED : 0);
        const bool two = P * q.row_bytes > SCALE_BLOCK;  // the pairs of scales need two blocks in the source
        if (two && spans_fit(q.row_bytes, 16)) {
            s->kind += TAKE_BY_16;
        } else {
            if (two && spans_fit(q.row_bytes, 4)) s->kind += TAKE_BY_4;
            per = TR_BYTES / 4;
        }
    } else if (spans_fit(q.row_bytes, 16)) {
        s->kind = TAKE_SPANS;
    } else {
        const uint64_t bits = (uint64_t)q.row_bytes | (uint64_t)(uintptr_t)q.src | (uint64_t)(uintptr_t)q.dst;
        while (unit < 2 && !(bits >> unit & 1)) unit++;  // rows of 8 bytes are spans
        s->kind = unit;
        per = TR_TILE;
    }
    s->row = (uint32_t)(q.row_bytes >> unit);
    s->inv_row = 1.0 / s->row;
    divide_by(s->row, &s->mul, &s->shift);
    s->units = K * (int64_t)s->row;
    return (s->units + per - 1) / per;
}

hipError_t launch_take_rows(const gsr_rows_segment *segs, int nseg, int64_t P, const int64_t *rows, int64_t K,
                            hipStream_t st) {
    TakeArgs a;
    a.rows = rows, a.P = P;
    for (int k = 0; k < nseg;) {
        int64_t blocks = 0;
        for (a.nseg = 0; k < nseg && a.nseg < TR_SEGS; k++) {
            if (segs[k].row_bytes == 0 || K == 0) continue;
            const int64_t b = take_entry(segs[k], P, K, &a.seg[a.nseg]);
            if (blocks && blocks + b > GSR_MAX_BLOCKS) break;  // the next launch takes it
            a.block0[a.nseg++] = (int)blocks;
            blocks += b;
        }
        if (!a.nseg) continue;
        a.block0[a.nseg] = (int)blocks;
        hipLaunchKernelGGL(take_rows_kernel, dim3((uint32_t)blocks), dim3(TR_THREADS), 0, st, a);
        if (hipError_t e = hipGetLastError()) return e;
    }
    return hipSuccess;
}

}  // namespace gsr
