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
#include "gsr_blockscale.hpp"
#include "gsr_kernels.hpp"
#include "gsr_wave.hpp"

#pragma clang fp contract(off)

namespace gsr {

constexpr int SR_THREADS = 256, SR_BINS = 2048;
constexpr int SR_TILE = 4096;  // scores per workgroup of the counting and writing kernels
constexpr int SR_BLOCKS = 1024;

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
__device__ __forceinline__ void resolve_digit(const uint32_t *hist, uint32_t keep, uint32_t *sh, uint32_t *bin,
                                              uint32_t *rest) {
    constexpr int PER = SR_BINS / SR_THREADS;
    uint32_t c[PER], sum = 0, tot;
    const int top = SR_BINS - 1 - (int)threadIdx.x * PER;
#pragma unroll
    for (int j = 0; j < PER; j++) sum += c[j] = hist[top - j];
    uint32_t before = block_inclusive_scan<SR_THREADS>(sum, sh, &tot) - sum;
    if (before < keep && keep <= before + sum) {
#pragma unroll
        for (int j = 0; j < PER; j++) {
            if (before < keep && keep <= before + c[j]) sh[8] = (uint32_t)(top - j), sh[9] = keep - before;
            before += c[j];
        }
    }
    __syncthreads();
    *bin = sh[8];
    *rest = sh[9];
    __syncthreads();
}

__global__ void __launch_bounds__(SR_THREADS) select_clear_kernel(SelectArgs a) {
    const int i = blockIdx.x * SR_THREADS + threadIdx.x;
    if (i < 3 * SR_BINS) a.hist[i] = 0;
    if (i == 0) a.ctrl[0] = 0, a.ctrl[1] = a.budget;
}

// digits of pass D: bits [SHIFT, SHIFT + BITS); the keys counted share the bits above
template <int D>
__device__ __forceinline__ void pass_state(const SelectArgs &a, uint32_t *sh, uint32_t *prefix, uint32_t *keep) {
    *prefix = a.ctrl[2 * (D ? D - 1 : 0)], *keep = a.ctrl[2 * (D ? D - 1 : 0) + 1];
    if (D > 0) {
        uint32_t bin, rest;
        resolve_digit(a.hist + (D - 1) * SR_BINS, *keep, sh, &bin, &rest);
        *prefix = *prefix << (D == 3 ? 10 : 11) | bin;
        *keep = rest;
        if (D < 3 && blockIdx.x == 0 && threadIdx.x == 0) a.ctrl[2 * D] = *prefix, a.ctrl[2 * D + 1] = *keep;
    }
}

template <int D>
__global__ void __launch_bounds__(SR_THREADS) select_hist_kernel(SelectArgs a) {
    __shared__ uint32_t h[SR_BINS], sh[16];
    constexpr int SHIFT = D == 0 ? 21 : (D == 1 ? 10 : 0), BITS = D == 2 ? 10 : 11;
    for (int i = threadIdx.x; i < SR_BINS; i += SR_THREADS) h[i] = 0;
    uint32_t prefix, keep;
    pass_state<D>(a, sh, &prefix, &keep);
    __syncthreads();
    const int64_t stride = (int64_t)gridDim.x * SR_THREADS * 4;
    for (int64_t i = ((int64_t)blockIdx.x * SR_THREADS + threadIdx.x) * 4; i < a.P; i += stride) {
        uint32_t key[4];
        const int live = score_keys(a, i, key);
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (j < live && (D == 0 || key[j] >> (SHIFT + BITS) == prefix))
                atomicAdd(&h[key[j] >> SHIFT & ((1u << BITS) - 1)], 1u);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < SR_BINS; i += SR_THREADS)
        if (h[i]) atomicAdd(&a.hist[D * SR_BINS + i], h[i]);
}

__global__ void __launch_bounds__(SR_THREADS) select_count_kernel(SelectArgs a) {
    __shared__ uint32_t sh[16];
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

__global__ void __launch_bounds__(SR_THREADS) select_write_kernel(SelectArgs a) {
    __shared__ uint32_t sh[16];
    uint32_t T, need;
    pass_state<3>(a, sh, &T, &need);
    uint32_t gt0 = a.gt[blockIdx.x], eq0 = a.eq[blockIdx.x];
    for (int u = 0; u < SR_TILE / (SR_THREADS * 4); u++) {
        const int64_t i = (int64_t)blockIdx.x * SR_TILE + (u * SR_THREADS + threadIdx.x) * 4;
        uint32_t key[4], own = 0, tot;
        const int live = score_keys(a, i, key);
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (j < live) own += key[j] > T ? 1u : (key[j] == T ? 0x10000u : 0u);  // gt low, eq high half: <= 1024 each
        const uint32_t before = block_inclusive_scan<SR_THREADS>(own, sh, &tot) - own;
        uint32_t g = gt0 + (before & 0xFFFFu), e = eq0 + (before >> 16);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (j >= live) continue;
            if (key[j] > T) a.rows[g++ + min(e, need)] = i + j;
            else if (key[j] == T) {
                if (e < need) a.rows[g + e] = i + j;
                e++;
            }
        }
        gt0 += tot & 0xFFFFu, eq0 += tot >> 16;
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
    a.tiles = (int)(((int64_t)P + SR_TILE - 1) / SR_TILE);
    a.hist = (uint32_t *)scratch;
    a.ctrl = a.hist + 3 * SR_BINS;
    a.gt = a.ctrl + 16;
    a.eq = a.gt + a.tiles;
    const dim3 t(SR_THREADS), hb(a.tiles < SR_BLOCKS ? a.tiles : SR_BLOCKS);
    hipLaunchKernelGGL(select_clear_kernel, dim3(3 * SR_BINS / SR_THREADS), t, 0, st, a);
    hipLaunchKernelGGL(select_hist_kernel<0>, hb, t, 0, st, a);
    hipLaunchKernelGGL(select_hist_kernel<1>, hb, t, 0, st, a);
    hipLaunchKernelGGL(select_hist_kernel<2>, hb, t, 0, st, a);
    hipLaunchKernelGGL(select_count_kernel, dim3(a.tiles), t, 0, st, a);
    hipLaunchKernelGGL(select_scan_kernel, dim3(2), dim3(1024), 0, st, a);
    hipLaunchKernelGGL(select_write_kernel, dim3(a.tiles), t, 0, st, a);
    return hipGetLastError();
}

// ------------------------------------------------------------ rows of many tensors
//
// dst[j] = src[rows[j]] for every segment, zeros where rows[j] is outside [0, P) (a
// fresh row; nothing is read).  Plain rows move in the largest power-of-two unit that
// their size and addresses allow.  8-bit states (gsr_blockscale.hpp): the rows' values
// land in other blocks of 64, whose scale is formed anew from what they hold; powers of
// two, so only values below 2^-13 of their new block's largest lose bits.
constexpr int TR_THREADS = 256, TR_SEGS = 48, TR_ITEMS = 8;
constexpr int TR_TILE = TR_THREADS * TR_ITEMS;   // units per workgroup
constexpr int TR_CODES = TR_THREADS * 4;         // codes per workgroup

struct TakeSeg {
    const void *src;
    void *dst;
    const uint8_t *src_scale;
    uint8_t *dst_scale;
    int64_t units;           // of dst
    uint32_t row, mul, shift;  // units per row; x / row = x * mul >> (31 + shift) for x < 2^31
    int32_t kind;            // log2 of the unit's bytes, or TAKE_CODES + signed
};
constexpr int TAKE_CODES = 8;
struct TakeArgs {
    const int64_t *rows;
    int64_t P;
    int nseg;
    int block0[TR_SEGS + 1];
    TakeSeg seg[TR_SEGS];
};

struct alignas(16) U128 { uint32_t x[4]; };

template <typename U>
__device__ __forceinline__ void take_units(const TakeArgs &a, const TakeSeg &s, int64_t tile) {
    const int64_t u0 = tile * TR_TILE, row0 = u0 / s.row;
    const uint32_t col0 = (uint32_t)(u0 - row0 * s.row);
    const U *src = (const U *)s.src;
    U *dst = (U *)s.dst;
    int64_t from[TR_ITEMS];
    U v[TR_ITEMS];
#pragma unroll
    for (int j = 0; j < TR_ITEMS; j++) {
        const uint32_t o = j * TR_THREADS + threadIdx.x, x = col0 + o;
        const uint32_t q = (uint32_t)((uint64_t)x * s.mul >> (31 + s.shift));
        from[j] = -1;
        if (u0 + o < s.units) {
            const int64_t r = a.rows[row0 + q];
            if ((uint64_t)r < (uint64_t)a.P) from[j] = r * s.row + (x - q * s.row);
        }
    }
#pragma unroll
    for (int j = 0; j < TR_ITEMS; j++) {
        v[j] = U{};
        if (from[j] >= 0) v[j] = src[from[j]];
    }
#pragma unroll
    for (int j = 0; j < TR_ITEMS; j++) {
        const uint32_t o = j * TR_THREADS + threadIdx.x;
        if (u0 + o < s.units) dst[u0 + o] = v[j];
    }
}

// 2^(byte - 129): a quarter of a block's scale, so that its largest code, 256, stays well in
// fp32 under the largest scale too.  A code's four bits are exact down to 2^-138.
__device__ __forceinline__ float quarter_scale(uint32_t byte) {
    return as_f32(byte > 2 ? (byte - 2) << 23 : 0x100000u << byte);
}

template <bool SIGNED>
__device__ __forceinline__ void take_codes(const TakeArgs &a, const TakeSeg &s, int64_t tile) {
    const int64_t u0 = tile * TR_CODES, row0 = u0 / s.row;
    const uint32_t col0 = (uint32_t)(u0 - row0 * s.row);
    const uint8_t *src = (const uint8_t *)s.src;
    uint32_t w = 0;
    float x[4], sc[4];
    int live = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const uint32_t o = threadIdx.x * 4 + j, c = col0 + o;
        const uint32_t q = (uint32_t)((uint64_t)c * s.mul >> (31 + s.shift));
        sc[j] = 0.f;
        if (u0 + o < s.units) {
            live++;
            const int64_t r = a.rows[row0 + q];
            if ((uint64_t)r < (uint64_t)a.P) {
                const int64_t f = r * s.row + (c - q * s.row);
                w |= (uint32_t)src[f] << 8 * j;
                sc[j] = quarter_scale(s.src_scale[f / SCALE_BLOCK]);
            }
        }
    }
    e4m3_decode4(w, x);
    uint32_t amax = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        x[j] *= sc[j];
        amax = max(amax, coded_bits(x[j]));
    }
    const uint32_t byte = scale_byte(row_max(amax) + (2u << 23));  // x is a quarter of the value
    w = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) w |= e4m3_nearest<SIGNED>(x[j], byte, 2) << 8 * j;
    const int64_t u = u0 + threadIdx.x * 4;
    uint8_t *dst = (uint8_t *)s.dst + u;
    if (live == 4) *reinterpret_cast<u32_u *>(dst) = w;
    else
        for (int j = 0; j < live; j++) dst[j] = (uint8_t)(w >> 8 * j);
    if (live && (threadIdx.x & 15) == 0) s.dst_scale[u / SCALE_BLOCK] = (uint8_t)byte;
}

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
        case 3: take_units<uint64_t>(a, s, tile); break;
        case 4: take_units<U128>(a, s, tile); break;
        case TAKE_CODES: take_codes<false>(a, s, tile); break;
        default: take_codes<true>(a, s, tile); break;
    }
}

hipError_t launch_take_rows(const gsr_rows_segment *segs, int nseg, int64_t P, const int64_t *rows, int64_t K,
                            hipStream_t st) {
    TakeArgs a;
    a.rows = rows, a.P = P;
    for (int k = 0; k < nseg;) {
        int blocks = 0;
        a.nseg = 0;
        for (; k < nseg && a.nseg < TR_SEGS; k++) {
            const gsr_rows_segment &q = segs[k];
            if (q.row_bytes == 0 || K == 0) continue;
            TakeSeg &s = a.seg[a.nseg];
            s.src = q.src, s.dst = q.dst, s.src_scale = q.src_scale, s.dst_scale = q.dst_scale;
            int unit = 0;
            if (q.kind == GSR_ROWS_PLAIN) {
                const uint64_t bits = (uint64_t)q.row_bytes | (uint64_t)(uintptr_t)q.src | (uint64_t)(uintptr_t)q.dst;
                while (unit < 4 && !(bits >> unit & 1)) unit++;
                s.kind = unit;
            } else {
                s.kind = TAKE_CODES + (q.kind == GSR_ROWS_E4M3_SIGNED ? 1 : 0);
            }
            s.row = (uint32_t)(q.row_bytes >> unit);
            s.shift = 0;
            while ((1ull << s.shift) < s.row) s.shift++;
            s.mul = (uint32_t)(((1ull << (31 + s.shift)) + s.row - 1) / s.row);
            s.units = K * (int64_t)s.row;
            const int64_t per = q.kind == GSR_ROWS_PLAIN ? TR_TILE : TR_CODES, b = (s.units + per - 1) / per;
            if (blocks && blocks + b > GSR_MAX_BLOCKS) break;  // the next launch takes it
            a.block0[a.nseg++] = blocks;
            blocks += (int)b;
        }
        if (!a.nseg) continue;
        a.block0[a.nseg] = blocks;
        hipLaunchKernelGGL(take_rows_kernel, dim3(blocks), dim3(TR_THREADS), 0, st, a);
        if (hipError_t e = hipGetLastError()) return e;
    }
    return hipSuccess;
}

}  // namespace gsr
