// adamw.hip — the AdamW step over any number of tensors, with its two moments in 32
// bits or in 8, and the global gradient norm that clips it.
//
//   g' = c g                                    c: the clip coefficient, on the device
//   m' = m + (1 - b1) (g' - m)                  v' = b2 v + (1 - b2) g'^2
//   p' = p (1 - lr wd) - lr / (1 - b1^t) m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
//
// The operations are those of torch.optim.AdamW in its order, in fp32, except that
// the bias correction of the root is a product with its reciprocal and, with 8-bit states, the
// quotient a product with the hardware's (one ulp; a division costs those 158 us instead
// of 153, at 59M elements, and the 32-bit ones nothing: 268 us either way).
//
// One pass over the data, 4 consecutive elements a lane; the tensors' table travels in the
// kernel's arguments (40 tensors a launch), so nothing is uploaded and nothing is kept.
// Memory bounds it: 28 bytes an element with 32-bit states, 16 with 8-bit ones.  59M
// elements (1M Gaussians): 265 us = 6.2 TB/s and 150 us = 6.3 TB/s, where a large copy
// reaches 4.8 and an addition of two arrays 5.85.  All of it streams non-temporally: 306
// us (32 bits) with ordinary accesses, 277 with the parameters alone kept in the caches (too
// large to be there at the next render).  Two or four vectors a lane: 282, 282 us.
//
// 8-bit states hold m and r = sqrt(v) (half the range of v's exponents) as e4m3 codes
// with a power-of-two scale for every 64 elements (gsr_blockscale.hpp).  They are
// rounded stochastically: an e4m3 step is 6-12 % of the value, one update moves v by
// (1 - b2) = 0.1 %, so rounding to nearest would never let a second moment fall, and
// would hold the first moments of Gaussians that no view sees at their last few codes,
// which then drift for ever.  The parameter is updated from the fp32 moments before
// they are rounded.  75 instructions an element leave it to memory, with the test for
// infinities and NaN made once a wave (for every element: 157 us instead of 153).  With bf16
// parameters, 87 instructions for 10 bytes, arithmetic bounds it: 125 us = 4.8 TB/s.
//
// Parameters and gradients are fp32 or bf16; a bf16 parameter is rounded
// stochastically too (an update below 2^-9 of the parameter would be lost).
#include <cmath>

#include "gsr_blockscale.hpp"
#include "gsr_kernels.hpp"

// every product and sum rounds by itself, as in the formulas above: the codes then do
// not depend on which of them the compiler would have fused
#pragma clang fp contract(off)

namespace gsr {

constexpr int AW_THREADS = 256, AW_VEC = 4, AW_SEGS = 40;  // 40 segments: 3.1 KB of kernel arguments
constexpr int AW_TILE = AW_THREADS * AW_VEC;               // elements per workgroup

struct AdamWSeg {
    void *p;
    const void *g;
    void *m, *v;           // float, or e4m3 codes of m and sqrt(v)
    uint8_t *ms, *vs;      // their scales
    int64_t n;
    float decay, neg_step, inv_bc2;
    uint32_t key;
};
struct AdamWArgs {
    int nseg;
    float w1, b2, w2, eps;
    const float *scale;  // NULL: 1
    int block0[AW_SEGS + 1];
    AdamWSeg seg[AW_SEGS];
};

template <typename T>
struct Elems;
template <>
struct Elems<float> {
    static __device__ __forceinline__ void load4(const float *s, float x[4]) {
        const f32x4_u *at = reinterpret_cast<const f32x4_u *>(s);
        const f32x4_u v = __builtin_nontemporal_load(at);
        x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
    }
    static __device__ __forceinline__ float load(const float *s) { return *s; }
    static __device__ __forceinline__ float round(float x, uint32_t) { return x; }
    static __device__ __forceinline__ void store4(float *d, const float x[4]) {
        f32x4_u v = {x[0], x[1], x[2], x[3]}, *at = reinterpret_cast<f32x4_u *>(d);
        __builtin_nontemporal_store(v, at);
    }
    static __device__ __forceinline__ void store(float *d, float x) { *d = x; }
};
template <>
struct Elems<uint16_t> {  // bf16
    static __device__ __forceinline__ void load4(const uint16_t *s, float x[4]) {
        const u16x4_u *at = reinterpret_cast<const u16x4_u *>(s);
        const u16x4_u v = __builtin_nontemporal_load(at);
        x[0] = as_f32((uint32_t)v.x << 16), x[1] = as_f32((uint32_t)v.y << 16);
        x[2] = as_f32((uint32_t)v.z << 16), x[3] = as_f32((uint32_t)v.w << 16);
    }
    static __device__ __forceinline__ float load(const uint16_t *s) { return as_f32((uint32_t)*s << 16); }
    // 16 more bits of the element's word (the moments take its halves) decide the rounding
    static __device__ __forceinline__ float round(float x, uint32_t word) {
        const uint32_t b = as_u32(x);
        if ((b & 0x7F800000u) == 0x7F800000u) return as_f32(b | ((b & 0x7FFFFFu) ? 0x400000u : 0u));  // a NaN stays one
        return as_f32(b + ((word * 0x9E3779B9u) >> 16));
    }
    static __device__ __forceinline__ void store4(uint16_t *d, const float x[4]) {
        u16x4_u v = {(uint16_t)(as_u32(x[0]) >> 16), (uint16_t)(as_u32(x[1]) >> 16), (uint16_t)(as_u32(x[2]) >> 16),
                     (uint16_t)(as_u32(x[3]) >> 16)};
        u16x4_u *at = reinterpret_cast<u16x4_u *>(d);
        __builtin_nontemporal_store(v, at);
    }
    static __device__ __forceinline__ void store(uint16_t *d, float x) { *d = (uint16_t)(as_u32(x) >> 16); }
};

// the segment of a workgroup: the last one that starts at or before it
__device__ __forceinline__ int segment_of(const int *block0, int nseg, int b) {
    int lo = 0, hi = nseg;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (block0[mid] <= b) lo = mid;
        else hi = mid;
    }
    return lo;
}

template <bool BITS8>
__device__ __forceinline__ void adamw_one(const AdamWArgs &a, const AdamWSeg &s, float c, float &p, float g, float &m,
                                          float &v, float &r) {
    const float x = g * c;
    m = m + (x - m) * a.w1;
    v = v * a.b2 + (x * x) * a.w2;
    r = sqrtf(v);
    const float d = r * s.inv_bc2 + a.eps;
    p = p * s.decay + (BITS8 ? m * __builtin_amdgcn_rcpf(d) : m / d) * s.neg_step;
}

// Four consecutive elements of a segment, as a lane holds them
template <typename T, bool BITS8>
struct AdamWLane {
    float P[4], G[4], M[4], V[4], R[4];
    uint32_t mw, rw, mb, rb;  // 8-bit states: codes and scale bytes
    int64_t i;
    int live;  // elements that exist

    __device__ __forceinline__ void load(const AdamWSeg &s, int64_t at) {
        i = at;
        live = (int)(s.n - i < AW_VEC ? (s.n - i > 0 ? s.n - i : 0) : AW_VEC);
        const T *p = (const T *)s.p + i, *g = (const T *)s.g + i;
        const uint8_t *mc = (const uint8_t *)s.m + i, *rc = (const uint8_t *)s.v + i;
        const float *m = (const float *)s.m + i, *v = (const float *)s.v + i;
#pragma unroll
        for (int j = 0; j < 4; j++) P[j] = G[j] = M[j] = V[j] = 0.f;
        mw = rw = mb = rb = 0;
        if (live == AW_VEC) {
            Elems<T>::load4(p, P);
            Elems<T>::load4(g, G);
            if (BITS8) {
                mw = __builtin_nontemporal_load(reinterpret_cast<const u32_u *>(mc));
                rw = __builtin_nontemporal_load(reinterpret_cast<const u32_u *>(rc));
            } else {
                Elems<float>::load4(m, M);
                Elems<float>::load4(v, V);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (j >= live) continue;
                P[j] = Elems<T>::load(p + j), G[j] = Elems<T>::load(g + j);
                if (BITS8) mw |= (uint32_t)mc[j] << 8 * j, rw |= (uint32_t)rc[j] << 8 * j;
                else M[j] = m[j], V[j] = v[j];
            }
        }
        if (BITS8 && live) mb = s.ms[i / SCALE_BLOCK], rb = s.vs[i / SCALE_BLOCK];
    }

    __device__ __forceinline__ void step(const AdamWArgs &a, const AdamWSeg &s, float c) {
        if (BITS8) {
            const float msc = block_scale(mb), rsc = block_scale(rb);
            e4m3_decode4(mw, M);
            e4m3_decode4(rw, R);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                M[j] *= msc;
                R[j] *= rsc;
                V[j] = R[j] * R[j];
            }
        }
#pragma unroll
        for (int j = 0; j < 4; j++) adamw_one<BITS8>(a, s, c, P[j], G[j], M[j], V[j], R[j]);
        if (BITS8) {
            uint32_t ma = 0, ra = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                ma = max(ma, as_u32(M[j]) & 0x7FFFFFFFu);
                ra = max(ra, as_u32(R[j]) & 0x7FFFFFFFu);
            }
            // a moment past the codes' range anywhere in the wave: every element is tested
            if (__any(max(ma, ra) >= E4M3_TOP)) {
                encode<true>(s);
            } else {
                mb = scale_byte(row_max(ma));
                rb = scale_byte(row_max(ra));
                encode<false>(s);
            }
        } else if (sizeof(T) == 2) {
#pragma unroll
            for (int j = 0; j < 4; j++) P[j] = Elems<T>::round(P[j], dither_word((uint64_t)(i + j), s.key));
        }
    }

    template <bool TEST>
    __device__ __forceinline__ void encode(const AdamWSeg &s) {
        if (TEST) {
            uint32_t ma = 0, ra = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                ma = max(ma, coded_bits(M[j]));
                ra = max(ra, coded_bits(R[j]));
            }
            mb = scale_byte(row_max(ma));
            rb = scale_byte(row_max(ra));
        }
        mw = rw = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint32_t w = dither_word((uint64_t)(i + j), s.key);
            mw |= e4m3_stochastic<true, TEST>(M[j], mb, w >> 16) << 8 * j;
            rw |= e4m3_stochastic<false, TEST>(R[j], rb, w & 0xFFFFu) << 8 * j;
            P[j] = Elems<T>::round(P[j], w);
        }
    }

    __device__ __forceinline__ void store(const AdamWSeg &s) const {
        T *p = (T *)s.p + i;
        uint8_t *mc = (uint8_t *)s.m + i, *rc = (uint8_t *)s.v + i;
        float *m = (float *)s.m + i, *v = (float *)s.v + i;
        if (live == AW_VEC) {
            Elems<T>::store4(p, P);
            if (BITS8) {
                __builtin_nontemporal_store(mw, reinterpret_cast<u32_u *>(mc));
                __builtin_nontemporal_store(rw, reinterpret_cast<u32_u *>(rc));
            } else {
                Elems<float>::store4(m, M);
                Elems<float>::store4(v, V);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (j >= live) continue;
                Elems<T>::store(p + j, P[j]);
                if (BITS8) mc[j] = (uint8_t)(mw >> 8 * j), rc[j] = (uint8_t)(rw >> 8 * j);
                else m[j] = M[j], v[j] = V[j];
            }
        }
        if (BITS8 && live && i % SCALE_BLOCK == 0) s.ms[i / SCALE_BLOCK] = (uint8_t)mb, s.vs[i / SCALE_BLOCK] = (uint8_t)rb;
    }
};

template <typename T, bool BITS8>
__global__ void __launch_bounds__(AW_THREADS) adamw_kernel(AdamWArgs a) {
    const int k = segment_of(a.block0, a.nseg, (int)blockIdx.x);
    const AdamWSeg &s = a.seg[k];
    const int64_t i = (int64_t)((int)blockIdx.x - a.block0[k]) * AW_TILE + threadIdx.x * AW_VEC;
    const float c = a.scale ? *a.scale : 1.f;
    AdamWLane<T, BITS8> e;
    e.load(s, i);
    e.step(a, s, c);
    e.store(s);
}

hipError_t launch_adamw(const gsr_adamw_segment *segs, int nseg, int dtype, int state_bits, double beta1, double beta2,
                        double eps, const float *grad_scale, uint64_t seed, hipStream_t st) {
    AdamWArgs a;
    a.w1 = (float)(1.0 - beta1);
    a.b2 = (float)beta2;
    a.w2 = (float)(1.0 - beta2);
    a.eps = (float)eps;
    a.scale = grad_scale;
    for (int k = 0; k < nseg;) {
        int blocks = 0;
        a.nseg = 0;
        for (; k < nseg && a.nseg < AW_SEGS; k++) {
            const gsr_adamw_segment &q = segs[k];
            const int64_t b = (q.n + AW_TILE - 1) / AW_TILE;
            if (b == 0) continue;
            if (blocks && blocks + b > GSR_MAX_BLOCKS) break;  // the next launch takes it
            AdamWSeg &s = a.seg[a.nseg];
            s.p = q.param, s.g = q.grad, s.m = q.exp_avg, s.v = q.exp_second;
            s.ms = q.avg_scale, s.vs = q.second_scale;
            s.n = q.n;
            s.decay = (float)(1.0 - q.lr * q.weight_decay);
            s.neg_step = (float)(-q.lr / (1.0 - std::pow(beta1, q.step)));
            s.inv_bc2 = (float)(1.0 / std::sqrt(1.0 - std::pow(beta2, q.step)));
            s.key = dither_key(seed, (uint32_t)q.step, (uint32_t)q.ordinal);
            a.block0[a.nseg++] = blocks;
            blocks += (int)b;
        }
        if (!a.nseg) continue;
        a.block0[a.nseg] = blocks;
        const dim3 g(blocks), t(AW_THREADS);
        if (dtype == GSR_DTYPE_F32 && state_bits == 32) hipLaunchKernelGGL((adamw_kernel<float, false>), g, t, 0, st, a);
        else if (dtype == GSR_DTYPE_F32) hipLaunchKernelGGL((adamw_kernel<float, true>), g, t, 0, st, a);
        else if (state_bits == 32) hipLaunchKernelGGL((adamw_kernel<uint16_t, false>), g, t, 0, st, a);
        else hipLaunchKernelGGL((adamw_kernel<uint16_t, true>), g, t, 0, st, a);
        if (hipError_t e = hipGetLastError()) return e;
    }
    return hipSuccess;
}

// ------------------------------------------------------------ global gradient norm
//
// norm = sqrt(sum g^2) over all tensors, c = min(1, max_norm / (norm + 1e-6)).  Squares
// and sums in 64 bits (the fp64 rate is far above what the stream of gradients needs): no
// overflow, the same bits for the same list of tensors, and for another split of the same
// values a sum that may differ in the last of its 53 bits.  Each workgroup leaves one partial
// sum; one workgroup adds them in a fixed order.  1180 MB in 193 us = 6.1 TB/s; 177 MB of 96
// bf16 tensors in 47 us = 3.8 TB/s: ten 16 KB tiles a workgroup, each behind a search of the table
// and its own loads.  2048 workgroups: 266 us instead of 249 a call for the large one, behind 1
// GB of writes.  The loads stay in the caches, for the step that follows: read non-temporally,
// both together cost 404 us instead of 385 (the 177 MB).
constexpr int GN_THREADS = 256, GN_SEGS = 128, GN_BLOCKS = 1024, GN_UNROLL = 4;
constexpr int64_t gn_tile(int dtype) { return GN_THREADS * GN_UNROLL * (dtype == GSR_DTYPE_F32 ? 4 : 8); }  // 16 KB
struct NormArgs {
    int nseg, tiles;
    double *partials;
    int tile0[GN_SEGS + 1];
    gsr_grad_segment seg[GN_SEGS];
};

__device__ __forceinline__ double add_square(double acc, float x) {
    return __builtin_fma((double)x, (double)x, acc);
}
// 16 bytes of gradients (cached: the step reads them again)
__device__ __forceinline__ double add_squares(double acc, u32x4_u v, float) {
#pragma unroll
    for (int j = 0; j < 4; j++) acc = add_square(acc, as_f32(v[j]));
    return acc;
}
__device__ __forceinline__ double add_squares(double acc, u32x4_u v, uint16_t) {
#pragma unroll
    for (int j = 0; j < 4; j++) acc = add_square(add_square(acc, as_f32(v[j] << 16)), as_f32(v[j] & 0xFFFF0000u));
    return acc;
}
template <typename T>
__device__ __forceinline__ double square_sum(const T *g, int64_t n) {
    constexpr int VEC = 16 / sizeof(T), TILE = GN_THREADS * GN_UNROLL * VEC;
    double acc = 0;
    if (n >= TILE) {
        u32x4_u v[GN_UNROLL];
#pragma unroll
        for (int u = 0; u < GN_UNROLL; u++)
            v[u] = *reinterpret_cast<const u32x4_u *>(g + (u * GN_THREADS + threadIdx.x) * VEC);
#pragma unroll
        for (int u = 0; u < GN_UNROLL; u++) acc = add_squares(acc, v[u], T(0));
    } else {
        for (int64_t i = threadIdx.x; i < n; i += GN_THREADS) acc = add_square(acc, Elems<T>::load(g + i));
    }
    return acc;
}

template <int THREADS>
__device__ __forceinline__ double block_sum_f64(double v, double *red) {
    for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    double t = 0;
    for (int k = 0; k < THREADS / 64; k++) t += red[k];
    return t;
}

__global__ void __launch_bounds__(GN_THREADS) grad_norm_kernel(NormArgs a) {
    __shared__ double red[GN_THREADS / 64];
    double acc = 0;
    for (int t = blockIdx.x; t < a.tiles; t += gridDim.x) {
        const int k = segment_of(a.tile0, a.nseg, t);
        const gsr_grad_segment &s = a.seg[k];
        const int64_t i = (t - a.tile0[k]) * gn_tile(s.dtype);
        acc += s.dtype == GSR_DTYPE_F32 ? square_sum((const float *)s.grad + i, s.n - i)
                                        : square_sum((const uint16_t *)s.grad + i, s.n - i);
    }
    const double t = block_sum_f64<GN_THREADS>(acc, red);
    if (threadIdx.x == 0) a.partials[blockIdx.x] = t;
}

constexpr int GNF_THREADS = 1024;
__global__ void __launch_bounds__(GNF_THREADS) grad_norm_finish_kernel(const double *partials, int n, double max_norm,
                                                                       float *out) {
    __shared__ double red[GNF_THREADS / 64];
    double acc = 0;
    for (int i = threadIdx.x; i < n; i += GNF_THREADS) acc += partials[i];
    const double norm = sqrt(block_sum_f64<GNF_THREADS>(acc, red));
    if (threadIdx.x == 0) {
        const double c = max_norm / (norm + 1e-6);
        out[0] = (float)norm;
        out[1] = c >= 1.0 ? 1.f : (float)c;  // a NaN norm stays NaN, as an infinite one gives 0
    }
}

size_t grad_norm_scratch_bytes(int nseg) {
    return (size_t)((nseg + GN_SEGS - 1) / GN_SEGS) * GN_BLOCKS * sizeof(double);
}

hipError_t launch_grad_norm(const gsr_grad_segment *segs, int nseg, double max_norm, void *scratch, float *out,
                            hipStream_t st) {
    NormArgs a;
    int parts = 0;
    for (int k = 0; k < nseg;) {
        a.nseg = 0, a.tiles = 0;
        // a launch takes GN_SEGS entries of the list, empty ones too: the scratch holds one
        // set of partial sums for each
        for (int q = 0; q < GN_SEGS && k < nseg; q++, k++) {
            const int64_t t = (segs[k].n + gn_tile(segs[k].dtype) - 1) / gn_tile(segs[k].dtype);
            if (t == 0) continue;
            a.seg[a.nseg] = segs[k];
            a.tile0[a.nseg++] = a.tiles;
            a.tiles += (int)t;
        }
        if (!a.nseg) continue;
        a.tile0[a.nseg] = a.tiles;
        const int blocks = a.tiles < GN_BLOCKS ? a.tiles : GN_BLOCKS;
        a.partials = (double *)scratch + parts;
        parts += blocks;
        hipLaunchKernelGGL(grad_norm_kernel, dim3(blocks), dim3(GN_THREADS), 0, st, a);
        if (hipError_t e = hipGetLastError()) return e;
    }
    hipLaunchKernelGGL(grad_norm_finish_kernel, dim3(1), dim3(GNF_THREADS), 0, st, (const double *)scratch, parts,
                       max_norm, out);
    return hipGetLastError();
}

}  // namespace gsr
