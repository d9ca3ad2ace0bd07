// Root-mean-square norm of rows with the residual's addition, its backward pass, and its output as
// e4m3 with scales.  A row operator like the softmax of softmax.cu (the leaves it stands beside are
// the reference's row reductions, apps/common/annot/functions.h:9-173); the reference has no norm.
//
//   h = x + residual,   r = 1 / sqrt(mean_j h_j^2 + eps),   y_j = h_j r w_j
//   dh_j = r (w_j dy_j - xhat_j mean_k(w_k dy_k xhat_k)) + dresidual_j,   xhat_j = h_j r
//   dw_j = sum over rows of dy_j xhat_j
//
// Bound: HBM.  Forward 8 bytes per bf16 element (x, residual in; y, h out), backward 8 (dy, h,
// dresidual in; dh out).  16384 x 4096 bf16: forward 80 us (6.7 TB/s), backward 92 us (5.8 TB/s, 4 of them
// the join of dweight's partial sums); e4m3 with a scale per 128 columns 4096 x 8192: 40-43 us (5.5-5.9 TB/s).
// A team of threads (8 lanes up to a block of 1024) owns a row and keeps it in
// registers, so every operand is read once; sums are fp32.  y is formed from the unrounded sum and
// rounded once; h is rounded once, where it is stored.  The backward pass takes the stored h and
// forms r from it again (the sum rides along with the one it needs anyway), so it is the exact
// gradient of the norm at that h and no per-row state is kept between the passes.
#include <algorithm>
#include <atomic>
#include <cuda_fp8.h>
#include <math.h>

#include "common.cuh"

namespace gb200 {
namespace {

// Smallest scale of a group in the e4m3 output: a group of zeros (or of values whose largest is below
// 448 * 2^-126) gets it, so that nothing is divided by zero or by a denormal.
constexpr float kScaleFloor = 1.17549435e-38f;   // 2^-126
constexpr float kE4m3Max = 448.0f;
constexpr int kLongCols = 16384;                 // longer rows are read again instead of kept

// Scale of a group whose largest |y| is `top`: top / 448 rounded once, whichever kernel the row goes through.  The product
// with the rounded reciprocal, corrected by the remainder it leaves (Markstein 1990), is that quotient for every
// significand (all 2^23 tried); an infinite one has no remainder.  4096 x 8192: 39.8 us, 40.7 with a division.
__device__ __forceinline__ float scale_of(float top) {
    constexpr float inv = 1.0f / kE4m3Max;
    const float q = top * inv, rest = fmaf(-kE4m3Max, q, top);
    return fmaxf(rest == rest ? fmaf(rest, inv, q) : q, kScaleFloor);
}

template <typename T, int V> struct Pack;        // V elements moved by one load
template <> struct Pack<float, 4> { using type = float4; };
template <> struct Pack<float, 1> { using type = float; };
struct alignas(32) Eight { uint32_t w[8]; };
template <> struct Pack<__nv_bfloat16, 16> { using type = Eight; };
template <> struct Pack<__nv_bfloat16, 8> { using type = uint4; };
template <> struct Pack<__nv_bfloat16, 2> { using type = uint32_t; };
template <> struct Pack<__nv_bfloat16, 1> { using type = unsigned short; };

__device__ __forceinline__ void widen(const float4 &p, float (&v)[4]) { v[0] = p.x; v[1] = p.y; v[2] = p.z; v[3] = p.w; }
__device__ __forceinline__ void widen(const float &p, float (&v)[1]) { v[0] = p; }
__device__ __forceinline__ void widen2(uint32_t w, float &lo, float &hi) {
    lo = __uint_as_float(w << 16);
    hi = __uint_as_float(w & 0xffff0000u);
}
__device__ __forceinline__ void widen(const uint4 &p, float (&v)[8]) {
    widen2(p.x, v[0], v[1]);
    widen2(p.y, v[2], v[3]);
    widen2(p.z, v[4], v[5]);
    widen2(p.w, v[6], v[7]);
}
__device__ __forceinline__ void widen(const Eight &p, float (&v)[16]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) widen2(p.w[i], v[2 * i], v[2 * i + 1]);
}
__device__ __forceinline__ void widen(const uint32_t &p, float (&v)[2]) { widen2(p, v[0], v[1]); }
__device__ __forceinline__ void widen(const unsigned short &p, float (&v)[1]) { v[0] = __uint_as_float(static_cast<uint32_t>(p) << 16); }

__device__ __forceinline__ void narrow(const float (&v)[4], float4 &p) { p = make_float4(v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ void narrow(const float (&v)[1], float &p) { p = v[0]; }
__device__ __forceinline__ void narrow(const float (&v)[8], uint4 &p) {
    p = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
}
__device__ __forceinline__ void narrow(const float (&v)[16], Eight &p) {
#pragma unroll
    for (int i = 0; i < 8; ++i) p.w[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
}
__device__ __forceinline__ void narrow(const float (&v)[2], uint32_t &p) { p = pack_bf16(v[0], v[1]); }
__device__ __forceinline__ void narrow(const float (&v)[1], unsigned short &p) { p = __bfloat16_as_ushort(__float2bfloat16_rn(v[0])); }

template <typename P> __device__ __forceinline__ P load_row(const P *p) { return __ldcs(p); }
template <typename P> __device__ __forceinline__ P load_weight(const P *p) { return __ldg(p); }
template <typename P> __device__ __forceinline__ void store_row(P *p, const P &v) { __stcs(p, v); }
template <> __device__ __forceinline__ Eight load_row(const Eight *p) {
    Eight v;
    ld_global_256(p, v.w);
    return v;
}
template <> __device__ __forceinline__ Eight load_weight(const Eight *p) { return load_row(p); }
template <> __device__ __forceinline__ void store_row(Eight *p, const Eight &v) {
    st_global_256(p, v.w[0], v.w[1], v.w[2], v.w[3], v.w[4], v.w[5], v.w[6], v.w[7]);
}

// V floats -> V e4m3 bytes (round to nearest even, saturating; NaN stays NaN)
template <int V>
__device__ __forceinline__ void store_e4m3(const float (&v)[V], uint8_t *dst) {
    if constexpr (V == 1) {
        *dst = __nv_cvt_float_to_fp8(v[0], __NV_SATFINITE, __NV_E4M3);
    } else {
        static_assert(V == 4 || V == 8 || V == 16);
        uint16_t w[V / 2];
#pragma unroll
        for (int i = 0; i < V / 2; ++i)
            w[i] = __nv_cvt_float2_to_fp8x2(make_float2(v[2 * i], v[2 * i + 1]), __NV_SATFINITE, __NV_E4M3);
        if constexpr (V == 16)
            *reinterpret_cast<uint4 *>(dst) = make_uint4(w[0] | (uint32_t)w[1] << 16, w[2] | (uint32_t)w[3] << 16,
                                                         w[4] | (uint32_t)w[5] << 16, w[6] | (uint32_t)w[7] << 16);
        else if constexpr (V == 8)
            *reinterpret_cast<uint2 *>(dst) = make_uint2(w[0] | (uint32_t)w[1] << 16, w[2] | (uint32_t)w[3] << 16);
        else
            *reinterpret_cast<uint32_t *>(dst) = w[0] | (uint32_t)w[1] << 16;
    }
}

// Sum over the TEAM lanes of a team that share a warp (the whole warp for larger teams).
template <int TEAM> __device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
    for (int o = (TEAM < 32 ? TEAM : 32) / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
template <int TEAM> __device__ __forceinline__ float lanes_max(float v) {    // of non-negative values
    if constexpr (TEAM >= 32) return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v)));
#pragma unroll
    for (int o = TEAM / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// Sum of K values over the team's threads.  Teams of more than a warp are whole blocks; `red` is
// double-buffered by `parity`, so one block barrier per call is enough as long as calls alternate it.
template <int TEAM, int K>
__device__ __forceinline__ void team_sum(float (&s)[K], float (*red)[2][32], int parity) {
#pragma unroll
    for (int k = 0; k < K; ++k) s[k] = lanes_sum<TEAM>(s[k]);
    if constexpr (TEAM > 32) {
        const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, warps = blockDim.x >> 5;
        if (lane == 0)
#pragma unroll
            for (int k = 0; k < K; ++k) red[k][parity][wid] = s[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k) s[k] = warp_sum(lane < warps ? red[k][parity][lane] : 0.0f);
    }
}

// Sum of the team's `s`, largest of its non-negative `m` (WITH_MAX) and union of its `flags`, in one block barrier.
template <int TEAM, bool WITH_MAX>
__device__ __forceinline__ void team_sum_max(float &s, float &m, unsigned &flags, float4 *red) {
    s = lanes_sum<TEAM>(s);
    flags = __reduce_or_sync(0xffffffffu, flags);
    if (WITH_MAX) m = lanes_max<TEAM>(m);
    if constexpr (TEAM > 32) {
        const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
        if (lane == 0) red[wid] = make_float4(s, __uint_as_float(flags), m, 0.0f);
        __syncthreads();
        const float4 v = lane < static_cast<int>(blockDim.x >> 5) ? red[lane] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        s = warp_sum(v.x);
        flags = __reduce_or_sync(0xffffffffu, __float_as_uint(v.y));
        if (WITH_MAX) m = lanes_max<32>(v.z);
    }
}

struct NormArgs {
    const void *x, *residual, *weight;
    int64_t ldx, ldr;
    void *y, *h;
    int64_t ldy, ldh;
    float *scales;
    int64_t lds;
    int64_t rows;
    int cols, group;     // group: columns per scale of the e4m3 output, 0 = the whole row
    float eps;
};

template <int TEAM> constexpr int kBlock = TEAM < 128 ? 128 : TEAM;

template <typename T> __device__ __forceinline__ float load_one(const T *p);
template <> __device__ __forceinline__ float load_one(const float *p) { return *p; }
template <> __device__ __forceinline__ float load_one(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
__device__ __forceinline__ void store_one(float v, float *p) { *p = v; }
__device__ __forceinline__ void store_one(float v, __nv_bfloat16 *p) { *p = __float2bfloat16_rn(v); }

// A vector's elements from any element's address.
__device__ __forceinline__ void load_any(const float *p, float4 &v) { v = make_float4(p[0], p[1], p[2], p[3]); }
__device__ __forceinline__ void load_any(const __nv_bfloat16 *p, uint4 &v) {
    if ((reinterpret_cast<uintptr_t>(p) & 3) == 0) {
        const uint32_t *q = reinterpret_cast<const uint32_t *>(p);
        v = make_uint4(q[0], q[1], q[2], q[3]);
    } else {
        const unsigned short *h = reinterpret_cast<const unsigned short *>(p);
        const uint32_t *q = reinterpret_cast<const uint32_t *>(h + 1);
        const uint32_t w0 = q[0], w1 = q[1], w2 = q[2];
        v = make_uint4(h[0] | w0 << 16, __funnelshift_l(w0, w1, 16), __funnelshift_l(w1, w2, 16),
                       w2 >> 16 | static_cast<uint32_t>(h[7]) << 16);
    }
}
// e4m3 bytes of a vector to any address.
template <int V>
__device__ __forceinline__ void store_e4m3_any(const float (&v)[V], uint8_t *dst) {
    uint8_t b[V];
#pragma unroll
    for (int i = 0; i < V; i += 2) {
        const uint16_t w = __nv_cvt_float2_to_fp8x2(make_float2(v[i], v[i + 1]), __NV_SATFINITE, __NV_E4M3);
        b[i] = static_cast<uint8_t>(w);
        b[i + 1] = static_cast<uint8_t>(w >> 8);
    }
    if ((reinterpret_cast<uintptr_t>(dst) & 3) == 0) {
#pragma unroll
        for (int i = 0; i < V; i += 4)
            *reinterpret_cast<uint32_t *>(dst + i) = b[i] | b[i + 1] << 8 | b[i + 2] << 16 | static_cast<uint32_t>(b[i + 3]) << 24;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) dst[i] = b[i];
    }
}

// QUANT: y is e4m3 with scales.  NV vectors of V elements per thread, TEAM threads per row (FIT: as many as the block
// has, TEAM at most; single elements keep their offsets constant, 96 against 126 us in the backward pass).
// PEEL: rows do not start on 16 bytes, but x, residual, y and residual_out lie alike: the elements before a
// row's first 16-byte boundary and behind its last (fewer than 2 V) are taken singly, one by a thread, and
// the vectors between them as if the row were aligned.  Loaded one by one, bf16 rows of 4095 columns ran at
// 27 % of the copy rate (16384 rows: 307 us).
// Blocks per SM that the e4m3 form's registers must leave room for.  Left alone it takes up to 64 registers with 16
// columns a thread, and the rows in flight get too few (4096 columns, a scale per 128: 86 us with 54, 76 with 48).
constexpr int min_blocks(int V, int NV, int TEAM, bool peel) {
    const int block = TEAM < 128 ? 128 : TEAM;
    if (V >= 8 && V * NV == 16 && TEAM < 1024) return (peel || V == 16 ? 1280 : 1536) / block;
    if (V == 16 && NV == 2 && TEAM >= 128) return (TEAM == 512 ? 1024 : 768) / block;
    return 0;    // no limit
}
template <typename T, int V, int NV, int TEAM, bool QUANT, bool PEEL, bool FIT>
__global__ void __launch_bounds__(kBlock<TEAM>, QUANT ? min_blocks(V, NV, TEAM, PEEL) : V == 16 && NV == 2 && TEAM == 512 ? 2 : 0)
rmsnorm_kernel(const NormArgs a) {
    using P = typename Pack<T, V>::type;
    constexpr int TEAMS = kBlock<TEAM> / TEAM;
    constexpr int SLOTS = TEAM * NV * V / 32 + (PEEL ? 1 : 0);       // groups a row can have
    __shared__ float4 red4[QUANT ? 32 : 1];
    __shared__ float red[1][2][32];
    __shared__ int amax[QUANT ? TEAMS * SLOTS : 1];                  // bits of non-negative floats order like ints
    pdl_launch_dependents();
    static_assert(TEAM >= 32 || (!PEEL && V >= 4), "teams that share a warp take whole vectors");
    const int width = FIT ? blockDim.x : TEAM;
    const int t = TEAM > 32 ? threadIdx.x : threadIdx.x % TEAM, team = TEAM > 32 ? 0 : threadIdx.x / TEAM;
    pdl_wait();
    const int64_t row = static_cast<int64_t>(blockIdx.x) * TEAMS + team;
    if (row - team % (TEAM < 32 ? 32 / TEAM : 1) >= a.rows) return;   // whole warps
    const bool live = TEAM >= 32 || row < a.rows;                     // (a dead team has no columns)
    const T *xr = static_cast<const T *>(a.x) + row * a.ldx;
    const T *rr = a.residual ? static_cast<const T *>(a.residual) + row * a.ldr : nullptr;
    T *hr = a.h ? static_cast<T *>(a.h) + row * a.ldh : nullptr;
    const T *wr = static_cast<const T *>(a.weight);
    const int head = PEEL ? min(static_cast<int>((16 - (reinterpret_cast<uintptr_t>(xr) & 15)) & 15) / static_cast<int>(sizeof(T)), a.cols) : 0;
    const int nvec = live ? (a.cols - head) / V : 0;
    // PEEL: this thread's single element, if it has one
    const int tail = head + nvec * V;
    const int one = t < head ? t : tail + t - head;
    const bool single = PEEL && one < a.cols && (t < head || one >= tail);
    const P *x = reinterpret_cast<const P *>(xr + head), *res = reinterpret_cast<const P *>(rr ? rr + head : nullptr);
    P px[NV], pr[NV], pw[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int idx = t + width * i;
        px[i] = P{};
        pr[i] = P{};
        if (idx < nvec) {
            px[i] = load_row(x + idx);
            if (rr) pr[i] = load_row(res + idx);
        }
    }
    if constexpr (QUANT && (PEEL || V < 4)) {    // groups' maxima meet in shared memory: zeroed while the loads are on their way
        for (int g = t; g < SLOTS; g += width) amax[team * SLOTS + g] = 0;
        if constexpr (TEAM > 32) __syncthreads();
        else __syncwarp();
    }
    float h1 = 0.0f, w1 = 0.0f;
    if (single) {
        h1 = load_one(xr + one);
        if (rr) h1 += load_one(rr + one);
        w1 = load_one(wr + one);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {   // the weight's load overlaps the reduction
        const int idx = t + width * i;
        pw[i] = P{};
        if (idx < nvec) {
            if constexpr (PEEL) load_any(wr + head + idx * V, pw[i]);
            else pw[i] = load_weight(reinterpret_cast<const P *>(wr) + idx);
        }
    }
    float h[NV][V];
    float s[1] = {h1 * h1};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        float r[V];
        widen(px[i], h[i]);
        widen(pr[i], r);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if (rr) h[i][j] += r[j];
            s[0] = fmaf(h[i][j], h[i][j], s[0]);
        }
    }
    auto store_h = [&] {
        if (!hr) return;
        P *dst = reinterpret_cast<P *>(hr + head);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int idx = t + width * i;
            P p;
            narrow(h[i], p);
            if (idx < nvec) store_row(dst + idx, p);
        }
        if (single) store_one(h1, hr + one);
    };
    if constexpr (!QUANT) {
        store_h();
        team_sum<TEAM>(s, red, 0);
        const float rs = rsqrtf(s[0] / static_cast<float>(a.cols) + a.eps);
        T *yr = static_cast<T *>(a.y) + row * a.ldy;
        P *dst = reinterpret_cast<P *>(yr + head);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int idx = t + width * i;
            float wv[V];
            widen(pw[i], wv);
#pragma unroll
            for (int j = 0; j < V; ++j) h[i][j] = h[i][j] * rs * wv[j];
            P p;
            narrow(h[i], p);
            if (idx < nvec) store_row(dst + idx, p);
        }
        if (single) store_one(h1 * rs * w1, yr + one);
    } else {
        // With m the largest |h w| of a group, y / scale = h w 448 / m and scale = m r / 448: the bytes do not need r,
        // and the maxima are found before the barrier that r waits for.  That holds while h w, m r and 448 / m are
        // well inside fp32's range, which is tested on the parts of the groups' maxima that warps hold, and on r.
        // A row where it does not hold is read again, and its bytes formed from y itself; so nothing that it is
        // read from is written before that is known.
        constexpr float kSmall = 8.6736174e-19f, kLarge = 1.2676506e30f;         // 2^-60, 2^100
        constexpr float kSmallR = 8.8817842e-16f, kLargeR = 1.1258999e15f;       // 2^-50, 2^50
        constexpr float kZeroR = 1024.0f;     // h w that is 0 in fp32 gives a y below 2^-139, which is 0 at the smallest scale
        constexpr unsigned kZero = 1, kUnsafe = 2;
        // groups are powers of two from 32 to 128 columns and vectors hold 4 to 16: whole lanes of one warp
        constexpr bool IN_WARP = !PEEL && V >= 4;
        const int g = a.group, shift = g ? 31 - __clz(g) : 0;
        int *mine = amax + team * SLOTS;
        uint8_t *qr = static_cast<uint8_t *>(a.y) + row * a.ldy;
        float *scales = a.scales + row * a.lds;
        auto meet = [] {
            if constexpr (TEAM > 32) __syncthreads();
            else __syncwarp();
        };
        auto spread = [](float top) { return top > 0.0f ? __fdividef(kE4m3Max, top) : 0.0f; };
        auto flags_of = [](float top) { return top == 0.0f ? kZero : top >= kSmall && top <= kLarge ? 0u : kUnsafe; };
        auto largest = [&](const float (&v)[V], int from, int to) {
            float r = 0.0f;
#pragma unroll
            for (int j = 0; j < V; ++j) r = fmaxf(r, j >= from && j < to ? fabsf(v[j]) : 0.0f);
            return r;
        };
        auto product = [&](int i, float (&v)[V]) {
            widen(pw[i], v);
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] *= h[i][j];
        };
        // Maxima of the groups into shared memory; returns their flags.  A warp's vectors cover 32 V columns in a row: one
        // reduction per group that can begin among them; a vector (PEEL) may lie in two groups.
        auto group_maxima = [&] {
            unsigned flags = 0;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int first = head + (t + width * i) * V, warp_first = head + ((t & ~31) + width * i) * V;
                if (warp_first >= a.cols) continue;    // the same for the whole warp
                const int mine_g = first >> shift, edge = ((mine_g + 1) << shift) - first;    // elements from `edge` on are in the next group
                float v[V];
                product(i, v);
                const float lo = largest(v, 0, edge), hi = edge < V ? largest(v, edge, V) : 0.0f;
                const int end = (min(warp_first + 32 * V, a.cols) + g - 1) >> shift;
                for (int k = warp_first >> shift; k < end; ++k) {
                    const unsigned top = __reduce_max_sync(0xffffffffu, __float_as_uint(mine_g == k ? lo : mine_g + 1 == k ? hi : 0.0f));
                    flags |= flags_of(__uint_as_float(top));
                    if ((t & 31) == 0) atomicMax(&mine[k], static_cast<int>(top));
                }
            }
            if (single) {
                const float top = fmaxf(fabsf(h1 * w1), 0.0f);    // (a NaN: 0)
                flags |= flags_of(top);
                atomicMax(&mine[one >> shift], __float_as_int(top));
            }
            return flags;
        };
        // the bytes of a vector: h times `factor(k)` for group k times w
        auto put = [&](int i, auto &&factor) {
            const int first = head + (t + width * i) * V, mine_g = first >> shift, edge = g ? ((mine_g + 1) << shift) - first : V;
            const float lo = factor(g ? mine_g : 0), hi = edge < V ? factor(mine_g + 1) : lo;
            float q[V];
            widen(pw[i], q);
#pragma unroll
            for (int j = 0; j < V; ++j) q[j] *= h[i][j] * (j < edge ? lo : hi);
            if constexpr (PEEL) store_e4m3_any<V>(q, qr + first);
            else store_e4m3<V>(q, qr + first);
        };
        auto put_single = [&](float factor) { qr[one] = __nv_cvt_float_to_fp8(h1 * factor * w1, __NV_SATFINITE, __NV_E4M3); };
        float m[NV];       // IN_WARP: the group's largest |h w|
        float top = 0.0f;  // g == 0: the row's
        unsigned flags = 0;
        if (g == 0) {
            top = fmaxf(fabsf(h1 * w1), 0.0f);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                float v[V];
                product(i, v);
                top = fmaxf(top, largest(v, 0, V));
            }
            if (t < nvec || single) flags = flags_of(top);
        } else if constexpr (IN_WARP) {
            const int span = g / V;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                float v[V];
                product(i, v);
                m[i] = largest(v, 0, V);
#pragma unroll
                for (int o = 1; o < 128 / V; o <<= 1)
                    if (o < span && o < TEAM) m[i] = fmaxf(m[i], __shfl_xor_sync(0xffffffffu, m[i], o));
            }
            if (TEAM < 32 && span > TEAM) {    // one group holds the row
#pragma unroll
                for (int i = 1; i < NV; ++i) m[0] = fmaxf(m[0], m[i]);
#pragma unroll
                for (int i = 1; i < NV; ++i) m[i] = m[0];
            }
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (t + width * i < nvec) {
                    flags |= flags_of(m[i]);
                    put(i, [&](int) { return spread(m[i]); });
                }
        } else {
            flags = group_maxima();
            if constexpr (TEAM <= 32) __syncwarp();    // (larger teams meet at the block's barrier below)
        }
        if (g == 0) team_sum_max<TEAM, true>(s[0], top, flags, red4);
        else team_sum_max<TEAM, false>(s[0], top, flags, red4);
        const float rs = rsqrtf(s[0] / static_cast<float>(a.cols) + a.eps);
        bool plain = !(flags & kUnsafe) && rs >= kSmallR && rs <= kLargeR && (!(flags & kZero) || rs <= kZeroR);
        if constexpr (TEAM < 32) plain = __all_sync(0xffffffffu, plain || !live);    // the rows of a warp go one way
        if (plain) {
            store_h();
            if (g == 0) {
                const float f = spread(top);
                if (t == 0 && live) scales[0] = scale_of(top * rs);
#pragma unroll
                for (int i = 0; i < NV; ++i)
                    if (t + width * i < nvec) put(i, [&](int) { return f; });
                if (single) put_single(f);
            } else if constexpr (IN_WARP) {
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int first = (t + width * i) * V;
                    if (first < nvec * V && (first & (g - 1)) == 0) scales[first >> shift] = scale_of(m[i] * rs);
                }
            } else {
#pragma unroll
                for (int i = 0; i < NV; ++i)
                    if (t + width * i < nvec) put(i, [&](int k) { return spread(__int_as_float(mine[k])); });
                if (single) put_single(spread(__int_as_float(mine[one >> shift])));
                for (int k = t; k << shift < a.cols; k += width) scales[k] = scale_of(__int_as_float(mine[k]) * rs);
            }
            return;
        }
        const int cols = live ? a.cols : 0;
        auto h_at = [&](int j) { return rr ? load_one(xr + j) + load_one(rr + j) : load_one(xr + j); };
        for (int k = t; k < SLOTS; k += width) mine[k] = 0;
        meet();
        for (int j = t; j < cols; j += width) {
            const float y = h_at(j) * rs * load_one(wr + j);
            atomicMax(&mine[g ? j >> shift : 0], __float_as_int(fmaxf(fabsf(y), 0.0f)));     // (a NaN: 0)
        }
        meet();
        for (int j = t; j < cols; j += width) {
            const float hv = h_at(j), y = hv * rs * load_one(wr + j);
            if (hr) store_one(hv, hr + j);
            qr[j] = __nv_cvt_float_to_fp8(y * (1.0f / scale_of(__int_as_float(mine[g ? j >> shift : 0]))), __NV_SATFINITE, __NV_E4M3);
        }
        for (int k = t; live && (k == 0 || (g && k << shift < cols)); k += width) scales[k] = scale_of(__int_as_float(mine[k]));
    }
}

// Rows longer than the registers of a block hold: x and residual are read again (from L2, where the
// row still is) for the groups' maxima and for the output.  Nothing is written before the last pass,
// and each element is written by the thread that reads it, so outputs may lie on their inputs.
template <typename T, bool QUANT>
__global__ void __launch_bounds__(1024)
rmsnorm_long_kernel(const NormArgs a) {
    __shared__ float red[1][2][32];
    pdl_launch_dependents();
    pdl_wait();
    const int wid = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *x = static_cast<const T *>(a.x) + row * a.ldx;
        const T *res = a.residual ? static_cast<const T *>(a.residual) + row * a.ldr : nullptr;
        const T *w = static_cast<const T *>(a.weight);
        T *hout = a.h ? static_cast<T *>(a.h) + row * a.ldh : nullptr;
        auto sum_at = [&](int j) { return load_one(x + j) + (res ? load_one(res + j) : 0.0f); };
        float s[1] = {0.0f};
        for (int j = threadIdx.x; j < a.cols; j += 1024) {
            const float v = sum_at(j);
            s[0] = fmaf(v, v, s[0]);
        }
        team_sum<1024>(s, red, 0);
        const float rs = rsqrtf(s[0] / static_cast<float>(a.cols) + a.eps);
        auto y_at = [&](float hv, int j) { return hv * rs * load_one(w + j); };
        if constexpr (!QUANT) {
            T *y = static_cast<T *>(a.y) + row * a.ldy;
            for (int j = threadIdx.x; j < a.cols; j += 1024) {
                const float hv = sum_at(j), yv = y_at(hv, j);
                if (hout) store_one(hv, hout + j);
                store_one(yv, y + j);
            }
        } else {
            uint8_t *y = static_cast<uint8_t *>(a.y) + row * a.ldy;
            auto put = [&](int j, float inv) {
                const float hv = sum_at(j), yv = y_at(hv, j);
                if (hout) store_one(hv, hout + j);
                y[j] = __nv_cvt_float_to_fp8(yv * inv, __NV_SATFINITE, __NV_E4M3);
            };
            if (a.group) {   // a warp owns a group
                const int groups = (a.cols + a.group - 1) / a.group;
                for (int g = wid; g < groups; g += 32) {
                    const int first = g * a.group, last = min(first + a.group, a.cols);
                    float m = 0.0f;
                    for (int j = first + lane; j < last; j += 32) m = fmaxf(m, fabsf(y_at(sum_at(j), j)));
                    const float scale = scale_of(warp_max(m));
                    for (int j = first + lane; j < last; j += 32) put(j, 1.0f / scale);
                    if (lane == 0) a.scales[row * a.lds + g] = scale;
                }
            } else {
                float m = 0.0f;
                for (int j = threadIdx.x; j < a.cols; j += 1024) m = fmaxf(m, fabsf(y_at(sum_at(j), j)));
                m = warp_max(m);
                if (lane == 0) red[0][1][wid] = m;
                __syncthreads();
                m = warp_max(red[0][1][lane]);
                const float scale = scale_of(m);
                for (int j = threadIdx.x; j < a.cols; j += 1024) put(j, 1.0f / scale);
                if (threadIdx.x == 0) a.scales[row * a.lds] = scale;
            }
        }
        __syncthreads();   // `red` is used again by the next row
    }
}


struct NormBackArgs {
    const void *dy, *h, *weight, *dres;
    int64_t lddy, ldh, lddres;
    void *dx;
    int64_t lddx;
    float *partial;      // [blocks][cols], NULL when dweight is not wanted
    int64_t rows;
    int cols;
    float eps;
};

// Persistent teams walk the rows; a thread owns the same columns of every row and keeps their dweight
// sums in registers, so the sum over rows needs one [cols] vector per block and no atomics: the same
// call gives the same bits.  AHEAD: the next row's loads are issued before this row's reduction.
template <typename T, int V, int NV, int TEAM, bool AHEAD, bool FIT>
__global__ void __launch_bounds__(kBlock<TEAM>, V == 16 && NV == 1 ? 512 / kBlock<TEAM> : 0)
rmsnorm_backward_kernel(const NormBackArgs a) {
    using P = typename Pack<T, V>::type;
    constexpr int TEAMS = kBlock<TEAM> / TEAM;
    __shared__ float red[2][2][32];
    pdl_launch_dependents();
    pdl_wait();
    const int width = FIT ? blockDim.x : TEAM;
    const int t = TEAM > 32 ? threadIdx.x : threadIdx.x % TEAM, team = TEAM > 32 ? 0 : threadIdx.x / TEAM;
    const int64_t mates = TEAM < 32 ? team % (32 / TEAM) : 0;     // teams of this warp before this one
    const int nvec = a.cols / V;
    const int64_t me = static_cast<int64_t>(blockIdx.x) * TEAMS + team, teams = static_cast<int64_t>(gridDim.x) * TEAMS;
    P pw[NV], pdy[NV], ph[NV], pd[NV];
    float dw[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int idx = t + width * i;
        pw[i] = idx < nvec ? load_weight(static_cast<const P *>(a.weight) + idx) : P{};
#pragma unroll
        for (int j = 0; j < V; ++j) dw[i][j] = 0.0f;
    }
    auto fetch = [&](int64_t row) {
        const P *dy = reinterpret_cast<const P *>(static_cast<const T *>(a.dy) + row * a.lddy);
        const P *h = reinterpret_cast<const P *>(static_cast<const T *>(a.h) + row * a.ldh);
        const P *d = a.dres ? reinterpret_cast<const P *>(static_cast<const T *>(a.dres) + row * a.lddres) : nullptr;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int idx = t + width * i;
            const bool in = idx < nvec && row < a.rows;
            pdy[i] = in ? load_row(dy + idx) : P{};
            ph[i] = in ? load_row(h + idx) : P{};
            pd[i] = in && d ? load_row(d + idx) : P{};
        }
    };
    if (AHEAD) fetch(me);
    int parity = 0;
    for (int64_t row = me; row - mates < a.rows; row += teams, parity ^= 1) {     // (the same number of rounds for a whole warp)
        P cdy[NV], ch[NV], cd[NV];
        if (!AHEAD) fetch(row);
        float s[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            cdy[i] = pdy[i];
            ch[i] = ph[i];
            cd[i] = pd[i];
        }
        if (AHEAD) fetch(row + teams);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float dy[V], h[V], w[V];
            widen(cdy[i], dy);
            widen(ch[i], h);
            widen(pw[i], w);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                s[0] = fmaf(h[j], h[j], s[0]);
                s[1] = fmaf(w[j] * dy[j], h[j], s[1]);
            }
        }
        team_sum<TEAM>(s, red, parity);
        const float inv = 1.0f / static_cast<float>(a.cols);
        const bool live = TEAM >= 32 || row < a.rows;
        const float rs = live ? rsqrtf(s[0] * inv + a.eps) : 0.0f;
        const float along = s[1] * rs * inv;          // mean(w dy xhat)
        P *dx = reinterpret_cast<P *>(static_cast<T *>(a.dx) + row * a.lddx);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int idx = t + width * i;
            float dy[V], h[V], w[V], d[V], o[V];
            widen(cdy[i], dy);
            widen(ch[i], h);
            widen(pw[i], w);
            widen(cd[i], d);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float xhat = h[j] * rs;
                o[j] = fmaf(rs, fmaf(-xhat, along, w[j] * dy[j]), d[j]);
                dw[i][j] = fmaf(dy[j], xhat, dw[i][j]);
            }
            P p;
            narrow(o, p);
            if (idx < nvec && live) store_row(dx + idx, p);
        }
    }
    if (!a.partial) return;
    if constexpr (TEAM > 32) {
        float *dst = a.partial + me * a.cols;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int idx = t + width * i;
            if (idx < nvec)
#pragma unroll
                for (int j = 0; j < V; ++j) dst[idx * V + j] = dw[i][j];
        }
    } else {    // the block's teams join: those of a warp by shuffles, then the warps
        __shared__ float joined[kBlock<TEAM> / 32][TEAM * NV * V];
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) {
#pragma unroll
                for (int o = TEAM; o < 32; o <<= 1) dw[i][j] += __shfl_xor_sync(0xffffffffu, dw[i][j], o);
                if ((threadIdx.x & 31) < TEAM) joined[threadIdx.x >> 5][(t + TEAM * i) * V + j] = dw[i][j];
            }
        __syncthreads();
        for (int c = threadIdx.x; c < a.cols; c += kBlock<TEAM>) {
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < kBlock<TEAM> / 32; ++w) v += joined[w][c];
            a.partial[static_cast<int64_t>(blockIdx.x) * a.cols + c] = v;
        }
    }
}

// The widest bf16 rows (more than 8192 columns), whose operands two rows deep do not fit the registers, on a
// ring of rows in shared memory that bulk copies fill ahead.  A block owns a row at a time, its threads 32
// columns each.  Needs 16-byte aligned rows.  4096 x 16384: 92 us, against 136 us without look-ahead.  (Narrower
// rows run faster from registers: 16384 x 4096 106 us on the ring, 94 us with a row's loads ahead in registers.)
constexpr int kRingFrom = 8192, kRingCols = 512 * 32, kRingStages = 2, kRingBytes = 3 * kRingCols * 2 * kRingStages;
static_assert(kRingBytes <= 220 * 1024, "the ring exceeds a block's shared memory");
__global__ void __launch_bounds__(512)
rmsnorm_backward_ring_kernel(const NormBackArgs a, int *status) {
    using T = __nv_bfloat16;
    constexpr int V = 8, NV = 4, stages = kRingStages;
    using P = typename Pack<T, V>::type;
    extern __shared__ __align__(16) unsigned char ring[];
    __shared__ uint64_t full[kRingStages];
    __shared__ float red[2][2][32];
    const int t = threadIdx.x, team = blockDim.x, lane = t & 31, wid = t >> 5, warps = team >> 5;
    const int nvec = a.cols / V, row_bytes = a.cols * (int)sizeof(T), operands = a.dres ? 3 : 2;
    if (t == 0) {
        for (int s = 0; s < stages; ++s) mbar_init(&full[s], 1);
        mbar_fence_init();
    }
    __syncthreads();
    pdl_launch_dependents();
    pdl_wait();
    auto fetch = [&](int64_t row, int s) {   // one thread
        unsigned char *dst = ring + s * operands * row_bytes;
        mbar_expect_tx(&full[s], operands * row_bytes);
        bulk_load(dst, static_cast<const T *>(a.dy) + row * a.lddy, row_bytes, &full[s]);
        bulk_load(dst + row_bytes, static_cast<const T *>(a.h) + row * a.ldh, row_bytes, &full[s]);
        if (a.dres) bulk_load(dst + 2 * row_bytes, static_cast<const T *>(a.dres) + row * a.lddres, row_bytes, &full[s]);
    };
    if (t == 0)
        for (int s = 0; s < stages; ++s) {
            const int64_t row = blockIdx.x + static_cast<int64_t>(s) * gridDim.x;
            if (row < a.rows) fetch(row, s);
        }
    P pw[NV];
    float dw[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int idx = t + team * i;
        pw[i] = idx < nvec ? __ldg(static_cast<const P *>(a.weight) + idx) : P{};
#pragma unroll
        for (int j = 0; j < V; ++j) dw[i][j] = 0.0f;
    }
    const float inv = 1.0f / static_cast<float>(a.cols);
    int s = 0, parity = 0;
    uint32_t phase = 0;
    bool ok = true;      // a wait that ran out is recorded and not repeated; the barriers below go on alike
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, parity ^= 1) {
        if (ok) ok = mbar_wait(&full[s], phase, status, 501);
        const unsigned char *src = ring + s * operands * row_bytes;
        float sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int idx = t + team * i;
            if (idx < nvec) {
                float dy[V], h[V], w[V];
                widen(reinterpret_cast<const P *>(src)[idx], dy);
                widen(reinterpret_cast<const P *>(src + row_bytes)[idx], h);
                widen(pw[i], w);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    sum[0] = fmaf(h[j], h[j], sum[0]);
                    sum[1] = fmaf(w[j] * dy[j], h[j], sum[1]);
                }
            }
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) sum[k] = warp_sum(sum[k]);
        if (lane == 0) {
            red[0][parity][wid] = sum[0];
            red[1][parity][wid] = sum[1];
        }
        __syncthreads();      // behind it every thread is done with the stage of the row before
        const int64_t next = row + static_cast<int64_t>(stages - 1) * gridDim.x;
        if (t == 0 && row != blockIdx.x && next < a.rows && ok) fetch(next, s == 0 ? stages - 1 : s - 1);
        if (++s == stages) {
            s = 0;
            phase ^= 1;
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) sum[k] = warp_sum(lane < warps ? red[k][parity][lane] : 0.0f);
        const float rs = rsqrtf(sum[0] * inv + a.eps);
        const float along = sum[1] * rs * inv;          // mean(w dy xhat)
        P *dx = reinterpret_cast<P *>(static_cast<T *>(a.dx) + row * a.lddx);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int idx = t + team * i;
            if (idx < nvec) {
                float dy[V], h[V], w[V], d[V], o[V];
                widen(reinterpret_cast<const P *>(src)[idx], dy);
                widen(reinterpret_cast<const P *>(src + row_bytes)[idx], h);
                widen(pw[i], w);
                widen(a.dres ? reinterpret_cast<const P *>(src + 2 * row_bytes)[idx] : P{}, d);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float xhat = h[j] * rs;
                    o[j] = fmaf(rs, fmaf(-xhat, along, w[j] * dy[j]), d[j]);
                    dw[i][j] = fmaf(dy[j], xhat, dw[i][j]);
                }
                P p;
                narrow(o, p);
                __stcs(dx + idx, p);
            }
        }
    }
    if (!ok && t == 0)     // no copy of this block may land in shared memory that is no longer its own
        for (int k = 0; k < stages; ++k) mbar_wait(&full[k], 0, nullptr, 0), mbar_wait(&full[k], 1, nullptr, 0);
    if (a.partial) {
        float *dst = a.partial + static_cast<int64_t>(blockIdx.x) * a.cols;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int idx = t + team * i;
            if (idx < nvec)
#pragma unroll
                for (int j = 0; j < V; j += 4)
                    *reinterpret_cast<float4 *>(dst + idx * V + j) = make_float4(dw[i][j], dw[i][j + 1], dw[i][j + 2], dw[i][j + 3]);
        }
    }
}

// Rows longer than the registers of a block hold take three launches: per row r and mean(w dy xhat),
// then the partial dweight sums, then dx (which may lie on dy or h, so it comes last).
template <typename T>
__global__ void __launch_bounds__(1024)
rmsnorm_backward_sums_kernel(const NormBackArgs a, float2 *row_sums) {
    __shared__ float red[2][2][32];
    pdl_launch_dependents();
    pdl_wait();
    const T *w = static_cast<const T *>(a.weight);
    int parity = 0;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, parity ^= 1) {
        const T *dy = static_cast<const T *>(a.dy) + row * a.lddy;
        const T *h = static_cast<const T *>(a.h) + row * a.ldh;
        float s[2] = {0.0f, 0.0f};
        for (int j = threadIdx.x; j < a.cols; j += 1024) {
            const float hv = load_one(h + j);
            s[0] = fmaf(hv, hv, s[0]);
            s[1] = fmaf(load_one(w + j) * load_one(dy + j), hv, s[1]);
        }
        team_sum<1024>(s, red, parity);
        const float inv = 1.0f / static_cast<float>(a.cols);
        const float rs = rsqrtf(s[0] * inv + a.eps);
        if (threadIdx.x == 0) row_sums[row] = make_float2(rs, s[1] * rs * inv);
    }
}

// A thread per column and stripe of rows.
template <typename T>
__global__ void __launch_bounds__(256)
rmsnorm_dweight_long_kernel(const NormBackArgs a, const float2 *row_sums) {
    pdl_launch_dependents();
    pdl_wait();
    const int col = blockIdx.x * 256 + threadIdx.x;
    if (col >= a.cols) return;
    float s = 0.0f;
    for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y)
        s = fmaf(load_one(static_cast<const T *>(a.dy) + row * a.lddy + col),
                 load_one(static_cast<const T *>(a.h) + row * a.ldh + col) * row_sums[row].x, s);
    a.partial[static_cast<int64_t>(blockIdx.y) * a.cols + col] = s;
}

template <typename T>
__global__ void __launch_bounds__(256)
rmsnorm_dx_long_kernel(const NormBackArgs a, const float2 *row_sums) {
    pdl_launch_dependents();
    pdl_wait();
    const int col = blockIdx.x * 256 + threadIdx.x;
    if (col >= a.cols) return;
    const float wv = load_one(static_cast<const T *>(a.weight) + col);
    for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const float2 rs = row_sums[row];
        const float xhat = load_one(static_cast<const T *>(a.h) + row * a.ldh + col) * rs.x;
        const float wdy = wv * load_one(static_cast<const T *>(a.dy) + row * a.lddy + col);
        const float d = a.dres ? load_one(static_cast<const T *>(a.dres) + row * a.lddres + col) : 0.0f;
        store_one(fmaf(rs.x, fmaf(-xhat, rs.y, wdy), d), static_cast<T *>(a.dx) + row * a.lddx + col);
    }
}

// dweight = (accumulate ? dweight : 0) + sum of the teams' partial vectors.  32 columns per block, 32
// threads deep: the partials (a few MB, in L2) are read once, in the same order every time.
__global__ void __launch_bounds__(1024)
rmsnorm_dweight_kernel(const float *__restrict__ partial, int64_t n, int cols, float *dweight, int accumulate) {
    __shared__ float part[32][33];
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31, deep = threadIdx.x >> 5;
    const int col = blockIdx.x * 32 + lane;
    float s = 0.0f;
    if (col < cols) {
        const float *p = partial + deep * static_cast<int64_t>(cols) + col;
        const int64_t step = 32 * static_cast<int64_t>(cols);
        int64_t i = deep;
        for (; i + 7 * 32 < n; i += 8 * 32, p += 8 * step) {   // eight loads in flight
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = __ldcs(p + k * step);
#pragma unroll
            for (int k = 0; k < 8; ++k) s += v[k];
        }
        for (; i < n; i += 32, p += step) s += __ldcs(p);
    }
    part[deep][lane] = s;
    __syncthreads();
    if (deep == 0 && col < cols) {
        s = 0.0f;
#pragma unroll
        for (int d = 0; d < 32; ++d) s += part[d][lane];
        dweight[col] = accumulate ? dweight[col] + s : s;
    }
}

// ---- dispatch ----------------------------------------------------------------------------------

// Calls f.template operator()<NV, TEAM>() for the team that takes rows of `cols` elements.  Rows of up to 1024 are a
// warp's or (SMALL, whole vectors only) a part's of one: 64 columns of bf16 306 us in a warp, 80 us in 8 lanes (2^26
// elements, as below).  Longer ones are a block's, with as many warps as they need, TEAM threads at most (10240 columns
// 111 us in 1024 threads, 80 in 640).  16 elements a thread keep the register count at about 40 and enough rows
// resident to cover the latency of HBM.  With 32-byte vectors (V = 16) a thread takes 32: half as many warps meet at the
// barrier, which pays where there is more to do behind it (e4m3, 4096 columns: 76 -> 72 us) and where 1024 threads would
// leave one row per SM (16384 columns: 92 -> 82 us).
template <int V, bool SMALL, typename F>
int with_team(int cols, F &&f) {
    constexpr int N8 = (8 + V - 1) / V, N16 = 16 / V, N32 = 32 / V;
    if constexpr (SMALL && V <= 8) {
        if (cols <= 8 * 8) return f.template operator()<N8, 8>();
        if (cols <= 16 * 8) return f.template operator()<N8, 16>();
        if (cols <= 32 * 8) return f.template operator()<N8, 32>();
    }
    if (cols <= 32 * 16) return f.template operator()<N16, 32>();
    if constexpr (V == 16) {
        if (cols <= 96 * 16) return f.template operator()<N16, 128>();
        if (cols <= 128 * 32) return f.template operator()<N32, 128>();
        if (cols <= 256 * 32) return f.template operator()<N32, 256>();
        return f.template operator()<N32, 512>();
    } else {
        if (cols <= 32 * 32) return f.template operator()<N32, 32>();
        if (cols <= 128 * 16) return f.template operator()<N16, 128>();
        if (cols <= 256 * 16) return f.template operator()<N16, 256>();
        if (cols <= 512 * 16) return f.template operator()<N16, 512>();
        return f.template operator()<N16, 1024>();
    }
}
static_assert(kLongCols == 1024 * 16, "with_team covers every row that is not long");

// The backward pass keeps three operands, the weight and the dweight sums of a thread's columns in
// registers, and the next row's operands where they fit (AHEAD): with bf16 pairs packed in a register
// 16 columns per thread, else 8.  Twice as many in teams of one warp, which have no block barrier to wait
// at (65536 x 1024 bf16: 91 us in warps of 32 columns per thread, 154 us in teams of 128 threads), and
// without the look-ahead in the widest rows.  32-byte vectors and at most 128 registers a thread leave 512 threads per
// SM (4096 columns 94 -> 91 us; with the 164 registers it takes unasked 123).  Short rows share a warp and longer ones take as many warps as they need,
// as in the forward pass (2^26 bf16 elements: 64 columns 375 -> 101 us, 1536 columns 124 -> 95 us); the teams of a
// block of warps join their dweight sums before they leave it.
template <typename T, int V> constexpr int kBackE = sizeof(T) == 2 && V > 1 ? 16 : 8;
template <typename T, int V> constexpr int kBackCols = 512 * 2 * kBackE<T, V>;    // the columns covered
template <typename T, int V, typename F>
int with_back_team(int cols, F &&f) {
    constexpr int E = kBackE<T, V>, N = E / V;
    if constexpr (V == 4 || V == 8) {
        if (cols <= 8 * 8) return f.template operator()<8 / V, 8, true>();
        if (cols <= 16 * 8) return f.template operator()<8 / V, 16, true>();
        if (cols <= 32 * 8) return f.template operator()<8 / V, 32, true>();
    }
    if (cols <= 32 * E) return f.template operator()<N, 32, true>();
    if (cols <= 64 * E) return f.template operator()<2 * N, 32, true>();
    if (cols <= 128 * E) return f.template operator()<N, 128, true>();
    if (cols <= 256 * E) return f.template operator()<N, 256, true>();
    if (cols <= 512 * E) return f.template operator()<N, 512, true>();
    return f.template operator()<2 * N, 512, false>();
}

bool aligned(const void *p, int64_t ld, int elem, int bytes) {
    return p == nullptr || (reinterpret_cast<uintptr_t>(p) % bytes == 0 && ld * elem % bytes == 0);
}

// Threads of a block whose rows hold `cols` elements, `each` a thread.
int fitting_threads(int cols, int each) { return (cols + 32 * each - 1) / (32 * each) * 32; }

template <typename T, int V, bool QUANT, bool PEEL>
struct Forward {
    gb200_ctx *ctx;
    const NormArgs &a;
    cudaStream_t stream;
    template <int NV, int TEAM>
    int operator()() const {
        constexpr int TEAMS = kBlock<TEAM> / TEAM;
        const int64_t blocks = (a.rows + TEAMS - 1) / TEAMS;
        const auto launch = [&](auto kern, int threads) {
            return launch_pdl(kern, dim3((unsigned)blocks), dim3((unsigned)threads), 0, stream, a);
        };
        const int threads = fitting_threads(a.cols, NV * V);
        // the e4m3 form's registers are worth a kernel of its own where a block is full (4096 x 8192: 41.1 against 40.3 us)
        constexpr bool MAY_FIT = TEAM > 32 && V >= 4 && !(QUANT && PEEL);
        if (MAY_FIT && !(QUANT && V == 16 && threads == TEAM))
            GB200_CUDA_TRY(launch(rmsnorm_kernel<T, V, NV, TEAM, QUANT, PEEL, MAY_FIT>, threads));
        else if constexpr (!MAY_FIT || (QUANT && V == 16))
            GB200_CUDA_TRY(launch(rmsnorm_kernel<T, V, NV, TEAM, QUANT, PEEL, false>, kBlock<TEAM>));
        return after_launch(ctx, "rmsnorm_kernel");
    }
};

template <typename T, bool QUANT>
int forward(gb200_ctx *ctx, const NormArgs &a, cudaStream_t stream) {
    constexpr int e = sizeof(T), wide = 16 / sizeof(T), ye = QUANT ? 1 : e;
    GB200_REQUIRE(a.rows <= 0x7fffffffll, GB200_ERR_TOO_LARGE, "more than 2^31 - 1 rows");
    if (a.cols > kLongCols) {
        int64_t blocks = a.rows;
        const int64_t cap = (int64_t)ctx->sm_count * 2;
        if (blocks > cap) blocks = cap;
        GB200_CUDA_TRY(launch_pdl(rmsnorm_long_kernel<T, QUANT>, dim3((unsigned)blocks), dim3(1024), 0, stream, a));
        return after_launch(ctx, "rmsnorm_long_kernel");
    }
    auto fits = [&](int v) {
        return a.cols % v == 0 && aligned(a.x, a.ldx, e, v * e) && aligned(a.residual, a.ldr, e, v * e) &&
               aligned(a.weight, 0, e, v * e) && aligned(a.y, a.ldy, ye, v * ye) && aligned(a.h, a.ldh, e, v * e);
    };
    if constexpr (e == 2)
        if (fits(16) && a.cols > (QUANT ? 256 : 12288)) return with_team<16, true>(a.cols, Forward<T, 16, QUANT, false>{ctx, a, stream});
    if (fits(wide)) return with_team<wide, true>(a.cols, Forward<T, wide, QUANT, false>{ctx, a, stream});
    // x, residual, y and residual_out as far from a 16-byte boundary as one another, in every row
    auto alike = [&](const void *p, int64_t ld) {
        return p == nullptr || ((reinterpret_cast<uintptr_t>(p) - reinterpret_cast<uintptr_t>(a.x)) % 16 == 0 &&
                                (a.rows == 1 || (ld - a.ldx) * e % 16 == 0));
    };
    if (alike(a.residual, a.ldr) && (QUANT || alike(a.y, a.ldy)) && alike(a.h, a.ldh))
        return with_team<wide, false>(a.cols, Forward<T, wide, QUANT, true>{ctx, a, stream});
    return with_team<1, false>(a.cols, Forward<T, 1, QUANT, false>{ctx, a, stream});
}

int finish_dweight(gb200_ctx *ctx, const float *partial, int64_t n, int cols, float *dweight, int accumulate, cudaStream_t stream) {
    GB200_CUDA_TRY(launch_pdl(rmsnorm_dweight_kernel, dim3((unsigned)((cols + 31) / 32)), dim3(1024), 0, stream, partial, n, cols,
                              dweight, accumulate));
    return after_launch(ctx, "rmsnorm_dweight_kernel");
}

template <typename T, int V>
struct Backward {
    gb200_ctx *ctx;
    NormBackArgs a;
    float *dweight;
    int accumulate;
    cudaStream_t stream;
    template <int NV, int TEAM, bool AHEAD>
    int operator()() const {
        constexpr int TEAMS = kBlock<TEAM> / TEAM;
        constexpr bool FIT = TEAM > 32 && V > 1;
        auto kern = rmsnorm_backward_kernel<T, V, NV, TEAM, AHEAD, FIT>;
        const int threads = FIT ? fitting_threads(a.cols, NV * V) : kBlock<TEAM>;
        static std::atomic<int> known[kBlock<TEAM> / 32 + 1];    // the same on every device this library runs on; asked once
        int per_sm = known[threads / 32];
        if (per_sm == 0) {
            if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, threads, 0) != cudaSuccess || per_sm < 1) per_sm = 1;
            known[threads / 32] = per_sm;
        }
        int64_t blocks = (a.rows + TEAMS - 1) / TEAMS;
        const int64_t cap = (int64_t)ctx->sm_count * per_sm;
        if (blocks > cap) blocks = cap;
        NormBackArgs args = a;
        if (dweight) {
            void *ws = nullptr;
            const int rc = scratch_reserve(ctx, (size_t)blocks * a.cols * sizeof(float), stream, &ws);
            if (rc) return rc;
            args.partial = static_cast<float *>(ws);
        }
        GB200_CUDA_TRY(launch_pdl(kern, dim3((unsigned)blocks), dim3((unsigned)threads), 0, stream, args));
        int rc = after_launch(ctx, "rmsnorm_backward_kernel");
        if (rc || !dweight) return rc;
        return finish_dweight(ctx, args.partial, blocks, a.cols, dweight, accumulate, stream);
    }
};

template <typename T>
int backward_long(gb200_ctx *ctx, NormBackArgs a, float *dweight, int accumulate, cudaStream_t stream) {
    const int64_t stripes = a.rows < 64 ? a.rows : 64;
    int64_t blocks = a.rows;
    const int64_t cap = (int64_t)ctx->sm_count * 2;
    if (blocks > cap) blocks = cap;
    void *ws = nullptr;
    int rc = scratch_reserve(ctx, (size_t)a.rows * sizeof(float2) + (dweight ? (size_t)stripes * a.cols * sizeof(float) : 0),
                             stream, &ws);
    if (rc) return rc;
    float2 *row_sums = static_cast<float2 *>(ws);
    a.partial = reinterpret_cast<float *>(row_sums + a.rows);
    const dim3 grid((unsigned)((a.cols + 255) / 256), (unsigned)stripes);
    GB200_CUDA_TRY(launch_pdl(rmsnorm_backward_sums_kernel<T>, dim3((unsigned)blocks), dim3(1024), 0, stream, a, row_sums));
    if ((rc = after_launch(ctx, "rmsnorm_backward_sums_kernel"))) return rc;
    if (dweight) {
        GB200_CUDA_TRY(launch_pdl(rmsnorm_dweight_long_kernel<T>, grid, dim3(256), 0, stream, a, row_sums));
        if ((rc = after_launch(ctx, "rmsnorm_dweight_long_kernel"))) return rc;
        if ((rc = finish_dweight(ctx, a.partial, stripes, a.cols, dweight, accumulate, stream))) return rc;
    }
    GB200_CUDA_TRY(launch_pdl(rmsnorm_dx_long_kernel<T>, grid, dim3(256), 0, stream, a, row_sums));
    return after_launch(ctx, "rmsnorm_dx_long_kernel");
}

template <typename T, int V>
int backward_vec(gb200_ctx *ctx, const NormBackArgs &a, float *dweight, int accumulate, cudaStream_t stream) {
    if (a.cols > kBackCols<T, V>) return backward_long<T>(ctx, a, dweight, accumulate, stream);
    return with_back_team<T, V>(a.cols, Backward<T, V>{ctx, a, dweight, accumulate, stream});
}

int backward_ring(gb200_ctx *ctx, NormBackArgs a, float *dweight, int accumulate, cudaStream_t stream) {
    const int threads = ((a.cols + 31) / 32 + 31) / 32 * 32;    // 8 elements x 4 vectors each
    const int64_t blocks = std::min<int64_t>(a.rows, ctx->sm_count);
    int rc = ensure_dynamic_smem(ctx, rmsnorm_backward_ring_kernel, kRingBytes);
    if (rc) return rc;
    if (dweight) {
        void *ws = nullptr;
        rc = scratch_reserve(ctx, (size_t)blocks * a.cols * sizeof(float), stream, &ws);
        if (rc) return rc;
        a.partial = static_cast<float *>(ws);
    }
    GB200_CUDA_TRY(launch_pdl(rmsnorm_backward_ring_kernel, dim3((unsigned)blocks), dim3((unsigned)threads),
                              (size_t)(kRingStages * (a.dres ? 3 : 2) * a.cols * 2), stream, a, ctx->d_status));
    rc = after_launch(ctx, "rmsnorm_backward_ring_kernel");
    if (rc || !dweight) return rc;
    return finish_dweight(ctx, a.partial, blocks, a.cols, dweight, accumulate, stream);
}

template <typename T>
int backward(gb200_ctx *ctx, const NormBackArgs &a, float *dweight, int accumulate, cudaStream_t stream) {
    constexpr int e = sizeof(T), wide = 16 / sizeof(T);
    auto fits = [&](int v) {
        return a.cols % v == 0 && aligned(a.dy, a.lddy, e, v * e) && aligned(a.h, a.ldh, e, v * e) &&
               aligned(a.weight, 0, e, v * e) && aligned(a.dres, a.lddres, e, v * e) && aligned(a.dx, a.lddx, e, v * e);
    };
    if constexpr (sizeof(T) == 2)
        if (fits(wide) && a.cols > kRingFrom && a.cols <= kRingCols) return backward_ring(ctx, a, dweight, accumulate, stream);
    if constexpr (sizeof(T) == 2)
        if (fits(16) && a.cols > 256 && a.cols <= kRingFrom) return backward_vec<T, 16>(ctx, a, dweight, accumulate, stream);
    if (fits(wide)) return backward_vec<T, wide>(ctx, a, dweight, accumulate, stream);
    if constexpr (sizeof(T) == 2)
        if (fits(2)) return backward_vec<T, 2>(ctx, a, dweight, accumulate, stream);
    return backward_vec<T, 1>(ctx, a, dweight, accumulate, stream);
}

// An output may be an input (same address and pitch: every element is read before the thread that read
// it writes it) but may not overlap one in any other way.
bool same_or_apart(const void *out, int64_t ldo, int eo, const void *in, int64_t ldi, int ei, int64_t rows, int64_t cols) {
    if (out == nullptr || in == nullptr || (out == in && (ldo == ldi || rows == 1) && eo == ei)) return true;
    return !Range(out, ldo, rows, cols, eo).overlaps(Range(in, ldi, rows, cols, ei));
}

int check_common(int64_t rows, int64_t cols, float eps) {
    GB200_REQUIRE(rows >= 0 && cols >= 0, GB200_ERR_INVALID_ARG, "negative extent");
    GB200_REQUIRE(eps >= 0.0f && isfinite(eps), GB200_ERR_INVALID_ARG, "eps must be finite and not negative");
    GB200_REQUIRE(cols <= 0x3fffffffll, GB200_ERR_TOO_LARGE, "more than 2^30 - 1 columns");
    GB200_REQUIRE(cols == 0 || rows <= (int64_t)0x3fffffffffffffffll / cols, GB200_ERR_TOO_LARGE, "rows x cols does not fit");
    return GB200_OK;
}

template <typename T, bool QUANT>
int forward_entry(gb200_ctx *ctx, const void *x, int64_t ldx, const void *residual, int64_t ldr, const void *weight, void *y,
                  int64_t ldy, float *scales, int64_t lds, void *h, int64_t ldh, int64_t rows, int64_t cols, int group,
                  float eps, void *stream) {
    GB200_REQUIRE(ctx != nullptr, GB200_ERR_INVALID_ARG, "ctx is NULL");
    int rc = check_common(rows, cols, eps);
    if (rc) return rc;
    constexpr int e = sizeof(T), ye = QUANT ? 1 : e;
    if (QUANT)
        GB200_REQUIRE(group == 0 || group == 32 || group == 64 || group == 128, GB200_ERR_UNSUPPORTED,
                      "a scale covers a whole row (group 0) or 32, 64 or 128 columns, not %d", group);
    if (rows == 0 || cols == 0) return GB200_OK;
    GB200_REQUIRE(x != nullptr && weight != nullptr && y != nullptr, GB200_ERR_INVALID_ARG, "NULL pointer");
    GB200_REQUIRE(ldx >= cols && ldy >= cols && (!residual || ldr >= cols) && (!h || ldh >= cols), GB200_ERR_INVALID_ARG,
                  "leading dimension smaller than the row");
    GB200_REQUIRE(aligned(x, 0, e, e) && aligned(residual, 0, e, e) && aligned(weight, 0, e, e) && aligned(y, 0, e, ye) &&
                      aligned(h, 0, e, e) && aligned(scales, 0, 4, 4),
                  GB200_ERR_INVALID_ARG, "pointer not aligned to its element");
    const int64_t groups = QUANT && group ? (cols + group - 1) / group : 1;
    if (QUANT) {
        GB200_REQUIRE(scales != nullptr, GB200_ERR_INVALID_ARG, "scales is NULL");
        GB200_REQUIRE(lds >= groups, GB200_ERR_INVALID_ARG, "leading dimension of the scales smaller than their row");
    }
    const Range ry(y, ldy, rows, cols, ye), rh(h, ldh, rows, cols, e), rs(scales, lds, rows, groups, 4),
        rw(weight, cols, 1, cols, e), rx(x, ldx, rows, cols, e), rr(residual, ldr, rows, cols, e);
    GB200_REQUIRE(same_or_apart(y, ldy, ye, x, ldx, e, rows, cols) && same_or_apart(y, ldy, ye, residual, ldr, e, rows, cols) &&
                      same_or_apart(h, ldh, e, x, ldx, e, rows, cols) &&
                      same_or_apart(h, ldh, e, residual, ldr, e, rows, cols) && !ry.overlaps(rh) && !ry.overlaps(rw) &&
                      !rh.overlaps(rw) && !rs.overlaps(ry) && !rs.overlaps(rh) && !rs.overlaps(rx) && !rs.overlaps(rr) &&
                      !rs.overlaps(rw),
                  GB200_ERR_INVALID_ARG, "an output overlaps another operand (it may only lie exactly on x or residual)");
    DeviceScope scope;
    rc = scope.enter(ctx);
    if (rc) return rc;
    const NormArgs a{x, residual, weight, ldx, ldr, y, h, ldy, ldh, scales, lds, rows, (int)cols, group, eps};
    return forward<T, QUANT>(ctx, a, static_cast<cudaStream_t>(stream));
}

template <typename T>
int backward_entry(gb200_ctx *ctx, const void *dy, int64_t lddy, const void *h, int64_t ldh, const void *weight, const void *dres,
                   int64_t lddres, void *dx, int64_t lddx, float *dweight, int accumulate, int64_t rows, int64_t cols,
                   float eps, void *stream) {
    GB200_REQUIRE(ctx != nullptr, GB200_ERR_INVALID_ARG, "ctx is NULL");
    int rc = check_common(rows, cols, eps);
    if (rc) return rc;
    constexpr int e = sizeof(T);
    if (cols == 0) return GB200_OK;
    DeviceScope scope;
    if (rows == 0) {   // no rows: no contribution to dweight
        rc = scope.enter(ctx);
        if (rc) return rc;
        if (dweight && !accumulate)
            GB200_CUDA_TRY(cudaMemsetAsync(dweight, 0, cols * sizeof(float), static_cast<cudaStream_t>(stream)));
        return GB200_OK;
    }
    GB200_REQUIRE(dy != nullptr && h != nullptr && weight != nullptr && dx != nullptr, GB200_ERR_INVALID_ARG, "NULL pointer");
    GB200_REQUIRE(lddy >= cols && ldh >= cols && lddx >= cols && (!dres || lddres >= cols), GB200_ERR_INVALID_ARG,
                  "leading dimension smaller than the row");
    GB200_REQUIRE(aligned(dy, 0, e, e) && aligned(h, 0, e, e) && aligned(weight, 0, e, e) && aligned(dres, 0, e, e) &&
                      aligned(dx, 0, e, e) && aligned(dweight, 0, 4, 4),
                  GB200_ERR_INVALID_ARG, "pointer not aligned to its element");
    const Range rdx(dx, lddx, rows, cols, e), rdw(dweight, cols, 1, cols, 4), rw(weight, cols, 1, cols, e),
        rdy(dy, lddy, rows, cols, e), rh(h, ldh, rows, cols, e), rdr(dres, lddres, rows, cols, e);
    GB200_REQUIRE(same_or_apart(dx, lddx, e, dy, lddy, e, rows, cols) && same_or_apart(dx, lddx, e, h, ldh, e, rows, cols) &&
                      same_or_apart(dx, lddx, e, dres, lddres, e, rows, cols) && !rdx.overlaps(rw) && !rdx.overlaps(rdw) &&
                      !rdw.overlaps(rw) && !rdw.overlaps(rdy) && !rdw.overlaps(rh) && !rdw.overlaps(rdr),
                  GB200_ERR_INVALID_ARG, "an output overlaps another operand (dx may only lie exactly on dy, h or dresidual)");
    rc = scope.enter(ctx);
    if (rc) return rc;
    const NormBackArgs a{dy, h, weight, dres, lddy, ldh, lddres, dx, lddx, nullptr, rows, (int)cols, eps};
    return backward<T>(ctx, a, dweight, accumulate, static_cast<cudaStream_t>(stream));
}

}  // namespace
}  // namespace gb200

using namespace gb200;

extern "C" {

int gb200_rmsnorm_f32(gb200_ctx *ctx, const float *x, int64_t ldx, const float *residual, int64_t ldr, const float *weight,
                      float *y, int64_t ldy, float *residual_out, int64_t ldro, int64_t rows, int64_t cols, float eps,
                      void *stream) {
    return forward_entry<float, false>(ctx, x, ldx, residual, ldr, weight, y, ldy, nullptr, 0, residual_out, ldro, rows, cols, 0,
                                       eps, stream);
}

int gb200_rmsnorm_bf16(gb200_ctx *ctx, const void *x, int64_t ldx, const void *residual, int64_t ldr, const void *weight,
                       void *y, int64_t ldy, void *residual_out, int64_t ldro, int64_t rows, int64_t cols, float eps,
                       void *stream) {
    return forward_entry<__nv_bfloat16, false>(ctx, x, ldx, residual, ldr, weight, y, ldy, nullptr, 0, residual_out, ldro, rows,
                                               cols, 0, eps, stream);
}

int gb200_rmsnorm_f32_e4m3(gb200_ctx *ctx, const float *x, int64_t ldx, const float *residual, int64_t ldr,
                           const float *weight, void *q, int64_t ldq, float *scales, int64_t lds, float *residual_out,
                           int64_t ldro, int64_t rows, int64_t cols, int group, float eps, void *stream) {
    return forward_entry<float, true>(ctx, x, ldx, residual, ldr, weight, q, ldq, scales, lds, residual_out, ldro, rows, cols,
                                      group, eps, stream);
}

int gb200_rmsnorm_bf16_e4m3(gb200_ctx *ctx, const void *x, int64_t ldx, const void *residual, int64_t ldr,
                            const void *weight, void *q, int64_t ldq, float *scales, int64_t lds, void *residual_out,
                            int64_t ldro, int64_t rows, int64_t cols, int group, float eps, void *stream) {
    return forward_entry<__nv_bfloat16, true>(ctx, x, ldx, residual, ldr, weight, q, ldq, scales, lds, residual_out, ldro, rows,
                                              cols, group, eps, stream);
}

int gb200_rmsnorm_backward_f32(gb200_ctx *ctx, const float *dy, int64_t lddy, const float *h, int64_t ldh,
                               const float *weight, const float *dresidual, int64_t lddr, float *dx, int64_t lddx,
                               float *dweight, int accumulate, int64_t rows, int64_t cols, float eps, void *stream) {
    return backward_entry<float>(ctx, dy, lddy, h, ldh, weight, dresidual, lddr, dx, lddx, dweight, accumulate, rows, cols, eps,
                                 stream);
}

int gb200_rmsnorm_backward_bf16(gb200_ctx *ctx, const void *dy, int64_t lddy, const void *h, int64_t ldh,
                                const void *weight, const void *dresidual, int64_t lddr, void *dx, int64_t lddx,
                                float *dweight, int accumulate, int64_t rows, int64_t cols, float eps, void *stream) {
    return backward_entry<__nv_bfloat16>(ctx, dy, lddy, h, ldh, weight, dresidual, lddr, dx, lddx, dweight, accumulate, rows,
                                         cols, eps, stream);
}

}  // extern "C"
