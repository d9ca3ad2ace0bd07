// Global norm of a list of gradient tensors, and clipping by it.
//
//   norm = sqrt(sum over all tensors and elements of g^2),   c = norm > max_norm ? max_norm / norm : 1,   out = c g
//
// The whole-list counterpart of the row reductions in softmax.cu; the reference has nothing like it.
//
// Bound: HBM.  The norm has to be known before anything can be scaled, so every gradient is read
// twice, and written once; the second pass walks the list backwards, so that what the first pass read
// last is still in the 126 MB L2 when it is wanted again.  537M bf16 gradients in 292 tensors: 168 us for the
// norm (6.4 TB/s), 501 us in all, the time of 3.2 GB at the copy rate being 492.  Tensors are cut into equal chunks; the
// list travels in the kernel's parameters (no table in device memory that a later call or a replayed
// graph could find changed), and a block finds its chunk's tensor by bisection.
//
// Numerics: squares of 16 elements at a time are added in fp32; a group whose sum over- or underflows
// there (gradients beyond 1e19 or below 1e-17) is added again in fp64.  Sums of groups are fp64, in
// an order that only the list and the device's SM count set: the same call gives the same bits.
#include <algorithm>
#include <math.h>
#include <vector>

#include "common.cuh"

namespace gb200 {
namespace {

struct Entry {
    const void *in;
    void *out;
    int64_t n;
    int32_t first_chunk;    // chunks of the tensors before it in this launch
    int32_t type;           // kIn16 | kOut16
};
enum { kIn16 = 1, kOut16 = 2 };

// Kernel parameters may take 32,764 bytes; lists of up to 100 tensors use the short form, whose
// launch is not slowed by the copy of 32 KB.
template <int CAP>
struct List {
    int count;
    int chunks;
    int chunk;              // elements, a multiple of 4096
    int pad;
    Entry e[CAP];
};
constexpr int kShort = 100, kFull = 1000;
static_assert(sizeof(List<kShort>) <= 4000 && sizeof(List<kFull>) <= 32600, "kernel parameter space");

constexpr int kThreads = 256;

struct NormOut {
    double *parts;          // one per block of every launch of the call
    int first_part, total_parts;
    int last;               // this launch finishes the sum
    float *norm;
    unsigned int *ticket;
};

template <int CAP>
__device__ __forceinline__ int find_tensor(const List<CAP> &l, int chunk) {
    int lo = 0, hi = l.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (l.e[mid].first_chunk <= chunk) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// W elements of T as floats, by one load where the address allows it.
template <typename T> struct Vec;
template <> struct Vec<float> {
    static constexpr int W = 4;
    using type = float4;
    __device__ static void widen(const float4 &p, float *v) { v[0] = p.x; v[1] = p.y; v[2] = p.z; v[3] = p.w; }
    __device__ static float one(const float *p) { return *p; }
};
template <> struct Vec<__nv_bfloat16> {
    static constexpr int W = 8;
    using type = uint4;
    __device__ static void widen(const uint4 &p, float *v) {
        const uint32_t w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    __device__ static float one(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
};

// Elements of T before the next 16-byte boundary at or after p.
template <typename T>
__device__ __forceinline__ int to_boundary(const T *p) {
    return static_cast<int>((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / static_cast<int>(sizeof(T));
}

template <int N>
__device__ __forceinline__ double squares(const float (&v)[N]) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) s = fmaf(v[i], v[i], s);
    if (s < 1e30f && s > 1e-30f) return static_cast<double>(s);
    double d = 0.0;      // out of fp32's comfortable range (or all zero, infinite, NaN): add again in fp64
#pragma unroll
    for (int i = 0; i < N; ++i) d = fma(static_cast<double>(v[i]), static_cast<double>(v[i]), d);
    return d;
}

__device__ __forceinline__ double block_sum(double v, double *red) {
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (lane == 0) red[wid] = v;
    __syncthreads();
    v = lane < kThreads / 32 ? red[lane] : 0.0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// One chunk's share of a thread: the elements up to the first 16-byte boundary and behind the last
// one singly, those between as vectors, 64 bytes in flight per thread.
template <typename T>
__device__ __forceinline__ double chunk_squares(const T *p, int n) {
    constexpr int W = Vec<T>::W, PER = 16 / W;   // vectors in a group of 16
    const int head = min(to_boundary(p), n);
    const int nvec = (n - head) / W, tail = head + nvec * W;
    const auto *q = reinterpret_cast<const typename Vec<T>::type *>(p + head);
    double sum = 0.0;
    for (int i = threadIdx.x; i < nvec; i += 4 * kThreads) {
        typename Vec<T>::type x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = i + k * kThreads < nvec ? q[i + k * kThreads] : typename Vec<T>::type{};
#pragma unroll
        for (int k = 0; k < 4; k += PER) {
            float v[16];
#pragma unroll
            for (int m = 0; m < PER; ++m) Vec<T>::widen(x[k + m], v + m * W);
            sum += squares(v);
        }
    }
    // fewer than 16 elements at either end
    const int i = threadIdx.x < head ? threadIdx.x : tail + static_cast<int>(threadIdx.x) - head;
    if (i < n) {
        const float v[1] = {Vec<T>::one(p + i)};
        sum += squares(v);
    }
    return sum;
}

template <int CAP>
__global__ void __launch_bounds__(kThreads)
grad_norm_kernel(const __grid_constant__ List<CAP> l, const NormOut o) {
    __shared__ double red[kThreads / 32];
    __shared__ bool last_block;
    pdl_launch_dependents();
    pdl_wait();
    double sum = 0.0;
    for (int c = blockIdx.x; c < l.chunks; c += gridDim.x) {
        const Entry &e = l.e[find_tensor(l, c)];
        const int64_t first = static_cast<int64_t>(c - e.first_chunk) * l.chunk;
        const int n = static_cast<int>(e.n - first < l.chunk ? e.n - first : l.chunk);
        if (e.type & kIn16) sum += chunk_squares(static_cast<const __nv_bfloat16 *>(e.in) + first, n);
        else sum += chunk_squares(static_cast<const float *>(e.in) + first, n);
    }
    sum = block_sum(sum, red);
    if (threadIdx.x == 0) {
        o.parts[o.first_part + blockIdx.x] = sum;
        last_block = false;
        if (o.last) {
            __threadfence();
            last_block = atomicAdd(o.ticket, 1u) == gridDim.x - 1;
        }
    }
    __syncthreads();
    if (!last_block) return;
    __threadfence();
    double total = 0.0;
    for (int i = threadIdx.x; i < o.total_parts; i += kThreads) total += __ldcg(o.parts + i);
    total = block_sum(total, red);
    if (threadIdx.x == 0) {
        *o.norm = static_cast<float>(sqrt(total));
        *o.ticket = 0;
    }
}

__device__ __forceinline__ void store_one(float v, __nv_bfloat16 *d) { *d = __float2bfloat16_rn(v); }
__device__ __forceinline__ void store_one(float v, float *d) { *d = v; }

// What one 16-byte store of the result takes from the gradient, and the scaled result.
template <typename TI, typename TO> struct Step;
template <> struct Step<float, float> {
    using in = float4;
    using out = float4;
    __device__ static out scale(const in &p, float c) { return make_float4(p.x * c, p.y * c, p.z * c, p.w * c); }
};
template <> struct Step<__nv_bfloat16, float> {
    using in = uint2;
    using out = float4;
    __device__ static out scale(const in &p, float c) {
        return make_float4(__uint_as_float(p.x << 16) * c, __uint_as_float(p.x & 0xffff0000u) * c, __uint_as_float(p.y << 16) * c,
                           __uint_as_float(p.y & 0xffff0000u) * c);
    }
};
template <> struct Step<__nv_bfloat16, __nv_bfloat16> {
    using in = uint4;
    using out = uint4;
    __device__ static uint32_t two(uint32_t w, float c) {
        return pack_bf16(__uint_as_float(w << 16) * c, __uint_as_float(w & 0xffff0000u) * c);
    }
    __device__ static out scale(const in &p, float c) { return make_uint4(two(p.x, c), two(p.y, c), two(p.z, c), two(p.w, c)); }
};

// Vectors aligned on the output, four in flight per thread, where the input lies alike; else element by
// element.  The ends before the first and behind the last 16-byte boundary are taken singly.
template <typename TI, typename TO>
__device__ __forceinline__ void chunk_scale(const TI *p, TO *d, int n, float c) {
    using S = Step<TI, TO>;
    constexpr int W = 16 / sizeof(TO);
    const int head = min(to_boundary(d), n);
    if (reinterpret_cast<uintptr_t>(p + head) % sizeof(typename S::in) != 0) {
#pragma unroll 8
        for (int i = threadIdx.x; i < n; i += kThreads) store_one(Vec<TI>::one(p + i) * c, d + i);
        return;
    }
    const int nvec = (n - head) / W, tail = head + nvec * W;
    const auto *in = reinterpret_cast<const typename S::in *>(p + head);
    auto *out = reinterpret_cast<typename S::out *>(d + head);
    for (int i = threadIdx.x; i < nvec; i += 4 * kThreads) {
        typename S::in x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (i + k * kThreads < nvec) x[k] = in[i + k * kThreads];
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (i + k * kThreads < nvec) __stcs(out + i + k * kThreads, S::scale(x[k], c));
    }
    const int i = threadIdx.x < head ? threadIdx.x : tail + static_cast<int>(threadIdx.x) - head;
    if (i < n) store_one(Vec<TI>::one(p + i) * c, d + i);
}

// Scales; chunks are taken from the last to the first.
template <int CAP>
__global__ void __launch_bounds__(kThreads)
grad_scale_kernel(const __grid_constant__ List<CAP> l, const float *norm, float max_norm) {
    pdl_launch_dependents();
    pdl_wait();
    const float have = *norm;
    // a norm that is not finite scales nothing: the caller sees it and drops the step
    const float c = have > max_norm && have < INFINITY ? max_norm / have : 1.0f;
    const int chunk = l.chunks - 1 - static_cast<int>(blockIdx.x);
    const Entry &e = l.e[find_tensor(l, chunk)];
    if (c == 1.0f && e.in == e.out) return;
    const int64_t first = static_cast<int64_t>(chunk - e.first_chunk) * l.chunk;
    const int n = static_cast<int>(e.n - first < l.chunk ? e.n - first : l.chunk);
    if ((e.type & kIn16) && (e.type & kOut16))
        chunk_scale(static_cast<const __nv_bfloat16 *>(e.in) + first, static_cast<__nv_bfloat16 *>(e.out) + first, n, c);
    else if (e.type & kIn16)
        chunk_scale(static_cast<const __nv_bfloat16 *>(e.in) + first, static_cast<float *>(e.out) + first, n, c);
    else
        chunk_scale(static_cast<const float *>(e.in) + first, static_cast<float *>(e.out) + first, n, c);
}

struct Span {
    uintptr_t lo, hi;
    bool written;
};

// Checks the list; `outputs`: the out pointers are used.
int check(const gb200_tensor *t, int64_t count, bool outputs, const float *norm, int64_t *elements) {
    GB200_REQUIRE(count >= 0, GB200_ERR_INVALID_ARG, "negative number of tensors");
    GB200_REQUIRE(count == 0 || t != nullptr, GB200_ERR_INVALID_ARG, "tensors is NULL");
    GB200_REQUIRE(count <= 1000000, GB200_ERR_TOO_LARGE, "more than 1000000 tensors");
    int64_t total = 0;
    for (int64_t i = 0; i < count; ++i) {
        GB200_REQUIRE(t[i].numel >= 0 && t[i].numel <= (1ll << 40), GB200_ERR_INVALID_ARG, "tensor %lld: %lld elements",
                      (long long)i, (long long)t[i].numel);
        GB200_REQUIRE((t[i].type == GB200_F32 || t[i].type == GB200_BF16) &&
                          (!outputs || !t[i].out || t[i].out_type == GB200_F32 || t[i].out_type == GB200_BF16),
                      GB200_ERR_UNSUPPORTED, "tensor %lld: element type is neither GB200_F32 nor GB200_BF16", (long long)i);
        if (t[i].numel == 0) continue;
        const uintptr_t in = reinterpret_cast<uintptr_t>(t[i].data), out = reinterpret_cast<uintptr_t>(t[i].out);
        GB200_REQUIRE(in != 0, GB200_ERR_INVALID_ARG, "tensor %lld: data is NULL", (long long)i);
        GB200_REQUIRE(in % (t[i].type == GB200_F32 ? 4 : 2) == 0, GB200_ERR_INVALID_ARG,
                      "tensor %lld: data is not aligned to its element", (long long)i);
        if (outputs && out) {
            GB200_REQUIRE(out % (t[i].out_type == GB200_F32 ? 4 : 2) == 0, GB200_ERR_INVALID_ARG,
                          "tensor %lld: out is not aligned to its element", (long long)i);
            GB200_REQUIRE(t[i].type == GB200_BF16 || t[i].out_type == GB200_F32, GB200_ERR_UNSUPPORTED,
                          "tensor %lld: an fp32 gradient has an fp32 result", (long long)i);
        }
        total += t[i].numel;
    }
    GB200_REQUIRE(total <= (1ll << 45), GB200_ERR_TOO_LARGE, "more than 2^45 elements");
    *elements = total;
    if (!outputs) return GB200_OK;
    // Two blocks may not write one element, nor one read what another writes.
    std::vector<Span> spans;
    spans.reserve((size_t)count * 2 + 1);
    spans.push_back({reinterpret_cast<uintptr_t>(norm), reinterpret_cast<uintptr_t>(norm) + sizeof(float), true});
    for (int64_t i = 0; i < count; ++i) {
        if (t[i].numel == 0) continue;
        const uintptr_t in = reinterpret_cast<uintptr_t>(t[i].data), out = reinterpret_cast<uintptr_t>(t[i].out);
        const uintptr_t in_bytes = (uintptr_t)t[i].numel * (t[i].type == GB200_F32 ? 4 : 2);
        if (out == 0 || (out == in && t[i].out_type == t[i].type)) {
            spans.push_back({in, in + in_bytes, true});
        } else {
            spans.push_back({in, in + in_bytes, false});
            spans.push_back({out, out + (uintptr_t)t[i].numel * (t[i].out_type == GB200_F32 ? 4 : 2), true});
        }
    }
    auto before = [](const Span &a, const Span &b) { return a.lo < b.lo; };
    if (!std::is_sorted(spans.begin(), spans.end(), before)) std::sort(spans.begin(), spans.end(), before);
    uintptr_t written = 0, any = 0;
    for (const Span &s : spans) {
        GB200_REQUIRE(s.lo >= (s.written ? any : written), GB200_ERR_INVALID_ARG,
                      "a tensor that is written overlaps another one of the list, is in it twice, or overlaps norm");
        any = std::max(any, s.hi);
        if (s.written) written = std::max(written, s.hi);
    }
    return GB200_OK;
}

// Elements per chunk of the norm: about four chunks per SM, between 4096 (a short list still spreads over
// the SMs) and 65536.
int pick_chunk(int64_t elements, int sm_count) {
    int64_t c = elements / ((int64_t)sm_count * 4);
    c = (c + 4095) / 4096 * 4096;
    return (int)std::min<int64_t>(std::max<int64_t>(c, 4096), 65536);
}
// Scaling gives every chunk a block of its own: blocks that come and go in the tensors' order keep the
// addresses in flight close together (536870912 bf16 in 292 tensors, norm and scaling: 502 us with 8192
// elements, 509 with 16384, 523 with 32768).
constexpr int kScaleChunk = 8192;
int pick_scale_chunk(int64_t elements) { return elements / kScaleChunk < (1ll << 30) ? kScaleChunk : 1 << 20; }

// Cuts the list into launches of up to CAP tensors and hands each to `f`.
template <int CAP, typename F>
int for_lists(const gb200_tensor *t, int64_t count, int chunk, F &&f) {
    List<CAP> l;
    int64_t i = 0;
    while (i < count) {
        l.count = 0;
        l.chunk = chunk;
        l.pad = 0;
        int64_t chunks = 0;
        for (; i < count && l.count < CAP; ++i) {
            if (t[i].numel == 0) continue;
            const int64_t more = (t[i].numel + chunk - 1) / chunk;
            Entry &e = l.e[l.count++];
            e.in = t[i].data;
            e.out = t[i].out ? t[i].out : const_cast<void *>(t[i].data);
            e.n = t[i].numel;
            e.first_chunk = (int32_t)chunks;
            e.type = (t[i].type == GB200_BF16 ? kIn16 : 0) | ((t[i].out ? t[i].out_type : t[i].type) == GB200_BF16 ? kOut16 : 0);
            chunks += more;
        }
        if (l.count == 0) break;
        l.chunks = (int)chunks;
        bool more_to_come = false;
        for (int64_t k = i; k < count && !more_to_come; ++k) more_to_come = t[k].numel != 0;
        const int rc = f(l, !more_to_come);
        if (rc) return rc;
    }
    return GB200_OK;
}

template <int CAP>
int norm_of(gb200_ctx *ctx, const gb200_tensor *t, int64_t count, int chunk, float *norm, cudaStream_t stream) {
    // parts: a grid of at most 8 blocks per SM for each launch of the list
    const int64_t launches = (count + CAP - 1) / CAP + 1;
    const int grid_cap = ctx->sm_count * 8;
    void *ws = nullptr;
    int rc = scratch_reserve(ctx, (size_t)launches * grid_cap * sizeof(double), stream, &ws);
    if (rc) return rc;
    int parts = 0;
    return for_lists<CAP>(t, count, chunk, [&](const List<CAP> &l, bool last) -> int {
        const int blocks = std::min(l.chunks, grid_cap);
        NormOut o{static_cast<double *>(ws), parts, parts + blocks, last ? 1 : 0, norm, ctx->tickets + kTicketNorm};
        parts += blocks;
        GB200_CUDA_TRY(launch_pdl(grad_norm_kernel<CAP>, dim3((unsigned)blocks), dim3(kThreads), 0, stream, l, o));
        return after_launch(ctx, "grad_norm_kernel");
    });
}

template <int CAP>
int scale_of(gb200_ctx *ctx, const gb200_tensor *t, int64_t count, int chunk, const float *norm, float max_norm,
             cudaStream_t stream) {
    return for_lists<CAP>(t, count, chunk, [&](const List<CAP> &l, bool) -> int {
        GB200_CUDA_TRY(launch_pdl(grad_scale_kernel<CAP>, dim3((unsigned)l.chunks), dim3(kThreads), 0, stream, l, norm, max_norm));
        return after_launch(ctx, "grad_scale_kernel");
    });
}

enum { kNorm = 1, kScale = 2 };

int entry(gb200_ctx *ctx, const gb200_tensor *t, int64_t count, int what, float max_norm, float *norm, void *stream_) {
    GB200_REQUIRE(ctx != nullptr, GB200_ERR_INVALID_ARG, "ctx is NULL");
    GB200_REQUIRE(norm != nullptr && reinterpret_cast<uintptr_t>(norm) % 4 == 0, GB200_ERR_INVALID_ARG,
                  "norm is NULL or not aligned to its element");
    if (what & kScale) GB200_REQUIRE(max_norm >= 0.0f, GB200_ERR_INVALID_ARG, "max_norm must not be negative or NaN");
    int64_t elements = 0;
    int rc = check(t, count, (what & kScale) != 0, norm, &elements);
    if (rc) return rc;
    DeviceScope scope;
    rc = scope.enter(ctx);
    if (rc) return rc;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    if (elements == 0) {
        if (what & kNorm) GB200_CUDA_TRY(cudaMemsetAsync(norm, 0, sizeof(float), stream));
        return GB200_OK;
    }
    const int chunk = pick_chunk(elements, ctx->sm_count);
    const bool short_list = count <= kShort;
    if (what & kNorm) {
        rc = short_list ? norm_of<kShort>(ctx, t, count, chunk, norm, stream) : norm_of<kFull>(ctx, t, count, chunk, norm, stream);
        if (rc) return rc;
    }
    if (what & kScale)
        rc = short_list ? scale_of<kShort>(ctx, t, count, pick_scale_chunk(elements), norm, max_norm, stream)
                        : scale_of<kFull>(ctx, t, count, pick_scale_chunk(elements), norm, max_norm, stream);
    return rc;
}

// No C++ exception leaves the C ABI.
int guarded(gb200_ctx *ctx, const gb200_tensor *t, int64_t count, int what, float max_norm, float *norm, void *stream) {
    try {
        return entry(ctx, t, count, what, max_norm, norm, stream);
    } catch (...) {
        set_error("out of host memory for the list of tensors");
        return GB200_ERR_TOO_LARGE;
    }
}

}  // namespace
}  // namespace gb200

using namespace gb200;

extern "C" {

int gb200_grad_norm(gb200_ctx *ctx, const gb200_tensor *tensors, int64_t count, float *norm, void *stream) {
    return guarded(ctx, tensors, count, kNorm, 0.0f, norm, stream);
}

int gb200_grad_scale(gb200_ctx *ctx, const gb200_tensor *tensors, int64_t count, float max_norm, const float *norm,
                     void *stream) {
    return guarded(ctx, tensors, count, kScale, max_norm, const_cast<float *>(norm), stream);
}

int gb200_grad_clip(gb200_ctx *ctx, const gb200_tensor *tensors, int64_t count, float max_norm, float *norm, void *stream) {
    return guarded(ctx, tensors, count, kNorm | kScale, max_norm, norm, stream);
}

}  // extern "C"
