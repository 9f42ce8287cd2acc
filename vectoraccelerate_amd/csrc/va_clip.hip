// va_clip.hip — the global 2-norm of a list of gradients, and the gradients clipped by it.
//
//   n = sqrt(sum over all values g^2)        out = g min(1, max_norm / (n + eps))
//
// Bound by memory: the gradients are read twice (the factor is known after the last of them) and
// written once.  The list travels in the kernels' arguments, kListMax tensors a launch, so a
// call leaves nothing behind that it would have to wait for.  A tensor is cut into chunks of
// kChunk values, whose loads are issued together; a workgroup takes a run of chunks and leaves one sum.  Sums are
// fp64 from the first product on (gradients of any magnitude, no overflow) and joined in a fixed order by every
// workgroup of the second pass, so results do not depend on the order in which workgroups run.  The second pass
// starts where the first one ended: what is left of it in the caches is read from there.
//
// Measured: 468 MB in bf16 110 us to read (4.2 TB/s, the cache writing back what a pass before left in it) and
// 165 us to scale (5.7 TB/s); 94 MB in 290 tensors 22 and 41 us; a few small tensors 4 and 5 us, the launches.
#include <algorithm>
#include <cmath>

#include "va_internal.hpp"

namespace va {
namespace {

constexpr uint32_t kChunk = 16384;
constexpr uint32_t kListMax = 166;    // just under 4 KiB of arguments
constexpr uint32_t kChunk0Max = 1u << 22;
// Workgroups of 256 threads a CU, all of them resident (72 registers): the two passes over 468 MB in bf16 take 289 us
// with 7, 291 with 6, 294 with 8 (64 registers); over 94 MB in 290 tensors 66, 68 and 67.
constexpr uint32_t kPerCu = 7;

// A tensor in 24 bytes: the more of them a launch holds, the fewer launches (290 tensors of 94 MB: 124 a launch
// 81 us, 166 a launch 72 us, before the grid above).
struct Entry {
    const void* in;
    void* out;
    uint64_t word;  // values (40 bits), first chunk among the launch's (22), type (2)
    __host__ __device__ uint64_t count() const { return word & ((1ull << 40) - 1); }
    __host__ __device__ uint32_t chunk0() const { return uint32_t(word >> 40) & (kChunk0Max - 1); }
    __host__ __device__ uint32_t dtype() const { return uint32_t(word >> 62); }
};
struct List {
    Entry e[kListMax];
    uint32_t n, chunks;
};
static_assert(sizeof(List) + 64 <= 4096, "kernel arguments");

template <class T>
using Vec8 = T __attribute__((ext_vector_type(8), aligned(sizeof(T))));
typedef float f32x8 __attribute__((ext_vector_type(8)));

// the tensor that holds chunk c, found by the whole wave: lane i looks at tensors i, 64 + i, ...
__device__ __forceinline__ uint32_t tensor_of(const List& l, uint32_t c) {
    uint32_t n = 0;
    for (uint32_t i = threadIdx.x & 63; i < (l.n + 63) / 64 * 64; i += 64) n += uint32_t(__popcll(__ballot(i < l.n && l.e[min(i, l.n - 1)].chunk0() <= c)));
    return __builtin_amdgcn_readfirstlane(n) - 1;
}

__device__ __forceinline__ double block_sum(double v, double* part) {
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0;
    for (uint32_t i = 0; i < blockDim.x / 64; ++i) v += part[i];
    return v;
}

template <class T>
__device__ __forceinline__ void add_squares(double (&s)[2], Vec8<T> v) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const double x = double(float(v[e]));
        s[e & 1] = fma(x, x, s[e & 1]);
    }
}
template <class T>
__device__ __forceinline__ double square_sum(const T* p, uint32_t n) {
    double s[2] = {0.0, 0.0};
    if (n == kChunk) {
        constexpr int R = sizeof(T) == 4 ? 4 : 8;  // 128 bytes a thread in flight
#pragma unroll
        for (uint32_t b = 0; b < kChunk / 2048; b += R) {
            Vec8<T> v[R];
#pragma unroll
            for (int r = 0; r < R; ++r) v[r] = *reinterpret_cast<const Vec8<T>*>(p + 2048 * (b + r) + 8 * threadIdx.x);
#pragma unroll
            for (int r = 0; r < R; ++r) add_squares<T>(s, v[r]);
        }
        return s[0] + s[1];
    }
    const uint32_t full = n / 8;
#pragma unroll 4
    for (uint32_t i = threadIdx.x; i < full; i += 256) add_squares<T>(s, *reinterpret_cast<const Vec8<T>*>(p + 8 * i));
    const uint32_t i = 8 * full + threadIdx.x;
    if (i < n) {
        const double x = double(float(p[i]));
        s[0] = fma(x, x, s[0]);
    }
    return s[0] + s[1];
}

__global__ __launch_bounds__(256, kPerCu) void clip_norm_kernel(List l, double* sums) {
    __shared__ double part[4];
    double s = 0.0;
    const uint32_t c0 = uint32_t(uint64_t(l.chunks) * blockIdx.x / gridDim.x), c1 = uint32_t(uint64_t(l.chunks) * (blockIdx.x + 1) / gridDim.x);
    uint32_t i = tensor_of(l, c0);
    for (uint32_t c = c0; c < c1; ++c) {
        if (i + 1 < l.n && l.e[i + 1].chunk0() <= c) ++i;  // (no tensor of a list is empty)
        const Entry& e = l.e[i];
        const uint64_t at = uint64_t(c - e.chunk0()) * kChunk;
        const uint32_t n = uint32_t(min(uint64_t(kChunk), e.count() - at));
        if (e.dtype() == VA_DTYPE_F32) s += square_sum(static_cast<const float*>(e.in) + at, n);
        else if (e.dtype() == VA_DTYPE_F16) s += square_sum(static_cast<const _Float16*>(e.in) + at, n);
        else s += square_sum(static_cast<const __bf16*>(e.in) + at, n);
    }
    s = block_sum(s, part);
    if (threadIdx.x == 0) sums[blockIdx.x] = s;
}

template <class T>
__device__ __forceinline__ void scale_chunk(const T* in, T* out, uint32_t n, float f) {
    auto put = [&](uint32_t at, Vec8<T> v) {
        const f32x8 x = __builtin_convertvector(v, f32x8) * f;
        *reinterpret_cast<Vec8<T>*>(out + at) = __builtin_convertvector(x, Vec8<T>);
    };
    if (n == kChunk) {
        constexpr int R = sizeof(T) == 4 ? 4 : 8;
#pragma unroll
        for (uint32_t b = 0; b < kChunk / 2048; b += R) {
            Vec8<T> v[R];
#pragma unroll
            for (int r = 0; r < R; ++r) v[r] = *reinterpret_cast<const Vec8<T>*>(in + 2048 * (b + r) + 8 * threadIdx.x);
#pragma unroll
            for (int r = 0; r < R; ++r) put(2048 * (b + r) + 8 * threadIdx.x, v[r]);
        }
        return;
    }
    const uint32_t full = n / 8;
#pragma unroll 4
    for (uint32_t i = threadIdx.x; i < full; i += 256) put(8 * i, *reinterpret_cast<const Vec8<T>*>(in + 8 * i));
    const uint32_t i = 8 * full + threadIdx.x;
    if (i < n) out[i] = T(float(in[i]) * f);
}

__global__ __launch_bounds__(256, kPerCu) void clip_scale_kernel(List l, const double* __restrict__ sums, uint32_t nsums, float max_norm, float eps,
                                                         float* out_norm) {
    __shared__ double part[4];
    double s = 0.0;
    for (uint32_t i = threadIdx.x; i < nsums; i += 256) s += sums[i];
    const double norm = sqrt(block_sum(s, part));
    // (a comparison that is false for NaN keeps it, as the quotient does)
    const double q = double(max_norm) / (norm + double(eps));
    const float f = q > 1.0 ? 1.0f : float(q);
    if (out_norm && blockIdx.x == 0 && threadIdx.x == 0) *out_norm = float(norm);
    if (!l.n) return;
    const uint32_t b = gridDim.x - 1 - blockIdx.x;
    const uint32_t c0 = uint32_t(uint64_t(l.chunks) * b / gridDim.x), c1 = uint32_t(uint64_t(l.chunks) * (b + 1) / gridDim.x);
    uint32_t i = tensor_of(l, c0);
    for (uint32_t c = c0; c < c1; ++c) {
        if (i + 1 < l.n && l.e[i + 1].chunk0() <= c) ++i;
        const Entry& e = l.e[i];
        if (f == 1.0f && e.in == e.out) continue;  // in place, and nothing changes
        const uint64_t at = uint64_t(c - e.chunk0()) * kChunk;
        const uint32_t n = uint32_t(min(uint64_t(kChunk), e.count() - at));
        if (e.dtype() == VA_DTYPE_F32) scale_chunk(static_cast<const float*>(e.in) + at, static_cast<float*>(e.out) + at, n, f);
        else if (e.dtype() == VA_DTYPE_F16) scale_chunk(static_cast<const _Float16*>(e.in) + at, static_cast<_Float16*>(e.out) + at, n, f);
        else scale_chunk(static_cast<const __bf16*>(e.in) + at, static_cast<__bf16*>(e.out) + at, n, f);
    }
}

// tensors [i, ...) of the list into one launch's arguments; the first tensor not taken
uint32_t take(const va_tensor_list* t, uint32_t i, List& l) {
    l.n = 0;
    uint64_t chunks = 0;
    for (; i < t->count && l.n < kListMax && chunks < kChunk0Max; ++i) {
        if (!t->sizes[i]) continue;
        l.e[l.n++] = Entry{t->tensors[i], t->outputs ? t->outputs[i] : t->tensors[i], t->sizes[i] | chunks << 40 | uint64_t(t->dtypes[i]) << 62};
        chunks += (t->sizes[i] + kChunk - 1) / kChunk;
    }
    l.chunks = uint32_t(chunks);  // (below 2^22 + 2^26)
    return i;
}

}  // namespace
}  // namespace va

using namespace va;

extern "C" {

va_status va_grad_clip(va_context* ctx, const va_tensor_list* t, float max_norm, float epsilon, float* out_norm) {
    if (!ctx) return VA_ERR_INVALID_ARG;
    VA_REQUIRE(ctx, t && (t->count == 0 || (t->tensors && t->sizes && t->dtypes)), "va_grad_clip: NULL list");
    VA_REQUIRE(ctx, max_norm >= 0.0f, "va_grad_clip: max_norm must not be negative or NaN");
    VA_REQUIRE(ctx, std::isfinite(epsilon) && epsilon >= 0.0f, "va_grad_clip: epsilon must be finite and not negative");
    uint64_t total = 0;
    for (uint32_t i = 0; i < t->count; ++i) {
        VA_REQUIRE(ctx, t->dtypes[i] == VA_DTYPE_F32 || t->dtypes[i] == VA_DTYPE_F16 || t->dtypes[i] == VA_DTYPE_BF16, "va_grad_clip: tensor %u: unknown type %d", i, int(t->dtypes[i]));
        const uintptr_t es = t->dtypes[i] == VA_DTYPE_F32 ? 4 : 2;
        const void* o = t->outputs ? t->outputs[i] : t->tensors[i];
        VA_REQUIRE(ctx, !t->sizes[i] || (t->tensors[i] && o), "va_grad_clip: tensor %u is NULL", i);
        VA_REQUIRE(ctx, reinterpret_cast<uintptr_t>(t->tensors[i]) % es == 0 && reinterpret_cast<uintptr_t>(o) % es == 0, "va_grad_clip: tensor %u is not aligned to its type", i);
        VA_REQUIRE(ctx, t->sizes[i] < 1ull << 40, "va_grad_clip: tensor %u: too many values", i);
        total += (t->sizes[i] + kChunk - 1) / kChunk;
    }
    DeviceGuard guard(ctx->device);
    // the launches are at most so many: each is closed by its tensors, or by its chunks
    const uint32_t most = kPerCu * uint32_t(ctx->num_cus);
    const uint64_t launches = ceil_div(t->count, kListMax) + total / kChunk0Max;
    Scratch sc(ctx);
    const uint64_t slots = std::min<uint64_t>(uint64_t(launches) * most, total);
    VA_CHECK_STATUS(sc.reserve(Scratch::round(slots * sizeof(double))));
    double* sums = sc.carve<double>(slots);
    uint32_t n = 0;
    List l;
    for (uint32_t i = 0; i < t->count;) {
        i = take(t, i, l);
        if (!l.n) break;
        const uint32_t grid = std::min(l.chunks, most);
        clip_norm_kernel<<<dim3(grid), dim3(256), 0, ctx->stream>>>(l, sums + n);
        VA_CHECK_LAUNCH(ctx);
        n += grid;
    }
    bool told = false;
    for (uint32_t i = 0; i < t->count || !told;) {
        i = take(t, i, l);
        if (!l.n && told) break;
        clip_scale_kernel<<<dim3(std::min(std::max(l.chunks, 1u), most)), dim3(256), 0, ctx->stream>>>(l, sums, n, max_norm, epsilon, told ? nullptr : out_norm);
        VA_CHECK_LAUNCH(ctx);
        told = true;
    }
    return VA_OK;
}

}  // extern "C"
