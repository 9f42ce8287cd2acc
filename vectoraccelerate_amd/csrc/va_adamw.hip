// va_adamw.hip — one AdamW step over a list of tensors, its moments in 32 bits or in 8.
//
//   g' = g s min(1, max_norm / (s norm + 1e-6))            (the factor only with a norm; s: grad_scale)
//   m = b1 m + (1 - b1) g'        v = b2 v + (1 - b2) g'^2
//   p = p (1 - rate decay) - rate m / (1 - b1^t) / (sqrt(v / (1 - b2^t)) + eps)
//
// Gradients, moments and parameters are read once, moments and parameters written once (fp32 28 bytes a value, bf16
// with fp32 moments 22, with 8-bit ones 10.1).  The list lies in device memory, laid out once when it is made, so a step is
// one launch whatever the number of tensors.  A tensor is cut into chunks of kChunk values; a workgroup takes a run of
// chunks and goes from tensor to tensor as they end, and a launch is as many workgroups as the CUs hold at once.
// Measured: 290 bf16 tensors, 38.6M values with fp32 moments and copies, 219 us, 4.9 TB/s, what a large copy reaches; 50 bf16
// tensors of 228M values with 8-bit moments 522-555 us, 4.1-4.4 TB/s (to 680 in the first milliseconds of work, while the clock is
// down): beside memory by the vector instructions, of which the random words' 64-bit products and the exact root are most; 6 tensors
// of a head 5 us, a launch.
//
// 8-bit moments: e4m3 codes with an fp32 scale for each group of 256 values (a tensor's first value starts one), of m
// and of r = sqrt(v), whose range is half of v's in binary orders.  Each group's largest value is code 448.  What
// lies between two codes goes to the upper one with the probability of the part cut off: with b2 = 0.999 a moment moves by
// less than a code's width a step, and rounded to the nearest it would never come down.  r > 0 never becomes 0, so no
// m is divided by eps alone.  The random bits are splitmix64 of (seed, step, place in the list), so a step repeats
// bit for bit.  p is computed from the moments before they are rounded.
#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

#include "va_internal.hpp"

struct va_adamw_list {
    int device = 0;
    void* table = nullptr;  // entries, then each entry's first chunk
    uint32_t count = 0, chunks = 0, bits = 32;
};

namespace va {
namespace {

constexpr uint32_t kChunk = 2048;
constexpr uint32_t kGroup = 256;  // values that share a scale

struct Entry {
    const void *param, *grad, *first, *second;
    const float *first_scales, *second_scales, *master;
    void *out_param, *out_first, *out_second;
    float *out_first_scales, *out_second_scales, *out_master;
    uint64_t size;
    uint64_t place;  // of the first value among the list's, each tensor from a multiple of a group on
    float rate, decay;
    uint32_t kind, pad;
};

struct Hyper {
    const int64_t* device_step;
    const float* device_rate;
    const float* norm;
    int64_t step;
    uint64_t seed;
    double rate, log_beta1, log_beta2;
    float beta1, rest1, beta2, rest2, eps, decay, scale, max_norm;
};

// The numbers of a step, the same for every thread of a launch.
struct Step {
    float factor, beta1, rest1, beta2, rest2, eps, decay, inv_root;  // inv_root: 1 / sqrt(1 - b2^t)
    double rate, corrected;                                             // rate, rate / (1 - b1^t)
    uint64_t random;
    bool skip;
};

__device__ __forceinline__ uint64_t mixed(uint64_t z) {
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
    z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
    return z ^ (z >> 31);
}
constexpr uint64_t kGolden = 0x9E3779B97F4A7C15ull;

__device__ __forceinline__ Step step_of(const Hyper& h) {
    Step s;
    const int64_t t = h.device_step ? max(*h.device_step, int64_t(1)) : h.step;
    s.rate = h.device_rate ? double(*h.device_rate) : h.rate;
    s.corrected = s.rate / (1.0 - exp2(double(t) * h.log_beta1));
    s.inv_root = float(1.0 / sqrt(1.0 - exp2(double(t) * h.log_beta2)));
    s.beta1 = h.beta1, s.rest1 = h.rest1, s.beta2 = h.beta2, s.rest2 = h.rest2, s.eps = h.eps, s.decay = h.decay;
    s.factor = h.scale;
    s.skip = false;
    if (h.norm) {
        const float n = *h.norm * h.scale;
        s.skip = !(fabsf(n) < __builtin_inff());
        s.factor *= fminf(1.0f, h.max_norm / (n + 1e-6f));
    }
    s.random = mixed(h.seed + kGolden * uint64_t(t));
    return s;
}

template <class T, int N>
using Vec = T __attribute__((ext_vector_type(N)));

// Values at their elements' alignment, in global memory: pointers that come out of a table are else taken for any memory's, whose
// loads and stores wait for each other.
template <class V>
struct __attribute__((packed)) Loose {
    V v;
};
template <class V>
__device__ __forceinline__ V load(const void* p) {
    return ((const __attribute__((address_space(1))) Loose<V>*)p)->v;
}
template <class V>
__device__ __forceinline__ void store(void* p, V v) {
    ((__attribute__((address_space(1))) Loose<V>*)p)->v = v;
}

// N values from i on of an array of n; behind its end: zeros
template <class T, int N>
__device__ __forceinline__ Vec<T, N> get(const void* p, uint64_t i, uint64_t n) {
    const T* at = static_cast<const T*>(p) + i;
    if (i + N <= n) return load<Vec<T, N>>(at);
    Vec<T, N> v;
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = i + e < n ? load<T>(at + e) : T(0);
    return v;
}
template <class T, int N>
__device__ __forceinline__ void put(void* p, uint64_t i, uint64_t n, Vec<T, N> v) {
    T* at = static_cast<T*>(p) + i;
    if (i + N <= n) {
        store<Vec<T, N>>(at, v);
        return;
    }
#pragma unroll
    for (int e = 0; e < N; ++e)
        if (i + e < n) store<T>(at + e, v[e]);
}

// e4m3 codes of four values that e4m3 has
__device__ __forceinline__ uint32_t pack_fp8(const float* v) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
    return uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], w, true));
}
__device__ __forceinline__ void unpack_fp8(uint32_t w, float* v) {
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(int(w), false), b = __builtin_amdgcn_cvt_pk_f32_fp8(int(w), true);
    v[0] = a[0], v[1] = a[1], v[2] = b[0], v[3] = b[1];
}

// The largest magnitude of a group, whose 256 values 32 lanes hold eight each; by bits, so that NaN is the largest.
__device__ __forceinline__ uint32_t group_top(uint32_t top) {
#pragma unroll
    for (int d = 16; d; d >>= 1) top = max(top, uint32_t(__shfl_xor(int(top), d)));
    return top;
}

// Eight values of a group as codes; LEAST: they are not negative, and one that is not zero stays so.  A code has three binary digits behind
// its first, so a value's last 20 go: 16 random ones are added above the last four, and what carries goes up.  Below 2^-6 codes
// are whole multiples of 2^-9: with 2^-6 added their last 20 digits are those.
template <bool LEAST>
__device__ __forceinline__ void code(const float (&x)[8], const uint32_t (&random)[8], uint32_t (&words)[2], float& scale) {
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[e]) & 0x7FFFFFFFu);
    float t = __uint_as_float(group_top(top));
    t = t < 0x1p-100f ? 0.0f : t;  // (its reciprocal would overflow)
    const float inv = t == 0.0f ? 0.0f : 448.0f / t;
    scale = t / 448.0f;
    const float least = t > 0.0f ? 0x1p-9f : 0.0f;
    float z[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        float a = fminf(fabsf(x[e]) * inv, 448.0f);
        const float low = a < 0x1p-6f ? 0x1p-6f : 0.0f;
        a = __uint_as_float((__float_as_uint(a + low) + (random[e] << 4)) & 0xFFF00000u) - low;
        z[e] = LEAST ? fmaxf(a, x[e] > 0.0f ? least : 0.0f) : copysignf(a, x[e]);
    }
    words[0] = pack_fp8(z);
    words[1] = pack_fp8(z + 4);
}

__device__ __forceinline__ void update(const Step& s, float g, float& m, float& v, float& root) {
    g *= s.factor;
    m = s.beta1 * m + s.rest1 * g;
    v = s.beta2 * v + s.rest2 * (g * g);
    root = sqrtf(v);
}
template <bool MASTER, bool DIVIDES>
__device__ __forceinline__ float moved(const Step& s, float keep, float rate, float p, float m, float root) {
    // (the reciprocal is off by a unit in its last place at most, beside moments of four binary digits)
    const float d = root * s.inv_root + s.eps;
    float next = p * keep - rate * (DIVIDES ? m / d : m * __builtin_amdgcn_rcpf(d));
    // the parameter is its copy's rounding: not that of a sum with more digits (v_fma_mixlo_f16)
    if (MASTER) asm("" : "+v"(next));
    return next;
}

// One chunk of a tensor.  32-bit moments: a thread takes four values at two places, whole lines everywhere;
// 8-bit ones: eight values, so that 32 lanes hold a group.
template <int BITS, bool DIVIDES, class P, class G, bool MASTER>
__device__ __forceinline__ void chunk(const Entry& e, const Step& s, uint64_t at) {
    const uint64_t n = e.size;
    const float rate = float(s.corrected * double(e.rate)), keep = float(1.0 - s.rate * double(e.rate) * double(s.decay) * double(e.decay));
    if constexpr (BITS == 32) {
        Vec<P, 4> p[2];
        Vec<G, 4> g[2];
        Vec<float, 4> m[2], v[2], w[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const uint64_t i = at + u * 1024 + 4 * threadIdx.x;
            g[u] = get<G, 4>(e.grad, i, n);
            m[u] = get<float, 4>(e.first, i, n);
            v[u] = get<float, 4>(e.second, i, n);
            if constexpr (MASTER) w[u] = get<float, 4>(e.master, i, n);
            else p[u] = get<P, 4>(e.param, i, n);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const uint64_t i = at + u * 1024 + 4 * threadIdx.x;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                float mm = m[u][c], vv = v[u][c], root;
                update(s, float(g[u][c]), mm, vv, root);
                m[u][c] = mm;
                v[u][c] = vv;
                const float next = moved<MASTER, DIVIDES>(s, keep, rate, MASTER ? w[u][c] : float(p[u][c]), mm, root);
                if constexpr (MASTER) w[u][c] = next;
                p[u][c] = P(next);
            }
            put<P, 4>(e.out_param, i, n, p[u]);
            put<float, 4>(e.out_first, i, n, m[u]);
            put<float, 4>(e.out_second, i, n, v[u]);
            if constexpr (MASTER) put<float, 4>(e.out_master, i, n, w[u]);
        }
    } else {
        const uint64_t i = at + 8 * threadIdx.x, group = i / kGroup;
        const bool any = group * kGroup < n;  // the group is the tensor's
        const Vec<G, 8> g = get<G, 8>(e.grad, i, n);
        const Vec<uint8_t, 8> cm = get<uint8_t, 8>(e.first, i, n), cr = get<uint8_t, 8>(e.second, i, n);
        const float sm = any ? load<float>(e.first_scales + group) : 0.0f, sr = any ? load<float>(e.second_scales + group) : 0.0f;
        Vec<P, 8> p;
        Vec<float, 8> w;
        if constexpr (MASTER) w = get<float, 8>(e.master, i, n);
        else p = get<P, 8>(e.param, i, n);
        float m[8], r[8];
        const uint2 wm = __builtin_bit_cast(uint2, cm), wr = __builtin_bit_cast(uint2, cr);
        unpack_fp8(wm.x, m), unpack_fp8(wm.y, m + 4);
        unpack_fp8(wr.x, r), unpack_fp8(wr.y, r + 4);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            m[c] *= sm;
            r[c] *= sr;
            float v = r[c] * r[c];
            update(s, float(g[c]), m[c], v, r[c]);
            const float next = moved<MASTER, DIVIDES>(s, keep, rate, MASTER ? w[c] : float(p[c]), m[c], r[c]);
            if constexpr (MASTER) w[c] = next;
            p[c] = P(next);
        }
        put<P, 8>(e.out_param, i, n, p);
        if constexpr (MASTER) put<float, 8>(e.out_master, i, n, w);
        uint32_t rm[8], rr[8];
        uint64_t state = s.random + kGolden * ((e.place + i) / 2);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const uint64_t z = mixed(state += kGolden);
            rm[2 * c] = uint32_t(z) & 0xFFFFu, rr[2 * c] = uint32_t(z) >> 16;
            rm[2 * c + 1] = uint32_t(z >> 32) & 0xFFFFu, rr[2 * c + 1] = uint32_t(z >> 48);
        }
        // (behind a tensor's end m and r are zero: they are no group's largest)
        uint32_t words[2];
        float scale;
        code<false>(m, rm, words, scale);
        put<uint8_t, 8>(e.out_first, i, n, __builtin_bit_cast(Vec<uint8_t, 8>, make_uint2(words[0], words[1])));
        const bool writes = any && threadIdx.x % 32 == 0;
        if (writes) store<float>(e.out_first_scales + group, scale);
        code<true>(r, rr, words, scale);
        put<uint8_t, 8>(e.out_second, i, n, __builtin_bit_cast(Vec<uint8_t, 8>, make_uint2(words[0], words[1])));
        if (writes) store<float>(e.out_second_scales + group, scale);
    }
}

// the values of a step that is not taken
__device__ __forceinline__ void carry(const void* from, void* to, uint64_t at, uint64_t n) {
    if (from == to) return;
    for (uint64_t i = at + threadIdx.x; i < n; i += 256) static_cast<uint8_t*>(to)[i] = static_cast<const uint8_t*>(from)[i];
}

enum Kind : uint32_t { F32 = 0, F16 = 1, BF16 = 2, F16_G32 = 3, BF16_G32 = 4, WITH_MASTER = 8 };

// Workgroups that a CU holds, by their registers, and that a launch has for it (8-bit moments in 64 registers spill: 568, not 541 us).
constexpr uint32_t kPerCu(int bits) { return bits == 32 ? 8 : 7; }

template <int BITS, bool DIVIDES>
__global__ __launch_bounds__(256, kPerCu(BITS)) void adamw_kernel(const Entry* __restrict__ entries, const uint32_t* __restrict__ first, uint32_t count,
                                                     uint32_t chunks, Hyper h) {
    const uint32_t c0 = uint32_t(uint64_t(chunks) * blockIdx.x / gridDim.x), c1 = uint32_t(uint64_t(chunks) * (blockIdx.x + 1) / gridDim.x);
    if (c0 >= c1) return;
    // the tensor that holds chunk c0: the whole wave looks at 64 tensors between the bounds at a time
    uint32_t lo = 0, hi = count;  // first[lo] <= c0; the answer lies in [lo, hi)
    while (hi - lo > 1) {
        const uint32_t width = (hi - lo + 63) / 64, l = lo + (threadIdx.x & 63) * width;
        const uint32_t c = uint32_t(__popcll(__ballot(l < hi && first[l] <= c0)));
        lo = __builtin_amdgcn_readfirstlane(lo + (c - 1) * width);
        hi = __builtin_amdgcn_readfirstlane(min(hi, lo + width));
    }
    uint32_t i = lo, next = i + 1 < count ? first[i + 1] : chunks;
    Entry e = entries[i];
    uint32_t begin = first[i];
    const Step s = step_of(h);
    for (uint32_t c = c0; c < c1; ++c) {
        if (c >= next) {  // (no tensor of a list is empty)
            ++i;
            e = entries[i];
            begin = next;
            next = i + 1 < count ? first[i + 1] : chunks;
        }
        const uint64_t at = uint64_t(c - begin) * kChunk;
        if (s.skip) {
            const uint64_t end = min(at + kChunk, e.size);
            const uint32_t ps = (e.kind & 7) == F32 ? 4 : 2, ms = BITS / 8;
            carry(e.param, e.out_param, at * ps, end * ps);
            carry(e.first, e.out_first, at * ms, end * ms);
            carry(e.second, e.out_second, at * ms, end * ms);
            if (e.kind & WITH_MASTER) carry(e.master, e.out_master, at * 4, end * 4);
            if (BITS == 8) {
                const uint64_t g0 = at / kGroup, g1 = (end + kGroup - 1) / kGroup;
                carry(e.first_scales, e.out_first_scales, g0 * 4, g1 * 4);
                carry(e.second_scales, e.out_second_scales, g0 * 4, g1 * 4);
            }
            continue;
        }
        switch (e.kind) {
            case F32: chunk<BITS, DIVIDES, float, float, false>(e, s, at); break;
            case F16: chunk<BITS, DIVIDES, _Float16, _Float16, false>(e, s, at); break;
            case BF16: chunk<BITS, DIVIDES, __bf16, __bf16, false>(e, s, at); break;
            case F16_G32: chunk<BITS, DIVIDES, _Float16, float, false>(e, s, at); break;
            case BF16_G32: chunk<BITS, DIVIDES, __bf16, float, false>(e, s, at); break;
            case F16 | WITH_MASTER: chunk<BITS, DIVIDES, _Float16, _Float16, true>(e, s, at); break;
            case BF16 | WITH_MASTER: chunk<BITS, DIVIDES, __bf16, __bf16, true>(e, s, at); break;
            case F16_G32 | WITH_MASTER: chunk<BITS, DIVIDES, _Float16, float, true>(e, s, at); break;
            case BF16_G32 | WITH_MASTER: chunk<BITS, DIVIDES, __bf16, float, true>(e, s, at); break;
        }
    }
}

struct Range {
    uintptr_t begin, end;
};

va_status create(va_context* ctx, const va_adamw_tensor* t, uint32_t count, uint32_t bits, va_adamw_list** out) {
    std::vector<Entry> entries;
    std::vector<uint32_t> first;
    std::vector<Range> written;
    entries.reserve(count), first.reserve(count), written.reserve(size_t(count) * 6);
    uint64_t chunks = 0, place = 0;
    const auto range = [](const void* p, uint64_t bytes) { return Range{reinterpret_cast<uintptr_t>(p), reinterpret_cast<uintptr_t>(p) + uintptr_t(bytes)}; };
    const auto aligned = [](const void* p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; };
    struct Pair {
        const void* in;
        void* out;
        uint64_t bytes;
        uint32_t align;
    };
    // (param is read only where there is no master)
    const auto pairs = [bits](const Entry& e, Pair (&p)[6]) {
        const uint32_t ps = (e.kind & 7) == F32 ? 4 : 2, ms = bits / 8;
        const uint64_t scales = bits == 8 ? 4 * ((e.size + kGroup - 1) / kGroup) : 0;
        p[0] = {e.param, e.out_param, e.size * ps, ps};
        p[1] = {e.first, e.out_first, e.size * ms, ms};
        p[2] = {e.second, e.out_second, e.size * ms, ms};
        p[3] = {e.first_scales, e.out_first_scales, scales, 4};
        p[4] = {e.second_scales, e.out_second_scales, scales, 4};
        p[5] = {e.master, e.out_master, e.kind & WITH_MASTER ? 4 * e.size : 0, 4};
    };
    for (uint32_t i = 0; i < count; ++i) {
        const va_adamw_tensor& a = t[i];
        const bool same = a.grad_dtype == a.param_dtype;
        VA_REQUIRE(ctx, a.param_dtype >= VA_DTYPE_F32 && a.param_dtype <= VA_DTYPE_BF16 && (same || a.grad_dtype == VA_DTYPE_F32),
                   "va_adamw_list_create: tensor %u: parameters of type %d with gradients of type %d", i, int(a.param_dtype), int(a.grad_dtype));
        VA_REQUIRE(ctx, std::isfinite(a.rate_factor) && a.rate_factor >= 0.0f && std::isfinite(a.decay_factor) && a.decay_factor >= 0.0f,
                   "va_adamw_list_create: tensor %u: factors must be finite and not negative", i);
        VA_REQUIRE(ctx, a.size < 1ull << 40, "va_adamw_list_create: tensor %u: too many values", i);
        VA_REQUIRE(ctx, !a.master || a.param_dtype != VA_DTYPE_F32, "va_adamw_list_create: tensor %u: fp32 parameters need no copy in fp32", i);
        const bool master = a.master != nullptr;
        if (!a.size) continue;
        Entry e{};
        e.param = a.param, e.grad = a.grad, e.first = a.first, e.second = a.second, e.first_scales = a.first_scales, e.second_scales = a.second_scales, e.master = a.master;
        e.out_param = a.out_param, e.out_first = a.out_first, e.out_second = a.out_second;
        e.out_first_scales = a.out_first_scales, e.out_second_scales = a.out_second_scales, e.out_master = a.out_master;
        e.size = a.size, e.place = place, e.rate = a.rate_factor, e.decay = a.decay_factor;
        e.kind = uint32_t(a.param_dtype) + (same ? 0u : 2u) + (master ? uint32_t(WITH_MASTER) : 0u);
        Pair p[6];
        pairs(e, p);
        for (int k = 0; k < 6; ++k) {
            if (!p[k].bytes) continue;
            VA_REQUIRE(ctx, p[k].in && p[k].out, "va_adamw_list_create: tensor %u: a pointer is NULL", i);
            VA_REQUIRE(ctx, aligned(p[k].in, p[k].align) && aligned(p[k].out, p[k].align), "va_adamw_list_create: tensor %u is not aligned to its type", i);
            written.push_back(range(p[k].out, p[k].bytes));
        }
        VA_REQUIRE(ctx, a.grad, "va_adamw_list_create: tensor %u: a pointer is NULL", i);
        VA_REQUIRE(ctx, aligned(a.grad, a.grad_dtype == VA_DTYPE_F32 ? 4 : 2), "va_adamw_list_create: tensor %u is not aligned to its type", i);
        entries.push_back(e);
        first.push_back(uint32_t(chunks));
        chunks += (a.size + kChunk - 1) / kChunk;
        VA_REQUIRE(ctx, chunks < 1ull << 32, "va_adamw_list_create: too many values");
        place += (a.size + kGroup - 1) / kGroup * kGroup;
    }
    // What is written is nothing else that is written, and nothing that is read but what it replaces.
    std::sort(written.begin(), written.end(), [](const Range& a, const Range& b) { return a.begin < b.begin; });
    for (size_t k = 1; k < written.size(); ++k) VA_REQUIRE(ctx, written[k - 1].end <= written[k].begin, "va_adamw_list_create: tensors that are written overlap");
    const auto hits = [&](const Range& r) {
        // (they are apart, so their ends are in order too)
        const auto at = std::upper_bound(written.begin(), written.end(), r.begin, [](uintptr_t b, const Range& w) { return b < w.end; });
        return at != written.end() && at->begin < r.end;
    };
    for (const Entry& e : entries) {
        Pair p[6];
        pairs(e, p);
        const uint32_t gs = (e.kind & 7) == F16 || (e.kind & 7) == BF16 ? 2 : 4;
        VA_REQUIRE(ctx, !hits(range(e.grad, e.size * gs)), "va_adamw_list_create: a gradient is written");
        for (int k = 0; k < 6; ++k)
            VA_REQUIRE(ctx, !p[k].bytes || p[k].in == p[k].out || !hits(range(p[k].in, p[k].bytes)), "va_adamw_list_create: what is read of a tensor is written elsewhere");
    }
    va_adamw_list* l = new va_adamw_list();
    l->device = ctx->device;
    l->count = uint32_t(entries.size()), l->chunks = uint32_t(chunks), l->bits = bits;
    if (l->count) {
        const size_t eb = entries.size() * sizeof(Entry), fb = first.size() * sizeof(uint32_t);
        hipError_t r = hipMalloc(&l->table, eb + fb);
        if (r == hipSuccess) r = hipMemcpy(l->table, entries.data(), eb, hipMemcpyHostToDevice);
        if (r == hipSuccess) r = hipMemcpy(static_cast<char*>(l->table) + eb, first.data(), fb, hipMemcpyHostToDevice);
        if (r != hipSuccess) {
            (void)hipGetLastError();
            if (l->table) (void)hipFree(l->table);
            delete l;
            return fail(ctx, r == hipErrorOutOfMemory ? VA_ERR_OOM : VA_ERR_HIP, "va_adamw_list_create: %s", hipGetErrorString(r));
        }
    }
    *out = l;
    return VA_OK;
}

}  // namespace
}  // namespace va

using namespace va;

extern "C" {

va_status va_adamw_list_create(va_context* ctx, const va_adamw_tensor* tensors, uint32_t count, uint32_t moment_bits, va_adamw_list** out) {
    if (!ctx) return VA_ERR_INVALID_ARG;
    VA_REQUIRE(ctx, out && (tensors || !count), "va_adamw_list_create: NULL pointer");
    *out = nullptr;
    VA_REQUIRE(ctx, moment_bits == 8 || moment_bits == 32, "va_adamw_list_create: moments of %u bits (8 or 32)", moment_bits);
    DeviceGuard guard(ctx->device);
    // (before anything is allocated: what a capture forbids would end it, and be an error of the caller's next calls)
    hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
    VA_CHECK_HIP(ctx, hipStreamIsCapturing(ctx->stream, &capture));
    VA_REQUIRE(ctx, capture == hipStreamCaptureStatusNone, "va_adamw_list_create: the context's stream is being captured");
    try {
        return create(ctx, tensors, count, moment_bits, out);
    } catch (const std::bad_alloc&) {
        return fail(ctx, VA_ERR_OOM, "va_adamw_list_create: out of host memory");
    }
}

va_status va_adamw_list_destroy(va_adamw_list* list) {
    if (!list) return VA_ERR_INVALID_ARG;
    DeviceGuard guard(list->device);
    if (list->table) (void)hipFree(list->table);  // (waits for the device)
    delete list;
    return VA_OK;
}

va_status va_adamw_step(va_context* ctx, const va_adamw_list* l, const va_adamw_params* p) {
    if (!ctx) return VA_ERR_INVALID_ARG;
    VA_REQUIRE(ctx, l && p, "va_adamw_step: NULL pointer");
    VA_REQUIRE(ctx, l->device == ctx->device, "va_adamw_step: the list is on device %d, the context on %d", l->device, ctx->device);
    VA_REQUIRE(ctx, p->beta1 >= 0.0 && p->beta1 < 1.0 && p->beta2 >= 0.0 && p->beta2 < 1.0, "va_adamw_step: beta1 and beta2 must lie in [0, 1)");
    VA_REQUIRE(ctx, std::isfinite(p->epsilon) && p->epsilon >= 0.0 && std::isfinite(p->weight_decay) && p->weight_decay >= 0.0,
               "va_adamw_step: epsilon and weight_decay must be finite and not negative");
    VA_REQUIRE(ctx, p->device_step || p->step >= 1, "va_adamw_step: steps count from 1");
    VA_REQUIRE(ctx, p->device_rate || (std::isfinite(p->rate) && p->rate >= 0.0), "va_adamw_step: the rate must be finite and not negative");
    VA_REQUIRE(ctx, std::isfinite(p->grad_scale) && p->grad_scale >= 0.0, "va_adamw_step: grad_scale must be finite and not negative");
    VA_REQUIRE(ctx, !p->grad_norm || p->max_norm >= 0.0, "va_adamw_step: max_norm must not be negative or NaN");
    if (!l->count) return VA_OK;
    DeviceGuard guard(ctx->device);
    Hyper h;
    h.device_step = p->device_step, h.device_rate = p->device_rate, h.norm = p->grad_norm;
    h.step = p->step, h.seed = p->seed, h.rate = p->rate;
    h.log_beta1 = std::log2(p->beta1), h.log_beta2 = std::log2(p->beta2);
    h.beta1 = float(p->beta1), h.rest1 = float(1.0 - p->beta1), h.beta2 = float(p->beta2), h.rest2 = float(1.0 - p->beta2);
    h.eps = float(p->epsilon), h.decay = float(p->weight_decay), h.scale = float(p->grad_scale), h.max_norm = float(p->max_norm);
    const Entry* entries = static_cast<const Entry*>(l->table);
    const uint32_t* first = reinterpret_cast<const uint32_t*>(entries + l->count);
    const uint32_t grid = std::min(l->chunks, kPerCu(int(l->bits)) * uint32_t(ctx->num_cus));
    // The divisor is epsilon at least and 2^91 more at most.  Of 8-bit moments a reciprocal takes its place (536, not 580 us for 50 tensors of
    // 228M values) where the instruction takes it: it has neither subnormal operands nor such results.  32-bit ones wait for
    // memory and gain nothing (218 and 219 us for 290 tensors).
    if (l->bits == 32) adamw_kernel<32, true><<<dim3(grid), dim3(256), 0, ctx->stream>>>(entries, first, l->count, l->chunks, h);
    else if (h.eps < 0x1p-126f || h.eps > 0x1p100f) adamw_kernel<8, true><<<dim3(grid), dim3(256), 0, ctx->stream>>>(entries, first, l->count, l->chunks, h);
    else adamw_kernel<8, false><<<dim3(grid), dim3(256), 0, ctx->stream>>>(entries, first, l->count, l->chunks, h);
    VA_CHECK_LAUNCH(ctx);
    return VA_OK;
}

}  // extern "C"
