// va_rmsnorm.hip — root-mean-square norm of rows with the residual's addition, its backward pass,
// and the output in 8 bits with scales.
//
//   r = x + residual     i = 1 / sqrt(mean_d r_d^2 + eps)     y_d = r_d i w_d
//   codes: s = max |y| over a group / M (M = 127 for int8, 448 for fp8 e4m3), code = round(y / s)
//   dx = i (w dy - n mean_d(w dy n)) + dresidual,  dw = sum_t dy n,  n = r i
//
// Bound by memory: every operand is read once and every result written once.  A row is held in registers by one
// wave (D <= 2048) or one workgroup (D <= 8192), 16 bytes a lane and chunk (8-bit outputs: 8 values, so that a
// group's largest value is a few lane exchanges away).  Longer rows are read twice, the second time from cache.  Values are loaded 16 bytes at a time whatever their
// alignment (global loads on gfx950 need none beyond the element's); a row's last, partial chunk element by
// element.  A row's sums are fp32 where it is held in registers (a lane's chain of at most 32 values, then a tree) and fp64
// in longer rows and where the squares leave fp32's range; the weight's gradient is a chain of fp32 over the rows of each share, then a tree.
//
// Measured: 65,536 x 1536 bf16 with residual to int8 by groups 156 us = 4.5 TB/s, and back 53 us = 5.7 TB/s; 10,007
// x 513 fp32 forward 18 us and backward 18 + 4 us (4.6 TB/s each); 37,289 x 768 bf16 forward 44 us = 5.2 TB/s.  One
// row: 5 us, the launch.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "va_internal.hpp"

namespace va {
namespace {

template <int E>
using F = float __attribute__((ext_vector_type(E)));  // E consecutive values of a row
using f32x8 = F<8>;

enum Out : int { OUT_SAME = 0, OUT_INT8 = 1, OUT_FP8 = 2 };

template <int DT>
struct Elem;
template <>
struct Elem<VA_DTYPE_F32> {
    using T = float;
};
template <>
struct Elem<VA_DTYPE_F16> {
    using T = _Float16;
};
template <>
struct Elem<VA_DTYPE_BF16> {
    using T = __bf16;
};
template <int DT>
using ElemT = typename Elem<DT>::T;

// E consecutive values with no alignment beyond the element's
template <class T, int E>
using Vec = T __attribute__((ext_vector_type(E), aligned(sizeof(T))));

// values [d, d + E) of a row, zeros from D on
template <int E, class T>
__device__ __forceinline__ Vec<T, E> raw(const T* row, uint32_t d, uint32_t D) {
    if (d + E <= D) return *reinterpret_cast<const Vec<T, E>*>(row + d);
    Vec<T, E> v;
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = d + e < D ? row[d + e] : T(0.0f);
    return v;
}
template <int E, class T>
__device__ __forceinline__ F<E> load(const T* row, uint32_t d, uint32_t D) {
    return __builtin_convertvector(raw<E>(row, d, D), F<E>);
}
template <int E, class T>
__device__ __forceinline__ void store(T* row, uint32_t d, uint32_t D, F<E> v) {
    typedef Vec<T, E> V;
    const V o = __builtin_convertvector(v, V);
    if (d + E <= D) {
        *reinterpret_cast<V*>(row + d) = o;
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (d + e < D) row[d + e] = o[e];
    }
}

template <int N, class S>
__device__ __forceinline__ S lanes_sum(S v) {
#pragma unroll
    for (int d = 1; d < N; d <<= 1) v += __shfl_xor(v, d);
    return v;
}
// the larger of two magnitudes; NaN stays
__device__ __forceinline__ float top(float a, float b) { return b > a || b != b ? b : a; }

// a sum over the row's threads (one wave, or the workgroup's four)
template <int WPR, class S>
__device__ __forceinline__ S row_sum(S v, S* part) {
    v = lanes_sum<64>(v);
    if constexpr (WPR > 1) {
        __syncthreads();  // the previous row's sums are read
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
        __syncthreads();
        v = (part[0] + part[1]) + (part[2] + part[3]);
    }
    return v;
}
template <int WPR>
__device__ __forceinline__ float row_top(float v, float* part) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v = top(v, __shfl_xor(v, d));
    if constexpr (WPR > 1) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
        __syncthreads();
        v = top(top(part[0], part[1]), top(part[2], part[3]));
    }
    return v;
}

struct RmsArgs {
    const void* x;
    const void* residual;  // or nullptr
    const void* weight;
    void* out_residual;  // or nullptr
    float* inverse;      // or nullptr
    void* out;
    float* scales;  // 8-bit outputs without a given scale
    uint64_t ldx, ldr, ldro, ldo;
    uint32_t t0, T, D, group, groups;  // the launch's first row; group 0: the row
    float eps, given;              // given > 0: the scale
};

// The codes of y / s (0 where s is), the quotient rounded to fp32 and then to the nearest code.  A division a value: by the
// reciprocal, a quotient next to a midpoint may come out on its other side (65,536 x 1536 to int8 by groups of 128 144 us
// that way and 156 divided, by rows 130 and 134).
__device__ __forceinline__ uint2 codes8(f32x8 y, float s, bool fp8) {
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float z[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            z[e] = s == 0.0f ? 0.0f : y[4 * h + e] / s;
            const float most = fp8 ? 448.0f : 127.0f;
            z[e] = z[e] != z[e] ? z[e] : fminf(fmaxf(z[e], -most), most);
        }
        if (fp8) {
            int p = __builtin_amdgcn_cvt_pk_fp8_f32(z[0], z[1], 0, false);
            w[h] = uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(z[2], z[3], p, true));
        } else {
            w[h] = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) w[h] |= (uint32_t(z[e] == z[e] ? int(rintf(z[e])) : 0) & 0xFFu) << (8 * e);
        }
    }
    return make_uint2(w[0], w[1]);
}
__device__ __forceinline__ void store_codes(uint8_t* row, uint32_t d, uint32_t D, uint2 c) {
    if (d + 8 <= D) {
        typedef uint32_t u32x2 __attribute__((ext_vector_type(2), aligned(1)));
        *reinterpret_cast<u32x2*>(row + d) = u32x2{c.x, c.y};
    } else {
        for (int e = 0; e < 8; ++e)
            if (d + e < D) row[d + e] = uint8_t((e < 4 ? c.x >> (8 * e) : c.y >> (8 * (e - 4))) & 0xFFu);
    }
}

// WPR waves a row; C chunks of E values a lane in registers, or (C == 0) any number, read again
template <int DT, int OUT, int WPR, int C>
__global__ __launch_bounds__(256) void rms_norm_kernel(RmsArgs a) {
    using T = ElemT<DT>;
    constexpr int NT = 64 * WPR, E = OUT == OUT_SAME ? 16 / int(sizeof(T)) : 8;
    __shared__ float part[4];
    __shared__ double wide[4];
    const uint32_t t = a.t0 + (WPR == 1 ? blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x);
    if (t >= a.T) return;  // (a whole wave, or the workgroup)
    const uint32_t tid = WPR == 1 ? threadIdx.x & 63 : threadIdx.x;
    const T* x = static_cast<const T*>(a.x) + t * a.ldx;
    const T* res = a.residual ? static_cast<const T*>(a.residual) + t * a.ldr : nullptr;
    const T* w = static_cast<const T*>(a.weight);
    T* ro = a.out_residual ? static_cast<T*>(a.out_residual) + t * a.ldro : nullptr;
    const uint32_t D = a.D, chunks = C ? C : (D + E * NT - 1) / (E * NT);
    auto sum_of = [&](uint32_t d) {
        F<E> v = load<E>(x, d, D);
        if (res) v += load<E>(res, d, D);
        return v;
    };
    F<E> r[C ? C : 1];
    double ds = 0.0;
    const auto add = [&](F<E> v) {
#pragma unroll
        for (int e = 0; e < E; ++e) ds = fma(double(v[e]), double(v[e]), ds);
    };
    const auto inverse = [&] { return float(1.0 / sqrt(row_sum<WPR>(ds, wide) / double(D) + double(a.eps))); };
    float inv;
    if constexpr (C > 0) {
        float ss = 0.0f;
#pragma unroll
        for (int c = 0; c < C; ++c) r[c] = sum_of((c * NT + tid) * E);
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int e = 0; e < E; ++e) ss = fmaf(r[c][e], r[c][e], ss);
        ss = row_sum<WPR>(ss, part);
        if (ss > 0x1p-100f && ss < 0x1p126f) {
            inv = 1.0f / sqrtf(ss / float(D) + a.eps);
        } else {  // (the whole row's threads) squares near or past the ends of fp32
#pragma unroll
            for (int c = 0; c < C; ++c) add(r[c]);
            inv = inverse();
        }
    } else {
        for (uint32_t c = 0; c < chunks; ++c) add(sum_of((c * NT + tid) * E));
        inv = inverse();
    }
    if (a.inverse && tid == 0) a.inverse[t] = inv;

    // y of a chunk, the new residual stored on the way (once)
    auto y_of = [&](uint32_t d, F<E> v, bool keep) {
        if (ro && keep) store<E>(ro, d, D, v);
        return v * inv * load<E>(w, d, D);
    };
    if constexpr (OUT == OUT_SAME) {
        T* o = static_cast<T*>(a.out) + t * a.ldo;
        if constexpr (C > 0) {
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const uint32_t d = (c * NT + tid) * E;
                store<E>(o, d, D, y_of(d, r[c], true));
            }
        } else {
            for (uint32_t c = 0; c < chunks; ++c) {
                const uint32_t d = (c * NT + tid) * E;
                store<E>(o, d, D, y_of(d, sum_of(d), true));
            }
        }
    } else {
        constexpr bool fp8 = OUT == OUT_FP8;
        constexpr float most = fp8 ? 448.0f : 127.0f;
        uint8_t* o = static_cast<uint8_t*>(a.out) + t * a.ldo;
        auto biggest = [&](F<E> y) {
            float m = fabsf(y[0]);
#pragma unroll
            for (int e = 1; e < E; ++e) m = top(m, fabsf(y[e]));
            return m;
        };
        // the scale of a whole row: one pass over y first
        float s = a.given;
        if (a.group == 0 && !(a.given > 0.0f)) {
            float m = 0.0f;
            if constexpr (C > 0) {
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    const uint32_t d = (c * NT + tid) * E;
                    r[c] = y_of(d, r[c], true);
                    m = top(m, biggest(r[c]));
                }
            } else {
                for (uint32_t c = 0; c < chunks; ++c) {
                    const uint32_t d = (c * NT + tid) * E;
                    m = top(m, biggest(y_of(d, sum_of(d), false)));
                }
            }
            s = row_top<WPR>(m, part) / most;
            if (tid == 0) a.scales[t] = s;
        }
        auto emit = [&](uint32_t d, F<E> y) {
            float sc = s;
            if (a.group) {
                float m = biggest(y);
                for (uint32_t k = 1; k < a.group / 8; k <<= 1) m = top(m, __shfl_xor(m, int(k)));
                sc = m / most;
                if (d < D && d % a.group == 0) a.scales[uint64_t(t) * a.groups + d / a.group] = sc;
            }
            store_codes(o, d, D, codes8(y, sc, fp8));
        };
        if constexpr (C > 0) {
            const bool have = a.group == 0 && !(a.given > 0.0f);  // r holds y
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const uint32_t d = (c * NT + tid) * E;
                emit(d, have ? r[c] : y_of(d, r[c], true));
            }
        } else {
            for (uint32_t c = 0; c < chunks; ++c) {
                const uint32_t d = (c * NT + tid) * E;
                emit(d, y_of(d, sum_of(d), true));
            }
        }
    }
}

// out = code scale, 8 values a thread
template <int DT>
__global__ __launch_bounds__(256) void rms_dequantize_kernel(const uint8_t* __restrict__ codes, const float* __restrict__ scales, uint64_t ldc,
                                                             uint64_t i0, uint32_t T, uint32_t D, uint32_t group, uint32_t groups, float given, bool fp8,
                                                             ElemT<DT>* __restrict__ out, uint64_t ldo) {
    const uint32_t per = (D + 7) / 8;
    const uint64_t i = i0 + uint64_t(blockIdx.x) * 256 + threadIdx.x;
    if (i >= uint64_t(T) * per) return;
    const uint32_t t = uint32_t(i / per), d = uint32_t(i % per) * 8;
    const float s = given > 0.0f ? given : scales[uint64_t(t) * groups + (group ? d / group : 0)];
    const uint8_t* c = codes + t * ldc + d;
    uint32_t w[2] = {0, 0};
    if (d + 8 <= D) {
        __builtin_memcpy(w, c, 8);
    } else {
        for (int e = 0; e < 8; ++e)
            if (d + e < D) w[e >> 2] |= uint32_t(c[e]) << (8 * (e & 3));
    }
    f32x8 v;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if (fp8) {
            v[4 * h] = __builtin_amdgcn_cvt_f32_fp8(int(w[h]), 0);
            v[4 * h + 1] = __builtin_amdgcn_cvt_f32_fp8(int(w[h]), 1);
            v[4 * h + 2] = __builtin_amdgcn_cvt_f32_fp8(int(w[h]), 2);
            v[4 * h + 3] = __builtin_amdgcn_cvt_f32_fp8(int(w[h]), 3);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[4 * h + e] = float(int8_t(w[h] >> (8 * e)));
        }
    }
    store<8>(out + t * ldo, d, D, f32x8(v * s));
}

// ---- backward ------------------------------------------------------------------------------------
struct RmsGradArgs {
    const void* grad;
    const void* r;  // the summed rows of the forward pass
    const void* weight;
    const void* grad_residual;  // or nullptr
    const float* inverse;
    void* out;    // dx, or nullptr
    float* part;  // [workgroups][D] shares of dw, or nullptr
    uint64_t ldg, ldr, ldgr, ldo;
    uint32_t T, D;
};

// A wave (or workgroup) takes rows in turn; the next row's loads are in flight while a row is worked on, and dw's
// shares stay in registers.  Rows of up to 64 E C WPR values.
template <int DT, int WPR, int C>
__global__ __launch_bounds__(256) void rms_grad_kernel(RmsGradArgs a) {
    using T = ElemT<DT>;
    constexpr int NT = 64 * WPR, E = 16 / int(sizeof(T));
    constexpr int ROWS = 4 / WPR;
    using V = Vec<T, E>;
    __shared__ float part[4];
    __shared__ F<E> join[WPR == 1 ? 256 : 1];
    const uint32_t tid = WPR == 1 ? threadIdx.x & 63 : threadIdx.x;
    const uint32_t D = a.D, step = gridDim.x * ROWS;
    const T* w = static_cast<const T*>(a.weight);
    F<E> dw[C], wv[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        dw[c] = F<E>(0.0f);
        wv[c] = load<E>(w, (c * NT + tid) * E, D);
    }
    struct Row {
        V g[C], r[C], gr[C];
        float inv;
    } next;
    auto fetch = [&](uint32_t t) {
        const T* g = static_cast<const T*>(a.grad) + t * a.ldg;
        const T* r = static_cast<const T*>(a.r) + t * a.ldr;
        const T* gr = static_cast<const T*>(a.grad_residual) + t * a.ldgr;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const uint32_t d = (c * NT + tid) * E;
            next.g[c] = raw<E>(g, d, D);
            next.r[c] = raw<E>(r, d, D);
            if (a.grad_residual) next.gr[c] = raw<E>(gr, d, D);
        }
        next.inv = a.inverse[t];
    };
    uint32_t t = blockIdx.x * ROWS + (WPR == 1 ? threadIdx.x >> 6 : 0);
    if (t < a.T) fetch(t);
    while (t < a.T) {
        const Row now = next;
        const uint32_t row = t;
        t += step;
        if (t < a.T) fetch(t);
        float along = 0.0f;
        F<E> gv[C], nv[C];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            gv[c] = __builtin_convertvector(now.g[c], F<E>);
            nv[c] = __builtin_convertvector(now.r[c], F<E>) * now.inv;
#pragma unroll
            for (int e = 0; e < E; ++e) along = fmaf(gv[c][e] * wv[c][e], nv[c][e], along);
            dw[c] += gv[c] * nv[c];
        }
        along = row_sum<WPR>(along, part) / float(D);
        if (!a.out) continue;
        T* o = static_cast<T*>(a.out) + row * a.ldo;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            F<E> v = (gv[c] * wv[c] - nv[c] * along) * now.inv;
            if (a.grad_residual) v += __builtin_convertvector(now.gr[c], F<E>);
            store<E>(o, (c * NT + tid) * E, D, v);
        }
    }
    if (!a.part) return;
    float* o = a.part + uint64_t(blockIdx.x) * D;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const uint32_t d = (c * NT + tid) * E;
        F<E> v = dw[c];
        if constexpr (WPR == 1) {
            __syncthreads();
            join[threadIdx.x] = v;
            __syncthreads();
            if (threadIdx.x >= 64) continue;
            v = (join[tid] + join[tid + 64]) + (join[tid + 128] + join[tid + 192]);
        }
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (d + e < D) o[d + e] = v[e];
    }
}

// dx of longer rows: a workgroup takes rows in turn and reads each twice, the second time from cache
template <int DT>
__global__ __launch_bounds__(256) void rms_long_grad_kernel(RmsGradArgs a) {
    using T = ElemT<DT>;
    constexpr int E = 16 / int(sizeof(T));
    __shared__ double part[4];
    const uint32_t D = a.D;
    const T* w = static_cast<const T*>(a.weight);
    for (uint32_t t = blockIdx.x; t < a.T; t += gridDim.x) {
        const T* g = static_cast<const T*>(a.grad) + t * a.ldg;
        const T* r = static_cast<const T*>(a.r) + t * a.ldr;
        const T* gr = a.grad_residual ? static_cast<const T*>(a.grad_residual) + t * a.ldgr : nullptr;
        T* o = static_cast<T*>(a.out) + t * a.ldo;
        const float inv = a.inverse[t];
        double sum = 0.0;
        for (uint32_t d = threadIdx.x * E; d < D; d += 256 * E) {
            const F<E> gg = load<E>(g, d, D), nn = load<E>(r, d, D) * inv, wc = load<E>(w, d, D);
#pragma unroll
            for (int e = 0; e < E; ++e) sum = fma(double(gg[e] * wc[e]), double(nn[e]), sum);
        }
        const float along = float(row_sum<4>(sum, part) / double(D));
        for (uint32_t d = threadIdx.x * E; d < D; d += 256 * E) {
            const F<E> gg = load<E>(g, d, D), nn = load<E>(r, d, D) * inv;
            F<E> v = (gg * load<E>(w, d, D) - nn * along) * inv;
            if (gr) v += load<E>(gr, d, D);
            store<E>(o, d, D, v);
        }
    }
}

// dw's shares of long rows: a workgroup takes 2048 columns of every gridDim.y-th row
template <int DT>
__global__ __launch_bounds__(256) void rms_weight_grad_kernel(RmsGradArgs a) {
    using T = ElemT<DT>;
    const uint32_t d = (blockIdx.x * 256 + threadIdx.x) * 8;
    f32x8 dw(0.0f);
    for (uint32_t t = blockIdx.y; t < a.T; t += gridDim.y)
        dw += load<8>(static_cast<const T*>(a.grad) + t * a.ldg, d, a.D) * (load<8>(static_cast<const T*>(a.r) + t * a.ldr, d, a.D) * a.inverse[t]);
    for (int e = 0; e < 8; ++e)
        if (d + e < a.D) a.part[uint64_t(blockIdx.y) * a.D + d + e] = dw[e];
}

// out[d] = sum of the shares, in a fixed order: 64 columns a workgroup, 16 groups of shares
template <int DT>
__global__ __launch_bounds__(1024) void rms_weight_sum_kernel(const float* __restrict__ part, uint32_t shares, uint32_t D, ElemT<DT>* __restrict__ out) {
    __shared__ float s[16][64];
    const uint32_t c = threadIdx.x & 63, g = threadIdx.x >> 6;
    for (uint32_t d0 = blockIdx.x * 64; d0 < D; d0 += gridDim.x * 64) {
        const uint32_t d = d0 + c;
        float v = 0.0f;
        if (d < D)
#pragma unroll 8
            for (uint32_t i = g; i < shares; i += 16) v += part[uint64_t(i) * D + d];
        s[g][c] = v;
        __syncthreads();
        if (g == 0 && d < D) {
            for (int i = 1; i < 16; ++i) v += s[i][c];
            out[d] = ElemT<DT>(v);
        }
        __syncthreads();  // the groups' sums are read
    }
}

// ---- host ------------------------------------------------------------------------------------------
// f(waves a row, chunks) for rows of D values, E a lane and chunk
template <int E, class Fn>
va_status by_shape(uint32_t D, Fn&& f) {
    using std::integral_constant;
    const integral_constant<int, 1> wave{};
    const integral_constant<int, 4> group{};
    switch (ceil_div(D, 64 * E)) {
        case 1: return f(wave, integral_constant<int, 1>());
        case 2: return f(wave, integral_constant<int, 2>());
        case 3: return f(wave, integral_constant<int, 3>());
        case 4: return f(wave, integral_constant<int, 4>());
        default: break;
    }
    if constexpr (E == 4) {
        if (D <= 64 * E * 6) return f(wave, integral_constant<int, 6>());
        if (D <= 64 * E * 8) return f(wave, integral_constant<int, 8>());
    }
    const uint32_t c = ceil_div(D, 256 * E);
    if (c <= 2) return f(group, integral_constant<int, 2>());
    if (c <= 4) return f(group, integral_constant<int, 4>());
    if constexpr (E == 4) {
        if (c <= 8) return f(group, integral_constant<int, 8>());
    }
    return f(group, integral_constant<int, 0>());
}
template <class Fn>
va_status by_dtype(va_dtype t, Fn&& f) {
    if (t == VA_DTYPE_F32) return f(std::integral_constant<int, VA_DTYPE_F32>());
    if (t == VA_DTYPE_F16) return f(std::integral_constant<int, VA_DTYPE_F16>());
    return f(std::integral_constant<int, VA_DTYPE_BF16>());
}
bool known(va_dtype t) { return t == VA_DTYPE_F32 || t == VA_DTYPE_F16 || t == VA_DTYPE_BF16; }
bool aligned(const void* p, va_dtype t) { return reinterpret_cast<uintptr_t>(p) % (t == VA_DTYPE_F32 ? 4 : 2) == 0; }

// Rows and dimensions that the kernels can count in 32 bits (a row's last chunk ends past it).
va_status check_sizes(va_context* ctx, uint32_t rows, uint32_t dim, const char* who) {
    VA_REQUIRE(ctx, rows <= 0x7FFFFFFFu && dim <= 0x7FFFFFFFu - 16384u, "%s: too many rows or dimensions (%u, %u)", who, rows, dim);
    return VA_OK;
}

// The description with the strides of a single row set, checked.
va_status check(va_context* ctx, const va_rms_desc* desc, const char* who, va_rms_desc& own) {
    VA_REQUIRE(ctx, desc, "%s: NULL description", who);
    own = *desc;
    for (uint64_t* stride : {&own.x_stride, &own.residual_stride, &own.out_residual_stride}) *stride = stride_of(own.rows, *stride, own.dim);
    const va_rms_desc* d = &own;
    VA_REQUIRE(ctx, d->x && d->weight, "%s: NULL pointer", who);
    VA_REQUIRE(ctx, d->rows > 0 && d->dim > 0, "%s: empty input (%u rows, %u dimensions)", who, d->rows, d->dim);
    VA_REQUIRE(ctx, known(d->dtype), "%s: unknown type %d", who, int(d->dtype));
    VA_REQUIRE(ctx, d->x_stride >= d->dim && (!d->residual || d->residual_stride >= d->dim) && (!d->out_residual || d->out_residual_stride >= d->dim),
               "%s: a row stride is below the dimension", who);
    VA_REQUIRE(ctx, aligned(d->x, d->dtype) && aligned(d->residual, d->dtype) && aligned(d->weight, d->dtype) && aligned(d->out_residual, d->dtype),
               "%s: an operand is not aligned to its type", who);
    VA_REQUIRE(ctx, std::isfinite(d->epsilon) && d->epsilon >= 0.0f, "%s: epsilon must be finite and not negative", who);
    return check_sizes(ctx, d->rows, d->dim, who);
}

template <int OUT>
va_status forward(va_context* ctx, const va_rms_desc* d, void* out, uint64_t ldo, uint32_t group, float given, float* scales) {
    RmsArgs a{d->x, d->residual, d->weight, d->out_residual, d->out_inverse_rms, out, scales, d->x_stride, d->residual_stride,
              d->out_residual_stride, ldo, 0, d->rows, d->dim, group, group ? ceil_div(d->dim, group) : 1u, d->epsilon, given};
    return by_dtype(d->dtype, [&](auto dt) {
        constexpr int E = OUT == OUT_SAME ? 16 / int(sizeof(ElemT<decltype(dt)::value>)) : 8;
        return by_shape<E>(d->dim, [&](auto wpr, auto c) {
            constexpr uint32_t rows = decltype(wpr)::value == 1 ? 4 : 1;  // a workgroup's
            for (a.t0 = 0; a.t0 < a.T;) {
                const uint32_t grid = std::min(ceil_div(a.T - a.t0, rows), kGridMax);
                rms_norm_kernel<decltype(dt)::value, OUT, decltype(wpr)::value, decltype(c)::value><<<dim3(grid), dim3(256), 0, ctx->stream>>>(a);
                VA_CHECK_LAUNCH(ctx);
                if (a.T - a.t0 <= grid * rows) break;
                a.t0 += grid * rows;
            }
            return VA_OK;
        });
    });
}

va_status check_codes(va_context* ctx, va_code code, uint32_t group, float given, const char* who) {
    VA_REQUIRE(ctx, code == VA_CODE_INT8 || code == VA_CODE_FP8_E4M3, "%s: unknown code type %d", who, int(code));
    VA_REQUIRE(ctx, group == 0 || (group >= 8 && group <= 512 && (group & (group - 1)) == 0),
               "%s: groups of %u (0, or a power of two from 8 to 512)", who, group);
    VA_REQUIRE(ctx, std::isfinite(given) && given >= 0.0f && (given == 0.0f || group == 0), "%s: a given scale is positive and for the whole tensor", who);
    return VA_OK;
}

}  // namespace
}  // namespace va

using namespace va;

extern "C" {

va_status va_rms_norm(va_context* ctx, const va_rms_desc* desc, void* out, uint64_t out_stride) {
    if (!ctx) return VA_ERR_INVALID_ARG;
    va_rms_desc own;
    VA_CHECK_STATUS(check(ctx, desc, "va_rms_norm", own));
    const va_rms_desc* d = &own;
    out_stride = stride_of(d->rows, out_stride, d->dim);
    VA_REQUIRE(ctx, out && out_stride >= d->dim && aligned(out, d->dtype), "va_rms_norm: the output is NULL, misaligned or its stride below the dimension");
    DeviceGuard guard(ctx->device);
    return forward<OUT_SAME>(ctx, d, out, out_stride, 0, 0.0f, nullptr);
}

va_status va_rms_norm_quantized(va_context* ctx, const va_rms_desc* desc, va_code code, uint32_t group, float given_scale, void* out_codes,
                                uint64_t codes_stride, float* out_scales) {
    if (!ctx) return VA_ERR_INVALID_ARG;
    va_rms_desc own;
    VA_CHECK_STATUS(check(ctx, desc, "va_rms_norm_quantized", own));
    const va_rms_desc* d = &own;
    codes_stride = stride_of(d->rows, codes_stride, d->dim);
    VA_CHECK_STATUS(check_codes(ctx, code, group, given_scale, "va_rms_norm_quantized"));
    VA_REQUIRE(ctx, out_codes && codes_stride >= d->dim, "va_rms_norm_quantized: the codes are NULL or their stride below the dimension");
    VA_REQUIRE(ctx, (given_scale > 0.0f) == (out_scales == nullptr), "va_rms_norm_quantized: scales are written unless one is given");
    DeviceGuard guard(ctx->device);
    return code == VA_CODE_INT8 ? forward<OUT_INT8>(ctx, d, out_codes, codes_stride, group, given_scale, out_scales)
                                : forward<OUT_FP8>(ctx, d, out_codes, codes_stride, group, given_scale, out_scales);
}

va_status va_rms_dequantize(va_context* ctx, const void* codes, uint64_t codes_stride, va_code code, const float* scales, float given_scale,
                            uint32_t rows, uint32_t dim, uint32_t group, va_dtype dtype, void* out, uint64_t out_stride) {
    if (!ctx) return VA_ERR_INVALID_ARG;
    VA_CHECK_STATUS(check_codes(ctx, code, group, given_scale, "va_rms_dequantize"));
    VA_REQUIRE(ctx, codes && out && (given_scale > 0.0f) == (scales == nullptr), "va_rms_dequantize: NULL pointer, or scales beside a given scale");
    VA_REQUIRE(ctx, rows > 0 && dim > 0, "va_rms_dequantize: empty input (%u rows, %u dimensions)", rows, dim);
    VA_CHECK_STATUS(check_sizes(ctx, rows, dim, "va_rms_dequantize"));
    VA_REQUIRE(ctx, known(dtype) && aligned(out, dtype), "va_rms_dequantize: unknown type or misaligned output");
    codes_stride = stride_of(rows, codes_stride, dim);
    out_stride = stride_of(rows, out_stride, dim);
    VA_REQUIRE(ctx, codes_stride >= dim && out_stride >= dim, "va_rms_dequantize: a row stride is below the dimension");
    const uint64_t blocks = (uint64_t(rows) * ((uint64_t(dim) + 7) / 8) + 255) / 256;
    DeviceGuard guard(ctx->device);
    return by_dtype(dtype, [&](auto dt) {
        for (uint64_t b = 0; b < blocks; b += kGridMax) {
            rms_dequantize_kernel<decltype(dt)::value><<<dim3(uint32_t(std::min<uint64_t>(blocks - b, kGridMax))), dim3(256), 0, ctx->stream>>>(
                static_cast<const uint8_t*>(codes), scales, codes_stride, b * 256, rows, dim, group, group ? ceil_div(dim, group) : 1u, given_scale,
                code == VA_CODE_FP8_E4M3, static_cast<ElemT<decltype(dt)::value>*>(out), out_stride);
            VA_CHECK_LAUNCH(ctx);
        }
        return VA_OK;
    });
}

va_status va_rms_norm_backward(va_context* ctx, const va_rms_desc* desc, const void* grad, uint64_t grad_stride, const void* grad_residual,
                               uint64_t grad_residual_stride, const float* inverse_rms, void* out_grad_x, uint64_t grad_x_stride,
                               void* out_grad_weight) {
    if (!ctx) return VA_ERR_INVALID_ARG;
    va_rms_desc own;
    VA_CHECK_STATUS(check(ctx, desc, "va_rms_norm_backward", own));
    const va_rms_desc* d = &own;
    for (uint64_t* stride : {&grad_stride, &grad_residual_stride, &grad_x_stride}) *stride = stride_of(d->rows, *stride, d->dim);
    VA_REQUIRE(ctx, grad && inverse_rms && (out_grad_x || out_grad_weight), "va_rms_norm_backward: NULL pointer");
    VA_REQUIRE(ctx, !d->residual && !d->out_residual && !d->out_inverse_rms, "va_rms_norm_backward: x is the summed row; the description has no residual and no output");
    VA_REQUIRE(ctx, grad_stride >= d->dim && (!grad_residual || grad_residual_stride >= d->dim) && (!out_grad_x || grad_x_stride >= d->dim),
               "va_rms_norm_backward: a row stride is below the dimension");
    VA_REQUIRE(ctx, aligned(grad, d->dtype) && aligned(grad_residual, d->dtype) && aligned(out_grad_x, d->dtype) && aligned(out_grad_weight, d->dtype),
               "va_rms_norm_backward: an operand is not aligned to its type");
    DeviceGuard guard(ctx->device);
    RmsGradArgs a{grad, d->x, d->weight, grad_residual, inverse_rms, out_grad_x, nullptr, grad_stride, d->x_stride, grad_residual_stride,
                  grad_x_stride, d->rows, d->dim};
    return by_dtype(d->dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        return by_shape<16 / int(sizeof(ElemT<DT>))>(d->dim, [&](auto wpr, auto c) {
            constexpr int WPR = decltype(wpr)::value, C = decltype(c)::value;
            // Workgroups a CU: 2-byte rows need more of them for as many bytes in flight.  37,289 x 768 bf16, forward and
            // backward: two 118 us, four 96; 30,000 x 512 fp32: 88 and 92.
            const uint32_t grid = std::min(ceil_div(a.T, 4 / WPR), (DT == VA_DTYPE_F32 ? 2u : 4u) * uint32_t(ctx->num_cus));
            const uint32_t shares = C ? grid : std::min(a.T, 256u);
            Scratch sc(ctx);
            if (out_grad_weight) {
                VA_CHECK_STATUS(sc.reserve(Scratch::round(uint64_t(shares) * a.D * 4)));
                a.part = sc.carve<float>(uint64_t(shares) * a.D);
            }
            if constexpr (C > 0) {
                rms_grad_kernel<DT, WPR, C><<<dim3(grid), dim3(256), 0, ctx->stream>>>(a);
                VA_CHECK_LAUNCH(ctx);
            } else {
                // (dw first: dx may be written over what it is the sum of)
                if (out_grad_weight) {
                    rms_weight_grad_kernel<DT><<<dim3(ceil_div(a.D, 2048), shares), dim3(256), 0, ctx->stream>>>(a);
                    VA_CHECK_LAUNCH(ctx);
                }
                if (a.out) {
                    rms_long_grad_kernel<DT><<<dim3(grid), dim3(256), 0, ctx->stream>>>(a);
                    VA_CHECK_LAUNCH(ctx);
                }
            }
            if (out_grad_weight) {
                rms_weight_sum_kernel<DT><<<dim3(std::min(ceil_div(a.D, 64), kGridMax / 4)), dim3(1024), 0, ctx->stream>>>(a.part, shares, a.D, static_cast<ElemT<DT>*>(out_grad_weight));
                VA_CHECK_LAUNCH(ctx);
            }
            return VA_OK;
        });
    });
}

}  // extern "C"
