// va_xent.hip — softmax cross entropy of hidden rows over all items of a collection, and its
// gradient, without the rows x items matrix.
//
//   l_tj = scale h_t . w_j + o_j          lse_t = log sum_j exp l_tj       loss_t = lse_t - l_{t, y_t}
//   dl_tj = g_t (exp(l_tj - lse_t) - [j = y_t])     dh = scale dl w        dw = scale dl^T h
//
// Forward: one product (va_gemm16.hpp) whose epilogue keeps, per row, the running maximum m and
// z = sum exp(l - m) of the items seen; the workgroups' (m, z) are joined by the finishing kernel.  Backward: the items are taken in
// pieces; for each piece the logits are computed again, dl leaves the product's epilogue as 16-bit
// values in a bounded workspace, and two more products read it, along its rows and across them: dh accumulates over
// the pieces in fp32, dw's rows of the piece are final.  So a training step is four products (one
// of them the recomputation), and the memory is that of one piece.
//
// Precision: fp16 / bf16 operands enter the matrix cores as they are, sums are fp32.  dl is rounded
// once to the operands' type for the second products (relative 2^-12 / 2^-9 a value, like the
// rounding of the result), after a scale that takes the largest |g| to 2^14: fp16's range then holds
// probabilities down to 2^-38 of it, and with one g for all rows the target's -g is exact.  fp32 operands, and dl with them, are two
// fp16 planes (va_gemm16.hpp).
//
// Masks: an item whose offset is -inf has no probability whatever its vector holds (NaN and inf
// included) and gets a zero gradient; a row without a target has loss 0 and a zero gradient whatever
// it holds.  When every item is masked, lse = -inf, the losses are 0 and so are the gradients.
#include <algorithm>
#include <cfloat>
#include <cmath>

#include "va_gemm16.hpp"

namespace va {
namespace {

using g16::f32x16;
using g16::f32x4;
using g16::u32x4;

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

// ---- element types -----------------------------------------------------------------------------
template <int DT>
struct Elem;
template <>
struct Elem<VA_DTYPE_F32> {
    using T = float;
    static __device__ float to_f(T v) { return v; }
    static __device__ T from_f(float v) { return v; }
};
template <>
struct Elem<VA_DTYPE_F16> {
    using T = _Float16;
    static __device__ float to_f(T v) { return float(v); }
    static __device__ T from_f(float v) { return T(v); }
};
template <>
struct Elem<VA_DTYPE_BF16> {
    using T = __bf16;
    static __device__ float to_f(T v) { return float(v); }
    static __device__ T from_f(float v) { return T(v); }
};
template <int DT>
using ElemT = typename Elem<DT>::T;
template <bool BF16>
__device__ __forceinline__ uint16_t bits16(float v) {
    if constexpr (BF16) return __builtin_bit_cast(uint16_t, __bf16(v));
    else return __builtin_bit_cast(uint16_t, _Float16(v));
}
// v = hi + lo in fp16
__device__ __forceinline__ void split16(float v, uint16_t& hi, uint16_t& lo) {
    const _Float16 h = _Float16(v);
    hi = __builtin_bit_cast(uint16_t, h);
    lo = __builtin_bit_cast(uint16_t, _Float16(v - float(h)));
}
// the power of two that puts |v| in [2^13, 2^14) (1 for 0, inf and NaN)
__device__ __forceinline__ float scale_to_2p14(float v) {
    v = fabsf(v);
    if (!(v > 0.0f) || !(v < INFINITY)) return 1.0f;
    int e;
    (void)frexpf(v, &e);  // v = f 2^e, f in [0.5, 1)
    return ldexpf(1.0f, min(14 - e, 126));
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v = fmaxf(v, __shfl_xor(v, d));
    return v;
}

// (m, z) of two disjoint sets of items, joined
__device__ __forceinline__ void join(float& m, float& z, float m2, float z2) {
    const float mm = fmaxf(m, m2);
    const float ref = mm == -INFINITY ? 0.0f : mm;
    z = z * exp2f((m - ref) * kLog2e) + z2 * exp2f((m2 - ref) * kLog2e);
    m = mm;
}

// ---- packing: operands whose rows are not whole 64-value stages, not 16-bit, or must not be read -----
// dst[r][k] = src[r][k], zeros for k in [D, Kp); rows whose drop value says so are zeros.  Nothing if *run_if is zero.
__global__ __launch_bounds__(256) void pack16_kernel(const uint16_t* __restrict__ src, uint64_t ld, uint32_t D, uint32_t Kp,
                                                     const float* __restrict__ drop, float drop_if, const uint32_t* run_if, uint16_t* __restrict__ dst, uint64_t n8) {
    if (run_if && *run_if == 0) return;
    typedef uint16_t u16x8 __attribute__((ext_vector_type(8), aligned(2)));
    const uint32_t per = Kp / 8;
    for (uint64_t i = uint64_t(blockIdx.x) * 256 + threadIdx.x; i < n8; i += uint64_t(gridDim.x) * 256) {
        const uint64_t r = i / per;
        const uint32_t k = uint32_t(i - r * per) * 8;
        u16x8 v = {};
        const uint16_t* s = src + r * ld + k;
        if (!(drop && drop[r] == drop_if)) {
            if (k + 8 <= D) {
                v = *reinterpret_cast<const u16x8*>(s);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = k + e < D ? s[e] : uint16_t(0);
            }
        }
        *reinterpret_cast<u32x4*>(dst + r * Kp + k) = __builtin_bit_cast(u32x4, v);
    }
}

// One wave per fp32 row: its planes dst[r] = {hi, lo} (Kp values each, zeros past D), scaled by the
// power of two that puts the row's largest entry, or the tensor's (absmax), near 2^14; inv[r] = the
// inverse.  Rows whose drop value says so are zeros.
__global__ __launch_bounds__(256) void pack32_kernel(const float* __restrict__ src, uint64_t ld, uint32_t R, uint32_t D, uint32_t Kp,
                                                     const uint32_t* __restrict__ absmax, const float* __restrict__ drop, float drop_if,
                                                     uint16_t* __restrict__ dst, float* __restrict__ inv) {
    typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
    const int lane = threadIdx.x & 63;
    const uint32_t r = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (r >= R) return;
    const float* s = src + r * ld;
    const bool none = drop && drop[r] == drop_if;
    auto load4 = [&](uint32_t k) {
        f32x4 v{0.0f, 0.0f, 0.0f, 0.0f};
        if (none) return v;
        if (k + 4 <= D) return f32x4(*reinterpret_cast<const f32x4u*>(s + k));
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = k + e < D ? s[k + e] : 0.0f;
        return v;
    };
    // up to 1024 values of the row stay in registers between the two passes
    f32x4 held[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) held[i] = load4(256 * i + 4 * lane);
    float sc;
    if (absmax) {
        sc = scale_to_2p14(__builtin_bit_cast(float, *absmax));
    } else {
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) m = fmaxf(m, fabsf(held[i][e]));
        for (uint32_t k = 1024 + 4 * lane; k < D; k += 256) {
            const f32x4 v = load4(k);
#pragma unroll
            for (int e = 0; e < 4; ++e) m = fmaxf(m, fabsf(v[e]));
        }
        sc = scale_to_2p14(wave_max(m));
    }
    if (lane == 0) inv[r] = 1.0f / sc;
    uint16_t* o = dst + uint64_t(r) * 2 * Kp;
    auto put = [&](uint32_t k, f32x4 v) {
        uint16_t h[4], l[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) split16(v[e] * sc, h[e], l[e]);
        *reinterpret_cast<uint2*>(o + k) = make_uint2(h[0] | uint32_t(h[1]) << 16, h[2] | uint32_t(h[3]) << 16);
        *reinterpret_cast<uint2*>(o + Kp + k) = make_uint2(l[0] | uint32_t(l[1]) << 16, l[2] | uint32_t(l[3]) << 16);
    };
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t k = 256 * i + 4 * lane;
        if (k < Kp) put(k, held[i]);
    }
    for (uint32_t k = 1024 + 4 * lane; k < Kp; k += 256) put(k, load4(k));
}

// *odd = 1 (0 before the launch) if a masked item holds NaN or inf, or if an offset is finite and beyond
// 1e37 (log2 e times it may not be).  One wave per 64 items; masked rows are read.
__global__ __launch_bounds__(256) void xent_odd_kernel(const uint16_t* __restrict__ items, uint64_t ld, const float* __restrict__ offsets, uint32_t V,
                                                       uint32_t D, uint32_t exponent, uint32_t* odd) {
    const uint32_t lane = threadIdx.x & 63, j0 = (blockIdx.x * 4 + (threadIdx.x >> 6)) * 64;
    const float o = j0 + lane < V ? offsets[j0 + lane] : 0.0f;
    bool bad = fabsf(o) > 1e37f && fabsf(o) < INFINITY;
    for (uint64_t masked = __ballot(o == -INFINITY); masked; masked &= masked - 1) {
        const uint16_t* row = items + (j0 + uint32_t(__builtin_ctzll(masked))) * ld;
        for (uint32_t d = lane; d < D; d += 64) bad |= (row[d] & exponent) == exponent;
    }
    if (__any(bad) && lane == 0) *odd = 1;
}

// out = the bits of the largest |src| (0 before the launch); rows whose drop value says so are left out
__global__ __launch_bounds__(256) void absmax_kernel(const float* __restrict__ src, uint64_t ld, uint32_t R, uint32_t D,
                                                     const float* __restrict__ drop, float drop_if, uint32_t* out) {
    typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
    __shared__ float part[4];
    float m = 0.0f;
    const int lane = threadIdx.x & 63;
    for (uint32_t r = blockIdx.x * 4 + (threadIdx.x >> 6); r < R; r += gridDim.x * 4) {
        if (drop && drop[r] == drop_if) continue;
        const float* s = src + r * ld;
        const uint32_t full = D / 4 * 4;
#pragma unroll 4
        for (uint32_t k = 4 * lane; k < full; k += 256) {
            const f32x4 v = *reinterpret_cast<const f32x4u*>(s + k);
            m = fmaxf(fmaxf(m, fmaxf(fabsf(v[0]), fabsf(v[1]))), fmaxf(fabsf(v[2]), fabsf(v[3])));
        }
        if (full + lane < D) m = fmaxf(m, fabsf(s[full + lane]));
    }
    m = wave_max(m);
    if (lane == 0) part[threadIdx.x >> 6] = m;
    __syncthreads();
    if (threadIdx.x == 0)
        atomicMax(out, __builtin_bit_cast(uint32_t, fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]))));
}

// ---- the logits' epilogues -------------------------------------------------------------------------
// The offsets of a launch: none, none but -inf for the items missing from the last tile, or any.
enum Offsets : int { OFF_NONE = 0, OFF_EDGE = 1, OFF_ANY = 2 };

struct LogitArgs {
    const float* offsets;  // of the launch's first item (nullptr: zeros)
    const uint32_t* odd;   // OFF_ANY: zero if no masked item holds NaN or inf and no offset is near fp32's
                           // limits (nullptr: not known)
    const float* qinv;     // fp32 operands: the rows' and the items' inverse scales
    const float* xinv;
    float scale;
    uint32_t rows, items;  // hidden rows; items of this launch
};

// The epilogues work on logits in the unit of a binary exponent (log2 e of them: one fma takes an
// accumulator there, and exp2 of a difference is one instruction more than the subtraction) unless that could
// go wrong: odd offsets (masked items are then told by their offset whatever their accumulator holds, and
// differences are taken before they are scaled: an offset of the type's lowest value stays in range) and fp32
// operands (whose items have scales of their own) keep natural units.
template <int OFF, bool PLANES, int TR>
struct LogitShared {
    float off[OFF ? TR : 1];
    float inv[PLANES ? TR : 1];
};
template <bool NATURAL, int OFF, bool PLANES, int TR>
__device__ __forceinline__ f32x4 logits4(const LogitShared<OFF, PLANES, TR>& sm, const f32x16& acc, int j, int r, float c) {
    f32x4 v;
    f32x4 o{}, x{};
    // these reads stay here, and the groups in order: mixed, a tile's would fill the registers
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (OFF != OFF_NONE) o = *reinterpret_cast<const f32x4*>(sm.off + r);
    if constexpr (PLANES) x = *reinterpret_cast<const f32x4*>(sm.inv + r);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float a = acc[4 * j + e];
        if constexpr (PLANES) a *= x[e];
        if constexpr (OFF == OFF_NONE) v[e] = a * c;
        else v[e] = NATURAL && o[e] == -INFINITY ? -INFINITY : fmaf(a, c, o[e]);
    }
    return v;
}
template <bool NATURAL>
__device__ __forceinline__ float exp_diff(float v, float ref) {
    return __builtin_amdgcn_exp2f(NATURAL ? (v - ref) * kLog2e : v - ref);
}
// whether a launch keeps natural units (uniform)
template <int OFF, bool PLANES>
__device__ __forceinline__ bool keeps_natural(const LogitArgs& a) {
    if constexpr (PLANES) return true;
    if constexpr (OFF != OFF_ANY) return false;
    return __builtin_amdgcn_readfirstlane(a.odd ? *a.odd : 1u) != 0u;
}
__device__ __forceinline__ float offset_of(const LogitArgs& a, bool in, uint32_t r, bool natural) {
    const float o = !in ? -INFINITY : a.offsets ? a.offsets[r] : 0.0f;
    return natural ? o : o * kLog2e;
}

// Forward: the running (m, z) of a lane's items per query; joined over the workgroup at the end of
// the item and written to part[row * slots + slot].  The target's logit is picked out on the way: with
// the loss a difference of two logits, both from the same sums, their errors cancel for a row whose
// target is far ahead of the other items.
template <class Sh, int OFF, bool PLANES>
struct LseEpi {
    using Shape = Sh;
    static constexpr int TQ = Sh::TQ, TR = Sh::TR;
    static constexpr bool kWalk = true, kStores = false;
    LogitArgs a;
    const int64_t* targets;
    uint32_t item0;  // of the launch
    float* picked;   // [rows] the target's logit
    float2* part;
    uint32_t slots, slot0;
    struct Shared : LogitShared<OFF, PLANES, TR> {
        float2 red[Sh::WR][TQ];
        uint32_t target[TQ];  // within the launch's items (any larger value: elsewhere)
        float qinv[PLANES ? TQ : 1];
    };
    struct State {
        float m[2], z[2];
        float off, inv;
        bool natural;
    };
    template <class Tile>
    __device__ void begin(State& s, Shared& sm, const Tile& t) {
        s.natural = keeps_natural<OFF, PLANES>(a);
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            s.m[n] = -INFINITY;
            s.z[n] = 0.0f;
        }
        const uint32_t i = threadIdx.x, q = t.qb * TQ + i;
        if (i >= uint32_t(TQ)) return;
        const int64_t y = q < a.rows ? targets[q] - int64_t(item0) : -1;
        sm.target[i] = y >= 0 && y < int64_t(a.items) ? uint32_t(y) : 0xFFFFFFFFu;
        if constexpr (PLANES) sm.qinv[i] = q < a.rows ? a.qinv[q] : 0.0f;
    }
    template <class Tile>
    __device__ void load(State& s, const Tile& t, int tid) {
        const uint32_t r = t.rb * TR + uint32_t(tid);
        const bool in = tid < TR && r < a.items;
        if constexpr (OFF != OFF_NONE) s.off = offset_of(a, in, r, s.natural);
        if constexpr (PLANES) s.inv = in ? a.xinv[r] : 0.0f;
    }
    __device__ void publish(State& s, Shared& sm, int tid) {
        if constexpr (OFF != OFF_NONE)
            if (tid < TR) sm.off[tid] = s.off;
        if constexpr (PLANES)
            if (tid < TR) sm.inv[tid] = s.inv;
    }
    template <bool NATURAL, class Tile>
    __device__ void block(State& s, Shared& sm, const g16::Lane& ln, f32x16 (&acc)[2][2], const Tile& t, int n) {
        const float c = (PLANES ? a.scale * sm.qinv[ln.q(n)] : a.scale) * (NATURAL ? 1.0f : kLog2e);
        float top = -INFINITY;
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                f32x4 v = logits4<NATURAL, OFF, PLANES, TR>(sm, acc[m][n], j, ln.r(m, j), c);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    top = fmaxf(top, v[e]);
                    acc[m][n][4 * j + e] = v[e];
                }
            }
        const float mm = fmaxf(s.m[n], top);
        const float ref = mm == -INFINITY ? 0.0f : mm;
        const float z = s.z[n] * exp_diff<NATURAL>(s.m[n], ref);
        // (a tile holds the target of few rows, most tiles of none of a wave's)
        const uint32_t y = sm.target[ln.q(n)] - t.rb * TR - uint32_t(ln.wr * 64);
        if (__any(y < 64u)) {
            const uint32_t i = y - 4u * uint32_t(ln.hh);  // 32 m + 8 j + e of the lane's values
            float v = 0.0f;
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int k = 0; k < 16; ++k) v = i == uint32_t(32 * m + 8 * (k >> 2) + (k & 3)) ? acc[m][n][k] : v;
            if (y < 64u && (i & 4u) == 0u) picked[t.qb * TQ + ln.q(n)] = NATURAL ? v : v * kLn2;
        }
        float zz[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int v = 0; v < 16; ++v) zz[v & 3] += exp_diff<NATURAL>(acc[m][n][v], ref);
        s.m[n] = mm;
        s.z[n] = z + ((zz[0] + zz[1]) + (zz[2] + zz[3]));
    }
    template <class Tile, class Settle>
    __device__ void tile(State& s, Shared& sm, const g16::Lane& ln, f32x16 (&acc)[2][2], const Tile& t, char*, Settle) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            if constexpr (PLANES) {
                block<true>(s, sm, ln, acc, t, n);
            } else if constexpr (OFF != OFF_ANY) {
                block<false>(s, sm, ln, acc, t, n);
            } else {
                if (s.natural) block<true>(s, sm, ln, acc, t, n);
                else block<false>(s, sm, ln, acc, t, n);
            }
        }
    }
    template <class Tile>
    __device__ void end(State& s, Shared& sm, const g16::Lane& ln, const Tile& t) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            // (natural units from here; a row's largest logit and its target's are scaled alike)
            float m = s.natural ? s.m[n] : s.m[n] * kLn2;
            join(m, s.z[n], __shfl_xor(m, 32), __shfl_xor(s.z[n], 32));
            if (ln.hh == 0) sm.red[ln.wr][ln.q(n)] = make_float2(m, s.z[n]);
        }
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        const uint32_t q = threadIdx.x;
        if (q < uint32_t(TQ) && t.qb * TQ + q < a.rows) {
            float2 v = sm.red[0][q];
#pragma unroll
            for (int w = 1; w < Sh::WR; ++w) join(v.x, v.y, sm.red[w][q].x, sm.red[w][q].y);
            part[uint64_t(t.qb * TQ + q) * slots + slot0 + t.part] = v;
        }
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    }
};

// Backward: dl of the piece's items, p[t][j]: Vp values a plane and row, zeros past the last item, rows
// `pitch` values apart.
template <class Sh, bool BF16, int OFF, bool PLANES>
struct GradEpi {
    using Shape = Sh;
    static constexpr int TQ = Sh::TQ, TR = Sh::TR;
    static constexpr bool kWalk = false, kStores = true;
    LogitArgs a;
    const float* gk;   // g_t times dl's factor (0: the row has no gradient)
    const float* lse;
    const int64_t* targets;
    uint32_t item0;    // the piece's first item
    uint16_t* p;
    uint32_t Vp, pitch;
    struct Shared : LogitShared<OFF, PLANES, TR> {
        float gk[TQ], lse[TQ];
        uint32_t target[TQ];  // within the piece (any larger value: elsewhere)
        float inv_q[PLANES ? TQ : 1];
    };
    struct State {
        float off, inv, gk, lse, qinv;
        uint32_t target;
        bool natural;
    };
    template <class Tile>
    __device__ void begin(State& s, Shared&, const Tile&) {
        s.natural = keeps_natural<OFF, PLANES>(a);
    }
    template <class Tile>
    __device__ void load(State& s, const Tile& t, int tid) {
        const uint32_t r = t.rb * TR + uint32_t(tid), q = t.qb * TQ + uint32_t(tid);
        const bool in = tid < TR && r < a.items, qin = tid < TQ && q < a.rows;
        if constexpr (OFF != OFF_NONE) s.off = offset_of(a, in, r, s.natural);
        if constexpr (PLANES) {
            s.inv = in ? a.xinv[r] : 0.0f;
            s.qinv = qin ? a.qinv[q] : 0.0f;
        }
        s.gk = qin ? gk[q] : 0.0f;
        s.lse = qin ? lse[q] : 0.0f;
        // a row without a gradient, or without any item: every probability is exp(-huge) = 0
        if (s.gk == 0.0f || s.lse == -INFINITY) {
            s.gk = 0.0f;
            s.lse = FLT_MAX;
        } else if (!s.natural) {
            s.lse *= kLog2e;
        }
        const int64_t y = qin ? targets[q] - int64_t(item0) : -1;
        s.target = y >= 0 && y < int64_t(a.items) ? uint32_t(y) : 0xFFFFFFFFu;
    }
    __device__ void publish(State& s, Shared& sm, int tid) {
        if constexpr (OFF != OFF_NONE)
            if (tid < TR) sm.off[tid] = s.off;
        if constexpr (PLANES)
            if (tid < TR) sm.inv[tid] = s.inv;
        if (tid >= TQ) return;
        if constexpr (PLANES) sm.inv_q[tid] = s.qinv;
        sm.gk[tid] = s.gk;
        sm.lse[tid] = s.lse;
        sm.target[tid] = s.target;
    }
    // One plane of the wave's 32 rows x 64 items from its 4 KiB of LDS: [t][j] rows of 128 bytes, 16-byte chunks
    // swizzled by t & 7 (the 8-byte writes and the reads then touch every bank equally); whole 128-byte
    // lines go out.  (Stored straight from the accumulators, 8 bytes a lane, a tile took three times as long.)
    __device__ void put(const char* spare, const g16::Lane& ln, const uint32_t q0, const uint32_t r0, uint32_t plane) {
        const int lane = ln.hh * 32 + ln.l32;
        asm volatile("" ::: "memory");  // the writes come first (a wave's LDS accesses execute in order)
        if (r0 < Vp) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int t = 8 * i + (lane >> 3), c = lane & 7;
                const u32x4 v = *reinterpret_cast<const u32x4*>(spare + t * 128 + 16 * (c ^ (t & 7)));
                if (q0 + t < a.rows)
                    *reinterpret_cast<u32x4*>(p + uint64_t(q0 + t) * pitch + plane * Vp + r0 + 8 * c) = v;
            }
        }
        asm volatile("" ::: "memory");  // and the reads before what is written next
    }
    static __device__ void write(char* spare, const g16::Lane& ln, int m, int j, const uint16_t (&v)[4]) {
        *reinterpret_cast<uint2*>(spare + ln.l32 * 128 + 16 * ((4 * m + j) ^ (ln.l32 & 7)) + 8 * ln.hh) =
            make_uint2(v[0] | uint32_t(v[1]) << 16, v[2] | uint32_t(v[3]) << 16);
    }
    // TARGETS: one of the wave's rows has its target among the block's items
    template <bool NATURAL, bool TARGETS>
    __device__ void block(Shared& sm, const g16::Lane& ln, f32x16 (&acc)[2][2], uint32_t y, int n, char* spare) {
        const float g = sm.gk[ln.q(n)], ref = sm.lse[ln.q(n)];
        const float c = (PLANES ? a.scale * sm.inv_q[ln.q(n)] : a.scale) * (NATURAL ? 1.0f : kLog2e);
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int r = ln.r(m, j);
                const f32x4 v = logits4<NATURAL, OFF, PLANES, TR>(sm, acc[m][n], j, r, c);
                uint16_t hi[4], lo[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float d = exp_diff<NATURAL>(v[e], ref);
                    if (TARGETS && y == uint32_t(r + e) && v[e] != -INFINITY) d -= 1.0f;
                    d *= g;
                    if constexpr (PLANES) {
                        split16(d, hi[e], lo[e]);
                        acc[m][n][4 * j + e] = d;
                    } else {
                        hi[e] = bits16<BF16>(d);
                    }
                }
                write(spare, ln, m, j, hi);
            }
    }
    template <class Tile, class Settle>
    __device__ void tile(State& s, Shared& sm, const g16::Lane& ln, f32x16 (&acc)[2][2], const Tile& t, char* spare, Settle settle) {
        const uint32_t r0 = t.rb * TR, rw = r0 + uint32_t(ln.wr * 64);
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const uint32_t q0 = t.qb * TQ + uint32_t(ln.wq * 64 + 32 * n), y = sm.target[ln.q(n)] - r0;
            const bool hit = __any(y - uint32_t(ln.wr * 64) < 64u);
            if constexpr (PLANES) {
                block<true, true>(sm, ln, acc, y, n, spare);
            } else {
                if (OFF == OFF_ANY && s.natural) block<true, true>(sm, ln, acc, y, n, spare);
                else if (hit) block<false, true>(sm, ln, acc, y, n, spare);
                else block<false, false>(sm, ln, acc, y, n, spare);
            }
            if (n == 0) settle();
            put(spare, ln, q0, rw, 0);
            if constexpr (PLANES) {
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        uint16_t hi[4], lo[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) split16(acc[m][n][4 * j + e], hi[e], lo[e]);
                        write(spare, ln, m, j, lo);
                    }
                put(spare, ln, q0, rw, 1);
            }
        }
    }
    template <class Tile>
    __device__ void end(State&, Shared&, const g16::Lane&, const Tile&) {}
};

// dh: fp32 shares [part][t][Dp], added to over the pieces (first: written)
template <class Sh>
struct ShareEpi {
    using Shape = Sh;
    static constexpr int TQ = Sh::TQ, TR = Sh::TR;
    static constexpr bool kWalk = false, kStores = true;
    float* out;
    uint32_t rows, D, Dp;
    bool first;
    struct Shared {};
    struct State {};
    template <class Tile>
    __device__ void begin(State&, Shared&, const Tile&) {}
    template <class Tile>
    __device__ void load(State&, const Tile&, int) {}
    __device__ void publish(State&, Shared&, int) {}
    template <class Tile, class Settle>
    __device__ void tile(State&, Shared&, const g16::Lane& ln, f32x16 (&acc)[2][2], const Tile& t, char*, Settle settle) {
        settle();
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const uint32_t q = t.qb * TQ + uint32_t(ln.q(n));
            if (q >= rows) continue;
            float* o = out + (uint64_t(t.part) * rows + q) * Dp;
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t d = t.rb * TR + uint32_t(ln.r(m, j));
                    if (d >= D) continue;  // (rows hold Dp = whole groups of 4)
                    f32x4 v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = acc[m][n][4 * j + e];
                    if (!first) v += *reinterpret_cast<const f32x4*>(o + d);
                    *reinterpret_cast<f32x4*>(o + d) = v;
                }
        }
    }
    template <class Tile>
    __device__ void end(State&, Shared&, const g16::Lane&, const Tile&) {}
};

// dw: the piece's rows, final
template <class Sh, int DT>
struct ItemGradEpi {
    using Shape = Sh;
    static constexpr int TQ = Sh::TQ, TR = Sh::TR;
    static constexpr bool kWalk = false, kStores = true;
    ElemT<DT>* out;
    uint64_t ld;
    uint32_t rows, D;
    const float* mul;        // scale over dl's factor
    const uint32_t* absmax;  // fp32: of the hidden rows (their planes' scale)
    bool vec;                // rows of four values are aligned
    struct Shared {
        float mul;
    };
    struct State {};
    template <class Tile>
    __device__ void begin(State&, Shared&, const Tile&) {}
    template <class Tile>
    __device__ void load(State&, const Tile&, int) {}
    __device__ void publish(State&, Shared& sm, int tid) {
        if (tid == 0) sm.mul = *mul / (DT == VA_DTYPE_F32 ? scale_to_2p14(__builtin_bit_cast(float, *absmax)) : 1.0f);
    }
    template <class Tile, class Settle>
    __device__ void tile(State&, Shared& sm, const g16::Lane& ln, f32x16 (&acc)[2][2], const Tile& t, char*, Settle settle) {
        settle();
        const float s = sm.mul;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const uint32_t q = t.qb * TQ + uint32_t(ln.q(n));
            if (q >= rows) continue;
            ElemT<DT>* o = out + q * ld;
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t d = t.rb * TR + uint32_t(ln.r(m, j));
                    if (d >= D) continue;
                    struct alignas(4 * sizeof(ElemT<DT>)) V4 {
                        ElemT<DT> v[4];
                    } v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v.v[e] = Elem<DT>::from_f(acc[m][n][4 * j + e] * s);
                    if (vec && d + 4 <= D) *reinterpret_cast<V4*>(o + d) = v;
                    else
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (d + e < D) o[d + e] = v.v[e];
                }
        }
    }
    template <class Tile>
    __device__ void end(State&, Shared&, const g16::Lane&, const Tile&) {}
};

// ---- finishing kernels ---------------------------------------------------------------------------
// One wave per row: the shares joined into lse, and the loss.
__global__ __launch_bounds__(256) void xent_finish_kernel(const int64_t* __restrict__ targets, uint32_t T, uint32_t V, int64_t ignore,
                                                          const float2* __restrict__ part, const float* __restrict__ picked,
                                                          uint32_t slots, float* __restrict__ loss, float* __restrict__ lse) {
    const int lane = threadIdx.x & 63;
    const uint32_t t = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (t >= T) return;
    float m = -INFINITY, z = 0.0f;
    for (uint32_t i = lane; i < slots; i += 64) {
        const float2 p = part[uint64_t(t) * slots + i];
        join(m, z, p.x, p.y);
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) join(m, z, __shfl_xor(m, d), __shfl_xor(z, d));
    if (lane) return;
    const float l = m == -INFINITY && z == 0.0f ? -INFINITY : m + logf(z);
    const int64_t y = targets[t];
    float out = 0.0f;
    if (y != ignore) {
        out = NAN;  // a target outside the collection
        if (y >= 0 && y < int64_t(V)) {
            const float v = picked[t];
            // log z + (m - v): the two large terms cancel before the small one is added
            out = l == -INFINITY ? 0.0f : v == -INFINITY ? INFINITY : logf(z) + (m - v);
        }
    }
    lse[t] = l;
    loss[t] = out;
}

// The sum or mean of the losses over the rows with a target.  One workgroup.
__global__ __launch_bounds__(1024) void xent_reduce_kernel(const float* __restrict__ loss, const int64_t* __restrict__ targets,
                                                           uint32_t T, int64_t ignore, bool mean, float* out) {
    __shared__ double sum[16];
    __shared__ uint32_t cnt[16];
    double s = 0.0;
    uint32_t c = 0;
    for (uint32_t t = threadIdx.x; t < T; t += 1024)
        if (targets[t] != ignore) {
            s += double(loss[t]);
            ++c;
        }
    for (int d = 32; d; d >>= 1) {
        s += __shfl_xor(s, d);
        c += __shfl_xor(c, d);
    }
    if ((threadIdx.x & 63) == 0) {
        sum[threadIdx.x >> 6] = s;
        cnt[threadIdx.x >> 6] = c;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 16; ++i) {
            s += sum[i];
            c += cnt[i];
        }
        *out = float(mean ? (c ? s / double(c) : 0.0) : s);
    }
}

// gk[t] = g_t c, *mul = scale / c: g_t is the gradient that reaches the row's loss, 0 for a row
// without a target, c takes the largest |g_t| to 2^14.  Clears absmax[0..3).  One workgroup.
__global__ __launch_bounds__(1024) void xent_gradient_kernel(const float* __restrict__ grad, const int64_t* __restrict__ targets,
                                                             uint32_t T, uint32_t V, int64_t ignore, int reduction, float scale,
                                                             float* __restrict__ gk, float* __restrict__ mul, uint32_t* absmax) {
    __shared__ float top[16];
    __shared__ uint32_t cnt[16];
    if (threadIdx.x < 3) absmax[threadIdx.x] = 0;
    float m = 0.0f;
    uint32_t c = 0;
    for (uint32_t t = threadIdx.x; t < T; t += 1024) {
        const int64_t y = targets[t];
        if (y == ignore) continue;
        ++c;
        if (reduction == VA_REDUCE_NONE && y >= 0 && y < int64_t(V)) m = fmaxf(m, fabsf(grad[t]));
    }
    for (int d = 32; d; d >>= 1) {
        m = fmaxf(m, __shfl_xor(m, d));
        c += __shfl_xor(c, d);
    }
    if ((threadIdx.x & 63) == 0) {
        top[threadIdx.x >> 6] = m;
        cnt[threadIdx.x >> 6] = c;
    }
    __syncthreads();
    m = top[0];
    c = cnt[0];
    for (int i = 1; i < 16; ++i) {
        m = fmaxf(m, top[i]);
        c += cnt[i];
    }
    float g = 1.0f;
    if (reduction != VA_REDUCE_NONE) {
        if (grad) g = *grad;
        if (reduction == VA_REDUCE_MEAN) g /= float(max(c, 1u));
        m = fabsf(g);
    }
    const bool plain = !(m > 0.0f) || !(m < INFINITY);
    if (plain) m = 16384.0f;
    for (uint32_t t = threadIdx.x; t < T; t += 1024) {
        const int64_t y = targets[t];
        const bool in = y != ignore && y >= 0 && y < int64_t(V);
        gk[t] = in ? (reduction == VA_REDUCE_NONE ? grad[t] : g) / m * 16384.0f : 0.0f;
    }
    if (threadIdx.x == 0) *mul = scale * (m / 16384.0f);
}

// dh[t][d] = mul sum over the shares (zero for a row without a gradient).  64 groups of four values a
// workgroup, its four waves a quarter of the shares each.
template <int DT>
__global__ __launch_bounds__(256) void share_sum_kernel(const float* __restrict__ share, uint32_t parts, uint32_t T, uint32_t D,
                                                        uint32_t Dp, const float* __restrict__ gk, const float* __restrict__ mul,
                                                        const uint32_t* __restrict__ absmax, ElemT<DT>* __restrict__ out, uint64_t ld) {
    __shared__ f32x4 part[4][64];
    const uint32_t per = Dp / 4, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const uint64_t i = uint64_t(blockIdx.x) * 64 + lane, n = uint64_t(T) * per;
    f32x4 v{0.0f, 0.0f, 0.0f, 0.0f};
    if (i < n)
#pragma unroll 8
        for (uint32_t s = w; s < parts; s += 4) v += *reinterpret_cast<const f32x4*>(share + (uint64_t(s) * n + i) * 4);
    part[w][lane] = v;
    __syncthreads();
    if (w || i >= n) return;
    v = (v + part[1][lane]) + (part[2][lane] + part[3][lane]);
    const uint32_t t = uint32_t(i / per), d = uint32_t(i % per) * 4;
    const float m = *mul / (DT == VA_DTYPE_F32 ? scale_to_2p14(__builtin_bit_cast(float, *absmax)) : 1.0f);
    const bool none = gk[t] == 0.0f;
    for (int e = 0; e < 4 && d + e < D; ++e) out[t * ld + d + e] = Elem<DT>::from_f(none ? 0.0f : v[e] * m);
}

// ---- host ------------------------------------------------------------------------------------------
size_t elem_size(va_dtype t) { return t == VA_DTYPE_F32 ? 4 : 2; }

// Rows that the product can read where they are: 16-bit, whole stages, aligned.
bool direct(va_dtype dt, const void* p, uint64_t ld, uint32_t D) {
    return dt != VA_DTYPE_F32 && D % g16::KC == 0 && ld % 8 == 0 && reinterpret_cast<uintptr_t>(p) % 16 == 0;
}
size_t packed_bytes(va_dtype dt, uint64_t rows, uint32_t Kp) { return rows * Kp * (dt == VA_DTYPE_F32 ? 4 : 2); }

va_status pack(va_context* ctx, va_dtype dt, const void* src, uint64_t ld, uint32_t R, uint32_t D, uint32_t Kp, const uint32_t* absmax,
               const float* drop, float drop_if, void* dst, float* inv, const uint32_t* run_if = nullptr) {
    if (dt == VA_DTYPE_F32) {
        pack32_kernel<<<dim3(ceil_div(R, 4)), dim3(256), 0, ctx->stream>>>(static_cast<const float*>(src), ld, R, D, Kp, absmax, drop, drop_if,
                                                                           static_cast<uint16_t*>(dst), inv);
    } else {
        const uint64_t n8 = uint64_t(R) * (Kp / 8);
        pack16_kernel<<<dim3(uint32_t(std::min<uint64_t>((n8 + 255) / 256, 16384))), dim3(256), 0, ctx->stream>>>(
            static_cast<const uint16_t*>(src), ld, D, Kp, drop, drop_if, run_if, static_cast<uint16_t*>(dst), n8);
    }
    VA_CHECK_LAUNCH(ctx);
    return VA_OK;
}

const char* at(const void* p, uint64_t ld, uint64_t row, va_dtype dt) { return static_cast<const char*>(p) + row * ld * elem_size(dt); }

// The shape of a product's workgroups: 256 x 256 tiles (the least operand traffic) where they fill most
// of the chip or the operands are that large; smaller ones where those would leave CUs without work.
template <class F>
va_status by_shape(int shape, F&& f) {
    if (shape == 0) return f(g16::Large());
    if (shape == 1) return f(g16::Shape<2, 2>());
    return f(g16::Shape<1, 2>());
}
struct Blocks {
    int shape;
    uint32_t tq, tr, grid;  // grid: the most workgroups of a launch
    uint32_t nq(uint64_t Q) const { return uint32_t((Q + tq - 1) / tq); }
    uint32_t nr(uint64_t R) const { return uint32_t((R + tr - 1) / tr); }
};
// `shares`: how many shares of the sum the caller can make of each tile
Blocks blocks_for(const va_context* ctx, uint64_t Q, uint64_t R, uint32_t shares = 1) {
    const Blocks all[3] = {{0, 256, 256, g16::grid_max<g16::Large>(ctx)},
                           {1, 128, 128, g16::grid_max<g16::Shape<2, 2>>(ctx)},
                           {2, 64, 128, g16::grid_max<g16::Shape<1, 2>>(ctx)}};
    const uint64_t enough = all[0].grid * 3 / 4;
    for (int i = 0; i < 2; ++i)
        if (Q > all[i].tq / 2 && uint64_t(all[i].nq(Q)) * all[i].nr(R) * shares >= enough) return all[i];
    return all[2];
}

// f(bf16, offsets, planes) of a launch over n items of a tile width
template <class F>
va_status by_type(va_dtype dt, bool offsets, bool edge, F&& f) {
    using std::integral_constant;
    const integral_constant<int, OFF_NONE> none{};
    const integral_constant<int, OFF_EDGE> some{};
    const integral_constant<int, OFF_ANY> any{};
    const std::false_type no{};
    const std::true_type yes{};
    if (dt == VA_DTYPE_F32) return offsets || edge ? f(no, any, yes) : f(no, none, yes);
    if (dt == VA_DTYPE_F16) return offsets ? f(no, any, no) : edge ? f(no, some, no) : f(no, none, no);
    return offsets ? f(yes, any, no) : edge ? f(yes, some, no) : f(yes, none, no);
}

va_status check_desc(va_context* ctx, const va_xent_desc* d, const char* who) {
    VA_REQUIRE(ctx, d != nullptr, "%s: NULL description", who);
    VA_REQUIRE(ctx, d->hidden && d->items && d->targets, "%s: NULL pointer", who);
    VA_REQUIRE(ctx, d->rows > 0 && d->num_items > 0 && d->dim > 0, "%s: empty input (%u rows, %u items, %u dimensions)", who, d->rows,
               d->num_items, d->dim);
    VA_REQUIRE(ctx, d->dtype == VA_DTYPE_F32 || d->dtype == VA_DTYPE_F16 || d->dtype == VA_DTYPE_BF16, "%s: unknown type %d", who, int(d->dtype));
    VA_REQUIRE(ctx, d->dim <= VA_XENT_MAX_DIM, "%s: %u dimensions (at most %u)", who, d->dim, VA_XENT_MAX_DIM);
    VA_REQUIRE(ctx, d->num_items < 0xFFFFFF00u && d->rows < 0xFFFFFF00u, "%s: too many rows or items", who);
    VA_REQUIRE(ctx, d->hidden_stride >= d->dim && d->items_stride >= d->dim, "%s: a row stride is below the dimension", who);
    VA_REQUIRE(ctx, std::isfinite(d->scale), "%s: the scale is not finite", who);
    const size_t es = elem_size(d->dtype);
    VA_REQUIRE(ctx, reinterpret_cast<uintptr_t>(d->hidden) % es == 0 && reinterpret_cast<uintptr_t>(d->items) % es == 0,
               "%s: rows or items are not aligned to their type", who);
    return VA_OK;
}

// A scale at which the logits' other unit might overflow: natural units (as with odd offsets).
bool wild_scale(const va_xent_desc* d) { return fabsf(d->scale) > 1e18f; }
// Whether offsets are looked over first, so that usual ones take the shorter epilogue: 16-bit operands, and
// products that are bound by the matrix cores (4096 rows x 262,144 items of 768: the check takes 10 us and
// saves 150; a product that streams its items hides the longer epilogue).
bool worth_checking(const va_xent_desc* d, const Blocks& b) {
    return d->offsets && d->dtype != VA_DTYPE_F32 && !wild_scale(d) && b.shape == 0;
}
va_status find_odd(va_context* ctx, const va_xent_desc* d, uint32_t* odd) {
    xent_odd_kernel<<<dim3(ceil_div(d->num_items, 256)), dim3(256), 0, ctx->stream>>>(
        static_cast<const uint16_t*>(d->items), d->items_stride, d->offsets, d->num_items, d->dim, d->dtype == VA_DTYPE_F16 ? 0x7C00u : 0x7F80u, odd);
    VA_CHECK_LAUNCH(ctx);
    return VA_OK;
}

uint32_t round_up(uint32_t v, uint32_t m) { return (v + m - 1) / m * m; }

// The largest piece of items (a multiple of 256) whose per-item workspace stays within `budget`.
uint32_t piece_items(uint32_t V, size_t per_item, size_t budget) {
    const uint64_t n = std::max<uint64_t>(budget / std::max<size_t>(per_item, 1) / 256, 1) * 256;
    return uint32_t(std::min<uint64_t>(n, round_up(V, 256)));
}

constexpr size_t kPackBudget = size_t(256) << 20;  // packed items of one piece
constexpr size_t kGradBudget = size_t(512) << 20;  // dl of one piece
// Values between dl's rows: with the rows a power of two apart, a tile's 256 rows meet in few memory
// channels.
constexpr uint32_t kRowPad = 64;

}  // namespace
}  // namespace va

using namespace va;

extern "C" {

va_status va_xent_forward(va_context* ctx, const va_xent_desc* d, float* out_loss, float* out_lse, va_reduction reduction, float* out_reduced) {
    if (!ctx) return VA_ERR_INVALID_ARG;
    VA_CHECK_STATUS(check_desc(ctx, d, "va_xent_forward"));
    VA_REQUIRE(ctx, out_loss && out_lse, "va_xent_forward: NULL output");
    VA_REQUIRE(ctx, reduction == VA_REDUCE_MEAN || reduction == VA_REDUCE_SUM || reduction == VA_REDUCE_NONE, "va_xent_forward: unknown reduction %d", int(reduction));
    VA_REQUIRE(ctx, (reduction == VA_REDUCE_NONE) == (out_reduced == nullptr), "va_xent_forward: a reduced loss goes with a reduction");
    DeviceGuard guard(ctx->device);
    const uint32_t T = d->rows, V = d->num_items, D = d->dim, Kp = round_up(D, g16::KC);
    const va_dtype dt = d->dtype;
    const size_t es = elem_size(dt), planes = dt == VA_DTYPE_F32 ? 2 : 1;
    const bool qd = direct(dt, d->hidden, d->hidden_stride, D), xd = direct(dt, d->items, d->items_stride, D);
    const uint32_t piece = xd ? round_up(V, 256) : piece_items(V, packed_bytes(dt, 1, Kp), kPackBudget);
    const uint32_t pieces = ceil_div(V, piece);
    const Blocks bl = blocks_for(ctx, T, std::min(piece, V));
    const bool wild = wild_scale(d), checks = worth_checking(d, bl);
    const uint32_t nq = bl.nq(T);
    // parts per query block: whole multiples of the XCDs when there are that many
    uint32_t parts = std::max(bl.grid / nq, 1u);
    if (parts > kXcds) parts = parts / kXcds * kXcds;
    parts = std::min(parts, bl.nr(std::min(piece, V)));
    const uint32_t last_parts = std::min(parts, bl.nr(V - (pieces - 1) * piece));  // (of the last piece)
    const uint32_t slots = parts * (pieces - 1) + last_parts;

    Scratch sc(ctx);
    const size_t need = (qd ? 0 : Scratch::round(packed_bytes(dt, T, Kp)) + Scratch::round(T * 4ull)) +
                        (xd ? 0 : Scratch::round(packed_bytes(dt, piece, Kp)) + Scratch::round(piece * 4ull)) +
                        Scratch::round(uint64_t(T) * slots * sizeof(float2)) + Scratch::round(T * 4ull) + Scratch::round(4);
    VA_CHECK_STATUS(sc.reserve(need));
    float2* part = sc.carve<float2>(uint64_t(T) * slots);
    float* picked = sc.carve<float>(T);
    uint32_t* odd = nullptr;
    if (checks) {
        odd = sc.carve<uint32_t>(1);
        VA_CHECK_STATUS(fill_u32(ctx, odd, 1, 0));
        VA_CHECK_STATUS(find_odd(ctx, d, odd));
    }
    char* qp = nullptr;
    char* xp = nullptr;
    float* qinv = nullptr;
    float* xinv = nullptr;
    if (!qd) {
        qp = sc.carve<char>(packed_bytes(dt, T, Kp));
        qinv = sc.carve<float>(T);
        VA_CHECK_STATUS(pack(ctx, dt, d->hidden, d->hidden_stride, T, D, Kp, nullptr, nullptr, 0.0f, qp, qinv));
    }
    if (!xd) {
        xp = sc.carve<char>(packed_bytes(dt, piece, Kp));
        xinv = sc.carve<float>(piece);
    }
    VA_CHECK_STATUS(sc.verify(need));
    for (uint32_t c = 0; c < pieces; ++c) {
        const uint32_t v0 = c * piece, n = std::min(piece, V - v0);
        const char* items = at(d->items, d->items_stride, v0, dt);
        if (!xd) VA_CHECK_STATUS(pack(ctx, dt, items, d->items_stride, n, D, Kp, nullptr, nullptr, 0.0f, xp, xinv));
        g16::Args a;
        a.q = g16::Operand{qd ? d->hidden : qp, qd ? d->hidden_stride * es : uint64_t(Kp) * 2 * planes, T, Kp * 2, Kp * 2};
        a.x = g16::Operand{xd ? items : xp, xd ? d->items_stride * es : uint64_t(Kp) * 2 * planes, n, Kp * 2, Kp * 2};
        a.kstages = Kp / g16::KC;
        a.nq = nq;
        a.nr = bl.nr(n);
        a.parts = c + 1 < pieces ? parts : last_parts;
        VA_CHECK_STATUS(by_shape(bl.shape, [&](auto sh) {
            using Sh = decltype(sh);
            return by_type(dt, d->offsets || wild, n % Sh::TR, [&](auto bf, auto off, auto pl) {
                LseEpi<Sh, decltype(off)::value, decltype(pl)::value> e;
                e.a = LogitArgs{d->offsets ? d->offsets + v0 : nullptr, odd, qinv, xinv, d->scale, T, n};
                e.targets = d->targets;
                e.item0 = v0;
                e.picked = picked;
                e.part = part;
                e.slots = slots;
                e.slot0 = c * parts;
                return g16::launch<decltype(bf)::value, decltype(pl)::value, false, false>(ctx, a, e);
            });
        }));
    }
    xent_finish_kernel<<<dim3(ceil_div(T, 4)), dim3(256), 0, ctx->stream>>>(d->targets, T, V, d->ignore_index, part, picked, slots, out_loss, out_lse);
    VA_CHECK_LAUNCH(ctx);
    if (out_reduced) {
        xent_reduce_kernel<<<dim3(1), dim3(1024), 0, ctx->stream>>>(out_loss, d->targets, T, d->ignore_index, reduction == VA_REDUCE_MEAN, out_reduced);
        VA_CHECK_LAUNCH(ctx);
    }
    return VA_OK;
}

va_status va_xent_backward(va_context* ctx, const va_xent_desc* d, const float* lse, va_reduction reduction, const float* grad,
                           void* out_grad_hidden, uint64_t grad_hidden_stride, void* out_grad_items, uint64_t grad_items_stride) {
    if (!ctx) return VA_ERR_INVALID_ARG;
    VA_CHECK_STATUS(check_desc(ctx, d, "va_xent_backward"));
    VA_REQUIRE(ctx, lse, "va_xent_backward: NULL log-sum-exp");
    VA_REQUIRE(ctx, reduction == VA_REDUCE_MEAN || reduction == VA_REDUCE_SUM || reduction == VA_REDUCE_NONE, "va_xent_backward: unknown reduction %d", int(reduction));
    VA_REQUIRE(ctx, reduction != VA_REDUCE_NONE || grad, "va_xent_backward: without a reduction the rows' gradients are needed");
    VA_REQUIRE(ctx, out_grad_hidden || out_grad_items, "va_xent_backward: no output");
    VA_REQUIRE(ctx, (!out_grad_hidden || grad_hidden_stride >= d->dim) && (!out_grad_items || grad_items_stride >= d->dim),
               "va_xent_backward: a gradient's row stride is below the dimension");
    DeviceGuard guard(ctx->device);
    const uint32_t T = d->rows, V = d->num_items, D = d->dim, Kp = round_up(D, g16::KC), Dp = round_up(D, 4);
    const va_dtype dt = d->dtype;
    const bool f32 = dt == VA_DTYPE_F32;
    const size_t es = elem_size(dt), planes = f32 ? 2 : 1;
    // masked items may hold anything, and dh sums over them: their rows are read as zeros, from a copy, unless
    // they are known to be finite
    const bool in_place = direct(dt, d->items, d->items_stride, D);
    const bool checks = worth_checking(d, blocks_for(ctx, T, V)), wild = wild_scale(d);
    const bool xd = in_place && !d->offsets;
    VA_REQUIRE(ctx, (!out_grad_hidden || reinterpret_cast<uintptr_t>(out_grad_hidden) % es == 0) &&
                        (!out_grad_items || reinterpret_cast<uintptr_t>(out_grad_items) % es == 0),
               "va_xent_backward: a gradient is not aligned to its type");
    // the piece: dl and the packed items within their budgets, dl's rows within the products' 32-bit offsets
    uint32_t piece = piece_items(V, uint64_t(T) * 2 * planes, kGradBudget);
    if (!xd) piece = std::min(piece, piece_items(V, packed_bytes(dt, 1, Kp), kPackBudget));
    piece = std::min<uint32_t>(piece, (uint32_t(kDmaMaxBytes / 256 / 2) - kRowPad) / uint32_t(planes) / 256 * 256);
    const uint32_t pieces = ceil_div(V, piece);
    const uint32_t Vpmax = round_up(std::min(piece, V), g16::KC);
    const uint32_t most = std::min(piece, V);
    // dh has few tiles and a long sum: shares of it until the chip is filled once, eight stages at least each
    const uint32_t kst = Vpmax / g16::KC * (f32 ? 3 : 1), shares = std::max(kst / 8, 1u);
    const Blocks lb = blocks_for(ctx, T, most), hb = blocks_for(ctx, T, D, shares), wb = blocks_for(ctx, most, D);
    const uint32_t parts = std::min(std::max(hb.grid / (hb.nq(T) * hb.nr(D)), 1u), shares);

    const size_t p_bytes = uint64_t(T) * (Vpmax * planes + kRowPad) * 2;
    const size_t share_n = out_grad_hidden ? uint64_t(parts) * T * Dp : 0;
    const size_t qp_bytes = packed_bytes(dt, T, Kp), xp_bytes = xd ? 0 : packed_bytes(dt, std::min(piece, V), Kp);
    Scratch sc(ctx);
    const size_t need = Scratch::round(p_bytes) + Scratch::round(share_n * 4) + Scratch::round(qp_bytes) + Scratch::round(xp_bytes) +
                        2 * Scratch::round(T * 4ull) + Scratch::round(piece * 4ull) + Scratch::round(32);
    VA_CHECK_STATUS(sc.reserve(need));
    uint16_t* p = sc.carve<uint16_t>(p_bytes / 2);
    float* share = sc.carve<float>(share_n);
    char* qp = sc.carve<char>(qp_bytes);
    char* xp = sc.carve<char>(xp_bytes);
    float* gk = sc.carve<float>(T);
    float* qinv = sc.carve<float>(T);
    float* xinv = sc.carve<float>(piece);
    float* mul = sc.carve<float>(8);
    uint32_t* absmax = reinterpret_cast<uint32_t*>(mul + 1);  // of the hidden rows, of the items
    uint32_t* odd = checks ? absmax + 2 : nullptr;
    VA_CHECK_STATUS(sc.verify(need));

    xent_gradient_kernel<<<dim3(1), dim3(1024), 0, ctx->stream>>>(grad, d->targets, T, V, d->ignore_index, int(reduction), d->scale, gk, mul, absmax);
    VA_CHECK_LAUNCH(ctx);
    if (f32) {
        // one scale a tensor: both tensors are summed over in the second products
        auto top = [&](const void* src, uint64_t ld, uint32_t R, const float* drop, float drop_if, uint32_t* out) {
            absmax_kernel<<<dim3(std::min<uint32_t>(ceil_div(R, 16), 512)), dim3(256), 0, ctx->stream>>>(static_cast<const float*>(src), ld, R, D, drop, drop_if, out);
        };
        top(d->hidden, d->hidden_stride, T, gk, 0.0f, absmax);
        top(d->items, d->items_stride, V, d->offsets, -INFINITY, absmax + 1);
        VA_CHECK_LAUNCH(ctx);
    }
    if (checks) VA_CHECK_STATUS(find_odd(ctx, d, odd));
    VA_CHECK_STATUS(pack(ctx, dt, d->hidden, d->hidden_stride, T, D, Kp, f32 ? absmax : nullptr, gk, 0.0f, qp, qinv));
    // read in place unless a masked item is odd (the copy then has the rows' own pitch)
    const bool either = in_place && checks && d->items_stride == Kp;
    for (uint32_t c = 0; c < pieces; ++c) {
        const uint32_t v0 = c * piece, n = std::min(piece, V - v0), Vp = round_up(n, g16::KC);
        const char* items = at(d->items, d->items_stride, v0, dt);
        const float* offsets = d->offsets ? d->offsets + v0 : nullptr;
        if (!xd) VA_CHECK_STATUS(pack(ctx, dt, items, d->items_stride, n, D, Kp, f32 ? absmax + 1 : nullptr, offsets, -INFINITY, xp, xinv, either ? odd : nullptr));
        const g16::Operand rows{qp, uint64_t(Kp) * 2 * planes, T, Kp * 2, Kp * 2};
        g16::Operand cols{xd || either ? items : xp, xd ? d->items_stride * es : uint64_t(Kp) * 2 * planes, n, Kp * 2, Kp * 2};
        if (either) {
            cols.other = xp;
            cols.choose = odd;
        }
        const uint32_t pitch = Vp * uint32_t(planes) + kRowPad;
        const g16::Operand dl{p, uint64_t(pitch) * 2, T, Vp * 2, Vp * 2};
        g16::Args a;
        a.q = rows;
        a.x = cols;
        a.kstages = Kp / g16::KC;
        a.nq = lb.nq(T);
        a.nr = lb.nr(n);
        a.parts = 1;
        VA_CHECK_STATUS(by_shape(lb.shape, [&](auto sh) {
            using Sh = decltype(sh);
            return by_type(dt, offsets || wild, n % Sh::TR, [&](auto bf, auto off, auto pl) {
                GradEpi<Sh, decltype(bf)::value, decltype(off)::value, decltype(pl)::value> e;
                e.a = LogitArgs{offsets, odd, qinv, xinv, d->scale, T, n};
                e.gk = gk;
                e.lse = lse;
                e.targets = d->targets;
                e.item0 = v0;
                e.p = p;
                e.Vp = Vp;
                e.pitch = pitch;
                return g16::launch<decltype(bf)::value, decltype(pl)::value, false, false>(ctx, a, e);
            });
        }));
        if (out_grad_hidden) {
            // dh[t][d] = sum_j dl[t][j] w[j][d]: the items are stored across the sum
            g16::Args b;
            b.q = dl;
            b.x = cols;
            b.kstages = Vp / g16::KC;
            b.nq = hb.nq(T);
            b.nr = hb.nr(D);
            b.parts = parts;
            VA_CHECK_STATUS(by_shape(hb.shape, [&](auto sh) {
                const ShareEpi<decltype(sh)> e{share, T, D, Dp, c == 0};
                return f32 ? g16::launch<false, true, false, true>(ctx, b, e)
                           : dt == VA_DTYPE_F16 ? g16::launch<false, false, false, true>(ctx, b, e) : g16::launch<true, false, false, true>(ctx, b, e);
            }));
        }
        if (out_grad_items) {
            // dw[j][d] = sum_t dl[t][j] h[t][d]: both are
            g16::Args b;
            b.q = dl;
            b.x = rows;
            b.kstages = ceil_div(T, g16::KC);
            b.nq = wb.nq(n);
            b.nr = wb.nr(D);
            b.parts = 1;
            const uintptr_t o = reinterpret_cast<uintptr_t>(out_grad_items) + uint64_t(v0) * grad_items_stride * es;
            const bool vec = o % (4 * es) == 0 && grad_items_stride % 4 == 0;
            VA_CHECK_STATUS(by_shape(wb.shape, [&](auto sh) {
                auto go = [&](auto DT, auto bf, auto pl) {
                    constexpr int kT = decltype(DT)::value;
                    ItemGradEpi<decltype(sh), kT> e{reinterpret_cast<ElemT<kT>*>(o), grad_items_stride, n, D, mul, absmax, vec};
                    return g16::launch<decltype(bf)::value, decltype(pl)::value, true, true>(ctx, b, e);
                };
                return f32 ? go(std::integral_constant<int, VA_DTYPE_F32>(), std::false_type(), std::true_type())
                           : dt == VA_DTYPE_F16 ? go(std::integral_constant<int, VA_DTYPE_F16>(), std::false_type(), std::false_type())
                                                : go(std::integral_constant<int, VA_DTYPE_BF16>(), std::true_type(), std::false_type());
            }));
        }
    }
    if (out_grad_hidden) {
        const dim3 grid(ceil_div(uint64_t(T) * (Dp / 4), 64));
        auto sum = [&](auto k, auto* o) {
            k<<<grid, dim3(256), 0, ctx->stream>>>(share, parts, T, D, Dp, gk, mul, absmax + 1, o, grad_hidden_stride);
        };
        if (f32) sum(&share_sum_kernel<VA_DTYPE_F32>, static_cast<float*>(out_grad_hidden));
        else if (dt == VA_DTYPE_F16) sum(&share_sum_kernel<VA_DTYPE_F16>, static_cast<_Float16*>(out_grad_hidden));
        else sum(&share_sum_kernel<VA_DTYPE_BF16>, static_cast<__bf16*>(out_grad_hidden));
        VA_CHECK_LAUNCH(ctx);
    }
    return VA_OK;
}

}  // extern "C"
