// va_xent.hpp — what the two directions of the softmax cross entropy share (va_xent.hip, va_xent_grad.hip):
// element types, the logits in a product's epilogue, the preparation of operands, the choice of tiles.
#pragma once

#include <algorithm>
#include <cfloat>
#include <cmath>

#include "va_gemm16.hpp"

namespace va {
namespace xent {

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

// ---- the logits' epilogues -------------------------------------------------------------------------
// The offsets of a launch: none, none but -inf for the items missing from the last tile, or any.
enum Offsets : int { OFF_NONE = 0, OFF_EDGE = 1, OFF_ANY = 2 };

struct LogitArgs {
    const float* offsets;  // of the launch's first item (nullptr: zeros)
    const uint32_t* odd;   // OFF_ANY: zero if no masked item's logit can be NaN or inf and no offset is near fp32's
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
// operands (whose results have the digits to show the extra rounding) keep natural units.
template <int KIND, int OFF, int TR>
struct LogitShared {
    float off[OFF ? TR : 1];
    float inv[KIND == g16::PLANES ? TR : 1];
};
template <bool NATURAL, int KIND, int OFF, int TR>
__device__ __forceinline__ f32x4 logits4(const LogitShared<KIND, OFF, TR>& sm, const f32x16& acc, int j, int r, float c) {
    f32x4 v;
    f32x4 o{}, x{};
    // these reads stay here, and the groups in order: mixed, a tile's would fill the registers
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (OFF != OFF_NONE) o = *reinterpret_cast<const f32x4*>(sm.off + r);
    if constexpr (KIND == g16::PLANES) x = *reinterpret_cast<const f32x4*>(sm.inv + r);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float a = acc[4 * j + e];
        // (the factors first: an item's alone may take the sum past fp32 where the row's brings it back)
        const float f = KIND == g16::PLANES ? x[e] * c : c;
        if constexpr (OFF == OFF_NONE) v[e] = a * f;
        else v[e] = NATURAL && o[e] == -INFINITY ? -INFINITY : fmaf(a, f, o[e]);
    }
    return v;
}
template <bool NATURAL>
__device__ __forceinline__ float exp_diff(float v, float ref) {
    return __builtin_amdgcn_exp2f(NATURAL ? (v - ref) * kLog2e : v - ref);
}
// whether a launch keeps natural units (uniform)
template <int KIND, int OFF>
__device__ __forceinline__ bool keeps_natural(const LogitArgs& a) {
    if constexpr (KIND >= g16::PLANES) return true;
    if constexpr (OFF != OFF_ANY) return false;
    return __builtin_amdgcn_readfirstlane(a.odd ? *a.odd : 1u) != 0u;
}
__device__ __forceinline__ float offset_of(const LogitArgs& a, bool in, uint32_t r, bool natural) {
    const float o = !in ? -INFINITY : a.offsets ? a.offsets[r] : 0.0f;
    return natural ? o : o * kLog2e;
}

// ---- host: operands and launches -----------------------------------------------------------------------
inline size_t elem_size(va_dtype t) { return t == VA_DTYPE_F32 ? 4 : 2; }
inline uint32_t round_up(uint32_t v, uint32_t m) { return (v + m - 1) / m * m; }
inline const char* row_at(const void* p, uint64_t ld, uint64_t row, va_dtype dt) { return static_cast<const char*>(p) + row * ld * elem_size(dt); }

// Rows that a product can read where they are: dwords, 256 of them (a tile's) within the reach of its loads' offsets.
inline bool in_place_rows(va_dtype dt, const void* p, uint64_t ld) {
    return ld * elem_size(dt) % 4 == 0 && reinterpret_cast<uintptr_t>(p) % 4 == 0 && ld <= kDmaMaxBytes / 256 / elem_size(dt);
}
// Bytes of a row of D values in place, and of one of a copy: whole stages.
inline uint32_t row_bytes(va_dtype dt, uint32_t D) { return round_up(D * uint32_t(elem_size(dt)), 4); }
inline uint32_t copy_bytes(int kind, uint32_t D) { return round_up(D * uint32_t(g16::size_of(kind)), g16::ROWB); }
// Operands over rows in place and over copies.
inline g16::Operand in_place(va_dtype dt, const void* p, uint64_t ld, uint32_t rows, uint32_t D) {
    g16::Operand o;
    o.p = p;
    o.pitch = ld * elem_size(dt);
    o.rows = rows;
    o.width = row_bytes(dt, D);
    return o;
}
inline g16::Operand copied(int kind, const void* p, uint32_t rows, uint32_t D) {
    g16::Operand o;
    o.p = p;
    o.pitch = copy_bytes(kind, D);
    o.rows = rows;
    o.width = uint32_t(o.pitch);
    return o;
}

// fp32 operands as they are or as planes.  Planes cost passes over the items that write copies
// (32 bytes a value of a training step, where fp32 as it is takes 16), and with the second products in SPLIT save
// 7/10 of the matrix cores' time: they win as soon as that counts.  Loss and gradients, as it is and in planes: 10 x 5000 x
// 512 56 and 75 us, 30 x 100,000 x 384 194 and 291, 48 x 100,000 x 768 546 and 614; 60 x 30,000 x 512 170 and 144,
// 33 x 5000 x 512 84 and 82.
inline int kind_of(va_dtype dt, uint32_t rows, uint32_t items) {
    if (dt == VA_DTYPE_F16) return g16::F16;
    if (dt == VA_DTYPE_BF16) return g16::BF16;
    return rows <= 32 || (rows <= 64 && items >= 65536) ? g16::F32 : g16::PLANES;
}

// Which rows of a copy are zeros: those whose drop value equals drop_if (drop may be nullptr: none).
struct Drop {
    const float* value = nullptr;
    float is = 0.0f;
};
// A copy of R rows as `kind` (not PLANES) wants them; nothing where *run_if is zero.
va_status make_copy(va_context* ctx, int kind, const void* src, uint64_t ld, uint32_t R, uint32_t D, Drop drop, void* dst,
                    const uint32_t* run_if = nullptr);
// The planes of R fp32 rows: scaled by the power of two that puts the row's largest entry near 2^14, and its
// inverse to inv[row].
struct Planes {
    const void* src = nullptr;
    uint64_t ld = 0;
    uint32_t R = 0;
    Drop drop;
    void* dst = nullptr;
    float* inv = nullptr;
};
// Of one matrix, or of two in one launch (b.R = 0: none).
va_status make_planes(va_context* ctx, uint32_t D, Planes a, Planes b = {});
// *odd = 1 (0 before) if a masked item holds NaN, inf or values whose products with the hidden rows may overflow, or an
// offset is finite and near fp32's limits
va_status find_odd(va_context* ctx, const va_xent_desc* d, uint32_t* odd);

// The description with the strides of single rows set, checked.
va_status check_desc(va_context* ctx, const va_xent_desc* desc, const char* who, va_xent_desc& d);
// A scale at which the logits' other unit might overflow: natural units (as with odd offsets).
inline bool wild_scale(const va_xent_desc* d) { return fabsf(d->scale) > 1e18f; }

// Stages of a product along rows of D values.
inline uint32_t stages_of(int kind, uint32_t D) { return copy_bytes(kind, D) / g16::ROWB; }

// The shapes of a product's workgroups.  Deep ones have four slots: alone on their CU, three stages in flight.
// Sliced ones (logits) have smaller tiles, with the stages of each shared among four waves.
using Medium = g16::Shape<2, 2>;
using Small = g16::Shape<1, 2>;
using DeepMedium = g16::Shape<2, 2, 2, 4>;
using DeepSmall = g16::Shape<1, 2, 2, 4>;
using Sliced = g16::Shape<1, 1, 2, 2, 4>;
// Planes' 256 x 256, for logits: eight waves of 128 x 64, whose registers hold both planes' fragments beside the sums.
// 4096 x 50,000 x 1024, loss: 1.03 ms, with 128 x 128 tiles 1.18; 2808 x 21,283 x 512 with gradients 846 and 860 us.
// (For dh too, 400 x 10,000 x 768 took 188 us instead of 182, the 2808 rows 833 instead of 846.)
using Wide = g16::Shape<2, 4, 4>;
// 32 queries, along k: fp32 products as they are, which 64 padded ones would bind to the matrix cores.
using Narrow = g16::Shape<1, 2, 1>;
using SlicedNarrow = g16::Shape<1, 1, 1, 2, 4>;
enum ShapeId : int { LARGE = 0, MEDIUM = 1, SMALL = 2, NARROW = 3, DEEP_MEDIUM = 4, DEEP_SMALL = 5, SLICED = 6, SLICED_NARROW = 7 };
template <int KIND, class F>
va_status by_shape(int shape, F&& f) {
    if constexpr (KIND != g16::PLANES && KIND != g16::SPLIT)
        if (shape == LARGE) return f(g16::Large());
    switch (shape) {
        case MEDIUM: return f(Medium());
        case SMALL: return f(Small());
        case DEEP_MEDIUM: return f(DeepMedium());
        default: return f(DeepSmall());
    }
}
template <int KIND, class F>
va_status by_shape_of(int shape, F&& f) {
    if constexpr (KIND == g16::F32)
        if (shape == NARROW) return f(Narrow());
    return by_shape<KIND>(shape, f);
}
template <int KIND, class F>
va_status by_logit_shape(int shape, F&& f) {
    if constexpr (KIND == g16::F32)
        if (shape == SLICED_NARROW) return f(SlicedNarrow());
    if constexpr (KIND == g16::PLANES)
        if (shape == LARGE) return f(Wide());
    if (shape == SLICED) return f(Sliced());
    return by_shape_of<KIND>(shape, f);
}
struct Blocks {
    int shape;              // ShapeId
    uint32_t tq, tr, grid;  // grid: the most workgroups of a launch
    uint32_t parts;         // shares of the sum of each tile
    uint32_t nq(uint64_t Q) const { return uint32_t((Q + tq - 1) / tq); }
    uint32_t nr(uint64_t R) const { return uint32_t((R + tr - 1) / tr); }
};
// The shape with the least time: rounds of the chip's workgroups, by what a round takes.  256 x 256 tiles move
// the fewest operand bytes, but a small or ragged product fills few of them: with as many stages each, a round of
// 128 x 128 tiles (two a CU) takes 0.50 to 0.56 of one of 256 x 256 in short products (0.61 to 0.75 in long ones
// of whole rounds, which the rule gives to the large tiles), one of 64 x 128 (three a CU) 0.48 to 0.59; measured on
// 1023 x 49,999 x 300 and 4096 x 262,144 x 768.  `shares`: how many shares of the sum the caller can make.  `stages`:
// those of a tile, where it may be sliced (logits; a sum shared among workgroups has short chains already: dh of
// 32 x 6979 x 1536 took 14 us sliced, 8 as it is).  Sliced pays where stages are many and tiles few.  64-query
// tiles, scoring, sliced and as they are: 32 x 6979 x 1536 (110 tiles, 24 stages; the
// logits alone) 12.6 and 16.4 us, 37 x 5510 x 1024 in fp32 (87, 32) 34 and 43; 64 x 9000 x 1024 (141, 16) 22.7 and 22.3,
// 64 x 16,000 x 640 (250, 10) 25.8 and 20.3, 1 x 10,000 x 512 (157, 8) 12.9 and 12.7 (but x 768 13.1 and 14.3).
// 32-query ones: 4 x 36,909 x 768 (577, 24) 38 and 58, 10 x 10,000 x 100 (157, 4) 15.0 and 16.4; 30 x 200,000 x 256
// (3125, 8) 70 and 63.
inline Blocks blocks_for(const va_context* ctx, int kind, uint64_t Q, uint64_t R, uint32_t shares = 1, bool narrow = false, uint32_t stages = 0) {
    Blocks all[4] = {{LARGE, 256, 256, g16::grid_max<g16::Large>(ctx), 1},
                     {MEDIUM, 128, 128, g16::grid_max<Medium>(ctx), 1},
                     {SMALL, 64, 128, g16::grid_max<Small>(ctx), 1},
                     {NARROW, 32, 128, g16::grid_max<Narrow>(ctx), 1}};
    const double round[4] = {1.0, 0.56, 0.5, 0.5};
    int best = -1;
    double least = 0.0;
    for (int i = narrow ? 3 : kind == g16::SPLIT ? 1 : 0; i < (narrow ? 4 : 3); ++i) {
        const uint64_t tiles = uint64_t(all[i].nq(Q)) * all[i].nr(R);
        all[i].parts = uint32_t(std::min<uint64_t>(std::max<uint64_t>(all[i].grid / tiles, 1), shares));
        const double t = double((tiles * all[i].parts + all[i].grid - 1) / all[i].grid) / all[i].parts * round[i];
        if (best < 0 || t < least) {
            best = i;
            least = t;
        }
    }
    Blocks b = all[best];
    // Fewer tiles than CUs: the time is that of one tile's loads, and of a wave's chain through its stages.
    const uint64_t cus = uint64_t(ctx->num_cus);
    if (narrow) {
        const Blocks f{SLICED_NARROW, 32, 64, g16::grid_max<SlicedNarrow>(ctx), 1};
        if (stages >= 4 && f.nr(R) * uint64_t(f.nq(Q)) <= 4 * cus) return f;
        return b;
    }
    const Blocks f{SLICED, 64, 64, g16::grid_max<Sliced>(ctx), 1};
    if (stages >= 12 && uint64_t(f.nq(Q)) * f.nr(R) <= cus / 2) return f;
    if (b.shape != LARGE && uint64_t(b.nq(Q)) * b.nr(R) * b.parts <= cus) {
        b.shape += DEEP_MEDIUM - MEDIUM;
        b.grid = g16::grid_max<DeepSmall>(ctx);
    }
    return b;
}

// f(kind, offsets) of a launch; edge: the last tile is not whole
template <class F>
va_status by_kind(int kind, bool offsets, bool edge, F&& f) {
    using std::integral_constant;
    const integral_constant<int, OFF_NONE> none{};
    const integral_constant<int, OFF_EDGE> some{};
    const integral_constant<int, OFF_ANY> any{};
    const auto go = [&](auto k) { return offsets ? f(k, any) : edge ? f(k, some) : f(k, none); };
    if (kind == g16::F16) return go(integral_constant<int, g16::F16>());
    if (kind == g16::BF16) return go(integral_constant<int, g16::BF16>());
    const auto full = [&](auto k) { return offsets || edge ? f(k, any) : f(k, none); };  // (natural units anyway)
    if (kind == g16::PLANES) return full(integral_constant<int, g16::PLANES>());
    return full(integral_constant<int, g16::F32>());
}
// f(kind) of a product with dl
template <class F>
va_status by_second(int kind, F&& f) {
    if (kind == g16::F16) return f(std::integral_constant<int, g16::F16>());
    if (kind == g16::BF16) return f(std::integral_constant<int, g16::BF16>());
    if (kind == g16::SPLIT) return f(std::integral_constant<int, g16::SPLIT>());
    return f(std::integral_constant<int, g16::F32>());
}
// The element type of a kind's tensors.
constexpr int dtype_of(int kind) { return kind == g16::F16 ? VA_DTYPE_F16 : kind == g16::BF16 ? VA_DTYPE_BF16 : VA_DTYPE_F32; }

// The largest piece of items (a multiple of 256) whose per-item workspace stays within `budget`.
inline uint32_t piece_items(uint32_t V, size_t per_item, size_t budget) {
    const uint64_t n = std::max<uint64_t>(budget / std::max<size_t>(per_item, 1) / 256, 1) * 256;
    return uint32_t(std::min<uint64_t>(n, round_up(V, 256)));
}
constexpr size_t kCopyBudget = size_t(256) << 20;  // copied items of one piece

}  // namespace xent
}  // namespace va
