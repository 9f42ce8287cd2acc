// va_xent_grad.hip — the gradient of the softmax cross entropy (va_xent.hip has the formulas).
//
// Launches of a call: the rows' factors and the hidden rows ended by zeros, then per piece of the items (fp32 rows
// for a product in planes: those first) the logits again with dl as their epilogue's result, dh += dl w,
// dw = dl^T h; at the end the shares of dh summed, where there are several.  dl of a piece stays within
// kGradBudget, or is that of 256 items where the rows are too many for it: a piece of 65,536 items for 4096 rows (pieces of 8,192 to 32,768, whose dl stays in the last
// level cache, ran 35 to 6 % slower: each product then ends in a round of half-idle CUs).
//
// What bounds it: the matrix cores.  A piece of 65,536 items by 4096 rows of 768 in bf16 takes 0.47 ms for the logits and dl
// (0.87 PFLOP/s; dl's 0.5 GB leave during the products), 0.39 for dh and 0.35 for dw (1.05 and 1.17); 1023 x 49,999 x
// 300 in fp16 63, 47 and 50 us.
#include "va_xent.hpp"

namespace va {
namespace {

using namespace xent;

// ---- preparation -----------------------------------------------------------------------------------------
struct PrepareArgs {
    const float* grad;
    const int64_t* targets;
    uint32_t T, V;
    int64_t ignore;
    int reduction;
    float scale, top;
    float* gk;
    float* mul;
    uint32_t* odd;  // cleared
};

// gk[t] = g_t c, *mul = scale / c: g_t is the gradient that reaches the row's loss, 0 for a row without a
// target, c takes the largest |g_t| to `top`.  Every workgroup finds c for itself and takes rows_per rows; with
// src it also copies them, ended by zeros (rows without a gradient: zeros).
template <class U>
__global__ __launch_bounds__(256) void xent_prepare_kernel(PrepareArgs a, uint32_t rows_per, const U* __restrict__ src, uint64_t ld, uint32_t D, uint32_t Kp,
                                                           U* __restrict__ dst) {
    __shared__ float tops[4];
    __shared__ uint32_t cnt[4];
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.odd = 0;
    float m = 0.0f;
    uint32_t c = 0;
    for (uint32_t t = threadIdx.x; t < a.T; t += 256) {
        const int64_t y = a.targets[t];
        if (y == a.ignore) continue;
        ++c;
        if (a.reduction == VA_REDUCE_NONE && y >= 0 && y < int64_t(a.V)) m = fmaxf(m, fabsf(a.grad[t]));
    }
    for (int d = 32; d; d >>= 1) {
        m = fmaxf(m, __shfl_xor(m, d));
        c += __shfl_xor(c, d);
    }
    if ((threadIdx.x & 63) == 0) {
        tops[threadIdx.x >> 6] = m;
        cnt[threadIdx.x >> 6] = c;
    }
    __syncthreads();
    m = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    c = (cnt[0] + cnt[1]) + (cnt[2] + cnt[3]);
    float g = 1.0f;
    if (a.reduction != VA_REDUCE_NONE) {
        if (a.grad) g = *a.grad;
        if (a.reduction == VA_REDUCE_MEAN) g /= float(max(c, 1u));
        m = fabsf(g);
    }
    if (!(m > 0.0f) || !(m < INFINITY)) m = a.top;
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.mul = a.scale * (m / a.top);
    auto of_row = [&](uint32_t t) {
        const int64_t y = a.targets[t];
        return y != a.ignore && y >= 0 && y < int64_t(a.V) ? (a.reduction == VA_REDUCE_NONE ? a.grad[t] : g) / m * a.top : 0.0f;
    };
    const uint32_t t0 = blockIdx.x * rows_per, t1 = min(a.T, t0 + rows_per);
    for (uint32_t t = t0 + threadIdx.x; t < t1; t += 256) a.gk[t] = of_row(t);
    if (!src) return;
    constexpr int E = 16 / sizeof(U);
    typedef U UxE __attribute__((ext_vector_type(E), aligned(sizeof(U))));
    const uint32_t per = Kp / E;
    for (uint32_t i = threadIdx.x; i < (t1 - t0) * per; i += 256) {
        const uint32_t t = t0 + i / per, k = i % per * E;
        const U* s = src + t * ld + k;
        UxE v = {};
        if (of_row(t) != 0.0f) {
            if (k + E <= D) {
                v = *reinterpret_cast<const UxE*>(s);
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) v[e] = k + e < D ? s[e] : U(0);
            }
        }
        *reinterpret_cast<u32x4*>(dst + uint64_t(t) * Kp + k) = __builtin_bit_cast(u32x4, v);
    }
}

// dl of the piece's items, p[t][j]: Vp values a row in 16 bits (fp32 rows: fp32), zeros past the last item, rows `pitch`
// bytes apart.
template <class Sh, int KIND, int OFF>
struct GradEpi {
    using Shape = Sh;
    static constexpr int TQ = Sh::TQ, TR = Sh::TR;
    static constexpr bool kWalk = false, kStores = true;
    LogitArgs a;
    const float* gk;   // g_t times dl's factor (0: the row has no gradient)
    const float* lse;
    const int64_t* targets;
    uint32_t item0;    // the piece's first item
    char* p;
    uint32_t Vp, pitch;
    struct Shared : LogitShared<KIND, OFF, TR> {
        float gk[TQ], lse[TQ];
        uint32_t target[TQ];  // within the piece (any larger value: elsewhere)
        float inv_q[KIND == g16::PLANES ? TQ : 1];
    };
    struct State {
        float off, inv, gk, lse, qinv;
        uint32_t target;
        bool natural;
    };
    template <class Tile>
    __device__ void begin(State& s, Shared&, const Tile&) {
        s.natural = keeps_natural<KIND, OFF>(a);
    }
    template <class Tile>
    __device__ void load(State& s, const Tile& t, int tid) {
        const uint32_t r = t.rb * TR + uint32_t(tid), q = t.qb * TQ + uint32_t(tid);
        const bool in = tid < TR && r < a.items, qin = tid < TQ && q < a.rows;
        if constexpr (OFF != OFF_NONE) s.off = offset_of(a, in, r, s.natural);
        if constexpr (KIND == g16::PLANES) {
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
        if constexpr (KIND == g16::PLANES)
            if (tid < TR) sm.inv[tid] = s.inv;
        if (tid >= TQ) return;
        if constexpr (KIND == g16::PLANES) sm.inv_q[tid] = s.qinv;
        sm.gk[tid] = s.gk;
        sm.lse[tid] = s.lse;
        sm.target[tid] = s.target;
    }
    // The wave's 4 KiB of LDS hold 32 rows of 128 bytes of dl (64 items in 16 bits, 32 in fp32), 16-byte chunks
    // swizzled by t & 7 (the writes and the reads then touch every bank equally); whole 128-byte lines go
    // out.  (Stored straight from the accumulators, 8 bytes a lane, a tile took three times as long.)
    __device__ void put(const char* spare, const g16::Lane<Sh::NB>& ln, const uint32_t q0, uint64_t at) {
        const int lane = ln.hh * 32 + ln.l32;
        asm volatile("" ::: "memory");  // the writes come first (a wave's LDS accesses execute in order)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int t = 8 * i + (lane >> 3), c = lane & 7;
            const u32x4 v = *reinterpret_cast<const u32x4*>(spare + t * 128 + 16 * (c ^ (t & 7)));
            if (q0 + t < a.rows) *reinterpret_cast<u32x4*>(p + uint64_t(q0 + t) * pitch + at + 16 * c) = v;
        }
        asm volatile("" ::: "memory");  // and the reads before what is written next
    }
    // dl of the lane's 16 items of one block (m) to LDS.  TARGETS: one of the wave's rows
    // has its target among the block's items
    template <bool NATURAL, bool TARGETS>
    __device__ void block(Shared& sm, const g16::Lane<Sh::NB>& ln, f32x16 (&acc)[2][Sh::NB], uint32_t y, int m, int n, char* spare) {
        const float g = sm.gk[ln.q(n)], ref = sm.lse[ln.q(n)];
        const float c = (KIND == g16::PLANES ? a.scale * sm.inv_q[ln.q(n)] : a.scale) * (NATURAL ? 1.0f : kLog2e);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int r = ln.r(m, j);
            const f32x4 v = logits4<NATURAL, KIND, OFF, TR>(sm, acc[m][n], j, r, c);
            uint16_t b[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float d = exp_diff<NATURAL>(v[e], ref);
                if (TARGETS && y == uint32_t(r + e) && v[e] != -INFINITY) d -= 1.0f;
                d *= g;
                if constexpr (KIND >= g16::PLANES) acc[m][n][4 * j + e] = d;
                else b[e] = bits16<KIND == g16::BF16>(d);
            }
            if constexpr (KIND >= g16::PLANES) {
                f32x4 d;
#pragma unroll
                for (int e = 0; e < 4; ++e) d[e] = acc[m][n][4 * j + e];
                *reinterpret_cast<f32x4*>(spare + ln.l32 * 128 + 16 * ((2 * j + ln.hh) ^ (ln.l32 & 7))) = d;
            } else {
                *reinterpret_cast<uint2*>(spare + ln.l32 * 128 + 16 * ((4 * m + j) ^ (ln.l32 & 7)) + 8 * ln.hh) =
                    make_uint2(b[0] | uint32_t(b[1]) << 16, b[2] | uint32_t(b[3]) << 16);
            }
        }
    }
    template <class Tile, class Settle>
    __device__ void tile(State& s, Shared& sm, const g16::Lane<Sh::NB>& ln, f32x16 (&acc)[2][Sh::NB], const Tile& t, char* spare, Settle settle) {
        const uint32_t r0 = t.rb * TR, rw = r0 + uint32_t(ln.wr * 64);
        constexpr int ES = g16::size_of(KIND);
#pragma unroll
        for (int n = 0; n < Sh::NB; ++n) {
            const uint32_t q0 = t.qb * TQ + uint32_t(ln.wq * 32 * Sh::NB + 32 * n), y = sm.target[ln.q(n)] - r0;
            const bool hit = __any(y - uint32_t(ln.wr * 64) < 64u);
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                if constexpr (KIND >= g16::PLANES) {
                    block<true, true>(sm, ln, acc, y, m, n, spare);
                } else {
                    if (OFF == OFF_ANY && s.natural) block<true, true>(sm, ln, acc, y, m, n, spare);
                    else if (hit) block<false, true>(sm, ln, acc, y, m, n, spare);
                    else block<false, false>(sm, ln, acc, y, m, n, spare);
                }
                if (n == 0 && m == (ES == 4 ? 0 : 1)) settle();
                // (dl's rows hold whole groups of 64 items: a wave's are inside or outside)
                if (ES == 4 && rw < Vp) put(spare, ln, q0, uint64_t(rw + 32 * m) * ES);
            }
            if (ES == 2 && rw < Vp) put(spare, ln, q0, uint64_t(rw) * ES);
        }
    }
    template <class Tile>
    __device__ void end(State&, Shared&, const g16::Lane<Sh::NB>&, const Tile&, bool) {}
};

// A product's rows as fp32 shares [part][row][Dp], dh's added to over the pieces (first: written)
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
    __device__ void tile(State&, Shared&, const g16::Lane<Sh::NB>& ln, f32x16 (&acc)[2][Sh::NB], const Tile& t, char*, Settle settle) {
        settle();
#pragma unroll
        for (int n = 0; n < Sh::NB; ++n) {
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
    __device__ void end(State&, Shared&, const g16::Lane<Sh::NB>&, const Tile&, bool) {}
};

// A product's rows, final: dw's, or dh's where its sum is not shared (gk: rows whose gradient is zero).  They leave
// through the wave's LDS as dl does, 128 bytes of a row at once (stored straight from the accumulators, 16 bytes
// of a row, a step of 11 rows, 155,134 items of 1536 in bf16 took 472 us, so 408; 40, 15,787 of 513 100 and 75).
template <class Sh, int KIND>
struct RowsEpi {
    static constexpr int DT = dtype_of(KIND);
    using Shape = Sh;
    using T = ElemT<DT>;
    static constexpr int TQ = Sh::TQ, TR = Sh::TR;
    static constexpr bool kWalk = false, kStores = true;
    T* out;
    uint64_t ld;
    uint32_t rows, D;
    const float* mul;  // scale over dl's factor
    const float* gk;   // nullptr: no such rows
    struct Shared {
        float mul;
    };
    struct State {};
    template <class Tile>
    __device__ void begin(State&, Shared&, const Tile&) {}
    template <class Tile>
    __device__ void load(State&, const Tile&, int) {}
    __device__ void publish(State&, Shared& sm, int tid) {
        if (tid == 0) sm.mul = *mul;
    }
    // 32 rows from q0, 128 bytes each from column d0
    __device__ void put(const char* spare, const g16::Lane<Sh::NB>& ln, uint32_t q0, uint32_t d0) {
        constexpr int E = 16 / int(sizeof(T));
        typedef T V __attribute__((ext_vector_type(E)));
        typedef T Vu __attribute__((ext_vector_type(E), aligned(sizeof(T))));  // (rows of any alignment)
        const int lane = ln.hh * 32 + ln.l32;
        asm volatile("" ::: "memory");  // the writes come first (a wave's LDS accesses execute in order)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int t = 8 * i + (lane >> 3), c = lane & 7;
            const u32x4 w = *reinterpret_cast<const u32x4*>(spare + t * 128 + 16 * (c ^ (t & 7)));
            const V v = __builtin_bit_cast(V, w);
            const uint32_t d = d0 + uint32_t(c * E);
            if (q0 + t >= rows || d >= D) continue;
            T* o = out + (q0 + t) * ld + d;
            if (d + E <= D) {
                *reinterpret_cast<Vu*>(o) = v;
            } else {
#pragma unroll
                for (int e = 0; e < E - 1; ++e)
                    if (d + e < D) o[e] = v[e];
            }
        }
        asm volatile("" ::: "memory");  // and the reads before what is written next
    }
    template <class Tile, class Settle>
    __device__ void tile(State&, Shared& sm, const g16::Lane<Sh::NB>& ln, f32x16 (&acc)[2][Sh::NB], const Tile& t, char* spare, Settle settle) {
        bool none[Sh::NB];
#pragma unroll
        for (int n = 0; n < Sh::NB; ++n) {
            const uint32_t q = t.qb * TQ + uint32_t(ln.q(n));
            none[n] = gk && q < rows && gk[q] == 0.0f;
        }
        settle();
        const float s = sm.mul;
        const uint32_t d0 = t.rb * TR + uint32_t(ln.wr * 64);
        if (d0 >= D) return;
#pragma unroll
        for (int n = 0; n < Sh::NB; ++n) {
            const uint32_t q0 = t.qb * TQ + uint32_t(ln.wq * 32 * Sh::NB + 32 * n);
            if (q0 >= rows) break;
#pragma unroll
            for (int m = 0; m < 2; ++m) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    struct alignas(4 * sizeof(T)) V4 {
                        T v[4];
                    } v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v.v[e] = Elem<DT>::from_f(none[n] ? 0.0f : acc[m][n][4 * j + e] * s);
                    const int c = sizeof(T) == 4 ? 2 * j + ln.hh : 4 * m + j;  // the four values' chunk of the row
                    *reinterpret_cast<V4*>(spare + ln.l32 * 128 + 16 * (c ^ (ln.l32 & 7)) + (sizeof(T) == 4 ? 0 : 8 * ln.hh)) = v;
                }
                if (sizeof(T) == 4) put(spare, ln, q0, d0 + 32 * m);
            }
            if (sizeof(T) == 2) put(spare, ln, q0, d0);
        }
    }
    template <class Tile>
    __device__ void end(State&, Shared&, const g16::Lane<Sh::NB>&, const Tile&, bool) {}
};

// out[t][d] = mul sum over the shares (zero for a row without a gradient, gk not NULL).  64 groups of four values a
// workgroup, its four waves a quarter of the shares each.
template <int KIND>
__global__ __launch_bounds__(256) void share_sum_kernel(const float* __restrict__ share, uint32_t parts, uint32_t T, uint32_t D,
                                                        uint32_t Dp, const float* __restrict__ gk, const float* __restrict__ mul,
                                                        ElemT<dtype_of(KIND)>* __restrict__ out, uint64_t ld) {
    __shared__ f32x4 part[4][64];
    const uint32_t per = Dp / 4, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const uint64_t n = uint64_t(T) * per;
    for (uint64_t i0 = uint64_t(blockIdx.x) * 64; i0 < n; i0 += uint64_t(gridDim.x) * 64) {
        const uint64_t i = i0 + lane;
        f32x4 v{0.0f, 0.0f, 0.0f, 0.0f};
        if (i < n)
#pragma unroll 8
            for (uint32_t s = w; s < parts; s += 4) v += *reinterpret_cast<const f32x4*>(share + (uint64_t(s) * n + i) * 4);
        part[w][lane] = v;
        __syncthreads();
        if (!w && i < n) {
            v = (v + part[1][lane]) + (part[2][lane] + part[3][lane]);
            const uint32_t t = uint32_t(i / per), d = uint32_t(i % per) * 4;
            const float m = *mul;
            const bool none = gk && gk[t] == 0.0f;
            for (int e = 0; e < 4 && d + e < D; ++e) out[t * ld + d + e] = Elem<dtype_of(KIND)>::from_f(none ? 0.0f : v[e] * m);
        }
        __syncthreads();  // the quarters are read
    }
}

constexpr size_t kGradBudget = size_t(512) << 20;  // dl of one piece
// Bytes between dl's rows: with the rows a power of two apart, a tile's 256 rows meet in few memory channels
// (4096 rows x 65,536 items of a piece: 7.17 ms a step without, 6.65 with).
constexpr uint32_t kRowPad = 128;
// Up to so many rows every workgroup of the preparation looks at all targets for itself.
constexpr uint32_t kPrepareRows = 8192;

}  // namespace
}  // namespace va

using namespace va;
using namespace va::xent;

extern "C" {

va_status va_xent_backward(va_context* ctx, const va_xent_desc* desc, const float* lse, va_reduction reduction, const float* grad,
                           void* out_grad_hidden, uint64_t grad_hidden_stride, void* out_grad_items, uint64_t grad_items_stride) {
    if (!ctx) return VA_ERR_INVALID_ARG;
    va_xent_desc own;
    VA_CHECK_STATUS(check_desc(ctx, desc, "va_xent_backward", own));
    const va_xent_desc* d = &own;
    grad_hidden_stride = stride_of(d->rows, grad_hidden_stride, d->dim);
    grad_items_stride = stride_of(d->num_items, grad_items_stride, d->dim);
    VA_REQUIRE(ctx, lse, "va_xent_backward: NULL log-sum-exp");
    VA_REQUIRE(ctx, reduction == VA_REDUCE_MEAN || reduction == VA_REDUCE_SUM || reduction == VA_REDUCE_NONE, "va_xent_backward: unknown reduction %d", int(reduction));
    VA_REQUIRE(ctx, reduction != VA_REDUCE_NONE || grad, "va_xent_backward: without a reduction the rows' gradients are needed");
    VA_REQUIRE(ctx, out_grad_hidden || out_grad_items, "va_xent_backward: no output");
    VA_REQUIRE(ctx, (!out_grad_hidden || grad_hidden_stride >= d->dim) && (!out_grad_items || grad_items_stride >= d->dim),
               "va_xent_backward: a gradient's row stride is below the dimension");
    const va_dtype dt = d->dtype;
    const size_t es = elem_size(dt);
    VA_REQUIRE(ctx, (!out_grad_hidden || reinterpret_cast<uintptr_t>(out_grad_hidden) % es == 0) &&
                        (!out_grad_items || reinterpret_cast<uintptr_t>(out_grad_items) % es == 0),
               "va_xent_backward: a gradient is not aligned to its type");
    DeviceGuard guard(ctx->device);
    const uint32_t T = d->rows, V = d->num_items, D = d->dim, Dp = round_up(D, 4);
    // The logits' kind, and the second products': dl's values reach from g down to the smallest probability, and each of its
    // columns is a sum of its own, so for fp32 rows it is fp32.  (Two fp16 planes of it would end 38 binary orders below
    // the largest |g|: probabilities of exp(-27) of it would be zeros.)
    const int kind = kind_of(dt, T, V), second = kind == g16::PLANES ? int(g16::SPLIT) : kind;
    const bool planes = kind == g16::PLANES, wild = wild_scale(d);
    const uint32_t ks = uint32_t(g16::size_of(second)), kv = uint32_t(g16::stage_of(second));
    const uint32_t row = copy_bytes(kind, D), tail = planes ? 0 : D * ks % g16::ROWB;
    // Masked items may hold anything, and dh sums over them: unless they are found to be finite, a copy is read in
    // which they are zeros.
    const bool xd = in_place_rows(dt, d->items, d->items_stride), checks = xd && d->offsets, copies = !xd || checks;

    // the piece: dl and the copied items within their budgets, dl's rows within the products' 32-bit offsets
    uint32_t piece = piece_items(V, uint64_t(T) * ks, kGradBudget);
    if (copies || planes) piece = std::min(piece, piece_items(V, row, kCopyBudget));
    piece = std::min<uint32_t>(piece, (uint32_t(kDmaMaxBytes / 256) - kRowPad) / ks / 256 * 256);
    const uint32_t pieces = ceil_div(V, piece), most = std::min(piece, V), Vpmax = round_up(most, 64);
    // dh has few tiles and a long sum, and so has dw of many rows and few items: shares of it until the chip is
    // filled once, eight stages at least each.  A short sum in one piece is not shared, its rows are final.
    const auto shares_of = [&](uint32_t k, bool once) {
        const uint32_t stages = ceil_div(k, kv);
        return stages <= 24 && once ? 1u : std::max(stages / 8, 1u);
    };
    const bool narrow = kind == g16::F32 && T <= 32;
    const Blocks lb = blocks_for(ctx, kind, T, most, 1, narrow, stages_of(kind, D)), hb = blocks_for(ctx, second, T, D, shares_of(Vpmax, pieces == 1), narrow),
                 wb = blocks_for(ctx, second, most, D, shares_of(T, true));
    const bool h_shared = out_grad_hidden && (hb.parts > 1 || pieces > 1), w_shared = out_grad_items && wb.parts > 1;

    const size_t p_bytes = uint64_t(T) * (uint64_t(Vpmax) * ks + kRowPad);
    const size_t share_n = h_shared ? uint64_t(hb.parts) * T * Dp : 0, w_share_n = w_shared ? uint64_t(wb.parts) * most * Dp : 0;
    const size_t q_bytes = uint64_t(T) * row, x_bytes = copies ? uint64_t(most) * row : 0;
    const size_t qs_bytes = planes ? q_bytes : 0, xs_bytes = planes ? uint64_t(most) * row : 0;
    Scratch sc(ctx);
    const size_t need = Scratch::round(p_bytes) + Scratch::round(share_n * 4) + Scratch::round(w_share_n * 4) + Scratch::round(q_bytes) + Scratch::round(x_bytes) +
                        Scratch::round(qs_bytes) + Scratch::round(xs_bytes) + 2 * Scratch::round(T * 4ull) + Scratch::round(most * 4ull) + Scratch::round(8);
    VA_CHECK_STATUS(sc.reserve(need));
    char* p = sc.carve<char>(p_bytes);
    float* share = sc.carve<float>(share_n);
    float* w_share = sc.carve<float>(w_share_n);
    char* qp = sc.carve<char>(q_bytes);
    char* xp = sc.carve<char>(x_bytes);
    char* qs = sc.carve<char>(qs_bytes);  // planes
    char* xs = sc.carve<char>(xs_bytes);
    float* gk = sc.carve<float>(T);
    float* qinv = sc.carve<float>(T);
    float* xinv = sc.carve<float>(most);
    float* mul = sc.carve<float>(2);
    uint32_t* odd = reinterpret_cast<uint32_t*>(mul + 1);
    VA_CHECK_STATUS(sc.verify(need));

    // gk, and the hidden rows ended by zeros
    // (dl's largest values: 2^14 in fp16, whose range is short; in types of fp32's range 1, so that no sum of dl w or dl h
    // passes fp32 where the gradient does not)
    const PrepareArgs pa{grad, d->targets, T, V, d->ignore_index, int(reduction), d->scale, dt == VA_DTYPE_F16 ? 0x1p14f : 1.0f, gk, mul, odd};
    const bool together = T <= kPrepareRows;
    const uint32_t rows_per = together ? std::max(4u, ceil_div(T, 512)) : T;
    if (dt == VA_DTYPE_F32)
        xent_prepare_kernel<uint32_t><<<dim3(ceil_div(T, rows_per)), dim3(256), 0, ctx->stream>>>(
            pa, rows_per, together ? static_cast<const uint32_t*>(d->hidden) : nullptr, d->hidden_stride, D, row / 4, reinterpret_cast<uint32_t*>(qp));
    else
        xent_prepare_kernel<uint16_t><<<dim3(ceil_div(T, rows_per)), dim3(256), 0, ctx->stream>>>(
            pa, rows_per, together ? static_cast<const uint16_t*>(d->hidden) : nullptr, d->hidden_stride, D, row / 2, reinterpret_cast<uint16_t*>(qp));
    VA_CHECK_LAUNCH(ctx);
    const Drop no_gradient{gk, 0.0f};
    if (!together) VA_CHECK_STATUS(make_copy(ctx, second, d->hidden, d->hidden_stride, T, D, no_gradient, qp));
    if (checks) VA_CHECK_STATUS(find_odd(ctx, d, odd));

    auto rows_out = [&](auto sh, auto k, auto qk, const g16::Args& b, uintptr_t o, uint64_t ld, uint32_t rows, const float* zero) {
        constexpr int kKind = decltype(k)::value;
        using E = ElemT<dtype_of(kKind)>;
        const RowsEpi<decltype(sh), kKind> e{reinterpret_cast<E*>(o), ld, rows, D, mul, zero};
        return g16::launch<kKind, decltype(qk)::value, true>(ctx, b, e);
    };
    auto sum_shares = [&](const float* from, uint32_t parts, uint32_t rows, const float* zero, uintptr_t o, uint64_t ld) {
        return by_second(second, [&](auto k) {
            constexpr int kKind = decltype(k)::value;
            share_sum_kernel<kKind><<<dim3(uint32_t(std::min<uint64_t>((uint64_t(rows) * (Dp / 4) + 63) / 64, kGridMax))), dim3(256), 0, ctx->stream>>>(
                from, parts, rows, D, Dp, zero, mul, reinterpret_cast<ElemT<dtype_of(kKind)>*>(o), ld);
            VA_CHECK_LAUNCH(ctx);
            return VA_OK;
        });
    };
    for (uint32_t c = 0; c < pieces; ++c) {
        const uint32_t v0 = c * piece, n = std::min(piece, V - v0), Vp = round_up(n, 64);
        const char* items = row_at(d->items, d->items_stride, v0, dt);
        const float* offsets = d->offsets ? d->offsets + v0 : nullptr;
        const Drop masked{offsets, -INFINITY};
        if (planes)
            VA_CHECK_STATUS(make_planes(ctx, D, Planes{d->hidden, d->hidden_stride, c ? 0 : T, no_gradient, qs, qinv},
                                        Planes{items, d->items_stride, n, masked, xs, xinv}));
        if (copies) VA_CHECK_STATUS(make_copy(ctx, second, items, d->items_stride, n, D, masked, xp, checks ? odd : nullptr));
        const g16::Operand rows = copied(second, qp, T, D);
        g16::Operand cols = xd ? in_place(dt, items, d->items_stride, n, D) : copied(second, xp, n, D);
        if (checks) {
            cols.other = xp;
            cols.other_pitch = row;
            cols.choose = odd;
        }
        g16::Operand dl;
        dl.p = p;
        dl.pitch = uint64_t(Vp) * ks + kRowPad;
        dl.rows = T;
        dl.width = Vp * ks;
        g16::Args a;
        a.q = planes ? copied(kind, qs, T, D) : rows;
        a.x = planes ? copied(kind, xs, n, D) : cols;
        a.kstages = row / g16::ROWB;
        a.tail = xd ? tail : 0;
        a.nq = lb.nq(T);
        a.nr = lb.nr(n);
        VA_CHECK_STATUS(by_kind(kind, offsets || wild, n % lb.tr, [&](auto k, auto off) {
            return by_logit_shape<decltype(k)::value>(lb.shape, [&](auto sh) {
                using Sh = decltype(sh);
                GradEpi<Sh, decltype(k)::value, decltype(off)::value> e;
                e.a = LogitArgs{offsets, checks && !wild ? odd : nullptr, qinv, xinv, d->scale, T, n};
                e.gk = gk;
                e.lse = lse;
                e.targets = d->targets;
                e.item0 = v0;
                e.p = p;
                e.Vp = Vp;
                e.pitch = uint32_t(dl.pitch);
                return g16::launch<decltype(k)::value, false, false>(ctx, a, e);
            });
        }));
        if (out_grad_hidden) {
            // dh[t][d] = sum_j dl[t][j] w[j][d]: the items are stored across the sum
            g16::Args b;
            b.q = dl;
            b.x = cols;
            b.kstages = Vp / kv;
            b.nq = hb.nq(T);
            b.nr = hb.nr(D);
            b.parts = hb.parts;
            VA_CHECK_STATUS(by_second(second, [&](auto k) {
                return by_shape_of<decltype(k)::value>(hb.shape, [&](auto sh) {
                    if (!h_shared) return rows_out(sh, k, std::false_type(), b, reinterpret_cast<uintptr_t>(out_grad_hidden), grad_hidden_stride, T, gk);
                    const ShareEpi<decltype(sh)> e{share, T, D, Dp, c == 0};
                    return g16::launch<decltype(k)::value, false, true>(ctx, b, e);
                });
            }));
        }
        if (out_grad_items) {
            // dw[j][d] = sum_t dl[t][j] h[t][d]: both are
            g16::Args b;
            b.q = dl;
            b.x = rows;
            b.kstages = ceil_div(T, kv);
            b.nq = wb.nq(n);
            b.nr = wb.nr(D);
            b.parts = wb.parts;
            const uintptr_t o = reinterpret_cast<uintptr_t>(out_grad_items) + uint64_t(v0) * grad_items_stride * es;
            VA_CHECK_STATUS(by_second(second, [&](auto k) {
                return by_shape<decltype(k)::value>(wb.shape, [&](auto sh) {
                    if (!w_shared) return rows_out(sh, k, std::true_type(), b, o, grad_items_stride, n, nullptr);
                    const ShareEpi<decltype(sh)> e{w_share, n, D, Dp, true};
                    return g16::launch<decltype(k)::value, true, true>(ctx, b, e);
                });
            }));
            if (w_shared) VA_CHECK_STATUS(sum_shares(w_share, wb.parts, n, nullptr, o, grad_items_stride));
        }
    }
    if (h_shared) VA_CHECK_STATUS(sum_shares(share, hb.parts, T, gk, reinterpret_cast<uintptr_t>(out_grad_hidden), grad_hidden_stride));
    return VA_OK;
}

}  // extern "C"
