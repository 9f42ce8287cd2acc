// va_xent.hip — softmax cross entropy of hidden rows over all items of a collection, and (va_xent_grad.hip) its
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
// of them the recomputation), and the memory is that of one piece and of dh's shares.
//
// Precision: fp16 / bf16 operands enter the matrix cores as they are, sums are fp32.  dl is rounded
// once to the operands' type for the second products (relative 2^-11 / 2^-8 a value, like the
// rounding of the result), after a scale that takes the largest |g| to 1, in fp16 to 2^14: its range then holds
// probabilities down to 2^-38 of it, and with one g for all rows the target's -g is exact.  What falls below would
// be below fp16's smallest gradient too, unless the largest is near its end: dl w scale of the largest |g| is at most
// 2^16, what is lost of it 2^-39, fp16's step 2^-24.  fp32 operands are
// multiplied as fp32 for few rows; for many, in the logits as two fp16 planes of each row, and in the second
// products split into three bf16 values (va_gemm16.hpp), dl being fp32 in both.
//
// Masks: an item whose offset is -inf has no probability whatever its vector holds (NaN and inf
// included) and gets a zero gradient; a row without a target has loss 0 and a zero gradient whatever
// it holds.  When every item is masked, lse = -inf, the losses are 0 and so are the gradients.
//
// What bounds it: few rows, the stream of the items (10 x 1M x 768 in fp16 258 us, 5.9 TB/s); many, the matrix cores and
// after them the exp of every logit, which share a SIMD's waves (4096 x 262,144 x 768 in bf16 1.60 ms, 1.03
// PFLOP/s; 1023 x 49,999 x 300 in fp16 53 us, 0.58 PFLOP/s with five stages a tile); fp32 rows in planes, three
// times the products and the copies (512 x 100,003 x 384: 111 + 52 us); a small collection, latency
// (1 x 10,000 x 768 in bf16: 10 + 4 us).
#include "va_xent.hpp"

namespace va {
namespace {

using namespace xent;

// ---- copies: rows a product cannot read in place, operands whose rows must end in zeros or may not be read, planes -------------
// dst[r][k] = src[r][k], zeros for k in [D, Kp) and in dropped rows.  Nothing if *run_if is zero.
template <class U>
__global__ __launch_bounds__(256) void copy_kernel(const U* __restrict__ src, uint64_t ld, uint32_t D, uint32_t Kp, Drop drop, const uint32_t* run_if,
                                                   U* __restrict__ dst, uint64_t n) {
    if (run_if && *run_if == 0) return;
    constexpr int E = 16 / sizeof(U);
    typedef U UxE __attribute__((ext_vector_type(E), aligned(sizeof(U))));
    const uint32_t per = Kp / E;
    for (uint64_t i = uint64_t(blockIdx.x) * 256 + threadIdx.x; i < n; i += uint64_t(gridDim.x) * 256) {
        const uint64_t r = i / per;
        const uint32_t k = uint32_t(i - r * per) * E;
        UxE v = {};
        const U* s = src + r * ld + k;
        if (!(drop.value && drop.value[r] == drop.is)) {
            if (k + E <= D) {
                v = *reinterpret_cast<const UxE*>(s);
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) v[e] = k + e < D ? s[e] : U(0);
            }
        }
        *reinterpret_cast<u32x4*>(dst + r * Kp + k) = __builtin_bit_cast(u32x4, v);
    }
}

// One wave per fp32 row: its planes dst[r] (16 values of hi, the same of lo, and so on; Kp values, zeros past D), scaled by the
// power of two that puts the row's largest entry near 2^14; inv[r] = the inverse.  Dropped rows are zeros.
// Rows of `a` in the first na workgroups, then of `b`.
__global__ __launch_bounds__(256) void planes_kernel(Planes a, Planes b, uint32_t na, uint32_t D, uint32_t Kp) {
    typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
    const int lane = threadIdx.x & 63;
    const bool second = blockIdx.x >= na;
    const uint32_t r = (second ? blockIdx.x - na : blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (r >= (second ? b.R : a.R)) return;
    const float* s = static_cast<const float*>(second ? b.src : a.src) + r * (second ? b.ld : a.ld);
    const float* drop = second ? b.drop.value : a.drop.value;
    const bool none = drop && drop[r] == (second ? b.drop.is : a.drop.is);
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
    const float sc = scale_to_2p14(wave_max(m));
    if (lane == 0) (second ? b.inv : a.inv)[r] = 1.0f / sc;
    uint16_t* o = static_cast<uint16_t*>(second ? b.dst : a.dst) + uint64_t(r) * 2 * Kp;
    auto put = [&](uint32_t k, f32x4 v) {
        uint16_t h[4], l[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) split16(v[e] * sc, h[e], l[e]);
        uint16_t* at = o + k / 16 * 32 + k % 16;
        *reinterpret_cast<uint2*>(at) = make_uint2(h[0] | uint32_t(h[1]) << 16, h[2] | uint32_t(h[3]) << 16);
        *reinterpret_cast<uint2*>(at + 16) = make_uint2(l[0] | uint32_t(l[1]) << 16, l[2] | uint32_t(l[3]) << 16);
    };
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t k = 256 * i + 4 * lane;
        if (k < Kp) put(k, held[i]);
    }
    for (uint32_t k = 1024 + 4 * lane; k < Kp; k += 256) put(k, load4(k));
}

// *odd = 1 (0 before the launch) if a masked item holds a value of magnitude `most` or more (bits; NaN and inf are), if
// an offset is finite and beyond 1e37 (log2 e times it may not be), or if a hidden value from `wide` to inf is among
// `hidden` (or nullptr).  One wave per 64 items, whose masked rows are read; then the workgroups behind the first
// `blocks`, a wave a hidden row in turn.
template <class U>
__global__ __launch_bounds__(256) void xent_odd_kernel(const U* __restrict__ items, uint64_t ld, const float* __restrict__ offsets, uint32_t V,
                                                       uint32_t D, U most, uint32_t blocks, const U* __restrict__ hidden, uint64_t ldh, uint32_t T,
                                                       U wide, U inf, uint32_t* odd) {
    constexpr U kSign = U(U(1) << (8 * sizeof(U) - 1));
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    bool bad = false;
    if (blockIdx.x < blocks) {
        const uint32_t j0 = (blockIdx.x * 4 + wave) * 64;
        const float o = j0 + lane < V ? offsets[j0 + lane] : 0.0f;
        bad = fabsf(o) > 1e37f && fabsf(o) < INFINITY;
        for (uint64_t masked = __ballot(o == -INFINITY); masked; masked &= masked - 1) {
            const U* row = items + (j0 + uint32_t(__builtin_ctzll(masked))) * ld;
            for (uint32_t d = lane; d < D; d += 64) bad |= U(row[d] & U(~kSign)) >= most;
        }
    } else {
        for (uint32_t t = (blockIdx.x - blocks) * 4 + wave; t < T; t += (gridDim.x - blocks) * 4) {
            const U* row = hidden + t * ldh;
#pragma unroll 4
            for (uint32_t d = lane; d < D; d += 64) {
                const U v = U(row[d] & U(~kSign));
                bad |= v >= wide && v <= inf;
            }
        }
    }
    if (__any(bad) && lane == 0) *odd = 1;
}

// Forward: the running (m, z) of a lane's items per query; joined over the workgroup at the end of
// the item and written to part[row * slots + slot].  The target's logit is picked out on the way: with
// the loss a difference of two logits, both from the same sums, their errors cancel for a row whose
// target is far ahead of the other items.
template <class Sh, int KIND, int OFF>
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
    struct Shared : LogitShared<KIND, OFF, TR> {
        float2 red[Sh::WR][TQ];
        uint32_t target[TQ];  // within the launch's items (any larger value: elsewhere)
        float qinv[KIND == g16::PLANES ? TQ : 1];
    };
    struct State {
        float m[Sh::NB], z[Sh::NB];
        float off, inv;
        bool natural;
    };
    template <class Tile>
    __device__ void begin(State& s, Shared& sm, const Tile& t) {
        s.natural = keeps_natural<KIND, OFF>(a);
#pragma unroll
        for (int n = 0; n < Sh::NB; ++n) {
            s.m[n] = -INFINITY;
            s.z[n] = 0.0f;
        }
        const uint32_t i = threadIdx.x, q = t.qb * TQ + i;
        if (i >= uint32_t(TQ)) return;
        const int64_t y = q < a.rows ? targets[q] - int64_t(item0) : -1;
        sm.target[i] = y >= 0 && y < int64_t(a.items) ? uint32_t(y) : 0xFFFFFFFFu;
        if constexpr (KIND == g16::PLANES) sm.qinv[i] = q < a.rows ? a.qinv[q] : 0.0f;
    }
    template <class Tile>
    __device__ void load(State& s, const Tile& t, int tid) {
        const uint32_t r = t.rb * TR + uint32_t(tid);
        const bool in = tid < TR && r < a.items;
        if constexpr (OFF != OFF_NONE) s.off = offset_of(a, in, r, s.natural);
        if constexpr (KIND == g16::PLANES) s.inv = in ? a.xinv[r] : 0.0f;
    }
    __device__ void publish(State& s, Shared& sm, int tid) {
        if constexpr (OFF != OFF_NONE)
            if (tid < TR) sm.off[tid] = s.off;
        if constexpr (KIND == g16::PLANES)
            if (tid < TR) sm.inv[tid] = s.inv;
    }
    template <bool NATURAL, class Tile>
    __device__ void block(State& s, Shared& sm, const g16::Lane<Sh::NB>& ln, f32x16 (&acc)[2][Sh::NB], const Tile& t, int n) {
        const float c = (KIND == g16::PLANES ? a.scale * sm.qinv[ln.q(n)] : a.scale) * (NATURAL ? 1.0f : kLog2e);
        float top = -INFINITY;
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                f32x4 v = logits4<NATURAL, KIND, OFF, TR>(sm, acc[m][n], j, ln.r(m, j), c);
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
    __device__ void tile(State& s, Shared& sm, const g16::Lane<Sh::NB>& ln, f32x16 (&acc)[2][Sh::NB], const Tile& t, char*, Settle) {
#pragma unroll
        for (int n = 0; n < Sh::NB; ++n) {
            if constexpr (KIND >= g16::PLANES) {
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
    __device__ void end(State& s, Shared& sm, const g16::Lane<Sh::NB>& ln, const Tile& t, bool mine) {
#pragma unroll
        for (int n = 0; n < Sh::NB; ++n) {
            // (natural units from here; a row's largest logit and its target's are scaled alike)
            float m = s.natural ? s.m[n] : s.m[n] * kLn2;
            join(m, s.z[n], __shfl_xor(m, 32), __shfl_xor(s.z[n], 32));
            if (mine && ln.hh == 0) sm.red[ln.wr][ln.q(n)] = make_float2(m, s.z[n]);
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

// ---- finishing kernels -----------------------------------------------------------------------------------
// The sum of the losses, or their mean over the rows with a target, by one workgroup.
__device__ void reduce_losses(const float* loss, const int64_t* __restrict__ targets, uint32_t T, int64_t ignore, bool mean, float* out) {
    __shared__ double sum[16];
    __shared__ uint32_t cnt[16];
    double s = 0.0;
    uint32_t c = 0;
    for (uint32_t t = threadIdx.x; t < T; t += blockDim.x)
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
    if (threadIdx.x) return;
    for (uint32_t i = 1; i < blockDim.x / 64; ++i) {
        s += sum[i];
        c += cnt[i];
    }
    *out = float(mean ? (c ? s / double(c) : 0.0) : s);
}
__global__ __launch_bounds__(1024) void xent_reduce_kernel(const float* __restrict__ loss, const int64_t* __restrict__ targets, uint32_t T,
                                                           int64_t ignore, bool mean, float* out) {
    reduce_losses(loss, targets, T, ignore, mean, out);
}

// One wave per row: the shares joined into lse, and the loss; launched as one workgroup (few rows), it also
// reduces the losses (reduced not NULL).
__global__ __launch_bounds__(1024) void xent_finish_kernel(const int64_t* __restrict__ targets, uint32_t T, uint32_t V, int64_t ignore,
                                                           const float2* __restrict__ part, const float* __restrict__ picked, uint32_t slots,
                                                           float* loss, float* __restrict__ lse, bool mean, float* reduced) {
    const int lane = threadIdx.x & 63;
    const uint32_t waves = blockDim.x / 64;
    for (uint32_t t = blockIdx.x * waves + (threadIdx.x >> 6); t < T; t += gridDim.x * waves) {
        float m = -INFINITY, z = 0.0f;
#pragma unroll 4
        for (uint32_t i = lane; i < slots; i += 64) {
            const float2 p = part[uint64_t(t) * slots + i];
            join(m, z, p.x, p.y);
        }
#pragma unroll
        for (int d = 32; d; d >>= 1) join(m, z, __shfl_xor(m, d), __shfl_xor(z, d));
        if (lane) continue;
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
    if (!reduced) return;
    __syncthreads();
    reduce_losses(loss, targets, T, ignore, mean, reduced);
}

// ---- host ------------------------------------------------------------------------------------------
}  // namespace

namespace xent {

// Up to so many rows one workgroup finishes and reduces them (one launch instead of two).
constexpr uint32_t kFinishRows = 64;

va_status make_copy(va_context* ctx, int kind, const void* src, uint64_t ld, uint32_t R, uint32_t D, Drop drop, void* dst, const uint32_t* run_if) {
    const uint32_t bytes = copy_bytes(kind, D);
    const uint64_t n = uint64_t(R) * (bytes / 16);
    const dim3 grid(uint32_t(std::min<uint64_t>((n + 255) / 256, 16384)));
    if (kind >= g16::F32)
        copy_kernel<uint32_t><<<grid, dim3(256), 0, ctx->stream>>>(static_cast<const uint32_t*>(src), ld, D, bytes / 4, drop, run_if, static_cast<uint32_t*>(dst), n);
    else
        copy_kernel<uint16_t><<<grid, dim3(256), 0, ctx->stream>>>(static_cast<const uint16_t*>(src), ld, D, bytes / 2, drop, run_if, static_cast<uint16_t*>(dst), n);
    VA_CHECK_LAUNCH(ctx);
    return VA_OK;
}

va_status make_planes(va_context* ctx, uint32_t D, Planes a, Planes b) {
    const uint32_t bytes = copy_bytes(g16::PLANES, D);
    auto rest = [&](Planes& p, uint32_t n) {  // what is left behind the first n rows
        p.src = static_cast<const float*>(p.src) + n * p.ld;
        p.dst = static_cast<char*>(p.dst) + uint64_t(n) * bytes;
        p.inv += n;
        if (p.drop.value) p.drop.value += n;
        p.R -= n;
    };
    while (a.R || b.R) {
        const uint32_t na = std::min(ceil_div(a.R, 4), kGridMax), nb = std::min(ceil_div(b.R, 4), kGridMax - na);
        planes_kernel<<<dim3(na + nb), dim3(256), 0, ctx->stream>>>(a, b, na, D, bytes / 4);
        VA_CHECK_LAUNCH(ctx);
        rest(a, std::min(a.R, 4 * na));
        rest(b, std::min(b.R, 4 * nb));
    }
    return VA_OK;
}

va_status find_odd(va_context* ctx, const va_xent_desc* d, uint32_t* odd) {
    const uint32_t blocks = ceil_div(d->num_items, 256);
    if (d->dtype == VA_DTYPE_F32) {
        xent_odd_kernel<uint32_t><<<dim3(blocks), dim3(256), 0, ctx->stream>>>(static_cast<const uint32_t*>(d->items), d->items_stride, d->offsets, d->num_items,
                                                                               d->dim, 0x7F800000u, blocks, nullptr, 0, 0, 0u, 0u, odd);
    } else {
        // A masked bf16 item's finite values may overflow its logits, which an offset of -inf then turns into NaN.  Items
        // below 2^64 and hidden values below 2^46 cannot: 2^16 products (VA_XENT_MAX_DIM) of less than 2^110 each.  Nor
        // can fp16's, 2^16 products of 2^32.
        static_assert(VA_XENT_MAX_DIM <= 1u << 16, "the bound on a logit's sum");
        const bool bf16 = d->dtype == VA_DTYPE_BF16;
        const uint16_t most = bf16 ? (127 + 64) << 7 : 0x7C00, wide = (127 + 46) << 7, inf = 0x7F80;
        const uint32_t more = bf16 ? std::min(ceil_div(d->rows, 4), 1024u) : 0u;
        xent_odd_kernel<uint16_t><<<dim3(blocks + more), dim3(256), 0, ctx->stream>>>(static_cast<const uint16_t*>(d->items), d->items_stride, d->offsets,
                                                                                      d->num_items, d->dim, most, blocks, static_cast<const uint16_t*>(d->hidden),
                                                                                      d->hidden_stride, d->rows, wide, inf, odd);
    }
    VA_CHECK_LAUNCH(ctx);
    return VA_OK;
}

va_status check_desc(va_context* ctx, const va_xent_desc* desc, const char* who, va_xent_desc& own) {
    VA_REQUIRE(ctx, desc != nullptr, "%s: NULL description", who);
    own = *desc;
    own.hidden_stride = stride_of(own.rows, own.hidden_stride, own.dim);
    own.items_stride = stride_of(own.num_items, own.items_stride, own.dim);
    const va_xent_desc* d = &own;
    VA_REQUIRE(ctx, d->hidden && d->items && d->targets, "%s: NULL pointer", who);
    VA_REQUIRE(ctx, d->rows > 0 && d->num_items > 0 && d->dim > 0, "%s: empty input (%u rows, %u items, %u dimensions)", who, d->rows,
               d->num_items, d->dim);
    VA_REQUIRE(ctx, d->dtype == VA_DTYPE_F32 || d->dtype == VA_DTYPE_F16 || d->dtype == VA_DTYPE_BF16, "%s: unknown type %d", who, int(d->dtype));
    VA_REQUIRE(ctx, d->dim <= VA_XENT_MAX_DIM, "%s: %u dimensions (at most %u)", who, d->dim, VA_XENT_MAX_DIM);
    VA_REQUIRE(ctx, d->num_items <= 0x7FFFFFFFu && d->rows <= 0x7FFFFFFFu, "%s: too many rows or items", who);
    VA_REQUIRE(ctx, d->hidden_stride >= d->dim && d->items_stride >= d->dim, "%s: a row stride is below the dimension", who);
    VA_REQUIRE(ctx, std::isfinite(d->scale), "%s: the scale is not finite", who);
    const size_t es = elem_size(d->dtype);
    VA_REQUIRE(ctx, reinterpret_cast<uintptr_t>(d->hidden) % es == 0 && reinterpret_cast<uintptr_t>(d->items) % es == 0,
               "%s: rows or items are not aligned to their type", who);
    return VA_OK;
}

}  // namespace xent
}  // namespace va

using namespace va;
using namespace va::xent;

extern "C" {

va_status va_xent_forward(va_context* ctx, const va_xent_desc* desc, float* out_loss, float* out_lse, va_reduction reduction, float* out_reduced) {
    if (!ctx) return VA_ERR_INVALID_ARG;
    va_xent_desc own;
    VA_CHECK_STATUS(check_desc(ctx, desc, "va_xent_forward", own));
    const va_xent_desc* d = &own;
    VA_REQUIRE(ctx, out_loss && out_lse, "va_xent_forward: NULL output");
    VA_REQUIRE(ctx, reduction == VA_REDUCE_MEAN || reduction == VA_REDUCE_SUM || reduction == VA_REDUCE_NONE, "va_xent_forward: unknown reduction %d", int(reduction));
    VA_REQUIRE(ctx, (reduction == VA_REDUCE_NONE) == (out_reduced == nullptr), "va_xent_forward: a reduced loss goes with a reduction");
    DeviceGuard guard(ctx->device);
    const uint32_t T = d->rows, V = d->num_items, D = d->dim;
    const va_dtype dt = d->dtype;
    const int kind = kind_of(dt, T, V);
    const uint32_t one = copy_bytes(kind, D), tail = kind == g16::PLANES ? 0 : D * uint32_t(elem_size(dt)) % g16::ROWB;
    // the hidden rows end in zeros, the items are cut in their fragments
    const bool qd = kind != g16::PLANES && tail == 0 && in_place_rows(dt, d->hidden, d->hidden_stride);
    const bool xd = kind != g16::PLANES && in_place_rows(dt, d->items, d->items_stride);
    const size_t q_bytes = qd ? 0 : uint64_t(T) * copy_bytes(kind, D), x_row = copy_bytes(kind, D);
    const uint32_t piece = xd ? round_up(V, 256) : piece_items(V, x_row, kCopyBudget), most = std::min(piece, V);
    const uint32_t pieces = ceil_div(V, piece);
    const Blocks bl = blocks_for(ctx, kind, T, most, 1, kind == g16::F32 && T <= 32, stages_of(kind, D));
    // Offsets are looked over first where the shorter epilogue counts: 16-bit products on the matrix cores'
    // time (4096 rows x 262,144 items of 768: the check takes 15 us and saves 100; a product that streams its
    // items hides the longer epilogue).
    const bool wild = wild_scale(d), checks = d->offsets && kind < g16::PLANES && !wild && bl.shape == LARGE;
    const uint32_t nq = bl.nq(T);
    // parts per query block: whole multiples of the XCDs where that costs no round of tiles
    uint32_t parts = std::min(std::max(bl.grid / nq, 1u), bl.nr(most));
    const uint32_t even = parts / kXcds * kXcds;
    if (even && ceil_div(bl.nr(most), even) == ceil_div(bl.nr(most), parts)) parts = even;
    const uint32_t last_parts = std::min(parts, bl.nr(V - (pieces - 1) * piece));  // (of the last piece)
    const uint32_t slots = parts * (pieces - 1) + last_parts;

    Scratch sc(ctx);
    const size_t need = Scratch::round(q_bytes) + (xd ? 0 : Scratch::round(x_row * most)) + Scratch::round(most * 4ull) + 2 * Scratch::round(T * 4ull) +
                        Scratch::round(uint64_t(T) * slots * sizeof(float2)) + Scratch::round(4);
    VA_CHECK_STATUS(sc.reserve(need));
    float2* part = sc.carve<float2>(uint64_t(T) * slots);
    float* picked = sc.carve<float>(T);
    float* qinv = sc.carve<float>(T);
    float* xinv = sc.carve<float>(most);
    uint32_t* odd = sc.carve<uint32_t>(1);
    char* qp = sc.carve<char>(q_bytes);
    char* xp = xd ? nullptr : sc.carve<char>(x_row * most);
    VA_CHECK_STATUS(sc.verify(need));
    if (checks) {
        VA_CHECK_STATUS(fill_u32(ctx, odd, 1, 0));
        VA_CHECK_STATUS(find_odd(ctx, d, odd));
    }
    const bool planes = kind == g16::PLANES;
    if (!qd && !planes) VA_CHECK_STATUS(make_copy(ctx, kind, d->hidden, d->hidden_stride, T, D, Drop{}, qp));
    for (uint32_t c = 0; c < pieces; ++c) {
        const uint32_t v0 = c * piece, n = std::min(piece, V - v0);
        const char* items = row_at(d->items, d->items_stride, v0, dt);
        if (planes)
            VA_CHECK_STATUS(make_planes(ctx, D, Planes{d->hidden, d->hidden_stride, c ? 0 : T, Drop{}, qp, qinv},
                                        Planes{items, d->items_stride, n, Drop{}, xp, xinv}));
        else if (!xd)
            VA_CHECK_STATUS(make_copy(ctx, kind, items, d->items_stride, n, D, Drop{}, xp));
        g16::Args a;
        a.q = qd ? in_place(dt, d->hidden, d->hidden_stride, T, D) : copied(kind, qp, T, D);
        a.x = xd ? in_place(dt, items, d->items_stride, n, D) : copied(kind, xp, n, D);
        a.kstages = one / g16::ROWB;
        a.tail = xd ? tail : 0;
        a.nq = nq;
        a.nr = bl.nr(n);
        a.parts = c + 1 < pieces ? parts : last_parts;
        VA_CHECK_STATUS(by_kind(kind, d->offsets || wild, n % bl.tr, [&](auto k, auto off) {
            return by_logit_shape<decltype(k)::value>(bl.shape, [&](auto sh) {
                using Sh = decltype(sh);
                LseEpi<Sh, decltype(k)::value, decltype(off)::value> e;
                e.a = LogitArgs{d->offsets ? d->offsets + v0 : nullptr, checks ? odd : nullptr, qinv, xinv, d->scale, T, n};
                e.targets = d->targets;
                e.item0 = v0;
                e.picked = picked;
                e.part = part;
                e.slots = slots;
                e.slot0 = c * parts;
                return g16::launch<decltype(k)::value, false, false>(ctx, a, e);
            });
        }));
    }
    const bool mean = reduction == VA_REDUCE_MEAN;
    if (T <= kFinishRows) {
        xent_finish_kernel<<<dim3(1), dim3(1024), 0, ctx->stream>>>(d->targets, T, V, d->ignore_index, part, picked, slots, out_loss, out_lse, mean, out_reduced);
    } else {
        xent_finish_kernel<<<dim3(std::min(ceil_div(T, 4), kGridMax)), dim3(256), 0, ctx->stream>>>(d->targets, T, V, d->ignore_index, part, picked, slots, out_loss, out_lse, mean, nullptr);
        VA_CHECK_LAUNCH(ctx);
        if (out_reduced) xent_reduce_kernel<<<dim3(1), dim3(1024), 0, ctx->stream>>>(out_loss, d->targets, T, d->ignore_index, mean, out_reduced);
    }
    VA_CHECK_LAUNCH(ctx);
    return VA_OK;
}

}  // extern "C"
