// va_mx.hip — rows in microscaled 4-bit floating point: coding, reading back, and the product of queries with items.
//
// A row is cut into blocks of 32 values; a value is e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign) times its block's power of two
// 2^(s - 127), s a byte (255: NaN).  s is the least for which no value of the block rounds past 6: the largest
// magnitude is below 7 2^(s - 127).  Rows are padded with zeros to whole groups of 128 values: 64 bytes of codes, two a
// byte with the even dimension in the low half, and 4 scale bytes.  So a lane's operand of
// v_mfma_scale_f32_32x32x64_f8f6f4 is 16 bytes as they lie, and its scale a byte of a dword.
//
//   out[t][v] = scale sum_d q[t][d] w[v][d] + offset[v]
#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "va_internal.hpp"
#include "va_mx_tile.hpp"

namespace va {
namespace {

template <class T, int N>
using Vec = T __attribute__((ext_vector_type(N)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

bool known(va_dtype d) { return d == VA_DTYPE_F32 || d == VA_DTYPE_F16 || d == VA_DTYPE_BF16; }
uint32_t size_of(va_dtype d) { return d == VA_DTYPE_F32 ? 4 : 2; }
bool aligned(const void* p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

constexpr uint32_t kGroup = 128;  // values of a group
constexpr uint32_t kCodes = kMxCodes;  // bytes of its codes
constexpr uint32_t groups_of(uint32_t dim) { return (dim + kGroup - 1) / kGroup; }

// values [d, d + 8) of a row of dim; behind its end: zeros
template <class T>
__device__ __forceinline__ void load8(const T* row, uint32_t d, uint32_t dim, float (&v)[8]) {
    if (d + 8 <= dim) {
        const auto x = loose_load<Vec<T, 8>>(row + d);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = float(x[e]);
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = d + e < dim ? float(row[d + e]) : 0.0f;
}

// 16 lanes take a group, eight values each; four lanes a block.  Bound by memory: 65,536 x 1536 in bf16 59 us, 4.3 TB/s, and back to bf16
// 45 us, 5.6 TB/s (mostly writes).
template <class T>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const T* __restrict__ x, uint64_t x_stride, uint32_t rows, uint32_t dim, uint32_t groups,
                                                          uint8_t* __restrict__ codes, uint64_t codes_stride, uint8_t* __restrict__ scales,
                                                          uint64_t scales_stride) {
    const uint64_t total = uint64_t(rows) * groups;
    for (uint64_t u = (uint64_t(blockIdx.x) * 256 + threadIdx.x) / 16; u < total; u += uint64_t(gridDim.x) * 16) {
        const uint32_t row = uint32_t(u / groups), group = uint32_t(u % groups), lane = threadIdx.x & 15;
        float v[8];
        load8(x + row * x_stride, group * kGroup + 8 * lane, dim, v);
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(v[e]) & 0x7FFFFFFFu);
        top = max(top, uint32_t(__shfl_xor(int(top), 1)));
        top = max(top, uint32_t(__shfl_xor(int(top), 2)));
        // from 1.75 of its binary order on the largest value would round past 6: the next order
        const uint32_t order = (top + 0x200000u) >> 23;
        const uint32_t s = top >= 0x7F800000u ? 255u : order > 2u ? order - 2u : 0u;
        const float inv = s == 255u ? 0.0f : __uint_as_float((254u - s) << 23);  // 2^(127 - s)
        uint32_t w = 0;
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0] * inv, v[1] * inv, 1.0f, 0);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2] * inv, v[3] * inv, 1.0f, 1);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4] * inv, v[5] * inv, 1.0f, 2);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6] * inv, v[7] * inv, 1.0f, 3);
        *reinterpret_cast<uint32_t*>(codes + row * codes_stride + group * kCodes + 4 * lane) = s == 255u ? 0u : w;
        uint32_t four = s << (8 * (lane >> 2));  // the lanes' blocks' bytes together
        four |= uint32_t(__shfl_xor(int(four), 4));
        four |= uint32_t(__shfl_xor(int(four), 8));
        if (lane == 0) *reinterpret_cast<uint32_t*>(scales + row * scales_stride + 4 * group) = four;
    }
}

__device__ __forceinline__ float scale_of(uint32_t s) { return s == 255u ? __builtin_nanf("") : ldexpf(1.0f, int(s) - 127); }

template <class T>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(const uint8_t* __restrict__ codes, uint64_t codes_stride, const uint8_t* __restrict__ scales,
                                                            uint64_t scales_stride, uint32_t rows, uint32_t dim, uint32_t groups, T* __restrict__ out,
                                                            uint64_t out_stride) {
    const uint64_t total = uint64_t(rows) * groups;
    for (uint64_t u = (uint64_t(blockIdx.x) * 256 + threadIdx.x) / 16; u < total; u += uint64_t(gridDim.x) * 16) {
        const uint32_t row = uint32_t(u / groups), group = uint32_t(u % groups), lane = threadIdx.x & 15, d = group * kGroup + 8 * lane;
        if (d >= dim) continue;
        const uint32_t w = *reinterpret_cast<const uint32_t*>(codes + row * codes_stride + group * kCodes + 4 * lane);
        const float s = scale_of(scales[row * scales_stride + 4 * group + (lane >> 2)]);
        Vec<T, 8> v;
        const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1),
                   c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 2), e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 3);
        v[0] = T(a[0] * s), v[1] = T(a[1] * s), v[2] = T(b[0] * s), v[3] = T(b[1] * s), v[4] = T(c[0] * s), v[5] = T(c[1] * s), v[6] = T(e[0] * s), v[7] = T(e[1] * s);
        T* at = out + row * out_stride + d;
        if (d + 8 <= dim) {
            loose_store(at, v);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (d + i < dim) at[i] = v[i];
        }
    }
}

struct Product {
    const uint8_t *codes, *scales;  // the items'
    uint64_t codes_stride, scales_stride;
    const void* queries;  // their codes, or the rows
    const uint8_t* query_scales;
    uint64_t query_stride, query_scales_stride;
    const float* offsets;
    void* out;
    uint64_t out_stride;
    uint32_t T, V, dim, groups;
    float scale;
};

// Eight values as P bf16 ones each, whose sum they are (fp16: two, fp32: three): the upper 8 binary digits cut off (a rounding
// could overflow), then the next ones.  NaN and inf are in the first alone.
template <int P>
__device__ __forceinline__ void planes(const float (&v)[8], bf16x8 (&o)[P]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        if constexpr (P == 1) {
            o[0][e] = __bf16(v[e]);
        } else {
            const bool odd = (__float_as_uint(v[e]) & 0x7F800000u) == 0x7F800000u;
            const float hi = odd ? v[e] : __uint_as_float(__float_as_uint(v[e]) & 0xFFFF0000u);
            float rest = odd ? 0.0f : v[e] - hi;
            o[0][e] = __bf16(hi);
#pragma unroll
            for (int p = 1; p < P; ++p) {
                o[p][e] = __bf16(rest);
                rest -= float(o[p][e]);
            }
        }
    }
}

// ---------------------------------------------------------------------------------------
// Coded queries: tiles through LDS
// ---------------------------------------------------------------------------------------
// A wave computes 64 queries x 64 items (2 x 2 blocks of v_mfma_scale_f32_32x32x64_f8f6f4, fp32 sums), a workgroup WQ x WI such
// waves.  One or two groups of 128 values of both operands (64 bytes of codes and 4 of scales a row each; two are a whole
// line of memory) are a stage; stages move global -> LDS by direct loads into three slots, three stages ahead, across tiles:
// the launch is persistent.  A group is two steps of 64 values, four products each; behind each product of the first one
// fragments of the second are read, behind those of the second the next group's first ones; where a stage ends, after its one
// barrier, the slot that it leaves is filled anew.
// Short rows make many scores of few products, so a launch is bound by their way to memory as much as by the matrix
// cores: a tile's sums stay in registers while the next tile's go to a second set, and are written between its products, a
// few at a time.  Written all at once they filled the memory pipe, and the loads behind them waited (4096 x 262,144 x 768
// to bf16: 410 us of stores and 500 us of products took 1000).
// The 16-byte chunks of an LDS row are swizzled by the row, so fragment reads meet in no bank.  An item goes to the LDS row that puts
// two neighbours into one lane: a half-wave writes 64 neighbouring scores of a query, whole lines, from its registers.
// Measured: 4096 x 262,144 x 768 to bf16 745-785 us, 2.2 PFLOP/s and 2.8 TB/s of scores (660 where the clock is up).  No unit is full: the
// matrix cores are busy for 27 % of the time, LDS for 17 %; a wave spends 30 % at waits and barriers.  What bounds it is how little the products
// (470 us without the stores; their instructions alone 300) and the stores (410 alone) overlap: a CU has one workgroup, whose eight
// waves meet at a barrier a stage.  512 x 100,003 x 384 to fp32: 43-45 us, its scores at 4.7 TB/s with the outputs in cache, 63 from memory:
// rows that begin inside lines are written in pieces of lines.
template <int WQ_, int WI_, int GS_>
struct Shape {
    static constexpr int WQ = WQ_, WI = WI_, GS = GS_, WAVES = WQ * WI, THREADS = 64 * WAVES;
    static constexpr int TQ = 64 * WQ, TI = 64 * WI;
    static constexpr int ROWB = GS * int(kCodes), CHUNKS = ROWB / 16;  // bytes of an LDS row
    // direct loads a wave and stage: of queries' codes, of all codes, of items' scales, of all scales
    static constexpr int LQ = TQ * ROWB / 1024 / WAVES, LC = (TQ + TI) * ROWB / 1024 / WAVES;
    static constexpr int LXS = (TI / 64 * GS + WAVES - 1) / WAVES, LS = LXS + (TQ / 64 * GS + WAVES - 1) / WAVES, L = LC + LS;
    static constexpr int SCALES = (TQ + TI) * ROWB, SLOT = SCALES + LS * WAVES * 256, LDS = 3 * SLOT;
    static constexpr int PER_SIMD = 2;  // waves, as the registers allow
    static constexpr int PER_CU = std::min(163840 / LDS, 4 * PER_SIMD / WAVES);
    static_assert(TQ * ROWB % (1024 * WAVES) == 0 && TI * ROWB % (1024 * WAVES) == 0 && (GS == 1 || GS == 2) && TI / 64 * GS % WAVES == 0, "shape");
};

// The tiles of a launch: every XCD takes a contiguous range of them, in strips of kStrip item blocks, along which the query
// blocks pass.  (Its workgroups, side by side in the strip, write neighbouring lines and read each operand's rows a few times
// each; with all query blocks of one item block at once their lines are a row of the output apart, and 4096 x 262,144 took
// a fifth longer.)
constexpr uint32_t kStrip = 8;
struct Tiles {
    uint32_t nq, ni;
    __device__ __forceinline__ uint32_t per() const { return (nq * ni + kXcds - 1) / kXcds; }
    // the place of the workgroup's i-th tile; false: there is none
    __device__ __forceinline__ bool at(uint32_t i, uint32_t& qb, uint32_t& ib) const {
        const uint32_t xcd = blockIdx.x % kXcds, seq = blockIdx.x / kXcds + i * (gridDim.x / kXcds), t = xcd * per() + seq;
        if (seq >= per() || t >= nq * ni) return false;
        const uint32_t strip = t / (kStrip * nq), in = t % (kStrip * nq), width = min(kStrip, ni - strip * kStrip);
        ib = strip * kStrip + in % width;
        qb = in / width;
        return true;
    }
};

// The scores of a wave: 32 QB queries x 64 items.
template <class O, int QB>
struct Sums {
    static constexpr int kStores = 16 * QB;
    f32x16 acc[QB][2];  // acc[m][n][4 j + e]: query 32 m + 8 j + 4 hh + e against item 2 l32 + n of the wave's
    O* to;             // of the lane's first query and item
    float offset[2];
    uint32_t q, i;     // the lane's first query and item

    __device__ __forceinline__ f32x16& sum(int m, int n) { return acc[m][n]; }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int m = 0; m < QB; ++m)
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[m][n][e] = 0.0f;
    }
    __device__ __forceinline__ void place(const Product& a, uint32_t q0, uint32_t i0, int l32, int hh) {
        q = q0 + 4 * uint32_t(hh);
        i = i0 + 2 * uint32_t(l32);
        to = static_cast<O*>(a.out) + q * a.out_stride + i;
#pragma unroll
        for (int n = 0; n < 2; ++n) offset[n] = a.offsets && i + n < a.V ? a.offsets[i + n] : 0.0f;
    }
    static __device__ __forceinline__ constexpr uint32_t row(int k) { return 32 * (k >> 4) + 8 * ((k & 15) >> 2) + (k & 3); }
    __device__ __forceinline__ O score(const Product& a, int k, int n) const {
        const float y = fmaf(acc[k >> 4][n][k & 15], a.scale, offset[n]);
        return O(offset[n] == -__builtin_inff() ? offset[n] : y);
    }
    // Store k, of a wave whose queries and items are all there: two neighbouring scores a lane.  LINES: the rows begin at lines
    // of memory; whole lines then pass the caches by and leave them to the operands (4096 x 262,144 x 768: 805, not 861 us; lines in
    // pieces, 512 x 100,003 x 384: 96, not 45).
    template <bool LINES>
    __device__ __forceinline__ void store(const Product& a, int k) const {
        using V2 = Vec<O, 2>;
        O* const p = to + row(k) * a.out_stride;
        const V2 v = {score(a, k, 0), score(a, k, 1)};
        if (LINES) __builtin_nontemporal_store(v, reinterpret_cast<V2*>(p));
        else loose_store(p, v);
    }
    __device__ __forceinline__ void store_some(const Product& a) const {
#pragma unroll
        for (int k = 0; k < kStores; ++k)
            if (q + row(k) < a.T) {
                O* const p = to + row(k) * a.out_stride;
                if (i < a.V) p[0] = score(a, k, 0);
                if (i + 1 < a.V) p[1] = score(a, k, 1);
            }
    }
};

template <class Sh, class O, bool LINES>
__global__ __launch_bounds__(Sh::THREADS, Sh::PER_SIMD) void mx_tile_kernel(Product a, Tiles tiles) {
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    constexpr int kStores = Sums<O, 2>::kStores;
    // rows of codes a direct load; loads a wave of queries' codes, of all codes, of items' scales, of all scales
    constexpr int WAVES = Sh::WAVES, GS = Sh::GS, CH = Sh::CHUNKS, RL = 64 / CH, LQ = Sh::LQ, LC = Sh::LC, LXS = Sh::LXS, LS = Sh::LS;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l32 = lane & 31, hh = lane >> 5, wq = wave % Sh::WQ, wi = wave / Sh::WQ;
    const uint32_t lds0 = lds_addr_of(lds), qp = uint32_t(a.query_stride), xp = uint32_t(a.codes_stride), qsp = uint32_t(a.query_scales_stride), xsp = uint32_t(a.scales_stride);
    const uint32_t groups = a.groups, stages = (groups + GS - 1) / GS;

    // Codes: RL LDS rows a load, first the queries', then the items'; lane: row l / CH of them, physical chunk l % CH = logical chunk
    // (l % CH) ^ (the row's swizzle).  Scales: a dword of 64 rows a load, one group's rows behind the other's, first the items'.
    uint32_t code_off[LC], scale_off[LS];
#pragma unroll
    for (int j = 0; j < LC; ++j) {
        const uint32_t row = uint32_t(wave + WAVES * (j < LQ ? j : j - LQ)) * RL + uint32_t(lane / CH);
        code_off[j] = j < LQ ? mx_code_offset<GS>(row, uint32_t(lane % CH), row, qp) : mx_code_offset<GS>(row, uint32_t(lane % CH), mx_item_of(row), xp);
    }
#pragma unroll
    for (int j = 0; j < LS; ++j) {
        const uint32_t g = uint32_t(wave + WAVES * (j < LXS ? j : j - LXS)), blocks = uint32_t(j < LXS ? Sh::TI : Sh::TQ) / 64;
        const uint32_t row = g % blocks * 64 + uint32_t(lane);
        // (a wave without rows of its own loads zeros into a place of its own)
        scale_off[j] = g < blocks * GS ? (j < LXS ? mx_scale_offset(g / blocks, mx_item_of(row), xsp) : mx_scale_offset(g / blocks, row, qsp)) : kDmaSkip;
    }
    dma_rsrc from_q, from_x, from_qs, from_xs;
    const auto open = [&](uint32_t i) {
        uint32_t qb = 0, ib = 0;
        const bool there = tiles.at(i, qb, ib);
        const uint32_t q0 = qb * Sh::TQ, i0 = ib * Sh::TI, nq = min(uint32_t(Sh::TQ), a.T - q0), ni = min(uint32_t(Sh::TI), a.V - i0);
        // (where there is no tile more: nothing lies behind the descriptors, and zeros arrive)
        from_q = make_dma_rsrc(static_cast<const char*>(a.queries) + uint64_t(q0) * qp, there ? mx_records(nq, qp, groups, kMxCodes) : 0);
        from_x = make_dma_rsrc(a.codes + uint64_t(i0) * xp, there ? mx_records(ni, xp, groups, kMxCodes) : 0);
        from_qs = make_dma_rsrc(a.query_scales + uint64_t(q0) * qsp, there ? mx_records(nq, qsp, groups, kMxScales) : 0);
        from_xs = make_dma_rsrc(a.scales + uint64_t(i0) * xsp, there ? mx_records(ni, xsp, groups, kMxScales) : 0);
        return there;
    };
    uint32_t ahead_tile = 0, ahead_stage = 0, ahead_slot = 0;
    // load j of the L of the stage that is three ahead
    const auto load = [&](int j) {
        const uint32_t to = lds0 + ahead_slot * uint32_t(Sh::SLOT) + uint32_t(wave) * (j < LC ? 1024u : 256u);
        if (j < LC) lds_dma16(j < LQ ? from_q : from_x, mx_stage_offset(code_off[j], ahead_stage, Sh::ROWB), to + uint32_t(j * WAVES * 1024));
        else lds_dma4(j - LC < LXS ? from_xs : from_qs, mx_stage_offset(scale_off[j - LC], ahead_stage, kMxScales * GS), to + uint32_t(Sh::SCALES + (j - LC) * WAVES * 256));
    };
    const auto loaded = [&] {
        ahead_slot = ahead_slot == 2 ? 0 : ahead_slot + 1;
        if (++ahead_stage == stages) {
            ahead_stage = 0;
            (void)open(++ahead_tile);
        }
    };
    const auto barrier = [] { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };

    // fragments: block b's lane reads row l32 of it, half hh of a step's 64 values
    const int swz = int(mx_swizzle<GS>(uint32_t(l32)));
    const char* const my_q = lds + (wq * 64 + l32) * Sh::ROWB;
    const char* const my_x = lds + (Sh::TQ + wi * 64 + l32) * Sh::ROWB;
    const char* const my_xs = lds + Sh::SCALES + (wi * 64 + l32) * 4;
    const char* const my_qs = lds + Sh::SCALES + LXS * WAVES * 256 + (wq * 64 + l32) * 4;
    u32x4 fq[2][2], fx[2][2];
    uint32_t sq[2], sx[2], nsq[2], nsx[2];
    uint32_t slot = 0;
    // fragment j of step t of the stage's group `sub`: a query block's, an item block's in turn; with the first step the group's scales
    const auto read = [&](int sub, int t, int j) {
        const int at = int(slot) * Sh::SLOT, chunk = 16 * ((4 * sub + 2 * t + hh) ^ swz), b = j >> 1;
        if (j & 1) {
            fx[t][b] = *reinterpret_cast<const u32x4*>(my_x + at + b * 32 * Sh::ROWB + chunk);
            if (t == 0) nsx[b] = *reinterpret_cast<const uint32_t*>(my_xs + at + sub * Sh::TI * 4 + b * 128);
        } else {
            fq[t][b] = *reinterpret_cast<const u32x4*>(my_q + at + b * 32 * Sh::ROWB + chunk);
            if (t == 0) nsq[b] = *reinterpret_cast<const uint32_t*>(my_qs + at + sub * Sh::TQ * 4 + b * 128);
        }
    };
    const auto multiply = [&](Sums<O, 2>& to, auto step, int j) {
        constexpr int t = decltype(step)::value;
        const auto wide = [](const u32x4& v) { return i32x8{int(v[0]), int(v[1]), int(v[2]), int(v[3]), 0, 0, 0, 0}; };
        const int m = j >> 1, n = (j ^ m) & 1;
        __builtin_amdgcn_sched_barrier(0);
        // (byte 2 t + hh of the group's scales: they are shifted by hh)
        to.acc[m][n] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wide(fq[t][m]), wide(fx[t][n]), to.acc[m][n], 4, 4, 2 * t, int(sq[m]), 2 * t, int(sx[n]));
        __builtin_amdgcn_sched_barrier(0);
    };
    const auto take_scales = [&] {
#pragma unroll
        for (int b = 0; b < 2; ++b) sq[b] = nsq[b] >> (8 * hh), sx[b] = nsx[b] >> (8 * hh);
    };
    const std::integral_constant<int, 0> first{};
    const std::integral_constant<int, 1> second{};

    // Stage s into `to`, and (part >= 0) half of the stores of `from`.
    const auto stage = [&](Sums<O, 2>& to, const Sums<O, 2>& from, uint32_t s, auto part) {
        constexpr int P = decltype(part)::value;
        const auto write = [&](int k, int n) {
            if constexpr (P >= 0) {
#pragma unroll
                for (int e = 0; e < n; ++e) from.template store<LINES>(a, P * (kStores / 2) + k + e);
            }
        };
        take_scales();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            multiply(to, first, j);
            read(0, 1, j);
            write(2 * j, 2);
        }
        if (GS == 2 && 2 * s + 1 < groups) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                multiply(to, second, j);
                read(GS - 1, 0, j);
                write(8 + 2 * j, 2);
            }
            take_scales();
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                multiply(to, first, j);
                read(GS - 1, 1, j);
            }
        } else {
            write(8, 8);
        }
        multiply(to, second, 0);
        // The next stage has arrived for every wave (loads and stores end in the order of their issue: what came behind its loads, the
        // next stage's and this tile's stores, need not have ended), and every wave has read this one, whose slot is filled anew.
        wait_vmcnt<Sh::L + (P + 1) * (kStores / 2)>();
        barrier();
        slot = slot == 2 ? 0 : slot + 1;
        read(0, 0, 0), read(0, 0, 1);
#pragma unroll
        for (int j = 0; j < Sh::L / 3; ++j) load(j);
        multiply(to, second, 1);
        read(0, 0, 2), read(0, 0, 3);
#pragma unroll
        for (int j = Sh::L / 3; j < 2 * Sh::L / 3; ++j) load(j);
        multiply(to, second, 2);
#pragma unroll
        for (int j = 2 * Sh::L / 3; j < Sh::L; ++j) load(j);
        multiply(to, second, 3);
        loaded();
    };
    // The workgroup's i-th tile into `to`, and the stores of `from` where they are still to be made; whether it has one more behind
    // it, and whether `to` is still to be stored.
    const auto tile = [&](Sums<O, 2>& to, const Sums<O, 2>& from, uint32_t i, bool& stores) {
        const std::integral_constant<int, -1> none{};
        to.clear();
        uint32_t s = 0;
        if (stores) {
            stage(to, from, 0, first);
            if (stages > 1) {
                stage(to, from, 1, second);
            } else {
#pragma unroll
                for (int k = kStores / 2; k < kStores; ++k) from.template store<LINES>(a, k);
            }
            s = 2;
        }
        for (; s < stages; ++s) stage(to, from, s, none);
        uint32_t qb = 0, ib = 0;
        (void)tiles.at(i, qb, ib);
        const uint32_t q0 = qb * Sh::TQ + wq * 64, i0 = ib * Sh::TI + wi * 64;
        to.place(a, q0, i0, l32, hh);
        stores = q0 + 64 <= a.T && i0 + 64 <= a.V;
        if (!stores) to.store_some(a);
        return tiles.at(i + 1, qb, ib);
    };

    if (!open(0)) return;
#pragma unroll
    for (int k = 0; k < 3; ++k) {
#pragma unroll
        for (int j = 0; j < Sh::L; ++j) load(j);
        loaded();
    }
    wait_vmcnt<2 * Sh::L>();
    barrier();
#pragma unroll
    for (int j = 0; j < 4; ++j) read(0, 0, j);
    Sums<O, 2> one, two;
    bool stores = false;
    for (uint32_t i = 0;; i += 2) {
        if (!tile(one, two, i, stores)) {
            two = one;
            break;
        }
        if (!tile(two, one, i + 1, stores)) break;
    }
    if (stores) {
#pragma unroll
        for (int k = 0; k < kStores; ++k) two.template store<LINES>(a, k);
    }
    wait_vmcnt<0>();
}

// The scores of a wave: 16 queries x 64 items, acc[n][e]: query 4 (l / 16) + e against item 4 (l % 16) + n.
template <class O>
struct Sums<O, 0> {
    f32x4 acc[4];
    O* to;
    float offset[4];
    uint32_t q, i;

    __device__ __forceinline__ f32x4& sum(int, int n) { return acc[n]; }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int n = 0; n < 4; ++n) acc[n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    __device__ __forceinline__ void write(const Product& a, uint32_t q0, uint32_t i0, int lane) {
        using V4 = Vec<O, 4>;
        q = q0 + 4 * uint32_t(lane >> 4);
        i = i0 + 4 * uint32_t(lane & 15);
        to = static_cast<O*>(a.out) + q * a.out_stride + i;
#pragma unroll
        for (int n = 0; n < 4; ++n) offset[n] = a.offsets && i + n < a.V ? a.offsets[i + n] : 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (q + e < a.T) {
                V4 v;
#pragma unroll
                for (int n = 0; n < 4; ++n) v[n] = O(offset[n] == -__builtin_inff() ? offset[n] : fmaf(acc[n][e], a.scale, offset[n]));
                if (i + 4 <= a.V) {
                    loose_store(to + e * a.out_stride, v);
                } else {
#pragma unroll
                    for (int n = 0; n < 4; ++n)
                        if (i + n < a.V) to[e * a.out_stride + n] = v[n];
                }
            }
    }
};

// ---------------------------------------------------------------------------------------
// Queries as they are
// ---------------------------------------------------------------------------------------
// The items' codes become bf16 values on their way to the matrix cores (v_cvt_scalef32_pk_bf16_fp4: e2m1 times a power of two has
// one exactly), the queries are P bf16 planes whose sum they are, so every product is exact, and the sums are fp32
// (v_mfma_f32_32x32x16_bf16).  A wave computes 32 QB queries x 64 items; a lane's 16 bytes of codes
// (a block) feed four products of each block of queries.  The queries' planes lie in LDS: all of them,
// loaded once for a workgroup's many tiles, where they fit (RESIDENT: no barrier, every wave streams by itself); else a
// group at a time in two slots, the next one's values in registers meanwhile, and the tiles in strips as above.  LDS rows are 256 bytes, chunks swizzled by the row.
// Measured: 1 x 10,000 x 768 8.3 us, a launch; 10 x 1M x 768 in fp16 107 us, the items at 4.1 TB/s; 32 x 1M x 768 in bf16 118 us; 4096 x
// 65,536 x 768 in bf16 567 us, 728 TFLOP/s, in fp16 816 us, twice 505: bound by the matrix cores and, beside them, the items'
// conversion for every 64 queries.
// Slots of a wave's items: three; of two waves, few in a launch, so many that a short row's loads are all under way; two where the
// queries are staged, whose groups take longer than a load.
constexpr int slots_of(int waves, bool resident) { return !resident ? 2 : waves == 2 ? 8 : 3; }
constexpr uint32_t items_lds(int waves, bool resident) { return uint32_t(waves * slots_of(waves, resident)) * (64 * kCodes + 256); }
template <class QT, int P, int QB, int WAVES, bool RESIDENT, class O>
__global__ __launch_bounds__(64 * WAVES, 2) void mx_rows_kernel(Product a, Tiles tiles) {
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    constexpr int TQ = QB ? 32 * QB : 16, TI = 64 * WAVES, THREADS = 64 * WAVES, UNITS = TQ * 16 / THREADS > 0 ? TQ * 16 / THREADS : 1;
    static_assert(RESIDENT || (QB && TQ * 16 % THREADS == 0), "whole units");
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l32 = lane & 31, hh = lane >> 5;
    const uint32_t groups = a.groups;
    // rows in LDS: those that there are (what a lane behind them computes is not written)
    const int held = int(min(uint32_t(TQ), a.T)), PLANE = held * 256, SLOT = P * PLANE;

    // eight values of a query row: unit u of a group is row u / 16, values 8 (u % 16) on
    const auto fetch = [&](uint32_t q0, uint32_t g, int u, float (&v)[8]) {
        const uint32_t r = q0 + uint32_t(u) / 16, d = g * kGroup + 8 * (uint32_t(u) % 16);
        if (r < a.T && d < a.dim) {
            load8(static_cast<const QT*>(a.queries) + r * a.query_stride, d, a.dim, v);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = 0.0f;
        }
    };
    const auto keep = [&](uint32_t slot, int u, const float (&v)[8]) {
        const int r = u / 16, c = u % 16;
        bf16x8 o[P];
        planes<P>(v, o);
#pragma unroll
        for (int p = 0; p < P; ++p) *reinterpret_cast<bf16x8*>(lds + slot * SLOT + p * PLANE + r * 256 + 16 * (c ^ (r & 15))) = o[p];
    };

    struct Items {
        u32x4 x[2][2];  // [block][half group]; 16 queries: four blocks
        uint32_t s[4];
    };
    // the workgroup's i-th tile: its first query, the wave's first item; false: there is none
    const auto place = [&](uint32_t i, uint32_t& q0, uint32_t& i0) {
        if constexpr (RESIDENT) {
            const uint32_t t = blockIdx.x + i * gridDim.x;
            q0 = 0, i0 = t * TI + wave * 64;
            return t < tiles.ni;
        } else {
            uint32_t qb = 0, ib = 0;
            const bool there = tiles.at(i, qb, ib);
            q0 = qb * TQ, i0 = ib * TI + wave * 64;
            return there;
        }
    };
    Sums<O, QB> sums;
    const auto widened = [](uint32_t c, float scale) {
        typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
        const bf16x2 w0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 0), w1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 1),
                     w2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 2), w3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 3);
        return bf16x8{w0[0], w0[1], w1[0], w1[1], w2[0], w2[1], w3[0], w3[1]};
    };
    const auto multiplied = [](bf16x8 q, bf16x8 w, auto c) {
        if constexpr (QB == 0) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(q, w, c, 0, 0, 0);
        else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(q, w, c, 0, 0, 0);
    };
    // A group.  32 queries a block: a lane has half hh of each half group of an item of two blocks.  16 queries: block l / 16 of the
    // group of an item of each of four blocks, and takes v_mfma_f32_16x16x32.
    constexpr int BLOCKS = QB ? 2 : 4, HALVES = QB ? 2 : 1, QBLOCKS = QB ? QB : 1;
    const int part = QB ? hh : lane >> 4;
    const auto code_of = [](const Items& o, int n, int h) { return QB ? o.x[n][h] : o.x[n >> 1][n & 1]; };
    const auto byte_of = [&](const Items& o, int n, int h) { return (o.s[n] >> (8 * (QB ? 2 * h + part : part))) & 255u; };
    const auto multiply = [&](uint32_t slot, const Items& o) {
        const char* at[QBLOCKS];
        int swz[QBLOCKS];
#pragma unroll
        for (int m = 0; m < QBLOCKS; ++m) {
            const int row = min(QB ? 32 * m + l32 : lane & 15, held - 1);
            at[m] = lds + slot * SLOT + row * 256;
            swz[m] = row & 15;
        }
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
            float scale[BLOCKS];
#pragma unroll
            for (int n = 0; n < BLOCKS; ++n) scale[n] = __uint_as_float(byte_of(o, n, h) << 23);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int chunk = (QB ? 8 * h : 0) + 4 * part + k;
                bf16x8 q[QBLOCKS][P], w[BLOCKS];
#pragma unroll
                for (int m = 0; m < QBLOCKS; ++m)
#pragma unroll
                    for (int p = 0; p < P; ++p) q[m][p] = *reinterpret_cast<const bf16x8*>(at[m] + p * PLANE + 16 * (chunk ^ swz[m]));
#pragma unroll
                for (int n = 0; n < BLOCKS; ++n) w[n] = widened(code_of(o, n, h)[k], scale[n]);
#pragma unroll
                for (int p = P - 1; p >= 0; --p)  // the smallest first
#pragma unroll
                    for (int n = 0; n < BLOCKS; ++n)
#pragma unroll
                        for (int m = 0; m < QBLOCKS; ++m) sums.sum(m, n) = multiplied(q[m][p], w[n], sums.sum(m, n));
            }
        }
    };
    // the sums; whether they went as whole stores, Sums::kStores of them
    const auto write = [&](uint32_t q0, uint32_t i0) {
        bool whole = false;
        if constexpr (QB == 0) {
            sums.write(a, q0, i0, lane);
        } else {
            sums.place(a, q0, i0, l32, hh);
            whole = q0 + TQ <= a.T && i0 + 64 <= a.V;
            if (whole) {
#pragma unroll
                for (int k = 0; k < Sums<O, QB>::kStores; ++k) sums.template store<false>(a, k);
            } else {
                sums.store_some(a);
            }
        }
        sums.clear();
        return whole;
    };

    uint32_t tile = 0, q0, i0;
    if (!place(0, q0, i0)) return;
    sums.clear();
    // A wave's items come through LDS of its own, kAhead groups ahead and across tiles: direct loads take a row's 64 bytes in four
    // neighbouring lanes, and 1M rows of 768 values pass at 5 TB/s; read straight into the lanes that multiply them, each of
    // which takes another row, at 3.4.
    constexpr int SLOT_X = 64 * int(kCodes) + 256, L = 5, kSlots = slots_of(WAVES, RESIDENT), kAhead = kSlots - 1;
    char* const mine = lds + (RESIDENT ? int(groups) : 2) * SLOT + wave * kSlots * SLOT_X;
    const uint32_t to0 = lds_addr_of(mine);
    const auto item_of = [](uint32_t r) { return QB ? r % 32u * 2u + r / 32u : r % 16u * 4u + r / 16u; };  // of an LDS row
    uint32_t code_off[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t row = 16u * j + uint32_t(lane >> 2);
        code_off[j] = item_of(row) * uint32_t(a.codes_stride) + 16u * (uint32_t(lane & 3) ^ ((row >> 2) & 3));
    }
    const uint32_t scale_off = item_of(uint32_t(lane)) * uint32_t(a.scales_stride);
    uint32_t ahead_tile = 0, ahead_g = 0, ahead_slot = 0, slot = 0;
    dma_rsrc from_x, from_s;
    const auto open = [&] {
        uint32_t q, i;
        const bool there = place(ahead_tile, q, i) && i < a.V;
        const uint32_t first = there ? i : 0, rows = there ? min(64u, a.V - i) - 1 : 0;
        from_x = make_dma_rsrc(a.codes + uint64_t(first) * a.codes_stride, there ? rows * uint32_t(a.codes_stride) + groups * kCodes : 0);
        from_s = make_dma_rsrc(a.scales + uint64_t(first) * a.scales_stride, there ? rows * uint32_t(a.scales_stride) + groups * 4 : 0);
    };
    const auto advance = [&] {
        const uint32_t to = to0 + ahead_slot * SLOT_X;
#pragma unroll
        for (int j = 0; j < 4; ++j) lds_dma16_so(from_x, code_off[j], ahead_g * kCodes, to + j * 1024u);
        lds_dma4_so(from_s, scale_off, ahead_g * 4u, to + 4096u);
        ahead_slot = ahead_slot + 1 == kSlots ? 0 : ahead_slot + 1;
        if (++ahead_g == groups) {
            ahead_g = 0;
            ++ahead_tile;
            open();
        }
    };
    // the next group's items, out of a slot that the group behind them may then fill
    const auto take = [&] {
        Items now;
        const char* const at = mine + slot * SLOT_X;
#pragma unroll
        for (int n = 0; n < BLOCKS; ++n) {
            const int row = QB ? 32 * n + l32 : 16 * n + (lane & 15);
            const auto chunk = [&](int c) { return *reinterpret_cast<const u32x4*>(at + row * int(kCodes) + 16 * (c ^ ((row >> 2) & 3))); };
            now.s[n] = *reinterpret_cast<const uint32_t*>(at + 4096 + 4 * row);
            if constexpr (QB == 0) {
                now.x[n >> 1][n & 1] = chunk(part);
            } else {
#pragma unroll
                for (int h = 0; h < 2; ++h) now.x[n][h] = chunk(2 * h + part);
            }
        }
        slot = slot + 1 == kSlots ? 0 : slot + 1;
        return now;
    };
    open();
#pragma unroll
    for (int k = 0; k < kAhead; ++k) advance();
    if constexpr (RESIDENT) {
        for (uint32_t g = 0; g < groups; ++g)
            for (int u = tid; u < held * 16; u += THREADS) {
                float v[8];
                fetch(0, g, u, v);
                keep(g, u, v);
            }
        __syncthreads();
        do {
            for (uint32_t g = 0; g < groups; ++g) {
                // (loads end in the order of their issue; a tile's stores between them only make this wait for those)
                wait_vmcnt<(kAhead - 1) * L>();
                const Items now = take();
                advance();  // (into the slot that the group before this one has left)
                multiply(g, now);
            }
            (void)write(q0, i0);
        } while (place(++tile, q0, i0));
    } else {
        // The queries' values, two groups ahead in registers, one in LDS; behind the last tile's zeros.
        float next[UNITS][8];
        uint32_t fetch_tile = 0, fetch_g = 0, fetch_q0 = q0;
        const auto fetch_all = [&] {
#pragma unroll
            for (int i = 0; i < UNITS; ++i) fetch(fetch_q0, fetch_g, tid + THREADS * i, next[i]);
            if (++fetch_g == groups) {
                uint32_t i;
                fetch_g = 0;
                if (!place(++fetch_tile, fetch_q0, i)) fetch_q0 = a.T;
            }
        };
        const auto keep_all = [&](uint32_t to) {
#pragma unroll
            for (int i = 0; i < UNITS; ++i)
                if (tid + THREADS * i < held * 16) keep(to, tid + THREADS * i, next[i]);
        };
        fetch_all();
        keep_all(0);
        fetch_all();
        uint32_t n = 0;
        bool whole = false;
        do {
            for (uint32_t g = 0; g < groups; ++g, n ^= 1) {
                asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // group g is there, and every wave is done with the one before it
                keep_all(n ^ 1);
                // (the items, loaded a group ago, have come; the stores of the tile before, issued behind those, need not have gone)
                if (whole) wait_vmcnt<Sums<O, QB>::kStores>();
                else wait_vmcnt<0>();
                whole = false;
                const Items now = take();
                advance();
                fetch_all();
                multiply(n, now);
            }
            whole = write(q0, i0);
        } while (place(++tile, q0, i0));
    }
    wait_vmcnt<0>();  // direct loads under way end before the LDS is another's
}

template <class QT, int P, int QB, int WAVES, bool RESIDENT, class O>
va_status launch_rows(va_context* ctx, const Product& a, uint32_t bytes) {
    const Tiles tiles{ceil_div(a.T, QB ? 32 * QB : 16), ceil_div(a.V, 64 * WAVES)};
    const uint64_t total = uint64_t(tiles.nq) * tiles.ni;
    if (total > 0x7FFFFFF0ull) return fail(ctx, VA_ERR_INVALID_ARG, "product too large: %u x %u", a.T, a.V);
    auto kern = &mx_rows_kernel<QT, P, QB, WAVES, RESIDENT, O>;
    static std::atomic<uint64_t> allowed{0};  // the kernel may take its LDS: asked once per device
    const uint64_t bit = ctx->device < 64 ? 1ull << ctx->device : 0;
    if (!(allowed.load(std::memory_order_relaxed) & bit)) {
        VA_CHECK_HIP(ctx, hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, 163840));
        allowed.fetch_or(bit, std::memory_order_relaxed);
    }
    const uint32_t per_cu = std::max(1u, std::min(163840u / std::max(bytes, 1u), 8u / WAVES));
    const uint32_t cus = std::max(uint32_t(ctx->num_cus), kXcds) / kXcds * kXcds;
    const uint32_t grid = uint32_t(std::min<uint64_t>(RESIDENT ? total : (total + kXcds - 1) / kXcds * kXcds, uint64_t(cus) * per_cu));
    kern<<<dim3(grid), dim3(64 * WAVES), bytes, ctx->stream>>>(a, tiles);
    VA_CHECK_LAUNCH(ctx);
    return VA_OK;
}
// At most 16 queries (QB 0; 10 x 1M x 768 in fp16: 108 us, with 32 a block 125) or 32 (QB 1).  fits: whether LDS holds them all (32 x 1M x
// 768 in bf16: 118 us, a group at a time 187).
template <class QT, int P, int QB, class O>
va_status few_rows(va_context* ctx, const Product& a, bool& fits) {
    const uint64_t all = uint64_t(a.groups) * P * a.T * 256;
    fits = true;
    // as many waves as LDS has room for; of two where there would be fewer of four than CUs (100,000 items: 11.0 us, of eight 11.6)
    if (a.V < 256u * uint32_t(ctx->num_cus)) {
        if (all + items_lds(2, true) <= 163840) return launch_rows<QT, P, QB, 2, true, O>(ctx, a, uint32_t(all) + items_lds(2, true));
    } else if (all + items_lds(8, true) <= 163840) {
        return launch_rows<QT, P, QB, 8, true, O>(ctx, a, uint32_t(all) + items_lds(8, true));
    } else if (all + items_lds(4, true) <= 163840) {
        return launch_rows<QT, P, QB, 4, true, O>(ctx, a, uint32_t(all) + items_lds(4, true));
    }
    fits = false;
    return VA_OK;
}
template <class QT, int P, class O>
va_status rows_of(va_context* ctx, const Product& a) {
    if (a.T <= 32) {
        bool fits;
        const va_status st = a.T <= 16 ? few_rows<QT, P, 0, O>(ctx, a, fits) : few_rows<QT, P, 1, O>(ctx, a, fits);
        if (fits) return st;
        return launch_rows<QT, P, 1, 8, false, O>(ctx, a, 2 * P * a.T * 256 + items_lds(8, false));
    }
    // (64 queries: an item's values, made once, meet 64 of them; 128 spilled, 4096 x 65,536 x 768 in bf16 took 636, not 567 us.  Three
    // planes of 64 do not fit beside the items.)
    constexpr int QB = P == 3 ? 1 : 2;
    return launch_rows<QT, P, QB, 8, false, O>(ctx, a, 2 * P * std::min(a.T, 32u * QB) * 256 + items_lds(8, false));
}
template <class QT, int P>
va_status product(va_context* ctx, const Product& a, va_dtype out) {
    if (out == VA_DTYPE_F32) return rows_of<QT, P, float>(ctx, a);
    if (out == VA_DTYPE_F16) return rows_of<QT, P, _Float16>(ctx, a);
    return rows_of<QT, P, __bf16>(ctx, a);
}

template <class Sh, class O, bool LINES>
va_status launch_tiles(va_context* ctx, const Product& a) {
    const Tiles tiles{ceil_div(a.T, Sh::TQ), ceil_div(a.V, Sh::TI)};
    const uint64_t total = uint64_t(tiles.nq) * tiles.ni;
    if (total > 0x7FFFFFF0ull) return fail(ctx, VA_ERR_INVALID_ARG, "product too large: %u x %u", a.T, a.V);
    auto kern = &mx_tile_kernel<Sh, O, LINES>;
    if (Sh::LDS > 65536) {
        static std::atomic<uint64_t> allowed{0};  // the kernel may take its LDS: asked once per device
        const uint64_t bit = ctx->device < 64 ? 1ull << ctx->device : 0;
        if (!(allowed.load(std::memory_order_relaxed) & bit)) {
            VA_CHECK_HIP(ctx, hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, Sh::LDS));
            allowed.fetch_or(bit, std::memory_order_relaxed);
        }
    }
    const uint64_t most = std::max(uint32_t(ctx->num_cus), kXcds) / kXcds * kXcds * uint64_t(Sh::PER_CU);
    const uint64_t grid = std::min<uint64_t>((total + kXcds - 1) / kXcds * kXcds, most);
    kern<<<dim3(uint32_t(grid)), dim3(Sh::THREADS), Sh::LDS, ctx->stream>>>(a, tiles);
    VA_CHECK_LAUNCH(ctx);
    return VA_OK;
}
template <class Sh>
va_status tiles_of(va_context* ctx, const Product& a, va_dtype out) {
    const bool lines = aligned(a.out, 128) && a.out_stride * size_of(out) % 128 == 0;
    const auto go = [&](auto o) {
        using O = decltype(o);
        return lines ? launch_tiles<Sh, O, true>(ctx, a) : launch_tiles<Sh, O, false>(ctx, a);
    };
    if (out == VA_DTYPE_F32) return go(0.0f);
    if (out == VA_DTYPE_F16) return go(_Float16(0));
    return go(__bf16(0));
}
va_status coded_product(va_context* ctx, const Product& a, va_dtype out) {
    // (16 x 1M x 768 to fp32: 116 us by the first, 128 by the second; 64 x 1M x 768 136 and 135; 128 x 300,000 x 768 58 and 46)
    if (a.T <= 64) return tiles_of<Shape<1, 4, 1>>(ctx, a, out);
    return tiles_of<Shape<2, 4, 2>>(ctx, a, out);
}

va_status check_rows(va_context* ctx, const va_mx_rows* r, const char* what, const char* name) {
    VA_REQUIRE(ctx, r, "%s: %s is NULL", what, name);
    VA_REQUIRE(ctx, r->dim >= 1 && r->dim <= VA_MX_MAX_DIM, "%s: %s: dimension %u (1 to %u)", what, name, r->dim, VA_MX_MAX_DIM);
    if (!r->rows) return VA_OK;
    VA_REQUIRE(ctx, r->codes && r->scales, "%s: %s: a pointer is NULL", what, name);
    VA_REQUIRE(ctx, aligned(r->codes, 16) && aligned(r->scales, 4), "%s: %s: codes lie at multiples of 16 bytes, scales at multiples of 4", what, name);
    if (r->rows > 1) {
        const uint32_t g = groups_of(r->dim);
        VA_REQUIRE(ctx, r->codes_stride >= uint64_t(g) * kCodes && r->codes_stride % 16 == 0 && r->codes_stride <= VA_MX_MAX_DIM, "%s: %s: a codes stride of %llu", what, name,
                   (unsigned long long)r->codes_stride);
        VA_REQUIRE(ctx, r->scales_stride >= uint64_t(g) * 4 && r->scales_stride % 4 == 0 && r->scales_stride <= VA_MX_MAX_DIM, "%s: %s: a scales stride of %llu", what, name,
                   (unsigned long long)r->scales_stride);
    }
    return VA_OK;
}
va_status check_matrix(va_context* ctx, const void* p, uint64_t stride, uint32_t rows, uint32_t dim, va_dtype dtype, const char* what, const char* name) {
    VA_REQUIRE(ctx, known(dtype), "%s: %s: unknown type %d", what, name, int(dtype));
    if (!rows || !dim) return VA_OK;
    VA_REQUIRE(ctx, p, "%s: %s is NULL", what, name);
    VA_REQUIRE(ctx, aligned(p, size_of(dtype)), "%s: %s is not aligned to its type", what, name);
    VA_REQUIRE(ctx, rows == 1 || (stride >= dim && stride < 1ull << 32), "%s: %s: a stride of %llu for rows of %u", what, name, (unsigned long long)stride, dim);
    return VA_OK;
}

va_status finish(va_context* ctx, Product& a, const va_mx_rows* items, float scale, const float* offsets, void* out, uint64_t out_stride, va_dtype out_dtype, const char* what) {
    VA_CHECK_STATUS(check_matrix(ctx, out, out_stride, a.T, items->rows, out_dtype, what, "out"));
    VA_REQUIRE(ctx, std::isfinite(scale), "%s: the scale must be finite", what);
    VA_REQUIRE(ctx, aligned(offsets, 4), "%s: offsets are not aligned to their type", what);
    a.codes = items->codes, a.scales = items->scales;
    a.codes_stride = stride_of(items->rows, items->codes_stride, 0), a.scales_stride = stride_of(items->rows, items->scales_stride, 0);
    a.offsets = offsets, a.out = out, a.out_stride = stride_of(a.T, out_stride, items->rows);
    a.V = items->rows, a.dim = items->dim, a.groups = groups_of(items->dim), a.scale = scale;
    return VA_OK;
}

}  // namespace
}  // namespace va

using namespace va;

extern "C" {

va_status va_mx_quantize(va_context* ctx, const void* x, uint64_t x_stride, va_dtype dtype, const va_mx_rows* out) {
    if (!ctx) return VA_ERR_INVALID_ARG;
    VA_CHECK_STATUS(check_rows(ctx, out, "va_mx_quantize", "out"));
    VA_CHECK_STATUS(check_matrix(ctx, x, x_stride, out->rows, out->dim, dtype, "va_mx_quantize", "x"));
    if (!out->rows) return VA_OK;
    DeviceGuard guard(ctx->device);
    const uint32_t groups = groups_of(out->dim);
    const uint32_t grid = uint32_t(std::min<uint64_t>((uint64_t(out->rows) * groups + 15) / 16, 16u * uint32_t(ctx->num_cus)));
    const uint64_t xs = stride_of(out->rows, x_stride, out->dim), cs = stride_of(out->rows, out->codes_stride, 0), ss = stride_of(out->rows, out->scales_stride, 0);
    const auto go = [&](auto* p) {
        mx_quantize_kernel<<<dim3(grid), dim3(256), 0, ctx->stream>>>(p, xs, out->rows, out->dim, groups, out->codes, cs, out->scales, ss);
    };
    if (dtype == VA_DTYPE_F32) go(static_cast<const float*>(x));
    else if (dtype == VA_DTYPE_F16) go(static_cast<const _Float16*>(x));
    else go(static_cast<const __bf16*>(x));
    VA_CHECK_LAUNCH(ctx);
    return VA_OK;
}

va_status va_mx_dequantize(va_context* ctx, const va_mx_rows* rows, va_dtype dtype, void* out, uint64_t out_stride) {
    if (!ctx) return VA_ERR_INVALID_ARG;
    VA_CHECK_STATUS(check_rows(ctx, rows, "va_mx_dequantize", "rows"));
    VA_CHECK_STATUS(check_matrix(ctx, out, out_stride, rows->rows, rows->dim, dtype, "va_mx_dequantize", "out"));
    if (!rows->rows) return VA_OK;
    DeviceGuard guard(ctx->device);
    const uint32_t groups = groups_of(rows->dim);
    const uint32_t grid = uint32_t(std::min<uint64_t>((uint64_t(rows->rows) * groups + 15) / 16, 16u * uint32_t(ctx->num_cus)));
    const uint64_t os = stride_of(rows->rows, out_stride, rows->dim), cs = stride_of(rows->rows, rows->codes_stride, 0), ss = stride_of(rows->rows, rows->scales_stride, 0);
    const auto go = [&](auto* p) {
        mx_dequantize_kernel<<<dim3(grid), dim3(256), 0, ctx->stream>>>(rows->codes, cs, rows->scales, ss, rows->rows, rows->dim, groups, p, os);
    };
    if (dtype == VA_DTYPE_F32) go(static_cast<float*>(out));
    else if (dtype == VA_DTYPE_F16) go(static_cast<_Float16*>(out));
    else go(static_cast<__bf16*>(out));
    VA_CHECK_LAUNCH(ctx);
    return VA_OK;
}

va_status va_mx_product(va_context* ctx, const va_mx_rows* queries, const va_mx_rows* items, float scale, const float* offsets, va_dtype out_dtype, void* out,
                        uint64_t out_stride) {
    if (!ctx) return VA_ERR_INVALID_ARG;
    VA_CHECK_STATUS(check_rows(ctx, queries, "va_mx_product", "queries"));
    VA_CHECK_STATUS(check_rows(ctx, items, "va_mx_product", "items"));
    if (queries->dim != items->dim) return fail(ctx, VA_ERR_DIMENSION_MISMATCH, "va_mx_product: queries of %u dimensions, items of %u", queries->dim, items->dim);
    Product a{};
    a.T = queries->rows, a.queries = queries->codes, a.query_scales = queries->scales;
    a.query_stride = stride_of(a.T, queries->codes_stride, 0), a.query_scales_stride = stride_of(a.T, queries->scales_stride, 0);
    VA_CHECK_STATUS(finish(ctx, a, items, scale, offsets, out, out_stride, out_dtype, "va_mx_product"));
    if (!a.T || !a.V) return VA_OK;
    DeviceGuard guard(ctx->device);
    return coded_product(ctx, a, out_dtype);
}

va_status va_mx_product_rows(va_context* ctx, const void* queries, uint64_t queries_stride, va_dtype dtype, uint32_t num_queries, const va_mx_rows* items, float scale,
                             const float* offsets, va_dtype out_dtype, void* out, uint64_t out_stride) {
    if (!ctx) return VA_ERR_INVALID_ARG;
    VA_CHECK_STATUS(check_rows(ctx, items, "va_mx_product_rows", "items"));
    VA_CHECK_STATUS(check_matrix(ctx, queries, queries_stride, num_queries, items->dim, dtype, "va_mx_product_rows", "queries"));
    Product a{};
    a.T = num_queries, a.queries = queries, a.query_stride = stride_of(num_queries, queries_stride, items->dim);
    VA_CHECK_STATUS(finish(ctx, a, items, scale, offsets, out, out_stride, out_dtype, "va_mx_product_rows"));
    if (!a.T || !a.V) return VA_OK;
    DeviceGuard guard(ctx->device);
    if (dtype == VA_DTYPE_F32) return product<float, 3>(ctx, a, out_dtype);
    if (dtype == VA_DTYPE_F16) return product<_Float16, 2>(ctx, a, out_dtype);
    return product<__bf16, 1>(ctx, a, out_dtype);
}

}  // extern "C"
