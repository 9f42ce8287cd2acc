// va_gemm16.hpp — the matrix product of two operands, with the epilogue a template argument: every product
// of the softmax cross entropy (va_xent.hip, va_xent_grad.hip) is one of these.
//
//   acc[q][r] = sum_k Q[q][k] X[r][k]        fp16, bf16 or fp32
//
// Either operand is stored with k along its rows (Q[q] is a row) or across them (k is the row: QK, XK).
//
// A wave computes 64 queries x 64 rows (2 x 2 blocks of v_mfma_f32_32x32x16, 64 fp32 accumulators a
// lane; NB = 1: 32 queries, 4: 128), a workgroup WQ x WR such waves: 4 x 4 for large products (256 x 256, four waves per
// SIMD, one workgroup a CU), fewer where tiles of that size would leave CUs without work.  128 bytes of k (a stage)
// of both operands move global -> LDS by direct loads into one of two slots while the other is computed on (four
// slots where a launch does not fill the chip and waits for each stage).  Where there are few tiles with many
// stages, SLICES groups of waves take a share of a tile's stages each, with slots of their own, and the sums
// join in the first one's registers.  LDS rows are 128 bytes with their 16-byte chunks swizzled by the row, so
// fragment reads are conflict-free.  An operand stored across k is staged as it lies, the stage's k-rows of the
// tile's width, and ds_read_tr16 turns it on the way into the fragments (a lane receives four k of one
// column); its 64-byte segments are swizzled by k, so that four k-rows meet in no bank.  Rows need no
// alignment but a dword's, and k may end anywhere: behind the end the row operand's values are cleared in its
// fragments, and the query operand's are zeros in memory.  The launch is persistent: a workgroup walks its tiles, and the
// next tile's first stage streams in during the epilogue.
//
// Bound by the matrix cores at the clock that the card's power leaves them: 8192^3 in bf16 runs at 1.3 PFLOP/s,
// 4096 x 262,144 x 768 with the loss's epilogue at 1.03 (the vendor library's plain products of those shapes: 1.56 and 1.02).
// Eight waves of 128 x 64 reach 1.30 and 1.05, four of 128 x 128 1.20 and 0.88, slots of half a stage 1.13
// and 0.97: MFMA busy times clock is nearly the same for all.
//
// fp32 operands come in three ways.  F32: as they are, on v_mfma_f32_32x32x2: a fragment's 16 bytes are four k-values
// instead of eight, everything else is alike; a sixteenth of the 16-bit rate, which is enough while the
// operands' bytes are what takes the time.  PLANES: as two fp16 planes (value = (hi + lo) 2^-e with one
// exponent a row): a product is then hi hi + hi lo + lo hi, into the same accumulators.  The planes
// alternate in memory, 16 values of hi and the same 16 of lo, so a stage holds both of 32 values and each
// fragment is read once for its two products.  lo lo is below 2^-22 of the product and is left out; a value is exact to
// 2^-22 of it, or, where that is more, to 2^-39 of its row's largest: fp32's exactness for rows whose values are
// within 17 binary orders of each other, and not its range.  So planes are for sums over a row's values alone.
// SPLIT: as they are in memory and LDS, and split in the fragments into three bf16 values, which have fp32's range and
// together all its digits; six products of 16-bit rate.  For the sums across rows, whose terms may be of any size.
// Loss and gradients of 4096 x 20,000 x 768 with these sums in SPLIT 2.29 ms, in F32 2.78; 100 x 10,000 x 768
// 118 and 137 us.
#pragma once

#include <algorithm>
#include <atomic>
#include <type_traits>
#include <utility>

#include "va_internal.hpp"

namespace va {
namespace g16 {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int ROWB = 128;  // bytes of an LDS row (k along the rows)

// What the operands are made of.
enum Kind : int { F16 = 0, BF16 = 1, PLANES = 2, F32 = 3, SPLIT = 4 };
constexpr int size_of(int kind) { return kind >= PLANES ? 4 : 2; }  // bytes of a value in memory
constexpr int stage_of(int kind) { return ROWB / size_of(kind); }     // k-values of a stage

template <int WQ_, int WR_, int NB_ = 2, int SLOTS_ = 2, int SLICES_ = 1>
struct Shape {
    static constexpr int SLOTS = SLOTS_;  // a power of two
    static constexpr int WQ = WQ_, WR = WR_, NB = NB_, SLICES = SLICES_;
    static constexpr int WPS = WQ * WR;  // waves of a slice
    static constexpr int WAVES = WPS * SLICES, THREADS = 64 * WAVES;
    static constexpr int TQ = 32 * NB * WQ, TR = 64 * WR;
    static constexpr int QB = TQ * ROWB, XB = TR * ROWB, STAGE = QB + XB, LDS = SLICES * SLOTS * STAGE;
    // waves per SIMD that the registers allow for: all of a CU's (16 waves), or two workgroups' and more
    static constexpr int PER_SIMD = WAVES == 16 ? 4 : LDS <= 80 * 1024 ? 2 : 1;
    static_assert(THREADS >= TQ && THREADS >= TR, "one thread per query and row");
    static_assert(WPS * 4096 <= STAGE, "the epilogue's LDS fits in one slot");
    static_assert(SLICES == 1 || WPS * NB * 8192 <= STAGE, "a slice's sums fit in one slot");
};
using Large = Shape<4, 4>;

struct Operand {
    const void* p = nullptr;   // row 0
    uint64_t pitch = 0;        // bytes between rows (a multiple of 16)
    uint32_t rows = 0;         // k along the rows: queries (rows) of the product; across: values of k
    uint32_t width = 0;        // bytes of a row that may be read (whole dwords)
    // read instead when *choose is not zero: a copy with rows of other_pitch bytes
    const void* other = nullptr;
    uint64_t other_pitch = 0;
    const uint32_t* choose = nullptr;
};

struct Args {
    Operand q, x;
    uint32_t kstages = 0;  // stages of k
    uint32_t tail = 0;     // bytes of k in the last stage (0: all of it); x along the rows only
    uint32_t nq = 0, nr = 0;  // blocks of the shape's queries and rows
    uint32_t parts = 1;  // walk: workgroups per query block; tiles: shares of the k-stages
};

// The order of a launch's tiles.  WALK: item i is (query block, part); a workgroup stays with its
// query block and takes row blocks part, part + parts, ... (running row statistics stay in
// registers).  The query blocks of one part are 8 apart in the grid, so they run on one XCD and
// share the part's rows in its L2.  Otherwise an item is one tile of one share of k; every XCD
// takes a contiguous range of the tiles, the operand with fewer blocks varying fastest.
template <bool WALK>
struct Tiles {
    uint32_t item, qb, rb, part;
    bool ok;
    __device__ void decode(const Args& a) {
        if constexpr (WALK) {
            const uint32_t total = a.nq * a.parts;
            ok = item < total;
            if (!ok) return;
            if (a.parts % kXcds == 0) {
                const uint32_t xcd = item % kXcds, seq = item / kXcds;
                qb = seq % a.nq;
                part = (seq / a.nq) * kXcds + xcd;
            } else {
                qb = item / a.parts;
                part = item % a.parts;
            }
            rb = part;
        } else {
            const uint32_t total = a.nq * a.nr * a.parts, per = (total + kXcds - 1) / kXcds;
            for (;; item += gridDim.x) {
                const uint32_t xcd = item % kXcds, seq = item / kXcds;
                ok = seq < per;
                if (!ok) return;
                const uint32_t t = xcd * per + seq;
                if (t >= total) continue;
                const uint32_t tile = t % (a.nq * a.nr);
                part = t / (a.nq * a.nr);
                if (a.nq < a.nr) {
                    qb = tile % a.nq;
                    rb = tile / a.nq;
                } else {
                    rb = tile % a.nr;
                    qb = tile / a.nr;
                }
                return;
            }
        }
    }
    __device__ void first(const Args& a) {
        item = blockIdx.x;
        decode(a);
    }
    // whether the next tile belongs to another item
    __device__ bool next(const Args& a) {
        if constexpr (WALK) {
            rb += a.parts;
            if (rb < a.nr) return false;
        }
        item += gridDim.x;
        decode(a);
        return true;
    }
};

// Eight fp32 values of a fragment as three bf16 ones each, v = o[0] + o[1] + o[2] exactly: the upper 8 binary digits cut off
// (a rounding could overflow), the next 8 rounded, the rest.
__device__ __forceinline__ void split3(const u32x4 (&v)[2], u32x4 (&o)[3]) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const auto as_f = [](uint32_t b) { return __builtin_bit_cast(float, b); };
    const auto pack = [](float a, float b) { return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2)); };
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t a = v[i >> 1][2 * i & 3], b = v[i >> 1][(2 * i + 1) & 3];
        o[0][i] = __builtin_amdgcn_perm(b, a, 0x07060302u);
        const float ra = as_f(a) - as_f(a & 0xFFFF0000u), rb = as_f(b) - as_f(b & 0xFFFF0000u);
        const uint32_t mid = pack(ra, rb);
        o[1][i] = mid;
        o[2][i] = pack(ra - as_f(mid << 16), rb - as_f(mid & 0xFFFF0000u));
    }
}

template <int KIND>
__device__ __forceinline__ f32x16 mfma(u32x4 x, u32x4 q, f32x16 c) {
    if constexpr (KIND == F32) {
        // (both operands' fragments hold the same four k of each half)
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(__builtin_bit_cast(f32x4, x)[e], __builtin_bit_cast(f32x4, q)[e], c, 0, 0, 0);
        return c;
    } else if constexpr (KIND == BF16 || KIND == SPLIT) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, q), c, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, x), __builtin_bit_cast(f16x8, q), c, 0, 0, 0);
    }
}

// The lane's place in a tile: acc[m][n][4 j + e] is query q(n) against row r(m, j) + e.
template <int NB>
struct Lane {
    int wq, wr, l32, hh;
    __device__ int q(int n) const { return wq * 32 * NB + 32 * n + l32; }
    __device__ int r(int m, int j) const { return wr * 64 + 32 * m + 8 * j + 4 * hh; }
};

// One operand's way into LDS and out of it: W waves of 32 N queries (rows) along it, of WAVES in the workgroup.
// KM: stored across k (N = 2).
template <bool KM, int KIND, int W, int WAVES, int N = 2>
struct Feed {
    static_assert((N == 2 && KIND != PLANES) || !KM, "narrow waves and planes only along k");
    static constexpr int ES = KIND >= F32 ? 4 : 2, KV = stage_of(KIND);  // bytes of a value in LDS
    static constexpr int LPW = 4 * N * W / WAVES;   // 1 KiB direct loads per wave and stage
    static constexpr int KROW = 64 * ES * W;        // bytes of a k-row, the columns of a tile (KM)
    // the place of a k-row's 16-byte chunk c: 16-bit values, its segment (four chunks) xored by k; fp32, its half
    // of 256 bytes by bit 2 of k (the two k-rows that a fragment reads at once are four apart)
    static __device__ uint32_t placed(uint32_t k, uint32_t c) {
        if constexpr (ES == 4) return c ^ ((k & 4u) << 1);
        else return W == 1 ? c ^ ((k << 1) & 4u) : c ^ ((k & 3u) << 2);
    }
    const char* p;
    const char* base;  // of the tile
    uint32_t records;  // bytes behind it (k along the rows)
    uint64_t left;     // (KM)
    uint32_t pitch;
    uint32_t voff[LPW];
    uint32_t lds_at;   // of the wave's first load, within a stage
    uint32_t frag[KM ? 2 : 1];  // fragment addresses within a stage
    int swz, hh;

    // Direct loads: wave w fills the 1 KiB groups g = w + WAVES i.  k along the rows: rows 8 g .. 8 g + 7, lane
    // L row 8 g + L / 8, physical chunk L % 8 = logical chunk (L % 8) ^ ((row >> 1) & 7).  Across: whole k-rows,
    // each lane one 16-byte chunk, the chunk's segment (four chunks) xored.  Rows past the operand's last one
    // lie past its descriptor and land as zeros.
    __device__ void init(const Operand& o, int wave, int lane, uint32_t at, int wtile) {
        const uint32_t* choose = o.choose;
        const void *one = o.p, *two = o.other;
        const uint64_t pitch1 = o.pitch, pitch2 = o.other_pitch;
        const bool copy = choose && *choose;
        p = static_cast<const char*>(copy ? two : one);
        pitch = uint32_t(copy ? pitch2 : pitch1);
        lds_at = at + uint32_t(wave) * 1024u;
        const int l32 = lane & 31;
        hh = lane >> 5;
        if constexpr (KM) {
#pragma unroll
            for (int i = 0; i < LPW; ++i) {
                const uint32_t byte = uint32_t(1024 * (wave + WAVES * i) + 16 * lane);
                const uint32_t k = byte / KROW, c = byte % KROW / 16;
                const uint32_t at_c = placed(k, c);
                voff[i] = k * pitch + 16u * at_c;
            }
            const int e = (lane & 15) >> 2;
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                if constexpr (ES == 4)  // column l32 of block n, k-row 4 hh (+ 8 t + e)
                    frag[n] = at + uint32_t(4 * hh * KROW) + 16u * placed(4u * uint32_t(hh), uint32_t(8 * (2 * wtile + n) + (l32 >> 2))) + 4u * uint32_t(l32 & 3);
                else  // k-row 8 hh + e, 4 columns of the half block (lane >> 4) & 1
                    frag[n] = at + uint32_t((8 * hh + e) * KROW) +
                              16u * placed(uint32_t(e), uint32_t(4 * (2 * wtile + n) + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1))) + 8u * uint32_t(lane & 1);
            }
        } else {
#pragma unroll
            for (int i = 0; i < LPW; ++i) {
                const uint32_t row = uint32_t(8 * (wave + WAVES * i) + (lane >> 3));
                voff[i] = row * pitch + 16u * uint32_t((lane & 7) ^ ((row >> 1) & 7));
            }
            frag[0] = at + uint32_t((wtile * 32 * N + l32) * ROWB);
            swz = (l32 >> 1) & 7;
        }
    }
    // the operand's block b of 32 N W queries (rows)
    __device__ void open(const Operand& o, uint32_t b) {
        if constexpr (KM) {
            base = p + uint64_t(b) * uint32_t(KROW);
            left = uint64_t(o.rows - 1) * pitch + o.width - uint64_t(b) * uint32_t(KROW);
        } else {
            base = p + uint64_t(b) * (32u * N * W) * pitch;
            records = (min(32u * N * W, o.rows - b * (32u * N * W)) - 1u) * pitch + o.width;
        }
    }
    // load i of stage k into the slot at LDS address `slot`; !ok: zeros
    __device__ void issue(uint32_t k, bool ok, uint32_t slot, int i) const {
        if constexpr (KM) {
            const uint64_t skip = uint64_t(k) * KV * pitch;
            const dma_rsrc r = make_dma_rsrc(base + skip, ok && skip < left ? uint32_t(min(left - skip, uint64_t(kDmaMaxBytes))) : 0u);
            lds_dma16(r, voff[i], slot + lds_at + uint32_t(1024 * WAVES * i));
        } else {
            const dma_rsrc r = make_dma_rsrc(base, records);
            lds_dma16_so(r, ok ? voff[i] : kDmaSkip, ok ? k * uint32_t(ROWB) : 0u, slot + lds_at + uint32_t(1024 * WAVES * i));
        }
    }
    // the fragment of the wave's 32-query (row) block n, k-step t of the slot (32 bytes of k: this lane's half)
    __device__ u32x4 read(const char* slot, int n, int t) const {
        if constexpr (KM && ES == 4) {
            const char* at = slot + frag[n] + t * 8 * KROW;
            u32x4 o;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = *reinterpret_cast<const uint32_t*>(at + e * KROW);
            return o;
        } else if constexpr (KM) {
            typedef short s16x4 __attribute__((ext_vector_type(4)));
            typedef __attribute__((address_space(3))) s16x4* lds_s16x4;
            struct alignas(16) {
                s16x4 v[2];
            } o;
            const uint32_t at = lds_addr_of(slot) + frag[n] + uint32_t(t * 16 * KROW);
            o.v[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_s16x4>(at));
            o.v[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_s16x4>(at + 4 * KROW));
            return __builtin_bit_cast(u32x4, o);
        } else {
            return *reinterpret_cast<const u32x4*>(slot + frag[0] + n * 32 * ROWB + 16 * ((2 * t + hh) ^ swz));
        }
    }
    // clears what a fragment of k-step t holds from byte `tail` of the stage on
    __device__ u32x4 cut(u32x4 v, int t, uint32_t tail) const {
        int have = int(tail) - 16 * (2 * t + hh);
        asm volatile("" : "+v"(have));  // computed here: kept through the main loop, the masks would spill its registers
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int b = have - 4 * e;
            v[e] &= b >= 4 ? ~0u : b == 2 ? 0xFFFFu : 0u;
        }
        return v;
    }
};

// Epi: struct with
//   Shape, static constexpr bool kWalk, kStores
//   struct State (per thread, lives through the main loop)
//   begin(State&, smem, tile)   a new item's first tile (barriers follow before the epilogue)
//   load(State&, tile, tid)     before the main loop: starts what the tile's epilogue reads
//   publish(State&, smem, tid)  after the main loop, before the barrier
//   tile(State&, smem, lane, acc, tile, spare, settle)  spare: 4 KiB of LDS of the wave's own; with kStores,
//                               settle() before the first store to memory
//   end(State&, smem, lane, tile, mine)  after an item's last tile; mine: the wave's state has the item's tiles
// With several slices, tile() runs in the first one's waves alone.
template <int KIND, bool QK, bool XK, class Epi>
__global__ __launch_bounds__(Epi::Shape::THREADS, Epi::Shape::PER_SIMD) void gemm16_kernel(Args a, Epi epi) {
    using Sh = typename Epi::Shape;
    constexpr int STAGE = Sh::STAGE;
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    __shared__ typename Epi::Shared smem;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int slice = wave / Sh::WPS, ws = wave % Sh::WPS;  // (uniform)
    const Lane<Sh::NB> ln{ws % Sh::WQ, ws / Sh::WQ, lane & 31, lane >> 5};
    constexpr int NB = Sh::NB;

    Tiles<Epi::kWalk> tile;
    tile.first(a);
    if (!tile.ok) return;

    const uint32_t total_stages = a.kstages;
    char* const mine = lds + slice * (Sh::SLOTS * STAGE);  // the slice's slots
    const uint32_t lds0 = lds_addr_of(mine);
    Feed<QK, KIND, Sh::WQ, Sh::WPS, Sh::NB> fq_;
    Feed<XK, KIND, Sh::WR, Sh::WPS> fx_;
    fq_.init(a.q, ws, lane, 0, ln.wq);
    fx_.init(a.x, ws, lane, Sh::QB, ln.wr);
    uint32_t s0, s1, ns;  // the slice's stages of the tile, and how many each slice takes
    auto open = [&]() {
        fq_.open(a.q, tile.qb);
        fx_.open(a.x, tile.rb);
        if constexpr (Epi::kWalk) {
            s0 = 0;
            s1 = total_stages;
        } else {
            s0 = uint32_t(uint64_t(total_stages) * tile.part / a.parts);
            s1 = uint32_t(uint64_t(total_stages) * (tile.part + 1) / a.parts);
        }
        ns = s1 - s0;
        if constexpr (Sh::SLICES > 1) {
            // even shares: all of a slice's ns stages but one at most are the tile's (past its share: zeros), so k ends within
            // the last two, where the loop below looks for it
            const uint32_t n = ns, from = s0;
            ns = (n + Sh::SLICES - 1) / Sh::SLICES;
            s0 = from + n * uint32_t(slice) / Sh::SLICES;
            s1 = from + n * uint32_t(slice + 1) / Sh::SLICES;
        }
    };
    // load i of the tile's stage s into slot `slot` (past the last stage: zeros)
    constexpr int LQ = decltype(fq_)::LPW, LX = decltype(fx_)::LPW;
    auto issue_one = [&](uint32_t s, uint32_t slot, int i) {
        const bool ok = s < s1;
        const uint32_t sb = lds0 + slot * uint32_t(STAGE);
        if (i < LQ) fq_.issue(s, ok, sb, i);
        else fx_.issue(s, ok, sb, i - LQ);
    };
    auto issue = [&](uint32_t s, uint32_t slot) {
#pragma unroll
        for (int i = 0; i < LQ + LX; ++i) issue_one(s, slot, i);
    };

    f32x16 acc[2][NB];
    constexpr int BUFS = KIND == PLANES ? 3 : 2;  // (SPLIT: the two halves of a k-step)
    u32x4 fx[BUFS][2], fq[BUFS][NB];
    auto read_one = [&](int buf, uint32_t slot, int t, int i) {
        const char* base = mine + slot * STAGE;
        if (i < 2) fx[buf][i] = fx_.read(base, i, t);
        else fq[buf][i - 2] = fq_.read(base, i - 2, t);
    };
    // One k-step: four MFMAs (NB = 1: two), and behind each of them, in this order, the read of one of the next k-step's
    // fragments and a share of the loads into the slot that this stage leaves.
    auto step = [&](int cur, uint32_t slot_next, int t_next, auto more, uint32_t s_load, uint32_t slot_load, bool ends) {
        if constexpr (!XK && !decltype(more)::value) {
            if (ends) {
                const int t = (t_next + 3) & 3;
#pragma unroll
                for (int m = 0; m < 2; ++m) fx[cur][m] = fx_.cut(fx[cur][m], t, a.tail);
            }
        }
#pragma unroll
        for (int i = 0; i < 2 * NB; ++i) {
            const int m = i & 1, n = i >> 1;
            acc[m][n] = mfma<KIND>(fx[cur][m], fq[cur][n], acc[m][n]);
            __builtin_amdgcn_sched_barrier(0);
            if (NB == 2) {
                read_one(cur ^ 1, slot_next, t_next, (i & 1) * 2 + (i >> 1));
            } else {
                read_one(cur ^ 1, slot_next, t_next, i);
                if (i) read_one(cur ^ 1, slot_next, t_next, 2);
            }
            if constexpr (decltype(more)::value) {
#pragma unroll
                for (int l = i * (LQ + LX) / (2 * NB); l < (i + 1) * (LQ + LX) / (2 * NB); ++l) issue_one(s_load, slot_load, l);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // The same of planes.  T even: hi hi, and the reads of the lo fragments (buffer 1); odd: lo hi and hi lo, and the reads
    // of the next hi ones (buffers 0 and 2 in turn).
    auto step_planes = [&](auto t, uint32_t slot_next, auto more, uint32_t s_load, uint32_t slot_load) {
        constexpr int T = decltype(t)::value, HI = T < 2 ? 0 : 2, NEXT = T & 1 ? 2 - HI : 1, N = T & 1 ? 4 * NB : 2 * NB;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int m = i & 1, n = (i >> 1) % NB;
            const bool second = i >= 2 * NB;
            acc[m][n] = mfma<KIND>(fx[T & 1 && !second ? 1 : HI][m], fq[second ? 1 : HI][n], acc[m][n]);
            __builtin_amdgcn_sched_barrier(0);
            if (i < 2 + NB) {
                if (NB == 4) {
                    read_one(NEXT, slot_next, (T + 1) & 3, i);
                } else if (NB == 2) {
                    read_one(NEXT, slot_next, (T + 1) & 3, (i & 1) * 2 + (i >> 1));
                } else if (i < 2) {
                    read_one(NEXT, slot_next, (T + 1) & 3, i);
                    if (i) read_one(NEXT, slot_next, (T + 1) & 3, 2);
                }
            }
            if constexpr (decltype(more)::value) {
#pragma unroll
                for (int l = i * (LQ + LX) / N; l < (i + 1) * (LQ + LX) / N; ++l) issue_one(s_load, slot_load, l);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // The same of fp32 values split into three bf16 ones: k-steps of 16 values, two fragments as they lie in LDS (any 16
    // values of k will do, as long as both operands' are the same).  Six of the nine products: the others are below
    // 2^-21 of the value, 2^-25 as a rule.  The fragments are split first, then the next ones read into their place.
    auto step_split = [&](uint32_t slot_next, int t_next, auto more, uint32_t s_load, uint32_t slot_load) {
        static_assert(KIND != SPLIT || XK, "k does not end within a stage");
        u32x4 px[2][3], pq[NB][3];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            const u32x4 v[2] = {fx[0][m], fx[1][m]};
            split3(v, px[m]);
        }
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            const u32x4 v[2] = {fq[0][n], fq[1][n]};
            split3(v, pq[n]);
        }
#pragma unroll
        for (int i = 0; i < 2 * (2 + NB); ++i) read_one(i / (2 + NB), slot_next, t_next + i / (2 + NB), i % (2 + NB));
        constexpr int PX[6] = {2, 0, 1, 1, 0, 0}, PQ[6] = {0, 2, 1, 0, 1, 0};  // the smallest products first
#pragma unroll
        for (int p = 0; p < 6; ++p) {
#pragma unroll
            for (int i = 0; i < 2 * NB; ++i) acc[i & 1][i >> 1] = mfma<KIND>(px[i & 1][PX[p]], pq[i >> 1][PQ[p]], acc[i & 1][i >> 1]);
            if constexpr (decltype(more)::value) {
#pragma unroll
                for (int l = p * (LQ + LX) / 6; l < (p + 1) * (LQ + LX) / 6; ++l) issue_one(s_load, slot_load, l);
            }
        }
    };
    // a workgroup barrier that leaves the direct loads in flight; this wave's LDS reads are done
    auto barrier = [&]() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
    // waits for all but the youngest `stages` stages of direct loads
    constexpr int SLOTS = Sh::SLOTS, L = LQ + LX;
    static_assert((SLOTS & (SLOTS - 1)) == 0 && L * (SLOTS - 1) < 64 && SLOTS <= 4, "slots");
    auto wait_but = [&](int stages) {
        if (SLOTS > 3 && stages >= 3) wait_vmcnt<(SLOTS > 3 ? 3 : 0) * L>();
        else if (SLOTS > 2 && stages == 2) wait_vmcnt<(SLOTS > 2 ? 2 : 0) * L>();
        else if (stages == 1) wait_vmcnt<L>();
        else wait_vmcnt<0>();
    };
    // stage i of the tile's ns; more: stage i + SLOTS follows; ends: k ends within it
    auto stage = [&](uint32_t i, uint32_t ns, auto more, bool ends) {
        const uint32_t slot = i & (SLOTS - 1);
        const std::integral_constant<bool, false> none{};
        if constexpr (KIND == PLANES) {
            step_planes(std::integral_constant<int, 0>(), slot, none, 0, 0);
            step_planes(std::integral_constant<int, 1>(), slot, none, 0, 0);
            step_planes(std::integral_constant<int, 2>(), slot, none, 0, 0);
        } else if constexpr (KIND == SPLIT) {
            step_split(slot, 2, none, 0, 0);
        } else {
#pragma unroll
            for (int t = 0; t < 3; ++t) step(t & 1, slot, t + 1, none, 0, 0, ends && !decltype(more)::value);
        }
        // the last k-step's fragments are in registers: publish the next stage, free this slot
        if (decltype(more)::value) wait_but(SLOTS - 2);
        else wait_but(min(SLOTS - 2, int(ns) - 2 - int(i)));
        barrier();
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (KIND == PLANES) step_planes(std::integral_constant<int, 3>(), (slot + 1) & (SLOTS - 1), more, s0 + i + SLOTS, slot);
        else if constexpr (KIND == SPLIT) step_split((slot + 1) & (SLOTS - 1), 0, more, s0 + i + SLOTS, slot);
        else step(1, (slot + 1) & (SLOTS - 1), 0, more, s0 + i + SLOTS, slot, ends);
    };

    typename Epi::State st;
    open();
    // the first tile's stages before anything that waits for memory; later tiles' first ones during the epilogues
#pragma unroll
    for (int k = 0; k < SLOTS; ++k)
        if (k == 0 || uint32_t(k) < ns) issue(s0 + k, k);
    epi.begin(st, smem, tile);
    bool settled = false, first = true;
    for (;;) {
        epi.load(st, tile, tid);
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int v = 0; v < 16; ++v) acc[m][n][v] = 0.0f;
        const uint32_t todo = ns;
        if (!first) {
            barrier();  // every wave is past the previous tile's epilogue: the other slots are free
#pragma unroll
            for (int k = 1; k < SLOTS; ++k)
                if (uint32_t(k) < todo) issue(s0 + k, k);
        }
        first = false;
        if (!settled) {
            wait_but(min(SLOTS, int(todo)) - 1);  // stage 0 (older than the others' loads)
            barrier();
        }
#pragma unroll
        for (int i = 0; i < (KIND == SPLIT ? 2 : 1) * (2 + NB); ++i) read_one(i / (2 + NB), 0, i / (2 + NB), i % (2 + NB));
        uint32_t i = 0;
        for (; i + SLOTS < todo; ++i) stage(i, todo, std::true_type(), false);
        for (; i < todo; ++i) stage(i, todo, std::false_type(), !XK && a.tail && s0 + i + 1 == total_stages);
        epi.publish(st, smem, tid);
        __syncthreads();  // every wave is past the main loop: slot 0 is free
        if constexpr (Sh::SLICES > 1) {
            // the slices' sums join in the first one's registers
            char* const at = mine + STAGE + ws * (NB * 8192) + lane * 16;
            if (slice) {
#pragma unroll
                for (int c = 0; c < 8 * NB; ++c) {
                    f32x4 v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = acc[c & 1][c / 8][4 * ((c >> 1) & 3) + e];
                    *reinterpret_cast<f32x4*>(at + 1024 * c) = v;
                }
            }
            __syncthreads();
            if (!slice) {
#pragma unroll
                for (int p = 1; p < Sh::SLICES; ++p)
#pragma unroll
                    for (int c = 0; c < 8 * NB; ++c) {
                        const f32x4 v = *reinterpret_cast<const f32x4*>(at + p * (Sh::SLOTS * STAGE) + 1024 * c);
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[c & 1][c / 8][4 * ((c >> 1) & 3) + e] += v[e];
                    }
            }
        }
        const Tiles<Epi::kWalk> here = tile;
        const bool last = tile.next(a);
        if (tile.ok) {
            open();
            issue(s0, 0);
        }
        // what the epilogue computes from the lane is computed there: kept through the main loop, its
        // addresses would take the registers that the fragments need
        Lane<Sh::NB> le = ln;
        asm volatile("" : "+v"(le.l32), "+v"(le.hh));
        // An epilogue that stores much waits for the next tile's first stage before its first store: behind the
        // stores, that wait would be for all of them.
        settled = Epi::kStores;
        if (Sh::SLICES == 1 || !slice) epi.tile(st, smem, le, acc, here, lds + STAGE + ws * 4096, [] { wait_vmcnt<0>(); });
        else if (Epi::kStores) wait_vmcnt<0>();
        if (last) {
            epi.end(st, smem, ln, here, Sh::SLICES == 1 || !slice);
            if (!tile.ok) break;
            epi.begin(st, smem, tile);
        }
    }
    wait_vmcnt<0>();
}

// Workgroups of a shape that a CU holds: its LDS (with up to 2 KiB of the epilogue's beside two slots; the
// largest shape is alone anyway), its registers, its 32 waves.
template <class Sh>
constexpr uint32_t per_cu() {
    constexpr uint32_t lds = 163840 / (Sh::LDS + 2048), waves = std::max(4 * Sh::PER_SIMD / Sh::WAVES, 1);
    return Sh::SLOTS > 2 ? 1u : std::max(std::min(lds, waves), 1u);
}
// Persistent launch: as many workgroups as the chip holds, a multiple of the XCDs.
template <class Sh>
uint32_t grid_max(const va_context* ctx) {
    return std::max(uint32_t(ctx->num_cus), kXcds) / kXcds * kXcds * per_cu<Sh>();
}
template <int KIND, bool QK, bool XK, class Epi>
va_status launch(va_context* ctx, const Args& a, const Epi& epi) {
    using Sh = typename Epi::Shape;
    static_assert(sizeof(typename Epi::Shared) + Sh::LDS <= 163840, "a workgroup's LDS");
    const uint64_t tiles = uint64_t(a.nq) * (Epi::kWalk ? a.parts : a.nr * uint64_t(a.parts));
    if (tiles == 0) return VA_OK;
    const uint64_t pitch = std::max(std::max(a.q.pitch, a.x.pitch), std::max(a.q.other_pitch, a.x.other_pitch));
    if (tiles > 0x7FFFFFF0ull || 256 * pitch > kDmaMaxBytes)
        return fail(ctx, VA_ERR_INVALID_ARG, "matrix product too large: %llu tiles, rows of %llu bytes", (unsigned long long)tiles,
                    (unsigned long long)pitch);
    const uint64_t grid = std::min<uint64_t>((tiles + kXcds - 1) / kXcds * kXcds, grid_max<Sh>(ctx));
    auto kern = &gemm16_kernel<KIND, QK, XK, Epi>;
    // the kernel may take its dynamic LDS: asked once per device
    static std::atomic<uint64_t> allowed{0};
    const uint64_t bit = ctx->device < 64 ? 1ull << ctx->device : 0;
    if (!(allowed.load(std::memory_order_relaxed) & bit)) {
        VA_CHECK_HIP(ctx, hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, Sh::LDS));
        allowed.fetch_or(bit, std::memory_order_relaxed);
    }
    kern<<<dim3(uint32_t(grid)), dim3(Sh::THREADS), Sh::LDS, ctx->stream>>>(a, epi);
    VA_CHECK_LAUNCH(ctx);
    return VA_OK;
}

}  // namespace g16
}  // namespace va
