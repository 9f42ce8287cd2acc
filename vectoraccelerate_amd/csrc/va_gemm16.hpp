// va_gemm16.hpp — the matrix product of two row-major 16-bit operands over their common (row)
// dimension, with the epilogue a template argument: every product of the softmax cross entropy
// (va_xent.hip) is one of these.
//
//   acc[q][r] = sum_k Q[q][k] X[r][k]        Q: [queries x pitch], X: [rows x pitch], fp16 or bf16
//
// One workgroup computes tiles of 256 queries x 256 rows with sixteen waves of 64 x 64 (2 x 2
// blocks of v_mfma_f32_32x32x16, 64 fp32 accumulators a lane, four waves per SIMD).  64 k-values
// of both operands move global -> LDS by direct loads into one of two 64 KiB slots while the
// other is computed on; LDS rows are 128 bytes with their 16-byte chunks swizzled by the row, so
// fragment reads are conflict-free.  The launch is persistent: a workgroup walks its tiles, and the
// next tile's first stage streams in during the epilogue.
//
// Operands of fp32 values come as two fp16 planes (value = (hi + lo) 2^-e with one exponent a row
// or tensor): a product is then hi hi + hi lo + lo hi, three passes over k with the same
// accumulators.  lo lo is below 2^-22 of the product and is left out; what remains is exact to
// about 2^-22 a term, the same as an fp32 fma chain of a few terms.
#pragma once

#include "va_internal.hpp"

namespace va {
namespace g16 {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int TQ = 256, TR = 256, KC = 64, WAVES = 16;
constexpr int ROWB = KC * 2;                 // bytes of an LDS row
constexpr int OPB = TQ * ROWB;               // bytes of one operand's stage
constexpr int STAGE = 2 * OPB;
constexpr int LDS_BYTES = 2 * STAGE;
constexpr int LPW = OPB / 1024 / WAVES;      // 1 KiB direct loads per wave, operand and stage

struct Operand {
    const void* p = nullptr;  // row 0
    uint64_t pitch = 0;       // bytes between rows (a multiple of 16)
    uint32_t rows = 0;
    uint32_t plane = 0;       // bytes from a row's hi plane to its lo plane (PLANES only)
};

struct Args {
    Operand q, x;
    uint32_t kstages = 0;  // stages of 64 k-values of one plane (rows are zero-padded to them)
    uint32_t nq = 0, nr = 0;  // blocks of 256
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

template <bool BF16>
__device__ __forceinline__ f32x16 mfma(u32x4 x, u32x4 q, f32x16 c) {
    if constexpr (BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, q), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, x), __builtin_bit_cast(f16x8, q), c, 0, 0, 0);
}

// The lane's place in a tile: acc[m][n][4 j + e] is query q(n) against row r(m, j) + e.
struct Lane {
    int wq, wr, l32, hh;
    __device__ int q(int n) const { return wq * 64 + 32 * n + l32; }
    __device__ int r(int m, int j) const { return wr * 64 + 32 * m + 8 * j + 4 * hh; }
};

// Epi: struct with
//   static constexpr bool kWalk
//   struct State (per thread, lives through the main loop)
//   begin(State&, smem, tile)   a new item's first tile (barriers follow before the epilogue)
//   load(State&, tile, tid)     before the main loop: starts what the tile's epilogue reads
//   publish(State&, smem, tid)  after the main loop, before the barrier
//   tile(State&, smem, lane, acc, tile, spare)  spare: 4 KiB of LDS of the wave's own
//   end(State&, smem, lane, tile)  after an item's last tile
template <bool BF16, bool PLANES, class Epi>
__global__ __launch_bounds__(64 * WAVES, 4) void gemm16_kernel(Args a, Epi epi) {
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    __shared__ typename Epi::Shared smem;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Lane ln{wave & 3, wave >> 2, lane & 31, lane >> 5};

    Tiles<Epi::kWalk> tile;
    tile.first(a);
    if (!tile.ok) return;

    // Direct loads: wave w fills the 1 KiB groups g = w + 16 i (rows 8 g .. 8 g + 7) of each operand;
    // lane L loads row 8 g + L / 8, physical chunk L % 8 = logical chunk (L % 8) ^ ((row >> 1) & 7).
    // Rows past the operand's last one lie past its descriptor and land as zeros.
    const uint32_t qpitch = uint32_t(a.q.pitch), xpitch = uint32_t(a.x.pitch);
    const uint32_t row0 = uint32_t(8 * wave + (lane >> 3));
    const uint32_t ch = 16u * uint32_t((lane & 7) ^ ((row0 >> 1) & 7));  // 8 * 16 rows on: the same swizzle
    const uint32_t total_stages = PLANES ? 3 * a.kstages : a.kstages;
    const uint32_t kbytes = a.kstages * uint32_t(ROWB);
    const uint32_t lds0 = lds_addr_of(lds);
    dma_rsrc qres, xres;
    uint32_t s0, s1;  // the tile's stages
    auto open = [&]() {
        const uint32_t q0 = tile.qb * TQ, r0 = tile.rb * TR;
        qres = make_dma_rsrc(static_cast<const char*>(a.q.p) + q0 * a.q.pitch,
                             (min(uint32_t(TQ), a.q.rows - q0) - 1u) * qpitch + kbytes + (PLANES ? a.q.plane : 0u));
        xres = make_dma_rsrc(static_cast<const char*>(a.x.p) + r0 * a.x.pitch,
                             (min(uint32_t(TR), a.x.rows - r0) - 1u) * xpitch + kbytes + (PLANES ? a.x.plane : 0u));
        if constexpr (Epi::kWalk) {
            s0 = 0;
            s1 = total_stages;
        } else {
            s0 = uint32_t(uint64_t(total_stages) * tile.part / a.parts);
            s1 = uint32_t(uint64_t(total_stages) * (tile.part + 1) / a.parts);
        }
    };
    // stage s of the tile into slot `slot` (past the last stage: zeros)
    auto issue = [&](uint32_t s, uint32_t slot) {
        const bool ok = s < s1;
        uint32_t qo, xo;
        if constexpr (PLANES) {
            const uint32_t seg = s / a.kstages, k = (s - seg * a.kstages) * uint32_t(ROWB);
            qo = k + (seg == 2 ? a.q.plane : 0u);
            xo = k + (seg == 1 ? a.x.plane : 0u);
        } else {
            qo = xo = s * uint32_t(ROWB);
        }
        const uint32_t sb = lds0 + slot * uint32_t(STAGE) + uint32_t(wave) * 1024u;
#pragma unroll
        for (int i = 0; i < LPW; ++i) {
            const uint32_t row = row0 + uint32_t(8 * WAVES * i), at = sb + uint32_t(1024 * WAVES * i);
            lds_dma16_so(qres, ok ? row * qpitch + ch : kDmaSkip, ok ? qo : 0u, at);
            lds_dma16_so(xres, ok ? row * xpitch + ch : kDmaSkip, ok ? xo : 0u, at + uint32_t(OPB));
        }
    };

    const int swz = (ln.l32 >> 1) & 7;
    const uint32_t q_at = uint32_t((ln.wq * 64 + ln.l32) * ROWB), x_at = uint32_t(OPB + (ln.wr * 64 + ln.l32) * ROWB);
    f32x16 acc[2][2];
    u32x4 fx[2][2], fq[2][2];
    auto read_frags = [&](int buf, uint32_t slot, int t) {
        const char* base = lds + slot * STAGE;
        const uint32_t ko = 16u * uint32_t((2 * t + ln.hh) ^ swz);
#pragma unroll
        for (int m = 0; m < 2; ++m) fx[buf][m] = *reinterpret_cast<const u32x4*>(base + x_at + m * 32 * ROWB + ko);
#pragma unroll
        for (int n = 0; n < 2; ++n) fq[buf][n] = *reinterpret_cast<const u32x4*>(base + q_at + n * 32 * ROWB + ko);
    };
    auto mma = [&](int buf) {
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int n = 0; n < 2; ++n) acc[m][n] = mfma<BF16>(fx[buf][m], fq[buf][n], acc[m][n]);
        // the next k-step's four fragment reads go between the four MFMAs
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
    };
    // a workgroup barrier that leaves the direct loads in flight; this wave's LDS reads are done
    auto barrier = [&]() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };

    typename Epi::State st;
    open();
    epi.begin(st, smem, tile);
    issue(s0, 0);  // later tiles: during the previous epilogue
    for (;;) {
        epi.load(st, tile, tid);
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int v = 0; v < 16; ++v) acc[m][n][v] = 0.0f;
        barrier();  // every wave is past the previous tile's main loop: slot 1 is free
        issue(s0 + 1, 1);
        wait_vmcnt<2 * LPW>();  // stage 0 (older than stage 1's loads)
        barrier();
        read_frags(0, 0, 0);
        const uint32_t ns = s1 - s0;
        for (uint32_t s = 0; s < ns; ++s) {
            const uint32_t slot = s & 1u;
#pragma unroll
            for (int t = 0; t < KC / 16; ++t) {
                const int cur = t & 1;
                if (t == KC / 16 - 1) {
                    // this k-step's fragments are in registers: publish the next stage, free this slot
                    wait_vmcnt<0>();
                    barrier();
                    if (s + 2 < ns) issue(s0 + s + 2, slot);
                    read_frags(cur ^ 1, slot ^ 1u, 0);
                } else {
                    read_frags(cur ^ 1, slot, t + 1);
                }
                mma(cur);
            }
        }
        epi.publish(st, smem, tid);
        __syncthreads();  // every wave is past the main loop: slot 0 is free
        const Tiles<Epi::kWalk> here = tile;
        const bool last = tile.next(a);
        if (tile.ok) {
            open();
            issue(s0, 0);
        }
        // what the epilogue computes from the lane is computed there: kept through the main loop, its
        // addresses would take the registers that the fragments need
        Lane le = ln;
        asm volatile("" : "+v"(le.l32), "+v"(le.hh));
        epi.tile(st, smem, le, acc, here, lds + STAGE + wave * 4096);
        if (last) {
            epi.end(st, smem, ln, here);
            if (!tile.ok) break;
            epi.begin(st, smem, tile);
        }
    }
    wait_vmcnt<0>();
}

// Persistent launch: one workgroup per CU (the LDS of a tile fills one), a multiple of the XCDs.
template <bool BF16, bool PLANES, class Epi>
va_status launch(va_context* ctx, const Args& a, const Epi& epi) {
    const uint64_t tiles = uint64_t(a.nq) * (Epi::kWalk ? a.parts : a.nr * uint64_t(a.parts));
    if (tiles == 0) return VA_OK;
    if (tiles > 0x7FFFFFF0ull || 256 * std::max(a.q.pitch, a.x.pitch) > kDmaMaxBytes)
        return fail(ctx, VA_ERR_INVALID_ARG, "matrix product too large: %llu tiles, rows of %llu and %llu bytes",
                    (unsigned long long)tiles, (unsigned long long)a.q.pitch, (unsigned long long)a.x.pitch);
    const uint64_t cus = std::max<uint64_t>(uint64_t(ctx->num_cus), kXcds) / kXcds * kXcds;
    const uint64_t grid = std::min((tiles + kXcds - 1) / kXcds * kXcds, cus);
    auto kern = &gemm16_kernel<BF16, PLANES, Epi>;
    VA_CHECK_HIP(ctx, hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, LDS_BYTES));
    kern<<<dim3(uint32_t(grid)), dim3(64 * WAVES), LDS_BYTES, ctx->stream>>>(a, epi);
    VA_CHECK_LAUNCH(ctx);
    return VA_OK;
}

}  // namespace g16
}  // namespace va
