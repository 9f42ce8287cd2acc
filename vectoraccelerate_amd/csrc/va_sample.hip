// va_sample.hip — an item for each row of logits, by temperature, top-k, top-p and min-p, from a given random number.
//
// With x_j the logits of a row, M their largest and T the temperature, item j weighs w_j = exp((x_j - M) / T).  Ordered by
// (x descending, j ascending) every truncation keeps a prefix:
//   top-k  the first k;        top-p  the fewest whose weights reach p of those that top-k keeps;        min-p  w_j >= m
// and the drawn item is the first, in the order of the items or in that of the truncations, at which the kept weights added up exceed u
// times their sum.  NaN and -inf are no items.
//
// Weights and their sums are fp64 throughout: an item next to a border has to fall on its side of it, and fp32's weights of
// 100,000 items would move one draw in a hundred.  A weight is off by 4e-14 of itself (exp2_of), and listed ones go to chunks in steps of
// 2^-50 of the largest: both are far below the distance of a border from a u of 24 digits.  A weight below 2^-1000 of the largest may be
// zero.  A sum's order is fixed, so results repeat bit for bit (a row's passes divided among workgroups and in one add up in other
// orders, and may part at a border by such a difference).
//
// Two passes over a row.  What weights refer to is the largest of a sample, so the first pass needs no other before it: it counts
// the items in 2048 bins of equal width, adds up all weights where top-p asks for the sum, and lists the few items
// above the sample's largest.  From the counts follow the bins that hold the cut.  The second pass lists their items, some dozens
// to some thousands, and adds up the weights above them by chunks of the row.  The list sorted gives the cut to the item, the
// chunks' sums the chunk that u falls into, and that chunk the item.  Where nothing is cut one pass gives the chunks' sums.
// Along falling logits (FALLING) the drawn item is the end of a prefix too, that whose weights exceed u times what is kept.  A list
// from the top holds it beside the cut.  Of long prefixes the list near the cut, or a pass without a list, gives what is kept, and a further
// pass, its bins chosen as before, lists the items around u times that; where nothing is cut the second pass does.
// A long row's passes are divided among workgroups, with a launch for each pass.  A row that the quick way cannot take goes through as many
// passes as it needs, by one workgroup: one with +inf, with no item in the sample, with more than 4096 items in the bins that hold the cut
// (equal logits, top-k beyond that), with more than 1024 items above the sample's largest, or, divided, with one that weighs 2^900
// times that (6.2 logits above it at a temperature of 0.01).  One row of 262,144: 51 us by the quick way at p 0.9, 2.3 ms so with a lone
// peak at a temperature of 0.01, 3.3 ms with all logits alike; along falling logits 75 us, 3.8 and 6.1 ms.
//
// Bound by the weights' fp64 instructions where there are many (2048 x 100,003 fp16, uncut: 190 us, 1.07 G weights a ms, 2.1 TB/s), by
// the chain of short steps where there are few (64 x 262,144 bf16, p 0.9: 78 us, of which clearing 5, the passes 25 and 35, the end
// 16; 1 x 10,000, top 50: 23 us in one launch).  Along falling logits 521 us, of each 1024 rows' 260 the passes 107 and 124 and the end
// 25; 60 us, as what min-p keeps is listed from the top and nothing above it weighed; 27 us.
#include <algorithm>
#include <cmath>
#include <cstddef>

#include "va_internal.hpp"

namespace va {
namespace {

struct Row {
    const void* logits;
    uint64_t stride;
    const float* uniforms;
    const float *temperatures, *top_ps, *min_ps;  // a value a row, or NULL
    const int32_t* top_ks;
    float temperature, top_p, min_p;
    uint32_t top_k;
    int64_t* items;
    float* log_probability;
    uint32_t rows, V;
};

// What a row is drawn by.  Values on the device that make no sense are taken as the nearest that does.
struct Settings {
    double c, p, m;  // weights are 2^((x - M) c)
    uint32_t k;
};
__device__ __forceinline__ Settings settings_of(const Row& a, uint32_t row) {
    Settings s;
    const float t = a.temperatures ? a.temperatures[row] : a.temperature, p = a.top_ps ? a.top_ps[row] : a.top_p, m = a.min_ps ? a.min_ps[row] : a.min_p;
    const int64_t k = a.top_ks ? int64_t(a.top_ks[row]) : int64_t(a.top_k);
    s.k = k > 0 ? uint32_t(min(k, int64_t(a.V))) : a.V;
    s.c = 1.4426950408889634;
    if (t > 0.0f) s.c /= double(t);
    else s.k = 1;  // the most likely item
    s.p = p > 0.0f ? double(p) : 0.0;
    if (!(p < 1.0f)) s.p = 1.0;
    s.m = m > 0.0f ? fmin(double(m), 1.0) : 0.0;
    return s;
}

// Along falling logits u is kept below 1, so that no rounding of what is kept takes the draw past its last item.
__device__ __forceinline__ double inner(float u) { return fmin(fmax(double(u), 0.0), 0x1.fffffep-1); }

// Larger logits have larger keys; 0: no item.
constexpr uint32_t kLowest = 0x00800000u;  // the key of the lowest finite value
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);  // (-0 is 0)
    const uint32_t k = b & 0x80000000u ? ~b : b | 0x80000000u;
    return x > -__builtin_inff() ? k : 0u;
}
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }

// 2^t, below 2^-1000 zero: the order as it is, and 1 + r q(r) for what is left of it, |r| <= 1/2, q through Chebyshev's points: off by 4e-14
__device__ __forceinline__ double exp2_of(double t) {
    const double shifted = t + 0x1.8p52, n = shifted - 0x1.8p52, r = t - n;
    double s = 1.0203115783547221e-07;
    s = fma(s, r, 1.325522487893318e-06);
    s = fma(s, r, 1.5252686876099085e-05);
    s = fma(s, r, 0.00015403455852451632);
    s = fma(s, r, 0.0013333558178986894);
    s = fma(s, r, 0.009618129159402562);
    s = fma(s, r, 0.05550410866476082);
    s = fma(s, r, 0.2402265069581299);
    s = fma(s, r, 0.6931471805599453);
    s = fma(s, r, 1.0);
    s = __hiloint2double(__double2hiint(s) + (__double2loint(shifted) << 20), __double2loint(s));
    return t >= -1000.0 ? s : 0.0;  // (false for what NaN gives)
}
__device__ __forceinline__ double weight(float x, double top, double c) { return double(x) == top ? 1.0 : exp2_of((double(x) - top) * c); }  // (x or top may be infinite)

// The logarithm of a weight's share, also of one whose quotient fp64 does not hold (u = 0 may draw it).
__device__ __forceinline__ float log_share(double w, double total) {
    const double r = w / total;
    return float(r >= 0x1p-1000 || !(w > 0.0) ? log(r) : log(w) - log(total));
}

constexpr int kThreads = 512, kWaves = kThreads / 64;
constexpr int kDigits = 4;       // of a level of the search by weight
constexpr uint32_t kMostChunks = 1024;

struct Shared {
    double digit[kDigits][kThreads];
    double chunk[kMostChunks];
    uint32_t count[256];
    double part[kWaves];
    uint32_t word[kWaves];
    double sum;
    uint32_t a, b;
};

template <class T>
struct Logits {
    const T* p;
    uint32_t n;
    __device__ __forceinline__ float operator()(uint32_t i) const { return float(p[i]); }
};

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    return v;
}
__device__ double block_sum(double v, Shared& sh) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0;
    for (int i = 0; i < kWaves; ++i) v += sh.part[i];
    return v;
}
__device__ uint32_t block_max(uint32_t v, Shared& sh) {
    for (int d = 32; d; d >>= 1) v = max(v, uint32_t(__shfl_xor(int(v), d)));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.word[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
    for (int i = 0; i < kWaves; ++i) v = max(v, sh.word[i]);
    return v;
}
__device__ uint32_t block_count(uint32_t v, Shared& sh) {
    for (int d = 32; d; d >>= 1) v += uint32_t(__shfl_xor(int(v), d));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.word[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
    for (int i = 0; i < kWaves; ++i) v += sh.word[i];
    return v;
}

// A prefix of the order: the items with larger keys, and the first `ties` with this one.
struct Cut {
    uint32_t key, ties;
    __device__ bool shorter(const Cut& o) const { return key != o.key ? key > o.key : ties < o.ties; }
};

// The first k items: four levels of eight bits, counted.
template <class T>
__device__ Cut cut_by_count(const Logits<T>& x, uint32_t k, Shared& sh) {
    uint32_t known = 0, left = k;
    for (int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        for (int i = threadIdx.x; i < 256; i += kThreads) sh.count[i] = 0;
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < x.n; i += kThreads) {
            const uint32_t key = key_of(x(i));
            if (key && (shift == 24 || key >> (shift + 8) == known)) atomicAdd(&sh.count[(key >> shift) & 255u], 1u);
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            uint32_t before = 0, d = 255;
            for (;; --d) {  // (the k-th item is there)
                if (before + sh.count[d] >= left || d == 0) break;
                before += sh.count[d];
            }
            sh.a = d;
            sh.b = left - before;
        }
        __syncthreads();
        known = known << 8 | sh.a;
        left = sh.b;
    }
    return {known, left};
}

// The fewest items whose weights reach `target` (past: exceed it), which those with keys of at least that of `most` do.
template <class T>
__device__ Cut cut_by_weight(const Logits<T>& x, double target, bool past, const Cut& most, double top, double c, Shared& sh) {
    uint32_t known = 0;
    double before = 0.0;
    for (int shift = 30; shift >= 0; shift -= 2) {
        for (int d = 0; d < kDigits; ++d) sh.digit[d][threadIdx.x] = 0.0;
        for (uint32_t i = threadIdx.x; i < x.n; i += kThreads) {
            const float v = x(i);
            const uint32_t key = key_of(v);
            if (key >= most.key && key && (shift == 30 || key >> (shift + 2) == known)) sh.digit[(key >> shift) & 3u][threadIdx.x] += weight(v, top, c);
        }
        double sums[kDigits];
#pragma unroll 1
        for (int d = 0; d < kDigits; ++d) sums[d] = block_sum(sh.digit[d][threadIdx.x], sh);
        int found = -1;
        double at = before;
        for (int d = kDigits - 1; d >= 0; --d) {
            if (sums[d] > 0.0) {  // (the last that holds something, should rounding leave the target beyond it)
                found = d;
                before = at;
                at += sums[d];
                if (past ? at > target : at >= target) break;
            }
        }
        if (found < 0) return most;  // nothing of these weighs anything
        known = known << 2 | uint32_t(found);
        __syncthreads();
    }
    const double w = weight(value_of(known), top, c), n = past ? floor((target - before) / w) + 1.0 : ceil((target - before) / w);
    return {known, n < 1.0 ? 1u : n < 4294967295.0 ? uint32_t(n) : 0xFFFFFFFFu};
}

// The index up to which items with the cut's key are kept; of: that of the last of them.
template <class T>
__device__ uint32_t last_tie(const Logits<T>& x, const Cut& cut, bool of, Shared& sh) {
    uint32_t n = 0;
    for (uint32_t i = threadIdx.x; i < x.n; i += kThreads) n += key_of(x(i)) == cut.key;
    n = block_count(n, sh);
    if (!of && n <= cut.ties) return x.n - 1;
    // a wave goes through the row; the others wait
    __syncthreads();
    if (threadIdx.x < 64) {
        uint32_t left = min(cut.ties, n);  // at least 1
        for (uint32_t b = 0; b < x.n; b += 64) {
            const uint32_t i = b + threadIdx.x;
            uint64_t m = __ballot(i < x.n && key_of(x(min(i, x.n - 1))) == cut.key);
            const uint32_t c = uint32_t(__popcll(m));
            if (c >= left) {
                for (; left > 1; --left) m &= m - 1;
                if (threadIdx.x == 0) sh.a = b + uint32_t(__ffsll((unsigned long long)m)) - 1;
                break;
            }
            left -= c;
        }
    }
    __syncthreads();
    return sh.a;
}

// Any row, whatever it holds, one pass after another: what the quick way below does not take.  (By value: by reference the caller keeps
// its arguments in private memory.)
template <bool FALLING, class T>
__device__ __noinline__ void sample_slowly(Row a, uint32_t row, Logits<T> x, Shared& sh) {
    const Settings s = settings_of(a, row);
    uint32_t top_key = 0, n = 0;
    for (uint32_t i = threadIdx.x; i < x.n; i += kThreads) {
        const uint32_t k = key_of(x(i));
        top_key = max(top_key, k);
        n += k != 0;
    }
    top_key = block_max(top_key, sh);
    n = block_count(n, sh);
    if (!n) {
        if (threadIdx.x == 0) {
            a.items[row] = -1;
            if (a.log_probability) a.log_probability[row] = -__builtin_inff();
        }
        return;
    }
    const double top = double(value_of(top_key));
    Cut cut{kLowest, 0xFFFFFFFFu};
    if (s.k < n) cut = cut_by_count(x, s.k, sh);
    if (s.p < 1.0) {
        double sum = 0.0;
        for (uint32_t i = threadIdx.x; i < x.n; i += kThreads) {
            const float v = x(i);
            if (key_of(v) > cut.key || (cut.ties == 0xFFFFFFFFu && key_of(v) == cut.key)) sum += weight(v, top, s.c);
        }
        sum = block_sum(sum, sh);
        if (cut.ties != 0xFFFFFFFFu) sum += double(cut.ties) * weight(value_of(cut.key), top, s.c);
        const Cut by = cut_by_weight(x, s.p * sum, false, cut, top, s.c, sh);
        if (by.shorter(cut)) cut = by;
    }
    if (s.m > 0.0) {
        // the least key whose weight reaches m: weights rise with keys
        uint32_t lo = kLowest, hi = top_key;
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo) / 2;
            if (weight(value_of(mid), top, s.c) >= s.m) hi = mid;
            else lo = mid + 1;
        }
        const Cut by{lo, 0xFFFFFFFFu};
        if (by.shorter(cut)) cut = by;
    }
    const uint32_t last = cut.ties == 0xFFFFFFFFu ? x.n - 1 : last_tie(x, cut, false, sh);
    const auto kept = [&](uint32_t i, float v) {
        const uint32_t k = key_of(v);
        return k > cut.key || (k == cut.key && i <= last);
    };
    if constexpr (FALLING) {
        double sum = 0.0;
        for (uint32_t i = threadIdx.x; i < x.n; i += kThreads) {
            const float v = x(i);
            if (kept(i, v)) sum += weight(v, top, s.c);
        }
        sum = block_sum(sum, sh);
        const Cut by = cut_by_weight(x, inner(a.uniforms[row]) * sum, true, cut, top, s.c, sh);
        const uint32_t item = last_tie(x, by, true, sh);
        if (threadIdx.x == 0) {
            a.items[row] = item;
            if (a.log_probability) a.log_probability[row] = log_share(weight(value_of(by.key), top, s.c), sum);
        }
        return;
    }
    // the kept weights of chunks of the row, then of one of them item by item
    uint32_t size = 64;
    while (uint64_t(size) * kMostChunks < x.n) size *= 2;
    const uint32_t chunks = (x.n + size - 1) / size, lane = threadIdx.x & 63;
    for (uint32_t j = threadIdx.x >> 6; j < chunks; j += kWaves) {
        double sum = 0.0;
        for (uint32_t i = j * size + lane; i < min(x.n, (j + 1) * size); i += 64) {
            const float v = x(i);
            if (kept(i, v)) sum += weight(v, top, s.c);
        }
        sum = wave_sum(sum);
        if (lane == 0) sh.chunk[j] = sum;
    }
    __syncthreads();
    if (threadIdx.x < 64) {
        double total = 0.0;
        for (uint32_t j = 0; j < chunks; ++j) total += sh.chunk[j];
        const double target = double(a.uniforms[row]) * total;
        double before = 0.0, start = 0.0;
        uint32_t at = 0;
        bool over = false;
        for (uint32_t j = 0; j < chunks && !over; ++j)
            if (sh.chunk[j] > 0.0) {  // (the last that holds something, should rounding leave the target beyond it)
                at = j;
                start = before;
                before += sh.chunk[j];
                over = before > target;
            }
        int64_t item = -1;
        double w = 0.0;
        for (uint32_t b = at * size; b < min(x.n, (at + 1) * size); b += 64) {
            const uint32_t i = b + lane;
            const float v = x(min(i, x.n - 1));
            const double mine = i < min(x.n, (at + 1) * size) && kept(i, v) ? weight(v, top, s.c) : 0.0;
            double upto = mine;
#pragma unroll
            for (int d = 1; d < 64; d *= 2) {
                const double o = __shfl_up(upto, d);
                if (int(lane) >= d) upto += o;
            }
            const uint64_t some = __ballot(mine > 0.0), past = __ballot(mine > 0.0 && start + upto > target);
            if (some) {
                const int l = past ? __ffsll((unsigned long long)past) - 1 : 63 - __clzll((long long)some);
                item = b + l;
                w = __shfl(mine, l);
            }
            if (past) break;
            start += __shfl(upto, 63);
        }
        if (lane == 0) {
            a.items[row] = item;
            if (a.log_probability) a.log_probability[row] = log_share(w, total);
        }
    }
}

// ---------------------------------------------------------------------------------------
// The quick way
// ---------------------------------------------------------------------------------------
constexpr uint32_t kBins = 2048;     // and one for what is no item
constexpr uint32_t kTops = 1024;     // items above the sample's largest that are listed
constexpr uint32_t kListed = 4096;   // items near a cut that are listed and sorted
// Items that are sorted, and drawn from, by counting: a wave's (the top 50 of 10,000 took 25.1 us, sorted by the network and drawn from
// the chunks 26.7; with 256 for the bound a top 200 took 36, not 28).
constexpr uint32_t kFew = 64;
constexpr uint32_t kSampled = 1u << 18;  // values of a row that a sample of 4096 stands for
constexpr uint32_t kStep = 512;      // values that a wave loads at a time, eight a lane

template <uint32_t LISTED>
struct QuickOf {
    union {
        uint32_t count[kBins + 4];
        unsigned long long fixed[kMostChunks];  // (when the counts have served)
    };
    uint64_t list[LISTED];
    double chunk[kMostChunks];
    double part[kWaves];
    uint32_t word[kWaves];
    uint32_t tops, listed;
    float low;
};
using Quick = QuickOf<kListed>;
using Brief = QuickOf<kTops>;  // what the first pass needs
union Both {
    Shared slow;
    Quick quick;
};

// Values [i, i + 8) of a row of n as they are in memory, -inf behind its end.
template <class T>
using Eight = T __attribute__((ext_vector_type(8)));
template <class T>
__device__ __forceinline__ Eight<T> load8(const T* p, uint32_t i, uint32_t n) {
    if (i + 8 <= n) return loose_load<Eight<T>>(p + i);
    Eight<T> v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = i + e < n ? p[i + e] : T(-__builtin_inff());
    return v;
}
template <class T>
__device__ __forceinline__ void widen(const Eight<T>& x, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = float(x[e]);
}

__device__ __forceinline__ bool is_item(float x) { return x > -__builtin_inff(); }
// the order of a list: larger logits first, then smaller indices
__device__ __forceinline__ uint64_t entry_of(uint32_t key, uint32_t i) { return uint64_t(~key) << 32 | i; }
__device__ __forceinline__ uint32_t entry_key(uint64_t e) { return ~uint32_t(e >> 32); }

template <class Q>
__device__ double quick_sum(double v, Q& q) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) q.part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0;
    for (int i = 0; i < kWaves; ++i) v += q.part[i];
    return v;
}
template <class Q>
__device__ uint32_t quick_count(uint32_t v, Q& q) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += uint32_t(__shfl_xor(int(v), d));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) q.word[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
    for (int i = 0; i < kWaves; ++i) v += q.word[i];
    return v;
}
// the largest value, NaN left out
template <class Q>
__device__ float quick_max(float v, Q& q) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v = fmaxf(v, __shfl_xor(v, d));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) q.word[threadIdx.x >> 6] = __float_as_uint(v);
    __syncthreads();
    v = -__builtin_inff();
    for (int i = 0; i < kWaves; ++i) v = fmaxf(v, __uint_as_float(q.word[i]));
    return v;
}
// the sum of the values of the threads before this one; total: of all
template <class N>
__device__ N quick_before(N v, N& total, N (&part)[kWaves]) {
    N upto = v;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const N o = __shfl_up(upto, d);
        if (int(threadIdx.x & 63) >= d) upto += o;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 63) part[threadIdx.x >> 6] = upto;
    __syncthreads();
    N before = 0;
    total = 0;
    for (int i = 0; i < kWaves; ++i) {
        if (i < int(threadIdx.x >> 6)) before += part[i];
        total += part[i];
    }
    return before + (upto - v);
}

// Ascending, by a bitonic network over E neighbours a thread: the exchanges within a thread and within a wave, most of them, need
// no memory and no barrier.
template <int E>
__device__ void sort_many(uint64_t* list, uint32_t n) {
    constexpr uint32_t SIZE = E * kThreads, WAVE = 64 * E;
    const uint32_t first = E * threadIdx.x;
    uint64_t v[E];
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = first + e < n ? list[first + e] : ~0ull;
    // one of the pair keeps the smaller: the lower one where the run ascends
    const auto exchange = [&](int e, uint64_t other, uint32_t j, uint32_t k) {
        const uint32_t i = first + e;
        const bool smaller = ((i & j) == 0) == ((i & k) == 0);
        v[e] = (v[e] < other) == smaller ? v[e] : other;
    };
    for (uint32_t k = 2; k <= SIZE; k *= 2) {
        uint32_t j = k / 2;
        for (; j >= WAVE; j /= 2) {
            __syncthreads();
#pragma unroll
            for (int e = 0; e < E; ++e) list[first + e] = v[e];
            __syncthreads();
#pragma unroll
            for (int e = 0; e < E; ++e) exchange(e, list[(first + e) ^ j], j, k);
        }
        for (; j >= E; j /= 2) {
#pragma unroll
            for (int e = 0; e < E; ++e) exchange(e, uint64_t(__shfl_xor((unsigned long long)v[e], int(j / E))), j, k);
        }
#pragma unroll
        for (int d = E / 2; d; d /= 2)
            if (uint32_t(d) < k) {
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (!(e & d)) {
                        const bool up = ((first + e) & k) == 0;
                        const uint64_t lo = v[e] < v[e | d] ? v[e] : v[e | d], hi = v[e] < v[e | d] ? v[e | d] : v[e];
                        v[e] = up ? lo : hi;
                        v[e | d] = up ? hi : lo;
                    }
            }
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e) list[first + e] = v[e];
    __syncthreads();
}
// Ascending; n <= kListed.  Few: each entry's place is the number of those before it (no two are alike), counted by a thread.
__device__ void quick_sort(uint64_t* list, uint32_t n) {
    if (n <= kFew) {
        __syncthreads();
        const uint64_t mine = threadIdx.x < n ? list[threadIdx.x] : 0;
        uint32_t place = 0;
        if ((threadIdx.x & ~63u) < n) {  // (broadcast reads: the waves without an entry leave LDS to the others)
#pragma unroll 4
            for (uint32_t i = 0; i < n; ++i) place += list[i] < mine;
        }
        __syncthreads();
        if (threadIdx.x < n) list[place] = mine;
        __syncthreads();
        return;
    }
    if (n <= kThreads) sort_many<1>(list, n);
    else if (n <= 2 * kThreads) sort_many<2>(list, n);
    else if (n <= 4 * kThreads) sort_many<4>(list, n);
    else sort_many<8>(list, n);
}

// A row's chunks of `size` values and those of them that a workgroup goes through.
struct Part {
    uint32_t size, chunks, from, to;
};
// Those chunks, the waves in turn: f(first index of the lane, its eight values), the next ones under way, and end(chunk) after each.
template <class T, class F, class E>
__device__ __forceinline__ void through(const Logits<T>& x, const Part& part, F f, E end) {
    const uint32_t lane = threadIdx.x & 63, size = part.size;
    uint32_t j = part.from + (threadIdx.x >> 6);
    if (j >= part.to) return;
    uint32_t b = j * size;
    Eight<T> next = load8(x.p, b + 8 * lane, x.n);
    for (;;) {
        const Eight<T> now = next;
        const uint32_t here = b, chunk = j;
        b += kStep;
        const bool ends = b >= min(uint64_t(x.n), uint64_t(chunk + 1) * size);
        if (ends) {
            j += kWaves;
            b = j * size;
        }
        if (j < part.to) next = load8(x.p, b + 8 * lane, x.n);
        float v[8];
        widen<T>(now, v);
        f(here + 8 * lane, v);
        if (ends) {
            end(chunk);
            if (j >= part.to) break;
        }
    }
}

// The key of the least value that weighs at least m beside `top`: found from the logarithm, 64 keys at a time.
__device__ uint32_t least_key(double m, float top, double c) {
    const uint32_t high = key_of(top);
    const float guess = float(double(top) + log2(m) / c);
    uint32_t at = guess > -__builtin_inff() ? min(max(key_of(guess), kLowest), high) : kLowest;
    uint32_t lo = kLowest, hi = high;  // the key lies within
    at = at > lo + 32 ? at - 32 : lo;
    const uint32_t mine = min(at + (threadIdx.x & 63), high);
    const uint64_t some = __ballot(weight(value_of(mine), double(top), c) >= m);
    if (some) {
        const int l = __ffsll((unsigned long long)some) - 1;
        hi = min(at + l, high);
        if (l > 0) return hi;
        if (at == lo) return lo;
    } else {
        lo = min(at + 64, high);
    }
    while (lo < hi) {
        const uint32_t mid = lo + (hi - lo) / 2;
        if (weight(value_of(mid), double(top), c) >= m) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

// The item that u draws from those that the cut keeps, whose weights the chunks' sums hold; by one wave.  A chunk's sum is zero only
// where none of its kept items weighs anything, so that an item is found within.
template <class T>
__device__ void draw(const Row& a, uint32_t row, const Logits<T>& x, const Part& part, uint32_t cut_key, uint32_t last, float ref, double c, const double* chunk) {
    const uint32_t lane = threadIdx.x & 63, per = (part.chunks + 63) / 64, from = lane * per, to = min(from + per, part.chunks);
    double mine = 0.0;
    for (uint32_t j = from; j < to; ++j) mine += chunk[j];
    double upto = mine;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const double o = __shfl_up(upto, d);
        if (int(lane) >= d) upto += o;
    }
    const double total = __shfl(upto, 63), target = double(a.uniforms[row]) * total;
    // the first chunk that brings the sum past the target, or the last that holds something
    double run = upto - mine, start = 0.0;
    uint32_t found = 0, some = 0;
    for (uint32_t j = from; j < to && !found; ++j) {
        const double v = chunk[j];
        if (v > 0.0) {
            some = j + 1;
            start = run;
            if (run + v > target) found = j + 1;
        }
        run += v;
    }
    const uint64_t past = __ballot(found != 0), any = __ballot(some != 0);
    const int at_lane = past ? __ffsll((unsigned long long)past) - 1 : 63 - __clzll((long long)any);
    const uint32_t at = uint32_t(__shfl(int(some), at_lane)) - 1;
    start = __shfl(start, at_lane);
    double w = 0.0;
    int64_t item = -1;
    const uint32_t stop = uint32_t(min(uint64_t(x.n), uint64_t(at + 1) * part.size));
    for (uint32_t b = at * part.size; b < stop; b += kStep) {
        const uint32_t i = b + 8 * lane;
        float v[8];
        widen<T>(load8(x.p, i, x.n), v);
        double ws[8], sum = 0.0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t k = key_of(v[e]);
            const bool kept = k > cut_key || (k == cut_key && i + e <= last);
            ws[e] = kept ? weight(v[e], double(ref), c) : 0.0;
            sum += ws[e];
        }
        double within = sum;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const double o = __shfl_up(within, d);
            if (int(lane) >= d) within += o;
        }
        const uint64_t holds = __ballot(sum > 0.0), over = __ballot(sum > 0.0 && start + within > target);
        if (holds) {
            const int l = over ? __ffsll((unsigned long long)over) - 1 : 63 - __clzll((long long)holds);
            // within the lane: the first past the target, or the last that weighs something
            double here = start + (within - sum), wm = 0.0;
            int im = 0;
            bool done = false;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                here += ws[e];
                if (!done && ws[e] > 0.0) {
                    im = int(i) + e;
                    wm = ws[e];
                    done = here > target;
                }
            }
            item = __shfl(im, l);
            w = __shfl(wm, l);
        }
        if (over) break;
        start += __shfl(within, 63);
    }
    if (lane == 0) {
        a.items[row] = item;
        if (a.log_probability) a.log_probability[row] = log_share(w, total);
    }
}

// What one pass over a row leaves for the next, alike in every thread.
struct Mid {
    float ref, low, top;   // what weights refer to: a sample's largest value; its least; the row's largest
    double all, above;     // the sum of all weights; of those above the listed ones
    uint32_t tops;         // items above ref
    int first, end;        // the bins whose items are listed (first -1: and what lies above them)
    uint32_t least;        // the least key that min-p keeps
    // along falling logits
    double kept;           // the sum of the kept weights; out of the second pass, of those above the listed items
    double target;         // the drawn item is the first at which the sum exceeds it; negative: not known yet
    bool whole;            // all that min-p keeps is listed
};
struct Kind {
    bool by_count, by_weight;
    __device__ bool sums() const { return !by_count && !by_weight; }
};
__device__ __forceinline__ Kind kind_of(const Settings& s, uint32_t n) { return {s.k < n, s.p < 1.0}; }

// Bins of equal width from ref down to the sample's least value, or over 64 binary orders of weight.
struct Bins {
    float ref, per;
    __device__ Bins(const Mid& m, const Settings& s) : ref(m.ref) {
        const double span = fmin(double(m.ref) - double(m.low), 64.0 / s.c);
        per = span > 0.0 ? float(double(kBins - 2) / span) : 0.0f;
    }
    __device__ __forceinline__ uint32_t of(float v) const {  // of values up to ref
        const float f = (ref - fmaxf(v, -3.4028235e38f)) * per;
        return is_item(v) ? (f < float(kBins - 1) ? uint32_t(f) : kBins - 1) : kBins;
    }
};

// The least value up to ref whose bin is at most b (b >= 0): bins fall as values rise; 64 keys at a time.
__device__ float edge_of(const Bins& bins, int b) {
    uint32_t lo = kLowest, hi = key_of(bins.ref);  // the key lies within
    while (lo < hi) {
        const uint32_t step = (hi - lo) / 64 + 1, at = min(uint64_t(lo) + uint64_t(step) * (threadIdx.x & 63), uint64_t(hi));
        const uint64_t in = __ballot(int(bins.of(value_of(at))) <= b);
        const int l = in ? __ffsll((unsigned long long)in) - 1 : 64;
        const uint32_t from = lo;
        if (l < 64) hi = min(uint64_t(from) + uint64_t(step) * l, uint64_t(hi));
        if (l > 0) lo = uint32_t(min(uint64_t(from) + uint64_t(step) * (l - 1) + 1, uint64_t(hi)));
    }
    return value_of(lo);
}

// A sample, 512 values at eight places (all of a short row; of a long one more, so that one row in 10^7 has more than kTops items above
// it): its largest value is what weights refer to.
template <class T, class Q>
__device__ bool begin(const Logits<T>& x, Q& q, Mid& m) {
    float ref = -__builtin_inff(), low = __builtin_inff();
    const auto look = [&](const float(&v)[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            ref = fmaxf(ref, v[e]);
            low = fminf(low, is_item(v[e]) ? v[e] : __builtin_inff());
        }
    };
    if (x.n <= kWaves * kStep) {
        const uint32_t chunks = (x.n + kStep - 1) / kStep;
        through(x, Part{kStep, chunks, 0, chunks}, [&](uint32_t, const float(&v)[8]) { look(v); }, [](uint32_t) {});
    } else {
        const uint32_t places = kWaves * ((x.n + kSampled - 1) / kSampled);
        for (uint32_t w = threadIdx.x >> 6; w < places; w += kWaves) {
            float v[8];
            widen<T>(load8(x.p, uint32_t(uint64_t(x.n - kStep) * w / (places - 1)) + 8 * (threadIdx.x & 63), x.n), v);
            look(v);
        }
    }
    m.ref = quick_max(ref, q);
    m.low = -quick_max(-low, q);
    return fabsf(m.ref) < __builtin_inff();
}

// The first pass.  Neither top-k nor top-p: the chunks' sums, or with min-p, which needs the row's largest value, that alone.  Else
// the bins' counts, what lies above ref listed, and, where top-k does not cut, the sum of all weights.  FALLING: these always.
template <bool FALLING, class T, class Q>
__device__ void pass_one(const Logits<T>& x, const Settings& s, const Part& part, Q& q, Mid& m) {
    const Kind kind = kind_of(s, x.n);
    const uint32_t lane = threadIdx.x & 63;
    float top = -__builtin_inff();
    m.all = 0.0;
    m.tops = 0;
    if (!FALLING && kind.sums()) {
        double sum = 0.0;
        through(x, part, [&](uint32_t, const float(&v)[8]) {
#pragma unroll
            for (int e = 0; e < 8; ++e) top = fmaxf(top, v[e]);
            if (s.m == 0.0) {
#pragma unroll
                for (int e = 0; e < 8; ++e) sum += exp2_of((double(v[e]) - double(m.ref)) * s.c);
            }
        }, [&](uint32_t j) {
            if (s.m == 0.0) {
                sum = wave_sum(sum);
                if (lane == 0) q.chunk[j] = sum;
                sum = 0.0;
            }
        });
        m.top = quick_max(top, q);
        return;
    }
    const Bins bins(m, s);
    __syncthreads();
    for (uint32_t i = threadIdx.x; i <= kBins; i += kThreads) q.count[i] = 0;
    if (threadIdx.x == 0) q.tops = 0;
    __syncthreads();
    double all = 0.0;
    through(x, part, [&](uint32_t i, const float(&v)[8]) {
        bool above = false;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            top = fmaxf(top, v[e]);
            above |= v[e] > m.ref;
            if (!(v[e] > m.ref)) atomicAdd(&q.count[bins.of(v[e])], 1u);
        }
        if (!kind.by_count) {
#pragma unroll
            for (int e = 0; e < 8; ++e) all += exp2_of((double(v[e]) - double(m.ref)) * s.c);
        }
        if (__any(above)) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (v[e] > m.ref) {
                    const uint32_t at = atomicAdd(&q.tops, 1u);
                    if (at < kTops) q.list[at] = entry_of(key_of(v[e]), i + e);
                }
        }
    }, [](uint32_t) {});
    m.top = quick_max(top, q);
    if (!kind.by_count) m.all = quick_sum(all, q);
    m.tops = q.tops;
}
// Whether weights that refer to ref have room in fp64, and the list held what lies above it.
__device__ __forceinline__ bool fits(const Settings& s, const Mid& m) { return m.top < __builtin_inff() && m.tops <= kTops && (double(m.top) - double(m.ref)) * s.c < 900.0; }

// The bins' counts added up: a thread's four sums (up to each bin and with it), what lies before them, the items of all bins and of the last.
struct Counts {
    uint32_t mine[4], before, items, last;
};
__device__ Counts counts_of(Quick& q) {
    Counts c;
    c.last = q.count[kBins - 1];
#pragma unroll
    for (int e = 0; e < 4; ++e) c.mine[e] = q.count[4 * threadIdx.x + e];
    c.before = quick_before(c.mine[0] + c.mine[1] + c.mine[2] + c.mine[3], c.items, q.word);
    c.mine[0] += c.before;
#pragma unroll
    for (int e = 1; e < 4; ++e) c.mine[e] += c.mine[e - 1];
    static_assert(kBins == 4 * kThreads, "four bins a thread");
    // (every thread has read its own, and the last one, before the barriers of quick_before)
#pragma unroll
    for (int e = 0; e < 4; ++e) q.count[4 * threadIdx.x + e] = c.mine[e];
    __syncthreads();
    return c;
}
// items of the bins up to b, whose counts are added up
__device__ __forceinline__ uint32_t upto(const Quick& q, int b) { return b < 0 ? 0u : q.count[min(b, int(kBins) - 1)]; }

// The bin with the k-th item, or, of a row that has fewer (a mask leaves them), with the last.
__device__ void range_by_count(uint32_t k, const Counts& counts, Quick& q, Mid& m) {
    uint32_t c = 0;
    k = min(k, m.tops + counts.items);
#pragma unroll
    for (int e = 0; e < 4; ++e) c += m.tops + counts.mine[e] < k;
    m.end = int(quick_count(c, q));
    if (k <= m.tops) m.end = -1;
}
// The bins in which what lies behind may come to weigh `need`, and the one where it likely does: from the least weights up, each item
// taken for one in its bin's middle and so off by at most half a bin's width (in the last bin, which has no lower end, for too large).
__device__ int range_by_weight(const Settings& s, double need, const Counts& counts, Quick& q, Mid& m) {
    const Bins bins(m, s);
    const double width = bins.per > 0.0f ? s.c / double(bins.per) : 0.0, off = exp2_of(0.501 * width);
    const double open = double(counts.last) * exp2_of(-(double(kBins) - 0.5) * width);
    double tail[4], sum;
    uint32_t above = 0, each = 0, within = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t c = counts.mine[e] - (e ? counts.mine[e - 1] : counts.before);
        tail[e] = c ? double(c) * exp2_of(-(double(4 * threadIdx.x + e) + 0.5) * width) : 0.0;
    }
    double have = quick_before(tail[0] + tail[1] + tail[2] + tail[3], sum, q.part);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        have += tail[e];
        const double behind = sum - have;
        above += behind - open > need * off;
        each += behind > need;
        within += behind * off > need;
    }
    above = quick_count(above, q), each = quick_count(each, q), within = quick_count(within, q);
    m.first = bins.per > 0.0f && sum - open > need * off ? int(above) : -1;
    m.end = sum * off > need ? int(min(within, kBins - 1)) : -1;
    return int(min(each, kBins - 1));
}
// As many of these bins as a list holds: from the top if that is few; of many items those in the middle, where errors cancel out.
__device__ bool narrow(int at, const Quick& q, Mid& m) {
    for (;;) {
        if (m.first <= 0 || m.tops + upto(q, m.end) <= kFew) m.first = -1;
        if ((m.first < 0 ? m.tops + upto(q, m.end) : upto(q, m.end) - upto(q, m.first - 1)) <= kListed) return true;
        const int first = m.first < 0 ? 0 : m.first;
        if (m.end <= at && first >= at && m.first >= 0) return false;
        m.first = min(first + max((at - first + 1) / 2, 1), max(at, 1));
        m.end = max(m.end - max((m.end - at + 1) / 2, 0), at);
    }
}

// From the counts, which bins' items are listed.
__device__ bool between(uint32_t n, const Settings& s, Quick& q, Mid& m) {
    const Kind kind = kind_of(s, n);
    m.above = 0.0;
    m.first = m.end = -1;
    if (kind.sums()) {
        if (s.m > 0.0) m.ref = m.top;
        m.least = s.m > 0.0 ? least_key(s.m, m.top, s.c) : kLowest;
        return true;
    }
    const Counts counts = counts_of(q);
    if (kind.by_count) {
        range_by_count(s.k, counts, q, m);
        if (m.tops + upto(q, m.end) > kListed) return false;
    } else if (!narrow(range_by_weight(s, (1.0 - s.p) * m.all, counts, q, m), q, m)) {
        return false;
    }
    m.least = s.m > 0.0 ? least_key(s.m, m.top, s.c) : kLowest;
    return true;
}

// The same along falling logits.  First: what the cut needs, or, where nothing is cut, what the draw does; -2 for the end: the second pass
// lists nothing and adds up what min-p keeps.
constexpr int kNoList = -2;
__device__ bool between_falling(uint32_t n, const Settings& s, double u, Quick& q, Mid& m) {
    const Kind kind = kind_of(s, n);
    m.above = m.kept = 0.0;
    m.target = -1.0;
    m.whole = false;
    m.first = m.end = -1;
    m.least = s.m > 0.0 ? least_key(s.m, m.top, s.c) : kLowest;
    const Counts counts = counts_of(q);
    if (kind.by_count) {
        range_by_count(s.k, counts, q, m);
        return m.tops + upto(q, m.end) <= kListed;
    }
    if (s.m == 0.0 && !kind.by_weight) {
        m.kept = m.all;
        m.target = u * m.all;
        return narrow(range_by_weight(s, m.all - m.target, counts, q, m), q, m);
    }
    int at = 0;
    m.end = int(kBins);
    if (kind.by_weight) at = range_by_weight(s, (1.0 - s.p) * m.all, counts, q, m);
    if (s.m > 0.0) {
        // what min-p keeps, if that is few, from the top, unless top-p's cut lies above its end
        const float least = value_of(m.least);
        const int end = least > m.ref ? -1 : min(int(Bins(m, s).of(least)), int(kBins) - 1);
        if (m.tops + upto(q, end) <= kListed && (m.first > 0 || end <= m.end)) {
            m.first = -1;
            m.end = end;
            m.whole = true;
            return true;
        }
    }
    if (kind.by_weight) return narrow(at, q, m);
    m.end = kNoList;
    return true;
}
// Again: the bins around the target.  summed: whether the counts are added up.
__device__ bool between_again(const Settings& s, bool summed, Quick& q, Mid& m) {
    Counts counts;
    if (!summed) {
        counts = counts_of(q);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) counts.mine[e] = q.count[4 * threadIdx.x + e];
        counts.before = threadIdx.x ? q.count[4 * threadIdx.x - 1] : 0u;
        counts.items = q.count[kBins - 1];
        counts.last = counts.items - q.count[kBins - 2];
    }
    m.above = 0.0;
    return narrow(range_by_weight(s, m.all - m.target, counts, q, m), q, m);
}

// The second pass: the items of the chosen bins are listed, and the sums of what lies above them and min-p keeps go to the chunks.
template <class T>
__device__ void pass_two(const Logits<T>& x, const Settings& s, const Part& part, Quick& q, Mid& m) {
    const uint32_t lane = threadIdx.x & 63;
    const float least = value_of(m.least);
    double sum = 0.0;
    if (kind_of(s, x.n).sums()) {
        if (s.m == 0.0) return;
        through(x, part, [&](uint32_t, const float(&v)[8]) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (v[e] >= least) sum += weight(v[e], double(m.ref), s.c);
        }, [&](uint32_t j) {
            sum = wave_sum(sum);
            if (lane == 0) q.chunk[j] = sum;
            sum = 0.0;
        });
        return;
    }
    if (m.first < 0 && m.end < 0) {  // what lies above ref, listed already
        if (threadIdx.x == 0) q.listed = m.tops;
        __syncthreads();
        return;
    }
    __syncthreads();
    if (threadIdx.x == 0) q.listed = 0;
    __syncthreads();
    const Bins bins(m, s);
    // what is listed lies from `down` on and below `up`
    const float up = m.first < 0 ? __builtin_inff() : m.first == 0 ? nextafterf(m.ref, __builtin_inff()) : edge_of(bins, m.first - 1), down = m.end < 0 ? nextafterf(m.ref, __builtin_inff()) : edge_of(bins, m.end);
    const bool apart = least > up;  // min-p leaves out some of what lies above
    double above = 0.0;
    through(x, part, [&](uint32_t i, const float(&v)[8]) {
        bool high = false, in = false;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            high |= v[e] >= up;
            in |= v[e] >= down && v[e] < up;
        }
        if (__any(high)) {
            if (!apart) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const double w = exp2_of((double(v[e]) - double(m.ref)) * s.c);
                    sum += v[e] >= up ? w : 0.0;
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const double w = exp2_of((double(v[e]) - double(m.ref)) * s.c);
                    above += v[e] >= up ? w : 0.0;
                    sum += v[e] >= least ? w : 0.0;
                }
            }
        }
        if (__any(in)) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (v[e] >= down && v[e] < up) {
                    const uint32_t at = atomicAdd(&q.listed, 1u);
                    if (at < kListed) q.list[at] = entry_of(key_of(v[e]), i + e);
                }
        }
    }, [&](uint32_t j) {
        if (m.first >= 0) {
            if (!apart) above += sum;
            sum = wave_sum(sum);
            if (lane == 0) q.chunk[j] = sum;
            sum = 0.0;
        }
    });
    m.above = quick_sum(above, q);
}

// The same along falling logits: the items of the chosen bins are listed, what lies above them is added up, and that of it which min-p keeps.
// again: the list is for the draw, and what is kept is known.
template <class T>
__device__ void pass_two_falling(const Logits<T>& x, const Settings& s, const Part& part, bool again, Quick& q, Mid& m) {
    if (!again && m.first < 0 && m.end == -1) {  // what lies above ref, listed already
        if (threadIdx.x == 0) q.listed = m.tops;
        __syncthreads();
        return;
    }
    __syncthreads();
    if (threadIdx.x == 0) q.listed = 0;
    __syncthreads();
    const float least = value_of(m.least);
    double above = 0.0, kept = 0.0;
    if (m.end == kNoList) {
        through(x, part, [&](uint32_t, const float(&v)[8]) {
            bool any = false;
#pragma unroll
            for (int e = 0; e < 8; ++e) any |= v[e] >= least;
            if (__any(any)) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const double w = exp2_of((double(v[e]) - double(m.ref)) * s.c);
                    kept += v[e] >= least ? w : 0.0;
                }
            }
        }, [](uint32_t) {});
        m.kept = quick_sum(kept, q);
        return;
    }
    const Bins bins(m, s);
    const float past = nextafterf(m.ref, __builtin_inff());
    const float up = m.first < 0 ? __builtin_inff() : m.first == 0 ? past : edge_of(bins, m.first - 1), down = m.end < 0 ? past : edge_of(bins, m.end);
    const bool apart = !again && least > up;  // min-p leaves out some of what lies above
    through(x, part, [&](uint32_t i, const float(&v)[8]) {
        bool high = false, in = false;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            high |= v[e] >= up;
            in |= v[e] >= down && v[e] < up;
        }
        if (__any(high)) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const double w = exp2_of((double(v[e]) - double(m.ref)) * s.c);
                above += v[e] >= up ? w : 0.0;
                if (apart) kept += v[e] >= least ? w : 0.0;
            }
        }
        if (__any(in)) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (v[e] >= down && v[e] < up) {
                    const uint32_t at = atomicAdd(&q.listed, 1u);
                    if (at < kListed) q.list[at] = entry_of(key_of(v[e]), i + e);
                }
        }
    }, [](uint32_t) {});
    m.above = quick_sum(above, q);
    if (!again && m.target < 0.0) m.kept = apart ? quick_sum(kept, q) : m.above;
}

// From the list, and from what lies above it, the cut and the item.
enum class Found { nothing, item, target };  // the row is one for the other way; it is drawn; what is kept is known, the item not listed
template <class T>
__device__ Found finish_falling(const Row& a, uint32_t row, const Logits<T>& x, const Settings& s, Quick& q, Mid& m) {
    const Kind kind = kind_of(s, x.n);
    const double u = inner(a.uniforms[row]);
    if (m.target < 0.0 && m.end == kNoList) {
        m.target = u * m.kept;
        return Found::target;
    }
    const uint32_t listed = q.listed;
    if (listed > kListed || !listed) return Found::nothing;
    quick_sort(q.list, listed);
    // their weights added up, eight neighbours a thread
    double w[8], sum = 0.0, total;
    const uint32_t from = 8 * threadIdx.x, held = kind.by_count ? min(listed, s.k) : listed;
    static_assert(kListed == 8 * kThreads, "eight entries a thread");
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        w[e] = from + e < held ? weight(value_of(entry_key(q.list[from + e])), double(m.ref), s.c) : 0.0;
        sum += w[e];
    }
    const double before = m.above + quick_before(sum, total, q.part);
    uint32_t n = held;  // entries among which the item is
    if (m.target < 0.0) {
        if (kind.by_weight) {
            const double enough = s.p * (kind.by_count ? total : m.all);
            double run = before;
            n = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                n += from + e < held && run < enough;
                run += w[e];
            }
            n = quick_count(n, q);
            if (!kind.by_count && m.above >= enough && m.above > 0.0) return Found::nothing;  // the cut lies above the list, or below it
            if (!kind.by_count && !m.whole && n == listed && m.above + total < enough && m.end < int(kBins) - 1) return Found::nothing;
            n = max(n, 1u);
        }
        uint32_t keep = 0;
        sum = 0.0;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (from + e < n && entry_key(q.list[from + e]) >= m.least) {
                ++keep;
                sum += w[e];
            }
        n = quick_count(keep, q);
        m.kept += quick_sum(sum, q);
        m.target = u * m.kept;
        if (m.first >= 0 && (!n || m.target < m.above)) return Found::target;
    } else {
        if (m.first >= 0 && m.above > m.target) return Found::nothing;  // the item lies above the list, or below it
        if (m.above + total <= m.target && m.end < int(kBins) - 1) return Found::nothing;
    }
    // the first that brings the sum past the target, or the last that weighs something
    uint32_t short_of = 0, some = 0;
    double run = before;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        run += w[e];
        const bool there = from + e < n && w[e] > 0.0;
        some += there;
        short_of += there && run <= m.target;
    }
    short_of = quick_count(short_of, q), some = quick_count(some, q);
    if (!some) return Found::nothing;
    const uint32_t at = min(short_of, some - 1);
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (from + e == at) {
            a.items[row] = int64_t(uint32_t(q.list[at]));
            if (a.log_probability) a.log_probability[row] = log_share(w[e], m.kept);
        }
    return Found::item;
}

// From the list and the chunks' sums: the cut, and the item.
template <class T>
__device__ bool finish(const Row& a, uint32_t row, const Logits<T>& x, const Settings& s, const Part& part, Quick& q, const Mid& m) {
    const Kind kind = kind_of(s, x.n);
    if (kind.sums()) {
        __syncthreads();
        if (threadIdx.x < 64) draw(a, row, x, part, m.least, x.n - 1, m.ref, s.c, q.chunk);
        return true;
    }
    const uint32_t listed = q.listed;
    if (listed > kListed || !listed) return false;
    for (uint32_t i = threadIdx.x; i < part.chunks; i += kThreads) q.fixed[i] = 0;
    quick_sort(q.list, listed);
    // their weights added up, eight neighbours a thread
    double w[8], sum = 0.0;
    const uint32_t from = 8 * threadIdx.x, held = kind.by_count ? min(listed, s.k) : listed;
    static_assert(kListed == 8 * kThreads, "eight entries a thread");
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        w[e] = from + e < held ? weight(value_of(entry_key(q.list[from + e])), double(m.ref), s.c) : 0.0;
        sum += w[e];
    }
    double total;
    double run = m.above + quick_before(sum, total, q.part);
    const double enough = kind.by_weight ? s.p * (kind.by_count ? total : m.all) : 0.0;
    uint32_t n = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        n += from + e < held && (!kind.by_weight || run < enough);
        run += w[e];
    }
    n = quick_count(n, q);
    if (kind.by_weight) {
        if (!kind.by_count && m.above >= enough && m.above > 0.0) return false;                                  // the cut lies above the list,
        if (!kind.by_count && n == listed && m.above + total < enough && m.end < int(kBins) - 1) return false;  // or below it
        n = max(n, 1u);
    }
    uint32_t cut = entry_key(q.list[n - 1]), last = uint32_t(q.list[n - 1]);
    if (m.least > cut) {
        cut = m.least;
        last = x.n - 1;
    }
    if (m.first < 0 && n <= kFew) {
        // All kept items are at hand: an item's kept weights up to its own, in the order of the items, added up by a thread.
        double* const ws = q.chunk;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (from + e < n) ws[from + e] = entry_key(q.list[from + e]) >= m.least ? w[e] : 0.0;
        __syncthreads();
        const bool mine = threadIdx.x < n && ws[threadIdx.x] > 0.0;
        const uint32_t index = mine ? uint32_t(q.list[threadIdx.x]) : 0xFFFFFFFFu;
        double upto = 0.0, kept = 0.0;
        if ((threadIdx.x & ~63u) < n) {
#pragma unroll 4
            for (uint32_t i = 0; i < n; ++i) {
                const double v = ws[i];
                kept += v;
                upto += uint32_t(q.list[i]) <= index ? v : 0.0;
            }
        }
        const double target = double(a.uniforms[row]) * kept;
        // the first that brings the sum past the target, or the last
        uint32_t best = mine && upto > target ? 0x80000000u - index : 0u, far = mine ? index + 1 : 0u;
#pragma unroll
        for (int d = 32; d; d >>= 1) {
            best = max(best, uint32_t(__shfl_xor(int(best), d)));
            far = max(far, uint32_t(__shfl_xor(int(far), d)));
        }
        __syncthreads();
        if ((threadIdx.x & 63) == 0) {
            q.count[threadIdx.x >> 6] = best;
            q.count[kWaves + (threadIdx.x >> 6)] = far;
        }
        __syncthreads();
        for (int i = 0; i < kWaves; ++i) {
            best = max(best, q.count[i]);
            far = max(far, q.count[kWaves + i]);
        }
        const uint32_t item = best ? 0x80000000u - best : far - 1;
        if (mine && index == item) {
            a.items[row] = int64_t(item);
            if (a.log_probability) a.log_probability[row] = log_share(ws[threadIdx.x], kept);
        }
        return true;
    }
    // the kept ones' weights go to their chunks as whole numbers of 2^-50 of the largest: no order of the additions changes those; the
    // upmost bit, which 4096 of them do not reach, tells a chunk whose items all round to zero from one without an item
    int order;
    (void)frexp(weight(value_of(entry_key(q.list[0])), double(m.ref), s.c), &order);
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (from + e < n && w[e] > 0.0 && entry_key(q.list[from + e]) >= m.least) {
            unsigned long long* const to = &q.fixed[uint32_t(q.list[from + e]) / part.size];
            atomicOr(to, 1ull << 63);
            atomicAdd(to, (unsigned long long)(ldexp(w[e], 50 - order) + 0.5));
        }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < part.chunks; i += kThreads) {
        const unsigned long long f = q.fixed[i];
        const double v = (m.first >= 0 ? q.chunk[i] : 0.0) + ldexp(double(f & ~(1ull << 63)), order - 50);
        q.chunk[i] = f && v == 0.0 ? 0x1p-1022 : v;
    }
    __syncthreads();
    if (threadIdx.x < 64) draw(a, row, x, part, cut, last, m.ref, s.c, q.chunk);
    return true;
}

__device__ __forceinline__ Part whole_of(uint32_t n) {
    uint32_t size = kStep;
    while (uint64_t(size) * kMostChunks < n) size *= 2;
    const uint32_t chunks = (n + size - 1) / size;
    return {size, chunks, 0, chunks};
}

// A row in one workgroup.  False: nothing is written, the row is one for the other way.
template <bool FALLING, class T>
__device__ bool sample_quickly(const Row& a, uint32_t row, const Logits<T>& x, Quick& q) {
    const Settings s = settings_of(a, row);
    const Part part = whole_of(x.n);
    Mid m;
    if (!begin(x, q, m)) return false;
#pragma nounroll
    for (int tries = 0;; ++tries) {
        pass_one<FALLING>(x, s, part, q, m);
        if (fits(s, m)) break;
        if (tries || !(m.top < __builtin_inff())) return false;
        m.ref = m.top;  // the sample was too far below
    }
    if constexpr (FALLING) {
#pragma nounroll
        for (bool again = false;; again = true) {
            if (!(again ? between_again(s, true, q, m) : between_falling(x.n, s, inner(a.uniforms[row]), q, m))) return false;
            pass_two_falling(x, s, part, again, q, m);
            const Found found = finish_falling(a, row, x, s, q, m);
            if (found != Found::target) return found == Found::item;
        }
    } else {
        if (!between(x.n, s, q, m)) return false;
        pass_two(x, s, part, q, m);
        return finish(a, row, x, s, part, q, m);
    }
}

template <class T, bool FALLING>
__global__ __launch_bounds__(kThreads, 4) void sample_kernel(Row a) {
    __shared__ Both sh;
    for (uint32_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const Logits<T> x{static_cast<const T*>(a.logits) + row * a.stride, a.V};
        if (!sample_quickly<FALLING>(a, row, x, sh.quick)) {
            __syncthreads();
            sample_slowly<FALLING>(a, row, x, sh.slow);
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------------------
// Much to do: a launch for each pass, few rows' chunks in several workgroups
// ---------------------------------------------------------------------------------------
// The same passes, what they leave joined in memory: counts and lists by whole-number atomics, sums and largest values a
// slot a workgroup, added up in the order of the workgroups.
constexpr uint32_t kSlices = 64;
struct Joined {
    // cleared before the first pass
    uint32_t count[kBins + 4];
    uint32_t tops, listed;
    uint32_t failed;   // set by the first pass alone: the sample holds no value to refer to
    uint32_t dropped;  // set by the second pass and read by the last kernel alone, so that a workgroup's waves see one `failed`
    uint32_t again;    // set by the kernel that ends a row: its draw needs a list of its own
    uint32_t pad[3];
    // written by it and the second
    Mid mid;
    float top[kSlices];
    double all[kSlices], above[kSlices], kept[kSlices];
    double chunk[kMostChunks];
    uint64_t top_list[kTops], list[kListed];
};
constexpr uint32_t kCleared = kBins + 12;  // words
static_assert(offsetof(Joined, mid) == 4 * kCleared, "what lies before it is cleared");

__global__ __launch_bounds__(256) void sample_clear_kernel(Joined* j) {
    uint32_t* const p = reinterpret_cast<uint32_t*>(j + blockIdx.y);
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i < kCleared) p[i] = 0;
}
__device__ __forceinline__ Part slice_of(uint32_t n) {
    Part p = whole_of(n);
    p.from = uint32_t(uint64_t(p.chunks) * blockIdx.x / gridDim.x);
    p.to = uint32_t(uint64_t(p.chunks) * (blockIdx.x + 1) / gridDim.x);
    return p;
}

template <class T, bool FALLING>
__global__ __launch_bounds__(kThreads, 8) void sample_one_kernel(Row a, Joined* joined) {
    __shared__ Brief q;
    __shared__ uint32_t base;
    const uint32_t row = blockIdx.y, tid = threadIdx.x;
    Joined& j = joined[row];
    const Logits<T> x{static_cast<const T*>(a.logits) + row * a.stride, a.V};
    const Settings s = settings_of(a, row);
    const Part part = slice_of(x.n);
    Mid m;
    if (!begin(x, q, m)) {
        if (blockIdx.x == 0 && tid == 0) {
            j.failed = 1;
            j.mid = m;
        }
        return;
    }
    pass_one<FALLING>(x, s, part, q, m);
    if (tid == 0) {
        j.top[blockIdx.x] = m.top;
        j.all[blockIdx.x] = m.all;
        if (blockIdx.x == 0) j.mid = m;
    }
    __syncthreads();
    if (!FALLING && kind_of(s, x.n).sums()) {
        if (s.m == 0.0)
            for (uint32_t i = part.from + tid; i < part.to; i += kThreads) j.chunk[i] = q.chunk[i];
        return;
    }
    for (uint32_t i = tid; i < kBins; i += kThreads)
        if (q.count[i]) atomicAdd(&j.count[i], q.count[i]);
    if (m.tops) {
        if (tid == 0) base = atomicAdd(&j.tops, m.tops);
        __syncthreads();
        for (uint32_t i = tid; i < min(m.tops, kTops); i += kThreads)
            if (base + i < kTops) j.top_list[base + i] = q.list[i];
    }
}

template <class T>
__global__ __launch_bounds__(kThreads, 6) void sample_two_kernel(Row a, Joined* joined) {
    __shared__ Quick q;
    __shared__ uint32_t base;
    const uint32_t row = blockIdx.y, tid = threadIdx.x;
    Joined& j = joined[row];
    if (j.failed) return;
    const Logits<T> x{static_cast<const T*>(a.logits) + row * a.stride, a.V};
    const Settings s = settings_of(a, row);
    const Kind kind = kind_of(s, x.n);
    const Part part = slice_of(x.n);
    Mid m = j.mid;
    m.top = -__builtin_inff();
    m.all = 0.0;
    for (uint32_t i = 0; i < gridDim.x; ++i) {
        m.top = fmaxf(m.top, j.top[i]);
        m.all += j.all[i];
    }
    m.tops = j.tops;
    bool good = fits(s, m);
    if (good) {
        if (!kind.sums()) {
            for (uint32_t i = tid; i < kBins; i += kThreads) q.count[i] = j.count[i];
            __syncthreads();
        }
        good = between(x.n, s, q, m);
    }
    if (!good) {  // (every workgroup of the row finds the same)
        if (blockIdx.x == 0 && tid == 0) j.dropped = 1;
        return;
    }
    pass_two(x, s, part, q, m);
    __syncthreads();
    if (tid == 0) {
        j.above[blockIdx.x] = m.above;
        // (what this kernel's other workgroups read of it, ref and low, is not among the changes but where min-p alone cuts, and there
        // they set ref themselves)
        if (blockIdx.x == 0) {
            j.mid.top = m.top;
            j.mid.all = m.all;
            j.mid.first = m.first;
            j.mid.end = m.end;
            j.mid.least = m.least;
        }
    }
    if (kind.sums()) {
        if (s.m > 0.0)
            for (uint32_t i = part.from + tid; i < part.to; i += kThreads) j.chunk[i] = q.chunk[i];
        return;
    }
    if (m.first < 0 && m.end < 0) return;
    if (m.first >= 0)
        for (uint32_t i = part.from + tid; i < part.to; i += kThreads) j.chunk[i] = q.chunk[i];
    const uint32_t n = q.listed;
    if (n) {
        if (tid == 0) base = atomicAdd(&j.listed, n);
        __syncthreads();
        for (uint32_t i = tid; i < min(n, kListed); i += kThreads)
            if (base + i < kListed) j.list[base + i] = q.list[i];
    }
}

template <class T>
__global__ __launch_bounds__(kThreads, 4) void sample_three_kernel(Row a, Joined* joined, uint32_t slices) {
    __shared__ Both sh;
    Quick& q = sh.quick;
    const uint32_t row = blockIdx.x, tid = threadIdx.x;
    const Joined& j = joined[row];
    const Logits<T> x{static_cast<const T*>(a.logits) + row * a.stride, a.V};
    bool done = false;
    if (!j.failed && !j.dropped) {
        const Settings s = settings_of(a, row);
        const Kind kind = kind_of(s, x.n);
        const Part part = whole_of(x.n);
        Mid m = j.mid;
        if (kind.sums() && s.m > 0.0) m.ref = m.top;
        m.above = 0.0;
        if (!kind.sums()) {
            const bool listed = !(m.first < 0 && m.end < 0);
            if (listed && m.first >= 0)
                for (uint32_t i = 0; i < slices; ++i) m.above += j.above[i];
            const uint32_t n = listed ? j.listed : j.tops;
            if (tid == 0) q.listed = n;
            for (uint32_t i = tid; i < min(n, kListed); i += kThreads) q.list[i] = listed ? j.list[i] : j.top_list[i];
        }
        if (kind.sums() || m.first >= 0)
            for (uint32_t i = tid; i < part.chunks; i += kThreads) q.chunk[i] = j.chunk[i];
        __syncthreads();
        done = finish(a, row, x, s, part, q, m);
    }
    if (!done) {
        __syncthreads();
        sample_slowly<false>(a, row, x, sh.slow);
    }
}

// The second pass and the end of a row along falling logits; again: of the rows whose draw needs a list of its own.
template <class T>
__global__ __launch_bounds__(kThreads, 6) void sample_two_falling_kernel(Row a, Joined* joined, bool again) {
    __shared__ Quick q;
    __shared__ uint32_t base;
    const uint32_t row = blockIdx.y, tid = threadIdx.x;
    Joined& j = joined[row];
    if (again ? !j.again : j.failed) return;
    const Logits<T> x{static_cast<const T*>(a.logits) + row * a.stride, a.V};
    const Settings s = settings_of(a, row);
    const Part part = slice_of(x.n);
    Mid m = j.mid;
    m.top = -__builtin_inff();
    m.all = 0.0;
    for (uint32_t i = 0; i < gridDim.x; ++i) {
        m.top = fmaxf(m.top, j.top[i]);
        m.all += j.all[i];
    }
    m.tops = j.tops;
    bool good = fits(s, m);
    if (good) {
        for (uint32_t i = tid; i < kBins; i += kThreads) q.count[i] = j.count[i];
        __syncthreads();
        good = again ? between_again(s, false, q, m) : between_falling(x.n, s, inner(a.uniforms[row]), q, m);
    }
    if (!good) {  // (every workgroup of the row finds the same)
        if (blockIdx.x == 0 && tid == 0) j.dropped = 1;
        return;
    }
    // (of what this kernel's other workgroups read of `mid` nothing changes: ref and low, and again also least, kept and target)
    if (blockIdx.x == 0 && tid == 0) {
        j.mid.top = m.top;
        j.mid.all = m.all;
        j.mid.first = m.first;
        j.mid.end = m.end;
        if (!again) {
            j.mid.least = m.least;
            j.mid.kept = m.kept;
            j.mid.target = m.target;
            j.mid.whole = m.whole;
        }
    }
    pass_two_falling(x, s, part, again, q, m);
    __syncthreads();
    if (tid == 0) {
        j.above[blockIdx.x] = m.above;
        j.kept[blockIdx.x] = m.kept;
    }
    if (!again && m.first < 0 && m.end == -1) return;
    const uint32_t n = q.listed;
    if (n) {
        if (tid == 0) base = atomicAdd(&j.listed, n);
        __syncthreads();
        for (uint32_t i = tid; i < min(n, kListed); i += kThreads)
            if (base + i < kListed) j.list[base + i] = q.list[i];
    }
}

template <class T>
__global__ __launch_bounds__(kThreads, 4) void sample_three_falling_kernel(Row a, Joined* joined, uint32_t slices, bool again) {
    __shared__ Both sh;
    Quick& q = sh.quick;
    const uint32_t row = blockIdx.x, tid = threadIdx.x;
    Joined& j = joined[row];
    if (again && !j.again) return;
    const Logits<T> x{static_cast<const T*>(a.logits) + row * a.stride, a.V};
    Found found = Found::nothing;
    if (!j.failed && !j.dropped) {
        const Settings s = settings_of(a, row);
        Mid m = j.mid;
        m.above = 0.0;
        if (m.first >= 0)
            for (uint32_t i = 0; i < slices; ++i) m.above += j.above[i];
        if (m.target < 0.0) {
            m.kept = 0.0;
            if (m.first >= 0 || m.end == kNoList)
                for (uint32_t i = 0; i < slices; ++i) m.kept += j.kept[i];
        }
        const bool listed = again || m.first >= 0 || m.end != -1;
        const uint32_t n = listed ? j.listed : j.tops;
        for (uint32_t i = tid; i < min(n, kListed); i += kThreads) q.list[i] = listed ? j.list[i] : j.top_list[i];
        if (tid == 0) q.listed = n;
        __syncthreads();
        found = finish_falling(a, row, x, s, q, m);
        if (found == Found::target) {
            __syncthreads();
            if (tid == 0) {
                j.mid.kept = m.kept;
                j.mid.target = m.target;
                j.listed = 0;
                j.again = 1;
            }
        }
    }
    if (found == Found::nothing) {
        __syncthreads();
        sample_slowly<true>(a, row, x, sh.slow);
    }
}

// Rows that are drawn from whole: after the first pass a wave each, eight a workgroup, which takes those together that the quick way does
// not.
template <class T>
__global__ __launch_bounds__(kThreads, 4) void sample_whole_kernel(Row a, Joined* joined, uint32_t slices) {
    __shared__ Shared slow;
    __shared__ uint32_t left[kWaves];
    const uint32_t wave = threadIdx.x >> 6, row = blockIdx.x * kWaves + wave;
    uint32_t mine = 0;
    if (row < a.rows) {
        const Joined& j = joined[row];
        const Logits<T> x{static_cast<const T*>(a.logits) + row * a.stride, a.V};
        const Settings s = settings_of(a, row);
        Mid m = j.mid;
        m.tops = 0;
        for (uint32_t i = 0; i < slices; ++i) m.top = i ? fmaxf(m.top, j.top[i]) : j.top[i];
        if (fabsf(m.ref) < __builtin_inff() && fits(s, m)) draw(a, row, x, whole_of(x.n), kLowest, x.n - 1, m.ref, s.c, j.chunk);
        else mine = 1;
    }
    if ((threadIdx.x & 63) == 0) left[wave] = mine;
    __syncthreads();
    for (uint32_t i = 0; i < uint32_t(kWaves); ++i)
        if (left[i]) {
            const uint32_t r = blockIdx.x * kWaves + i;
            sample_slowly<false>(a, r, Logits<T>{static_cast<const T*>(a.logits) + r * a.stride, a.V}, slow);
            __syncthreads();
        }
}

// The workgroups that a row is divided among; 0: the row's passes are one launch.  That costs less where rows are short (one of 8000
// values, p 0.9: 29, not 36 us; of 40,000: 53, not 39).  Many rows that are not cut gain from more waves on a CU than all passes in
// one have room for (512 x 8000: 22, not 16 us); others do not (35, not 42).
uint32_t slices_of(const va_context* ctx, uint32_t rows, uint32_t V, bool whole) {
    if (V < 24576 && !(whole && rows >= 128 && V > kWaves * kStep)) return 0;
    return std::max(std::min(std::min(2u * uint32_t(ctx->num_cus) / rows, V / (kWaves * kStep)), kSlices), 1u);
}
constexpr uint32_t kBatch = 1024;  // rows that share a launch, and a workspace

template <class T, bool FALLING>
va_status run(va_context* ctx, const Row& all, bool whole, Joined* joined, uint32_t slices) {
    if (!slices) {
        sample_kernel<T, FALLING><<<dim3(std::min<uint32_t>(all.rows, 1u << 20)), dim3(kThreads), 0, ctx->stream>>>(all);
        VA_CHECK_LAUNCH(ctx);
        return VA_OK;
    }
    for (uint32_t r = 0; r < all.rows; r += kBatch) {
        Row a = all;
        a.rows = std::min(all.rows - r, kBatch);
        a.logits = static_cast<const T*>(all.logits) + r * all.stride;
        a.uniforms += r, a.items += r;
        if (a.log_probability) a.log_probability += r;
        if (a.temperatures) a.temperatures += r;
        if (a.top_ps) a.top_ps += r;
        if (a.min_ps) a.min_ps += r;
        if (a.top_ks) a.top_ks += r;
        if (whole && !FALLING) {
            sample_one_kernel<T, false><<<dim3(slices, a.rows), dim3(kThreads), 0, ctx->stream>>>(a, joined);
            VA_CHECK_LAUNCH(ctx);
            sample_whole_kernel<T><<<dim3(ceil_div(a.rows, kWaves)), dim3(kThreads), 0, ctx->stream>>>(a, joined, slices);
            VA_CHECK_LAUNCH(ctx);
            continue;
        }
        sample_clear_kernel<<<dim3((kCleared + 255) / 256, a.rows), dim3(256), 0, ctx->stream>>>(joined);
        VA_CHECK_LAUNCH(ctx);
        sample_one_kernel<T, FALLING><<<dim3(slices, a.rows), dim3(kThreads), 0, ctx->stream>>>(a, joined);
        VA_CHECK_LAUNCH(ctx);
        if constexpr (FALLING) {
            // (top-k's list holds the item, and of whole rows the first list does)
            const bool by_count = !a.top_ks && ((a.top_k > 0 && a.top_k < a.V) || (!a.temperatures && a.temperature == 0.0f));
            for (int again = 0; again < (whole || by_count ? 1 : 2); ++again) {
                sample_two_falling_kernel<T><<<dim3(slices, a.rows), dim3(kThreads), 0, ctx->stream>>>(a, joined, again != 0);
                VA_CHECK_LAUNCH(ctx);
                sample_three_falling_kernel<T><<<dim3(a.rows), dim3(kThreads), 0, ctx->stream>>>(a, joined, slices, again != 0);
                VA_CHECK_LAUNCH(ctx);
            }
            continue;
        }
        sample_two_kernel<T><<<dim3(slices, a.rows), dim3(kThreads), 0, ctx->stream>>>(a, joined);
        VA_CHECK_LAUNCH(ctx);
        sample_three_kernel<T><<<dim3(a.rows), dim3(kThreads), 0, ctx->stream>>>(a, joined, slices);
        VA_CHECK_LAUNCH(ctx);
    }
    return VA_OK;
}

}  // namespace
}  // namespace va

using namespace va;

extern "C" {

va_status va_sample(va_context* ctx, const va_sample_desc* d, int64_t* out_items, float* out_log_probability) {
    return va_sample_in_order(ctx, d, VA_SAMPLE_BY_ITEM, out_items, out_log_probability);
}

va_status va_sample_in_order(va_context* ctx, const va_sample_desc* d, va_sample_order order, int64_t* out_items, float* out_log_probability) {
    if (!ctx) return VA_ERR_INVALID_ARG;
    VA_REQUIRE(ctx, d, "va_sample: NULL description");
    VA_REQUIRE(ctx, d->dtype == VA_DTYPE_F32 || d->dtype == VA_DTYPE_F16 || d->dtype == VA_DTYPE_BF16, "va_sample: unknown type %d", int(d->dtype));
    VA_REQUIRE(ctx, d->num_items >= 1 && d->num_items < 0x80000000u, "va_sample: %u items (1 to 2^31 - 1)", d->num_items);
    VA_REQUIRE(ctx, d->temperatures || (std::isfinite(d->temperature) && d->temperature >= 0.0f), "va_sample: the temperature must be finite and not negative");
    VA_REQUIRE(ctx, d->top_ks || d->top_k >= 0, "va_sample: top_k must not be negative");
    VA_REQUIRE(ctx, d->top_ps || (d->top_p > 0.0f && d->top_p <= 1.0f), "va_sample: top_p must lie in (0, 1]");
    VA_REQUIRE(ctx, order == VA_SAMPLE_BY_ITEM || order == VA_SAMPLE_BY_LOGIT, "va_sample_in_order: unknown order %d", int(order));
    VA_REQUIRE(ctx, d->min_ps || (d->min_p >= 0.0f && d->min_p <= 1.0f), "va_sample: min_p must lie in [0, 1]");
    if (!d->rows) return VA_OK;
    VA_REQUIRE(ctx, d->logits && d->uniforms && out_items, "va_sample: NULL pointer");
    const uintptr_t es = d->dtype == VA_DTYPE_F32 ? 4 : 2;
    VA_REQUIRE(ctx, reinterpret_cast<uintptr_t>(d->logits) % es == 0 && reinterpret_cast<uintptr_t>(out_items) % 8 == 0, "va_sample: a pointer is not aligned to its type");
    VA_REQUIRE(ctx, d->rows == 1 || (d->stride >= d->num_items && d->stride < 1ull << 40), "va_sample: a stride of %llu for rows of %u", (unsigned long long)d->stride,
               d->num_items);
    DeviceGuard guard(ctx->device);
    Row a;
    a.logits = d->logits, a.stride = stride_of(d->rows, d->stride, d->num_items), a.uniforms = d->uniforms;
    a.temperatures = d->temperatures, a.top_ps = d->top_ps, a.min_ps = d->min_ps, a.top_ks = d->top_ks;
    a.temperature = d->temperature, a.top_p = d->top_p, a.min_p = d->min_p, a.top_k = uint32_t(d->top_k);
    a.items = out_items, a.log_probability = out_log_probability, a.rows = d->rows, a.V = d->num_items;
    const bool falling = order == VA_SAMPLE_BY_LOGIT;
    // no row is cut, as the host can tell
    const bool whole = !a.temperatures && !a.top_ps && !a.min_ps && !a.top_ks && a.temperature > 0.0f && a.top_p >= 1.0f && a.min_p == 0.0f && (a.top_k == 0 || a.top_k >= a.V);
    uint32_t slices = slices_of(ctx, d->rows, d->num_items, whole && !falling);
    Joined* joined = nullptr;
    if (slices) {
        const uint64_t need = uint64_t(std::min(d->rows, kBatch)) * sizeof(Joined);
        if (d->workspace) {
            VA_REQUIRE(ctx, d->workspace_bytes >= need && reinterpret_cast<uintptr_t>(d->workspace) % 16 == 0, "va_sample: a workspace of %llu bytes, at a multiple of 16, is needed",
                       (unsigned long long)need);
            joined = static_cast<Joined*>(d->workspace);
        } else {
            // a captured call must not keep the arena, which may be replaced: without a workspace of its own it is one launch
            hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
            VA_CHECK_HIP(ctx, hipStreamIsCapturing(ctx->stream, &capture));
            if (capture != hipStreamCaptureStatusNone) {
                slices = 0;
            } else {
                Scratch sc(ctx);
                VA_CHECK_STATUS(sc.reserve(Scratch::round(need)));
                joined = sc.carve<Joined>(std::min(d->rows, kBatch));
            }
        }
    }
    const auto go = [&](auto t) {
        using T = decltype(t);
        return falling ? run<T, true>(ctx, a, whole, joined, slices) : run<T, false>(ctx, a, whole, joined, slices);
    };
    if (d->dtype == VA_DTYPE_F32) return go(0.0f);
    if (d->dtype == VA_DTYPE_F16) return go(_Float16(0));
    return go(__bf16(0));
}

uint64_t va_sample_workspace(va_context* ctx, uint32_t rows, uint32_t num_items) {
    if (!ctx || !rows) return 0;
    return slices_of(ctx, rows, num_items, true) ? uint64_t(std::min(rows, kBatch)) * sizeof(Joined) : 0;
}

}  // extern "C"
