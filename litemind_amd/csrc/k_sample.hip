// k_sample.hip -- the next token of a row of logits from temperature, top-k,
// top-p, min-p and one given random number (litemind_serving.h, lm_sample).
//
//   e_i = exp((x_i - max) / temperature), as whole numbers of 2^-bits: sums of
//   them are exact in any order, so are the cuts, and the token does not depend
//   on how the row was shared out.  bits = 46 for up to 2^17 tokens (their sum
//   stays under 2^63), one less per doubling past that: an e is off by at most
//   half a unit, 7e-15 of the largest.
//
// The kept tokens are a prefix of the order (logit down, index up), found
// without a sort.  A sweep counts the row, or adds up its e, by 2048 equal
// stretches of the logits' range; the stretch in which the k-th token lies, or
// top-p is reached, is listed in LDS and searched by the bits of its logits.
// The kept tokens' e are then added up by stretches of the row's indices, and the
// stretch that the random number falls into is cut up again until one is left.
//
// A row is a workgroup's; its sweeps after the first come from the caches. What
// they cost is the e: 11 steps of 64-bit arithmetic and as many others, 22 us for
// 102400 on one CU. By temperature alone a row has one such sweep (35 us by
// itself, 256 rows 49 us), by top-k none (29 us), by top-p two (78 us); a greedy row
// takes 12. Sharing a row among workgroups, a kernel for each sweep, was no faster:
// 40 us for top-k and 76 for 32 rows of any settings, where this takes 70.
#include "serve_internal.h"

#include <algorithm>

namespace lm {
namespace {

constexpr int kThreads = 1024;
constexpr int64_t kMostRows = int64_t{1} << 21;
constexpr int kWaves = kThreads / 64;
constexpr int kBins = 2048;  // two a thread where they are added up
constexpr int kTable = 1024;
constexpr int kList = 4096;
constexpr float kMost = 3.4028234663852886e38f;
constexpr uint64_t kRaw = 0x4330000000000000ull;  // the bits of 2^52
constexpr int kSpan = 256;  // what a wave loads at once

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));  // rows of any alignment

// 2^(j / 1024) for 0 <= j < 1024: the root of it over 2^(1/2) by the power series
// of exp to the 11th power (|f| <= 0.17: f^12 / 12! = 2e-18), squared.
__device__ inline double exp2_entry(int j) {
    const double f = (j - kTable / 2) * (0.693147180559945309417 / (2 * kTable));
    double p = 1.0 / 39916800.0;
    p = __builtin_fma(p, f, 1.0 / 3628800.0);
    p = __builtin_fma(p, f, 1.0 / 362880.0);
    p = __builtin_fma(p, f, 1.0 / 40320.0);
    p = __builtin_fma(p, f, 1.0 / 5040.0);
    p = __builtin_fma(p, f, 1.0 / 720.0);
    p = __builtin_fma(p, f, 1.0 / 120.0);
    p = __builtin_fma(p, f, 1.0 / 24.0);
    p = __builtin_fma(p, f, 1.0 / 6.0);
    p = __builtin_fma(p, f, 0.5);
    p = __builtin_fma(p, f, 1.0);
    p = __builtin_fma(p, f, 1.0);
    return j == 0 ? 1.0 : p * p * 1.41421356237309504880;
}

// Whole numbers in the order of the floats; NaN below -infinity.
__device__ inline uint32_t order_key(float x) {
    if (x != x) {
        return 0;
    }
    const uint32_t b = __float_as_uint(x + 0.0f);  // -0 as +0
    return (b & 0x80000000u) != 0 ? ~b : b | 0x80000000u;
}
__device__ inline float key_float(uint32_t k) { return __uint_as_float((k & 0x80000000u) != 0 ? k & 0x7fffffffu : ~k); }
constexpr uint32_t kKeyMinusInf = 0x007fffffu;

struct Shared {
    double table[kTable];  // 2^(bits + j / 1024)
    uint64_t bins[kBins];
    uint32_t list_key[kList];
    int32_t list_at[kList];
    uint64_t part[kWaves];
    uint64_t found[3];
    uint32_t key_part[kWaves], key_part2[kWaves];
    int32_t at_part[kWaves];
    uint32_t listed;
};

template <class T, class F>
__device__ inline T wave_reduce(T v, F f) {
    for (int o = 32; o >= 1; o >>= 1) {
        v = f(v, __shfl_xor(v, o));
    }
    return v;
}
template <class T, class F>
__device__ inline T block_reduce(T v, T* part, F f) {
    v = wave_reduce(v, f);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
        part[threadIdx.x >> 6] = v;
    }
    __syncthreads();
    v = part[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) {
        v = f(v, part[w]);
    }
    return v;
}
struct Add {
    __device__ uint64_t operator()(uint64_t a, uint64_t b) const { return a + b; }
};
// The exclusive prefix of v over the wave's lanes.
__device__ inline uint64_t wave_before(uint64_t v) {
    uint64_t sum = v;
    for (int o = 1; o < 64; o <<= 1) {
        const uint64_t up = __shfl_up(sum, o);
        sum += (threadIdx.x & 63) >= static_cast<unsigned>(o) ? up : 0;
    }
    return sum - v;
}

// What a row's sweeps share.
struct Row {
    const float* x;
    int32_t n;
    double top, rate;  // largest logit, 1024 log2(e) / temperature
    float top_f, scale, offset;  // stretches per logit, and where the largest lies
    uint64_t one;      // e = 1
    bool top_inf;
    const double* table;  // in LDS

    // e in units, to the nearest, as the bits of e + 2^52: t = 1024 log2 e = j + f with
    // |f| <= 1/2; 2^(f / 1024) by its power series (cut off at 6e-16), 2^(j / 1024) from
    // the table and the exponent. Under 2^-64, and for NaN, it is 2^52.
    __device__ __forceinline__ uint64_t raw(float v) const {
        constexpr double kC1 = 0.693147180559945309417 / kTable, kC2 = kC1 * kC1 / 2, kC3 = kC1 * kC1 * kC1 / 6;
        const double t = fmax((static_cast<double>(v) - top) * rate, -64.0 * kTable);
        const double z = t + 0x1.8p52;
        const double f = t - (z - 0x1.8p52);
        const int32_t j = static_cast<int32_t>(__double_as_longlong(z));
        const double p = f * __builtin_fma(f, __builtin_fma(f, kC3, kC2), kC1);
        const int64_t whole = __double_as_longlong(table[j & (kTable - 1)]) + (static_cast<int64_t>(j >> 10) << 52);
        const double e = __longlong_as_double(whole);
        return static_cast<uint64_t>(__double_as_longlong(__builtin_fma(e, p, e) + 0x1p52));
    }
    __device__ __forceinline__ uint64_t units(float v) const {
        if (top_inf) {
            return v == __builtin_inff() ? one : 0;
        }
        return raw(v) - kRaw;
    }
    __device__ __forceinline__ void units(f32x4 v, uint64_t* w) const {
        if (top_inf) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                w[j] = v[j] == __builtin_inff() ? one : 0;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                w[j] = raw(v[j]) - kRaw;
            }
        }
    }
    // The stretch of the range, kBins - 1 at the largest: one rounding and a cut, so
    // that a larger logit is never in a lower one, whatever the range.
    __device__ int bin(float v) const {
        return static_cast<int>(__builtin_amdgcn_fmed3f(__builtin_fmaf(v, scale, offset), 0.0f, static_cast<float>(kBins - 1)));
    }
    // A logit that no logit of the stretch lies under, and one that none lies over: a
    // stretch more, and two steps for the roundings.
    __device__ float under(int stretch) const {
        return near((static_cast<float>(stretch) - 1.0f - offset) / scale, -1, stretch == 0);
    }
    __device__ float over(int stretch) const { return near((static_cast<float>(stretch) + 2.0f - offset) / scale, 1, false); }
    __device__ static float near(float v, int way, bool all) {
        if (all || !(v > -kMost && v < kMost)) {
            return way < 0 ? -kMost : kMost;
        }
        return key_float(order_key(v) + 2 * way);
    }
};

// f(index, four logits) for the wave's share [from, to) of a row: whole spans but
// at the row's end, past which the logits are NaN.
__device__ __forceinline__ f32x4 load4(const Row& r, int32_t first, int32_t i) {
    f32x4 v = __builtin_nanf("");
    if (first + kSpan <= r.n) {
        v = *reinterpret_cast<const f32x4_any*>(r.x + i);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (i + j < r.n) {
                v[j] = r.x[i + j];
            }
        }
    }
    return v;
}
template <class F>
__device__ __forceinline__ void sweep(const Row& r, int32_t from, int32_t to, F f) {
    const int lane = threadIdx.x & 63;
    from = __builtin_amdgcn_readfirstlane(from);
    to = __builtin_amdgcn_readfirstlane(to);
#pragma unroll 1
    for (int32_t base = from; base < to; base += 4 * kSpan) {
        f32x4 v[4];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int32_t first = base + g * kSpan;
            if (first < to) {
                v[g] = load4(r, first, first + 4 * lane);
            }
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int32_t first = base + g * kSpan;
            if (first < to) {
                f(first + 4 * lane, v[g]);
            }
        }
    }
}
// The wave's share of [from, to), whole spans.
__device__ inline int32_t share_of(int32_t from, int32_t to) {
    return ((to - from + kWaves - 1) / kWaves + kSpan - 1) / kSpan * kSpan;
}
template <class F>
__device__ __forceinline__ void sweep_row(const Row& r, F f) {
    const int32_t share = share_of(0, r.n), from = static_cast<int32_t>(threadIdx.x >> 6) * share;
    sweep(r, from, min(from + share, r.n), f);
}

// The bin, from the highest down, at which the bins' sum reaches want.
struct Found {
    int bin;
    uint64_t above, own;  // the sums of the bins above it and of itself
};
__device__ inline Found find_bin(Shared& sh, uint64_t want) {
    __syncthreads();
    const int b = kBins - 1 - 2 * static_cast<int>(threadIdx.x);
    const uint64_t hi = sh.bins[b], lo = sh.bins[b - 1], own = hi + lo;
    uint64_t ahead = wave_before(own);
    if ((threadIdx.x & 63) == 63) {
        sh.part[threadIdx.x >> 6] = ahead + own;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        ahead += w < static_cast<int>(threadIdx.x >> 6) ? sh.part[w] : 0;
    }
    if (ahead < want && ahead + own >= want) {
        const bool second = ahead + hi < want;
        sh.found[0] = static_cast<uint64_t>(second ? b - 1 : b);
        sh.found[1] = second ? ahead + hi : ahead;
        sh.found[2] = second ? lo : hi;
    }
    __syncthreads();
    return Found{static_cast<int>(sh.found[0]), sh.found[1], sh.found[2]};
}
__device__ inline void clear_bins(Shared& sh) {
    __syncthreads();
    sh.bins[threadIdx.x] = sh.bins[threadIdx.x + kThreads] = 0;
    __syncthreads();
}
__device__ inline void add_bin(Shared& sh, int b, uint64_t w) {
    atomicAdd(reinterpret_cast<unsigned long long*>(&sh.bins[b]), static_cast<unsigned long long>(w));
}

// The key at which the weight of the keys from the highest down reaches want, by
// eleven bits at a time; each(f) calls f(key, weight) for all, lo and hi are bounds
// of the keys.
struct Selected {
    uint32_t key;
    uint64_t above, own;  // the weights of the keys above it and of itself
};
template <class Each>
__device__ __forceinline__ Selected select(Shared& sh, uint32_t lo, uint32_t hi, uint64_t want, Each each) {
    int bits = max(32 - __clz(static_cast<int>(lo ^ hi)), 1);
    Selected s{bits == 32 ? 0 : hi >> bits << bits, 0, 0};
#pragma unroll 1
    while (bits > 0) {
        const int shift = max(bits - 11, 0);
        clear_bins(sh);
        each([&](uint32_t key, uint64_t weight) {
            if (static_cast<uint64_t>(key ^ s.key) >> bits == 0) {
                add_bin(sh, static_cast<int>((key ^ s.key) >> shift), weight);
            }
        });
        const Found f = find_bin(sh, want - s.above);
        s.key |= static_cast<uint32_t>(f.bin) << shift;
        s.above += f.above;
        s.own = f.own;
        bits = shift;
    }
    return s;
}

// The first index up to which the weights add up to more than target, of
// weights that do in the end.  weigh(index, four logits, four weights) gives them.
struct Located {
    int32_t at;
    uint64_t weight;
};
template <class Weigh, class Target>
__device__ __forceinline__ Located locate(Shared& sh, const Row& r, Weigh weigh, Target target_of) {
    const int wave = threadIdx.x >> 6;
    int32_t from = 0, to = r.n;
    uint64_t target = 0;
    bool first = true;
    while (first || to - from > kSpan) {
        const int32_t share = share_of(from, to), mine = from + wave * share;
        uint64_t sum = 0;
        sweep(r, min(mine, to), min(mine + share, to), [&](int32_t i, f32x4 v) {
            uint64_t w[4];
            weigh(i, v, w);
            sum += w[0] + w[1] + w[2] + w[3];
        });
        sum = wave_reduce(sum, Add());
        __syncthreads();
        if ((threadIdx.x & 63) == 0) {
            sh.part[wave] = sum;
        }
        __syncthreads();
        if (first) {
            uint64_t total = 0;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                total += sh.part[w];
            }
            target = target_of(total);
            first = false;
        }
        int w = 0;
        while (w < kWaves - 1 && target >= sh.part[w]) {
            target -= sh.part[w];
            ++w;
        }
        from = min(from + w * share, to);
        to = min(from + share, to);
    }
    __syncthreads();
    if (wave == 0) {
        const int32_t i = from + 4 * static_cast<int32_t>(threadIdx.x);
        uint64_t w[4];
        weigh(i, load4(r, from, i), w);
        const uint64_t own = w[0] + w[1] + w[2] + w[3];
        uint64_t before = wave_before(own);
        if (target >= before && target - before < own) {
            int at = 0;
            uint64_t weight = w[0];
#pragma unroll
            for (int j = 0; j < 3; ++j) {
                if (at == j && target - before >= w[j]) {
                    before += w[j];
                    at = j + 1;
                    weight = w[j + 1];
                }
            }
            sh.found[0] = static_cast<uint64_t>(i + at);
            sh.found[1] = weight;
        }
    }
    __syncthreads();
    return Located{static_cast<int32_t>(sh.found[0]), sh.found[1]};
}

// A prefix of the order: keys above `key`, and of those equal to it the ones up
// to index `last`.
struct Cut {
    uint32_t key;
    int32_t last;
    __device__ bool keeps(uint32_t k, int32_t i) const { return k > key || (k == key && i <= last); }
};

__global__ __launch_bounds__(kThreads) void sample_kernel(const SampleArgs a, int64_t row0, int bits) {
    __shared__ Shared sh;
    const int64_t row = row0 + blockIdx.x;
    const lm_sampling set = a.settings[row];
    Row r;
    r.x = a.logits + row * a.stride;
    r.n = static_cast<int32_t>(a.vocab);
    r.table = sh.table;
    r.one = 1ull << bits;
    sh.table[threadIdx.x] = __builtin_ldexp(exp2_entry(threadIdx.x), bits);
    // the largest logit and the least; -infinity, where there is one, and NaN are not
    // told from each other
    float own = -__builtin_inff(), least = __builtin_inff();
    sweep_row(r, [&](int32_t, f32x4 v) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            own = v[j] > own ? v[j] : own;
            least = v[j] < least ? v[j] : least;
        }
    });
    auto larger = [](uint32_t x, uint32_t y) { return max(x, y); };
    auto smaller = [](uint32_t x, uint32_t y) { return min(x, y); };
    const uint32_t best = block_reduce(order_key(own), sh.key_part, larger);
    least = key_float(block_reduce(order_key(least), sh.key_part2, smaller));
    const float top = key_float(best);
    if (best <= kKeyMinusInf || !(set.temperature > 0.0f) || set.min_p > 1.0f) {
        int32_t at = 0x7fffffff;
        if (best > kKeyMinusInf) {
            sweep_row(r, [&](int32_t i, f32x4 v) {
                if (v[0] == top || v[1] == top || v[2] == top || v[3] == top) {
                    at = min(at, i + (v[0] == top ? 0 : v[1] == top ? 1 : v[2] == top ? 2 : 3));
                }
            });
            at = block_reduce(at, sh.at_part, [](int32_t x, int32_t y) { return min(x, y); });
        }
        if (threadIdx.x == 0) {
            a.token[row] = best <= kKeyMinusInf ? -1 : at;
            if (a.probability != nullptr) {
                a.probability[row] = best <= kKeyMinusInf ? 0.0f : 1.0f;
            }
        }
        return;
    }
    const double temperature = static_cast<double>(set.temperature);
    r.top = static_cast<double>(top);
    r.top_f = top;
    r.top_inf = top == __builtin_inff();
    r.rate = kTable * 1.4426950408889634074 / temperature;
    // Logits that lie 48 powers of two under the largest weigh nothing. Up to there,
    // or to the least one, the range is cut into stretches kBins - 1 .. 1; what lies
    // further below is in stretch 0.
    r.scale = static_cast<float>(48 * 0.6931471805599453 * temperature);
    r.scale = (kBins - 2) / (least > -__builtin_inff() ? fminf(r.scale, top - least) : r.scale);
    r.scale = fminf(r.scale, 1e30f / fmaxf(fabsf(r.top_inf ? 0.0f : top), 1.0f));
    if (r.top_inf) {
        // (temperatures past 1e37 leave no scale, and infinity times 0 is in no stretch)
        r.scale = fmaxf(r.scale, 1e-30f);
    }
    r.offset = static_cast<float>(kBins) - 0.5f - (r.top_inf ? 0.0f : top) * r.scale;

    Cut cut{kKeyMinusInf + 1, 0x7fffffff};
    // Lists the kept ones of a stretch, or of it and those above it; false: too many.
    auto gather = [&](int stretch, bool upwards) __attribute__((always_inline)) {
        const float loose = r.under(stretch);
        __syncthreads();
        if (threadIdx.x == 0) {
            sh.listed = 0;
        }
        __syncthreads();
        sweep_row(r, [&](int32_t i, f32x4 v) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (v[j] >= loose) {
                    const int b = r.bin(v[j]);
                    const uint32_t key = order_key(v[j]);
                    if ((b == stretch || (upwards && b > stretch)) && cut.keeps(key, i + j)) {
                        const uint32_t at = atomicAdd(&sh.listed, 1u);
                        if (at < kList) {
                            sh.list_key[at] = key;
                            sh.list_at[at] = i + j;
                        }
                    }
                }
            }
        });
        __syncthreads();
        return sh.listed <= kList;
    };
    auto listed_share = [&](auto f) {
#pragma unroll 1
        for (uint32_t t = threadIdx.x; t < sh.listed; t += kThreads) {
            f(sh.list_key[t], sh.list_at[t]);
        }
    };
    // The list holds all that the cut keeps. For a short row that is any cut; for
    // top-k of fewer than there are threads, each thread's largest logit bounds the
    // k-th largest from below (a row of 102400 by itself, with the token drawn from the
    // list: 29 us, and 68 by counts over the whole row).
    bool whole = r.n <= kList && (set.top_k > 0 || set.top_p < 1.0f);
    if (whole) {
        gather(0, true);
    } else if (set.top_k > 0 && set.top_k <= kThreads) {
        clear_bins(sh);
        if (own > -__builtin_inff()) {
            add_bin(sh, r.bin(own), 1);
        }
        if (__syncthreads_count(own > -__builtin_inff()) >= set.top_k) {
            whole = gather(find_bin(sh, static_cast<uint64_t>(set.top_k)).bin, true);
        }
    }
    // The cut of top-k by counts, then that of top-p by sums of e within it.
#pragma unroll 1
    for (int step = 0; step < 2; ++step) {
        const bool mass = step == 1;
        if (mass ? !(set.top_p < 1.0f) : set.top_k <= 0 || set.top_k >= r.n) {
            continue;
        }
        auto weight = [&](float v) { return mass ? r.units(v) : uint64_t{1}; };
        uint64_t total = 0, above = 0;  // (total: this thread's share of it)
        int stretch = 0;
        if (whole) {
            listed_share([&](uint32_t key, int32_t i) { total += cut.keeps(key, i) ? weight(key_float(key)) : 0; });
        } else {
            clear_bins(sh);
            const float least_f = key_float(cut.key);
            sweep_row(r, [&](int32_t i, f32x4 v) {
                uint64_t w[4] = {1, 1, 1, 1};
                if (mass) {
                    r.units(v, w);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (v[j] > least_f || (v[j] == least_f && i + j <= cut.last)) {
                        add_bin(sh, r.bin(v[j]), w[j]);
                    }
                }
            });
            __syncthreads();
            total = sh.bins[threadIdx.x] + sh.bins[threadIdx.x + kThreads];
        }
        total = block_reduce(total, sh.part, Add());
        // a token is kept while the e before it are under top_p of the total
        const uint64_t want =
            mass ? max(static_cast<uint64_t>(__builtin_ceil(fmax(static_cast<double>(set.top_p), 0.0) * static_cast<double>(total))), uint64_t{1})
                 : static_cast<uint64_t>(set.top_k);
        if (want > total) {
            continue;
        }
        bool listed = true;
        if (!whole) {
            const Found f = find_bin(sh, want);
            if (f.bin == 0 && !mass && r.over(0) < top && r.units(r.over(0)) == 0) {
                continue;  // a cut among those that weigh nothing
            }
            stretch = f.bin;
            // Of 4096 logits in or above it thrown at 1024 threads, 19 threads would get
            // none; with fewer such threads the list would not hold them (32 rows by
            // themselves: 86 us, and 110 where it was always tried).
            const bool reaches = own > -__builtin_inff() && r.bin(own) >= stretch;
            whole = __syncthreads_count(reaches) <= kThreads - 19 && gather(stretch, true);
            if (!whole) {
                above = f.above;
                listed = gather(stretch, false);
            }
        }
        uint32_t lo = 0xffffffffu, hi = 0;
        if (listed) {
            listed_share([&](uint32_t key, int32_t) {
                lo = min(lo, key);
                hi = max(hi, key);
            });
        }
        // a stretch of too many is read from the row again
        lo = listed ? block_reduce(lo, sh.key_part, smaller) : cut.key;
        hi = listed ? block_reduce(hi, sh.key_part2, larger) : best;
        // the key at the cut, then, where only some of it are kept, the last one's index
        uint64_t goal = want - above;
        uint32_t key = 0;
#pragma unroll 1
        for (bool by_index = false;; by_index = true) {
            const Selected s = select(sh, lo, hi, goal, [&](auto add) {
                auto one = [&](uint32_t k, int32_t i) {
                    if (cut.keeps(k, i) && (!by_index || k == key)) {
                        add(by_index ? ~static_cast<uint32_t>(i) : k, by_index ? uint64_t{1} : weight(key_float(k)));
                    }
                };
                const int32_t many = listed ? static_cast<int32_t>(sh.listed) : r.n;
#pragma unroll 1
                for (int32_t t = threadIdx.x; t < many; t += kThreads) {
                    if (listed) {
                        one(sh.list_key[t], sh.list_at[t]);
                    } else if (r.x[t] > -__builtin_inff() && r.bin(r.x[t]) == stretch) {
                        one(order_key(r.x[t]), t);
                    }
                }
            });
            if (by_index) {
                cut = Cut{key, static_cast<int32_t>(~s.key)};
                break;
            }
            key = s.key;
            const uint64_t unit = weight(key_float(key)), equal = (goal - s.above + unit - 1) / unit;
            if (equal * unit >= s.own) {
                cut = Cut{key, key > cut.key ? 0x7fffffff : cut.last};
                break;
            }
            goal = equal;
            lo = ~static_cast<uint32_t>(r.n);
            hi = ~0u;
        }
    }
    if (set.min_p > 0.0f) {
        // the lowest key whose e is at least min_p, between one whose is not and
        // the largest's, by as many probes as there are threads; close to where the
        // logarithm has it, if that is borne out
        auto kept = [&](double x) { return exp((x - r.top) / temperature) >= static_cast<double>(set.min_p); };
        uint32_t under = kKeyMinusInf, least_kept = best;
        const double guess = r.top + temperature * log(static_cast<double>(set.min_p));
        const double room = 1e-13 * (fabs(r.top) + fabs(guess));
        const float below = static_cast<float>(guess - room), above = static_cast<float>(guess + room);
        if (!r.top_inf && below > -kMost && above < top) {
            const uint32_t low = order_key(below) - 1, high = order_key(above) + 1;
            if (!kept(static_cast<double>(key_float(low))) && kept(static_cast<double>(key_float(high)))) {
                under = low;
                least_kept = high;
            }
        }
#pragma unroll 1
        while (!r.top_inf && least_kept - under > 1) {
            const uint32_t step = (least_kept - under + kThreads - 1) / kThreads;
            const uint64_t probe = under + static_cast<uint64_t>(threadIdx.x + 1) * step;
            const double x = static_cast<double>(key_float(static_cast<uint32_t>(min(probe, static_cast<uint64_t>(least_kept)))));
            const int fewer = __syncthreads_count(probe < least_kept && !kept(x));
            under += static_cast<uint32_t>(fewer) * step;
            least_kept = static_cast<uint32_t>(min(under + static_cast<uint64_t>(step), static_cast<uint64_t>(least_kept)));
        }
        if (least_kept > cut.key) {
            cut = Cut{least_kept, 0x7fffffff};
            whole = whole || gather(r.bin(key_float(least_kept)), true);
        }
    }
    // running > u total: over the whole number below it
    auto target_of = [&](uint64_t total) {
        const float u = a.uniform[row];
        return min(static_cast<uint64_t>((u > 0.0f ? static_cast<double>(u) : 0.0) * static_cast<double>(total)), total - 1);
    };
    Located drawn;
    uint64_t total = 0;
    if (whole) {
        listed_share([&](uint32_t key, int32_t i) { total += cut.keeps(key, i) ? r.units(key_float(key)) : 0; });
        total = block_reduce(total, sh.part, Add());
        const Selected s = select(sh, ~static_cast<uint32_t>(r.n), ~0u, target_of(total) + 1, [&](auto add) {
            listed_share([&](uint32_t key, int32_t i) {
                if (cut.keeps(key, i)) {
                    add(~static_cast<uint32_t>(i), r.units(key_float(key)));
                }
            });
        });
        drawn = Located{static_cast<int32_t>(~s.key), s.own};
    } else {
        const float least_f = key_float(cut.key), next_f = key_float(cut.key + 1);
        drawn = locate(sh, r, [&](int32_t i, f32x4 v, uint64_t* w) {
            // (a span before the last kept index, after it, or both)
            const int32_t first = __builtin_amdgcn_readfirstlane(i);
            const float from = first <= cut.last ? least_f : next_f;
            if (first <= cut.last && cut.last - first < kSpan) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    v[j] = v[j] == least_f && i + j > cut.last ? __builtin_nanf("") : v[j];
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                w[j] = 0;
            }
            const bool kept[4] = {v[0] >= from, v[1] >= from, v[2] >= from, v[3] >= from};
            if (kept[0] || kept[1] || kept[2] || kept[3]) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    v[j] = kept[j] ? v[j] : __builtin_nanf("");
                }
                r.units(v, w);
            }
        }, [&](uint64_t all) {
            total = all;
            return target_of(all);
        });
    }
    if (threadIdx.x == 0) {
        a.token[row] = drawn.at;
        if (a.probability != nullptr) {
            a.probability[row] = static_cast<float>(static_cast<double>(drawn.weight) / static_cast<double>(total));
        }
    }
}

}  // namespace

hipError_t launch_sample(const SampleArgs& a, hipStream_t s) {
    int bits = 46;
    while (a.vocab > int64_t{1} << (63 - bits)) {
        --bits;
    }
    // (a launch takes less than 2^32 threads)
    hipError_t err = hipSuccess;
    for (int64_t row0 = 0; row0 < a.rows && err == hipSuccess; row0 += kMostRows) {
        hipLaunchKernelGGL(sample_kernel, dim3(static_cast<unsigned>(std::min(a.rows - row0, kMostRows))), dim3(kThreads), 0, s,
                           a, row0, bits);
        err = hipGetLastError();
    }
    return err;
}

}  // namespace lm
