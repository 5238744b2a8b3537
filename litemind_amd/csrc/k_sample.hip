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
// without a sort by descending through the bits of the logits, eight at a time:
// counts per value of the eight bits give the k-th largest logit, sums of e the
// one at which top-p is reached.  Equal logits at a cut are told apart by index.
#include "serve_internal.h"

namespace lm {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kBins = 256;

// 2^t in units of 2^-bits, to the nearest, for t <= 0: t split into n + f with
// |f| <= 1/2, 2^f by its power series to the 11th power (cut off at 4e-15), and
// the unit taken from the double's mantissa next to 2^52.
__device__ inline uint64_t exp2_units(double t, int bits) {
    if (!(t > -64.0)) {
        return 0;
    }
    const double n = __builtin_rint(t);
    const double f = (t - n) * 0.693147180559945309417;
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
    const double scaled = __builtin_ldexp(p, static_cast<int>(n) + bits);
    return static_cast<uint64_t>(__double_as_longlong(scaled + 0x1p52)) & 0xfffffffffffffull;
}

// Whole numbers in the order of the floats; NaN below -infinity.
__device__ inline uint32_t order_key(float x) {
    if (x != x) {
        return 0;
    }
    const uint32_t b = __float_as_uint(x + 0.0f);  // -0 as +0
    return (b & 0x80000000u) != 0 ? ~b : b | 0x80000000u;
}
constexpr uint32_t kKeyMinusInf = 0x007fffffu;

// What a row's passes share.
struct Row {
    const float* x;
    int32_t n;
    double top, rate;  // largest logit, log2(e) / temperature
    int bits;
    bool top_inf;
    __device__ uint64_t units(float v) const {
        if (!(v > -__builtin_inff())) {
            return 0;
        }
        if (top_inf) {
            return v == __builtin_inff() ? 1ull << bits : 0;
        }
        return exp2_units((static_cast<double>(v) - top) * rate, bits);
    }
};

template <class T, class F>
__device__ inline T block_reduce(T v, T* part, F f) {
    for (int o = 32; o >= 1; o >>= 1) {
        v = f(v, __shfl_xor(v, o));
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
        part[threadIdx.x >> 6] = v;
    }
    __syncthreads();
    v = part[0];
    for (int w = 1; w < kWaves; ++w) {
        v = f(v, part[w]);
    }
    return v;
}

__device__ inline uint64_t block_sum(uint64_t v, uint64_t* part) {
    return block_reduce(v, part, [](uint64_t a, uint64_t b) { return a + b; });
}

// The exclusive prefix of v over the workgroup's threads.
__device__ inline uint64_t block_before(uint64_t v, uint64_t* part) {
    uint64_t sum = v;
    for (int o = 1; o < 64; o <<= 1) {
        const uint64_t up = __shfl_up(sum, o);
        if ((threadIdx.x & 63) >= static_cast<unsigned>(o)) {
            sum += up;
        }
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 63) {
        part[threadIdx.x >> 6] = sum;
    }
    __syncthreads();
    uint64_t base = 0;
    for (int w = 0; w < static_cast<int>(threadIdx.x >> 6); ++w) {
        base += part[w];
    }
    return base + sum - v;
}

// A prefix of the order: keys above `key`, and of those equal to it the
// `equal` of lowest index.
struct Cut {
    uint32_t key;
    uint64_t equal;
};

// Descends to the key at which the weight of the keys above it, within
// `outer`, reaches `want`: the largest key with weight(keys > key) < want <=
// weight(keys >= key).  Weights: 1 each, or units.  *above: weight(keys > key).
template <bool MASS>
__device__ uint32_t descend(const Row& r, uint32_t floor_key, uint64_t want, uint64_t* bins, uint64_t* part,
                            uint64_t* above) {
    uint32_t prefix = 0;
    uint64_t before = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        for (int b = threadIdx.x; b < kBins; b += kThreads) {
            bins[b] = 0;
        }
        __syncthreads();
        for (int32_t i = threadIdx.x; i < r.n; i += kThreads) {
            const uint32_t key = order_key(r.x[i]);
            if (key >= floor_key && key > kKeyMinusInf &&
                (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8)))) {
                const uint64_t w = MASS ? r.units(r.x[i]) : 1;
                if (w != 0) {
                    atomicAdd(reinterpret_cast<unsigned long long*>(&bins[(key >> shift) & 255]), w);
                }
            }
        }
        __syncthreads();
        // the highest bin whose sum from above reaches want
        const int b = 255 - static_cast<int>(threadIdx.x & 255);
        const uint64_t own = threadIdx.x < kBins ? bins[b] : 0;
        const uint64_t ahead = block_before(own, part) + before;
        __syncthreads();
        if (threadIdx.x < kBins && ahead < want && ahead + own >= want) {
            part[kWaves] = static_cast<uint64_t>(b);
            part[kWaves + 1] = ahead;
        }
        __syncthreads();
        prefix |= static_cast<uint32_t>(part[kWaves]) << shift;
        before = part[kWaves + 1];
    }
    *above = before;
    return prefix;
}

__global__ __launch_bounds__(kThreads) void sample_kernel(const SampleArgs a, int bits) {
    __shared__ uint64_t bins[kBins], part[kWaves + 2];
    __shared__ uint32_t keys[kWaves];
    const int64_t row = blockIdx.x;
    const lm_sampling set = a.settings[row];
    Row r;
    r.x = a.logits + row * a.stride;
    r.n = static_cast<int32_t>(a.vocab);
    r.bits = bits;
    uint32_t best = 0;
    for (int32_t i = threadIdx.x; i < r.n; i += kThreads) {
        best = max(best, order_key(r.x[i]));
    }
    best = block_reduce(best, keys, [](uint32_t x, uint32_t y) { return max(x, y); });
    if (best <= kKeyMinusInf) {
        if (threadIdx.x == 0) {
            a.token[row] = -1;
            if (a.probability != nullptr) {
                a.probability[row] = 0.0f;
            }
        }
        return;
    }
    const float top = __uint_as_float((best & 0x80000000u) != 0 ? best & 0x7fffffffu : ~best);
    const bool greedy = !(set.temperature > 0.0f);
    r.top = static_cast<double>(top);
    r.top_inf = top == __builtin_inff();
    r.rate = greedy ? 0.0 : 1.4426950408889634074 / static_cast<double>(set.temperature);
    // the cut of top-k, then of top-p within it
    const uint64_t all = ~0ull;
    Cut cut{kKeyMinusInf + 1, all};
    if (greedy) {
        cut = Cut{best, 1};
    } else {
        if (set.top_k > 0 && set.top_k < r.n) {
            uint64_t candidates = 0;
            for (int32_t i = threadIdx.x; i < r.n; i += kThreads) {
                candidates += order_key(r.x[i]) > kKeyMinusInf ? 1 : 0;
            }
            candidates = block_sum(candidates, part);
            if (static_cast<uint64_t>(set.top_k) < candidates) {
                uint64_t above = 0;
                const uint32_t key = descend<false>(r, 0, static_cast<uint64_t>(set.top_k), bins, part, &above);
                cut = Cut{key, static_cast<uint64_t>(set.top_k) - above};
            }
        }
        if (set.top_p < 1.0f) {
            // mass of the prefix: keys above the cut, and `equal` times the cut's
            uint64_t mass = 0, ties = 0;
            for (int32_t i = threadIdx.x; i < r.n; i += kThreads) {
                const uint32_t key = order_key(r.x[i]);
                mass += key > cut.key ? r.units(r.x[i]) : 0;
                ties += key == cut.key ? 1 : 0;
            }
            mass = block_sum(mass, part);
            ties = block_sum(ties, part);
            const uint32_t k = cut.key;
            const uint64_t each = r.units(__uint_as_float((k & 0x80000000u) != 0 ? k & 0x7fffffffu : ~k));
            const uint64_t tied = min(cut.equal, ties);
            const uint64_t total = mass + tied * each;
            // a token is kept while the mass before it is under top_p of the total
            const double share = fmax(static_cast<double>(set.top_p), 0.0) * static_cast<double>(total);
            const uint64_t want = max(static_cast<uint64_t>(__builtin_ceil(share)), uint64_t{1});
            if (want <= mass) {
                uint64_t above = 0;
                const uint32_t key = descend<true>(r, 0, want, bins, part, &above);
                const uint64_t unit = r.units(__uint_as_float((key & 0x80000000u) != 0 ? key & 0x7fffffffu : ~key));
                cut = Cut{key, (want - above + unit - 1) / unit};
            } else if (want <= total) {
                cut = Cut{cut.key, (want - mass + each - 1) / each};
            }
        }
        if (set.min_p > 1.0f) {
            cut = Cut{best, 1};
        } else if (set.min_p > 0.0f) {
            // the lowest key whose e is at least min_p; the largest logit's always
            uint32_t lowest = best;
            for (int32_t i = threadIdx.x; i < r.n; i += kThreads) {
                const uint32_t key = order_key(r.x[i]);
                if (key >= cut.key && key > kKeyMinusInf && !r.top_inf &&
                    exp((static_cast<double>(r.x[i]) - r.top) / static_cast<double>(set.temperature)) >=
                        static_cast<double>(set.min_p)) {
                    lowest = min(lowest, key);
                }
            }
            lowest = block_reduce(lowest, keys, [](uint32_t x, uint32_t y) { return min(x, y); });
            if (lowest > cut.key) {
                cut = Cut{lowest, all};
            }
        }
    }
    // the kept tokens in index order, a stretch of the row per thread
    const int32_t per = (r.n + kThreads - 1) / kThreads;
    const int32_t i0 = min(static_cast<int32_t>(threadIdx.x) * per, r.n), i1 = min(i0 + per, r.n);
    uint64_t ties = 0;
    for (int32_t i = i0; i < i1; ++i) {
        ties += order_key(r.x[i]) == cut.key ? 1 : 0;
    }
    const uint64_t ties_before = block_before(ties, part);
    auto weight = [&](int32_t i, uint64_t& seen) -> uint64_t {
        const uint32_t key = order_key(r.x[i]);
        const bool kept = key > cut.key || (key == cut.key && seen < cut.equal);
        seen += key == cut.key ? 1 : 0;
        return kept ? r.units(r.x[i]) : 0;
    };
    uint64_t sum = 0, seen = ties_before;
    for (int32_t i = i0; i < i1; ++i) {
        sum += weight(i, seen);
    }
    const uint64_t before = block_before(sum, part);
    const uint64_t total = block_sum(sum, part);
    // running > u total: over the whole number below it
    const float u = a.uniform[row];
    const double at = (u > 0.0f ? static_cast<double>(u) : 0.0) * static_cast<double>(total);
    const uint64_t target = min(static_cast<uint64_t>(at), total - 1);
    __syncthreads();
    if (target >= before && target - before < sum) {
        uint64_t running = before;
        seen = ties_before;
        for (int32_t i = i0; i < i1; ++i) {
            const uint64_t w = weight(i, seen);
            running += w;
            if (running > target) {
                a.token[row] = i;
                if (a.probability != nullptr) {
                    a.probability[row] = static_cast<float>(static_cast<double>(w) / static_cast<double>(total));
                }
                break;
            }
        }
    }
}

}  // namespace

hipError_t launch_sample(const SampleArgs& a, hipStream_t s) {
    int bits = 46;
    while (a.vocab > int64_t{1} << (63 - bits)) {
        --bits;
    }
    hipLaunchKernelGGL(sample_kernel, dim3(static_cast<unsigned>(a.rows)), dim3(kThreads), 0, s, a, bits);
    return hipGetLastError();
}

}  // namespace lm
