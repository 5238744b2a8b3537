// k_pages.hip -- the plan of a step: pages, starts, positions and slots of the
// requests' new tokens from their lengths.
//
//   length = cached + added;  start = sum of added before;  pages taken =
//   ceil(length / P) - ceil(cached / P), their place in the ring the sum of
//   those before;  slot of position p = table[p / P] P + p % P
//
// Three sums over the requests; per four tokens, and per taken and returned page,
// one search in them.  Latency bound: a decode step of 48 requests reads and
// writes 2 KB and takes 10 us by itself, 4.0 among others' calls; 509 requests of
// up to 64 new tokens take 15.9 and 5.3.  One workgroup; requests in chunks of one
// per thread.
#include "serve_internal.h"

namespace lm {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;

struct Sums {
    int32_t tokens, taken, back;
};

__device__ inline Sums operator+(const Sums& a, const Sums& b) {
    return Sums{a.tokens + b.tokens, a.taken + b.taken, a.back + b.back};
}

__device__ inline Sums wave_up(const Sums& v, int by) {
    return Sums{__shfl_up(v.tokens, by), __shfl_up(v.taken, by), __shfl_up(v.back, by)};
}

// A request's share of the step, in 64 bits where the caller's numbers could
// overflow 32.
struct Request {
    int32_t cached, added;
    bool over, bad_length, bad_added;
    int32_t had, taken;  // pages before, pages taken
};

__device__ inline Request load_request(const lm_paged_step& s, int64_t r) {
    Request q{};
    if (r >= s.requests) {
        return q;
    }
    q.cached = s.cached[r];
    q.added = s.added[r];
    q.over = q.added < 0;
    q.added = max(q.added, 0);
    const int64_t length = static_cast<int64_t>(q.cached) + q.added;
    q.bad_length = q.cached < 0 || length > static_cast<int64_t>(s.table_width) * s.page_size;
    q.bad_added = q.added > s.max_added;
    if (!q.bad_length) {
        const uint32_t size = static_cast<uint32_t>(s.page_size);
        q.had = static_cast<int32_t>((static_cast<uint32_t>(q.cached) + size - 1) / size);
        q.taken = static_cast<int32_t>((static_cast<uint32_t>(length) + size - 1) / size) - q.had;
    }
    return q;
}

// Last entry of the ascending at[0 .. n) that is <= i (at[0] <= i).
__device__ inline int find(const int32_t* at, int n, int32_t i) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (at[mid] <= i) {
            lo = mid;
        } else {
            hi = mid;
        }
    }
    return lo;
}

__global__ __launch_bounds__(kThreads) void page_plan_kernel(const lm_paged_step s) {
    __shared__ int32_t starts[kThreads], firsts[kThreads], backs[kThreads], had[kThreads], cached[kThreads];
    __shared__ Sums wave_sums[kWaves];
    __shared__ int64_t wave_tokens[kWaves], wave_taken[kWaves], wave_back[kWaves];
    __shared__ int32_t flags[2];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // places in the ring in 32 bits: a division of 64 takes 150 instructions
    const int32_t count = s.queue_in[1];
    const uint32_t ring = static_cast<uint32_t>(s.pages);
    const int32_t head = s.queue_in[0] % static_cast<int32_t>(ring);
    const uint32_t front = static_cast<uint32_t>(head) + (head < 0 ? ring : 0);
    const uint32_t behind = (front + static_cast<uint32_t>(max(count, 0))) % ring;
    const Request mine = load_request(s, tid);  // of the first chunk
    // can the step be served: totals in 64 bits
    if (tid < 2) {
        flags[tid] = 0;
    }
    __syncthreads();
    int64_t tokens = 0, taken = 0, back = 0;
    for (int64_t r = tid; r < s.requests; r += kThreads) {
        const Request q = r < kThreads ? mine : load_request(s, r);
        if (q.bad_length) {
            flags[0] = 1;
        }
        if (q.bad_added) {
            flags[1] = 1;
        }
        tokens += q.added;
        taken += q.taken;
        back += q.over ? q.had : 0;
    }
    for (int o = 32; o >= 1; o >>= 1) {
        tokens += __shfl_xor(tokens, o);
        taken += __shfl_xor(taken, o);
        back += __shfl_xor(back, o);
    }
    if (lane == 0) {
        wave_tokens[wave] = tokens;
        wave_taken[wave] = taken;
        wave_back[wave] = back;
    }
    __syncthreads();
    tokens = taken = back = 0;
    for (int w = 0; w < kWaves; ++w) {
        tokens += wave_tokens[w];
        taken += wave_taken[w];
        back += wave_back[w];
    }
    // (returned pages go behind the free ones while taken ones are read: both have to
    // have their own places in the ring)
    const int32_t status = flags[0] != 0                             ? LM_STEP_LENGTH
                           : flags[1] != 0 || tokens > s.tokens      ? LM_STEP_TOKENS
                           : taken > max(static_cast<int64_t>(count), int64_t{0}) ? LM_STEP_PAGES
                           : count < 0 || count + back > s.pages ? LM_STEP_RING
                                                                       : LM_STEP_OK;
    Sums before{};  // of the requests in earlier chunks
    if (status == LM_STEP_OK) {
        for (int64_t r0 = 0; r0 < s.requests; r0 += kThreads) {
            const int64_t r = r0 + tid;
            const int n = static_cast<int>(min(s.requests - r0, static_cast<int64_t>(kThreads)));
            const Request q = r0 == 0 ? mine : load_request(s, r);
            const Sums own{q.added, q.over ? 0 : q.taken, q.over ? q.had : 0};
            Sums sum = own;
            for (int o = 1; o < 64; o <<= 1) {
                const Sums up = wave_up(sum, o);
                if (lane >= o) {
                    sum = sum + up;
                }
            }
            __syncthreads();  // the chunk before has been read
            if (lane == 63) {
                wave_sums[wave] = sum;
            }
            __syncthreads();
            Sums base = before;
            for (int w = 0; w < kWaves; ++w) {
                if (w < wave) {
                    base = base + wave_sums[w];
                }
                before = before + wave_sums[w];
            }
            sum = base + sum;
            starts[tid] = sum.tokens - own.tokens;
            firsts[tid] = sum.taken - own.taken;
            backs[tid] = sum.back - own.back;
            had[tid] = q.had;
            cached[tid] = q.cached;
            if (r < s.requests) {
                s.lengths[r] = q.over ? 0 : q.cached + q.added;
                s.starts[r] = sum.tokens - own.tokens;
            }
            __syncthreads();
            const Sums from{starts[0], firsts[0], backs[0]};
            for (int32_t i = from.taken + tid; i < before.taken; i += kThreads) {
                const int k = find(firsts, n, i);
                s.table[(r0 + k) * s.table_width + had[k] + i - firsts[k]] = s.ring[(front + i) % ring];
            }
            for (int32_t i = from.back + tid; i < before.back; i += kThreads) {
                const int k = find(backs, n, i);
                s.ring[(behind + i) % ring] = s.table[(r0 + k) * s.table_width + i - backs[k]];
            }
            // (unsigned: rows past 2^31 - 1 are stepped to, not written)
            const uint32_t end = static_cast<uint32_t>(before.tokens);
            for (uint32_t t = static_cast<uint32_t>(from.tokens) + 4u * tid; t < end; t += 4u * kThreads) {
                int k = find(starts, n, static_cast<int32_t>(t));
                int32_t page[4], place[4];
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) {
                    if (t + j < end) {
                        while (k + 1 < n && static_cast<uint32_t>(starts[k + 1]) <= t + j) {
                            ++k;
                        }
                        place[j] = static_cast<int32_t>(cached[k] + t + j - starts[k]);
                        const int32_t column = place[j] / s.page_size;
                        page[j] = column < had[k] ? s.table[(r0 + k) * s.table_width + column]
                                                  : s.ring[(front + static_cast<uint32_t>(firsts[k] + column - had[k])) % ring];
                    }
                }
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) {
                    if (t + j < end) {
                        s.positions[t + j] = place[j];
                        s.slots[t + j] = static_cast<uint32_t>(page[j]) < ring
                                             ? page[j] * s.page_size + place[j] % s.page_size
                                             : -1;
                    }
                }
            }
        }
    } else {
        for (int64_t r = tid; r < s.requests; r += kThreads) {
            s.lengths[r] = s.cached[r];
            s.starts[r] = 0;
        }
    }
    for (int64_t t = static_cast<int64_t>(before.tokens) + tid; t < s.tokens; t += kThreads) {
        s.positions[t] = 0;
        s.slots[t] = -1;
    }
    if (tid == 0) {
        s.starts[s.requests] = before.tokens;
        s.queue_out[0] = static_cast<int32_t>((front + static_cast<uint32_t>(before.taken)) % ring);
        s.queue_out[1] = status == LM_STEP_OK ? count - before.taken + before.back : count;
        s.info[0] = status;
        s.info[1] = before.tokens;
        s.info[2] = before.taken;
        s.info[3] = before.back;
    }
}

}  // namespace

hipError_t launch_page_plan(const lm_paged_step& step, hipStream_t s) {
    hipLaunchKernelGGL(page_plan_kernel, dim3(1), dim3(kThreads), 0, s, step);
    return hipGetLastError();
}

}  // namespace lm
