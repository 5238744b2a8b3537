// k_paged.hip -- attention of the requests' new tokens over a latent cache in
// pages (litemind_serving.h, lm_paged_attention).
//
// Per token t of request r at position p and per head h, with pool rows
// (c_j, k_j) and queries absorbed into the latent space:
//     s_j = scale q . (c_j, k_j), j <= p;   out = sum_j softmax(s)_j c_j
#include "serve_internal.h"

namespace lm {
namespace {

typedef __bf16 bf16;

// ---- any widths ----
// One workgroup per token and head, its four waves on alternate keys, a lane on
// channels lane + 64 i; running maximum and sum per wave, joined at the end.
constexpr int kMaxRank = 1024, kMaxRope = 256;

template <class E>
__global__ __launch_bounds__(256) void paged_any_kernel(const PagedAttention a) {
    constexpr int kC = kMaxRank / 64, kR = kMaxRope / 64;
    __shared__ float part[4][kMaxRank], stats[4][2];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int32_t t = static_cast<int32_t>(blockIdx.x / a.heads), h = static_cast<int32_t>(blockIdx.x % a.heads);
    const PagedView& v = a.view;
    // the token's request: the last whose rows start at or before it
    int32_t lo = 0, hi = v.requests;
    while (hi - lo > 1) {
        const int32_t mid = lo + (hi - lo) / 2;
        if (v.starts[mid] <= t) {
            lo = mid;
        } else {
            hi = mid;
        }
    }
    const PagedRequest r = paged_request(v, lo);
    if (t < r.first || t >= r.first + r.added) {
        return;  // past the last request's rows
    }
    const int width = a.rank + a.rope;
    const E* const q = static_cast<const E*>(a.q) + (static_cast<int64_t>(t) * a.heads + h) * width;
    float qc[kC], qr[kR], o[kC];
#pragma unroll
    for (int i = 0; i < kC; ++i) {
        qc[i] = lane + 64 * i < a.rank ? static_cast<float>(q[lane + 64 * i]) : 0.0f;
        o[i] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < kR; ++i) {
        qr[i] = lane + 64 * i < a.rope ? static_cast<float>(q[a.rank + lane + 64 * i]) : 0.0f;
    }
    float m = -__builtin_inff(), l = 0.0f;
    const int32_t keys = r.cached + t - r.first + 1;
    for (int32_t j = wave; j < keys; j += 4) {
        const int64_t page = checked_page(v, v.table[static_cast<int64_t>(lo) * v.table_width + j / v.page_size]);
        const E* const row = static_cast<const E*>(a.pool) + (page * v.page_size + j % v.page_size) * width;
        float c[kC], s = 0.0f;
#pragma unroll
        for (int i = 0; i < kC; ++i) {
            c[i] = lane + 64 * i < a.rank ? static_cast<float>(row[lane + 64 * i]) : 0.0f;
            s = __builtin_fmaf(qc[i], c[i], s);
        }
#pragma unroll
        for (int i = 0; i < kR; ++i) {
            s = __builtin_fmaf(qr[i], lane + 64 * i < a.rope ? static_cast<float>(row[a.rank + lane + 64 * i]) : 0.0f,
                               s);
        }
        for (int w = 32; w >= 1; w >>= 1) {
            s += __shfl_xor(s, w);
        }
        s *= a.scale;
        const float top = fmaxf(m, s);
        // no score above -infinity yet: nothing to rescale, and no weight
        const float alpha = m == -__builtin_inff() ? 1.0f : __expf(m - top);
        const float p = s == -__builtin_inff() ? 0.0f : __expf(s - top);
        l = __builtin_fmaf(l, alpha, p);
#pragma unroll
        for (int i = 0; i < kC; ++i) {
            o[i] = __builtin_fmaf(o[i], alpha, p * c[i]);
        }
        m = top;
    }
#pragma unroll
    for (int i = 0; i < kC; ++i) {
        part[wave][lane + 64 * i] = o[i];
    }
    if (lane == 0) {
        stats[wave][0] = m;
        stats[wave][1] = l;
    }
    __syncthreads();
    float top = -__builtin_inff(), total = 0.0f, w[4];
    for (int i = 0; i < 4; ++i) {
        top = fmaxf(top, stats[i][0]);
    }
    for (int i = 0; i < 4; ++i) {
        w[i] = stats[i][0] == -__builtin_inff() ? 0.0f : __expf(stats[i][0] - top);
        total = __builtin_fmaf(w[i], stats[i][1], total);
    }
    E* const out = static_cast<E*>(a.out) + (static_cast<int64_t>(t) * a.heads + h) * a.rank;
    for (int i = threadIdx.x; i < a.rank; i += 256) {
        float sum = 0.0f;
        for (int k = 0; k < 4; ++k) {
            sum = __builtin_fmaf(w[k], part[k][i], sum);
        }
        out[i] = static_cast<E>(sum / total);
    }
}

template <class E>
hipError_t launch(const PagedAttention& a, hipStream_t s) {
    hipLaunchKernelGGL(paged_any_kernel<E>, dim3(static_cast<unsigned>(a.view.tokens * a.heads)), dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_paged_attention(const PagedAttention& a, hipStream_t s) {
    return a.bf16 != 0 ? launch<bf16>(a, s) : launch<_Float16>(a, s);
}

}  // namespace lm
