// k_latent.hip -- what lies between the projections of an attention layer and
// its latents in pages (k_paged.hip): the new tokens' latents into their slots,
// and kv_b_proj, whose key half W_k [head][nope][rank] is taken into the query
// and whose value half W_v [head][vh][rank] into the output:
//   q . (W_k c) = (W_k^T q) . c        sum_j p_j (W_v c_j) = W_v (sum_j p_j c_j)
// Reference: Attention::forward (src/Attention.cpp:33-98), within the MFMA
// path's tolerance: fp16 operands, fp32 sums, norms and rotations in fp32.
#include "mfma_tile.h"
#include "serve_internal.h"

namespace lm {
namespace {

typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// Pair i of a row of `rope` channels at `from`, rotated into `to`; positions
// past the tables stay as they are (and where they are).
__device__ inline void rotate_to(const LatentArgs& a, const float* from, int i, int32_t pos, _Float16* to) {
    const float e = from[2 * i], o = from[2 * i + 1];
    const int half = a.rope / 2;
    if (pos < 0 || pos >= a.max_positions) {
        to[2 * i] = static_cast<_Float16>(e);
        to[2 * i + 1] = static_cast<_Float16>(o);
        return;
    }
    const int64_t at = static_cast<int64_t>(pos) * half + i;
    float lo, hi;
    rotate_pair(e, o, a.cos_t[at], a.sin_t[at], lo, hi);
    to[i] = static_cast<_Float16>(lo);
    to[i + half] = static_cast<_Float16>(hi);
}

// A workgroup per token: its normalised latent and rotated key into its slot of
// the pool, its heads' rotated query channels behind the absorbed ones. Rows
// without a slot in the pool store nothing there. Bound by its launch: 14 KB read
// and 3 KB written a token (16 heads; one token 4.6 us, 2048 10 us).
__global__ __launch_bounds__(256) void latent_rows_kernel(const LatentArgs a) {
    __shared__ double part[4];
    const int64_t t = blockIdx.x;
    const int32_t pos = a.positions[t], slot = a.slots[t];
    const float* const row = a.lat + t * (a.rank + a.rope);
    const bool stored = slot >= 0 && slot < a.pool_rows && t < a.live[0];
    _Float16* const to = a.pool + static_cast<int64_t>(stored ? slot : 0) * (a.rank + a.rope);
    const float inverse = rms_inverse_256(row, a.rank, a.eps, part);
    if (stored) {
        for (int c = threadIdx.x; c < a.rank; c += 256) {
            float x = row[c] * inverse;
            x = x * a.norm[c];
            asm volatile("" : "+v"(x));  // round to fp32 first: no mixed-precision product
            to[c] = static_cast<_Float16>(x);
        }
        for (int i = threadIdx.x; i < a.rope / 2; i += 256) {
            rotate_to(a, row + a.rank, i, pos, to + a.rank);
        }
    }
    const float* const q = a.q + t * a.heads * (a.nope + a.rope);
    _Float16* const q16 = a.q16 + t * a.heads * (a.rank + a.rope);
    for (int n = threadIdx.x; n < a.heads * (a.rope / 2); n += 256) {
        const int h = n / (a.rope / 2), i = n - h * (a.rope / 2);
        rotate_to(a, q + h * (a.nope + a.rope) + a.nope, i, pos, q16 + h * (a.rank + a.rope) + a.rank);
    }
}

// Zeros into rows of `width` floats from live[0] on.
__global__ __launch_bounds__(256) void clear_rows_kernel(float* rows, const int32_t* live, int32_t width) {
    if (static_cast<int64_t>(blockIdx.x) >= live[0]) {
        for (int c = threadIdx.x; c < width; c += 256) {
            rows[blockIdx.x * static_cast<int64_t>(width) + c] = 0.0f;
        }
    }
}

// Key halves transposed into panels [heads rank][nope], from kv_b's panels
// [heads (nope + vh)][rank]; once per upload.
__global__ __launch_bounds__(256) void absorb_kernel(const _Float16* __restrict__ kvb, _Float16* __restrict__ out,
                                                     int32_t heads, int32_t nope, int32_t vh, int32_t rank) {
    const int64_t n = blockIdx.x * int64_t{256} + threadIdx.x;
    if (n >= static_cast<int64_t>(heads) * nope * rank) {
        return;
    }
    const int64_t row = n / nope;  // h rank + r
    const int d = static_cast<int>(n - row * nope);
    const int64_t h = row / rank;
    const int r = static_cast<int>(row - h * rank);
    out[panel_index(row, d, static_cast<int64_t>(heads) * rank)] =
        kvb[panel_index(h * (nope + vh) + d, r, static_cast<int64_t>(heads) * (nope + vh))];
}

__device__ inline half8 load8(const float* p) {
    const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
    half8 h;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        h[e] = static_cast<_Float16>(a[e]);
        h[4 + e] = static_cast<_Float16>(b[e]);
    }
    return h;
}
__device__ inline half8 load8(const _Float16* p) { return *reinterpret_cast<const half8*>(p); }

// Per head: out[t][n] = sum_k x[t][k] w[n][k]. A wave takes B x B of a head, as
// products of 16 x 16 x 32 whose operands come straight from memory: the weights of
// all heads (2 MB a side on V2-Lite) stay in each L2, and K is 128 or 512, so there
// is no loop long enough to pay for staging in LDS. Row m of a product's weights is
// row B / 4 (m / 4) + 4 j + m % 4 of the tile, so that a lane's sums of all products
// are B / 4 successive channels of a token (queries of 2048 tokens: 33.1 -> 31.4 us).
// Bound by those loads: 200 MB from the caches for that call, 4.3 GFLOP.
template <class X, int B>
__global__ __launch_bounds__(256) void heads_kernel(const HeadsArgs a) {
    constexpr int S = B / 16;
    const int lane = threadIdx.x & 63, low = lane & 15, grp = lane >> 4;
    const int nt = a.N / B;
    const int64_t tt = (a.tokens + B - 1) / B;
    // weight tiles of a token tile side by side: its tokens are read from L2 once
    const int64_t tile = blockIdx.x * int64_t{4} + (threadIdx.x >> 6);
    if (tile >= tt * nt * a.heads) {
        return;
    }
    const int n0 = static_cast<int>(tile % nt) * B;
    const int h = static_cast<int>(tile / nt % a.heads);
    const int64_t t0 = tile / nt / a.heads * B;
    const X* x[S];
    const _Float16* w[S];
#pragma unroll
    for (int i = 0; i < S; ++i) {
        x[i] = static_cast<const X*>(a.x) + min(t0 + 16 * i + low, a.tokens - 1) * a.x_token + h * a.x_head + 8 * grp;
        w[i] = a.w + panel_index(static_cast<int64_t>(h) * a.w_head + a.w_first + n0 + B / 4 * (low >> 2) + 4 * i + (low & 3), 8 * grp, a.w_rows);
    }
    f32x4 sums[S][S] = {};
#pragma unroll 4
    for (int k = 0; k < a.K; k += 32) {
        half8 xs[S], ws[S];
#pragma unroll
        for (int i = 0; i < S; ++i) {
            xs[i] = load8(x[i] + k);
            ws[i] = load8(w[i] + k * a.w_rows);
        }
#pragma unroll
        for (int i = 0; i < S; ++i) {
#pragma unroll
            for (int j = 0; j < S; ++j) {
                sums[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ws[j], xs[i], sums[i][j], 0, 0, 0);
            }
        }
    }
    const int64_t live = a.live != nullptr ? a.live[0] : a.tokens;
#pragma unroll
    for (int i = 0; i < S; ++i) {
        const int64_t t = t0 + 16 * i + low;
        if (t < a.tokens) {
#pragma unroll
            for (int j = 0; j < S; ++j) {
                const int n = n0 + B / 4 * grp + 4 * j;
                half4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    // rows that the attention left as they were give zeros
                    v[e] = static_cast<_Float16>(t < live ? sums[i][j][e] : 0.0f);
                }
                _Float16* const to = a.out_panels != 0 ? a.out + panel_index(t, h * a.N + n, a.tokens)
                                                       : a.out + t * a.out_token + h * a.out_head + n;
                *reinterpret_cast<half4*>(to) = v;
            }
        }
    }
}

template <class X, int B>
void launch_heads_tiles(const HeadsArgs& a, hipStream_t s) {
    const int64_t tiles = (a.tokens + B - 1) / B * (a.N / B) * a.heads;
    hipLaunchKernelGGL((heads_kernel<X, B>), dim3(static_cast<unsigned>((tiles + 3) / 4)), dim3(256), 0, s, a);
}

}  // namespace

hipError_t launch_latent_rows(const LatentArgs& a, hipStream_t s) {
    hipLaunchKernelGGL(latent_rows_kernel, dim3(static_cast<unsigned>(a.tokens)), dim3(256), 0, s, a);
    return hipGetLastError();
}

hipError_t launch_clear_rows(float* rows, const int32_t* live, int64_t tokens, int32_t width, hipStream_t s) {
    hipLaunchKernelGGL(clear_rows_kernel, dim3(static_cast<unsigned>(tokens)), dim3(256), 0, s, rows, live, width);
    return hipGetLastError();
}

hipError_t launch_absorb(const _Float16* kvb, _Float16* out, int32_t heads, int32_t nope, int32_t vh, int32_t rank,
                         hipStream_t s) {
    const int64_t n = static_cast<int64_t>(heads) * nope * rank;
    hipLaunchKernelGGL(absorb_kernel, dim3(static_cast<unsigned>((n + 255) / 256)), dim3(256), 0, s, kvb, out, heads,
                       nope, vh, rank);
    return hipGetLastError();
}

// The largest tiles that still give every SIMD one. V2-Lite's queries and outputs
// with B = 16, 32, 64 (us): 32 tokens 4.2, 5.5, 7.9 and 7.4, 8.6, 12.4; 128 tokens
// 7.7, 5.9, 9.4 and 7.2, 8.5, 15.0; 512 tokens 23.4, 14.2, 10.5 and 13.9, 9.0, 15.4;
// 2048 tokens 84.7, 47.2, 33.1 and 49.8, 27.6, 18.9.
hipError_t launch_heads(const HeadsArgs& a, hipStream_t s) {
    const auto tiles = [&](int b) { return a.N % b == 0 ? (a.tokens + b - 1) / b * (a.N / b) * a.heads : 0; };
    const int b = tiles(64) >= 1024 ? 64 : tiles(32) >= 1024 ? 32 : 16;
    if (a.x_f32 != 0) {
        b == 64   ? launch_heads_tiles<float, 64>(a, s)
        : b == 32 ? launch_heads_tiles<float, 32>(a, s)
                  : launch_heads_tiles<float, 16>(a, s);
    } else {
        b == 64   ? launch_heads_tiles<_Float16, 64>(a, s)
        : b == 32 ? launch_heads_tiles<_Float16, 32>(a, s)
                  : launch_heads_tiles<_Float16, 16>(a, s);
    }
    return hipGetLastError();
}

}  // namespace lm
