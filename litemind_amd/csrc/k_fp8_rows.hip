// k_fp8_rows.hip -- rows and matrices into FP8 blocks (lm_fp8_quantize).
//
// A block's scale is max(m / 448, 2^-126), m the largest magnitude of its finite
// values, and its codes are RNE_e4m3(x * (1 / scale)): one read of x, a
// reduction over the block, one write of a byte an element.
#include "fp8_internal.h"

#include <algorithm>

namespace lm {
namespace {

// Eight values of a row from element c0 on: the lane's own, `vec` by 16-byte
// loads (all eight or none in the row), else element by element. Values past
// the row are 0, which no scale notices and nothing stores.
template <class T>
__device__ inline void load8(const T* __restrict__ row, int64_t c0, int64_t width, bool vec, float (&v)[8]) {
    if (vec) {
        if (c0 < width) {
            T t[8];
#pragma unroll
            for (int i = 0; i < static_cast<int>(sizeof(t) / 16); ++i) {
                reinterpret_cast<uint4*>(t)[i] = reinterpret_cast<const uint4*>(row + c0)[i];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                v[i] = static_cast<float>(t[i]);
            }
            return;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v[i] = c0 + i < width ? static_cast<float>(row[c0 + i]) : 0.0f;
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        v[i] = 0.0f;
    }
}

__device__ inline void store8(uint8_t* __restrict__ row, int64_t c0, int64_t width, bool vec, const float (&v)[8],
                              float inverse) {
    float s[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        s[i] = fp8_finite_or_nan(v[i]) * inverse;
    }
    const uint2 codes = make_uint2(fp8_pack4(s[0], s[1], s[2], s[3]), fp8_pack4(s[4], s[5], s[6], s[7]));
    if (vec) {
        if (c0 < width) {
            *reinterpret_cast<uint2*>(row + c0) = codes;
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (c0 + i < width) {
            row[c0 + i] = static_cast<uint8_t>((i < 4 ? codes.x : codes.y) >> (8 * (i & 3)));
        }
    }
}

__device__ inline float most8(const float (&v)[8], float most) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        most = __builtin_fmaxf(most, fp8_magnitude(v[i]));
    }
    return most;
}

// Blocks of 1 x 128: sixteen lanes a block, eight values a lane.
template <class T>
__global__ __launch_bounds__(256) void fp8_rows_kernel(Fp8Rows a, bool vec, int64_t items, int32_t wide) {
    for (int64_t first = blockIdx.x * int64_t{16}; first < items; first += gridDim.x * int64_t{16}) {
        const int64_t item = first + (threadIdx.x >> 4);
        const int64_t at = item < items ? item : items - 1;  // every lane takes part in the shuffles
        // 32-bit division where the items allow it
        const int64_t r = items <= 0x7fffffff ? static_cast<uint32_t>(at) / static_cast<uint32_t>(wide) : at / wide;
        const int64_t c0 = (at - r * wide) * kFp8Block + 8 * (threadIdx.x & 15);
        float v[8];
        load8(static_cast<const T*>(a.x) + r * a.stride, c0, a.width, vec, v);
        float most = most8(v, 0.0f);
#pragma unroll
        for (int o = 8; o >= 1; o >>= 1) {
            most = __builtin_fmaxf(most, __shfl_xor(most, o));
        }
        const float scale = fp8_scale(most);
        if (item < items) {
            store8(a.q + r * a.width, c0, a.width, vec, v, 1.0f / scale);
            if ((threadIdx.x & 15) == 0) {
                a.scale[item] = scale;
            }
        }
    }
}

// Blocks of 128 x 128: a workgroup a block, which stays in registers.
template <class T>
__global__ __launch_bounds__(256) void fp8_matrix_kernel(Fp8Rows a, bool vec, int32_t wide) {
    __shared__ float part[4];
    const int64_t tall = blockIdx.y, b = blockIdx.x;
    const int64_t c0 = b * kFp8Block + 8 * (threadIdx.x & 15);
    const int64_t r0 = tall * kFp8Block + (threadIdx.x >> 4);
    float v[8][8];
    float most = 0.0f;
#pragma unroll
    for (int p = 0; p < 8; ++p) {
        const int64_t r = min(r0 + 16 * p, a.rows - 1);
        const int64_t at = a.group == 0 ? r : r / a.group * (2 * a.group) + r % a.group;
        load8(static_cast<const T*>(a.x) + at * a.stride, c0, a.width, vec, v[p]);
    }
#pragma unroll
    for (int p = 0; p < 8; ++p) {
        most = most8(v[p], most);  // a row past the last repeats the last, which is of this block
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        most = __builtin_fmaxf(most, __shfl_xor(most, o));
    }
    if ((threadIdx.x & 63) == 0) {
        part[threadIdx.x >> 6] = most;
    }
    __syncthreads();
    most = __builtin_fmaxf(__builtin_fmaxf(part[0], part[1]), __builtin_fmaxf(part[2], part[3]));
    const float scale = fp8_scale(most);
    const float inverse = 1.0f / scale;
#pragma unroll
    for (int p = 0; p < 8; ++p) {
        const int64_t r = r0 + 16 * p;
        if (r < a.rows) {
            store8(a.q + r * a.width, c0, a.width, vec, v[p], inverse);
        }
    }
    if (threadIdx.x == 0) {
        a.scale[tall * wide + b] = scale;
    }
}

template <class T>
hipError_t launch_rows(const Fp8Rows& a, hipStream_t s) {
    const int64_t wide = fp8_blocks(a.width);
    const int64_t items = a.rows * wide;
    // sixteen bytes at a time where every row's start and end allow it
    const bool vec = reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && a.stride * static_cast<int64_t>(sizeof(T)) % 16 == 0 &&
                     a.width % 8 == 0;
    if (a.block_rows == 1) {
        const unsigned blocks = static_cast<unsigned>(std::min<int64_t>((items + 15) / 16, 1 << 20));
        hipLaunchKernelGGL(HIP_KERNEL_NAME(fp8_rows_kernel<T>), dim3(blocks), dim3(256), 0, s, a, vec, items,
                           static_cast<int32_t>(wide));
    } else {
        const int64_t tall = fp8_blocks(a.rows);  // under 2^16, as the grid's second axis has to be
        hipLaunchKernelGGL(HIP_KERNEL_NAME(fp8_matrix_kernel<T>),
                           dim3(static_cast<unsigned>(wide), static_cast<unsigned>(tall)), dim3(256), 0, s, a, vec,
                           static_cast<int32_t>(wide));
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_fp8_quantize(const Fp8Rows& a, hipStream_t s) {
    switch (a.dtype) {
        case LM_DT_F32:
            return launch_rows<float>(a, s);
        case LM_DT_F16:
            return launch_rows<_Float16>(a, s);
        default:
            return launch_rows<__bf16>(a, s);
    }
}

}  // namespace lm
