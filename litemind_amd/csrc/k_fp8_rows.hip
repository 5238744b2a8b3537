// k_fp8_rows.hip -- rows and matrices into FP8 blocks (lm_fp8_quantize).
//
// A block's scale is max(m / 448, 2^-126), m the largest magnitude of its finite
// values, and its codes are RNE_e4m3(448 x / m): one read of x, a reduction over
// the block, one write of a byte an element.
//
// fp32's x * (448 / m) is off by up to 3 2^-24 of itself, and on the wrong side of
// a middle between two codes once in 2^20. So eight values' codes are made at both
// ends of +- 2^-22. 448 x = 7 2^6 x and a middle (five bits) times m are the same or
// far apart: with x and m of eleven bits by 2^-16 of themselves, so that where a
// pair of codes differs the quotient is a middle, and the even one is right. With x
// and m of 24 bits by 2^-29: there the quotients are computed in two floats, which
// are off by 2^-45 (past m = 2^100, where the second is subnormal, by up to 2^-31),
// and rounded to the nearest odd float before their rounding to e4m3.
//
// What bounds it: its way through memory, and beside it the vector units. Magnitudes
// are compared as whole numbers, which finds NaN and infinities too: only blocks that
// hold one look at each value.  10.5 M fp32 values 7.4 us, 7.1 TB/s (8.5 with every
// quotient in two floats); 22.4 M BF16 ones in blocks of 128 x 128 9.6 us, 7.0 TB/s
// (12.0 with middles in two floats).
#include "fp8_internal.h"

#include <algorithm>

namespace lm {
namespace {

// Eight neighbouring values of a row, and what their magnitudes are as whole
// numbers: of 16-bit types two to a word.
template <class T>
struct Eight {
    static constexpr bool kWide = sizeof(T) == 4;
    static constexpr uint32_t kInfinity = kWide ? 0x7f800000u : __is_same(T, __bf16) ? 0x7f80u : 0x7c00u;
    uint32_t word[2 * sizeof(T)];
    // From element c0 on, VEC by 16-byte loads (all eight or none in the row).
    // Values past the row are 0, which no scale notices and nothing stores.
    template <bool VEC>
    __device__ void load(const T* __restrict__ row, int64_t c0, int64_t width) {
#pragma unroll
        for (int i = 0; i < static_cast<int>(2 * sizeof(T)); ++i) {
            word[i] = 0;
        }
        if constexpr (VEC) {
            if (c0 < width) {
#pragma unroll
                for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) {
                    const uint4 four = reinterpret_cast<const uint4*>(row + c0)[i];
                    word[4 * i] = four.x;
                    word[4 * i + 1] = four.y;
                    word[4 * i + 2] = four.z;
                    word[4 * i + 3] = four.w;
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (c0 + i < width) {
                    if constexpr (kWide) {
                        word[i] = __builtin_bit_cast(uint32_t, row[c0 + i]);
                    } else {
                        word[i / 2] |= static_cast<uint32_t>(__builtin_bit_cast(uint16_t, row[c0 + i])) << (16 * (i & 1));
                    }
                }
            }
        }
    }
    __device__ float value(int i) const {
        if constexpr (kWide) {
            return __builtin_bit_cast(float, word[i]);
        } else if constexpr (__is_same(T, __bf16)) {
            return __builtin_bit_cast(float, i % 2 == 0 ? word[i / 2] << 16 : word[i / 2] & 0xffff0000u);
        } else {
            return static_cast<float>(__builtin_bit_cast(T, static_cast<uint16_t>(word[i / 2] >> (16 * (i & 1)))));
        }
    }
    // The larger of `most` and the magnitudes.
    __device__ uint32_t most(uint32_t most) const {
#pragma unroll
        for (int i = 0; i < static_cast<int>(2 * sizeof(T)); ++i) {
            if constexpr (kWide) {
                most = max(most, word[i] & 0x7fffffffu);
            } else {
                typedef uint16_t pair __attribute__((ext_vector_type(2)));
                most = __builtin_bit_cast(
                    uint32_t, __builtin_elementwise_max(__builtin_bit_cast(pair, most),
                                                        __builtin_bit_cast(pair, word[i] & 0x7fff7fffu)));
            }
        }
        return most;
    }
    // Of a word of magnitudes the larger, and its value.
    __device__ static uint32_t one(uint32_t most) { return kWide ? most : max(most & 0xffffu, most >> 16); }
    __device__ static float magnitude(uint32_t one) {
        if constexpr (kWide) {
            return __builtin_bit_cast(float, one);
        } else {
            return static_cast<float>(__builtin_bit_cast(T, static_cast<uint16_t>(one)));
        }
    }
    __device__ float most_finite(float most) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            most = __builtin_fmaxf(most, fp8_magnitude(value(i)));
        }
        return most;
    }
};

// 1 over a block's scale before its rounding, as a sum of two, and around it.
struct Inverse {
    float high, low, under, over;
    __device__ explicit Inverse(float most) {
        const bool least = most < kFp8Largest * 0x1p-126f;
        high = least ? 0x1p126f : kFp8Largest / most;
        low = least ? 0.0f : __builtin_fmaf(-high, most, kFp8Largest) * (high * (1.0f / kFp8Largest));
        under = high * (1.0f - 0x1p-22f);
        over = high * (1.0f + 0x1p-22f);
    }
    // x over the scale, and where that is no float (by 2^-30 of it) the odd one of
    // its neighbours, which lies on the same side of every middle.
    __device__ float exact(float x) const {
        const float first = x * high;
        const float second = __builtin_fmaf(x, low, __builtin_fmaf(x, high, -first));  // up to a step of the first
        const float v = first + second;
        const float rest = second - (v - first);
        const int32_t bits = __builtin_bit_cast(int32_t, v);
        const int32_t odd = (bits + ((bits ^ __builtin_bit_cast(int32_t, rest)) >> 31)) | 1;
        const float whole = __builtin_fabsf(rest) <= 0x1p-30f * __builtin_fabsf(v) ? v : __builtin_bit_cast(float, odd);
        return __builtin_copysignf(whole, x);  // -0 + 0 is 0
    }
};

// The codes of eight finite values; false where one of them lies so near to a
// middle that its code may be another.
template <class T>
__device__ inline bool codes8(const Eight<T>& v, const Inverse& inverse, uint2& codes) {
    const auto pack4 = [&](int i, float by) {
        return fp8_pack4_finite(v.value(i) * by, v.value(i + 1) * by, v.value(i + 2) * by, v.value(i + 3) * by);
    };
    codes = make_uint2(pack4(0, inverse.under), pack4(4, inverse.under));
    const uint2 others = make_uint2(pack4(0, inverse.over), pack4(4, inverse.over));
    if constexpr (Eight<T>::kWide) {
        return codes.x == others.x && codes.y == others.y;
    } else {  // of each two the even one
        const auto even = [](uint32_t a, uint32_t b) { return a ^ ((a ^ b) & ((a & 0x01010101u) * 0xffu)); };
        codes = make_uint2(even(codes.x, others.x), even(codes.y, others.y));
        return true;
    }
}
// The codes of any eight values.
template <class T>
__device__ inline uint2 exact_codes8(const Eight<T>& v, const Inverse& inverse) {
    const auto pack4 = [&](int i) {
        const auto quotient = [&](int at) { return inverse.exact(fp8_finite_or_nan(v.value(at))); };
        return fp8_pack4(quotient(i), quotient(i + 1), quotient(i + 2), quotient(i + 3));
    };
    return make_uint2(pack4(0), pack4(4));
}
template <bool VEC>
__device__ inline void store8(uint8_t* __restrict__ row, int64_t c0, int64_t width, uint2 codes) {
    if constexpr (VEC) {
        if (c0 < width) {
            *reinterpret_cast<uint2*>(row + c0) = codes;
        }
    } else {
        const uint64_t all = codes.x | static_cast<uint64_t>(codes.y) << 32;
#pragma unroll 1
        for (int i = 0; i < 8 && c0 + i < width; ++i) {
            row[c0 + i] = static_cast<uint8_t>(all >> (8 * i));
        }
    }
}

// Blocks of 1 x 128: sixteen lanes a block, eight values a lane.
template <class T, bool VEC>
__global__ __launch_bounds__(256) void fp8_rows_kernel(Fp8Rows a, int64_t items, int32_t wide) {
    for (int64_t first = blockIdx.x * int64_t{16}; first < items; first += gridDim.x * int64_t{16}) {
        const int64_t item = first + (threadIdx.x >> 4);
        const int64_t at = item < items ? item : items - 1;  // every lane takes part in the shuffles
        // 32-bit division where the items allow it
        const int64_t r = items <= 0x7fffffff ? static_cast<uint32_t>(at) / static_cast<uint32_t>(wide) : at / wide;
        const int64_t c0 = (at - r * wide) * kFp8Block + 8 * (threadIdx.x & 15);
        Eight<T> v;
        v.template load<VEC>(static_cast<const T*>(a.x) + r * a.stride, c0, a.width);
        uint32_t bits = v.one(v.most(0));
#pragma unroll
        for (int o = 8; o >= 1; o >>= 1) {
            bits = max(bits, static_cast<uint32_t>(__shfl_xor(static_cast<int>(bits), o)));
        }
        const bool finite = bits < v.kInfinity;
        float most = v.magnitude(bits);
        if (__any(!finite)) {
            most = v.most_finite(0.0f);
#pragma unroll
            for (int o = 8; o >= 1; o >>= 1) {
                most = __builtin_fmaxf(most, __shfl_xor(most, o));
            }
        }
        if (item < items) {
            const Inverse inverse(most);
            uint2 codes;
            if (!finite || !codes8(v, inverse, codes)) {
                codes = exact_codes8(v, inverse);
            }
            store8<VEC>(a.q + r * a.width, c0, a.width, codes);
            if ((threadIdx.x & 15) == 0) {
                a.scale[item] = fp8_scale(most);
            }
        }
    }
}

// Blocks of 128 x 128: a workgroup a block, which stays in registers.
template <class T, bool VEC>
__global__ __launch_bounds__(256) void fp8_matrix_kernel(Fp8Rows a, int32_t wide) {
    __shared__ uint32_t part[4];
    __shared__ float part_finite[4];
    const int64_t tall = blockIdx.y, b = blockIdx.x;
    const int64_t c0 = b * kFp8Block + 8 * (threadIdx.x & 15);
    const int32_t r0 = static_cast<int32_t>(blockIdx.y) * kFp8Block + static_cast<int32_t>(threadIdx.x >> 4);
    const auto load = [&](int p, Eight<T>& to) {
        const int32_t r = min(r0 + 16 * p, static_cast<int32_t>(a.rows) - 1);
        to.template load<VEC>(static_cast<const T*>(a.x) + (r + (r & ~(a.group - 1))) * a.stride, c0, a.width);
    };
    Eight<T> v[8];
#pragma unroll
    for (int p = 0; p < 8; ++p) {
        load(p, v[p]);
    }
    uint32_t bits = 0;
#pragma unroll
    for (int p = 0; p < 8; ++p) {
        bits = v[p].most(bits);  // a row past the last repeats the last, which is of this block
    }
    bits = v[0].one(bits);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        bits = max(bits, static_cast<uint32_t>(__shfl_xor(static_cast<int>(bits), o)));
    }
    if ((threadIdx.x & 63) == 0) {
        part[threadIdx.x >> 6] = bits;
    }
    __syncthreads();
    bits = max(max(part[0], part[1]), max(part[2], part[3]));
    const bool finite = bits < v[0].kInfinity;
    float most = v[0].magnitude(bits);
    if (!finite) {  // the whole workgroup
        most = 0.0f;
#pragma unroll 1
        for (int p = 0; p < 8; ++p) {
            Eight<T> one;
            load(p, one);
            most = one.most_finite(most);
        }
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) {
            most = __builtin_fmaxf(most, __shfl_xor(most, o));
        }
        if ((threadIdx.x & 63) == 0) {
            part_finite[threadIdx.x >> 6] = most;
        }
        __syncthreads();
        most = __builtin_fmaxf(__builtin_fmaxf(part_finite[0], part_finite[1]),
                               __builtin_fmaxf(part_finite[2], part_finite[3]));
    }
    const Inverse inverse(most);
    uint32_t again = finite ? 0 : 0xff;
    if (finite) {
#pragma unroll
        for (int p = 0; p < 8; ++p) {
            const int32_t r = r0 + 16 * p;
            uint2 codes;
            again |= codes8(v[p], inverse, codes) ? 0 : 1u << p;
            if (r < a.rows) {
                store8<VEC>(a.q + r * a.width, c0, a.width, codes);
            }
        }
    }
    // few: from memory again, so that the code for them is there once
    while (again != 0) {
        const int p = __builtin_ctz(again);
        again &= again - 1;
        if (r0 + 16 * p < a.rows) {
            Eight<T> one;
            load(p, one);
            store8<VEC>(a.q + (r0 + 16 * p) * a.width, c0, a.width, exact_codes8(one, inverse));
        }
    }
    if (threadIdx.x == 0) {
        a.scale[tall * wide + b] = fp8_scale(most);
    }
}

template <class T, bool VEC>
hipError_t launch_blocks(const Fp8Rows& a, hipStream_t s) {
    const int64_t wide = fp8_blocks(a.width);
    const int64_t items = a.rows * wide;
    if (a.block_rows == 1) {
        const unsigned blocks = static_cast<unsigned>(std::min<int64_t>((items + 15) / 16, 1 << 20));
        hipLaunchKernelGGL(HIP_KERNEL_NAME(fp8_rows_kernel<T, VEC>), dim3(blocks), dim3(256), 0, s, a, items,
                           static_cast<int32_t>(wide));
    } else {
        const int64_t tall = fp8_blocks(a.rows);  // under 2^16, as the grid's second axis has to be
        hipLaunchKernelGGL(HIP_KERNEL_NAME(fp8_matrix_kernel<T, VEC>),
                           dim3(static_cast<unsigned>(wide), static_cast<unsigned>(tall)), dim3(256), 0, s, a,
                           static_cast<int32_t>(wide));
    }
    return hipGetLastError();
}

template <class T>
hipError_t launch_rows(const Fp8Rows& a, hipStream_t s) {
    // sixteen bytes at a time where every row's start and end allow it
    const bool vec = reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && a.stride * static_cast<int64_t>(sizeof(T)) % 16 == 0 &&
                     a.width % 8 == 0;
    return vec ? launch_blocks<T, true>(a, s) : launch_blocks<T, false>(a, s);
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
