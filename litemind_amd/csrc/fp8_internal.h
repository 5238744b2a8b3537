// fp8_internal.h -- what the FP8 kernels (k_fp8.hip, k_fp8_rows.hip) share with
// the ABI over them (lm_fp8.hip).
#pragma once

#include "litemind_fp8.h"
#include "lm_internal.h"

namespace lm {

constexpr int kFp8Block = LM_FP8_BLOCK;
constexpr float kFp8Largest = 448.0f;      // of e4m3
constexpr int kFp8MaxGroups = 512;
constexpr int64_t kFp8MaxInner = 1 << 20;  // reduced channels of a product

inline int64_t fp8_blocks(int64_t n) { return (n + kFp8Block - 1) / kFp8Block; }

struct Fp8Rows {
    const void* x;
    int32_t dtype;  // LM_DT_F32, LM_DT_F16 or LM_DT_BF16
    int64_t rows, width, stride;
    int32_t block_rows;  // 1 or 128
    int32_t group;       // of a matrix: 0, or its rows lie in groups of so many (a power of two), as many others between
    uint8_t* q;
    float* scale;
};
hipError_t launch_fp8_quantize(const Fp8Rows& a, hipStream_t s);

// A product of FP8 rows with the matrix of each group.
struct Fp8Product {
    const uint8_t* a;        // [a_rows][k]
    const float* a_scale;    // [a_rows][kb]
    const uint8_t* w;        // [groups][n][k], SwiGLU: [groups][2][n][k]
    const float* w_scale;    // [groups][nb][kb], SwiGLU: [groups][2][nb][kb]
    int64_t a_rows;
    int32_t n, k, nb, kb;    // SwiGLU: n is one of the two products' features
    int32_t groups;
    int32_t divisor;         // of source
    int64_t rows;
    const int32_t* offsets;  // [groups + 1], or null: one group of all rows
    const int32_t* source;   // or null
    const int32_t* target;   // or null
    void* out;               // [out_rows][n] of out_dtype
    int64_t out_rows;
    int32_t out_dtype;
    uint8_t* q;              // SwiGLU: [rows][n] codes
    float* q_scale;          // SwiGLU: [rows][nb]
    int32_t exact;           // 1: fp32 sums; 0: large tiles on the FP8 matrix cores
    uint32_t* error;         // set to 1 (host memory) by an index outside its range; null without offsets
};
// Sums of products whose reduced axis several workgroups share.
constexpr int64_t kFp8WorkspaceBytes = 32 << 20;
// The kernel that a product takes.
constexpr int64_t kFp8MaxTiles = int64_t{1} << 22;  // of a launch: 2^31 threads
struct Fp8Plan {
    int32_t tile;            // which of the kernels of tiles, -1: the kernel of few rows
    int32_t rows, features;  // of a tile (SwiGLU: features of gate and up each)
    int32_t shares;          // workgroups that share a tile's reduced axis
    bool exact;              // fp32 sums
    int64_t tiles;           // that the launch has room for: refused past kFp8MaxTiles
};
Fp8Plan plan_fp8_gemm(const Fp8Product& p, const Fp8Product* beside = nullptr);
Fp8Plan plan_fp8_swiglu(const Fp8Product& p, const Fp8Product* beside = nullptr);
// `beside`: another product of the same kind without offsets, in the same launch
// (p has offsets then, and neither exact sums but SwiGLU's).
hipError_t launch_fp8_gemm(const Fp8Product& p, void* workspace, hipStream_t s, const Fp8Product* beside = nullptr);
hipError_t launch_fp8_swiglu(const Fp8Product& p, hipStream_t s, const Fp8Product* beside = nullptr);

#if defined(__HIPCC__)
// The scale of a block whose finite values' largest magnitude is `most`.
__device__ inline float fp8_scale(float most) { return __builtin_fmaxf(most / kFp8Largest, 0x1p-126f); }

// The codes of four values already divided by their scale, the first in the
// lowest byte.  |v| <= 448 (1 + 2^-21), which rounds to 448.
__device__ inline uint32_t fp8_pack4_finite(float a, float b, float c, float d) {
    const int low = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, low, true));
}
// The same, NaN too.  The conversion makes it 0xff: bytes of magnitude 0x7f, the
// only ones that 1 carries into their sign bit, lose their sign.
__device__ inline uint32_t fp8_pack4(float a, float b, float c, float d) {
    const uint32_t v = fp8_pack4_finite(a, b, c, d);
    return v & ~(((v & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u);
}

// A value with infinities made NaN, and its magnitude, 0 where it is not finite.
__device__ inline float fp8_finite_or_nan(float x) { return x - x == 0.0f ? x : __builtin_nanf(""); }
__device__ inline float fp8_magnitude(float x) { return x - x == 0.0f ? __builtin_fabsf(x) : 0.0f; }
#endif

// ---- services of lm_fp8.hip ----
struct Fp8State;
Fp8State*& context_fp8(lm_context* ctx);
void fp8_release(Fp8State* st);
// What products need of the context, made at its first call (not while the stream
// is being captured).
struct Fp8Scratch {
    uint32_t* error;
    void* workspace;
};
int fp8_scratch(lm_context* ctx, Fp8Scratch* out);
// The status of a product's launch.
int fp8_launched(hipError_t e);
// A plan as the ABI gives it, LM_EINVAL where the product would be.
int fp8_plan_out(const Fp8Plan& plan, lm_fp8_plan* out);
// LM_EKERNEL, once, where a kernel met an index outside its range.
int fp8_check_error(lm_context* ctx);

}  // namespace lm
