// lm_fp8.hip -- the C ABI of include/litemind_fp8.h but for the layers' path:
// argument checks and launches.
#include "fp8_internal.h"
#include "lm_error.h"

#include <algorithm>
#include <new>
#include <string>

#define LM_FP8_HIP(call)                                                                                     \
    do {                                                                                                     \
        const hipError_t lm_status_ = (call);                                                                \
        if (lm_status_ != hipSuccess) {                                                                      \
            return lm::set_error(LM_EHIP, std::string(#call) + ": " + hipGetErrorString(lm_status_));        \
        }                                                                                                    \
    } while (0)

namespace lm {

struct Fp8State {
    // Host memory that the grouped kernels write when an index lies outside its
    // range: read without a copy once the stream has drained.
    uint32_t* error = nullptr;
    // Sums of products whose reduced axis several workgroups share: of a fixed
    // size, so captured graphs keep its pointer. Calls on the stream take turns.
    void* workspace = nullptr;
};

void fp8_release(Fp8State* st) {
    if (st == nullptr) {
        return;
    }
    (void)hipHostFree(st->error);
    (void)hipFree(st->workspace);
    delete st;
}

int fp8_check_error(lm_context* ctx) {
    Fp8State* st = context_fp8(ctx);
    if (st == nullptr || __atomic_load_n(st->error, __ATOMIC_ACQUIRE) == 0) {
        return LM_OK;
    }
    __atomic_store_n(st->error, 0u, __ATOMIC_RELEASE);
    return set_error(LM_EKERNEL, "offsets that fall, or a row index outside the rows of an FP8 product by groups; its output is invalid");
}

}  // namespace lm

namespace {

int fail(int code, const std::string& message) { return lm::set_error(code, message); }

bool aligned(const void* p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

struct Range {
    const void* at;
    int64_t bytes;
};

// Whether an output meets an input or another output.
bool overlap(const Range& a, const Range& b) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a.at), y = reinterpret_cast<uintptr_t>(b.at);
    return a.at != nullptr && b.at != nullptr && x < y + static_cast<uintptr_t>(b.bytes) &&
           y < x + static_cast<uintptr_t>(a.bytes);
}

int64_t element_bytes(int32_t dtype) {
    return dtype == LM_DT_F32 ? 4 : dtype == LM_DT_F16 || dtype == LM_DT_BF16 ? 2 : 0;
}

constexpr int64_t kMost32 = int64_t{1} << 32;

// The sizes of a product: p's n, k, nb, kb, a_rows and rows on success.
int product_sizes(lm::Fp8Product& p, int64_t a_rows, int64_t n, int64_t k, int64_t parts) {
    if (k < 16 || k > lm::kFp8MaxInner || k % 16 != 0) {
        return fail(LM_EINVAL, "in_features must be a multiple of 16 up to 2^20");
    }
    if (n < 1 || n > (int64_t{1} << 24) || parts * n * k >= kMost32) {
        return fail(LM_EINVAL, "the weights must have 1 .. 2^24 rows and under 2^32 codes a matrix");
    }
    if (a_rows < 0 || a_rows > INT32_MAX || a_rows * k >= kMost32) {
        return fail(LM_EINVAL, "the rows must be 0 .. 2^31 - 1, with under 2^32 codes");
    }
    p.a_rows = a_rows;
    p.n = static_cast<int32_t>(n);
    p.k = static_cast<int32_t>(k);
    p.nb = static_cast<int32_t>(lm::fp8_blocks(n));
    p.kb = static_cast<int32_t>(lm::fp8_blocks(k));
    return LM_OK;
}

// The same for gate and up, whose outputs are the next product's rows.
int swiglu_sizes(lm::Fp8Product& p, int64_t a_rows, int64_t inter, int64_t k) {
    if (inter < 16 || inter > lm::kFp8MaxInner || inter % 16 != 0 || p.rows * inter >= kMost32) {
        return fail(LM_EINVAL, "inter must be a multiple of 16 up to 2^20, with under 2^32 codes");
    }
    return product_sizes(p, a_rows, inter, k, 2);
}

// The operands' pointers.
int product_inputs(lm::Fp8Product& p, const uint8_t* a, const float* a_scale, const uint8_t* w, const float* w_scale) {
    if (a == nullptr || w == nullptr || !aligned(a, 16) || !aligned(w, 16)) {
        return fail(LM_EINVAL, "rows and weights must be 16-byte aligned device memory");
    }
    if (a_scale == nullptr || w_scale == nullptr || !aligned(a_scale, 4) || !aligned(w_scale, 4)) {
        return fail(LM_EINVAL, "null or misaligned scales");
    }
    p.a = a;
    p.a_scale = a_scale;
    p.w = w;
    p.w_scale = w_scale;
    return LM_OK;
}

int product_groups(lm::Fp8Product& p, const lm_fp8_groups* g) {
    if (g == nullptr) {
        return fail(LM_EINVAL, "null groups");
    }
    if (g->groups < 1 || g->groups > lm::kFp8MaxGroups || g->rows < 0 || g->rows > INT32_MAX) {
        return fail(LM_EINVAL, "groups must be 1 .. 512, their rows 0 .. 2^31 - 1");
    }
    if (g->source == nullptr ? g->divisor != 0 : g->divisor < 1) {
        return fail(LM_EINVAL, "divisor must be positive with source, 0 without");
    }
    if (g->offsets == nullptr || !aligned(g->offsets, 4) || !aligned(g->source, 4) || !aligned(g->target, 4)) {
        return fail(LM_EINVAL, "null or misaligned offsets, or misaligned source or target");
    }
    p.groups = g->groups;
    p.divisor = g->divisor;
    p.rows = g->rows;
    p.offsets = g->offsets;
    p.source = g->source;
    p.target = g->target;
    return LM_OK;
}

// LM_EINVAL where one of the outputs meets an input or the other output.
int product_overlap(const lm::Fp8Product& p, int64_t parts, const Range& out, const Range& second) {
    const int64_t matrix = parts * p.n * p.k, scales = 4 * parts * p.nb * p.kb;
    const Range in[] = {{p.a, p.a_rows * p.k},
                        {p.a_scale, 4 * p.a_rows * p.kb},
                        {p.w, p.groups * matrix},
                        {p.w_scale, p.groups * scales},
                        {p.offsets, 4 * (int64_t{p.groups} + 1)},
                        {p.source, 4 * p.rows},
                        {p.target, 4 * p.rows}};
    for (const Range& r : in) {
        if (overlap(out, r) || overlap(second, r)) {
            return fail(LM_EINVAL, "an output overlaps an input");
        }
    }
    return overlap(out, second) ? fail(LM_EINVAL, "codes and scales overlap") : LM_OK;
}

}  // namespace

int lm::fp8_scratch(lm_context* ctx, Fp8Scratch* out) {
    Fp8State*& st = context_fp8(ctx);
    if (st == nullptr) {
        const lm::ContextInfo info = context_info(ctx);
        hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
        LM_FP8_HIP(hipStreamIsCapturing(info.stream, &capture));
        if (capture != hipStreamCaptureStatusNone) {  // an allocation would end the capture
            return fail(LM_EINVAL, "the context's first FP8 product cannot be captured: call one before");
        }
        auto* made = new Fp8State();
        hipError_t err = hipHostMalloc(reinterpret_cast<void**>(&made->error), sizeof(uint32_t),
                                       hipHostMallocMapped | hipHostMallocCoherent);
        if (err == hipSuccess) {
            err = hipMalloc(&made->workspace, kFp8WorkspaceBytes);
            made->workspace = err == hipSuccess ? made->workspace : nullptr;
        } else {
            made->error = nullptr;
        }
        if (err != hipSuccess) {
            (void)hipGetLastError();  // or the next launch would report it
            fp8_release(made);
            return fail(LM_ENOMEM, std::string("FP8 products' error word and workspace: ") + hipGetErrorString(err));
        }
        *made->error = 0;
        st = made;
    }
    *out = Fp8Scratch{st->error, st->workspace};
    return LM_OK;
}

int lm::fp8_launched(hipError_t e) {
    if (e == hipErrorInvalidConfiguration) {
        return fail(LM_EINVAL, "more than 2^22 output tiles: call it for fewer rows, groups or features at a time");
    }
    LM_FP8_HIP(e);
    return LM_OK;
}

int lm::fp8_plan_out(const Fp8Plan& plan, lm_fp8_plan* out) {
    if (plan.tiles > kFp8MaxTiles) {
        return fp8_launched(hipErrorInvalidConfiguration);
    }
    *out = lm_fp8_plan{plan.rows, plan.features, plan.shares, plan.exact ? 1 : 0, plan.tile, 0, plan.tiles};
    return LM_OK;
}

extern "C" {

int lm_fp8_quantize(lm_context* ctx, const void* x_dev, int32_t dtype, int64_t rows, int64_t width, int64_t row_stride,
                    int32_t block_rows, uint8_t* q_dev, float* scale_dev) try {
    const int64_t bytes = element_bytes(dtype);
    if (bytes == 0) {
        return fail(LM_EINVAL, "dtype must be LM_DT_F32, LM_DT_F16 or LM_DT_BF16");
    }
    if (block_rows != 1 && block_rows != LM_FP8_BLOCK) {
        return fail(LM_EINVAL, "block_rows must be 1 or 128");
    }
    const int64_t most = block_rows == 1 ? INT32_MAX : (int64_t{1} << 23) - 128;
    if (rows < 0 || rows > most || width < 1 || width > (int64_t{1} << 24) || row_stride < width ||
        row_stride > (int64_t{1} << 28)) {
        return fail(LM_EINVAL, "rows must be 0 .. 2^31 - 1 (2^23 - 128 of a matrix), width 1 .. 2^24, row_stride width .. 2^28");
    }
    if (rows == 0) {
        return ctx != nullptr ? LM_OK : fail(LM_EINVAL, "null context");
    }
    if (x_dev == nullptr || !aligned(x_dev, static_cast<uintptr_t>(bytes)) || q_dev == nullptr || !aligned(q_dev, 16) ||
        scale_dev == nullptr || !aligned(scale_dev, 4)) {
        return fail(LM_EINVAL, "null or misaligned values, codes (16 bytes) or scales");
    }
    const Range x{x_dev, ((rows - 1) * row_stride + width) * bytes}, q{q_dev, rows * width},
        scale{scale_dev, 4 * (block_rows == 1 ? rows : lm::fp8_blocks(rows)) * lm::fp8_blocks(width)};
    if (overlap(x, q) || overlap(x, scale) || overlap(q, scale)) {
        return fail(LM_EINVAL, "values, codes and scales must not overlap");
    }
    if (ctx == nullptr) {
        return fail(LM_EINVAL, "null context");
    }
    const lm::ContextInfo info = lm::context_info(ctx);
    LM_FP8_HIP(hipSetDevice(info.device));
    LM_FP8_HIP(lm::launch_fp8_quantize(
        lm::Fp8Rows{x_dev, dtype, rows, width, row_stride, block_rows, 0, q_dev, scale_dev}, info.stream));
    return LM_OK;
} catch (const std::bad_alloc&) {
    return fail(LM_ENOMEM, "host allocation failed");
}

int lm_fp8_gemm(lm_context* ctx, const uint8_t* a_dev, const float* a_scale_dev, int64_t rows, const uint8_t* w_dev,
                const float* w_scale_dev, int64_t out_features, int64_t in_features, void* out_dev,
                int32_t out_dtype) try {
    lm::Fp8Product p{};
    int rc = product_sizes(p, rows, out_features, in_features, 1);
    if (rc != LM_OK) {
        return rc;
    }
    const int64_t bytes = element_bytes(out_dtype);
    if (bytes == 0) {
        return fail(LM_EINVAL, "out_dtype must be LM_DT_F32, LM_DT_F16 or LM_DT_BF16");
    }
    p.groups = 1;
    p.rows = rows;
    p.out_rows = rows;
    p.out = out_dev;
    p.out_dtype = out_dtype;
    p.exact = out_dtype == LM_DT_F32 ? 1 : 0;
    if (rows == 0) {
        return ctx != nullptr ? LM_OK : fail(LM_EINVAL, "null context");
    }
    rc = product_inputs(p, a_dev, a_scale_dev, w_dev, w_scale_dev);
    if (rc != LM_OK) {
        return rc;
    }
    if (out_dev == nullptr || !aligned(out_dev, 16)) {
        return fail(LM_EINVAL, "the output must be 16-byte aligned device memory");
    }
    rc = product_overlap(p, 1, Range{out_dev, rows * out_features * bytes}, Range{nullptr, 0});
    if (rc != LM_OK) {
        return rc;
    }
    if (ctx == nullptr) {
        return fail(LM_EINVAL, "null context");
    }
    const lm::ContextInfo info = lm::context_info(ctx);
    LM_FP8_HIP(hipSetDevice(info.device));
    lm::Fp8Scratch sc{};
    rc = lm::fp8_scratch(ctx, &sc);
    if (rc != LM_OK) {
        return rc;
    }
    return lm::fp8_launched(lm::launch_fp8_gemm(p, sc.workspace, info.stream));
} catch (const std::bad_alloc&) {
    return fail(LM_ENOMEM, "host allocation failed");
}

int lm_fp8_grouped_gemm(lm_context* ctx, const lm_fp8_groups* groups, const uint8_t* a_dev, const float* a_scale_dev,
                        int64_t a_rows, const uint8_t* w_dev, const float* w_scale_dev, int64_t out_features,
                        int64_t in_features, void* out_dev, int64_t out_rows, int32_t out_dtype) {
    try {
        lm::Fp8Product p{};
        int rc = product_groups(p, groups);
        if (rc != LM_OK) {
            return rc;
        }
        rc = product_sizes(p, a_rows, out_features, in_features, 1);
        if (rc != LM_OK) {
            return rc;
        }
        const int64_t bytes = element_bytes(out_dtype);
        if (bytes == 0) {
            return fail(LM_EINVAL, "out_dtype must be LM_DT_F32, LM_DT_F16 or LM_DT_BF16");
        }
        if (out_rows < 0 || out_rows > INT32_MAX) {
            return fail(LM_EINVAL, "out_rows must be 0 .. 2^31 - 1");
        }
        if (p.rows == 0) {
            return ctx != nullptr ? LM_OK : fail(LM_EINVAL, "null context");
        }
        if (a_rows == 0 || out_rows == 0) {
            return fail(LM_EINVAL, "rows of groups need rows of a and of the output");
        }
        rc = product_inputs(p, a_dev, a_scale_dev, w_dev, w_scale_dev);
        if (rc != LM_OK) {
            return rc;
        }
        if (out_dev == nullptr || !aligned(out_dev, 16)) {
            return fail(LM_EINVAL, "the output must be 16-byte aligned device memory");
        }
        rc = product_overlap(p, 1, Range{out_dev, out_rows * out_features * bytes}, Range{nullptr, 0});
        if (rc != LM_OK) {
            return rc;
        }
        if (ctx == nullptr) {
            return fail(LM_EINVAL, "null context");
        }
        const lm::ContextInfo info = lm::context_info(ctx);
        LM_FP8_HIP(hipSetDevice(info.device));
        lm::Fp8Scratch sc{};
        rc = lm::fp8_scratch(ctx, &sc);
        if (rc != LM_OK) {
            return rc;
        }
        p.out = out_dev;
        p.out_rows = out_rows;
        p.out_dtype = out_dtype;
        p.exact = out_dtype == LM_DT_F32 ? 1 : 0;
        p.error = sc.error;
        return lm::fp8_launched(lm::launch_fp8_gemm(p, sc.workspace, info.stream));
    } catch (const std::bad_alloc&) {
        return fail(LM_ENOMEM, "host allocation failed");
    }
}

int lm_fp8_grouped_swiglu(lm_context* ctx, const lm_fp8_groups* groups, const uint8_t* a_dev, const float* a_scale_dev,
                          int64_t a_rows, const uint8_t* w_dev, const float* w_scale_dev, int64_t inter,
                          int64_t in_features, uint8_t* q_dev, float* scale_dev) {
    try {
        lm::Fp8Product p{};
        int rc = product_groups(p, groups);
        if (rc != LM_OK) {
            return rc;
        }
        if (p.target != nullptr) {
            return fail(LM_EINVAL, "target must be NULL: row i of the groups is row i of the codes");
        }
        rc = swiglu_sizes(p, a_rows, inter, in_features);
        if (rc != LM_OK) {
            return rc;
        }
        if (p.rows == 0) {
            return ctx != nullptr ? LM_OK : fail(LM_EINVAL, "null context");
        }
        if (a_rows == 0) {
            return fail(LM_EINVAL, "rows of groups need rows of a");
        }
        rc = product_inputs(p, a_dev, a_scale_dev, w_dev, w_scale_dev);
        if (rc != LM_OK) {
            return rc;
        }
        if (q_dev == nullptr || !aligned(q_dev, 16) || scale_dev == nullptr || !aligned(scale_dev, 4)) {
            return fail(LM_EINVAL, "null or misaligned codes (16 bytes) or scales");
        }
        rc = product_overlap(p, 2, Range{q_dev, p.rows * inter}, Range{scale_dev, 4 * p.rows * p.nb});
        if (rc != LM_OK) {
            return rc;
        }
        if (ctx == nullptr) {
            return fail(LM_EINVAL, "null context");
        }
        const lm::ContextInfo info = lm::context_info(ctx);
        LM_FP8_HIP(hipSetDevice(info.device));
        lm::Fp8Scratch sc{};
        rc = lm::fp8_scratch(ctx, &sc);
        if (rc != LM_OK) {
            return rc;
        }
        p.q = q_dev;
        p.q_scale = scale_dev;
        p.exact = 1;
        p.error = sc.error;
        return lm::fp8_launched(lm::launch_fp8_swiglu(p, info.stream));
    } catch (const std::bad_alloc&) {
        return fail(LM_ENOMEM, "host allocation failed");
    }
}

int lm_fp8_plan_gemm(int32_t groups, int64_t rows, int64_t out_features, int64_t in_features, int32_t out_dtype,
                     lm_fp8_plan* out) try {
    lm::Fp8Product p{};
    const int32_t none = 0;
    const lm_fp8_groups g{groups, 0, rows, &none, nullptr, nullptr};
    int rc = groups == 0 ? LM_OK : product_groups(p, &g);
    if (rc == LM_OK) {
        rc = product_sizes(p, groups == 0 ? rows : 1, out_features, in_features, 1);
    }
    if (rc != LM_OK) {
        return rc;
    }
    if (out == nullptr || rows < 1 || element_bytes(out_dtype) == 0) {
        return fail(LM_EINVAL, "null output, no rows, or not LM_DT_F32, LM_DT_F16 or LM_DT_BF16");
    }
    p.groups = std::max(groups, 1);
    p.rows = rows;
    p.exact = out_dtype == LM_DT_F32 ? 1 : 0;
    return lm::fp8_plan_out(lm::plan_fp8_gemm(p), out);
} catch (const std::bad_alloc&) {
    return fail(LM_ENOMEM, "host allocation failed");
}

int lm_fp8_plan_swiglu(int32_t groups, int64_t rows, int64_t inter, int64_t in_features, lm_fp8_plan* out) try {
    lm::Fp8Product p{};
    const int32_t none = 0;
    const lm_fp8_groups g{groups, 0, rows, &none, nullptr, nullptr};
    int rc = product_groups(p, &g);
    if (rc == LM_OK) {
        rc = swiglu_sizes(p, 1, inter, in_features);
    }
    if (rc != LM_OK) {
        return rc;
    }
    if (out == nullptr || rows < 1) {
        return fail(LM_EINVAL, "null output or no rows");
    }
    p.exact = 1;
    return lm::fp8_plan_out(lm::plan_fp8_swiglu(p), out);
} catch (const std::bad_alloc&) {
    return fail(LM_ENOMEM, "host allocation failed");
}

}  // extern "C"
