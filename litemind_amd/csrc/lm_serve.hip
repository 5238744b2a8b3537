// lm_serve.hip -- the C ABI of include/litemind_serving.h but for the model's
// layers (lm_attn.hip): argument checks and launches.
#include "lm_error.h"
#include "serve_internal.h"

#include <new>
#include <string>

#define LM_SERVE_HIP(call)                                                                                   \
    do {                                                                                                     \
        const hipError_t lm_status_ = (call);                                                                \
        if (lm_status_ != hipSuccess) {                                                                      \
            return lm::set_error(LM_EHIP, std::string(#call) + ": " + hipGetErrorString(lm_status_));        \
        }                                                                                                    \
    } while (0)

namespace lm {

struct ServeState {
    // Host memory that the kernels write when a table names a page outside the
    // pool: read without a copy once the stream has drained.
    uint32_t* error = nullptr;
    // Sums of blocks whose keys are shared by several workgroups, for blocks of
    // 16 and of 64 query rows (17 and 67 MB): of a fixed size each, so captured
    // graphs keep their pointers. Steps on the stream take turns.
    void* parts16 = nullptr;
    void* parts64 = nullptr;
};

void serve_release(ServeState* st) {
    if (st == nullptr) {
        return;
    }
    (void)hipHostFree(st->error);
    (void)hipFree(st->parts16);
    (void)hipFree(st->parts64);
    delete st;
}

int serve_check_error(lm_context* ctx) {
    ServeState* st = context_serve(ctx);
    if (st == nullptr || st->error == nullptr || __atomic_load_n(st->error, __ATOMIC_ACQUIRE) == 0) {
        return LM_OK;
    }
    __atomic_store_n(st->error, 0u, __ATOMIC_RELEASE);
    return set_error(LM_EKERNEL, "a block table named a page outside the pool; the attention's output is invalid");
}

}  // namespace lm

namespace {

int fail(int code, const std::string& message) { return lm::set_error(code, message); }

bool aligned(const void* p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

bool overlap(const void* a, int64_t a_bytes, const void* b, int64_t b_bytes) {
    const char* x = static_cast<const char*>(a);
    const char* y = static_cast<const char*>(b);
    return x < y + b_bytes && y < x + a_bytes;
}

// The context's serving state, and with `rows` the workspace of blocks of that
// many query rows, made at the first call that needs them (not while the stream
// is being captured: an allocation would end the capture).
int serve_state(lm_context* ctx, int rows, lm::ServeState** out, void** parts) {
    lm::ServeState*& st = lm::context_serve(ctx);
    *parts = nullptr;
    void** const at = st == nullptr || rows == 0 ? nullptr : rows == 16 ? &st->parts16 : &st->parts64;
    if (st != nullptr && (at == nullptr || *at != nullptr)) {
        *out = st;
        *parts = at == nullptr ? nullptr : *at;
        return LM_OK;
    }
    const lm::ContextInfo info = lm::context_info(ctx);
    hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
    LM_SERVE_HIP(hipStreamIsCapturing(info.stream, &capture));
    if (capture != hipStreamCaptureStatusNone) {
        return fail(LM_EINVAL, "the context's first paged attention of a kind cannot be captured: call it once before");
    }
    hipError_t err = hipSuccess;
    if (st == nullptr) {
        auto* made = new lm::ServeState();
        err = hipHostMalloc(reinterpret_cast<void**>(&made->error), sizeof(uint32_t),
                            hipHostMallocMapped | hipHostMallocCoherent);
        if (err == hipSuccess) {
            *made->error = 0;
            st = made;
        } else {
            delete made;
        }
    }
    if (err == hipSuccess && rows != 0) {
        void** const to = rows == 16 ? &st->parts16 : &st->parts64;
        err = hipMalloc(to, static_cast<size_t>(lm::paged_workspace_bytes(rows)));
        if (err != hipSuccess) {
            *to = nullptr;
        }
        *parts = *to;
    }
    if (err != hipSuccess) {
        (void)hipGetLastError();  // or the next launch would report it
        return fail(LM_ENOMEM, std::string("paged attention's workspace: ") + hipGetErrorString(err));
    }
    *out = st;
    return LM_OK;
}

int check_work(const lm_paged_step& s, int32_t heads) {
    if (s.tokens * heads > INT32_MAX / 2 ||
        !lm::paged_shares_out(s.tokens, heads, static_cast<int64_t>(s.table_width) * s.page_size)) {
        return fail(LM_EINVAL, "tokens * heads must stay under 2^30, and with the keys of a table row under 2^62");
    }
    return LM_OK;
}

}  // namespace

int lm::paged_attention_ready(lm_context* ctx, const lm_paged_step& step, int32_t heads, int32_t rank, int32_t rope) {
    ServeState* st = nullptr;
    void* parts = nullptr;
    const int rc = check_work(step, heads);
    return rc != LM_OK ? rc
                       : serve_state(ctx, paged_tiled(rank, rope) ? paged_block_rows(step.max_added, heads) : 0, &st, &parts);
}

int lm::check_step_sizes(const lm_paged_step* s) {
    if (s == nullptr) {
        return fail(LM_EINVAL, "null step");
    }
    if (s->requests < 1 || s->requests > INT32_MAX - 1 || s->tokens < 0 || s->tokens > INT32_MAX) {
        return fail(LM_EINVAL, "a step needs 1 .. 2^31 - 2 requests and 0 .. 2^31 - 1 tokens");
    }
    if (s->page_size < 16 || s->page_size > 4096 || s->page_size % 16 != 0) {
        return fail(LM_EINVAL, "page_size must be a multiple of 16 up to 4096");
    }
    if (s->pages < 1 || s->pages > INT32_MAX || s->pages * s->page_size > INT32_MAX) {
        return fail(LM_EINVAL, "the pool must hold 1 page at least and 2^31 - 1 tokens at most");
    }
    if (s->table_width < 1 || static_cast<int64_t>(s->table_width) * s->page_size > INT32_MAX) {
        return fail(LM_EINVAL, "table_width must be positive and cover at most 2^31 - 1 tokens");
    }
    if (s->max_added < 0 || s->reserved != 0) {
        return fail(LM_EINVAL, "max_added must not be negative, reserved must be 0");
    }
    return LM_OK;
}

extern "C" {

int lm_page_plan(lm_context* ctx, const lm_paged_step* step) try {
    const int rc = lm::check_step_sizes(step);
    if (rc != LM_OK) {
        return rc;
    }
    const lm_paged_step& s = *step;
    for (const void* p : {static_cast<const void*>(s.cached), static_cast<const void*>(s.added),
                          static_cast<const void*>(s.table), static_cast<const void*>(s.ring),
                          static_cast<const void*>(s.queue_in), static_cast<const void*>(s.queue_out),
                          static_cast<const void*>(s.lengths), static_cast<const void*>(s.starts),
                          static_cast<const void*>(s.info)}) {
        if (p == nullptr || !aligned(p, 4)) {
            return fail(LM_EINVAL, "a null or misaligned array of the step");
        }
    }
    if (s.tokens > 0 && (s.positions == nullptr || s.slots == nullptr || !aligned(s.positions, 4) ||
                         !aligned(s.slots, 4))) {
        return fail(LM_EINVAL, "null or misaligned positions or slots");
    }
    if (ctx == nullptr) {
        return fail(LM_EINVAL, "null context");
    }
    const lm::ContextInfo info = lm::context_info(ctx);
    LM_SERVE_HIP(hipSetDevice(info.device));
    LM_SERVE_HIP(lm::launch_page_plan(s, info.stream));
    return LM_OK;
} catch (const std::bad_alloc&) {
    return fail(LM_ENOMEM, "host allocation failed");
}

int lm_paged_attention(lm_context* ctx, const lm_paged_step* step, const void* q_dev, const void* pool_dev,
                       int32_t dtype, int32_t heads, int32_t rank, int32_t rope, float scale, void* out_dev) {
    try {
        int rc = lm::check_step_sizes(step);
        if (rc != LM_OK) {
            return rc;
        }
        if (dtype != LM_DT_F16 && dtype != LM_DT_BF16) {
            return fail(LM_EINVAL, "dtype must be LM_DT_F16 or LM_DT_BF16");
        }
        if (heads < 1 || rank < 8 || rank > 1024 || rank % 8 != 0 || rope < 0 || rope > 256 || rope % 8 != 0) {
            return fail(LM_EINVAL, "heads must be positive, rank a multiple of 8 up to 1024, rope of 8 up to 256");
        }
        if (!(scale - scale == 0.0f)) {
            return fail(LM_EINVAL, "scale must be finite");
        }
        const lm_paged_step& s = *step;
        if (s.tokens == 0) {
            return ctx != nullptr ? LM_OK : fail(LM_EINVAL, "null context");
        }
        rc = check_work(s, heads);
        if (rc != LM_OK) {
            return rc;
        }
        if (s.table == nullptr || s.lengths == nullptr || s.starts == nullptr || !aligned(s.table, 4) ||
            !aligned(s.lengths, 4) || !aligned(s.starts, 4)) {
            return fail(LM_EINVAL, "a null or misaligned array of the step");
        }
        for (const void* p : {q_dev, pool_dev, static_cast<const void*>(out_dev)}) {
            if (p == nullptr || !aligned(p, 16)) {
                return fail(LM_EINVAL, "queries, pool and output must be 16-byte aligned device memory");
            }
        }
        const int64_t width = rank + rope, rows = s.tokens * heads;
        const int64_t pool_bytes = 2 * s.pages * s.page_size * width;
        if (overlap(out_dev, 2 * rows * rank, q_dev, 2 * rows * width) ||
            overlap(out_dev, 2 * rows * rank, pool_dev, pool_bytes)) {
            return fail(LM_EINVAL, "out_dev overlaps the queries or the pool");
        }
        if (ctx == nullptr) {
            return fail(LM_EINVAL, "null context");
        }
        const lm::ContextInfo info = lm::context_info(ctx);
        LM_SERVE_HIP(hipSetDevice(info.device));
        lm::ServeState* st = nullptr;
        void* parts = nullptr;
        rc = serve_state(ctx, lm::paged_tiled(rank, rope) ? lm::paged_block_rows(s.max_added, heads) : 0, &st, &parts);
        if (rc != LM_OK) {
            return rc;
        }
        lm::PagedAttention a;
        a.view = lm::PagedView{s.table, s.lengths, s.starts, s.pages, static_cast<int32_t>(s.requests),
                               static_cast<int32_t>(s.tokens), s.page_size, s.table_width, st->error};
        a.q = q_dev;
        a.pool = pool_dev;
        a.out = out_dev;
        a.bf16 = dtype == LM_DT_BF16 ? 1 : 0;
        a.heads = heads;
        a.rank = rank;
        a.rope = rope;
        a.max_added = s.max_added;
        a.scale = scale;
        LM_SERVE_HIP(lm::launch_paged_attention(a, parts, info.stream));
        return LM_OK;
    } catch (const std::bad_alloc&) {
        return fail(LM_ENOMEM, "host allocation failed");
    }
}

int lm_sample(lm_context* ctx, const float* logits_dev, int64_t rows, int64_t vocab, int64_t row_stride,
              const lm_sampling* settings_dev, const float* uniform_dev, int32_t* token_dev, float* probability_dev) try {
    if (rows < 0 || rows > INT32_MAX || vocab < 1 || vocab > (int64_t{1} << 24) || row_stride < vocab) {
        return fail(LM_EINVAL, "rows must be 0 .. 2^31 - 1, vocab 1 .. 2^24, row_stride at least vocab");
    }
    if (rows == 0) {
        return ctx != nullptr ? LM_OK : fail(LM_EINVAL, "null context");
    }
    for (const void* p : {static_cast<const void*>(logits_dev), static_cast<const void*>(settings_dev),
                          static_cast<const void*>(uniform_dev), static_cast<const void*>(token_dev)}) {
        if (p == nullptr || !aligned(p, 4)) {
            return fail(LM_EINVAL, "null or misaligned logits, settings, random numbers or tokens");
        }
    }
    if (!aligned(probability_dev, 4)) {
        return fail(LM_EINVAL, "misaligned probabilities");
    }
    if (ctx == nullptr) {
        return fail(LM_EINVAL, "null context");
    }
    const lm::ContextInfo info = lm::context_info(ctx);
    LM_SERVE_HIP(hipSetDevice(info.device));
    lm::SampleArgs a;
    a.logits = logits_dev;
    a.rows = rows;
    a.vocab = vocab;
    a.stride = row_stride;
    a.settings = settings_dev;
    a.uniform = uniform_dev;
    a.token = token_dev;
    a.probability = probability_dev;
    LM_SERVE_HIP(lm::launch_sample(a, info.stream));
    return LM_OK;
} catch (const std::bad_alloc&) {
    return fail(LM_ENOMEM, "host allocation failed");
}

}  // extern "C"
