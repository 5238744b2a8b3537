// serve_internal.h -- what the kernels of the paged cache and of sampling
// (k_pages.hip, k_paged.hip, k_sample.hip) share with the ABI over them
// (lm_serve.hip, lm_attn.hip).
#pragma once

#include "litemind_serving.h"
#include "lm_internal.h"

namespace lm {

// A planned step as the attention reads it: lm_paged_step's device arrays, with
// the sizes that every kernel checks what it reads against.
struct PagedView {
    const int32_t* table;
    const int32_t* lengths;
    const int32_t* starts;
    int64_t pages;
    int32_t requests, tokens, page_size, table_width;
    uint32_t* error;  // set to 1 (host memory) where a page id lies outside the pool
};

// Tokens that request r has in its pages and adds, within the arrays' bounds:
// rows first .. first + added - 1 of the step, which see keys 0 .. cached + i.
struct PagedRequest {
    int32_t first, added, cached;
};
__device__ inline PagedRequest paged_request(const PagedView& v, int32_t r) {
    PagedRequest q;
    const int64_t room = static_cast<int64_t>(v.table_width) * v.page_size;
    const int32_t length = static_cast<int32_t>(min(static_cast<int64_t>(v.lengths[r]), room));
    q.first = min(max(v.starts[r], 0), v.tokens);
    const int32_t end = min(max(v.starts[r + 1], q.first), v.tokens);
    q.added = max(0, min(end - q.first, length));
    q.cached = length - q.added;
    return q;
}

// A page id of the table: ids outside the pool read page 0 and set the error word.
__device__ inline int64_t checked_page(const PagedView& v, int32_t page) {
    if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(v.pages)) {
        __hip_atomic_store(v.error, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
        return 0;
    }
    return page;
}

hipError_t launch_page_plan(const lm_paged_step& step, hipStream_t s);

// Attention of the step's tokens: q [tokens][heads][rank + rope], pool
// [pages][page_size][rank + rope], out [tokens][heads][rank], BF16 or fp16.
struct PagedAttention {
    PagedView view;
    const void* q;
    const void* pool;
    void* out;
    int32_t bf16;
    int32_t heads, rank, rope;
    int32_t max_added;
    float scale;
};
// Whether rows of this width go to the matrix cores, in blocks of
// paged_block_rows() query rows (16 or 64) that need a workspace of
// paged_workspace_bytes(), whatever the step.
bool paged_tiled(int32_t rank, int32_t rope);
int paged_block_rows(int32_t max_added, int32_t heads);
// Whether the costs of a step's blocks fit in 64 bits (room: tokens that a table row covers).
bool paged_shares_out(int64_t tokens, int32_t heads, int64_t room);
int64_t paged_workspace_bytes(int rows);
hipError_t launch_paged_attention(const PagedAttention& a, void* workspace, hipStream_t s);

struct SampleArgs {
    const float* logits;
    int64_t rows, vocab, stride;
    const lm_sampling* settings;
    const float* uniform;
    int32_t* token;
    float* probability;  // or null
};
hipError_t launch_sample(const SampleArgs& a, hipStream_t s);

// ---- the model's layers over pages (k_latent.hip) ----
struct LatentArgs {
    int64_t tokens;
    int32_t heads, nope, rope, rank;
    const float* q;    // [tokens][heads][nope + rope]
    const float* lat;  // [tokens][rank + rope]
    const float* norm; // [rank]
    float eps;
    const int32_t* positions;
    const int32_t* slots;
    const int32_t* live;  // the number of new tokens
    int64_t max_positions;
    const float* cos_t;
    const float* sin_t;
    _Float16* pool;
    int64_t pool_rows;
    _Float16* q16;  // [tokens][heads][rank + rope]: the rope part is written
};
hipError_t launch_latent_rows(const LatentArgs& a, hipStream_t s);
// Zeros into the rows of [tokens][width] from live[0] on.
hipError_t launch_clear_rows(float* rows, const int32_t* live, int64_t tokens, int32_t width, hipStream_t s);
hipError_t launch_absorb(const _Float16* kvb, _Float16* out, int32_t heads, int32_t nope, int32_t vh, int32_t rank,
                         hipStream_t s);
// out[t][h][n] = sum_k x[t][h][k] w[h w_head + w_first + n][k], K % 32 == 0, N % 16 == 0
struct HeadsArgs {
    int64_t tokens;
    int32_t heads, K, N;
    const void* x;  // fp32 or fp16
    int32_t x_f32;
    int64_t x_token, x_head;
    const _Float16* w;  // panels [w_rows][K]
    int64_t w_rows;
    int32_t w_head, w_first;
    _Float16* out;
    int32_t out_panels;  // panels [tokens][heads N], or rows:
    int64_t out_token, out_head;
    const int32_t* live;  // rows from here on give zeros (null: none)
};
hipError_t launch_heads(const HeadsArgs& a, hipStream_t s);

// ---- services of lm_serve.hip ----
// LM_OK where a step's sizes can be relied on.
int check_step_sizes(const lm_paged_step* step);
// Whether lm_paged_attention can run a step of good sizes: its work fits in 64 bits,
// its workspace is made.
int paged_attention_ready(lm_context* ctx, const lm_paged_step& step, int32_t heads, int32_t rank, int32_t rope);
struct ServeState;
ServeState*& context_serve(lm_context* ctx);
void serve_release(ServeState* st);
// LM_EKERNEL, once, where a kernel met a page id outside the pool.
int serve_check_error(lm_context* ctx);

}  // namespace lm
