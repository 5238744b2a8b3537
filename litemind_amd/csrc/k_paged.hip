// k_paged.hip -- attention of the requests' new tokens over a latent cache in
// pages (litemind_serving.h, lm_paged_attention).
//
// Per token t of request r at position p and per head h, with pool rows
// (c_j, k_j) and queries absorbed into the latent space:
//     s_j = scale q . (c_j, k_j), j <= p;   out = sum_j softmax(s)_j c_j
// All heads read the same rows, so the query rows of a request, token by token
// and head by head, are one matrix Q against K = (c, k) and V = c: S^T = K Q^T
// leaves a lane the scores of one query row, running maximum and sum are one
// value per lane, and the lane's weights are already the B operand of
// out^T = V^T P^T, whose order of keys is free. V^T is read from the row-major
// tile by transposing LDS reads. Scores never leave the registers.
//
// Rows of 576 values (rank 512, rope 64: DeepSeek-V2's) go to the matrix cores,
// in blocks of query rows of one request:
//   few rows (paged_rows16_kernel): 16 rows, each wave on key tiles of its own
//   many (paged_rows128_kernel): 128 rows, 32 per wave, tiles shared by the waves
// Any other widths take paged_any_kernel.
//
// The blocks' key tiles are shared out evenly: the grid's workgroups cut the
// line of all blocks' costs into equal pieces, found from the lengths on the
// GPU, so neither lengths nor the cut pass through the host. A block cut by a
// border leaves unnormalised sums, which paged_join_kernel adds in order.
#include "serve_internal.h"

#include <algorithm>
#include <cmath>

namespace lm {
namespace {

typedef __bf16 bf16;
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef short short8v __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) short4v lds_short4;

constexpr int kRank = 512, kRope = 64, kWidth = kRank + kRope;
constexpr int kRowBytes = kWidth * 2;        // 1152
constexpr int kUnits = kRowBytes / 16;       // 16-byte units of a row
constexpr int kTile = 32;                    // keys of a tile
constexpr int kTileBytes = kTile * kRowBytes;
constexpr int kGrid = 256;                   // workgroups that share out the tiles: one per CU
constexpr float kNone = -__builtin_inff();

template <class E>
struct Half;
template <>
struct Half<_Float16> {
    typedef half8 vec8;
    typedef half4 vec4;
    static __device__ f32x4 mfma16(vec8 a, vec8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
    static __device__ f32x16 mfma32(vec8 a, vec8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Half<bf16> {
    typedef bf16x8 vec8;
    typedef bf16x4 vec4;
    static __device__ f32x4 mfma16(vec8 a, vec8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    static __device__ f32x16 mfma32(vec8 a, vec8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
};

// ---- sharing out the tiles ----
// Block b of a request (rows b M .. of its added heads rows) costs the keys that
// its last token sees, as a line in b: cached + kExtra + (b + 1) M / heads, in
// whole numbers below. kExtra stands for what a block costs besides its tiles.
constexpr int kExtra = 64;
// Cost per workgroup below which fewer take part.
constexpr int kLeast = 128;

struct Shares {
    int32_t heads, rows;  // rows: M
    __device__ int32_t blocks(const PagedRequest& r) const {
        return static_cast<int32_t>((static_cast<int64_t>(r.added) * heads + rows - 1) / rows);
    }
    // Cost of the request's first b blocks.
    __device__ int64_t cost(const PagedRequest& r, int32_t b) const {
        return static_cast<int64_t>(b) * (r.cached + kExtra) + static_cast<int64_t>(b) * (b + 1) / 2 * rows / heads;
    }
    // Tiles of block b.
    __device__ int32_t tiles(const PagedRequest& r, int32_t b) const {
        const int64_t last = min(static_cast<int64_t>(b + 1) * rows, static_cast<int64_t>(r.added) * heads) - 1;
        return (r.cached + static_cast<int32_t>(last / heads) + kTile) / kTile;
    }
};

// A workgroup's piece of the line, begin .. end, of `total` in `parts` pieces.
struct Piece {
    int64_t total;
    int64_t begin, end;
    int32_t parts;
    int32_t request;  // that `begin` lies in
    int64_t base;     // cost of the requests before it
};
__device__ inline int64_t border(int64_t total, int32_t parts, int32_t g) {
    return total / parts * g + total % parts * g / parts;
}

// Every thread of the 256-thread workgroup calls it. Threads take stretches of
// requests; `scratch` (8 + 3 words of 64 bits) passes the sums.
__device__ inline Piece find_piece(const PagedView& v, const Shares& sh, int32_t g, int64_t* scratch) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int32_t per = (v.requests + 255) / 256;
    const int32_t r0 = min(tid * per, v.requests), r1 = min(r0 + per, v.requests);
    int64_t own = 0;
    for (int32_t r = r0; r < r1; ++r) {
        const PagedRequest q = paged_request(v, r);
        own += sh.cost(q, sh.blocks(q));
    }
    int64_t sum = own;
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t up = __shfl_up(sum, o);
        sum += lane >= o ? up : 0;
    }
    if (lane == 63) {
        scratch[wave] = sum;
    }
    __syncthreads();
    int64_t before = sum - own, total = 0;
    for (int w = 0; w < 4; ++w) {
        before += w < wave ? scratch[w] : 0;
        total += scratch[w];
    }
    Piece p;
    p.total = total;
    p.parts = static_cast<int32_t>(max(int64_t{1}, min(static_cast<int64_t>(kGrid), total / kLeast)));
    p.begin = g < p.parts ? border(total, p.parts, g) : total;
    p.end = g < p.parts ? border(total, p.parts, g + 1) : total;
    if (p.begin >= before && p.begin < before + own) {
        for (int32_t r = r0; r < r1; ++r) {
            const PagedRequest q = paged_request(v, r);
            const int64_t c = sh.cost(q, sh.blocks(q));
            if (p.begin < before + c) {
                scratch[4] = r;
                scratch[5] = before;
                break;
            }
            before += c;
        }
    }
    __syncthreads();
    p.request = static_cast<int32_t>(scratch[4]);
    p.base = scratch[5];
    return p;
}

// A stretch of one block's tiles.
struct Segment {
    PagedRequest req;
    int32_t request, block;
    int32_t tile0, tile1;
    bool begins, ends;    // the block begins and ends in this piece
    int32_t parts_after;  // pieces after this one that hold more of the block
};

// Walks a piece's segments.
struct Walk {
    Piece p;
    Shares sh;
    PagedRequest req;
    int32_t request, block, blocks;
    int64_t at;  // cost at the block's begin
    __device__ void start(const PagedView& v) {
        request = p.request;
        req = paged_request(v, request);
        blocks = sh.blocks(req);
        // the block that `begin` lies in: the last whose cost line starts at or before it
        int32_t lo = 0, hi = blocks;
        while (hi - lo > 1) {
            const int32_t mid = lo + (hi - lo) / 2;
            if (p.base + sh.cost(req, mid) <= p.begin) {
                lo = mid;
            } else {
                hi = mid;
            }
        }
        block = lo;
        at = p.base + sh.cost(req, lo);
    }
    __device__ bool next(const PagedView& v, Segment& s) {
        if (at >= p.end) {
            return false;
        }
        while (block >= blocks) {  // (only where `at` is below `end`: a later request has blocks)
            ++request;
            req = paged_request(v, request);
            blocks = sh.blocks(req);
            block = 0;
        }
        const int64_t cost = sh.cost(req, block + 1) - sh.cost(req, block);
        s.req = req;
        s.request = request;
        s.block = block;
        const int32_t tiles = sh.tiles(req, block);
        s.begins = p.begin <= at;
        s.ends = p.end >= at + cost;
        s.tile0 = s.begins ? 0 : static_cast<int32_t>((p.begin - at) * tiles / cost);
        s.tile1 = s.ends ? tiles : static_cast<int32_t>((p.end - at) * tiles / cost);
        s.parts_after = 0;
        if (s.begins && !s.ends) {
            int32_t g = static_cast<int32_t>(blockIdx.x) + 1;
            while (g < p.parts && border(p.total, p.parts, g) < at + cost) {
                ++g;
            }
            s.parts_after = g - static_cast<int32_t>(blockIdx.x) - 1;
        }
        at += cost;
        ++block;
        return true;
    }
};

// Sums of cut blocks. Workgroup g leaves those of a block that began in an
// earlier piece in slot 2 g, those of one that began in its own in slot 2 g + 1,
// with a head that says what follows.
struct PartHead {
    int64_t row0;   // first output row of the block
    int32_t rows;   // its rows; 0: nothing was cut here
    int32_t after;  // slots 2 (g + 1), 2 (g + 2), .. that hold the rest
};
struct Parts {
    float* sums;      // [2 kGrid][M][512], unnormalised
    float* stats;     // [2 kGrid][M][2] maximum (times c) and total
    PartHead* heads;  // [kGrid]
};

struct TileArgs {
    PagedView view;
    const void* q;
    const void* pool;
    void* out;
    int32_t heads;
    int32_t negative;  // the scale is negative: the queries change sign
    uint32_t page_mul; // 2^32 / (page_size / 16), rounded up
    float c;           // |scale| log2(e)
    Parts parts;
};

// Where 16-byte unit u of row r lies in a tile in LDS. A 16-lane group of a key
// read takes one unit of 16 rows, a transposing read two or four neighbouring
// units of eight or four rows: with the unit's low three bits XORed by the
// reversed bits of r / 2, and rows 8 units apart modulo the 16 that the banks
// hold, all are free of conflicts.
__device__ inline int swizzle(int r) {
    const int k = (r >> 1) & 7;
    return (k & 1) << 2 | (k & 2) | k >> 2;
}
__device__ inline int unit_at(int r, int u) { return r * kRowBytes + ((u ^ swizzle(r)) << 4); }

// The pages of one request's keys, 64 table entries at a time in the lanes.
struct PageWalk {
    const int32_t* row;  // the request's table row
    int32_t base;        // first entry held; a multiple of 64, or -1
    int32_t held;        // this lane's
    __device__ void start(const PagedView& v, int32_t request) {
        row = v.table + static_cast<int64_t>(request) * v.table_width;
        base = -1;
    }
    // Pool row of key (a multiple of 16; the 15 after it lie in the same page).
    __device__ int64_t at(const PagedView& v, uint32_t page_mul, int32_t key) {
        const uint32_t d = static_cast<uint32_t>(v.page_size) / 16, n = static_cast<uint32_t>(key) / 16;
        uint32_t page = __umulhi(n, page_mul);
        if (d == 1) {
            page = n;
        } else if (page * d > n) {
            --page;
        }
        const int32_t from = static_cast<int32_t>(page & ~63u);
        if (from != base) {
            base = from;
            const int32_t i = from + static_cast<int32_t>(threadIdx.x & 63);
            held = row[min(i, v.table_width - 1)];
        }
        const int32_t id = __builtin_amdgcn_readlane(held, static_cast<int>(page & 63));
        return checked_page(v, id) * v.page_size + static_cast<int64_t>(n - page * d) * 16;
    }
};

// ---- few rows ----
// 16 query rows, four waves. A wave takes every fourth tile of the segment into
// a buffer of its own, without a barrier: S^T of 2 x 18 and out^T of 32 products
// of 16 x 16 x 32 a tile. The waves' sums meet in LDS at the segment's end.
constexpr int kRows16 = 16;

template <class E>
__global__ __launch_bounds__(256) void paged_rows16_kernel(const TileArgs a) {
    using H = Half<E>;
    typedef typename H::vec8 vec8;
    __shared__ __align__(16) char tiles[4][kTileBytes];
    __shared__ float stats[4][kRows16][2];
    __shared__ int64_t scratch[8];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, grp = lane >> 4;
    Walk walk;
    walk.sh = Shares{a.heads, kRows16};
    walk.p = find_piece(a.view, walk.sh, blockIdx.x, scratch);
    if (tid == 0) {
        a.parts.heads[blockIdx.x].rows = 0;
    }
    if (walk.p.begin >= walk.p.end) {
        return;
    }
    walk.start(a.view);
    char* const tile = tiles[wave];
    // Loads: 16 rows are 18 loads of 64 units; load j's lane takes position
    // 64 j + lane, row and unit as below.
    auto place = [&](int j, int& row, int& unit) {
        const int at = 64 * j + lane;
        row = at / kUnits;
        unit = (at - row * kUnits) ^ swizzle(row);
    };
    unsigned from[18];
#pragma unroll
    for (int j = 0; j < 18; ++j) {
        int row, unit;
        place(j, row, unit);
        from[j] = static_cast<unsigned>(row * kRowBytes + unit * 16);
    }
    Segment s;
    while (walk.next(a.view, s)) {
        const int64_t row0 = static_cast<int64_t>(s.req.first) * a.heads + static_cast<int64_t>(s.block) * kRows16;
        const int rows = static_cast<int>(min(static_cast<int64_t>(kRows16),
                                              static_cast<int64_t>(s.req.added) * a.heads - s.block * int64_t{kRows16}));
        const int32_t keys = s.req.cached + s.req.added;
        // this lane's query row; the last key that it sees, and that all rows see
        const int own = min(col, rows - 1);
        const int32_t sees = s.req.cached + static_cast<int32_t>((s.block * int64_t{kRows16} + own) / a.heads);
        const int32_t all_see = s.req.cached + static_cast<int32_t>(s.block * int64_t{kRows16} / a.heads);
        vec8 q[18];
        {
            const E* const from_q = static_cast<const E*>(a.q) + (row0 + own) * kWidth + 8 * grp;
#pragma unroll
            for (int ks = 0; ks < 18; ++ks) {
                q[ks] = *reinterpret_cast<const vec8*>(from_q + 32 * ks);
            }
            if (a.negative) {
#pragma unroll
                for (int ks = 0; ks < 18; ++ks) {
                    q[ks] = -q[ks];
                }
            }
        }
        PageWalk pages;
        pages.start(a.view, s.request);
        f32x4 o[32] = {};
        float m = kNone, l = 0.0f;
        for (int32_t t = s.tile0 + wave; t < s.tile1; t += 4) {
            // the tile before has been read
            __builtin_amdgcn_s_waitcnt(0xc07f);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int32_t key = t * kTile + 16 * half, last = keys - 1;
                const int32_t first = min(key, last & ~15);
                const char* const base =
                    static_cast<const char*>(a.pool) + pages.at(a.view, a.page_mul, first) * kRowBytes;
                const __amdgpu_buffer_rsrc_t res =
                    __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, 16 * kRowBytes, kBufferWord3);
                char* const to = tile + half * 16 * kRowBytes;
                if (key + 15 <= last) {
#pragma unroll
                    for (int j = 0; j < 18; ++j) {
                        buffer_lds16(res, to + j * 1024, from[j], 0);
                    }
                } else {  // rows past the last key: the last key's once more
#pragma unroll
                    for (int j = 0; j < 18; ++j) {
                        int row, unit;
                        place(j, row, unit);
                        const int r = min(key + row, last) - first;
                        buffer_lds16(res, to + j * 1024, static_cast<unsigned>(r * kRowBytes + unit * 16), 0);
                    }
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_waitcnt(0x0070 | 0x0F00);  // vmcnt(0)
            __builtin_amdgcn_sched_barrier(0);
            f32x4 sc[2] = {};
#pragma unroll
            for (int ks = 0; ks < 18; ++ks) {
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) {
                    const vec8 k = *reinterpret_cast<const vec8*>(tile + unit_at(16 * kb + col, 4 * ks + grp));
                    sc[kb] = H::mfma16(k, q[ks], sc[kb]);
                }
            }
            // register e of sc[kb]: key 32 t + 16 kb + 4 grp + e
            bool guard = false;
            uint32_t bad = 0;  // bit 4 kb + e: a key that some row must not see is not finite
            if (t * kTile + kTile - 1 > all_see) {
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float v = sc[kb][e];
                        const uint64_t odd = __ballot(!(v - v == 0.0f));
                        bad |= (odd >> (16 * grp) & 0xffff) != 0 ? 1u << (4 * kb + e) : 0u;
                        if (t * kTile + 16 * kb + 4 * grp + e > sees) {
                            sc[kb][e] = kNone;
                        }
                    }
                }
                guard = __any(bad != 0);
            }
            float top = kNone;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                top = fmaxf(top, fmaxf(sc[0][e], sc[1][e]));
            }
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            const float up = fmaxf(m, top);
            if (__any(up > m)) {
                const float alpha = up == kNone ? 1.0f : __builtin_amdgcn_exp2f((m - up) * a.c);
                l *= alpha;
#pragma unroll
                for (int ct = 0; ct < 32; ++ct) {
                    o[ct] *= alpha;
                }
                m = up;
            }
            const float mc = m == kNone ? 0.0f : m * a.c;
            vec8 p;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i / 4][i % 4], a.c, -mc));
                l += w;
                p[i] = static_cast<E>(w);
            }
            const int vrow = 4 * grp + (col >> 2), vlow = (col & 3) >> 1, vbyte = (col & 1) * 8;
#pragma unroll
            for (int ct = 0; ct < 32; ++ct) {
                short8v v;
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) {
                    const short4v part = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (lds_short4*)(tile + unit_at(16 * kb + vrow, 2 * ct + vlow) + vbyte));
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        v[4 * kb + e] = part[e];
                    }
                }
                if (guard) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        v[i] = (bad >> i & 1) != 0 ? short{0} : v[i];
                    }
                }
                o[ct] = H::mfma16(__builtin_bit_cast(vec8, v), p, o[ct]);
            }
        }
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        // join the waves: o[ct] register e is channel 16 ct + 4 grp + e of row `col`
        __syncthreads();
        float* const mine = reinterpret_cast<float*>(tile);
#pragma unroll
        for (int ct = 0; ct < 32; ++ct) {
            *reinterpret_cast<f32x4*>(mine + col * kRank + ((16 * ct + 4 * grp) ^ (col << 2 & 28))) = o[ct];
        }
        if (grp == 0) {
            stats[wave][col][0] = m == kNone ? kNone : m * a.c;
            stats[wave][col][1] = l;
        }
        __syncthreads();
        const bool whole = s.begins && s.ends;
        const int slot = 2 * static_cast<int>(blockIdx.x) + (s.begins ? 1 : 0);
        for (int i = tid; i < rows * (kRank / 4); i += 256) {
            const int r = i / (kRank / 4), ch = i % (kRank / 4) * 4;
            float high = kNone, total = 0.0f;
            for (int w = 0; w < 4; ++w) {
                high = fmaxf(high, stats[w][r][0]);
            }
            f32x4 sum = {};
            for (int w = 0; w < 4; ++w) {
                const float weight = stats[w][r][0] == kNone ? 0.0f : __builtin_amdgcn_exp2f(stats[w][r][0] - high);
                total = __builtin_fmaf(weight, stats[w][r][1], total);
                const f32x4 v = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(tiles[w]) + r * kRank +
                                                                (ch ^ (r << 2 & 28)));
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    sum[e] = __builtin_fmaf(weight, v[e], sum[e]);
                }
            }
            if (whole) {
                typename H::vec4 out;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    out[e] = static_cast<E>(sum[e] / total);
                }
                *reinterpret_cast<typename H::vec4*>(static_cast<E*>(a.out) + (row0 + r) * kRank + ch) = out;
            } else {
                *reinterpret_cast<f32x4*>(a.parts.sums + (static_cast<int64_t>(slot) * kRows16 + r) * kRank + ch) = sum;
                if (ch == 0) {
                    float* const st = a.parts.stats + (static_cast<int64_t>(slot) * kRows16 + r) * 2;
                    st[0] = high;
                    st[1] = total;
                }
            }
        }
        if (s.begins && !s.ends && tid == 0) {
            a.parts.heads[blockIdx.x] = PartHead{row0, rows, s.parts_after};
        }
        __syncthreads();
    }
}

// The parts of cut blocks added up: workgroup (g, y) takes rows y, y + gridDim.y, ..
// of the block that piece g began and did not end. 64 lanes hold 512 channels,
// the four waves alternate parts.
template <class E, int M>
__global__ __launch_bounds__(256) void paged_join_kernel(const TileArgs a) {
    __shared__ float sums[4][kRank], totals[4];
    const int g = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const PartHead head = a.parts.heads[g];
    for (int r = blockIdx.y; r < head.rows; r += gridDim.y) {
        auto slot = [&](int k) { return static_cast<int64_t>(k == 0 ? 2 * g + 1 : 2 * (g + k)) * M + r; };
        float high = kNone;
        for (int k = lane; k <= head.after; k += 64) {
            high = fmaxf(high, a.parts.stats[slot(k) * 2]);
        }
        for (int o = 32; o >= 1; o >>= 1) {
            high = fmaxf(high, __shfl_xor(high, o));
        }
        float total = 0.0f, sum[8] = {};
        for (int k = wave; k <= head.after; k += 4) {
            const float top = a.parts.stats[slot(k) * 2];
            if (top == kNone) {
                // no score above -infinity here: a total that is not 0 is NaN
                total += a.parts.stats[slot(k) * 2 + 1];
                continue;
            }
            const float w = __builtin_amdgcn_exp2f(top - high);
            total = __builtin_fmaf(w, a.parts.stats[slot(k) * 2 + 1], total);
            const float* const from = a.parts.sums + slot(k) * kRank + 8 * lane;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                sum[i] = __builtin_fmaf(w, from[i], sum[i]);
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            sums[wave][8 * lane + i] = sum[i];
        }
        if (lane == 0) {
            totals[wave] = total;
        }
        __syncthreads();
        total = (totals[0] + totals[1]) + (totals[2] + totals[3]);
        E* const out = static_cast<E*>(a.out) + (head.row0 + r) * kRank;
        for (int i = threadIdx.x; i < kRank; i += 256) {
            out[i] = static_cast<E>(((sums[0][i] + sums[1][i]) + (sums[2][i] + sums[3][i])) / total);
        }
    }
}

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
    float m = kNone, l = 0.0f;
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
        const float alpha = m == kNone ? 1.0f : __expf(m - top);
        const float p = s == kNone ? 0.0f : __expf(s - top);
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
    float top = kNone, total = 0.0f, w[4];
    for (int i = 0; i < 4; ++i) {
        top = fmaxf(top, stats[i][0]);
    }
    for (int i = 0; i < 4; ++i) {
        w[i] = stats[i][0] == kNone ? 0.0f : __expf(stats[i][0] - top);
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
hipError_t launch(const PagedAttention& a, void* workspace, hipStream_t s) {
    if (!paged_tiled(a.rank, a.rope)) {
        hipLaunchKernelGGL(paged_any_kernel<E>, dim3(static_cast<unsigned>(a.view.tokens * a.heads)), dim3(256), 0, s,
                           a);
        return hipGetLastError();
    }
    TileArgs t;
    t.view = a.view;
    t.q = a.q;
    t.pool = a.pool;
    t.out = a.out;
    t.heads = a.heads;
    t.negative = a.scale < 0.0f ? 1 : 0;
    t.page_mul = static_cast<uint32_t>(((uint64_t{1} << 32) + a.view.page_size / 16 - 1) / (a.view.page_size / 16));
    // a scale of 0 weighs all keys alike, as one this small does, and leaves -infinity what it is
    t.c = std::max(std::fabs(a.scale) * 1.4426950408889634f, 1e-30f);
    char* w = static_cast<char*>(workspace);
    t.parts.heads = reinterpret_cast<PartHead*>(w);
    w += round_up(sizeof(PartHead) * kGrid, 256);
    t.parts.stats = reinterpret_cast<float*>(w);
    w += round_up(sizeof(float) * 2 * kGrid * kRows16 * 2, 256);
    t.parts.sums = reinterpret_cast<float*>(w);
    hipLaunchKernelGGL(paged_rows16_kernel<E>, dim3(kGrid), dim3(256), 0, s, t);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) {
        return err;
    }
    hipLaunchKernelGGL((paged_join_kernel<E, kRows16>), dim3(kGrid, kRows16), dim3(256), 0, s, t);
    return hipGetLastError();
}

}  // namespace

bool paged_tiled(int32_t rank, int32_t rope) { return rank == kRank && rope == kRope; }

int64_t paged_workspace_bytes() {
    return round_up(sizeof(PartHead) * kGrid, 256) + round_up(sizeof(float) * 2 * kGrid * kRows16 * 2, 256) +
           static_cast<int64_t>(sizeof(float)) * 2 * kGrid * kRows16 * kRank;
}

hipError_t launch_paged_attention(const PagedAttention& a, void* workspace, hipStream_t s) {
    return a.bf16 != 0 ? launch<bf16>(a, workspace, s) : launch<_Float16>(a, workspace, s);
}

}  // namespace lm
