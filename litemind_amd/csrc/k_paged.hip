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
// in blocks of 64 query rows of one request, or of 16 where no request has more
// (paged_rows_kernel). Any other widths take paged_any_kernel.
//
// The blocks' key tiles are shared out evenly: the grid's workgroups cut the
// line of all blocks' costs into equal pieces, found from the lengths on the
// GPU, so neither lengths nor the cut pass through the host. A block cut by a
// border leaves unnormalised sums, which paged_join_kernel adds in order.
#include "serve_internal.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

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
// its last token sees, as a line in b and times heads, which keeps it whole:
// (cached + kExtra) heads + (b + 1) M. kExtra stands for what a block costs
// besides its tiles.
constexpr int kExtra = 64;
// Keys per workgroup below which fewer take part.
constexpr int kLeast = 128;

struct Shares {
    int32_t heads, rows;  // rows: M
    __device__ int32_t blocks(const PagedRequest& r) const { return (r.added * heads + rows - 1) / rows; }
    // Cost of the request's first b blocks.
    __device__ int64_t cost(const PagedRequest& r, int32_t b) const {
        return static_cast<int64_t>(b) * (r.cached + kExtra) * heads + static_cast<int64_t>(b) * (b + 1) / 2 * rows;
    }
    // Tiles of block b.
    __device__ int32_t tiles(const PagedRequest& r, int32_t b) const {
        const int32_t last = min((b + 1) * rows, r.added * heads) - 1;
        return (r.cached + last / heads + kTile) / kTile;
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
// Begin of piece g. (In doubles, as the cuts of blocks below: a 64-bit division
// is 150 instructions. Neighbours form a border from the same numbers, so they
// agree on it however it rounds.)
__device__ inline int64_t border(int64_t total, int32_t parts, int32_t g) {
    return g >= parts ? total : static_cast<int64_t>(static_cast<double>(total) * g / parts);
}
// Tile of a block at which a border `x` past the block's begin cuts it.
__device__ inline int32_t cut(int64_t x, int64_t cost, int32_t tiles) {
    return min(tiles, static_cast<int32_t>(static_cast<double>(x) * tiles / static_cast<double>(cost)));
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
    p.parts = static_cast<int32_t>(max(int64_t{1}, min(static_cast<int64_t>(kGrid), total / (int64_t{kLeast} * sh.heads))));
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
        s.tile0 = s.begins ? 0 : cut(p.begin - at, cost, tiles);
        s.tile1 = s.ends ? tiles : cut(p.end - at, cost, tiles);
        s.parts_after = 0;
        if (s.begins && !s.ends) {
            // the last piece that begins before the block's end, from its share of the line
            const int32_t own = static_cast<int32_t>(blockIdx.x);
            int32_t g = static_cast<int32_t>(static_cast<double>(at + cost) * p.parts / static_cast<double>(p.total));
            g = max(own, min(g, p.parts - 1));
            while (g + 1 < p.parts && border(p.total, p.parts, g + 1) < at + cost) {
                ++g;
            }
            while (g > own && border(p.total, p.parts, g) >= at + cost) {
                --g;
            }
            s.parts_after = g - own;
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

// A tile in LDS: per eight rows their 64 units of latent (16 bytes each), a row
// after the other, then their eight units of rotary key. A load fills 64 units,
// so a row's latent is one load and eight rotary keys are one. Units are XORed by
// row so that LDS reads are free of bank conflicts: a 16-lane group of a key read
// takes one unit of 16 rows; 32 lanes of a transposing read four neighbouring
// units of four rows, or two of eight. Bits 2 and 3 come from the row within
// four, bits 0 and 1 from the fours; rotary rows are 8 units apart.
constexpr int kEightBytes = 8 * kRowBytes;  // 9216
__device__ inline int swizzle(int r) { return (r & 3) << 2 | (r >> 2 & 2) | (r >> 2 & 1); }
__device__ inline int latent_at(int r, int u) {
    return (r >> 3) * kEightBytes + (r & 7) * 1024 + ((u ^ swizzle(r)) << 4);
}
__device__ inline int rotary_at(int r, int u) {
    return (r >> 3) * kEightBytes + 8192 + (r & 7) * 128 + ((u ^ (r >> 1 & 7)) << 4);
}

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

// The same value, made anew where it stands: kept from becoming a register that
// lives through a loop for every constant that is added to it.
__device__ inline int here(int v) {
    asm volatile("" : "+v"(v));
    return v;
}

// ---- blocks of query rows ----
// M = 64 rows, four waves. The waves share tiles of 32 keys, which come straight
// to LDS four deep, and split each product differently:
//   S^T   wave (kh, rh): keys 16 kh .. + 15 for rows 32 rh .. + 31; its queries
//         stay in 144 registers, 36 products of 16 x 16 x 32 a tile
//   out^T channels 128 w .. + 127 of wave w for all rows; 128 registers of sums,
//         16 products of 32 x 32 x 16 a tile
// (M = 16: keys 16 kh .. for all rows, on both rh; 32 registers, 8 products of
// 16 x 16 x 32.) The weights pass through LDS. One barrier a tile: between two,
// the waves run the scores of tile t + 1 and the context of tile t, which do not
// depend on each other, and the weights of t + 1 beside the last of the context.
// A wave with 32 rows and all channels would need no exchange, but 256 + 16
// registers of sums, where the matrix cores' results go to 256.
//
// The weights' reference m, one per row, has to be the same for all waves: it is
// moved only where a row's scores pass it by more than kSlack (in powers of
// two), which a wave tells the others at the next barrier; the tile's weights
// are then made anew. fp32 sums do not mind the factor, and 16-bit weights up to
// 2^kSlack round as those up to 1 do.
constexpr float kSlack = 10.0f;
constexpr float kUnset = -1e30f;  // reference of a row without a score yet: any finite one passes it

// Non-finite values as 0: keys that some row must not see weigh 0 there, and 0
// times NaN or infinity is not 0. (Rows that see such a key have a NaN weight.)
template <class E>
__device__ inline short8v finite_or_zero(short8v v) {
    constexpr short kExponent = std::is_same_v<E, bf16> ? 0x7f80 : 0x7c00;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        v[e] = (v[e] & kExponent) == kExponent ? short{0} : v[e];
    }
    return v;
}

template <class E, int M>
__global__ __launch_bounds__(256, 1) void paged_rows_kernel(const TileArgs a) {
    static_assert(M == 64 || M == 16);
    using H = Half<E>;
    typedef typename H::vec8 vec8;
    typedef typename H::vec4 vec4;
    constexpr bool kWide = M == 64;
    constexpr int NB = kWide ? 2 : 1;        // blocks of 16 rows in a wave's scores
    constexpr int NO = 8;                    // sums: [2][4] of 32 x 32, or [8] of 16 x 16
    using Sum = std::conditional_t<kWide, f32x16, f32x4>;
    // one array per stage: the compiler tracks loads to LDS per array
    __shared__ __align__(16) char s0[kTileBytes], s1[kTileBytes], s2[kTileBytes], s3[kTileBytes];
    __shared__ __align__(16) char weights[2][M * kTile * 2];
    __shared__ float tops[2][M];
    __shared__ int late_flags[4];
    __shared__ int64_t scratch[8];
    char* const ring[4] = {s0, s1, s2, s3};
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kh = wave & 1, rh = kWide ? wave >> 1 : 0;
    const int col = lane & 15, grp = lane >> 4;     // of 16 x 16 products
    const int col32 = lane & 31, half = lane >> 5;  // of 32 x 32 products
    Walk walk;
    walk.sh = Shares{a.heads, M};
    walk.p = find_piece(a.view, walk.sh, blockIdx.x, scratch);
    if (tid == 0) {
        a.parts.heads[blockIdx.x].rows = 0;
    }
    if (walk.p.begin >= walk.p.end) {
        return;
    }
    walk.start(a.view);
    // The wave loads rows 8 wave .. + 7 of a tile: eight latents, and their rotary
    // keys in one load, of which this lane takes
    const int rotary_from = (lane >> 3) * kRowBytes + 1024 + (((lane & 7) ^ ((8 * wave + (lane >> 3)) >> 1 & 7)) << 4);
    // Where the lane's reads of a tile begin. The scores' k-step ks reads latent
    // unit 4 ks + grp, bits 2 and 3 of which the swizzle changes: ks & 3 is XORed
    // in, the rest is a constant offset; so are channel tiles below. A row of
    // weights is 64 bytes, its four units XORed by row / 4.
    const int key_at = latent_at(16 * kh + col, grp);
    const int rotary_key_at = rotary_at(16 * kh + col, grp);
    int value_at[2], weight_from[NB], weight_to[NB];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        // the first or second four of the lane's eight keys
        const int r = 8 * (kWide ? half : grp) + 4 * i + ((lane & 15) >> 2);
        const int u = kWide ? 2 * (lane >> 4 & 1) + ((lane & 3) >> 1) : (lane & 3) >> 1;
        value_at[i] = latent_at(r, u) + (lane & 1) * 8 + wave * 256;
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const int row = kWide ? 32 * b + col32 : col, to = 32 * rh + 16 * b + col;
        weight_from[b] = row * 64 + (((kWide ? half : grp) ^ (row >> 2 & 3)) << 4);
        weight_to[b] = to * 64 + (((2 * kh + (grp >> 1)) ^ (to >> 2 & 3)) << 4) + (grp & 1) * 8;
    }
    Segment s;
    while (walk.next(a.view, s)) {
        const int in_request = s.block * M;  // the block's first row
        const int64_t row0 = static_cast<int64_t>(s.req.first) * a.heads + in_request;
        const int rows = min(M, s.req.added * a.heads - in_request);
        const int32_t last = s.req.cached + s.req.added - 1;
        const int32_t all_see = s.req.cached + in_request / a.heads;
        PageWalk pages;
        pages.start(a.view, s.request);
        auto issue = [&](int32_t t, char* to) {
            const int32_t key = t * kTile + 16 * (wave >> 1);
            const int32_t first = min(key, last & ~15);
            const char* const base =
                static_cast<const char*>(a.pool) + pages.at(a.view, a.page_mul, first) * kRowBytes;
            const __amdgpu_buffer_rsrc_t res =
                __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, 16 * kRowBytes, kBufferWord3);
            to += wave * kEightBytes;
            const int eight = 8 * (wave & 1), of = here(lane * 16);
            if (key + 15 <= last) {
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    buffer_lds16(res, to + r * 1024, static_cast<unsigned>(of ^ (swizzle(r) | (wave & 1) << 1) << 4),
                                 static_cast<unsigned>((eight + r) * kRowBytes));
                }
                buffer_lds16(res, to + 8192, static_cast<unsigned>(rotary_from),
                             static_cast<unsigned>(eight * kRowBytes));
            } else {  // rows past the last key: the last key's once more
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    buffer_lds16(res, to + r * 1024, static_cast<unsigned>(of ^ (swizzle(r) | (wave & 1) << 1) << 4),
                                 static_cast<unsigned>((min(key + eight + r, last) - first) * kRowBytes));
                }
                const int r = of >> 7;  // lane / 8
                buffer_lds16(res, to + 8192,
                             static_cast<unsigned>(rotary_from + (min(key + eight + r, last) - first - r) * kRowBytes),
                             0);
            }
        };
        auto meet = [] {
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_waitcnt(0xc07f);  // this wave's LDS writes are done
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_sched_barrier(0);
        };
        __syncthreads();  // the block before is done with LDS
        if (tid < 4) {
            late_flags[tid] = 0;
        }
        if (s.tile0 < s.tile1) {
            issue(s.tile0, ring[0]);
        }
        if (s.tile0 + 1 < s.tile1) {
            issue(s.tile0 + 1, ring[1]);
        }
        int32_t sees[NB];
        vec8 q[NB][18];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int own = min(32 * rh + 16 * b + col, rows - 1);
            sees[b] = s.req.cached + (in_request + own) / a.heads;
            const E* const from_q = static_cast<const E*>(a.q) + (row0 + own) * kWidth + 8 * grp;
#pragma unroll
            for (int ks = 0; ks < 18; ++ks) {
                q[b][ks] = *reinterpret_cast<const vec8*>(from_q + 32 * ks);
            }
        }
        if (a.negative) {
#pragma unroll
            for (int b = 0; b < NB; ++b) {
#pragma unroll
                for (int ks = 0; ks < 18; ++ks) {
                    q[b][ks] = -q[b][ks];
                }
            }
        }
        Sum o[NO] = {};
        f32x4 sc[NB];             // scores of the newest tile
        float m = kNone;          // reference of row `lane`, the same in every wave
        float ref[NB], l[NB], sum[NB];  // of this lane's rows: reference times c, total, the newest tile's
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            ref[b] = kUnset;
            l[b] = sum[b] = 0.0f;
        }
        // the newest tile's weights; tells whether a score passes the reference
        auto weigh = [&](char* wt) {
            float over = kNone;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                vec4 p;
                float w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float x = __builtin_fmaf(sc[b][e], a.c, -ref[b]);
                    over = fmaxf(over, x);
                    w[e] = __builtin_amdgcn_exp2f(x);
                    p[e] = static_cast<E>(w[e]);
                }
                sum[b] = (w[0] + w[1]) + (w[2] + w[3]);
                *reinterpret_cast<vec4*>(wt + weight_to[b]) = p;
            }
            return over;
        };
        auto tell = [&](float over, int u) {
            if (__builtin_expect(__any(over > kSlack), 0)) {
                if (lane == 0) {
                    late_flags[u] = 1;
                }
            }
        };
        // The products of an interval: scores of the tile in `next` (S), context of
        // the tile in `now` (C), each step's operands read during the one before.
        // The scores take the first half, so that `weights_of` runs beside the
        // second half of the context.
        auto products = [&](auto with_scores, const char* next, auto with_context, const char* now, const char* wt,
                            bool sanitize, auto middle, auto weights_of) {
            constexpr bool S = decltype(with_scores)::value, C = decltype(with_context)::value;
            // step i: k-steps 3 i .. + 2 of the scores (i < 6), part `unit(i)` of the context
            auto unit = [](int i) { return i < 5 ? i : i == 5 ? -1 : i - 1; };
            vec8 kf[2][3], vf[2], pf[NB];
            const int k_at = here(key_at), r_at = here(rotary_key_at);
            const int v_at[2] = {here(value_at[0]), here(value_at[1])};
            auto read = [&](int i) {
                if (S && i < 6) {
#pragma unroll
                    for (int k = 0; k < 3; ++k) {
                        const int ks = 3 * i + k;
                        kf[i & 1][k] = *reinterpret_cast<const vec8*>(
                            next + (ks < 16 ? (k_at ^ (ks & 3) << 6) + (ks >> 2) * 256 : r_at ^ (ks & 1) << 6));
                    }
                }
                const int n = unit(i);
                if (C && n >= 0) {
                    // M = 64: keys 16 st .. + 15, channels 32 ct ..; M = 16: all keys, channels 16 ct ..
                    const int st = kWide ? n / 4 : 0, ct = kWide ? n % 4 : n;
                    short8v v;
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        // a channel tile is four units (M = 16: two), a wave's channels 16
                        const int from_here =
                            kWide ? (v_at[k] ^ ct << 6) + st * 2 * kEightBytes : v_at[k] ^ ct << 5;
                        const short4v part = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(now + from_here));
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            v[4 * k + e] = part[e];
                        }
                    }
                    vf[n & 1] = __builtin_bit_cast(vec8, v);
                }
            };
            auto read_weights = [&](int st) {
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    pf[b] = *reinterpret_cast<const vec8*>(wt + (weight_from[b] ^ st * 32));
                }
            };
            if constexpr (S) {
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    sc[b] = f32x4{};
                }
            }
            if constexpr (C) {
                read_weights(0);
            }
            read(0);
            middle();
#pragma unroll
            for (int i = 0; i < 9; ++i) {
                if (i < 8) {
                    read(i + 1);
                }
                if (i <= 6) {
                    __builtin_amdgcn_sched_barrier(0);
                }
                const int n = unit(i);
                if (C && n >= 0) {
                    vec8 f = vf[n & 1];
                    if (sanitize) {
                        f = __builtin_bit_cast(vec8, finite_or_zero<E>(__builtin_bit_cast(short8v, f)));
                    }
                    if constexpr (kWide) {
                        o[n % 4] = H::mfma32(f, pf[0], o[n % 4]);
                        o[4 + n % 4] = H::mfma32(f, pf[NB - 1], o[4 + n % 4]);
                    } else {
                        o[n] = H::mfma16(f, pf[0], o[n]);
                    }
                    if (kWide && n == 3) {
                        read_weights(1);
                    }
                }
                if (S && i < 6) {
#pragma unroll
                    for (int k = 0; k < 3; ++k) {
#pragma unroll
                        for (int b = 0; b < NB; ++b) {
                            sc[b] = H::mfma16(kf[i & 1][k], q[b][3 * i + k], sc[b]);
                        }
                    }
                }
                if (i < 6) {
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (i == 6) {
                    weights_of();
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        };
        const std::true_type yes;
        const std::false_type no;
        const auto nothing = [] {};
        auto mask = [&](int32_t t) {
            if (t * kTile + kTile - 1 > all_see) {
#pragma unroll
                for (int b = 0; b < NB; ++b) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        sc[b][e] = t * kTile + 16 * kh + 4 * grp + e > sees[b] ? kNone : sc[b][e];
                    }
                }
            }
        };
        // moves the reference to the rows' largest scores of the newest tile;
        // returns the factor of row `lane`'s sums so far
        auto follow = [&] {
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                float high = fmaxf(fmaxf(sc[b][0], sc[b][1]), fmaxf(sc[b][2], sc[b][3]));
                high = fmaxf(high, __shfl_xor(high, 16));
                high = fmaxf(high, __shfl_xor(high, 32));
                if (grp == 0) {
                    tops[kh][32 * rh + 16 * b + col] = high;
                }
            }
            meet();
            const int row = min(lane, rows - 1);  // (rows past the last are the last once more)
            const float up = fmaxf(m, fmaxf(tops[0][row], tops[1][row]));
            const float alpha = up == kNone ? 1.0f : __builtin_amdgcn_exp2f((m - up) * a.c);
            m = up;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const float mine = __shfl(up, 32 * rh + 16 * b + col);
                ref[b] = mine == kNone ? kUnset : mine * a.c;
            }
            return alpha;
        };
        // tile t's weights and tile t + 1 are in
        auto arrive = [&](int32_t t) {
            __builtin_amdgcn_sched_barrier(0);
            if (t + 2 < s.tile1) {
                __builtin_amdgcn_s_waitcnt(0x0F70 | 9);
            } else {
                __builtin_amdgcn_s_waitcnt(0x0F70);
            }
            meet();
        };
        if (s.tile0 < s.tile1) {
            arrive(s.tile0 - 1);
            if (s.tile0 + 2 < s.tile1) {
                issue(s.tile0 + 2, ring[2]);
            }
            products(yes, ring[0], no, nullptr, nullptr, false, nothing, nothing);
            mask(s.tile0);
            follow();
            weigh(weights[0]);
            // tiles up to here are seen by all rows, and the next one too
            const int32_t full = min(s.tile1 - 1, (all_see + 1) / kTile - 1);
            int32_t t = s.tile0;
            while (t < s.tile1) {
                // A reference left behind, or a tile that rows may not see, is
                // for the loop after this one: the sums are touched by products
                // alone here, and stay in the registers that products use.
                int stop = 0;
                bool here_already = false;
                while (stop == 0) {
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        if (t + u >= full) {
                            stop = u + 1;
                            break;
                        }
                        arrive(t + u);
                        if (__builtin_expect(late_flags[u] != 0, 0)) {
                            stop = u + 1;
                            here_already = true;
                            break;
                        }
                        if (tid == 0) {
                            late_flags[(u + 2) & 3] = 0;
                        }
#pragma unroll
                        for (int b = 0; b < NB; ++b) {
                            l[b] += sum[b];
                        }
                        float over;
                        products(
                            yes, ring[(u + 1) & 3], yes, ring[u], weights[u & 1], false,
                            [&] {
                                if (t + u + 3 < s.tile1) {
                                    issue(t + u + 3, ring[(u + 3) & 3]);
                                }
                            },
                            [&] { over = weigh(weights[(u + 1) & 1]); });
                        tell(over, (u + 1) & 3);
                    }
                    t += stop == 0 ? 4 : 0;
                }
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    if (u + 1 >= stop && t + u < s.tile1) {
                        if (u + 1 != stop || !here_already) {
                            arrive(t + u);
                        }
                        if (late_flags[u] != 0) {
                            const float alpha = follow();
#pragma unroll
                            for (int b = 0; b < NB; ++b) {
                                const float f = __shfl(alpha, kWide ? 32 * b + col32 : col);
#pragma unroll
                                for (int i = 0; i < NO / NB; ++i) {
                                    o[NO / NB * b + i] *= f;
                                }
                            }
#pragma unroll
                            for (int b = 0; b < NB; ++b) {
                                l[b] *= __shfl(alpha, 32 * rh + 16 * b + col);
                            }
                            weigh(weights[u & 1]);
                            meet();
                        }
                        if (tid == 0) {
                            late_flags[(u + 2) & 3] = 0;
                        }
#pragma unroll
                        for (int b = 0; b < NB; ++b) {
                            l[b] += sum[b];
                        }
                        if (t + u + 3 < s.tile1) {
                            issue(t + u + 3, ring[(u + 3) & 3]);
                        }
                        if (t + u + 1 < s.tile1) {
                            products(yes, ring[(u + 1) & 3], no, nullptr, nullptr, false, nothing, nothing);
                            mask(t + u + 1);
                        }
                        products(no, nullptr, yes, ring[u], weights[u & 1], (t + u) * kTile + kTile - 1 > all_see, nothing,
                                 nothing);
                        if (t + u + 1 < s.tile1) {
                            tell(weigh(weights[(u + 1) & 1]), (u + 1) & 3);
                        }
                    }
                }
                t += 4;
            }
        }
        // the totals: the rows' parts of both key halves meet in `tops`
        __syncthreads();
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            l[b] += __shfl_xor(l[b], 16);
            l[b] += __shfl_xor(l[b], 32);
            if (grp == 0) {
                tops[kh][32 * rh + 16 * b + col] = l[b];
            }
        }
        __syncthreads();
        const bool whole = s.begins && s.ends;
        const int64_t slot = 2 * static_cast<int64_t>(blockIdx.x) + (s.begins ? 1 : 0);
        // o[4 rb + ct] register e: channel 128 wave + 32 ct + 8 (e / 4) + 4 half + e % 4
        // of row 32 rb + col32 (M = 16: o[ct], channel 128 wave + 16 ct + 4 grp + e of row col)
#pragma unroll
        for (int i = 0; i < NO; ++i) {
            const int row = kWide ? 32 * (i / 4) + col32 : col;
            if (row < rows) {
                const float inv = whole ? 1.0f / (tops[0][row] + tops[1][row]) : 1.0f;
                const int ch = 128 * wave + (kWide ? 32 * (i % 4) + 4 * half : 16 * i + 4 * grp);
#pragma unroll
                for (int g = 0; g < (kWide ? 4 : 1); ++g) {
                    if (whole) {
                        vec4 out;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            out[e] = static_cast<E>(o[i][4 * g + e] * inv);
                        }
                        *reinterpret_cast<vec4*>(static_cast<E*>(a.out) + (row0 + row) * kRank + ch + 8 * g) = out;
                    } else {
                        f32x4 out;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            out[e] = o[i][4 * g + e];
                        }
                        *reinterpret_cast<f32x4*>(a.parts.sums + (slot * M + row) * kRank + ch + 8 * g) = out;
                    }
                }
            }
        }
        if (!whole && tid < rows) {
            float* const to = a.parts.stats + (slot * M + tid) * 2;
            to[0] = m == kNone ? kNone : m * a.c;
            to[1] = tops[0][tid] + tops[1][tid];
        }
        if (s.begins && !s.ends && tid == 0) {
            a.parts.heads[blockIdx.x] = PartHead{row0, rows, s.parts_after};
        }
    }
}

// The parts of cut blocks added up. An item of work is four rows of a block, a
// wave each with 64 lanes for 512 channels; of a block in kMany parts or more (a
// long request, few rows) it is 128 channels of one row, 32 lanes for them and
// the parts dealt to the workgroup's eight half waves. The workgroups take
// items in turn, so a step with one cut block uses as many as one with 256.
constexpr int kMany = 16;
constexpr int kJoinGrid = 1024;

template <class E, int M>
__global__ __launch_bounds__(256) void paged_join_kernel(const TileArgs a) {
    __shared__ int32_t first[kGrid], wave_items[4];
    __shared__ float sums[8][128], totals[8], tops[8];
    static_assert(kGrid == 256, "a piece per thread");
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const PartHead own = a.parts.heads[tid];
    const int32_t items = own.rows == 0 ? 0 : own.after + 1 >= kMany ? own.rows * 4 : (own.rows + 3) / 4;
    int32_t sum_items = items;
    for (int o = 1; o < 64; o <<= 1) {
        const int32_t up = __shfl_up(sum_items, o);
        sum_items += lane >= o ? up : 0;
    }
    if (lane == 63) {
        wave_items[wave] = sum_items;
    }
    __syncthreads();
    int32_t total_items = 0;
    for (int w = 0; w < 4; ++w) {
        sum_items += w < wave ? wave_items[w] : 0;
        total_items += wave_items[w];
    }
    first[tid] = sum_items - items;
    __syncthreads();
    for (int32_t item = blockIdx.x; item < total_items; item += gridDim.x) {
        int g = 0;  // the last piece whose items start at or before this one
        for (int step = 128; step >= 1; step >>= 1) {
            g += first[g + step] <= item ? step : 0;
        }
        const PartHead head = a.parts.heads[g];
        const int32_t at = item - first[g];
        auto slot = [&](int k, int r) { return static_cast<int64_t>(k == 0 ? 2 * g + 1 : 2 * (g + k)) * M + r; };
        // parts k0, k0 + by, ..; four loads at a time, those past the last weigh 0
        auto add = [&](int k0, int by, int r, int channel, float high, f32x4 (&sum)[2], bool second, float& total) {
            for (int k = k0; k <= head.after; k += 4 * by) {
                f32x4 v[4][2];
                float st[4][2];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int64_t from = slot(min(k + i * by, head.after), r);
                    st[i][0] = a.parts.stats[from * 2];
                    st[i][1] = a.parts.stats[from * 2 + 1];
                    v[i][0] = *reinterpret_cast<const f32x4*>(a.parts.sums + from * kRank + channel);
                    if (second) {
                        v[i][1] = *reinterpret_cast<const f32x4*>(a.parts.sums + from * kRank + channel + 256);
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    // no score above -infinity: weighs 0 (NaN in the total or the sums stays)
                    const float w = st[i][0] == kNone || k + i * by > head.after
                                        ? 0.0f
                                        : __builtin_amdgcn_exp2f(st[i][0] - high);
                    total = __builtin_fmaf(w, st[i][1], total);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        sum[0][e] = __builtin_fmaf(w, v[i][0][e], sum[0][e]);
                        if (second) {
                            sum[1][e] = __builtin_fmaf(w, v[i][1][e], sum[1][e]);
                        }
                    }
                }
            }
        };
        auto highest = [&](int k0, int by, int r) {
            float high = kNone;
            for (int k = k0; k <= head.after; k += by) {
                high = fmaxf(high, a.parts.stats[slot(k, r) * 2]);
            }
            return high;
        };
        auto store = [&](int r, int channel, const f32x4& sum, float total) {
            const float inv = 1.0f / total;
            typename Half<E>::vec4 out;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                out[e] = static_cast<E>(sum[e] * inv);
            }
            *reinterpret_cast<typename Half<E>::vec4*>(static_cast<E*>(a.out) + (head.row0 + r) * kRank + channel) = out;
        };
        f32x4 sum[2] = {};
        float total = 0.0f;
        if (head.after + 1 < kMany) {
            const int r = min(4 * at + wave, head.rows - 1);  // (a wave past the last row repeats it)
            add(0, 1, r, 4 * lane, highest(0, 1, r), sum, true, total);
            store(r, 4 * lane, sum[0], total);
            store(r, 256 + 4 * lane, sum[1], total);
            continue;
        }
        const int r = at >> 2, channel = (at & 3) * 128 + (tid & 31) * 4, eighth = tid >> 5;
        float high = highest(tid, 256, r);
        for (int o = 32; o >= 1; o >>= 1) {
            high = fmaxf(high, __shfl_xor(high, o));
        }
        __syncthreads();  // the item before has been read
        if (lane == 0) {
            tops[wave] = high;
        }
        __syncthreads();
        high = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
        add(eighth, 8, r, channel, high, sum, false, total);
        *reinterpret_cast<f32x4*>(&sums[eighth][(tid & 31) * 4]) = sum[0];
        if ((tid & 31) == 0) {
            totals[eighth] = total;
        }
        __syncthreads();
        if (tid < 32) {
            sum[0] = f32x4{};
            total = 0.0f;
            for (int i = 0; i < 8; ++i) {
                const f32x4 v = *reinterpret_cast<const f32x4*>(&sums[i][tid * 4]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    sum[0][e] += v[e];
                }
                total += totals[i];
            }
            store(r, channel, sum[0], total);
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
    const int m = paged_block_rows(a.max_added, a.heads);
    t.parts.heads = reinterpret_cast<PartHead*>(w);
    w += round_up(sizeof(PartHead) * kGrid, 256);
    t.parts.stats = reinterpret_cast<float*>(w);
    w += round_up(sizeof(float) * 2 * kGrid * m * 2, 256);
    t.parts.sums = reinterpret_cast<float*>(w);
    if (m == 16) {
        hipLaunchKernelGGL((paged_rows_kernel<E, 16>), dim3(kGrid), dim3(256), 0, s, t);
    } else {
        hipLaunchKernelGGL((paged_rows_kernel<E, 64>), dim3(kGrid), dim3(256), 0, s, t);
    }
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) {
        return err;
    }
    if (m == 16) {
        hipLaunchKernelGGL((paged_join_kernel<E, 16>), dim3(kJoinGrid), dim3(256), 0, s, t);
    } else {
        hipLaunchKernelGGL((paged_join_kernel<E, 64>), dim3(kJoinGrid), dim3(256), 0, s, t);
    }
    return hipGetLastError();
}

}  // namespace

bool paged_tiled(int32_t rank, int32_t rope) { return rank == kRank && rope == kRope; }

int paged_block_rows(int32_t max_added, int32_t heads) {
    return static_cast<int64_t>(max_added) * heads <= 16 ? 16 : 64;
}

int64_t paged_workspace_bytes(int rows) {
    return round_up(sizeof(PartHead) * kGrid, 256) + round_up(sizeof(float) * 2 * kGrid * rows * 2, 256) +
           static_cast<int64_t>(sizeof(float)) * 2 * kGrid * rows * kRank;
}

hipError_t launch_paged_attention(const PagedAttention& a, void* workspace, hipStream_t s) {
    return a.bf16 != 0 ? launch<bf16>(a, workspace, s) : launch<_Float16>(a, workspace, s);
}

}  // namespace lm
