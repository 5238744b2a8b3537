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
//
// Measured, 16 heads, calls of three contexts in turn: one token over 131072 keys
// 35 us, 4.3 TB/s (large reads reach 6.4); one each of 32 requests of up to 4000
// keys 21.8 us; 512 tokens after 3001 84 us, 0.70 PFLOP/s, and 2048 after none 117
// us, 0.63 (large library products reach 1.2). A call by itself takes 20 us at
// least: the lengths, the tables, the first tiles and the sums each wait for the
// one before.
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
typedef __attribute__((address_space(3))) short4v lds_short4;
typedef __attribute__((address_space(3))) char lds_char;

constexpr int kRank = 512, kRope = 64, kWidth = kRank + kRope;
constexpr int kRowBytes = kWidth * 2;        // 1152
constexpr int kTile = 32;                    // keys of a tile
constexpr int kTileBytes = kTile * kRowBytes;
constexpr int kGrid = 256;                   // workgroups that share out the tiles: one per CU
constexpr int kWaves = 8;                    // of each, two per SIMD
constexpr int kThreads = 64 * kWaves;
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
};
template <>
struct Half<bf16> {
    typedef bf16x8 vec8;
    typedef bf16x4 vec4;
    static __device__ f32x4 mfma16(vec8 a, vec8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
};

// ---- sharing out the tiles ----
// Block b of a request (rows b M .. of its added heads rows) costs the keys that
// its last token sees, as a line in b and times heads, which keeps it whole:
// (cached + kExtra) heads + (b + 1) M. kExtra, ten tiles, stands for what a block
// costs besides its tiles and comes first, so that a workgroup which begins a
// second block has so many tiles fewer. (By itself, with 64, 128, 192, 256, 320,
// 384 keys: a prompt of 2048 tokens, 16 heads 235, 168, 137, 127, 122, 122 us; one
// token of 32 requests after up to 4000 31.1, 30.0, 28.0, 25.9, 25.4, 25.6; of 128
// requests after 1000 31.6, 30.6, 29.6, 28.2, 29.4, 29.9. Spread over the block's
// tiles 256 keys made these 132, 33.4 and 32.3.)
constexpr int kExtra = 320;
// Keys per workgroup below which fewer take part (one token after 4000 by itself,
// with the join: 64 keys 18.5 us, 128 18.8, 256 21.9, 512 29.6; after 500 19.3,
// 19.4, 21.4, 28.2).
constexpr int kLeast = 128;

struct Shares {
    int32_t heads, rows;  // rows: M
    __device__ int32_t blocks(const PagedRequest& r) const { return (r.added * heads + rows - 1) / rows; }
    // Cost of the request's first b blocks.
    __device__ int64_t cost(const PagedRequest& r, int32_t b) const {
        return b * (static_cast<int64_t>(r.cached) + kExtra) * heads + static_cast<int64_t>(b) * (b + 1) / 2 * rows;
    }
    // Tiles of block b.
    __device__ int32_t tiles(const PagedRequest& r, int32_t b) const {
        const int32_t last = min((b + 1) * rows, r.added * heads) - 1;
        return static_cast<int32_t>((static_cast<uint32_t>(r.cached + last / heads) + kTile) / kTile);
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
// Tile of a block at which a border `x` past the block's begin cuts it: what the
// block costs besides its tiles comes first, and a border in that does not cut.
__device__ inline int32_t cut(int64_t x, int64_t cost, int32_t tiles, int32_t heads) {
    const int64_t extra = static_cast<int64_t>(kExtra) * heads;
    return x <= extra ? 0
                      : min(tiles, static_cast<int32_t>(static_cast<double>(x - extra) * tiles /
                                                        static_cast<double>(cost - extra)));
}

// Every thread of the workgroup calls it. Threads take stretches of requests;
// `scratch` (kWaves + 2 words of 64 bits) passes the sums.
__device__ inline Piece find_piece(const PagedView& v, const Shares& sh, int32_t g, int64_t* scratch) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t requests = static_cast<uint32_t>(v.requests), per = (requests + kThreads - 1) / kThreads;
    const int32_t r0 = static_cast<int32_t>(min(tid * per, requests)), r1 = static_cast<int32_t>(min(r0 + per, requests));
    int64_t own = 0;
#pragma unroll 1
    for (int32_t r = r0; r < r1; ++r) {
        const PagedRequest q = paged_request(v, r);
        own += sh.cost(q, sh.blocks(q));
    }
    int64_t sum = own;
#pragma unroll 1
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t up = __shfl_up(sum, o);
        sum += lane >= o ? up : 0;
    }
    if (lane == 63) {
        scratch[wave] = sum;
    }
    __syncthreads();
    int64_t before = sum - own, total = 0;
    for (int w = 0; w < kWaves; ++w) {
        before += w < wave ? scratch[w] : 0;
        total += scratch[w];
    }
    Piece p;
    p.total = total;
    p.parts = static_cast<int32_t>(max(int64_t{1}, min(static_cast<int64_t>(kGrid), static_cast<int64_t>(static_cast<double>(total) / (kLeast * static_cast<double>(sh.heads))))));
    p.begin = g < p.parts ? border(total, p.parts, g) : total;
    p.end = g < p.parts ? border(total, p.parts, g + 1) : total;
    if (p.begin >= before && p.begin < before + own) {
#pragma unroll 1
        for (int32_t r = r0; r < r1; ++r) {
            const PagedRequest q = paged_request(v, r);
            const int64_t c = sh.cost(q, sh.blocks(q));
            if (p.begin < before + c) {
                scratch[kWaves] = r;
                scratch[kWaves + 1] = before;
                break;
            }
            before += c;
        }
    }
    __syncthreads();
    p.request = __builtin_amdgcn_readfirstlane(static_cast<int32_t>(scratch[kWaves]));
    p.base = scratch[kWaves + 1];
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
#pragma unroll 1
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
        s.ends = p.end >= at + cost;
        s.tile0 = cut(p.begin - at, cost, tiles, sh.heads);
        s.tile1 = s.ends ? tiles : cut(p.end - at, cost, tiles, sh.heads);
        s.begins = s.tile0 == 0;
        if (s.tile1 == 0) {
            return false;  // the block begins in the next piece
        }
        s.parts_after = 0;
        if (s.begins && !s.ends) {
            // the last piece that begins before the block's end, from its share of the line
            const int32_t own = static_cast<int32_t>(blockIdx.x);
            int32_t g = static_cast<int32_t>(static_cast<double>(at + cost) * p.parts / static_cast<double>(p.total));
            g = max(own, min(g, p.parts - 1));
#pragma unroll 1
            while (g + 1 < p.parts && border(p.total, p.parts, g + 1) < at + cost) {
                ++g;
            }
#pragma unroll 1
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
    int32_t sign;      // of the scale, or 0: the queries are multiplied by it
    uint32_t page_mul; // 2^32 / (page_size / 16), rounded up
    float c;           // |scale| log2(e)
    Parts parts;
};

// A tile in LDS: per eight rows their 64 units of latent (16 bytes each), a row
// after the other, then their eight units of rotary key. A load fills 64 units,
// so a row's latent is one load and eight rotary keys are one. Units are XORed by
// row so that LDS reads are free of bank conflicts (16 units to a cycle). A key
// read's cycles take 16 rows: 0 - 3 and 12 - 15 of one unit and 4 - 11 of the next,
// or the other way round (measured: with the units of rows 4 - 11 not closed under
// XOR 1, a third of the cycles were conflicts). A transposing read's take four
// units of four rows, or two of eight. Bits 2 and 3 come from the row within
// four, bits 0 and 1 from the fours; rotary rows are 8 units apart.
constexpr int kEightBytes = 8 * kRowBytes;  // 9216
__device__ inline int swizzle(int r) { return (r & 3) << 2 | ((r >> 2 ^ r >> 3) & 1) << 1 | (r >> 3 & 1); }
__device__ inline int latent_at(int r, int u) {
    return (r >> 3) * kEightBytes + (r & 7) * 1024 + ((u ^ swizzle(r)) << 4);
}
__device__ inline int rotary_at(int r, int u) {
    return (r >> 3) * kEightBytes + 8192 + (r & 7) * 128 + ((u ^ (r >> 1 & 7)) << 4);
}

// The pages of one request's keys, a step ahead of their loads: look(key) reads
// the table entry, take() the pool row of that key (a multiple of 16; the 15 after
// it lie in the same page). The entry is a scalar load: a vector load's wait would
// be one for all tiles in flight.
typedef __attribute__((address_space(4))) const int32_t scalar_int;
struct PageWalk {
    const int32_t* row;  // the request's table row
    int32_t id, in_page;
    __device__ void start(const PagedView& v, int32_t request) {
        row = v.table + static_cast<int64_t>(request) * v.table_width;
    }
    __device__ void look(const PagedView& v, uint32_t page_mul, uint32_t key) {
        const uint32_t d = static_cast<uint32_t>(v.page_size) / 16, n = key / 16;
        uint32_t page = __umulhi(n, page_mul);
        if (d == 1) {
            page = n;
        } else if (page * d > n) {
            --page;
        }
        id = ((scalar_int*)row)[page];
        in_page = static_cast<int32_t>(n - page * d) * 16;
    }
    __device__ int64_t take(const PagedView& v) const {
        return checked_page(v, id) * v.page_size + in_page;
    }
};

// The same value, made anew where it stands: kept from becoming a register that
// lives through a loop for every constant that is added to it.
__device__ inline int here(int v) {
    asm volatile("" : "+v"(v));
    return v;
}
__device__ inline int lds_address(const char* p) {
    return static_cast<int>(reinterpret_cast<uintptr_t>((const lds_char*)p));
}

// ---- blocks of query rows ----
// M = 64 rows, eight waves, two per SIMD, so that one's products run beside the
// other's loads, exponentials and addresses. The waves share tiles of 32 keys,
// which come straight to LDS four deep, and split each product differently, in
// products of 16 x 16 x 32:
//   S^T   wave (kh, rq): keys 16 kh .. + 15 for rows 16 rq .. + 15, 18 products a
//         tile; its queries stay in 72 registers
//   out^T channels 64 w .. + 63 of wave w for all rows, 16 products a tile; 64
//         registers of sums
// (M = 16: keys 16 kh .. for all rows, on every rq; 4 products, 16 registers.)
// The weights pass through LDS. One barrier a tile: between two, the waves run
// the scores of tile t + 1 and the context of tile t, which do not depend on each
// other. LDS reads are 208 KB a tile, 191 bytes per clock of the products' time
// against the 254 that a CU reads; four waves of twice the work each would need
// 110, but have no second wave to fill a SIMD, and were no faster. Products of
// 32 x 32 x 16 take 19.4 ns on numbers as they come, two of 16 x 16 x 32 16.2
// (the clock gives way to the power drawn; on zeros 13.4 and 14.4).
// An interval takes 1.3 us: 0.55 of products, 0.8 for the tile's loads alone, 1.1
// without them; the rest is what a barrier a tile leaves unfilled.
//
// The weights' reference m, one per row, has to be the same for all waves: it is
// moved only where a row's scores pass it by more than kSlack (in powers of
// two), which a wave tells the others at the next barrier; the tile's weights
// are then made anew. A score at the reference weighs 2^kLift. In bf16, whose latents
// may lie near the end of the range of their fp32 sums, that is 2^-kSlack, so that no
// weight passes 1. In fp16 the weights, which end at 2^16, keep 11 bits down to
// 2^-(14 + kLift) of a row's largest and are rounded to steps of 2^-(24 + kLift) of it
// below: of n keys far under a first one, n 2^-30 of the row at most is lost, less than
// its output's rounding for up to 2^18 keys to a workgroup. (More lift needs less slack,
// and references move more often: a prompt of 2048 takes 1 % longer with 8 and 7, 4 %
// with 6 and 9, 15 % with 4 and 11.)
constexpr float kSlack = 10.0f;
template <class E>
constexpr float kLift = std::is_same_v<E, bf16> ? -kSlack : 5.0f;
// Reference of a row without a score yet: finite ones pass it, or weigh against it as
// against any other where the scale is that small; -infinity weighs 0.
constexpr float kLowest = -0x1.fffffep127f;

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
__global__ __launch_bounds__(kThreads, 2) void paged_rows_kernel(const TileArgs a) {
    static_assert(M == 64 || M == 16);
    using H = Half<E>;
    typedef typename H::vec8 vec8;
    typedef typename H::vec4 vec4;
    constexpr int RB = M / 16;  // blocks of 16 rows
    // one array per stage: the compiler tracks loads to LDS per array
    __shared__ __align__(16) char s0[kTileBytes], s1[kTileBytes], s2[kTileBytes], s3[kTileBytes];
    __shared__ __align__(16) char weights[2][M * kTile * 2];
    __shared__ float tops[2][M];
    __shared__ int late_flags[4];
    __shared__ int64_t scratch[kWaves + 2];
    char* const ring[4] = {s0, s1, s2, s3};
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kh = wave & 1, rq = M == 64 ? wave >> 1 : 0;
    const int col = lane & 15, grp = lane >> 4;
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
    // The wave loads rows 4 wave .. + 3 of a tile: a load for each latent, one of
    // half a wave for their rotary keys, of which this lane takes
    const int rotary_from = (lane >> 3) * kRowBytes + 1024 + (((lane & 7) ^ ((4 * wave + (lane >> 3)) >> 1 & 7)) << 4);
    // Where the lane's reads of a tile begin. The scores' k-step ks reads latent
    // unit 4 ks + grp, bits 2 and 3 of which the swizzle changes: ks & 3 is XORed
    // in, the rest is a constant offset; so are channel tiles below. A row of
    // weights is 64 bytes, its four units XORed by row / 4.
    const int key_at = latent_at(16 * kh + col, grp);
    const int rotary_key_at = rotary_at(16 * kh + col, grp);
    int value_at[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        // the first or second four of the lane's eight keys; the wave's 64 channels are eight units
        const int r = 8 * grp + 4 * i + (col >> 2);
        value_at[i] = latent_at(r, ((lane & 3) >> 1) + 8 * (wave & 1)) + (lane & 1) * 8 + (wave >> 1) * 256;
    }
    const int weight_from = col * 64 + ((grp ^ (col >> 2 & 3)) << 4);
    const int score_row = 16 * rq + col;  // this lane's row of the scores
    const int weight_to = score_row * 64 + (((2 * kh + (grp >> 1)) ^ (score_row >> 2 & 3)) << 4) + (grp & 1) * 8;
    auto meet = [] {
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_waitcnt(0xc07f);  // this wave's LDS accesses are done
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
    };
    Segment s;
    PageWalk pages;
    int32_t last = 0;  // key
    // Tile t's loads in five parts, so that they can be spread between products: a
    // queue that takes 16 cycles a load would hold up the wave. Of a tile past the
    // segment's they read nothing.
    struct Loads {
        __amdgpu_buffer_rsrc_t res;
        char* eight;
        int from, past;
    };
    auto prepare = [&](int32_t t, char* to) {
        // (unsigned: tiles past a segment's end may begin past 2^31 - 1)
        const uint32_t key = static_cast<uint32_t>(t) * kTile + 16 * (wave >> 2);
        const uint32_t final16 = static_cast<uint32_t>(last) & ~15u, first = min(key, final16);
        // (tiles are prepared in order: the row looked up is this one's)
        const char* const base = static_cast<const char*>(a.pool) + pages.take(a.view) * kRowBytes;
        pages.look(a.view, a.page_mul, min(key + kTile, final16));
        Loads d;
        d.res = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, t < s.tile1 ? 16 * kRowBytes : 0, kBufferWord3);
        d.eight = to + (wave >> 1) * kEightBytes;
        // rows past the last key: the last key's once more
        d.from = static_cast<int32_t>(key - first) + 4 * (wave & 3);
        d.past = static_cast<int32_t>(static_cast<uint32_t>(last) - first);
        return d;
    };
    auto load = [&](const Loads& d, int part) {
        if (part < 4) {
            buffer_lds16(d.res, d.eight + ((wave & 1) * 4 + part) * 1024,
                         static_cast<unsigned>(here(lane * 16) ^ swizzle(4 * (wave & 3) + part) << 4),
                         static_cast<unsigned>(min(d.from + part, d.past) * kRowBytes));
        } else if (lane < 32) {
            const int r = lane >> 3;
            buffer_lds16(d.res, d.eight + 8192 + (wave & 1) * 512,
                         static_cast<unsigned>(rotary_from + (min(d.from + r, d.past) - r) * kRowBytes), 0);
        }
    };
    auto issue = [&](int32_t t, char* to) {
        const Loads d = prepare(t, to);
#pragma unroll
        for (int part = 0; part < 5; ++part) {
            load(d, part);
        }
    };
    int in_request = 0, rows = 0;  // the block's first row in its request, and its rows
    int64_t row0 = 0;              // and in the output
    int32_t all_see = 0, sees = 0;
    vec8 q[18];
    // The next block's first tiles and queries.
    auto open = [&] {
        in_request = s.block * M;
        row0 = static_cast<int64_t>(s.req.first) * a.heads + in_request;
        rows = min(M, s.req.added * a.heads - in_request);
        last = s.req.cached + s.req.added - 1;
        pages.start(a.view, s.request);
        pages.look(a.view, a.page_mul, min(static_cast<uint32_t>(s.tile0) * kTile + 16 * (wave >> 2), static_cast<uint32_t>(last) & ~15u));
        if (s.tile0 < s.tile1) {
            issue(s.tile0, ring[0]);
        }
        if (s.tile0 + 1 < s.tile1) {
            issue(s.tile0 + 1, ring[1]);
        }
        const int own = min(score_row, rows - 1);
        const E* const from_q = static_cast<const E*>(a.q) + (row0 + own) * kWidth + 8 * grp;
#pragma unroll
        for (int ks = 0; ks < 18; ++ks) {
            q[ks] = *reinterpret_cast<const vec8*>(from_q + 32 * ks);
        }
        all_see = s.req.cached + in_request / a.heads;
        sees = s.req.cached + (in_request + own) / a.heads;
    };
    bool more = walk.next(a.view, s);
    if (more) {
        open();
    }
    if (tid < 4) {
        late_flags[tid] = 0;
    }
    while (more) {
        if (a.sign != 1) {
#pragma unroll
            for (int ks = 0; ks < 18; ++ks) {
                q[ks] = q[ks] * static_cast<E>(static_cast<float>(a.sign));
            }
        }
        f32x4 o[RB][4] = {};
        f32x4 sc;                 // scores of the newest tile
        float m = kLowest;        // reference of row `lane`, the same in every wave
        float ref = kLowest;      // of this lane's row of the scores
        float l = 0.0f, sum = 0.0f;  // its total, and the newest tile's
        // the newest tile's weights; their total is that of the rounded ones, so that what
        // is rounded away of a key that outweighs the others goes from both
        float over = kNone;
        auto exps = [&](char* wt) {
            vec4 p;
            float w[4];
            over = kNone;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                // (the difference first: c times a reference of 2^28 and more is off by more
                // than the range of the weights)
                const float x = __builtin_fmaf(sc[e] - ref, a.c, kLift<E>);
                over = fmaxf(over, x);
                p[e] = static_cast<E>(__builtin_amdgcn_exp2f(x));
                w[e] = static_cast<float>(p[e]);
            }
            sum = (w[0] + w[1]) + (w[2] + w[3]);
            *reinterpret_cast<vec4*>(wt + weight_to) = p;
        };
        // tells the others where a score passed the reference
        auto tell = [&](int u) {
            if (__builtin_expect(__any(over > kSlack + kLift<E>), 0)) {
                if (lane == 0) {
                    late_flags[u] = 1;
                }
            }
        };
        auto weigh = [&](char* wt, int u) {
            exps(wt);
            tell(u);
        };
        // The products of an interval: scores of the tile in `next` (S) in six steps,
        // then context of the tile in `now` (C) in four, each step's operands read
        // during the one before; `between(i)` runs ahead of step i's products. With
        // the scores first, their exponentials run beside the context's products (512
        // tokens after 3001: 93 us, and 99 with both kinds side by side).
        auto products = [&](auto with_scores, const char* next, auto with_context, const char* now, const char* wt,
                            bool sanitize, auto between) {
            constexpr bool S = decltype(with_scores)::value, C = decltype(with_context)::value;
            constexpr int kFrom = S ? 0 : 6, kTo = C ? 10 : 6;
            vec8 kf[2][3], vf[2], pf[RB];
            const int k_at = here(key_at), r_at = here(rotary_key_at);
            const int v_at[2] = {here(value_at[0]), here(value_at[1])};
            auto read = [&](int i) {
                if (i < 6) {
#pragma unroll
                    for (int k = 0; k < 3; ++k) {
                        const int ks = 3 * i + k;
                        kf[i & 1][k] = *reinterpret_cast<const vec8*>(
                            next + (ks < 16 ? (k_at ^ (ks & 3) << 6) + (ks >> 2) * 256 : r_at ^ (ks & 1) << 6));
                    }
                } else {  // channels 16 (i - 6) ..
                    if (i == 6) {
#pragma unroll
                        for (int rb = 0; rb < RB; ++rb) {
                            pf[rb] = *reinterpret_cast<const vec8*>(wt + weight_from + rb * 1024);
                        }
                    }
                    short8v v;
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const short4v part =
                            __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(now + (v_at[k] ^ (i - 6) << 5)));
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            v[4 * k + e] = part[e];
                        }
                    }
                    vf[i & 1] = __builtin_bit_cast(vec8, v);
                }
            };
            f32x4 odd{};
            if constexpr (S) {
                sc = f32x4{};
            }
            read(kFrom);
#pragma unroll
            for (int i = kFrom; i < kTo; ++i) {
                if (i + 1 < kTo) {
                    read(i + 1);
                }
                between(i);
                __builtin_amdgcn_sched_barrier(0);
                if (i >= 6) {
                    vec8 f = vf[i & 1];
                    if (sanitize) {
                        f = __builtin_bit_cast(vec8, finite_or_zero<E>(__builtin_bit_cast(short8v, f)));
                    }
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb) {
                        o[rb][i - 6] = H::mfma16(f, pf[rb], o[rb][i - 6]);
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < 3; ++k) {
                        f32x4& to = (3 * i + k) % 2 == 0 ? sc : odd;
                        to = H::mfma16(kf[i & 1][k], q[3 * i + k], to);
                    }
                    if (i == 5) {
                        sc += odd;
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        const std::true_type yes;
        const std::false_type no;
        const auto nothing = [](int) {};
        auto mask = [&](int32_t t) {
            if (t * kTile + kTile - 1 > all_see) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    sc[e] = t * kTile + 16 * kh + 4 * grp + e > sees ? kNone : sc[e];
                }
            }
        };
        // moves the reference to the rows' largest scores of the newest tile;
        // returns the factor of row `lane`'s sums so far
        auto follow = [&] {
            float high = fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3]));
            high = fmaxf(high, __shfl_xor(high, 16));
            high = fmaxf(high, __shfl_xor(high, 32));
            if (grp == 0) {
                tops[kh][score_row] = high;
            }
            meet();
            const int row = min(lane, rows - 1);  // (rows past the last are the last once more)
            const float up = fmaxf(m, fmaxf(tops[0][row], tops[1][row]));
            const float alpha = __builtin_amdgcn_exp2f((m - up) * a.c);
            m = up;
            ref = __shfl(up, score_row);
            return alpha;
        };
        // tile t's weights and tile t + 1 are in: all but tile t + 2's loads have come
        auto arrive = [&](int32_t t) {
            __builtin_amdgcn_sched_barrier(0);
            if (t + 2 >= s.tile1) {
                __builtin_amdgcn_s_waitcnt(0x0F70);
            } else {
                __builtin_amdgcn_s_waitcnt(0x0F70 | 5);
            }
            meet();
        };
        if (s.tile0 < s.tile1) {
            arrive(s.tile0 - 1);
            if (s.tile0 + 2 < s.tile1) {
                issue(s.tile0 + 2, ring[2]);
            }
            products(yes, ring[0], no, nullptr, nullptr, false, nothing);
            mask(s.tile0);
            follow();
            weigh(weights[0], 0);
            // tiles up to here are seen by all rows, and the next one too
            const int32_t full = min(s.tile1 - 1, (all_see + 1) / kTile - 1);
            int32_t t = s.tile0;
            while (t < s.tile1) {
                // A reference left behind, or a tile that rows may not see, is
                // for the loop after this one: the sums are touched by products
                // alone here, and stay in the registers that products use.
                int stop = 0;
                bool arrived = false;
                while (stop == 0) {
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        if (t + u >= full) {
                            stop = u + 1;
                            break;
                        }
                        arrive(t + u);
                        if (__builtin_expect(__builtin_amdgcn_readfirstlane(late_flags[u]) != 0, 0)) {
                            stop = u + 1;
                            arrived = true;
                            break;
                        }
                        if (tid == 0) {
                            late_flags[(u + 2) & 3] = 0;
                        }
                        l += sum;
                        const Loads d = prepare(t + u + 3, ring[(u + 3) & 3]);
                        products(yes, ring[(u + 1) & 3], yes, ring[u], weights[u & 1], false, [&](int i) {
                            if (i > 0 && i < 6) {
                                load(d, i - 1);
                            }
                            if (i == 7) {
                                exps(weights[(u + 1) & 1]);
                            }
                        });
                        tell((u + 1) & 3);
                    }
                    t += stop == 0 ? 4 : 0;
                }
                // one copy of the code for all stages, to which the compiler's
                // tracking does not reach: it waits for every load here
#pragma unroll 1
                for (int u = stop - 1; u < 4 && t + u < s.tile1; ++u) {
                    if (!arrived) {
                        arrive(t + u);
                    }
                    arrived = false;
                    auto stage = [&](int i) {
                        const int at = (i & 3) == 0   ? lds_address(s0)
                                       : (i & 3) == 1 ? lds_address(s1)
                                       : (i & 3) == 2 ? lds_address(s2)
                                                      : lds_address(s3);
                        return (const char*)(lds_char*)static_cast<uintptr_t>(here(at));
                    };
                    if (__builtin_amdgcn_readfirstlane(late_flags[u]) != 0) {
                        const float alpha = follow();
#pragma unroll
                        for (int rb = 0; rb < RB; ++rb) {
                            const float f = __shfl(alpha, 16 * rb + col);
#pragma unroll
                            for (int ct = 0; ct < 4; ++ct) {
                                o[rb][ct] *= f;
                            }
                        }
                        l *= __shfl(alpha, score_row);
                        weigh(weights[u & 1], u);
                        meet();
                    }
                    if (tid == 0) {
                        late_flags[(u + 2) & 3] = 0;
                    }
                    l += sum;
                    if (t + u + 3 < s.tile1) {
                        if (u == 0) {
                            issue(t + u + 3, ring[3]);
                        } else if (u == 1) {
                            issue(t + u + 3, ring[0]);
                        } else if (u == 2) {
                            issue(t + u + 3, ring[1]);
                        } else {
                            issue(t + u + 3, ring[2]);
                        }
                    }
                    if (t + u + 1 < s.tile1) {
                        products(yes, stage(u + 1), no, nullptr, nullptr, false, nothing);
                        mask(t + u + 1);
                    }
                    products(no, nullptr, yes, stage(u), weights[u & 1], (t + u) * kTile + kTile - 1 > all_see, nothing);
                    if (t + u + 1 < s.tile1) {
                        weigh(weights[(u + 1) & 1], (u + 1) & 3);
                    }
                }
                t += 4;
            }
        }
        // The totals: the rows' parts of both key halves meet in `tops`. The next
        // block's loads start before this one's results go out.
        meet();
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        if (grp == 0) {
            tops[kh][score_row] = l;
        }
        if (tid < 4) {
            late_flags[tid] = 0;
        }
        const bool whole = s.begins && s.ends;
        const int32_t parts_after = s.begins && !s.ends ? s.parts_after : -1;
        const int64_t slot = 2 * static_cast<int64_t>(blockIdx.x) + (s.begins ? 1 : 0);
        const int64_t out_row = row0;
        const int out_rows = rows;
        more = walk.next(a.view, s);
        if (more) {
            open();
        }
        meet();
        // o[rb][ct] register e: channel 64 wave + 16 ct + 4 grp + e of row 16 rb + col
        if (whole) {
            // through LDS (stages 2 and 3: the next block's first tiles are in 0 and
            // 1), so that rows go out whole; units XORed by row
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                const int row = min(16 * rb + col, out_rows - 1);
                const float inv = 1.0f / (tops[0][row] + tops[1][row]);
                char* const to = (rb < 2 ? s2 : s3) + (16 * (rb & 1) + col) * 1024;
#pragma unroll
                for (int ct = 0; ct < 4; ++ct) {
                    vec4 out;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        out[e] = static_cast<E>(o[rb][ct][e] * inv);
                    }
                    *reinterpret_cast<vec4*>(to + (((8 * wave + 2 * ct + (grp >> 1)) ^ col) << 4) + (grp & 1) * 8) = out;
                }
            }
            meet();
#pragma unroll
            for (int i = 0; i < M / kWaves; ++i) {
                const int row = M / kWaves * wave + i;
                if (row < out_rows) {
                    const char* const from = (row < 32 ? s2 : s3) + (row & 31) * 1024 + ((lane ^ (row & 15)) << 4);
                    *reinterpret_cast<u32x4*>(static_cast<E*>(a.out) + (out_row + row) * kRank + 8 * lane) =
                        *reinterpret_cast<const u32x4*>(from);
                }
            }
        } else {
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                const int row = 16 * rb + col;
                if (row < out_rows) {
                    float* const to = a.parts.sums + (slot * M + row) * kRank + 64 * wave + 4 * grp;
#pragma unroll
                    for (int ct = 0; ct < 4; ++ct) {
                        *reinterpret_cast<f32x4*>(to + 16 * ct) = o[rb][ct];
                    }
                }
            }
            if (tid < out_rows) {
                float* const to = a.parts.stats + (slot * M + tid) * 2;
                to[0] = m * a.c;
                to[1] = tops[0][tid] + tops[1][tid];
            }
            if (parts_after >= 0 && tid == 0) {
                a.parts.heads[blockIdx.x] = PartHead{out_row, out_rows, parts_after};
            }
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
// A workgroup per token and head (in turn, past 2^20 of them), its four waves on alternate keys, a lane on
// channels lane + 64 i; running maximum and sum per wave, joined at the end.
constexpr int kMaxRank = 1024, kMaxRope = 256;

template <class E>
__global__ __launch_bounds__(256) void paged_any_kernel(const PagedAttention a) {
    constexpr int kC = kMaxRank / 64, kR = kMaxRope / 64;
    __shared__ float part[4][kMaxRank], stats[4][2];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t rows = static_cast<int64_t>(a.view.tokens) * a.heads;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const int32_t t = static_cast<int32_t>(row / a.heads), h = static_cast<int32_t>(row % a.heads);
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
            continue;  // past the last request's rows
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
        for (uint32_t j = wave; j < static_cast<uint32_t>(keys); j += 4) {
            const uint32_t size = static_cast<uint32_t>(v.page_size);
            const int64_t page = checked_page(v, v.table[static_cast<int64_t>(lo) * v.table_width + j / size]);
            const E* const key = static_cast<const E*>(a.pool) + (page * v.page_size + j % size) * width;
            float c[kC], s = 0.0f;
#pragma unroll
            for (int i = 0; i < kC; ++i) {
                c[i] = lane + 64 * i < a.rank ? static_cast<float>(key[lane + 64 * i]) : 0.0f;
                s = __builtin_fmaf(qc[i], c[i], s);
            }
#pragma unroll
            for (int i = 0; i < kR; ++i) {
                s = __builtin_fmaf(qr[i], lane + 64 * i < a.rope ? static_cast<float>(key[a.rank + lane + 64 * i]) : 0.0f,
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
        __syncthreads();  // `part` is free again
    }
}

template <class E>
hipError_t launch(const PagedAttention& a, void* workspace, hipStream_t s) {
    if (!paged_tiled(a.rank, a.rope)) {
        hipLaunchKernelGGL(paged_any_kernel<E>, dim3(static_cast<unsigned>(std::min(static_cast<int64_t>(a.view.tokens) * a.heads, int64_t{1} << 20))),
                           dim3(256), 0, s, a);
        return hipGetLastError();
    }
    TileArgs t;
    t.view = a.view;
    t.q = a.q;
    t.pool = a.pool;
    t.out = a.out;
    t.heads = a.heads;
    t.sign = a.scale < 0.0f ? -1 : a.scale > 0.0f ? 1 : 0;
    t.page_mul = static_cast<uint32_t>(((uint64_t{1} << 32) + a.view.page_size / 16 - 1) / (a.view.page_size / 16));
    // (above 0 for any scale: scores of keys that a row may not see are -infinity times it)
    t.c = t.sign == 0 ? 1.0f : std::fabs(a.scale) * 1.4426950408889634f;
    char* w = static_cast<char*>(workspace);
    const int m = paged_block_rows(a.max_added, a.heads);
    t.parts.heads = reinterpret_cast<PartHead*>(w);
    w += round_up(sizeof(PartHead) * kGrid, 256);
    t.parts.stats = reinterpret_cast<float*>(w);
    w += round_up(sizeof(float) * 2 * kGrid * m * 2, 256);
    t.parts.sums = reinterpret_cast<float*>(w);
    if (m == 16) {
        hipLaunchKernelGGL((paged_rows_kernel<E, 16>), dim3(kGrid), dim3(kThreads), 0, s, t);
    } else {
        hipLaunchKernelGGL((paged_rows_kernel<E, 64>), dim3(kGrid), dim3(kThreads), 0, s, t);
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

bool paged_shares_out(int64_t tokens, int32_t heads, int64_t room) {
    const double rows = static_cast<double>(tokens) * heads;
    return (rows / 16 + static_cast<double>(tokens)) * ((static_cast<double>(room) + kExtra) * heads + rows + 64) < 0x1p62;
}

// 16 rows where no request has more (one token of 32 requests, 16 heads, three
// contexts in turn: 22 us, in blocks of 64 25), or else 64 (32 heads: 28 us, in
// blocks of 16 34).
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
