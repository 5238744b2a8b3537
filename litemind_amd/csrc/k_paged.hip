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
//   many (paged_rows64_kernel): 64 rows, tiles and products shared by the waves
// Any other widths take paged_any_kernel.
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

// The same value, made anew where it stands: kept from becoming a register that
// lives through a loop for every constant that is added to it.
__device__ inline int here(int v) {
    asm volatile("" : "+v"(v));
    return v;
}

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
        const int rows = min(kRows16, s.req.added * a.heads - s.block * kRows16);
        const int32_t keys = s.req.cached + s.req.added;
        // this lane's query row; the last key that it sees, and that all rows see
        const int own = min(col, rows - 1);
        const int32_t sees = s.req.cached + (s.block * kRows16 + own) / a.heads;
        const int32_t all_see = s.req.cached + s.block * kRows16 / a.heads;
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

// ---- many rows ----
// 64 query rows, four waves. The waves share tiles of 32 keys, which come straight
// to LDS four deep, and split each product differently:
//   S^T   wave (kh, rh): keys 16 kh .. + 15 for rows 32 rh .. + 31; its queries
//         stay in 144 registers, 36 products of 16 x 16 x 32 a tile
//   out^T channels 128 w .. + 127 of wave w for all rows; 128 registers of sums,
//         16 products of 32 x 32 x 16 a tile
// The weights pass through LDS. One barrier a tile: between two, the waves run
// the scores of tile t + 1 and the context of tile t, which do not depend on each
// other, so either's latencies are filled by the other's products. 32 rows with
// all 512 channels per wave, without the exchange, would take 256 + 16 registers
// of sums, and the matrix cores' results go to 256.
//
// The weights' reference m, one per row, has to be the same for all waves: it
// follows the rows' maxima one barrier late, and only where a row passed it by
// more than 2^kSlack, which keeps the weights in 16 bits' range; the tile's
// weights are then made anew. (fp32 sums do not mind the factor.)
constexpr int kRows64 = 64;
constexpr float kSlack = 10.0f;

// Non-finite values as 0: keys that some row must not see weigh 0 there, and 0
// times NaN or infinity is not 0. (Rows that see such a key have a NaN weight.)
template <class E>
__device__ inline short8v finite_or_zero(short8v v) {
    constexpr short kExponent = sizeof(E) == 2 && __is_same(E, bf16) ? 0x7f80 : 0x7c00;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        v[e] = (v[e] & kExponent) == kExponent ? short{0} : v[e];
    }
    return v;
}

template <class E>
__global__ __launch_bounds__(256, 1) void paged_rows64_kernel(const TileArgs a) {
    using H = Half<E>;
    typedef typename H::vec8 vec8;
    typedef typename H::vec4 vec4;
    // one array per stage: the compiler tracks loads to LDS per array
    __shared__ __align__(16) char s0[kTileBytes], s1[kTileBytes], s2[kTileBytes], s3[kTileBytes];
    __shared__ __align__(16) char weights[2][kRows64 * kTile * 2];
    __shared__ float tops[2][2][kRows64];
    __shared__ int64_t scratch[8];
    char* const ring[4] = {s0, s1, s2, s3};
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kh = wave & 1, rh = wave >> 1;
    const int col = lane & 15, grp = lane >> 4;     // of 16 x 16 products
    const int col32 = lane & 31, half = lane >> 5;  // of 32 x 32 products
    Walk walk;
    walk.sh = Shares{a.heads, kRows64};
    walk.p = find_piece(a.view, walk.sh, blockIdx.x, scratch);
    if (tid == 0) {
        a.parts.heads[blockIdx.x].rows = 0;
    }
    if (walk.p.begin >= walk.p.end) {
        return;
    }
    walk.start(a.view);
    // The wave loads rows 8 wave .. + 7 of a tile, 9 loads of 64 units.
    auto place = [&](int j, int of, int& row, int& unit) {
        const int at = 64 * j + of;
        const int r = at / kUnits;
        row = 8 * (wave & 1) + r;  // of 16
        unit = (at - r * kUnits) ^ swizzle(row);
    };
    unsigned from[9];
#pragma unroll
    for (int j = 0; j < 9; ++j) {
        int row, unit;
        place(j, lane, row, unit);
        from[j] = static_cast<unsigned>(row * kRowBytes + unit * 16);
    }
    // Where the lane's reads of a tile begin; the rest is constant offsets, since
    // the swizzle changes the low three bits of a unit only.
    int key_at[2], value_at[2][2], weight_from[2], weight_to[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        key_at[i] = unit_at(16 * kh + col, 4 * i + grp);
        const int row = 32 * i + col32, to = 32 * rh + 16 * i + col;
        weight_from[i] = row * 64 + ((half ^ (row >> 2 & 1)) * 16 | (row >> 3 & 1) * 32);
        weight_to[i] = to * 64 + ((2 * kh + (grp >> 1)) ^ (to >> 2 & 3)) * 16 + (grp & 1) * 8;
#pragma unroll
        for (int odd = 0; odd < 2; ++odd) {
            const int r = 8 * half + 4 * i + ((lane & 15) >> 2);
            value_at[i][odd] = unit_at(r, 4 * odd + 2 * (lane >> 4 & 1) + ((lane & 3) >> 1)) + (lane & 1) * 8 +
                               wave * 256;
        }
    }
    Segment s;
    while (walk.next(a.view, s)) {
        const int in_request = s.block * kRows64;  // the block's first row
        const int64_t row0 = static_cast<int64_t>(s.req.first) * a.heads + in_request;
        const int rows = min(kRows64, s.req.added * a.heads - in_request);
        const int32_t last = s.req.cached + s.req.added - 1;
        const int32_t all_see = s.req.cached + in_request / a.heads;
        int32_t sees[2];
        vec8 q[2][18];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
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
            for (int ks = 0; ks < 18; ++ks) {
                q[0][ks] = -q[0][ks];
                q[1][ks] = -q[1][ks];
            }
        }
        PageWalk pages;
        pages.start(a.view, s.request);
        auto issue = [&](int32_t t, char* to) {
            const int32_t key = t * kTile + 16 * (wave >> 1);
            const int32_t first = min(key, last & ~15);
            const char* const base =
                static_cast<const char*>(a.pool) + pages.at(a.view, a.page_mul, first) * kRowBytes;
            const __amdgpu_buffer_rsrc_t res =
                __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, 16 * kRowBytes, kBufferWord3);
            to += 8 * wave * kRowBytes;
            if (key + 15 <= last) {
#pragma unroll
                for (int j = 0; j < 9; ++j) {
                    buffer_lds16(res, to + j * 1024, from[j], 0);
                }
            } else {  // rows past the last key: the last key's once more
                const int of = here(lane);
#pragma unroll
                for (int j = 0; j < 9; ++j) {
                    int row, unit;
                    place(j, of, row, unit);
                    const int r = min(key + row, last) - first;
                    buffer_lds16(res, to + j * 1024, static_cast<unsigned>(r * kRowBytes + unit * 16), 0);
                }
            }
        };
        f32x16 o[2][4] = {};
        f32x4 sc[2];             // scores of the newest tile
        float m = kNone;         // reference of row `lane`, the same in every wave
        float ref[2];            // times c, of this lane's rows of the scores
        float l[2] = {0.0f, 0.0f};
        ref[0] = ref[1] = 0.0f;
        // The products of an interval in eight steps, each step's operands read
        // during the one before: k-steps 9 i / 4 .. of the scores of the tile in
        // `next`, channel tile i % 4 of keys 16 (i / 4) .. of the context of the
        // tile in `now`.
        auto products = [&](auto with_scores, const char* next, auto with_context, const char* now, const char* wt,
                            auto sanitize) {
            constexpr bool S = decltype(with_scores)::value, C = decltype(with_context)::value;
            vec8 kf[2][3], vf[2], pf[2][2];
            const int k_at[2] = {here(key_at[0]), here(key_at[1])};
            const int v_at[2][2] = {{here(value_at[0][0]), here(value_at[0][1])},
                                    {here(value_at[1][0]), here(value_at[1][1])}};
            auto read = [&](int i) {
                if constexpr (S) {
#pragma unroll
                    for (int ks = 9 * i / 4; ks < 9 * (i + 1) / 4; ++ks) {
                        kf[i & 1][ks - 9 * i / 4] =
                            *reinterpret_cast<const vec8*>(next + k_at[ks & 1] + (ks >> 1) * 128);
                    }
                }
                if constexpr (C) {
                    const int st = i / 4, ct = i % 4;
                    if (ct == 0) {
#pragma unroll
                        for (int rb = 0; rb < 2; ++rb) {
                            pf[st][rb] = *reinterpret_cast<const vec8*>(wt + (weight_from[rb] ^ st * 32));
                        }
                    }
                    short8v v;
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const short4v part = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (lds_short4*)(now + v_at[k][ct & 1] + st * 16 * kRowBytes + (ct >> 1) * 128));
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            v[4 * k + e] = part[e];
                        }
                    }
                    vf[i & 1] = __builtin_bit_cast(vec8, v);
                }
            };
            if constexpr (S) {
                sc[0] = sc[1] = f32x4{};
            }
            read(0);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (i < 7) {
                    read(i + 1);
                }
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (C) {
                    vec8 f = vf[i & 1];
                    if constexpr (decltype(sanitize)::value) {
                        f = __builtin_bit_cast(vec8, finite_or_zero<E>(__builtin_bit_cast(short8v, f)));
                    }
                    o[0][i % 4] = H::mfma32(f, pf[i / 4][0], o[0][i % 4]);
                    o[1][i % 4] = H::mfma32(f, pf[i / 4][1], o[1][i % 4]);
                }
                if constexpr (S) {
#pragma unroll
                    for (int ks = 9 * i / 4; ks < 9 * (i + 1) / 4; ++ks) {
                        const vec8 k = kf[i & 1][ks - 9 * i / 4];
                        sc[0] = H::mfma16(k, q[0][ks], sc[0]);
                        sc[1] = H::mfma16(k, q[1][ks], sc[1]);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        auto mask = [&](int32_t t) {
            if (t * kTile + kTile - 1 > all_see) {
#pragma unroll
                for (int b = 0; b < 2; ++b) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        sc[b][e] = t * kTile + 16 * kh + 4 * grp + e > sees[b] ? kNone : sc[b][e];
                    }
                }
            }
        };
        // the rows' maxima of the newest tile
        auto pass = [&](float (*top)[kRows64]) {
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                float high = fmaxf(fmaxf(sc[b][0], sc[b][1]), fmaxf(sc[b][2], sc[b][3]));
                high = fmaxf(high, __shfl_xor(high, 16));
                high = fmaxf(high, __shfl_xor(high, 32));
                if (grp == 0) {
                    top[kh][32 * rh + 16 * b + col] = high;
                }
            }
        };
        auto weigh = [&](char* wt, float (&sum)[2]) {
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                vec4 p;
                sum[b] = 0.0f;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[b][e], a.c, -ref[b]));
                    sum[b] += w;
                    p[e] = static_cast<E>(w);
                }
                *reinterpret_cast<vec4*>(wt + weight_to[b]) = p;
            }
        };
        auto meet = [] {
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_waitcnt(0xc07f);  // the weights are written
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_sched_barrier(0);
        };
        __syncthreads();  // the block before is done with the ring
        if (s.tile0 < s.tile1) {
            issue(s.tile0, ring[0]);
        }
        if (s.tile0 + 1 < s.tile1) {
            issue(s.tile0 + 1, ring[1]);
        }
        float sum[2] = {0.0f, 0.0f};  // of the newest tile's weights
        // Between two barriers: context of tile t (stage u), scores of t + 1.
        const std::true_type yes;
        const std::false_type no;
        // tile t's weights and tile t + 1 are in
        auto arrive = [&](int32_t t, int u) {
            __builtin_amdgcn_sched_barrier(0);
            if (t + 2 < s.tile1) {
                __builtin_amdgcn_s_waitcnt(0x0F70 | 9);
            } else {
                __builtin_amdgcn_s_waitcnt(0x0F70);
            }
            meet();
            if (t + 3 < s.tile1) {
                issue(t + 3, ring[(u + 3) & 3]);
            }
        };
        // the largest score of row `lane` in the tile whose maxima are in `top`
        auto largest = [&](const float (*top)[kRows64]) {
            return lane < rows ? fmaxf(top[0][lane], top[1][lane]) : kNone;
        };
        auto follow = [&](float high, float* alpha) {
            const float up = fmaxf(m, high);
            *alpha = up == kNone ? 1.0f : __builtin_amdgcn_exp2f((m - up) * a.c);
            m = up;
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const float mine = __shfl(up, 32 * rh + 16 * b + col);
                ref[b] = mine == kNone ? 0.0f : mine * a.c;
            }
        };
        if (s.tile0 < s.tile1) {
            arrive(s.tile0 - 1, 3);
            products(yes, ring[0], no, nullptr, nullptr, no);
            mask(s.tile0);
            pass(tops[0]);
            meet();
            float alpha;
            follow(largest(tops[0]), &alpha);
            weigh(weights[0], sum);
            // tiles up to here are seen by all rows, and the next one too
            const int32_t full = min(s.tile1 - 1, (all_see + 1) / kTile - 1);
            int32_t t = s.tile0;
            while (t < s.tile1) {
                // A reference left behind, or a tile that rows may not see, is
                // for the loop after this one: the sums are touched by products
                // alone here, and stay in the registers that products use.
                int late = 0;
                float high = kNone;
                for (; t + 4 <= full; t += 4) {
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        arrive(t + u, u);
                        high = largest(tops[u & 1]);
                        if (__builtin_expect(__any((high - m) * a.c > kSlack), 0)) {
                            late = u + 1;
                            break;
                        }
                        l[0] += sum[0];
                        l[1] += sum[1];
                        products(yes, ring[(u + 1) & 3], yes, ring[u], weights[u & 1], no);
                        pass(tops[(u + 1) & 1]);
                        weigh(weights[(u + 1) & 1], sum);
                    }
                    if (late != 0) {
                        break;
                    }
                }
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    if (u + 1 >= late && t + u < s.tile1) {
                        if (u + 1 != late) {
                            arrive(t + u, u);
                            high = largest(tops[u & 1]);
                        }
                        if (__any((high - m) * a.c > kSlack)) {
                            follow(high, &alpha);
#pragma unroll
                            for (int rb = 0; rb < 2; ++rb) {
                                const float f = __shfl(alpha, 32 * rb + col32);
#pragma unroll
                                for (int ct = 0; ct < 4; ++ct) {
                                    o[rb][ct] *= f;
                                }
                            }
                            l[0] *= __shfl(alpha, 32 * rh + col);
                            l[1] *= __shfl(alpha, 32 * rh + 16 + col);
                            weigh(weights[u & 1], sum);
                            meet();
                        }
                        l[0] += sum[0];
                        l[1] += sum[1];
                        if (t + u + 1 < s.tile1) {
                            products(yes, ring[(u + 1) & 3], no, nullptr, nullptr, no);
                            mask(t + u + 1);
                        }
                        products(no, nullptr, yes, ring[u], weights[u & 1], yes);
                        if (t + u + 1 < s.tile1) {
                            pass(tops[(u + 1) & 1]);
                            weigh(weights[(u + 1) & 1], sum);
                        }
                    }
                }
                t += 4;
            }
        }
        // the totals: the rows' parts of both key halves meet in `tops`
        __syncthreads();
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            l[b] += __shfl_xor(l[b], 16);
            l[b] += __shfl_xor(l[b], 32);
            if (grp == 0) {
                tops[0][kh][32 * rh + 16 * b + col] = l[b];
            }
        }
        __syncthreads();
        const bool whole = s.begins && s.ends;
        const int slot = 2 * static_cast<int>(blockIdx.x) + (s.begins ? 1 : 0);
        // o[rb][ct] register e: channel 128 wave + 32 ct + 8 (e / 4) + 4 half + e % 4 of row 32 rb + col32
#pragma unroll
        for (int rb = 0; rb < 2; ++rb) {
            const int row = 32 * rb + col32;
            if (row < rows) {
                if (whole) {
                    const float inv = 1.0f / (tops[0][0][row] + tops[0][1][row]);
                    E* const to = static_cast<E*>(a.out) + (row0 + row) * kRank + 128 * wave + 4 * half;
#pragma unroll
                    for (int ct = 0; ct < 4; ++ct) {
#pragma unroll
                        for (int g = 0; g < 4; ++g) {
                            vec4 out;
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                out[e] = static_cast<E>(o[rb][ct][4 * g + e] * inv);
                            }
                            *reinterpret_cast<vec4*>(to + 32 * ct + 8 * g) = out;
                        }
                    }
                } else {
                    float* const to = a.parts.sums + (static_cast<int64_t>(slot) * kRows64 + row) * kRank + 128 * wave +
                                      4 * half;
#pragma unroll
                    for (int ct = 0; ct < 4; ++ct) {
#pragma unroll
                        for (int g = 0; g < 4; ++g) {
                            f32x4 out;
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                out[e] = o[rb][ct][4 * g + e];
                            }
                            *reinterpret_cast<f32x4*>(to + 32 * ct + 8 * g) = out;
                        }
                    }
                }
            }
        }
        if (!whole && tid < rows) {
            float* const to = a.parts.stats + (static_cast<int64_t>(slot) * kRows64 + tid) * 2;
            to[0] = m == kNone ? kNone : m * a.c;
            to[1] = tops[0][0][tid] + tops[0][1][tid];
        }
        if (s.begins && !s.ends && tid == 0) {
            a.parts.heads[blockIdx.x] = PartHead{row0, rows, s.parts_after};
        }
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
    const int m = paged_block_rows(a.max_added, a.heads);
    t.parts.heads = reinterpret_cast<PartHead*>(w);
    w += round_up(sizeof(PartHead) * kGrid, 256);
    t.parts.stats = reinterpret_cast<float*>(w);
    w += round_up(sizeof(float) * 2 * kGrid * m * 2, 256);
    t.parts.sums = reinterpret_cast<float*>(w);
    if (m == kRows16) {
        hipLaunchKernelGGL(paged_rows16_kernel<E>, dim3(kGrid), dim3(256), 0, s, t);
    } else {
        hipLaunchKernelGGL(paged_rows64_kernel<E>, dim3(kGrid), dim3(256), 0, s, t);
    }
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) {
        return err;
    }
    if (m == kRows16) {
        hipLaunchKernelGGL((paged_join_kernel<E, kRows16>), dim3(kGrid, kRows16), dim3(256), 0, s, t);
    } else {
        hipLaunchKernelGGL((paged_join_kernel<E, kRows64>), dim3(kGrid, 16), dim3(256), 0, s, t);
    }
    return hipGetLastError();
}

}  // namespace

bool paged_tiled(int32_t rank, int32_t rope) { return rank == kRank && rope == kRope; }

int paged_block_rows(int32_t max_added, int32_t heads) {
    return static_cast<int64_t>(max_added) * heads <= kRows16 ? kRows16 : kRows64;
}

int64_t paged_workspace_bytes(int rows) {
    return round_up(sizeof(PartHead) * kGrid, 256) + round_up(sizeof(float) * 2 * kGrid * rows * 2, 256) +
           static_cast<int64_t>(sizeof(float)) * 2 * kGrid * rows * kRank;
}

hipError_t launch_paged_attention(const PagedAttention& a, void* workspace, hipStream_t s) {
    return a.bf16 != 0 ? launch<bf16>(a, workspace, s) : launch<_Float16>(a, workspace, s);
}

}  // namespace lm
