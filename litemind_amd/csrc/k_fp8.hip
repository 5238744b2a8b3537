// k_fp8.hip -- products of FP8 rows with FP8 matrices, one matrix or one for
// each group of rows (lm_fp8_gemm, lm_fp8_grouped_gemm), and the gate and up
// products that end in SwiGLU and FP8 blocks again (lm_fp8_grouped_swiglu).
//
// Mathematics.  Rows and weights carry a scale per block of 128 reduced
// channels, so
//     out[r][n] = sum_b (sa[r][b] sw[n / 128][b]) sum_{k in b} a[r][k] w[n][k].
// The inner sum over a block starts from zero on the matrix cores, and its
// results are taken into the fp32 sums by a fused multiply-add with the product
// of the two scales.  The weights are the matrix instruction's first operand and
// the rows its second, so a lane's four results are four neighbouring features
// of one row, which share both scales: 4 FMAs (16 clocks) beside 32 clocks (FP8)
// or 64 (fp16) of the matrix core.
//
// Two kinds of inner sums.  v_mfma_f32_16x16x128_f8f6f4 takes a block at once,
// but adds its products in groups of eight neighbours, each cut 13 bits under
// the largest exponent of its group (measured, instruction by itself): the sums
// are off by 1.4e-5 of their norm (2.7e-5 to 3.7e-5 where a few channels are far
// larger), at most 7 2^-13 of the sum of magnitudes.  That is a hundredth of what
// rounding to BF16 takes and a fifteenth of fp16's, so outputs of 16 bits use it.
// Outputs that keep more of their sums (fp32, and SwiGLU's fp32 scales) convert
// the codes to fp16, exactly, and take four v_mfma_f32_16x16x32_f16, whose
// sums are fp32's, at half the rate.
//
// Operand layout.  Lane l holds 32 codes of row l & 15: the 16-byte chunks
// l >> 4 and 4 + (l >> 4) of the row's 128 bytes.  Which 32 of the 128 channels a
// lane quarter holds does not matter as long as both operands agree, and so
// four lanes read 64 contiguous bytes of a row.
//
// A reduced axis that ends inside a block: the chunks past it are zeros in the
// rows' operand and the row's first chunk in the weights' (never bytes of
// another row, whose NaN would come through).
#include "fp8_internal.h"

#include <algorithm>
#include <cmath>

namespace lm {
namespace {

typedef int intx8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef _Float16 halfx2 __attribute__((ext_vector_type(2)));
typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));

constexpr int kXcds = 8;

// s_waitcnt with only vmcnt (expcnt and lgkmcnt at their maxima)
#define LM_WAIT_VM(n) __builtin_amdgcn_s_waitcnt(((n) & 15) | (((n) >> 4) << 14) | 0x0F70)

// Thirty-two codes of a lane as a matrix operand, and the sum over a block.
template <bool EXACT>
struct Operand;
template <>
struct Operand<false> {
    intx8 v;
    __device__ void set(uint4 lo, uint4 hi) {
        v = intx8{static_cast<int>(lo.x), static_cast<int>(lo.y), static_cast<int>(lo.z), static_cast<int>(lo.w),
                  static_cast<int>(hi.x), static_cast<int>(hi.y), static_cast<int>(hi.z), static_cast<int>(hi.w)};
    }
};
template <>
struct Operand<true> {
    halfx8 v[4];
    __device__ static halfx8 widen(uint32_t lo, uint32_t hi) {
        const halfx2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false),
                     b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true),
                     c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false),
                     d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
        return halfx8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
    }
    __device__ void set(uint4 lo, uint4 hi) {
        v[0] = widen(lo.x, lo.y);
        v[1] = widen(lo.z, lo.w);
        v[2] = widen(hi.x, hi.y);
        v[3] = widen(hi.z, hi.w);
    }
};
__device__ inline floatx4 block_sum(const Operand<false>& w, const Operand<false>& a) {
    const floatx4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w.v, a.v, zero, 0, 0, 0, 0, 0, 0);
}
__device__ inline floatx4 block_sum(const Operand<true>& w, const Operand<true>& a) {
    floatx4 d = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        d = __builtin_amdgcn_mfma_f32_16x16x32_f16(w.v[q], a.v[q], d, 0, 0, 0);
    }
    return d;
}

__device__ inline void report(const Fp8Product& p) {
    __hip_atomic_store(p.error, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
}

__device__ inline void take(floatx4& acc, floatx4 d, float scale) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        acc[u] = __builtin_fmaf(d[u], scale, acc[u]);
    }
}

// ---- which rows and features a workgroup computes ----

struct Tile {
    int32_t g;      // group
    int32_t mt, nt; // row tile and feature tile inside the group
    int32_t first;  // the group's first row
    int32_t rows;   // its rows
};

// First row and rows of group g, within the arrays whatever the offsets say.
__device__ inline void group_rows(const Fp8Product& p, int g, int32_t& first, int32_t& rows) {
    const int32_t from = p.offsets[g], to = p.offsets[g + 1];
    const int32_t most = static_cast<int32_t>(p.rows);
    first = min(max(from, 0), most);
    rows = max(0, min(to, most) - first);
    if (from < 0 || to < from || to > most) {
        report(p);
    }
}

// The tile of workgroup blockIdx.x, the same in every wave (each looks for it
// by itself: no barrier). Workgroup b runs on XCD b % 8; every XCD takes a
// contiguous eighth of the tiles, in which the row tiles of one feature tile
// follow each other, so that their weights are read from one L2. The first `beside`
// tiles are another product's, whose group is -1 here, of rows_beside rows.
__device__ inline bool find_tile(const Fp8Product& p, int bm, int nts, Tile& t, int32_t beside = 0,
                                 int32_t rows_beside = 0) {
    const int lane = threadIdx.x & 63;
    // the workgroup's place among all tiles, from which `beside` count back; none: INT32_MIN
    auto share = [&](int32_t total) {
        total += beside;
        const int32_t xcd = blockIdx.x % kXcds, idx = blockIdx.x / kXcds;
        const int32_t per = total / kXcds, extra = total % kXcds;
        return idx < per + (xcd < extra ? 1 : 0) ? xcd * per + min(xcd, extra) + idx - beside : INT32_MIN;
    };
    auto take_beside = [&](int32_t tile) {
        const int32_t mts = (rows_beside + bm - 1) / bm;
        t = Tile{-1, (tile + beside) % mts, (tile + beside) / mts, 0, rows_beside};
        return true;
    };
    if (p.offsets == nullptr) {
        const int32_t mts = static_cast<int32_t>((p.rows + bm - 1) / bm);
        const int32_t tile = share(mts * nts);
        t = Tile{0, tile % mts, tile / mts, 0, static_cast<int32_t>(p.rows)};
        return tile >= 0;
    }
    // The host's bound on the tiles keeps every sum of good offsets under kMost;
    // offsets that fall may count rows twice, and then sums stay there.
    constexpr int32_t kMost = 1 << 28;
    auto inclusive = [&](int32_t v) {
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int32_t u = __shfl_up(v, o);
            v = min(v + (lane >= o ? u : 0), kMost);
        }
        return v;
    };
    int32_t first = 0, rows = 0, sum = 0, total = 0;
    for (int g0 = 0; g0 < p.groups; g0 += 64) {
        rows = 0;
        if (g0 + lane < p.groups) {
            group_rows(p, g0 + lane, first, rows);
        }
        sum = inclusive((rows + bm - 1) / bm * nts);
        total = min(total + __builtin_amdgcn_readlane(sum, 63), kMost);
    }
    const int32_t tile = share(total);
    if (tile < 0) {
        return tile != INT32_MIN && take_beside(tile);
    }
    int32_t before = 0;
    for (int g0 = 0; g0 < p.groups; g0 += 64) {
        if (p.groups > 64) {  // else they are there
            rows = 0;
            if (g0 + lane < p.groups) {
                group_rows(p, g0 + lane, first, rows);
            }
            sum = inclusive((rows + bm - 1) / bm * nts);
        }
        const uint64_t past = __ballot(before + sum > tile);
        if (past != 0) {
            const int at = static_cast<int>(__builtin_ctzll(past));
            const int32_t mts = (rows + bm - 1) / bm;
            const int32_t tiles = __builtin_amdgcn_readlane(mts, at);
            const int32_t local = tile - before - (__builtin_amdgcn_readlane(sum, at) - tiles * nts);
            t = Tile{g0 + at, local % tiles, local / tiles, __builtin_amdgcn_readlane(first, at),
                     __builtin_amdgcn_readlane(rows, at)};
            return t.mt >= 0 && t.nt >= 0 && t.nt < nts;
        }
        before = min(before + __builtin_amdgcn_readlane(sum, 63), kMost);
    }
    return false;
}

// Floats from one share's sums to the next one's: 16-byte aligned.
__host__ __device__ inline int64_t plane(int64_t count) { return (count + 3) / 4 * 4; }

__host__ __device__ inline int32_t tiles_beside(const Fp8Product& q, int bm, int bn) {
    return static_cast<int32_t>((q.rows + bm - 1) / bm) * ((q.n + bn - 1) / bn);
}

// The row of a that row i of the groups reads.
__device__ inline uint32_t source_row(const Fp8Product& p, int32_t i) {
    const int32_t from = p.source == nullptr ? i : p.source[i];
    const uint32_t row = static_cast<uint32_t>(from) / static_cast<uint32_t>(p.source == nullptr ? 1 : p.divisor);
    if (from < 0 || row >= static_cast<uint64_t>(p.a_rows)) {
        report(p);
        return 0;
    }
    return row;
}

// The output row that row i is written to, -1 for none.
__device__ inline int64_t target_row(const Fp8Product& p, int32_t i) {
    const int32_t to = p.target == nullptr ? i : p.target[i];
    if (static_cast<uint32_t>(to) >= static_cast<uint64_t>(p.out_rows)) {
        report(p);
        return -1;
    }
    return to;
}

// Features n .. n + 3 of an output row: sixteen or eight bytes where rows allow
// it, rounded once.
__device__ inline void store4(const Fp8Product& p, int64_t row, int32_t n, floatx4 v) {
    const int64_t at = row * p.n + n;
    if (p.n % 4 == 0) {
        if (p.out_dtype == LM_DT_F32) {
            *reinterpret_cast<floatx4*>(static_cast<float*>(p.out) + at) = v;
        } else if (p.out_dtype == LM_DT_F16) {
            typedef _Float16 half4 __attribute__((ext_vector_type(4)));
            *reinterpret_cast<half4*>(static_cast<_Float16*>(p.out) + at) = __builtin_convertvector(v, half4);
        } else {
            typedef __bf16 bf4 __attribute__((ext_vector_type(4)));
            *reinterpret_cast<bf4*>(static_cast<__bf16*>(p.out) + at) = __builtin_convertvector(v, bf4);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (n + i < p.n) {
            if (p.out_dtype == LM_DT_F32) {
                static_cast<float*>(p.out)[at + i] = v[i];
            } else if (p.out_dtype == LM_DT_F16) {
                static_cast<_Float16*>(p.out)[at + i] = static_cast<_Float16>(v[i]);
            } else {
                static_cast<__bf16*>(p.out)[at + i] = static_cast<__bf16>(v[i]);
            }
        }
    }
}

// gate / (1 + exp(-gate)) * up.  The exponential is taken of gate / ln 2 in fp32 and
// is off by 2^-23 (2 + |gate|) of itself; what of that reaches the quotient, its
// share of 1 + exp(-gate), is at most 2^-16 (at -87, under which the quotient is
// subnormal and taken as 0) and far below the rounding to e4m3 (2^-4).
__device__ inline float swiglu(float gate, float up) {
    return gate * __builtin_amdgcn_rcpf(1.0f + __expf(-gate)) * up;
}

// ---- the kernel of large tiles ----
//
// A tile has BM rows and BN weight rows (SwiGLU: blocks of 16 gate rows and the
// 16 up rows of the same channels in turn). A stage is one scale block, 128
// bytes of every row, loaded straight to LDS STAGES - 1 stages ahead, with the
// rows' and the weights' scales of the block.
//
// What bounds it: many rows the matrix cores and the FMAs or conversions beside them,
// under whose load the clock falls (2048 x 5120 x 16384 160 us in turn with others,
// 2.14 PFLOP/s; fp32 sums, experts of 12288 rows, 104 and 189 us, 0.7 PFLOP/s of rows
// that count); few rows of many experts their weights (187 MB 31 us, 1731 MB 278 us:
// 6.0 and 6.2 TB/s). Larger tiles read less and wait longer: which is taken is decided
// by their costs below.
//
// LDS rows are 128 bytes: chunk c of row r lies at chunk position c ^ (r / 2).
// A 16-byte read takes sixteen lanes a clock over 64 banks (256 bytes, two
// rows); whether those are lanes 0 .. 15 or, as it seems, 0 .. 3, 12 .. 15 and
// 20 .. 27, they hold sixteen different rows, and land on different banks.
// (c ^ (r & 7) ^ (r >> 3 & 1), free of conflicts in the first order alone, had one
// a read: 1680 clocks of LDS a stage of 256 x 256 where this has 912.)
__device__ inline int chunk_swizzle(int r) { return (r >> 1) & 7; }

template <bool SWIGLU_, int BM_, int BN_, int WAVES_, int STAGES_>
struct Shape {
    static constexpr bool SWIGLU = SWIGLU_;
    static constexpr int BM = BM_, BN = BN_, WAVES = WAVES_, STAGES = STAGES_;
    static constexpr int CN = SWIGLU ? BN / 2 : BN;  // output features of a tile
    static constexpr int kABytes = BM * 128, kBBytes = BN * 128;
    static constexpr int kScales = (BM + 63) / 64;  // 64-lane loads of row scales
    static constexpr int kBlocks = (BN + kFp8Block - 1) / kFp8Block;  // weight scales
    static constexpr int kRowScales = kABytes + kBBytes, kWeightScales = kRowScales + kScales * 256;
    static constexpr int kStageBytes = kWeightScales + 256;
    static_assert(STAGES >= 2 && STAGES <= 4 && kScales < WAVES, "a scale load per wave");
    static_assert(!SWIGLU || CN == kFp8Block, "a SwiGLU tile is one output block wide");
    static_assert(kFp8Block % CN == 0 || CN % kFp8Block == 0, "tiles end where scale blocks do");
};

// What every wave of a tile needs.
template <class Z>
struct Stage {
    char* const (&bufs)[4];
    Tile t;
    int m0, n0;  // the tile's first row in its group, its first feature
    int lane, wave;
    int first, stages;  // the tile's share of the reduced axis, in scale blocks
};

// The products of a tile: WM x WN waves of MI x NJ blocks of 16 rows x 16 weight
// rows.
template <class Z, bool EXACT, int WM, int WN, int MI, int NJ>
struct Work {
    static constexpr bool SWIGLU = Z::SWIGLU;
    static constexpr int STAGES = Z::STAGES, BM = Z::BM;
    // 1 KB loads of a wave and stage; where the rows have fewer than there are
    // waves, two waves load the same
    static constexpr int AL = BM / 8 > Z::WAVES ? BM / 8 / Z::WAVES : 1, BL = Z::BN / 8 / Z::WAVES;
    static constexpr int L = AL + BL + 1;
    static_assert(WM * WN == Z::WAVES && 16 * WM * MI == BM && 16 * WN * NJ == Z::BN);
    static_assert((AL * 8 * Z::WAVES == BM || Z::WAVES * 8 % BM == 0) && BL * 8 * Z::WAVES == Z::BN,
                  "whole loads per wave");
    static_assert((STAGES - 1) * L < 64, "vmcnt");
    static_assert(SWIGLU ? NJ % 2 == 0 : (16 * NJ <= kFp8Block && kFp8Block % (16 * NJ) == 0),
                  "gate and up in one wave, one weight scale otherwise");

    __amdgpu_buffer_rsrc_t ra, rb, rs;  // rows, weights, the scales that this wave loads
    unsigned va[AL], vb[BL], vs;        // this lane's byte offsets in stage 0
    unsigned ta[AL], tb[BL];            // the same in the last block's stage
    int scales_at;                      // where the scales go in a stage
    int lane, wave, wm, wn;
    int blocks;          // scale blocks of the reduced axis
    int last_chunks;     // chunks of the last one that hold channels
    bool idle;           // none of this wave's rows is the group's: it loads for the others
    int fa, fb, fs, ws;  // this lane's row chunk, weight chunk, row scale and weight scale in a stage
    floatx4 acc[MI][NJ];

    __device__ __forceinline__ Work(const Fp8Product& p, const Stage<Z>& st) {
        const Tile& t = st.t;
        lane = st.lane;
        wave = st.wave;
        wm = wave / WN;
        wn = wave % WN;
        blocks = p.kb;
        last_chunks = (p.k - (p.kb - 1) * kFp8Block) / 16;
        idle = st.m0 + 16 * MI * wm >= t.rows;
        const int chunk = (lane & 15) * 128 + (((lane >> 4) ^ chunk_swizzle(lane & 15)) << 4);
        fa = 2048 * MI * wm + chunk;
        fb = Z::kABytes + 2048 * NJ * wn + chunk;
        fs = Z::kRowScales + 64 * MI * wm + 4 * (lane & 15);
        ws = Z::kWeightScales + (SWIGLU ? 0 : wn * 16 * NJ / kFp8Block * 4);
        constexpr int kParts = SWIGLU ? 2 : 1;
        const int64_t matrix = static_cast<int64_t>(p.n) * p.k, scales = static_cast<int64_t>(kParts) * p.nb * p.kb;
        ra = __builtin_amdgcn_make_buffer_rsrc((void*)p.a, 0, static_cast<int>(p.a_rows * p.k), kBufferWord3);
        rb = __builtin_amdgcn_make_buffer_rsrc((void*)(p.w + t.g * kParts * matrix), 0,
                                               static_cast<int>(kParts * matrix), kBufferWord3);
        // rows past the group's last repeat it, and are not stored
        const auto row_of = [&](int r) { return source_row(p, t.first + min(st.m0 + r, t.rows - 1)); };
#pragma unroll
        for (int q = 0; q < AL; ++q) {
            const int r = load_row(q);
            const int c = (lane & 7) ^ chunk_swizzle(r);
            const unsigned row = row_of(r) * static_cast<unsigned>(p.k);
            va[q] = row + 16 * c;
            ta[q] = c < last_chunks ? va[q] : row;
        }
#pragma unroll
        for (int q = 0; q < BL; ++q) {
            const int r = 8 * (Z::WAVES * q + wave) + (lane >> 3);
            const int c = (lane & 7) ^ chunk_swizzle(r);
            const int n = SWIGLU ? st.n0 + (r >> 5) * 16 + (r & 15) : st.n0 + r;
            const unsigned part = SWIGLU ? (r >> 4) & 1 : 0;
            const unsigned row = (part * static_cast<unsigned>(p.n) + min(n, p.n - 1)) * static_cast<unsigned>(p.k);
            vb[q] = row + 16 * c;
            tb[q] = c < last_chunks ? vb[q] : row;
        }
        // The first waves load 64 rows' scales each, a line of memory for every
        // row; the others the weights', one or two lines, all of them the same.
        if (wave < Z::kScales) {
            rs = __builtin_amdgcn_make_buffer_rsrc((void*)p.a_scale, 0, static_cast<int>(p.a_rows * p.kb * 4),
                                                   kBufferWord3);
            vs = row_of(min(64 * wave + lane, BM - 1)) * static_cast<unsigned>(p.kb) * 4u;
            scales_at = Z::kRowScales + wave * 256;
        } else {
            rs = __builtin_amdgcn_make_buffer_rsrc((void*)(p.w_scale + t.g * scales), 0, static_cast<int>(4 * scales),
                                                   kBufferWord3);
            const int block = SWIGLU ? (lane & 1) * p.nb + t.nt : min(st.n0 / kFp8Block + lane % Z::kBlocks, p.nb - 1);
            vs = static_cast<unsigned>(block) * static_cast<unsigned>(p.kb) * 4u;
            scales_at = Z::kWeightScales;
        }
#pragma unroll
        for (int i = 0; i < MI; ++i) {
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                acc[i][j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
            }
        }
    }

    // The row of which load q of the rows has this lane's chunk.
    __device__ __forceinline__ int load_row(int q) const { return 8 * ((Z::WAVES * q + wave) % (BM / 8)) + (lane >> 3); }
    // Load q of this wave's stage loads: rows, weights, then the scales.
    __device__ __forceinline__ void load1(int ks, char* buf, bool last, int q) {
        const unsigned at = static_cast<unsigned>(ks) * 128u;
        if (q < AL) {
            buffer_lds16(ra, buf + (Z::WAVES * q + wave) % (BM / 8) * 1024, last ? ta[q] : va[q], at);
        } else if (q < AL + BL) {
            const int w = q - AL;
            buffer_lds16(rb, buf + Z::kABytes + (Z::WAVES * w + wave) * 1024, last ? tb[w] : vb[w], at);
        } else {
            buffer_lds4(rs, buf + scales_at, vs, at / 32);
        }
    }
    // Sixteen rows' fragment: `at` is this lane's first chunk in the stage (one
    // addition from the array's start, so that the compiler sees which it is).
    __device__ __forceinline__ void read(const char* cur, int at, Operand<EXACT>& to) const {
        to.set(*reinterpret_cast<const uint4*>(cur + at), *reinterpret_cast<const uint4*>(cur + (at ^ 64)));
    }
    // Zeros past the reduced axis in the last stage, each lane into the chunks
    // that it loaded.
    __device__ __forceinline__ void clear_past(char* buf) {
#pragma unroll
        for (int q = 0; q < AL; ++q) {
            const int r = load_row(q);
            if (((lane & 7) ^ chunk_swizzle(r)) >= last_chunks) {
                *reinterpret_cast<uint4*>(buf + r * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
            }
        }
        __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
    }
    // No read of one stage's buffer may cross it, in either direction.
    __device__ __forceinline__ void barrier() {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    }
    // The products of a stage: row block i's on the matrix cores beside block
    // i - 1's FMAs and the reads of block i + 1. between(i) issues a part of the
    // next loads: a wave's run of them would wait for each to be accepted (2048 x
    // 5120 x 16384 in tiles of 256 x 256: 209 -> 201 us, of 128 x 256 265 -> 223).
    template <class Between>
    __device__ __forceinline__ void multiply(const char* cur, Between between) {
        const float w0 = *reinterpret_cast<const float*>(cur + ws);
        const float w1 = SWIGLU ? *reinterpret_cast<const float*>(cur + (ws + 4)) : w0;
        Operand<EXACT> b[NJ], a[2];
        floatx4 d[2][NJ];
        float scale[2], s0[2], s1[2];
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            read(cur, fb + 2048 * j, b[j]);
        }
        read(cur, fa, a[0]);
        scale[0] = *reinterpret_cast<const float*>(cur + fs);
#pragma unroll
        for (int i = 0; i <= MI; ++i) {
            const int now = i & 1, before = now ^ 1;
            if (i < MI) {
                if (i + 1 < MI) {
                    read(cur, fa + 2048 * (i + 1), a[before]);
                    scale[before] = *reinterpret_cast<const float*>(cur + (fs + 64 * (i + 1)));
                }
                s0[now] = scale[now] * w0;
                s1[now] = SWIGLU ? scale[now] * w1 : s0[now];
            }
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                if (i < MI) {
                    d[now][j] = block_sum(b[j], a[now]);
                }
                if (i > 0) {
                    take(acc[i - 1][j], d[before][j], SWIGLU && j % 2 == 1 ? s1[before] : s0[before]);
                }
            }
            if (i < MI) {
                between(i);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    // The nk stages from `first` on: stage ks lives in buffer ks % STAGES; its loads
    // are issued STAGES - 1 stages before, into the buffer that every wave has read
    // when it passes the barrier of stage ks - STAGES + 1. The first loop's stages
    // have later ones behind them that are not the last block's.
    __device__ __forceinline__ void run(char* const (&bufs)[4], int first, int nk) {
        const auto spread = [&](int ks, char* buf, bool last, int i) {
            // two stages: the next one's loads go out in the first half of this one, or
            // they are still on their way at its end (256 x 256: 1.55 -> 1.32 us a stage)
            constexpr int kSteps = STAGES == 2 ? (MI + 1) / 2 : MI;
#pragma unroll
            for (int q = i * L / kSteps; q < (i + 1) * L / kSteps && q < L; ++q) {
                load1(first + ks, buf, last, q);
            }
        };
#pragma unroll
        for (int d = 0; d < STAGES - 1; ++d) {
            if (d < nk) {
#pragma unroll
                for (int i = 0; i < MI; ++i) {
                    spread(d, bufs[d], first + d == blocks - 1, i);
                }
            }
        }
        int ks = 0;
        for (; ks + 2 * STAGES - 1 < nk; ks += STAGES) {
#pragma unroll
            for (int j = 0; j < STAGES; ++j) {
                LM_WAIT_VM((STAGES - 2) * L);
                barrier();
                const auto next = [&](int i) { spread(ks + j + STAGES - 1, bufs[(j + STAGES - 1) % STAGES], false, i); };
                if (idle) {
#pragma unroll
                    for (int i = 0; i < MI; ++i) {
                        next(i);
                    }
                } else {
                    multiply(bufs[j], next);
                }
            }
        }
        for (; ks < nk; ks += STAGES) {
#pragma unroll
            for (int j = 0; j < STAGES; ++j) {
                const int k = ks + j;
                if (k < nk) {
                    if (STAGES > 2 && k + STAGES - 2 < nk) {
                        LM_WAIT_VM((STAGES - 2) * L);
                    } else {
                        LM_WAIT_VM(0);
                    }
                    if (first + k == blocks - 1 && last_chunks < 8) {
                        clear_past(bufs[j]);
                    }
                    barrier();
                    if (k + STAGES - 1 < nk) {
#pragma unroll
                        for (int i = 0; i < MI; ++i) {
                            spread(k + STAGES - 1, bufs[(j + STAGES - 1) % STAGES], first + k + STAGES == blocks, i);
                        }
                    }
                    if (!idle) {
                        multiply(bufs[j], [](int) {});
                    }
                }
            }
        }
    }
    __device__ __forceinline__ void store(const Fp8Product& p, const Stage<Z>& st) {
        const int quad = 4 * (lane >> 4);
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            const int m = st.m0 + 16 * (wm * MI + i) + (lane & 15);
            const int64_t row = m < st.t.rows ? target_row(p, st.t.first + m) : -1;
            if (row >= 0) {
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    const int n = st.n0 + 16 * (wn * NJ + j) + quad;
                    if (n < p.n) {
                        store4(p, row, n, acc[i][j]);
                    }
                }
            }
        }
    }
    // SwiGLU, each row's largest magnitude over the tile's 128 channels from the
    // waves that share the row, and the codes through LDS to 16-byte stores. The
    // quotients are fp32's: the sums are off by more.
    __device__ __forceinline__ void store_swiglu(const Fp8Product& p, const Stage<Z>& st, char* codes, float* most_of) {
        constexpr int kPitch = kFp8Block + 16;  // a row's 16 lanes write to 16 different banks
        static_assert(BM * kPitch <= Z::kStageBytes);
        const int quad = 4 * (lane >> 4);
        const int rows = st.t.rows - st.m0;
        const int64_t first = st.t.first + st.m0;
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            float most = 0.0f;
#pragma unroll
            for (int j = 0; j < NJ; j += 2) {
                const bool in = st.n0 + 8 * (wn * NJ + j) + quad < p.n;  // p.n is a multiple of 16
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const float v = in ? swiglu(acc[i][j][u], acc[i][j + 1][u]) : 0.0f;
                    acc[i][j][u] = v;
                    most = __builtin_fmaxf(most, fp8_magnitude(v));
                }
            }
            most = __builtin_fmaxf(most, __shfl_xor(most, 16));
            most = __builtin_fmaxf(most, __shfl_xor(most, 32));
            if (lane < 16) {
                most_of[wn * BM + 16 * (wm * MI + i) + lane] = most;
            }
        }
        __syncthreads();  // `codes` is a stage's buffer: every wave's products are done
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            const int r = 16 * (wm * MI + i) + (lane & 15);
            float most = most_of[r];
#pragma unroll
            for (int w = 1; w < WN; ++w) {
                most = __builtin_fmaxf(most, most_of[w * BM + r]);
            }
            const float scale = fp8_scale(most), inverse = 1.0f / scale;
#pragma unroll
            for (int j = 0; j < NJ; j += 2) {
                float v[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    v[u] = fp8_finite_or_nan(acc[i][j][u]) * inverse;
                }
                *reinterpret_cast<uint32_t*>(codes + r * kPitch + 8 * (wn * NJ + j) + quad) =
                    fp8_pack4(v[0], v[1], v[2], v[3]);
            }
            if (wn == 0 && lane < 16 && r < rows) {
                p.q_scale[(first + r) * p.nb + st.t.nt] = scale;
            }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < BM * 8; i += 64 * Z::WAVES) {
            const int r = i / 8, n = st.n0 + 16 * (i % 8);
            if (r < rows && n < p.n) {
                *reinterpret_cast<uint4*>(p.q + (first + r) * p.n + n) =
                    *reinterpret_cast<const uint4*>(codes + r * kPitch + 16 * (i % 8));
            }
        }
    }
};

// BESIDE: the tiles of q, which has no offsets, are computed beside p's.
template <class Z, bool EXACT, int WM, int WN, int MI, int NJ, bool BESIDE>
__global__ __launch_bounds__(64 * WM * WN) __attribute__((amdgpu_waves_per_eu(2, 2))) void fp8_tile_kernel(Fp8Product p,
                                                                                                         Fp8Product q) {
    // one LDS array per stage: the compiler tracks the asynchronous writes by array
    __shared__ __attribute__((aligned(1024))) char s0[Z::kStageBytes], s1[Z::kStageBytes],
        s2[Z::STAGES > 2 ? Z::kStageBytes : 16], s3[Z::STAGES > 3 ? Z::kStageBytes : 16];
    __shared__ float most_of[Z::SWIGLU ? WN * Z::BM : 1];
    char* const bufs[4] = {s0, s1, s2, s3};
    Tile t;
    if (!find_tile(p, Z::BM, (p.n + Z::CN - 1) / Z::CN, t, BESIDE ? tiles_beside(q, Z::BM, Z::CN) : 0,
                   BESIDE ? static_cast<int32_t>(q.rows) : 0)) {
        return;
    }
    if (BESIDE && t.g < 0) {
        p = q;
        t.g = 0;
    }
    int first = 0, stages = p.kb;
    if (gridDim.y > 1) {  // a share of the reduced axis, into a plane of fp32 sums of its own
        const int per = (p.kb + gridDim.y - 1) / gridDim.y;
        first = blockIdx.y * per;
        stages = min(per, p.kb - first);
        p.out = static_cast<float*>(p.out) + blockIdx.y * plane(p.rows * p.n);
    }
    const Stage<Z> st{bufs, t, t.mt * Z::BM, t.nt * Z::CN, static_cast<int>(threadIdx.x & 63),
                      __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6)), first, stages};
    Work<Z, EXACT, WM, WN, MI, NJ> work(p, st);
    work.run(st.bufs, st.first, st.stages);
    if constexpr (Z::SWIGLU) {
        work.store_swiglu(p, st, s0, most_of);
    } else {
        work.store(p, st);
    }
}

// Tiles of bm rows and bn features that a launch has room for: a group of n rows
// takes ceil(n / bm) row tiles, at most one more than n / bm for each group that
// has any.
int64_t most_tiles(const Fp8Product& p, const Fp8Product* beside, int bm, int bn) {
    const int64_t mts = p.offsets == nullptr ? (p.rows + bm - 1) / bm : p.rows / bm + std::min<int64_t>(p.groups, p.rows);
    return mts * ((p.n + bn - 1) / bn) + (beside != nullptr ? tiles_beside(*beside, bm, bn) : 0);
}

template <bool SWIGLU, bool EXACT, int WM, int WN, int MI, int NJ, int STAGES>
hipError_t launch_tiles(const Fp8Product& p, const Fp8Product* beside, hipStream_t s, int shares = 1) {
    using Z = Shape<SWIGLU, 16 * WM * MI, 16 * WN * NJ, WM * WN, STAGES>;
    const int64_t tiles = most_tiles(p, beside, Z::BM, Z::CN);
    if (tiles > kFp8MaxTiles) {
        return hipErrorInvalidConfiguration;
    }
    const dim3 grid(static_cast<unsigned>(round_up(tiles, kXcds)), static_cast<unsigned>(shares)), block(64 * Z::WAVES);
    if constexpr (SWIGLU || !EXACT) {  // a layer's products
        if (beside != nullptr) {
            hipLaunchKernelGGL(HIP_KERNEL_NAME(fp8_tile_kernel<Z, EXACT, WM, WN, MI, NJ, true>), grid, block, 0, s, p, *beside);
            return hipGetLastError();
        }
    }
    hipLaunchKernelGGL(HIP_KERNEL_NAME(fp8_tile_kernel<Z, EXACT, WM, WN, MI, NJ, false>), grid, block, 0, s, p, p);
    return hipGetLastError();
}

// ---- the kernel of few rows ----
//
// Tiles of 16 rows at most by 16 features: the weights are read once, straight to
// registers, and the waves of a workgroup take turns at the scale blocks of the
// reduced axis; their sums are added up in LDS, wave by wave. What counts is the
// bytes in flight: U blocks of 2 KB a wave. One row by 10944 x 2048 (22 MB) 8.8 us,
// 5.4 in turn with others (4.2 TB/s), six experts of 2048 x 1408 (17 MB) 7.3 and 5.5;
// by themselves a round trip to memory and its waiting make up half of it.
//
// Scale blocks b0, b0 + step, ... (U of them, as far as there are any) of 16
// weight rows and the rows of a.
template <int U>
__device__ __forceinline__ void stream_blocks(const Fp8Product& p, int b0, int step, const uint8_t* a, const float* a_scale,
                                              bool live, const uint8_t* w, const float* w_scale, floatx4& acc) {
    const int lane = threadIdx.x & 63, chunks = p.k / 16;
    uint4 wv[U][2], av[U][2];
    float sa[U], sw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int b = min(b0 + u * step, p.kb - 1);  // past the last block: it again, which counts for nothing
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int c = 8 * b + 4 * h + (lane >> 4);
            wv[u][h] = load_stream16(w + (c < chunks ? 16 * c : 0));
            av[u][h] = make_uint4(0, 0, 0, 0);
            if (live && c < chunks) {
                av[u][h] = *reinterpret_cast<const uint4*>(a + 16 * c);
            }
        }
        sa[u] = live && b0 + u * step < p.kb ? a_scale[b] : 0.0f;
        sw[u] = w_scale[b];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        Operand<true> rows, weights;
        rows.set(av[u][0], av[u][1]);
        weights.set(wv[u][0], wv[u][1]);
        take(acc, block_sum(weights, rows), sa[u] * sw[u]);
    }
}

template <int WAVES, int U, bool BESIDE>
__global__ __launch_bounds__(64 * WAVES) void fp8_stream_kernel(Fp8Product p, Fp8Product q) {
    __shared__ floatx4 sums[WAVES][64];
    Tile t;
    if (!find_tile(p, 16, (p.n + 15) / 16, t, BESIDE ? tiles_beside(q, 16, 16) : 0,
                   BESIDE ? static_cast<int32_t>(q.rows) : 0)) {
        return;
    }
    if (BESIDE && t.g < 0) {
        p = q;
        t.g = 0;
    }
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    const int m = t.mt * 16 + (lane & 15), n0 = t.nt * 16;
    const bool live = m < t.rows;
    const int64_t row = live ? source_row(p, t.first + m) : 0;
    const uint8_t* const w = p.w + (static_cast<int64_t>(t.g) * p.n + min(n0 + (lane & 15), p.n - 1)) * p.k;
    const float* const w_scale = p.w_scale + (static_cast<int64_t>(t.g) * p.nb + n0 / kFp8Block) * p.kb;
    floatx4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int b0 = wave; b0 < p.kb; b0 += WAVES * U) {
        stream_blocks<U>(p, b0, WAVES, p.a + row * p.k, p.a_scale + row * p.kb, live, w, w_scale, acc);
    }
    sums[wave][lane] = acc;
    __syncthreads();
    const int n = n0 + 4 * (lane >> 4);
    if (wave == 0 && live && n < p.n) {
#pragma unroll
        for (int i = 1; i < WAVES; ++i) {
            acc += sums[i][lane];
        }
        const int64_t to = target_row(p, t.first + m);
        if (to >= 0) {
            store4(p, to, n, acc);
        }
    }
}

// Rows and features of a tile of the kernel of few rows.
constexpr int kStreamTile = 16;

template <int WAVES, int U>
hipError_t launch_stream(const Fp8Product& p, const Fp8Product* beside, hipStream_t s) {
    const int64_t tiles = most_tiles(p, beside, kStreamTile, kStreamTile);
    const dim3 grid(static_cast<unsigned>(round_up(tiles, kXcds))), block(64 * WAVES);
    if (beside != nullptr) {
        hipLaunchKernelGGL(HIP_KERNEL_NAME(fp8_stream_kernel<WAVES, U, true>), grid, block, 0, s, p, *beside);
    } else {
        hipLaunchKernelGGL(HIP_KERNEL_NAME(fp8_stream_kernel<WAVES, U, false>), grid, block, 0, s, p, p);
    }
    return hipGetLastError();
}

// out = the shares' sums, added up in order.
__global__ __launch_bounds__(256) void fp8_join_kernel(Fp8Product p, const float* __restrict__ sums, int64_t count,
                                                       int32_t shares) {
    const int64_t at = 4 * (blockIdx.x * int64_t{256} + threadIdx.x);
    if (at >= count) {
        return;
    }
    // rows follow each other without a gap: a row of all values, cut in fours
    p.n = static_cast<int32_t>(min(count - at, int64_t{4}));
    constexpr int kAtOnce = 4;  // loads in flight
    floatx4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int i = 0; i < shares; i += kAtOnce) {
        floatx4 part[kAtOnce];
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) {
            part[j] = *reinterpret_cast<const floatx4*>(sums + min(i + j, shares - 1) * plane(count) + at);
        }
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) {
            v += i + j < shares ? part[j] : floatx4{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }
    p.out = static_cast<char*>(p.out) + at * (p.out_dtype == LM_DT_F32 ? 4 : 2);
    store4(p, 0, 0, v);
}

// ---- which kernel ----

// What a tile costs, in microseconds: a stage where at most half the places of
// workgroups are taken and where all are (measured with 1408 to 16384 reduced
// channels), a stage with weights for each group, and what is no stage's (finding
// the tile, its first loads, its outputs). A group's few row tiles wait together
// for weights from memory that no tile has read before, so that the larger tile
// gains there: fitted to the experts of layers with 64 x 1408 x 2048 and 160 x 1536
// x 5120 at 32 to 4096 tokens (gate and up of 1024 tokens by the latter: 648 us by
// two 32 x 256 tiles a CU, which the other figures take, 548 by 128 x 256; at 256
// tokens 483 and 519). Up to 128 x 128 two workgroups share a CU.
struct TileCost {
    int bm, bn, places;
    float solo, full, grouped, fixed;
};
constexpr TileCost kFp8Tiles[] = {{32, 128, 512, 0.33f, 0.62f, 0.90f, 1.5f},
                                  {64, 128, 512, 0.38f, 0.85f, 1.25f, 3.0f},
                                  {128, 128, 512, 0.71f, 1.05f, 1.80f, 5.0f},
                                  {128, 256, 256, 0.79f, 1.02f, 1.70f, 7.0f},
                                  {256, 256, 256, 1.32f, 1.72f, 2.15f, 11.0f}};
constexpr TileCost kExactTiles[] = {{32, 128, 512, 0.41f, 0.69f, 0.90f, 1.5f},
                                    {64, 128, 512, 0.59f, 1.15f, 1.25f, 3.0f},
                                    {128, 128, 512, 0.90f, 1.80f, 1.85f, 5.0f},
                                    {128, 256, 256, 1.44f, 1.73f, 1.75f, 7.0f}};
constexpr TileCost kSwigluTiles[] = {{32, 128, 256, 0.62f, 0.69f, 1.10f, 3.0f},
                                     {32, 128, 512, 0.87f, 1.22f, 1.85f, 3.0f},
                                     {64, 128, 256, 0.94f, 1.11f, 1.60f, 4.0f},
                                     {128, 128, 256, 1.45f, 1.80f, 1.80f, 6.0f}};
// SwiGLU on the FP8 matrix cores: the small tiles wait for their weights, and
// keep fp32 sums.
constexpr TileCost kSwigluFp8Tiles[] = {{32, 128, 256, 0.62f, 0.69f, 1.10f, 3.0f},
                                        {32, 128, 512, 0.87f, 1.22f, 1.85f, 3.0f},
                                        {64, 128, 256, 0.94f, 1.11f, 1.60f, 4.0f},
                                        {128, 128, 256, 0.80f, 1.05f, 1.40f, 7.0f},
                                        {256, 128, 256, 1.35f, 1.75f, 2.10f, 9.0f}};

// Groups that have rows, at most.
int64_t active_groups(const Fp8Product& p) { return p.offsets == nullptr ? 1 : std::min<int64_t>(p.groups, p.rows); }

// About how many row tiles there are: the host does not know the groups' sizes,
// and takes the last tile of each for half full.
double row_tiles(const Fp8Product& p, int bm) {
    if (p.offsets == nullptr) {
        return static_cast<double>((p.rows + bm - 1) / bm);
    }
    const double groups = static_cast<double>(active_groups(p));
    return std::max(groups, static_cast<double>(p.rows) / bm + 0.5 * groups);
}

// The time of all tiles: rounds in which all places are taken, and one of the rest.
// Where two workgroups share a CU, one more tile than CUs makes some CUs run two (128
// stages in 258 tiles of 64 x 128, fp32 sums, 120 us; 79 in 240); one to a CU, they
// share the memory and the clock alone. (700 rows by 10944 x 16384 in 258 tiles of 128
// x 256, a round and two tiles, 399 us; in 946 of 64 x 128 280.) Of groups the number
// of tiles is a guess: half a round more.
double tile_time(const TileCost& c, double tiles, int64_t stages, bool grouped) {
    const double n = static_cast<double>(stages);
    if (grouped) {
        const double per = n * (2.0 * tiles <= c.places ? c.solo : c.grouped) + c.fixed;
        return tiles <= c.places ? per : per * (tiles / c.places + 0.5);
    }
    const double rounds = std::floor(tiles / c.places), rest = tiles / c.places - rounds;
    const double past = 2.0 * rest - 1.0;
    const double stage = past <= 0.0       ? c.solo
                         : c.places > 256 ? std::max<double>(c.solo, (0.8 + 0.2 * past) * c.full)
                                          : c.solo + past * (c.full - c.solo);
    return rounds * (n * c.full + c.fixed) + (rest > 0.0 ? n * stage + c.fixed : 0.0);
}

// Where tiles leave places empty and the reduced axis is long, several
// workgroups share a tile's reduced axis, and a second launch joins their sums:
// that costs 5 us and their way through memory (6 TB/s). 80 rows by 16384 channels
// and 10944 features, fp32: 69 us in two shares, 60 in four; 40 by 10944 and 2048:
// 13.4 in four, 10.7 in eight.
struct TileChoice {
    int tile = 0;
    int shares = 1;
};
template <size_t N>
TileChoice choose_tile(const Fp8Product& p, const Fp8Product* beside, const TileCost (&tiles)[N], bool split) {
    constexpr int kShares[] = {1, 2, 3, 4, 6, 8, 12};
    TileChoice best{static_cast<int>(N) - 1, 1};
    double least = 1e30;
    for (size_t i = 0; i < N; ++i) {
        const TileCost& c = tiles[i];
        if (most_tiles(p, beside, c.bm, c.bn) > kFp8MaxTiles) {
            continue;  // a launch of larger ones may have room
        }
        double count = row_tiles(p, c.bm) * static_cast<double>((p.n + c.bn - 1) / c.bn);
        if (beside != nullptr) {  // by their stages
            count += static_cast<double>(tiles_beside(*beside, c.bm, c.bn)) * beside->kb / p.kb;
        }
        for (const int shares : kShares) {
            const int64_t stages = (p.kb + shares - 1) / shares;
            double t = tile_time(c, count * shares, stages, p.offsets != nullptr);
            if (shares > 1) {
                const int64_t sums = plane(p.rows * p.n) * shares;
                if (!split || stages < 4 || count * shares > c.places || 4 * sums > kFp8WorkspaceBytes) {
                    break;
                }
                t += 5.0 + 4.0 * static_cast<double>(2 * sums + p.rows * p.n) / 6e6;
            }
            if (t < least) {
                least = t;
                best = TileChoice{static_cast<int>(i), shares};
            }
        }
    }
    // every share has a part of the reduced axis
    const int per = (p.kb + best.shares - 1) / best.shares;
    best.shares = (p.kb + per - 1) / per;
    return best;
}

template <bool EXACT>
hipError_t launch_gemm_tile(const Fp8Product& p, const Fp8Product* beside, const Fp8Plan& c, hipStream_t s) {
    switch (c.tile) {
        case 0:
            return launch_tiles<false, EXACT, 1, 4, 2, 2, 3>(p, beside, s, c.shares);
        case 1:
            return launch_tiles<false, EXACT, 1, 4, 4, 2, 3>(p, beside, s, c.shares);
        case 2:
            return launch_tiles<false, EXACT, 2, 2, 4, 4, 2>(p, beside, s, c.shares);
        case 4:
            if constexpr (!EXACT) {
                return launch_tiles<false, false, 2, 4, 8, 4, 2>(p, beside, s, c.shares);
            }
            [[fallthrough]];
        default:
            return launch_tiles<false, EXACT, 2, 4, 4, 4, 3>(p, beside, s, c.shares);
    }
}

// Whether the kernel of few rows is the faster: what its workgroups read, each
// the weights of its 16 features and its rows, stays under 28 MB. A call in turn
// with others' and by itself, and the same in tiles: four rows by 10944 channels
// and 2048 features (27 MB) 5.7 and 10.6 us, 9.1 and 11.3; by 2048 and 10944 5.3
// and 6.9, 5.4 and 7.8; twelve (37 MB) 6.1 and 8.6, 5.3 and 7.8; six experts of
// 2048 features (18 MB) 5.6 and 5.9, 5.5 and 7.3, of 5120 (48 MB) 13 and 17, 6.3
// and 12.
int64_t stream_bytes(const Fp8Product& p) {
    const int64_t groups = active_groups(p), rows = std::min<int64_t>(16, (p.rows + groups - 1) / groups);
    const int64_t tiles = most_tiles(p, nullptr, kStreamTile, kStreamTile);
    return tiles <= 4096 ? tiles * p.kb * (16 + rows) * kFp8Block : INT32_MAX;
}
bool streams(const Fp8Product& p, const Fp8Product* beside) {
    return stream_bytes(p) + (beside != nullptr ? stream_bytes(*beside) : 0) <= (28 << 20);
}

}  // namespace

Fp8Plan plan_fp8_gemm(const Fp8Product& p, const Fp8Product* beside) {
    if (streams(p, beside)) {
        return Fp8Plan{-1, kStreamTile, kStreamTile, 1, true, most_tiles(p, beside, kStreamTile, kStreamTile)};
    }
    const bool exact = p.exact != 0, split = p.offsets == nullptr;
    const TileChoice c = exact ? choose_tile(p, beside, kExactTiles, split) : choose_tile(p, beside, kFp8Tiles, split);
    const TileCost& t = exact ? kExactTiles[c.tile] : kFp8Tiles[c.tile];
    return Fp8Plan{c.tile, t.bm, t.bn, c.shares, exact, most_tiles(p, beside, t.bm, t.bn)};
}

Fp8Plan plan_fp8_swiglu(const Fp8Product& p, const Fp8Product* beside) {
    const bool exact = p.exact != 0;
    const TileChoice c = exact ? choose_tile(p, beside, kSwigluTiles, false) : choose_tile(p, beside, kSwigluFp8Tiles, false);
    const TileCost& t = exact ? kSwigluTiles[c.tile] : kSwigluFp8Tiles[c.tile];
    return Fp8Plan{c.tile, t.bm, t.bn, 1, exact || c.tile < 3, most_tiles(p, beside, t.bm, t.bn)};
}

hipError_t launch_fp8_gemm(const Fp8Product& p, void* workspace, hipStream_t s, const Fp8Product* beside) {
    const Fp8Plan plan = plan_fp8_gemm(p, beside);
    if (plan.tile < 0) {
        // all of a wave's loads in flight at once where the axis is short, many
        // waves where it is long (10944 channels: 9.5 us, 11 with four waves)
        return p.kb <= 12   ? launch_stream<4, 3>(p, beside, s)
               : p.kb <= 16 ? launch_stream<4, 4>(p, beside, s)
               : p.kb <= 40 ? launch_stream<8, 2>(p, beside, s)
                            : launch_stream<16, 2>(p, beside, s);
    }
    Fp8Product q = p;
    if (plan.shares > 1) {
        q.out = workspace;
        q.out_dtype = LM_DT_F32;
    }
    const hipError_t e = plan.exact ? launch_gemm_tile<true>(q, beside, plan, s) : launch_gemm_tile<false>(q, beside, plan, s);
    if (e != hipSuccess || plan.shares == 1) {
        return e;
    }
    const int64_t count = p.rows * p.n;
    hipLaunchKernelGGL(fp8_join_kernel, dim3(static_cast<unsigned>((count + 1023) / 1024)), dim3(256), 0, s, p,
                       static_cast<const float*>(workspace), count, plan.shares);
    return hipGetLastError();
}

hipError_t launch_fp8_swiglu(const Fp8Product& p, hipStream_t s, const Fp8Product* beside) {
    const Fp8Plan plan = plan_fp8_swiglu(p, beside);
    switch (plan.tile) {
        case 0:
            return launch_tiles<true, true, 1, 8, 2, 2, 3>(p, beside, s);
        case 1:
            return launch_tiles<true, true, 1, 4, 2, 4, 2>(p, beside, s);
        case 2:
            return launch_tiles<true, true, 1, 8, 4, 2, 3>(p, beside, s);
        case 3:
            return plan.exact ? launch_tiles<true, true, 2, 4, 4, 4, 3>(p, beside, s)
                              : launch_tiles<true, false, 2, 4, 4, 4, 3>(p, beside, s);
        default:
            return launch_tiles<true, false, 2, 4, 8, 4, 2>(p, beside, s);
    }
}

}  // namespace lm
