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
// follow each other, so that their weights are read from one L2.
__device__ inline bool find_tile(const Fp8Product& p, int bm, int nts, Tile& t) {
    const int lane = threadIdx.x & 63;
    auto share = [&](int32_t total) {
        const int32_t xcd = blockIdx.x % kXcds, idx = blockIdx.x / kXcds;
        const int32_t per = total / kXcds, extra = total % kXcds;
        return idx < per + (xcd < extra ? 1 : 0) ? xcd * per + min(xcd, extra) + idx : -1;
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
        return false;
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

// gate / (1 + exp(-gate)) * up; the hardware's exponential and reciprocal are
// off by a few 2^-24, far below the rounding to e4m3 (2^-4).
__device__ inline float swiglu(float gate, float up) {
    return gate * __builtin_amdgcn_rcpf(1.0f + __expf(-gate)) * up;
}

// ---- the kernel of large tiles ----
//
// WM x WN waves, each MI x NJ blocks of 16 rows x 16 features, so a tile has
// 16 WM MI rows and 16 WN NJ weight rows (SwiGLU: half of each wave's are gate
// rows and half the up rows of the same channels). A stage is one scale block,
// 128 bytes of every row, loaded straight to LDS STAGES - 1 stages ahead, with
// the rows' and the weights' scales of the block.
//
// LDS rows are 128 bytes: chunk c of row r lies at chunk position c ^ f(r),
// f(r) = (r & 7) ^ (r >> 3 & 1), which puts any eight rows at eight positions
// (32 banks) and any sixteen at sixteen places of two rows (64 banks).
__device__ inline int chunk_swizzle(int r) { return (r & 7) ^ ((r >> 3) & 1); }

template <bool SWIGLU, int WM, int WN, int MI, int NJ, int STAGES>
struct Shape {
    static constexpr int WAVES = WM * WN;
    static constexpr int BM = 16 * WM * MI, BN = 16 * WN * NJ;
    static constexpr int CN = SWIGLU ? BN / 2 : BN;  // output features of a tile
    static constexpr int kABytes = BM * 128, kBBytes = BN * 128;
    static constexpr int kScales = (BM + 63) / 64;  // 64-lane loads of row scales
    static constexpr int kBlocks = (BN + kFp8Block - 1) / kFp8Block;  // weight scales
    static constexpr int kRowScales = kABytes + kBBytes, kWeightScales = kRowScales + kScales * 256;
    static constexpr int kStageBytes = kWeightScales + 256;
    static constexpr int AL = BM / 8 / WAVES, BL = BN / 8 / WAVES;
    static constexpr int L = AL + BL + 2;
    static_assert(AL * 8 * WAVES == BM && BL * 8 * WAVES == BN, "whole 1 KB loads per wave");
    static_assert(kScales <= WAVES && (STAGES - 1) * L < 64, "a scale load per wave, vmcnt");
    static_assert(!SWIGLU || CN == kFp8Block, "a SwiGLU tile is one output block wide");
    static_assert(16 * NJ <= (SWIGLU ? 2 : 1) * kFp8Block && CN % (SWIGLU ? 1 : 16 * NJ) == 0, "one weight scale per wave and part");
};

template <bool SWIGLU, bool EXACT, int WM, int WN, int MI, int NJ, int STAGES>
struct Pipeline {
    using Z = Shape<SWIGLU, WM, WN, MI, NJ, STAGES>;
    __amdgpu_buffer_rsrc_t ra, rs, rb, rw;  // rows, their scales, weights, their scales
    unsigned va[Z::AL], vb[Z::BL], vs, vw;  // this lane's byte offsets in stage 0
    unsigned ta[Z::AL], tb[Z::BL];      // the same in the last stage
    int lane, wave, wm, wn, nk;
    int live;                           // this wave's 16-row blocks that hold rows
    int last_chunks;                    // chunks of the last stage that hold channels
    int fa, fb, fs, ws;                 // this lane's row chunk, weight chunk, row scale and weight scale in a stage
    floatx4 acc[MI][NJ];

    __device__ void load(int ks, char* buf, bool last) {
#pragma unroll
        for (int q = 0; q < Z::AL; ++q) {
            buffer_lds16(ra, buf + (Z::WAVES * q + wave) * 1024, last ? ta[q] : va[q], static_cast<unsigned>(ks) * 128u);
        }
#pragma unroll
        for (int q = 0; q < Z::BL; ++q) {
            buffer_lds16(rb, buf + Z::kABytes + (Z::WAVES * q + wave) * 1024, last ? tb[q] : vb[q],
                         static_cast<unsigned>(ks) * 128u);
        }
        buffer_lds4(rs, buf + Z::kRowScales + (wave % Z::kScales) * 256, vs, static_cast<unsigned>(ks) * 4u);
        buffer_lds4(rw, buf + Z::kWeightScales, vw, static_cast<unsigned>(ks) * 4u);
    }
    // Sixteen rows' fragment: `at` is this lane's first chunk in the stage (one
    // addition from the array's start, so that the compiler sees which it is).
    __device__ void read(const char* cur, int at, Operand<EXACT>& to) const {
        to.set(*reinterpret_cast<const uint4*>(cur + at), *reinterpret_cast<const uint4*>(cur + (at ^ 64)));
    }
    // Zeros past the reduced axis in the last stage, each lane into the chunks
    // that it loaded.
    __device__ void clear_past(char* buf) {
#pragma unroll
        for (int q = 0; q < Z::AL; ++q) {
            const int r = 8 * (Z::WAVES * q + wave) + (lane >> 3);
            if (((lane & 7) ^ chunk_swizzle(r)) >= last_chunks) {
                *reinterpret_cast<uint4*>(buf + r * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
            }
        }
        __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
    }
    // No read of one stage's buffer may cross it, in either direction.
    __device__ void barrier() {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    }
    // The products of a stage. FULL: all of the wave's row blocks hold rows.
    template <bool FULL>
    __device__ void multiply(const char* cur) {
        const float w0 = *reinterpret_cast<const float*>(cur + ws);
        const float w1 = SWIGLU ? *reinterpret_cast<const float*>(cur + (ws + 4)) : w0;
        Operand<EXACT> b[NJ];
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            read(cur, fb + 2048 * j, b[j]);
        }
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            if (FULL || i < live) {
                Operand<EXACT> a;
                read(cur, fa + 2048 * i, a);
                const float scale = *reinterpret_cast<const float*>(cur + (fs + 64 * i));
                const float s0 = scale * w0, s1 = SWIGLU ? scale * w1 : s0;
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    const floatx4 d = block_sum(b[j], a);
                    const float s = SWIGLU && j >= NJ / 2 ? s1 : s0;
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        acc[i][j][u] = __builtin_fmaf(d[u], s, acc[i][j][u]);
                    }
                }
            }
        }
    }
    // All nk stages: stage ks lives in buffer ks % STAGES; its loads are issued
    // STAGES - 1 stages before, into the buffer that every wave has read when it
    // passes the barrier of stage ks - STAGES + 1. The first loop's stages have
    // later ones behind them that are not the last.
    template <bool FULL>
    __device__ void run(char* const (&bufs)[4]) {
#pragma unroll
        for (int d = 0; d < STAGES - 1; ++d) {
            if (d < nk) {
                load(d, bufs[d], d == nk - 1);
            }
        }
        int ks = 0;
        for (; ks + 2 * STAGES - 1 < nk; ks += STAGES) {
#pragma unroll
            for (int j = 0; j < STAGES; ++j) {
                LM_WAIT_VM((STAGES - 2) * Z::L);
                barrier();
                load(ks + j + STAGES - 1, bufs[(j + STAGES - 1) % STAGES], false);
                multiply<FULL>(bufs[j]);
            }
        }
        for (; ks < nk; ks += STAGES) {
#pragma unroll
            for (int j = 0; j < STAGES; ++j) {
                const int k = ks + j;
                if (k < nk) {
                    if (STAGES > 2 && k + STAGES - 2 < nk) {
                        LM_WAIT_VM((STAGES - 2) * Z::L);
                    } else {
                        LM_WAIT_VM(0);
                    }
                    if (k == nk - 1 && last_chunks < 8) {
                        clear_past(bufs[j]);
                    }
                    barrier();
                    if (k + STAGES - 1 < nk) {
                        load(k + STAGES - 1, bufs[(j + STAGES - 1) % STAGES], k + STAGES == nk);
                    }
                    multiply<FULL>(bufs[j]);
                }
            }
        }
    }
};

template <bool SWIGLU, bool EXACT, int WM, int WN, int MI, int NJ, int STAGES, int PER_EU>
__global__ __launch_bounds__(64 * WM * WN) __attribute__((amdgpu_waves_per_eu(PER_EU, PER_EU))) void fp8_tile_kernel(
    Fp8Product p) {
    using Z = Shape<SWIGLU, WM, WN, MI, NJ, STAGES>;
    static_assert(STAGES >= 2 && STAGES <= 4);
    // one LDS array per stage: the compiler tracks the asynchronous writes by array
    __shared__ __attribute__((aligned(1024))) char s0[Z::kStageBytes], s1[Z::kStageBytes],
        s2[STAGES > 2 ? Z::kStageBytes : 16], s3[STAGES > 3 ? Z::kStageBytes : 16];
    char* const bufs[4] = {s0, s1, s2, s3};
    Tile t;
    if (!find_tile(p, Z::BM, (p.n + Z::CN - 1) / Z::CN, t)) {
        return;
    }
    Pipeline<SWIGLU, EXACT, WM, WN, MI, NJ, STAGES> pipe;
    const int lane = pipe.lane = threadIdx.x & 63;
    const int wave = pipe.wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    const int wm = pipe.wm = wave / WN;
    const int wn = pipe.wn = wave % WN;
    pipe.nk = p.kb;
    pipe.last_chunks = (p.k - (p.kb - 1) * kFp8Block) / 16;
    const int m0 = t.mt * Z::BM, n0 = t.nt * Z::CN;
    const int chunk = (lane & 15) * 128 + (((lane >> 4) ^ chunk_swizzle(lane & 15)) << 4);
    pipe.fa = 2048 * MI * wm + chunk;
    pipe.fb = Z::kABytes + 2048 * NJ * wn + chunk;
    pipe.fs = Z::kRowScales + 64 * MI * wm + 4 * (lane & 15);
    pipe.ws = Z::kWeightScales + (SWIGLU ? 0 : wn * 16 * NJ / kFp8Block * 4);
    pipe.live = (t.rows - m0 - 16 * MI * wm + 15) / 16;
    constexpr int kParts = SWIGLU ? 2 : 1;
    const int64_t matrix = static_cast<int64_t>(p.n) * p.k;
    pipe.ra = __builtin_amdgcn_make_buffer_rsrc((void*)p.a, 0, static_cast<int>(p.a_rows * p.k), kBufferWord3);
    pipe.rs = __builtin_amdgcn_make_buffer_rsrc((void*)p.a_scale, 0, static_cast<int>(p.a_rows * p.kb * 4), kBufferWord3);
    pipe.rb = __builtin_amdgcn_make_buffer_rsrc((void*)(p.w + t.g * kParts * matrix), 0,
                                                static_cast<int>(kParts * matrix), kBufferWord3);
    const int64_t blocks = static_cast<int64_t>(kParts) * p.nb * p.kb;
    pipe.rw = __builtin_amdgcn_make_buffer_rsrc((void*)(p.w_scale + t.g * blocks), 0, static_cast<int>(4 * blocks),
                                                kBufferWord3);
    // rows past the group's last repeat it, and are not stored
    const auto row_of = [&](int r) { return source_row(p, t.first + min(m0 + r, t.rows - 1)); };
#pragma unroll
    for (int q = 0; q < Z::AL; ++q) {
        const int r = 8 * (Z::WAVES * q + wave) + (lane >> 3);
        const int c = (lane & 7) ^ chunk_swizzle(r);
        const unsigned row = row_of(r) * static_cast<unsigned>(p.k);
        pipe.va[q] = row + 16 * c;
        pipe.ta[q] = c < pipe.last_chunks ? pipe.va[q] : row;
    }
    pipe.vs = row_of(min(64 * (wave % Z::kScales) + lane, Z::BM - 1)) * static_cast<unsigned>(p.kb) * 4u;
#pragma unroll
    for (int q = 0; q < Z::BL; ++q) {
        const int r = 8 * (Z::WAVES * q + wave) + (lane >> 3);
        const int c = (lane & 7) ^ chunk_swizzle(r);
        int n = n0 + r;
        unsigned part = 0;
        if (SWIGLU) {  // wave r / (16 NJ): its gate rows, then the up rows of the same channels
            const int in = r % (16 * NJ);
            part = in >= 8 * NJ ? 1u : 0u;
            n = n0 + r / (16 * NJ) * 8 * NJ + in % (8 * NJ);
        }
        const unsigned row = (part * static_cast<unsigned>(p.n) + min(n, p.n - 1)) * static_cast<unsigned>(p.k);
        pipe.vb[q] = row + 16 * c;
        pipe.tb[q] = c < pipe.last_chunks ? pipe.vb[q] : row;
    }
    const int block = SWIGLU ? (lane & 1) * p.nb + t.nt : min(n0 / kFp8Block + lane % Z::kBlocks, p.nb - 1);
    pipe.vw = static_cast<unsigned>(block) * static_cast<unsigned>(p.kb) * 4u;
#pragma unroll
    for (int i = 0; i < MI; ++i) {
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            pipe.acc[i][j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }
    if (pipe.live >= MI) {
        pipe.template run<true>(bufs);
    } else {
        pipe.template run<false>(bufs);
    }

    const int quad = 4 * (lane >> 4);
    if constexpr (!SWIGLU) {
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            const int m = m0 + 16 * (wm * MI + i) + (lane & 15);
            const int64_t row = m < t.rows ? target_row(p, t.first + m) : -1;
            if (row >= 0) {
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    const int n = n0 + 16 * (wn * NJ + j) + quad;
                    if (n < p.n) {
                        store4(p, row, n, pipe.acc[i][j]);
                    }
                }
            }
        }
    } else {
        // Each row's largest magnitude over the tile's 128 channels, from the
        // waves that share the row, then the codes through LDS to 16-byte stores.
        constexpr int kPitch = kFp8Block + 16;  // a row's 16 lanes write to 16 different banks
        static_assert(Z::BM * kPitch <= Z::kStageBytes);
        __shared__ float most_of[WN][Z::BM];
        char* const codes = s0;  // written once every wave has passed a barrier after its products
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            float most = 0.0f;
#pragma unroll
            for (int j = 0; j < NJ / 2; ++j) {
                const bool in = n0 + 8 * NJ * wn + 16 * j + quad < p.n;  // p.n is a multiple of 16
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const float v = in ? swiglu(pipe.acc[i][j][u], pipe.acc[i][j + NJ / 2][u]) : 0.0f;
                    pipe.acc[i][j][u] = v;
                    most = __builtin_fmaxf(most, fp8_magnitude(v));
                }
            }
            most = __builtin_fmaxf(most, __shfl_xor(most, 16));
            most = __builtin_fmaxf(most, __shfl_xor(most, 32));
            if (lane < 16) {
                most_of[wn][16 * (wm * MI + i) + lane] = most;
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            const int r = 16 * (wm * MI + i) + (lane & 15);
            float most = most_of[0][r];
#pragma unroll
            for (int w = 1; w < WN; ++w) {
                most = __builtin_fmaxf(most, most_of[w][r]);
            }
            const float scale = fp8_scale(most), inverse = 1.0f / scale;
#pragma unroll
            for (int j = 0; j < NJ / 2; ++j) {
                float v[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    v[u] = fp8_finite_or_nan(pipe.acc[i][j][u]) * inverse;
                }
                *reinterpret_cast<uint32_t*>(codes + r * kPitch + 8 * NJ * wn + 16 * j + quad) =
                    fp8_pack4(v[0], v[1], v[2], v[3]);
            }
            if (wn == 0 && lane < 16 && m0 + r < t.rows) {
                p.q_scale[static_cast<int64_t>(t.first + m0 + r) * p.nb + t.nt] = scale;
            }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < Z::BM * 8; i += 64 * Z::WAVES) {
            const int r = i / 8, n = n0 + 16 * (i % 8);
            if (m0 + r < t.rows && n < p.n) {
                *reinterpret_cast<uint4*>(p.q + static_cast<int64_t>(t.first + m0 + r) * p.n + n) =
                    *reinterpret_cast<const uint4*>(codes + r * kPitch + 16 * (i % 8));
            }
        }
    }
}

template <bool SWIGLU, bool EXACT, int WM, int WN, int MI, int NJ, int STAGES, int PER_EU>
hipError_t launch_tiles(const Fp8Product& p, hipStream_t s) {
    using Z = Shape<SWIGLU, WM, WN, MI, NJ, STAGES>;
    // a group of n rows takes ceil(n / BM) row tiles: at most one more than
    // n / BM for each group that has any
    const int64_t mts = p.offsets == nullptr ? (p.rows + Z::BM - 1) / Z::BM
                                             : p.rows / Z::BM + std::min<int64_t>(p.groups, p.rows);
    const int64_t tiles = mts * ((p.n + Z::CN - 1) / Z::CN);
    if (tiles > (1 << 22)) {
        return hipErrorInvalidValue;
    }
    hipLaunchKernelGGL(HIP_KERNEL_NAME(fp8_tile_kernel<SWIGLU, EXACT, WM, WN, MI, NJ, STAGES, PER_EU>),
                       dim3(static_cast<unsigned>(round_up(tiles, kXcds))), dim3(64 * Z::WAVES), 0, s, p);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_fp8_gemm(const Fp8Product& p, hipStream_t s) {
    return p.out_dtype == LM_DT_F32 ? launch_tiles<false, true, 1, 8, 4, 2, 2, 2>(p, s)
                                    : launch_tiles<false, false, 1, 8, 4, 2, 2, 2>(p, s);
}

hipError_t launch_fp8_swiglu(const Fp8Product& p, hipStream_t s) {
    return launch_tiles<true, true, 1, 8, 4, 2, 2, 2>(p, s);
}

}  // namespace lm
