// What the block-scaled products share (gfx950): the operands, the tiles and their k-steps, and which form a call runs in.
// gemm_blocks.hip has the products themselves, gemm_blocks_act.hip those with an activation and a residual behind them.
#pragma once

#include <algorithm>

#include "gemm_core.h"

namespace h3b {

using namespace h3g;

struct BlocksParams {
    const uint8_t* a;           // [M, K] e4m3
    const uint8_t* w;           // [E, N, K] e4m3
    const float* sa;            // [M, KB], element strides sa_m, sa_k
    const float* sw;            // [E, NB, KB], element strides sw_e, sw_n, sw_k
    const void* bias;           // [N] in the output's type, or null
    uint16_t* y;                // [M, N] bf16 / fp16
    const void* offsets;        // grouped: [E + 1] int32 / int64; null: one group of all rows
    int64_t lda, ldw, w_e, ldy;
    int64_t sa_m, sa_k, sw_e, sw_n, sw_k;
    int64_t M;
    int N, K, E;
    int idx_bytes;
    int fp16;                   // output type
};

__device__ __forceinline__ int64_t offset_at(const BlocksParams& p, int e) {
    const int64_t v = p.idx_bytes == 8 ? reinterpret_cast<const int64_t*>(p.offsets)[e]
                                       : (int64_t)reinterpret_cast<const int32_t*>(p.offsets)[e];
    return v < 0 ? 0 : v > p.M ? p.M : v;                 // whatever the offsets hold, no row outside [0, M) is touched
}

// Rows of one tile: `rows` (<= TT) from row0 on, of expert e.
struct TileRows {
    int e, rows;
    int64_t row0;
};

// Inclusive prefix sums over the 64 lanes: within rows of 16 by shifts, then across rows.
__device__ __forceinline__ int wave_prefix(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);        // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);        // row_bcast 15 into rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);        // row_bcast 31 into rows 2 and 3
    return v;
}

// By expert: row tile t (TT rows each, no tile spans two experts, an expert without rows has none); false past the last one.  A wave
// looks at 64 experts at a time.
__device__ __forceinline__ bool locate_rows(const BlocksParams& p, int TT, int64_t t, int lane, TileRows& r) {
    for (int e0 = 0; e0 < p.E; e0 += 64) {
        const int e = e0 + lane;
        int64_t lo = 0, hi = 0;
        if (e < p.E) {
            lo = offset_at(p, e);
            hi = offset_at(p, e + 1);
        }
        const int n = hi > lo ? (int)((hi - lo + TT - 1) / TT) : 0;
        const int sum = wave_prefix(n);
        const uint64_t past = __ballot(sum > t);
        if (past) {
            const int f = __ffsll((unsigned long long)past) - 1;
            // offsets are at most M < 2^31
            const int first = __builtin_amdgcn_readlane((int)lo, f), last = __builtin_amdgcn_readlane((int)hi, f);
            r.e = e0 + f;
            r.row0 = first + (t - (__builtin_amdgcn_readlane(sum, f) - __builtin_amdgcn_readlane(n, f))) * TT;
            r.rows = (int)min<int64_t>(TT, last - r.row0);
            return true;
        }
        t -= __builtin_amdgcn_readlane(sum, 63);
    }
    return false;
}

// ---- the tiled form -------------------------------------------------------------------------------------------------
//
// A workgroup of WN x WM waves, one per CU, walks tiles of TW channels x TT tokens (persistent: tile b, b + G, ...); a wave
// owns NI x NJ MFMA blocks, its 16 NI channels within one 128-channel weight block.  Two waves share a SIMD, so each has
// 256 registers; acc takes 4 NI NJ of them.
//   * Operands go global -> LDS by LDS-DMA (whole 128-byte lines, 8 rows an instruction) into NST stages of one k-block each;
//     the loads run NST k-steps ahead of the MFMAs, across tile boundaries.
//   * Two barriers per k-step.  The first, when its token fragments and scales are in registers: their part of stage g is free
//     and takes those of k-step g + NST, one load per MFMA.  The second, when its channel fragments are, and this wave's share
//     of stage g + 1 has landed: the weights' part follows, and the next first fragments are read behind the remaining MFMAs.
//     The last load then stands 28 of a k-step's 32 MFMAs before the wait for it.  (One barrier, the nine loads of a k-step
//     one per MFMA behind it, the last 18 MFMAs ahead: 18 880 x 21 504 x 5376 1890 us against 1814; two loads per MFMA: 1977.)
//     The last two channel blocks go token by token, so that a token's fragment registers are free for the next k-step's as
//     early as possible.
//   * A wave whose tokens all lie behind the tile's rows only loads: the other wave of its SIMD runs alone.
//   * The fmas of an MFMA's four results stand LAG MFMAs behind it (it needs 24 wait states), also across k-steps; per MFMA
//     (32 cycles of the matrix pipe) they cost 16 cycles of the vector pipe.
//   * Channel of MFMA block i, row 4 g + r: 32 (i / 2) + 8 g + 4 (i % 2) + r, so that two blocks' results of a lane are 8
//     consecutive channels: the epilogue stores 16 bytes per lane, 64-byte pieces of a row, without going through LDS.
//   * LDS rows are 128 bytes; logical 16-byte chunk c of row r is stored at c ^ (weights: swz_w(r), tokens: swz(r)), which
//     puts the 16 rows of a fragment read on different banks.
//     A 16-byte read serves lanes 0-3, 12-15 and 20-27 together, and 4-11, 16-19 and 28-31: lane groups g and g ^ 1 read chunks
//     that differ in bit 0, so that those 16 lanes meet 16 places (with chunks 2 g, 2 g + 1: twice the LDS cycles; 200 x 5376
//     x 7168 23.7 us against 22.6).  The order of k within a block is the operands' common one and changes no product.
//   * Every tile has buffer descriptors of its own from its own base: rows past the tile's read zeros and store nothing,
//     and nothing else is limited to 32-bit offsets.
// What bounds it: with operands in the caches the return path from L2 to LDS (64 KiB a k-step and CU) beside the matrix pipe,
// busy 0.54 of the time at 2.0 GHz and 0.63 at the 1.5 GHz that the power limit leaves under a lasting load: 18 880 x 21 504 x
// 5376 in 1780-1890 us (2.3-2.45 PFLOP/s), 32 768 rows over 32 experts of 4096 x 4096 in 550-600 (2.0-1.8: every expert's last tile
// is partly empty).  With few rows per expert the weights' way from memory: 4100 rows over 16 experts 111 us; 16 x 128 rows 76 us
// from memory, 44 from the caches.  Fetching the weights' lines into L2 some k-steps ahead by one more load per wave (a dword
// of each line) made every case slower (1890 -> 2244 us): the requests that are under way are the limit.
__device__ __forceinline__ int swz_w(int r) { return ((r >> 1) & 1) | (((r >> 3) & 3) << 1); }

constexpr int LAG = 5;
constexpr int AHEAD = 3;                                  // channel blocks read ahead of their MFMAs

template <int WN_, int WM_, int NI_, int NJ_, int NST_>
struct BTile {
    static constexpr int WN = WN_, WM = WM_, NI = NI_, NJ = NJ_, NST = NST_;
    static constexpr bool PAIRS = NI % 2 == 0;
    static constexpr int WAVES = WN * WM, NM = NI * NJ;
    static constexpr int TW = 16 * NI * WN, TT = 16 * NJ * WM;
    static constexpr int WL = TW / 8 / WAVES, AL = TT / 8 / WAVES;   // LDS-DMA instructions per wave and k-step
    static constexpr int SC_A = (TT + 63) / 64;                      // 64-token pieces of scales, one more piece: the weight's
    static constexpr int SL = (SC_A + WAVES) / WAVES;                // ... and the scales' per wave
    static constexpr int LOADS = WL + AL + SL;
    static constexpr int STAGE = (TW + TT) * ROWB, A_OFF = TW * ROWB;
    static constexpr int SC_OFF = NST * STAGE, SC_STAGE = SL * WAVES * 256;
    static constexpr int LDS = SC_OFF + NST * SC_STAGE;
    static_assert(LDS <= 160 * 1024, "LDS");
    __device__ static int swz_of_w(int r) { return PAIRS ? swz_w(r) : swz(r); }
};

// NT (both kinds of tiles): the weight loads carry the non-temporal hint.
template <int WN, int WM, int NI, int NJ, int NST, bool NT_ = false>
struct BigTile : BTile<WN, WM, NI, NJ, NST> {
    using B = BTile<WN, WM, NI, NJ, NST>;
    static constexpr bool NT = NT_;
    static constexpr int U0 = (NI - 2) * NJ;                         // MFMAs before the last two channel blocks
    static constexpr int EARLY = NJ;                                 // the MFMA that the first barrier stands behind
    static constexpr int BAR = (NI - 1 - AHEAD) * NJ + NJ;           // ... and the second
    static_assert(NI % 2 == 0 && NI > AHEAD && B::NM > LAG && B::SL == 1 && B::TW % 128 == 0 && 128 % (16 * NI) == 0, "wave tile");
    static_assert(B::TW % (8 * B::WAVES) == 0 && B::TT % (8 * B::WAVES) == 0 && B::WL <= 15 && B::AL <= 15, "whole loads per wave");
    static_assert(B::LOADS * (NST - 1) <= 63, "vmcnt range");
    static constexpr int mi(int u) { return u < U0 ? u / NJ : NI - 2 + (u - U0) % 2; }
    static constexpr int mj(int u) { return u < U0 ? u % NJ : (u - U0) / 2; }
};

// KS: k-steps per barrier.
template <int WN, int WM, int NI, int NJ, int NST, int KS_, bool NT_ = false>
struct SmallTile : BTile<WN, WM, NI, NJ, NST> {
    using B = BTile<WN, WM, NI, NJ, NST>;
    static constexpr int KS = KS_;
    static constexpr bool NT = NT_;
    static constexpr int PIECES = B::SC_A + 1;                       // of scales: 64 tokens' each, and the weight blocks'
    static constexpr int SL = (PIECES + B::WAVES - 1) / B::WAVES;    // ... per wave, in the first PIECES waves at least
    static constexpr bool EVEN = PIECES % B::WAVES == 0;             // ... and in every wave
    static constexpr int LOADS = B::WL + B::AL + SL;                 // instructions of those waves; one fewer in the others
    static constexpr int SC_OFF = B::STAGE, STAGE = SC_OFF + PIECES * 256;   // a stage's scales behind its operands
    static constexpr int LDS = NST * STAGE;
    static_assert(B::TW % (8 * B::WAVES) == 0 && B::TT % (8 * B::WAVES) == 0, "whole load instructions per wave");
    static_assert(128 % (16 * NI) == 0 && (B::TW % 128 == 0 || 128 % B::TW == 0), "a wave's channels in one weight block");
    static_assert(LDS <= 160 * 1024 && LOADS * (NST - 1) <= 63 && KS <= 2 && NST >= 2 * KS, "LDS, vmcnt range, ring");
    static constexpr int mi(int u) { return u / NJ; }
    static constexpr int mj(int u) { return u % NJ; }
};

// The tile whose operands are loaded next, and its k-step.
template <class T>
struct BCursor {
    v4u rw, ra, rs;             // buffer descriptors of the weight rows, the token rows and this wave's scales
    uint32_t vw[T::WL], va[T::AL];  // lane offsets of the wave's 8-row groups
    uint32_t cut;               // bit i (weights) / 16 + j (tokens): the lane's chunk lies at or past K in the last k-step
    uint32_t vs;                // lane offset of the scale load
    uint32_t k0, s0;            // byte offsets of the k-step: operands, scales
    int ks, c;
    bool valid;
};

template <class T>
struct BFrags {
    v8i w[2], t[T::NJ];         // the next k-step's first two channel blocks and its tokens
    float sa[T::NJ], sw;        // ... and its scales
};

struct TileSpace {
    int rt, tiles_n, total;     // row tiles, channel tiles
    const int* tab;             // grouped: row tiles of experts 0 .. e, then their first rows and the rows behind their last, in LDS
};

constexpr int MAX_TAB = 256;    // experts of the LDS table; more are counted from the offsets at every tile

// The table, by one wave; returns all experts' row tiles.
__device__ __forceinline__ int fill_table(const BlocksParams& p, int TT, int lane, int* tab) {
    int base = 0;
    for (int e0 = 0; e0 < p.E; e0 += 64) {
        const int e = e0 + lane;
        int n = 0, lo = 0, hi = 0;
        if (e < p.E) {
            lo = (int)offset_at(p, e), hi = (int)offset_at(p, e + 1);
            n = hi > lo ? (int)(((int64_t)hi - lo + TT - 1) / TT) : 0;
        }
        const int sum = wave_prefix(n);
        if (e < MAX_TAB && e < p.E) {
            tab[e] = base + sum;
            tab[MAX_TAB + e] = lo;
            tab[2 * MAX_TAB + e] = hi;
        }
        base += __builtin_amdgcn_readlane(sum, 63);
    }
    return base;
}

// Tile `id` of the launch: its rows and channel tile.
template <class T, bool GROUPED>
__device__ __forceinline__ bool tile_at(const BlocksParams& p, const TileSpace& sp, int id, int lane, TileRows& r, int& tn) {
    if (id >= sp.total) return false;
    int tm;
    tile_of(id, sp.total, sp.rt, sp.tiles_n, 4, tm, tn);
    if (!GROUPED) {
        r.e = 0;
        r.row0 = (int64_t)tm * T::TT;
        r.rows = (int)min<int64_t>(T::TT, p.M - r.row0);
        return true;
    }
    if (p.E > MAX_TAB) return locate_rows(p, T::TT, tm, lane, r);
    int before = 0;
    for (int e0 = 0; e0 < p.E; e0 += 64) {
        const int v = e0 + lane < p.E ? sp.tab[e0 + lane] : 0x7fffffff;
        const uint64_t past = __ballot(v > tm);
        if (past) {
            const int f = __builtin_ctzll(past);
            if (f) before = __builtin_amdgcn_readlane(v, f - 1);
            r.e = e0 + f;
            break;
        }
        before = __builtin_amdgcn_readlane(v, 63);
    }
    const int lo = __builtin_amdgcn_readfirstlane(sp.tab[MAX_TAB + r.e]), hi = __builtin_amdgcn_readfirstlane(sp.tab[2 * MAX_TAB + r.e]);
    r.row0 = lo + (int64_t)(tm - before) * T::TT;
    r.rows = (int)min<int64_t>(T::TT, hi - r.row0);
    return true;
}

template <class T, bool GROUPED>
__device__ __forceinline__ void cursor_tile(BCursor<T>& I, const BlocksParams& p, const TileSpace& sp, int c, int wave, int lane) {
    I.c = c;
    I.ks = 0;
    I.k0 = I.s0 = 0;
    TileRows r;
    int tn = 0;
    I.valid = tile_at<T, GROUPED>(p, sp, (int)blockIdx.x + c * (int)gridDim.x, lane, r, tn);
    if (!I.valid) {                                       // the loads still run, read nothing and fill the stage with zeros
        I.rw[2] = I.ra[2] = I.rs[2] = 0;
        return;
    }
    const int n0 = tn * T::TW, nrows = min(T::TW, p.N - n0);
    const int kb = (p.K + BK - 1) / BK;
    I.rw = buffer_desc(p.w + r.e * p.w_e + (int64_t)n0 * p.ldw, (uint32_t)((nrows - 1) * p.ldw + p.K));
    I.ra = buffer_desc(p.a + r.row0 * p.lda, (uint32_t)((r.rows - 1) * p.lda + p.K));
    const bool tok = wave < T::SC_A;                      // the first wave past the token scales': the weight's
    const int nb = (nrows + 127) / 128;
    const float* base = tok ? p.sa + r.row0 * p.sa_m : p.sw + r.e * p.sw_e + (int64_t)(n0 / 128) * p.sw_n;
    const int64_t st = tok ? p.sa_m : p.sw_n, sk = tok ? p.sa_k : p.sw_k;
    const int entries = tok ? r.rows : nb, first = tok ? 64 * wave : 64 * (wave - T::SC_A);
    I.rs = buffer_desc(base, (uint32_t)(((entries - 1) * st + (kb - 1) * sk) * 4 + 4));
    I.vs = first + lane < entries ? (uint32_t)((first + lane) * st * 4) : OOB;
}

template <class T, bool GROUPED>
__device__ __forceinline__ void cursor_next(BCursor<T>& I, const BlocksParams& p, const TileSpace& sp, int nk, int wave, int lane) {
    if (!I.valid) return;                                 // empty descriptors: offset 0
    ++I.ks;
    I.k0 += BK;
    I.s0 += (uint32_t)__builtin_amdgcn_readfirstlane((int)((wave < T::SC_A ? p.sa_k : p.sw_k) * 4));
    if (__builtin_expect(I.ks == nk, 0)) cursor_tile<T, GROUPED>(I, p, sp, I.c + 1, wave, lane);
}

// What the load instructions of the cursor's k-step share: their uniform byte offsets and LDS addresses, in scalar registers
// for inline asm (the compiler may keep a uniform value in a vector register, and does not move it back for an asm operand).
// The wait states that asm leaves to the program: one between a vector write and its readfirstlane, two between that and a
// vector instruction that reads the scalar, five before a memory instruction that does.
struct BIssue {
    uint32_t k0, s0, w, a, sc, cut;
};

template <class T>
__device__ __forceinline__ BIssue bissue(const BCursor<T>& I, int nk, uint32_t st, uint32_t sc, int wave) {
    BIssue S;
    asm volatile("s_nop 0\n\tv_readfirstlane_b32 %0, %5\n\tv_readfirstlane_b32 %1, %6\n\tv_readfirstlane_b32 %2, %7\n\t"
                 "v_readfirstlane_b32 %3, %8\n\tv_readfirstlane_b32 %4, %9\n\ts_nop 4"
                 : "=&s"(S.k0), "=&s"(S.s0), "=&s"(S.w), "=&s"(S.a), "=&s"(S.sc)
                 : "v"(I.k0), "v"(I.s0), "v"(st + (uint32_t)(wave * T::WL * 8 * ROWB)),
                   "v"(st + (uint32_t)(T::A_OFF + wave * T::AL * 8 * ROWB)), "v"(sc + 256u * (uint32_t)wave));
    S.cut = I.ks == nk - 1 ? I.cut : 0u;
    return S;
}

// Load instruction i of the k-step.  The hardware checks the lane's offset against the buffer's size less the uniform offset,
// so that one (k0, s0) never exceeds the size: the rows are in the lane's.
template <class T>
__device__ __forceinline__ void bload(const BCursor<T>& I, const BIssue& S, int i) {
    if (i < T::WL) {
        const uint32_t at = S.w + (uint32_t)(i * 8 * ROWB), v = I.vw[i] | ((S.cut << (31 - i)) & OOB);
        if (T::NT) dma16_at_nt(I.rw, at, v, S.k0);
        else dma16_at(I.rw, at, v, S.k0);
    } else if (i < T::WL + T::AL) {
        const int j = i - T::WL;
        dma16_at(I.ra, S.a + (uint32_t)(j * 8 * ROWB), I.va[j] | ((S.cut << (15 - j)) & OOB), S.k0);
    } else {
        dma4_at(I.rs, S.sc, I.vs, S.s0);
    }
}

__device__ __forceinline__ v8i frag16(const uint8_t* p0, const uint8_t* p1, int off) {
    const uint4 lo = *reinterpret_cast<const uint4*>(p0 + off);
    const uint4 hi = *reinterpret_cast<const uint4*>(p1 + off);
    v8i f;
    f[0] = (int)lo.x; f[1] = (int)lo.y; f[2] = (int)lo.z; f[3] = (int)lo.w;
    f[4] = (int)hi.x; f[5] = (int)hi.y; f[6] = (int)hi.z; f[7] = (int)hi.w;
    return f;
}

// A wave's fragment addresses within a stage: lane l reads row c = l & 15 of a block, logical chunks k0 and k0 + 2, k0 = 0, 1, 4, 5
// by g = l >> 4.
template <class T>
struct BAddr {
    uint32_t w0, w1, t0, t1, sa, sw;
};

template <class T>
__device__ __forceinline__ BAddr<T> baddr(int wn, int wm, int lane) {
    const int c = lane & 15, g = lane >> 4, k0 = 4 * (g >> 1) + (g & 1);
    const int wr = T::PAIRS ? 8 * (c >> 2) + (c & 3) : c; // + 32 (i / 2) + 4 (i % 2), or + 16 i; neither changes the swizzle
    const int tr = c;                                     // + 16 j; neither changes swz
    BAddr<T> A;
    A.w0 = (uint32_t)((wn * 16 * T::NI + wr) * ROWB + (k0 ^ T::swz_of_w(wr)) * 16);
    A.w1 = (uint32_t)((wn * 16 * T::NI + wr) * ROWB + ((k0 + 2) ^ T::swz_of_w(wr)) * 16);
    A.t0 = (uint32_t)(T::A_OFF + (wm * 16 * T::NJ + tr) * ROWB + (k0 ^ swz(tr)) * 16);
    A.t1 = (uint32_t)(T::A_OFF + (wm * 16 * T::NJ + tr) * ROWB + ((k0 + 2) ^ swz(tr)) * 16);
    A.sa = (uint32_t)((wm * 16 * T::NJ + c) * 4);
    A.sw = (uint32_t)(T::SC_A * 256 + (wn * 16 * T::NI / 128) * 4);
    return A;
}

template <class T>
__device__ __forceinline__ v8i read_w(const uint8_t* st, const BAddr<T>& A, int i) {
    return frag16(st + A.w0, st + A.w1, (T::PAIRS ? 32 * (i >> 1) + 4 * (i & 1) : 16 * i) * ROWB);
}

template <class T>
__device__ __forceinline__ v8i read_t(const uint8_t* st, const BAddr<T>& A, int j) {
    return frag16(st + A.t0, st + A.t1, 16 * j * ROWB);
}

template <class T>
__device__ __forceinline__ void bfma(v4f (&acc)[T::NI][T::NJ], const v4f& b, float s, int u) {
    v4f& a = acc[T::mi(u)][T::mj(u)];
#pragma unroll
    for (int r = 0; r < 4; ++r) a[r] = __builtin_fmaf(b[r], s, a[r]);
    asm volatile("" : "+v"(a));                           // here, not wherever the sum is needed next
}

// One k-step: F holds its first fragments and scales and receives the next one's; pend and sp the last LAG MFMAs' results
// and scales.  cur / nxt: this stage and the next; ld: the stage that the loads of the cursor's k-step go to (this one).
template <class T>
__device__ __forceinline__ void bkstep(const uint8_t* lds, uint32_t lds0, uint32_t cur, uint32_t nxt, uint32_t cur_sc, uint32_t nxt_sc,
                                       const BCursor<T>& I, int nk, const BAddr<T>& A, int wave,
                                       v4f (&acc)[T::NI][T::NJ], BFrags<T>& F, v4f (&pend)[LAG], float (&sp)[T::NJ]) {
    v8i w[T::NI], t[T::NJ];
    v4f b[T::NM];
    float s[T::NJ];
    const BIssue S = bissue<T>(I, nk, lds0 + cur, lds0 + cur_sc, wave);
    w[0] = F.w[0];
    w[1] = F.w[1];
#pragma unroll
    for (int j = 0; j < T::NJ; ++j) t[j] = F.t[j];
#pragma unroll
    for (int u = 0; u < T::NM; ++u) {
        b[u] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w[T::mi(u)], t[T::mj(u)], v4f{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);                // the fmas behind it: 25 wait states to the MFMA they read
        if (u == LAG - 2) {
#pragma unroll
            for (int j = 0; j < T::NJ; ++j) s[j] = F.sa[j] * F.sw;
        }
        if (u < LAG) bfma<T>(acc, pend[u], sp[T::mj(T::NM - LAG + u)], T::NM - LAG + u);
        else bfma<T>(acc, b[u - LAG], s[T::mj(u - LAG)], u - LAG);
#pragma unroll
        for (int i = 2; i < T::NI; ++i)                   // this stage's channel blocks, AHEAD of their MFMAs
            if (u == (i < AHEAD ? 0 : (i - AHEAD) * T::NJ + (i == AHEAD ? 1 : 0))) w[i] = read_w<T>(lds + cur, A, i);
        if (u == T::BAR) {
            wait_lgkm0();                                 // this wave's reads of the stage have returned
            __builtin_amdgcn_s_waitcnt(vmcnt_imm(T::LOADS * (T::NST - 2) + T::AL + T::SL));   // its share of the next one has landed
            barrier_nofence();
        }
        if (u == T::EARLY) barrier_nofence();              // the first MFMAs waited for the tokens, read behind the scales
        if (u > T::EARLY && u <= T::EARLY + T::AL + T::SL) bload<T>(I, S, T::WL + u - T::EARLY - 1);
        if (u > T::BAR) {
            if (u <= T::BAR + T::WL) bload<T>(I, S, u - T::BAR - 1);
            if (u == T::BAR + 1) F.w[0] = read_w<T>(lds + nxt, A, 0);
            if (u == T::BAR + 2) F.w[1] = read_w<T>(lds + nxt, A, 1);
            if (u == T::BAR + 3) {
#pragma unroll
                for (int j = 0; j < T::NJ; ++j) F.sa[j] = *reinterpret_cast<const float*>(lds + nxt_sc + A.sa + 64 * j);
                F.sw = *reinterpret_cast<const float*>(lds + nxt_sc + A.sw);
            }
            if (u > T::U0 && (u - T::U0) % 2 == 1) F.t[(u - T::U0) / 2] = read_t<T>(lds + nxt, A, (u - T::U0) / 2);
        }
        __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int k = 0; k < LAG; ++k) pend[k] = b[T::NM - LAG + k];
#pragma unroll
    for (int j = 0; j < T::NJ; ++j) sp[j] = s[j];
}

// The first fragments and the scales of a tile, from its first stage.
template <class T>
__device__ __forceinline__ void bfirst(const uint8_t* lds, uint32_t st, uint32_t sc, const BAddr<T>& A, BFrags<T>& F) {
    F.w[0] = read_w<T>(lds + st, A, 0);
    F.w[1] = read_w<T>(lds + st, A, 1);
#pragma unroll
    for (int j = 0; j < T::NJ; ++j) F.sa[j] = *reinterpret_cast<const float*>(lds + sc + A.sa + 64 * j);
    F.sw = *reinterpret_cast<const float*>(lds + sc + A.sw);
    __builtin_amdgcn_sched_barrier(0);                    // the tokens last, as in a k-step
#pragma unroll
    for (int j = 0; j < T::NJ; ++j) F.t[j] = read_t<T>(lds + st, A, j);
}

// One k-step of a wave whose tokens lie behind the tile's rows: its loads and the barriers.
template <class T>
__device__ __forceinline__ void bidle(uint32_t lds0, uint32_t cur, uint32_t cur_sc, const BCursor<T>& I, int nk, int wave) {
    const BIssue S = bissue<T>(I, nk, lds0 + cur, lds0 + cur_sc, wave);
    wait_lgkm0();
    barrier_nofence();
#pragma unroll
    for (int f = T::WL; f < T::LOADS; ++f) bload<T>(I, S, f);
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(T::LOADS * (T::NST - 2) + T::AL + T::SL));
    barrier_nofence();
#pragma unroll
    for (int f = 0; f < T::WL; ++f) bload<T>(I, S, f);
}

template <class T, bool FP16, bool BIAS>
__device__ __forceinline__ void bstore(const BlocksParams& p, const TileRows& r, int tn, int wn, int wm, int lane,
                                       const v4f (&acc)[T::NI][T::NJ]) {
    const int c = lane & 15, g = lane >> 4;
    const __amdgpu_buffer_rsrc_t yr = make_rsrc(p.y + r.row0 * p.ldy, (uint32_t)(((r.rows - 1) * p.ldy + p.N) * 2));
    if constexpr (!T::PAIRS) {                            // 4 consecutive channels a lane and block
#pragma unroll
        for (int i = 0; i < T::NI; ++i) {
            const int n = tn * T::TW + wn * 16 * T::NI + 16 * i + 4 * g;
            const bool in = n < p.N;
            float bias[4] = {0.f, 0.f, 0.f, 0.f};
            if (BIAS) {
#pragma unroll
                for (int e = 0; e < 4; ++e) bias[e] = load_bias(p.bias, (in ? n : 0) + e, FP16);
            }
#pragma unroll
            for (int j = 0; j < T::NJ; ++j) {
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = (acc[i][j][e] + 0.0f) + (BIAS ? bias[e] : 0.0f);
                const v2u32 o = FP16 ? v2u32{fp16_rne(v[0]) | (fp16_rne(v[1]) << 16), fp16_rne(v[2]) | (fp16_rne(v[3]) << 16)}
                                     : v2u32{cvt_bf16x2(v[0], v[1]), cvt_bf16x2(v[2], v[3])};
                const uint32_t off = (uint32_t)(wm * 16 * T::NJ + 16 * j + c) * (uint32_t)p.ldy * 2u + (uint32_t)n * 2u;
                __builtin_amdgcn_raw_buffer_store_b64(o, yr, in ? off : OOB, 0, 0);
            }
        }
        return;
    }
    const int n0 = tn * T::TW + wn * 16 * T::NI + 8 * g;
#pragma unroll
    for (int q = 0; q < T::NI / 2; ++q) {
        const int n = n0 + 32 * q;
        const bool in = n < p.N;
        float bias[8];
        if (BIAS) {
#pragma unroll
            for (int e = 0; e < 8; ++e) bias[e] = load_bias(p.bias, (in ? n : 0) + e, FP16);
        }
#pragma unroll
        for (int j = 0; j < T::NJ; ++j) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = (acc[2 * q + (e >> 2)][j][e & 3] + 0.0f) + (BIAS ? bias[e] : 0.0f);
            v4u o;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                o[e] = FP16 ? fp16_rne(v[2 * e]) | (fp16_rne(v[2 * e + 1]) << 16) : cvt_bf16x2(v[2 * e], v[2 * e + 1]);
            const uint32_t off = (uint32_t)(wm * 16 * T::NJ + 16 * j + c) * (uint32_t)p.ldy * 2u + (uint32_t)n * 2u;
            __builtin_amdgcn_raw_buffer_store_b128(o, yr, in ? off : OOB, 0, 0);
        }
    }
}

// The kernel; `store` writes a tile's sums (REREAD: it takes more than a few registers).
template <class T, bool GROUPED>
constexpr int tile_lds() { return T::LDS + (GROUPED ? 3 * MAX_TAB * 4 : 0); }

template <class T, bool GROUPED, class Store>
__device__ __forceinline__ void tile_kernel(const BlocksParams& p, uint8_t* lds, const Store& store) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int wn = wave % T::WN, wm = wave / T::WN;
    const uint32_t lds0 = lds_addr(lds);
    const int nk = (p.K + BK - 1) / BK, ktail = p.K % BK;
    TileSpace sp;
    sp.tiles_n = (p.N + T::TW - 1) / T::TW;
    sp.rt = (int)((p.M + T::TT - 1) / T::TT);
    sp.tab = reinterpret_cast<const int*>(lds + T::LDS);
    if (GROUPED) {                                        // every wave counts, and writes the same table
        sp.rt = fill_table(p, T::TT, lane, reinterpret_cast<int*>(lds + T::LDS));
        __syncthreads();
    }
    sp.total = sp.rt * sp.tiles_n;

    BCursor<T> I;
    {
        // lane l moves LDS chunk l & 7 of row l >> 3 of an 8-row group: logical chunk (l & 7) ^ swizzle(row)
        const int lrow = lane >> 3;
        I.cut = 0;
#pragma unroll
        for (int i = 0; i < T::WL; ++i) {
            const int row = 8 * (wave * T::WL + i) + lrow, ch = (lane & 7) ^ T::swz_of_w(row);
            I.vw[i] = (uint32_t)(row * p.ldw) + 16u * (uint32_t)ch;
            I.cut |= ktail && 16 * ch >= ktail ? 1u << i : 0u;
        }
#pragma unroll
        for (int j = 0; j < T::AL; ++j) {
            const int row = 8 * (wave * T::AL + j) + lrow, ch = (lane & 7) ^ swz(row);
            I.va[j] = (uint32_t)(row * p.lda) + 16u * (uint32_t)ch;
            I.cut |= ktail && 16 * ch >= ktail ? 1u << (16 + j) : 0u;
        }
    }
    I.rw = buffer_desc(nullptr, 0);
    I.ra = I.rs = I.rw;
    I.vs = OOB;
    cursor_tile<T, GROUPED>(I, p, sp, 0, wave, lane);
    if (!I.valid) return;
#pragma unroll 1
    for (int s = 0; s < T::NST; ++s) {
        const BIssue S = bissue<T>(I, nk, lds0 + (uint32_t)s * T::STAGE, lds0 + T::SC_OFF + (uint32_t)s * T::SC_STAGE, wave);
#pragma unroll
        for (int i = 0; i < T::LOADS; ++i) bload<T>(I, S, i);
        cursor_next<T, GROUPED>(I, p, sp, nk, wave, lane);
    }
    const BAddr<T> A = baddr<T>(wn, wm, lane);
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(T::LOADS * (T::NST - 1)));
    barrier_nofence();
    uint32_t cur = 0, cur_sc = T::SC_OFF;
    auto next_stage = [&](uint32_t& n, uint32_t& n_sc) {
        n = cur == (T::NST - 1) * T::STAGE ? 0u : cur + T::STAGE;
        n_sc = n == 0 ? T::SC_OFF : cur_sc + T::SC_STAGE;
    };
    BFrags<T> F;
    bfirst<T>(lds, 0, T::SC_OFF, A, F);

    for (int c = 0;; ++c) {
        TileRows r;
        int tn = 0;
        if (!tile_at<T, GROUPED>(p, sp, (int)blockIdx.x + c * (int)gridDim.x, lane, r, tn)) break;
        if (r.rows <= wm * 16 * T::NJ) {                  // the other waves of the SIMDs have the matrix pipes to themselves
            for (int ks = 0; ks < nk; ++ks) {
                uint32_t nxt, nxt_sc;
                next_stage(nxt, nxt_sc);
                bidle<T>(lds0, cur, cur_sc, I, nk, wave);
                cursor_next<T, GROUPED>(I, p, sp, nk, wave, lane);
                cur = nxt;
                cur_sc = nxt_sc;
            }
            bfirst<T>(lds, cur, cur_sc, A, F);            // the next tile's, as the last k-step of the others reads them
            continue;
        }
        v4f acc[T::NI][T::NJ], pend[LAG];
        float sp_[T::NJ];
#pragma unroll
        for (int i = 0; i < T::NI; ++i)
#pragma unroll
            for (int j = 0; j < T::NJ; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < LAG; ++k) pend[k] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < T::NJ; ++j) sp_[j] = 0.f;
        for (int ks = 0; ks < nk; ++ks) {
            uint32_t nxt, nxt_sc;
            next_stage(nxt, nxt_sc);
            bkstep<T>(lds, lds0, cur, nxt, cur_sc, nxt_sc, I, nk, A, wave, acc, F, pend, sp_);
            cursor_next<T, GROUPED>(I, p, sp, nk, wave, lane);
            cur = nxt;
            cur_sc = nxt_sc;
        }
        // the last results: 24 wait states behind their MFMAs, as a dependence
        asm volatile("s_nop 15\n\ts_nop 7" : "+v"(pend[LAG - 1]));
#pragma unroll
        for (int k = 0; k < LAG; ++k) {
            asm volatile("" : "+v"(pend[k]));
            bfma<T>(acc, pend[k], sp_[T::mj(T::NM - LAG + k)], T::NM - LAG + k);
        }
        store(p, r, tn, wn, wm, lane, acc);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (Store::REREAD) {                    // the store needs the next fragments' registers: they are read again
            asm volatile("" ::: "memory");
            bfirst<T>(lds, cur, cur_sc, A, F);
        }
    }
    wait_vm0();                                           // the loads behind the last k-step have landed before the exit
}

// ---- the forms of small tiles ---------------------------------------------------------------------------------------
//
// Few tiles, or few rows per tile: the time is that of streaming the operands (the weights, mostly) and of a k-step's chain of
// barrier, fragment reads and MFMAs.  One workgroup per tile, a deep ring of stages, fragments read a whole k-step ahead (two
// sets of registers, the loop unrolled by two) and the fmas a whole k-step behind their MFMAs.
// 200 x 5376 x 7168 22.6 us (128 x 64 tiles on 168 CUs, 0.4 us a k-step: 225 MB from L2 at 10 TB/s); 1 x 21 504 x 5376 19.5 us
// (5.9 TB/s of weights); 64 rows over 32 experts of 2048 x 4096 52 us with two rows in each (5.2 TB/s), 45 with rows in 25 of them (4.7).
// The LDS is the launch's: a size that the compiler knew would let it give a lone workgroup 512 registers a lane and put the
// MFMAs' results into the accumulation half, a copy away from the fmas.
template <class T>
struct SFrags {
    v8i w[T::NI], t[T::NJ];
    float s[T::NJ], sw;
};

template <class T>
__device__ __forceinline__ void sread(SFrags<T>& F, const uint8_t* lds, uint32_t st, const BAddr<T>& A) {
#pragma unroll
    for (int j = 0; j < T::NJ; ++j) F.t[j] = read_t<T>(lds + st, A, j);
#pragma unroll
    for (int i = 0; i < T::NI; ++i) F.w[i] = read_w<T>(lds + st, A, i);
#pragma unroll
    for (int j = 0; j < T::NJ; ++j) F.s[j] = *reinterpret_cast<const float*>(lds + st + T::SC_OFF + A.sa + 64 * j);
    F.sw = *reinterpret_cast<const float*>(lds + st + T::SC_OFF + A.sw);
}

// The tile's loads: descriptors, lane offsets at k = 0 (OOB: nothing), the next k-step's offsets, the k-steps left.
template <class T>
struct SLoader {
    v4u rw, ra, rs[T::SL];
    uint32_t vw[T::WL], va[T::AL], vs[T::SL], step[T::SL];
    uint32_t k0, k_step, s0[T::SL];
    uint32_t dw, da, ds;
    int left, ktail;
    bool full;                                            // this wave loads SL pieces of scales (else one fewer)
};

template <class T>
__device__ __forceinline__ void sload_set(SLoader<T>& L, const BlocksParams& p, const TileRows& r, int tn, int wave, int lane) {
    const int kb = (p.K + BK - 1) / BK, lrow = lane >> 3;
    const int n0 = tn * T::TW, nrows = min(T::TW, p.N - n0);
    L.rw = buffer_desc(p.w + r.e * p.w_e + (int64_t)n0 * p.ldw, (uint32_t)((nrows - 1) * p.ldw + p.K));
    L.ra = buffer_desc(p.a + r.row0 * p.lda, (uint32_t)((r.rows - 1) * p.lda + p.K));
#pragma unroll
    for (int i = 0; i < T::WL; ++i) {
        const int row = 8 * (wave * T::WL + i) + lrow;
        L.vw[i] = (uint32_t)(row * p.ldw) + 16u * (uint32_t)((lane & 7) ^ T::swz_of_w(row));
    }
#pragma unroll
    for (int j = 0; j < T::AL; ++j) {
        const int row = 8 * (wave * T::AL + j) + lrow;
        L.va[j] = (uint32_t)(row * p.lda) + 16u * (uint32_t)((lane & 7) ^ swz(row));
    }
    const int nb = (nrows + 127) / 128;
#pragma unroll
    for (int i = 0; i < T::SL; ++i) {                     // piece q: 64 tokens' scales, piece SC_A the weight blocks'
        const int q = wave + i * T::WAVES;
        const bool tok = q < T::SC_A;
        const float* base = tok ? p.sa + r.row0 * p.sa_m : p.sw + r.e * p.sw_e + (int64_t)(n0 / 128) * p.sw_n;
        const int64_t st = tok ? p.sa_m : p.sw_n, sk = tok ? p.sa_k : p.sw_k;
        const int entries = tok ? r.rows : nb, first = tok ? 64 * q : 64 * (q - T::SC_A);
        L.rs[i] = buffer_desc(base, (uint32_t)(((entries - 1) * st + (kb - 1) * sk) * 4 + 4));
        L.vs[i] = first + lane < entries ? (uint32_t)((first + lane) * st * 4) : OOB;
        L.step[i] = (uint32_t)(sk * 4);
        L.s0[i] = 0;
    }
    L.k0 = 0;
    L.k_step = BK;
    L.left = kb;
    L.ktail = p.K % BK;
    L.dw = (uint32_t)(wave * T::WL * 8 * ROWB);
    L.da = (uint32_t)(T::A_OFF + wave * T::AL * 8 * ROWB);
    L.ds = T::SC_OFF + 256u * (uint32_t)wave;
    L.full = wave + (T::SL - 1) * T::WAVES < T::PIECES;
}

// Before the next k-step's loads.  The last k-step of a K that is no multiple of 128 cuts the lanes past K off for good; past the
// last one the descriptors are empty and the uniform offsets 0, so that the loads read zeros.
template <class T>
__device__ __forceinline__ void sload_edge(SLoader<T>& L, int wave, int lane) {
    if (__builtin_expect(L.left == 1 && L.ktail != 0, 0)) {
        const int lrow = lane >> 3;
#pragma unroll
        for (int i = 0; i < T::WL; ++i)
            if (16 * ((lane & 7) ^ T::swz_of_w(8 * (wave * T::WL + i) + lrow)) >= L.ktail) L.vw[i] = OOB;
#pragma unroll
        for (int j = 0; j < T::AL; ++j)
            if (16 * ((lane & 7) ^ swz(8 * (wave * T::AL + j) + lrow)) >= L.ktail) L.va[j] = OOB;
    }
}
template <class T>
__device__ __forceinline__ void sload_end(SLoader<T>& L) {
    const bool live = L.left > 0;
    L.rw[2] = live ? L.rw[2] : 0;
    L.ra[2] = live ? L.ra[2] : 0;
    L.k0 = live ? L.k0 : 0;
    L.k_step = live ? BK : 0;
#pragma unroll
    for (int i = 0; i < T::SL; ++i) {
        L.rs[i][2] = live ? L.rs[i][2] : 0;
        L.s0[i] = live ? L.s0[i] : 0;
        L.step[i] = live ? L.step[i] : 0;
    }
}

// Load instruction i of the k-step into stage `st`.
template <class T>
__device__ __forceinline__ void sload_one(const SLoader<T>& L, uint32_t st, int i) {
    if (i < T::WL) {
        if (T::NT) dma16_at_nt(L.rw, st + L.dw + (uint32_t)(i * 8 * ROWB), L.vw[i], L.k0);
        else dma16_at(L.rw, st + L.dw + (uint32_t)(i * 8 * ROWB), L.vw[i], L.k0);
    } else if (i < T::WL + T::AL) {
        const int j = i - T::WL;
        dma16_at(L.ra, st + L.da + (uint32_t)(j * 8 * ROWB), L.va[j], L.k0);
    } else {
        const int k = i - T::WL - T::AL;
        if (T::EVEN || k < T::SL - 1 || L.full) dma4_at(L.rs[k], st + L.ds + (uint32_t)(k * T::WAVES * 256), L.vs[k], L.s0[k]);
    }
}

template <class T>
__device__ __forceinline__ void sload_next(SLoader<T>& L) {
    --L.left;
    L.k0 += L.k_step;
#pragma unroll
    for (int i = 0; i < T::SL; ++i) L.s0[i] += L.step[i];
}

// All but the youngest N k-steps' loads of this wave have landed.
template <class T, int N>
__device__ __forceinline__ void swait(const SLoader<T>& L) {
    if (T::EVEN || L.full) __builtin_amdgcn_s_waitcnt(vmcnt_imm(T::LOADS * N));
    else __builtin_amdgcn_s_waitcnt(vmcnt_imm((T::LOADS - 1) * N));
    asm volatile("" ::: "memory");
}

// The next place in the ring.
template <class T>
__device__ __forceinline__ uint32_t snext(uint32_t st) { return st == (T::NST - 1) * T::STAGE ? 0u : st + T::STAGE; }

// One k-step on the fragments F (its results go to b): the next one's are read into G; pend and ps are the results and scales of
// the k-step before.  BAR: a barrier first, behind which the next KS k-steps have landed in every wave and the stages of the
// last KS whose fragments are read are free.  Each k-step loads one of those (ring place `ld`), between its MFMAs and its fmas: a
// load holds the wave up for 16 to 30 cycles, and in a burst behind the barrier they held up everything (200 x 5376 x 7168 in
// 128 x 64 tiles: 980 cycles a k-step, most of them 54 loads in a row).
template <class T, bool BAR>
__device__ __forceinline__ void skstep(const uint8_t* lds, uint32_t lds0, uint32_t& rd, uint32_t& ld, SLoader<T>& L,
                                       const BAddr<T>& A, int wave, int lane, v4f (&acc)[T::NI][T::NJ], const SFrags<T>& F, SFrags<T>& G,
                                       const v4f (&pend)[T::NM], v4f (&b)[T::NM], float (&ps)[T::NJ]) {
    wait_lgkm0();                                         // this wave's reads of F have returned
    if (BAR) {
        swait<T, T::NST - 2 * T::KS>(L);
        barrier_nofence();
    }
    rd = snext<T>(rd);
    if (__builtin_expect(L.left <= 1, 0)) {
        sload_edge<T>(L, wave, lane);
        sload_end<T>(L);
    }
    sread<T>(G, lds, rd, A);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < 2 * T::NM; ++u) {
        if (u < T::NM)
            b[u] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(F.w[T::mi(u)], F.t[T::mj(u)], v4f{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
        else
            bfma<T>(acc, pend[u - T::NM], ps[T::mj(u - T::NM)], u - T::NM);
#pragma unroll
        for (int i = u * T::LOADS / (2 * T::NM); i < (u + 1) * T::LOADS / (2 * T::NM); ++i) sload_one<T>(L, lds0 + ld, i);
        __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int j = 0; j < T::NJ; ++j) ps[j] = F.s[j] * F.sw;
    sload_next<T>(L);
    ld = snext<T>(ld);
    __builtin_amdgcn_sched_barrier(0);
}

// The last k-step's results, 24 wait states behind their MFMAs as a dependence.
template <class T>
__device__ __forceinline__ void sdrain(v4f (&acc)[T::NI][T::NJ], v4f (&pend)[T::NM], const float (&ps)[T::NJ]) {
    asm volatile("s_nop 15\n\ts_nop 7" : "+v"(pend[T::NM - 1]));
#pragma unroll
    for (int u = 0; u < T::NM; ++u) {
        asm volatile("" : "+v"(pend[u]));
        bfma<T>(acc, pend[u], ps[T::mj(u)], u);
    }
}

template <class T, bool GROUPED, class Store>
__device__ __forceinline__ void small_kernel(const BlocksParams& p, const uint8_t* lds, int tiles_n, int rt, const Store& store) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int wn = wave % T::WN, wm = wave / T::WN;
    const uint32_t lds0 = lds_addr(lds);
    int tm, tn;
    tile_of((int)blockIdx.x, (int)gridDim.x, rt, tiles_n, 8, tm, tn);
    TileRows r;
    if (GROUPED) {
        if (!locate_rows(p, T::TT, tm, lane, r)) return;
    } else {
        r.e = 0;
        r.row0 = (int64_t)tm * T::TT;
        r.rows = (int)min<int64_t>(T::TT, p.M - r.row0);
    }
    SLoader<T> L;
    sload_set<T>(L, p, r, tn, wave, lane);
    uint32_t rd = 0, ld = 0;
#pragma unroll
    for (int s = 0; s < T::NST - (T::KS - 1); ++s) {
        sload_edge<T>(L, wave, lane);
        sload_end<T>(L);
#pragma unroll
        for (int i = 0; i < T::LOADS; ++i) sload_one<T>(L, lds0 + ld, i);
        sload_next<T>(L);
        ld = snext<T>(ld);
    }
    const BAddr<T> A = baddr<T>(wn, wm, lane);
    v4f acc[T::NI][T::NJ], pa[T::NM], pb[T::NM];
    float ps[T::NJ];
#pragma unroll
    for (int u = 0; u < T::NM; ++u) acc[T::mi(u)][T::mj(u)] = pa[u] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < T::NJ; ++j) ps[j] = 0.f;
    swait<T, T::NST - T::KS>(L);
    barrier_nofence();
    SFrags<T> F, G;
    sread<T>(F, lds, 0, A);
    // in pairs: an odd count takes one more k-step, of zeros, which adds +0
    for (int left = (p.K + 2 * BK - 1) / (2 * BK); left > 0; --left) {
        skstep<T, true>(lds, lds0, rd, ld, L, A, wave, lane, acc, F, G, pa, pb, ps);
        skstep<T, T::KS == 1>(lds, lds0, rd, ld, L, A, wave, lane, acc, G, F, pb, pa, ps);
    }
    sdrain<T>(acc, pa, ps);
    wait_vm0();                                           // the loads behind the last k-step have landed before the exit
    store(p, r, tn, wn, wm, lane, acc);
}

constexpr int64_t kMaxSpan = 0x7fff0000LL;                // byte offsets within a tile are 32-bit

inline int check(const BlocksParams& p, const char* who, int out_dtype, int64_t N, int64_t K, int64_t E) {
    H3_REQUIRE(p.M >= 0 && N >= 0 && K >= 0 && E >= 0, "%s: negative size", who);
    H3_REQUIRE(out_dtype == H3FP8_DT_BF16 || out_dtype == H3FP8_DT_FP16, "%s: bad out_dtype %d", who, out_dtype);
    H3_REQUIRE(K % 16 == 0 && N % 16 == 0, "%s: K=%lld and N=%lld must be multiples of 16", who, (long long)K, (long long)N);
    H3_REQUIRE(p.M <= 0x7fffffff && N <= 0x7fffffff && K <= 0x7fffffff && E <= 0x7fffffff, "%s: size too large", who);
    if (p.M == 0 || N == 0 || E == 0) return H3FP8_OK;
    H3_REQUIRE(K > 0, "%s: K must be positive (got 0)", who);
    H3_REQUIRE(p.a && p.w && p.sa && p.sw && p.y, "%s: null pointer", who);
    H3_REQUIRE(p.lda >= K && p.lda % 16 == 0 && p.ldw >= K && p.ldw % 16 == 0 && p.w_e % 16 == 0,
               "%s: the row strides of a and w must be >= K and multiples of 16, w's expert stride too", who);
    H3_REQUIRE(p.ldy >= N && p.ldy % 8 == 0, "%s: the row stride of y must be >= N and a multiple of 8", who);
    H3_REQUIRE(((uintptr_t)p.a & 15) == 0 && ((uintptr_t)p.w & 15) == 0 && ((uintptr_t)p.y & 15) == 0,
               "%s: a, w and y must be 16-byte aligned", who);
    H3_REQUIRE(((uintptr_t)p.sa & 3) == 0 && ((uintptr_t)p.sw & 3) == 0 && ((uintptr_t)p.bias & 1) == 0,
               "%s: misaligned scales or bias", who);
    H3_REQUIRE(p.sa_m >= 0 && p.sa_k >= 0 && p.sw_e >= 0 && p.sw_n >= 0 && p.sw_k >= 0 && p.w_e >= 0, "%s: negative stride", who);
    const int64_t kb = (K + 127) / 128;
    // tiles are addressed from their own base: 256 rows of each operand and all of their scales within 2 GiB
    H3_REQUIRE(256 * p.lda + K <= kMaxSpan && 256 * p.ldw + K <= kMaxSpan && 256 * p.ldy * 2 + 2 * N <= kMaxSpan &&
                   (256 * p.sa_m + kb * p.sa_k) * 4 <= kMaxSpan && (2 * p.sw_n + kb * p.sw_k) * 4 <= kMaxSpan,
               "%s: a stride is too large", who);
    return H3FP8_OK;
}

// Row tiles of TT rows at most: every expert adds at most one that is not full.
inline int64_t row_tiles(const BlocksParams& p, int TT) {
    const int64_t full = (p.M + TT - 1) / TT;
    return p.offsets ? std::min<int64_t>(p.M, p.M / TT + p.E) : full;
}

// ---- which form runs --------------------------------------------------------------------------------------------------
//
// Small tiles, channels x tokens (one-shot workgroups), in ascending order of their area: the calls that take them (kernels are
// compiled for those only) and how many of them a CU holds.
constexpr int DENSE = 1, EXPERTS = 2;
#define H3_SMALL_FORMS(X)                                                                                              \
    X(F_32x16, DENSE | EXPERTS, 3, 2, 1, 1, 1, 6, 1)                                                                   \
    X(F_32x32, DENSE, 2, 2, 1, 1, 2, 8, 2)                                                                             \
    X(F_64x32, EXPERTS, 2, 2, 1, 2, 2, 5, 1)                                                                           \
    X(F_32x64, DENSE, 2, 2, 2, 1, 2, 6, 2)                                                                             \
    X(F_64x64, EXPERTS, 1, 2, 2, 2, 2, 4, 1)                                                                           \
    X(F_128x64, DENSE, 1, 4, 2, 2, 2, 6, 2)                                                                            \
    X(F_128x64_PAIR, DENSE, 2, 2, 2, 4, 2, 3, 1)
enum Form {
#define X(id, ...) id,
    H3_SMALL_FORMS(X)
#undef X
    F_256x128, F_256x256
};
struct FormDims { int calls, per_cu, tw, tt; };
constexpr FormDims kForms[] = {
#define X(id, calls, per, WN, WM, NI, NJ, NST, KS) {calls, per, 16 * NI * WN, 16 * NJ * WM},
    H3_SMALL_FORMS(X)
#undef X
    {DENSE | EXPERTS, 1, 256, 128}, {DENSE | EXPERTS, 1, 256, 256}};

inline int64_t tiles_of(int form, int64_t row_tiles, int64_t N) { return row_tiles * ((N + kForms[form].tw - 1) / kForms[form].tw); }

// The large tiles by rounds over the CUs: one of 256 x 128 tiles takes 0.66 to 0.69 of the time of one of 256 x 256 (M x 5376 x
// 7168 in 256 x 128 / 256 x 256, us: 1024 rows 55 / 75 in one round each, 2048 103 / 80 in 2 and 1, 4096 170 / 167 in 3 and 2).
inline int large_form(int64_t rows128, int64_t rows256, int64_t N, int G) {
    const int64_t r128 = (tiles_of(F_256x128, rows128, N) + G - 1) / G, r256 = (tiles_of(F_256x256, rows256, N) + G - 1) / G;
    return 16 * r256 < 11 * r128 ? F_256x256 : F_256x128;
}

// One problem: the smallest form whose tiles the CUs hold at once; with 16 tokens or fewer always 32 x 16 (the weights' bytes
// count).  Past that the large tiles.  64 x 32 and 64 x 64 are compiled for experts (below).  Measured on 256 CUs, the weights in
// turn from copies that together exceed the last-level cache, us, [taken]; 64 x 32 and 64 x 64 from a build that had them:
//   M x N x K           32 x 16  32 x 32  64 x 32  32 x 64  64 x 64  128 x 64  in pairs  256 x 128  256 x 256
//   32 x 5376 x 7168     [17.3]     13.6     17.5     17.0     20.5      26.6      31.3       46.5       62.8
//   64 x 5376 x 7168     [21.5]     21.0     17.4     18.1     21.7      30.1      32.7       49.6       63.3
//   128 x 5376 x 7168      36.6     30.0     27.6   [27.9]     21.3      29.2      32.1       56.3       65.0
//   200 x 5376 x 7168         -        -        -     34.3     29.3    [25.4]      31.4       52.7       75.9
//   512 x 5376 x 7168         -        -        -     65.3     49.1      53.6    [47.0]       54.1       75.9
//   1024 x 5376 x 7168        -        -        -        -        -      75.8      67.8     [54.3]       77.0
//   2048 x 5376 x 7168        -        -        -        -        -     150.6     119.0      107.9     [78.9]
//   32 x 21 504 x 5376     38.0     34.0     26.3     32.0     27.0    [26.8]      29.0       40.5       53.9
//   128 x 21 504 x 5376    98.9     71.0     61.7     59.0     45.6      47.4    [43.7]       48.6       55.5
//   256 x 21 504 x 5376       -        -        -     94.8     75.0      65.8      59.2     [48.1]       62.4
// So it takes the best form or one within a few per cent of it from 200 rows on and on wide outputs, but not at 17 to 128 rows of
// 5376 channels: workgroups that share a CU share its load path too, which this rule does not count.
inline int dense_form(int64_t M, int64_t N, int G) {
    if (M <= 16) return F_32x16;
    for (int f = 0; f < F_256x128; ++f)
        if ((kForms[f].calls & DENSE) && tiles_of(f, (M + kForms[f].tt - 1) / kForms[f].tt, N) <= (int64_t)kForms[f].per_cu * G) return f;
    return large_form((M + 127) / 128, (M + 255) / 256, N, G);
}

// By expert, from the mean rows per expert, since the host does not know the counts (each expert's last tile taken as half
// full).  While an expert has few rows the time is its weights', and a tile should hold all of its rows.  4096 x 4096 weights,
// 32 experts, us in 32 x 16 / 64 x 32 / 64 x 64 / 256 x 128 tiles: 4 rows each 101 / 112 / 121 / 122, 8: 120 / 111 / 117 / 122,
// 16: 149 / 131 / 122 / 124, 24: 201 / 145 / 133 / 124, 48: 277 / 203 / 162 / 128; 16 experts in 64 x 64 / 256 x 128 / 256 x
// 256: 32 rows 76 / 70 / 73, 128: 129 / 76 / 78, 200: 167 / 88 / 84, 384: - / 130 / 123.
inline int grouped_form(int64_t M, int64_t N, int64_t E, int G) {
    if (M <= 5 * E) return F_32x16;
    if (M <= 12 * E) return F_64x32;
    if (M <= 20 * E) return F_64x64;
    return large_form(M / 128 + (E + 1) / 2, M / 256 + (E + 1) / 2, N, G);
}

// The non-temporal hint on the weight loads that stream them once: for more than 64 MiB of weights, of which a next call finds
// little in the last-level cache (256 MiB) whatever this one leaves there.  With / without it, us: 1 x 21 504 x 5376 19.6 / 21.7;
// by expert 64 rows x 32 x 2048 x 4096 46.5 / 49.7, 256 x 32 x 4096 x 4096 106 / 116 (64 x 32); but weights that are still in
// that cache come slower: two sets of 8 x 4096 x 4096 in turn, 20 rows, 25.9 / 21.7.
inline bool streams(const BlocksParams& p) { return (int64_t)p.N * p.K * std::min<int64_t>(p.E, p.M) > (64LL << 20); }

// ... and of the large tiles, by expert, while one row tile holds a mean expert's rows.  16 experts of 4096 x 4096: 64 rows each 67
// / 73, 128: 77 / 80, 256: 85 / 92; but with two row tiles that share the weights in L2, 384: 137 / 127, and 32 768 rows
// over 32 experts 585 / 557.
inline bool once(const BlocksParams& p, int64_t rows) { return p.M <= rows * p.E; }

inline int form_for(int64_t M, int64_t N, int64_t E, bool grouped, int G) { return grouped ? grouped_form(M, N, E, G) : dense_form(M, N, G); }

}  // namespace h3b
