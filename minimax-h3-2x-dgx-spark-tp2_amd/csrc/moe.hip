// A whole layer of block-scaled FP8 experts for a few tokens (gfx950), in two or three kernels.
//
//   y[t] = residual[t] + sum_j weight[t, j] * W2[e] h,  h = silu(g) * u,  g | u = W1[e] x[t],  e = experts[t, j]
//
// Every weight is read once, the tokens of an expert together, and the floor is the weights' bytes.  The tokens stay as
// they are (bf16 / fp16), unlike in the path of many tokens, whose products quantise them: the weights' e4m3 codes are
// widened in registers (bf16 and fp16 hold them exactly), MFMAs 16x16x32 make the sum of one block of 128 from a zero
// accumulator, the weight rows as the A operand and the tokens as B, and one fma per element adds it with the block's
// scale in fp32.  Kernel 1 leaves h times the pair's weight as two bf16 numbers, the value and what its rounding left (16 bits
// in all), so that the layer has one rounding to the output's type and none that counts before.
//
// Up to 8 or 16 pairs (a token or a few) what counts is the latency up to the first bytes: kernels that find their rows by ballots.
// Past that a workgroup's waves share the tokens' values through LDS, and its items follow each other without a pause.
//
// us of a layer, and the weights' bytes over that: 4 experts of 4096 x 2048 (1 token) 24, 4.3 TB/s; 2 of 1536 x 2304 (1 token)
// 13.5, 1.6; 12 of 1200 x 1040 (37 tokens, fp16) 24, 1.9; 23 to 28 of 4096 x 2048 (16 tokens) 113 to 136, 5.2; 32 of them (128
// tokens, 1024 pairs) 186 to 215, 3.7 to 4.3.  A copy of 2 GiB runs at 5.0 TB/s, read and written together.
#include <algorithm>
#include <type_traits>

#include "gemm_core.h"

namespace {

using namespace h3g;

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8hf __attribute__((ext_vector_type(8)));

constexpr int MAX_T = 128, MAX_K = 16, MAX_E = 512;

struct MoeParams {
    const void* x;              // [T, H], row stride ldx
    int64_t ldx;
    const uint8_t* w1;          // [E, 2F, H]
    const float* s1;            // [E, ceil(2F / 128), ceil(H / 128)], strides s1_e, s1_n, s1_k
    const uint8_t* w2;          // [E, H, F]
    const float* s2;
    int64_t w1_e, ld1, w2_e, ld2;
    int64_t s1_e, s1_n, s1_k, s2_e, s2_n, s2_k;
    const float* weights;       // [T, k]
    const int* experts;         // [T, k]
    const int* offsets;         // [E + 1]
    const int* order;           // [T k]
    const void* residual;       // [T, H] or null
    int64_t ldr;
    uint16_t* y;                // [T, H]
    int64_t ldy;
    char* h;                    // [T k, F] pairs of bf16: 16 values, then what they leave
    float* z;                   // [T k, H]: the pairs' results (more rows per expert)
    int T, E, k, H, F;
    int fp16;
};

__device__ __forceinline__ int offset_at(const MoeParams& p, int e) {
    return min(max(p.offsets[e], 0), p.T * p.k);          // whatever the offsets hold, no pair outside [0, T k) is read
}

// Eight e4m3 codes as an MFMA operand.
__device__ __forceinline__ v8bf widen_bf16(uint32_t lo, uint32_t hi) {
    typedef __bf16 v2 __attribute__((ext_vector_type(2)));
    const v2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
    const v2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
    return v8bf{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ __forceinline__ v8hf widen_fp16(uint32_t lo, uint32_t hi) {
    typedef _Float16 v2 __attribute__((ext_vector_type(2)));
    const v2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
    const v2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
    return v8hf{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// c (FIRST: zero) + the product of 32 of k.  In asm, so that c stays where it is: the compiler moves the sums of a chain between
// registers, and takes those they leave for other values sooner than 24 wait states behind the MFMA that wrote them.  A vector
// instruction's result goes into an MFMA two wait states behind it.
template <bool FP16, bool FIRST>
__device__ __forceinline__ void mfma(v4f& c, uint32_t w_lo, uint32_t w_hi, v4u b) {
    if constexpr (FP16) {
        const v8hf a = widen_fp16(w_lo, w_hi);
        if constexpr (FIRST) asm volatile("s_nop 1\n\tv_mfma_f32_16x16x32_f16 %0, %1, %2, 0" : "=&v"(c) : "v"(a), "v"(b));
        else asm volatile("s_nop 1\n\tv_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "v"(b));
    } else {
        const v8bf a = widen_bf16(w_lo, w_hi);
        if constexpr (FIRST) asm volatile("s_nop 1\n\tv_mfma_f32_16x16x32_bf16 %0, %1, %2, 0" : "=&v"(c) : "v"(a), "v"(b));
        else asm volatile("s_nop 1\n\tv_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "v"(b));
    }
}

// The blocks' sums are read 24 wait states behind the last MFMA, and after this.
template <int A, int B>
__device__ __forceinline__ void sums_ready(v4f (&b)[A][B]) {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 15\n\ts_nop 7" : "+v"(b[A - 1][B - 1]));
#pragma unroll
    for (int i = 0; i < A; ++i)
#pragma unroll
        for (int j = 0; j < B; ++j) asm volatile("" : "+v"(b[i][j]));
}

__device__ __forceinline__ int wave_prefix(int v) {       // inclusive
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
    return v;
}


// ---- the routing, in LDS ------------------------------------------------------------------------------------------------
//
// All that a workgroup needs of the routing is loaded at once, and looked up from then on: one trip to memory before the first
// weights can be asked for instead of one per step (offsets, order, experts).

// An expert that has pairs: sorted rows r0 .. r0 + rows - 1, in blocks; `start`: its first item (see Item).
struct Expert { uint16_t e, r0, rows, none; int start; };

struct Routed {
    int* count;                                           // of experts that have pairs, of the workgroup's XCD's items
    Expert* list;
    float* weight;                                        // [P] of a sorted row: of all its token's choices of its expert (the
                                                          // second of two equal ones has the same, and is not read)
    uint16_t* pair;                                       // [P] of a sorted row
};

constexpr size_t routed_bytes(int E, int P, bool weights) {
    return 16 + (size_t)(E < P ? E : P) * sizeof(Expert) + (size_t)P * (weights ? 6 : 2);
}
constexpr int TEMP_BYTES = 8 * MAX_T * MAX_K;             // what load_routing needs besides, before the first stage is loaded

// The items of a launch are a block of up to ROWS rows of an expert and a tile of its output channels.  Blocks of one expert read
// the same weights, so they run at the same time on the same XCD, whose L2 then has them: tile t of the s-th expert is XCD
// (s tiles + t) % 8's (workgroups are dealt over the XCDs in turn), and a XCD's items are ordered by expert, tile, block.
struct Item {
    int e, r0, n, tile;                                   // n = 0: past the last one
};

constexpr int XCDS = 8;

// By all threads, with barriers.  temp: experts and weights of the pairs, while the weights are added up.
template <int ROWS, bool WEIGHTS>
__device__ __forceinline__ Routed load_routing(const MoeParams& p, char* lds, char* temp, int threads, int tiles) {
    const int P = p.T * p.k, lane = threadIdx.x & 63, cap = min(p.E, P), xcd = (int)blockIdx.x % XCDS;
    Routed r;
    r.count = reinterpret_cast<int*>(lds);
    r.list = reinterpret_cast<Expert*>(r.count + 4);
    r.weight = reinterpret_cast<float*>(r.list + cap);
    r.pair = reinterpret_cast<uint16_t*>(r.weight + (WEIGHTS ? P : 0));
    int* experts_of = reinterpret_cast<int*>(temp);
    float* weights_of = reinterpret_cast<float*>(experts_of + P);
    for (int i = threadIdx.x; i < P; i += threads) {
        const int o = p.order[i];
        if (WEIGHTS) {
            const int e = p.experts[i];
            const float w = p.weights[i];
            experts_of[i] = e;
            weights_of[i] = w;
        }
        r.pair[i] = (uint16_t)min(max(o, 0), P - 1);      // whatever it holds, no row outside the tokens is read
    }
    if (threadIdx.x < 64) {
        int experts = 0, items = 0;
        for (int e0 = 0; e0 < p.E; e0 += 64) {
            int lo = 0, hi = 0;
            if (e0 + lane < p.E) lo = offset_at(p, e0 + lane), hi = offset_at(p, e0 + lane + 1);
            const int n = max(hi - lo, 0);
            const uint64_t has = __ballot(n > 0);
            const int s = experts + __popcll(has & ((1ull << lane) - 1));
            const int t0 = (xcd + XCDS - s * tiles % XCDS) % XCDS, mine = n > 0 && t0 < tiles ? (tiles - t0 + XCDS - 1) / XCDS : 0;
            const int m = mine * ((n + ROWS - 1) / ROWS), at = items + wave_prefix(m) - m;
            // (offsets that are not ascending may name more experts than there are pairs)
            if (n > 0 && s < cap) r.list[s] = Expert{(uint16_t)(e0 + lane), (uint16_t)lo, (uint16_t)n, 0, at};
            experts += __popcll(has);
            items = __builtin_amdgcn_readlane(at + m, 63);
        }
        if (lane == 0) r.count[0] = min(experts, cap), r.count[1] = items;
    }
    __syncthreads();
    if (WEIGHTS) {
        for (int i = threadIdx.x; i < P; i += threads) {
            const int pair = r.pair[i], e = experts_of[pair];
            float w = 0.0f;
            for (int j = 0, q = pair / p.k * p.k; j < p.k; ++j) w += experts_of[q + j] == e ? weights_of[q + j] : 0.0f;
            r.weight[i] = w;
        }
        __syncthreads();
    }
    return r;
}

// Item i of the workgroup's XCD, by a wave; all scalars.
template <int ROWS>
__device__ __forceinline__ Item item_at(const Routed& r, int experts, int items, int i, int tiles, int lane) {
    if (i >= items) return Item{0, 0, 0, 0};
    int s = -1;
    for (int s0 = 0; s0 < experts; s0 += 64)              // the last expert that starts no later
        s += __popcll(__ballot(s0 + lane < experts && r.list[min(s0 + lane, experts - 1)].start <= i));
    // experts without a tile here start where the next one does, and are not the last
    const Expert& x = r.list[s];
    const int e = __builtin_amdgcn_readfirstlane(x.e), r0 = __builtin_amdgcn_readfirstlane(x.r0);
    const int rows = __builtin_amdgcn_readfirstlane(x.rows), k = i - __builtin_amdgcn_readfirstlane(x.start);
    const int nb = (rows + ROWS - 1) / ROWS, t = k / nb, b = k - t * nb;
    const int t0 = ((int)blockIdx.x % XCDS + XCDS - s * tiles % XCDS) % XCDS;
    return Item{e, r0 + b * ROWS, min(ROWS, rows - b * ROWS), t0 + XCDS * t};
}

// silu(g) u w of 4 consecutive channels f .. f + 3 of a pair, as two bf16 numbers each.
__device__ __forceinline__ void store_h(const MoeParams& p, int pair, int f, float weight, const v4f& gate, const v4f& up) {
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const float h = times_sigmoid(gate[r], gate[r]) * up[r] * weight;
        hi[r] = bf16_rne(h);
        const float rest = h - bf16_to_f32(hi[r]);
        lo[r] = (hi[r] & 0x7f80u) == 0x7f80u ? 0u : bf16_rne(rest);       // infinite or NaN: nothing is left
    }
    char* at = p.h + (int64_t)pair * p.F * 4 + f / 16 * 64 + f % 16 * 2;
    *reinterpret_cast<uint2*>(at) = uint2{hi[0] | (hi[1] << 16), hi[2] | (hi[3] << 16)};
    *reinterpret_cast<uint2*>(at + 32) = uint2{lo[0] | (lo[1] << 16), lo[2] | (lo[3] << 16)};
}

// The residual's 4 channels n .. n + 3 of a token; zeros without one.
__device__ __forceinline__ uint2 residual_at(const MoeParams& p, int t, int n) {
    return p.residual ? *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(p.residual) + t * p.ldr + n) : uint2{0u, 0u};
}

// 4 consecutive channels of a token, with the residual.
__device__ __forceinline__ void store_y(const MoeParams& p, int t, int n, v4f v, uint2 r) {
    if (p.residual) {
        const uint32_t b[4] = {r.x & 0xffffu, r.x >> 16, r.y & 0xffffu, r.y >> 16};
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] += p.fp16 ? fp16_to_f32(b[q]) : bf16_to_f32(b[q]);
    }
    const uint2 o = p.fp16 ? uint2{fp16_rne(v[0]) | (fp16_rne(v[1]) << 16), fp16_rne(v[2]) | (fp16_rne(v[3]) << 16)}
                           : uint2{cvt_bf16x2(v[0], v[1]), cvt_bf16x2(v[2], v[3])};
    *reinterpret_cast<uint2*>(p.y + t * p.ldy + n) = o;
}

// ---- a token or a few -----------------------------------------------------------------------------------------------------
//
// What counts is how soon the weights' bytes are asked for.  The pairs, at most 16, are a lane each: the experts that have
// pairs, the pairs of one and their tokens come out of ballots on one load of `experts`, by every wave for itself.

// LDS place of 16-byte chunk i of weight row r (128 bytes): i ^ this.
__device__ __forceinline__ int weight_swz(int r) { return (r & 2) | ((r >> 1) & 4); }

// LDS place of 16-byte chunk i of row r: the 16 lanes that are served together (0-3, 12-15 and 20-27; 4-11, 16-19 and 28-31) meet 16
// places.  Kernel 1: lane group g reads chunks 2 g + ..; kernel 2: 4 g + ..
template <bool UP>
__device__ __forceinline__ int chunk_at(int r, int i) {
    const int c = r & 15;
    return i ^ (UP ? c : (((c >> 2) ^ (c >> 3)) & 1) | ((c & 3) << 1) | (c & 8));
}

// Each token's first pair among the pairs `same` (of one expert): the second of two equal choices is not a row of its own.
__device__ __forceinline__ uint64_t first_pairs(uint64_t same, int lane, int k) {
    const int t = lane / k;
    return same & __ballot(((same >> (t * k)) & ((1ull << (lane - t * k)) - 1)) == 0);
}

// A wave has two units under way, in LDS of its own: weights in whole lines, the values of up to TOKENS tokens (more columns of the
// MFMAs repeat them), scales.  (Straight into registers, a lane 16 bytes of its row, the memory pipe took a clock per lane: 1 token,
// 4 experts of 4096 x 2048 29 us in place of 24, 8 of 1536 x 2304 42 in place of 28.)
template <bool UP, int TOKENS>
struct Few {
    static constexpr int WAVES = UP ? 8 : TOKENS > 2 ? 8 : 16;
    static constexpr int ROW = UP ? 256 : 512, LPR = ROW / 16, RPI = 64 / LPR;        // bytes of a token's block; lanes; tokens of an instruction
    static constexpr int DW = UP ? 4 : 2, DX = TOKENS > RPI ? TOKENS / RPI : 1;
    static constexpr int X = DW * 1024, S = X + TOKENS * ROW, STAGE = S + 16, LDS = 2 * STAGE * WAVES;
    static constexpr int LOADS = DW + DX + 1;
    static_assert(LDS >= WAVES * 64 * 16 * (UP ? 2 : 1), "the waves' sums take the place of the stages");
};

// All but the last N loads have landed; LDS is read behind this.
template <int N>
__device__ __forceinline__ void stage_landed() {
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(N));
    asm volatile("" ::: "memory");
}

// Kernel 1: a workgroup takes 16 gate rows and the up rows that belong to them, of one expert; its 8 waves share out the blocks of K
// and join through LDS.
template <bool FP16, int TOKENS>
__global__ void __launch_bounds__((Few<true, TOKENS>::WAVES * 64)) moe_few_up_kernel(MoeParams p, int tiles) {
    using C = Few<true, TOKENS>;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[C::LDS];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int c = lane & 15, g = lane >> 4, P = p.T * p.k;
    const int mine = lane < P ? p.experts[lane] : -1;
    const float weight = lane < P ? p.weights[lane] : 0.0f;
    int slot = (int)blockIdx.x / tiles;
    const int tile = (int)blockIdx.x - slot * tiles, f0 = tile * 16;
    uint64_t left = __ballot(mine >= 0 && mine < p.E), same = 0;
    int e = 0;
    for (; left; --slot) {
        e = __builtin_amdgcn_readlane(mine, __builtin_ctzll(left));
        same = __ballot(mine == e);
        if (slot == 0) break;
        left &= ~same;
    }
    if (!left) return;
    const uint64_t rows = first_pairs(same, lane, p.k);
    const int n = __popcll(rows);
    // column c: the c-th of the rows
    const int at = (rows >> lane) & 1 ? __popcll(rows & ((1ull << lane) - 1)) : 63;
    const int pair = __builtin_amdgcn_ds_permute(4 * at, lane), col = __shfl(pair, c, 64);
    const int kb = (p.H + BK - 1) / BK;
    const uint8_t* w0 = p.w1 + e * p.w1_e + f0 * p.ld1;
    const uint32_t bytes = (uint32_t)(15 * p.ld1 + p.H), row_bytes = (uint32_t)p.H * 2u;
    const v4u qg = buffer_desc(w0, bytes), qu = buffer_desc(w0 + p.F * p.ld1, bytes), qs = buffer_desc(p.s1, 0x7fffffffu);
    const v4u qx = buffer_desc(p.x, (uint32_t)(((p.T - 1) * p.ldx + p.H) * 2));
    uint32_t cw[2], vw[2], cx[C::DX], vx[C::DX];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = 8 * i + (lane >> 3);
        cw[i] = 16u * (uint32_t)((lane & 7) ^ weight_swz(r));
        vw[i] = (uint32_t)(r * p.ld1) + cw[i];
    }
#pragma unroll
    for (int i = 0; i < C::DX; ++i) {
        const int r = C::RPI * i + lane / C::LPR, token = __shfl(pair, r, 64) / p.k;
        cx[i] = 16u * (uint32_t)chunk_at<true>(r, lane % C::LPR);
        vx[i] = r < n ? (uint32_t)token * (uint32_t)(p.ldx * 2) + cx[i] : OOB;
    }
    const uint32_t sv = (uint32_t)(e * p.s1_e + (lane & 1 ? p.F + f0 : f0) / BK * p.s1_n) * 4u;
    const uint8_t* own = lds + wave * 2 * C::STAGE;
    const uint32_t own0 = (uint32_t)__builtin_amdgcn_readfirstlane((int)lds_addr(own));
    const int turn = (3 * e + 5 * tile) % kb;
    // always the same loads, past the last block of nothing, so that the count of those under way is known
    auto load = [&](int d, int b) {
        const int blk = b < kb ? (b + turn < kb ? b + turn : b + turn - kb) : 0;
        const uint32_t k0 = (uint32_t)(blk * BK), left = b < kb ? (uint32_t)p.H - k0 : 0u, at0 = own0 + (uint32_t)(d * C::STAGE);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            dma16_at(i < 2 ? qg : qu, __builtin_amdgcn_readfirstlane(at0 + 1024u * i), cw[i & 1] < left ? vw[i & 1] : OOB, __builtin_amdgcn_readfirstlane(k0));
#pragma unroll
        for (int i = 0; i < C::DX; ++i)
            if (C::RPI * (i + 1) <= TOKENS || lane < TOKENS * C::LPR)
                dma16(qx, __builtin_amdgcn_readfirstlane(at0 + C::X + 1024u * i),
                      b < kb && vx[i] != OOB && 2 * k0 + cx[i] < row_bytes ? vx[i] + 2 * k0 : OOB);
        if (lane < 2) dma4(qs, __builtin_amdgcn_readfirstlane(at0 + C::S), sv + (uint32_t)(blk * p.s1_k) * 4u);
    };
#pragma unroll
    for (int d = 0; d < 2; ++d) load(d, wave + d * C::WAVES);
    v4f acc[2] = {v4f{0.f, 0.f, 0.f, 0.f}, v4f{0.f, 0.f, 0.f, 0.f}};
    int d = 0;
    for (int b = wave; b < kb; b += C::WAVES, d ^= 1) {
        stage_landed<C::LOADS>();
        const uint8_t *ws = own + d * C::STAGE + c * 128, *xs = own + d * C::STAGE + C::X + (c & (TOKENS - 1)) * C::ROW;
        v4u w[2][2], x[2][2];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
#pragma unroll
            for (int i = 0; i < 2; ++i) w[i][s] = *reinterpret_cast<const v4u*>(ws + 2048 * i + 16 * ((4 * s + g) ^ weight_swz(c)));
#pragma unroll
            for (int q = 0; q < 2; ++q) x[s][q] = *reinterpret_cast<const v4u*>(xs + 16 * chunk_at<true>(c & (TOKENS - 1), 8 * s + 2 * g + q));
        }
        const float sg = *reinterpret_cast<const float*>(own + d * C::STAGE + C::S), su = *reinterpret_cast<const float*>(own + d * C::STAGE + C::S + 4);
        wait_lgkm0();
        __builtin_amdgcn_sched_barrier(0);
        load(d, b + 2 * C::WAVES);
        v4f sum[2][1];
#pragma unroll
        for (int q = 0; q < 4; ++q)                       // 32 of the block's k each
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const v4u& a = w[i][q >> 1];
                if (q == 0) mfma<FP16, true>(sum[i][0], a[0], a[1], x[0][0]);
                else mfma<FP16, false>(sum[i][0], a[2 * (q & 1)], a[2 * (q & 1) + 1], x[q >> 1][q & 1]);
            }
        sums_ready(sum);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            acc[0][r] = __builtin_fmaf(sum[0][0][r], sg, acc[0][r]);
            acc[1][r] = __builtin_fmaf(sum[1][0][r], su, acc[1][r]);
        }
    }
    wait_vm0();                                           // the loads behind the last unit
    __syncthreads();
    v4f* part = reinterpret_cast<v4f*>(lds);              // [wave][gate, up][lane]
#pragma unroll
    for (int i = 0; i < 2; ++i) part[(wave * 2 + i) * 64 + lane] = acc[i];
    __syncthreads();
    if (wave != 0) return;
    v4f gate = part[lane], up = part[64 + lane];
#pragma unroll
    for (int v = 1; v < C::WAVES; ++v) {
        gate += part[2 * v * 64 + lane];
        up += part[(2 * v + 1) * 64 + lane];
    }
    float sum = 0.0f;                                     // of all the token's choices of this expert
    for (uint64_t m = same; m; m &= m - 1) {
        const int q = __builtin_ctzll(m);
        const float wq = u2f(__builtin_amdgcn_readlane((int)f2u(weight), q));
        sum += q / p.k == col / p.k ? wq : 0.0f;
    }
    if (c < n) store_h(p, col, f0 + 4 * g, sum, gate, up);
}

// Kernel 2: a workgroup takes 16 channels for all experts; its waves share out the units, the blocks of F of every expert that has
// pairs.  Column c of the MFMAs is token c, zero where it is not the expert's, so that the accumulators run over all experts.
template <int TOKENS>
__global__ void __launch_bounds__((Few<false, TOKENS>::WAVES * 64)) moe_few_down_kernel(MoeParams p) {
    using C = Few<false, TOKENS>;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[C::LDS];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int c = lane & 15, g = lane >> 4, P = p.T * p.k, n0 = (int)blockIdx.x * 16;
    const int mine = lane < P ? p.experts[lane] : -1;
    const uint2 residual = wave == 0 && c < p.T ? residual_at(p, c, n0 + 4 * g) : uint2{0u, 0u};      // on its way from here on
    const uint64_t all = __ballot(mine >= 0 && mine < p.E), choices = (1ull << p.k) - 1;
    const int fb = (p.F + BK - 1) / BK;
    const uint32_t row_bytes = (uint32_t)p.F * 4u;
    const v4u qh = buffer_desc(p.h, (uint32_t)P * row_bytes), qs = buffer_desc(p.s2, 0x7fffffffu);
    const uint32_t wbytes = (uint32_t)(15 * p.ld2 + p.F);
    const uint8_t* w0 = p.w2 + n0 * p.ld2;
    const uint32_t s0 = (uint32_t)(n0 / BK * p.s2_n) * 4u;
    uint32_t cw[2], vw[2], cx[C::DX];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = 8 * i + (lane >> 3);
        cw[i] = 16u * (uint32_t)((lane & 7) ^ weight_swz(r));
        vw[i] = (uint32_t)(r * p.ld2) + cw[i];
    }
#pragma unroll
    for (int i = 0; i < C::DX; ++i) cx[i] = 16u * (uint32_t)chunk_at<false>(C::RPI * i + lane / C::LPR, lane % C::LPR);
    const uint8_t* own = lds + wave * 2 * C::STAGE;
    const uint32_t own0 = (uint32_t)__builtin_amdgcn_readfirstlane((int)lds_addr(own));
    // the units of a wave: block b of the expert at hand, whose pairs are the first of `left`
    struct Unit { uint64_t left, same; int e, b; };
    auto settle = [&](Unit& u) {                          // ... to where b is one of the expert's blocks, or nothing is left
        for (;;) {
            if (u.left) {
                u.e = __builtin_amdgcn_readlane(mine, __builtin_ctzll(u.left));
                u.same = __ballot(mine == u.e);
            }
            if (!u.left || u.b < fb) return;
            u.b -= fb;
            u.left &= ~u.same;
        }
    };
    Unit next{all, 0, 0, wave}, now = next;
    settle(next);
    now = next;
    auto step = [&](Unit& u) { u.b += C::WAVES; settle(u); };
    // always the same loads, past the last unit of nothing, so that the count of those under way is known
    auto load = [&](int d) {
        const bool live = next.left != 0;
        const int b = live ? next.b : 0, e = live ? next.e : 0;
        const uint32_t k0 = (uint32_t)(b * BK), left = live ? (uint32_t)p.F - k0 : 0u, at0 = own0 + (uint32_t)(d * C::STAGE);
        const v4u qw = buffer_desc(w0 + e * p.w2_e, live ? wbytes : 0u);
#pragma unroll
        for (int i = 0; i < 2; ++i)
            dma16_at(qw, __builtin_amdgcn_readfirstlane(at0 + 1024u * i), cw[i] < left ? vw[i] : OOB, __builtin_amdgcn_readfirstlane(k0));
#pragma unroll
        for (int i = 0; i < C::DX; ++i) {
            const int t = C::RPI * i + lane / C::LPR;
            const uint64_t pairs = live && t < p.T ? (next.same >> (t * p.k)) & choices : 0;
            dma16(qh, __builtin_amdgcn_readfirstlane(at0 + C::X + 1024u * i),
                  pairs && 4 * k0 + cx[i] < row_bytes ? (uint32_t)(t * p.k + __builtin_ctzll(pairs)) * row_bytes + 4 * k0 + cx[i] : OOB);
        }
        if (lane == 0) dma4(qs, __builtin_amdgcn_readfirstlane(at0 + C::S), (uint32_t)(e * p.s2_e + b * p.s2_k) * 4u + s0);
        step(next);
    };
    v4f acc = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int d = 0; d < 2; ++d) load(d);
    for (int d = 0; now.left; step(now), d ^= 1) {
        stage_landed<C::LOADS>();
        const uint8_t *ws = own + d * C::STAGE + c * 128, *xs = own + d * C::STAGE + C::X + (c & (TOKENS - 1)) * C::ROW;
        v4u w[2], h[2][4];                                // h: 16 values, what they leave
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            w[s] = *reinterpret_cast<const v4u*>(ws + 16 * ((4 * s + g) ^ weight_swz(c)));
#pragma unroll
            for (int q = 0; q < 4; ++q) h[s][q] = *reinterpret_cast<const v4u*>(xs + 16 * chunk_at<false>(c & (TOKENS - 1), 4 * (4 * s + g) + q));
        }
        const float scale = *reinterpret_cast<const float*>(own + d * C::STAGE + C::S);
        const bool has = c < p.T && ((now.same >> (c * p.k)) & choices) != 0;
        wait_lgkm0();
        __builtin_amdgcn_sched_barrier(0);
        load(d);
        v4f sum[1][1];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const uint32_t lo = w[q >> 1][2 * (q & 1)], hi = w[q >> 1][2 * (q & 1) + 1];
            if (q == 0) mfma<false, true>(sum[0][0], lo, hi, h[0][0]);
            else mfma<false, false>(sum[0][0], lo, hi, h[q >> 1][q & 1]);
            mfma<false, false>(sum[0][0], lo, hi, h[q >> 1][2 + (q & 1)]);
        }
        sums_ready(sum);
        if (has) {                                        // an expert's NaN is not another token's
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[r] = __builtin_fmaf(sum[0][0][r], scale, acc[r]);
        }
    }
    wait_vm0();                                           // the loads behind the last unit
    __syncthreads();
    v4f* part = reinterpret_cast<v4f*>(lds);              // [wave][lane]
    part[wave * 64 + lane] = acc;
    __syncthreads();
    if (wave != 0) return;
    v4f v = part[lane];
#pragma unroll
    for (int q = 1; q < C::WAVES; ++q) v += part[q * 64 + lane];
    if (c < p.T) store_y(p, c, n0 + 4 * g, v, residual);
}

// ---- more rows per expert -----------------------------------------------------------------------------------------------
//
// With many rows the tokens' values, read again for every 16 weight rows, are more than the weights.  So the waves of a workgroup
// (4 or 8) take neighbouring tiles of weight rows, the whole of K each (no join), and share the tokens' values through LDS: an item
// is a block of up to 16 NT rows of an expert and a tile of 16 output channels (kernel 1, gate and up rows) or 32 (kernel 2) per
// wave; of a few items two groups of 4 waves take alternate units each.  A unit is a block of 128 of K.  Tokens, weights and scales
// come by LDS-DMA, two units ahead of their use in a ring of three, one barrier per unit; the loads of the next item follow those
// of the last without a pause.
//
// What bounded the steps before, us of the layer at 32 experts of 4096 x 2048, 64 / 1024 pairs: a workgroup per item, the weights
// straight into registers, 216 / 709; items one behind the other, the tokens shared through LDS, 145 / 330 (a lane had 16 bytes of its
// row, which the memory pipe takes one by one); weights in whole lines of 128 bytes through LDS, blocks of one expert at the same
// time on one XCD, so that its L2 has the weights, and each item's K from a start of its own, (3 e + 5 tile) units in (rows a
// power of two apart meet the same channels: 7 to 8 %), 115 / 200.  What bounds it now: up to 20 rows per expert the weights' bytes
// (5.2 TB/s; kernel 1 5.8); past that the largest XCD's items, whole rounds of blocks over its 32 CUs.  Blocks of 64 rows make those rounds
// coarser: 110 to 140 us in kernel 1 against 114, 83 to 105 in kernel 2 against 78; two waves to a block of K in kernel 2, so that
// each reads half the tokens' values from LDS, take 79.

// Kernel 2 leaves the pairs' results in fp32, and a third kernel adds up the choices of each token, in their order.

// KS groups of WV waves share out the units of an item; AH: units under way, of each.
template <bool UP, int NT, int CT, int WV, int KS, int AH>
struct Rows {
    static constexpr int RT = UP ? 2 : CT;                // tiles of 16 weight rows of a wave: gate and up; channels
    static constexpr int SC = UP ? 2 : 1;                 // scales of a block, per wave
    static constexpr int OUT = UP ? 16 : 16 * CT;         // output channels of a wave
    static constexpr int ROW = UP ? 256 : 512;            // bytes of a token's block
    static constexpr int STAGES = AH + 1;
    static constexpr int XSTAGE = 16 * NT * ROW, DX = XSTAGE / 1024 / WV;             // of the tokens: bytes, load instructions of a wave
    static constexpr int WSTAGE = RT * 16 * 128, DW = WSTAGE / 1024;                  // of a wave's weights
    static constexpr int W_OFF = STAGES * XSTAGE, S_OFF = W_OFF + STAGES * WV * WSTAGE;      // behind them the waves' scales, 256 bytes a stage
    static constexpr int RING = S_OFF + STAGES * 256, USED = KS * RING, LDS = !UP || USED > TEMP_BYTES ? USED : TEMP_BYTES;
    static constexpr int LOADS = DX + DW + 1;
    static_assert(DX >= 1 && (AH - 1) * LOADS <= 63, "vmcnt range");
    static_assert(RT * NT * 1024 <= WSTAGE, "a wave's sums take the place of a unit's weights");
};

template <bool UP, bool FP16, int NT, int CT, int WV, int KS, int AH>
__global__ void __launch_bounds__(WV * KS * 64) moe_rows_kernel(MoeParams p, int tiles) {
    using C = Rows<UP, NT, CT, WV, KS, AH>;
    constexpr int BLOCK = 16 * NT, DX = C::DX, DW = C::DW, LPR = C::ROW / 16, RPI = 64 / LPR;       // lanes of a token, tokens of an instruction
    extern __shared__ __attribute__((aligned(1024))) uint8_t rows_lds[];
    const int lane = threadIdx.x & 63;
    const int all = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), wave = all % WV, part = all / WV;      // in its group; the group
    const uint8_t* lds = rows_lds + part * C::RING;
    const int c = lane & 15, g = lane >> 4;
    const uint32_t lds0 = (uint32_t)__builtin_amdgcn_readfirstlane((int)lds_addr(lds));
    const Routed R = load_routing<BLOCK, UP>(p, reinterpret_cast<char*>(rows_lds + C::LDS), reinterpret_cast<char*>(rows_lds), WV * KS * 64, tiles);
    const int experts = __builtin_amdgcn_readfirstlane(R.count[0]), items = __builtin_amdgcn_readfirstlane(R.count[1]);
    const int K = UP ? p.H : p.F, N = UP ? p.F : p.H, kb = (K + BK - 1) / BK, units = ((kb + KS - 1) / KS + AH - 1) / AH * AH;
    const int64_t ld = UP ? p.ld1 : p.ld2;
    const uint32_t row_bytes = UP ? (uint32_t)p.H * 2u : (uint32_t)p.F * 4u;
    const v4u qx = buffer_desc(UP ? p.x : p.h, UP ? (uint32_t)(((p.T - 1) * p.ldx + p.H) * 2) : (uint32_t)(p.T * p.k) * (uint32_t)p.F * 4u);
    const v4u qs = buffer_desc(UP ? p.s1 : p.s2, 0x7fffffffu);
    // what the next loads need: the weights' buffers, lane offsets of the tokens' and of the weights' chunks (OOB: nothing), offsets
    // of the scales, the unit
    v4u qw, qu;
    uint32_t vx[DX], vw[UP ? 2 : DW], s_at, s_up;
    int lu = 0, first = 0, blocks = 0;
    // the chunk that a lane's 16 bytes of its token are; of its weight row (8 rows an instruction)
    uint32_t cx[DX], cw[2];
#pragma unroll
    for (int i = 0; i < DX; ++i) cx[i] = 16u * (uint32_t)chunk_at<UP>(RPI * (wave * DX + i) + lane / LPR, lane % LPR);
#pragma unroll
    for (int i = 0; i < 2; ++i) cw[i] = 16u * (uint32_t)((lane & 7) ^ weight_swz(8 * i + (lane >> 3)));
    auto aim = [&](const Item& it) {
        const int n0 = (it.tile * WV + wave) * C::OUT, rows = min(C::OUT, N - n0);
        const bool alive = it.n > 0 && rows > 0;
        const int at = alive ? n0 : 0;
        const uint32_t bytes = alive ? (uint32_t)((rows - 1) * ld + K) : 0u;
        const uint8_t* w = (UP ? p.w1 + it.e * p.w1_e : p.w2 + it.e * p.w2_e) + at * ld;
        qw = buffer_desc(w, bytes);
        if (UP) qu = buffer_desc(w + p.F * ld, bytes);
        blocks = alive ? kb : 0;
#pragma unroll
        for (int i = 0; i < (UP ? 2 : DW); ++i) {
            const int row = 8 * i + (lane >> 3);
            vw[i] = row < rows ? (uint32_t)(row * ld) + cw[i & 1] : OOB;
        }
        s_at = (uint32_t)(UP ? it.e * p.s1_e + at / BK * p.s1_n : it.e * p.s2_e + at / BK * p.s2_n) * 4u;
        s_up = UP ? (uint32_t)(it.e * p.s1_e + (p.F + at) / BK * p.s1_n) * 4u : 0u;
#pragma unroll
        for (int i = 0; i < DX; ++i) {
            const int row = RPI * (wave * DX + i) + lane / LPR;
            uint32_t v = OOB;
            if (row < it.n) v = UP ? (uint32_t)(R.pair[it.r0 + row] / p.k) * (uint32_t)(p.ldx * 2) : (uint32_t)R.pair[it.r0 + row] * row_bytes;
            vx[i] = v;
        }
        lu = 0;
        first = (3 * it.e + 5 * it.tile) % (units * KS);
    };
    // a unit of the next loads into a stage: always the same instructions, past the last block or item of nothing
    auto load = [&](int stage, int u) {
        const int at = KS * u + part + first, blk = at >= units * KS ? at - units * KS : at;
        const uint32_t x0 = (uint32_t)(blk * C::ROW), xs = lds0 + (uint32_t)(stage * C::XSTAGE + wave * DX * 1024);
#pragma unroll
        for (int i = 0; i < DX; ++i)
            dma16(qx, __builtin_amdgcn_readfirstlane(xs + 1024u * i), vx[i] != OOB && x0 + cx[i] < row_bytes ? vx[i] + x0 + cx[i] : OOB);
        const uint32_t k0 = blk < blocks ? (uint32_t)(blk * BK) : 0u, left = blk < blocks ? (uint32_t)K - k0 : 0u;
        const uint32_t ws = lds0 + (uint32_t)(C::W_OFF + (stage * WV + wave) * C::WSTAGE);
#pragma unroll
        for (int i = 0; i < DW; ++i)
            dma16_at(UP && i >= 2 ? qu : qw, __builtin_amdgcn_readfirstlane(ws + 1024u * i), cw[i & 1] < left ? vw[UP ? i & 1 : i] : OOB,
                     __builtin_amdgcn_readfirstlane(k0));
        // the wave's scales (of the gate rows, of the up rows), by lanes of its own; past the last block 0, so that nothing times an
        // infinite one is no NaN
        const uint32_t sb = (uint32_t)(blk * (UP ? p.s1_k : p.s2_k)) * 4u;
        if (lane / C::SC == wave)
            dma4(qs, __builtin_amdgcn_readfirstlane(lds0 + (uint32_t)(C::S_OFF + stage * 256)),
                 blk < blocks ? (UP && (lane & 1) ? s_up : s_at) + sb : OOB);
    };
    v4f acc[C::RT][NT];
    // a block of K on the first J blocks of 16 tokens
    auto block_sums = [&](auto blocks_of_16, int stage) {
        constexpr int J = decltype(blocks_of_16)::value, PARTS = UP ? 1 : 2;
        const uint8_t *xs = lds + stage * C::XSTAGE + c * C::ROW, *ws = lds + C::W_OFF + (stage * WV + wave) * C::WSTAGE + c * 128;
        v4f sum[C::RT][J];
        v4u w[C::RT][2];
        float scale[C::SC];
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int i = 0; i < C::RT; ++i)
                w[i][s] = *reinterpret_cast<const v4u*>(ws + 2048 * i + 16 * ((4 * s + g) ^ weight_swz(c)));
#pragma unroll
        for (int i = 0; i < C::SC; ++i) scale[i] = *reinterpret_cast<const float*>(lds + C::S_OFF + stage * 256 + 4 * (wave * C::SC + i));
#pragma unroll
        for (int s = 0; s < 2; ++s) {                     // half a block's values first, then its products
            v4u t[2][J][PARTS];
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int j = 0; j < J; ++j)
#pragma unroll
                    for (int h = 0; h < PARTS; ++h)
                        t[q][j][h] = *reinterpret_cast<const v4u*>(
                            xs + 16 * j * C::ROW + 16 * chunk_at<UP>(c, UP ? 8 * s + 2 * g + q : 4 * (4 * s + g) + q + 2 * h));
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int h = 0; h < PARTS; ++h)
#pragma unroll
                    for (int j = 0; j < J; ++j)
#pragma unroll
                        for (int i = 0; i < C::RT; ++i) {
                            const uint32_t lo = w[i][s][2 * q], hi = w[i][s][2 * q + 1];
                            if (s + q + h == 0) mfma<UP && FP16, true>(sum[i][j], lo, hi, t[q][j][h]);
                            else mfma<UP && FP16, false>(sum[i][j], lo, hi, t[q][j][h]);
                        }
        }
        sums_ready(sum);
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
            for (int i = 0; i < C::RT; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k) acc[i][j][k] = __builtin_fmaf(sum[i][j][k], scale[UP ? i : 0], acc[i][j][k]);
    };
    const int step = (int)gridDim.x / XCDS;
    int next = (int)blockIdx.x / XCDS;
    Item it = item_at<BLOCK>(R, experts, items, next, tiles, lane);
    if (it.n == 0) return;
    aim(it);
#pragma unroll
    for (int d = 0; d < AH; ++d) load(d, d);
    for (int stage = 0;;) {
#pragma unroll
        for (int i = 0; i < C::RT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
        Item nx = it;
        for (int u = 0; u < units; u += AH) {
            if (u + AH < units) {
                lu += AH;
            } else {
                next += step;
                nx = item_at<BLOCK>(R, experts, items, next, tiles, lane);
                aim(nx);
            }
#pragma unroll
            for (int d = 0; d < AH; ++d) {
                // this wave's share of the unit has landed, its reads of the last one have returned, and so have all waves'
                __builtin_amdgcn_s_waitcnt(vmcnt_imm((AH - 1) * C::LOADS));
                wait_lgkm0();
                barrier_nofence();
                load(stage == 0 ? C::STAGES - 1 : stage - 1, lu + d);         // in the last one's place
                if (NT == 1 || it.n <= 16) block_sums(std::integral_constant<int, 1>(), stage);
                else block_sums(std::integral_constant<int, NT>(), stage);
                stage = stage == C::STAGES - 1 ? 0 : stage + 1;
            }
        }
        if constexpr (KS > 1) {                           // the groups join, by way of the last unit's weights, where nothing is on its way to
            const int done = stage == 0 ? C::STAGES - 1 : stage - 1;
            v4f* sums = reinterpret_cast<v4f*>(rows_lds + C::RING + C::W_OFF + (done * WV + wave) * C::WSTAGE) + lane;
#pragma unroll
            for (int i = 0; i < C::RT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j)
                    if (part == 1) sums[64 * (i * NT + j)] = acc[i][j];
            wait_lgkm0();
            barrier_nofence();
#pragma unroll
            for (int i = 0; i < C::RT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j)
                    if (part == 0) acc[i][j] += sums[64 * (i * NT + j)];
        }
        const int n0 = (it.tile * WV + wave) * C::OUT + 4 * g;
#pragma unroll
        for (int j = 0; j < NT; ++j)
            if (part == 0 && 16 * j + c < it.n) {
                const int pair = R.pair[it.r0 + 16 * j + c];
                if constexpr (UP) {
                    if (n0 < N) store_h(p, pair, n0, R.weight[it.r0 + 16 * j + c], acc[0][j], acc[1][j]);
                } else {
#pragma unroll
                    for (int i = 0; i < C::RT; ++i)
                        if (n0 + 16 * i < N) *reinterpret_cast<v4f*>(p.z + (int64_t)pair * p.H + n0 + 16 * i) = acc[i][j];
                }
            }
        it = nx;
        if (it.n == 0) break;
    }
    wait_vm0();                                           // the loads behind the last unit have landed before the exit
}

// y: the sum over a token's choices, in their order; of equal experts the first counts (it has both weights).  What bounds it is the
// trip to memory: eight choices are asked for at once, those that do not count too, and left out of the sum.
__global__ void __launch_bounds__(256) moe_combine_kernel(MoeParams p) {
    constexpr int AT_ONCE = 8;
    const int t = blockIdx.y, n = 4 * (int)(blockIdx.x * 256 + threadIdx.x), lane = threadIdx.x & 63;
    const int e = lane < p.k ? p.experts[t * p.k + lane] : -1;
    bool first = true;
    for (int i = 0; i < p.k; ++i) first = first && (i >= lane || __builtin_amdgcn_readlane(e, i) != e);
    const uint64_t count = __ballot(first && e >= 0 && e < p.E);
    if (n >= p.H) return;
    const uint2 residual = residual_at(p, t, n);
    const float* z = p.z + (int64_t)t * p.k * p.H + n;
    v4f v = {0.f, 0.f, 0.f, 0.f};
    for (int j0 = 0; j0 < p.k; j0 += AT_ONCE) {
        v4f c[AT_ONCE];
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) c[j] = *reinterpret_cast<const v4f*>(z + (int64_t)min(j0 + j, p.k - 1) * p.H);
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j)
            if ((count >> (j0 + j)) & 1) v += c[j];
    }
    store_y(p, t, n, v, residual);
}

template <bool UP, bool FP16, int NT, int WV, int KS>
int launch_rows(const MoeParams& p, hipStream_t st) {
    constexpr int CT = 2, AH = 2;
    using C = Rows<UP, NT, CT, WV, KS, AH>;
    const int out = WV * C::OUT, tiles = ((UP ? p.F : p.H) + out - 1) / out, P = p.T * p.k, most = std::min(p.E, P) + P / (16 * NT);
    const size_t lds = C::LDS + routed_bytes(p.E, P, UP);
    // 8 waves per CU
    const int64_t grid = std::min<int64_t>(((int64_t)tiles * most + XCDS - 1) / XCDS * XCDS, std::max(XCDS, 8 / (WV * KS) * h3host::cu_count() / XCDS * XCDS));
    hipLaunchKernelGGL((moe_rows_kernel<UP, FP16, NT, CT, WV, KS, AH>), dim3((unsigned)grid), dim3(WV * KS * 64), lds, st, p, tiles);
    H3_CHECK_HIP(hipGetLastError());
    return H3FP8_OK;
}

int launch_combine(const MoeParams& p, hipStream_t st) {
    hipLaunchKernelGGL(moe_combine_kernel, dim3((unsigned)((p.H + 1023) / 1024), (unsigned)p.T), dim3(256), 0, st, p);
    H3_CHECK_HIP(hipGetLastError());
    return H3FP8_OK;
}

template <bool FP16, int TOKENS>
int launch_few(const MoeParams& p, hipStream_t st) {
    const int tiles = p.F / 16;
    hipLaunchKernelGGL((moe_few_up_kernel<FP16, TOKENS>), dim3((unsigned)(tiles * std::min(p.E, p.T * p.k))), dim3(Few<true, TOKENS>::WAVES * 64), 0, st,
                       p, tiles);
    H3_CHECK_HIP(hipGetLastError());
    hipLaunchKernelGGL((moe_few_down_kernel<TOKENS>), dim3((unsigned)(p.H / 16)), dim3(Few<false, TOKENS>::WAVES * 64), 0, st, p);
    H3_CHECK_HIP(hipGetLastError());
    return H3FP8_OK;
}

// ---- which kernels run --------------------------------------------------------------------------------------------------
//
// A token or a few, while launches and first loads count: one or two tokens up to 16 pairs, up to 8 tokens at 8 pairs and 128 MiB of
// their experts' weights; then by rows.  us of the kernels, few / by rows, for 1 x 4 (token x choices), 2 x 4, 2 x 8, 8 x 1, 4 x 4:
// 32 experts of 4096 x 2048 24 / 40, 41 / 47, 74 / 79, 47 / 42, 87 / 73; 8 of 2048 x 2048 18 / 33, 24 / 33, 29 / 33, 31 / 32,
// 39 / 33; 16 of 1200 x 1040 13 / 23, 20 / 25, 26 / 26, 20 / 25, 33 / 26; 128 of 2048 x 1024 14 / 28, 18 / 29, 29 / 30, 23 / 28,
// 40 / 30.
bool few(int64_t T, int64_t k, int64_t H, int64_t F, int64_t E) {
    return T <= 2 ? T * k <= 16 : T * k <= 8 && 3 * H * F * std::min(T * k, E) <= (128LL << 20);
}

template <bool FP16>
int run(const MoeParams& p, hipStream_t st) {
    if (few(p.T, p.k, p.H, p.F, p.E)) return p.T <= 2 ? launch_few<FP16, 2>(p, st) : launch_few<FP16, 8>(p, st);
    // Blocks of 32 rows and 8 waves past 20 rows per expert, in kernel 2 while they are items enough for the CUs (one of 256
    // channels and all rows of an expert at least); else blocks of 16 and 4 waves.  us, 16 rows and 4 waves / 32 and 8, kernel 1 and
    // kernel 2: 32 experts of 4096 x 2048, 12 rows each 104 / 98 and 58 / 58, 16 110 / 122 and 64 / 71, 24 132 / 117 and 77 / 75,
    // 32 150 / 115 and 110 / 79; 8 experts of 2048 x 2048, 32 rows 27 / 22 and 19 / 25; 16 of 1200 x 1040, 32 rows 21 / 17 and 15 / 19.
    const bool many = p.T * p.k > 20 * p.E, wide = (int64_t)p.H * p.E >= 256 * h3host::cu_count();
    // Two groups of 4 waves to an item where the items leave half the CUs alone and have 12 blocks of K or more.  us, one / two, kernel
    // 1: 4 experts of 4096 x 1024 (64 items, 32 blocks) 21.7 / 17.5, 8 of 4096 x 512 (64) 21.8 / 17.4, but 8 of 2048 x 2048 (256 items,
    // 16 blocks) 15.1 / 16.6, 2 of 1024 x 512 (16, 8) 8.9 / 8.4; kernel 2: 8 of 2048 x 2048 (128, 16) 13.7 / 11.7, 8 of 1536 x 2304
    // (96, 18) 14.9 / 13.0, but 16 of 1024 x 512 (128, 4) 5.9 / 6.3, 12 of 1200 x 1040 (120, 9) 10.5 / 10.6.
    const int blocks = std::max(std::min(p.E, p.T * p.k), p.T * p.k / 16);
    const auto two = [&](int64_t tiles, int K) { return 2 * tiles * blocks <= h3host::cu_count() && K > 11 * BK; };
    int rc = many                        ? launch_rows<true, FP16, 2, 8, 1>(p, st)
             : two((p.F + 63) / 64, p.H) ? launch_rows<true, FP16, 1, 4, 2>(p, st)
                                         : launch_rows<true, FP16, 1, 4, 1>(p, st);
    if (rc) return rc;
    rc = many && wide                  ? launch_rows<false, false, 2, 8, 1>(p, st)
         : two((p.H + 127) / 128, p.F) ? launch_rows<false, false, 1, 4, 2>(p, st)
                                       : launch_rows<false, false, 1, 4, 1>(p, st);
    return rc ? rc : launch_combine(p, st);
}

constexpr int64_t kMaxSpan = 0x7fff0000LL;

}  // namespace

extern "C" int64_t h3fp8_moe_blocks_workspace(int64_t T, int64_t k, int64_t H, int64_t F, int64_t E) {
    return T < 0 || k < 0 || H < 0 || F < 0 || E < 0 ? 0 : T * k * 4 * (few(T, k, H, F, E) ? F : F + H);
}

extern "C" int h3fp8_moe_blocks(const void* x, int64_t ldx, int dtype, int64_t T, int64_t H, int64_t F, int64_t E, int k,
                                const void* w1, int64_t w1_e, int64_t ld1, const float* s1, int64_t s1_e, int64_t s1_n, int64_t s1_k,
                                const void* w2, int64_t w2_e, int64_t ld2, const float* s2, int64_t s2_e, int64_t s2_n, int64_t s2_k,
                                const float* weights, const int32_t* experts, const int32_t* offsets, const int32_t* order,
                                const void* residual, int64_t ldr, void* y, int64_t ldy, void* workspace, int64_t workspace_bytes,
                                void* stream) {
    const char* who = "h3fp8_moe_blocks";
    H3_REQUIRE(T >= 0 && T <= MAX_T, "%s: %lld tokens (at most %d; more go by h3fp8_grouped_gemm_blocks)", who, (long long)T, MAX_T);
    H3_REQUIRE(E >= 1 && E <= MAX_E && k >= 1 && k <= MAX_K && k <= E, "%s: k = %d of %lld experts (at most %d of %d)", who, k,
               (long long)E, MAX_K, MAX_E);
    H3_REQUIRE(dtype == H3FP8_DT_BF16 || dtype == H3FP8_DT_FP16, "%s: bad dtype %d", who, dtype);
    H3_REQUIRE(H >= 16 && F >= 16 && H % 16 == 0 && F % 16 == 0 && H <= (1 << 22) && F <= (1 << 22),
               "%s: H=%lld and F=%lld must be positive multiples of 16, at most 2^22", who, (long long)H, (long long)F);
    if (T == 0) return H3FP8_OK;
    H3_REQUIRE(x && w1 && s1 && w2 && s2 && weights && experts && offsets && order && y && workspace, "%s: null pointer", who);
    H3_REQUIRE(((((uintptr_t)x | (uintptr_t)w1 | (uintptr_t)w2 | (uintptr_t)workspace) & 15) | (((uintptr_t)y | (uintptr_t)residual) & 7)) == 0,
               "%s: x, w1, w2 and the workspace must be 16-byte, y and the residual 8-byte aligned", who);
    H3_REQUIRE((((uintptr_t)s1 | (uintptr_t)s2 | (uintptr_t)weights | (uintptr_t)experts | (uintptr_t)offsets | (uintptr_t)order) & 3) == 0,
               "%s: misaligned scales or routing", who);
    H3_REQUIRE((T == 1 || (ldx >= H && ldy >= H)) && ldx % 8 == 0 && ldy % 4 == 0 && (!residual || (ldr >= 0 && ldr % 4 == 0)),
               "%s: the row strides of x and y must be >= H, x's a multiple of 8, y's and the residual's of 4", who);
    H3_REQUIRE(ld1 >= H && ld2 >= F && ld1 % 16 == 0 && ld2 % 16 == 0 && w1_e >= 0 && w2_e >= 0 && w1_e % 16 == 0 && w2_e % 16 == 0,
               "%s: the weights' row strides must cover their rows, theirs and the expert strides be multiples of 16", who);
    H3_REQUIRE(s1_e >= 0 && s1_n >= 0 && s1_k >= 0 && s2_e >= 0 && s2_n >= 0 && s2_k >= 0, "%s: negative stride", who);
    const int64_t span = kMaxSpan;
    H3_REQUIRE(ldx <= span / 512 && ld1 <= span / 128 && ld2 <= span / 128 && T * k * F * 4 <= span, "%s: a stride or size is too large", who);
    // the scales' offsets are 32 bits of bytes
    const auto bounded = [&](int64_t n, int64_t kb, int64_t se, int64_t sn, int64_t sk) {
        return se <= span / 4 && sn <= span / 4 && sk <= span / 4 && ((E - 1) * se + (n - 1) * sn + (kb - 1) * sk) * 4 <= span / 2;
    };
    const int64_t hb = (H + 127) / 128, fb = (F + 127) / 128, f2 = (2 * F + 127) / 128;
    H3_REQUIRE(bounded(f2, hb, s1_e, s1_n, s1_k) && bounded(hb, fb, s2_e, s2_n, s2_k), "%s: a scale stride is too large", who);
    const int64_t need = h3fp8_moe_blocks_workspace(T, k, H, F, E);
    H3_REQUIRE(workspace_bytes >= need, "%s: the workspace needs %lld bytes", who, (long long)need);
    MoeParams p{};
    p.x = x; p.ldx = ldx;
    p.w1 = (const uint8_t*)w1; p.s1 = s1; p.w2 = (const uint8_t*)w2; p.s2 = s2;
    p.w1_e = w1_e; p.ld1 = ld1; p.w2_e = w2_e; p.ld2 = ld2;
    p.s1_e = s1_e; p.s1_n = s1_n; p.s1_k = s1_k; p.s2_e = s2_e; p.s2_n = s2_n; p.s2_k = s2_k;
    p.weights = weights; p.experts = experts; p.offsets = offsets; p.order = order;
    p.residual = residual; p.ldr = ldr; p.y = (uint16_t*)y; p.ldy = ldy; p.h = (char*)workspace; p.z = (float*)(p.h + T * k * F * 4);
    p.T = (int)T; p.E = (int)E; p.k = k; p.H = (int)H; p.F = (int)F; p.fp16 = dtype == H3FP8_DT_FP16;
    return p.fp16 ? run<true>(p, (hipStream_t)stream) : run<false>(p, (hipStream_t)stream);
}
