// A whole layer of block-scaled FP8 experts for a few tokens (gfx950), in two kernels.
//
//   y[t] = residual[t] + sum_j weight[t, j] * W2[e] h,  h = silu(g) * u,  g | u = W1[e] x[t],  e = experts[t, j]
//
// Every weight is read once, the tokens of an expert together, and the time is that of the weights' bytes.  The tokens stay as
// they are (bf16 / fp16), unlike in the path of many tokens, whose products quantise them: the weights' e4m3 codes are
// widened in registers (bf16 and fp16 hold them exactly), MFMAs 16x16x32 make the sum of one block of 128 from a zero
// accumulator, the weight rows as the A operand and the tokens as B, and one fma per element adds it with the block's
// scale in fp32.
//
// Kernel 1: a workgroup takes 16 NI gate rows and the up rows that belong to them, of one expert that has tokens, and all of
// that expert's tokens; its 8 waves share out the blocks of K and join through LDS.  h times the pair's weight leaves as two
// bf16 numbers, the value and what its rounding left (16 bits in all, so that the layer has one rounding to the output's
// type and none that counts before).
// Kernel 2: a workgroup takes 16 CT rows of W2 for all experts, and its waves share out the (expert, block of F) units; the
// MFMA's 16 columns are tokens by their own number, zero where a token is not the expert's, so that the sums over experts
// stay in the accumulators and no order of workgroups shows in the result.
#include <algorithm>

#include "gemm_core.h"

namespace {

using namespace h3g;

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8hf __attribute__((ext_vector_type(8)));

constexpr int WAVES = 8;
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

// 16 bytes per lane; OOB (and up to 64 KiB past it) and what lies past the buffer read as zeros.  The hardware checks the lane's
// offset against the buffer's size less the uniform offset: that one is the start of a block that there is.
template <bool NT>
__device__ __forceinline__ v4u load16(__amdgpu_buffer_rsrc_t r, uint32_t voff, uint32_t soff) {
    return __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(r, (int)voff, (int)soff, NT ? 2 : 0));
}

// One number for all lanes.
__device__ __forceinline__ float load4(__amdgpu_buffer_rsrc_t r, uint32_t off) {
    return u2f(__builtin_amdgcn_raw_buffer_load_b32(r, (int)off, 0, 0));
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

struct Block { int e, r0, n; };                           // n sorted rows from r0 on, of expert e

struct Routed {
    int* count;                                           // of blocks
    int* pair;                                            // [P] of a sorted row
    float* weight;                                        // [P] of a sorted row: of all its token's choices of its expert (the
                                                          // second of two equal ones has the same, and is not read)
    Block* blocks;                                        // the experts' rows in blocks of at most ROWS
    int* experts;                                         // [P] of a pair
    float* weights;                                       // [P]
};

template <int ROWS>
constexpr int max_blocks(int E, int P) { return (E < P ? E : P) + P / ROWS; }

template <int ROWS>
constexpr size_t routed_bytes(int E, int P) { return (size_t)P * 16 + (size_t)max_blocks<ROWS>(E, P) * sizeof(Block) + 16; }

// By all threads, with barriers.
template <int ROWS>
__device__ __forceinline__ Routed load_routing(const MoeParams& p, char* lds, int threads) {
    const int P = p.T * p.k, lane = threadIdx.x & 63, cap = max_blocks<ROWS>(p.E, P);
    Routed r;
    r.count = reinterpret_cast<int*>(lds);
    r.pair = r.count + 4;
    r.weight = reinterpret_cast<float*>(r.pair + P);
    r.experts = reinterpret_cast<int*>(r.weight + P);
    r.weights = reinterpret_cast<float*>(r.experts + P);
    r.blocks = reinterpret_cast<Block*>(r.weights + P);
    for (int i = threadIdx.x; i < P; i += threads) {
        const int o = p.order[i], e = p.experts[i];
        const float w = p.weights[i];
        r.pair[i] = min(max(o, 0), P - 1);                // whatever it holds, no row outside the tokens is read
        r.experts[i] = e;
        r.weights[i] = w;
    }
    if (threadIdx.x < 64) {
        int blocks = 0;
        for (int e0 = 0; e0 < p.E; e0 += 64) {
            int lo = 0, hi = 0;
            if (e0 + lane < p.E) lo = offset_at(p, e0 + lane), hi = offset_at(p, e0 + lane + 1);
            const int n = max(hi - lo, 0), nb = (n + ROWS - 1) / ROWS, at = blocks + wave_prefix(nb) - nb;
            for (int i = 0; i < nb; ++i)                  // (offsets that are not ascending may name more blocks than there are pairs)
                if (at + i < cap) r.blocks[at + i] = Block{e0 + lane, lo + i * ROWS, min(ROWS, n - i * ROWS)};
            blocks = __builtin_amdgcn_readlane(at + nb, 63);
        }
        if (lane == 0) *r.count = min(blocks, cap);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < P; i += threads) {
        const int e = r.experts[r.pair[i]];
        float w = 0.0f;
        for (int j = 0, q = r.pair[i] / p.k * p.k; j < p.k; ++j) w += r.experts[q + j] == e ? r.weights[q + j] : 0.0f;
        r.weight[i] = w;
    }
    __syncthreads();
    return r;
}

// An item of a persistent workgroup: a block of rows and a tile of output channels.
struct Item {
    int blk, tile;

    __device__ __forceinline__ void next(int step_blk, int step_tile, int tiles) {
        blk += step_blk;
        tile += step_tile;
        if (tile >= tiles) tile -= tiles, ++blk;
    }
};

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

// 4 consecutive channels n .. n + 3 of a token, with the residual.
__device__ __forceinline__ void store_y(const MoeParams& p, int t, int n, v4f v) {
    if (p.residual) {
        const uint2 r = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(p.residual) + t * p.ldr + n);
        const uint32_t b[4] = {r.x & 0xffffu, r.x >> 16, r.y & 0xffffu, r.y >> 16};
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] += p.fp16 ? fp16_to_f32(b[q]) : bf16_to_f32(b[q]);
    }
    const uint2 o = p.fp16 ? uint2{fp16_rne(v[0]) | (fp16_rne(v[1]) << 16), fp16_rne(v[2]) | (fp16_rne(v[3]) << 16)}
                           : uint2{cvt_bf16x2(v[0], v[1]), cvt_bf16x2(v[2], v[3])};
    *reinterpret_cast<uint2*>(p.y + t * p.ldy + n) = o;
}

// ---- kernel 1 ---------------------------------------------------------------------------------------------------------
//
// An item is a block of up to 16 rows of one expert and 16 gate rows; the workgroup's 8 waves share out the blocks of K.  Two
// workgroups per CU, persistent: a wave's loads run D of its units (blocks of K) ahead, across items.

template <bool FP16, int D>
__global__ void __launch_bounds__(WAVES * 64, 4) moe_up_kernel(MoeParams p, int tiles, int step_blk, int step_tile) {
    extern __shared__ __attribute__((aligned(16))) char up_lds[];
    __shared__ v4f part[2][WAVES][2][64];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int c = lane & 15, g = lane >> 4;
    const Routed R = load_routing<16>(p, up_lds, WAVES * 64);
    const int blocks = __builtin_amdgcn_readfirstlane(*R.count);
    const int kb = (p.H + BK - 1) / BK, rounds = (kb + D * WAVES - 1) / (D * WAVES);
    const __amdgpu_buffer_rsrc_t rx = make_rsrc(p.x, (uint32_t)(((p.T - 1) * p.ldx + p.H) * 2));
    const __amdgpu_buffer_rsrc_t rs = make_rsrc(p.s1, 0x7fffffffu);
    // what the next loads need: buffers, lane offsets of the weight row and the token, offsets of the scales, the block
    __amdgpu_buffer_rsrc_t rg, ru;
    uint32_t vw, vx, sg, su;
    int lb, lend;                                         // (past the last item no block is there)
    auto aim = [&](const Item& it) {
        const bool live = it.blk < blocks;
        const Block& B = R.blocks[live ? it.blk : 0];
        const int e = __builtin_amdgcn_readfirstlane(B.e), r0 = __builtin_amdgcn_readfirstlane(B.r0), n = __builtin_amdgcn_readfirstlane(B.n);
        const int f0 = it.tile * 16;
        const uint32_t bytes = live ? (uint32_t)(15 * p.ld1 + p.H) : 0u;
        const uint8_t* w = p.w1 + e * p.w1_e + f0 * p.ld1;
        rg = make_rsrc(w, bytes);
        ru = make_rsrc(w + p.F * p.ld1, bytes);
        vx = live && c < n ? (uint32_t)(R.pair[r0 + min(c, n - 1)] / p.k) * (uint32_t)(p.ldx * 2) + 32u * g : OOB;
        sg = (uint32_t)(e * p.s1_e + f0 / BK * p.s1_n) * 4u;
        su = (uint32_t)(e * p.s1_e + (p.F + f0) / BK * p.s1_n) * 4u;
        lb = wave;
        lend = live ? kb : 0;
    };
    vw = (uint32_t)(c * p.ld1) + 16u * g;
    v4u w[D][2][2], x[D][2][2];
    float sc[D][2];
    // always the same loads, past the last block of nothing, so that the count of those under way is known
    auto load = [&](int d) {
        const int b = lb + d * WAVES, at = b < lend ? b * BK : 0, left = b < lend ? p.H - at : 0;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const bool in = 64 * s + 16 * g < left;
            w[d][0][s] = load16<true>(rg, (in ? vw : OOB) + 64 * s, at);
            w[d][1][s] = load16<true>(ru, (in ? vw : OOB) + 64 * s, at);
#pragma unroll
            for (int q = 0; q < 2; ++q) x[d][s][q] = load16<false>(rx, (in ? vx : OOB) + 128 * s + 16 * q, 2 * at);
        }
        const uint32_t sb = (uint32_t)(min(b, kb - 1) * p.s1_k) * 4u;
        sc[d][0] = load4(rs, sg + sb);
        sc[d][1] = load4(rs, su + sb);
        __builtin_amdgcn_sched_barrier(0);                // in this order: the waits count them
    };
    Item it{(int)blockIdx.x / tiles, (int)blockIdx.x % tiles}, nx = it;
    if (it.blk >= blocks) return;
    aim(it);
#pragma unroll
    for (int d = 0; d < D; ++d) load(d);
    for (int buf = 0;; buf ^= 1) {
        v4f acc[2] = {v4f{0.f, 0.f, 0.f, 0.f}, v4f{0.f, 0.f, 0.f, 0.f}};
        for (int r = 0; r < rounds; ++r) {
            if (r + 1 < rounds) lb += D * WAVES;
            else nx.next(step_blk, step_tile, tiles), aim(nx);
#pragma unroll
            for (int d = 0; d < D; ++d) {
                v4f sum[2][1];
#pragma unroll
                for (int q = 0; q < 4; ++q)               // 32 of the block's k each
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const v4u& a = w[d][i][q >> 1];
                        if (q == 0) mfma<FP16, true>(sum[i][0], a[0], a[1], x[d][0][0]);
                        else mfma<FP16, false>(sum[i][0], a[2 * (q & 1)], a[2 * (q & 1) + 1], x[d][q >> 1][q & 1]);
                    }
                sums_ready(sum);
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int k = 0; k < 4; ++k) acc[i][k] = __builtin_fmaf(sum[i][0][k], sc[d][i], acc[i][k]);
                __builtin_amdgcn_sched_barrier(0);
                load(d);
            }
        }
        // join the waves' sums; the other buffer is the next item's
#pragma unroll
        for (int i = 0; i < 2; ++i) part[buf][wave][i][lane] = acc[i];
        wait_lgkm0();
        barrier_nofence();
        if (wave == (it.tile & (WAVES - 1))) {
            v4f gate = part[buf][0][0][lane], up = part[buf][0][1][lane];
#pragma unroll
            for (int v = 1; v < WAVES; ++v) {
                gate += part[buf][v][0][lane];
                up += part[buf][v][1][lane];
                asm volatile("" : "+v"(gate), "+v"(up)::"memory");        // not all of them in registers at once
            }
            const Block& B = R.blocks[it.blk];
            if (c < B.n) store_h(p, R.pair[B.r0 + c], it.tile * 16 + 4 * g, R.weight[B.r0 + c], gate, up);
        }
        it.next(step_blk, step_tile, tiles);
        if (it.blk >= blocks) return;
    }
}

// ---- kernel 2, few rows per expert --------------------------------------------------------------------------------------
//
// A workgroup takes 16 channels for all experts; its 16 waves share out the units, the blocks of F of every expert that has rows.
// Column c of the MFMAs is token 16 j + c, zero where it is not the expert's, so that the accumulators run over all experts.

constexpr int DOWN_WAVES = 16;

// NT: blocks of 16 tokens (all of them); D: units in flight per wave.
template <int NT, int D>
__global__ void __launch_bounds__(DOWN_WAVES * 64) moe_down_kernel(MoeParams p) {
    constexpr int THREADS = DOWN_WAVES * 64;
    extern __shared__ __attribute__((aligned(16))) char down_lds[];
    v4f(*part)[NT][64] = reinterpret_cast<v4f(*)[NT][64]>(down_lds);                            // [DOWN_WAVES]
    int* s_expert = reinterpret_cast<int*>(down_lds + sizeof(v4f) * DOWN_WAVES * NT * 64);      // the experts that have pairs
    uint16_t* s_slot = reinterpret_cast<uint16_t*>(s_expert + MAX_E);                           // ... and where an expert is among them
    uint8_t* s_map = reinterpret_cast<uint8_t*>(s_slot + MAX_E);                                // [slots][16 NT]: 1 + the token's choice, or 0
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int n0 = (int)blockIdx.x * 16, P = p.T * p.k, cap = min(p.E, P);
    // the pairs' experts, under way together with the offsets
    constexpr int MINE = (16 * NT * MAX_K + THREADS - 1) / THREADS;
    int experts[MINE];
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
        const int q = threadIdx.x + i * THREADS;
        experts[i] = q < P ? p.experts[q] : -1;
    }
    for (int i = threadIdx.x; i < cap * 4 * NT; i += THREADS) reinterpret_cast<uint32_t*>(s_map)[i] = 0;
    int active = 0;
    for (int e0 = 0; e0 < p.E; e0 += 64) {                // every wave counts, the first one writes
        const int e = e0 + lane;
        const bool in = e < p.E && offset_at(p, e + 1) > offset_at(p, e);
        const uint64_t has = __ballot(in);
        const int at = active + __popcll(has & ((1ull << lane) - 1));
        if (wave == 0 && e < p.E) {
            s_slot[e] = in && at < cap ? (uint16_t)at : (uint16_t)0xffff;
            if (in && at < cap) s_expert[at] = e;
        }
        active += __popcll(has);
    }
    active = min(active, cap);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
        const int q = threadIdx.x + i * THREADS, e = experts[i];
        if (e >= 0 && e < p.E && s_slot[e] != 0xffff) s_map[s_slot[e] * 16 * NT + q / p.k] = (uint8_t)(1 + q % p.k);
    }
    __syncthreads();
    const int fb = (p.F + BK - 1) / BK, units = active * fb;
    const __amdgpu_buffer_rsrc_t rh = make_rsrc(p.h, (uint32_t)P * (uint32_t)p.F * 4u), rs = make_rsrc(p.s2, 0x7fffffffu);
    const uint32_t vw = (uint32_t)(c * p.ld2) + 16u * g, wbytes = (uint32_t)(15 * p.ld2 + p.F);
    const uint8_t* w0 = p.w2 + n0 * p.ld2;
    const uint32_t s0 = (uint32_t)(n0 / BK * p.s2_n) * 4u;
    v4u w[D][2], h[D][NT][2][4];                          // h: 16 values, what they leave
    float sc[D];
    int ls = 0, lb = wave;                                // the next unit's expert and block
    while (lb >= fb && ls < active) lb -= fb, ++ls;
    // always the same loads, past the last unit of nothing, so that the count of those under way is known
    auto load = [&](int d) {
        const bool live = ls < active;
        const int slot = live ? ls : 0, b = live ? lb : 0, e = __builtin_amdgcn_readfirstlane(s_expert[slot]);
        const int left = live ? p.F - b * BK : 0;
        const __amdgpu_buffer_rsrc_t rw = make_rsrc(w0 + e * p.w2_e, live ? wbytes : 0u);
        uint32_t vh[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int m = s_map[slot * 16 * NT + 16 * j + c];
            vh[j] = m ? (uint32_t)((16 * j + c) * p.k + m - 1) * (uint32_t)p.F * 4u + 64u * g : OOB;
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const bool in = 64 * s + 16 * g < left;
            w[d][s] = load16<true>(rw, (in ? vw : OOB) + 64 * s, b * BK);
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) h[d][j][s][q] = load16<false>(rh, (in ? vh[j] : OOB) + 256 * s + 16 * q, 4 * b * BK);
        }
        sc[d] = load4(rs, (uint32_t)(e * p.s2_e + b * p.s2_k) * 4u + s0);
        lb += DOWN_WAVES;
        while (lb >= fb && ls < active) lb -= fb, ++ls;
        __builtin_amdgcn_sched_barrier(0);                // in this order: the waits count them
    };
    v4f acc[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[j] = v4f{0.f, 0.f, 0.f, 0.f};
    if (units > 0) {
#pragma unroll
        for (int d = 0; d < D; ++d) load(d);
    }
    int slot = 0, b = wave;                               // of the unit at hand
    while (b >= fb && slot < active) b -= fb, ++slot;
    for (int u0 = wave; u0 < units; u0 += D * DOWN_WAVES) {
#pragma unroll
        for (int d = 0; d < D; ++d) {
            v4f sum[1][NT];
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    const uint32_t lo = w[d][q >> 1][2 * (q & 1)], hi = w[d][q >> 1][2 * (q & 1) + 1];
                    if (q == 0) mfma<false, true>(sum[0][j], lo, hi, h[d][j][0][0]);
                    else mfma<false, false>(sum[0][j], lo, hi, h[d][j][q >> 1][q & 1]);
                    mfma<false, false>(sum[0][j], lo, hi, h[d][j][q >> 1][2 + (q & 1)]);
                }
            sums_ready(sum);
#pragma unroll
            for (int j = 0; j < NT; ++j)
                if (slot < active && s_map[slot * 16 * NT + 16 * j + c] != 0) {       // an expert's NaN is not another token's
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[j][r] = __builtin_fmaf(sum[0][j][r], sc[d], acc[j][r]);
                }
            __builtin_amdgcn_sched_barrier(0);
            load(d);
            b += DOWN_WAVES;
            while (b >= fb && slot < active) b -= fb, ++slot;
        }
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) part[wave][j][lane] = acc[j];
    __syncthreads();
    if (threadIdx.x < NT * 64) {
        const int j = threadIdx.x >> 6, t = 16 * j + c, n = n0 + 4 * g;
        v4f v = part[0][j][lane];
#pragma unroll
        for (int q = 1; q < DOWN_WAVES; ++q) v += part[q][j][lane];
        if (t < p.T) store_y(p, t, n, v);
    }
}

// ---- more rows per expert -----------------------------------------------------------------------------------------------
//
// With many rows the tokens' values, read again for every 16 weight rows, are more than the weights.  So the 8 waves of a workgroup
// take 8 neighbouring tiles of weight rows, the whole of K each (no join), and share the tokens' values through LDS: an item is a
// block of up to 16 NT rows and 8 tiles.  A unit is 256 (NT = 1) or 128 of K in kernel 1, 128 of F (both numbers) in kernel 2.  It comes by LDS-DMA, two units ahead of its use in a ring of three, one barrier per unit; the weights come two units
// ahead into registers.  Kernel 2 leaves the pairs' results in fp32, and a third kernel adds up the choices of each token, in their
// order.

template <bool UP, int NT, int CT>
struct Rows {
    static constexpr int RT = UP ? 2 : CT;                // tiles of 16 weight rows of a wave: gate and up; channels
    static constexpr int KB = UP && NT == 1 ? 2 : 1;      // blocks of 128 of a unit
    static constexpr int ROW = UP ? 256 * KB : 512;       // bytes of a row's unit
    static constexpr int STAGE = 16 * NT * ROW, DX = STAGE / 1024 / WAVES;    // LDS-DMA instructions of a wave, 1 KiB each
    static constexpr int SC = UP ? 2 : 1;                 // scales of a block
    static constexpr int OUT = UP ? 16 : 16 * CT;         // output channels of a wave
    static constexpr int LOADS = KB * (2 * RT + SC);      // of a unit, per wave
};

// LDS place of 16-byte chunk i of row r: the 16 lanes that are served together (0-3, 12-15 and 20-27; 4-11, 16-19 and 28-31) meet 16
// places.  Kernel 1: lane group g reads chunks 2 g + ..; kernel 2: 4 g + ..
template <bool UP>
__device__ __forceinline__ int chunk_at(int r, int i) {
    const int c = r & 15;
    return i ^ (UP ? c : (((c >> 2) ^ (c >> 3)) & 1) | ((c & 3) << 1) | (c & 8));
}

constexpr int STAGES = 3, AHEAD = 2;

template <bool UP, bool FP16, int NT, int CT>
__global__ void __launch_bounds__(WAVES * 64, NT <= 2 ? 4 : 2) moe_rows_kernel(MoeParams p, int tiles, int step_blk, int step_tile, int cap) {
    using C = Rows<UP, NT, CT>;
    constexpr int STAGE = C::STAGE, DX = C::DX, LPR = C::ROW / 16, RPI = 64 / LPR;     // lanes of a row, rows of an instruction
    extern __shared__ __attribute__((aligned(1024))) uint8_t rows_lds[];
    uint8_t* lds = rows_lds;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int c = lane & 15, g = lane >> 4;
    const uint32_t lds0 = lds_addr(lds);
    const Routed R = load_routing<16 * NT>(p, reinterpret_cast<char*>(lds + STAGES * STAGE), WAVES * 64);
    const int blocks = __builtin_amdgcn_readfirstlane(*R.count);
    const int K = UP ? p.H : p.F, N = UP ? p.F : p.H, kb = (K + BK - 1) / BK, units = (kb + AHEAD * C::KB - 1) / (AHEAD * C::KB) * AHEAD;
    const int64_t ld = UP ? p.ld1 : p.ld2;
    const v4u rx = buffer_desc(UP ? p.x : p.h, UP ? (uint32_t)(((p.T - 1) * p.ldx + p.H) * 2) : (uint32_t)(p.T * p.k) * (uint32_t)p.F * 4u);
    const __amdgpu_buffer_rsrc_t rs = make_rsrc(UP ? p.s1 : p.s2, 0x7fffffffu);
    const uint32_t row_bytes = UP ? (uint32_t)p.H * 2u : (uint32_t)p.F * 4u;
    // what the next loads need: buffers, lane offsets of the tokens' chunks, offsets of the scales, the unit
    __amdgpu_buffer_rsrc_t rw, ru;
    uint32_t vx[DX], vc[DX], s_at, s_up;
    int lu = 0;
    bool alive;
    const uint32_t vw = (uint32_t)(c * ld) + 16u * g;
#pragma unroll
    for (int i = 0; i < DX; ++i)                          // the chunk that the lane's 16 bytes of its row are
        vc[i] = 16u * (uint32_t)chunk_at<UP>(RPI * (wave * DX + i) + lane / LPR, lane % LPR);
    auto aim = [&](const Item& it) {
        const bool live = it.blk < blocks;
        const Block& B = R.blocks[live ? it.blk : 0];
        const int e = __builtin_amdgcn_readfirstlane(B.e), r0 = __builtin_amdgcn_readfirstlane(B.r0), n = __builtin_amdgcn_readfirstlane(B.n);
        const int n0 = (it.tile * WAVES + wave) * C::OUT, rows = min(C::OUT, N - n0);
        alive = live && rows > 0;
        const uint32_t bytes = alive ? (uint32_t)((rows - 1) * ld + K) : 0u;
        const int at = alive ? n0 : 0;
        const uint8_t* w = (UP ? p.w1 + e * p.w1_e : p.w2 + e * p.w2_e) + at * ld;
        rw = make_rsrc(w, bytes);
        if (UP) ru = make_rsrc(w + p.F * ld, bytes);
        s_at = (uint32_t)(UP ? e * p.s1_e + at / BK * p.s1_n : e * p.s2_e + at / BK * p.s2_n) * 4u;
        s_up = UP ? (uint32_t)(e * p.s1_e + (p.F + at) / BK * p.s1_n) * 4u : 0u;
#pragma unroll
        for (int i = 0; i < DX; ++i) {
            const int row = RPI * (wave * DX + i) + lane / LPR;
            uint32_t v = OOB;
            if (live && row < n) v = UP ? (uint32_t)(R.pair[r0 + row] / p.k) * (uint32_t)(p.ldx * 2) : (uint32_t)R.pair[r0 + row] * row_bytes;
            vx[i] = v;
        }
        lu = 0;
    };
    v4u w[AHEAD][C::KB][C::RT][2];
    float sc[AHEAD][C::KB][C::SC];
    // the tokens' values of the unit into a stage, the weights of the unit: always the same loads, past the last of nothing
    auto fetch = [&](int stage, int u) {
        const uint32_t at = lds0 + (uint32_t)(stage * STAGE + wave * DX * 1024), k0 = (uint32_t)(u * C::ROW);
#pragma unroll
        for (int i = 0; i < DX; ++i) dma16(rx, __builtin_amdgcn_readfirstlane(at + 1024u * i), vx[i] != OOB && k0 + vc[i] < row_bytes ? vx[i] + k0 + vc[i] : OOB);
        __builtin_amdgcn_sched_barrier(0);
    };
    auto load = [&](int d, int u) {
#pragma unroll
        for (int b = 0; b < C::KB; ++b) {
            const int blk = u * C::KB + b, k0 = alive && blk < kb ? blk * BK : 0, left = alive && blk < kb ? K - k0 : 0;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const bool in = 64 * s + 16 * g < left;
#pragma unroll
                for (int i = 0; i < C::RT; ++i)
                    w[d][b][i][s] = load16<true>(UP && i ? ru : rw, (in ? vw + (UP ? 0u : (uint32_t)(16 * i * ld)) : OOB) + 64 * s, k0);
            }
            const uint32_t sb = (uint32_t)(min(blk, kb - 1) * (UP ? p.s1_k : p.s2_k)) * 4u;
            sc[d][b][0] = load4(rs, s_at + sb);
            if (UP) sc[d][b][C::SC - 1] = load4(rs, s_up + sb);
        }
        __builtin_amdgcn_sched_barrier(0);                // in this order: the waits count them
    };
    Item it{(int)blockIdx.x / tiles, (int)blockIdx.x % tiles}, nx = it;
    if (it.blk >= blocks) return;
    aim(it);
#pragma unroll
    for (int d = 0; d < AHEAD; ++d) {
        fetch(d, d);
        load(d, d);
    }
    for (int stage = 0;;) {
        const Block B = R.blocks[it.blk];
        const int n = __builtin_amdgcn_readfirstlane(B.n);
        v4f acc[C::RT][NT];
#pragma unroll
        for (int i = 0; i < C::RT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
        for (int u = 0; u < units; u += AHEAD) {
            if (u + AHEAD < units) lu += AHEAD;
            else nx.next(step_blk, step_tile, tiles), aim(nx);
#pragma unroll
            for (int d = 0; d < AHEAD; ++d) {
                // this wave's share of the unit has landed (behind it: its weights, the next unit's both), and its reads of the last one
                __builtin_amdgcn_s_waitcnt(vmcnt_imm(AHEAD * C::LOADS + (AHEAD - 1) * DX));
                wait_lgkm0();
                barrier_nofence();
                const int free = stage == 0 ? STAGES - 1 : stage - 1;             // the last one's place
                fetch(free, lu + d);
                const uint8_t* st = lds + stage * STAGE;
#pragma unroll
                for (int b = 0; b < C::KB; ++b) {
                    v4f sum[C::RT][NT];
#pragma unroll
                    for (int q = 0; q < 4; ++q)
#pragma unroll
                        for (int j = 0; j < NT; ++j) {
                            if (j && 16 * j >= n) continue;   // uniform
                            const int chunk = UP ? 16 * b + 8 * (q >> 1) + 2 * g + (q & 1) : 4 * (4 * (q >> 1) + g) + (q & 1);
                            const uint8_t* row = st + (16 * j + c) * C::ROW;
                            const v4u t = *reinterpret_cast<const v4u*>(row + 16 * chunk_at<UP>(c, chunk));
#pragma unroll
                            for (int i = 0; i < C::RT; ++i) {
                                const uint32_t lo = w[d][b][i][q >> 1][2 * (q & 1)], hi = w[d][b][i][q >> 1][2 * (q & 1) + 1];
                                if (q == 0) mfma<UP && FP16, true>(sum[i][j], lo, hi, t);
                                else mfma<UP && FP16, false>(sum[i][j], lo, hi, t);
                            }
                            if (!UP) {
                                const v4u t2 = *reinterpret_cast<const v4u*>(row + 16 * chunk_at<UP>(c, chunk + 2));
#pragma unroll
                                for (int i = 0; i < C::RT; ++i)
                                    mfma<false, false>(sum[i][j], w[d][b][i][q >> 1][2 * (q & 1)], w[d][b][i][q >> 1][2 * (q & 1) + 1], t2);
                            }
                        }
                    sums_ready(sum);
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        if (j && 16 * j >= n) continue;
#pragma unroll
                        for (int i = 0; i < C::RT; ++i)
#pragma unroll
                            for (int k = 0; k < 4; ++k) acc[i][j][k] = __builtin_fmaf(sum[i][j][k], sc[d][b][UP ? i : 0], acc[i][j][k]);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                load(d, lu + d);
                stage = stage == STAGES - 1 ? 0 : stage + 1;
            }
        }
        const int n0 = (it.tile * WAVES + wave) * C::OUT + 4 * g;
#pragma unroll
        for (int j = 0; j < NT; ++j)
            if (16 * j + c < n) {
                const int pair = R.pair[B.r0 + 16 * j + c];
                if constexpr (UP) {
                    if (n0 < N) store_h(p, pair, n0, R.weight[B.r0 + 16 * j + c], acc[0][j], acc[1][j]);
                } else {
#pragma unroll
                    for (int i = 0; i < C::RT; ++i)
                        if (n0 + 16 * i < N) *reinterpret_cast<v4f*>(p.z + (int64_t)pair * p.H + n0 + 16 * i) = acc[i][j];
                }
            }
        it.next(step_blk, step_tile, tiles);
        if (it.blk >= blocks) break;
    }
    wait_vm0();                                           // the loads behind the last unit have landed before the exit
}

// y: the sum over a token's choices, in their order; of equal experts the first counts (it has both weights).
__global__ void __launch_bounds__(256) moe_combine_kernel(MoeParams p) {
    const int t = blockIdx.y, n = 4 * (int)(blockIdx.x * 256 + threadIdx.x);
    if (n >= p.H) return;
    v4f v = {0.f, 0.f, 0.f, 0.f};
    for (int j = 0; j < p.k; ++j) {
        const int q = t * p.k + j, e = p.experts[q];
        bool count = e >= 0 && e < p.E;
        for (int i = 0; i < j; ++i) count = count && p.experts[t * p.k + i] != e;
        if (count) v += *reinterpret_cast<const v4f*>(p.z + (int64_t)q * p.H + n);
    }
    store_y(p, t, n, v);
}

template <bool UP, bool FP16, int NT, int CT>
int launch_rows(const MoeParams& p, hipStream_t st) {
    const int out = WAVES * Rows<UP, NT, CT>::OUT, tiles = ((UP ? p.F : p.H) + out - 1) / out, P = p.T * p.k, cap = max_blocks<16 * NT>(p.E, P);
    const size_t lds = STAGES * Rows<UP, NT, CT>::STAGE + routed_bytes<16 * NT>(p.E, P);
    const int grid = (int)std::min<int64_t>((int64_t)tiles * cap, (NT <= 2 ? 2 : 1) * h3host::cu_count());
    hipLaunchKernelGGL((moe_rows_kernel<UP, FP16, NT, CT>), dim3(grid), dim3(WAVES * 64), lds, st, p, tiles, grid / tiles, grid % tiles, cap);
    H3_CHECK_HIP(hipGetLastError());
    return H3FP8_OK;
}

int launch_combine(const MoeParams& p, hipStream_t st) {
    hipLaunchKernelGGL(moe_combine_kernel, dim3((unsigned)((p.H + 1023) / 1024), (unsigned)p.T), dim3(256), 0, st, p);
    H3_CHECK_HIP(hipGetLastError());
    return H3FP8_OK;
}

template <bool FP16, int D>
int launch_up(const MoeParams& p, hipStream_t st) {
    const int tiles = p.F / 16, P = p.T * p.k;
    const int grid = (int)std::min<int64_t>((int64_t)tiles * max_blocks<16>(p.E, P), 2 * h3host::cu_count());
    hipLaunchKernelGGL((moe_up_kernel<FP16, D>), dim3(grid), dim3(WAVES * 64), routed_bytes<16>(p.E, P), st, p, tiles, grid / tiles,
                       grid % tiles);
    H3_CHECK_HIP(hipGetLastError());
    return H3FP8_OK;
}

template <int NT, int D>
int launch_down(const MoeParams& p, hipStream_t st) {
    const size_t lds = sizeof(v4f) * DOWN_WAVES * NT * 64 + 6 * MAX_E + (size_t)std::min(p.E, p.T * p.k) * 16 * NT;
    hipLaunchKernelGGL((moe_down_kernel<NT, D>), dim3((unsigned)(p.H / 16)), dim3(DOWN_WAVES * 64), lds, st, p);
    H3_CHECK_HIP(hipGetLastError());
    return H3FP8_OK;
}

// Which kernels run (host only; for the workspace too).
bool by_rows(int64_t T, int64_t k, int64_t E) { return T > 16 || T * k > 4 * E; }

template <bool FP16, int NT>
int run_rows(const MoeParams& p, hipStream_t st) {
    int rc = launch_rows<true, FP16, NT, 1>(p, st);
    if (!rc) rc = launch_rows<false, false, NT, 2>(p, st);
    return rc ? rc : launch_combine(p, st);
}

template <bool FP16>
int run(const MoeParams& p, hipStream_t st) {
    if (by_rows(p.T, p.k, p.E)) {
        const int mean = (p.T * p.k + p.E - 1) / p.E;
        if (mean <= 8) return run_rows<FP16, 1>(p, st);
        if (mean <= 24) return run_rows<FP16, 2>(p, st);
        return run_rows<FP16, 4>(p, st);
    }
    const int rc = launch_up<FP16, 2>(p, st);
    return rc ? rc : launch_down<1, 2>(p, st);
}

constexpr int64_t kMaxSpan = 0x7fff0000LL;

}  // namespace

extern "C" int64_t h3fp8_moe_blocks_workspace(int64_t T, int64_t k, int64_t H, int64_t F, int64_t E) {
    return T < 0 || k < 0 || H < 0 || F < 0 ? 0 : T * k * 4 * (by_rows(T, k, E) ? F + H : F);
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
    H3_REQUIRE(H >= 16 && F >= 16 && H % 16 == 0 && F % 16 == 0 && H <= (1 << 24) && F <= (1 << 24),
               "%s: H=%lld and F=%lld must be positive multiples of 16", who, (long long)H, (long long)F);
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
    H3_REQUIRE(128 * ldx * 2 + 2 * H <= kMaxSpan && 64 * ld1 + H <= kMaxSpan && 64 * ld2 + F <= kMaxSpan && T * k * F * 4 <= kMaxSpan,
               "%s: a stride or size is too large", who);
    const int64_t hb = (H + 127) / 128, fb = (F + 127) / 128, f2 = (2 * F + 127) / 128;
    H3_REQUIRE((E * s1_e + f2 * s1_n) * 4 <= kMaxSpan / 2 && hb * s1_k * 4 <= kMaxSpan / 2 && hb * s2_n * 4 <= kMaxSpan / 2 && fb * s2_k * 4 <= kMaxSpan / 2,
               "%s: a scale stride is too large", who);
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
