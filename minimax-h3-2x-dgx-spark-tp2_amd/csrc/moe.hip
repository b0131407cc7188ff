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

// The slot-th expert that has pairs, and its pairs' places.
__device__ __forceinline__ bool find_expert(const MoeParams& p, int slot, int lane, int& e, int& r0, int& r1) {
    for (int e0 = 0; e0 < p.E; e0 += 64) {
        int lo = 0, hi = 0;
        if (e0 + lane < p.E) lo = offset_at(p, e0 + lane), hi = offset_at(p, e0 + lane + 1);
        const uint64_t has = __ballot(hi > lo);
        const int n = __popcll(has);
        if (slot < n) {
            const uint64_t at = __ballot(hi > lo && __popcll(has & ((1ull << lane) - 1)) == slot);
            const int f = __builtin_ctzll(at);
            e = e0 + f;
            r0 = __builtin_amdgcn_readlane(lo, f);
            r1 = __builtin_amdgcn_readlane(hi, f);
            return true;
        }
        slot -= n;
    }
    return false;
}

// ---- kernel 1 ---------------------------------------------------------------------------------------------------------

// NI: blocks of 16 gate rows; NT: blocks of 16 tokens; D: k-blocks in flight per wave.
template <bool FP16, int NI, int NT, int D>
__global__ void __launch_bounds__(WAVES * 64) moe_up_kernel(MoeParams p, int tiles) {
    constexpr int ITEMS = NI * NT * 64;                   // results of 4 channels x 1 token
    __shared__ v4f part[WAVES][2 * NI * NT][64];
    __shared__ int s_pair[16 * NT];
    __shared__ float s_weight[16 * NT];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int slot = (int)blockIdx.x / tiles, f0 = ((int)blockIdx.x - slot * tiles) * 16 * NI;
    int e, r0, r1;
    if (!find_expert(p, slot, lane, e, r0, r1)) return;
    const int c = lane & 15, g = lane >> 4;
    const int kb = (p.H + BK - 1) / BK, frows = min(16 * NI, p.F - f0);
    const uint32_t wbytes = (uint32_t)((frows - 1) * p.ld1 + p.H);
    const uint8_t* wg = p.w1 + e * p.w1_e + (int64_t)f0 * p.ld1;
    const __amdgpu_buffer_rsrc_t rg = make_rsrc(wg, wbytes), ru = make_rsrc(wg + (int64_t)p.F * p.ld1, wbytes);
    // in the vector memory's order of loads: a scalar load's wait is for all that are under way
    const __amdgpu_buffer_rsrc_t rs = make_rsrc(p.s1 + e * p.s1_e, 0x7fffffffu);
    const __amdgpu_buffer_rsrc_t rx = make_rsrc(p.x, (uint32_t)(((p.T - 1) * p.ldx + p.H) * 2));
    uint32_t vw[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) vw[i] = 16 * i + c < frows ? (uint32_t)((16 * i + c) * p.ld1) + 16u * g : OOB;
    for (int rt = r0; rt < r1; rt += 16 * NT) {
        uint32_t vx[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int r = rt + 16 * j + c;
            const int pair = r < r1 ? p.order[r] : -1;
            vx[j] = pair >= 0 && pair < p.T * p.k ? (uint32_t)(pair / p.k * p.ldx * 2) + 32u * g : OOB;
        }
        if (threadIdx.x < 16 * NT) {                      // the pair of each column and its weight (of every choice of this expert)
            const int r = rt + (int)threadIdx.x;
            int pair = r < r1 ? p.order[r] : -1;
            float w = 0.0f;
            if (pair < 0 || pair >= p.T * p.k) pair = -1;
            else
                for (int j = 0, q = pair / p.k * p.k; j < p.k; ++j) w += p.experts[q + j] == e ? p.weights[q + j] : 0.0f;
            s_pair[threadIdx.x] = pair;
            s_weight[threadIdx.x] = w;
        }
        v4u w[D][2 * NI][2], x[D][NT][2][2];
        float sc[D][2][NI];
        // always the same loads, past the last block of nothing, so that the count of those under way is known
        auto load = [&](int d, int b) {
            const int at = b < kb ? b * BK : 0;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const bool in = b * BK + 64 * s + 16 * g < p.H;
#pragma unroll
                for (int i = 0; i < NI; ++i) {
                    w[d][i][s] = load16<true>(rg, (in ? vw[i] : OOB) + 64 * s, at);
                    w[d][NI + i][s] = load16<true>(ru, (in ? vw[i] : OOB) + 64 * s, at);
                }
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int q = 0; q < 2; ++q) x[d][j][s][q] = load16<false>(rx, (in ? vx[j] : OOB) + 128 * s + 16 * q, 2 * at);
            }
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int n = f0 + 16 * i < p.F ? f0 + 16 * i : f0;
                const int bb = min(b, kb - 1);
                sc[d][0][i] = load4(rs, (uint32_t)(n / BK * p.s1_n + bb * p.s1_k) * 4u);
                sc[d][1][i] = load4(rs, (uint32_t)((p.F + n) / BK * p.s1_n + bb * p.s1_k) * 4u);
            }
            __builtin_amdgcn_sched_barrier(0);            // in this order: the waits count them
        };
        v4f acc[2 * NI][NT];
#pragma unroll
        for (int i = 0; i < 2 * NI; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int d = 0; d < D; ++d) load(d, wave + d * WAVES);
        for (int b0 = wave; b0 < kb; b0 += D * WAVES) {
#pragma unroll
            for (int d = 0; d < D; ++d) {
                const int b = b0 + d * WAVES;
                if (b < kb) {
                    v4f sum[2 * NI][NT];
#pragma unroll
                    for (int q = 0; q < 4; ++q)           // 32 of the block's k each
#pragma unroll
                        for (int i = 0; i < 2 * NI; ++i)
#pragma unroll
                            for (int j = 0; j < NT; ++j) {
                                const v4u& a = w[d][i][q >> 1];
                                if (q == 0) mfma<FP16, true>(sum[i][j], a[0], a[1], x[d][j][0][0]);
                                else mfma<FP16, false>(sum[i][j], a[2 * (q & 1)], a[2 * (q & 1) + 1], x[d][j][q >> 1][q & 1]);
                            }
                    sums_ready(sum);
#pragma unroll
                    for (int i = 0; i < 2 * NI; ++i)
#pragma unroll
                        for (int j = 0; j < NT; ++j)
#pragma unroll
                            for (int r = 0; r < 4; ++r) acc[i][j][r] = __builtin_fmaf(sum[i][j][r], sc[d][i / NI][i % NI], acc[i][j][r]);
                }
                load(d, b + D * WAVES);
            }
        }
#pragma unroll
        for (int i = 0; i < 2 * NI; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) part[wave][i * NT + j][lane] = acc[i][j];
        __syncthreads();
        for (int it = threadIdx.x; it < ITEMS; it += WAVES * 64) {
            const int l = it & 63, ij = it >> 6, col = ij % NT * 16 + (l & 15), f = f0 + ij / NT * 16 + 4 * (l >> 4);
            v4f gate = part[0][ij][l], up = part[0][NI * NT + ij][l];
#pragma unroll
            for (int v = 1; v < WAVES; ++v) {
                gate += part[v][ij][l];
                up += part[v][NI * NT + ij][l];
            }
            const int pair = s_pair[col];
            if (pair >= 0 && f < p.F) {
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float h = gate[r] / (1.0f + expf(-gate[r])) * up[r] * s_weight[col];
                    hi[r] = bf16_rne(h);
                    const float rest = h - bf16_to_f32(hi[r]);
                    lo[r] = (hi[r] & 0x7f80u) == 0x7f80u ? 0u : bf16_rne(rest);     // infinite or NaN: nothing is left
                }
                char* at = p.h + (int64_t)pair * p.F * 4 + f / 16 * 64 + f % 16 * 2;
                *reinterpret_cast<uint2*>(at) = uint2{hi[0] | (hi[1] << 16), hi[2] | (hi[3] << 16)};
                *reinterpret_cast<uint2*>(at + 32) = uint2{lo[0] | (lo[1] << 16), lo[2] | (lo[3] << 16)};
            }
        }
        __syncthreads();
    }
}

// ---- kernel 2 ---------------------------------------------------------------------------------------------------------

// CT: blocks of 16 channels; NT: blocks of 16 tokens (all of them); D: units in flight per wave.
template <int CT, int NT, int D>
__global__ void __launch_bounds__(WAVES * 64) moe_down_kernel(MoeParams p) {
    extern __shared__ __attribute__((aligned(16))) char down_lds[];
    v4f(*part)[CT * NT][64] = reinterpret_cast<v4f(*)[CT * NT][64]>(down_lds);                // [WAVES]
    int* s_expert = reinterpret_cast<int*>(down_lds + sizeof(v4f) * WAVES * CT * NT * 64);      // the experts that have pairs
    uint16_t* s_slot = reinterpret_cast<uint16_t*>(s_expert + MAX_E);                           // ... and where an expert is among them
    uint8_t* s_map = reinterpret_cast<uint8_t*>(s_slot + MAX_E);                                // [slots][16 NT]: 1 + the token's choice, or 0
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int n0 = (int)blockIdx.x * 16 * CT, rows = min(16 * CT, p.H - n0), P = p.T * p.k;
    const int cap = min(p.E, P);
    for (int i = threadIdx.x; i < cap * 16 * NT / 4; i += WAVES * 64) reinterpret_cast<uint32_t*>(s_map)[i] = 0;
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
    for (int q = threadIdx.x; q < P; q += WAVES * 64) {
        const int e = p.experts[q], t = q / p.k;
        if (e >= 0 && e < p.E && s_slot[e] != 0xffff) s_map[s_slot[e] * 16 * NT + t] = (uint8_t)(1 + q - t * p.k);
    }
    __syncthreads();
    const int fb = (p.F + BK - 1) / BK, units = active * fb;
    const __amdgpu_buffer_rsrc_t rh = make_rsrc(p.h, (uint32_t)P * (uint32_t)p.F * 4u);
    uint32_t vw[CT];
#pragma unroll
    for (int i = 0; i < CT; ++i) vw[i] = 16 * i + c < rows ? (uint32_t)((16 * i + c) * p.ld2) + 16u * g : OOB;
    constexpr bool AHEAD = NT <= 2;                       // the tokens' values are loaded with the weights, else when they are needed
    v4u w[D][CT][2], h[AHEAD ? D : 1][AHEAD ? NT : 1][2][4];          // h: 16 values, what they leave
    float sc[D];
    auto load_h = [&](int d, int j, int m, int b, int width) {
        const uint32_t vh = (uint32_t)((16 * j + c) * p.k + m - 1) * (uint32_t)p.F * 4u + 64u * g;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const uint32_t v = m && b * BK + 64 * s + 16 * g < width ? vh : OOB;
#pragma unroll
            for (int q = 0; q < 4; ++q) h[d][AHEAD ? j : 0][s][q] = load16<false>(rh, v + 256 * s + 16 * q, 4 * b * BK);
        }
    };
    // always the same loads, past the last unit of nothing, so that the count of those under way is known
    auto load = [&](int d, int u) {
        int width = u < units ? p.F : 0;
        asm("" : "+v"(width));                            // a value, so that it selects offsets and does not branch around loads
        const int v = min(u, units - 1), slot = v / fb, b = v - slot * fb, e = __builtin_amdgcn_readfirstlane(s_expert[slot]);
        const __amdgpu_buffer_rsrc_t rw = make_rsrc(p.w2 + e * p.w2_e + (int64_t)n0 * p.ld2, (uint32_t)((rows - 1) * p.ld2 + p.F));
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const bool in = b * BK + 64 * s + 16 * g < width;
#pragma unroll
            for (int i = 0; i < CT; ++i) w[d][i][s] = load16<true>(rw, (in ? vw[i] : OOB) + 64 * s, b * BK);
        }
        if constexpr (AHEAD) {
#pragma unroll
            for (int j = 0; j < NT; ++j) load_h(d, j, s_map[slot * 16 * NT + 16 * j + c], b, width);
        }
        sc[d] = load4(make_rsrc(p.s2 + e * p.s2_e, 0x7fffffffu), (uint32_t)(n0 / BK * p.s2_n + b * p.s2_k) * 4u);
        __builtin_amdgcn_sched_barrier(0);                // in this order: the waits count them
    };
    v4f acc[CT][NT];
#pragma unroll
    for (int i = 0; i < CT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
    if (units > 0) {
#pragma unroll
        for (int d = 0; d < D; ++d) load(d, wave + d * WAVES);
    }
    for (int u0 = wave; u0 < units; u0 += D * WAVES) {
#pragma unroll
        for (int d = 0; d < D; ++d) {
            const int u = u0 + d * WAVES;
            if (u < units) {
                const int slot = u / fb;
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    const int m = s_map[slot * 16 * NT + 16 * j + c];
                    if (__ballot(m != 0) == 0) continue;  // none of these tokens is the expert's
                    const int hd = AHEAD ? d : 0, hj = AHEAD ? j : 0;
                    if constexpr (!AHEAD) load_h(0, j, m, u - slot * fb, p.F);
                    v4f sum[CT][1];
#pragma unroll
                    for (int q = 0; q < 4; ++q)
#pragma unroll
                        for (int i = 0; i < CT; ++i) {
                            const uint32_t lo = w[d][i][q >> 1][2 * (q & 1)], hi = w[d][i][q >> 1][2 * (q & 1) + 1];
                            if (q == 0) mfma<false, true>(sum[i][0], lo, hi, h[hd][hj][0][0]);
                            else mfma<false, false>(sum[i][0], lo, hi, h[hd][hj][q >> 1][q & 1]);
                            mfma<false, false>(sum[i][0], lo, hi, h[hd][hj][q >> 1][2 + (q & 1)]);
                        }
                    sums_ready(sum);
                    if (m) {                              // an expert's NaN is not another token's
#pragma unroll
                        for (int i = 0; i < CT; ++i)
#pragma unroll
                            for (int r = 0; r < 4; ++r) acc[i][j][r] = __builtin_fmaf(sum[i][0][r], sc[d], acc[i][j][r]);
                    }
                }
            }
            load(d, u + D * WAVES);
        }
    }
#pragma unroll
    for (int i = 0; i < CT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) part[wave][i * NT + j][lane] = acc[i][j];
    __syncthreads();
    for (int it = threadIdx.x; it < CT * NT * 64; it += WAVES * 64) {
        const int l = it & 63, ij = it >> 6, t = ij % NT * 16 + (l & 15), n = n0 + ij / NT * 16 + 4 * (l >> 4);
        v4f v = part[0][ij][l];
#pragma unroll
        for (int q = 1; q < WAVES; ++q) v += part[q][ij][l];
        if (t >= p.T || n >= p.H) continue;
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
}

template <bool FP16, int NI, int NT, int D>
int launch_up(const MoeParams& p, hipStream_t st) {
    const int tiles = (p.F + 16 * NI - 1) / (16 * NI);
    const int64_t blocks = (int64_t)tiles * std::min(p.E, p.T * p.k);
    hipLaunchKernelGGL((moe_up_kernel<FP16, NI, NT, D>), dim3((unsigned)blocks), dim3(WAVES * 64), 0, st, p, tiles);
    H3_CHECK_HIP(hipGetLastError());
    return H3FP8_OK;
}

template <int CT, int NT, int D>
int launch_down(const MoeParams& p, hipStream_t st) {
    const size_t lds = sizeof(v4f) * WAVES * CT * NT * 64 + 6 * MAX_E + (size_t)std::min(p.E, p.T * p.k) * 16 * NT;
    hipLaunchKernelGGL((moe_down_kernel<CT, NT, D>), dim3((unsigned)((p.H + 16 * CT - 1) / (16 * CT))), dim3(WAVES * 64), lds, st, p);
    H3_CHECK_HIP(hipGetLastError());
    return H3FP8_OK;
}

template <bool FP16>
int run(const MoeParams& p, hipStream_t st) {
    const int rc = p.T <= 16 ? launch_up<FP16, 1, 1, 4>(p, st) : launch_up<FP16, 1, 2, 2>(p, st);
    if (rc) return rc;
    if (p.T <= 16) return launch_down<1, 1, 3>(p, st);
    if (p.T <= 32) return launch_down<1, 2, 2>(p, st);
    if (p.T <= 64) return launch_down<1, 4, 4>(p, st);
    return launch_down<1, 8, 4>(p, st);
}

constexpr int64_t kMaxSpan = 0x7fff0000LL;

}  // namespace

extern "C" int64_t h3fp8_moe_blocks_workspace(int64_t T, int64_t k, int64_t F) { return T < 0 || k < 0 || F < 0 ? 0 : T * k * F * 4; }

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
    H3_REQUIRE(f2 * s1_n * 4 <= kMaxSpan / 2 && hb * s1_k * 4 <= kMaxSpan / 2 && hb * s2_n * 4 <= kMaxSpan / 2 && fb * s2_k * 4 <= kMaxSpan / 2,
               "%s: a scale stride is too large", who);
    H3_REQUIRE(workspace_bytes >= h3fp8_moe_blocks_workspace(T, k, F), "%s: the workspace needs %lld bytes", who,
               (long long)h3fp8_moe_blocks_workspace(T, k, F));
    MoeParams p{};
    p.x = x; p.ldx = ldx;
    p.w1 = (const uint8_t*)w1; p.s1 = s1; p.w2 = (const uint8_t*)w2; p.s2 = s2;
    p.w1_e = w1_e; p.ld1 = ld1; p.w2_e = w2_e; p.ld2 = ld2;
    p.s1_e = s1_e; p.s1_n = s1_n; p.s1_k = s1_k; p.s2_e = s2_e; p.s2_n = s2_n; p.s2_k = s2_k;
    p.weights = weights; p.experts = experts; p.offsets = offsets; p.order = order;
    p.residual = residual; p.ldr = ldr; p.y = (uint16_t*)y; p.ldy = ldy; p.h = (char*)workspace;
    p.T = (int)T; p.E = (int)E; p.k = k; p.H = (int)H; p.F = (int)F; p.fp16 = dtype == H3FP8_DT_FP16;
    return p.fp16 ? run<true>(p, (hipStream_t)stream) : run<false>(p, (hipStream_t)stream);
}
