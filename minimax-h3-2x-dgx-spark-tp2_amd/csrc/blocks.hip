// The e4m3 quant with one scale per block of 128 columns, of a tensor or of the SwiGLU of a [gate | up] tensor.
//
//   amax = max |x| over the block (NaN propagating), scale = max(amax / 448, 1/(448*512)),
//   q    = e4m3fn_rne(clamp(x * (1 / scale), -448, 448))          (kernel 1's arithmetic, per block instead of per row)
//
// A block is 1 x 128 (activations: one scale per token and 128 columns) or 128 x 128 (weights).  A row or column count
// that is no multiple of 128 leaves the last block smaller.  The SwiGLU form quantises h = g / (1 + exp(-g)) * u held in
// fp32: the only rounding of h is its code's.
//
// HBM-bound: every input is read once and every code written once.  The 1 x 128 form: a wave holds four blocks of a row,
// 16 lanes x 8 elements each (16-byte loads, 8-byte code stores, the maximum over 16 lanes by row rotations), and takes
// ROWS / 4 tokens of the same four blocks, all loads in flight before the first use; the four waves of a workgroup share
// a tile of ROWS tokens, whose scales go through LDS so that the scale tensor, token-contiguous as the product reads it,
// is written in pieces of ROWS consecutive entries.  ROWS = 8: quant of 42848 x 7168 bf16 141 us (6.6 TB/s), SwiGLU of 18880 x
// 2 x 14336 204 us (6.7 TB/s), of 64 x 2 x 2048 2.8 us; with 32 rows 152, 220 and 5.3 (few and long waves), 16 rows 146
// and 217, 4 rows 151, 230 and 2.4 (a scale line in more pieces).  (All in one run, in turn; a kernel trace gives the 64 tokens 3.4-3.7
// us, and the large ones are 10 us slower on new inputs.)  From fp32 42848 x 7168 276 us (5.6 TB/s).  128 x 128: 21504 x 5376 bf16
// 54 us (6.4 TB/s), fp32 112 us (5.2 TB/s); with 256 threads of 8 loads each, behind branches, bf16 was 64.
#include "h3fp8_common.h"

namespace {

using namespace h3;

typedef unsigned int v2u __attribute__((ext_vector_type(2)));

constexpr uint32_t OUTSIDE = 0x80000000u;                 // an offset past every buffer range: loads zeros, stores nothing

template <int DT> struct Elem { static constexpr int BYTES = DT == H3FP8_DT_F32 ? 4 : 2; };

// 8 consecutive elements at byte offset `off` of a buffer, in fp32.
template <int DT>
__device__ __forceinline__ void unpack8(const v4u* t, float f[8]) {
    if (DT == H3FP8_DT_F32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = u2f(t[i >> 2][i & 3]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (DT == H3FP8_DT_BF16) {
                f[2 * i] = u2f(t[0][i] << 16);
                f[2 * i + 1] = u2f(t[0][i] & 0xffff0000u);
            } else {
                f[2 * i] = fp16_to_f32(t[0][i] & 0xffffu);
                f[2 * i + 1] = fp16_to_f32(t[0][i] >> 16);
            }
        }
    }
}

template <int DT>
__device__ __forceinline__ void load8(__amdgpu_buffer_rsrc_t r, uint32_t off, v4u* t) {
    t[0] = __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 2);                    // nt: read once
    if (DT == H3FP8_DT_F32) t[1] = __builtin_amdgcn_raw_buffer_load_b128(r, off + 16u, 0, 2);
}

// max(m, |a|, |b|), NaN propagating.
__device__ __forceinline__ float max3_abs(float m, float a, float b) {
    float r;
    asm("v_maximum3_f32 %0, %1, |%2|, |%3|" : "=v"(r) : "v"(m), "v"(a), "v"(b));
    return r;
}

__device__ __forceinline__ float absmax8(const float f[8], float m) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) m = max3_abs(m, f[i], f[i + 1]);
    return m;
}

// The maximum over each row of 16 lanes (rotations within the row); non-negative floats and NaN by their bits.
__device__ __forceinline__ uint32_t row16_max(uint32_t m) {
    uint32_t o;
    o = (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x128, 0xf, 0xf, true); m = m > o ? m : o;      // row_ror 8, 4, 2, 1
    o = (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x124, 0xf, 0xf, true); m = m > o ? m : o;
    o = (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x122, 0xf, 0xf, true); m = m > o ? m : o;
    o = (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x121, 0xf, 0xf, true); m = m > o ? m : o;
    return m;
}

// FINITE: the block's maximum is finite.  Then no clamp is needed: |x| <= amax, so |x (1 / scale)| <= 448 (1 + 3 2^-24), and
// everything below 464 rounds to 448.  Otherwise the compare / select clamp, which keeps NaN.
template <bool FINITE>
__device__ __forceinline__ v2u codes8(const float f[8], float inv) {
    float c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = FINITE ? f[i] * inv : quant_clamp(f[i], inv);
    return v2u{e4m3x4(c[0], c[1], c[2], c[3]), e4m3x4(c[4], c[5], c[6], c[7])};
}

// g / (1 + exp(-g)) * u.  exp(-g) = exp2(y + d): y = -g log2(e) rounded, d what the rounding and the constant's own lost, applied
// as a factor 1 + d ln 2 (with g held to +-200, where the exponential is 0 or inf, d stays finite).  exp2 and the reciprocal are
// the hardware's, 1 ulp each.  The reciprocal returns 0 where its result is subnormal, which is so from an exponential of 2^126
// on (g < -87.3), short of its overflow at 2^128 (g < -88.7): denominator and gate are held as quarters, exactly, so that it
// stays normal (one product more: 209 us against 206 at 18880 x 2 x 14336 timed in turn, the least of each 203.6 and 203.9).  From the overflow on the result is -0, as the division by inf gives.  Without d
// the exponential is |g| / 2 ulp off and four times as many codes at a rounding border fall on its other side.  With it 43 to
// 59 of 36 M codes differ from those of float64, with a library exponential and IEEE division 41 to 52; a Newton step on the rcp
// (36 to 63) costs 6 % of the time, the sum's lost bits on top (41 to 52) 24 %.
__device__ __forceinline__ float swiglu(float g, float u) {
    constexpr float L = -1.44269504088896340736f, LL = -1.92596299112661746887e-8f;       // -log2(e) = L + LL
    const float c = __builtin_amdgcn_fmed3f(g, -200.0f, 200.0f);
    const float y = c * L;
    const float d = __builtin_fmaf(c, LL, __builtin_fmaf(c, L, -y));
    const float e = __builtin_amdgcn_exp2f(y) * __builtin_fmaf(d, 0.69314718055994530942f / 4, 0.25f);        // exp(-g) / 4
    return 0.25f * g * __builtin_amdgcn_rcpf(0.25f + e) * u;
}

struct RowsArgs {
    const uint8_t* x;
    int64_t ldx;                // bytes
    int64_t M;
    int K;                      // columns of q (SWIGLU: F, x has 2F)
    uint8_t* q;
    int64_t ldq;
    float* scale;
    int64_t ss_m, ss_k;         // scale strides (elements) along tokens and column blocks
    int groups;                 // groups of four blocks per row
};

constexpr int ROWS = 8;         // tokens per workgroup

template <int DT, bool SWIGLU>
__global__ void __launch_bounds__(256) quant_blocks_kernel(RowsArgs a) {
    constexpr int EB = Elem<DT>::BYTES, PER = ROWS / 4, NV = DT == H3FP8_DT_F32 ? 2 : 1;
    __shared__ float tile[4][ROWS + 1];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int grp = (int)(blockIdx.x % (unsigned)a.groups);
    const int64_t m0 = (int64_t)(blockIdx.x / (unsigned)a.groups) * ROWS;
    const int64_t mw = m0 + wave * PER;                       // the wave's first token
    const int col = grp * 512 + lane * 8;                     // the lane's first column
    const bool in = col < a.K;
    v4u t[PER][NV], u[SWIGLU ? PER : 1][NV];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const bool live = mw + i < a.M;
        const __amdgpu_buffer_rsrc_t r = make_rsrc(a.x + (live ? mw + i : 0) * a.ldx,
                                                   live ? (uint32_t)a.K * EB * (SWIGLU ? 2 : 1) : 0u);
        load8<DT>(r, in ? (uint32_t)col * EB : OUTSIDE, t[i]);
        if (SWIGLU) load8<DT>(r, in ? (uint32_t)(col + a.K) * EB : OUTSIDE, u[i]);
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        float f[8];
        unpack8<DT>(t[i], f);
        if (SWIGLU) {
            float up[8];
            unpack8<DT>(u[i], up);
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = swiglu(f[e], up[e]);
        }
        const uint32_t mx = row16_max(f2u(absmax8(f, 0.0f)));
        const float s = row_scale(u2f(mx)), inv = inv_scale(s);
        const v2u c = __all(mx < 0x7f800000u) ? codes8<true>(f, inv) : codes8<false>(f, inv);
        const bool live = mw + i < a.M;
        const __amdgpu_buffer_rsrc_t qr = make_rsrc(a.q + (live ? mw + i : 0) * a.ldq, live ? (uint32_t)a.K : 0u);
        __builtin_amdgcn_raw_buffer_store_b64(c, qr, in ? (uint32_t)col : OUTSIDE, 0, 16);
        if ((lane & 15) == 0) tile[lane >> 4][wave * PER + i] = s;
    }
    __syncthreads();
    if (threadIdx.x < 4 * ROWS) {
        const int b = threadIdx.x / ROWS, i = threadIdx.x % ROWS;
        const int kb = grp * 4 + b;
        if (kb * 128 < a.K && m0 + i < a.M) a.scale[(m0 + i) * a.ss_m + kb * a.ss_k] = tile[b][i];
    }
}

// One 128 x 128 block per workgroup: thread t holds 8 columns 8 (t & 15) of rows (t >> 4) + 32 i.  Threads past the last row
// or column read the block's last ones again, which does not change its maximum, and store nothing.
constexpr int SQ_THREADS = 512;

template <int DT>
__global__ void __launch_bounds__(SQ_THREADS) quant_squares_kernel(RowsArgs a) {
    constexpr int EB = Elem<DT>::BYTES, NV = DT == H3FP8_DT_F32 ? 2 : 1, STEP = SQ_THREADS / 16, N = 128 / STEP;
    __shared__ uint32_t part[SQ_THREADS / 64];
    const int kb = (int)(blockIdx.x % (unsigned)a.groups);
    const int64_t mb = blockIdx.x / (unsigned)a.groups;
    const int col = kb * 128 + 8 * (threadIdx.x & 15), row = (int)threadIdx.x >> 4;
    const int rows = (int)min((int64_t)128, a.M - mb * 128);
    const bool in = col < a.K;
    const uint8_t* src = a.x + mb * 128 * a.ldx + (int64_t)(in ? col : a.K - 8) * EB;
    v4u t[N][NV];
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int v = 0; v < NV; ++v)
            t[i][v] = __builtin_nontemporal_load(reinterpret_cast<const v4u*>(src + min(row + STEP * i, rows - 1) * a.ldx + 16 * v));
    float fm = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        float f[8];
        unpack8<DT>(t[i], f);
        fm = absmax8(f, fm);
    }
    uint32_t mx = wave_max_u32(f2u(fm));
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = mx;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < SQ_THREADS / 64; ++i) mx = mx > part[i] ? mx : part[i];
    const float s = row_scale(u2f(mx));
    const float inv = inv_scale(s);
    uint8_t* dst = a.q + mb * 128 * a.ldq + col;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        float f[8];
        unpack8<DT>(t[i], f);
        const v2u c = mx < 0x7f800000u ? codes8<true>(f, inv) : codes8<false>(f, inv);     // one side for the workgroup
        if (in && row + STEP * i < rows) *reinterpret_cast<v2u*>(dst + (row + STEP * i) * a.ldq) = c;
    }
    if (threadIdx.x == 0) a.scale[mb * a.ss_m + kb * a.ss_k] = s;
}

int check_blocks(const char* who, const void* x, int64_t ldx, int dtype, int64_t M, int64_t K, int64_t width, const void* q,
                 int64_t ldq, const float* scale, int64_t ss_m, int64_t ss_k) {
    H3_REQUIRE(M >= 0 && K >= 0, "%s: negative size", who);
    H3_REQUIRE(K % 16 == 0 && K <= (1 << 28), "%s: the width %lld must be a multiple of 16 (at most 2^28)", who, (long long)K);
    if (M == 0 || K == 0) return H3FP8_OK;
    const int eb = dtype == H3FP8_DT_F32 ? 4 : 2, vec = 16 / eb;
    H3_REQUIRE(x && q && scale, "%s: null pointer", who);
    H3_REQUIRE(ldx >= width && ldx % vec == 0, "%s: the row stride of x must be >= %lld and a multiple of 16 bytes", who,
               (long long)width);
    H3_REQUIRE(ldq >= K && ldq % 8 == 0, "%s: the row stride of q must be >= %lld and a multiple of 8", who, (long long)K);
    H3_REQUIRE(((uintptr_t)x & 15) == 0 && ((uintptr_t)q & 7) == 0 && ((uintptr_t)scale & 3) == 0,
               "%s: x must be 16-byte, q 8-byte and the scales 4-byte aligned", who);
    H3_REQUIRE(ss_m >= 0 && ss_k >= 0, "%s: negative scale stride", who);
    return H3FP8_OK;
}

template <bool SWIGLU>
int launch_rows(RowsArgs a, int dtype, hipStream_t st) {
    a.groups = (a.K + 511) / 512;
    const int64_t blocks = (a.M + ROWS - 1) / ROWS * a.groups;
    H3_REQUIRE(blocks < ((int64_t)1 << 24), "quant_blocks: too many rows for one launch");       // 2^32 threads
    const dim3 grid((unsigned)blocks), block(256);
    if (dtype == H3FP8_DT_BF16) hipLaunchKernelGGL((quant_blocks_kernel<H3FP8_DT_BF16, SWIGLU>), grid, block, 0, st, a);
    else if (dtype == H3FP8_DT_FP16) hipLaunchKernelGGL((quant_blocks_kernel<H3FP8_DT_FP16, SWIGLU>), grid, block, 0, st, a);
    else if constexpr (!SWIGLU) hipLaunchKernelGGL((quant_blocks_kernel<H3FP8_DT_F32, SWIGLU>), grid, block, 0, st, a);
    H3_CHECK_HIP(hipGetLastError());
    return H3FP8_OK;
}

RowsArgs rows_args(const void* x, int64_t ldx, int dtype, int64_t M, int64_t K, void* q, int64_t ldq, float* scale,
                   int64_t ss_m, int64_t ss_k) {
    return RowsArgs{(const uint8_t*)x, ldx * (dtype == H3FP8_DT_F32 ? 4 : 2), M, (int)K, (uint8_t*)q, ldq, scale, ss_m, ss_k, 0};
}

bool dtype_ok(int dtype) { return dtype == H3FP8_DT_BF16 || dtype == H3FP8_DT_FP16 || dtype == H3FP8_DT_F32; }

}  // namespace

extern "C" {

int h3fp8_quant_blocks(const void* x, int64_t ldx, int dtype, int64_t M, int64_t K, int rows, void* q, int64_t ldq,
                       float* scale, int64_t ss_m, int64_t ss_k, void* stream) {
    H3_REQUIRE(dtype_ok(dtype), "h3fp8_quant_blocks: bad dtype %d", dtype);
    H3_REQUIRE(rows == 1 || rows == 128, "h3fp8_quant_blocks: blocks have 1 or 128 rows, got %d", rows);
    const int rc = check_blocks("h3fp8_quant_blocks", x, ldx, dtype, M, K, K, q, ldq, scale, ss_m, ss_k);
    if (rc || M == 0 || K == 0) return rc;
    RowsArgs a = rows_args(x, ldx, dtype, M, K, q, ldq, scale, ss_m, ss_k);
    hipStream_t st = (hipStream_t)stream;
    if (rows == 1) return launch_rows<false>(a, dtype, st);
    a.groups = (int)((K + 127) / 128);
    const int64_t blocks = (M + 127) / 128 * a.groups;
    H3_REQUIRE(blocks < ((int64_t)1 << 23), "h3fp8_quant_blocks: too many blocks for one launch");
    const dim3 grid((unsigned)blocks), block(SQ_THREADS);
    if (dtype == H3FP8_DT_BF16) hipLaunchKernelGGL((quant_squares_kernel<H3FP8_DT_BF16>), grid, block, 0, st, a);
    else if (dtype == H3FP8_DT_FP16) hipLaunchKernelGGL((quant_squares_kernel<H3FP8_DT_FP16>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((quant_squares_kernel<H3FP8_DT_F32>), grid, block, 0, st, a);
    H3_CHECK_HIP(hipGetLastError());
    return H3FP8_OK;
}

int h3fp8_silu_mul_quant_blocks(const void* x, int64_t ldx, int dtype, int64_t M, int64_t F, void* q, int64_t ldq,
                                float* scale, int64_t ss_m, int64_t ss_k, void* stream) {
    H3_REQUIRE(dtype == H3FP8_DT_BF16 || dtype == H3FP8_DT_FP16, "h3fp8_silu_mul_quant_blocks: bad dtype %d", dtype);
    const int rc = check_blocks("h3fp8_silu_mul_quant_blocks", x, ldx, dtype, M, F, 2 * F, q, ldq, scale, ss_m, ss_k);
    if (rc || M == 0 || F == 0) return rc;
    return launch_rows<true>(rows_args(x, ldx, dtype, M, F, q, ldq, scale, ss_m, ss_k), dtype, (hipStream_t)stream);
}

}  // extern "C"
