// The FP8 product of block-scaled operands, dense and grouped by expert (gfx950).
//
//   y[m, n] = round(sum_b sa[m, b] * sw[n / 128, b] * P_b[m, n] (+ bias[n])),  P_b = sum over the 128 k of block b of
//   a[m, k] w[n, k];  grouped: row m of expert e (offsets[e] <= m < offsets[e + 1]) takes w[e], sw[e].
//
// One MFMA makes one P_b: v_mfma 16x16x128 on e4m3 from a zero accumulator, the weight rows as its A operand and the
// tokens as its B operand, so that lane l holds channels 4 (l >> 4) + r (r = 0 .. 3) of token l & 15 and the block's scale
// sa * sw is one number per lane: acc = fma(P_b, sa * sw, acc) in fp32, b ascending.  Every form below computes every
// element by this sequence, so all give the same bits.
#include <algorithm>

#include "gemm_core.h"

namespace {

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

// Row tile t (TT rows each, no tile spans two experts, an expert without rows has none); false past the last one.  A wave
// looks at 64 experts at a time.
__device__ __forceinline__ bool locate_rows(const BlocksParams& p, int TT, int64_t t, int lane, TileRows& r) {
    if (!p.offsets) {
        r.e = 0;
        r.row0 = t * TT;
        r.rows = (int)min<int64_t>(TT, p.M - r.row0);
        return r.row0 < p.M;
    }
    for (int e0 = 0; e0 < p.E; e0 += 64) {
        const int e = e0 + lane;
        int64_t lo = 0, hi = 0;
        if (e < p.E) {
            lo = offset_at(p, e);
            hi = offset_at(p, e + 1);
        }
        const int n = hi > lo ? (int)((hi - lo + TT - 1) / TT) : 0;
        int sum = n;                                      // inclusive prefix over the lanes
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int v = __shfl_up(sum, o, 64);
            if (lane >= o) sum += v;
        }
        const uint64_t past = __ballot(sum > t);
        if (past) {
            const int f = __ffsll((unsigned long long)past) - 1;
            const int64_t first = __shfl(lo, f, 64), last = __shfl(hi, f, 64);
            r.e = e0 + f;
            r.row0 = first + (t - (__shfl(sum, f, 64) - __shfl(n, f, 64))) * TT;
            r.rows = (int)min<int64_t>(TT, last - r.row0);
            return true;
        }
        t -= __shfl(sum, 63, 64);
    }
    return false;
}

// One wave per 16 channels x 16 tokens, operands from global memory.  Two waves per SIMD at least leave a wave 256 registers,
// and the compiler then puts an MFMA's result into vector registers, where the fmas read it.
__global__ void __launch_bounds__(64, 2) gemm_blocks_kernel(BlocksParams p, int tiles_n) {
    const int lane = threadIdx.x;
    const int tn = (int)(blockIdx.x % (unsigned)tiles_n);
    TileRows r;
    if (!locate_rows(p, 16, blockIdx.x / (unsigned)tiles_n, lane, r)) return;
    const int c = lane & 15, g = lane >> 4;
    const int64_t m = r.row0 + c;
    const bool mok = c < r.rows;
    const uint8_t* wp = p.w + r.e * p.w_e + (int64_t)(tn * 16 + c) * p.ldw + 32 * g;
    const uint8_t* ap = p.a + (mok ? m : r.row0) * p.lda + 32 * g;
    const float* swp = p.sw + r.e * p.sw_e + (tn * 16 / 128) * p.sw_n;
    const float* sap = p.sa + (mok ? m : r.row0) * p.sa_m;
    v4f acc = {0.f, 0.f, 0.f, 0.f};
    for (int k = 0; k < p.K; k += BK) {
        v8i wf = {}, af = {};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (k + 32 * g + 16 * i >= p.K) continue;      // K % 16 == 0: a chunk is wholly in or out
            const int4 x = *reinterpret_cast<const int4*>(wp + k + 16 * i), y = *reinterpret_cast<const int4*>(ap + k + 16 * i);
            wf[4 * i] = x.x; wf[4 * i + 1] = x.y; wf[4 * i + 2] = x.z; wf[4 * i + 3] = x.w;
            af[4 * i] = y.x; af[4 * i + 1] = y.y; af[4 * i + 2] = y.z; af[4 * i + 3] = y.w;
        }
        const float s = sap[(k / BK) * p.sa_k] * swp[(k / BK) * p.sw_k];
        v4f b = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf, af, v4f{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
        asm volatile("s_nop 15\n\ts_nop 7" : "+v"(b));
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = __builtin_fmaf(b[i], s, acc[i]);
    }
    if (!mok) return;
    const int n = tn * 16 + 4 * g;
    uint32_t o[2];
    if (p.bias) {
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] += load_bias(p.bias, n + i, p.fp16);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
        o[i] = p.fp16 ? fp16_rne(acc[2 * i]) | (fp16_rne(acc[2 * i + 1]) << 16) : cvt_bf16x2(acc[2 * i], acc[2 * i + 1]);
    *reinterpret_cast<uint2*>(p.y + m * p.ldy + n) = make_uint2(o[0], o[1]);
}

constexpr int64_t kMaxSpan = 0x7fff0000LL;                // byte offsets within a tile are 32-bit

int check(const BlocksParams& p, const char* who, int out_dtype, int64_t N, int64_t K, int64_t E) {
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
int64_t row_tiles(const BlocksParams& p, int TT) {
    const int64_t full = (p.M + TT - 1) / TT;
    return p.offsets ? std::min<int64_t>(p.M, p.M / TT + p.E) : full;
}

int run(const BlocksParams& p, const char* who, hipStream_t st) {
    if (p.M == 0 || p.N == 0 || p.E == 0) return H3FP8_OK;
    const int tiles_n = p.N / 16;
    const int64_t tiles = row_tiles(p, 16) * tiles_n;
    H3_REQUIRE(tiles < ((int64_t)1 << 31), "%s: too many tiles for one launch", who);
    hipLaunchKernelGGL(gemm_blocks_kernel, dim3((unsigned)tiles), dim3(64), 0, st, p, tiles_n);
    H3_CHECK_HIP(hipGetLastError());
    return H3FP8_OK;
}

}  // namespace

extern "C" {

int h3fp8_gemm_blocks(const void* a, int64_t lda, const void* w, int64_t ldw, const float* sa, int64_t sa_m, int64_t sa_k,
                      const float* sw, int64_t sw_n, int64_t sw_k, const void* bias, void* y, int64_t ldy, int out_dtype,
                      int64_t M, int64_t N, int64_t K, void* stream) {
    BlocksParams p{};
    p.a = (const uint8_t*)a; p.w = (const uint8_t*)w; p.sa = sa; p.sw = sw; p.bias = bias; p.y = (uint16_t*)y;
    p.lda = lda; p.ldw = ldw; p.ldy = ldy;
    p.sa_m = sa_m; p.sa_k = sa_k; p.sw_n = sw_n; p.sw_k = sw_k;
    p.M = M; p.N = (int)N; p.K = (int)K; p.E = 1; p.fp16 = out_dtype == H3FP8_DT_FP16;
    const int rc = check(p, "h3fp8_gemm_blocks", out_dtype, N, K, 1);
    return rc ? rc : run(p, "h3fp8_gemm_blocks", (hipStream_t)stream);
}

int h3fp8_grouped_gemm_blocks(const void* a, int64_t lda, const void* w, int64_t w_e, int64_t ldw, const float* sa,
                              int64_t sa_m, int64_t sa_k, const float* sw, int64_t sw_e, int64_t sw_n, int64_t sw_k,
                              const void* offsets, int idx_bytes, void* y, int64_t ldy, int out_dtype, int64_t M, int64_t N,
                              int64_t K, int64_t E, void* stream) {
    BlocksParams p{};
    p.a = (const uint8_t*)a; p.w = (const uint8_t*)w; p.sa = sa; p.sw = sw; p.y = (uint16_t*)y;
    p.lda = lda; p.ldw = ldw; p.w_e = w_e; p.ldy = ldy;
    p.sa_m = sa_m; p.sa_k = sa_k; p.sw_e = sw_e; p.sw_n = sw_n; p.sw_k = sw_k;
    p.M = M; p.N = (int)N; p.K = (int)K; p.E = (int)E; p.fp16 = out_dtype == H3FP8_DT_FP16;
    p.offsets = offsets; p.idx_bytes = idx_bytes;
    const int rc = check(p, "h3fp8_grouped_gemm_blocks", out_dtype, N, K, E);
    if (rc) return rc;
    H3_REQUIRE(idx_bytes == 4 || idx_bytes == 8, "h3fp8_grouped_gemm_blocks: offsets must be int32 or int64");
    H3_REQUIRE(M == 0 || N == 0 || E == 0 || offsets, "h3fp8_grouped_gemm_blocks: null offsets");
    return run(p, "h3fp8_grouped_gemm_blocks", (hipStream_t)stream);
}

}  // extern "C"
